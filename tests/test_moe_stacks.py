"""A fused layer of routed experts computes with the weights that its experts have, however those got there: loads into a child, experts and projections put in
another's place, tensors that were set.  The stacks themselves on the CPU; what the layer then computes on the GPU."""
import copy
import gc
import io
import weakref

import pytest
import torch
import torch.nn as nn

from khaosz_amd import QuantLinear, fuse_shared_inputs
from khaosz_amd.block import MLP, MoE

DEV = "cuda:0"
E, DIM, FFN = 4, 64, 48


def _quantized(seed, dev, bias=False):
    """An MLP of quantized layers with random codes."""
    g = torch.Generator().manual_seed(seed)
    m = MLP(DIM, FFN)
    for name, out, width in (("up", FFN, DIM), ("gate", FFN, DIM), ("down", DIM, FFN)):
        q = QuantLinear(width, out, bias=bias, device=dev)
        q.qweight.copy_(torch.randint(-127, 128, (out, width), generator=g))
        q.w_scale.copy_(torch.rand(out, generator=g) * 0.005 + 0.0005)
        setattr(m, name, q)
    return m


def _layer(dev, fused=True):
    torch.manual_seed(0)
    m = MoE(DIM, FFN, E, 2).to(dev)
    m.router.reset_parameters()
    for i in range(E):
        m.routed_experts[i] = _quantized(i, dev)
    if fused:
        fuse_shared_inputs(m, experts=True)
        assert m._experts is not None and m._stacked()
    return m


class Adapter(nn.Module):
    """A projection with a low-rank product beside it, of zeros and ones with one term to a sum: exact in any order."""

    def __init__(self, base):
        super().__init__()
        self.base, dev = base, base.qweight.device
        self.register_buffer("a", torch.eye(base.in_dim, device=dev)[:4])
        self.register_buffer("b", torch.eye(4, device=dev).repeat(base.out_dim // 4, 1))

    def forward(self, x, **kw):
        return self.base(x, **kw) + (x @ self.a.t()) @ self.b.t()


def _dict(dev, seed=90):
    return {k: v.clone() for k, v in _quantized(seed, dev).state_dict().items()}


def _set(m, i, name, buffer, how):
    p = getattr(m.routed_experts[i], name)
    t = getattr(_quantized(95, p.qweight.device), name)._buffers[buffer].clone()
    if how == "set":
        setattr(p, buffer, t)
    elif how == "entry":
        p._buffers[buffer] = t
    else:
        getattr(p, buffer).data = t


def _all(m, dev):
    return {k: v.clone() for k, v in {**m.state_dict(), **{f"routed_experts.{i}.{k}": v for i in range(E) for k, v in _dict(dev, 80 + i).items()}}.items()}


STACKED = {
    "nothing": lambda m, dev: None,
    "load": lambda m, dev: m.load_state_dict(_all(m, dev)),
    "load that assigns": lambda m, dev: m.load_state_dict(_all(m, dev), assign=True),
    "expert's load": lambda m, dev: m.routed_experts[1].load_state_dict(_dict(dev)),
    "expert's load that assigns": lambda m, dev: m.routed_experts[1].load_state_dict(_dict(dev), assign=True),
    "projection's load that assigns": lambda m, dev: m.routed_experts[3].down.load_state_dict(
        {k[5:]: v for k, v in _dict(dev).items() if k.startswith("down.")}, assign=True),
    "list's load that assigns": lambda m, dev: m.routed_experts.load_state_dict(
        {f"{i}.{k}": v for i in range(E) for k, v in _dict(dev, 60 + i).items()}, assign=True),
    "another expert": lambda m, dev: m.routed_experts.__setitem__(2, _quantized(91, dev)),
    "two experts exchanged": lambda m, dev: m.routed_experts.__init__([m.routed_experts[i] for i in (0, 2, 1, 3)]),
    "another projection": lambda m, dev: setattr(m.routed_experts[0], "gate", _quantized(92, dev).gate),
    "codes set": lambda m, dev: _set(m, 1, "up", "qweight", "set"),
    "scales set": lambda m, dev: _set(m, 0, "down", "w_scale", "set"),
    "a buffer's entry": lambda m, dev: _set(m, 3, "gate", "w_scale", "entry"),
    "a tensor's data": lambda m, dev: _set(m, 2, "gate", "qweight", "data"),
    "a float weight's load": lambda m, dev: m.routed_experts[1].up.load_float_weight(torch.randn(FFN, DIM, device=dev)),
    "projections fused afterwards": lambda m, dev: fuse_shared_inputs(m),
    "moved and back": lambda m, dev: m.cpu().to(dev),
    "an expert moved and back": lambda m, dev: m.routed_experts[0].double().float(),
}
APART = {
    "a bias": lambda m, dev: setattr(m.routed_experts[1], "down", QuantLinear(FFN, DIM, bias=True, device=dev)),
    "a bias set": lambda m, dev: setattr(m.routed_experts[1].up, "bias", nn.Parameter(torch.ones(FFN, device=dev), requires_grad=False)),
    "an adapter": lambda m, dev: setattr(m.routed_experts[2], "gate", Adapter(m.routed_experts[2].gate)),
    "an adapter behind": lambda m, dev: setattr(m.routed_experts[2], "down", Adapter(m.routed_experts[2].down)),
    "a float expert": lambda m, dev: m.routed_experts.__setitem__(0, MLP(DIM, FFN).to(dev).apply(lambda x: getattr(x, "reset_parameters", lambda: None)())),
    "a module of another kind": lambda m, dev: m.routed_experts.__setitem__(0, nn.Identity()),
    "an expert in two places": lambda m, dev: m.routed_experts.__setitem__(3, m.routed_experts[1]),
    "a fused projection's bias set": lambda m, dev: setattr(m.routed_experts[3].gate, "bias", nn.Parameter(torch.ones(FFN, device=dev), requires_grad=False)),
    "a wider expert": lambda m, dev: m.routed_experts.__setitem__(1, _wider(dev)),
}


def _wider(dev):
    m = MLP(DIM, 2 * FFN)
    for name, out, width in (("up", 2 * FFN, DIM), ("gate", 2 * FFN, DIM), ("down", DIM, 2 * FFN)):
        q = QuantLinear(width, out, device=dev)
        q.qweight.random_(-127, 128)
        q.w_scale.fill_(0.002)
        setattr(m, name, q)
    return m


def _current(m):
    return [[getattr(getattr(e, n), b) for e in m.routed_experts] for n in ("up", "gate", "down") for b in ("qweight", "w_scale")]


@pytest.mark.parametrize("projections", [False, True])
@pytest.mark.parametrize("how", list(STACKED))
def test_the_stacks_follow(how, projections):
    if how == "a float weight's load":
        pytest.skip("the quantizer is a kernel")
    m = _layer("cpu")
    if projections:
        m = _layer("cpu", False)
        fuse_shared_inputs(m)
        fuse_shared_inputs(m, experts=True)
    STACKED[how](m, "cpu")
    want = [[t.clone() for t in ts] for ts in _current(m)]
    assert m._stacked() and m._stacked()
    up, up_s, gate, gate_s, down, down_s = want
    stacks = m._experts
    for i in range(E):
        assert torch.equal(stacks[0][i], torch.cat([up[i], gate[i]])) and torch.equal(stacks[1][i], torch.cat([up_s[i], gate_s[i]]))
        assert torch.equal(stacks[2][i], down[i]) and torch.equal(stacks[3][i], down_s[i])
    assert all(torch.equal(a, b) for ts, us in zip(want, _current(m)) for a, b in zip(ts, us))
    # one copy: what is written through a child is in the stacks
    m.routed_experts[1].gate.qweight.fill_(7)
    assert m._stacked() and m._experts[0][1, FFN:].eq(7).all() and (m.routed_experts[1]._upgate is None or m.routed_experts[1]._upgate.qweight[FFN:].eq(7).all())


def test_projections_fused_behind_the_stacks_keep_no_second_copy():
    torch.manual_seed(0)
    m = MoE(DIM, FFN, E, 2)
    for i in range(E):
        m.routed_experts[i] = _quantized(i, "cpu")
    assert m.fuse_experts()
    stacks = m._experts
    codes = [[e.up.qweight.clone(), e.gate.qweight.clone(), e.up.w_scale.clone(), e.gate.w_scale.clone()] for e in m.routed_experts]
    assert fuse_shared_inputs(m) == E
    for i, (e, (u, g, us, gs)) in enumerate(zip(m.routed_experts, codes)):
        fused = e._upgate
        assert fused.qweight.data_ptr() == stacks[0][i].data_ptr() and fused.w_scale.data_ptr() == stacks[1][i].data_ptr()
        assert torch.equal(fused.qweight, torch.cat([u, g])) and torch.equal(fused.w_scale, torch.cat([us, gs]))
        assert torch.equal(e.up.qweight, u) and torch.equal(e.gate.qweight, g)
    assert m._stacked() and m._experts is stacks
    m.load_state_dict(_all(m, "cpu"))
    assert torch.equal(stacks[0][2, :FFN], _quantized(82, "cpu").up.qweight)  # through the child, without a forward in between
    # parts that lie where the kernels cannot read are copied
    flat, c = torch.randint(-127, 128, (2 * FFN * DIM + 4,), dtype=torch.int8), _quantized(3, "cpu")  # (its base is at a multiple of 64)
    c.up.qweight, c.gate.qweight = flat[4:].view(2, FFN, DIM)
    assert c.up.qweight.data_ptr() % 16 and QuantLinear.concat([c.up, c.gate]).qweight.data_ptr() % 16 == 0
    # parts elsewhere, in another order or with a gap are copied
    a, b = _quantized(1, "cpu"), _quantized(2, "cpu")
    whole = QuantLinear.concat([a.up, a.gate])
    for parts in ([a.gate, a.up], [a.up, b.up], [b.up, b.gate]):
        want = torch.cat([p.qweight for p in parts])
        again = QuantLinear.concat(parts)
        assert torch.equal(again.qweight, want) and again.qweight.data_ptr() != whole.qweight.data_ptr()


@pytest.mark.parametrize("how", list(APART))
def test_experts_that_no_longer_fit_take_the_layer_apart(how):
    m = _layer("cpu")
    APART[how](m, "cpu")
    assert not m._stacked() and m._experts is None and not m.fuse_experts()
    m.load_state_dict(m.state_dict())
    m.load_state_dict(m.state_dict(), assign=True)


def test_a_load_on_a_layer_with_a_float_expert():
    m = _layer("cpu")
    APART["a float expert"](m, "cpu")
    m.load_state_dict({k: v.clone() for k, v in m.state_dict().items()})  # (stacks are looked at behind every load)
    assert m._experts is None


@pytest.mark.parametrize("dim,ffn,fits", [(32768, 32752, True), (32768, 32768, False), (16, 1 << 24, True), (32, (1 << 24) + 16, False), (1 << 25, 16, False), (64, 40, False), (40, 64, False)])
def test_experts_of_sizes_that_the_operators_do_not_take_are_not_stacked(dim, ffn, fits):
    """What the operators would refuse at every call (2 F dim past 31 bits, rows past 2^24, not whole pieces of 16) stays a loop."""
    from khaosz_amd import _abi
    with torch.device("meta"):
        m = MoE(dim, ffn, 2, 1)
        for e in m.routed_experts:
            e.up, e.gate, e.down = QuantLinear(dim, ffn, device="meta"), QuantLinear(dim, ffn, device="meta"), QuantLinear(ffn, dim, device="meta")
    assert m.fuse_experts() == fits
    p = 1 << 20  # a fake, aligned pointer: what is taken ends at the workspace's size, before any launch
    rc = _abi.load().aq_experts_w8a8(p, 1, 1, dim, p, 2, p, p, p, 1, p, p, p, p, ffn, None, p, p, 0, None)
    assert (rc == -5) == fits and rc in (-2, -5, -6)


def test_limits_of_a_batch_are_the_librarys():
    """The largest batches that the layer hands over in one call are taken, and one more of each is not."""
    from khaosz_amd import _abi, ops
    p = 1 << 20

    def experts(T, k, dim, ffn):
        return _abi.load().aq_experts_w8a8(p, 1, T, dim, p, 2, p, p, p, k, p, p, p, p, ffn, None, p, p, 0, None)
    assert experts(ops.EXPERTS_MAX_TOKENS, 1, 16, 16) == -5 and experts(ops.EXPERTS_MAX_TOKENS + 1, 1, 16, 16) == -6
    assert experts(ops.EXPERTS_MAX_ROWS // 16, 16, 16, 16) == -5 and experts(ops.EXPERTS_MAX_ROWS // 16 + 1, 16, 16, 16) == -6
    for k, dim, ffn in ((2, 2048, 14336), (1, 4096, 16), (6, 2048, 1408)):
        most = ops.EXPERTS_MAX_VALUES // max(dim, k * ffn)
        assert experts(most, k, dim, ffn) == -5 and experts(most + 2, k, dim, ffn) == -6
    route = lambda T: _abi.load().aq_route_topk(p, 1, T, 8, 8, 2, 1, p, p, p, p, p, p, 0, None)
    assert route(ops.EXPERTS_MAX_TOKENS) == -5 and route(ops.EXPERTS_MAX_TOKENS + 1) == -6


def test_stacks_of_copies_are_their_own():
    m = _layer("cpu")
    twin = copy.deepcopy(m)
    assert twin._stacked() and m._stacked()
    twin.routed_experts[0].up.qweight.fill_(3)
    assert twin._experts[0][0, :FFN].eq(3).all() and not m._experts[0][0, :FFN].eq(3).all()
    buf = io.BytesIO()
    torch.save(m, buf)  # (after a look: what native code remembers is not the layer's state)
    buf.seek(0)
    again = torch.load(buf, weights_only=False)
    assert again._stacked() and torch.equal(again._experts[0], m._experts[0])
    again.routed_experts[2].down.qweight.fill_(5)
    assert again._stacked()[2][2].eq(5).all()


def test_a_moved_layer_keeps_nothing_of_the_stacks_it_had():
    m = _layer("cpu")
    assert m._stacked()
    old, slices = [weakref.ref(t) for t in m._experts], [weakref.ref(e.up.qweight) for e in m.routed_experts]
    m.double().float()
    gc.collect()
    assert all(r() is None for r in old + slices) and m._stacked()


def test_stacks_made_in_inference_mode_can_be_written_outside():
    m = _layer("cpu")
    with torch.inference_mode():
        STACKED["another expert"](m, "cpu")
        assert m._stacked()
    m.load_state_dict(_all(m, "cpu"))
    assert m._stacked()


@pytest.mark.gpu
@pytest.mark.parametrize("projections", [False, True])
@pytest.mark.parametrize("how", list(STACKED) + list(APART))
def test_the_layer_computes_with_what_its_experts_have(how, projections):
    """After each change: a fused layer's bits are those of a new layer of the same weights; one that is apart has the plain forward's."""
    m = _layer(DEV, not projections)
    if projections:
        assert fuse_shared_inputs(m, experts=True) == E and m._stacked()
    x = torch.randn(11, DIM, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    with torch.inference_mode():
        before = m(x)
    {**STACKED, **APART}[how](m, DEV)
    if how == "a module of another kind":
        m.routed_experts[0].up = m.routed_experts[0].gate = m.routed_experts[0].down = None
    with torch.inference_mode():
        got = m(x)
        assert torch.equal(got, m(x)) and torch.equal(got, before) == (how in ("nothing", "projections fused afterwards", "moved and back", "an expert moved and back"))
        if how in STACKED:
            assert m._experts is not None
            new = _layer(DEV, False)
            new.load_state_dict(m.state_dict())
            assert new.fuse_experts() and torch.equal(got, new(x))
        else:
            assert m._experts is None
            probs = torch.softmax(m.router(x).float(), -1)
            w, idx = torch.topk(probs, 2, dim=-1)
            w = (w / w.sum(-1, keepdim=True)).double()
            want, size = (torch.zeros(11, DIM, device=DEV, dtype=torch.float64) for _ in range(2))
            for e, expert in enumerate(m.routed_experts):
                one = x if type(expert) is not MLP else expert.down(expert.up(x) * torch.nn.functional.silu(expert.gate(x)))
                term = one.double() * (w * (idx == e)).sum(-1, keepdim=True)
                want, size = want + term, size + term.abs()
            # the weight's softmax, sum and quotient are the same numbers; then its product and one addition a choice.  A float expert's products are
            # sums of 64 and 48 terms in another order, of numbers below 30
            tol = 8 * 2.0 ** -24 * size if how != "a float expert" else 256 * 2.0 ** -24 * (size + 30.0)
            assert ((got - want).abs() <= tol).all()


@pytest.mark.gpu
def test_a_router_of_fewer_experts():
    """An expert that the router does not know is never chosen, fused or not."""
    m = _layer(DEV)
    x = torch.randn(11, DIM, device=DEV)
    with torch.inference_mode():
        before = m(x)
        m.routed_experts.append(_quantized(70, DEV))
        after = m(x)
        assert (after.double() - before.double()).norm() / before.double().norm() < 3e-2  # (the loop's roundings of h and sums)


@pytest.mark.gpu
def test_a_call_with_weights_of_its_own():
    """torch.func.functional_call puts tensors in the place of buffers for one call."""
    m = _layer(DEV)
    x = torch.randn(11, DIM, device=DEV)
    with torch.inference_mode():
        before, other = m(x), _all(m, DEV)
        new = _layer(DEV, False)
        new.load_state_dict(other)
        assert new.fuse_experts()
        assert torch.equal(torch.func.functional_call(m, other, (x,)), new(x))
        assert torch.equal(m(x), before)


@pytest.mark.gpu
def test_moved_weights_are_refused_under_capture():
    m = _layer(DEV)
    x = torch.randn(3, DIM, device=DEV)
    with torch.inference_mode():
        m(x)
        torch.cuda.synchronize()
        STACKED["codes set"](m, DEV)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="captured"):
            with torch.cuda.graph(graph):
                m(x)
        want = m(x).clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(m(x), want)


@pytest.mark.gpu
def test_a_compiled_layer_and_threads_that_share_one():
    import threading
    m = _layer(DEV)
    x = torch.randn(11, DIM, device=DEV)
    with torch.inference_mode():
        want = m(x)
        torch._dynamo.reset()
        compiled = torch.compile(m, backend="eager")
        assert torch.equal(compiled(x), want)
        STACKED["codes set"](m, DEV)
        after = compiled(x)
        assert torch.equal(after, m(x)) and not torch.equal(after, want)
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()), torch.inference_mode():
            for i in range(50):
                if i % 10 == 0:
                    m.routed_experts[1].train(i % 20 == 0)  # (looked through again)
                if not torch.equal(m(x), after):
                    wrong.append(i)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
def test_a_layer_on_one_stream_behind_a_change_seen_on_another():
    """The call that stacks the weights again does so on its stream; a call on another stream, with nothing between the two, reads whole stacks."""
    m, other = _layer(DEV), _layer(DEV, False)
    x = torch.randn(11, DIM, device=DEV)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.inference_mode():
        for i in range(5):
            for e in range(E):
                m.routed_experts[e].load_state_dict(_dict(DEV, 200 + 10 * i + e), assign=True)
            other.load_state_dict({k: v.clone() for k, v in m.state_dict().items()})
            other._experts = None
            assert other.fuse_experts()
            want = other(x)
            torch.cuda.synchronize()
            with torch.cuda.stream(a):
                big = torch.randn(4096, 4096, device=DEV)
                for _ in range(8):
                    big = big @ big  # the stream is busy
                one = m(x)
            with torch.cuda.stream(b):
                two = m(x)
            torch.cuda.synchronize()
            assert torch.equal(one, want) and torch.equal(two, want)
