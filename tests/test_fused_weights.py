"""Fused projections (q/k/v, up/gate, siblings behind share_inputs) compute with the weights that their parts have, however those got there: loads that
assign, projections put in another's place, tensors that were set, moves.  What is fused on the CPU; what blocks then compute on the GPU."""
import copy

import pytest
import torch
import torch.nn as nn

from khaosz_amd import QuantLinear, fuse_shared_inputs, quantize_model, share_inputs
from khaosz_amd.block import MLP, DecoderBlock, GQA, PagedKV, _settled, rotary_table

DEV = "cuda:0"
DIM, HEADS, KV, FFN = 512, 8, 2, 704


def _projection(seed, out, width, dev, bias=False):
    g = torch.Generator().manual_seed(seed)
    q = QuantLinear(width, out, bias=bias, device=dev)
    q.qweight.copy_(torch.randint(-127, 128, (out, width), generator=g))
    q.w_scale.copy_(torch.rand(out, generator=g) * 0.001 + 0.0002)
    return q


def _gqa(dev, bias=False):
    m = GQA(64, 4, 2)
    for i, (n, out) in enumerate((("q_proj", 64), ("k_proj", 32), ("v_proj", 32))):
        setattr(m, n, _projection(i, out, 64, dev, bias))
    return m, "_qkv", ("q_proj", "k_proj", "v_proj")


def _mlp(dev, bias=False):
    m = MLP(64, 48)
    for i, n in enumerate(("up", "gate")):
        setattr(m, n, _projection(i, 48, 64, dev, bias))
    m.down = _projection(5, 64, 48, dev)
    return m, "_upgate", ("up", "gate")


def _new(p, seed=77):
    return _projection(seed, p.out_dim, p.in_dim, p.qweight.device, p.bias is not None)


CHANGES = {
    "nothing": lambda m, n: None,
    "load": lambda m, n: m.load_state_dict({k: torch.ones_like(v) for k, v in m.state_dict().items()}),
    "load that assigns": lambda m, n: m.load_state_dict({k: torch.ones_like(v) for k, v in m.state_dict().items()}, assign=True),
    "part's load that assigns": lambda m, n: getattr(m, n).load_state_dict(_new(getattr(m, n)).state_dict(), assign=True),
    "another part": lambda m, n: setattr(m, n, _new(getattr(m, n))),
    "codes set": lambda m, n: setattr(getattr(m, n), "qweight", _new(getattr(m, n)).qweight),
    "scales set": lambda m, n: setattr(getattr(m, n), "w_scale", _new(getattr(m, n)).w_scale),
    "a tensor's data": lambda m, n: setattr(getattr(m, n).qweight, "data", _new(getattr(m, n)).qweight),
    "moved": lambda m, n: m.double().float(),
}


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("make", [_gqa, _mlp])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("how", list(CHANGES))
def test_fused_rows_follow_their_parts(how, which, make, bias):
    m, name, parts = make("cpu", bias)
    assert m.fuse_projections()
    first = _settled(m, name, parts)
    assert first is getattr(m, name)
    CHANGES[how](m, parts[which])
    now = [getattr(m, p) for p in parts]
    want = [[t.clone() for t in (p.qweight, p.w_scale)] + [None if p.bias is None else p.bias.clone()] for p in now]
    whole = _settled(m, name, parts)
    assert whole is getattr(m, name) and whole is _settled(m, name, parts) and (whole is first) == (how in ("nothing", "load"))
    assert torch.equal(whole.qweight, torch.cat([w[0] for w in want])) and torch.equal(whole.w_scale, torch.cat([w[1] for w in want]))
    assert not bias or torch.equal(whole.bias, torch.cat([w[2] for w in want]))
    now[which].qweight.fill_(9)  # one copy
    lo = sum(p.out_dim for p in now[:which])
    assert whole.qweight[lo:lo + now[which].out_dim].eq(9).all()


@pytest.mark.parametrize("make", [_gqa, _mlp])
def test_rows_fused_in_inference_mode_can_be_written_outside(make):
    m, name, parts = make("cpu", True)
    m.fuse_projections()
    CHANGES["another part"](m, parts[1])
    with torch.inference_mode():
        whole = _settled(m, name, parts)
    m.load_state_dict({k: torch.ones_like(v) for k, v in m.state_dict().items()})
    assert whole.qweight.eq(1).all() and whole.bias.eq(1).all() and _settled(m, name, parts) is whole


class Doubled(nn.Module):
    def __init__(self, base):
        super().__init__()
        self.base = base

    def forward(self, x, **kw):
        return self.base(x, **kw) * 2


@pytest.mark.parametrize("make", [_gqa, _mlp])
def test_parts_of_another_kind_are_not_fused(make):
    for change in (lambda m, n: setattr(m, n, Doubled(getattr(m, n))), lambda m, n: setattr(m, n, nn.Linear(64, getattr(m, n).out_dim)),
                   lambda m, n: setattr(m, n, _projection(3, getattr(m, n).out_dim, 64, "cpu", True))):
        m, name, parts = make("cpu")
        m.fuse_projections()
        change(m, parts[1])
        assert _settled(m, name, parts) is None and getattr(m, name) is None


def _block(norms, seed=3, **kw):
    torch.manual_seed(seed)
    b = DecoderBlock(DIM, HEADS, FFN, KV, **kw)
    b.reset_parameters()
    b = b.to(DEV).to(torch.bfloat16)
    quantize_model(b)
    fuse_shared_inputs(b, norms=norms, decode_attention=True, residuals=True)
    return b


def _run(b, B, S, cached, norms):
    d = DIM // HEADS
    g = torch.Generator(device=DEV).manual_seed(B + S)
    cache = PagedKV(B * 4, 32, KV, d, DEV, torch.bfloat16)
    cache.k_layers.normal_(generator=g)
    cache.v_layers.normal_(generator=g)
    cache.bind(torch.arange(B * 4, device=DEV).view(B, 4), cached + S)
    fr = rotary_table(d, 256, device=DEV)[cached:cached + S].unsqueeze(0).expand(B, -1, -1)
    x = torch.randn(B, S, DIM, generator=g, device=DEV).to(torch.bfloat16)
    with torch.inference_mode():
        return b(x, fr, None, cache)


PARTS = [("attention", "q_proj"), ("attention", "v_proj"), ("mlp", "up"), ("mlp", "gate")]


@pytest.mark.gpu
@pytest.mark.parametrize("norms", [True, False])
@pytest.mark.parametrize("part", PARTS)
@pytest.mark.parametrize("how", [h for h in CHANGES if h not in ("load", "load that assigns", "moved")] + ["block's load that assigns", "block moved"])
def test_a_fused_block_computes_with_what_its_projections_have(how, part, norms):
    """Decode steps (one native call with ``norms``) and prompts: the bits of a new block of the same weights."""
    b = _block(norms)
    before = [_run(b, 3, 1, 40, norms), _run(b, 2, 20, 0, norms)]
    if how == "block's load that assigns":
        b.load_state_dict({k: v.clone() for k, v in _block(norms, 4).state_dict().items()}, assign=True)
    elif how == "block moved":
        b.cpu().to(DEV)
    else:
        CHANGES[how](getattr(b, part[0]), part[1])
    new = _block(norms, 5)
    new.load_state_dict(b.state_dict())
    got, again, want = ([_run(m, 3, 1, 40, norms), _run(m, 2, 20, 0, norms)] for m in (b, b, new))
    for g, a, w, f in zip(got, again, want, before):
        assert torch.equal(g, w) and torch.equal(a, w) and torch.equal(g, f) == (how in ("nothing", "block moved"))


@pytest.mark.gpu
@pytest.mark.parametrize("part", PARTS)
def test_a_block_with_a_projection_of_another_kind(part):
    """Twice the projection's output is that of twice its scales, to the bit."""
    b, twice = _block(False), _block(False)
    setattr(getattr(b, part[0]), part[1], Doubled(getattr(getattr(b, part[0]), part[1])))
    getattr(getattr(twice, part[0]), part[1]).w_scale.mul_(2.0)
    for B, S, cached in ((3, 1, 40), (2, 20, 0), (2, 5, 31)):
        assert torch.equal(_run(b, B, S, cached, False), _run(twice, B, S, cached, False))
    b, plain = _block(True), _run(_block(True), 3, 1, 40, True)
    setattr(getattr(b, part[0]), part[1], Doubled(getattr(getattr(b, part[0]), part[1])))  # (with norms fused: inside their quantisation's noise)
    twice = _block(True)
    getattr(getattr(twice, part[0]), part[1]).w_scale.mul_(2.0)
    got, want = _run(b, 3, 1, 40, True), _run(twice, 3, 1, 40, True)
    assert (got.double() - want.double()).norm() < 2e-2 * want.double().norm() and not torch.equal(got, plain)


@pytest.mark.gpu
def test_moved_rows_are_refused_under_capture():
    m, name, parts = _mlp(DEV)
    m.fuse_projections()
    x = torch.randn(3, 64, device=DEV)
    with torch.inference_mode():
        m(x)
        CHANGES["codes set"](m, "up")
        torch.cuda.synchronize()
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
def test_codes_need_the_fused_projection():
    for make, call in ((_gqa, lambda m, x, c: m(x.view(1, 3, 64), None, codes=c)), (_mlp, lambda m, x, c: m(x, codes=c))):
        m, name, parts = make(DEV)
        x = torch.randn(3, 64, device=DEV)
        with pytest.raises(ValueError, match="pre-quantised"):
            call(m, x, (torch.zeros(3, 64, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV)))


@pytest.mark.gpu
@pytest.mark.parametrize("how", [h for h in CHANGES if h not in ("load", "load that assigns", "moved")])
def test_siblings_behind_a_shared_input_follow(how):
    """The reference's modules call their projections themselves: each gives what it has, and nothing outlives the forward."""
    parent = nn.Module()
    for i, n in enumerate(("q_proj", "k_proj", "v_proj")):
        setattr(parent, n, _projection(i, 64, 64, DEV))
    assert share_inputs(parent, ("q_proj", "k_proj", "v_proj"))
    x = torch.randn(5, 64, device=DEV)
    with torch.inference_mode():
        [getattr(parent, n)(x) for n in ("q_proj", "k_proj", "v_proj")]
        CHANGES[how](parent, "k_proj")
        group = parent.q_proj._shared[0]
        for _ in range(2):
            for n in ("q_proj", "k_proj", "v_proj"):
                p = getattr(parent, n)
                alone = QuantLinear(64, 64, device=DEV)
                alone.load_state_dict(p.state_dict())
                assert torch.equal(p(x), alone(x)), n
            if how != "another part":
                assert group._x is None and group._y is None


@pytest.mark.gpu
def test_threads_that_share_a_block_whose_weights_move():
    """Every call, fused or projection by projection (the same bits without fused norms), has each projection's old weights or its new ones, whole."""
    import threading

    def replace(m, n, p):
        setattr(getattr(m, n[0]), n[1], p)
    b, allowed = _block(False), []
    for mask in range(16):  # any of the four replaced or not yet
        c = _block(False)
        for i, n in enumerate(PARTS):
            if mask >> i & 1:
                replace(c, n, _new(getattr(getattr(c, n[0]), n[1])))
        allowed.append(_run(c, 3, 1, 40, False))
    wrong, stop = [], threading.Event()

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            while not stop.is_set():
                y = _run(b, 3, 1, 40, False)
                if not any(torch.equal(y, a) for a in allowed):
                    wrong.append(min(float((y.double() - a.double()).norm() / a.double().norm()) for a in allowed))
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for n in PARTS:
        p = _new(getattr(getattr(b, n[0]), n[1]))
        torch.cuda.synchronize()
        replace(b, n, p)
        _run(b, 3, 1, 40, False)
    stop.set()
    for t in threads:
        t.join()
    assert not wrong, wrong
    assert torch.equal(_run(b, 3, 1, 40, False), allowed[15])
