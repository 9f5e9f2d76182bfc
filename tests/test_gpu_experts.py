"""Routed experts (DeepSeekMoE, mlp.py:31-93) without the host in between: routing, grouped W8A8 products, the weighted sum, and the whole
layer, against plain implementations: choices, rows and products bit for bit, weights, SwiGLU and sums within bounds taken from their roundings."""
import math
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from khaosz_amd import ops  # noqa: E402

DEV = "cuda:0"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # a rounding is off by at most half a step


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


# ---- routing --------------------------------------------------------------------------------------------------------

def _route(x, k, renormalize):
    """Plain: (weights in 64 bits, experts, rows, tokens, offsets) of logits on the CPU."""
    x = x.double().cpu().numpy()
    T, E = x.shape
    with np.errstate(invalid="ignore"):
        able = x > -np.inf  # (not NaN either)
    key = np.where(able, x, -np.inf)
    experts = np.argsort(-key, axis=1, kind="stable")[:, :k]
    experts = np.where(np.take_along_axis(able, experts, 1), experts, -1).astype(np.int64)
    weights = np.zeros((T, k))
    for t in range(T):
        live = [e for e in experts[t] if e >= 0]
        if not live:
            continue
        most = x[t, live[0]]
        p = np.array([1.0 if able[t, e] and x[t, e] == most else math.exp(x[t, e] - most) if able[t, e] else 0.0 for e in range(E)])
        total = p[live].sum() if renormalize else p.sum()
        weights[t, :len(live)] = p[live] / total
    rows = np.full((T, k), -1, np.int64)
    tokens = np.full((T * k,), -1, np.int64)
    offsets, r = [0], 0
    for e in range(E):
        for t, j in zip(*np.nonzero(experts == e)):
            rows[t, j], tokens[r], r = r, t, r + 1
        offsets.append(r)
    return weights, experts, rows, tokens, np.array(offsets)


def _check_route(x, k, renormalize, got):
    weights, experts, rows, tokens, offsets = _route(x, k, renormalize)
    for name, want in (("experts", experts), ("rows", rows), ("tokens", tokens), ("offsets", offsets)):
        g = getattr(got, name)
        assert g.dtype == torch.int32 and tuple(g.shape) == want.shape, name
        assert np.array_equal(g.cpu().numpy(), want), name
    # a weight: x - max rounded (|x - max| half steps of the exponential), the exponential (one step), a sum of up to 512 / 16 + 4
    # rounded additions of such numbers, and a quotient
    xs = x.double().cpu().numpy()
    real = xs[np.isfinite(xs)]
    spread = float(real.max() - real.min()) if real.size else 0.0
    tol = (2 * spread + 2 + 2 + 36 + 1) * HALF[torch.float32]
    assert got.weights.dtype == torch.float32
    assert np.all(np.abs(got.weights.double().cpu().numpy() - weights) <= tol * weights + 1e-40)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 6), (2, 3, 3), (7, 8, 2), (63, 60, 4), (64, 65, 5), (65, 16, 16), (256, 17, 3), (257, 64, 6),
                                   (333, 60, 4), (511, 200, 8), (700, 256, 8), (130, 128, 7), (1500, 512, 16), (4100, 9, 2), (3000, 512, 9), (3000, 401, 5), (2100, 64, 6)])
def test_route(T, E, k, dtype):
    _say("route", T, E, k, dtype)
    g = torch.Generator().manual_seed(T * 1000 + E)
    x = torch.randn(T, E, generator=g) * 2.0
    for renormalize in (True, False):
        d = x.to(dtype).to(DEV)
        _check_route(d, k, renormalize, ops.route_topk(d, k, renormalize))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [9, 300])
def test_route_ties_masks_infinities_and_nan(T, dtype):
    _say("route edges", T, dtype)
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-2, 3, (T, 24), generator=g).float()  # ties everywhere, zeros of both signs
    x[::3] *= -1.0
    x[1] = -math.inf                                        # a padded token
    x[2, 3:] = -math.inf                                    # fewer than k experts
    x[3, :] = torch.finfo(dtype).min                        # the type's lowest value is a number
    x[4, 5] = math.nan
    x[5, :] = math.nan
    x[6, 7] = math.inf
    x[7, 3:9] = math.inf
    x[8, ::2] = torch.finfo(dtype).min
    d = x.to(dtype).to(DEV)
    for renormalize in (True, False):
        got = ops.route_topk(d, 6, renormalize)
        _check_route(d, 6, renormalize, got)
    assert got.experts[1].eq(-1).all() and got.weights[1].eq(0).all() and got.experts[5].eq(-1).all()
    none = ops.route_topk(torch.full((T, 24), -math.inf, device=DEV, dtype=dtype), 6)
    assert none.offsets.eq(0).all() and none.tokens.eq(-1).all() and none.rows.eq(-1).all()


def test_route_of_everything_to_one_expert_of_no_token_and_of_strided_logits():
    x = torch.zeros(1000, 40, device=DEV)
    x[:, 13] = 5.0
    _check_route(x, 1, True, ops.route_topk(x, 1))
    empty = ops.route_topk(torch.empty(0, 40, device=DEV), 3)
    assert empty.offsets.eq(0).all() and empty.rows.shape == (0, 3) and empty.tokens.numel() == 0
    wide = torch.randn(100, 96, device=DEV)
    for view in (wide[:, 5:45], wide[::2, :40], wide.t()[:40, :].t()):
        _check_route(view, 4, True, ops.route_topk(view, 4))
        got, want = ops.route_topk(view, 4), ops.route_topk(view.contiguous(), 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_route_of_a_large_batch_against_torch():
    """Chunks of several passes: 40000 tokens are 625 times 64."""
    g = torch.Generator(device=DEV).manual_seed(3)
    T, E, k = 40000, 48, 3
    x = torch.randn(T, E, generator=g, device=DEV)
    got = ops.route_topk(x, k)
    top, at = torch.sort(x, dim=1, descending=True, stable=True)
    assert torch.equal(got.experts, at[:, :k].int())
    group, order = torch.sort(at[:, :k].reshape(-1), stable=True)
    assert torch.equal(got.tokens, (order // k).int())
    assert torch.equal(got.rows.flatten().long()[order], torch.arange(T * k, device=DEV))
    assert torch.equal(got.offsets, torch.searchsorted(group, torch.arange(E + 1, device=DEV)).int())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,E,k", [(32768, 64, 3), (32769, 64, 3), (40000, 64, 4), (70000, 255, 7), (33000, 512, 2)])
def test_route_of_chunks_of_several_passes_whose_counts_are_summed_apart(T, E, k, dtype):
    """More than 32768 tokens are two passes or more to a chunk; more than 16384 chunks times experts, and the counts have a launch of their own."""
    _say("large route", T, E, k, dtype)
    g = torch.Generator(device=DEV).manual_seed(T + E)
    x = torch.randn(T, E, generator=g, device=DEV).to(dtype)
    x[:, E // 3] += 1.0  # one that is asked often
    x[torch.rand(T, generator=g, device=DEV) < 0.1] = -math.inf
    got = ops.route_topk(x, k)
    top, at = torch.sort(x.float(), dim=1, descending=True, stable=True)
    experts = torch.where(top[:, :k] > -math.inf, at[:, :k], -1)
    assert torch.equal(got.experts, experts.int())
    group, order = torch.sort(torch.where(experts < 0, E, experts).reshape(-1), stable=True)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(T * k, device=DEV)
    assert torch.equal(got.rows, torch.where(experts < 0, -1, rows.view(T, k)).int())
    assert torch.equal(got.tokens, torch.where(group < E, order // k, -1).int())
    assert torch.equal(got.offsets, torch.searchsorted(group, torch.arange(E + 1, device=DEV)).int())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E", [64, 128, 256, 512])
@pytest.mark.parametrize("T", [1, 2, 100, 300, 2500])
def test_route_of_whole_vectors_in_strided_and_shifted_views(T, E, dtype):
    """Logits whose rows are whole vectors of a lane, at every stride and base: read as vectors where both are aligned."""
    g = torch.Generator(device=DEV).manual_seed(T + E)
    buf = torch.randn((T + 2) * (E + 24), generator=g, device=DEV).to(dtype)
    k = 6
    for stride in (E, E + 4, E + 8, E + 1, E + 2, E + 7):
        for base in (0, 1, 2, 4, 8, 5):
            view = buf[base:].as_strided((T, E), (stride, 1))
            got, want = ops.route_topk(view, k), ops.route_topk(view.clone(memory_format=torch.contiguous_format), k)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (stride, base)
    _check_route(view[:300], k, True, ops.route_topk(view[:300], k))


# ---- grouped products -----------------------------------------------------------------------------------------------

def _operands(counts, K, N, seed, tokens=None, dtype=torch.bfloat16, bias=None, loud=False):
    """Codes, scales and groups for experts with the given numbers of rows; tokens: rows come from that many tokens, in any order."""
    g = torch.Generator().manual_seed(seed)
    E, R = len(counts), sum(counts)
    rows = R if tokens is None else tokens
    xq = torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8) if not loud else torch.full((rows, K), 127, dtype=torch.int8)
    wq = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8) if not loud else torch.full((E, N, K), -127, dtype=torch.int8)
    sx = torch.rand(rows, generator=g) * 0.02 + 0.001
    sw = torch.rand(E, N, generator=g) * 0.02 + 0.001
    b = None if bias is None else (torch.randn(E, N, generator=g) * 2).to(bias)
    tok = None if tokens is None else torch.randint(0, rows, (R,), generator=g, dtype=torch.int32)
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    return xq, sx, wq, sw, offsets, tok, b


def _projections(xq, sx, wq, sw, offsets, tok, b):
    """fp32 [R, N], operation by operation; whole-number sums exactly."""
    R = int(offsets[-1])
    y = torch.empty(R, wq.shape[1])
    for e in range(wq.shape[0]):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        if lo == hi:
            continue
        at = torch.arange(lo, hi) if tok is None else tok[lo:hi].long()
        acc = xq[at].double() @ wq[e].double().t()  # below 2^53: exact
        v = (acc.float() * sx[at][:, None]) * sw[e]
        y[lo:hi] = v if b is None else v + b[e].float()
    return y


def _on(*ts):
    return tuple(None if t is None else t.to(DEV) for t in ts)


@pytest.fixture(params=["by size", "rows of 16", "walked 256", "walked 128", "walked 64"])
def kernel(request):
    """The kernel that the library takes for the sizes, and each of them whatever the sizes."""
    from khaosz_amd import _abi
    if request.param == "by size":
        yield request.param
        return
    with _abi.lab_library() as lab:
        assert lab.aq_lab_set_grouped_kernel({"rows of 16": 1, "walked 256": 2, "walked 128": 3, "walked 64": 4}[request.param]) == 0
        yield request.param


GROUPS = {
    "one row": [1],
    "one expert": [37],
    "all empty but one": [0, 0, 5, 0],
    "empty ends": [0, 16, 17, 0, 1, 0],
    "tile edges": [15, 16, 17, 31, 32, 33, 63, 64, 65],
    "a large one": [3, 300, 0, 129, 128, 127, 1],
    "65 experts": [i % 4 for i in range(65)],
    "200 experts": [(7 * i) % 5 if i % 3 else 0 for i in range(200)],
    "512 experts": [1 if i % 7 == 0 else 0 for i in range(512)],
}


@pytest.mark.parametrize("K,N", [(16, 1), (48, 33), (128, 64), (208, 100), (1408, 31), (512, 200), (1040, 257)])
@pytest.mark.parametrize("groups", list(GROUPS))
def test_grouped_linear_bits(kernel, groups, K, N):
    _say("grouped linear", kernel, groups, K, N)
    counts = GROUPS[groups]
    for tokens, dtype, bias in ((None, torch.bfloat16, None), (50, torch.float32, torch.float32), (3, torch.bfloat16, torch.bfloat16)):
        xq, sx, wq, sw, offsets, tok, b = _operands(counts, K, N, K + N, tokens, bias=bias)
        want = _projections(xq, sx, wq, sw, offsets, tok, b).to(dtype)
        d = _on(xq, sx, wq, sw, offsets, tok, b)
        got = ops.linear_w8a8_grouped(*d[:5], d[5], bias=d[6], out_dtype=dtype)
        assert got.shape == want.shape and got.dtype == dtype
        assert torch.equal(got.cpu(), want), (tokens, dtype)


def test_more_rows_than_one_grid_axis_has_tiles():
    """1.1 million rows are more than 65535 tiles of 16, of narrow layers the few-rows kernel is the quickest for."""
    R = 1_100_000
    xq, sx, wq, sw, offsets, tok, _ = _operands([R], 16, 1, 77)
    y = ops.linear_w8a8_grouped(*_on(xq, sx, wq, sw, offsets), out_dtype=torch.float32)
    want = (xq.float() @ wq[0].float().t()) * sx[:, None] * sw[0]
    assert torch.equal(y.cpu(), want)
    _, _, uq, us, dq, ds = _layer(2, 16, 16, 78)
    x = torch.randn(R // 2, 16, device=DEV).bfloat16()
    r = ops.route_topk(torch.randn(R // 2, 2, device=DEV), 2)
    got = ops.experts_w8a8(x, r, uq, us, dq, ds)
    assert torch.equal(got, _composed(x, r, uq, us, dq, ds, None))


@pytest.mark.parametrize("K,N", [(2048, 272), (4096, 96), (528, 514)])
def test_grouped_linear_bits_many_rows(kernel, K, N):
    """Enough rows an expert for whole tiles of any kernel."""
    _say("grouped linear, many rows", kernel, K, N)
    counts = [700, 0, 513, 260, 1, 256, 255, 1000]
    for tokens, dtype in ((None, torch.bfloat16), (777, torch.float32)):
        xq, sx, wq, sw, offsets, tok, b = _operands(counts, K, N, K, tokens, bias=torch.float32)
        want = _projections(xq, sx, wq, sw, offsets, tok, b).to(dtype)
        d = _on(xq, sx, wq, sw, offsets, tok, b)
        assert torch.equal(ops.linear_w8a8_grouped(*d[:5], d[5], bias=d[6], out_dtype=dtype).cpu(), want)


def test_grouped_linear_is_the_single_linear():
    counts = [5, 40, 0, 300]
    xq, sx, wq, sw, offsets, tok, b = _on(*_operands(counts, 512, 192, 3, 100, bias=torch.bfloat16))
    got = ops.linear_w8a8_grouped(xq, sx, wq, sw, offsets, tok, bias=b)
    for e in range(4):
        lo, hi = int(offsets[e]), int(offsets[e + 1])
        at = tok[lo:hi].long()
        if hi > lo:
            assert torch.equal(got[lo:hi], ops.linear_w8a8(xq[at], sx[at], wq[e], sw[e], b[e]))


def test_grouped_linear_largest_sums(kernel):
    """Codes of one sign throughout: sums of 4096 * 127^2, past what fp32 holds exactly."""
    xq, sx, wq, sw, offsets, tok, b = _operands([3, 20, 140], 4096, 40, 1, loud=True)
    want = _projections(xq, sx, wq, sw, offsets, tok, b).to(torch.float32)
    assert torch.equal(ops.linear_w8a8_grouped(*_on(xq, sx, wq, sw, offsets), out_dtype=torch.float32).cpu(), want)


@pytest.mark.parametrize("counts", [[2, 1, 0], [30, 200, 0]])
def test_grouped_rows_behind_the_last_are_left_and_odd_tokens_are_zeros(kernel, counts):
    from khaosz_amd import _abi
    R, live, K, N = sum(counts) + 37, sum(counts), 64, 48
    xq, sx, wq, sw, offsets, _, _ = _operands(counts, K, N, 9, 50)
    tok = torch.randint(0, 50, (R,), dtype=torch.int32)
    tok[1], tok[2] = -1, 50
    d = _on(xq, sx, wq, sw, offsets, tok)
    for swiglu in (False, True):
        out = torch.full((R, N), 7.0, device=DEV, dtype=torch.bfloat16)
        if swiglu:
            out = torch.full((R, 16), 7.0, device=DEV, dtype=torch.bfloat16)
            d2 = (d[0], d[1], d[2][:, :32].contiguous(), d[3][:, :32].contiguous(), d[4], d[5])
            rc = _abi.load().aq_swiglu_w8a8_grouped(d2[0].data_ptr(), d2[1].data_ptr(), 50, d2[2].data_ptr(), d2[3].data_ptr(), d2[4].data_ptr(), 3,
                                                    d2[5].data_ptr(), R, out.data_ptr(), _abi.AQ_BF16, 16, K, torch.cuda.current_stream().cuda_stream)
        else:
            rc = _abi.load().aq_linear_w8a8_grouped(d[0].data_ptr(), d[1].data_ptr(), 50, d[2].data_ptr(), d[3].data_ptr(), None, 0, d[4].data_ptr(), 3,
                                                    d[5].data_ptr(), R, out.data_ptr(), _abi.AQ_BF16, N, K, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert out[live:].eq(7.0).all()
        assert out[1].eq(0).all() and out[2].eq(0).all() and not out[0].eq(0).all()
        ok = tok.clamp(0, 49)
        if not swiglu:
            want = _projections(xq, sx, wq, sw, offsets, ok, None).to(torch.bfloat16)
            keep = [r for r in range(live) if r not in (1, 2)]
            assert torch.equal(out.cpu()[keep], want[keep])


def test_grouped_offsets_out_of_bounds_touch_nothing_else(kernel):
    """Offsets below 0, past R or falling are the caller's mistake: other rows and other memory stay as they are."""
    from khaosz_amd import _abi
    R, K, N = 40, 32, 16
    for bad in ([-5, 10, 100, 30, 1 << 30], [0, 40, 20, 40, 40], [50, 60, 70, 80, 90], [-9, -8, -7, -6, -5]):
        xq, sx, wq, sw, _, _, _ = _on(*_operands([10] * 4, K, N, 2))
        offsets = torch.tensor(bad, dtype=torch.int32, device=DEV)
        out = torch.full((3 * R, N), 7.0, device=DEV)
        rc = _abi.load().aq_linear_w8a8_grouped(xq.data_ptr(), sx.data_ptr(), R, wq.data_ptr(), sw.data_ptr(), None, 0, offsets.data_ptr(), 4, None, R,
                                                out[R:2 * R].data_ptr(), _abi.AQ_F32, N, K, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert out[:R].eq(7.0).all() and out[2 * R:].eq(7.0).all()


@pytest.mark.parametrize("K,F", [(16, 16), (64, 48), (208, 112), (1536, 96), (1040, 272)])
@pytest.mark.parametrize("groups", ["one row", "empty ends", "tile edges", "a large one", "200 experts"])
def test_grouped_swiglu(kernel, groups, K, F):
    """h is up silu(gate) of the projections as stored: off by the exponential's two steps, a sum, a quotient, a product (7 half steps of fp32; a
    bf16 result by a faster exponential, within 2^-16), and the rounding to the output's type."""
    _say("grouped swiglu", kernel, groups, K, F)
    for tokens, dtype in ((None, torch.bfloat16), (29, torch.float32)):
        xq, sx, wq, sw, offsets, tok, _ = _operands(GROUPS[groups], K, 2 * F, K + F, tokens)
        sw *= 30.0 / math.sqrt(K)  # gates from -50 to 50
        ug = _projections(xq, sx, wq, sw, offsets, tok, None).to(dtype).double()
        up, gate = ug.chunk(2, dim=1)
        want = up * (gate / (1.0 + torch.exp(-gate)))
        got = ops.swiglu_w8a8_grouped(*_on(xq, sx, wq, sw, offsets), None if tok is None else tok.to(DEV), out_dtype=dtype)
        assert got.shape == want.shape and got.dtype == dtype
        tol = HALF[dtype] + (2.0 ** -16 if dtype == torch.bfloat16 else 7 * HALF[dtype])
        # (exponentials past 87 are taken as that: silu there is below 1e-35)
        assert ((got.cpu().double() - want).abs() <= tol * want.abs() + 1e-34 * up.abs() + 1e-38).all()


def test_grouped_swiglu_over_every_gate(kernel):
    """Every bf16 gate, each beside 256 ups, in bf16: nothing but the 7 half steps of fp32 that the layer's frozen form takes (the exponential's two steps, a sum, a
    quotient, a product) before the rounding of h.  Gates below -87 have the exponential of 87."""
    F = 256
    gates = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    gates = gates[gates.abs() < 1e18]  # (beyond, a product with an up overflows; what is not finite: below)
    R = gates.numel()
    g = torch.Generator(device=DEV).manual_seed(11)
    xq, wq = torch.zeros(R, 16, dtype=torch.int8, device=DEV), torch.zeros(1, 2 * F, 16, dtype=torch.int8, device=DEV)
    xq[:, 0], wq[:, :, 0] = 1, 1
    sw = torch.ones(1, 2 * F, device=DEV)
    sw[0, :F] = 1.0 + torch.rand(F, generator=g, device=DEV)
    sx = gates.float()
    offsets = torch.tensor([0, R], dtype=torch.int32, device=DEV)
    got = ops.swiglu_w8a8_grouped(xq, sx, wq, sw, offsets).double()
    up, gate = (sx[:, None] * sw[:, :F]).to(torch.bfloat16).double(), gates.double()[:, None]
    want = up * gate / (1.0 + torch.exp(-gate.clamp(min=-87.0)))
    tol = HALF[torch.bfloat16] + 7 * HALF[torch.float32]
    assert ((got - want).abs() <= tol * want.abs() + 1e-37).all()  # (1e-37: of numbers below fp32's normal ones)
    # what is not finite, as a division has it
    sx = torch.tensor([math.inf, -math.inf, math.nan], device=DEV)
    odd = ops.swiglu_w8a8_grouped(xq[:3], sx, wq, sw, torch.tensor([0, 3], dtype=torch.int32, device=DEV))
    assert odd[:2].eq(math.inf).all() and odd[2].isnan().all()


# ---- the weighted sum -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (3, 2, 7), (11, 6, 2048), (5, 9, 33), (40, 16, 1536), (130, 8, 264), (2, 64, 40), (700, 3, 520)])
def test_combine(T, k, N, dtype):
    _say("combine", T, k, N, dtype)
    g = torch.Generator().manual_seed(T + k + N)
    R = T * k
    y = torch.randn(R, N, generator=g).to(dtype)
    rows = torch.randperm(R, generator=g).view(T, k).int()
    rows[torch.rand(T, k, generator=g) < 0.2] = -1
    rows[0, 0] = R  # outside: as -1
    if T > 2:
        rows[2] = -1
    w = torch.rand(T, k, generator=g)
    res = torch.randn(T, N, generator=g).to(dtype)
    live = ((rows >= 0) & (rows < R))[:, :, None]
    terms = torch.where(live, y.double()[rows.clamp(0, R - 1).long()], 0.0) * w.double()[:, :, None]
    for r in (None, res):
        want, size = terms.sum(1), terms.abs().sum(1)
        if r is not None:
            want, size = want + r.double(), size + r.double().abs()
        got = ops.combine_rows(y.to(DEV), rows.to(DEV), w.to(DEV), None if r is None else r.to(DEV)).cpu()
        assert got.dtype == dtype and got.shape == (T, N)
        # each term: a product and at most k + 1 additions in fp32; then the output's rounding
        assert ((got.double() - want).abs() <= (k + 2) * HALF[torch.float32] * size + HALF[dtype] * want.abs() + 1e-40).all()


@pytest.mark.parametrize("kernel_of", [2, 3, 4])
def test_outputs_past_32_bits(kernel_of):
    """1.1 million rows of 2056 bf16 values are 4.5 GB: products that write them, and sums that read the last of them."""
    from khaosz_amd import _abi
    R, K, N = 1_100_000, 16, 2056
    g = torch.Generator().manual_seed(1)
    xq = torch.randint(-127, 128, (64, K), generator=g, dtype=torch.int8)
    wq = torch.randint(-127, 128, (2, N, K), generator=g, dtype=torch.int8)
    sx, sw = torch.rand(64, generator=g), torch.rand(2, N, generator=g)
    tok = (torch.arange(R, dtype=torch.int32) * 7) % 64
    offsets = torch.tensor([0, 1_000_003, R], dtype=torch.int32)
    with _abi.lab_library() as lab:
        lab.aq_lab_set_grouped_kernel(kernel_of)
        y = ops.linear_w8a8_grouped(*_on(xq, sx, wq, sw, offsets, tok))
    each = torch.stack([((xq.float() @ wq[e].float().t()) * sx[:, None]) * sw[e] for e in range(2)]).to(torch.bfloat16)
    for lo, hi in ((0, 500), (1_000_000, 1_000_500), (1_044_000, 1_045_500), (R - 700, R)):
        at = torch.arange(lo, hi)
        assert torch.equal(y[lo:hi].cpu(), each[(at >= 1_000_003).long(), tok[at].long()])
    rows = torch.tensor([[R - 1, 0], [R - 2, 1_044_500], [-1, R - 3]], dtype=torch.int32)
    got = ops.combine_rows(y, rows.to(DEV), torch.ones(3, 2, device=DEV))
    last = lambda r: y[r].float().cpu()
    assert torch.equal(got.cpu(), torch.stack([last(R - 1) + last(0), last(R - 2) + last(1_044_500), last(R - 3)]).to(torch.bfloat16))


def test_weights_past_32_bits(kernel):
    """260 experts of 4096 x 4096 codes: the last one's begin 4.3 GB behind the first's."""
    E, K, N = 260, 4096, 4096
    g = torch.Generator(device=DEV).manual_seed(2)
    wq = torch.zeros(E, N, K, dtype=torch.int8, device=DEV)
    wq[0], wq[-1] = (torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8, device=DEV) for _ in range(2))
    sw = torch.rand(E, N, generator=g, device=DEV) * 1e-4
    xq, sx = torch.randint(-127, 128, (5, K), generator=g, dtype=torch.int8, device=DEV), torch.rand(5, generator=g, device=DEV)
    offsets = torch.full((E + 1,), 2, dtype=torch.int32, device=DEV)
    offsets[0], offsets[-1] = 0, 5
    y = ops.linear_w8a8_grouped(xq, sx, wq, sw, offsets, out_dtype=torch.float32)
    h = ops.swiglu_w8a8_grouped(xq, sx, wq, sw, offsets, out_dtype=torch.float32)
    for lo, hi, e in ((0, 2, 0), (2, 5, -1)):
        one = ops.linear_w8a8(xq[lo:hi], sx[lo:hi], wq[e], sw[e], out_dtype=torch.float32)
        assert torch.equal(y[lo:hi], one)
        up, gate = one.double().chunk(2, 1)
        want = up * gate / (1 + torch.exp(-gate))
        assert ((h[lo:hi].double() - want).abs() <= 8 * HALF[torch.float32] * want.abs() + 1e-34 * up.abs() + 1e-38).all()  # (as above)


def test_combine_ignores_what_no_row_names():
    y = torch.full((6, 64), math.nan, device=DEV)
    y[4] = 1.0
    rows = torch.tensor([[4, -1], [-1, -1]], dtype=torch.int32, device=DEV)
    w = torch.tensor([[0.5, math.nan], [math.inf, 1.0]], device=DEV)
    out = ops.combine_rows(y, rows, w)
    assert out[0].eq(0.5).all() and out[1].eq(0).all()
    assert ops.combine_rows(y, rows[:0], w[:0]).shape == (0, 64)


# ---- the whole layer ------------------------------------------------------------------------------------------------

def _layer(E, dim, F, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    up_gate = torch.randn(E, 2 * F, dim, generator=g, device=DEV) / math.sqrt(dim)
    down = torch.randn(E, dim, F, generator=g, device=DEV) / math.sqrt(F)
    (uq, us), (dq, ds) = (ops.quant_rowwise_i8(w.view(-1, w.shape[2])) for w in (up_gate, down))
    return up_gate, down, uq.view(E, 2 * F, dim), us.view(E, -1), dq.view(E, dim, F), ds.view(E, -1)


def _composed(x, r, uq, us, dq, ds, residual):
    xq, sx = ops.quant_rowwise_i8(x)
    h = ops.swiglu_w8a8_grouped(xq, sx, uq, us, r.offsets, r.tokens, out_dtype=x.dtype)
    h[int(r.offsets[-1]):] = 0
    hq, sh = ops.quant_rowwise_i8(h)
    y = ops.linear_w8a8_grouped(hq, sh, dq, ds, r.offsets, out_dtype=x.dtype)
    return ops.combine_rows(y, r.rows, r.weights, residual)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k,dim,F", [(1, 64, 6, 2048, 1408), (1, 8, 1, 64, 16), (2, 8, 2, 256, 352), (5, 60, 4, 1536, 704), (16, 64, 6, 512, 208), (17, 4, 4, 128, 64),
                                         (60, 16, 3, 1040, 144), (300, 8, 2, 256, 352), (900, 16, 4, 512, 288)])
def test_layer_is_its_parts(T, E, k, dim, F, dtype):
    _say("layer", T, E, k, dim, F, dtype)
    up_gate, down, *q = _layer(E, dim, F, T)
    g = torch.Generator(device=DEV).manual_seed(T + 1)
    x = torch.randn(T, dim, generator=g, device=DEV).to(dtype)
    x[:, 3] *= 5.0
    logits = torch.randn(T, E, generator=g, device=DEV)
    if T > 4:
        logits[1] = -math.inf  # padding
        logits[T // 2:, E // 2:] = -math.inf if E // 2 >= k else 0.0
    res = torch.randn(T, dim, generator=g, device=DEV).to(dtype)
    r = ops.route_topk(logits, k)
    for residual in (None, res):
        got = ops.experts_w8a8(x, r, *q, residual=residual)
        assert torch.equal(got, _composed(x, r, *q, residual))
    assert torch.equal(got, ops.experts_w8a8(x, r, *q, residual=residual))  # the same bits again
    if T > 4:
        assert torch.equal(got[1], res[1]) and ops.experts_w8a8(x, r, *q)[1].eq(0).all()
    # and near the layer in floating point: the noise of codes of activations, weights and h
    want = res.double()
    p = torch.zeros(T, E, device=DEV, dtype=torch.float64)
    live = r.experts >= 0
    t, j = live.nonzero(as_tuple=True)
    p[t, r.experts[t, j].long()] = r.weights[t, j].double()
    for e in range(E):
        at = p[:, e].nonzero()[:, 0]
        if at.numel():
            up, gate = (x[at].double() @ up_gate[e].double().t()).chunk(2, 1)
            want[at] += p[at, e, None] * ((up * torch.nn.functional.silu(gate)) @ down[e].double().t())
    assert (got.double() - want).norm() / want.norm() < 4e-2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,k", [(63, 1), (64, 1), (65, 1), (32, 2), (33, 2), (16, 4)])
def test_layer_whose_tokens_fit_a_wavefront_and_do_not(T, k, dtype):
    """63 to 66 rows of 3 experts, tiles of up to 16: the tokens beside the offsets, or read row by row; and a row of a token that there is not."""
    _, _, uq, us, dq, ds = _layer(3 + k, 144, 80, T)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, 144, generator=g, device=DEV).to(dtype)
    r = ops.route_topk(torch.randn(T, 3 + k, generator=g, device=DEV), k)
    assert torch.equal(ops.experts_w8a8(x, r, uq, us, dq, ds), _composed(x, r, uq, us, dq, ds, None))
    tokens = r.tokens.clone()
    tokens[0], tokens[T // 2], tokens[-1] = -1, T, 1 << 30
    odd = r._replace(tokens=tokens)
    got = ops.experts_w8a8(x, odd, uq, us, dq, ds)
    assert torch.equal(got, _composed(x, odd, uq, us, dq, ds, None))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k,dim,F", [(1, 4, 2, 128, 6912), (1, 2, 1, 8192, 48), (1, 2, 1, 8208, 48), (2, 4, 4, 64, 8192), (2, 4, 4, 64, 8208), (3, 4, 3, 4112, 4112),
                                         (4, 8, 2, 64, 6912), (5, 8, 2, 6912, 64), (7, 4, 2, 96, 4128), (16, 4, 4, 4112, 32), (16, 4, 4, 32, 4112), (40, 4, 1, 2064, 2064)])
def test_layer_of_long_rows(T, E, k, dim, F, dtype):
    """Rows of x or of h of more than 4096 (fp32: 2048) are quantised in the products' launches while a workgroup has room for them."""
    _say("long rows", T, E, k, dim, F, dtype)
    _, _, uq, us, dq, ds = _layer(E, dim, F, T)
    g = torch.Generator(device=DEV).manual_seed(T)
    x, res = (torch.randn(T, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    r = ops.route_topk(torch.randn(T, E, generator=g, device=DEV), k)
    assert torch.equal(ops.experts_w8a8(x, r, uq, us, dq, ds, residual=res), _composed(x, r, uq, us, dq, ds, res))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k,dim,F", [(1, 64, 8, 64, 8192), (1, 64, 16, 64, 8192), (2, 128, 9, 16, 8192), (1, 64, 8, 64, 4096), (3, 256, 16, 32, 4096), (1, 64, 16, 8192, 16)])
def test_layer_of_long_rows_and_many_choices(T, E, k, dim, F, dtype):
    """A row of codes for each of eight wavefronts: more than 64 KB of a compute unit's LDS."""
    _say("long rows, many choices", T, E, k, dim, F, dtype)
    _, _, uq, us, dq, ds = _layer(E, dim, F, T)
    g = torch.Generator(device=DEV).manual_seed(T)
    x, res = (torch.randn(T, dim, generator=g, device=DEV).to(dtype) for _ in range(2))
    r = ops.route_topk(torch.randn(T, E, generator=g, device=DEV), k)
    assert torch.equal(ops.experts_w8a8(x, r, uq, us, dq, ds, residual=res), _composed(x, r, uq, us, dq, ds, res))


@pytest.mark.parametrize("T,E,k,dim,F", [(54, 128, 1, 3568, 80), (16, 60, 1, 1936, 80), (2, 16, 2, 4096, 48), (2, 16, 2, 4112, 48), (512, 2, 1, 16, 16), (513, 2, 1, 16, 16)])
def test_layer_of_many_columns_and_narrow_experts(T, E, k, dim, F):
    """The second product and the sum in one launch, or not: the same bits; and never in a launch of so many workgroups that the layer takes far longer than its parts
    one after the other (the first of these took three times as long)."""
    _say("many columns", T, E, k, dim, F)
    _, _, uq, us, dq, ds = _layer(E, dim, F, T)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, dim, generator=g, device=DEV).bfloat16()
    r = ops.route_topk(torch.randn(T, E, generator=g, device=DEV), k)

    def parts():
        xq, sx = ops.quant_rowwise_i8(x)
        hq, sh = ops.quant_rowwise_i8(ops.swiglu_w8a8_grouped(xq, sx, uq, us, r.offsets, r.tokens))
        return ops.combine_rows(ops.linear_w8a8_grouped(hq, sh, dq, ds, r.offsets), r.rows, r.weights)
    assert torch.equal(ops.experts_w8a8(x, r, uq, us, dq, ds), parts())
    us_of = []
    for call in (lambda: ops.experts_w8a8(x, r, uq, us, dq, ds), parts):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(10):
                call()
        times = []
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            graph.replay()
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b) * 100)
        us_of.append(min(times))
    assert us_of[0] < 1.8 * us_of[1], us_of


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 5, 40, 700])
def test_layer_with_infinities_and_nan_in_a_row(T, dtype):
    """The same bits, or NaN in the same places, whichever launch quantises the rows; the other rows as without them."""
    _say("odd rows", T, dtype)
    _, _, uq, us, dq, ds = _layer(8, 256, 352, T)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = torch.randn(T, 256, generator=g, device=DEV).to(dtype)
    r = ops.route_topk(torch.randn(T, 8, generator=g, device=DEV), 2)
    clean = ops.experts_w8a8(x, r, uq, us, dq, ds)
    others = torch.arange(T, device=DEV) != T // 2
    for odd in (math.inf, -math.inf, math.nan, 3e38):
        x[T // 2, 7] = odd
        got, want = ops.experts_w8a8(x, r, uq, us, dq, ds), _composed(x, r, uq, us, dq, ds, None)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
        assert torch.equal(got[others], clean[others])


def test_layer_of_no_tokens():
    _, _, uq, us, dq, ds = _layer(3, 64, 32, 1)
    r = ops.route_topk(torch.empty(0, 3, device=DEV), 2)
    x = torch.empty(0, 64, device=DEV)
    assert ops.experts_w8a8(x, r, uq, us, dq, ds).shape == (0, 64)
    assert ops.linear_w8a8_grouped(x.to(torch.int8), x[:, 0], uq, us, r.offsets).shape == (0, 64)
    assert ops.combine_rows(x, r.rows, r.weights).shape == (0, 64)


def test_layer_under_a_graph_on_another_stream_and_twice_at_once():
    """One captured pass (routing and experts) replayed over new inputs beside eager work; two streams at once."""
    E, k, dim, F = 16, 4, 256, 128
    _, _, *q = _layer(E, dim, F, 3)
    g = torch.Generator(device=DEV).manual_seed(8)
    for T in (3, 40, 600):
        x = torch.randn(T, dim, generator=g, device=DEV).to(torch.bfloat16)
        logits = torch.randn(T, E, generator=g, device=DEV).to(torch.bfloat16)

        def go(a, b):
            return ops.experts_w8a8(a, ops.route_topk(b, k), *q, residual=a)
        want = go(x, logits)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = go(x, logits)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = go(x, logits)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(beside, want)
        for i in range(4):
            x.copy_(torch.randn(T, dim, generator=g, device=DEV))
            logits.copy_(torch.randn(T, E, generator=g, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, go(x, logits)), (T, i)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        x2, l2 = x.flip(0).contiguous(), logits.flip(0).contiguous()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            a = [go(x, logits) for _ in range(5)]
        b = [go(x2, l2) for _ in range(5)]
        torch.cuda.synchronize()
        assert all(torch.equal(v, go(x, logits)) for v in a) and all(torch.equal(v, go(x2, l2)) for v in b)


def test_general_path_gives_the_same_bits():
    """Non-contiguous operands and dtypes the native path leaves to the Python one."""
    E, k, dim, F, T = 8, 2, 128, 64, 20
    _, _, uq, us, dq, ds = _layer(E, dim, F, 4)
    x = torch.randn(T, 2 * dim, device=DEV).to(torch.bfloat16)[:, ::2]
    logits = torch.randn(T, 2 * E, device=DEV)[:, ::2]
    r = ops.route_topk(logits, k)
    want = ops.experts_w8a8(x.contiguous(), ops.route_topk(logits.contiguous(), k), uq, us, dq, ds)
    assert torch.equal(ops.experts_w8a8(x, r, uq, us, dq, ds), want)
    assert torch.equal(ops.experts_w8a8(x, ops.Routing(*(t.clone() for t in r)), uq, us.t().contiguous().t(), dq, ds), want)
    assert ops.experts_w8a8(x[:0], ops.route_topk(logits[:0], k), uq, us, dq, ds).shape == (0, dim)
    xq, sx = ops.quant_rowwise_i8(x)
    a = ops.linear_w8a8_grouped(xq, sx, uq, us, r.offsets, r.tokens)
    b = ops.linear_w8a8_grouped(xq.t().contiguous().t(), sx, uq, us, r.offsets, torch.stack([r.tokens, r.tokens], 1)[:, 0])
    assert torch.equal(a, b)


def test_refusals_on_the_device():
    E, k, dim, F, T = 4, 2, 64, 32, 6
    _, _, uq, us, dq, ds = _layer(E, dim, F, 4)
    x, logits = torch.randn(T, dim, device=DEV), torch.randn(T, E, device=DEV)
    r = ops.route_topk(logits, k)
    xq, sx = ops.quant_rowwise_i8(x)
    bad = [
        lambda: ops.route_topk(logits, 0),
        lambda: ops.route_topk(logits, E + 1),
        lambda: ops.route_topk(logits.half(), k),
        lambda: ops.route_topk(logits[0], k),
        lambda: ops.route_topk(torch.zeros(2, 513, device=DEV), 2),
        lambda: ops.route_topk(torch.zeros(2, 64, device=DEV), 17),
        lambda: ops.linear_w8a8_grouped(xq, sx, uq, us, r.offsets.long(), r.tokens),
        lambda: ops.linear_w8a8_grouped(xq, sx, uq, us, r.offsets[:-1], r.tokens),
        lambda: ops.linear_w8a8_grouped(xq, sx, uq, us, r.offsets, r.tokens.long()),
        lambda: ops.linear_w8a8_grouped(xq, sx, uq[:, :, :32], us, r.offsets, r.tokens),
        lambda: ops.linear_w8a8_grouped(xq, sx, uq, us[:, :-1], r.offsets, r.tokens),
        lambda: ops.linear_w8a8_grouped(xq, sx[:-1], uq, us, r.offsets, r.tokens),
        lambda: ops.linear_w8a8_grouped(xq, sx, uq, us, r.offsets, r.tokens, bias=us[0]),
        lambda: ops.linear_w8a8_grouped(xq, sx, uq, us, r.offsets, r.tokens, out_dtype=torch.float16),
        lambda: ops.linear_w8a8_grouped(xq[:, 8:24], sx, uq[:, :, 8:32], us, r.offsets, r.tokens),
        lambda: ops.linear_w8a8_grouped(xq.view(torch.uint8), sx, uq, us, r.offsets, r.tokens),
        lambda: ops.swiglu_w8a8_grouped(xq, sx, uq[:, :48], us[:, :48], r.offsets, r.tokens),
        lambda: ops.swiglu_w8a8_grouped(xq, sx, uq, us, r.offsets, r.tokens, out_dtype=None),
        lambda: ops.combine_rows(x, r.rows.long(), r.weights),
        lambda: ops.combine_rows(x, r.rows, r.weights.double()),
        lambda: ops.combine_rows(x, r.rows, r.weights[:, :1]),
        lambda: ops.combine_rows(x.half(), r.rows, r.weights),
        lambda: ops.combine_rows(x, r.rows, r.weights, residual=x[:, :32]),
        lambda: ops.combine_rows(x, r.rows, r.weights, residual=x.to(torch.bfloat16)),
        lambda: ops.experts_w8a8(x[:3], r, uq, us, dq, ds),
        lambda: ops.experts_w8a8(x.half(), r, uq, us, dq, ds),
        lambda: ops.experts_w8a8(x, r, uq[:, :48], us[:, :48], dq, ds),
        lambda: ops.experts_w8a8(x, r, uq, us, dq[:, :32], ds[:, :32]),
        lambda: ops.experts_w8a8(x, r, uq, us, dq[:3], ds[:3]),
        lambda: ops.experts_w8a8(x, r, uq.float(), us, dq, ds),
        lambda: ops.experts_w8a8(x, r._replace(offsets=r.offsets[1:]), uq, us, dq, ds),
        lambda: ops.experts_w8a8(x, r._replace(tokens=r.tokens[1:]), uq, us, dq, ds),
        lambda: ops.experts_w8a8(x, r._replace(weights=r.weights[:, :1]), uq, us, dq, ds),
        lambda: ops.experts_w8a8(x, r, uq, us, dq, ds, residual=x[:, :32]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            _say("not refused:", i)
    with pytest.raises(RuntimeError):
        ops.experts_w8a8(x.cpu(), r, uq, us, dq, ds)
    with pytest.raises(RuntimeError):
        ops.linear_w8a8_grouped(xq, sx, uq, us, r.offsets.cpu(), r.tokens)
