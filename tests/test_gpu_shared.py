"""Decode attention of a batch that shares its first pages, against the definition in 64 bits (GPU).

The tolerance, per element: the output's own rounding, half a bf16 step (2^-8 of it); every probability of a shared position rounded
by at most half a step, so at most 2^-8 of sum p |v| / sum p; and, on the same scale, the scores' and sums' fp32 error: a score is a
sum of D products, off by at most (D + 4) 2^-24 of scale * sum |q k| (log2(e) and the maximum's subtraction included: 4), which
moves a weight by that much of itself, once in the numerator and once in the denominator; each of them is a sum of T terms, off by at
most T 2^-24 of sum p |v|; exponentials, weights of the slices and the reciprocal stay within 8 steps of 2^-24 each."""
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

from khaosz_amd import ops  # noqa: E402

DEV = "cuda:0"
MASKED = -1.0e30


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def _expected(q, kc, vc, table, T, lens=None, scale=None):
    """(out, tolerance) [B, Hq, D] in 64 bits: one sequence at a time, everything gathered, no page twice."""
    B, Hq, D = q.shape
    n_pages, page, Hkv, _ = kc.shape
    scale = D ** -0.5 if scale is None else scale
    out, tol = torch.empty(B, Hq, D, dtype=torch.float64), torch.empty(B, Hq, D, dtype=torch.float64)
    for b in range(B):
        pos = torch.arange(T)
        col = pos // page
        ids = torch.where(col < table.shape[1], table[b].cpu()[col.clamp(max=table.shape[1] - 1)], -1)
        ok = (ids >= 0) & (ids < n_pages)
        at = (ids.clamp(0, n_pages - 1), pos % page)
        n = T if lens is None else max(0, min(T, int(lens[b])))
        seen = n if n else T
        k, v = (torch.where(ok[:, None, None], c.cpu()[at].double(), 0.0)[:seen] for c in (kc, vc))
        for h in range(Hq):
            kh, vh, qh = k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)], q[b, h].cpu().double()
            s = scale * (kh @ qh) if n else torch.zeros(T, dtype=torch.float64)
            p = torch.exp(s - s.max())
            p = p / p.sum()
            out[b, h] = p @ vh
            size = scale * (kh.abs() @ qh.abs())
            size = float(size[size.isfinite()].max()) if n and bool(size.isfinite().any()) else 0.0
            near = 2.0 ** -8 + 2 * size * (D + 4) * 2.0 ** -24 + 2 * T * 2.0 ** -24 + 24 * 2.0 ** -24
            tol[b, h] = 2.0 ** -8 * out[b, h].abs() * (1 + near) + near * (p @ vh.abs())
    return out, tol


def _check(got, want, tol):
    err = (got.cpu().double() - want).abs()
    worst = (err / tol.clamp(min=1e-300)).max().item()
    assert bool((err <= tol).all()), f"error is {worst:.2f} times the tolerance"


def _case(B, Hq, Hkv, D, page, shared, T, seed=0, extra=3, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    P, common = -(-T // page) + 1, -(-shared // page)
    mine = P - common
    n_pages = common + B * mine + extra
    ids = torch.randperm(n_pages, generator=g)
    table = torch.cat([ids[:common].expand(B, -1), ids[common:common + B * mine].view(B, mine)], 1).contiguous()
    q = (torch.randn(B, Hq, D, generator=g) * gain).to(torch.bfloat16)
    k, v = (torch.randn(n_pages, page, Hkv, D, generator=g).to(torch.bfloat16) for _ in range(2))
    return [t.to(DEV) for t in (q, k, v, table)]


def _is_shared(q, k, T, shared):
    """Whether the call reads the shared positions once: it then keeps other partial results than the decode kernel, which takes calls that
    would gain nothing."""
    (B, Hq, D), Hkv = q.shape, k.shape[2]
    return ops.paged_attn_shared_workspace_bytes(B, Hq, Hkv, D, T, shared, DEV) != ops.paged_attn_workspace_bytes(B, Hq, Hkv, T)


@pytest.mark.parametrize("B,Hq,Hkv,D,page,shared,T", [
    (2, 1, 1, 64, 64, 2048, 2049),      # two rows, one own position
    (2, 24, 4, 64, 128, 2432, 2500),
    (3, 16, 4, 128, 64, 2112, 2112),    # everything is shared
    (2, 4, 4, 128, 1, 2070, 2131),      # pages of one position
    (9, 6, 2, 128, 16, 2160, 2161),     # three heads a KV head, one own position
    (5, 8, 1, 64, 24, 2088, 2150),      # pages end inside a block
    (33, 24, 4, 64, 16, 1008, 1401),
    (17, 16, 2, 128, 48, 2064, 2300),   # 136 rows a KV head: two tiles and a piece of one
    (17, 16, 4, 128, 48, 960, 1300),    # 68 rows
    (70, 4, 2, 128, 256, 1024, 1030),
    (128, 2, 2, 64, 64, 640, 660),
    (130, 3, 1, 128, 64, 640, 700),     # 390 rows
    (66, 16, 8, 128, 64, 4096, 4170),   # 132 rows of many: tiles of 128
    (34, 32, 8, 64, 32, 8192, 8200),    # the same, pages of half a block
    (66, 16, 8, 128, 24, 4104, 4110),   # pages of another size
    (2, 2, 2, 128, 3, 20001, 20300),    # more pages in a slice than are kept in LDS: 20001 positions of one tile
    (300, 8, 1, 64, 128, 512, 777),
    (2, 8, 1, 128, 4096, 4096, 9000),   # one page holds all that is shared; long tails
    (4, 4, 4, 64, 1, 2600, 30000),      # tails with pages of one position
    (8, 16, 4, 128, 64, 2048, 2591),
    (4, 32, 8, 128, 128, 4096, 4100),
    (2, 2, 2, 128, 100, 20000, 20001),  # long, pages of an odd size
])
def test_against_64_bits(B, Hq, Hkv, D, page, shared, T):
    _say("shared", B, Hq, Hkv, D, page, shared, T)
    q, k, v, table = _case(B, Hq, Hkv, D, page, shared, T, seed=T + B)
    assert _is_shared(q, k, T, shared)
    want, tol = _expected(q, k, v, table, T)
    _check(ops.paged_attn_decode_shared(q, k, v, table, T, shared), want, tol)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shared", [0, 1, 63, 64, 65, 900, 1500, 1535, 1536, 1537, 2000, 2239, 2240, 2299, 2300, 1 << 40])
def test_any_shared_length_means_the_same(D, shared):
    """The promise may cut a page or a block anywhere, or reach past the last position."""
    _say("shared lengths", D, shared)
    q, k, v, table = _case(5, 8, 2, D, 40, 2300, 2300)
    want, tol = _expected(q, k, v, table, 2300)
    got = ops.paged_attn_decode_shared(q, k, v, table, 2300, shared)
    _check(got, want, tol)
    assert _is_shared(q, k, 2300, shared) == (shared >= 64)
    if shared < 64:
        assert torch.equal(got, ops.paged_attn_decode(q, k, v, table, 2300))


@pytest.mark.parametrize("B,Hq,Hkv,D,page,shared,T", [(2, 24, 4, 64, 128, 512, 576), (8, 16, 4, 128, 64, 512, 700), (3, 4, 2, 64, 16, 64, 65)])
def test_calls_that_gain_nothing_by_it_are_the_decode_kernels(B, Hq, Hkv, D, page, shared, T):
    q, k, v, table = _case(B, Hq, Hkv, D, page, shared, T)
    lens = torch.randint(0, T + 1, (B,)).to(DEV)
    assert not _is_shared(q, k, T, shared)
    assert torch.equal(ops.paged_attn_decode_shared(q, k, v, table, T, shared, seq_lens=lens), ops.paged_attn_decode(q, k, v, table, T, seq_lens=lens))


def test_one_sequence_shares_nothing():
    q, k, v, table = _case(1, 16, 4, 128, 64, 512, 700)
    assert torch.equal(ops.paged_attn_decode_shared(q, k, v, table, 700, 512), ops.paged_attn_decode(q, k, v, table, 700))


@pytest.mark.parametrize("B,Hq,Hkv,D,page,shared,T,lens", [
    (4, 8, 2, 64, 64, 1792, 2300, [2300, 1793, 1900, 2299]),
    (4, 8, 2, 128, 64, 1792, 2300, [2300, 1792, 1791, 1]),              # ends at the border, inside, at once
    (6, 4, 4, 64, 16, 2048, 2056, [2056, 0, 64, 65, 130, 2047]),        # one without any length: the average of all positions
    (3, 4, 2, 128, 64, 1920, 2212, [0, -5, 100000]),                    # cut to 0 .. T
    (70, 6, 2, 64, 24, 1032, 1101, None),
    (150, 4, 4, 128, 64, 640, 677, None),
    (66, 16, 8, 128, 64, 4096, 4170, None),
    (66, 16, 8, 64, 20, 8200, 8230, None),
])
def test_sequences_at_different_positions(B, Hq, Hkv, D, page, shared, T, lens):
    _say("shared lens", B, Hq, Hkv, D, page, shared, T)
    q, k, v, table = _case(B, Hq, Hkv, D, page, shared, T, seed=B)
    lens = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B)) if lens is None else torch.tensor(lens)
    assert _is_shared(q, k, T, shared)
    want, tol = _expected(q, k, v, table, T, lens)
    _check(ops.paged_attn_decode_shared(q, k, v, table, T, shared, seq_lens=lens.to(DEV)), want, tol)


def test_all_sequences_without_any_length():
    q, k, v, table = _case(3, 4, 2, 64, 16, 2048, 2101)
    lens = torch.zeros(3, dtype=torch.int64)
    assert _is_shared(q, k, 2101, 2048)
    want, tol = _expected(q, k, v, table, 2101, lens)
    _check(ops.paged_attn_decode_shared(q, k, v, table, 2101, 2048, seq_lens=lens.to(DEV)), want, tol)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_lies_behind_every_length_may_hold_anything(page, value):
    """Shared positions that no sequence sees, and each sequence's own behind its length."""
    T, shared = 2500, 2176
    q, k, v, table = _case(4, 8, 2, 128, page, shared, T, seed=page)
    assert _is_shared(q, k, T, shared)
    lens = torch.tensor([300, 500, 20, 499])
    got = ops.paged_attn_decode_shared(q, k, v, table, T, shared, seq_lens=lens.to(DEV))
    own = torch.tensor([2500, 2300, 2177, 2400])
    far = ops.paged_attn_decode_shared(q, k, v, table, T, shared, seq_lens=own.to(DEV))
    k2, v2, k3, v3 = k.clone(), v.clone(), k.clone(), v.clone()
    pos = torch.arange(T, device=DEV)
    for b in range(4):
        behind = pos[500:]
        k2[table[b, behind // page], behind % page] = value
        v2[table[b, behind // page], behind % page] = value
        behind = pos[int(own[b]):]
        k3[table[b, behind // page], behind % page] = value
        v3[table[b, behind // page], behind % page] = value
    assert torch.equal(ops.paged_attn_decode_shared(q, k2, v2, table, T, shared, seq_lens=lens.to(DEV)), got)
    assert torch.equal(ops.paged_attn_decode_shared(q, k3, v3, table, T, shared, seq_lens=own.to(DEV)), far)


def _check_odd(got, want, tol):
    """The same where some of it is infinite or NaN: infinite or NaN there, near everywhere else."""
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    ok = want.isfinite()
    assert bool((got[want.isinf()] == want[want.isinf()]).all())
    _check(got[ok], want[ok], tol[ok])


@pytest.mark.parametrize("B,Hq,Hkv,D,page,shared,T", [
    (4, 8, 2, 128, 16, 2176, 2500), (4, 8, 2, 64, 64, 2176, 2500), (66, 16, 8, 128, 64, 4096, 4140), (66, 16, 8, 64, 24, 4104, 4140)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["keys", "values"])
def test_what_lies_behind_a_length_changes_nothing_of_its_result(B, Hq, Hkv, D, page, shared, T, value, where):
    """... though other sequences see it and have it in theirs: one element of shared position 450, one of a sequence's own."""
    _say("odd", B, Hq, Hkv, D, page, shared, T, value, where)
    q, k, v, table = _case(B, Hq, Hkv, D, page, shared, T, seed=page + B)
    assert _is_shared(q, k, T, shared)
    lens = torch.randint(200, T + 1, (B,), generator=torch.Generator().manual_seed(B))
    lens[:4] = torch.tensor([300, 450, 451, T])
    if B > 4:
        lens[9] = 0
    c = k if where == "keys" else v
    c[table[0, 450 // page], 450 % page, 1, 5] = value
    c[table[3, (T - 1) // page], (T - 1) % page, 0, D - 1] = value
    want, tol = _expected(q, k, v, table, T, lens)
    assert bool(want[:2].isfinite().all()) and (where == "keys" or not bool(want[2:4].isfinite().all()))
    _check_odd(ops.paged_attn_decode_shared(q, k, v, table, T, shared, seq_lens=lens.to(DEV)), want, tol)


@pytest.mark.parametrize("D", [64, 128])
def test_scores_without_a_bound(D):
    """Queries that are infinite or NaN, and whole blocks of keys whose scores are -infinity, first ones of a slice among them."""
    q, k, v, table = _case(5, 8, 2, D, 64, 2176, 2400)
    assert _is_shared(q, k, 2400, 2176)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    for first in (0, 512, 1111, 2304):
        for pos in range(first, first + 96):
            k[table[1, pos // 64], pos % 64, 0, 0] = -float("inf")
    lens = torch.tensor([2400, 2400, 64, 2399, 30])  # two of them see nothing else: NaN, with the heads of KV head 0
    for n in (None, lens):
        want, tol = _expected(q, k, v, table, 2400, n)
        assert n is None or bool(want[2, 0].isnan().all()) and bool(want[2, 7].isfinite().all())
        _check_odd(ops.paged_attn_decode_shared(q, k, v, table, 2400, 2176, seq_lens=None if n is None else n.to(DEV)), want, tol)
    q[1, 2, 7] = float("nan")
    q[3, 5, 1] = float("inf")  # scores of both infinities
    want, tol = _expected(q, k, v, table, 2400)
    assert bool(want[1, 2].isnan().all()) and bool(want[3, 5].isnan().all()) and bool(want[0].isfinite().all())
    _check_odd(ops.paged_attn_decode_shared(q, k, v, table, 2400, 2176), want, tol)


@pytest.mark.parametrize("page", [16, 64, 200])
def test_unmapped_pages_are_zero_keys_and_values(page):
    q, k, v, table = _case(6, 8, 2, 128, page, 1800, 2201, seed=page)
    assert _is_shared(q, k, 2201, 1800)
    table[:, 1] = -1                          # shared
    table[:, 2] = k.shape[0]                  # a page past the cache
    table[2, 1800 // page + 1] = -7           # one sequence's own
    table[3, -1] = 1 << 40
    want, tol = _expected(q, k, v, table, 2201)
    _check(ops.paged_attn_decode_shared(q, k, v, table, 2201, 1800), want, tol)


def test_positions_past_the_page_table_are_unmapped():
    for page in (64, 24):
        q, k, v, table = _case(3, 4, 2, 64, page, 2112, 2200)
        short = table[:, :1000 // page].contiguous()
        assert _is_shared(q, k, 2200, 2112)
        want, tol = _expected(q, k, v, short, 2200)
        _check(ops.paged_attn_decode_shared(q, k, v, short, 2200, 2112), want, tol)


def test_large_scores_and_a_scale():
    """Scores of some hundreds: the running maximum is raised block by block."""
    q, k, v, table = _case(7, 4, 2, 128, 64, 2048, 2080, gain=20.0)
    assert _is_shared(q, k, 2080, 2048)
    k[table[0, 5], 3] = k[table[0, 5], 3] * 4
    for scale in (None, 0.02, 1.0):
        want, tol = _expected(q, k, v, table, 2080, scale=scale)
        _check(ops.paged_attn_decode_shared(q, k, v, table, 2080, 2048, scale=scale), want, tol)


def test_strided_inputs_and_a_workspace():
    q, k, v, table = _case(5, 8, 2, 64, 32, 2240, 2300)
    want = ops.paged_attn_decode_shared(q, k, v, table, 2300, 2240)
    wide = torch.zeros(5, 8, 100, dtype=torch.bfloat16, device=DEV)
    wide[..., 8:72] = q
    tall = torch.zeros(5, 90, dtype=torch.int64, device=DEV)
    tall[:, 3:3 + table.shape[1]] = table
    assert torch.equal(ops.paged_attn_decode_shared(wide[..., 8:72], k, v, tall[:, 3:3 + table.shape[1]], 2300, 2240), want)
    need = ops.paged_attn_shared_workspace_bytes(5, 8, 2, 64, 2300, 2240, DEV)
    ws = torch.full((need // 4 + 64,), float("nan"), device=DEV)
    assert torch.equal(ops.paged_attn_decode_shared(q, k, v, table, 2300, 2240, workspace=ws), want)
    assert bool(ws[need // 4:].isnan().all())
    assert torch.equal(ops.paged_attn_decode_shared(q, k, v, table, 2300, 2240, workspace=ws[:16]), want)  # too small: one of its own


def test_the_same_bits_each_time_and_on_another_stream():
    q, k, v, table = _case(40, 16, 4, 128, 64, 2048, 2300)
    want = ops.paged_attn_decode_shared(q, k, v, table, 2300, 2048)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = ops.paged_attn_decode_shared(q, k, v, table, 2300, 2048)
    b = ops.paged_attn_decode_shared(q, k, v, table, 2300, 2048)  # both at once
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def test_pages_beyond_32_bits():
    """Offsets of the last pages pass 2^32 elements."""
    page, Hkv, D = 64, 8, 128
    n_pages = (1 << 32) // (page * Hkv * D) + 60
    k, v = (torch.empty(n_pages, page, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(1)
    k[-60:].normal_(generator=g)
    v[-60:].normal_(generator=g)
    q = torch.randn(3, 16, D, generator=g, device=DEV).to(torch.bfloat16)
    table = (n_pages - 60 + torch.cat([torch.arange(32).expand(3, -1), 32 + torch.arange(9).view(3, 3)], 1)).to(DEV)
    assert _is_shared(q, k, 2200, 2048)
    got = ops.paged_attn_decode_shared(q, k, v, table, 2200, 2048)
    near = ops.paged_attn_decode_shared(q, k[-60:].clone(), v[-60:].clone(), table - (n_pages - 60), 2200, 2048)
    assert torch.equal(got, near)


def test_captured_and_replayed():
    """Two graphs and eager calls in turn, on new inputs each time."""
    cases = [_case(8, 16, 4, 128, 64, 2048, 2200, seed=s) for s in range(3)]
    lens = torch.randint(2049, 2201, (8,), generator=torch.Generator().manual_seed(0)).to(DEV)
    want = [ops.paged_attn_decode_shared(*c, 2200, 2048, seq_lens=lens) for c in cases]
    held = [t.clone() for t in cases[0]]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_attn_decode_shared(*held, 2200, 2048, seq_lens=lens)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attn_decode_shared(*held, 2200, 2048, seq_lens=lens))
        graphs.append(g)
    for turn in range(6):
        c = turn % 3
        for t, x in zip(held, cases[c]):
            t.copy_(x)
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        other = ops.paged_attn_decode_shared(*cases[(c + 1) % 3], 2200, 2048, seq_lens=lens)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[c]) and torch.equal(outs[1], want[c]) and torch.equal(other, want[(c + 1) % 3]), turn


def test_empty_batch():
    q, k, v, table = _case(2, 4, 2, 64, 16, 64, 80)
    out = ops.paged_attn_decode_shared(q[:0], k, v, table[:0], 80, 64)
    assert out.shape == (0, 4, 64)


def test_refusals():
    q, k, v, table = _case(2, 4, 2, 64, 16, 64, 80)
    call = ops.paged_attn_decode_shared
    with pytest.raises(RuntimeError, match="GPU only"):
        call(q.cpu(), k, v, table, 80, 64)
    with pytest.raises(ValueError, match="bfloat16"):
        call(q.float(), k, v, table, 80, 64)
    with pytest.raises(ValueError, match="caches"):
        call(q, k, v[:1], table, 80, 64)
    with pytest.raises(ValueError, match="contiguous"):
        call(q, k[:, ::2], v[:, ::2], table, 80, 64)
    with pytest.raises(ValueError, match="int64"):
        call(q, k, v, table.int(), 80, 64)
    with pytest.raises(ValueError, match="int64"):
        call(q, k, v, table[:1], 80, 64)
    with pytest.raises(ValueError, match="seq_lens"):
        call(q, k, v, table, 80, 64, seq_lens=torch.ones(2, device=DEV))
    for bad in (dict(total_len=0, shared_len=0), dict(total_len=80, shared_len=-1), dict(total_len=(1 << 30) + 1, shared_len=64),
                dict(total_len=80, shared_len=64, scale=-1.0), dict(total_len=80, shared_len=64, scale=float("nan"))):
        with pytest.raises(ValueError):
            call(q, k, v, table, **bad)
    with pytest.raises(ValueError):  # five query heads per KV head
        call(torch.zeros(2, 10, 64, dtype=torch.bfloat16, device=DEV), k, v, table, 80, 64)
    with pytest.raises(ValueError):  # head dimension
        call(q[..., :32].contiguous(), k[..., :32].contiguous(), v[..., :32].contiguous(), table, 80, 64)
