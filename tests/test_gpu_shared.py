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
            size = float((scale * (kh.abs() @ qh.abs())).max()) if n else 0.0
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


@pytest.mark.parametrize("B,Hq,Hkv,D,page,shared,T", [
    (2, 1, 1, 64, 64, 64, 65),          # the smallest shared block
    (2, 24, 4, 64, 128, 512, 576),
    (3, 16, 4, 128, 64, 64, 64),        # everything is shared
    (2, 4, 4, 128, 1, 70, 131),         # pages of one position
    (9, 6, 2, 128, 16, 160, 161),       # three heads a KV head, one own position
    (5, 8, 1, 64, 24, 456, 500),        # pages end inside a block
    (33, 24, 4, 64, 16, 1008, 1401),
    (17, 16, 2, 128, 48, 960, 1300),    # 136 rows a KV head: a tile and a piece of one
    (70, 4, 2, 128, 256, 1024, 1030),   # 140 rows
    (128, 2, 2, 64, 64, 320, 333),      # 128 rows, one head each
    (130, 3, 1, 128, 64, 640, 700),     # 390 rows
    (8, 16, 4, 128, 64, 2048, 2591),
    (4, 32, 8, 128, 128, 4096, 4100),
    (3, 2, 1, 64, 4096, 4096, 4200),    # one page holds all that is shared
    (2, 2, 2, 128, 100, 20000, 20001),  # long, pages of an odd size
])
def test_against_64_bits(B, Hq, Hkv, D, page, shared, T):
    _say("shared", B, Hq, Hkv, D, page, shared, T)
    q, k, v, table = _case(B, Hq, Hkv, D, page, shared, T, seed=T + B)
    want, tol = _expected(q, k, v, table, T)
    _check(ops.paged_attn_decode_shared(q, k, v, table, T, shared), want, tol)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shared", [0, 1, 63, 64, 65, 127, 128, 200, 255, 256, 300, 399, 400, 1 << 40])
def test_any_shared_length_means_the_same(D, shared):
    """The promise may cut a page or a block anywhere, or reach past the last position."""
    _say("shared lengths", D, shared)
    q, k, v, table = _case(5, 8, 2, D, 40, 400, 400)
    want, tol = _expected(q, k, v, table, 400)
    got = ops.paged_attn_decode_shared(q, k, v, table, 400, shared)
    _check(got, want, tol)
    if shared < 64:
        assert torch.equal(got, ops.paged_attn_decode(q, k, v, table, 400))


def test_one_sequence_shares_nothing():
    q, k, v, table = _case(1, 16, 4, 128, 64, 512, 700)
    assert torch.equal(ops.paged_attn_decode_shared(q, k, v, table, 700, 512), ops.paged_attn_decode(q, k, v, table, 700))


@pytest.mark.parametrize("B,Hq,Hkv,D,page,shared,T,lens", [
    (4, 8, 2, 64, 64, 256, 700, [700, 257, 300, 699]),
    (4, 8, 2, 128, 64, 256, 700, [700, 256, 255, 1]),            # ends at the border, inside, at once
    (6, 4, 4, 64, 16, 512, 520, [520, 0, 64, 65, 130, 511]),     # one without any length: the average of all positions
    (3, 4, 2, 128, 64, 128, 512, [0, -5, 100000]),               # cut to 0 .. T
    (70, 6, 2, 64, 24, 240, 301, None),
    (150, 4, 4, 128, 64, 320, 330, None),
])
def test_sequences_at_different_positions(B, Hq, Hkv, D, page, shared, T, lens):
    _say("shared lens", B, Hq, Hkv, D, page, shared, T)
    q, k, v, table = _case(B, Hq, Hkv, D, page, shared, T, seed=B)
    lens = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B)) if lens is None else torch.tensor(lens)
    want, tol = _expected(q, k, v, table, T, lens)
    _check(ops.paged_attn_decode_shared(q, k, v, table, T, shared, seq_lens=lens.to(DEV)), want, tol)


def test_all_sequences_without_any_length():
    q, k, v, table = _case(3, 4, 2, 64, 16, 320, 400)
    lens = torch.zeros(3, dtype=torch.int64)
    want, tol = _expected(q, k, v, table, 400, lens)
    _check(ops.paged_attn_decode_shared(q, k, v, table, 400, 320, seq_lens=lens.to(DEV)), want, tol)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_what_lies_behind_every_length_may_hold_anything(page, value):
    """Shared positions that no sequence sees, and each sequence's own behind its length."""
    q, k, v, table = _case(4, 8, 2, 128, page, 640, 900, seed=page)
    lens = torch.tensor([300, 500, 20, 499])
    got = ops.paged_attn_decode_shared(q, k, v, table, 900, 640, seq_lens=lens.to(DEV))
    own = torch.tensor([900, 700, 641, 800])
    far = ops.paged_attn_decode_shared(q, k, v, table, 900, 640, seq_lens=own.to(DEV))
    k2, v2, k3, v3 = k.clone(), v.clone(), k.clone(), v.clone()
    pos = torch.arange(900, device=DEV)
    for b in range(4):
        behind = pos[500:]
        k2[table[b, behind // page], behind % page] = value
        v2[table[b, behind // page], behind % page] = value
        behind = pos[int(own[b]):]
        k3[table[b, behind // page], behind % page] = value
        v3[table[b, behind // page], behind % page] = value
    assert torch.equal(ops.paged_attn_decode_shared(q, k2, v2, table, 900, 640, seq_lens=lens.to(DEV)), got)
    assert torch.equal(ops.paged_attn_decode_shared(q, k3, v3, table, 900, 640, seq_lens=own.to(DEV)), far)


@pytest.mark.parametrize("page", [16, 64, 200])
def test_unmapped_pages_are_zero_keys_and_values(page):
    q, k, v, table = _case(6, 8, 2, 128, page, 600, 1001, seed=page)
    table[:, 1] = -1                          # shared
    table[:, 2] = k.shape[0]                  # a page past the cache
    table[2, 600 // page + 1] = -7            # one sequence's own
    table[3, -1] = 1 << 40
    want, tol = _expected(q, k, v, table, 1001)
    _check(ops.paged_attn_decode_shared(q, k, v, table, 1001, 600), want, tol)


def test_positions_past_the_page_table_are_unmapped():
    q, k, v, table = _case(3, 4, 2, 64, 64, 256, 300)
    short = table[:, :3].contiguous()
    want, tol = _expected(q, k, v, short, 300)
    _check(ops.paged_attn_decode_shared(q, k, v, short, 300, 256), want, tol)


def test_large_scores_and_a_scale():
    """Scores of some hundreds: the running maximum is raised block by block."""
    q, k, v, table = _case(7, 4, 2, 128, 64, 768, 800, gain=20.0)
    k[table[0, 5], 3] = k[table[0, 5], 3] * 4
    for scale in (None, 0.02, 1.0):
        want, tol = _expected(q, k, v, table, 800, scale=scale)
        _check(ops.paged_attn_decode_shared(q, k, v, table, 800, 768, scale=scale), want, tol)


def test_strided_inputs_and_a_workspace():
    q, k, v, table = _case(5, 8, 2, 64, 32, 448, 500)
    want = ops.paged_attn_decode_shared(q, k, v, table, 500, 448)
    wide = torch.zeros(5, 8, 100, dtype=torch.bfloat16, device=DEV)
    wide[..., 8:72] = q
    tall = torch.zeros(5, 40, dtype=torch.int64, device=DEV)
    tall[:, 3:3 + table.shape[1]] = table
    assert torch.equal(ops.paged_attn_decode_shared(wide[..., 8:72], k, v, tall[:, 3:3 + table.shape[1]], 500, 448), want)
    need = ops.paged_attn_shared_workspace_bytes(5, 8, 2, 64, 500, 448, DEV)
    ws = torch.full((need // 4 + 64,), float("nan"), device=DEV)
    assert torch.equal(ops.paged_attn_decode_shared(q, k, v, table, 500, 448, workspace=ws), want)
    assert bool(ws[need // 4:].isnan().all())
    assert torch.equal(ops.paged_attn_decode_shared(q, k, v, table, 500, 448, workspace=ws[:16]), want)  # too small: one of its own


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
    n_pages = (1 << 32) // (page * Hkv * D) + 40
    k, v = (torch.empty(n_pages, page, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(1)
    k[-40:].normal_(generator=g)
    v[-40:].normal_(generator=g)
    q = torch.randn(3, 16, D, generator=g, device=DEV).to(torch.bfloat16)
    table = (n_pages - 40 + torch.cat([torch.arange(8).expand(3, -1), 8 + torch.arange(9).view(3, 3)], 1)).to(DEV)
    got = ops.paged_attn_decode_shared(q, k, v, table, 700, 512)
    near = ops.paged_attn_decode_shared(q, k[-40:].clone(), v[-40:].clone(), table - (n_pages - 40), 700, 512)
    assert torch.equal(got, near)


def test_captured_and_replayed():
    """Two graphs and eager calls in turn, on new inputs each time."""
    cases = [_case(8, 16, 4, 128, 64, 1024, 1200, seed=s) for s in range(3)]
    lens = torch.randint(1025, 1201, (8,), generator=torch.Generator().manual_seed(0)).to(DEV)
    want = [ops.paged_attn_decode_shared(*c, 1200, 1024, seq_lens=lens) for c in cases]
    held = [t.clone() for t in cases[0]]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_attn_decode_shared(*held, 1200, 1024, seq_lens=lens)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.paged_attn_decode_shared(*held, 1200, 1024, seq_lens=lens))
        graphs.append(g)
    for turn in range(6):
        c = turn % 3
        for t, x in zip(held, cases[c]):
            t.copy_(x)
        graphs[turn % 2].replay()
        graphs[1 - turn % 2].replay()
        other = ops.paged_attn_decode_shared(*cases[(c + 1) % 3], 1200, 1024, seq_lens=lens)
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
