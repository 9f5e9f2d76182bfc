"""Decode steps of a fused block on long contexts, with and without a shared prefix: queued natively in one call, a block has to give the bits
of the step-by-step path, whose operators get scratch memory of their own (GPU)."""
import sys

import pytest
import torch

from khaosz_amd import block, fuse_shared_inputs, ops, quantize_model
from khaosz_amd.block import DecoderBlock, PagedKV, rotary_table

DEV, DT = "cuda:0", torch.bfloat16


def _block(heads, kv_heads, dim, **options):
    torch.manual_seed(11)
    b = DecoderBlock(heads * dim, heads, 704, kv_heads, **options)
    b.reset_parameters()
    b = b.to(DEV).to(DT)
    quantize_model(b)
    fuse_shared_inputs(b, norms=True, decode_attention=True, residuals=True)
    return b


def _step(batch, heads, kv_heads, dim, page, total, shared=0, mixed=False):
    """Tokens, angles, and a cache bound for a step whose rows share their first `shared` positions (whole pages)."""
    g = torch.Generator(device=DEV).manual_seed(total + batch)
    common = shared // page
    mine = -(-total // page) - common
    n_pages = common + batch * mine
    ids = torch.randperm(n_pages, generator=g, device=DEV)
    table = torch.cat([ids[:common].expand(batch, -1), ids[common:].view(batch, mine)], 1).contiguous()
    cache = PagedKV(n_pages, page, kv_heads, dim, DEV, DT)
    cache.k_layers.normal_(generator=g)
    cache.v_layers.normal_(generator=g)
    lens = torch.randint(total // 2, total + 1, (batch,), generator=g, device=DEV) if mixed else None
    angles = rotary_table(dim, total, device=DEV)[total - 1:].unsqueeze(0).expand(batch, -1, -1)
    x = torch.randn(batch, 1, heads * dim, generator=g, device=DEV).to(DT)
    return x, angles, cache.bind(table, total, seq_lens=lens, share_prefix=shared > 0)


def _counted(monkeypatch, name):
    calls, real = [], getattr(ops, name)
    monkeypatch.setattr(ops, name, lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    return calls


def _native_and_step_by_step(monkeypatch, b, x, angles, cache, operator):
    k0, v0 = cache.k_layers.clone(), cache.v_layers.clone()
    with torch.inference_mode():
        got = block._native()(b, x, angles, cache)
        assert got is not None  # queued natively
        held = cache.k_layers.clone(), cache.v_layers.clone()
        cache.k_layers.copy_(k0)
        cache.v_layers.copy_(v0)
        calls = _counted(monkeypatch, operator)
        want = b(x, angles, None, cache)
    assert len(calls) == 1
    assert bool(want.isfinite().all()) and torch.equal(got, want)
    assert torch.equal(held[0], cache.k_layers) and torch.equal(held[1], cache.v_layers)
    assert not torch.equal(held[0], k0)  # the step's own key


# contexts on which reading all positions once, were they shared, would take less scratch memory than the decode kernel does, and some where not
@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv_heads,dim,page,total", [
    (8, 24, 4, 64, 128, 4096), (8, 24, 4, 64, 16, 4097), (32, 24, 4, 64, 64, 769), (32, 24, 4, 64, 24, 800), (16, 24, 4, 64, 64, 1601),
    (64, 32, 8, 128, 64, 2113), (64, 16, 4, 128, 64, 4161), (8, 16, 4, 128, 64, 700), (1, 16, 4, 128, 64, 9000)])
@pytest.mark.parametrize("mixed", [False, True])
def test_steps_without_a_shared_prefix(monkeypatch, batch, heads, kv_heads, dim, page, total, mixed):
    print("step", batch, heads, kv_heads, dim, page, total, mixed, file=sys.stderr, flush=True)
    b = _block(heads, kv_heads, dim)
    x, angles, cache = _step(batch, heads, kv_heads, dim, page, total, mixed=mixed)
    assert cache.shared_len == 0
    _native_and_step_by_step(monkeypatch, b, x, angles, cache, "rope_paged_attn_decode")


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv_heads,dim,page,total,shared", [
    (64, 32, 8, 128, 64, 8448, 8192), (16, 16, 4, 128, 128, 65600, 65536), (40, 8, 2, 64, 64, 4200, 2048), (70, 6, 2, 64, 24, 4500, 4104),
    (8, 16, 4, 128, 64, 2591, 2048), (33, 24, 4, 64, 16, 1401, 1296)])
@pytest.mark.parametrize("mixed", [False, True])
def test_steps_over_a_shared_prefix(monkeypatch, batch, heads, kv_heads, dim, page, total, shared, mixed):
    print("shared step", batch, heads, kv_heads, dim, page, total, shared, mixed, file=sys.stderr, flush=True)
    b = _block(heads, kv_heads, dim)
    x, angles, cache = _step(batch, heads, kv_heads, dim, page, total, shared, mixed)
    assert cache.shared_len == shared
    _native_and_step_by_step(monkeypatch, b, x, angles, cache, "paged_attn_decode_shared")


@pytest.mark.gpu
def test_a_replaced_rule_of_sharing_is_asked_by_fused_blocks(monkeypatch):
    """A program that replaces the rule has its blocks read the prefix once, or not, as its own rule says."""
    b = _block(8, 2, 64)
    x, angles, cache = _step(40, 8, 2, 64, 16, 2101, 2096)
    table = cache.page_table
    with torch.inference_mode():
        shared = b(x, angles, None, cache)
        apart = b(x, angles, None, cache.bind(table, 2101))
        assert not torch.equal(shared, apart)  # (probabilities are rounded in one of them)
        cache.bind(table, 2101, share_prefix=True)
        asked, rule = [], ops.paged_attn_shared_positions
        monkeypatch.setattr(ops, "paged_attn_shared_positions", lambda *a: (asked.append(a), 0)[1])
        assert torch.equal(b(x, angles, None, cache), apart)
        assert asked == [(40, 8, 2, 64, 2101, 2096, True)]
        monkeypatch.setattr(ops, "paged_attn_shared_positions", lambda *a: (asked.append(a), rule(*a))[1])
        assert torch.equal(b(x, angles, None, cache), shared) and len(asked) == 2


def test_sizes_whose_steps_share():
    """A step shares no more than the operator does, and less often: it has a launch more then."""
    rule = ops.paged_attn_shared_positions
    for sizes in ((40, 8, 2, 64, 2101, 2096), (3, 8, 2, 64, 2101, 2096), (64, 32, 8, 128, 8448, 8192), (2, 16, 4, 128, 65600, 65536)):
        assert rule(*sizes, step=True) == rule(*sizes) == sizes[5] // 64 * 64
    for sizes in ((57, 32, 8, 128, 217, 208), (49, 8, 8, 64, 1162, 400), (3, 32, 8, 128, 2097, 592), (120, 16, 4, 128, 254, 208)):
        assert rule(*sizes) == sizes[5] // 64 * 64 and rule(*sizes, step=True) == 0
    for sizes in ((0, 4, 2, 64, 3000, 2990), (2, 5, 2, 64, 3000, 2990), (2, 4, 2, 96, 3000, 2990), (2, 4, 2, 64, 3000, -1), (2, 4, 2, 64, 0, 0),
                  (1, 4, 2, 64, 3000, 2990), (2, 4, 2, 64, 3000, 63)):
        assert rule(*sizes, step=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("batch,heads,kv_heads,dim,page,total,shared", [(57, 32, 8, 128, 16, 217, 208), (49, 8, 8, 64, 16, 1162, 400)])
def test_steps_that_gain_nothing_by_sharing_are_as_ever(monkeypatch, batch, heads, kv_heads, dim, page, total, shared):
    """Sizes at which the operator alone gains by reading the prefix once and a step does not (in a graph a block of 106 us loses 10, one of 47 loses 4)."""
    assert ops.paged_attn_shared_positions(batch, heads, kv_heads, dim, total, shared) > 0
    b = _block(heads, kv_heads, dim)
    x, angles, cache = _step(batch, heads, kv_heads, dim, page, total, shared)
    assert cache.shared_len == shared
    _native_and_step_by_step(monkeypatch, b, x, angles, cache, "rope_paged_attn_decode")
    with torch.inference_mode():
        got = b(x, angles, None, cache)
        assert torch.equal(got, b(x, angles, None, cache.bind(cache.page_table, total)))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_probabilities_of_own_positions_are_rounded_too(dim):
    """The probabilities of each sequence's own positions are rounded to bf16 (by half a step, 2^-8 of themselves at most), as those of the
    shared ones are, and the denominator sums them unrounded.  Weights are taken relative to the largest of a range: where all scores
    are 0 they are 1, nothing is rounded, and the sums of small whole numbers are exact.  Where every second own position has the score 1/2, own
    weights are 1 and 2^-1/2: the own positions may move the result by that rounding, the shared ones, whose weights are 1, not at all."""
    batch, page, shared, total = 6, 64, 2048, 2560
    g = torch.Generator().manual_seed(dim)
    common, mine = shared // page, (total - shared) // page
    n_pages = common + batch * mine
    table = torch.cat([torch.arange(common).expand(batch, -1), common + torch.arange(batch * mine).view(batch, mine)], 1).cuda()
    v = torch.randint(-3, 4, (n_pages, page, 2, dim), generator=g).to(DT).cuda()
    k = torch.zeros_like(v)
    k[common:, ::2, :, 0] = 1.0  # every second of the sequences' own positions
    q = torch.zeros(batch, 8, dim, dtype=DT, device=DEV)
    for weight in (0.0, 0.5):
        q[:, :, 0] = weight  # scores 0 and weight in the exp2 domain: a scale of ln 2
        got = ops.paged_attn_decode_shared(q, k, v, table, total, shared, scale=0.6931471805599453)
        assert ops.paged_attn_shared_positions(batch, 8, 2, dim, total, shared) == shared
        for b in range(batch):
            values = v[table[b]].flatten(0, 1).double()  # [total, heads, dim]
            p = torch.where(k[table[b]].flatten(0, 1)[:, :1, :1] > 0, 2.0 ** weight, 1.0).double()
            want = (p * values).sum(0) / p.sum()
            moved = (2.0 ** -8 if weight else 0.0) * (p * values.abs())[shared:].sum(0) / p.sum()
            # fp32: T terms in each sum, the exponential and the division 8 steps of 2^-24 each; then the result's own half step
            near = moved + (2 * total + 16) * 2.0 ** -24 * (p * values.abs()).sum(0) / p.sum()
            tol = (near + 2.0 ** -8 * (want.abs() + near)).repeat_interleave(4, 0)
            assert bool(((got[b].double() - want.repeat_interleave(4, 0)).abs() <= tol).all())


@pytest.mark.gpu
def test_a_row_rolled_back_into_a_page_that_others_read():
    """Such a row is named twice: its second child has a copy of what is written, and what it writes reaches no other row.  Its first child is
    dropped in the next fork, which leaves the counts as if it had not been."""
    page, n_pages = 16, 12
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, n_pages, page, 2, 64, generator=g).to(DT).cuda() for _ in range(2))
    table = torch.tensor([[3, 5, 7, -1], [3, 5, 2, -1]], device=DEV)  # both hold page 5 as a full one ..
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    refs[table[0, :2]], refs[table[:, 2]] = 2, 1
    lens = torch.tensor([40, 21], device=DEV)  # .. and the second is set back to its 5th position in it
    k0, v0 = k.clone(), v.clone()
    one = ops.fork_pages(table, refs, torch.tensor([0, 1, 1], device=DEV), k, v, 48, seq_lens=lens)
    assert one.page_table.tolist() == [[3, 5, 7, -1], [3, 5, 2, -1], [3, 0, -1, -1]] and one.missing.item() == 0
    assert torch.equal(k[:, 0, :5], k0[:, 5, :5]) and torch.equal(v[:, 0, :5], v0[:, 5, :5])
    lens = torch.tensor([40, 21, 21], device=DEV)
    two = ops.fork_pages(one.page_table, one.refs, torch.tensor([0, 2], device=DEV), k, v, 48, seq_lens=lens)
    assert two.page_table.tolist() == [[3, 5, 7, -1], [3, 0, -1, -1]]
    want = torch.zeros(n_pages, dtype=torch.int32)
    want[3], want[5], want[7], want[0] = 2, 1, 1, 1
    assert torch.equal(two.refs.cpu(), want)
    qkv = torch.randn(2, (2 + 2 * 2) * 64, generator=g).to(DT).cuda()  # a token at position 21 of the row that was set back
    ops.rope_kv_write(qkv[1:], rotary_table(64, 22, device=DEV)[21:], two.page_table[1:], 21, k[0], v[0], 2, 2)
    assert not torch.equal(k[0, 0, 5], k0[0, 0, 5])
    others = [x for x in range(n_pages) if x != 0]
    assert torch.equal(k[:, others], k0[:, others]) and torch.equal(v[:, others], v0[:, others])
