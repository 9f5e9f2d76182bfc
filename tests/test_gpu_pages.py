"""Forks of page-table rows and the compaction of pages, against plain Python on the host (GPU).  Tables, counts and every byte of the
caches have to be equal."""
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

from khaosz_amd import ops  # noqa: E402

DEV = "cuda:0"


def _say(*a):
    print(*a, file=sys.stderr, flush=True)


def _caches(layers, n_pages, page, heads, dim, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(-100, 100, (layers, n_pages, page, heads, dim), generator=g).to(dtype) for _ in range(2)]


def _forked(table, refs, parents, k, v, total, lens=None):
    """The definition, one row after the other, in place on copies."""
    B, P = table.shape
    n_pages, page = refs.numel(), k.shape[2]
    rows = [[e if 0 <= e < n_pages else -1 for e in r] for r in table.tolist()]
    refs, k, v = refs.tolist(), k.clone(), v.clone()
    for row in rows:
        for e in row:
            if e >= 0:
                refs[e] -= 1
    refs = [max(r, 0) for r in refs]
    new, wants, seen = [], [], set()
    for i, p in enumerate(parents.tolist()):
        if not 0 <= p < B:
            new.append([-1] * P)
            continue
        n = total if lens is None else max(0, min(total, int(lens[p])))
        whole, rest = divmod(n, page)
        if p not in seen:
            row = list(rows[p])
        else:
            row = rows[p][:whole] + [-1] * (P - whole)
            if rest and whole < P and rows[p][whole] >= 0:
                wants.append((i, whole, rest, rows[p][whole]))
        seen.add(p)
        new.append(row)
        for e in row:
            if e >= 0:
                refs[e] += 1
    free = [x for x, r in enumerate(refs) if r == 0]
    for (i, whole, rest, source), to in zip(wants, free):
        new[i][whole], refs[to] = to, 1
        k[:, to, :rest], v[:, to, :rest] = k[:, source, :rest], v[:, source, :rest]
    return (torch.tensor(new, dtype=torch.int64).view(-1, P), torch.tensor(refs, dtype=torch.int32),
            torch.tensor([max(0, len(wants) - len(free))], dtype=torch.int32), k, v)


def _compacted(table, refs, k, v):
    n_pages = refs.numel()
    r, k, v = refs.tolist(), k.clone(), v.clone()
    live = sum(x > 0 for x in r)
    where = [x if r[x] > 0 else -1 for x in range(n_pages)]
    holes = [x for x in range(live) if r[x] <= 0]
    out = [x for x in reversed(range(live, n_pages)) if r[x] > 0]
    counts = [max(0, x) for x in r]
    for source, to in zip(out, holes):
        where[source], counts[to], counts[source] = to, r[source], 0
        k[:, to], v[:, to] = k[:, source], v[:, source]
    new = [[where[e] if 0 <= e < n_pages else -1 for e in row] for row in table.tolist()]
    return (torch.tensor(new, dtype=torch.int64).view(table.shape), torch.tensor(counts, dtype=torch.int32),
            torch.tensor(where), torch.tensor([live], dtype=torch.int32), k, v)


def _equal(got, want, k, v):
    for name, a, b in zip(want._fields if hasattr(want, "_fields") else range(9), (*got, k, v), want):
        assert torch.equal(a.cpu(), b), name


def _fork_check(table, refs, parents, k, v, total, lens=None):
    want = _forked(table, refs, parents, k, v, total, lens)
    kd, vd, td, rd = k.to(DEV), v.to(DEV), table.to(DEV), refs.to(DEV)
    got = ops.fork_pages(td, rd, parents.to(DEV), kd, vd, total, seq_lens=None if lens is None else lens.to(DEV))
    _equal(got, want, kd, vd)
    assert torch.equal(td.cpu(), table) and torch.equal(rd.cpu(), refs)  # left as they were
    return want


def _state(B, P, n_pages, page, layers=2, heads=2, dim=16, seed=0, common=0, dtype=torch.bfloat16, extra_refs=3):
    """Rows that share their first `common` columns, and a few pages that someone else holds."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(n_pages, generator=g)
    own = common + B * (P - common)
    assert own + extra_refs <= n_pages
    table = torch.cat([ids[:common].expand(B, -1), ids[common:own].view(B, P - common)], 1).contiguous()
    refs = torch.zeros(n_pages, dtype=torch.int32)
    refs[ids[:common]] = B
    refs[ids[common:own]] = 1
    refs[ids[own:own + extra_refs]] = 2
    return (table, refs, *_caches(layers, n_pages, page, heads, dim, dtype, seed))


@pytest.mark.parametrize("page,total", [(16, 40), (16, 48), (16, 1), (1, 3), (24, 70), (128, 300), (7, 20)])
@pytest.mark.parametrize("parents", [[0], [0, 0, 0, 0], [2, 1, 0], [1, 1, 2, 1, 2], [], [-1, 0, 3, 99, 2, 2], [2] * 9])
def test_fork_small(page, total, parents):
    _say("fork", page, total, parents)
    P = -(-total // page) + 1
    table, refs, k, v = _state(3, P, 3 * P + 16, page, common=1)
    _fork_check(table, refs, torch.tensor(parents, dtype=torch.int64), k, v, total)


@pytest.mark.parametrize("B,R,P,page,n_pages,layers,seed", [(64, 64, 23, 16, 2000, 2, 0), (1, 300, 5, 64, 400, 1, 1), (200, 40, 30, 4, 6100, 1, 2),
                                                           (256, 300, 17, 16, 9000, 3, 3), (2, 2, 2049, 2, 4200, 1, 4),
                                                           (70, 90, 200, 4, 14500, 1, 5), (4, 9, 3, 16, 8193, 1, 6), (300, 5000, 2, 4, 5700, 1, 7),
                                                           (5, 7, 4, 16, 8190, 1, 8), (64, 2100, 3, 4, 4097, 2, 9),
                                                           (300, 700, 3600, 2, 1100003, 1, 10), (4000, 4090, 4, 4, 8190, 1, 11),
                                                           (4096, 4095, 4, 4, 4110, 1, 12), (256, 256, 2, 4, 1024, 2, 13),
                                                           (100, 1, 8, 16, 1021, 1, 14), (3, 253, 4, 16, 1024, 3, 15), (256, 256, 2, 4, 1025, 1, 16)])
def test_fork_rows_at_lengths_of_their_own(B, R, P, page, n_pages, layers, seed):
    _say("fork lens", B, R, P, page, n_pages)
    table, refs, k, v = _state(B, P, n_pages, page, layers=layers, seed=seed, common=min(3, P - 1), heads=1)
    g = torch.Generator().manual_seed(seed)
    parents = torch.randint(0, max(1, B // 3), (R,), generator=g)
    lens = torch.randint(-3, P * page + 9, (B,), generator=g)
    lens[0] = P * page - 1
    _fork_check(table, refs, parents, k, v, P * page, lens)


def test_fork_takes_pages_that_have_just_become_free():
    """No page is free before: the dropped rows' pages are handed out, lowest first."""
    table = torch.tensor([[4, 1], [3, 0], [5, 2]])
    refs = torch.ones(6, dtype=torch.int32)
    k, v = _caches(1, 6, 8, 1, 8)
    want = _fork_check(table, refs, torch.tensor([1, 1, 1]), k, v, 12)
    assert want[0].tolist() == [[3, 0], [3, 1], [3, 2]] and want[1].tolist() == [1, 1, 1, 3, 0, 0]


def test_fork_without_enough_free_pages():
    table = torch.tensor([[0, 1], [0, 2]])
    refs = torch.tensor([2, 1, 1, 0, 7], dtype=torch.int32)
    k, v = _caches(2, 5, 8, 1, 8)
    want = _fork_check(table, refs, torch.tensor([0, 0, 1, 0, 1]), k, v, 13)
    assert want[2].tolist() == [2] and want[0].tolist() == [[0, 1], [0, 3], [0, 2], [0, -1], [0, -1]]


def test_fork_of_tables_and_counts_that_do_not_fit_each_other():
    """Unmapped entries, entries past the cache, pages named twice, counts below what the table names: nothing outside is touched and
    no page in use is handed out."""
    table = torch.tensor([[0, -1, 9, 3], [1 << 40, 2, 2, -(1 << 60)], [3, 4, 4, 4]])
    refs = torch.tensor([0, 0, 1, 0, 2, -7, 0, 0], dtype=torch.int32)
    k, v = _caches(2, 8, 4, 1, 8)
    for total in (0, 3, 6, 10, 15, 16):
        _fork_check(table, refs, torch.tensor([2, 2, 0, 0, 1, 1, 5]), k, v, total)


def test_fork_an_empty_table():
    k, v = _caches(1, 6, 4, 1, 8)
    _fork_check(torch.zeros(0, 3, dtype=torch.int64), torch.tensor([1, 0, 2, 0, 0, 0], dtype=torch.int32), torch.tensor([0, 1]), k, v, 5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16, torch.int8])
def test_fork_and_compact_one_layer_of_any_type(dtype):
    table, refs, k, v = _state(4, 3, 40, 12, layers=1, heads=2, dim=40, dtype=dtype, seed=5)
    want = _forked(table, refs, torch.tensor([0, 0, 3, 3, 3]), k, v, 30)
    kd, vd = k[0].to(DEV), v[0].to(DEV)
    got = ops.fork_pages(table.to(DEV), refs.to(DEV), torch.tensor([0, 0, 3, 3, 3], device=DEV), kd, vd, 30)
    _equal(got, want, kd.unsqueeze(0), vd.unsqueeze(0))
    want = _compacted(want[0], want[1], *want[3:])
    got = ops.compact_pages(got.page_table, got.refs, kd, vd)
    _equal(got, want, kd.unsqueeze(0), vd.unsqueeze(0))


@pytest.mark.parametrize("n_pages,live", [(1, 0), (1, 1), (8, 3), (100, 0), (100, 100), (1000, 1), (1023, 500), (1024, 512), (1025, 1024), (4095, 2047), (4096, 4096), (4096, 2000), (4097, 4096), (5000, 1), (16384, 9000), (16385, 16000), (20000, 11111), (70001, 35000), (1100003, 600001)])
def test_compact(n_pages, live):
    _say("compact", n_pages, live)
    g = torch.Generator().manual_seed(n_pages + live)
    refs = torch.zeros(n_pages, dtype=torch.int32)
    held = torch.randperm(n_pages, generator=g)[:live]
    refs[held] = torch.randint(1, 9, (live,), generator=g, dtype=torch.int32)
    table = torch.randint(-2, n_pages + 2, (7, 13), generator=g)
    k, v = _caches(2, n_pages, 2, 1, 8, seed=live)
    want = _compacted(table, refs, k, v)
    kd, vd = k.to(DEV), v.to(DEV)
    got = ops.compact_pages(table.to(DEV), refs.to(DEV), kd, vd)
    _equal(got, want, kd, vd)


def test_compact_pages_larger_than_a_turn_and_layers_apart():
    """Pages of several turns of a workgroup and a piece of one; layers that are a slice of a larger allocation."""
    g = torch.Generator().manual_seed(0)
    k, v = _caches(3, 30, 50, 3, 72, seed=2)  # 21600 bytes a page
    refs = (torch.rand(30, generator=g) < 0.4).int()
    table = torch.randint(0, 30, (2, 5), generator=g)
    want = _compacted(table, refs, k[:, :22], v[:, :22]) if int(refs[22:].sum()) == 0 else None
    refs, table = refs[:22].contiguous(), table.clamp(max=21)
    want = _compacted(table, refs, k[:, :22], v[:, :22])
    kd, vd = k.to(DEV), v.to(DEV)
    got = ops.compact_pages(table.to(DEV), refs.to(DEV), kd[:, :22], vd[:, :22])
    _equal(got, want, kd[:, :22], vd[:, :22])
    assert torch.equal(kd[:, 22:].cpu(), k[:, 22:]) and torch.equal(vd[:, 22:].cpu(), v[:, 22:])


def test_compact_without_a_table():
    refs = torch.tensor([0, 1, 0, 2], dtype=torch.int32)
    k, v = _caches(1, 4, 4, 1, 8)
    want = _compacted(torch.zeros(0, 2, dtype=torch.int64), refs, k, v)
    kd, vd = k.to(DEV), v.to(DEV)
    _equal(ops.compact_pages(torch.zeros(0, 2, dtype=torch.int64, device=DEV), refs.to(DEV), kd, vd), want, kd, vd)


def test_captured_and_replayed():
    """A fork and a compaction in one graph, replayed on new tables, eager work between; another stream too."""
    B, P, n_pages, page = 16, 9, 400, 16
    states = [_state(B, P, n_pages, page, seed=s, common=2) for s in range(3)]
    parents = [torch.randint(0, B, (20,), generator=torch.Generator().manual_seed(s)) for s in range(3)]

    def expected(s):
        t, r, m, k, v = _forked(states[s][0], states[s][1], parents[s], states[s][2], states[s][3], 130)
        return (m, *_compacted(t, r, k, v))

    want = [expected(s) for s in range(3)]
    held = [t.to(DEV) for t in (*states[0], parents[0])]

    def step():
        f = ops.fork_pages(held[0], held[1], held[4], held[2], held[3], 130)
        return f.missing, ops.compact_pages(f.page_table, f.refs, held[2], held[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        missing, out = step()
    for turn in range(5):
        s = turn % 3
        for t, x in zip(held, (*states[s], parents[s])):
            t.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((missing, *out, held[2], held[3]), want[s]):
            assert torch.equal(a.cpu(), b), turn
        if turn % 2:
            for t, x in zip(held, (*states[s], parents[s])):
                t.copy_(x)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                m2, o2 = step()
            torch.cuda.synchronize()
            for a, b in zip((m2, *o2, held[2], held[3]), want[s]):
                assert torch.equal(a.cpu(), b), turn


def test_pages_beyond_32_bits():
    """The last pages' offsets pass 2^32 bytes and 2^32 elements."""
    page, heads, dim = 64, 8, 128
    n_pages = (1 << 32) // (page * heads * dim) + 8
    k, v = (torch.zeros(n_pages, page, heads, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    k[-2:].normal_()
    v[-2:].normal_()
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    refs[-2:] = 1
    refs[:n_pages - 7] = 1
    table = torch.tensor([[n_pages - 2, n_pages - 1]], device=DEV)
    ka, va = k[-2:].clone(), v[-2:].clone()
    f = ops.fork_pages(table, refs, torch.tensor([0, 0], device=DEV), k, v, 100)
    to = n_pages - 7
    assert f.page_table.tolist() == [[n_pages - 2, n_pages - 1], [n_pages - 2, to]] and f.missing.item() == 0
    assert torch.equal(k[to, :36], ka[1, :36]) and torch.equal(v[to, :36], va[1, :36]) and not bool(k[to, 36:].any())
    c = ops.compact_pages(f.page_table, f.refs, k, v)
    assert c.live.item() == n_pages - 4 and c.page_table.tolist() == [[n_pages - 5, n_pages - 6], [n_pages - 5, to]]
    assert torch.equal(k[n_pages - 6], ka[1]) and torch.equal(k[n_pages - 5], ka[0]) and torch.equal(v[n_pages - 6], va[1])


def test_counts_at_any_address():
    table, refs, k, v = _state(3, 4, 40, 16)
    want = _forked(table, refs, torch.tensor([0, 0, 2]), k, v, 50)
    kd, vd = k.to(DEV), v.to(DEV)
    odd = torch.zeros(43, dtype=torch.int32, device=DEV)[3:]
    odd.copy_(refs)
    got = ops.fork_pages(table.to(DEV), odd, torch.tensor([0, 0, 2], device=DEV), kd, vd, 50)
    _equal(got, want, kd, vd)


def test_refusals():
    table, refs, k, v = (t.to(DEV) for t in _state(2, 2, 12, 16))
    parents = torch.tensor([0, 1], device=DEV)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.fork_pages(table, refs, parents.cpu(), k, v, 20)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.compact_pages(table.cpu(), refs, k, v)
    for bad_table in (table.int(), table[0], table[:, :0]):
        with pytest.raises(ValueError, match="page_table"):
            ops.fork_pages(bad_table, refs, parents, k, v, 0)
        with pytest.raises(ValueError, match="page_table"):
            ops.compact_pages(bad_table, refs, k, v)
    for bad_refs in (refs.long(), refs[:-1], refs.view(3, 4)):
        with pytest.raises(ValueError, match="refs"):
            ops.fork_pages(table, bad_refs, parents, k, v, 20)
        with pytest.raises(ValueError, match="refs"):
            ops.compact_pages(table, bad_refs, k, v)
    for bad in ((k, v[:, :5]), (k, v.float()), (k[0, 0], v[0, 0]), (k[:, ::2], v[:, ::2]), (k[:0], v[:0]), (k[..., :4], v[..., :4])):
        with pytest.raises(ValueError, match="caches|contiguous"):
            ops.compact_pages(table, refs, *bad)
    with pytest.raises(ValueError, match="16 bytes"):
        ops.compact_pages(table, refs, k[..., :1, :4].contiguous(), v[..., :1, :4].contiguous())
    with pytest.raises(ValueError, match="parents"):
        ops.fork_pages(table, refs, parents.int(), k, v, 20)
    with pytest.raises(ValueError, match="parents"):
        ops.fork_pages(table, refs, parents.view(1, 2), k, v, 20)
    for total in (-1, 33):
        with pytest.raises(ValueError, match="outside"):
            ops.fork_pages(table, refs, parents, k, v, total)
    with pytest.raises(ValueError, match="seq_lens"):
        ops.fork_pages(table, refs, parents, k, v, 20, seq_lens=torch.ones(3, dtype=torch.int64, device=DEV))
