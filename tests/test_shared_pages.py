"""Shared pages: what the C ABI refuses before any launch, and what a cache finds out about its table (CPU); a generation that samples,
drops and goes on from shared pages (GPU)."""
import pytest
import torch

from khaosz_amd import _abi, AutoRegressiveLM, LMConfig, fuse_shared_inputs, ops, quantize_model
from khaosz_amd.block import PagedKV
from test_gpu_shared import _check, _expected

P = 1 << 20  # a fake, aligned pointer: refused before any launch


def _attn(**change):
    a = dict(q=P, k=P, v=P, table=P, cols=200, total=3000, shared=2990, lens=None, page=16, n_pages=9, scale=0.1, out=P, B=2, Hq=4, Hkv=2, D=64,
             ws=P, ws_bytes=1 << 30, stream=None)
    a.update(change)
    return _abi.load().aq_paged_attn_decode_shared(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(D=96), -2), (dict(Hq=5), -2), (dict(Hq=10, Hkv=2), -2), (dict(Hkv=0), -2), (dict(B=-1), -2), (dict(cols=0), -2), (dict(total=0), -2),
    (dict(shared=-1), -2), (dict(page=0), -2), (dict(n_pages=0), -2), (dict(scale=0.0), -2), (dict(scale=float("nan")), -2), (dict(q=None), -1),
    (dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1), (dict(out=None), -1), (dict(ws=None), -1), (dict(q=P + 2), -4), (dict(k=P + 8), -4),
    (dict(v=P + 8), -4), (dict(out=P + 8), -4), (dict(ws=P + 4), -4), (dict(ws_bytes=100), -5), (dict(total=(1 << 30) + 1), -6),
    (dict(n_pages=1 << 31), -6), (dict(B=1 << 24), -6), (dict(Hkv=1 << 19, Hq=1 << 19), -6), (dict(B=0), 0),
    (dict(shared=0, total=300, ws_bytes=8), -5),  # nothing shared: the decode kernel's own checks
])
def test_attention_is_refused_before_any_launch(change, code):
    assert _attn(**change) == code


def _fork(**change):
    a = dict(table=P, B=2, cols=3, refs=P, parents=P, R=4, total=30, lens=None, k=P, v=P, layers=2, layer_bytes=9 * 16 * 64, n_pages=9, page=16,
             row_bytes=64, new_table=P, new_refs=P, missing=P, ws=P, ws_bytes=1 << 20, stream=None)
    a.update(change)
    return _abi.load().aq_fork_pages(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(B=-1), -2), (dict(R=-1), -2), (dict(cols=0), -2), (dict(total=-1), -2), (dict(layers=0), -2), (dict(n_pages=0), -2), (dict(page=0), -2),
    (dict(row_bytes=0), -2), (dict(row_bytes=24), -4), (dict(layer_bytes=9 * 16 * 64 - 16), -2), (dict(layer_bytes=9 * 16 * 64 + 8), -4),
    (dict(table=None), -1), (dict(refs=None), -1), (dict(parents=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(new_table=None), -1),
    (dict(new_refs=None), -1), (dict(missing=None), -1), (dict(ws=None), -1), (dict(k=P + 8), -4), (dict(v=P + 4), -4), (dict(table=P + 4), -4),
    (dict(parents=P + 4), -4), (dict(lens=P + 4), -4), (dict(refs=P + 2), -4), (dict(new_refs=P + 2), -4), (dict(new_table=P + 4), -4),
    (dict(ws=P + 8), -4), (dict(refs=P + 8), -4), (dict(total=49), -2), (dict(ws_bytes=100), -5), (dict(n_pages=0x7fffffff, layer_bytes=1 << 62), -6), (dict(R=1 << 25), -6), (dict(R=(1 << 16) + 1), -6), (dict(B=1 << 25), -6),
])
def test_forks_are_refused_before_any_launch(change, code):
    assert _fork(**change) == code


def _compact(**change):
    a = dict(table=P, entries=6, refs=P, k=P, v=P, layers=1, layer_bytes=0, n_pages=9, page=16, row_bytes=64, new_table=P, new_refs=P, where=P,
             live=P, ws=P, ws_bytes=1 << 20, stream=None)
    a.update(change)
    return _abi.load().aq_compact_pages(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(entries=-1), -2), (dict(layers=-1), -2), (dict(layers=2), -2), (dict(n_pages=-4), -2), (dict(page=-1), -2), (dict(row_bytes=8), -4),
    (dict(table=None), -1), (dict(refs=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(new_table=None), -1), (dict(new_refs=None), -1),
    (dict(where=None), -1), (dict(live=None), -1), (dict(ws=None), -1), (dict(where=P + 4), -4), (dict(refs=P + 4), -4), (dict(live=P + 2), -4), (dict(ws_bytes=99), -5),
    (dict(layers=1 << 17), -6),
])
def test_compaction_is_refused_before_any_launch(change, code):
    assert _compact(**change) == code


def test_sizes_of_workspaces():
    lib = _abi.load()
    assert lib.aq_fork_pages_workspace_bytes(0, 4) == 0 and lib.aq_fork_pages_workspace_bytes(5, -1) == 0
    assert lib.aq_compact_pages_workspace_bytes(-1) == 0
    size = lib.aq_paged_attn_decode_shared_workspace_bytes
    assert size(0, 4, 2, 64, 100, 64) == 0 and size(2, 5, 2, 64, 100, 64) == 0 and size(2, 4, 2, 64, 0, 0) == 0
    for total, shared in ((100, 0), (100, 64), (3000, 0), (3000, 63)):  # nothing to gain: the decode kernel's
        assert size(2, 4, 2, 64, total, shared) == lib.aq_paged_attn_decode_workspace_bytes(2, 4, 2, total)
    # 256 compute units where there is no device: 23 slices of 128 positions of the first 2944, whole blocks of 64, and a tail a sequence
    assert size(2, 4, 2, 64, 3000, 2990) == 4 * (23 * 2 * 68 * 32 + 2 * 2 * 68 * 2)


def test_positions_that_are_read_once():
    f = _abi.load().aq_paged_attn_decode_shared_positions
    assert f(0, 4, 2, 64, 3000, 2990) == 0 and f(2, 5, 2, 64, 3000, 2990) == 0 and f(2, 10, 2, 64, 3000, 2990) == 0 and f(2, 4, 2, 96, 3000, 2990) == 0 and f(2, 4, 2, 64, 3000, -1) == 0
    assert f(2, 4, 2, 64, 3000, 2990) == 2944 and f(2, 4, 2, 64, 3000, 1 << 40) == 2944 and f(1, 4, 2, 64, 3000, 2990) == 0
    assert f(2, 4, 2, 64, 100, 64) == 0 and f(2, 4, 2, 64, 3000, 63) == 0
    assert ops.paged_attn_shared_positions(2, 4, 2, 64, 3000, 2990) == 2944


def test_cpu_tensors_are_refused():
    cache = PagedKV(8, 16, 2, 64, "cpu", torch.bfloat16).bind(torch.arange(8).view(2, 4), 40)
    with pytest.raises(RuntimeError, match="GPU only"):
        cache.fork(torch.zeros(8, dtype=torch.int32), torch.tensor([0]))
    with pytest.raises(RuntimeError, match="GPU only"):
        cache.compact(torch.zeros(8, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.paged_attn_decode_shared(torch.zeros(2, 2, 64, dtype=torch.bfloat16), cache.k, cache.v, cache.page_table, 40, 16)
    unbound = PagedKV(8, 16, 2, 64, "cpu", torch.bfloat16)
    for call in (lambda: unbound.fork(torch.zeros(8, dtype=torch.int32), torch.tensor([0])), lambda: unbound.compact(torch.zeros(8, dtype=torch.int32))):
        with pytest.raises(ValueError, match="page table"):
            call()


def test_a_cache_finds_what_its_rows_share():
    cache = PagedKV(40, 16, 2, 64, "cpu", torch.bfloat16)
    table = torch.tensor([[5, 6, 7, 1], [5, 6, 8, 1], [5, 6, 9, 1]])  # the last column is the same again, behind one that is not
    assert cache.bind(table, 60).shared_len == 0                     # not asked for
    assert cache.bind(table, 60, share_prefix=True).shared_len == 32
    assert cache.bind(table, 20, share_prefix=True).shared_len == 19  # the new token's position is not shared
    assert cache.bind(table, 0, share_prefix=True).shared_len == 0
    assert cache.bind(table, 60).shared_len == 0                     # holds until the next bind
    table[1, 0] = 4
    assert cache.bind(table, 60, share_prefix=True, refresh=True).shared_len == 0
    assert cache.bind(table[:1], 60, share_prefix=True).shared_len == 0  # one sequence
    assert cache.bind(torch.full((2, 3), -1), 40, share_prefix=True).shared_len == 0
    table = torch.tensor([[5, -1, -1], [5, -1, -1]])  # pages that are still to come are not shared
    assert cache.bind(table, 40, share_prefix=True).shared_len == 16
    table[0, 1], table[1, 1] = 7, 8
    assert cache.bind(table, 40, share_prefix=True).shared_len == 16


def _model(**options):
    torch.manual_seed(0)
    m = AutoRegressiveLM(LMConfig(vocab_size=97, dim=512, n_layers=2, n_heads=8, n_kv_heads=2, dim_ffn=704, max_len=2304, **options)).to("cuda", torch.bfloat16).eval()
    quantize_model(m)
    fuse_shared_inputs(m, norms=True, decode_attention=True, residuals=True)
    return m


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"use_qk_norm": True}, {"use_gated_attention": True}])
@pytest.mark.parametrize("mixed", [False, True])
def test_samples_of_a_prompt(options, mixed, monkeypatch):
    """A prompt, forked into samples; steps over the shared pages; samples dropped and forked again; the cache compacted; steps again.
    Every attention that the model runs is checked against 64 bits on the tensors it was given.  (The logits are not compared with those of
    unshared sequences: int8 codes that fall the other way grow through the layers.)  What is exact: the first layer's keys and values
    depend on the tokens alone, and samples that were given the same tokens so far have the same logits, bit for bit."""
    page, prompt, full = 16, 2100, 131  # the last of the prompt's 132 pages is begun
    m = _model(**options)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 97, (1, prompt), generator=g).cuda()
    cache, plain = m.new_cache(800, page), m.new_cache(800, page)
    run, calls = ops.paged_attn_decode_shared, []

    def checked(q, k, v, table, total, shared, seq_lens=None):
        got = run(q, k, v, table, total, shared, seq_lens=seq_lens)
        assert ops.paged_attn_shared_workspace_bytes(*q.shape[:2], k.shape[2], 64, total, shared, "cuda") != \
            ops.paged_attn_workspace_bytes(*q.shape[:2], k.shape[2], total)  # read once, not the decode kernel
        assert shared == full * page and (seq_lens is not None) == mixed
        want, tol = _expected(q, k, v, table, total, None if seq_lens is None else seq_lens.cpu())
        _check(got, want, tol)
        calls.append(total)
        return got

    monkeypatch.setattr(ops, "paged_attn_decode_shared", checked)

    def step(tokens, table, total, lens, alone):
        tokens = tokens.cuda().view(-1, 1)
        outs = []
        for c, t, share in ((cache, table, True), (plain, alone, False)):
            c.bind(t, total, share_prefix=share)
            where = dict(start_pos=total - 1) if lens is None else dict(position_ids=(lens - 1).view(-1, 1))
            with torch.inference_mode():
                outs.append(m(tokens, paged_cache=c, **where)["logits"])
        for a, b in ((cache.k_layers, plain.k_layers), (cache.v_layers, plain.v_layers)):
            at = (total - 1) // page, (total - 1) % page
            assert torch.equal(a[0, table[:, at[0]], at[1]], b[0, alone[:, at[0]], at[1]])
        return outs[0]

    def copied(table, n):  # rows with pages of their own, holding what the shared ones hold
        own = torch.randperm(800, generator=g)[:table.shape[0] * n].view(-1, n).cuda()
        plain.k_layers[:, own], plain.v_layers[:, own] = cache.k_layers[:, table[:, :n]], cache.v_layers[:, table[:, :n]]
        return own.contiguous()

    table = torch.full((1, full + 2), -1, dtype=torch.int64, device="cuda")
    table[0, :full + 1] = torch.randperm(800, generator=g)[:full + 1].cuda()
    refs = torch.zeros(800, dtype=torch.int32, device="cuda")
    refs[table[0, :full + 1]] = 1
    with torch.inference_mode():
        m(ids, paged_cache=cache.bind(table[:, :full + 1].contiguous(), prompt), start_pos=0)
    cache.bind(table, prompt)
    forked = cache.fork(refs, torch.zeros(5, dtype=torch.int64, device="cuda"))  # five samples
    assert forked.missing.item() == 0 and forked.refs.sum().item() == 5 * (full + 1)
    table, refs, total = forked.page_table, forked.refs, prompt
    alone = copied(table, full + 1)
    lens = torch.tensor([prompt] * 5, device="cuda") if mixed else None
    for _ in range(4):
        total += 1
        if lens is not None:
            lens = lens + 1
        tokens = torch.randint(0, 97, (5,), generator=g)
        tokens[4] = tokens[0]
        logits = step(tokens, table, total, lens, alone)
        assert torch.equal(logits[4], logits[0]) and not torch.equal(logits[1], logits[0])
    cache.bind(table, total)
    parents = torch.tensor([3, 1, 3, 3], device="cuda")  # two go on, one of them three times
    forked = cache.fork(refs, parents)
    assert forked.missing.item() == 0 and forked.refs.sum().item() == 4 * (full + 1)
    cache.bind(forked.page_table, total)
    packed = cache.compact(forked.refs)
    table = packed.page_table
    assert packed.live.item() == full + 4 and int(table.max()) == full + 3
    alone = copied(table, full + 1)
    lens = lens[parents] if mixed else None
    for _ in range(3):
        total += 1
        if lens is not None:
            lens = lens + 1
        tokens = torch.randint(0, 97, (4,), generator=g)
        tokens[3] = tokens[0]
        logits = step(tokens, table, total, lens, alone)
        assert torch.equal(logits[3], logits[0]) and not torch.equal(logits[1], logits[0])
    assert calls == [t for t in range(2101, 2108) for _ in range(2)]


@pytest.mark.gpu
@pytest.mark.parametrize("options", [{}, {"use_qk_norm": True}])
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("batch", [3, 40])
def test_native_blocks_share_too(options, mixed, batch, monkeypatch):
    """A step with the blocks queued natively, and operator by operator: the same bits, in the logits and in the cache."""
    m = _model(**options)
    g = torch.Generator().manual_seed(5)
    cache = m.new_cache(140 + batch, 16)
    for c in (cache.k_layers, cache.v_layers):
        c.copy_(torch.randn(c.shape, generator=g))
    table = torch.cat([torch.arange(131).expand(batch, -1), 131 + torch.arange(batch)[:, None]], 1).cuda()
    total = 2101
    lens = torch.randint(1500, total + 1, (batch,), generator=g).cuda() if mixed else None
    where = dict(start_pos=total - 1) if lens is None else dict(position_ids=(lens - 1).view(-1, 1))
    tokens = torch.randint(0, 97, (batch, 1), generator=g).cuda()
    run, calls, outs, held = ops.paged_attn_decode_shared, [], [], []
    assert ops.paged_attn_shared_positions(batch, 8, 2, 64, total, 2096) == 2048
    for alone in (False, True):
        if alone:
            monkeypatch.setattr(ops, "paged_attn_decode_shared", lambda *a, **k: (calls.append(a[5]), run(*a, **k))[1])
        cache.bind(table, total, share_prefix=True)
        assert cache.shared_len == 2096
        with torch.inference_mode():
            outs.append(m(tokens, paged_cache=cache, **where)["logits"])
        held.append((cache.k_layers.clone(), cache.v_layers.clone()))
    assert calls == [2096, 2096]
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(held[0][0], held[1][0]) and torch.equal(held[0][1], held[1][1])


@pytest.mark.gpu
def test_a_prefix_that_gains_nothing_is_read_as_ever():
    m = _model()
    g = torch.Generator().manual_seed(6)
    cache = m.new_cache(40, 16)
    for c in (cache.k_layers, cache.v_layers):
        c.copy_(torch.randn(c.shape, generator=g))
    table = torch.cat([torch.arange(10).expand(2, -1), 10 + torch.arange(2)[:, None]], 1).cuda()
    assert ops.paged_attn_shared_positions(2, 8, 2, 64, 165, 160) == 0
    outs = []
    for share in (False, True):
        cache.bind(table, 165, share_prefix=share)
        assert cache.shared_len == (160 if share else 0)
        with torch.inference_mode():
            outs.append(m(torch.tensor([[3], [5]]).cuda(), paged_cache=cache, start_pos=164)["logits"])
    assert torch.equal(outs[0], outs[1])


@pytest.mark.gpu
def test_a_captured_step():
    """A step of the model over a shared prefix in a graph, replayed on new tokens and new pages, with eager steps between."""
    m = _model()
    g = torch.Generator().manual_seed(7)
    cache = m.new_cache(160, 16)
    table = torch.cat([torch.arange(131).expand(6, -1), 131 + torch.arange(6)[:, None]], 1).cuda()
    cache.bind(table, 2101, share_prefix=True)
    assert ops.paged_attn_shared_positions(6, 8, 2, 64, 2101, cache.shared_len) == 2048
    fills = [torch.randn(cache.k_layers.shape, generator=g) for _ in range(3)]
    tokens = [torch.randint(0, 97, (6, 1), generator=g).cuda() for _ in range(3)]
    held = tokens[0].clone()

    def fill(i):
        cache.k_layers.copy_(fills[i])
        cache.v_layers.copy_(fills[(i + 1) % 3])

    def step(t):
        with torch.inference_mode():
            return m(t, paged_cache=cache, start_pos=2100)["logits"]

    want = []
    for i in range(3):
        fill(i)
        want.append(step(tokens[i]).clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for turn in range(5):
        i = turn % 3
        fill(i)
        held.copy_(tokens[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), turn
        fill((i + 1) % 3)
        assert torch.equal(step(tokens[(i + 1) % 3]), want[(i + 1) % 3]), turn
