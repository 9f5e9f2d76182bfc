"""Operators on a paged KV cache whose sequences share pages, as measurable cases: what a serving program does once one
prompt has several continuations (samples of a prompt, beams of a search, requests behind one system prompt).

* ``attn``: a decode step's attention for a batch whose sequences begin with the same pages; the shared positions are
  read and multiplied once for all of them, each sequence's own positions through its own row of the page table.
* ``fork``: the rows of a page table replaced by forks of them: a new row holds its parent's whole pages with it, and has
  a copy of the page that the parent is still writing (the first child goes on in that page itself).  Rows without a child
  are let go; the pages that nobody holds any more can be taken again.
* ``compact``: the pages that are held moved to the front of the cache, and the page table renumbered.

Caches are ``[layers, pages, page, kv_heads, head_dim]`` in bf16, page tables and lengths int64, reference counts int32.
The package is inference only: there is no backward direction.
"""
import math

import torch

own = False
DEVICE = "cuda"
MASKED = -1.0e30  # score of a position behind a sequence's length: a number, so that a sequence without any averages all


def _attn(name, batch, heads, kv_heads, head_dim, page, shared, total, mixed=False):
    return dict(name=name, kind="attn", batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, shared=shared,
                total=total, mixed=mixed)


def _fork(name, layers, kv_heads, head_dim, page, pages, batch, rows, parents, total, mixed=False):
    return dict(name=name, kind="fork", layers=layers, kv_heads=kv_heads, head_dim=head_dim, page=page, pages=pages, batch=batch,
                rows=rows, parents=parents, total=total, mixed=mixed)


def _compact(name, layers, kv_heads, head_dim, page, pages, live, batch):
    return dict(name=name, kind="compact", layers=layers, kv_heads=kv_heads, head_dim=head_dim, page=page, pages=pages, live=live, batch=batch)


def listed():
    return [
        # two samples of one prompt of the 24-layer model, 64 tokens on
        _attn("attn_2x576_of_512", 2, 24, 4, 64, 128, 512, 576),
        # eight samples of a long prompt on the 2048-wide block
        _attn("attn_8x2591_of_2048", 8, 16, 4, 128, 64, 2048, 2591),
        # requests behind one system prompt, each at its own position, small pages
        _attn("attn_33x1401_of_1008_mixed", 33, 24, 4, 64, 16, 1008, 1401, mixed=True),
        # a large batch on a long document, eight KV heads
        _attn("attn_64x8448_of_8192", 64, 32, 8, 128, 64, 8192, 8448),
        # a few questions to a very long one, just begun
        _attn("attn_16x65600_of_65536", 16, 16, 4, 128, 128, 65536, 65600),
        # many requests behind a few-shot prompt, at all lengths
        _attn("attn_256x4500_of_4096_mixed", 256, 16, 4, 128, 64, 4096, 4500, mixed=True),
        # one prompt becomes eight samples: the 24-layer model's cache, 63 tokens into a page
        _fork("fork_1_to_8", 24, 4, 64, 128, 64, 1, 8, 1, 575),
        # a step of a search over 64 beams, of which 24 go on
        _fork("fork_beams_64", 24, 4, 128, 64, 2048, 64, 64, 24, 1400),
        # a serving batch that is thinned out and filled again: small pages, every row at its own length
        _fork("fork_256_mixed", 4, 4, 64, 16, 40000, 256, 300, 180, 2040, mixed=True),
        # a block's small cache
        _compact("compact_40_of_128", 1, 4, 128, 64, 128, 40, 4),
        # the 24-layer model's cache, half full
        _compact("compact_500_of_1024", 24, 4, 64, 128, 1024, 500, 37),
        # small pages, a third of them held
        _compact("compact_20011_of_60000", 4, 4, 64, 16, 60000, 20011, 200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_attn(rng):
    heads, kv_heads, head_dim = rng.choice(((16, 4, 128), (24, 4, 64), (32, 8, 128), (16, 2, 128), (8, 8, 64), (12, 4, 64), (16, 8, 128), (6, 6, 128)))
    page = rng.choice((16, 24, 64, 128, 256))
    batch, own_tokens = _log(rng, 2, 256), _log(rng, 1, 1024)
    shared = page * max(1, _log(rng, 64, 65536) // page)
    while batch * heads * head_dim * (shared + own_tokens) * 4 > 8.6e9:
        shared, own_tokens = page * max(1, shared // 2 // page), max(1, own_tokens * 3 // 4)
    return _attn("", batch, heads, kv_heads, head_dim, page, shared, shared + own_tokens, rng.random() < 0.5)


def _draw_fork(rng):
    layers, page = _log(rng, 1, 24), rng.choice((16, 24, 64, 128))
    kv_heads, head_dim = rng.choice(((4, 64), (4, 128), (8, 128), (2, 64)))
    batch = _log(rng, 1, 256)
    rows = max(1, min(300, int(batch * rng.uniform(0.5, 2.0)) + rng.randint(0, 8)))
    parents = rng.randint(1, min(batch, rows))
    total = _log(rng, 1, 2048)
    need = -(-total // page) * batch + rows + 8
    while layers > 1 and layers * need * page * kv_heads * head_dim * 4 > 4e9:
        layers //= 2
    pages = min(int(need * rng.uniform(1.0, 1.5)), max(need, int(4e9 / (layers * page * kv_heads * head_dim * 4))))
    return _fork("", layers, kv_heads, head_dim, page, pages, batch, rows, parents, total, rng.random() < 0.5)


def _draw_compact(rng):
    page = rng.choice((16, 24, 64, 128))
    kv_heads, head_dim = rng.choice(((4, 64), (4, 128), (8, 128), (2, 64)))
    each = page * kv_heads * head_dim * 4
    layers = _log(rng, 1, 24)
    pages = max(8, min(_log(rng, 32, 60000), int(3e9 / (layers * each))))
    return _compact("", layers, kv_heads, head_dim, page, pages, max(1, int(pages * rng.uniform(0.05, 0.95))), _log(rng, 1, 256))


def draw(rng):
    case = rng.choices((_draw_attn, _draw_fork, _draw_compact), (5, 3, 2))[0](rng)
    del case["name"]
    return case


# ---- what is in hand before the call -----------------------------------------------------------------------------

def _caches(gen, *shape):
    return tuple(torch.empty(*shape, device=DEVICE, dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))


def _prepare_attn(case, gen):
    batch, page, total = case["batch"], case["page"], case["total"]
    common = case["shared"] // page
    mine = -(-total // page) - common
    pages = common + batch * mine
    ids = torch.randperm(pages, generator=gen, device=DEVICE)  # as a pool that has been in use hands them out
    table = torch.cat([ids[:common].expand(batch, -1), ids[common:].view(batch, mine)], 1).contiguous()
    k, v = _caches(gen, pages, page, case["kv_heads"], case["head_dim"])
    # as trained models have them: a loud channel, and a first token that many heads look at
    k[..., 3] *= 4.0
    q = torch.randn(batch, case["heads"], case["head_dim"], generator=gen, device=DEVICE)
    first = k[table[0, 0], 0].float().repeat_interleave(case["heads"] // case["kv_heads"], 0)
    q = (q + first * 0.3 * torch.rand(batch, case["heads"], 1, generator=gen, device=DEVICE)).to(torch.bfloat16)
    lens = None
    if case["mixed"]:
        lens = torch.randint(case["shared"] + 1, total + 1, (batch,), generator=gen, device=DEVICE)
        lens[0] = total
    return {"kind": "attn", "q": q, "k": k, "v": v, "table": table, "total": total, "shared": case["shared"], "lens": lens}


def _prepare_fork(case, gen):
    batch, page, total, pages = case["batch"], case["page"], case["total"], case["pages"]
    columns = -(-total // page)
    common = columns // 2
    ids = torch.randperm(pages, generator=gen, device=DEVICE)
    held = common + batch * (columns - common)
    table = torch.full((batch, columns + 1), -1, device=DEVICE, dtype=torch.int64)  # a column for the tokens to come
    table[:, :common] = ids[:common]
    table[:, common:columns] = ids[common:held].view(batch, -1)
    refs = torch.zeros(pages, device=DEVICE, dtype=torch.int32)
    refs[ids[:common]] = batch
    refs[ids[common:held]] = 1
    refs[ids[:max(1, common // 2)]] += 1  # a cache of prompts holds some of them too
    lens = torch.randint(1, total + 1, (batch,), generator=gen, device=DEVICE) if case["mixed"] else None
    chosen = torch.randperm(batch, generator=gen, device=DEVICE)[:case["parents"]]
    more = torch.randint(0, case["parents"], (case["rows"] - case["parents"],), generator=gen, device=DEVICE)
    parents = torch.cat([chosen, chosen[more]])[torch.randperm(case["rows"], generator=gen, device=DEVICE)]
    k, v = _caches(gen, case["layers"], pages, page, case["kv_heads"], case["head_dim"])
    return {"kind": "fork", "table": table, "refs": refs, "parents": parents, "k": k, "v": v, "total": total, "lens": lens}


def _prepare_compact(case, gen):
    pages, live, batch = case["pages"], case["live"], case["batch"]
    held = torch.randperm(pages, generator=gen, device=DEVICE)[:live]
    refs = torch.zeros(pages, device=DEVICE, dtype=torch.int32)
    refs[held] = torch.randint(1, 4, (live,), generator=gen, device=DEVICE, dtype=torch.int32)
    columns = -(-live // batch)
    table = torch.full((batch * columns,), -1, device=DEVICE, dtype=torch.int64)
    table[:live] = held
    k, v = _caches(gen, case["layers"], pages, case["page"], case["kv_heads"], case["head_dim"])
    return {"kind": "compact", "table": table.view(batch, columns), "refs": refs, "k": k, "v": v}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"attn": _prepare_attn, "fork": _prepare_fork, "compact": _prepare_compact}[case["kind"]](case, gen)


# ---- the call ------------------------------------------------------------------------------------------------------

def _plain_attn(s):
    q, k, v, table, total = s["q"], s["k"], s["v"], s["table"], s["total"]
    (batch, heads, dim), (_, page, kv_heads, _) = q.shape, k.shape
    group, common = heads // kv_heads, s["shared"] // page
    qs = q.float().view(batch, kv_heads, group, dim) * dim ** -0.5
    rows = qs.transpose(0, 1).reshape(kv_heads, batch * group, dim)

    def shared(c):  # [kv_heads, positions, dim]
        return c[table[0, :common]].flatten(0, 1).float().transpose(0, 1).contiguous()

    def mine(c):  # [batch, kv_heads, positions, dim]
        return c[table[:, common:]].flatten(1, 2)[:, :total - common * page].float().transpose(1, 2).contiguous()

    near = torch.matmul(rows, shared(k).transpose(1, 2).contiguous()).view(kv_heads, batch, group, -1).transpose(0, 1)
    far = torch.matmul(qs, mine(k).transpose(2, 3).contiguous())
    score = torch.cat([near, far], 3)
    if s["lens"] is not None:
        behind = torch.arange(total, device=q.device) >= s["lens"][:, None]
        score = score.masked_fill(behind[:, None, None], MASKED)
    p = torch.exp(score - score.amax(3, keepdim=True))
    p = p / p.sum(3, keepdim=True)
    split = common * page
    out = torch.matmul(p[..., :split].transpose(0, 1).reshape(kv_heads, batch * group, split), shared(v))
    out = out.view(kv_heads, batch, group, dim).transpose(0, 1) + torch.matmul(p[..., split:].contiguous(), mine(v))
    return out.reshape(batch, heads, dim).to(q.dtype)


def _counts(entries, pages):
    """How many of the entries name each page."""
    entries = entries.flatten()
    at = torch.where(entries < 0, pages, entries)
    return torch.zeros(pages + 1, device=entries.device, dtype=torch.int32).index_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:pages]


def _plain_fork(s):
    table, refs, parents, k, v = s["table"], s["refs"], s["parents"], s["k"], s["v"]
    (batch, columns), pages, page = table.shape, refs.numel(), k.shape[2]
    known = (parents >= 0) & (parents < batch)
    at = parents.clamp(0, batch - 1)
    first = known & ~(parents[:, None] == parents[None, :]).tril(-1).any(1)
    entries = torch.where((table >= 0) & (table < pages), table, -1)
    length = torch.full_like(parents, s["total"]) if s["lens"] is None else s["lens"].clamp(0, s["total"])[at]
    whole, rest = length // page, length % page
    rows = entries[at]
    keep = first[:, None] | (torch.arange(columns, device=table.device) < whole[:, None])
    new = torch.where(keep & known[:, None], rows, -1)
    counts = (refs - _counts(entries, pages)).clamp(min=0) + _counts(new, pages)
    source = rows.gather(1, whole.clamp(max=columns - 1)[:, None])[:, 0]
    wants = known & ~first & (rest > 0) & (whole < columns) & (source >= 0)
    rank = wants.cumsum(0) - 1
    free = (counts == 0).nonzero()[:, 0]
    row = (wants & (rank < free.numel())).nonzero()[:, 0]
    fresh = free[rank[row]]
    new[row, whole[row]] = fresh
    counts[fresh] = 1
    written = (torch.arange(page, device=table.device) < rest[row, None])[None, :, :, None, None]
    k[:, fresh] = torch.where(written, k[:, source[row]], k[:, fresh])
    v[:, fresh] = torch.where(written, v[:, source[row]], v[:, fresh])
    return new, counts, (wants.sum(dtype=torch.int32) - row.numel()).view(1), k, v


def _plain_compact(s):
    table, refs, k, v = s["table"], s["refs"], s["k"], s["v"]
    pages = refs.numel()
    held = refs > 0
    live = held.sum()
    ids = torch.arange(pages, device=refs.device)
    to = (~held & (ids < live)).nonzero()[:, 0]
    source = (held & (ids >= live)).nonzero()[:, 0].flip(0)  # the last page held goes into the first hole
    where = torch.where(held, ids, -1)
    where[source] = to
    counts = torch.where(ids < live, refs, 0)
    counts[to] = refs[source]
    k[:, to] = k[:, source]
    v[:, to] = v[:, source]
    new = torch.where((table >= 0) & (table < pages), where[table.clamp(0, pages - 1)], -1)
    return new, counts, where, live.to(torch.int32).view(1), k, v


def run(state):
    s = state
    if own:
        from khaosz_amd import ops

        if s["kind"] == "attn":
            return ops.paged_attn_decode_shared(s["q"], s["k"], s["v"], s["table"], s["total"], s["shared"], seq_lens=s["lens"])
        if s["kind"] == "fork":
            f = ops.fork_pages(s["table"], s["refs"], s["parents"], s["k"], s["v"], s["total"], seq_lens=s["lens"])
            return f.page_table, f.refs, f.missing, s["k"], s["v"]
        c = ops.compact_pages(s["table"], s["refs"], s["k"], s["v"])
        return c.page_table, c.refs, c.where, c.live, s["k"], s["v"]
    return {"attn": _plain_attn, "fork": _plain_fork, "compact": _plain_compact}[s["kind"]](s)


# ---- what it cannot do without -----------------------------------------------------------------------------------

def work(case):
    token = case["kv_heads"] * case["head_dim"] * 2 * 2  # bytes of a token's key and value in one layer
    if case["kind"] == "attn":
        batch, heads, dim = case["batch"], case["heads"], case["head_dim"]
        tail = case["total"] - case["shared"]
        tail = batch * (tail if not case["mixed"] else (tail + 1) / 2)
        table = 8 * batch * -(-case["total"] // case["page"])
        return {"bytes": (case["shared"] + tail) * token + 2 * 2 * batch * heads * dim + table,
                "flops": 4.0 * heads * dim * (batch * case["shared"] + tail)}
    if case["kind"] == "fork":
        copies, rest = case["rows"] - case["parents"], case["total"] % case["page"]
        if case["mixed"]:  # lengths are spread evenly
            rest = sum(n % case["page"] for n in range(1, case["total"] + 1)) / case["total"]
        tables = 8 * (-(-case["total"] // case["page"]) + 1) * (case["batch"] + case["rows"])
        return {"bytes": 2 * copies * rest * token * case["layers"] + tables + 8 * case["pages"] + 8 * case["rows"], "flops": 0}
    moved = case["live"] * (1 - case["live"] / case["pages"])  # of pages held anywhere, those behind the last place
    tables = 16 * -(-case["live"] // case["batch"]) * case["batch"]
    return {"bytes": 2 * moved * case["page"] * token * case["layers"] + tables + 16 * case["pages"], "flops": 0}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------

def _exact_attn(s):
    q, total = s["q"].double(), s["total"]
    out = torch.empty_like(q)
    group = q.shape[1] // s["k"].shape[2]
    for b in range(q.shape[0]):
        n = total if s["lens"] is None else int(s["lens"][b])
        n = min(max(n, 0), total)
        keys, values = (c[s["table"][b]].flatten(0, 1)[:n or total].double() for c in (s["k"], s["v"]))
        for h in range(keys.shape[1]):
            heads = slice(h * group, (h + 1) * group)
            x = q[b, heads] @ keys[:, h].t() / math.sqrt(q.shape[2])
            out[b, heads] = (torch.softmax(x, 1) if n else torch.full_like(x, 1 / total)) @ values[:, h]
    return out


def _exact_fork(s):
    table, refs, parents = s["table"].tolist(), s["refs"].tolist(), s["parents"].tolist()
    page = s["k"].shape[2]
    lens = [s["total"]] * len(table) if s["lens"] is None else s["lens"].tolist()
    for row in table:
        for e in row:
            if e >= 0:
                refs[e] -= 1
    new, copies, seen = [], [], set()
    for i, p in enumerate(parents):
        whole, rest = divmod(lens[p], page)
        row = list(table[p]) if p not in seen else table[p][:whole] + [-1] * (len(table[p]) - whole)
        if p in seen and rest and table[p][whole] >= 0:
            copies.append((i, whole, rest, table[p][whole]))
        seen.add(p)
        new.append(row)
        for e in row:
            if e >= 0:
                refs[e] += 1
    free = [i for i, r in enumerate(refs) if r == 0]
    for (i, whole, rest, source), to in zip(copies, free):
        new[i][whole] = to
        refs[to] = 1
        s["k"][:, to, :rest] = s["k"][:, source, :rest]
        s["v"][:, to, :rest] = s["v"][:, source, :rest]
    missing = max(0, len(copies) - len(free))
    return (torch.tensor(new), torch.tensor(refs, dtype=torch.int32), torch.tensor([missing], dtype=torch.int32), s["k"], s["v"])


def _exact_compact(s):
    refs, table = s["refs"].tolist(), s["table"].tolist()
    where = [i if r > 0 else -1 for i, r in enumerate(refs)]
    low, high = 0, len(refs) - 1
    moves = []
    while True:  # from both ends: the first hole takes the last page held
        while low < high and refs[low] > 0:
            low += 1
        while low < high and refs[high] <= 0:
            high -= 1
        if low >= high:
            break
        moves.append((high, low))
        refs[low], refs[high], where[high] = refs[high], 0, low
    if moves:
        source, to = torch.tensor(moves, device=DEVICE).unbind(1)
        for c in (s["k"], s["v"]):
            for layer in c:
                layer[to] = layer[source]
    new = [[where[e] if e >= 0 else -1 for e in row] for row in table]
    live = sum(r > 0 for r in refs)
    return (torch.tensor(new), torch.tensor(refs, dtype=torch.int32), torch.tensor(where), torch.tensor([live], dtype=torch.int32),
            s["k"], s["v"])


def exact(case, seed):
    return {"attn": _exact_attn, "fork": _exact_fork, "compact": _exact_compact}[case["kind"]](prepare(case, seed))
