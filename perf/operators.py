"""Operators of a serving program around the paged decode: what is timed.

Four families:

  prefix   decode attention of a batch whose sequences share long prefixes,
           each read once for all of its sequences
           (`pa_decode_shared_prefix`)
  copy     pages of a cache copied in every layer (`copy_cache_pages`)
  branch   sequences forked off others, grown by their next tokens -- which
           copies the partial page a fork shares -- and freed again
           (`fork_cache_pages`, `extend_cache_pages`, `free_cache_pages`)
  compact  the live pages of a cache moved to its front
           (`compact_cache_pages`)

With ``own`` false, `run` computes the plain forms: elementary torch
operations, attention in 32 bits.  Lengths, tables and page numbers belong to
the case (drawn from its `lengths` seed); the seed of `prepare` gives the
values.
"""

import math

import numpy as np
import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
DEV = "cuda"


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------


def _prefix(name, groups, batch, ql, heads, kv_heads, page, prefix, suffix, *, loose=0, head=128, per_token=False,
            dtype="bf16", lengths=7):
    c = {"family": "prefix", "groups": groups, "batch": batch, "ql": ql, "heads": heads, "kv_heads": kv_heads,
         "page": page, "prefix": prefix, "suffix": suffix, "loose": loose, "head": head, "per_token": per_token,
         "dtype": dtype, "lengths": lengths}
    return dict(c, name=name) if name else c


def _pages(name, family, layers, kv_heads, page, blocks, *, head=128, per_token=False, lengths=7, **more):
    c = {"family": family, "layers": layers, "kv_heads": kv_heads, "page": page, "blocks": blocks, "head": head,
         "per_token": per_token, "lengths": lengths, **more}
    return dict(c, name=name) if name else c


def listed():
    return [
        # Four samples of a short prompt: launches and host work count.
        _prefix("prefix_small", 1, 4, 1, 8, 2, 16, "fixed:500", "uniform:1:64"),
        # A serving batch of chats behind one system prompt.
        _prefix("prefix_chat", 1, 64, 1, 32, 8, 16, "fixed:2048", "uniform:16:1024"),
        # Questions about one long document.
        _prefix("prefix_document", 1, 32, 1, 32, 8, 64, "fixed:32768", "uniform:64:2048"),
        # Speculative decode (four query tokens) of several prompts' samples,
        # per-token scales; eight sequences of the batch share nothing.
        _prefix("prefix_mtp", 4, 128, 4, 64, 4, 64, "uniform:2000:12000", "uniform:4:2048", loose=8,
                per_token=True),
        # Many samples of one long prompt: rows enough to be bound by the
        # matrix products.
        _prefix("prefix_samples", 1, 256, 1, 32, 8, 16, "fixed:16383", "uniform:1:512"),
        # 64-wide heads in half precision, 1024-token pages.
        _prefix("prefix_d64", 2, 48, 1, 32, 8, 1024, "uniform:3000:9000", "uniform:1:700", head=64, dtype="f16"),
        # Two pages of a small cache, where the launch is what counts.
        _pages("copy_small", "copy", 2, 2, 16, 64, pairs=2),
        # Pages of every layer of a model, as many as a batch swaps.
        _pages("copy_large", "copy", 32, 8, 16, 4096, pairs=512),
        # Four samples start from one short prompt.
        _pages("branch_small", "branch", 2, 2, 16, 256, parents=1, children=4, ctx="fixed:300", grow=1),
        # Parallel samples of eight prompts, every layer, 64-token pages.
        _pages("branch_large", "branch", 32, 4, 64, 6144, parents=8, children=256, ctx="uniform:1000:32768", grow=4),
        # A small pool, and one of a serving cache with a third of it free.
        _pages("compact_small", "compact", 2, 2, 16, 256, seqs=8, fill=0.6),
        _pages("compact_large", "compact", 8, 8, 16, 16384, seqs=128, fill=0.7),
    ]


# (query heads, kv heads): the shapes of the listed cases and shards of them.
_HEADS = ((8, 2), (32, 8), (64, 8), (64, 4), (8, 1), (16, 1))
# What a drawn case may cost: rows x tokens of the prefixes (times kv heads),
# (token, kv head) pairs read, and bytes copied or held by a cache.
_MOST_ROWS = 256 * 4 * 8 * 16384
_MOST_PAIRS = 128 * 1024 * 4 + 4 * 7000 * 4
_MOST_COPY = 400 << 20
_MOST_CACHE = 4 << 30


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _page_bytes(kv_heads, page, head, per_token):
    """Bytes of one page in one layer (keys, values, their scales)."""
    return kv_heads * page * (2 * head + (8 if per_token else 0))


def draw(rng):
    family = rng.choice(("prefix",) * 6 + ("copy", "branch", "branch", "compact"))
    lengths = rng.randrange(1, 1 << 30)
    if family == "prefix":
        heads, kv_heads = rng.choice(_HEADS)
        ql = rng.choice((1, 1, 1, 2, 4))
        batch = _log_int(rng, 2, 256)
        loose = rng.choice((0, 0, batch // 8))
        groups = max(1, min(batch - loose, _log_int(rng, 1, 8)))
        head = rng.choice((128,) * 5 + (64, 256))
        page = rng.choice((16, 16, 64, 1024))
        top = min(32768, _MOST_ROWS * 128 // head // (batch * ql * heads), _MOST_PAIRS * 64 // head // kv_heads // groups)
        top = _log_int(rng, 64, max(65, top))
        prefix = rng.choice(("fixed:%d" % top, "uniform:%d:%d" % (max(1, top // 4), top)))
        most = max(ql + 1, min(4096, _MOST_PAIRS * 64 // head // kv_heads // batch))
        suffix = "uniform:%d:%d" % (ql, _log_int(rng, ql + 1, most + 1))
        return _prefix(None, groups, batch, ql, heads, kv_heads, page, prefix, suffix, loose=loose, head=head,
                       per_token=rng.random() < 0.4, dtype=rng.choice(("bf16", "bf16", "f16")), lengths=lengths)
    kv_heads = rng.choice((1, 2, 4, 8))
    page = rng.choice((16, 16, 64, 1024))
    head = rng.choice((128, 128, 64))
    per_token = rng.random() < 0.4
    layers = _log_int(rng, 1, 40)
    one = _page_bytes(kv_heads, page, head, per_token) * layers
    while one > (64 << 20):
        layers = (layers + 1) // 2
        one = _page_bytes(kv_heads, page, head, per_token) * layers
    room = max(8, min(16384, _MOST_CACHE // one))
    if family == "copy":
        pairs = _log_int(rng, 1, max(2, min(512, room // 2, _MOST_COPY // one)))
        return _pages(None, family, layers, kv_heads, page, max(2 * pairs, _log_int(rng, 8, room)), head=head,
                      per_token=per_token, lengths=lengths, pairs=pairs)
    if family == "branch":
        children = _log_int(rng, 1, max(2, min(256, room // 8, _MOST_COPY // one)))
        parents = _log_int(rng, 1, max(1, min(8, children)))
        grow = rng.choice((1, 1, 4, page + 3))
        more = children * (2 + -(-grow // page))
        most = max(1, min(32768, (room - more) // parents * page))
        top = _log_int(rng, 1, most)
        return _pages(None, family, layers, kv_heads, page, more + parents * -(-top // page), head=head,
                      per_token=per_token, lengths=lengths, parents=parents, children=children,
                      ctx="uniform:%d:%d" % (max(1, top // 4), top), grow=grow)
    blocks = _log_int(rng, 8, room)
    while blocks * one > 4 * _MOST_COPY:
        blocks = max(8, blocks // 2)
    return _pages(None, family, layers, kv_heads, page, blocks, head=head, per_token=per_token, lengths=lengths,
                  seqs=_log_int(rng, 1, max(2, min(256, blocks // 4))), fill=rng.uniform(0.3, 0.95))


# ---------------------------------------------------------------------------
# Lengths and tables of a case (host)
# ---------------------------------------------------------------------------


def _sizes(spec, n, rng):
    kind, *p = spec.split(":")
    if kind == "fixed":
        return [int(p[0])] * n
    return [int(x) for x in rng.integers(int(p[0]), int(p[1]) + 1, size=n)]


def _batch(case):
    """(groups' first sequences and end, prefix lengths, context lengths) of a
    prefix case; sequences behind the last group share nothing."""
    rng = np.random.default_rng(case["lengths"])
    grouped = case["batch"] - case["loose"]
    cuts = sorted(rng.choice(np.arange(1, grouped), size=case["groups"] - 1, replace=False)) if grouped > 1 else []
    indptr = [0] + [int(x) for x in cuts] + [grouped]
    prefix = _sizes(case["prefix"], len(indptr) - 1, rng)
    suffix = _sizes(case["suffix"], case["batch"], rng)
    ctx = []
    for g, p in enumerate(prefix):
        ctx += [p + s for s in suffix[indptr[g]:indptr[g + 1]]]
    return indptr, prefix, ctx + suffix[grouped:]


def _batch_tables(case):
    """Block tables of a prefix case: a group's full prefix pages are the same
    in every row; the page its prefix ends in is each row's own, a copy of the
    first row's.  Returns (tables, pages, copies [(from, to)])."""
    indptr, prefix, ctx = _batch(case)
    page = case["page"]
    rng = np.random.default_rng(case["lengths"] + 1)
    rows, copies, n = [], [], 0
    for g in range(len(prefix) + 1):
        b0, b1 = (indptr[g], indptr[g + 1]) if g < len(prefix) else (indptr[-1], case["batch"])
        full, part = divmod(prefix[g], page) if g < len(prefix) else (0, 0)
        shared = list(range(n, n + full))
        n += full
        for b in range(b0, b1):
            more = -(-ctx[b] // page) - full
            rows.append(shared + list(range(n, n + more)))
            if part and b > b0:
                copies.append((rows[b0][full], n))
            n += more
    names = rng.permutation(n)
    table = np.zeros((case["batch"], max(len(r) for r in rows)), dtype=np.int32)
    for b, r in enumerate(rows):
        table[b, :len(r)] = names[r]
    return table, n, [(int(names[a]), int(names[b])) for a, b in copies]


def _pool(case):
    """(tables, context lengths, reference counts) of a branch or compact case."""
    rng = np.random.default_rng(case["lengths"])
    page, blocks = case["page"], case["blocks"]
    names = rng.permutation(blocks)
    if case["family"] == "branch":
        ctx = _sizes(case["ctx"], case["parents"], rng)
        total = case["parents"] + case["children"]
        width = max(-(-(c + case["grow"]) // page) for c in ctx)
    else:
        total = case["seqs"]
        live = max(total, min(blocks, int(blocks * case["fill"])))
        cuts = np.sort(rng.choice(np.arange(1, live), size=total - 1, replace=False)) if total > 1 else []
        per = np.diff(np.concatenate([[0], cuts, [live]])).astype(int)
        ctx = [int((k - 1) * page + rng.integers(1, page + 1)) for k in per]
        width = int(max(per)) + 1
    table = np.zeros((total, width), dtype=np.int32)
    refs = np.zeros(blocks, dtype=np.int32)
    n = 0
    for s, c in enumerate(ctx):
        k = -(-c // page)
        table[s, :k] = names[n:n + k]
        refs[names[n:n + k]] = 1
        n += k
    return table, ctx + [0] * (total - len(ctx)), refs


def _forks(case):
    """(parents, children) of a branch case."""
    rng = np.random.default_rng(case["lengths"] + 2)
    p = np.concatenate([np.arange(case["parents"]), rng.integers(0, case["parents"], case["children"])])
    return p[:case["children"]], case["parents"] + rng.permutation(case["children"])


def _copied(case):
    """Pages that one pass of a copy, branch or compact case copies."""
    if case["family"] == "copy":
        return case["pairs"]
    table, ctx, refs = _pool(case)
    if case["family"] == "branch":  # the parents keep the page they share
        return sum(1 for p in _forks(case)[0] if ctx[p] % case["page"])
    live = int((refs > 0).sum())
    return int((refs[live:] > 0).sum())


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _quantised(shape, gen, per_token):
    """fp8 rows [..., D] of normal values and their float32 scales."""
    x = torch.randn(shape, generator=gen, device=DEV)
    amax = x.abs().amax(dim=-1, keepdim=True) if per_token else x.abs().amax().reshape(1)
    scale = amax / FP8_MAX
    return (x / scale).to(FP8).view(torch.uint8), scale.contiguous()


def _bytes(shape, gen):
    """fp8 values of every exponent, no NaN."""
    x = torch.randint(0, 127, shape, generator=gen, device=DEV, dtype=torch.uint8)
    return x.add_(torch.randint(0, 2, shape, generator=gen, device=DEV, dtype=torch.uint8).mul_(128)).view(FP8)


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def _prepare_prefix(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    indptr, prefix, ctx = _batch(case)
    table, pages, copies = _batch_tables(case)
    h, bs, d = case["kv_heads"], case["page"], case["head"]
    dt = torch.float16 if case["dtype"] == "f16" else torch.bfloat16
    q = torch.randn(case["batch"] * case["ql"], case["heads"], d, generator=gen, device=DEV).to(dt)
    k, ks = _quantised((pages, h, bs, d), gen, case["per_token"])
    v, vs = _quantised((pages, h, bs, d), gen, case["per_token"])
    kc = k.view(pages, h, bs, d // 16, 16).permute(0, 1, 3, 2, 4).contiguous()
    vc = v.view(pages, h, bs // 16, 16, d).permute(0, 1, 2, 4, 3).contiguous()
    del k, v
    if copies:
        a = torch.tensor(copies, device=DEV)
        for t in (kc, vc) + ((ks, vs) if case["per_token"] else ()):
            t[a[:, 1]] = t[a[:, 0]]
    return {"case": case, "indptr": indptr, "prefix": prefix, "ctx": ctx, "query": q, "out": torch.empty_like(q),
            "key_cache": kc.view(FP8), "value_cache": vc.view(FP8), "key_scale": ks, "value_scale": vs,
            "tables": _ints(table), "lengths": _ints(ctx), "prefix_indptr": _ints(indptr),
            "prefix_lengths": _ints(prefix), "scale": 1.0 / math.sqrt(d)}


def _stores(case, gen):
    """The caches of all layers: keys and values (and their scales), each one
    allocation [layers, pages, ...]."""
    n, nb, h, bs, d = case["layers"], case["blocks"], case["kv_heads"], case["page"], case["head"]
    out = [_bytes((n, nb, h, d // 16, bs, 16), gen), _bytes((n, nb, h, bs // 16, d, 16), gen)]
    if case["per_token"]:
        out += [torch.rand((n, nb, h, bs, 1), generator=gen, device=DEV) for _ in range(2)]
    return out


def prepare(case, seed):
    if case["family"] == "prefix":
        return _prepare_prefix(case, seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    stores = _stores(case, gen)
    st = {"case": case, "stores": stores, "caches": [s[i] for i in range(case["layers"]) for s in stores]}
    if case["family"] == "copy":
        p = np.random.default_rng(case["lengths"]).permutation(case["blocks"])
        n = case["pairs"]
        return dict(st, source=_ints(p[:n]), target=_ints(p[n:2 * n]))
    table, ctx, refs = _pool(case)
    st.update(tables=_ints(table), lengths=_ints(ctx), refs=_ints(refs))
    if case["family"] == "branch":
        parents, children = _forks(case)
        st.update(parents=_ints(parents), children=_ints(children),
                  grown=_ints([ctx[p] + case["grow"] for p in parents]))
    return st


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------


def _rows(cache, scale, pages, values):
    """Dequantised rows [..., H, tokens, D] of the pages [..., n], float32."""
    x = cache.view(torch.uint8)[pages].view(FP8).float()
    lead, n = pages.shape[:-1], pages.shape[-1]
    if values:  # [..., n, H, bs/16, D, 16]
        h, nb, d = x.shape[-4], x.shape[-3], x.shape[-2]
        x = x.movedim(-5, -4).transpose(-1, -2).reshape(*lead, h, n * nb * 16, d)
    else:  # [..., n, H, D/16, bs, 16]
        h, nc, bs = x.shape[-4], x.shape[-3], x.shape[-2]
        x = x.movedim(-5, -4).transpose(-3, -2).reshape(*lead, h, n * bs, nc * 16)
    if scale.dim() > 1:
        s = scale[pages].movedim(-4, -3).reshape(*lead, h, -1, 1)
        return x * s
    return x * scale


def _part(q, k, v, seen, scale):
    """Softmax attention over one part of the tokens: (maximum, sum, output)
    of rows q [..., R, D]; seen [..., R, T] says which tokens a row sees."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.clamp_min(-3.0e38))
    return m, p.sum(-1, keepdim=True), torch.matmul(p, v)


def _plain_prefix(st):
    c = st["case"]
    ql, h, page, d = c["ql"], c["kv_heads"], c["page"], c["head"]
    gqa = c["heads"] // h
    q = st["query"].float().view(c["batch"], ql, h, gqa, d).permute(0, 2, 1, 3, 4).reshape(c["batch"], h, ql * gqa, d)
    out = torch.empty_like(q)
    step = torch.arange(ql, device=DEV).repeat_interleave(gqa)
    tables = st["tables"].long()
    for g in range(len(st["prefix"]) + 1):
        b0, b1 = (st["indptr"][g], st["indptr"][g + 1]) if g < len(st["prefix"]) else (st["indptr"][-1], c["batch"])
        if b0 == b1:
            continue
        P = st["prefix"][g] if g < len(st["prefix"]) else 0
        n, R = b1 - b0, ql * gqa
        limit = st["lengths"][b0:b1, None] - ql + 1 + step  # [n, R]
        parts = []
        if P:
            pages = tables[b0, :-(-P // page)]
            k = _rows(st["key_cache"], st["key_scale"], pages, False)[:, :P]
            v = _rows(st["value_cache"], st["value_scale"], pages, True)[:, :P]
            rows = q[b0:b1].transpose(0, 1).reshape(h, n * R, d)
            seen = torch.arange(P, device=DEV) < limit.reshape(n * R, 1)
            parts = [x.view(h, n, R, -1).transpose(0, 1) for x in _part(rows, k, v, seen, st["scale"])]
        first, last = P // page, -(-max(st["ctx"][b0:b1]) // page)
        at = torch.arange(first * page, last * page, device=DEV)
        seqs = max(1, (1 << 28) // max(1, (last - first) * page * h * d))
        for s0 in range(b0, b1, seqs):
            s1 = min(b1, s0 + seqs)
            pages = tables[s0:s1, first:last]
            lim = limit[s0 - b0:s1 - b0, None, :, None]
            k = _rows(st["key_cache"], st["key_scale"], pages, False)
            v = _rows(st["value_cache"], st["value_scale"], pages, True)
            m, l, o = _part(q[s0:s1], k, v, (at >= P) & (at < lim), st["scale"])
            if P:
                m0, l0, o0 = (x[s0 - b0:s1 - b0] for x in parts)
                top = torch.maximum(m, m0).clamp_min(-3.0e38)
                w, w0 = torch.exp(m - top), torch.exp(m0 - top)
                l, o = l * w + l0 * w0, o * w + o0 * w0
            out[s0:s1] = o / l
    return out.view(c["batch"], h, ql, gqa, d).permute(0, 2, 1, 3, 4).reshape(st["query"].shape).to(st["query"].dtype)


def _plain_copy(caches, source, target):
    s, t = source.long(), target.long()
    for c in caches:
        c = c.view(torch.uint8) if c.dtype == FP8 else c
        c[t] = c[s]


def _plain_fork(st):
    table, ctx, refs, page = st["tables"], st["lengths"], st["refs"], st["case"]["page"]
    p, c = st["parents"].long(), st["children"].long()
    length = ctx[p]
    use = torch.arange(table.shape[1], device=DEV) < ((length + page - 1) // page)[:, None]
    rows = torch.where(use, table[p], table[c])
    table[c] = rows
    refs.scatter_add_(0, rows.reshape(-1).long(), use.reshape(-1).int())
    ctx[c] = length
    return torch.ones_like(st["parents"])


def _plain_extend(st):
    table, ctx, refs, page = st["tables"], st["lengths"], st["refs"], st["case"]["page"]
    s, new = st["children"].long(), st["grown"]
    length = ctx[s]
    last = table[s, (length // page).clamp_max(table.shape[1] - 1).long()].long()
    shared = (length % page != 0) & (new > length) & (refs[last] > 1)
    same = (last[:, None] == last) & shared[:, None] & shared
    rank = same.tril(-1).sum(1)
    copy = shared & (rank < refs[last] - 1)
    need = (new + page - 1) // page - (length + page - 1) // page + copy.int()
    end = need.cumsum(0)
    free = (refs == 0).nonzero()[:, 0].int()
    fits = end <= free.numel()
    need, copy = need * fits, copy & fits
    k = torch.arange(int(need.max()), device=DEV)
    row, k = ((k < need[:, None]).nonzero()).unbind(1)
    got = free[(end[row] - need[row] + k).long()]
    col = torch.where(copy, length // page, (length + page - 1) // page)
    table[s[row], (col[row] + k).long()] = got
    which = copy.nonzero()[:, 0]
    _plain_copy(st["caches"], last[which], table[s[which], (length[which] // page).long()])
    refs[got.long()] = 1
    refs.scatter_add_(0, last, -copy.int())
    ctx[s] = torch.where(fits, new, length)
    return fits.int()


def _plain_free(st):
    table, ctx, refs, page = st["tables"], st["lengths"], st["refs"], st["case"]["page"]
    s = st["children"].long()
    use = torch.arange(table.shape[1], device=DEV) < ((ctx[s] + page - 1) // page)[:, None]
    refs.scatter_add_(0, table[s].reshape(-1).long(), -use.reshape(-1).int())
    ctx[s] = 0
    return torch.ones_like(st["children"])


def _plain_compact(st):
    table, ctx, refs, page = st["tables"], st["lengths"], st["refs"], st["case"]["page"]
    held = refs > 0
    live = held.sum()
    at = torch.arange(refs.numel(), device=DEV)
    source = (held & (at >= live)).nonzero()[:, 0]
    target = (~held & (at < live)).nonzero()[:, 0]
    where = torch.where(held, at, -1).int()
    where[source] = target.int()
    counts = refs * (at < live)
    counts[target] = refs[source]
    use = torch.arange(table.shape[1], device=DEV) < ((ctx + page - 1) // page)[:, None]
    tables = torch.where(use, where[table.long()], table)
    _plain_copy(st["caches"], source, target)
    return tables, counts, where, live.reshape(1).int()


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def run(st):
    case = st["case"]
    family, page = case["family"], case["page"]
    if not own:
        if family == "prefix":
            return _plain_prefix(st)
        if family == "copy":
            _plain_copy(st["caches"], st["source"], st["target"])
            return st["stores"]
        if family == "compact":
            return list(_plain_compact(st)) + st["stores"]
        did = [_plain_fork(st), _plain_extend(st), _plain_free(st)]
        return did + [st["tables"], st["lengths"], st["refs"]] + st["stores"]
    import flydsl_amd as fa

    if family == "prefix":
        fa.pa_decode_shared_prefix(st["out"], st["query"], st["key_cache"], st["value_cache"], st["lengths"],
                                   st["tables"], st["prefix_indptr"], st["prefix_lengths"], st["scale"],
                                   st["key_scale"], st["value_scale"])
        return st["out"]
    if family == "copy":
        fa.copy_cache_pages(st["caches"], st["source"], st["target"])
        return st["stores"]
    if family == "compact":
        return list(fa.compact_cache_pages(st["caches"], st["tables"], st["lengths"], st["refs"], page)) + st["stores"]
    did = [
        fa.fork_cache_pages(st["tables"], st["lengths"], st["refs"], st["parents"], st["children"], page),
        fa.extend_cache_pages(st["caches"], st["tables"], st["lengths"], st["refs"], st["children"], st["grown"], page),
        fa.free_cache_pages(st["tables"], st["lengths"], st["refs"], st["children"], page),
    ]
    return did + [st["tables"], st["lengths"], st["refs"]] + st["stores"]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    page = case["page"]
    if case["family"] == "prefix":
        indptr, prefix, ctx = _batch(case)
        h, d = case["kv_heads"], case["head"]
        rows = case["batch"] * case["ql"] * case["heads"]
        tokens = sum(prefix) + sum(ctx) - sum(p * (indptr[g + 1] - indptr[g]) for g, p in enumerate(prefix))
        per = h * (2 * d + (8 if case["per_token"] else 0))
        return {"bytes": tokens * per + 2 * rows * d * 2, "flops": 4 * d * case["heads"] * case["ql"] * sum(ctx)}
    one = _page_bytes(case["kv_heads"], page, case["head"], case["per_token"]) * case["layers"]
    moved = 2 * _copied(case) * one
    if case["family"] == "copy":
        return {"bytes": moved + 8 * case["pairs"], "flops": 0}
    _, ctx, refs = _pool(case)
    used = lambda n: -(-n // page)
    if case["family"] == "compact":  # counts in and out, the map, the tables
        return {"bytes": moved + 12 * case["blocks"] + 8 * sum(used(c) for c in ctx), "flops": 0}
    # a row in and out and its counts for each fork, the row and its counts
    # again for each sequence freed
    forked = sum(used(ctx[p]) for p in _forks(case)[0])
    return {"bytes": moved + forked * (8 + 8 + 4 + 8), "flops": 0}


# ---------------------------------------------------------------------------
# The definition, in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    """Attention of each sequence over all of its tokens by itself, float64;
    the other families only move what they are given."""
    if case["family"] != "prefix":
        return None
    st = _prepare_prefix(case, seed)
    ql, h, bs, d = case["ql"], case["kv_heads"], case["page"], case["head"]
    gqa = case["heads"] // h
    out = torch.empty(st["query"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(st["ctx"]):
        t = torch.arange(n, device=DEV)
        pg, off = st["tables"][b].long()[t // bs], t % bs
        kc, vc = st["key_cache"].view(torch.uint8), st["value_cache"].view(torch.uint8)
        k = kc[pg, :, :, off].view(FP8).double().reshape(n, h, d)
        v = vc[pg, :, off // 16, :, off % 16].view(FP8).double()
        if case["per_token"]:
            k = k * st["key_scale"][pg, :, off].double()
            v = v * st["value_scale"][pg, :, off].double()
        else:
            k, v = k * st["key_scale"].double(), v * st["value_scale"].double()
        for i in range(ql):
            see = n - ql + i + 1
            q = st["query"][b * ql + i].double().view(h, gqa, d)
            w = torch.softmax(torch.einsum("hgd,thd->hgt", q, k[:see]) * st["scale"], dim=-1)
            out[b * ql + i] = torch.einsum("hgt,thd->hgd", w, v[:see]).reshape(case["heads"], d)
    return out
