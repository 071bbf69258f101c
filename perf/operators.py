"""Workloads of the cache operators: drafted-token trees, page operations, page-selected sparse decode.

Five kinds of case, all over the paged K/V cache ``[layers, pages, 2, page_size, kv_heads, head_dim]`` in bf16:

* ``tree``: a verification step's ancestor mask, then the attention of every drafted token of every row over
  its context and its ancestors, ``layers`` layers of it.
* ``sparse``: one decode token per row over the pages that the integer bound score selects, per kv head.
* ``bounds``: the int8 bounds of pages that prefill or decode just filled, which that score reads.
* ``fork``: a branching step: losing rows give their pages back, winners fork into them (full pages shared, the
  partial last one copied in every layer), then every live row reserves its next slots.
* ``compact``: the kept tokens of every row move together in every layer; after a verified draft ("accept",
  where the longest accepted path is found first) or after an eviction that keeps scattered tokens ("evict").

With ``own`` false, :func:`run` computes them in elementary torch operations, in fp32; with ``own`` true it calls
the framework.
"""

import math

import numpy as np
import torch

own = False

INV127 = float(np.float32(1.0) / np.float32(127.0))


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One interactive sequence with a small draft: latency counts.
        dict(name="tree 1x8 ctx 600", kind="tree", rows=1, n_lo=8, n_hi=8, ctx_lo=600, ctx_hi=600, hq=32, hkv=8,
             d=128, ps=16, layers=1),
        # A ragged batch of a multi-head (no GQA) model.
        dict(name="tree 12x5-33 ctx 300-4100 mha", kind="tree", rows=12, n_lo=5, n_hi=33, ctx_lo=300, ctx_hi=4100,
             hq=32, hkv=32, d=128, ps=16, layers=2),
        # Long contexts with wide trees: the K/V of 8 x 32768 tokens, 64 drafted tokens each.
        dict(name="tree 8x64 ctx 32768", kind="tree", rows=8, n_lo=64, n_hi=64, ctx_lo=32768, ctx_hi=32768, hq=32,
             hkv=8, d=128, ps=16, layers=2),
        # One interactive sequence of a few thousand tokens.
        dict(name="sparse 1 row ctx 5003", kind="sparse", rows=1, ctx_lo=5003, ctx_hi=5003, hq=32, hkv=8, d=128,
             ps=16, select=48, sink=1, recent=4),
        # A ragged serving batch, some rows shorter than the page budget.
        dict(name="sparse 24 rows ctx 500-40000", kind="sparse", rows=24, ctx_lo=500, ctx_hi=40000, hq=32, hkv=8,
             d=128, ps=16, select=64, sink=1, recent=8),
        # Long documents: 8 x 131072 tokens, 256 pages (4096 tokens) read of each.
        dict(name="sparse 8 rows ctx 131072", kind="sparse", rows=8, ctx_lo=131072, ctx_hi=131072, hq=32, hkv=8,
             d=128, ps=16, select=256, sink=4, recent=16),
        # The pages that a decode batch of 64 rows filled in one step.
        dict(name="bounds 64 pages", kind="bounds", pages=64, hkv=8, d=128, ps=16),
        # The pages of 8 prompts of 32768 tokens, after prefill.
        dict(name="bounds 16384 pages", kind="bounds", pages=16384, hkv=8, d=128, ps=16),
        # A small beam of a small model.
        dict(name="fork 4 of 8 rows 2 layers", kind="fork", rows=8, forks=4, ctx_lo=130, ctx_hi=700, hkv=2, d=64,
             ps=16, layers=2, reserve=1),
        # A branching batch: half of 96 rows lost, the other half forks.
        dict(name="fork 48 of 96 rows 32 layers", kind="fork", rows=96, forks=48, ctx_lo=30, ctx_hi=500, hkv=8,
             d=128, ps=16, layers=32, reserve=4),
        # After one verification step of a serving batch.
        dict(name="compact accept 16x32", kind="compact", mode="accept", rows=16, n_lo=9, n_hi=32, ctx_lo=200,
             ctx_hi=900, hkv=8, d=128, ps=16, layers=32),
        # A cache eviction that keeps every second token or so of 12 contexts.
        dict(name="compact evict 12x4096", kind="compact", mode="evict", rows=12, n_lo=0, n_hi=0, ctx_lo=3800,
             ctx_hi=4096, hkv=8, d=128, ps=16, layers=16),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "sparse", "sparse", "bounds", "fork", "compact"])
    ps = rng.choice([16, 16, 32])
    d = rng.choice([128, 128, 64])
    if kind in ("tree", "sparse"):
        hq, hkv = rng.choice([(32, 8), (32, 32), (28, 4), (8, 2), (16, 1)])
    else:
        hkv = rng.choice([8, 2, 4, 1])
    if kind == "tree":
        rows = _logint(rng, 1, 24)
        n_hi = _logint(rng, 1, 64)
        # at most the largest listed case's rows x context x heads
        ctx_hi = _logint(rng, 40, max(60, min(33000, 8 * 8 * 32768 // (rows * hkv))))
        return dict(kind=kind, rows=rows, n_lo=max(1, n_hi // 3), n_hi=n_hi, ctx_lo=max(1, ctx_hi // rng.choice([1, 2, 8])),
                    ctx_hi=ctx_hi, hq=hq, hkv=hkv, d=d, ps=ps, layers=rng.choice([1, 2]))
    if kind == "sparse":
        rows = _logint(rng, 1, 48)
        ctx_hi = _logint(rng, 300, max(400, min(131072, 8 * 8 * 131072 // (rows * hkv))))
        select = _logint(rng, 12, 256)
        return dict(kind=kind, rows=rows, ctx_lo=max(1, ctx_hi // rng.choice([1, 2, 10])), ctx_hi=ctx_hi, hq=hq,
                    hkv=hkv, d=d, ps=ps, select=select, sink=rng.randint(0, 4), recent=rng.randint(1, min(8, select - 4)))
    if kind == "bounds":
        return dict(kind=kind, pages=_logint(rng, 1, 16384 * 16 // ps), hkv=hkv, d=d, ps=ps)
    if kind == "fork":
        forks = _logint(rng, 1, 48)
        return dict(kind=kind, rows=2 * forks + rng.randint(0, 9), forks=forks, ctx_lo=1, ctx_hi=_logint(rng, 20, 500),
                    hkv=hkv, d=d, ps=ps, layers=_logint(rng, 1, 32), reserve=rng.randint(1, 7))
    mode = rng.choice(["accept", "evict"])
    rows = _logint(rng, 1, 12)
    ctx_hi = _logint(rng, 20, 4096)
    n_hi = _logint(rng, 1, 48) if mode == "accept" else 0
    return dict(kind=kind, mode=mode, rows=rows, n_lo=n_hi // 3 if n_hi < 3 else 1, n_hi=n_hi, ctx_lo=max(1, ctx_hi // 2),
                ctx_hi=ctx_hi, hkv=hkv, d=d, ps=ps, layers=_logint(rng, 1, 16))


def _lengths(case, lo, hi, salt):
    """One length per row, spread over [lo, hi]: by the case alone, so that work() knows them."""

    r = np.random.RandomState(1000 * salt + case["rows"] + 7 * hi)
    out = r.randint(lo, hi + 1, case["rows"])
    out[0] = hi
    return out.astype(np.int64)


def _pages(length, ps):
    return (length + ps - 1) // ps


# ----------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _kv(g, shape):
    """Keys and values as a decoder's cache holds them: channels of unequal size, a few of them large."""

    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    ch = 0.5 + torch.rand(shape[-2:], generator=g, device="cuda")
    ch = ch * torch.where(torch.rand(shape[-2:], generator=g, device="cuda") < 0.03, 4.0, 1.0)
    return x.mul_(ch.to(torch.bfloat16))


def _i32(a):
    return torch.as_tensor(np.asarray(a, np.int32), device="cuda")


def _table(rng, lens, ps, spare):
    """Row page lists over a shuffled pool: (pool size, per-row lists, last page lengths)."""

    n = _pages(lens, ps)
    pool = int(n.sum()) + spare
    perm = rng.permutation(pool)
    at = np.concatenate([[0], np.cumsum(n)])
    rows = [perm[at[i]:at[i + 1]] for i in range(len(lens))]
    return pool, rows, at, np.where(lens > 0, lens - (n - 1) * ps, 0)


def _parents(rng, n):
    """A drafted tree in topological order: node 0 is the last sampled token, the others hang below earlier ones."""

    p = np.full(n, -1, np.int64)
    for i in range(1, n):
        p[i] = rng.randint(max(0, i - 6), i)
    return p


def prepare(case, seed):
    rng = np.random.RandomState(seed % (2**31 - 1))
    g = _gen(seed)
    kind, ps, d, hkv = case["kind"], case["ps"], case["d"], case["hkv"]
    if kind == "tree":
        n = _lengths(case, case["n_lo"], case["n_hi"], 1)
        lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 2) + n
        pool, rows, at, last = _table(rng, lens, ps, 3)
        total, layers = int(n.sum()), case["layers"]
        kv = _kv(g, (layers, pool, 2, ps, hkv, d))
        q = torch.randn(layers, total, case["hq"], d, generator=g, device="cuda", dtype=torch.bfloat16)
        return dict(kind=kind, q=q, kv=kv, parents=_i32(np.concatenate([_parents(rng, k) for k in n])),
                    qo_indptr=_i32(np.concatenate([[0], np.cumsum(n)])), kv_indptr=_i32(at),
                    kv_indices=_i32(np.concatenate(rows)), kv_last=_i32(last), words=(int(n.max()) + 31) // 32,
                    max_n=int(n.max()), max_pages=int(_pages(lens, ps).max()), out=torch.empty_like(q),
                    lse=torch.empty(layers, total, case["hq"], device="cuda"))
    if kind == "sparse":
        lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 3)
        pool, rows, at, last = _table(rng, lens, ps, 3)
        kv = _kv(g, (pool, 2, ps, hkv, d))
        q = torch.randn(case["rows"], case["hq"], d, generator=g, device="cuda", dtype=torch.bfloat16)
        bounds, scale = _bounds(kv)
        return dict(kind=kind, q=q, kv=kv, bounds=bounds, scale=scale, kv_indptr=_i32(at),
                    kv_indices=_i32(np.concatenate(rows)), kv_last=_i32(last), select=case["select"],
                    sink=case["sink"], recent=case["recent"], max_pages=int(_pages(lens, ps).max()),
                    out=torch.empty_like(q), lse=torch.empty(case["rows"], case["hq"], device="cuda"),
                    selected=torch.empty(case["rows"], hkv, case["select"], device="cuda", dtype=torch.int32))
    if kind == "bounds":
        pool = case["pages"] + 5
        return dict(kind=kind, kv=_kv(g, (pool, 2, ps, hkv, d)),
                    page_ids=_i32(rng.permutation(pool)[:case["pages"]]),
                    bounds=torch.zeros(pool, hkv, 2, d, device="cuda", dtype=torch.int8),
                    scale=torch.zeros(pool, hkv, device="cuda"))
    return _prepare_pages(case, rng, g)


def _prepare_pages(case, rng, g):
    """Rows over a reference-counted pool.  The state that the operators change (counts, tables) is one buffer,
    so that a pass begins from the same state with one copy."""

    kind, ps, R, layers = case["kind"], case["ps"], case["rows"], case["layers"]
    lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 4)
    if kind == "fork":
        n = np.zeros(R, np.int64)
        spare = case["forks"] + R * (_pages(case["reserve"], ps) + 1) + 3
        idle = R - 2 * case["forks"]  # rows that neither fork nor end
        lens[R - idle // 2:] = 0      # some of them not in use
    elif case["mode"] == "accept":
        n = _lengths(case, case["n_lo"], case["n_hi"], 5)
        spare = int(_pages(n, ps).sum()) + 2 * R + 3
    else:
        n = np.zeros(R, np.int64)
        spare = int(_pages(lens, ps).sum()) + 3
    lens = lens + n
    pool, rows, at, last = _table(rng, lens, ps, spare)
    cap = int(_pages(lens, ps).max()) + _pages(case.get("reserve", 0), ps) + 2
    table = np.zeros((R, cap), np.int64)
    for r, pg in enumerate(rows):
        table[r, :len(pg)] = pg
    count = np.zeros(pool, np.int64)
    np.add.at(count, np.concatenate(rows), 1)
    meta = _i32(np.concatenate([count, table.reshape(-1), _pages(lens, ps), last]))
    s = dict(kind=kind, pool=_kv(g, (layers, pool, 2, ps, case["hkv"], case["d"])), meta0=meta, meta=meta.clone(),
             pages=pool, rows=R, cap=cap, ps=ps)
    if kind == "fork":
        order = rng.permutation(2 * case["forks"])
        s["released"] = _i32(order[:case["forks"]])
        s["src"], s["dst"] = _i32(order[case["forks"]:][rng.randint(0, case["forks"], case["forks"])]), _i32(order[:case["forks"]])
        live = np.array([case["reserve"] if r < 2 * case["forks"] or lens[r] > 0 else 0 for r in range(R)])
        total = int(live.sum())
        s.update(tok_indptr=_i32(np.concatenate([[0], np.cumsum(live)])), total=total,
                 slot_page=torch.zeros(total, device="cuda", dtype=torch.int32),
                 slot_off=torch.zeros(total, device="cuda", dtype=torch.int32),
                 indptr=torch.zeros(R + 1, device="cuda", dtype=torch.int32),
                 indices=torch.zeros(R * cap, device="cuda", dtype=torch.int32))
    elif case["mode"] == "accept":
        par = [_parents(rng, k) for k in n]
        tok = [rng.randint(0, 32000, k) for k in n]
        tgt = [rng.randint(0, 32000, k) for k in n]
        for p, t, w in zip(par, tok, tgt):
            for i in range(1, len(p)):  # the target model agrees with most drafted tokens
                if rng.rand() < 0.7:
                    t[i] = w[p[i]]
        s.update(mode="accept", parents=_i32(np.concatenate(par)), qo_indptr=_i32(np.concatenate([[0], np.cumsum(n)])),
                 tokens=torch.as_tensor(np.concatenate(tok), device="cuda"),
                 targets=torch.as_tensor(np.concatenate(tgt), device="cuda"), max_n=int(n.max()),
                 keep_from=_i32(lens - n), keep=torch.full((R, int(n.max())), -1, device="cuda", dtype=torch.int32),
                 keep_count=torch.zeros(R, device="cuda", dtype=torch.int32),
                 next_token=torch.zeros(R, device="cuda", dtype=torch.int64))
    else:
        keep_from = np.minimum(lens, 4)
        kept = [keep_from[r] + np.flatnonzero(rng.rand(lens[r] - keep_from[r]) < 0.5) for r in range(R)]
        keep = np.full((R, max(1, max(len(k) for k in kept))), -1, np.int64)
        for r, k in enumerate(kept):
            keep[r, :len(k)] = k
        s.update(mode="evict", keep_from=_i32(keep_from), keep=_i32(keep), keep_count=_i32([len(k) for k in kept]))
    return s


def _meta(s):
    p, r, c = s["pages"], s["rows"], s["cap"]
    m = s["meta"]
    return m[:p], m[p:p + r * c].view(r, c), m[p + r * c:p + r * c + r], m[p + r * c + r:]


# -------------------------------------------------------------------- run
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from pagelora_b200 import kernels as K

    if s["kind"] == "tree":
        mask, depth = K.tree_mask(s["parents"], s["qo_indptr"], s["words"])
        for q, kv, out, lse in zip(s["q"], s["kv"], s["out"], s["lse"]):
            K.paged_tree_attention(q, kv, s["qo_indptr"], s["kv_indptr"], s["kv_indices"], s["kv_last"], mask,
                                   out=out, out_lse=lse)
        return dict(out=s["out"], lse=s["lse"], mask=mask, depth=depth)
    if s["kind"] == "sparse":
        K.paged_sparse_decode(s["q"], s["kv"], s["kv_indptr"], s["kv_indices"], s["kv_last"], s["bounds"], s["scale"],
                              num_select=s["select"], sink_pages=s["sink"], recent_pages=s["recent"],
                              max_pages=s["max_pages"], out=s["out"], out_lse=s["lse"], selected=s["selected"])
        return dict(out=s["out"], lse=s["lse"], selected=s["selected"])
    if s["kind"] == "bounds":
        K.page_bounds(s["kv"], s["page_ids"], s["bounds"], s["scale"])
        return dict(bounds=s["bounds"], scale=s["scale"])
    s["meta"].copy_(s["meta0"])
    count, table, num, last = _meta(s)
    got = dict(pool=s["pool"].view(torch.int16), meta=s["meta"])
    if s["kind"] == "fork":
        K.page_release(count, table, num, last, s["released"])
        K.page_fork(s["pool"], count, table, num, last, s["src"], s["dst"])
        K.page_reserve(count, table, num, last, s["tok_indptr"], s["ps"], slot_page=s["slot_page"],
                       slot_offset=s["slot_off"], out_indptr=s["indptr"], out_indices=s["indices"])
        return dict(got, slot_page=s["slot_page"], slot_off=s["slot_off"], indptr=s["indptr"], indices=s["indices"])
    if s["mode"] == "accept":
        K.tree_accept(s["parents"], s["tokens"], s["targets"], s["qo_indptr"], s["keep_from"], keep=s["keep"],
                      keep_count=s["keep_count"], next_token=s["next_token"])
        got.update(keep=s["keep"], keep_count=s["keep_count"], next_token=s["next_token"])
    K.cache_compact(s["pool"], count, table, num, last, s["keep_from"], s["keep"], s["keep_count"])
    return got


def _run_plain(s):
    if s["kind"] == "tree":
        return _plain_tree(s)
    if s["kind"] == "sparse":
        return _plain_sparse(s)
    if s["kind"] == "bounds":
        ids = s["page_ids"].long()
        s["bounds"][ids], s["scale"][ids] = _bounds(s["kv"][ids])
        return dict(bounds=s["bounds"], scale=s["scale"])
    s["meta"].copy_(s["meta0"])
    return _plain_fork(s) if s["kind"] == "fork" else _plain_compact(s)


# ------------------------------------------------------------ plain forms
def _padded(indptr, width):
    """Positions of ragged rows as a padded matrix: (flat index [rows, width], inside)."""

    n = (indptr[1:] - indptr[:-1]).long()
    at = torch.arange(width, device=indptr.device)
    inside = at < n[:, None]
    return torch.where(inside, indptr[:-1].long()[:, None] + at, 0), inside


def _square(m):
    return ((m @ m) > 0).float()


def _closure(parents, qo_indptr, max_n):
    """Ancestor-or-self matrix of every row's drafted tokens, [rows, max_n, max_n] (0 / 1), at most 128 tokens."""

    flat, inside = _padded(qo_indptr, max_n)
    p = torch.where(inside, parents[flat].long(), -1)
    at = torch.arange(max_n, device=p.device)
    m = ((p[..., None] == at) | ((at[:, None] == at) & inside[..., None])).float()
    return _square(_square(_square(_square(_square(_square(_square(m))))))), flat, inside, p


def _plain_tree(s):
    q, kv = s["q"].float(), s["kv"]
    layers, total, hq, d = q.shape
    ps, hkv = kv.shape[3], kv.shape[4]
    c, flat, inside, _ = _closure(s["parents"], s["qo_indptr"], s["max_n"])
    rows, n = flat.shape
    tok_row = torch.searchsorted(s["qo_indptr"][1:].long(), torch.arange(total, device=q.device), right=True)
    tok_at = torch.arange(total, device=q.device) - s["qo_indptr"].long()[tok_row]
    bits = torch.zeros(total, s["words"] * 32, device=q.device, dtype=torch.int64)
    bits[:, :n] = c[tok_row, tok_at].long()
    mask = (bits.view(total, -1, 32) << torch.arange(32, device=q.device)).sum(-1).to(torch.int32)
    depth = (bits.sum(-1) - 1).to(torch.int32)

    at, has = _padded(s["kv_indptr"], s["max_pages"])
    pages = s["kv_indices"].long()[at]
    npg = has.sum(-1)
    kv_len = torch.where(npg > 0, (npg - 1) * ps + s["kv_last"].long(), 0)
    k = kv[:, pages, 0].reshape(layers, rows, -1, hkv, d).float()
    v = kv[:, pages, 1].reshape(layers, rows, -1, hkv, d).float()
    pos = torch.arange(k.shape[2], device=q.device)
    ctx = kv_len - (s["qo_indptr"][1:] - s["qo_indptr"][:-1]).long()
    j = (pos - ctx[:, None]).clamp(0, n - 1)
    draft = torch.gather(c, 2, j[:, None].expand(rows, n, -1)) > 0
    see = (pos < ctx[:, None])[:, None] | ((pos >= ctx[:, None]) & (pos < kv_len[:, None]))[:, None] & draft
    # [layers, rows, kv head, token x group, positions]
    qp = q[:, flat].view(layers, rows, n, hkv, hq // hkv, d).permute(0, 1, 3, 2, 4, 5).reshape(layers, rows, hkv, -1, d)
    sc = (qp @ k.permute(0, 1, 3, 4, 2)).mul_(1.0 / math.sqrt(d)).view(layers, rows, hkv, n, hq // hkv, -1)
    sc.masked_fill_(~see[:, None, :, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    p = sc.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(layers, rows, hkv, -1, p.shape[-1]) @ v.permute(0, 1, 3, 2, 4)).view(layers, rows, hkv, n, hq // hkv, d)
    o = torch.where(l > 0, o / l, 0.0).permute(0, 1, 3, 2, 4, 5).reshape(layers, rows, n, hq, d)
    lse = (m + l.log())[..., 0].permute(0, 1, 3, 2, 4).reshape(layers, rows, n, hq)
    return dict(out=o[:, tok_row, tok_at].to(torch.bfloat16), lse=lse[:, tok_row, tok_at], mask=mask, depth=depth)


def _bounds(kv):
    """int8 bounds [pages, kv heads, 2, d] (lo, hi) of the keys of full pages, and their scale."""

    k = kv[:, 0]  # minima and maxima of bf16 values are bf16 values: nothing is rounded
    lo, hi = k.amin(1).float(), k.amax(1).float()
    scale = torch.maximum(lo.abs(), hi.abs()).amax(-1) * INV127
    div = torch.where(scale > 0, scale, 1.0)[..., None]
    return (torch.stack([(lo / div).floor().clamp(-127, 127), (hi / div).ceil().clamp(-127, 127)], -2).to(torch.int8),
            scale)


def _plain_sparse(s):
    q, kv = s["q"].float(), s["kv"]
    rows, hq, d = q.shape
    ps, hkv = kv.shape[2], kv.shape[3]
    at, has = _padded(s["kv_indptr"], s["max_pages"])
    pages = s["kv_indices"].long()[at]
    npg = has.sum(-1)
    # integer score: fp32 holds every product and sum exactly (|sum| < 2^24)
    qg = q.view(rows, hkv, hq // hkv, d)
    qs = qg.abs().amax((-1, -2), keepdim=True) * INV127
    qi = (qg / torch.where(qs > 0, qs, 1.0)).round().clamp(-127, 127)
    bd = s["bounds"][pages].permute(0, 2, 3, 4, 1).float()  # [rows, hkv, 2, d, pages]
    dot = (qi.clamp(min=0) @ bd[:, :, 1] + qi.clamp(max=0) @ bd[:, :, 0]).amax(2)
    score = dot * s["scale"][pages].transpose(1, 2)
    idx = torch.arange(s["max_pages"], device=q.device)
    forced = (idx < s["sink"]) | (idx >= npg[:, None] - s["recent"])
    score = score.masked_fill(forced[:, None], float("inf")).masked_fill(~has[:, None], float("-inf"))
    width = s["select"]
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :width]
    order = torch.where(order < npg[:, None, None], order, s["max_pages"]).sort(-1).values
    order = torch.nn.functional.pad(order, (0, max(0, width - order.shape[-1])), value=s["max_pages"])
    live = order < s["max_pages"]
    pick = torch.where(live, order, 0)
    pg = torch.gather(pages[:, None].expand(-1, hkv, -1), 2, pick)
    head = torch.arange(hkv, device=q.device)[None, :, None]
    k = kv[pg, 0, :, head].float().reshape(rows, hkv, -1, d)
    v = kv[pg, 1, :, head].float().reshape(rows, hkv, -1, d)
    used = torch.where(pick == npg[:, None, None] - 1, s["kv_last"][:, None, None].long(), ps)
    see = (live[..., None] & (torch.arange(ps, device=q.device) < used[..., None])).reshape(rows, hkv, 1, -1)
    sc = (qg @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    sc = sc.masked_fill(~see, float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    p = (sc - m).exp()
    l = p.sum(-1, keepdim=True)
    o = torch.where(l > 0, (p @ v) / l, 0.0)
    return dict(out=o.reshape(rows, hq, d).to(torch.bfloat16), lse=(m + l.log()).reshape(rows, hq),
                selected=torch.where(live, order, -1).to(torch.int32))


def _free(count, most):
    """The lowest `most` free page ids."""

    order = torch.sort((count > 0).to(torch.int8), stable=True).indices
    return order[:most].to(torch.int32)


def _drop(count, table, num, first):
    """One reference less for the pages first[r] .. num[r] of every row."""

    at = torch.arange(table.shape[1], device=table.device)
    gone = (at >= first[:, None]) & (at < num[:, None])
    count.scatter_add_(0, torch.where(gone, table, 0).long().view(-1), -gone.to(torch.int32).view(-1))


def _csr(table, num, indptr, indices):
    at = torch.arange(table.shape[1], device=table.device)
    indptr[1:] = num.cumsum(0)
    to = torch.where(at < num[:, None], indptr[:-1, None] + at, indices.numel())
    indices.copy_(torch.nn.functional.pad(indices, (0, 1)).scatter(0, to.long().view(-1), table.view(-1))[:-1])


def _plain_fork(s):
    count, table, num, last = _meta(s)
    ps, cap = s["ps"], s["cap"]
    at = torch.arange(cap, device=table.device)
    # release
    rows = s["released"].long()
    _drop(count, table[rows], num[rows], torch.zeros_like(num[rows]))
    num[rows], last[rows] = 0, 0
    # fork
    src, dst = s["src"].long(), s["dst"].long()
    n, tail = num[src], last[src]
    copied = (n > 0) & (tail < ps)
    full = n - copied.int()
    pages = _free(count, len(src))[(copied.cumsum(0) - 1).clamp(min=0)]
    shared = at < full[:, None]
    old = table[src]
    count.scatter_add_(0, torch.where(shared, old, 0).long().view(-1), shared.to(torch.int32).view(-1))
    count.scatter_add_(0, pages.long(), copied.to(torch.int32))
    new = torch.where(shared, old, table[dst])
    table[dst] = torch.where((at == full[:, None]) & copied[:, None], pages[:, None], new)
    num[dst], last[dst] = n, tail
    a = torch.gather(old, 1, full.long().clamp(max=cap - 1)[:, None])[:, 0].long()
    used = (torch.arange(ps, device=table.device) < tail[:, None]) & copied[:, None]
    job, tok = used.nonzero(as_tuple=True)
    s["pool"][:, pages.long()[job], :, tok] = s["pool"][:, a[job], :, tok]
    # reserve
    n = s["tok_indptr"][1:] - s["tok_indptr"][:-1]
    length = torch.where(num > 0, (num - 1) * ps + last, 0)
    grown = (length + n + ps - 1) // ps
    want = grown - num
    first = want.cumsum(0) - want
    fresh = (at >= num[:, None]) & (at < grown[:, None])
    pages = _free(count, s["rows"] * cap)
    ids = pages[(first[:, None] + at - num[:, None]).clamp(0, len(pages) - 1).long()]
    table.copy_(torch.where(fresh, ids, table))
    count.scatter_add_(0, torch.where(fresh, ids, 0).long().view(-1), fresh.to(torch.int32).view(-1))
    row = torch.searchsorted(s["tok_indptr"][1:].long(), torch.arange(s["total"], device=table.device), right=True)
    pos = length[row] + torch.arange(s["total"], device=table.device) - s["tok_indptr"][row]
    s["slot_page"].copy_(table[row, pos // ps])
    s["slot_off"].copy_(pos % ps)
    num.copy_(grown)
    last.copy_(torch.where(n > 0, (length + n - 1) % ps + 1, last))
    _csr(table, num, s["indptr"], s["indices"])
    return dict(pool=s["pool"].view(torch.int16), meta=s["meta"], slot_page=s["slot_page"], slot_off=s["slot_off"],
                indptr=s["indptr"], indices=s["indices"])


def _plain_accept(s):
    n = s["max_n"]
    c, flat, inside, p = _closure(s["parents"], s["qo_indptr"], n)
    tok, tgt = s["tokens"][flat], s["targets"][flat]
    match = (p < 0) | (tok == torch.gather(tgt, 1, p.clamp(min=0)))
    taken = inside & ((c @ (~match).float()[..., None])[..., 0] == 0)
    depth = c.sum(-1)
    at = torch.arange(n, device=p.device)
    best = (taken * (depth * (n + 1) + (n - at))).argmax(-1)
    some = taken.any(-1)
    path = (torch.gather(c, 1, best[:, None, None].expand(-1, 1, n))[:, 0] > 0) & some[:, None]
    # the path's own order is the index order: parents come first
    idx = torch.where(path, at, n).sort(-1).values
    s["keep"].copy_(torch.where(idx < n, idx + s["keep_from"][:, None], -1))
    s["keep_count"].copy_(path.sum(-1))
    s["next_token"].copy_(torch.where(some, torch.gather(tgt, 1, best[:, None])[:, 0], -1))


def _plain_compact(s):
    got = dict(pool=s["pool"].view(torch.int16), meta=s["meta"])
    if s["mode"] == "accept":
        _plain_accept(s)
        got.update(keep=s["keep"], keep_count=s["keep_count"], next_token=s["next_token"])
    count, table, num, last = _meta(s)
    ps, cap = s["ps"], s["cap"]
    keep, k, kf = s["keep"].long(), s["keep_count"].long(), s["keep_from"].long()
    i = torch.arange(keep.shape[1], device=table.device)
    stays = ((keep == kf[:, None] + i) & (i < k[:, None])).to(torch.int64).cumprod(-1).sum(-1)
    length = kf + k
    full = (kf + stays) // ps
    rest = length - full * ps
    at_full = torch.gather(table, 1, full.clamp(max=cap - 1)[:, None])[:, 0].long()
    # nothing moves and the new last page is whole or the row's own: cut in place
    cut = (stays == k) & ((rest == 0) | (count[at_full] == 1))
    want = torch.where(cut, 0, (rest + ps - 1) // ps)
    first = want.cumsum(0) - want
    at = torch.arange(cap, device=table.device)
    fresh = (at >= full[:, None]) & (at < (full + want)[:, None])
    pages = _free(count, s["rows"] * cap)
    ids = pages[(first[:, None] + at - full[:, None]).clamp(0, len(pages) - 1)]
    # the tokens that move
    pos = torch.arange(cap * ps, device=table.device)
    moved = (pos >= (full * ps)[:, None]) & (pos < length[:, None]) & ~cut[:, None]
    row, to = moved.nonzero(as_tuple=True)
    frm = torch.where(to < kf[row], to, keep[row, (to - kf[row]).clamp(min=0)])
    old = table[row, frm // ps].long()
    s["pool"][:, ids[row, to // ps].long(), :, to % ps] = s["pool"][:, old, :, frm % ps]
    held = torch.where(cut & (rest > 0), full + 1, full)
    _drop(count, table, num, held)
    count.scatter_add_(0, torch.where(fresh, ids, 0).long().view(-1), fresh.to(torch.int32).view(-1))
    table.copy_(torch.where(fresh, ids, table))
    num.copy_((length + ps - 1) // ps)
    last.copy_(torch.where(length > 0, (length - 1) % ps + 1, 0))
    return got


# ------------------------------------------------------------------- work
def work(case):
    kind, ps, d, hkv = case["kind"], case["ps"], case["d"], case["hkv"]
    if kind == "tree":
        n = _lengths(case, case["n_lo"], case["n_hi"], 1)
        lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 2) + n
        per = int(lens.sum()) * 4 * hkv * d + int(n.sum()) * case["hq"] * (4 * d + 4)
        return dict(bytes=case["layers"] * per, flops=4 * case["layers"] * case["hq"] * d * int((n * lens).sum()))
    if kind == "sparse":
        lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 3)
        npg = _pages(lens, ps)
        scored = np.where(npg > case["select"], npg - case["sink"] - case["recent"], 0)
        toks = np.minimum(lens, case["select"] * ps)
        q = case["rows"] * case["hq"]
        return dict(bytes=hkv * (int(scored.sum()) * (2 * d + 4) + int(toks.sum()) * 4 * d) + q * (4 * d + 4)
                    + case["rows"] * hkv * case["select"] * 4,
                    flops=case["hq"] * d * (4 * int(toks.sum()) + 4 * int(scored.sum())))
    if kind == "bounds":
        return dict(bytes=case["pages"] * hkv * (ps * d * 2 + 2 * d + 4), flops=case["pages"] * hkv * ps * d * 2)
    token = 2 * case["hkv"] * d * 2 * case["layers"]  # K and V of one token in every layer
    lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 4)
    if kind == "fork":
        return dict(bytes=case["forks"] * (ps // 2) * 2 * token + 4 * int(_pages(lens, ps).sum()), flops=0)
    if case["mode"] == "evict":
        return dict(bytes=int(lens.sum()) * token, flops=0)  # half of the tokens, read and written
    return dict(bytes=case["rows"] * (ps // 2 + 3) * 2 * token, flops=0)


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The floating outputs in 64 bits, from the definitions, one row at a time.  Copies of cache contents and
    whole numbers have no such value."""

    s = prepare(case, seed)
    if s["kind"] == "tree":
        return _exact_tree(s)
    if s["kind"] == "sparse":
        return _exact_sparse(s)
    if s["kind"] == "bounds":
        ids = s["page_ids"].long()
        a = s["kv"][ids, 0].abs().amax((1, 3)).double()
        scale = s["scale"].double()
        scale[ids] = a / 127.0
        return dict(bounds=None, scale=scale)
    return None


def _row_tokens(s, kv, r):
    ps = kv.shape[2]
    i0, i1 = int(s["kv_indptr"][r]), int(s["kv_indptr"][r + 1])
    n = (i1 - i0 - 1) * ps + int(s["kv_last"][r]) if i1 > i0 else 0
    return s["kv_indices"][i0:i1].long(), n


def _exact_attention(q, k, v, see):
    """softmax(q k^T / sqrt(d)) v of one head in 64 bits; see: [queries, keys] or None."""

    x = q @ k.t() / math.sqrt(q.shape[1])
    if see is not None:
        x = x.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(x, 1)
    return torch.exp(x - lse[:, None]) @ v, lse


def _exact_tree(s):
    layers, total, hq, d = s["q"].shape
    hkv = s["kv"].shape[4]
    out = torch.zeros(layers, total, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(layers, total, hq, dtype=torch.float64, device="cuda")
    par = s["parents"].tolist()
    for r in range(len(s["kv_last"])):
        a, b = int(s["qo_indptr"][r]), int(s["qo_indptr"][r + 1])
        see = np.zeros((b - a, b - a), bool)
        for i in range(b - a):
            j = i
            while j >= 0:
                see[i, j] = True
                j = par[a + j]
        for l in range(layers):
            pages, n = _row_tokens(s, s["kv"][l], r)
            full = torch.ones(b - a, n, dtype=torch.bool, device="cuda")
            full[:, n - (b - a):] = torch.as_tensor(see, device="cuda")
            for h in range(hkv):
                kv = s["kv"][l][pages, :, :, h].double()
                k, v = kv[:, 0].reshape(-1, d)[:n], kv[:, 1].reshape(-1, d)[:n]
                for m in range(hq // hkv):
                    x = h * (hq // hkv) + m
                    out[l, a:b, x], lse[l, a:b, x] = _exact_attention(s["q"][l, a:b, x].double(), k, v, full)
    return dict(out=out, lse=lse, mask=None, depth=None)


def _exact_sparse(s):
    rows, hq, d = s["q"].shape
    ps, hkv = s["kv"].shape[2], s["kv"].shape[3]
    out = torch.zeros(rows, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(rows, hq, dtype=torch.float64, device="cuda")
    g = hq // hkv
    for r in range(rows):
        pages, n = _row_tokens(s, s["kv"], r)
        cnt = len(pages)
        b = s["bounds"][pages].cpu().numpy().astype(np.int64)
        sc = s["scale"][pages].cpu().numpy()
        for h in range(hkv):
            q = s["q"][r, h * g:(h + 1) * g].double()
            if cnt > s["select"]:
                x = q.float().cpu().numpy()
                qs = np.float32(np.abs(x).max()) * np.float32(INV127)
                qi = np.clip(np.rint(x / qs), -127, 127).astype(np.int64)
                dot = np.maximum(qi[:, None] * b[None, :, h, 0], qi[:, None] * b[None, :, h, 1]).sum(-1).max(0)
                val = dot.astype(np.float32) * sc[:, h]
                mid = np.arange(s["sink"], cnt - s["recent"])
                top = mid[np.lexsort((mid, -val[mid].astype(np.float64)))][:s["select"] - s["sink"] - s["recent"]]
                pick = np.sort(np.concatenate([np.arange(s["sink"]), top, np.arange(cnt - s["recent"], cnt)]))
            else:
                pick = np.arange(cnt)
            tok = (pick[:, None] * ps + np.arange(ps)).reshape(-1)
            kv = s["kv"][pages[torch.as_tensor(pick, device="cuda")], :, :, h].double()
            ok = torch.as_tensor(tok < n, device="cuda")
            k, v = kv[:, 0].reshape(-1, d)[ok], kv[:, 1].reshape(-1, d)[ok]
            out[r, h * g:(h + 1) * g], lse[r, h * g:(h + 1) * g] = _exact_attention(q, k, v, None)
    return dict(out=out, lse=lse, selected=None)
