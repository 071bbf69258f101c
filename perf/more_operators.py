"""Workloads of the operators that keep a paged cache small: windows with sinks, a 4-bit cache, eviction by weight.

Seven kinds of case over the paged cache ``[pages, 2, page_size, kv_heads, head_dim]``:

* ``wdec`` / ``wprompt``: attention with a sliding window and a few first tokens that stay visible, of one token per
  row and of ragged prompts behind cached prefixes.
* ``kv4dec``: one token per row over a cache held in 4 bits, with and without a window.
* ``kv4put``: the K/V of a prompt chunk quantised into its pages, and these pages expanded again, as the attention of
  the next chunk reads them.
* ``wtdec`` / ``wtprompt``: the attention weight that every cached token receives, accumulated over heads and tokens:
  with the attention of a decode step, and of a prompt from its log sums.
* ``select``: the positions that every row keeps, by that weight, and the weights moved with them.

A 4-bit record of one head of one token is head_dim / 2 bytes of codes (two channels a byte, the even one low), four
scales and four minima in bf16. Channel c belongs to group c % 4: value = minimum + scale * code.

With ``own`` false, :func:`run` computes them in elementary torch operations, in fp32; with ``own`` true it calls
the framework.
"""

import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One interactive sequence: latency counts.
        dict(name="window decode 1 row ctx 5003", kind="wdec", rows=1, ctx_lo=5003, ctx_hi=5003, hq=32, hkv=8, d=128,
             ps=16, window=1024, sinks=4),
        # A ragged serving batch, some rows shorter than the window.
        dict(name="window decode 48 rows ctx 700-30000", kind="wdec", rows=48, ctx_lo=700, ctx_hi=30000, hq=32, hkv=8,
             d=128, ps=16, window=4096, sinks=4),
        # Chunks of several requests behind cached prefixes, a group of seven heads.
        dict(name="window prompt 7 rows of 37-2500", kind="wprompt", rows=7, n_lo=37, n_hi=2500, ctx_lo=0, ctx_hi=5000,
             hq=28, hkv=4, d=128, ps=16, window=515, sinks=4),
        # One long document.
        dict(name="window prompt 1x32768", kind="wprompt", rows=1, n_lo=32768, n_hi=32768, ctx_lo=0, ctx_hi=0, hq=32,
             hkv=8, d=128, ps=16, window=4096, sinks=16),
        # One interactive sequence over a 4-bit cache.
        dict(name="kv4 decode 1 row ctx 600", kind="kv4dec", rows=1, ctx_lo=600, ctx_hi=600, hq=32, hkv=8, d=128, ps=16,
             window=0, sinks=0),
        # A ragged serving batch.
        dict(name="kv4 decode 24 rows ctx 500-40000", kind="kv4dec", rows=24, ctx_lo=500, ctx_hi=40000, hq=32, hkv=8,
             d=128, ps=16, window=0, sinks=0),
        # A batch of a multi-head model: the cache that 4 bits are for.
        dict(name="kv4 decode 64 rows ctx 8192 mha", kind="kv4dec", rows=64, ctx_lo=8192, ctx_hi=8192, hq=32, hkv=32,
             d=128, ps=16, window=0, sinks=0),
        # A long prompt chunk put into a 4-bit cache.
        dict(name="kv4 put 16384 tokens", kind="kv4put", tokens=16384, hkv=8, d=128, ps=16),
        # One interactive sequence that will evict.
        dict(name="weights decode 1 row ctx 2000", kind="wtdec", rows=1, ctx_lo=2000, ctx_hi=2000, hq=32, hkv=8, d=128,
             ps=16),
        # A ragged serving batch that will evict.
        dict(name="weights decode 32 rows ctx 1000-12000", kind="wtdec", rows=32, ctx_lo=1000, ctx_hi=12000, hq=32,
             hkv=8, d=128, ps=16),
        # The weights that a prompt gives its own tokens.
        dict(name="weights prompt 1x8192", kind="wtprompt", rows=1, n_lo=8192, n_hi=8192, ctx_lo=0, ctx_hi=0, hq=32,
             hkv=8, d=128, ps=16),
        # Long contexts cut to a sixteenth.
        dict(name="select 12 rows ctx 131072", kind="select", rows=12, ctx_lo=100000, ctx_hi=131072, budget=8192,
             sinks=4, recent=1000),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["wdec", "wprompt", "kv4dec", "kv4dec", "kv4put", "wtdec", "wtprompt", "select"])
    if kind == "select":
        ctx_hi = _logint(rng, 20, 131072)
        budget = _logint(rng, 12, max(13, ctx_hi))
        sinks = rng.randint(0, min(8, budget // 2))
        return dict(kind=kind, rows=_logint(rng, 1, 12), ctx_lo=max(1, ctx_hi // rng.choice([1, 2, 30])), ctx_hi=ctx_hi,
                    budget=budget, sinks=sinks, recent=rng.randint(0, (budget - sinks) // 2))
    ps = rng.choice([16, 16, 32])
    d = rng.choice([128, 128, 64])
    if kind == "kv4put":
        hkv = rng.choice([8, 2, 4, 1])
        return dict(kind=kind, tokens=_logint(rng, 1, 16384), hkv=hkv, d=d, ps=ps)
    hq, hkv = rng.choice([(32, 8), (32, 32), (28, 4), (8, 2), (16, 1)])
    case = dict(kind=kind, hq=hq, hkv=hkv, d=d, ps=ps)
    if kind in ("wdec", "kv4dec", "wtdec"):
        rows = _logint(rng, 1, 64)
        # at most the largest listed case's rows x context x heads
        most = {"wdec": 48 * 30000 * 8, "kv4dec": 64 * 8192 * 32, "wtdec": 32 * 12000 * 8}[kind]
        ctx_hi = _logint(rng, 20, max(40, min(60000, most // (rows * hkv))))
        case.update(rows=rows, ctx_lo=max(1, ctx_hi // rng.choice([1, 2, 10])), ctx_hi=ctx_hi)
    else:
        rows = _logint(rng, 1, 8)
        most = {"wprompt": 8192, "wtprompt": 6000}[kind]
        n_hi = _logint(rng, 1, max(8, most // rows))
        ctx_hi = rng.choice([0, _logint(rng, 1, max(2, most // rows))])
        case.update(rows=rows, n_lo=max(1, n_hi // rng.choice([1, 2, 10])), n_hi=n_hi, ctx_lo=ctx_hi // 2, ctx_hi=ctx_hi)
    if kind in ("wdec", "wprompt"):
        case.update(window=_logint(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 17]))
    elif kind == "kv4dec":
        case.update(window=rng.choice([0, 0, _logint(rng, 1, 4096)]), sinks=rng.choice([0, 4]))
    return case


def _lengths(case, lo, hi, salt):
    """One length per row, spread over [lo, hi]: by the case alone, so that work() knows them."""

    r = np.random.RandomState(1000 * salt + case["rows"] + 7 * hi)
    out = r.randint(lo, hi + 1, case["rows"])
    out[0] = hi
    return out.astype(np.int64)


def _row_lengths(case):
    """(query tokens, cached tokens with them) of every row."""

    n = _lengths(case, case["n_lo"], case["n_hi"], 1) if "n_hi" in case else np.ones(case["rows"], np.int64)
    ctx = _lengths(case, case["ctx_lo"], case["ctx_hi"], 2)
    return n, ctx if "n_hi" not in case else ctx + n


def _pages(length, ps):
    return (length + ps - 1) // ps


# ----------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _channels(g, shape):
    """Sizes of the channels of a decoder's keys and values: unequal, a few of them large."""

    ch = 0.5 + torch.rand(shape, generator=g, device="cuda")
    return (ch * torch.where(torch.rand(shape, generator=g, device="cuda") < 0.03, 4.0, 1.0)).to(torch.bfloat16)


def _kv(g, shape):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    return x.mul_(_channels(g, shape[-2:]))


def _i32(a):
    return torch.as_tensor(np.asarray(a, np.int32), device="cuda")


def _table(rng, lens, ps, spare):
    """Row page lists over a shuffled pool: (pool size, indptr, indices, last page lengths)."""

    n = _pages(lens, ps)
    pool = int(n.sum()) + spare
    at = np.concatenate([[0], np.cumsum(n)])
    return pool, at, rng.permutation(pool)[:at[-1]], np.where(lens > 0, lens - (n - 1) * ps, 0)


def prepare(case, seed):
    rng = np.random.RandomState(seed % (2**31 - 1))
    g = _gen(seed)
    kind = case["kind"]
    if kind == "select":
        lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 2)
        width = case["ctx_hi"] + 16
        # a few tokens hold most of the weight
        w = torch.rand(case["rows"], width, generator=g, device="cuda").pow_(8).mul_(50.0)
        w *= torch.arange(width, device="cuda") < _i32(lens)[:, None]
        most = case["budget"] - case["sinks"]
        return dict(kind=kind, weight=w, lens=_i32(lens), budget=case["budget"], sinks=case["sinks"],
                    recent=case["recent"], keep_from=torch.zeros(case["rows"], device="cuda", dtype=torch.int32),
                    keep=torch.zeros(case["rows"], most, device="cuda", dtype=torch.int32),
                    keep_count=torch.zeros(case["rows"], device="cuda", dtype=torch.int32),
                    out_weight=torch.zeros_like(w))
    ps, d, hkv = case["ps"], case["d"], case["hkv"]
    if kind == "kv4put":
        t = case["tokens"]
        n = _pages(t, ps)
        ids = rng.permutation(n + 3)[:n]
        at = np.arange(t)
        k, v = _kv(g, (t, hkv, d)), _kv(g, (t, hkv, d))
        return dict(kind=kind, k=k, v=v, ps=ps, page_id=_i32(ids[at // ps]), page_off=_i32(at % ps), page_ids=_i32(ids),
                    cache=torch.zeros(n + 3, 2, ps, hkv, d // 2 + 16, device="cuda", dtype=torch.uint8),
                    out=torch.zeros(n, 2, ps, hkv, d, device="cuda", dtype=torch.bfloat16))
    n, lens = _row_lengths(case)
    pool, at, ids, last = _table(rng, lens, ps, 3)
    total = int(n.sum())
    q = torch.randn(total, case["hq"], d, generator=g, device="cuda", dtype=torch.bfloat16)
    s = dict(kind=kind, q=q, kv_indptr=_i32(at), kv_indices=_i32(ids), kv_last=_i32(last), lens=lens, n=n, ps=ps,
             hkv=hkv, out=torch.empty_like(q), lse=torch.empty(total, case["hq"], device="cuda"))
    if kind == "kv4dec":
        s["cache"] = torch.empty(pool, 2, ps, hkv, d // 2 + 16, device="cuda", dtype=torch.uint8)
        ch = _channels(g, (2, 1, hkv, d))
        step = max(1, (1 << 27) // (2 * ps * hkv * d))
        for p in range(0, pool, step):
            part = s["cache"][p:p + step]
            x = torch.randn(*part.shape[:-1], d, generator=g, device="cuda", dtype=torch.bfloat16) * ch
            part.copy_(_pack4(x))
        s.update(window=case["window"], sinks=case["sinks"])
        return s
    s["kv"] = _kv(g, (pool, 2, ps, hkv, d))
    if kind in ("wdec", "wprompt"):
        s.update(window=case["window"], sinks=case["sinks"])
    if kind in ("wprompt", "wtprompt"):
        s["qo_indptr"] = _i32(np.concatenate([[0], np.cumsum(n)]))
    if kind in ("wtdec", "wtprompt"):
        live = torch.arange(int(lens.max()) + 5, device="cuda") < _i32(lens)[:, None]
        s["weight0"] = torch.rand(len(lens), live.shape[1], generator=g, device="cuda").pow_(4) * live
        s["weight"] = s["weight0"].clone()
    if kind == "wtprompt":  # the prompt's attention came before: its log sums are in hand
        s["lse"] = _plain_attention(s, want_out=False)[1]
    return s


# -------------------------------------------------------------------- run
def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from pagelora_b200 import kernels as K

    kind = s["kind"]
    if kind == "select":
        K.evict_select(s["weight"], s["lens"], s["budget"], sinks=s["sinks"], recent=s["recent"],
                       keep_from=s["keep_from"], keep=s["keep"], keep_count=s["keep_count"], out_weight=s["out_weight"])
        return dict(keep_from=s["keep_from"], keep=s["keep"], keep_count=s["keep_count"], weight=s["out_weight"])
    if kind == "kv4put":
        K.kv4_append(s["k"], s["v"], s["cache"], s["page_id"], s["page_off"])
        return K.kv4_expand(s["cache"], s["page_ids"], out=s["out"])
    table = (s["kv_indptr"], s["kv_indices"], s["kv_last"])
    if kind == "wtprompt":
        s["weight"].copy_(s["weight0"])
        return K.paged_prefill_weights(s["q"], s["kv"], s["qo_indptr"], *table, s["lse"], s["weight"])
    to = dict(out=s["out"], out_lse=s["lse"])
    if kind == "wdec":
        K.paged_window_decode(s["q"], s["kv"], *table, window=s["window"], sinks=s["sinks"], **to)
    elif kind == "wprompt":
        K.paged_window_prefill(s["q"], s["kv"], s["qo_indptr"], *table, window=s["window"], sinks=s["sinks"], **to)
    elif kind == "kv4dec":
        K.paged_kv4_decode(s["q"], s["cache"], *table, window=s["window"] or None, sinks=s["sinks"], **to)
    else:
        s["weight"].copy_(s["weight0"])
        K.paged_decode_weights(s["q"], s["kv"], *table, s["weight"], **to)
        return dict(out=s["out"], lse=s["lse"], weight=s["weight"])
    return dict(out=s["out"], lse=s["lse"])


def _run_plain(s):
    kind = s["kind"]
    if kind == "select":
        return _plain_select(s)
    if kind == "kv4put":
        s["cache"][s["page_id"].long(), :, s["page_off"].long()] = _pack4(torch.stack([s["k"], s["v"]], 1))
        s["out"].copy_(_unpack4(s["cache"][s["page_ids"].long()]).to(torch.bfloat16))
        return s["out"]
    if kind == "wtprompt":
        s["weight"].copy_(s["weight0"])
        _plain_prompt_weights(s)
        return s["weight"]
    if kind == "wtdec":
        s["weight"].copy_(s["weight0"])
    out, lse = _plain_attention(s)
    got = dict(out=out, lse=lse)
    return dict(got, weight=s["weight"]) if kind == "wtdec" else got


# ------------------------------------------------------------ plain forms
def _pack4(x):
    """bf16 [..., d] as 4-bit records [..., d / 2 + 16]. Halves, so that no difference of two values overflows."""

    d = x.shape[-1]
    half = x.float().mul_(0.5).view(*x.shape[:-1], d // 4, 4)
    lo, hi = half.amin(-2), half.amax(-2)
    scale = ((hi - lo) / 7.5).to(torch.bfloat16)
    step = 0.5 * scale.float()
    step = torch.where(step > 0, step, math.inf)
    code = ((half - lo[..., None, :]) / step[..., None, :]).round_().clamp_(0, 15).to(torch.uint8).view(x.shape)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    tail = torch.cat([scale, (2.0 * lo).to(torch.bfloat16)], -1)
    return torch.cat([codes, tail.view(torch.uint8)], -1)


def _unpack4(rec):
    """The fp32 values [..., d] that records stand for."""

    half = rec.shape[-1] - 16
    code = torch.stack([rec[..., :half] & 15, rec[..., :half] >> 4], -1).view(*rec.shape[:-1], half // 2, 4).float()
    tail = rec[..., half:].contiguous().view(torch.bfloat16).float()
    return (code * tail[..., None, :4] + tail[..., None, 4:]).view(*rec.shape[:-1], 2 * half)


def _tokens(s, part, rows, pages):
    """K or V (part 0 / 1) of the pages [rows, n], fp32 [rows, kv heads, n x page_size, d]."""

    if "cache" in s:
        x = _unpack4(s["cache"][pages, part])
    else:
        x = s["kv"][pages, part].float()
    return x.reshape(rows, -1, s["hkv"], x.shape[-1]).transpose(1, 2)


def _plain_attention(s, want_out=True):
    """Attention of every kind, in blocks of rows (one token each) or of a row's queries."""

    return _plain_prompts(s, want_out) if "qo_indptr" in s else _plain_decode(s)


def _plain_decode(s):
    q, ps, hkv = s["q"].float(), s["ps"], s["hkv"]
    rows, hq, d = q.shape
    window, sinks = s.get("window", 0), s.get("sinks", 0)
    out, lse = torch.empty_like(q), torch.empty(rows, hq, device=q.device)
    first = np.maximum(s["lens"] - window, 0) // ps if window else np.zeros(rows, np.int64)
    early = np.minimum(_pages(sinks, ps), first)  # pages of the first tokens in front of the window's
    count = early + _pages(s["lens"], ps) - first
    step = max(1, (1 << 29) // max(1, int(count.max()) * ps * hkv * d))
    for r in range(0, rows, step):
        b = slice(r, min(rows, r + step))
        most = int(count[b].max())
        at = torch.arange(most, device=q.device)
        f, e, c = (torch.as_tensor(x[b], device=q.device)[:, None] for x in (first, early, count))
        n = torch.as_tensor(s["lens"][b], device=q.device)[:, None]
        page = torch.where(at < e, at, at - e + f)
        entry = s["kv_indptr"][b].long()[:, None] + torch.where(at < c, page, 0)
        pages = s["kv_indices"].long()[torch.where(n > 0, entry, 0)]
        pos = (page[..., None] * ps + torch.arange(ps, device=q.device)).view(len(n), -1)
        see = (pos < n) & (at < c).repeat_interleave(ps, 1)
        if window:
            see &= (pos >= n - window) | (pos < sinks)
        k = _tokens(s, 0, len(n), pages)
        x = (q[b].view(len(n), hkv, hq // hkv, d) @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
        x.masked_fill_(~see[:, None, None], -math.inf)
        m = x.amax(-1, keepdim=True)
        m = torch.where(torch.isinf(m), 0.0, m)
        p = x.sub_(m).exp_()
        l = p.sum(-1, keepdim=True)
        out[b] = torch.where(l > 0, (p @ _tokens(s, 1, len(n), pages)) / l, 0.0).view(len(n), hq, d)
        lse[b] = (m + l.log()).view(len(n), hq)
        if "weight" in s:
            w = torch.where(l > 0, p / l, 0.0).sum((1, 2))
            take = min(w.shape[1], s["weight"].shape[1])
            s["weight"][b, :take] += w[:, :take]
    return out.to(torch.bfloat16), lse


def _blocks(s, most):
    """Blocks of a row's queries: (row, queries of the flat matrix, their positions, keys [a, b) of the row)."""

    at = 0
    for r, (n, length) in enumerate(zip(s["n"].tolist(), s["lens"].tolist())):
        for i in range(0, n, most):
            j = min(n, i + most)
            p0 = length - n + i
            lo = max(0, p0 - s["window"] + 1) if s.get("window") else 0
            yield r, slice(at + i, at + j), (p0, length - n + j), (lo, length - n + j)
        at += n


def _row_keys(s, r, part, a, b):
    """K or V of positions [a, b) of row r: [kv heads, b - a, d] fp32."""

    ps, i0 = s["ps"], s["kv_indptr_host"][r]
    pages = s["kv_indices"][i0 + a // ps:i0 + _pages(b, ps)].long()
    return _tokens(s, part, 1, pages[None])[0][:, a % ps:a % ps + b - a]


def _plain_prompts(s, want_out=True):
    q, hkv = s["q"].float(), s["hkv"]
    total, hq, d = q.shape
    s.setdefault("kv_indptr_host", np.concatenate([[0], np.cumsum(_pages(s["lens"], s["ps"]))]))
    sinks = s.get("sinks", 0)
    out = torch.empty_like(q) if want_out else None
    lse = torch.empty(total, hq, device=q.device)
    for r, rows, (p0, p1), (a, b) in _blocks(s, 2048 if "window" in s else 1024):
        early = min(sinks, a)
        qb = q[rows].view(-1, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        key = torch.cat([_row_keys(s, r, 0, 0, early), _row_keys(s, r, 0, a, b)], 1)
        pos = torch.cat([torch.arange(early, device=q.device), torch.arange(a, b, device=q.device)])
        at = torch.arange(p0, p1, device=q.device)[:, None]
        see = pos <= at
        if "window" in s:
            see &= (pos > at - s["window"]) | (pos < sinks)
        x = (qb @ key.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(hkv, hq // hkv, p1 - p0, -1)
        x.masked_fill_(~see, -math.inf)
        m = x.amax(-1, keepdim=True)
        p = x.sub_(m).exp_()
        l = p.sum(-1, keepdim=True)
        lse[rows] = (m + l.log())[..., 0].permute(2, 0, 1).reshape(-1, hq)
        if want_out:
            v = torch.cat([_row_keys(s, r, 1, 0, early), _row_keys(s, r, 1, a, b)], 1)
            o = (p.view(hkv, -1, p.shape[-1]) @ v).view(hkv, hq // hkv, p1 - p0, d) / l
            out[rows] = o.permute(2, 0, 1, 3).reshape(-1, hq, d)
    return out.to(torch.bfloat16) if want_out else None, lse


def _plain_prompt_weights(s):
    q, hkv = s["q"].float(), s["hkv"]
    _, hq, d = q.shape
    for r, rows, (p0, p1), (a, b) in _blocks(s, 1024):
        qb = q[rows].view(-1, hkv, hq // hkv, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        x = (qb @ _row_keys(s, r, 0, a, b).transpose(-1, -2)).mul_(1.0 / math.sqrt(d))
        x = x.view(hkv, hq // hkv, p1 - p0, -1)
        x.sub_(s["lse"][rows].view(-1, hkv, hq // hkv).permute(1, 2, 0)[..., None])
        see = torch.arange(a, b, device=q.device) <= torch.arange(p0, p1, device=q.device)[:, None]
        s["weight"][r, a:b] += x.masked_fill_(~see, -math.inf).exp_().sum((0, 1, 2))


def _plain_select(s):
    w, n = s["weight"], s["lens"].long()[:, None]
    rows, width = w.shape
    budget, sinks, recent = s["budget"], s["sinks"], s["recent"]
    at = torch.arange(width, device=w.device)
    forced = (at < sinks) | (at >= n - recent)
    score = torch.where(forced, math.inf, w).masked_fill(at >= n, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :budget]
    cut = n > budget
    kept = torch.sort(torch.where(torch.arange(order.shape[1], device=w.device) < n, order, width), dim=-1).values
    s["keep_from"].copy_(torch.where(cut, sinks, n)[:, 0])
    s["keep_count"].copy_(torch.where(cut, budget - sinks, 0)[:, 0])
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[1]), value=width)
    s["keep"].copy_(torch.where(cut, kept[:, sinks:], -1))
    src = torch.nn.functional.pad(kept[:, :width], (0, max(0, width - budget)), value=width)
    src = torch.where(cut, src, torch.where(at < n, at, width))
    s["out_weight"].copy_(torch.gather(torch.nn.functional.pad(w, (0, 1)), 1, src))
    return dict(keep_from=s["keep_from"], keep=s["keep"], keep_count=s["keep_count"], weight=s["out_weight"])


# ------------------------------------------------------------------- work
def _seen(case):
    """(keys that at least one query of the row sees, visible pairs) over all rows."""

    n, lens = _row_lengths(case)
    keys = pairs = 0
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    for k, length in zip(n.tolist(), lens.tolist()):
        p = np.arange(length - k, length, dtype=np.int64)
        if window:
            lo = np.maximum(p - window + 1, 0)
            pairs += int((p + 1 - lo + np.minimum(sinks, lo)).sum())
            keys += length - int(lo[0]) + min(sinks, int(lo[0])) if k else 0
        else:
            pairs += int((p + 1).sum())
            keys += length
    return keys, pairs


def work(case):
    kind = case["kind"]
    if kind == "select":
        lens = _lengths(case, case["ctx_lo"], case["ctx_hi"], 2)
        kept = np.minimum(lens, case["budget"])
        width = case["rows"] * (case["ctx_hi"] + 16)
        return dict(bytes=4 * int(lens.sum() + kept.sum()) + 4 * width, flops=0)
    d, hkv = case["d"], case["hkv"]
    if kind == "kv4put":
        # K/V in, records out; records in, pages out
        pages = _pages(case["tokens"], case["ps"]) * case["ps"]
        return dict(bytes=2 * hkv * (case["tokens"] * (2 * d + d // 2 + 16) + pages * (d // 2 + 16 + 2 * d)), flops=0)
    n, lens = _row_lengths(case)
    keys, pairs = _seen(case)
    q = int(n.sum()) * case["hq"]
    per_key = 2 * hkv * (d // 2 + 16) if kind == "kv4dec" else 4 * hkv * d
    if kind == "wtprompt":
        return dict(bytes=keys * (2 * hkv * d + 8) + q * (2 * d + 4), flops=2 * d * case["hq"] * pairs)
    extra = 8 * keys if kind == "wtdec" else 0
    return dict(bytes=keys * per_key + extra + q * (4 * d + 4), flops=4 * d * case["hq"] * pairs)


# ------------------------------------------------------------------ exact
def exact(case, seed):
    """The floating outputs in 64 bits, from the definitions, one row and one head at a time."""

    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "select":
        return None  # whole numbers, and copies of weights
    if kind == "kv4put":
        return _exact_put(s)
    if kind == "wtprompt":
        return _exact_rows(s)["weight"]
    got = _exact_rows(s)
    return got if kind == "wtdec" else dict(out=got["out"], lse=got["lse"])


def _exact_put(s):
    out = s["out"].double()
    for part, x in enumerate((s["k"], s["v"])):
        for grp in range(4):
            c = x[:, :, grp::4].double()
            lo, hi = c.amin(-1, keepdim=True), c.amax(-1, keepdim=True)
            scale = ((hi - lo) / 15.0).to(torch.bfloat16).double()
            code = torch.where(scale > 0, torch.round((c - lo) / torch.where(scale > 0, scale, 1.0)), 0.0)
            page = torch.arange(x.shape[0], device=x.device)
            out[page // s["ps"], part, page % s["ps"], :, grp::4] = lo + scale * code
    if s["k"].shape[0] % s["ps"]:  # slots of the last page that hold no token: all-zero records
        out[-1, :, s["k"].shape[0] % s["ps"]:] = 0.0
    return out


def _exact_values(s, pages, part, h):
    """Positions of a row's pages of one kv head in 64 bits, [tokens, d]."""

    if "cache" not in s:
        return s["kv"][pages, part, :, h].double().reshape(-1, s["kv"].shape[-1])
    rec = s["cache"][pages, part, :, h].reshape(-1, s["cache"].shape[-1])
    half = rec.shape[1] - 16
    code = torch.empty(rec.shape[0], 2 * half, dtype=torch.float64, device=rec.device)
    code[:, 0::2] = (rec[:, :half] % 16).double()
    code[:, 1::2] = (rec[:, :half] // 16).double()
    tail = rec[:, half:].contiguous().view(torch.bfloat16).double()
    grp = torch.arange(2 * half, device=rec.device) % 4
    return tail[:, 4 + grp] + tail[:, grp] * code


def _exact_rows(s):
    total, hq, d = s["q"].shape
    group = hq // s["hkv"]
    window, sinks = s.get("window", 0), s.get("sinks", 0)
    out = torch.zeros(total, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((total, hq), -math.inf, dtype=torch.float64, device="cuda")
    weight = s["weight0"].double() if "weight0" in s else None
    starts = np.concatenate([[0], np.cumsum(s["n"])])
    for r in range(len(s["lens"])):
        n, length = int(s["n"][r]), int(s["lens"][r])
        i0, i1 = int(s["kv_indptr"][r]), int(s["kv_indptr"][r + 1])
        pages = s["kv_indices"][i0:i1].long()
        for h in range(s["hkv"]):
            k = _exact_values(s, pages, 0, h)[:length]
            v = _exact_values(s, pages, 1, h)[:length] if s["kind"] != "wtprompt" else None
            for a in range(0, n, 4096):
                b = min(n, a + 4096)
                p = torch.arange(length - n + a, length - n + b, device="cuda")[:, None]
                lo = max(0, length - n + a - window + 1) if window else 0
                early = min(lo, sinks)
                pos = torch.cat([torch.arange(early, device="cuda"), torch.arange(lo, length - n + b, device="cuda")])
                hide = pos > p
                if window:
                    hide |= (pos <= p - window) & (pos >= sinks)
                rows = slice(starts[r] + a, starts[r] + b)
                for x in range(h * group, h * group + group):
                    sc = s["q"][rows, x].double() @ k[pos].t() / math.sqrt(d)
                    sc.masked_fill_(hide, -math.inf)
                    if s["kind"] == "wtprompt":
                        weight[r, pos] += torch.exp(sc - s["lse"][rows, x].double()[:, None]).sum(0)
                        continue
                    lse[rows, x] = torch.logsumexp(sc, 1)
                    pr = torch.exp(sc - lse[rows, x][:, None])
                    out[rows, x] = pr @ v[pos]
                    if weight is not None:
                        weight[r, pos] += pr.sum(0)
    return dict(out=out, lse=lse, weight=weight)
