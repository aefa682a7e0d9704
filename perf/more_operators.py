"""Timed cases of the 4-bit block cache and of the care of cache pages on one MI355X.

A stream's frames (or single query tokens) are written into a cache that
holds keys and values in 4 bits (``write``), and attended to there
(``attend``); ``step`` is one streamed frame through write, choice and
attention. ``compact`` moves the tokens that a sequence keeps to the front of
other pages. ``pages`` is one turn of a batch of branches: last turn's
branches are freed, sequences forked into new ones that share their pages,
pages reserved for the next tokens, and the shared pages among them copied.

``run`` computes them from elementary torch operations where ``own`` is
false, and through ``vasc_amd.ops`` where it is true.

The 4-bit cache, in both forms: pages of 64 tokens, found through a page
table ``[B, max_pages]``. A token's row of a head, of k and of v, is held in
groups of 32 features: e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
opposites, nearest, ties to the even code) times 2^e, e the smallest in
[-60, 60] with max|x| <= 7 * 2^e, what passes 6 * 2^e being held as that. A
value row's groups have e at least the largest of the row less 14. A token
with a value that is not finite is NaN in k and v. A page has the mean of its
keys in bf16. An 8-bit cache holds a row as e4m3 values times one such power,
max|x| <= 448 * 2^e.
"""
import math

import torch

own = False

PAGE = 64
GROUP = 32
PER_FRAME = 1041  # 5 special tokens + 28 x 37 patches of a 392x518 frame


def listed():
    return [
        # one token for each of 64 streams of uneven length: every page is touched for one row
        dict(name="write_tokens", kind="write", batch=64, tokens=1, kept=4096, heads=8, dim=128, dtype="bfloat16",
             ragged=True),
        # a clip of 32 frames behind a short one: whole pages, the first and last in part
        dict(name="write_clip", kind="write", batch=1, tokens=32 * PER_FRAME, kept=PER_FRAME, heads=16, dim=64,
             dtype="bfloat16", ragged=False),
        # one query token over four frames: latency
        dict(name="attend_token", kind="attend", batch=1, tokens=1, kept=4 * PER_FRAME, heads=16, group=1, dim=64,
             block_q=1, keep=16, causal=False, dtype="bfloat16", ragged=False),
        # single tokens of 16 long streams over every key, four query heads to a key head
        dict(name="attend_tokens", kind="attend", batch=16, tokens=1, kept=131072, heads=8, group=4, dim=128, block_q=0,
             keep=0, causal=False, dtype="bfloat16", ragged=True),
        # every key of eight streams of uneven length, float16 queries
        dict(name="attend_all_fp16", kind="attend", batch=8, tokens=1, kept=32 * PER_FRAME, heads=16, group=1, dim=64,
             block_q=0, keep=0, causal=False, dtype="float16", ragged=True),
        # a frame's queries over 128 frames, in the query blocks of the global layers, a quarter of the pages kept
        dict(name="attend_frame", kind="attend", batch=1, tokens=PER_FRAME, kept=128 * PER_FRAME, heads=16, group=1,
             dim=64, block_q=128, keep=520, causal=False, dtype="bfloat16", ragged=False),
        # a causal chunk over every key before it, the queries' own keys the last of the cache
        dict(name="attend_chunk_causal", kind="attend", batch=2, tokens=250, kept=20001, heads=8, group=4, dim=128,
             block_q=0, keep=0, causal=True, dtype="bfloat16", ragged=False),
        # one streamed frame through write, choice and attention over 32 frames
        dict(name="step_frame", kind="step", batch=1, tokens=PER_FRAME, kept=31 * PER_FRAME, heads=16, group=1, dim=64,
             block_q=128, keep=128, causal=False, dtype="bfloat16", ragged=False),
        # every head of 16 sequences keeps the quarter of its tokens that it attended to most
        dict(name="compact_heads", kind="compact", batch=16, kept=16384, share=0.25, heads=8, dim=128, bits=4,
             per_head=True, run=1, ragged=True, dtype="bfloat16"),
        # a stream forgets three of every four of its 128 frames, an 8-bit cache
        dict(name="compact_frames", kind="compact", batch=1, kept=128 * PER_FRAME, share=0.25, heads=16, dim=64, bits=8,
             per_head=False, run=PER_FRAME, ragged=False, dtype="bfloat16"),
        # eight branches of a few short sequences, a token each: latency
        dict(name="pages_branch", kind="pages", batch=4, branches=8, kept=4096, tokens=1, spare=64, heads=8, dim=128,
             bits=4, ragged=True, dtype="bfloat16"),
        # 256 branches of 64 long sequences, chunks of 250 tokens
        dict(name="pages_beams", kind="pages", batch=64, branches=256, kept=65536, tokens=250, spare=2048, heads=2,
             dim=64, bits=8, ragged=True, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _candidate(rng):
    kind = rng.choice(["write", "write", "attend", "attend", "attend", "step", "compact", "compact", "pages", "pages"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    dim = rng.choice([64, 128])
    if kind == "write":
        single = rng.random() < 0.4
        return dict(kind=kind, batch=_log_int(rng, 1, 128) if single else rng.choice([1, 1, 2, 5]),
                    tokens=1 if single else _log_int(rng, 2, 34000), kept=_log_int(rng, 1, 8000),
                    heads=rng.choice([1, 2, 8, 16]), dim=dim, dtype=rng.choice([dtype, dtype, "float32"]),
                    ragged=rng.random() < 0.5)
    if kind == "compact":
        return dict(kind=kind, batch=_log_int(rng, 1, 24), kept=_log_int(rng, 100, 60000),
                    share=rng.choice([0.05, 0.25, 0.6, 0.9]), heads=rng.choice([1, 2, 8, 16]), dim=dim,
                    bits=rng.choice([4, 8]), per_head=rng.random() < 0.5, run=rng.choice([1, 1, 7, 64, PER_FRAME]),
                    ragged=rng.random() < 0.5, dtype=dtype)
    if kind == "pages":
        batch = _log_int(rng, 1, 64)
        branches = _log_int(rng, 1, 256)
        # now and then too few pages for all
        spare = rng.choice([branches * 6, branches * 6, max(1, branches // 2)])
        return dict(kind=kind, batch=batch, branches=branches, kept=_log_int(rng, 10, 65536),
                    tokens=rng.choice([1, 1, _log_int(rng, 2, 300)]), spare=spare, heads=rng.choice([1, 2, 4]), dim=dim,
                    bits=rng.choice([4, 8]), ragged=rng.random() < 0.7, dtype=dtype)
    kept = _log_int(rng, 200, 133000)
    if kind == "step":
        return dict(kind=kind, batch=1, tokens=rng.randint(200, 1400), kept=min(kept, 40000), heads=rng.choice([4, 16]),
                    group=1, dim=64, block_q=rng.choice([64, 128]), keep=max(1, kept // PAGE // 4), causal=False,
                    dtype=dtype, ragged=False)
    group = rng.choice([1, 1, 2, 4, 5, 8])
    heads = rng.choice([1, 2, 8]) if group > 1 else rng.choice([4, 16])
    frame = rng.random() < 0.4
    tokens = _log_int(rng, 2, 1400) if frame else 1
    block_q = rng.choice([16, 64, 128]) if frame else 1
    while block_q * group > 128:
        block_q //= 2
    causal = frame and rng.random() < 0.5
    case = dict(kind=kind, batch=rng.choice([1, 2]) if frame else _log_int(rng, 1, 64), tokens=tokens,
                kept=max(kept, tokens), heads=heads, group=group, dim=dim, block_q=block_q,
                keep=max(1, round(kept / PAGE * rng.choice([0.05, 0.125, 0.25]))), causal=causal, dtype=dtype,
                ragged=rng.random() < 0.5)
    if rng.random() < 0.4:
        case["keep"], case["block_q"] = 0, 0
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def _held(case):
    """Values of the history, as a bound on what a state holds."""
    return case["kept"] * case["batch"] * case["heads"] * case["dim"]


def draw(rng):
    most, held = max(_cost(c) for c in listed()), max(_held(c) for c in listed())
    while True:
        case = _candidate(rng)
        if _cost(case) <= most and _held(case) <= held:
            return case


# ------------------------------------------------------------------ inputs
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _bits(case):
    return case.get("bits", 4)


def _lengths(case):
    """Tokens that each sequence of the case holds before the call (write, step, compact, pages) or at it (attend)."""
    n, B = case["kept"], case["batch"]
    if not case["ragged"]:
        return [n] * B
    least = case["tokens"] if case["kind"] in ("step", "attend") else 0
    return [max(least, n - (n * b * 3) // (4 * B) - 7 * b) for b in range(B)]


def _counts(case):
    """New tokens of each sequence: a padded batch where lengths are uneven."""
    T, B = case["tokens"], case["batch"]
    return [T - (T * b) // (3 * B) if case["ragged"] else T for b in range(B)]


def _max_pages(case):
    most = max(_lengths(case)) + (case["tokens"] if case["kind"] in ("write", "step", "pages") else 0)
    return max(1, -(-most // PAGE))


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, B, H, T, D, dtype):
    """[B,H,T,D]: unit rows with a slow part that neighbours share and some features larger than others, as keys have."""
    x = torch.randn(B, H, T, D, device="cuda", generator=g, dtype=torch.float32 if B * H * T * D < 1 << 28 else dtype)
    slow = torch.randn(B, H, -(-T // 48), D, device="cuda", generator=g).to(x.dtype)
    x += slow.repeat_interleave(48, 2)[:, :, :T]
    x *= torch.exp(0.5 * torch.randn(1, H, 1, D, device="cuda", generator=g)).to(x.dtype)
    return x.to(dtype)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _cache_inputs(case, seed):
    """History rows, new rows, queries, page table and lists of a case (what none of the forms changes)."""
    g = _gen(seed)
    B, H, D = case["batch"], case["heads"], case["dim"]
    dt = DTYPES[case["dtype"]]
    kind, lens, mp = case["kind"], _lengths(case), _max_pages(case)
    out = dict(case=case, lens=lens)
    if kind == "pages":
        return _pages_inputs(case, g, out)
    pages = B * mp + 3
    out_pages = -(-_kept_tokens(case) // PAGE) if kind == "compact" else 0
    shuffled = torch.randperm(pages + B * out_pages, device="cuda", generator=g).to(torch.int32)
    out.update(pages=pages + B * out_pages, table=shuffled[:B * mp].view(B, mp).contiguous())
    L = max(max(lens), 1)
    out["hk"], out["hv"] = _rows(g, B, H, L, D, dt), _rows(g, B, H, L, D, dt)
    if kind in ("write", "step"):
        out["k"], out["v"] = (_rows(g, B, H, case["tokens"], D, dt) for _ in range(2))
    if kind in ("attend", "step"):
        qd = torch.bfloat16 if dt == torch.float32 else dt
        out["q"] = _rows(g, B, H * case["group"], case["tokens"], D, qd)
    if kind == "compact":
        out["out_table"] = shuffled[B * mp:B * (mp + out_pages)].view(B, out_pages).contiguous()
        out["index"], out["count"] = _kept_lists(case, g, lens)
    elif kind == "attend":
        out["index"] = out["count"] = None
        if case["keep"]:
            # lists of a selection: the first page, the last, and `keep` others, ascending
            U = -(-case["tokens"] // case["block_q"])
            W = min(case["keep"] + 2, mp)
            r = torch.rand(B, H, U, mp, device="cuda", generator=g)
            valid = torch.tensor([-(-n // PAGE) for n in lens], device="cuda").view(B, 1, 1, 1)
            at = torch.arange(mp, device="cuda")
            r = torch.where(at < valid, r, -1.0)
            r = torch.where((at == 0) | (at == valid - 1), 2.0, r)
            idx = r.topk(W, -1).indices.sort(-1).values
            cnt = torch.minimum((r >= 0).sum(-1), torch.tensor(W, device="cuda"))
            # blocks behind the sequence sort to the end: they are no part of the list
            idx = torch.where(torch.arange(W, device="cuda") < cnt.unsqueeze(-1), idx, -1)
            out["index"], out["count"] = idx.to(torch.int32), cnt.to(torch.int32)
    return out


def _kept_counts(case):
    return [max(1, round(n * case["share"])) if n else 0 for n in _lengths(case)]


def _kept_tokens(case):
    return max(1, max(_kept_counts(case)))


def _kept_lists(case, g, lens):
    """(tokens that are kept, ascending, -1 behind them: [B,n] or [B,H,n]; how many [B]): runs of `run` tokens by chance."""
    B, H, n, run = case["batch"], case["heads"] if case["per_head"] else 1, _kept_tokens(case), case["run"]
    counts = _kept_counts(case)
    L = max(max(lens), 1)
    r = torch.rand(B, H, -(-L // run), device="cuda", generator=g).repeat_interleave(run, 2)[:, :, :L].contiguous()
    r = torch.where(torch.arange(L, device="cuda") < _ints(lens).view(B, 1, 1), r, -1.0)
    # the tokens of highest chance; equal ones (of a run) in order
    order = torch.argsort(r, dim=-1, descending=True, stable=True)[..., :n]
    kept = torch.arange(n, device="cuda") < _ints(counts).view(B, 1, 1)
    order = torch.where(kept, order, L).sort(-1).values
    order = torch.where(kept, order, -1).to(torch.int32)
    return (order if case["per_head"] else order[:, 0]).contiguous(), _ints(counts)


def _pages_inputs(case, g, out):
    """Sequences whose pages lie anywhere, holders' counts, the sequence of each branch (some have none), and the rows of
    each sequence's last page in part, which is all that a turn reads of the cache."""
    B, H, D, lens, mp = case["batch"], case["heads"], case["dim"], out["lens"], _max_pages(case)
    held = [-(-n // PAGE) for n in lens]
    pages = sum(held) + case["spare"]
    at = torch.arange(mp, device="cuda")
    live = at < _ints(held).view(B, 1)
    taken = torch.randperm(pages, device="cuda", generator=g)[:sum(held)].to(torch.int32)
    table = torch.full((B, mp), -1, device="cuda", dtype=torch.int32)
    table[live] = taken
    refs = torch.zeros(pages, device="cuda", dtype=torch.int32)
    refs[taken.long()] = 1
    source = torch.randint(0, B, (case["branches"],), device="cuda", generator=g, dtype=torch.int32)
    source = torch.where(torch.rand(case["branches"], device="cuda", generator=g) < 1 / 32, -1, source)
    out.update(pages=pages, table=table, refs=refs, source=source)
    out["hk"], out["hv"] = (_rows(g, B, H, PAGE, D, DTYPES[case["dtype"]]) for _ in range(2))
    return out


def prepare(case, seed):
    s = _cache_inputs(case, seed)
    lens, new = s["lens"], _counts(case) if case["kind"] in ("write", "step") else None
    s["start"] = _ints(lens)
    s["new"] = None if new is None else _ints(new)
    s["after"] = lens if new is None else [n + c for n, c in zip(lens, new)]
    s["lengths"] = _ints(s["after"])
    # what the cache holds of the sequences: everything, or the last page in part
    begin = [n // PAGE * PAGE if case["kind"] == "pages" else 0 for n in lens]
    size = [n - b for n, b in zip(lens, begin)]
    hk, hv = s.pop("hk"), s.pop("hv")
    if own:
        from vasc_amd import ops
        from vasc_amd.streaming import BlockCache, PagePool
        s["cache"] = BlockCache(s["pages"], case["heads"], case["dim"], bits=_bits(case))
        ops.cache_write(s["cache"], hk, hv, s["table"], _ints(begin), count=_ints(size))
        if case["kind"] == "pages":
            s["pool"] = PagePool(s["pages"])
            s["pool"].refs.copy_(s["refs"])
    else:
        s["cache"] = _plain_cache(s["pages"], case["heads"], case["dim"])
        _plain_write(s["cache"], hk, hv, s["table"], begin, size, _bits(case))
    if case["kind"] == "pages":
        s["branch"] = None
        run(s)
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from vasc_amd import ops
    case = s["case"]
    kind, cache, table = case["kind"], s["cache"], s["table"]
    if kind == "write":
        ops.cache_write(cache, s["k"], s["v"], table, s["start"], count=s["new"])
        k, v = ops.cache_read(cache, table, s["start"], case["tokens"], count=s["new"], dtype=s["k"].dtype)
        return [k, v, cache.mean]
    if kind == "compact":
        ops.cache_compact(cache, table, s["index"], s["out_table"], count=s["count"])
        k, v = ops.cache_read(cache, s["out_table"], torch.zeros_like(s["count"]), s["index"].shape[-1], count=s["count"],
                              dtype=DTYPES[case["dtype"]])
        return [k, v, cache.mean]
    if kind == "pages":
        pool, T = s["pool"], case["tokens"]
        if s["branch"] is not None:
            ops.pages_free(pool, *s["branch"])
        branch, lengths = s["branch"] = ops.pages_fork(pool, table, s["lengths"], s["source"])
        granted, src, dst = ops.pages_reserve(pool, branch, lengths, T)
        ops.cache_copy(cache, src, dst)
        k, v = ops.cache_read(cache, branch, lengths // PAGE * PAGE, PAGE, count=lengths % PAGE,
                              dtype=DTYPES[case["dtype"]])
        return [branch, lengths, granted, src, dst, pool.refs, k, v]
    rule = dict(block_q=case["block_q"], causal=case["causal"])
    if kind == "attend":
        if s["index"] is None:
            return ops.cache_attn(s["q"], cache, table, s["lengths"], causal=case["causal"])
        return ops.cache_attn(s["q"], cache, table, s["lengths"], s["index"], s["count"], **rule)
    ops.cache_write(cache, s["k"], s["v"], table, s["start"])
    index, count = ops.cache_select(s["q"], cache, table, s["lengths"], case["keep"], **rule)
    o = ops.cache_attn(s["q"], cache, table, s["lengths"], index, count, **rule)
    return [cache.mean, index, count, o]


# ------------------------------------------------------------------ the plain form
def _plain(s):
    case = s["case"]
    kind, cache, table, new = case["kind"], s["cache"], s["table"], [b - a for a, b in zip(s["lens"], s["after"])]
    if kind == "write":
        _plain_write(cache, s["k"], s["v"], table, s["lens"], new, 4)
        k, v = _plain_read(cache, table, s["lens"], case["tokens"], new, s["k"].dtype)
        return [k, v, cache["mean"]]
    if kind == "compact":
        counts, n = _kept_counts(case), s["index"].shape[-1]
        _plain_compact(cache, table, s["index"], s["out_table"], counts)
        k, v = _plain_read(cache, s["out_table"], [0] * len(counts), n, counts, DTYPES[case["dtype"]])
        return [k, v, cache["mean"]]
    if kind == "pages":
        return _plain_pages(s)
    if kind == "attend":
        block_q = case["block_q"] or case["tokens"]
        return _plain_attend(s["q"], cache, table, s["after"], s["index"], s["count"], block_q, case["causal"])
    _plain_write(cache, s["k"], s["v"], table, s["lens"], new, 4)
    index, count = _plain_select(s["q"], cache, table, s["after"], case["keep"], case["block_q"])
    o = _plain_attend(s["q"], cache, table, s["after"], index, count, case["block_q"], False)
    return [cache["mean"], index, count, o]


def _plain_cache(pages, heads, dim):
    """The values that the cache holds, which are exact in bf16."""
    return {name: torch.zeros(pages, heads, *row, dim, device="cuda", dtype=torch.bfloat16)
            for name, row in (("k", (PAGE,)), ("v", (PAGE,)), ("mean", ()))}


def _power(e):
    """2^e in float32, from its bits (a library's pow may be off in the last place)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _exponent(top, limit):
    """The smallest e in [-60, 60] with top <= limit * 2^e; limit: 7 (0.875 * 2^3) or 448 (0.875 * 2^9)."""
    m, e = torch.frexp(top)
    e = e - (3 if limit == 7 else 9) + (m > 0.875).to(e.dtype)
    return torch.where(top == 0, torch.full_like(e, -60), e.clamp(-60, 60))


def _to_e2m1(y):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code; what passes 6 is 6."""
    a = y.abs()
    low = torch.round(a * 2) * 0.5               # steps of 0.5 up to 2
    mid = torch.round(a)                         # of 1 up to 4
    high = torch.round(a * 0.5) * 2              # of 2
    v = torch.where(a < 2, low, torch.where(a < 4, mid, high)).clamp_max(6.0)
    return torch.where(y < 0, -v, v)


def _quantise(x, fine, bits, value):
    """What the cache holds of rows [..., D]; rows that are not `fine` are NaN."""
    x = torch.where(fine.unsqueeze(-1), x.float(), torch.zeros((), device=x.device))
    if bits == 8:
        e = _exponent(x.abs().amax(-1, keepdim=True), 448)
        y = (x * _power(-e)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float() * _power(e)
    else:
        xg = x.unflatten(-1, (-1, GROUP))
        e = _exponent(xg.abs().amax(-1, keepdim=True), 7)
        if value:
            e = torch.maximum(e, e.amax(-2, keepdim=True) - 14)
        y = (_to_e2m1(xg * _power(-e)) * _power(e)).flatten(-2)
    return torch.where(fine.unsqueeze(-1), y, math.nan).bfloat16()


def _places(table, start, new):
    """(sequence, token, page, slot) of every new token."""
    b = torch.cat([torch.full((n,), i) for i, n in enumerate(new)]).cuda()
    t = torch.cat([torch.arange(n) for n in new]).cuda()
    pos = torch.tensor(start, device="cuda")[b] + t
    return b, t, table[b, pos // PAGE].long(), pos % PAGE


def _plain_write(cache, k, v, table, start, new, bits):
    b, t, page, slot = _places(table, start, new)
    for lo in range(0, b.numel(), 1 << 17):
        part = slice(lo, lo + (1 << 17))
        rk, rv = k[b[part], :, t[part]], v[b[part], :, t[part]]
        fine = rk.isfinite().all(-1) & rv.isfinite().all(-1)
        cache["k"][page[part], :, slot[part]] = _quantise(rk, fine, bits, False)
        cache["v"][page[part], :, slot[part]] = _quantise(rv, fine, bits, True)
    _plain_means(cache, table, start, new)


def _plain_means(cache, table, start, new):
    # the pages that were touched: (sequence, page of it, tokens it holds now)
    touched = [(i, j, min(PAGE, at + n - j * PAGE)) for i, (at, n) in enumerate(zip(start, new)) if n
               for j in range(at // PAGE, (at + n - 1) // PAGE + 1)]
    for lo in range(0, len(touched), 1024):
        i, j, filled = torch.tensor(touched[lo:lo + 1024], device="cuda").unbind(1)
        ids = table[i, j].long()
        live = torch.arange(PAGE, device="cuda") < filled[:, None]
        vals = cache["k"][ids].double()
        total = torch.where(live[:, None, :, None], vals, torch.zeros_like(vals)).sum(2)
        cache["mean"][ids] = (total / filled[:, None, None]).float().bfloat16()


def _plain_read(cache, table, start, tokens, new, dtype):
    B, (H, _, D) = table.shape[0], cache["k"].shape[1:]
    out = [torch.zeros(B, H, tokens, D, device="cuda", dtype=dtype) for _ in range(2)]
    b, t, page, slot = _places(table, start, new)
    for o, name in zip(out, ("k", "v")):
        o[b, :, t] = cache[name][page, :, slot].to(dtype)
    return out


def _plain_compact(cache, table, index, out_table, counts):
    H = cache["k"].shape[1]
    head = torch.arange(H, device="cuda")
    index = index if index.dim() == 3 else index.unsqueeze(1).expand(-1, H, -1)
    b, t, page, slot = _places(out_table, [0] * len(counts), counts)
    for lo in range(0, b.numel(), 1 << 17):
        part = slice(lo, lo + (1 << 17))
        at = index[b[part], :, t[part]].long()  # [n,H]
        ids = table[b[part].unsqueeze(1), at // PAGE].long()
        for name in ("k", "v"):
            cache[name][page[part], :, slot[part]] = cache[name][ids, head, at % PAGE]
    _plain_means(cache, out_table, [0] * len(counts), counts)


def _plain_pages(s):
    """Free, fork, reserve, copy: the pages' holders are counted, free pages are handed out from the lowest."""
    case, table, lens, source, refs, cache = s["case"], s["table"], s["lengths"], s["source"], s["refs"], s["cache"]
    T, P = case["tokens"], s["pages"]
    mp = table.shape[1]
    if s["branch"] is not None:
        last = s["branch"][0]
        refs.index_add_(0, last.clamp_min(0).flatten().long(), -(last >= 0).flatten().int())
    # a branch shares the pages that hold its sequence's tokens
    at = torch.arange(mp, device="cuda")
    live = source >= 0
    lengths = torch.where(live, lens[source.clamp_min(0).long()], 0).to(torch.int32)
    shared = at < ((lengths + PAGE - 1) // PAGE).unsqueeze(1)
    branch = torch.where(shared, table[source.clamp_min(0).long()], -1)
    refs.index_add_(0, branch.clamp_min(0).flatten().long(), shared.flatten().int())
    # pages of the next T tokens: those that are missing, and those that others hold too
    fit = (mp * PAGE - lengths).clamp(0, T)
    span = (T + PAGE - 2) // PAGE + 1
    j = (lengths // PAGE).unsqueeze(1) + torch.arange(span, device="cuda")
    touched = (j * PAGE < (lengths + fit).unsqueeze(1)) & (fit > 0).unsqueeze(1)
    have = branch.gather(1, j.clamp_max(mp - 1).long())
    alone = (have >= 0) & (refs[have.clamp_min(0).long()] == 1)
    need = touched & ~alone
    wanted = need.sum(1)
    end = wanted.cumsum(0)
    ok = end <= (refs <= 0).sum()
    granted = torch.where(ok, fit, 0).to(torch.int32)
    take = need & ok.unsqueeze(1)
    rank = (end - wanted).unsqueeze(1) + need.long().cumsum(1) - 1
    free = torch.argsort((refs > 0).int(), stable=True)
    page = torch.where(take, free[rank.clamp(0, P - 1)].int(), have)
    keep_row = torch.cat([branch, torch.zeros(branch.shape[0], 1, device="cuda", dtype=torch.int32)], 1)
    keep_row.scatter_(1, torch.where(touched, j, mp).long(), page)  # a last column takes what is not written
    branch = keep_row[:, :mp].contiguous()
    refs.index_add_(0, have.clamp_min(0).flatten().long(), -(take & (have >= 0)).flatten().int())
    refs.index_add_(0, page.clamp_min(0).flatten().long(), take.flatten().int())
    # the page that holds tokens in part is copied
    part = take[:, 0] & (lengths % PAGE > 0) & (have[:, 0] >= 0)
    src, dst = torch.where(part, have[:, 0], -1), torch.where(part, page[:, 0], -1)
    at = part.nonzero().flatten()
    for name in ("k", "v", "mean"):
        cache[name][dst[at].long()] = cache[name][src[at].long()]
    s["branch"] = branch, lengths
    slot = torch.arange(PAGE, device="cuda")
    ids = branch.gather(1, (lengths // PAGE).clamp_max(mp - 1).unsqueeze(1).long()).squeeze(1)
    seen = (slot < (lengths % PAGE).unsqueeze(1)) & (ids >= 0).unsqueeze(1)
    seen = seen & (lengths // PAGE < mp).unsqueeze(1)
    k, v = (torch.where(seen[:, None, :, None], cache[name][ids.clamp_min(0).long()], 0.0).to(DTYPES[case["dtype"]])
            for name in ("k", "v"))
    return [branch, lengths, granted, src, dst, refs, k, v]


def _plain_select(q, cache, table, lens, keep, block_q):
    """Per query block and key head: the first page, the last, and the `keep` of largest score among the others,
    ascending, -1 behind."""
    B, H, T, D = q.shape
    mp, U = table.shape[1], -(-T // block_q)
    W = min(1 + keep + 1, mp)
    index = torch.full((B, H, U, W), -1, device="cuda", dtype=torch.int32)
    count = torch.zeros(B, H, U, device="cuda", dtype=torch.int32)
    at = torch.arange(mp, device="cuda")
    for b in range(B):
        means = cache["mean"][table[b].long()].double().permute(1, 2, 0).contiguous()  # [H,D,mp]
        seen = -(-lens[b] // PAGE)
        for u in range(U):
            t0, t1 = u * block_q, min((u + 1) * block_q, T)
            qm = (q[b, :, t0:t1].double().sum(1) / (t1 - t0)).float().bfloat16().double()
            score = torch.matmul(qm.unsqueeze(1), means).squeeze(1).float()
            forced = ((at < 1) | (at >= seen - 1)) & (at < seen)
            free = (~forced & (at < seen)).expand(H, mp)
            # equal scores: the stable order keeps the lowest index first
            key = torch.where(free & ~score.isnan(), score, torch.full_like(score, -math.inf))
            order = torch.argsort(key, dim=-1, descending=True, stable=True)
            order = order.gather(1, torch.argsort((~free).gather(1, order).int(), dim=-1, stable=True))
            rank = torch.empty_like(order).scatter_(1, order, at.expand(H, mp))
            chosen = forced | (free & (rank < keep))
            n = chosen.sum(-1)
            first = torch.argsort((~chosen).int(), dim=-1, stable=True)[:, :W]
            index[b, :, u] = torch.where(at[:W] < n[:, None], first, -1).to(torch.int32)
            count[b, :, u] = n.to(torch.int32)
    return index, count


def _plain_attend(q, cache, table, lens, index, count, block_q, causal):
    B, Hq, T, D = q.shape
    H = cache["k"].shape[1]
    G, scale = Hq // H, D ** -0.5
    out = torch.zeros(B, Hq, T, D, device="cuda", dtype=q.dtype)
    head = torch.arange(H, device="cuda")[:, None]
    for b in range(B):
        qb, ob = q[b].reshape(H, G, T, D), out[b].view(H, G, T, D)
        for t0 in range(0, T, block_q):
            t1, u = min(t0 + block_q, T), t0 // block_q
            if index is None:
                pages = torch.arange(-(-lens[b] // PAGE), device="cuda").expand(H, -1)
                live = torch.ones_like(pages, dtype=torch.bool)
            else:
                pages = index[b, :, u].long()
                live = torch.arange(pages.shape[1], device="cuda") < count[b, :, u][:, None]
                pages = torch.where(live, pages, 0)
            ids = table[b].long()[pages]
            k = cache["k"][ids, head].float().flatten(1, 2)  # [H,W*64,D]
            v = cache["v"][ids, head].float().flatten(1, 2)
            key = (pages[..., None] * PAGE + torch.arange(PAGE, device="cuda")).flatten(1)
            seen = (live[..., None].expand(-1, -1, PAGE).flatten(1) & (key < lens[b]))[:, None, :]
            if causal:
                row = lens[b] - T + torch.arange(t0, t1, device="cuda").repeat(G)
                seen = seen & (key[:, None, :] <= row[None, :, None])
            x = torch.matmul(qb[:, :, t0:t1].reshape(H, -1, D).float(), k.transpose(1, 2).contiguous()) * scale
            x = torch.where(seen, x, -math.inf)
            top = x.amax(-1, keepdim=True)
            e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = e.sum(-1, keepdim=True)
            v = torch.where(seen.any(1).unsqueeze(-1), v, torch.zeros_like(v))
            o = torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)
            ob[:, :, t0:t1] = o.view(H, G, t1 - t0, D).to(q.dtype)
    return out


# ------------------------------------------------------------------ work
def work(case):
    size = {"bfloat16": 2, "float16": 2, "float32": 4}[case["dtype"]]
    D, B, H, bits = case["dim"], case["batch"], case["heads"], _bits(case)
    # bytes of a row of k or of v in the cache
    row = D + 1 if bits == 8 else D // 2 + D // GROUP
    lens = _lengths(case)
    if case["kind"] == "write":
        n = sum(_counts(case))
        pages = sum(-(-(s + c) // PAGE) - s // PAGE for s, c in zip(lens, _counts(case)))
        # read, written, read back, written out; a touched page's key mean
        return {"bytes": 2 * n * H * (2 * size * D + 2 * row) + 2 * pages * H * D, "flops": 6 * n * H * D}
    if case["kind"] == "compact":
        n = sum(_kept_counts(case))
        # read, written, read back, written out; a touched page's key mean; the lists
        return {"bytes": n * H * (2 * 3 * row + 2 * size * D) + 2 * (n // PAGE + B) * H * D
                + 4 * n * (H if case["per_head"] else 1), "flops": n * H * D}
    if case["kind"] == "pages":
        # table rows read and written, holders' counts of the pages read and written, twice; the copied pages, read again
        entries = case["branches"] * sum(-(-x // PAGE) for x in lens) // B
        pages = sum(-(-x // PAGE) for x in lens) + case["spare"]
        copied = case["branches"] * H * (2 * PAGE * row + 2 * D)
        out = 2 * case["branches"] * H * PAGE * D * size
        return {"bytes": 2 * 2 * 4 * entries + 2 * 2 * 4 * pages + 3 * copied + out, "flops": 2 * entries}
    T, G = case["tokens"], case["group"]
    lens = [n + (T if case["kind"] == "step" else 0) for n in lens]
    block_q = case["block_q"] or T
    units = -(-T // block_q)
    nbytes = 2 * 2 * B * T * H * G * D
    nflops = 0
    for L in lens:
        held = -(-L // PAGE)
        if case["kind"] == "step":
            nbytes += held * H * D * 2 + units * H * 4 * min(held, case["keep"] + 2)
            nflops += 2 * units * held * H * D
        w = min(held, case["keep"] + 2) if case["keep"] else held
        # pages that any of the units lists, were the lists drawn apart
        union = held * (1.0 - (1.0 - w / held) ** units) if held else 0
        nbytes += int(min(union * PAGE, L)) * H * 2 * row
        keys = min(w * PAGE, L) - (T / 2 if case["causal"] else 0)
        nflops += int(4 * D * T * H * G * keys)
    if case["kind"] == "step":
        nbytes += 2 * B * T * H * (size * D + row)
    return {"bytes": int(nbytes), "flops": int(nflops)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _two(n):
    return ((n.long() + 1023) << 52).view(torch.float64)  # 2^n, exactly


def _exact_power(top, limit):
    """The smallest exponent in [-60, 60] with top <= limit * 2^e, by trying."""
    e = torch.ceil(torch.log2(top / limit)).clamp(-60, 60)
    e = torch.where((top > limit * _two(e)) & (e < 60), e + 1, e)
    return torch.where((top <= limit * _two(e - 1)) & (e > -60), e - 1, e)


def _exact_rows(x, bits, value):
    """float64 values that a cached row stands for: each value to the nearest multiple of its step."""
    x = x.double()
    if bits == 8:
        e, steps, least, largest = _exact_power(x.abs().amax(-1, keepdim=True), 448.0), 3, -6, 448.0
    else:
        x = x.unflatten(-1, (-1, GROUP))
        e, steps, least, largest = _exact_power(x.abs().amax(-1, keepdim=True), 7.0), 1, 0, 6.0
        if value:
            e = torch.maximum(e, e.amax(-2, keepdim=True) - 14)
    y = x / _two(e)
    binade = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20)))
    binade = torch.where(y.abs() >= _two(binade + 1), binade + 1, binade)
    binade = torch.where(y.abs() < _two(binade), binade - 1, binade)
    step = _two(binade.clamp_min(least) - steps)
    y = (torch.round(y / step) * step).clamp(-largest, largest) * _two(e)
    return y if bits == 8 else y.flatten(-2)


def _exact_means(case, rows, lens, table, mean):
    """Means of the pages of 64 rows each [H,L,D] that every sequence has."""
    for b, n in enumerate(lens):
        for j, part in enumerate(rows[b][:, :n].split(PAGE, 1) if n else ()):
            mean[table[b, j]] = part.mean(1)


def exact(case, seed):
    s = _cache_inputs(case, seed)
    lens, bits, kind = s["lens"], _bits(case), case["kind"]
    B, H, D = case["batch"], case["heads"], case["dim"]
    zeros = dict(device="cuda", dtype=torch.float64)
    if kind == "pages":
        lengths = [lens[b] if b >= 0 else 0 for b in s["source"].tolist()]
        k, v = torch.zeros(len(lengths), H, PAGE, D, **zeros), torch.zeros(len(lengths), H, PAGE, D, **zeros)
        for i, b in enumerate(s["source"].tolist()):
            n = lengths[i] % PAGE
            if n:  # a branch that gets no pages keeps the one that it shares
                k[i, :, :n] = _exact_rows(s["hk"][b, :, :n], bits, False)
                v[i, :, :n] = _exact_rows(s["hv"][b, :, :n], bits, True)
        return [None, None, None, None, None, None, k, v]
    table = s["table"].long()
    mean = torch.zeros(s["pages"], H, D, **zeros)
    if kind == "compact":
        out_table, counts, n = s["out_table"].long(), _kept_counts(case), s["index"].shape[-1]
        ko, vo = torch.zeros(B, H, n, D, **zeros), torch.zeros(B, H, n, D, **zeros)
        for b in range(B):
            for h in range(H):
                at = (s["index"][b, h] if case["per_head"] else s["index"][b])[:counts[b]].long()
                kr = _exact_rows(s["hk"][b, h, :lens[b]], bits, False)
                ko[b, h, :counts[b]] = kr[at]
                vo[b, h, :counts[b]] = _exact_rows(s["hv"][b, h].index_select(0, at), bits, True)
                whole = lens[b] // PAGE
                mean[table[b, :whole], h] = kr[:whole * PAGE].view(-1, PAGE, D).mean(1)
                if lens[b] % PAGE:
                    mean[table[b, whole], h] = kr[whole * PAGE:].mean(0)
        _exact_means(case, ko, counts, out_table, mean)
        return [ko, vo, mean]
    if kind in ("write", "step"):
        ko = torch.zeros(s["k"].shape, **zeros)
        vo = torch.zeros_like(ko)
        stream = []
        for b, (old, new) in enumerate(zip(lens, _counts(case))):
            kb = _exact_rows(torch.cat([s["hk"][b, :, :old], s["k"][b, :, :new]], 1), bits, False)
            ko[b, :, :new] = kb[:, old:]
            vo[b, :, :new] = _exact_rows(s["v"][b, :, :new], bits, True)
            _exact_means(case, kb.unsqueeze(0), [old + new], table[b:b + 1], mean)
            if kind == "step":
                stream.append((kb, torch.cat([_exact_rows(s["hv"][b, :, :old], bits, True), vo[b]], 1)))
        if kind == "write":
            return [ko, vo, mean]
        means = mean.float().bfloat16().double()  # the score is defined on what the cache holds
        return [mean, None, None, _exact_attend(case, s["q"], lambda b, h: (stream[b][0][h], stream[b][1][h]),
                                                lambda b, h, u: _exact_choice(case, s["q"], means, table, b, h, u))]
    if s["index"] is None:
        def pages(b, h, u):
            return torch.arange(-(-lens[b] // PAGE), device="cuda")
    else:
        def pages(b, h, u):
            return s["index"][b, h, u, :s["count"][b, h, u]].long()
    return _exact_attend(case, s["q"], lambda b, h: (_exact_rows(s["hk"][b, h, :lens[b]], bits, False),
                                                     _exact_rows(s["hv"][b, h, :lens[b]], bits, True)), pages)


def _exact_choice(case, q, means, table, b, h, u):
    """Pages that query block u of a step's one sequence chooses."""
    n = -(-(_lengths(case)[b] + case["tokens"]) // PAGE)
    qm = q[b, h, u * case["block_q"]:(u + 1) * case["block_q"]].double().mean(0).float().bfloat16().double()
    score = ((means[table[b, 1:n - 1], h] * qm).sum(-1).float().tolist()) if n > 2 else []
    best = sorted(range(len(score)), key=lambda j: (-score[j], j))[:case["keep"]]
    return torch.tensor(sorted({0, n - 1, *(j + 1 for j in best)}), device="cuda")


def _exact_attend(case, q, rows, pages):
    B, Hq, T, D = q.shape
    G, block_q = case["group"], case["block_q"] or T
    out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
    for b in range(B):
        for h in range(Hq // G):
            k, v = rows(b, h)
            L = k.shape[0]
            for t0 in range(0, T, block_q):
                t1 = min(t0 + block_q, T)
                p = pages(b, h, t0 // block_q)
                at = (p[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()
                at = at[at < L]
                kk, vv = (k, v) if at.numel() == L else (k[at], v[at])
                for g in range(G):
                    x = q[b, h * G + g, t0:t1].double() @ kk.T / math.sqrt(D)
                    if case["causal"]:
                        x = x.masked_fill(at[None, :] > (L - T + torch.arange(t0, t1, device="cuda"))[:, None], -math.inf)
                    out[b, h * G + g, t0:t1] = torch.softmax(x, -1) @ vv
    return out
