"""Timed cases of the streamed global layer's operators on one MI355X.

A stream's frames (or single query tokens) go through four operators: the
rotary embedding over several axes (``rotary``), the write into an 8-bit
block cache and the read of it (``write``), the choice of cache blocks by a
cheap score (``select``), and attention over the chosen blocks (``attend``).
``step`` is one streamed frame through write, choice and attention.

``run`` computes them from elementary torch operations where ``own`` is
false, and through ``vasc_amd.ops`` where it is true.

The cache, in both forms: pages of 64 tokens, found through a page table
``[B, max_pages]``; each (token, head) row of k and of v is held as e4m3
values times a power of two (a token's row with a value that is not finite,
in k or in v, as NaN in both); each page has the mean of its keys in bf16.
"""
import math

import torch

own = False

PAGE = 64
E4M3_MAX = 448.0
PER_FRAME = 1041  # 5 special tokens + 28 x 37 patches of a 392x518 frame


def listed():
    return [
        # q and k of one streamed frame: the smallest rotary call, launch-bound
        dict(name="rotary_frame", kind="rotary", batch=1, tokens=PER_FRAME, heads_q=16, heads_k=16, dim=64, st=16, sh=24,
             sw=24, dtype="bfloat16", train=False, first=1000),
        # a clip of 24 frames, forward and backward as a training step calls them
        dict(name="rotary_clip_train", kind="rotary", batch=1, tokens=24 * PER_FRAME, heads_q=16, heads_k=16, dim=64,
             st=16, sh=24, sw=24, dtype="bfloat16", train=True, first=0),
        # one token for each of 64 streams of uneven length: every page is touched for one row
        dict(name="write_tokens", kind="write", batch=64, tokens=1, kept=4096, heads=8, dim=128, dtype="bfloat16",
             ragged=True),
        # a clip of 32 frames behind a short one: whole pages, the first and last in part
        dict(name="write_clip", kind="write", batch=1, tokens=32 * PER_FRAME, kept=PER_FRAME, heads=16, dim=64,
             dtype="bfloat16", ragged=False),
        # single tokens of 16 long streams, four query heads to a key head
        dict(name="select_tokens", kind="select", batch=16, tokens=1, kept=131072, heads=8, group=4, dim=128, block_q=1,
             keep=256, causal=False, dtype="bfloat16", ragged=True),
        # a frame's queries over 128 frames, in the query blocks of the global layers, a quarter of the pages kept
        dict(name="select_frame", kind="select", batch=1, tokens=PER_FRAME, kept=128 * PER_FRAME, heads=16, group=1,
             dim=64, block_q=128, keep=520, causal=False, dtype="bfloat16", ragged=False),
        # one query token over four frames: latency
        dict(name="attend_token", kind="attend", batch=1, tokens=1, kept=4 * PER_FRAME, heads=16, group=1, dim=64,
             block_q=1, keep=16, causal=False, dtype="bfloat16", ragged=False),
        # the lists of select_tokens
        dict(name="attend_tokens", kind="attend", batch=16, tokens=1, kept=131072, heads=8, group=4, dim=128, block_q=1,
             keep=256, causal=False, dtype="bfloat16", ragged=True),
        # the lists of select_frame
        dict(name="attend_frame", kind="attend", batch=1, tokens=PER_FRAME, kept=128 * PER_FRAME, heads=16, group=1,
             dim=64, block_q=128, keep=520, causal=False, dtype="bfloat16", ragged=False),
        # every key of eight streams of uneven length, float16 queries
        dict(name="attend_all_fp16", kind="attend", batch=8, tokens=1, kept=32 * PER_FRAME, heads=16, group=1, dim=64,
             block_q=1, keep=0, causal=False, dtype="float16", ragged=True),
        # a causal chunk over every key before it, the queries' own keys the last of the cache
        dict(name="attend_chunk_causal", kind="attend", batch=2, tokens=250, kept=20001, heads=8, group=4, dim=128,
             block_q=0, keep=0, causal=True, dtype="bfloat16", ragged=False),
        # one streamed frame through write, choice and attention over 32 frames
        dict(name="step_frame", kind="step", batch=1, tokens=PER_FRAME, kept=31 * PER_FRAME, heads=16, group=1, dim=64,
             block_q=128, keep=128, causal=False, dtype="bfloat16", ragged=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _candidate(rng):
    kind = rng.choice(["rotary", "rotary", "write", "write", "select", "select", "attend", "attend", "attend", "step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    dim = rng.choice([64, 128])
    if kind == "rotary":
        quarter = rng.choice([dim // 4, dim // 8, 6])
        side = (dim - quarter) // 2 // 2 * 2
        heads = rng.choice([4, 8, 16, 32])
        return dict(kind=kind, batch=rng.choice([1, 1, 2, 3]), tokens=_log_int(rng, 1, 30000), heads_q=heads,
                    heads_k=rng.choice([heads, max(1, heads // 4)]), dim=dim, st=quarter, sh=side, sw=side,
                    dtype=rng.choice([dtype, dtype, "float32"]), train=rng.random() < 0.5, first=_log_int(rng, 1, 100000))
    if kind == "write":
        single = rng.random() < 0.4
        return dict(kind=kind, batch=_log_int(rng, 1, 128) if single else rng.choice([1, 1, 2, 5]),
                    tokens=1 if single else _log_int(rng, 2, 34000), kept=_log_int(rng, 1, 8000),
                    heads=rng.choice([1, 2, 8, 16]), dim=dim, dtype=rng.choice([dtype, dtype, "float32"]),
                    ragged=rng.random() < 0.5)
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
    if kind == "attend" and rng.random() < 0.3:
        case["keep"], case["block_q"] = 0, 0
    return case


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def _held(case):
    """Values of the history, as a bound on what a state holds."""
    return case.get("kept", 0) * case["batch"] * case.get("heads", 1) * case["dim"]


def draw(rng):
    most, held = max(_cost(c) for c in listed()), max(_held(c) for c in listed())
    while True:
        case = _candidate(rng)
        if _cost(case) <= most and _held(case) <= held:
            return case


# ------------------------------------------------------------------ inputs
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def _lengths(case):
    """Tokens that each sequence of the case holds before the call (write, step) or at it (select, attend)."""
    n, B = case["kept"], case["batch"]
    if not case["ragged"]:
        return [n] * B
    return [max(case["tokens"] if case["kind"] != "write" else 0, n - (n * b * 3) // (4 * B) - 7 * b) for b in range(B)]


def _counts(case):
    """New tokens of each sequence: a padded batch where lengths are uneven."""
    T, B = case["tokens"], case["batch"]
    return [T - (T * b) // (3 * B) if case["ragged"] else T for b in range(B)]


def _max_pages(case):
    most = max(_lengths(case)) + (case["tokens"] if case["kind"] in ("write", "step") else 0)
    return -(-most // PAGE)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, B, H, T, D, dtype):
    """[B,H,T,D]: unit rows with a slow part that neighbours share and some features larger than others, as keys have."""
    x = torch.randn(B, H, T, D, device="cuda", generator=g, dtype=torch.float32 if B * H * T * D < 1 << 28 else dtype)
    slow = torch.randn(B, H, -(-T // 48), D, device="cuda", generator=g).to(x.dtype)
    x += slow.repeat_interleave(48, 2)[:, :, :T]
    x *= torch.exp(0.5 * torch.randn(1, H, 1, D, device="cuda", generator=g)).to(x.dtype)
    return x.to(dtype)


def _rotary_inputs(case, seed):
    g = _gen(seed)
    B, T, D = case["batch"], case["tokens"], case["dim"]
    dt = DTYPES[case["dtype"]]

    def heads(n):
        # the projection's rows [B,T,H,D] seen as [B,H,T,D]
        return torch.randn(B, T, n, D, device="cuda", generator=g).to(dt).transpose(1, 2)

    q, k = heads(case["heads_q"]), heads(case["heads_k"])
    gq, gk = (heads(case["heads_q"]), heads(case["heads_k"])) if case["train"] else (None, None)
    t = torch.arange(T, device="cuda")
    cell = t % PER_FRAME - 5
    pos = torch.stack([case["first"] + t // PER_FRAME, torch.where(cell < 0, 0, cell // 37 + 1),
                       torch.where(cell < 0, 0, cell % 37 + 1)], -1).to(torch.int32)
    pos = pos.unsqueeze(0).repeat(B, 1, 1)
    pos[:, :, 0] += torch.randint(0, 1000, (B, 1), device="cuda", generator=g, dtype=torch.int32)
    sections = (case["st"], case["sh"], case["sw"])
    freq = torch.cat([base ** (-torch.arange(0, s, 2, dtype=torch.float64) / s)
                      for s, base in zip(sections, (10000.0, 100.0, 100.0))]).cuda()
    return q, k, gq, gk, pos, sections, freq


def _cache_inputs(case, seed):
    """History rows, new rows, queries, page table and lists of a case (what none of the forms changes)."""
    g = _gen(seed)
    B, H, D, T = case["batch"], case["heads"], case["dim"], case["tokens"]
    dt = DTYPES[case["dtype"]]
    lens, mp = _lengths(case), _max_pages(case)
    pages = B * mp + 3
    table = torch.randperm(pages, device="cuda", generator=g)[:B * mp].view(B, mp).to(torch.int32)
    out = dict(case=case, lens=lens, pages=pages, table=table)
    L = max(max(lens), 1)
    out["hk"], out["hv"] = _rows(g, B, H, L, D, dt), _rows(g, B, H, L, D, dt)
    if case["kind"] in ("write", "step"):
        out["k"], out["v"] = _rows(g, B, H, T, D, dt), _rows(g, B, H, T, D, dt)
    if case["kind"] != "write":
        qd = torch.bfloat16 if dt == torch.float32 else dt
        out["q"] = _rows(g, B, H * case["group"], T, D, qd)
    out["index"] = out["count"] = None
    if case["kind"] == "attend" and case["keep"]:
        # lists of a selection: the first page, the last, and `keep` others, ascending
        U = -(-T // case["block_q"])
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


def prepare(case, seed):
    if case["kind"] == "rotary":
        q, k, gq, gk, pos, sections, freq = _rotary_inputs(case, seed)
        if own and case["train"]:
            q, k = q.requires_grad_(), k.requires_grad_()
        return dict(case=case, q=q, k=k, gq=gq, gk=gk, pos=pos, sections=sections, freq=freq)
    s = _cache_inputs(case, seed)
    dev = dict(device="cuda", dtype=torch.int32)
    s["start"] = torch.tensor(s["lens"], **dev)
    counts = _counts(case) if case["kind"] in ("write", "step") else None
    s["new"] = None if counts is None else torch.tensor(counts, **dev)
    after = s["lens"] if counts is None else [n + c for n, c in zip(s["lens"], counts)]
    s["after"], s["lengths"] = after, torch.tensor(after, **dev)
    zero = torch.zeros_like(s["start"])
    hk, hv = s.pop("hk"), s.pop("hv")
    if own:
        from vasc_amd import ops
        from vasc_amd.streaming import BlockCache
        s["cache"] = BlockCache(s["pages"], case["heads"], case["dim"])
        ops.cache_write(s["cache"], hk, hv, s["table"], zero, count=s["start"])
    else:
        s["cache"] = _plain_cache(s["pages"], case["heads"], case["dim"])
        _plain_write(s["cache"], hk, hv, s["table"], [0] * len(s["lens"]), s["lens"])
    return s


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from vasc_amd import ops
    case = s["case"]
    kind = case["kind"]
    if kind == "rotary":
        qo, ko = ops.rotary_axes(s["q"], s["k"], s["pos"], s["sections"], s["freq"])
        if not case["train"]:
            return [qo, ko]
        dq, dk = torch.autograd.grad([qo, ko], [s["q"], s["k"]], [s["gq"], s["gk"]])
        return [qo.detach(), ko.detach(), dq, dk]
    cache, table = s["cache"], s["table"]
    if kind == "write":
        ops.cache_write(cache, s["k"], s["v"], table, s["start"], count=s["new"])
        k, v = ops.cache_read(cache, table, s["start"], case["tokens"], count=s["new"], dtype=s["k"].dtype)
        return [k, v, cache.mean]
    rule = dict(block_q=case["block_q"], causal=case["causal"])
    if kind == "select":
        return list(ops.cache_select(s["q"], cache, table, s["lengths"], case["keep"], want_score=True, **rule))
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
    kind = case["kind"]
    if kind == "rotary":
        out = [_plain_rotary(s["q"], s["pos"], s["sections"], s["freq"], 1.0),
               _plain_rotary(s["k"], s["pos"], s["sections"], s["freq"], 1.0)]
        if case["train"]:
            out += [_plain_rotary(s["gq"], s["pos"], s["sections"], s["freq"], -1.0),
                    _plain_rotary(s["gk"], s["pos"], s["sections"], s["freq"], -1.0)]
        return out
    cache, table, new = s["cache"], s["table"], [b - a for a, b in zip(s["lens"], s["after"])]
    if kind == "write":
        _plain_write(cache, s["k"], s["v"], table, s["lens"], new)
        k, v = _plain_read(cache, table, s["lens"], case["tokens"], new, s["k"].dtype)
        return [k, v, cache["mean"]]
    if kind == "select":
        return list(_plain_select(s["q"], cache, table, s["after"], case["keep"], case["block_q"], case["causal"]))
    if kind == "attend":
        block_q = case["block_q"] or case["tokens"]
        return _plain_attend(s["q"], cache, table, s["after"], s["index"], s["count"], block_q, case["causal"])
    _plain_write(cache, s["k"], s["v"], table, s["lens"], new)
    index, count, _ = _plain_select(s["q"], cache, table, s["after"], case["keep"], case["block_q"], False)
    o = _plain_attend(s["q"], cache, table, s["after"], index, count, case["block_q"], False)
    return [cache["mean"], index, count, o]


def _plain_rotary(x, pos, sections, freq, sign):
    """Pairs (j, j + d/2) of each axis' section turned by position * frequency; angles in float64."""
    xf = x.float()
    out = xf.clone()
    at = f = 0
    for a, d in enumerate(sections):
        h = d // 2
        ang = pos[..., a].double()[:, None, :, None] * freq[f:f + h]  # [B,1,T,h]
        c, s = ang.cos().float(), sign * ang.sin().float()
        lo, hi = xf[..., at:at + h], xf[..., at + h:at + d]
        out[..., at:at + h] = lo * c - hi * s
        out[..., at + h:at + d] = hi * c + lo * s
        at, f = at + d, f + h
    return out.to(x.dtype)


def _plain_cache(pages, heads, dim):
    z = dict(device="cuda")
    return dict(k=torch.zeros(pages, heads, PAGE, dim, dtype=torch.uint8, **z),
                v=torch.zeros(pages, heads, PAGE, dim, dtype=torch.uint8, **z),
                ke=torch.zeros(pages, heads, PAGE, dtype=torch.int16, **z),
                ve=torch.zeros(pages, heads, PAGE, dtype=torch.int16, **z),
                mean=torch.zeros(pages, heads, dim, dtype=torch.bfloat16, **z))


def _power(e):
    """2^e in float32, from its bits (a library's pow may be off in the last place)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x, fine):
    """(e4m3 codes, exponents) of rows: the smallest power of two that brings a row's largest value to 448 or below.
    Rows that are not `fine` are held as zeros times 2^128, which is NaN."""
    x = torch.where(fine.unsqueeze(-1), x.float(), torch.zeros((), device=x.device))
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-60, 60)
    e = torch.where(top == 0, torch.full_like(e, -60), e)
    y = (x * _power(-e).unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX)
    return y.to(torch.float8_e4m3fn).view(torch.uint8), torch.where(fine, e, 128).to(torch.int16)


def _values(codes, e):
    return codes.view(torch.float8_e4m3fn).float() * _power(e).unsqueeze(-1)


def _plain_write(cache, k, v, table, start, new):
    b, t, page, slot = _places(table, start, new)
    for lo in range(0, b.numel(), 1 << 17):
        part = slice(lo, lo + (1 << 17))
        rows = dict(k=k[b[part], :, t[part]], v=v[b[part], :, t[part]])
        fine = rows["k"].isfinite().all(-1) & rows["v"].isfinite().all(-1)
        for name, x in rows.items():
            codes, e = _quantise(x, fine)
            cache[name][page[part], :, slot[part]] = codes
            cache[name + "e"][page[part], :, slot[part]] = e
    # the pages that were touched: (sequence, page of it, tokens it holds now)
    touched = [(i, j, min(PAGE, at + n - j * PAGE)) for i, (at, n) in enumerate(zip(start, new)) if n
               for j in range(at // PAGE, (at + n - 1) // PAGE + 1)]
    for lo in range(0, len(touched), 1024):
        i, j, filled = torch.tensor(touched[lo:lo + 1024], device="cuda").unbind(1)
        ids = table[i, j].long()
        live = torch.arange(PAGE, device="cuda") < filled[:, None]
        vals = _values(cache["k"][ids], cache["ke"][ids]).double()
        total = torch.where(live[:, None, :, None], vals, torch.zeros_like(vals)).sum(2)
        cache["mean"][ids] = (total / filled[:, None, None]).float().bfloat16()


def _places(table, start, new):
    """(sequence, token, page, slot) of every new token."""
    b = torch.cat([torch.full((n,), i) for i, n in enumerate(new)]).cuda()
    t = torch.cat([torch.arange(n) for n in new]).cuda()
    pos = torch.tensor(start, device="cuda")[b] + t
    return b, t, table[b, pos // PAGE].long(), pos % PAGE


def _plain_read(cache, table, start, tokens, new, dtype):
    B, H, D = table.shape[0], cache["k"].shape[1], cache["k"].shape[3]
    out = [torch.zeros(B, H, tokens, D, device="cuda", dtype=dtype) for _ in range(2)]
    b, t, page, slot = _places(table, start, new)
    for o, name in zip(out, ("k", "v")):
        o[b, :, t] = _values(cache[name][page, :, slot], cache[name + "e"][page, :, slot]).to(dtype)
    return out


def _plain_select(q, cache, table, lens, keep, block_q, causal):
    """Per query block and key head: the first page, the last (from the first row's own page on where causal), and the
    `keep` of largest score among the others, ascending, -1 behind."""
    B, Hq, T, D = q.shape
    H, mp = cache["mean"].shape[1], table.shape[1]
    G, U = Hq // H, -(-T // block_q)
    W = min(1 + keep + 1 + ((block_q + 62) // PAGE if causal else 0), mp)
    index = torch.full((B, H, U, W), -1, device="cuda", dtype=torch.int32)
    count = torch.zeros(B, H, U, device="cuda", dtype=torch.int32)
    scores = torch.full((B, H, U, mp), -math.inf, device="cuda")
    at = torch.arange(mp, device="cuda")
    for b in range(B):
        means = cache["mean"][table[b].long()].double().permute(1, 2, 0).contiguous()  # [H,D,mp]
        for u in range(U):
            t0, t1 = u * block_q, min((u + 1) * block_q, T)
            rows = q[b].view(H, G, T, D)[:, :, t0:t1].double()
            qm = (rows.sum((1, 2)) / (G * (t1 - t0))).float().bfloat16().double()
            score = torch.matmul(qm.unsqueeze(1), means).squeeze(1).float()
            if causal:
                seen = (lens[b] - T + t1 - 1) // PAGE + 1
                recent = max(0, lens[b] - T + t0) // PAGE
            else:
                seen = -(-lens[b] // PAGE)
                recent = seen - 1
            if seen <= 0:
                continue
            forced = ((at < 1) | (at >= recent)) & (at < seen)
            score = torch.where(score.isnan() | (at >= seen), torch.full_like(score, -math.inf), score)
            scores[b, :, u] = score
            free = (~forced & (at < seen)).expand(H, mp)
            # equal scores: the stable order keeps the lowest index first
            key = torch.where(free, score, torch.full_like(score, -math.inf))
            order = torch.argsort(key, dim=-1, descending=True, stable=True)
            order = order.gather(1, torch.argsort((~free).gather(1, order).int(), dim=-1, stable=True))
            rank = torch.empty_like(order).scatter_(1, order, at.expand(H, mp))
            chosen = forced | (free & (rank < keep))
            n = chosen.sum(-1)
            first = torch.argsort((~chosen).int(), dim=-1, stable=True)[:, :W]
            index[b, :, u] = torch.where(at[:W] < n[:, None], first, -1).to(torch.int32)
            count[b, :, u] = n.to(torch.int32)
    return index, count, scores


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
            k = _values(cache["k"][ids, head], cache["ke"][ids, head]).flatten(1, 2)  # [H,W*64,D]
            v = _values(cache["v"][ids, head], cache["ve"][ids, head]).flatten(1, 2)
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
    D, B, T = case["dim"], case["batch"], case["tokens"]
    if case["kind"] == "rotary":
        elems = B * T * (case["heads_q"] + case["heads_k"]) * D
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * size * elems + 12 * B * T), "flops": passes * 3 * elems}
    H = case["heads"]
    row = D + 1  # a row of k or of v in the cache
    if case["kind"] == "write":
        n = sum(_counts(case))
        pages = sum(-(-(s + c) // PAGE) - s // PAGE for s, c in zip(_lengths(case), _counts(case)))
        # read, written, read back, written out; a touched page's key mean
        return {"bytes": 2 * n * H * (2 * size * D + 2 * row) + 2 * pages * H * D, "flops": 6 * n * H * D}
    lens = [n + (T if case["kind"] == "step" else 0) for n in _lengths(case)]
    G = case["group"]
    block_q = case["block_q"] or T
    units = -(-T // block_q)
    qbytes = 2 * B * T * H * G * D
    nbytes = nflops = 0
    for L in lens:
        held = -(-L // PAGE)
        if case["kind"] in ("select", "step"):
            nbytes += held * H * D * 2 + units * H * 4 * min(held, case["keep"] + 2)
            nflops += 2 * units * held * H * D
        if case["kind"] in ("attend", "step"):
            w = min(held, case["keep"] + 2) if case["keep"] else held
            # pages that any of the units lists, were the lists drawn apart
            union = held * (1.0 - (1.0 - w / held) ** units) if held else 0
            nbytes += int(min(union * PAGE, L)) * H * 2 * row
            keys = min(w * PAGE, L) - (T / 2 if case["causal"] else 0)
            nflops += int(4 * D * T * H * G * keys)
    nbytes += qbytes * (1 if case["kind"] == "select" else 2)
    if case["kind"] == "step":
        nbytes += 2 * B * T * H * (size * D + row)
    return {"bytes": int(nbytes), "flops": int(nflops)}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_rows(x):
    """float64 values that a row's 8-bit form stands for: each value to the nearest multiple of its e4m3 step."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    two = lambda n: ((n.long() + 1023) << 52).view(torch.float64)  # noqa: E731  2^n, exactly
    power = torch.ceil(torch.log2(top / E4M3_MAX)).clamp(-59, 59)
    power = torch.where(top > E4M3_MAX * two(power), power + 1, power)
    power = torch.where(top <= E4M3_MAX * two(power - 1), power - 1, power)
    y = x / two(power)
    binade = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20)))
    binade = torch.where(y.abs() >= two(binade + 1), binade + 1, binade)
    binade = torch.where(y.abs() < two(binade), binade - 1, binade)
    step = two(binade.clamp_min(-6.0) - 3.0)
    return torch.round(y / step) * step * two(power)


def exact(case, seed):
    if case["kind"] == "rotary":
        q, k, gq, gk, pos, sections, freq = _rotary_inputs(case, seed)

        def turn(x, sign):
            # each pair as a complex number times exp(i angle)
            parts, at, f = [], 0, 0
            for a, d in enumerate(sections):
                h = d // 2
                z = torch.complex(x[..., at:at + h].double(), x[..., at + h:at + d].double())
                ang = sign * pos[..., a].double().unsqueeze(-1) * freq[f:f + h]
                z = z * torch.polar(torch.ones_like(ang), ang).unsqueeze(1)
                parts += [z.real, z.imag]
                at, f = at + d, f + h
            return torch.cat([*parts, x[..., at:].double()], -1)

        return [turn(q, 1.0), turn(k, 1.0)] + ([turn(gq, -1.0), turn(gk, -1.0)] if case["train"] else [])
    s = _cache_inputs(case, seed)
    lens, table = s["lens"], s["table"].long()
    if case["kind"] == "select":
        return [None, None, _exact_score(case, s)]
    if case["kind"] in ("write", "step"):
        mean = torch.zeros(s["pages"], case["heads"], case["dim"], device="cuda", dtype=torch.float64)
        ko = torch.zeros(s["k"].shape, device="cuda", dtype=torch.float64)
        vo = torch.zeros_like(ko)
        stream = []
        for b, (old, new) in enumerate(zip(lens, _counts(case))):
            kb = torch.cat([s["hk"][b, :, :old], s["k"][b, :, :new]], 1)
            kb = _exact_rows(kb)
            ko[b, :, :new] = kb[:, old:]
            vo[b, :, :new] = _exact_rows(s["v"][b, :, :new])
            for j, part in enumerate(kb.split(PAGE, 1)):
                mean[table[b, j]] = part.mean(1)
            if case["kind"] == "step":
                stream.append((kb, torch.cat([_exact_rows(s["hv"][b, :, :old]), vo[b]], 1)))
        if case["kind"] == "write":
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
    return _exact_attend(case, s["q"], lambda b, h: (_exact_rows(s["hk"][b, h, :lens[b]]),
                                                     _exact_rows(s["hv"][b, h, :lens[b]])), pages)


def _exact_score(case, s):
    """Score of each page that a query block sees, -inf for the others: the definition rounds both means to bf16."""
    T, G, n, lens = case["tokens"], case["group"], case["block_q"], s["lens"]
    B, H, mp = case["batch"], case["heads"], s["table"].shape[1]
    U = -(-T // n)
    out = torch.full((B, H, U, mp), -math.inf, device="cuda", dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            part = _exact_rows(s["hk"][b, h, :lens[b]]).split(PAGE)
            mean = torch.stack([p.mean(0) for p in part]) if len(part) < 2 else \
                torch.cat([torch.stack(part[:-1]).mean(1), part[-1].mean(0, keepdim=True)])
            mean = mean.float().bfloat16().double()
            for u in range(U):
                last = min((u + 1) * n, T) - 1
                seen = -(-(lens[b] - T + last + 1 if case["causal"] else lens[b]) // PAGE)
                qm = s["q"][b, h * G:(h + 1) * G, u * n:last + 1].double().mean((0, 1)).float().bfloat16().double()
                out[b, h, u, :seen] = (mean[:seen] * qm).sum(-1)
    return out


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
