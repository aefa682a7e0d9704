"""The 4-bit block cache against its definitions in float64 (oracle/streaming.py), as tests/test_gpu_streaming.py has them for
the 8-bit one; the attention's bound is that one's: the widened keys and values are exact here too."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

from oracle import streaming as O
from test_gpu_streaming import _check_attend, _gen, _i32, _np, _randn, _same, _table
from vasc_amd import _lib, ops
from vasc_amd.streaming import BlockCache

pytestmark = pytest.mark.gpu

BUFFERS = ("kc", "vc", "ks", "vs", "vo", "mean")


def _fill(cache, g, table, lens, k=None, v=None):
    B, H, D, L = len(lens), cache.heads, cache.head_dim, max(max(lens), 1)
    k = _randn(g, B, H, L, D) if k is None else k
    v = _randn(g, B, H, L, D) if v is None else v
    ops.cache_write(cache, k.cuda(), v.cuda(), table, _i32([0] * B), count=_i32(lens))
    return [O.quantise4(_np(k[b, :, :n]), _np(v[b, :, :n])) for b, n in enumerate(lens)]


@pytest.mark.parametrize("dtype,powers", [(torch.float32, (-60, 0, 37)), (torch.bfloat16, (-60, 0, 37)), (torch.float16, (-12, 0, 9))])
@pytest.mark.parametrize("D", [64, 128])
def test_every_code_and_tie(D, dtype, powers):
    """Each e2m1 value, each tie between two and one step beside it, both signs, under several powers: the conversion's
    rounding. A value of 6 (or 7) beside them holds the power in place."""
    codes = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    ties = [(a + b) / 2 for a, b in zip(codes, codes[1:])]
    near = [t * (1 + s * 2.0 ** -k) for t in ties + codes for s in (-1, 1) for k in (22, 10, 7)]
    values = [s * x for x in codes + ties + near for s in (1, -1)]
    values += [6.5, -6.5, 7.0, 6.9999995]
    rows = [values[i:i + 31] for i in range(0, len(values), 31)]
    tops = (6.0, 7.0, 5.0)
    x = torch.zeros(1, 1, len(rows) * len(tops) * 3, D)
    at = 0
    for row in rows:
        for top in tops:
            for e in powers:
                for gr in range(D // 32):
                    x[0, 0, at, gr * 32:gr * 32 + len(row)] = torch.tensor(row) * 2.0 ** e
                    x[0, 0, at, gr * 32 + 31] = top * 2.0 ** e
                at += 1
    x = x.to(dtype)
    table = _i32([list(range(-(-at // 64)))])
    cache = BlockCache(8, 1, D, bits=4)
    ops.cache_write(cache, x.cuda(), x.flip(3).contiguous().cuda(), table, _i32([0]))
    k, v = ops.cache_read(cache, table, _i32([0]), at, dtype=torch.float32)
    ko, vo = O.quantise4(_np(x), _np(x.flip(3)))
    assert _same(_np(k), ko) and _same(_np(v), vo)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,H", [(64, 3), (128, 2)])
def test_write_then_read(dtype, D, H):
    """Values of many magnitudes, other ones in each group, at ragged places, from strided rows; every other slot and page
    keeps what it held."""
    g = _gen(D)
    B, T, mp = 4, 150, 6
    table, pages = _table(g, B, mp)
    start, count = [0, 61, 130, 64], [150, 70, 0, 1]
    cache = BlockCache(pages, H, D, bits=4)
    for t in (cache.kc, cache.vc, cache.vo):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (cache.ks, cache.vs):
        t.copy_(torch.randint(110, 140, t.shape, generator=g, dtype=torch.uint8))
    cache.mean.copy_(torch.randn(cache.mean.shape, generator=g))
    before = {n: getattr(cache, n).clone() for n in BUFFERS}
    mag = torch.exp2(torch.randint(-12, 12, (B, T, H, D // 32), generator=g).float()).repeat_interleave(32, 3)
    k = (torch.randn(B, T, H, D, generator=g) * mag).to(dtype).cuda().transpose(1, 2)
    v = (torch.randn(B, T, H, D, generator=g) * mag.flip(1)).to(dtype).cuda().transpose(1, 2)
    old_k, old_v = ops.cache_read(cache, table, _i32([0] * B), mp * 64, dtype=torch.float32)
    ops.cache_write(cache, k, v, table, _i32(start), count=_i32(count))
    rk, rv = ops.cache_read(cache, table, _i32(start), T, count=_i32(count), dtype=torch.float32)
    all_k, all_v = ops.cache_read(cache, table, _i32([0] * B), mp * 64, dtype=torch.float32)
    touched = set()
    for b in range(B):
        s, n = start[b], count[b]
        ko, vo = O.quantise4(_np(k[b, :, :n]), _np(v[b, :, :n]))
        assert _same(_np(rk[b, :, :n]), ko) and _same(_np(rv[b, :, :n]), vo)
        assert not rk[b, :, n:].any() and not rv[b, :, n:].any()
        want_k, want_v = _np(old_k[b]), _np(old_v[b])
        want_k[:, s:s + n], want_v[:, s:s + n] = ko, vo
        assert _same(_np(all_k[b]), want_k) and _same(_np(all_v[b]), want_v)
        for j in range(s // 64, (s + n - 1) // 64 + 1 if n else s // 64):
            p = int(table[b, j])
            touched.add(p)
            part = want_k[:, j * 64:min(j * 64 + 64, s + n)]
            mean = O.round_bf16((part.sum(1) / part.shape[1]).astype(np.float32))
            assert _same(_np(cache.mean[p]), mean.astype(np.float64))
    rest = [p for p in range(pages) if p not in touched]
    for n, t in before.items():
        assert torch.equal(getattr(cache, n)[rest], t[rest]), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_write_edge_values(D, dtype):
    """Groups at the borders of the format: 7 * 2^e and one step past it, the exponents' ends, groups of a value row farther
    apart than the offsets reach, zeros, float32's largest and smallest; tokens that are not finite."""
    step = 1 + 2.0 ** -10
    rows = [[7.0], [7.0 * step], [6.0], [3.5, 0.4375], [3.5 * step, 1.0], [0.0], [-0.0], [2.0 ** -62, 2.0 ** -63],
            [2.0 ** -61, 3 * 2.0 ** -62], [2.0 ** -126, 2.0 ** -149], [3.0e38, 1.0], [7 * 2.0 ** 60, 2.0 ** 53], [2.0 ** 127],
            [1.0, 0.3, 2.5, 0.7], [float("inf")], [1.0, float("nan")], [-float("inf"), 1.0], [float("nan")]]
    x = torch.zeros(1, 1, len(rows), D)
    for i, r in enumerate(rows):
        x[0, 0, i, :len(r)] = torch.tensor(r, dtype=torch.float64).float()
        # the next group 13, 14, 15 and more powers lower, in turn
        x[0, 0, i, 32:32 + len(r)] = x[0, 0, i, :len(r)] * 2.0 ** -(11 + i % 7)
        x[0, 0, i, D - 1] = x[0, 0, i, 0]
    x = x.to(dtype)
    y = torch.full_like(x, 0.5)
    y[0, 0, 2, 5] = float("nan")  # a value that is not finite marks the token's key too
    table = _i32([[1]])
    for a, b in ((x, y), (y, x)):
        cache = BlockCache(2, 1, D, bits=4)
        ops.cache_write(cache, a.cuda(), b.cuda(), table, _i32([0]))
        k, v = ops.cache_read(cache, table, _i32([0]), len(rows), dtype=torch.float32)
        ko, vo = O.quantise4(_np(a), _np(b))
        assert _same(_np(k), ko) and _same(_np(v), vo)
        assert cache.mean[1].isnan().all()  # NaN tokens in the page
        ops.cache_write(cache, a[:, :, :2].cuda(), b[:, :, :2].cuda(), table, _i32([0]))  # written again, shorter
        mean = O.round_bf16((ko[0, 0, :2].sum(0) / 2).astype(np.float32))
        assert _same(_np(cache.mean[1, 0]), mean.astype(np.float64))
        k16, _ = ops.cache_read(cache, table, _i32([0]), len(rows), dtype=torch.float16)
        with np.errstate(over="ignore"):
            assert _same(_np(k16), ko.astype(np.float16).astype(np.float64))


def test_write_in_any_portions_gives_the_same_bytes():
    g = _gen(17)
    for D in (64, 128):
        H, n = 2, 200
        k, v = _randn(g, 1, H, n, D).cuda(), _randn(g, 1, H, n, D).cuda()
        table, pages = _table(g, 1, 4)
        caches = []
        for cuts in ([n], list(range(1, n + 1)), [3, 63, 64, 65, 127, 130, 192, n]):
            c, at = BlockCache(pages, H, D, bits=4), 0
            for e in cuts:
                ops.cache_write(c, k[:, :, at:e], v[:, :, at:e], table, _i32([at]))
                at = e
            caches.append(c)
        for c in caches[1:]:
            for name in BUFFERS:
                assert torch.equal(getattr(c, name), getattr(caches[0], name)), name


def test_write_and_read_outside_the_table():
    g = _gen(23)
    cache = BlockCache(4, 1, 64, bits=4)
    table = _i32([[3, -1, 99, 0]])
    k, v = _randn(g, 1, 1, 300, 64).cuda(), _randn(g, 1, 1, 300, 64).cuda()
    before = {n: getattr(cache, n).clone() for n in BUFFERS}
    ops.cache_write(cache, k, v, table, _i32([-1]))
    ops.cache_write(cache, k, v, table, _i32([256]))
    ops.cache_write(cache, k, v, table, _i32([0]), count=_i32([-5]))
    assert all(torch.equal(getattr(cache, n), t) for n, t in before.items())
    ops.cache_write(cache, k, v, table, _i32([10]))
    rk, rv = ops.cache_read(cache, table, _i32([10]), 300, dtype=torch.float32)
    ko, vo = O.quantise4(_np(k), _np(v))
    live = np.zeros(300, bool)
    pos = np.arange(300) + 10
    live[(pos < 64) | ((pos >= 192) & (pos < 256))] = True
    assert _same(_np(rk), np.where(live[:, None], ko, 0)) and _same(_np(rv), np.where(live[:, None], vo, 0))
    assert not cache.kc[1:3].any() and not cache.vc[1:3].any()
    rk, _ = ops.cache_read(cache, table, _i32([-3]), 70)
    assert not rk.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,G", [(64, 2, 1), (128, 1, 4), (64, 1, 20), (128, 1, 32), (128, 2, 1)])
def test_attend_single_tokens(dtype, D, H, G):
    g = _gen(D + G)
    lens = [1, 63, 64, 65, 0, 700, 1300]
    table, pages = _table(g, len(lens), 21)
    cache = BlockCache(pages, H, D, bits=4)
    held = _fill(cache, g, table, lens)
    q = _randn(g, len(lens), H * G, 1, D, dtype=dtype).cuda()
    o = ops.cache_attn(q, cache, table, _i32(lens))
    assert o.dtype == dtype
    _check_attend(o, q, held, lens, None, 1, False, H=H)
    assert not o[4].any()
    for keep in (0, 3):
        index, count = ops.cache_select(q, cache, table, _i32(lens), keep)
        for b in range(len(lens)):  # the choice is by the 4-bit cache's means
            means = _np(cache.mean)[table[b].cpu().numpy()]
            n = -(-lens[b] // 64)
            for h in range(H):
                want, _ = O.select(_np(q)[b, h * G:(h + 1) * G, 0], means[:n, h], n, n - 1, keep, 1, 1)
                assert index[b, h, 0, :count[b, h, 0]].tolist() == want
        lists = [[[index[b, h, 0, :count[b, h, 0]].tolist()] for h in range(H)] for b in range(len(lens))]
        o = ops.cache_attn(q, cache, table, _i32(lens), index, count)
        _check_attend(o, q, held, lens, lists, 1, False, H=H)


@pytest.mark.parametrize("D,H,G,T,block_q,L", [(64, 2, 1, 300, 128, 1200), (64, 1, 1, 40, 32, 500), (128, 1, 4, 70, 32, 600),
                                               (64, 1, 2, 50, 16, 50), (128, 1, 8, 5, 2, 330), (128, 2, 1, 130, 64, 700)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_chunks(D, H, G, T, block_q, L, causal, dtype):
    g = _gen(D + T + L)
    lens = [L, max(T, L - 77)]
    table, pages = _table(g, 2, -(-L // 64) + 1)
    cache = BlockCache(pages, H, D, bits=4)
    held = _fill(cache, g, table, lens)
    q = _randn(g, 2, H * G, T, D, dtype=dtype).cuda()
    n_q = [T, T - T // 3]
    o = ops.cache_attn(q, cache, table, _i32(lens), causal=causal, q_count=_i32(n_q))
    _check_attend(o, q, held, lens, None, block_q, causal, n_q=n_q, H=H)
    index, count = ops.cache_select(q, cache, table, _i32(lens), 2, block_q=block_q, causal=causal, q_count=_i32(n_q))
    lists = [[[index[b, h, u, :count[b, h, u]].tolist() for u in range(index.shape[2])] for h in range(H)] for b in range(2)]
    o = ops.cache_attn(q, cache, table, _i32(lens), index, count, block_q=block_q, causal=causal, q_count=_i32(n_q))
    _check_attend(o, q, held, lens, lists, block_q, causal, n_q=n_q, H=H)


@pytest.mark.parametrize("D,H,G,T,L", [(64, 1, 1, 1, 9000), (128, 1, 3, 1, 7000), (64, 1, 1, 90, 5000), (128, 2, 1, 2, 2600)])
def test_attend_many_parts(D, H, G, T, L):
    g = _gen(L)
    table, pages = _table(g, 2, -(-L // 64))
    cache = BlockCache(pages, H, D, bits=4)
    lens = [L, 100]  # most parts of the second have no page
    held = _fill(cache, g, table, lens)
    q = _randn(g, 2, H * G, T, D).cuda()
    o = ops.cache_attn(q, cache, table, _i32(lens))
    _check_attend(o, q, held, lens, None, 1, False, H=H)
    assert not ops.cache_attn(q, cache, table, _i32([0, 0])).any()


@pytest.mark.parametrize("D,G,T", [(64, 1, 1), (128, 20, 1), (64, 1, 100), (128, 4, 30)])
def test_attend_groups_far_apart(D, G, T):
    """Groups of keys and values that are powers of two apart, other ones in each token and up to all that the offsets hold;
    rows of zeros among them; a small value row's token that has most of the weight."""
    g = _gen(D + G)
    L = 300
    mag = torch.exp2(torch.randint(-20, 3, (1, 1, L, D // 32), generator=g).float()).repeat_interleave(32, 3)
    k, v = torch.randn(1, 1, L, D, generator=g), torch.randn(1, 1, L, D, generator=g) * mag
    k = k * torch.exp2(torch.randint(-3, 1, (1, 1, L, D // 32), generator=g).float()).repeat_interleave(32, 3)
    v[0, 0, ::17] = 0
    v[0, 0, 5] *= 2.0 ** -40
    k[0, 0, 5] = 3.0
    table, pages = _table(g, 1, 5)
    cache = BlockCache(pages, 1, D, bits=4)
    held = _fill(cache, g, table, [L], k.bfloat16(), v.bfloat16())
    q = (torch.randn(1, G, T, D, generator=g) + 0.3).bfloat16().cuda()
    o = ops.cache_attn(q, cache, table, _i32([L]))
    _check_attend(o, q, held, [L], None, 128 // G, False, H=1)


@pytest.mark.parametrize("D,G,T", [(64, 1, 1), (128, 20, 1), (64, 1, 100), (128, 4, 30)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_nan_tokens_and_queries(D, G, T, dtype):
    """A NaN token makes the rows that see it NaN and touches no other; a query that is not finite makes its own row NaN."""
    g = _gen(D + T)
    L, B = 200, 2
    table, pages = _table(g, B, 4)
    cache = BlockCache(pages, 1, D, bits=4)
    k, v = _randn(g, B, 1, L, D), _randn(g, B, 1, L, D)
    k[1, 0, L - 3, 7] = float("nan")
    v[0, 0, 150, 3] = float("inf")
    held = _fill(cache, g, table, [L, L], k, v)
    q = _randn(g, B, G, T, D, dtype=dtype).cuda()
    q[1, 0, T - 1, 5] = float("-inf")
    o = ops.cache_attn(q, cache, table, _i32([140, L - 3]))
    bad = torch.zeros_like(o, dtype=torch.bool)
    bad[1, 0, T - 1] = True
    assert torch.equal(o.isnan(), bad)
    clean = q.clone()
    clean[1, 0, T - 1, 5] = 0
    oc = ops.cache_attn(clean, cache, table, _i32([140, L - 3]))
    _check_attend(oc, clean, [tuple(x[:, :140] for x in held[0]), tuple(x[:, :L - 3] for x in held[1])], [140, L - 3], None,
                  128 // G, False, H=1)
    assert ops.cache_attn(clean, cache, table, _i32([L, L])).isnan().all()


def test_attend_missing_pages_and_lists():
    """Entries of the table that are no page, and of a list that repeat, fall back or lie outside, are not seen."""
    g = _gen(31)
    D, L = 128, 640
    table, pages = _table(g, 1, 10)
    cache = BlockCache(pages, 2, D, bits=4)
    held = _fill(cache, g, table, [L])
    holes = table.clone()
    holes[0, 3], holes[0, 7] = -1, pages
    q = _randn(g, 1, 2, 1, D).cuda()
    o = ops.cache_attn(q, cache, holes, _i32([L]))
    there = [[[[0, 1, 2, 4, 5, 6, 8, 9]]] * 2]
    _check_attend(o, q, held, [L], there, 1, False, H=2)
    index = _i32([4, 4, 2, 5, 12, -1, 9, 0]).view(1, 1, 1, 8).expand(1, 2, 1, 8)
    o = ops.cache_attn(q, cache, table, _i32([L]), index, _i32([8, 8]).view(1, 2, 1))
    _check_attend(o, q, held, [L], [[[[4, 5, 9]]] * 2], 1, False, H=2)


@pytest.mark.parametrize("how", ["deepcopy", "copy", "pickle"])
def test_copied_cache(how):
    g = _gen(59)
    table, pages = _table(g, 1, 3)
    cache = BlockCache(pages, 2, 64, bits=4)
    held = _fill(cache, g, table, [100])
    other = {"deepcopy": copy.deepcopy, "copy": copy.copy, "pickle": lambda c: pickle.loads(pickle.dumps(c))}[how](cache)
    assert other.bits == 4 and other.pointers == tuple(getattr(other, n).data_ptr() for n in BUFFERS[:-1])
    assert (other.pointers == cache.pointers) == (how == "copy")
    q = _randn(g, 1, 2, 1, 64).cuda()
    _check_attend(ops.cache_attn(q, other, table, _i32([100])), q, held, [100], None, 1, False, H=2)


def test_offsets_past_32_bits():
    """A cache whose codes lie past 2^32 bytes, written, attended to, copied and compacted at both ends."""
    g = _gen(47)
    H, D = 8, 128
    pages = (2 ** 32) // (H * 64 * D // 2) + 40
    cache = BlockCache(pages, H, D, bits=4)
    table = torch.stack([torch.arange(pages - 12, pages), torch.arange(12)]).to(torch.int32).cuda()
    lens = [700, 650]
    held = _fill(cache, g, table, lens)
    q = _randn(g, 2, H, 1, D).cuda()
    _check_attend(ops.cache_attn(q, cache, table, _i32(lens)), q, held, lens, None, 1, False, H=H)
    ops.cache_copy(cache, table.flip(0)[:, :11].flatten(), torch.arange(20, 42, device="cuda"))
    swapped = torch.arange(20, 42, device="cuda", dtype=torch.int32).view(2, 11)
    for t, order in ((table, (0, 1)), (swapped, (1, 0))):
        rk, rv = ops.cache_read(cache, t, _i32([0, 0]), 640, dtype=torch.float32)
        for i, b in enumerate(order):
            assert _same(_np(rk[i]), held[b][0][:, :640]) and _same(_np(rv[i]), held[b][1][:, :640])
    out = torch.arange(pages - 20, pages - 12, device="cuda", dtype=torch.int32).view(2, 4)
    index = torch.arange(0, 500, 2, device="cuda").expand(2, 250)
    ops.cache_compact(cache, table, index, out)
    rk, rv = ops.cache_read(cache, out, _i32([0, 0]), 250, dtype=torch.float32)
    for b in range(2):
        assert _same(_np(rk[b]), held[b][0][:, :500:2]) and _same(_np(rv[b]), held[b][1][:, :500:2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,H", [(64, 16), (128, 8)])
@pytest.mark.parametrize("bits", [4, 8])
def test_reads_of_much_and_little(bits, D, H, dtype):
    """Outputs of 128 MB and more are stored in another way than smaller ones (half types); the rows are the same."""
    T = (1 << 27) // (2 * H * D * dtype.itemsize)
    cache = BlockCache(-(-T // 64) + 1, H, D, bits=bits)
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(1, H, T, D, device="cuda", generator=g, dtype=torch.bfloat16) for _ in range(2))
    table = torch.arange(1, cache.pages, device="cuda", dtype=torch.int32).view(1, -1)
    ops.cache_write(cache, k, v, table, _i32([0]))
    ko, vo = ops.cache_read(cache, table, _i32([0]), T, count=_i32([T - 5]), dtype=dtype)
    for at, n in ((0, T // 2), (T // 2, T - 5 - T // 2)):
        a, b = ops.cache_read(cache, table, _i32([at]), n, dtype=dtype)
        assert torch.equal(ko[:, :, at:at + n], a) and torch.equal(vo[:, :, at:at + n], b)
    assert not ko[:, :, -5:].any() and not vo[:, :, -5:].any()


@pytest.mark.parametrize("D,H", [(64, 16), (128, 8)])
@pytest.mark.parametrize("bits", [4, 8])
def test_writes_of_much_and_little(bits, D, H):
    """Float32 rows of 256 MB and more are loaded in another way than fewer; the cache's bytes are the same."""
    T = (1 << 28) // (2 * H * D * 4)
    a, b = (BlockCache(-(-T // 64), H, D, bits=bits) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.randn(1, H, T, D, device="cuda", generator=g) for _ in range(2))
    k[0, 1, 77, 3] = float("nan")
    table = torch.arange(a.pages, device="cuda", dtype=torch.int32).view(1, -1)
    ops.cache_write(a, k, v, table, _i32([0]))
    for at, n in ((0, T // 2 + 9), (T // 2 + 9, T - T // 2 - 9)):
        ops.cache_write(b, k[:, :, at:at + n], v[:, :, at:at + n], table, _i32([at]))
    for name in ("kc", "vc", "ks", "vs", "vo", "mean"):
        x, y = getattr(a, name), getattr(b, name)
        assert x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)), name


def test_step_captured_in_graphs():
    """Write, choice and attention in two graphs with their own memory, replayed in turn with eager work between."""
    g = _gen(3)
    H, G, D, T, block_q, steps = 2, 2, 128, 5, 4, 4
    table, pages = _table(g, 2, 10)
    qs, ks, vs = ([_randn(g, 2, n, T, D).cuda() for _ in range(steps)] for n in (H * G, H, H))
    start0 = [70, 3]

    def history():
        c = BlockCache(pages, H, D, bits=4)
        gg = _gen(99)
        k, v = _randn(gg, 2, H, 70, D).cuda(), _randn(gg, 2, H, 70, D).cuda()
        ops.cache_write(c, k, v, table, _i32([0, 0]), count=_i32(start0))
        return c

    def step(c, q, k, v, start, lengths):
        ops.cache_write(c, k, v, table, start)
        index, count = ops.cache_select(q, c, table, lengths, 2, block_q=block_q)
        return ops.cache_attn(q, c, table, lengths, index, count, block_q=block_q)

    eager, cache = [], history()
    for i in range(steps):
        s = _i32(start0) + i * T
        eager.append(step(cache, qs[i], ks[i], vs[i], s, s + T))
    graphs = []
    for _ in range(2):
        c = history()
        st = dict(cache=c, q=qs[0].clone(), k=ks[0].clone(), v=vs[0].clone(), start=_i32(start0), lengths=_i32(start0) + T)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(c, *(st[n] for n in ("q", "k", "v", "start", "lengths")))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(c, *(st[n] for n in ("q", "k", "v", "start", "lengths")))
        graphs.append((graph, st, out))
    for i in range(steps):
        for graph, st, out in graphs:
            for name, src in (("q", qs), ("k", ks), ("v", vs)):
                st[name].copy_(src[i])
            st["start"].copy_(_i32(start0) + i * T)
            st["lengths"].copy_(st["start"] + T)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager[i]), i
            torch.randn(1 << 16, device="cuda").sum().item()


def test_rounding_of_normal_rows():
    """A value is off by at most a fifth of itself (the widest: 5 between 4 and 6, 1.25 between 1 and 1.5) or by half a
    subnormal step, 2^e / 4, where the group's largest is above 3.5 * 2^e."""
    g = _gen(5)
    x = torch.randn(1, 2, 256, 128, generator=g)
    table = _i32([[0, 1, 2, 3]])
    cache = BlockCache(4, 2, 128, bits=4)
    ops.cache_write(cache, x.cuda(), x.cuda(), table, _i32([0]))
    for r in ops.cache_read(cache, table, _i32([0]), 256, dtype=torch.float32):
        err, size = (r.cpu() - x).double().view(-1, 32).abs(), x.double().view(-1, 32).abs()
        assert (err <= torch.maximum(size / 5, size.amax(-1, keepdim=True) / 14)).all()


@pytest.mark.parametrize("D,G,T", [(64, 1, 1), (64, 2, 40), (128, 1, 1), (128, 4, 30)])
def test_attend_strided_tensors_out_and_scales(D, G, T):
    """Queries cut from wider rows, written to a strided `out` whose other elements stay; scales of both signs, 0 and large; a
    causal chunk longer than its sequence, whose first rows see nothing."""
    g = _gen(D + G + T)
    H, lens = 2, [700, 9]
    table, pages = _table(g, 2, 11)
    cache = BlockCache(pages, H, D, bits=4)
    held = _fill(cache, g, table, lens)
    wide = _randn(g, 2, T, H * G + 3, D + 24).cuda()
    q = wide[:, :, 1:1 + H * G, 8:8 + D].transpose(1, 2)
    store = torch.full((2, T + 2, H * G, D + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    out = store[:, 1:T + 1, :, 4:4 + D].transpose(1, 2)
    n_q = [T, max(1, T - 5)]
    for causal in (False, True):
        for scale in (None, -0.3, 0.0, 1.0):
            got = ops.cache_attn(q, cache, table, _i32(lens), causal=causal, q_count=_i32(n_q), scale=scale, out=out)
            assert got is out
            # the bound's part of the logits is their size, scale times sum |q| |k|: below 0 for a negative scale, which would
            # take 2 (D + 8) 2^-24 30 = 5e-4 from it here; the opposite queries have the same logits with the positive one
            sign = -1 if scale is not None and scale < 0 else 1
            _check_attend(got.contiguous(), sign * q.contiguous(), held, lens, None, 128 // G, causal,
                          scale=None if scale is None else abs(scale), n_q=n_q, H=H)
            if causal and T > lens[1]:
                assert not got[1, :, :n_q[1] - lens[1]].any()
            seen = store.clone()
            seen[:, 1:T + 1, :, 4:4 + D] = 7.0
            assert (seen == 7.0).all()


def test_two_streams_at_once():
    """Attention over one 4-bit cache and writes into another on streams of their own: as one after the other."""
    g = _gen(53)
    H, D, L = 2, 128, 4000
    table, pages = _table(g, 2, 63)
    cache, other = BlockCache(pages, H, D, bits=4), BlockCache(pages, H, D, bits=4)
    k, v = _randn(g, 2, H, L, D).cuda(), _randn(g, 2, H, L, D).cuda()
    ops.cache_write(cache, k, v, table, _i32([0, 0]))
    q, n, start = _randn(g, 2, H, 1, D).cuda(), _i32([L]), _i32([0, 0])
    want = [ops.cache_attn(q[b:b + 1], cache, table[b:b + 1], n) for b in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], [[], []]
    for _ in range(6):
        for b in range(2):
            with torch.cuda.stream(streams[b]):
                got[b].append(ops.cache_attn(q[b:b + 1], cache, table[b:b + 1], n))
        with torch.cuda.stream(streams[2]):
            ops.cache_write(other, k, v, table, start)
    torch.cuda.synchronize()
    for b in range(2):
        assert all(torch.equal(x, want[b]) for x in got[b])
    assert all(torch.equal(getattr(other, name), getattr(cache, name)) for name in BUFFERS)


def test_inputs_that_need_a_gradient_are_refused():
    cache = BlockCache(2, 1, 64, bits=4)
    x = torch.zeros(1, 1, 3, 64, device="cuda", requires_grad=True)
    table, n = _i32([[0, 1]]), _i32([0])
    with pytest.raises(ValueError, match="gradient"):
        ops.cache_write(cache, x, x, table, n)
    with pytest.raises(ValueError, match="gradient"):
        ops.cache_attn(x.bfloat16(), cache, table, n)
    with pytest.raises(ValueError, match="heads"):
        ops.cache_write(cache, x.detach().expand(1, 2, 3, 64), x.detach().expand(1, 2, 3, 64), table, n)
    with torch.no_grad():
        ops.cache_write(cache, x, x, table, n)
    assert cache.nbytes == sum(getattr(cache, name).numel() * getattr(cache, name).element_size() for name in BUFFERS)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["lists", "causal"])
def test_attend_frame_with_short_last_unit(how, dtype):
    """A frame of 1041 queries over many pages, whose last unit of 17 rows has a launch of its own: lists of every unit, or a
    causal chunk with a shorter count, against float64 on the GPU. The bound is _check_attend's."""
    g = _gen(7)
    H, D, T, L, block = 16, 64, 1041, 133200, 128
    table, pages = _table(g, 1, -(-L // 64))
    cache = BlockCache(pages, H, D, bits=4)
    k, v = _randn(g, 1, H, L, D).cuda(), _randn(g, 1, H, L, D).cuda()
    ops.cache_write(cache, k, v, table, _i32([0]))
    k, v = (x[0].double() for x in ops.cache_read(cache, table, _i32([0]), L))
    q = _randn(g, 1, H, T, D, dtype=dtype).cuda()
    n_q = T if how == "lists" else T - 9
    size = _lib.fn("vasc_cache4_attn_workspace_size")
    sizes = [size(1, H, H, t, D, block, table.shape[1], 522 if how == "lists" else 0) for t in (T, T + 15, T + 16, 9 * block)]
    # 17 and 32 rows are a launch of their own, of other parts; 33 are not, and take what 128 do
    assert sizes[0] != sizes[2] and sizes[1] != sizes[2] and sizes[2] == sizes[3]
    if how == "lists":
        index, count = ops.cache_select(q, cache, table, _i32([L]), 520, block_q=block)
        o = ops.cache_attn(q, cache, table, _i32([L]), index, count, block_q=block)
    else:
        o = ops.cache_attn(q, cache, table, _i32([L]), causal=True, q_count=_i32([n_q]))
    pos = torch.arange(L, device="cuda")
    for h in range(H):
        for u in range(-(-T // block)):
            rows = torch.arange(u * block, min(T, (u + 1) * block), device="cuda")
            if how == "lists":
                listed = torch.zeros(table.shape[1], dtype=torch.bool, device="cuda")
                listed[index[0, h, u, :count[0, h, u]].long()] = True
                seen = listed[pos // 64].expand(len(rows), L)
            else:
                seen = (pos[None] <= (L - n_q + rows)[:, None]) & (rows < n_q)[:, None]
            qd = q[0, h, rows].double()
            x = torch.where(seen, qd @ k[h].T.contiguous() * D ** -0.5, -math.inf)
            w = torch.nan_to_num(torch.softmax(x, -1))
            ref, mag = w @ v[h], w @ v[h].abs()
            logit = torch.where(seen, qd.abs() @ k[h].abs().T.contiguous() * D ** -0.5, 0.0).amax(-1, keepdim=True)
            n = seen.sum(-1, keepdim=True)
            rel = 2.0 ** -11 + 2 * ((D + 8) * 2.0 ** -24 * logit + n * 2.0 ** -24) + 2.0 ** -14.5
            half = torch.finfo(dtype).eps / 2
            bound = rel * mag + half * (ref.abs() + rel * mag) + n * 2.0 ** -36 * v[h].abs().max() + 2.0 ** -25
            assert ((o[0, h, rows].double() - ref).abs() <= bound).all(), (h, u)
    assert not o[:, :, n_q:].any()
