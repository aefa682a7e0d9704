"""The streaming operators against their definitions in float64 (oracle/streaming.py)."""
import copy
import math
import pickle

import numpy as np
import pytest
import torch

from oracle import streaming as O
from vasc_amd import _lib, ops
from vasc_amd.streaming import BlockCache

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -9 * 2, torch.float16: 2.0 ** -12 * 2, torch.float32: 2.0 ** -25 * 2}  # half a step


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _np(t):
    return t.detach().double().cpu().numpy()


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g).to(dtype)


def _table(g, B, mp, spare=3):
    """(page table with pages in random order, pages of the cache)."""
    pages = B * mp + spare
    return torch.randperm(pages, generator=g)[:B * mp].view(B, mp).to(torch.int32).cuda(), pages


# ------------------------------------------------------------------ rotary
def _freq(sections, bases):
    return torch.cat([b ** (-torch.arange(0, s, 2, dtype=torch.float64) / s) for s, b in zip(sections, bases)])


def _rotary_bound(x, ref, sections, dtype):
    """Output rounding, and float32 arithmetic on the pair: cos and sin within 2^-22 of exact (the correction term leaves
    sincosf's last place and the reduction's 2^-24), two products and a sum of three roundings."""
    x = _np(x)
    size = np.abs(x).copy()
    at = 0
    for d in sections:
        h = d // 2
        s = np.abs(x[..., at:at + h]) + np.abs(x[..., at + h:at + d])
        size[..., at:at + h] = size[..., at + h:at + d] = s
        at += d
    size[..., at:] = 0
    return HALF[dtype] * np.abs(ref) + (2.0 ** -22 + 3 * 2.0 ** -24) * size * (1 + HALF[dtype]) + 2.0 ** -25


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,sections,T", [(64, (16, 24, 24), 37), (128, (32, 48, 48), 9), (64, (32, 32), 1),
                                          (64, (6, 28, 28), 130), (80, (16, 16, 16, 16), 21), (64, (2, 6, 10), 50),
                                          (64, (64,), 600)])
def test_rotary_matches_float64(dtype, D, sections, T):
    g = _gen(D + T)
    B, Hq, Hk = 2, 5, 3
    q, k = _randn(g, B, T, Hq, D, dtype=dtype).cuda().transpose(1, 2), _randn(g, B, Hk, T, D, dtype=dtype).cuda()
    pos = torch.randint(-50, 5000, (B, T, len(sections)), generator=g)
    freq = _freq(sections, (10000.0, 100.0, 100.0, 50.0))
    qo, ko = ops.rotary_axes(q, k, pos.cuda(), sections, freq.cuda())
    for x, y in ((q, qo), (k, ko)):
        ref = O.rotate(_np(x), pos.numpy(), sections, freq.numpy())
        assert y.shape == x.shape and y.dtype == dtype
        assert (np.abs(_np(y) - ref) <= _rotary_bound(x, ref, sections, dtype)).all()
        assert torch.equal(y[..., sum(sections):], x[..., sum(sections):])
    assert qo.stride() == q.stride() and ko.stride() == k.stride()


def test_rotary_far_positions_and_shared_rows():
    """Positions of 2^31 - 1: a float32 angle would be off by tens of radians. One row of positions for all sequences."""
    g = _gen(3)
    sections = (16, 24, 24)
    x = _randn(g, 3, 2, 40, 64, dtype=torch.float32).cuda()
    pos = torch.randint(2 ** 30, 2 ** 31 - 1, (40, 3), generator=g)
    pos[0] = 2 ** 31 - 1
    pos[1] = -2 ** 31
    freq = _freq(sections, (10000.0, 100.0, 100.0))
    y, none = ops.rotary_axes(x, None, pos.cuda(), sections, freq.cuda())
    assert none is None
    ref = O.rotate(_np(x), pos.numpy()[None], sections, freq.numpy())
    # the float64 angle itself is rounded: 2^31 * 2^-53 on both sides
    bound = _rotary_bound(x, ref, sections, torch.float32) + 2 ** -21 * (np.abs(_np(x)).max() * 2)
    assert (np.abs(_np(y) - ref) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotary_gradients(dtype):
    """Against the formula (the inverse turn), with shared and broadcast inputs, one gradient missing, and differences."""
    g = _gen(11)
    sections, D, T = (16, 24, 24), 72, 33
    freq = _freq(sections, (10000.0, 100.0, 100.0)).cuda()
    pos = torch.randint(0, 900, (2, T, 3), generator=g).cuda()
    q = _randn(g, 2, 4, T, D, dtype=dtype).cuda().requires_grad_()
    k = _randn(g, 1, 1, T, D, dtype=dtype).cuda().requires_grad_()
    gq, gk = _randn(g, 2, 4, T, D, dtype=dtype).cuda(), _randn(g, 2, 3, T, D, dtype=dtype).cuda()
    qo, ko = ops.rotary_axes(q, k.expand(2, 3, T, D), pos, sections, freq)
    dq, dk = torch.autograd.grad([qo, ko], [q, k], [gq, gk])
    ref = O.rotate(_np(gq), pos.cpu().numpy(), sections, freq.cpu().numpy(), -1.0)
    assert (np.abs(_np(dq) - ref) <= _rotary_bound(gq, ref, sections, dtype)).all()
    each = O.rotate(_np(gk), pos.cpu().numpy(), sections, freq.cpu().numpy(), -1.0)
    # six gradients summed by torch (a rounding for each of at most two sums of partial results, and their own)
    bound = _rotary_bound(gk, each, sections, dtype).sum((0, 1)) + 6 * HALF[dtype] * np.abs(each).sum((0, 1))
    assert (np.abs(_np(dk)[0, 0] - each.sum((0, 1))) <= bound).all()
    # only one of the outputs is used
    _, ko = ops.rotary_axes(q, k.expand(2, 3, T, D), pos, sections, freq)
    dq, dk2 = torch.autograd.grad([ko], [q, k], [gk], allow_unused=True)
    assert dq is None and torch.equal(dk2, dk)
    if dtype == torch.float32:  # differences: the map is linear, so a difference of a long step is its rounding off
        d = _randn(g, 2, 4, T, D, dtype=dtype).cuda()
        with torch.no_grad():
            up = ops.rotary_axes(q + d, None, pos, sections, freq)[0].double()
            dn = ops.rotary_axes(q - d, None, pos, sections, freq)[0].double()
        qo = ops.rotary_axes(q, None, pos, sections, freq)[0]
        dq, = torch.autograd.grad(qo, q, gq)
        lhs = ((up - dn) / 2 * gq.double()).sum().item()
        rhs = (dq.double() * d.double()).sum().item()
        n = gq.numel()
        assert abs(lhs - rhs) <= 2.0 ** -20 * math.sqrt(n) * 40
    # a second derivative: of |turn(q)|^2 / 2 along gq, which is gq itself (a turn keeps lengths)
    qo = ops.rotary_axes(q, None, pos, sections, freq)[0]
    grad, = torch.autograd.grad(qo, q, qo, create_graph=True)
    again, = torch.autograd.grad(grad, q, gq)
    bound = 2 * _rotary_bound(gq, _np(gq), sections, dtype) + 2 ** -20
    if dtype == torch.float32:
        assert (np.abs(_np(again) - _np(gq)) <= 8 * bound).all()
    # broadcast gradient (stride 0 everywhere)
    qo = ops.rotary_axes(q, None, pos, sections, freq)[0]
    dq, = torch.autograd.grad(qo.sum(), q)
    ref = O.rotate(np.ones(q.shape), pos.cpu().numpy(), sections, freq.cpu().numpy(), -1.0)
    assert (np.abs(_np(dq) - ref) <= _rotary_bound(torch.ones(q.shape), ref, sections, dtype)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rotary_tangents(dtype):
    """A forward-mode tangent is the turn of the tangent, bit for bit; the cache operators refuse one."""
    import torch.autograd.forward_ad as fwd
    g = _gen(13)
    sections, T = (16, 24, 24), 21
    freq = _freq(sections, (10000.0, 100.0, 100.0)).cuda()
    pos = torch.randint(0, 900, (2, T, 3), generator=g).cuda()
    q, tq = (_randn(g, 2, T, 4, 64, dtype=dtype).cuda().transpose(1, 2) for _ in range(2))
    k, tk = (_randn(g, 2, 2, T, 64, dtype=dtype).cuda() for _ in range(2))
    want = ops.rotary_axes(tq, tk, pos, sections, freq)
    plain = ops.rotary_axes(q, k, pos, sections, freq)
    with fwd.dual_level():
        for grad in (False, True):
            out = ops.rotary_axes(fwd.make_dual(q.clone().requires_grad_(grad), tq), fwd.make_dual(k, tk), pos, sections, freq)
            for x, t, p in zip(out, want, plain):
                x = fwd.unpack_dual(x)
                assert torch.equal(x.primal, p) and torch.equal(x.tangent, t)
        qo, ko = ops.rotary_axes(q, fwd.make_dual(k, tk), pos, sections, freq)
        assert torch.equal(fwd.unpack_dual(ko).tangent, want[1]) and not fwd.unpack_dual(qo).tangent.any()
        if dtype != torch.float32:
            cache, table = BlockCache(1, 2, 64), _i32([[0], [0]])
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                ops.cache_attn(fwd.make_dual(q, tq), cache, table, _i32([0, 0]))
            with pytest.raises(ValueError, match="tangent"):
                ops.cache_write(cache, k, fwd.make_dual(k, tk), table, _i32([0, 0]))


def test_rotary_odd_strides_and_empty():
    """Rows that start at odd elements, a transposed layout, no tokens, no heads."""
    g = _gen(5)
    sections = (8, 8)
    freq = _freq(sections, (100.0, 100.0))
    pos = torch.randint(0, 40, (1, 19, 2), generator=g)
    wide = _randn(g, 2, 3, 19, 37).cuda()
    for x in (wide[..., 1:21], wide[..., 2:34], wide.permute(0, 2, 3, 1)[:, :, :19, :].transpose(1, 2)[..., :2]):
        if x.shape[-1] < 16:
            with pytest.raises(ValueError, match="sections"):
                ops.rotary_axes(x, None, pos.cuda(), sections, freq.cuda())
            continue
        y = ops.rotary_axes(x, None, pos.cuda(), sections, freq.cuda())[0]
        ref = O.rotate(_np(x), pos.numpy(), sections, freq.numpy())
        assert (np.abs(_np(y) - ref) <= _rotary_bound(x, ref, sections, torch.bfloat16)).all()
    e = torch.zeros(2, 3, 0, 32, device="cuda")
    out, _ = ops.rotary_axes(e, None, pos[:, :0].cuda(), sections, freq.cuda())
    assert out.shape == e.shape


# ------------------------------------------------------------------ the cache: write and read
def _fill(cache, g, table, lens, k=None, v=None):
    """Random history; returns the held values, float64 [B][H,len,D]."""
    B, H, D, L = len(lens), cache.heads, cache.head_dim, max(max(lens), 1)
    k = _randn(g, B, H, L, D) if k is None else k
    v = _randn(g, B, H, L, D) if v is None else v
    ops.cache_write(cache, k.cuda(), v.cuda(), table, _i32([0] * B), count=_i32(lens))
    held = [O.quantise(_np(k[b, :, :n]), _np(v[b, :, :n])) for b, n in enumerate(lens)]
    return held


def _same(a, b):
    return np.array_equal(a, b, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,H", [(64, 3), (128, 2)])
def test_write_then_read(dtype, D, H):
    """Values of many magnitudes at ragged places, from strided rows; every other byte of the cache stays."""
    g = _gen(D)
    B, T, mp = 4, 150, 6
    table, pages = _table(g, B, mp)
    start, count = [0, 61, 130, 64], [150, 70, 0, 1]
    cache = BlockCache(pages, H, D)
    for t in (cache.kc, cache.vc):  # finite codes everywhere
        t.copy_(torch.randint(0, 0x7e, t.shape, generator=g, dtype=torch.uint8))
    for t in (cache.ks, cache.vs):
        t.copy_(torch.randint(110, 140, t.shape, generator=g, dtype=torch.uint8))
    cache.mean.copy_(torch.randn(cache.mean.shape, generator=g))
    before = {n: getattr(cache, n).clone() for n in ("kc", "vc", "ks", "vs", "mean")}
    mag = torch.exp2(torch.randint(-12, 12, (B, T, H, 1), generator=g).float())
    k = (torch.randn(B, T, H, D, generator=g) * mag).to(dtype).cuda().transpose(1, 2)
    v = (torch.randn(B, T, H, D, generator=g) * mag.flip(1)).to(dtype).cuda().transpose(1, 2)
    old_k, old_v = ops.cache_read(cache, table, _i32([0] * B), mp * 64, dtype=torch.float32)
    ops.cache_write(cache, k, v, table, _i32(start), count=_i32(count))
    rk, rv = ops.cache_read(cache, table, _i32(start), T, count=_i32(count), dtype=torch.float32)
    all_k, all_v = ops.cache_read(cache, table, _i32([0] * B), mp * 64, dtype=torch.float32)
    touched = set()
    for b in range(B):
        s, n = start[b], count[b]
        ko, vo = O.quantise(_np(k[b, :, :n]), _np(v[b, :, :n]))
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


@pytest.mark.parametrize("D", [64, 128])
def test_write_edge_values(D):
    """Rows at the borders of the format: powers of two, 448 * 2^e and one step past it, e4m3 ties and subnormals, zero,
    the exponents' ends, float32's largest and smallest; tokens that are not finite."""
    step = 1 + 2.0 ** -10
    rows = [[448.0], [448.0 * step], [1.75, 0.4375], [1.75 * step, 1.0], [0.0], [-0.0], [2.0 ** -70, 2.0 ** -69],
            [2.0 ** -126, 2.0 ** -149], [3.0e38, 1.0], [448 * 2.0 ** 60, 2.0 ** 53], [2.0 ** 127],
            [17.0, 19.0, 21.0, 23.0, -17.0], [448.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11],
            [float("inf")], [1.0, float("nan")], [-float("inf"), 1.0]]
    x = torch.zeros(1, 1, len(rows), D)
    for i, r in enumerate(rows):
        x[0, 0, i, :len(r)] = torch.tensor(r, dtype=torch.float64).float()
        x[0, 0, i, D - 1] = x[0, 0, i, 0]
    y = torch.full_like(x, 0.5)
    y[0, 0, 2, 5] = float("nan")  # a value that is not finite marks the token's key too
    table = _i32([[1]])
    for a, b in ((x, y), (y, x)):
        cache = BlockCache(2, 1, D)
        ops.cache_write(cache, a.cuda(), b.cuda(), table, _i32([0]))
        k, v = ops.cache_read(cache, table, _i32([0]), len(rows), dtype=torch.float32)
        ko, vo = O.quantise(_np(a), _np(b))
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
    H, D, n = 2, 64, 200
    k, v = _randn(g, 1, H, n, D).cuda(), _randn(g, 1, H, n, D).cuda()
    table, pages = _table(g, 1, 4)
    caches = []
    for cuts in ([n], list(range(1, n + 1)), [3, 63, 64, 65, 127, 130, 192, n]):
        c, at = BlockCache(pages, H, D), 0
        for e in cuts:
            ops.cache_write(c, k[:, :, at:e], v[:, :, at:e], table, _i32([at]))
            at = e
        caches.append(c)
    for c in caches[1:]:
        for name in ("kc", "vc", "ks", "vs", "mean"):
            assert torch.equal(getattr(c, name), getattr(caches[0], name)), name


def test_write_and_read_outside_the_table():
    """Entries that are no page, a start past the table or below 0, more tokens than the table holds: nothing is written
    there, and zeros are read."""
    g = _gen(23)
    cache = BlockCache(3, 1, 64)
    table = _i32([[0, -1], [7, 1], [2, 3], [-5, -5], [5, 4]])
    k, v = _randn(g, 5, 1, 200, 64).cuda(), _randn(g, 5, 1, 200, 64).cuda()
    ops.cache_write(cache, k, v, table, _i32([0, 0, 0, 10, -3]))
    rk, rv = ops.cache_read(cache, table, _i32([0, 0, 0, 10, -3]), 200, dtype=torch.float32)
    for b, (lo, hi) in enumerate(((0, 64), (64, 128), (0, 64), (0, 0), (0, 0))):
        ko, vo = O.quantise(_np(k[b, :, lo:hi]), _np(v[b, :, lo:hi]))
        assert _same(_np(rk[b, :, lo:hi]), ko) and _same(_np(rv[b, :, lo:hi]), vo)
        for r in (rk, rv):
            assert not r[b, :, :lo].any() and not r[b, :, hi:].any()
    before = cache.kc.clone()
    ops.cache_write(cache, k, v, table, _i32([128, 2 ** 31 - 1, 1000, -2 ** 31, -1]))
    assert torch.equal(before, cache.kc)
    far, _ = ops.cache_read(cache, table, _i32([128, 2 ** 31 - 1, 1000, -2 ** 31, -1]), 70)
    assert not far.any()


# ------------------------------------------------------------------ choice
def _check_select(q, cache, table, lens, held, keep, block_q, sink, recent, causal, n_q=None):
    B, Hq, T, D = q.shape
    H, mp = cache.heads, table.shape[1]
    G, U = Hq // H, -(-T // block_q)
    index, count, score = ops.cache_select(q, cache, table, _i32(lens), keep, block_q=block_q, sink=sink, recent=recent,
                                           causal=causal, q_count=None if n_q is None else _i32(n_q), want_score=True)
    assert index.shape == (B, H, U, min(mp, sink + keep + recent + ((block_q + 62) // 64 if causal else 0)))
    i2, c2 = ops.cache_select(q, cache, table, _i32(lens), keep, block_q=block_q, sink=sink, recent=recent, causal=causal,
                              q_count=None if n_q is None else _i32(n_q))
    assert torch.equal(index, i2) and torch.equal(count, c2)
    qn, index, count, score = _np(q), index.cpu().numpy(), count.cpu().numpy(), score.cpu().numpy()
    for b in range(B):
        nq = T if n_q is None else n_q[b]
        for h in range(H):
            means = O.page_means(held[b][0][h])
            for u in range(U):
                t0, t1 = u * block_q, min((u + 1) * block_q, nq)
                seen, own = O.unit_pages(lens[b], nq, t0, t1, causal)
                if seen == 0:
                    want, s = [], np.zeros(0, np.float32)
                else:
                    rows = qn[b, h * G:(h + 1) * G, t0:t1].reshape(-1, D)
                    want, s = O.select(rows, means, seen, own, keep, sink, recent)
                n = count[b, h, u]
                assert n == len(want), (b, h, u)
                assert list(index[b, h, u, :n]) == want and (index[b, h, u, n:] == -1).all(), (b, h, u)
                assert np.array_equal(score[b, h, u, :seen], s) and (score[b, h, u, seen:] == -np.inf).all()


@pytest.mark.parametrize("D,H,G,T,block_q,causal", [(64, 2, 1, 1, 1, False), (128, 1, 5, 1, 1, False),
                                                    (64, 1, 1, 300, 128, False), (128, 2, 4, 70, 32, True),
                                                    (64, 2, 2, 130, 64, True), (64, 1, 128, 2, 1, False),
                                                    (64, 1, 1, 9, 3, True)])
def test_select_matches_definition(D, H, G, T, block_q, causal):
    g = _gen(D + G + T)
    lens = [1500, 64, 1, 0, 777, T]
    if causal:
        lens = [max(n, T) for n in lens]
    table, pages = _table(g, len(lens), 25)
    cache = BlockCache(pages, H, D)
    held = _fill(cache, g, table, lens)
    q = _randn(g, len(lens), H * G, T, D).cuda()
    for keep, sink, recent in ((5, 1, 1), (0, 2, 3), (40, 0, 1)):
        _check_select(q, cache, table, lens, held, keep, block_q, sink, recent, causal)


@pytest.mark.parametrize("mp", [1, 255, 257, 2049, 8200])
def test_select_long_tables(mp):
    """Around the sizes at which the list kernel changes."""
    g = _gen(mp)
    H, D = 1, 64
    table, pages = _table(g, 2, mp)
    cache = BlockCache(pages, H, D)
    lens = [mp * 64, mp * 64 - min(mp * 64, 100)]
    means = torch.randn(pages, H, D, generator=g).bfloat16()
    cache.mean.copy_(means)
    q = _randn(g, 2, 2, 1, D).cuda()
    for keep in (max(1, mp // 4), 3, mp - 1):
        index, count, score = ops.cache_select(q, cache, table, _i32(lens), keep, want_score=True)
        for b in range(2):
            m = _np(means)[table[b].cpu().numpy(), 0]
            want, s = O.select(_np(q)[b, :, 0], m, -(-lens[b] // 64), -(-lens[b] // 64) - 1, keep, 1, 1)
            assert count[b, 0, 0] == len(want) and index[b, 0, 0, :len(want)].tolist() == want
            assert np.array_equal(score[b, 0, 0, :len(s)].cpu().numpy(), s)


def test_select_ties_nan_and_missing_pages():
    """Equal scores go by page; NaN and missing pages come last; +0 and -0 are equal; queries past q_count choose nothing."""
    H, D, mp = 1, 64, 600
    cache = BlockCache(mp, H, D)
    g = _gen(9)
    level = torch.randint(-2, 3, (mp,), generator=g).float()
    cache.mean[:, 0, 0] = level.cuda().bfloat16()
    cache.mean[50, 0, 3] = float("nan")
    cache.mean[60, 0, 0] = -0.0
    table = torch.arange(mp, dtype=torch.int32).view(1, mp).cuda()
    table[0, 70] = -1
    table[0, 80] = mp
    q = torch.zeros(1, 1, 3, D, dtype=torch.bfloat16, device="cuda")
    q[0, 0, :, 0] = torch.tensor([1.0, -1.0, 0.0], device="cuda")
    means = _np(cache.mean)[:, 0]
    means[70] = means[80] = np.nan
    for keep in (1, 100, 130, 350, 595, 598):
        index, count = ops.cache_select(q, cache, table, _i32([mp * 64 - 5]), keep, sink=1, recent=1, q_count=_i32([2]))
        for t in range(2):
            want, _ = O.select(_np(q)[0, :, t], means, mp, mp - 1, keep, 1, 1)
            assert index[0, 0, t, :len(want)].tolist() == want and count[0, 0, t] == len(want)
        assert count[0, 0, 2] == 0 and (index[0, 0, 2] == -1).all()


@pytest.mark.parametrize("mp", [200, 600, 4000, 9000])
def test_select_equal_and_close_scores(mp):
    """All scores equal (the list is the first pages), equal in two halves, and apart in their last bits only."""
    g = _gen(mp)
    cache = BlockCache(mp, 1, 64)
    table = torch.arange(mp, dtype=torch.int32).view(1, mp).cuda()
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda")
    q[..., 0], q[..., 1] = 1.0, 2.0 ** -9
    for kind in range(3):
        m = torch.zeros(mp, 64)
        if kind == 1:
            m[::2, 0] = -1.0
        if kind == 2:
            m[:, 0] = -1.0
            m[:, 1] = torch.randint(0, 200, (mp,), generator=g).float() * 2.0 ** -7
        cache.mean[:, 0] = m.bfloat16().cuda()
        for keep in (1, 7, mp // 2 - 1, mp // 2, mp - 3):
            index, count = ops.cache_select(q, cache, table, _i32([mp * 64]), keep)
            want, _ = O.select(_np(q)[0, :, 0], _np(cache.mean)[:, 0], mp, mp - 1, keep, 1, 1)
            assert count.item() == len(want) and index[0, 0, 0, :len(want)].tolist() == want


# ------------------------------------------------------------------ attention
def _check_attend(o, q, held, lens, lists, block_q, causal, scale=None, n_q=None, H=None):
    """o against float64 over the held values. Bound for an element: the output's rounding; weights rounded to half
    (2^-11 of each term); an error of the float32 logits in weights and sum, (D + 8) 2^-24 of the products' magnitudes;
    float32 sums over n keys, n 2^-24 of the terms' magnitudes, twice (weights and their sum), and 2^-14.5 for exp2,
    the powers, the division and the exponents: logits are summed on top of a reference whose size is up to 2^8 + 2 |logit| (the
    values' biased exponents, up to 187, and the largest logit), so each of its two roundings is up to 2^-24 (2^8 + 2
    |logit|) ln 2 of a weight, and again in the sum: 4 * 2^-24 * 2^8 ln 2 < 2^-14.5; the logits' part
    is in (D + 8). Weights under 2^-36 of the largest, at most n of them."""
    B, Hq, T, D = q.shape
    G = Hq // H
    scale = D ** -0.5 if scale is None else scale
    qn, on = _np(q), _np(o)
    assert not np.isnan(on).any()
    worst = 0.0
    for b in range(B):
        nq = T if n_q is None else n_q[b]
        for h in range(H):
            k, v = held[b][0][h], held[b][1][h]
            pos = np.arange(len(k))
            for t in range(T):
                seen = pos < lens[b]
                if lists is not None:
                    seen &= np.isin(pos // 64, lists[b][h][t // block_q])
                if causal:
                    seen &= pos <= lens[b] - nq + t
                if t >= nq:
                    seen &= False
                for gi in range(G):
                    ref, mag, logit = O.attend(qn[b, h * G + gi, t], k, v, seen, scale)
                    n = int(seen.sum())
                    rel = 2.0 ** -11 + 2 * ((D + 8) * 2.0 ** -24 * logit + n * 2.0 ** -24) + 2.0 ** -14.5
                    bound = rel * mag + HALF[o.dtype] * (np.abs(ref) + rel * mag) + n * 2.0 ** -36 * np.abs(v).max(initial=0)
                    if o.dtype == torch.float16:
                        bound = bound + 2.0 ** -25
                    err = np.abs(on[b, h * G + gi, t] - ref)
                    assert (err <= bound).all(), (b, h, t, gi, (err - bound).max())
                    worst = max(worst, float((err / (bound + 1e-30)).max()))
    return worst


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,G", [(64, 2, 1), (128, 1, 4), (64, 1, 12), (128, 2, 1)])
def test_attend_single_tokens(dtype, D, H, G):
    g = _gen(D + G)
    lens = [1, 63, 64, 65, 0, 700, 1300]
    table, pages = _table(g, len(lens), 21)
    cache = BlockCache(pages, H, D)
    held = _fill(cache, g, table, lens)
    q = _randn(g, len(lens), H * G, 1, D, dtype=dtype).cuda()
    o = ops.cache_attn(q, cache, table, _i32(lens))
    assert o.dtype == dtype
    _check_attend(o, q, held, lens, None, 1, False, H=H)
    assert not o[4].any()
    for keep in (0, 3):
        index, count = ops.cache_select(q, cache, table, _i32(lens), keep)
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
    cache = BlockCache(pages, H, D)
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
    """Few units over many pages: each split over some dozens of workgroups, joined by groups that share a row."""
    g = _gen(L)
    table, pages = _table(g, 2, -(-L // 64))
    cache = BlockCache(pages, H, D)
    lens = [L, 100]  # most parts of the second have no page
    held = _fill(cache, g, table, lens)
    q = _randn(g, 2, H * G, T, D).cuda()
    o = ops.cache_attn(q, cache, table, _i32(lens))
    _check_attend(o, q, held, lens, None, 1, False, H=H)
    assert not ops.cache_attn(q, cache, table, _i32([0, 0])).any()


def test_attend_list_rules():
    """Entries that repeat, fall back, lie outside or have no page are skipped; counts are cut to the list; rows that see
    nothing are zero."""
    g = _gen(31)
    D, H, L = 64, 1, 640
    table, pages = _table(g, 1, 12)
    cache = BlockCache(pages, H, D)
    held = _fill(cache, g, table, [L])
    table[0, 4] = -1
    q = _randn(g, 1, 1, 8, D).cuda()
    rows = [[0, 2, 2, 5, 9, -1], [3, 1, 5, 5, 5, 5], [-1, -1, 7, 8, 9, 10], [4, 10, 11, 12, 300, 7], [0, 1, 2, 3, 4, 5],
            [6, 7, 8, 9, 10, 11], [0, 1, 2, 3, 4, 5], [2, -7, 5, 6, 7, 8]]
    counts = [6, 6, 6, 6, 3, 99, 0, -4]
    want = [[0, 2, 5, 9], [3, 5], [7, 8, 9], [], [0, 1, 2], [6, 7, 8, 9], [], []]
    o = ops.cache_attn(q, cache, table, _i32([L]), _i32(rows).view(1, 1, 8, 6), _i32(counts).view(1, 1, 8), block_q=1)
    _check_attend(o, q, held, [L], [[want]], 1, False, H=1)
    for t in (3, 6, 7):
        assert not o[0, 0, t].any()


def test_attend_masked_values_do_not_matter():
    """NaN tokens past the length or behind a causal row change nothing; seen ones make exactly their rows NaN. Keys whose
    logits are far apart, values whose powers are far apart, zero rows."""
    g = _gen(37)
    D, H, T, L = 64, 1, 40, 200
    table, pages = _table(g, 1, 4)
    k, v = _randn(g, 1, H, L, D), _randn(g, 1, H, L, D)
    v[0, 0, 10:20] *= 2.0 ** 40
    v[0, 0, 20:30] *= 2.0 ** -40
    v[0, 0, 64:128] = 0
    k[0, 0, 30:40] *= 40
    cache = BlockCache(pages, H, D)
    held = _fill(cache, g, table, [L], k, v)
    q = _randn(g, 1, H, T, D).cuda()
    base = ops.cache_attn(q, cache, table, _i32([L]), causal=True)
    _check_attend(base, q, held, [L], None, 1, True, H=1)
    v[0, 0, 190, 5] = float("nan")
    _fill(cache, g, table, [L], k, v)
    o = ops.cache_attn(q, cache, table, _i32([L]), causal=True)
    # rows up to position 189 do not see token 190
    assert torch.equal(o[0, 0, :30], base[0, 0, :30]) and o[0, 0, 30:].isnan().all()
    o = ops.cache_attn(q[:, :, :5], cache, table, _i32([190]))
    _check_attend(o, q[:, :, :5], [(held[0][0][:, :190], held[0][1][:, :190])], [190], None, 1, False, H=1)


@pytest.mark.parametrize("D,G,T", [(64, 1, 1), (128, 20, 1), (64, 1, 100), (128, 4, 30)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend_nan_tokens_and_queries(D, G, T, dtype):
    """In every kernel: a NaN token makes the rows that see it NaN and no others, as does an infinite query."""
    g = _gen(D + T)
    table, pages = _table(g, 2, 5)
    cache = BlockCache(pages, 1, D)
    k, v = _randn(g, 2, 1, 300, D), _randn(g, 2, 1, 300, D)
    k[1, 0, 150, 3] = float("inf")
    held = _fill(cache, g, table, [300, 300], k, v)
    q = _randn(g, 2, G, T, D, dtype=dtype).cuda()
    o = ops.cache_attn(q, cache, table, _i32([300, 300]))
    assert o[1].isnan().all()
    _check_attend(o[:1], q[:1], held[:1], [300], None, 1, False, H=1)
    o = ops.cache_attn(q, cache, table, _i32([300, 150]))
    cut = [held[0], (held[1][0][:, :150], held[1][1][:, :150])]
    _check_attend(o, q, cut, [300, 150], None, 1, False, H=1)
    q[0, G - 1, T - 1, 7] = float("inf")
    o2 = ops.cache_attn(q, cache, table, _i32([300, 150]))
    assert o2[0, G - 1, T - 1].isnan().all()
    o2[0, G - 1, T - 1] = o[0, G - 1, T - 1]
    assert torch.equal(o2, o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,G,T,mp,parts", [(64, 1, 1, 1, 8, 1), (64, 64, 1, 1, 200, 8), (64, 1, 1, 1, 140, 35),
                                              (128, 64, 20, 1, 200, 4), (128, 1, 20, 1, 140, 35), (64, 1, 1, 50, 8, 8),
                                              (64, 1, 1, 100, 24, 24), (128, 1, 4, 30, 3, 3), (128, 1, 4, 30, 100, 100)])
def test_attend_nan_in_split_pages(D, H, G, T, mp, parts, dtype):
    """The pages of a unit on one workgroup or on some, joined a row a lane group or a row a workgroup: rows that see a NaN
    token are NaN where it shares its part with others, fills it, fills the first parts or is all there is, and so are NaN
    queries; every other row is as without them."""
    block_q = max(1, min(T, 128 // G))
    units = 2 * H * -(-T // block_q)
    size = _lib.fn("vasc_cache_attn_workspace_size")(2, H * G, H, T, D, block_q, mp, 0)
    assert size == (units * block_q * G * parts * (D + 2) * 4 if parts > 1 else 0)
    g = _gen(D + T + mp)
    table, pages = _table(g, 2, mp)
    full = min(mp, 7) * 64
    k, v = _randn(g, 2, H, full, D), _randn(g, 2, H, full, D)
    q = _randn(g, 2, H * G, T, D, dtype=dtype).cuda()

    def attend(bad, length, queries=q, **rule):
        """With NaN in the tokens `bad` of the second sequence."""
        cache = BlockCache(pages, H, D)
        kn = k.clone()
        kn[1, :, bad, 5] = float("nan")
        ops.cache_write(cache, kn.cuda(), v.cuda(), table, _i32([0, 0]))
        return ops.cache_attn(queries, cache, table, _i32([full, length]), **rule)

    for bad, length in ((slice(70, 71), full), (slice(64, 128), full), (slice(0, full - 64), full), (slice(64, 65), 65),
                        (slice(0, 1), 1), (slice(0, full), full)):
        base, o = attend(slice(0, 0), length), attend(bad, length)
        assert torch.equal(o[0], base[0]) and base.isfinite().all()
        assert o[1].isnan().all(), (bad, length)
        # masked for every row
        cut = bad.start
        assert torch.equal(attend(bad, cut), attend(slice(0, 0), cut)), (bad, cut)
        if T > 1:  # the queries are the last T tokens: those before the first bad token do not see it
            base, o = attend(slice(0, 0), length, causal=True), attend(bad, length, causal=True)
            blind = min(max(0, bad.start - (length - T)), T)
            assert torch.equal(o[0], base[0]) and torch.equal(o[1, :, :blind], base[1, :, :blind])
            assert o[1, :, blind:].isnan().all(), (bad, length)
    base = attend(slice(0, 0), full)
    qn = q.clone()
    qn[1, H * G - 1, T - 1, 3] = float("nan")
    o = attend(slice(0, 0), full, qn)
    assert o[1, H * G - 1, T - 1].isnan().all()
    o[1, H * G - 1, T - 1] = base[1, H * G - 1, T - 1]
    assert torch.equal(o, base)
    assert not attend(slice(0, 0), 0, qn)[1].any()  # it sees no key


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,G,T,mp", [(64, 1, 1, 6), (64, 1, 1, 140), (128, 20, 1, 6), (64, 1, 100, 6), (128, 4, 30, 140)])
def test_attend_infinite_queries(D, G, T, mp, dtype):
    """An infinite query has no softmax over any key, also where all its logits are minus infinity: its rows are NaN, or zero
    where they see no key."""
    g = _gen(D + T + mp)
    L = 300
    table, pages = _table(g, 1, mp)
    cache = BlockCache(pages, 1, D)
    k = _randn(g, 1, 1, L, D)
    k[..., 7] = -k[..., 7].abs() - 0.25
    held = _fill(cache, g, table, [L], k)
    q = _randn(g, 1, G, T, D, dtype=dtype).cuda()
    base = ops.cache_attn(q, cache, table, _i32([L]))
    _check_attend(base, q, held, [L], None, 1, False, H=1)
    for value in (float("inf"), -float("inf")):
        bad = q.clone()
        bad[0, 0, T - 1, 7] = value
        o = ops.cache_attn(bad, cache, table, _i32([L]))
        assert o[0, 0, T - 1].isnan().all()
        o[0, 0, T - 1] = base[0, 0, T - 1]
        assert torch.equal(o, base)
        assert not ops.cache_attn(bad, cache, table, _i32([0])).any()


def test_attend_wide_logits_and_scale():
    """Logits of hundreds: one key takes all; the running maximum moves many times; a scale of the caller's."""
    g = _gen(41)
    D, H, L = 128, 1, 900
    table, pages = _table(g, 1, 15)
    cache = BlockCache(pages, H, D)
    k = _randn(g, 1, H, L, D) * torch.linspace(0.1, 6, L).view(1, 1, L, 1).bfloat16()
    held = _fill(cache, g, table, [L], k)
    q = (_randn(g, 1, 3, 1, D) * 4).cuda()
    for scale in (1.0, 0.01, 0.0):
        o = ops.cache_attn(q, cache, table, _i32([L]), scale=scale)
        _check_attend(o, q, held, [L], None, 1, False, scale=scale, H=1)


def test_integers_of_64_bits():
    """Starts, lengths, tables and lists past 32 bits on the GPU: nothing is written or seen there; within it, as int32."""
    g = _gen(107)
    cache = BlockCache(3, 1, 64)
    k = _randn(g, 2, 1, 70, 64).cuda()
    far = torch.tensor([[2 ** 32, 2 ** 33 + 1], [1, -2 ** 32 + 2]], device="cuda")
    ops.cache_write(cache, k, k, far, torch.tensor([2 ** 32, -2 ** 32], device="cuda"))
    assert not cache.kc.any()
    ops.cache_write(cache, k, k, far, torch.tensor([0, 0], device="cuda"))
    assert not cache.kc[[0, 2]].any() and cache.kc[1].any()
    held = [(np.zeros((1, 0, 64)),) * 2, O.quantise(_np(k[1, :, :64]), _np(k[1, :, :64]))]
    q = _randn(g, 2, 1, 1, 64).cuda()
    lists, count = torch.tensor([0, 2 ** 32 + 1, 1], device="cuda").expand(2, 1, 1, 3), torch.tensor([3], device="cuda").expand(2, 1, 1)
    for length in (64, 2 ** 40):
        n = torch.tensor([length] * 2, device="cuda")
        assert not ops.cache_attn(q[:1], cache, far[:1], n[:1]).any()
        _check_attend(ops.cache_attn(q, cache, far, n, lists, count), q, held, [0, 64], [[[[]]], [[[0]]]], 1, False, H=1)
    assert not ops.cache_attn(q, cache, far, torch.tensor([-2 ** 32 + 64] * 2, device="cuda")).any()


@pytest.mark.parametrize("D,G,T,mp", [(64, 1, 1, 6), (64, 1, 1, 140), (128, 20, 1, 6), (64, 1, 100, 6), (128, 4, 30, 6)])
def test_attend_scales(D, G, T, mp):
    """Scales below zero, hardly above it and far above one, in every kernel."""
    g = _gen(D + T + mp)
    L = 300
    table, pages = _table(g, 1, mp)
    cache = BlockCache(pages, 1, D)
    held = _fill(cache, g, table, [L])
    q = _randn(g, 1, G, T, D).cuda()
    for scale in (-0.125, 1e-29, -1e-29, 3.0):
        o = ops.cache_attn(q, cache, table, _i32([L]), scale=scale)
        # of the bound, what grows with the logits goes by their magnitude
        _check_attend(o, q if scale > 0 else -q, held, [L], None, 1, False, scale=abs(scale), H=1)


def test_rows_cut_from_wider_ones():
    """One token of one sequence and head out of rows of odd width, written and asked for: strides of dimensions of size one."""
    g = _gen(83)
    wide = _randn(g, 3, 1, 1, 1, 65).cuda()
    for shift in (0, 1):  # aligned rows, and rows that are not
        q, k, v = (t[..., shift:shift + 64] for t in wide)
        cache, table = BlockCache(1, 1, 64), _i32([[0]])
        ops.cache_write(cache, k, v, table, _i32([0]))
        held = [O.quantise(_np(k[0]), _np(v[0]))]
        _check_attend(ops.cache_attn(q, cache, table, _i32([1])), q, held, [1], None, 1, False, H=1)
        index, count = ops.cache_select(q, cache, table, _i32([1]), 1)
        assert index.tolist() == [[[[0]]]] and count.item() == 1


@pytest.mark.parametrize("L,apart", [(400, 7), (400, -56), (20000, 18)])
@pytest.mark.parametrize("D,G,T,wide", [(64, 1, 1, False), (64, 1, 1, True), (128, 20, 1, False), (64, 1, 40, False),
                                        (64, 2, 60, True), (128, 4, 30, False)])
def test_attend_values_far_apart(L, apart, D, G, T, wide):
    """One key whose value row is at the exponents' upper end, `apart` powers of two more likely than all the others, whose
    rows are zero or at the lower end: they count in the softmax's sum with all their weight (300 of 2^-7 are 3 times the one,
    20000 of 2^-18 are 7 % of it). It is the first key, the last, or in the middle; pages on one workgroup or split."""
    mp = -(-L // 64) + (140 if wide else 0)
    g = _gen(L)
    table, pages = _table(g, 4, mp)
    q = torch.zeros(4, G, T, D, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    k, v = torch.zeros(4, 1, L, D), torch.zeros(4, 1, L, D)
    for b, at in enumerate((0, L // 2 + 5, L - 1, 70)):
        k[b, 0, at, 0] = apart
        v[b, 0, :, 1] = 0.0 if b % 2 else 448 * 2.0 ** -60
        v[b, 0, at] = torch.linspace(224, 448, 8).repeat(D // 8) * 2.0 ** 60
        v[b, 0, at, 1] = -448 * 2.0 ** 60
    cache = BlockCache(pages, 1, D)
    ops.cache_write(cache, k.cuda(), v.cuda(), table, _i32([0] * 4))
    hk, hv = ops.cache_read(cache, table, _i32([0] * 4), L, dtype=torch.float32)
    assert torch.equal(hk.cpu(), k) and torch.equal(hv.cpu(), v)  # all of it is what 8 bits hold
    held = [(_np(k[b]), _np(v[b])) for b in range(4)]
    o = ops.cache_attn(q.cuda(), cache, table, _i32([L] * 4), scale=math.log(2.0))
    _check_attend(o[:, :1, :1], q[:, :1, :1], held, [L] * 4, None, 1, False, scale=math.log(2.0), H=1)
    assert (o == o[:, :1, :1]).all()
    lists = torch.arange(-(-L // 64), dtype=torch.int32, device="cuda")[1:].expand(4, 1, T, -1)
    count = _i32([lists.shape[3]]).expand(4, 1, T)
    o = ops.cache_attn(q.cuda(), cache, table, _i32([L] * 4), lists, count, block_q=1, scale=math.log(2.0))
    _check_attend(o[:, :1, :1], q[:, :1, :1], held, [L] * 4, [[[list(range(1, -(-L // 64)))]]] * 4, 1, False,
                  scale=math.log(2.0), H=1)


def test_attend_strided_tensors_and_out():
    g = _gen(43)
    D, H, T, L = 64, 2, 6, 333
    table, pages = _table(g, 2, 6)
    wide = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, :6] = table
    cache = BlockCache(pages, H, D)
    held = _fill(cache, g, table, [L, L - 9])
    qkv = _randn(g, 2, T, 3, H * 2, D).cuda()
    q = qkv[:, :, 1].transpose(1, 2)
    rows = torch.full((2, T, H * 2, D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    out = rows[..., :D].transpose(1, 2)
    o = ops.cache_attn(q, cache, wide[:, :6], _i32([L, L - 9]), out=out)
    assert o.data_ptr() == rows.data_ptr() and (rows[..., D:] == 7.0).all()
    _check_attend(o, q, held, [L, L - 9], None, 1, False, H=H)
    again = ops.cache_attn(q, cache, wide[:, :6], torch.tensor([L, L - 9], device="cuda"))  # int64 lengths
    assert torch.equal(again, o)


@pytest.mark.parametrize("how", ["deepcopy", "copy", "pickle", "save"])
def test_copied_cache(how, tmp_path):
    """A deep copy, a pickled and a saved cache have buffers of their own, at their own addresses; a shallow copy shares them."""
    g = _gen(59)
    table, pages = _table(g, 1, 3)
    cache = BlockCache(pages, 2, 64)
    held = _fill(cache, g, table, [100])
    if how == "save":
        torch.save(cache, tmp_path / "cache")
        other = torch.load(tmp_path / "cache", weights_only=False)
    else:
        other = {"deepcopy": copy.deepcopy, "copy": copy.copy, "pickle": lambda c: pickle.loads(pickle.dumps(c))}[how](cache)
    buffers = ("kc", "vc", "ks", "vs")
    assert other.pointers == tuple(getattr(other, n).data_ptr() for n in buffers)
    assert other.mean_pointer == other.mean.data_ptr() and other.device_index == cache.device_index
    assert (other.pointers == cache.pointers) == (how == "copy")
    more = _randn(g, 1, 2, 30, 64).cuda()
    before = {n: getattr(cache, n).clone() for n in (*buffers, "mean")}
    ops.cache_write(other, more, more, table, _i32([100]))
    assert all(torch.equal(getattr(cache, n), t) for n, t in before.items()) == (how != "copy")
    q = _randn(g, 1, 2, 1, 64).cuda()
    new = O.quantise(_np(more[0]), _np(more[0]))
    both = [tuple(np.concatenate([a, b], 1) for a, b in zip(held[0], new))]
    _check_attend(ops.cache_attn(q, other, table, _i32([130])), q, both, [130], None, 1, False, H=2)
    _check_attend(ops.cache_attn(q, cache, table, _i32([100])), q, held, [100], None, 1, False, H=2)


def test_offsets_past_32_bits():
    """A cache whose codes lie past 2^32 bytes, written, chosen from and attended to at both ends."""
    g = _gen(47)
    H, D = 8, 128
    pages = (2 ** 32) // (H * 64 * D) + 40
    cache = BlockCache(pages, H, D)
    table = torch.stack([torch.arange(pages - 12, pages), torch.arange(12)]).to(torch.int32).cuda()
    lens = [700, 650]
    held = _fill(cache, g, table, lens)
    rk, rv = ops.cache_read(cache, table, _i32([0, 0]), 700, count=_i32(lens), dtype=torch.float32)
    for b, n in enumerate(lens):
        assert _same(_np(rk[b, :, :n]), held[b][0]) and _same(_np(rv[b, :, :n]), held[b][1])
    q = _randn(g, 2, H, 1, D).cuda()
    _check_select(q, cache, table, lens, held, 3, 1, 1, 1, False)
    o = ops.cache_attn(q, cache, table, _i32(lens))
    _check_attend(o, q, held, lens, None, 1, False, H=H)


def test_rotary_backward_captured():
    """A captured forward and backward is refused while an eager graph of its leaves lives; without one, every replay
    equals the eager result."""
    g = _gen(71)
    sections, T = (16, 24, 24), 50
    freq = _freq(sections, (10000.0, 100.0, 100.0)).cuda()
    pos = torch.randint(0, 900, (1, T, 3), generator=g).cuda().int()
    q, k = _randn(g, 1, 4, T, 64).cuda().requires_grad_(), _randn(g, 1, 2, T, 64).cuda().requires_grad_()
    gq, gk = _randn(g, 1, 4, T, 64).cuda(), _randn(g, 1, 2, T, 64).cuda()

    def both():
        out = ops.rotary_axes(q, k, pos, sections, freq)
        return [*(x.detach() for x in out), *torch.autograd.grad(out, (q, k), (gq, gk))]

    eager = ops.rotary_axes(q, None, pos, sections, freq)[0]
    refused = None
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        try:
            ops.rotary_axes(q, k, pos, sections, freq)
        except ValueError as e:
            refused = str(e)
    assert refused is not None and "eager graph" in refused
    del eager
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(4):
        with torch.no_grad():
            for x in (q, k, gq, gk):
                x.copy_(_randn(g, *x.shape))
        graph.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        torch.randn(1 << 16, device="cuda").sum().item()  # other work between replays


# ------------------------------------------------------------------ a run of them
def _step(cache, q, k, v, pos, table, start, lengths, freq, sections, block_q):
    q, k = ops.rotary_axes(q, k, pos, sections, freq)
    ops.cache_write(cache, k, v, table, start)
    index, count = ops.cache_select(q, cache, table, lengths, 2, block_q=block_q)
    return ops.cache_attn(q, cache, table, lengths, index, count, block_q=block_q)


@pytest.mark.parametrize("T", [1, 37])
def test_step_captured_in_graphs(T):
    """rotary, write, choice and attention in two graphs with their own memory, replayed in turn with eager work between:
    each replay equals the eager run. The lengths live on the device, so one graph serves every step."""
    g = _gen(T)
    H, G, D, block_q = 2, 2, 64, 32
    sections = (16, 24, 24)
    freq = _freq(sections, (10000.0, 100.0, 100.0)).cuda()
    table, pages = _table(g, 2, 10)
    steps = 5
    qs = [_randn(g, 2, H * G, T, D).cuda() for _ in range(steps)]
    ks = [_randn(g, 2, H, T, D).cuda() for _ in range(steps)]
    vs = [_randn(g, 2, H, T, D).cuda() for _ in range(steps)]
    ps = [torch.randint(0, 99, (2, T, 3), generator=g).cuda().int() for _ in range(steps)]
    start0 = [70, 3]

    def history():
        c = BlockCache(pages, H, D)
        gg = _gen(99)
        k, v = _randn(gg, 2, H, 70, D).cuda(), _randn(gg, 2, H, 70, D).cuda()
        ops.cache_write(c, k, v, table, _i32([0, 0]), count=_i32(start0))
        return c

    eager, cache = [], history()
    for i in range(steps):
        s = _i32(start0) + i * T
        eager.append(_step(cache, qs[i], ks[i], vs[i], ps[i], table, s, s + T, freq, sections, block_q))
    graphs = []
    for _ in range(2):
        c = history()
        # the cache and the inputs live as long as their graph does
        st = dict(cache=c, q=qs[0].clone(), k=ks[0].clone(), v=vs[0].clone(), pos=ps[0].clone(), start=_i32(start0),
                  lengths=_i32(start0) + T)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(c, st["q"], st["k"], st["v"], st["pos"], table, st["start"], st["lengths"], freq, sections, block_q)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(c, st["q"], st["k"], st["v"], st["pos"], table, st["start"], st["lengths"], freq, sections, block_q)
        graphs.append((graph, st, out))
    for i in range(steps):
        for graph, st, out in graphs:
            for name, src in (("q", qs), ("k", ks), ("v", vs), ("pos", ps)):
                st[name].copy_(src[i])
            st["start"].copy_(_i32(start0) + i * T)
            st["lengths"].copy_(st["start"] + T)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager[i]), i
            torch.randn(1 << 16, device="cuda").sum().item()  # other work between replays


def test_two_streams_at_once():
    """Two sequences' attention on streams of their own: separate workspaces, same results as one after the other."""
    g = _gen(53)
    H, D, L = 2, 64, 4000
    table, pages = _table(g, 2, 63)
    cache = BlockCache(pages, H, D)
    k, v = _randn(g, 2, H, L, D).cuda(), _randn(g, 2, H, L, D).cuda()
    ops.cache_write(cache, k, v, table, _i32([0, 0]))
    q = _randn(g, 2, H, 1, D).cuda()
    n = _i32([L])
    want = [ops.cache_attn(q[b:b + 1], cache, table[b:b + 1], n) for b in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for b, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[b].append(ops.cache_attn(q[b:b + 1], cache, table[b:b + 1], n))
    torch.cuda.synchronize()
    for b in range(2):
        assert all(torch.equal(x, want[b]) for x in got[b])


# ------------------------------------------------------------------ the modules
def _module(dim=256, heads=4, rope=None, seed=0):
    from vasc_amd.aggregator import Attention
    torch.manual_seed(seed)
    m = Attention(dim, heads, rope=rope).cuda().to(torch.bfloat16)
    with torch.no_grad():
        for n in (m.q_norm, m.k_norm):
            n.weight.normal_(1.0, 0.2)
            n.bias.normal_(0.0, 0.2)
    return m


def test_rotary_axes_module_is_the_2d_one():
    """Two sections of half a head, one frequency: RotaryPositionEmbedding2D, whose float32 tables and products are within a
    step of these (float32 tokens: cos and sin off by 2^-24, two products and a sum, on both sides)."""
    from vasc_amd.aggregator import RotaryPositionEmbedding2D, RotaryPositionEmbeddingAxes
    g = _gen(61)
    x = torch.randn(2, 3, 50, 64, generator=g).cuda()
    pos = torch.randint(0, 4000, (2, 50, 2), generator=g).cuda()
    a = RotaryPositionEmbedding2D(100.0)(x, pos)
    b = RotaryPositionEmbeddingAxes((32, 32), 100.0)(x, pos)
    assert (a - b).abs().max().item() <= 2 * (2.0 ** -22 + 3 * 2.0 ** -24) * 2 * x.abs().max().item()
    with pytest.raises(ValueError):
        RotaryPositionEmbeddingAxes((31, 32))
    with pytest.raises(ValueError):
        RotaryPositionEmbeddingAxes((16, 16), (1.0, 2.0, 3.0))


def test_rope_module_across_modes(tmp_path):
    """First called in inference mode, then trained with; saved, loaded onto the host and moved back."""
    from vasc_amd.aggregator import RotaryPositionEmbeddingAxes
    g = _gen(89)
    rope = RotaryPositionEmbeddingAxes((32, 32))
    x, pos = _randn(g, 1, 2, 9, 64).cuda(), torch.randint(0, 40, (1, 9, 2), generator=g).cuda()
    with torch.inference_mode():
        want = rope(x, pos).clone()
    leaf = x.clone().requires_grad_()
    y = rope(leaf, pos)
    y.sum().backward()
    assert torch.equal(y, want) and leaf.grad.isfinite().all()
    torch.save(rope, tmp_path / "rope")
    back = torch.load(tmp_path / "rope", map_location="cpu", weights_only=False).cuda()
    assert torch.equal(back(x, pos), want)


@pytest.mark.parametrize("axes", [2, 3])
@pytest.mark.parametrize("special", [0, 5])
def test_stream_attention_layer(axes, special):
    """Three pushes of a layer against float64 attention over the held keys and values, projection in float32."""
    from vasc_amd.aggregator import RotaryPositionEmbedding2D, RotaryPositionEmbeddingAxes
    from vasc_amd.streaming import _layer_qkv, stream_attention
    g = _gen(67)
    rope = RotaryPositionEmbedding2D(100.0) if axes == 2 else RotaryPositionEmbeddingAxes((16, 24, 24), (1e4, 100.0, 100.0))
    m = _module(rope=rope)
    B, frames, P = 2, 2, 100
    T = frames * P
    table, pages = _table(g, B, 10)
    cache = BlockCache(pages, 4, 64)
    held = None
    for step in range(3):
        x = _randn(g, B, T, 256).cuda()
        pos = torch.randint(0, 40, (B, T, axes), generator=g).int().cuda()
        start, lengths = _i32([step * T] * B), _i32([step * T + T] * B)
        with torch.no_grad():
            qp, qs, k, v = _layer_qkv(m, x, pos, frames, special)
        new = [O.quantise(_np(k[b]), _np(v[b])) for b in range(B)]
        held = new if held is None else [tuple(np.concatenate([o, n], 1) for o, n in zip(held[b], new[b])) for b in range(B)]
        keep = None if step == 0 else 1
        y = stream_attention(m, x, pos, cache, table, start, lengths, keep=keep, frames=frames, special=special)
        assert y.shape == x.shape and not y.requires_grad
        lists = None
        n = step * T + T
        if keep is not None:
            index, count = ops.cache_select(qp, cache, table, lengths, keep, block_q=128)
            lists = [[[index[b, h, u, :count[b, h, u]].tolist() for u in range(index.shape[2])] for h in range(4)] for b in range(B)]
            o = ops.cache_attn(qp, cache, table, lengths, index, count, block_q=128)
        else:
            o = ops.cache_attn(qp, cache, table, lengths)
        _check_attend(o, qp, held, [n] * B, lists, 128, False, H=4)
        o_s = None
        if special:
            o_s = ops.cache_attn(qs, cache, table, lengths)
            _check_attend(o_s, qs, held, [n] * B, None, 1, False, H=4)
        rows = ops.restore_tokens(o, o_s, frames, P, special)
        with torch.no_grad():
            assert torch.equal(y, m.proj(rows))


@pytest.mark.parametrize("axes", [2, 3])
def test_stream_attention_of_special_tokens_only(axes):
    """Frames whose tokens are all special attend to everything, with and without a choice of pages."""
    from vasc_amd.aggregator import RotaryPositionEmbedding2D, RotaryPositionEmbeddingAxes
    from vasc_amd.streaming import stream_attention
    g = _gen(109)
    m = _module(rope=RotaryPositionEmbedding2D(100.0) if axes == 2 else RotaryPositionEmbeddingAxes((16, 24, 24)))
    x, pos = _randn(g, 2, 3 * 30, 256).cuda(), torch.randint(0, 40, (2, 90, axes), generator=g).int().cuda()
    table, pages = _table(g, 2, 2)
    want = stream_attention(m, x, pos, BlockCache(pages, 4, 64), table, _i32([0, 0]), _i32([90, 90]), keep=None)
    for keep in (None, 1):
        got = stream_attention(m, x, pos, BlockCache(pages, 4, 64), table, _i32([0, 0]), _i32([90, 90]), keep=keep, frames=3,
                               special=30)
        # the same rows in units of another size: bf16 of the attention and of the projection, whose sums it moves by as much
        assert (got.float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()


@pytest.mark.parametrize("axes", [2, 3])
def test_stream_attention_captured(axes):
    """One captured layer serves every step: the lengths and the inputs are device tensors that move on."""
    from vasc_amd.aggregator import RotaryPositionEmbedding2D, RotaryPositionEmbeddingAxes
    from vasc_amd.streaming import stream_attention
    g = _gen(113)
    m = _module(rope=RotaryPositionEmbedding2D(100.0) if axes == 2 else RotaryPositionEmbeddingAxes((16, 24, 24)))
    B, T, steps = 2, 105, 5
    table, pages = _table(g, B, -(-steps * T // 64))
    xs = [_randn(g, B, T, 256).cuda() for _ in range(steps)]
    ps = [torch.randint(0, 40, (B, T, axes), generator=g).int().cuda() for _ in range(steps)]

    def layer(cache, x, pos, start, lengths):
        return stream_attention(m, x, pos, cache, table, start, lengths, keep=2, special=5)

    cache = BlockCache(pages, 4, 64)
    eager = [layer(cache, xs[i], ps[i], _i32([i * T] * B), _i32([i * T + T] * B)) for i in range(steps)]
    st = dict(cache=BlockCache(pages, 4, 64), x=xs[0].clone(), pos=ps[0].clone(), start=_i32([0] * B), lengths=_i32([T] * B))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(**st)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(**st)
    for i in range(steps):
        st["x"].copy_(xs[i])
        st["pos"].copy_(ps[i])
        st["start"].fill_(i * T)
        st["lengths"].copy_(st["start"] + T)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), i
        torch.randn(1 << 16, device="cuda").sum().item()  # other work between replays


def test_dense_layer_with_three_axes():
    """Attention.forward with RoPE over (time, row, column) against torch in float32 on the same bf16 q, k, v."""
    from vasc_amd.aggregator import RotaryPositionEmbeddingAxes
    g = _gen(71)
    m = _module(rope=RotaryPositionEmbeddingAxes((16, 24, 24), (1e4, 100.0, 100.0)))
    x = _randn(g, 2, 90, 256).cuda()
    pos = torch.randint(0, 60, (2, 90, 3), generator=g).cuda()
    with torch.no_grad():
        y = m(x, pos=pos)
        qkv = m.qkv(x).view(2, 90, 3, 4, 64)
        q, k = m.rope.rotate(m.q_norm(qkv[:, :, 0].transpose(1, 2)), m.k_norm(qkv[:, :, 1].transpose(1, 2)), pos)
        v = qkv[:, :, 2].transpose(1, 2).float()
        p = torch.softmax((q.float() @ k.float().transpose(2, 3).contiguous()) / 8, -1)
        o = p @ v
        # bf16 weights (2^-8 of each term) and output (2^-8) of the dense kernel, then the projection's 256 terms
        slack = 2.0 ** -8 * (p @ v.abs()) + 2.0 ** -8 * o.abs()
        w = m.proj.weight.float()
        ref = o.transpose(1, 2).reshape(2, 90, 256) @ w.T.contiguous() + m.proj.bias.float()
        bound = slack.transpose(1, 2).reshape(2, 90, 256) @ w.T.contiguous().abs()
        assert ((y.float() - ref).abs() <= bound + 2.0 ** -8 * (ref.abs() + bound) + 1e-4).all()


@pytest.mark.parametrize("params", [torch.float32, torch.float16])
def test_axes_rope_with_norms_of_another_type(params):
    """Norm parameters that are not bf16 go with either rope: normed and turned in float32, rounded to bf16 once, on both sides
    (half a step each, and float32's share as in _rotary_bound and a norm of 64 terms). Dense, sparse and streamed layers."""
    from vasc_amd.aggregator import Attention, RotaryPositionEmbedding2D, RotaryPositionEmbeddingAxes
    from vasc_amd.attention import adaptive_sparse_attention_forward
    from vasc_amd.streaming import _layer_qkv, stream_attention
    g = _gen(79)
    torch.manual_seed(3)
    m = Attention(256, 4).cuda()
    m.q_norm, m.k_norm = (torch.nn.LayerNorm(64, eps=1e-6).cuda().to(params) for _ in range(2))
    with torch.no_grad():
        for n in (m.q_norm, m.k_norm):
            n.weight.normal_(1.0, 0.2)
            n.bias.normal_(0.0, 0.2)
    B, P = 2, 6 * 7
    x = torch.randn(B, 2 * P, 256, generator=g).cuda()
    cell = torch.arange(P)
    pos = torch.stack([cell // 7 + 1, cell % 7 + 1], -1).repeat(B, 2, 1).cuda()
    got = {}
    for name, rope in (("table", RotaryPositionEmbedding2D(100.0)), ("axes", RotaryPositionEmbeddingAxes((32, 32), 100.0))):
        m.rope = rope
        with torch.no_grad():
            got[name] = _layer_qkv(m, x, pos, 2, 0)
    for a, b in zip(got["axes"], got["table"]):
        if a is not None:
            a, b = a.float(), b.float()
            side = 2.0 ** -18 * (a.abs() + a.roll(16, -1).abs() + a.roll(-16, -1).abs() + 1)
            assert ((a - b).abs() <= 2 * 2.0 ** -8 * torch.maximum(a.abs(), b.abs()) + side).all()
    q, _, k, v = (None if t is None else t.float() for t in got["axes"])
    p = torch.softmax((q @ k.transpose(2, 3).contiguous()) / 8, -1)
    o = p @ v
    slack = 2.0 ** -8 * (p @ v.abs()) + 2.0 ** -8 * o.abs()  # as for three axes
    with torch.no_grad():
        w = m.proj.weight
        flat = lambda t: t.transpose(1, 2).reshape(B, 2 * P, 256)  # noqa: E731
        ref, bound = flat(o) @ w.T.contiguous() + m.proj.bias, flat(slack) @ w.T.contiguous().abs() + 1e-4
        assert ((m(x, pos=pos) - ref).abs() <= bound).all()
        sparse = adaptive_sparse_attention_forward(m, x, pos, sparse_ratio=0.0, num_special_tokens=0, num_heads=4)
        sparse = sparse[0] if isinstance(sparse, tuple) else sparse
        assert ((sparse - ref).abs() <= bound).all()
        cache = BlockCache(4, 4, 64)
        y = stream_attention(m, x, pos, cache, _i32([[0, 1], [2, 3]]), _i32([0, 0]), _i32([2 * P] * 2), keep=None, frames=2)
    assert y.dtype == torch.float32 and y.isfinite().all()


@pytest.mark.parametrize("axes", [2, 3])
def test_aggregator_stream(axes):
    """Pushes run, repeat after reset bit for bit, do not see stale cache contents, and refuse what does not fit."""
    from vasc_amd.aggregator import Aggregator, RotaryPositionEmbeddingAxes
    from vasc_amd.streaming import AggregatorStream
    torch.manual_seed(4)
    model = Aggregator(dim=512, depth=2, num_heads=8, intermediate_layer_idx=(0, 1)).cuda().to(torch.bfloat16)
    if axes == 3:
        rope = RotaryPositionEmbeddingAxes((16, 24, 24), (1e4, 100.0, 100.0))
        for blk in (*model.frame_blocks, *model.global_blocks):
            blk.attn.rope = rope
    g = _gen(73)
    images = torch.rand(2, 5, 3, 112, 140, generator=g).cuda()
    stream = AggregatorStream(model, 5, sparse_ratio=0.5)

    def run():
        got = []
        for a, b in ((0, 1), (1, 3), (3, 5)):
            outs, s = stream.push(images[:, a:b])
            assert s == 5 and all(o.shape == (2, b - a, 85, 1024) and o.isfinite().all() for o in outs)
            got += outs
        return got

    first = run()
    with pytest.raises(ValueError, match="holds"):
        stream.push(images[:, :1])
    stream.reset()
    with pytest.raises(ValueError, match="another"):
        stream.push(images[:, :1])
        stream.push(images[:1, :1])
    stream.reset()
    for c in stream.caches:  # what is left in the pages is not seen again
        c.ks.fill_(255)
    for a, b in zip(run(), first):
        assert torch.equal(a, b)
    if axes == 2:
        # one frame, every page: the whole-clip aggregator, up to the 8-bit keys and values of its global layers. A value is off
        # by at most 2^-4 of itself, so an attention output (about unit size) by some percent; two layers scaled by 0.01.
        dense = AggregatorStream(model, 1, sparse_ratio=0.0)
        with torch.no_grad():
            want, _ = model(images[:, :1])
        got, _ = dense.push(images[:, :1])
        for a, b in zip(got, want):
            assert (a.float() - b.float()).abs().max() <= 0.02 * b.float().abs().max()


def _float64_norm(x, norm):
    x = x - x.mean(-1, keepdims=True)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + norm.eps) * _np(norm.weight) + _np(norm.bias)


def _layer_positions(B, first, n, grid, special, axes):
    """Positions of n frames from `first` on, written out: (frame,) row, column, special tokens at 0, 0."""
    rows = []
    for f in range(first, first + n):
        cells = [(0, 0)] * special + [(r + 1, c + 1) for r in range(grid[0]) for c in range(grid[1])]
        rows += [((f,) if axes == 3 else ()) + cell for cell in cells]
    return np.broadcast_to(np.array(rows), (B, len(rows), axes))


@pytest.mark.parametrize("sparse_ratio", [0.0, 0.6])
@pytest.mark.parametrize("axes", [2, 3])
def test_aggregator_stream_against_float64(axes, sparse_ratio, monkeypatch):
    """Every global block of every push, from the projection's rows up: norms, positions (time from the stream's start), the
    keys and values held, and attention over all that was seen or over the pages chosen, in float64 with code of its own.
    Frame blocks pass the tokens through (their scales are 0), so the first one shows the special tokens of first and later
    frames; a global block adds its attention to them (scales 1 and 0, an identity for the projection).

    Keys: a bf16 rounding (2^-8) and an e4m3 one (2^-4 of the value, or half the smallest step 2^-9 of the row's power,
    which is below top / 224), float32's share as in _rotary_bound and a norm of 64 terms. Output: a rounding of q in every logit,
    2^-8 of sum |q k| scale, in weights and their sum; the rounding of half weights and the rest, 2^-10; bf16 of the
    attention and of the sum with the tokens, 2^-8 each. With three axes the norms are torch's, which round to bf16 before the
    turn: a pair's two roundings, 2^-8 of each value, turn with it, so either value is off by at most 2^-8 (|lo| + |hi|) more
    (|cos| and |sin| up to 1); the layout kernel of two axes rounds once."""
    from vasc_amd.aggregator import Aggregator, RotaryPositionEmbeddingAxes
    from vasc_amd.streaming import AggregatorStream
    torch.manual_seed(8)
    C, H, D, grid, S = 512, 8, 64, (8, 10), 5
    P = S + grid[0] * grid[1]
    model = Aggregator(dim=C, depth=2, num_heads=H, intermediate_layer_idx=(0, 1)).cuda().to(torch.bfloat16)
    sections, bases = ((16, 24, 24), (1e4, 100.0, 100.0)) if axes == 3 else ((32, 32), (100.0, 100.0))
    with torch.no_grad():
        model.camera_token.normal_()
        model.register_token.normal_()
        for blk in model.frame_blocks:
            blk.ls1.gamma.zero_()
            blk.ls2.gamma.zero_()
        for blk in model.global_blocks:
            blk.ls1.gamma.fill_(1)
            blk.ls2.gamma.zero_()
            blk.attn.proj.weight.copy_(torch.eye(C))
            blk.attn.proj.bias.zero_()
            blk.norm1.weight.normal_(1.0, 0.2)
            blk.norm1.bias.normal_(0.0, 0.2)
            for n in (blk.attn.q_norm, blk.attn.k_norm):
                n.weight.normal_(1.5, 0.3)
                n.bias.normal_(0.0, 0.3)
    if axes == 3:
        rope = RotaryPositionEmbeddingAxes(sections, bases)
        for blk in (*model.frame_blocks, *model.global_blocks):
            blk.attn.rope = rope
    freq = _freq(sections, bases).numpy()

    def early(rows):
        """What a rounding before the turn adds to each value."""
        off, at = np.zeros_like(rows), 0
        for d in sections if axes == 3 else ():
            pair = np.abs(rows[..., at:at + d // 2]) + np.abs(rows[..., at + d // 2:at + d])
            off[..., at:at + d // 2] = off[..., at + d // 2:at + d] = 2.0 ** -8 * pair
            at += d
        return off

    seen_qkv, lists = [], []
    for blk in model.global_blocks:
        blk.attn.qkv.register_forward_hook(lambda m, args, out: seen_qkv.append((args[0], out)))
    choose = ops.cache_select
    monkeypatch.setattr(ops, "cache_select", lambda *a, **kw: lists.append(choose(*a, **kw)) or lists[-1])
    B, total = 2, 5
    images = torch.rand(B, total, 3, grid[0] * 14, grid[1] * 14, generator=_gen(97)).cuda()
    stream = AggregatorStream(model, total, sparse_ratio=sparse_ratio)
    missed_time = missed_attention = False
    for lo, hi in ((0, 1), (1, 3), (3, 5)):
        seen_qkv.clear()
        lists.clear()
        n, L = hi - lo, hi * P
        outs, _ = stream.push(images[:, lo:hi])
        first = _np(outs[0][..., :C])  # [B,n,P,C]
        for f in range(n):
            which = 0 if lo + f == 0 else 1
            assert np.array_equal(first[:, f, 0], np.broadcast_to(_np(model.camera_token[:, which, 0]), (B, C)))
            assert np.array_equal(first[:, f, 1:S], np.broadcast_to(_np(model.register_token[:, which]), (B, S - 1, C)))
        assert (first[:, :, S:].std((0, 1, 2)) > 0).all()
        assert torch.equal(outs[1][..., :C], outs[0][..., C:])
        pos = _layer_positions(B, lo, n, grid, S, axes)
        pages = -(-L // 64)
        keep = None if sparse_ratio == 0 else max(0, max(1, int(pages * (1 - sparse_ratio))) - 2)
        for i, blk in enumerate(model.global_blocks):
            x, y = (_np(outs[i][..., s]).reshape(B, n * P, C) for s in (slice(0, C), slice(C, 2 * C)))
            h, qkv = (_np(t).reshape(B, n * P, -1) for t in seen_qkv[i])
            want = _float64_norm(x, blk.norm1)
            assert (np.abs(h - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -16 * (1 + np.abs(want))).all()
            q, k, v = (qkv.reshape(B, n * P, 3, H, D)[:, :, j].transpose(0, 2, 1, 3) for j in range(3))
            q, k = _float64_norm(q, blk.attn.q_norm), _float64_norm(k, blk.attn.k_norm)
            side = 2.0 ** -17 * (1 + np.abs(k).max())
            k0, q_off, k_off = k, early(q), early(k)
            q, k = O.rotate(q, pos, sections, freq), O.rotate(k, pos, sections, freq)
            q_off += 2.0 ** -8 * np.abs(q)
            zero = _i32([0] * B)
            hk, hv = (_np(t) for t in ops.cache_read(stream.caches[i], stream.page_table, zero, L, dtype=torch.float32))
            # a push is held in the global layers' order, its patches and behind them its special tokens
            t = np.arange(n * P)
            held = np.concatenate([t[t % P >= S], t[t % P < S]])
            assert np.array_equal(hv[:, :, lo * P:], O.quantise(v, v)[1][:, :, held])

            def off(kk):
                kk = kk[:, :, held]
                top = np.abs(kk).max(-1, keepdims=True) * (1 + 2.0 ** -8)
                bound = (2.0 ** -4 * (1 + 2.0 ** -8) + 2.0 ** -8) * np.abs(kk) + top / 224 * 2.0 ** -10 + side + 1.07 * k_off[:, :, held]
                return (np.abs(hk[:, :, lo * P:] - kk) > bound).any()

            assert not off(k)
            if axes == 3:  # the check sees a time that is off by one
                later = pos + np.array([1, 0, 0])
                missed_time = missed_time or not off(O.rotate(k0, later, sections, freq))
            for b in range(B):
                for head in range(H):
                    logits = q[b, head] @ hk[b, head].T / 8
                    live = np.ones((n * P, L), bool)
                    if keep is not None:
                        index, count = (z.cpu().numpy() for z in lists[i])
                        patch = t % P >= S
                        unit = (t // P * (P - S) + t % P - S) // 128
                        for u in range(index.shape[2]):
                            got = index[b, head, u, :count[b, head, u]].tolist()
                            assert len(got) == min(pages, keep + 2) and got[0] == 0 and got[-1] == pages - 1
                            live[patch & (unit == u)] = np.isin(np.arange(L) // 64, got)
                    logits[~live] = -np.inf
                    p = np.exp(logits - logits.max(-1, keepdims=True))
                    p /= p.sum(-1, keepdims=True)
                    o, mag = p @ hv[b, head], p @ np.abs(hv[b, head])
                    off_logit = (q_off[b, head] @ np.abs(hk[b, head]).T).max(-1, keepdims=True) / 8 + side
                    off_o = (np.expm1(2 * off_logit) + 2.0 ** -10) * mag
                    off_o = off_o + 2.0 ** -8 * (np.abs(o) + off_o)
                    xs, ys = (t[b][:, head * D:(head + 1) * D] for t in (x, y))
                    bound = off_o + 2.0 ** -8 * (np.abs(xs + o) + off_o)
                    assert (np.abs(ys - (xs + o)) <= bound).all(), (lo, i, b, head)
                    missed_attention = missed_attention or not (np.abs(ys - xs) > bound).any()
    assert not missed_time and not missed_attention


def test_aggregator_stream_forked():
    """A deep copy goes its own way: neither sees the other's frames."""
    from vasc_amd.aggregator import Aggregator
    from vasc_amd.streaming import AggregatorStream
    torch.manual_seed(9)
    model = Aggregator(dim=512, depth=2, num_heads=8, intermediate_layer_idx=(0, 1)).cuda().to(torch.bfloat16)
    with torch.no_grad():
        for blk in model.global_blocks:
            blk.ls1.gamma.fill_(1)
    images = torch.rand(1, 4, 3, 112, 140, generator=_gen(101)).cuda()

    def straight(order):
        stream = AggregatorStream(model, 3)
        return [stream.push(images[:, i:i + 1])[0] for i in order]

    one, two = straight((0, 1, 2)), straight((0, 3, 2))
    stream = AggregatorStream(model, 3)
    stream.push(images[:, :1])
    fork = copy.deepcopy(stream)
    for order in (1, 2):
        a, b = stream.push(images[:, order:order + 1])[0], fork.push(images[:, [3, 2][order - 1]:][:, :1])[0]
        for x, y, wx, wy in zip(a, b, one[order], two[order]):
            assert torch.equal(x, wx) and torch.equal(y, wy)
    assert not torch.equal(one[2][1], two[2][1])


@pytest.mark.parametrize("axes", [2, 3])
@pytest.mark.parametrize("how", ["bf16", "float32", "autocast"])
def test_aggregator_stream_types_and_layouts(how, axes):
    """float32 models, with autocast or without, as the whole-clip aggregator takes them; a model without a camera token; frames
    of any memory order, whose results are those of contiguous ones."""
    import contextlib
    from vasc_amd.aggregator import Aggregator, RotaryPositionEmbeddingAxes
    from vasc_amd.streaming import AggregatorStream
    torch.manual_seed(11)
    model = Aggregator(dim=512, depth=2, num_heads=8, intermediate_layer_idx=(0, 1), camera_token=how != "float32").cuda()
    model = model.to(torch.bfloat16) if how == "bf16" else model
    if axes == 3:
        rope = RotaryPositionEmbeddingAxes((16, 24, 24), (1e4, 100.0, 100.0))
        for blk in (*model.frame_blocks, *model.global_blocks):
            blk.attn.rope = rope
    images = torch.rand(2, 3, 3, 70, 84, generator=_gen(127)).cuda()
    other = images.permute(1, 0, 3, 4, 2).contiguous().permute(1, 0, 4, 2, 3)
    cast = torch.autocast("cuda", torch.bfloat16) if how == "autocast" else contextlib.nullcontext()
    got = []
    with cast:
        for x in (images, other):
            stream = AggregatorStream(model, 3, sparse_ratio=0.5)
            got.append([o for a, b in ((0, 1), (1, 3)) for o in stream.push(x[:, a:b])[0]])
        if axes == 2:
            with torch.no_grad():
                want, _ = model(images[:, :1].contiguous())
            dense = AggregatorStream(model, 1, sparse_ratio=0.0).push(images[:, :1])[0]
            for a, b in zip(dense, want):
                assert a.dtype == b.dtype and (a.float() - b.float()).abs().max() <= 0.02 * b.float().abs().max()
    for a, b in zip(*got):
        assert a.isfinite().all() and torch.equal(a, b)


def test_sparse_layer_with_three_axes():
    """The sparse layer over (time, row, column) positions, nothing left out: float32 attention on the same q, k, v, special
    tokens among the keys, as test_dense_layer_with_three_axes bounds it."""
    from vasc_amd.aggregator import RotaryPositionEmbeddingAxes
    from vasc_amd.attention import adaptive_sparse_attention_forward
    g = _gen(131)
    m = _module(rope=RotaryPositionEmbeddingAxes((16, 24, 24), (1e4, 100.0, 100.0)))
    B, n, grid, S = 2, 3, (6, 7), 5
    P = S + grid[0] * grid[1]
    x = _randn(g, B, n * P, 256).cuda()
    pos = torch.from_numpy(_layer_positions(B, 40, n, grid, S, 3).copy()).cuda()
    with torch.no_grad():
        y = adaptive_sparse_attention_forward(m, x, pos, sparse_ratio=0.0, num_special_tokens=S, num_heads=4)
        y = y[0] if isinstance(y, tuple) else y
        qkv = m.qkv(x).view(B, n * P, 3, 4, 64)
        q, k = m.rope.rotate(m.q_norm(qkv[:, :, 0].transpose(1, 2)), m.k_norm(qkv[:, :, 1].transpose(1, 2)), pos)
        v = qkv[:, :, 2].transpose(1, 2).float()
        p = torch.softmax((q.float() @ k.float().transpose(2, 3).contiguous()) / 8, -1)
        o = p @ v
        slack = 2.0 ** -8 * (p @ v.abs()) + 2.0 ** -8 * o.abs()
        w = m.proj.weight.float()
        flat = lambda t: t.transpose(1, 2).reshape(B, n * P, 256)  # noqa: E731
        ref, bound = flat(o) @ w.T.contiguous() + m.proj.bias.float(), flat(slack) @ w.T.contiguous().abs()
    assert ((y.float() - ref).abs() <= bound + 2.0 ** -8 * (ref.abs() + bound) + 1e-4).all()
