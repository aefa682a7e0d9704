"""What the 4-bit cache and the page operators refuse, on the CPU: bad arguments at the C boundary (which returns before it
touches a pointer), host tensors, tables that cannot be changed in place; and oracle/streaming.py's 4-bit form and page tables
against definitions of their own."""
import math
import types

import numpy as np
import pytest
import torch

from oracle import streaming as O
from vasc_amd import _lib, ops
from vasc_amd.streaming import AggregatorStream, BlockCache, PagePool

FAKE = 1 << 20  # an aligned address that nothing reads


def _write(name="vasc_cache4_write", **kw):
    a = dict(k=FAKE, st=64, B=1, H=2, T=4, D=64, dtype=0, table=FAKE, ts=8, mp=8, start=FAKE, kc=FAKE, vo=FAKE, pages=9)
    a.update(kw)
    if name == "vasc_cache4_write":
        _lib.call(name, a["k"], 512, 256, a["st"], FAKE, 512, 256, 64, a["B"], a["H"], a["T"], a["D"], a["dtype"],
                  a["table"], a["ts"], a["mp"], a["start"], None, a["kc"], FAKE, FAKE, FAKE, a["vo"], FAKE, a["pages"], None)
    else:
        _lib.call(name, a["kc"], FAKE, FAKE, FAKE, a["vo"], a["pages"], a["table"], a["ts"], a["mp"], a["start"], None, a["B"],
                  a["H"], a["T"], a["D"], a["dtype"], a["k"], FAKE, None)


@pytest.mark.parametrize("name", ["vasc_cache4_write", "vasc_cache4_read"])
@pytest.mark.parametrize("kw,match", [
    (dict(k=None), "NULL"), (dict(table=None), "required"), (dict(start=None), "required"), (dict(kc=None), "required"),
    (dict(vo=None), "vo"), (dict(vo=FAKE + 8), "vo"), (dict(B=0), "empty"), (dict(T=0), "empty"), (dict(D=80), "not built"),
    (dict(D=32), "not built"), (dict(dtype=7), "dtype"), (dict(pages=0), "positive"), (dict(mp=0), "positive"),
    (dict(mp=1 << 24, ts=1 << 24), "too large"), (dict(ts=4), "table_stride"), (dict(k=FAKE + 8), "aligned"),
    (dict(kc=FAKE + 4), "aligned"), (dict(T=1 << 30), "too many"), (dict(B=1 << 24), "too many"),
])
def test_write_and_read_refuse(name, kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _write(name, **kw)


def _attn(**kw):
    a = dict(q=FAKE, o=FAKE, B=1, Hq=4, H=2, T=1, D=64, dtype=0, kc=FAKE, vo=FAKE, mp=5000, ts=5000, lengths=FAKE, block_q=1,
             index=None, width=0, count=None, ws=None, bytes=0, qst=256, ost=256, scale=0.125)
    a.update(kw)
    _lib.call("vasc_cache4_attn", a["q"], 512, 64, a["qst"], a["o"], 512, 64, a["ost"], a["B"], a["Hq"], a["H"], a["T"],
              a["D"], a["dtype"], a["kc"], FAKE, FAKE, FAKE, a["vo"], 9, FAKE, a["ts"], a["mp"], a["lengths"], None,
              a["block_q"], a["index"], a["width"], a["count"], 0, a["scale"], a["ws"], a["bytes"], None)


@pytest.mark.parametrize("kw,match", [
    (dict(q=None), "NULL"), (dict(kc=None), "NULL"), (dict(vo=None), "vo"), (dict(lengths=None), "NULL"),
    (dict(D=96), "not built"), (dict(dtype=2), "dtype"), (dict(index=FAKE), "together"), (dict(width=3), "together"),
    (dict(Hq=3), "sizes"), (dict(block_q=65), "sizes"), (dict(T=0), "sizes"), (dict(B=1 << 24), "sizes"),
    (dict(q=FAKE + 2), "aligned"), (dict(o=FAKE + 4), "aligned"), (dict(qst=260), "multiples"), (dict(ost=258), "multiples"),
    (dict(ts=7), "table_stride"), (dict(scale=math.inf), "scale"), (dict(scale=1e-35), "scale"), (dict(), "workspace"),
    (dict(ws=FAKE, bytes=64), "workspace"),
])
def test_attn_refuses(kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _attn(**kw)


def _copy(**kw):
    a = dict(bits=4, kc=FAKE, vo=FAKE, mean=FAKE, pages=9, H=2, D=64, src=FAKE, dst=FAKE, n=3)
    a.update(kw)
    _lib.call("vasc_cache_copy", a["bits"], a["kc"], FAKE, FAKE, FAKE, a["vo"], a["mean"], a["pages"], a["H"], a["D"], a["src"],
              a["dst"], a["n"], None)


@pytest.mark.parametrize("kw,match", [
    (dict(bits=6), "not built"), (dict(bits=8), "vo"), (dict(vo=None), "vo"), (dict(vo=FAKE + 4), "aligned"),
    (dict(kc=None), "required"), (dict(mean=None), "mean"), (dict(src=None), "required"), (dict(dst=None), "required"),
    (dict(pages=0), "positive"), (dict(D=32), "not built"), (dict(H=0), "no heads"), (dict(n=0), "no heads"),
    (dict(n=1 << 31), "too many"),
])
def test_copy_refuses(kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _copy(**kw)


def _compact(**kw):
    a = dict(bits=4, kc=FAKE, vo=FAKE, mean=FAKE, pages=9, H=2, D=64, table=FAKE, ts=8, mp=8, index=FAKE, isb=64, ish=0, B=1,
             n=64, out=FAKE, os=2, omp=2)
    a.update(kw)
    _lib.call("vasc_cache_compact", a["bits"], a["kc"], FAKE, FAKE, FAKE, a["vo"], a["mean"], a["pages"], a["H"], a["D"],
              a["table"], a["ts"], a["mp"], a["index"], a["isb"], a["ish"], None, a["B"], a["n"], a["out"], a["os"], a["omp"], None)


@pytest.mark.parametrize("kw,match", [
    (dict(bits=2), "not built"), (dict(bits=8), "vo"), (dict(vo=None), "vo"), (dict(kc=None), "required"),
    (dict(mean=None), "required"), (dict(table=None), "required"), (dict(index=None), "required"), (dict(out=None), "required"),
    (dict(ts=3), "table_stride"), (dict(os=1), "out_stride"), (dict(omp=0), "out_stride"), (dict(isb=-1), "negative"),
    (dict(B=0), "empty"), (dict(n=0), "empty"), (dict(n=1 << 30), "empty"), (dict(B=1 << 24), "too many"),
])
def test_compact_refuses(kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _compact(**kw)


def _pool(name, **kw):
    a = dict(refs=FAKE, pages=9, table=FAKE, ts=8, mp=8, lengths=FAKE, B=2, source=FAKE, rows=3, out=FAKE, tokens=5, ws=FAKE,
             bytes=1 << 20, src=FAKE)
    a.update(kw)
    head = (a["refs"], a["pages"], a["table"], a["ts"], a["mp"], a["lengths"], a["B"])
    if name == "fork":
        _lib.call("vasc_pages_fork", *head, a["source"], a["rows"], a["out"], FAKE, None)
    elif name == "free":
        _lib.call("vasc_pages_free", *head, None, None)
    else:
        _lib.call("vasc_pages_reserve", *head, a["tokens"], None, FAKE, a["src"], FAKE, a["ws"], a["bytes"], None)


@pytest.mark.parametrize("name", ["fork", "free", "reserve"])
@pytest.mark.parametrize("kw,match", [
    (dict(refs=None), "required"), (dict(table=None), "required"), (dict(lengths=None), "required"), (dict(pages=0), "pages"),
    (dict(pages=1 << 26), "pages"), (dict(mp=0), "max_pages"), (dict(ts=7), "stride"), (dict(mp=1 << 24, ts=1 << 24), "max_pages"),
    (dict(B=0), "B 0"), (dict(B=65537), "B 65537"),
])
def test_pool_refuses(name, kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _pool(name, **kw)


@pytest.mark.parametrize("name,kw,match", [
    ("fork", dict(source=None), "required"), ("fork", dict(out=None), "required"), ("fork", dict(rows=0), "rows"),
    ("fork", dict(rows=1 << 31), "rows"), ("reserve", dict(tokens=0), "tokens"), ("reserve", dict(tokens=1 << 30), "tokens"),
    ("reserve", dict(B=65536, mp=1 << 23, ts=1 << 23, tokens=1 << 29), "too many"), ("reserve", dict(src=None), "required"), ("reserve", dict(ws=None), "workspace"), ("reserve", dict(bytes=100), "workspace"),
    ("reserve", dict(ws=FAKE + 4), "aligned"),
])
def test_pool_calls_refuse(name, kw, match):
    with pytest.raises(_lib.VascError, match=match):
        _pool(name, **kw)


def test_workspace_sizes():
    size = _lib.fn("vasc_pages_reserve_workspace_size")
    assert size(9, 8, 2, 5) > 0
    # free bits, a count a chunk, needs, lists of the pages that the tokens can touch or the table can hold
    assert size(8193, 4, 300, 1 << 20) >= 8193 // 8 + 3 * 4 + 300 * 4 + 300 * 4 * 4
    for bad in ((0, 8, 2, 5), (1 << 26, 8, 2, 5), (9, 0, 2, 5), (9, 8, 0, 5), (9, 8, 2, 0), (9, 8, 65537, 5), (9, 8, 2, 1 << 30),
                (9, 1 << 23, 65536, 1 << 29)):
        assert size(*bad) == -1
    attn = _lib.fn("vasc_cache4_attn_workspace_size")
    assert attn(1, 4, 2, 1, 64, 1, 5000, 0) > 0 and attn(1, 4, 2, 1, 64, 1, 5000, 4) == 0
    for bad in ((0, 4, 2, 1, 64, 1, 10, 0), (1, 5, 2, 1, 64, 1, 10, 0), (1, 4, 2, 1, 60, 1, 10, 0), (1, 4, 2, 1, 64, 65, 10, 0)):
        assert attn(*bad) == -1


def test_host_tensors_and_constructors():
    for bad in (3, 16):
        with pytest.raises(ValueError, match="bits"):
            BlockCache(4, 2, 64, bits=bad)
    with pytest.raises(ValueError, match="GPU"):
        BlockCache(4, 2, 64, device="cpu", bits=4)
    for pages in (0, 1 << 26):
        with pytest.raises(ValueError, match="pages"):
            PagePool(pages)
    with pytest.raises(ValueError, match="GPU"):
        PagePool(4, device="cpu")
    for kw in (dict(bits=5), dict(branches=0)):
        with pytest.raises(ValueError, match="bits"):
            AggregatorStream(None, 4, **kw)
    stream = AggregatorStream(None, 4, branches=2)
    with pytest.raises(ValueError, match="nothing"):
        stream.fork()
    with pytest.raises(ValueError, match="held"):
        stream.keep([0])
    stream.close()
    with pytest.raises(ValueError, match="closed"):
        stream.reset()
    x = torch.zeros(2, 8, dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    cache = types.SimpleNamespace(device_index=0, pointers=(FAKE,) * 5, mean_pointer=FAKE, bits=4, pages=4, heads=2, head_dim=64)
    pool = types.SimpleNamespace(device_index=0, pointer=FAKE, pages=4)
    for call in (lambda: ops.cache_copy(cache, n, n), lambda: ops.cache_compact(cache, x, x, x),
                 lambda: ops.pages_fork(pool, x, n, n), lambda: ops.pages_free(pool, x, n),
                 lambda: ops.pages_reserve(pool, x, n, 3)):
        with pytest.raises(ValueError, match="GPU"):
            call()


# ------------------------------------------------------------------ the oracle
def test_e2m1_is_the_nearest_of_all_values():
    values = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    codes = np.concatenate([-values[:0:-1], values])
    g = np.random.default_rng(0)
    y = np.concatenate([g.uniform(-7, 7, 500), codes, (codes[1:] + codes[:-1]) / 2, [6.9, -7.0]])
    got = O.e2m1(y)
    assert np.isin(got, codes).all()
    assert (np.abs(got - y) == np.abs(y[:, None] - codes[None]).min(1)).all()
    # ties go to the even code: an even place among the magnitudes
    ties = np.abs((codes[1:] + codes[:-1]) / 2)
    assert (np.searchsorted(values, np.abs(O.e2m1(ties))) % 2 == 0).all()


@pytest.mark.parametrize("top", [6.0, 7.0, 7.001, 3.5, 3.5001, 0.0, 2.0 ** -60, 7 * 2.0 ** 60, 1e30, 2.0 ** -140])
def test_exponent4_is_the_smallest_that_holds(top):
    e = O.exponent4(np.array([0.0, -top]))
    assert O.E_MIN <= e <= O.E_MAX
    assert e == O.E_MAX or top <= 7 * 2.0 ** e
    assert e == O.E_MIN or top > 7 * 2.0 ** (e - 1)


def test_quantise4_groups():
    g = np.random.default_rng(1)
    x = g.normal(size=(40, 64)) * np.repeat(np.exp2(g.integers(-20, 20, (40, 2))), 32, 1)
    k, v = O.quantise4(x, x)
    top = np.abs(x).reshape(40, 2, 32).max(-1)
    row = np.abs(x).max(-1, keepdims=True)
    size = np.abs(x).reshape(40, 2, 32)
    assert (np.abs(k.reshape(40, 2, 32) - size * np.sign(x.reshape(40, 2, 32))) <=
            np.maximum(size / 5, top[..., None] / 14)).all()
    # value groups more than 14 powers below the row's largest have steps of that: a quarter of the row's power, 2^-14 less
    bound = np.maximum(np.maximum(size / 5, top[..., None] / 14), row[..., None] / 14 * 2.0 ** -O.LOWEST)
    assert (np.abs(v.reshape(40, 2, 32) - x.reshape(40, 2, 32)) <= bound).all()
    x[3, 5], x[7, 0] = np.inf, np.nan
    k, v = O.quantise4(x, np.ones_like(x))
    assert np.isnan(k).all(-1).nonzero()[0].tolist() == [3, 7] and np.isnan(v).all(-1).nonzero()[0].tolist() == [3, 7]


def test_pool_counts_its_holders():
    """After any turns the count of a page is the number of entries that name it, and no two rows share a page that a reserve
    has given."""
    g = np.random.default_rng(2)
    for _ in range(20):
        pages, mp = 30, 4
        pool = O.Pool([0] * pages)
        tables = [([[-1] * mp for _ in range(3)], [0, 0, 0])]
        for _ in range(8):
            rows, lengths = tables[-1]
            rows, granted, src, dst = pool.reserve(rows, lengths, g.integers(0, 90, len(rows)).tolist())
            lengths = [n + c for n, c in zip(lengths, granted)]
            assert all((s < 0) == (d < 0) for s, d in zip(src, dst))
            tables[-1] = rows, lengths
            if g.random() < 0.5:
                tables.append(pool.fork(rows, lengths, g.integers(-1, len(rows) + 1, 3).tolist()))
            elif len(tables) > 1:
                rows, lengths = tables.pop(0)
                pool.free(rows, lengths, [0] * len(rows))
            named = np.bincount([p for rows, _ in tables for row in rows for p in row if p >= 0], minlength=pages)
            assert named.tolist() == pool.refs


def test_oracle_reserve_of_any_table():
    """Counts and entries that do not agree: what is given was free, is given once and counted once; refused rows stay; counted
    pages lose a holder for each entry that is replaced; nothing is both copied from and given."""
    g = np.random.default_rng(3)
    for _ in range(200):
        pages, B, mp = 12, int(g.integers(1, 6)), 3
        before = g.choice([-1, 0, 0, 1, 1, 2, 3], pages).tolist()
        rows = g.integers(-2, pages + 1, (B, mp)).tolist()
        lengths, counts = g.integers(-1, mp * 64 + 2, B).tolist(), g.integers(-1, 150, B).tolist()
        pool = O.Pool(before)
        new, granted, src, dst = pool.reserve(rows, lengths, counts)
        lost = np.zeros(pages, int)
        for old, row, n, c in zip(rows, new, lengths, granted):
            assert c > 0 or row == old
            touched = range(max(n, 0) // 64, -(-(max(n, 0) + c) // 64) if c else 0)
            for j in range(mp):
                if j not in touched:
                    assert row[j] == old[j]
                elif not (0 <= old[j] < pages and before[old[j]] == 1):
                    assert before[row[j]] <= 0 and pool.refs[row[j]] == 1
                    if 0 <= old[j] < pages and before[old[j]] > 0:
                        lost[old[j]] += 1
                else:
                    assert row[j] == old[j]
        fresh = [row[j] for old, row, n, c in zip(rows, new, lengths, granted) if c
                 for j in range(max(n, 0) // 64, -(-(max(n, 0) + c) // 64)) if before[row[j]] <= 0]
        assert len(fresh) == len(set(fresh))
        assert sorted(fresh) == [p for p in range(pages) if before[p] <= 0][:len(fresh)]
        for p in range(pages):
            assert pool.refs[p] == (1 if p in fresh else before[p] - lost[p])
        copied = {p for p in src if p >= 0}
        assert not copied & {p for p in dst if p >= 0} and not copied & set(fresh)
