"""oracle/streaming.py against definitions of their own: torch's e4m3 conversion, a search over all 8-bit values, float64
softmax, brute-force choice."""
import math

import numpy as np
import pytest
import torch

from oracle import streaming as O


def test_e4m3_is_the_nearest_of_all_values():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    codes = np.unique(codes[np.isfinite(codes)])
    g = np.random.default_rng(0)
    y = np.concatenate([g.uniform(-448, 448, 400), np.exp2(g.uniform(-12, 8.8, 400)) * g.choice([-1, 1], 400), codes,
                        (codes[1:] + codes[:-1]) / 2])
    got = O.e4m3(y)
    assert np.isin(got, codes).all()
    best = np.abs(y[:, None] - codes[None]).min(1)
    assert (np.abs(got - y) == best).all()
    # ties as torch rounds them: to the even code
    want = torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn).double().numpy()
    exact = y.astype(np.float32).astype(np.float64) == y
    assert np.array_equal(got[exact], want[exact])


@pytest.mark.parametrize("top", [448.0, 448.5, 1.75, 1.7500001, 0.0, 2.0 ** -60, 448 * 2.0 ** 60, 1e30, 2.0 ** -140])
def test_exponent_is_the_smallest_that_holds(top):
    e = O.exponent(np.array([0.0, -top]))
    assert O.E_MIN <= e <= O.E_MAX
    assert e == O.E_MAX or top <= 448 * 2.0 ** e
    assert e == O.E_MIN or top > 448 * 2.0 ** (e - 1)


def test_quantise_error_and_nan_rows():
    g = np.random.default_rng(1)
    k, v = g.normal(size=(50, 64)) * np.exp2(g.integers(-20, 20, (50, 1))), g.normal(size=(50, 64))
    ko, vo = O.quantise(k, v)
    for x, o in ((k, ko), (v, vo)):
        top = np.abs(x).max(-1, keepdims=True)
        # half a step of a normal value, or half the subnormal step at the row's power (its largest is above 224 of it)
        assert (np.abs(o - x) <= np.maximum(2.0 ** -4 * np.abs(x), top / 224 * 2.0 ** -10)).all()
    v[3, 5], k[7, 0] = np.inf, np.nan
    ko, vo = O.quantise(k, v)
    bad = np.isnan(ko).all(-1)
    assert np.array_equal(bad, np.isnan(vo).all(-1)) and bad.nonzero()[0].tolist() == [3, 7]


def test_select_by_brute_force():
    g = np.random.default_rng(2)
    means = O.round_bf16(g.normal(size=(12, 8)).astype(np.float32)).astype(np.float64)
    means[4] = means[9]
    means[6, 0] = np.nan
    rows = g.normal(size=(3, 8)).astype(np.float32)
    for keep in range(0, 13):
        got, score = O.select(rows, means, 11, 10, keep, 2, 2)
        free = [j for j in range(11) if j not in (0, 1, 9, 10)]
        for j in free:
            ahead = sum(1 for i in free if score[i] > score[j] or (score[i] == score[j] and i < j))
            assert (j in got) == (ahead < keep)
        assert {0, 1, 9, 10} <= set(got) and got == sorted(got)


def test_attend_and_rotate():
    g = np.random.default_rng(3)
    q, k, v = g.normal(size=16), g.normal(size=(40, 16)), g.normal(size=(40, 16))
    seen = g.random(40) < 0.5
    o, mag, _ = O.attend(q, k, v, seen, 0.3)
    w = [math.exp(0.3 * float(q @ k[j])) if seen[j] else 0.0 for j in range(40)]
    want = sum(w[j] * v[j] for j in range(40)) / sum(w)
    assert np.allclose(o, want, rtol=1e-12, atol=1e-14) and (mag >= np.abs(o) - 1e-12).all()
    assert not O.attend(q, k, v, np.zeros(40, bool), 0.3)[0].any()
    x = g.normal(size=(1, 2, 5, 12))
    pos = g.integers(0, 9, (1, 5, 2))
    freq = np.array([1.0, 0.1, 0.5])
    y = O.rotate(x, pos, (4, 2), freq)
    for t in range(5):
        for a, (lo, hi), f in ((0, (0, 2), 1.0), (0, (1, 3), 0.1), (1, (4, 5), 0.5)):
            z = complex(*x[0, 1, t, [lo, hi]]) * np.exp(1j * pos[0, t, a] * f)
            assert np.allclose(y[0, 1, t, [lo, hi]], [z.real, z.imag])
    assert np.array_equal(y[..., 6:], x[..., 6:]) and np.allclose(O.rotate(y, pos, (4, 2), freq, -1.0), x)
    assert O.unit_pages(100, 3, 0, 2, True) == (2, 1) and O.unit_pages(100, 3, 0, 3, False) == (2, 1)
    assert O.unit_pages(0, 0, 0, 0, True) == (0, 0) and O.unit_pages(1, 3, 0, 1, True) == (0, 0)
