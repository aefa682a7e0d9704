"""Streamed global attention in float64: the definitions behind
``include/vasc_stream.h``, from the formulas, one row at a time.

``quantise`` and ``quantise4`` are exact (every step is a power of two times a small integer),
``select`` decides on scores that float64 holds to far less than a float32
step; ``attend`` and ``rotate`` are what the kernels are within rounding of.
"""
from __future__ import annotations

import math

import numpy as np

PAGE = 64
E_MIN, E_MAX = -60, 60


def round_bf16(x: np.ndarray) -> np.ndarray:
    """float32 -> the nearest bfloat16 (ties to even), as float32; NaN stays."""
    x = np.asarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def e4m3(y: np.ndarray) -> np.ndarray:
    """The nearest e4m3 value (ties to even) of |y| <= 448."""
    y = np.asarray(y, np.float64)
    _, e = np.frexp(y)  # |y| in [2^(e-1), 2^e)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.rint(y / step) * step


def exponent(row: np.ndarray) -> int:
    """Smallest e in [E_MIN, E_MAX] with max|row| <= 448 * 2^e (E_MAX where none is)."""
    top = float(np.abs(row).max(initial=0.0))
    for e in range(E_MIN, E_MAX):
        if top <= math.ldexp(448.0, e):
            return e
    return E_MAX


def quantise(k: np.ndarray, v: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """What the cache holds for rows k, v ``[..., D]`` of one token and head each."""
    k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)
    ko, vo = np.empty_like(k), np.empty_like(v)
    for at in np.ndindex(k.shape[:-1]):
        if not (np.isfinite(k[at]).all() and np.isfinite(v[at]).all()):
            ko[at] = vo[at] = np.nan
            continue
        for x, o in ((k, ko), (v, vo)):
            e = exponent(x[at])
            o[at] = e4m3(np.clip(np.ldexp(x[at], -e), -448.0, 448.0)) * math.ldexp(1.0, e)
    return ko, vo


GROUP, LOWEST = 32, 14  # features under one power; powers of two that a value row's groups may lie below its largest


def e2m1(y: np.ndarray) -> np.ndarray:
    """The nearest e2m1 value (ties to the even code); past 6: 6."""
    y = np.asarray(y, np.float64)
    _, e = np.frexp(y)
    step = np.ldexp(1.0, np.maximum(e - 1, 0) - 1)
    return np.clip(np.rint(y / step) * step, -6.0, 6.0)


def exponent4(group: np.ndarray) -> int:
    """Smallest e in [E_MIN, E_MAX] with max|group| <= 7 * 2^e (E_MAX where none is)."""
    top = float(np.abs(group).max(initial=0.0))
    for e in range(E_MIN, E_MAX):
        if top <= math.ldexp(7.0, e):
            return e
    return E_MAX


def quantise4(k: np.ndarray, v: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """What the 4-bit cache holds for rows k, v ``[..., D]`` of one token and head each."""
    k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)
    ko, vo = np.empty_like(k), np.empty_like(v)
    for at in np.ndindex(k.shape[:-1]):
        if not (np.isfinite(k[at]).all() and np.isfinite(v[at]).all()):
            ko[at] = vo[at] = np.nan
            continue
        for x, o, below in ((k, ko, None), (v, vo, LOWEST)):
            groups = x[at].reshape(-1, GROUP)
            es = [exponent4(g) for g in groups]
            if below is not None:
                es = [max(e, max(es) - below) for e in es]
            o[at] = np.concatenate([e2m1(np.ldexp(g, -e)) * math.ldexp(1.0, e) for g, e in zip(groups, es)])
    return ko, vo


class Pool:
    """Page tables that share pages, one entry at a time: lists of rows, -1 for no page."""

    def __init__(self, refs):
        self.refs = list(refs)

    def fork(self, table, lengths, source):
        out, tokens = [], []
        for s in source:
            inside = 0 <= s < len(table)
            mp = len(table[0])
            n = max(0, min(lengths[s], mp * PAGE)) if inside else 0
            row = [table[s][j] if inside and j * PAGE < n else -1 for j in range(mp)]
            row = [p if 0 <= p < len(self.refs) else -1 for p in row]
            for p in row:
                if p >= 0:
                    self.refs[p] += 1
            out.append(row)
            tokens.append(n)
        return out, tokens

    def free(self, table, lengths, keep):
        """(table, lengths) afterwards."""
        out, tokens = [], []
        for row, n, k in zip(table, lengths, keep):
            n = min(max(0, min(n, len(row) * PAGE)), max(0, k))
            for p in row[-(-n // PAGE):]:
                if 0 <= p < len(self.refs):
                    self.refs[p] -= 1
            out.append(row[:-(-n // PAGE)] + [-1] * (len(row) - -(-n // PAGE)))
            tokens.append(n)
        return out, tokens

    def reserve(self, table, lengths, counts):
        """(table, granted, src, dst): decided on the holders before the call."""
        before = list(self.refs)
        free = [p for p, r in enumerate(before) if r <= 0]
        table = [list(row) for row in table]
        granted, src, dst, wanted = [], [], [], 0

        def held(p):
            return 0 <= p < len(before) and before[p] > 0

        for row, n, c in zip(table, lengths, counts):
            mp = len(row)
            n = max(0, min(n, mp * PAGE))
            c = max(0, min(c, mp * PAGE - n))
            if c and n % PAGE and 0 <= row[n // PAGE] < len(before) and not held(row[n // PAGE]):
                c = 0  # the last page's tokens are in one that is free
            lacking = [j for j in range(n // PAGE, -(-(n + c) // PAGE) if c else 0)
                       if not (held(row[j]) and before[row[j]] == 1)]
            at, wanted = wanted, wanted + len(lacking)
            ok = not lacking or wanted <= len(free)
            granted.append(c if ok else 0)
            s = d = -1
            for i, j in enumerate(lacking if ok else ()):
                if held(row[j]):
                    self.refs[row[j]] -= 1
                    if j * PAGE < n:
                        s, d = row[j], free[at + i]
                row[j] = free[at + i]
                self.refs[row[j]] = 1
            src.append(s)
            dst.append(d)
        return table, granted, src, dst


def page_means(k: np.ndarray) -> np.ndarray:
    """bf16 mean of each page of the held keys ``[T, D]``, as float64 ``[ceil(T/64), D]``."""
    return np.stack([round_bf16((p.sum(0) / len(p)).astype(np.float32)).astype(np.float64)
                     for p in (k[i:i + PAGE] for i in range(0, len(k), PAGE))]) if len(k) else np.zeros((0, k.shape[1]))


def unit_pages(length: int, n_q: int, t0: int, t1: int, causal: bool) -> tuple[int, int]:
    """(pages seen, first of the rows' own pages) of query tokens [t0, t1)."""
    if t1 <= t0:
        return 0, 0
    if not causal:
        seen = -(-length // PAGE)
        return seen, seen - 1
    return max(0, -(-(length - n_q + t1) // PAGE)), max(0, length - n_q + t0) // PAGE


def select(rows: np.ndarray, means: np.ndarray, seen: int, own: int, keep: int, sink: int, recent: int):
    """(listed pages, float32 scores of the seen pages) of a unit with query rows ``[n, D]``."""
    qm = round_bf16((rows.astype(np.float64).sum(0) / len(rows)).astype(np.float32)).astype(np.float64)
    with np.errstate(invalid="ignore"):
        score = (means[:seen] @ qm).astype(np.float32)
    score = np.where(np.isnan(score), np.float32(-np.inf), score)
    forced = {j for j in range(seen) if j < sink or j >= own - (recent - 1)}
    free = sorted((j for j in range(seen) if j not in forced), key=lambda j: (-float(score[j]), j))
    return sorted(forced | set(free[:keep])), score


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, seen: np.ndarray, scale: float):
    """(o, sum p|v|, largest sum |q||k| scale) of one row over the keys where ``seen``."""
    if not seen.any():
        return np.zeros(v.shape[1]), np.zeros(v.shape[1]), 0.0
    k, v = k[seen], v[seen]
    x = (k @ q) * scale
    p = np.exp(x - x.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max()) * scale


def rotate(x: np.ndarray, pos: np.ndarray, sections, inv_freq: np.ndarray, sign: float = 1.0) -> np.ndarray:
    """x ``[B,H,T,D]``, pos ``[B,T,A]``."""
    x = np.asarray(x, np.float64)
    out = x.copy()
    at = f = 0
    for a, d in enumerate(sections):
        h = d // 2
        ang = pos[:, None, :, a, None].astype(np.float64) * inv_freq[f:f + h]
        c, s = np.cos(ang), sign * np.sin(ang)
        lo, hi = x[..., at:at + h], x[..., at + h:at + d]
        out[..., at:at + h], out[..., at + h:at + d] = lo * c - hi * s, hi * c + lo * s
        at, f = at + d, f + h
    return out
