"""Torch-facing wrappers of the C-ABI kernels (one per entry point).

Each wrapper validates shapes and dtypes, allocates outputs with torch's
caching allocator, and launches on ``torch.cuda.current_stream()``. Inputs
must be device tensors; nothing here falls back to the CPU.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib

BLOCK_Q = 128
BLOCK_K = 64
HEAD_DIM = 64
# the attention kernels' softmax runs in base 2: queries packed with
# q_scale = LOG2E * scale take scale = LN2 there
LOG2E, LN2 = 1.4426950408889634, 0.6931471805599453


def _stream() -> int:
    # torch.cuda.current_stream().cuda_stream without the two Python objects
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _dev(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError(f"{name} must be a GPU tensor (the HIP path has no CPU fallback)")


def _bhtd(t: torch.Tensor, name: str, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``dtype`` [B,H,T,D] with unit stride on D and 16-byte aligned rows."""
    _dev(t, name)
    if t.dim() != 4:
        raise ValueError(f"{name} must be [B,H,T,D], got {tuple(t.shape)}")
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.stride(-1) != 1 or any(s % 8 for s in t.stride()[:3]) or t.data_ptr() % 16:
        t = t.contiguous()
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


# ----------------------------------------------------------------- kernel 1
def pool_qk_max(q: torch.Tensor, k: torch.Tensor):
    """Block max pooling of Q (128 tokens) and K (64 tokens), bf16:
    ``predict_attention(pool_mode="max")``'s pooling."""
    q = _bhtd(q, "q")
    k = _bhtd(k, "k")
    B, H, nq, D = q.shape
    nk = k.shape[2]
    pq = torch.empty(B, H, math.ceil(nq / BLOCK_Q), D, device=q.device, dtype=torch.bfloat16)
    pk = torch.empty(B, H, math.ceil(nk / BLOCK_K), D, device=q.device, dtype=torch.bfloat16)
    _lib.call("vasc_pool_qk_max", q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], B, H, nq, nk, D,
              BLOCK_Q, BLOCK_K, pq.data_ptr(), pk.data_ptr(), _stream())
    return pq, pk


def pool_qkv(q=None, k=None, v=None, *, innovation: bool = True):
    """Block mean pooling (bf16-rounded) of Q (128) and K, V (64) + V pair innovation.

    Returns ``(pooled_q, pooled_k, pooled_v, innovation)`` with ``None`` for
    skipped inputs.
    """
    given = [t for t in (q, k, v) if t is not None]
    ref = given[0]
    # float16 tensors are rounded to bf16 as the kernel reads them
    half = all(isinstance(t, torch.Tensor) and t.dtype == torch.float16 for t in given)
    dtype = torch.float16 if half else torch.bfloat16
    q = None if q is None else _bhtd(q, "q", dtype)
    k = None if k is None else _bhtd(k, "k", dtype)
    v = None if v is None else _bhtd(v, "v", dtype)
    B, H, _, D = ref.shape
    nq = q.shape[2] if q is not None else 0
    nk = (k if k is not None else v).shape[2] if (k is not None or v is not None) else 0
    dev = ref.device
    pq = torch.empty(B, H, math.ceil(nq / BLOCK_Q), D, device=dev, dtype=torch.bfloat16) if q is not None else None
    pk = torch.empty(B, H, math.ceil(nk / BLOCK_K), D, device=dev, dtype=torch.bfloat16) if k is not None else None
    pv = torch.empty(B, H, math.ceil(nk / BLOCK_K), D, device=dev, dtype=torch.bfloat16) if v is not None else None
    inn = None
    if v is not None and innovation:
        inn = torch.empty(B, H, math.ceil(math.ceil(nk / BLOCK_K) / 2), device=dev, dtype=torch.float32)
    st = lambda t: (0, 0, 0) if t is None else tuple(t.stride()[:3])  # noqa: E731
    _lib.call("vasc_pool_qkv_f16" if half else "vasc_pool_qkv", _ptr(q), *st(q), _ptr(k), *st(k), _ptr(v), *st(v),
              B, H, nq, nk, D, BLOCK_Q, BLOCK_K, _ptr(pq), _ptr(pk), _ptr(pv), _ptr(inn), _stream())
    return pq, pk, pv, inn


def pooled_softmax(pooled_q: torch.Tensor, pooled_k: torch.Tensor, *, scale: float | None = None,
                   round_bf16: bool = True, priority: bool = False):
    """fp32 ``softmax(bf16(bf16(pq.pk) * scale))`` over key blocks, ``[B,H,Qb,Kb]``.

    ``priority=True`` returns ``(prob, priority)`` with ``priority`` the
    VASC ledger's QK-order priority ``max(prob, 0)``, NaN -> 0, written by
    the same launch.
    """
    _dev(pooled_q, "pooled_q")
    _dev(pooled_k, "pooled_k")
    pq = pooled_q.to(torch.bfloat16).contiguous()
    pk = pooled_k.to(torch.bfloat16).contiguous()
    B, H, qb, D = pq.shape
    kb = pk.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    prob = torch.empty(B, H, qb, kb, device=pq.device, dtype=torch.float32)
    prio = torch.empty_like(prob) if priority else None
    size = _lib.load().vasc_pooled_softmax_workspace_size(B, H, qb, kb)
    ws = torch.empty(size, device=pq.device, dtype=torch.uint8) if size else None
    _lib.call("vasc_pooled_softmax", pq.data_ptr(), pk.data_ptr(), B, H, qb, kb, D, float(scale),
              int(bool(round_bf16)), prob.data_ptr(), _ptr(prio), _ptr(ws), _stream())
    return (prob, prio) if priority else prob


def pair_innovation(pooled_value: torch.Tensor) -> torch.Tensor:
    """Pair innovation of float32 pooled values ``[B,H,Kb,D]`` -> ``[B,H,ceil(Kb/2)]``."""
    _dev(pooled_value, "pooled_value")
    pv = pooled_value.float().contiguous()
    B, H, kb, D = pv.shape
    out = torch.empty(B, H, (kb + 1) // 2, device=pv.device, dtype=torch.float32)
    _lib.call("vasc_pair_innovation", pv.data_ptr(), B, H, kb, D, out.data_ptr(), _stream())
    return out


# ----------------------------------------------------------------- kernel 2
def select_workspace(B: int, H: int, Q: int, K: int, device) -> torch.Tensor:
    n = _lib.fn("vasc_select_workspace_size")(B, H, Q, K)
    return torch.empty(max(int(n), 256), device=device, dtype=torch.uint8)


def select_workspace_region(workspace: torch.Tensor, B: int, H: int, Q: int, K: int, region: int) -> torch.Tensor:
    """A result region of the VASC selection workspace after a VASC call
    (``vasc_select_workspace_offset``): per-row totals, pair sums (float32
    ``[B,H,Q]``), capacities (int32 ``[B,H,Q]``) or the admitted debt
    (float32 ``[B,H,P]``)."""
    off = int(_lib.fn("vasc_select_workspace_offset")(B, H, Q, K, int(region)))
    if off < 0:
        raise ValueError(f"unknown workspace region {region}")
    P = (K + 1) // 2
    n, dtype = {_lib.WS_ROW_TOTAL: (B * H * Q, torch.float32), _lib.WS_ROW_PAIR_SUM: (B * H * Q, torch.float32),
                _lib.WS_ROW_CAPACITY: (B * H * Q, torch.int32), _lib.WS_ADMITTED_DEBT: (B * H * P, torch.float32)}[region]
    shape = (B, H, P) if region == _lib.WS_ADMITTED_DEBT else (B, H, Q)
    return workspace[off:off + 4 * n].view(dtype).view(shape)


def select_blocks(score: torch.Tensor, *, mode: int, topk: int, innovation=None, row_cap=None,
                  protected_mask=None, force_last: bool = False, max_capacity: int = 0,
                  sink_blocks: int = 0, debt=None, pending_arrival=None, prev_service=None,
                  want_priority: bool = False, want_mask: bool = False, width: int | None = None,
                  workspace: torch.Tensor | None = None):
    """Block selection (kernel 2). Returns a dict of device tensors.

    Keys: ``index`` [B,H,Q,width] int32 ascending, ``count`` [B,H,Q] int32,
    and in VASC mode ``debt``, ``arrival``, ``service`` [B,H,P] float32,
    ``gate`` int32 [1]; optional ``priority`` / ``mask``.
    """
    _dev(score, "score")
    s = score.float().contiguous()
    B, H, Q, K = s.shape
    P = (K + 1) // 2
    vasc = mode == _lib.MODE_VASC
    dev = s.device
    if vasc:
        maxc = mc_arg = min(int(max_capacity), K)
    elif row_cap is not None:  # per-row counts, each at most max_capacity (0 = K), plus the forced tail
        mc_arg = int(max_capacity)
        maxc = min((mc_arg if mc_arg > 0 else K) + int(bool(force_last)), K)
    else:
        maxc = mc_arg = min(max(int(topk), 1) + int(bool(force_last)), K)
    width = maxc + sink_blocks if width is None else int(width)
    out = {
        "index": torch.empty(B, H, Q, max(width, 1), device=dev, dtype=torch.int32),
        "count": torch.empty(B, H, Q, device=dev, dtype=torch.int32),
    }
    f32 = lambda t: None if t is None else t.float().contiguous()  # noqa: E731
    inn = f32(innovation)
    if vasc:
        if inn is None or tuple(inn.shape) != (B, H, P):
            raise ValueError(f"innovation must be [B,H,{P}] for K={K}")
        out["debt"] = torch.empty(B, H, P, device=dev, dtype=torch.float32)
        out["arrival"] = torch.empty(B, H, P, device=dev, dtype=torch.float32)
        out["service"] = torch.empty(B, H, P, device=dev, dtype=torch.float32)
        out["gate"] = torch.empty(1, device=dev, dtype=torch.int32)
        if workspace is None:
            workspace = select_workspace(B, H, Q, K, dev)
        out["workspace"] = workspace
    if want_priority:
        out["priority"] = torch.empty(B, H, Q, K, device=dev, dtype=torch.float32)
    if want_mask:
        out["mask"] = torch.empty(B, H, Q, K, device=dev, dtype=torch.uint8)
    rc = None if row_cap is None else row_cap.to(torch.int32).contiguous()
    pm = None if protected_mask is None else protected_mask.to(torch.uint8).contiguous()
    state = [f32(debt), f32(pending_arrival), f32(prev_service)]
    for t, name in zip(state, ("debt", "pending_arrival", "prev_service")):
        if t is not None and t.numel() != B * H * P:
            raise ValueError(f"{name} must hold B*H*P={B * H * P} values")
    ws_bytes = workspace.numel() if workspace is not None else 0
    _lib.call("vasc_select_blocks", s.data_ptr(), _ptr(inn), B, H, Q, K, int(mode), int(topk), _ptr(rc),
              _ptr(pm), int(bool(force_last)), int(mc_arg), int(sink_blocks), _ptr(state[0]),
              _ptr(state[1]), _ptr(state[2]), _ptr(out.get("debt")), _ptr(out.get("arrival")),
              _ptr(out.get("service")), _ptr(out.get("gate")), _ptr(out.get("priority")),
              _ptr(out.get("mask")), out["index"].data_ptr(), width, out["count"].data_ptr(),
              _ptr(workspace), ws_bytes, _stream())
    return out


def cdf_counts(score: torch.Tensor, cdf_threshold, *, min_count: int = 0, force_last: bool = False,
               eps: float = 1e-5, want_base: bool = False):
    """Per-row counts of ``get_block_mask``'s cdf-threshold branch (kernel 2).

    ``cdf_threshold``: a number or ``H`` per-head values
    (``hyperparameter_check``); the kernel compares against
    ``f32(f32(thr) + f32(eps))``. Returns ``(count, base)`` int32 ``[B,H,Q]``
    (``base`` adds the forced mixed tail, ``None`` unless ``want_base``).
    """
    _dev(score, "score")
    s = score.float().contiguous()
    B, H, Q, K = s.shape
    thr = cdf_threshold.detach().float().cpu().numpy() if isinstance(cdf_threshold, torch.Tensor) else cdf_threshold
    thr = np.asarray(thr, dtype=np.float32)
    if thr.ndim == 0:
        thr = np.full(H, thr, dtype=np.float32)
    if thr.ndim != 1 or thr.size != H:
        raise ValueError(f"cdf_threshold must be a number or hold {H} values")
    T = torch.from_numpy((thr + np.float32(eps)).astype(np.float32)).to(s.device)
    count = torch.empty(B, H, Q, device=s.device, dtype=torch.int32)
    base = torch.empty_like(count) if want_base else None
    _lib.call("vasc_cdf_counts", s.data_ptr(), B, H, Q, K, T.data_ptr(), int(min_count), int(bool(force_last)),
              count.data_ptr(), _ptr(base), _stream())
    return count, base


def priority_order(priority: torch.Tensor, M: int, index: torch.Tensor | None = None,
                   count: torch.Tensor | None = None, sink: int = 0) -> torch.Tensor:
    """The selector's selected indices (kernel 2): per row the ``M`` blocks
    of largest priority, largest first, equal priorities in ascending block
    index, as ``priority.topk(M, dim=-1, sorted=True).indices``
    (SW:3887-3894). ``priority`` float32 ``[..., K]``; returns int64
    ``[..., M]``. ``index`` / ``count`` / ``sink``: the ``select_blocks``
    lists of the same selection; rows that kept exactly ``M`` patch blocks
    take them from there."""
    _dev(priority, "priority")
    p = priority.float().contiguous()
    K = p.shape[-1]
    if not 0 <= int(M) <= K:
        raise ValueError(f"M={M} outside [0, {K}]")
    out = torch.empty(p.shape[:-1] + (int(M),), device=p.device, dtype=torch.int64)
    rows = p.numel() // K if K else 0
    width = 0
    if index is not None:
        if count is None or index.dtype != torch.int32 or count.dtype != torch.int32:
            raise ValueError("index and count must be the int32 lists of select_blocks")
        if index.shape[:-1] != p.shape[:-1] or count.shape != p.shape[:-1]:
            raise ValueError("index and count must match the priority rows")
        index, count = index.contiguous(), count.contiguous()
        width = index.shape[-1]
    if rows and M:
        _lib.call("vasc_priority_order", p.data_ptr(), _ptr(index), _ptr(count), width, int(sink), rows, K, int(M),
                  out.data_ptr(), _stream())
    return out


def settle_terminal(debt, pending_arrival, service) -> torch.Tensor:
    pend = pending_arrival.float().contiguous()
    svc = service.float().contiguous()
    d = None if debt is None else debt.float().contiguous()
    out = torch.empty_like(pend)
    _lib.call("vasc_settle_terminal", _ptr(d), pend.data_ptr(), svc.data_ptr(), pend.numel(),
              out.data_ptr(), _stream())
    return out


# ----------------------------------------------------------------- kernel 3
def pack_v(v: torch.Tensor) -> torch.Tensor:
    """Packed, transposed, key-permuted V tiles ``[B,H,ceil(T/64),64,64]`` (bf16)."""
    if isinstance(v, torch.Tensor) and v.dtype == torch.float16:
        return pack_kv_half(None, v)[1]
    v = _bhtd(v, "v")
    B, H, T, D = v.shape
    nkb = math.ceil(T / BLOCK_K)
    vt = torch.empty(B, H, nkb, D, BLOCK_K, device=v.device, dtype=torch.bfloat16)
    _lib.call("vasc_pack_v", v.data_ptr(), *v.stride()[:3], B, H, T, D, vt.data_ptr(), _stream())
    return vt


def pack_kv_half(k: torch.Tensor | None, v: torch.Tensor):
    """``(k in bf16 or None, pack_v(v))`` of float16 K and V in one pass."""
    v = _bhtd(v, "v", torch.float16)
    B, H, T, D = v.shape
    vt = torch.empty(B, H, math.ceil(T / BLOCK_K), D, BLOCK_K, device=v.device, dtype=torch.bfloat16)
    ko, ks = None, (None, 0, 0, 8)
    if k is not None:
        k = _bhtd(k, "k", torch.float16)
        if k.shape != v.shape:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        ko = torch.empty(B, H, T, D, device=v.device, dtype=torch.bfloat16)
        ks = (k.data_ptr(), *k.stride()[:3])
    _lib.call("vasc_pack_kv_f16", *ks, v.data_ptr(), *v.stride()[:3], B, H, T, D, _ptr(ko), vt.data_ptr(), _stream())
    return ko, vt


# ----------------------------------------------------------------- kernel 4
def block_sparse_attn(q: torch.Tensor, k: torch.Tensor, vt: torch.Tensor, index: torch.Tensor,
                      count: torch.Tensor, *, scale: float | None = None, delta: bool = False,
                      out: torch.Tensor | None = None, half_out: bool = False) -> torch.Tensor:
    """Block-sparse attention over listed 64-key blocks; bf16 output ``[B,H,Nq,D]``.
    ``half_out``: the bf16 result as float16, for float16 q (which the kernel
    then reads as it is)."""
    half = half_out and q.dtype == torch.float16 and out is None
    q = _bhtd(q, "q", torch.float16 if half else torch.bfloat16)
    k = _bhtd(k, "k")
    _dev(vt, "vt")
    B, H, nq, D = q.shape
    nk = k.shape[2]
    if vt.shape != (B, H, math.ceil(nk / BLOCK_K), D, BLOCK_K):
        raise ValueError(f"vt shape {tuple(vt.shape)} does not match K {tuple(k.shape)}")
    qb = math.ceil(nq / BLOCK_Q)
    index = index.to(torch.int32).contiguous()
    count = count.to(torch.int32).contiguous()
    if index.shape[:3] != (B, H, qb) or count.shape != (B, H, qb):
        raise ValueError(f"index/count must be [B,H,{qb},W]/[B,H,{qb}]")
    o = out if out is not None else torch.empty(B, H, nq, D, device=q.device, dtype=q.dtype)
    scale = D ** -0.5 if scale is None else scale
    _lib.call("vasc_block_sparse_attn_f16_fwd" if half else "vasc_block_sparse_attn_fwd", q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3],
              vt.data_ptr(), o.data_ptr(), *o.stride()[:3], B, H, nq, nk, D, index.data_ptr(),
              index.shape[-1], count.data_ptr(), int(bool(delta)), float(scale), _stream())
    if half_out and not half:
        o = o.to(torch.float16)
    return o


def block_sparse_attn_pv(q: torch.Tensor, k: torch.Tensor, vt: torch.Tensor, index: torch.Tensor,
                         count: torch.Tensor, pv_threshold, *, scale: float | None = None, delta: bool = False):
    """``block_sparse_attn`` with the PV post-cut; ``pv_threshold`` is a
    number or ``H`` values in log2 units. Returns ``(o, pv_map)`` with the
    int32 execution map ``[B, H, ceil(Nq/128)*4, ceil(Nk/64)]``."""
    q = _bhtd(q, "q")
    k = _bhtd(k, "k")
    _dev(vt, "vt")
    B, H, nq, D = q.shape
    nk = k.shape[2]
    if vt.shape != (B, H, math.ceil(nk / BLOCK_K), D, BLOCK_K):
        raise ValueError(f"vt shape {tuple(vt.shape)} does not match K {tuple(k.shape)}")
    qb, kb = math.ceil(nq / BLOCK_Q), math.ceil(nk / BLOCK_K)
    index = index.to(torch.int32).contiguous()
    count = count.to(torch.int32).contiguous()
    if index.shape[:3] != (B, H, qb) or count.shape != (B, H, qb):
        raise ValueError(f"index/count must be [B,H,{qb},W]/[B,H,{qb}]")
    thr = torch.as_tensor(pv_threshold, dtype=torch.float32).reshape(-1)
    thr = (thr.expand(H) if thr.numel() == 1 else thr).contiguous().to(q.device)
    if thr.numel() != H:
        raise ValueError(f"pv_threshold must be a number or hold {H} values")
    o = torch.empty(B, H, nq, D, device=q.device, dtype=torch.bfloat16)
    pv_map = torch.zeros(B, H, qb * 4, kb, device=q.device, dtype=torch.int32)
    scale = D ** -0.5 if scale is None else scale
    _lib.call("vasc_block_sparse_attn_pv_fwd", q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3],
              vt.data_ptr(), o.data_ptr(), *o.stride()[:3], B, H, nq, nk, D, index.data_ptr(),
              index.shape[-1], count.data_ptr(), int(bool(delta)), float(scale), thr.data_ptr(),
              pv_map.data_ptr(), _stream())
    return o, pv_map


def dense_attn(q: torch.Tensor, k: torch.Tensor, vt: torch.Tensor, *, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Dense attention with the same MFMA kernel (every key block)."""
    q = _bhtd(q, "q")
    k = _bhtd(k, "k")
    _dev(vt, "vt")
    B, H, nq, D = q.shape
    nk = k.shape[2]
    if vt.shape != (B, H, math.ceil(nk / BLOCK_K), D, BLOCK_K):
        raise ValueError(f"vt shape {tuple(vt.shape)} does not match K {tuple(k.shape)}")
    if out is not None:
        _dev(out, "out")
        if out.shape != (B, H, nq, D) or out.dtype != torch.bfloat16 or out.stride(3) != 1:
            raise ValueError(f"out must be bf16 {(B, H, nq, D)} with unit stride over D, "
                             f"got {out.dtype} {tuple(out.shape)} strides {out.stride()}")
    o = out if out is not None else torch.empty(B, H, nq, D, device=q.device, dtype=torch.bfloat16)
    scale = D ** -0.5 if scale is None else scale
    _lib.call("vasc_dense_attn_fwd", q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3],
              vt.data_ptr(), o.data_ptr(), *o.stride()[:3], B, H, nq, nk, D, float(scale), _stream())
    return o


def _global_ws(B: int, H: int, n_patch: int, n_special: int, nk: int, width: int, device) -> tuple:
    """The special queries' split workspace: (tensor or None, pointer, bytes).
    Fewer than 64 key blocks are never split: not asked for, the call is host time."""
    if not n_special or nk <= 63 * BLOCK_K:
        return None, None, 0
    size = _lib.fn("vasc_global_attn_workspace_size")(B, H, n_patch, n_special, nk, width)
    ws = torch.empty(size, device=device, dtype=torch.uint8) if size else None
    return ws, _ptr(ws), size


def global_attn(q_patch: torch.Tensor, q_special: torch.Tensor | None, k: torch.Tensor, vt: torch.Tensor,
                index: torch.Tensor, count: torch.Tensor, *, scale: float | None = None):
    """Patch queries over their listed blocks and special queries over every
    key, in one launch. Returns ``(o_patch, o_special or None)`` (bf16)."""
    q_patch = _bhtd(q_patch, "q_patch")
    k = _bhtd(k, "k")
    _dev(vt, "vt")
    B, H, n_patch, D = q_patch.shape
    nk = k.shape[2]
    if vt.shape != (B, H, math.ceil(nk / BLOCK_K), D, BLOCK_K):
        raise ValueError(f"vt shape {tuple(vt.shape)} does not match K {tuple(k.shape)}")
    qb = math.ceil(n_patch / BLOCK_Q)
    index = index.to(torch.int32).contiguous()
    count = count.to(torch.int32).contiguous()
    if index.shape[:3] != (B, H, qb) or count.shape != (B, H, qb):
        raise ValueError(f"index/count must be [B,H,{qb},W]/[B,H,{qb}]")
    o_patch = torch.empty(B, H, n_patch, D, device=q_patch.device, dtype=torch.bfloat16)
    n_special = 0
    o_special = None
    qs_args = (None, 0, 0, 8)
    os_args = (None, 0, 0, 8)
    if q_special is not None and q_special.shape[2] > 0:
        q_special = _bhtd(q_special, "q_special")
        n_special = q_special.shape[2]
        o_special = torch.empty(B, H, n_special, D, device=q_patch.device, dtype=torch.bfloat16)
        qs_args = (q_special.data_ptr(), *q_special.stride()[:3])
        os_args = (o_special.data_ptr(), *o_special.stride()[:3])
    scale = D ** -0.5 if scale is None else scale
    ws, ws_ptr, ws_bytes = _global_ws(B, H, n_patch, n_special, nk, index.shape[-1], q_patch.device)
    _lib.call("vasc_global_attn_ws_fwd", q_patch.data_ptr(), *q_patch.stride()[:3], *qs_args, k.data_ptr(),
              *k.stride()[:3], vt.data_ptr(), o_patch.data_ptr(), *o_patch.stride()[:3], *os_args, B, H, n_patch,
              n_special, nk, D, index.data_ptr(), index.shape[-1], count.data_ptr(), float(scale), ws_ptr, ws_bytes,
              _stream())
    return o_patch, o_special


def global_attn_tokens(q_patch: torch.Tensor, q_special: torch.Tensor | None, k: torch.Tensor, vt: torch.Tensor,
                       index: torch.Tensor, count: torch.Tensor, frames: int, tokens_per_frame: int, special: int,
                       *, scale: float | None = None) -> torch.Tensor:
    """``global_attn`` followed by ``restore_tokens`` in one launch: the
    results land on their frame-major token rows of ``[B, N*P, H*D]`` bf16."""
    q_patch = _bhtd(q_patch, "q_patch")
    k = _bhtd(k, "k")
    _dev(vt, "vt")
    B, H, n_patch, D = q_patch.shape
    N, P, S = int(frames), int(tokens_per_frame), int(special)
    nk = k.shape[2]
    if n_patch != N * (P - S) or nk != N * P:
        raise ValueError(f"q_patch/k hold {n_patch}/{nk} tokens, expected {N * (P - S)}/{N * P}")
    if k.shape[:2] != (B, H) or k.shape[3] != D:
        raise ValueError(f"k {tuple(k.shape)} does not match q_patch {tuple(q_patch.shape)}")
    if vt.shape != (B, H, math.ceil(nk / BLOCK_K), D, BLOCK_K):
        raise ValueError(f"vt shape {tuple(vt.shape)} does not match K {tuple(k.shape)}")
    qb = math.ceil(n_patch / BLOCK_Q)
    index = index.to(torch.int32).contiguous()
    count = count.to(torch.int32).contiguous()
    if index.shape[:3] != (B, H, qb) or count.shape != (B, H, qb):
        raise ValueError(f"index/count must be [B,H,{qb},W]/[B,H,{qb}]")
    qs_args = (None, 0, 0, 8)
    if S > 0:
        if q_special is None or tuple(q_special.shape) != (B, H, N * S, D):
            raise ValueError(f"q_special must be [B, H, {N * S}, {D}]")
        q_special = _bhtd(q_special, "q_special")
        qs_args = (q_special.data_ptr(), *q_special.stride()[:3])
    out = torch.empty(B, N * P, H * D, device=q_patch.device, dtype=torch.bfloat16)
    scale = D ** -0.5 if scale is None else scale
    ws, ws_ptr, ws_bytes = _global_ws(B, H, n_patch, N * S, nk, index.shape[-1], q_patch.device)
    _lib.call("vasc_global_attn_tokens_ws_fwd", q_patch.data_ptr(), *q_patch.stride()[:3], *qs_args, k.data_ptr(),
              *k.stride()[:3], vt.data_ptr(), out.data_ptr(), B, H, N, P, S, nk, D, index.data_ptr(),
              index.shape[-1], count.data_ptr(), float(scale), ws_ptr, ws_bytes, _stream())
    return out


# ----------------------------------------------------------------- kernel 5
def _btht(t: torch.Tensor, name: str) -> tuple:
    """(pointer, sb, st, sh) of a bf16 ``[B,T,H,D]`` view with unit stride on D."""
    _dev(t, name)
    if t.dtype != torch.bfloat16 or t.stride(-1) != 1 or any(s % 8 for s in t.stride()[:3]) or t.data_ptr() % 16:
        raise ValueError(f"{name} must be bf16 [B,T,H,D] with unit stride on D, 16-byte aligned rows")
    return t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)


def _param(t: torch.Tensor, name: str, numel: int, dtypes: tuple) -> torch.Tensor:
    """A [numel] parameter as a contiguous device tensor of one of ``dtypes``
    (converted to the first when it is none of them). Nothing is cached: the
    kernel reads the parameter's current values on every call."""
    t = t.detach()
    _dev(t, name)
    if t.numel() != numel:
        raise ValueError(f"{name} must hold {numel} values")
    if t.dtype not in dtypes:
        t = t.to(dtypes[0])
    return t.contiguous()


def residual_norm(x: torch.Tensor, y: torch.Tensor, gamma: torch.Tensor | None = None, norm=None):
    """Residual update of a pre-norm block and the next LayerNorm in one pass:
    ``x_new = bf16(x + bf16(y * gamma))`` (torch's bf16 LayerScale multiply and
    add) and, with ``norm = (weight or None, bias or None, eps)``, its
    LayerNorm over the last dimension (fp32 statistics, bf16 output).
    x, y: ``[..., dim]`` bf16 of one shape; gamma, weight, bias: ``[dim]``.
    Returns ``(x_new, normed or None)``; x is not modified."""
    _dev(x, "x")
    _dev(y, "y")
    if x.shape != y.shape:
        raise ValueError(f"x {tuple(x.shape)} and y {tuple(y.shape)} differ")
    if x.dtype != torch.bfloat16 or y.dtype != torch.bfloat16:
        raise ValueError("residual_norm computes on bf16 rows")
    dim = x.shape[-1]
    xr, yr = x.reshape(-1, dim), y.reshape(-1, dim)
    if xr.stride(-1) != 1:
        xr = xr.contiguous()
    if yr.stride(-1) != 1:
        yr = yr.contiguous()
    rows = xr.shape[0]
    keep = []

    def param(t, name):
        if t is None:
            return None
        if t.dtype != torch.bfloat16:
            raise ValueError(f"{name} must be bf16: the pass rounds as torch's bf16 ops on bf16 parameters")
        t = _param(t, name, dim, (torch.bfloat16,))
        keep.append(t)
        return t.data_ptr()

    xo = torch.empty(x.shape, device=x.device, dtype=torch.bfloat16)
    no = torch.empty(x.shape, device=x.device, dtype=torch.bfloat16) if norm is not None else None
    w, b, eps = norm if norm is not None else (None, None, 0.0)
    _lib.call("vasc_residual_norm", xr.data_ptr(), xr.stride(0), yr.data_ptr(), yr.stride(0), param(gamma, "gamma"),
              param(w, "norm weight"), param(b, "norm bias"), float(eps), xo.data_ptr(), dim,
              no.data_ptr() if no is not None else None, dim, rows, dim, _stream())
    return xo, no


def _layout_args(B: int, T: int, D: int, q_norm, k_norm, pos, rope_tables) -> tuple[list, tuple]:
    """The norm and rotary arguments of the layout entry points:
    ``(tensors to keep alive, (q norm x4, k norm x4, rope x6))``."""
    keep = []

    def norm_args(nrm, name):
        if nrm is None:
            return (None, None, 0.0, 0)
        w, b, eps = nrm
        given = [t for t in (w, b) if t is not None]
        # both parameters in one dtype the kernel reads directly: bf16 (2) or float32 (1)
        kind = 2 if given and all(t.dtype == torch.bfloat16 for t in given) else 1
        out = []
        for t in (w, b):
            if t is None:
                out.append(None)
            else:
                t = _param(t, f"{name} parameters", D, (torch.bfloat16,) if kind == 2 else (torch.float32,))
                keep.append(t)
                out.append(t.data_ptr())
        return (out[0], out[1], float(eps), kind)

    rope = (None, 0, 2, None, None, 0)
    if pos is not None:
        if rope_tables is None:
            raise ValueError("rope_tables are required with pos")
        _dev(pos, "pos")
        pos32 = pos.to(torch.int32)
        if pos32.dim() == 2:
            pos32 = pos32.unsqueeze(0)
        if pos32.shape[-2:] != (T, 2) or pos32.stride(-1) != 1:
            pos32 = pos32.reshape(-1, T, 2).contiguous()
        if pos32.dim() != 3 or pos32.shape[0] not in (1, B):
            raise ValueError(f"pos must be [{B} or 1, {T}, 2], got {tuple(pos.shape)}")
        cos, sin = (t.float().contiguous() for t in rope_tables)
        if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] != D // 4:
            raise ValueError(f"rope tables must be [n, {D // 4}]")
        keep += [pos32, cos, sin]
        rope = (pos32.data_ptr(), pos32.stride(0) if pos32.shape[0] > 1 else 0, pos32.stride(1), cos.data_ptr(),
                sin.data_ptr(), cos.shape[0])
    return keep, (*norm_args(q_norm, "q_norm"), *norm_args(k_norm, "k_norm"), *rope)


def pack_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, frames: int, tokens_per_frame: int,
             special: int, *, q_norm=None, k_norm=None, pos: torch.Tensor | None = None,
             rope_tables: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Frame-major ``[B,T,H,D]`` q/k/v views -> ``(q_patch, q_special, k, v)``
    in the global layer's ``[patch; special]`` order, ``[B,H,*,D]`` bf16.
    ``v=None`` packs only q and k (the returned v is None).

    ``q_norm`` / ``k_norm``: ``(weight or None, bias or None, eps)`` of a
    per-head LayerNorm, or None. ``pos`` int ``[B,T,2]`` (row, column) with
    ``rope_tables = (cos, sin)`` float32 ``[n, D/4]``: 2D rotary embedding.
    """
    B, T, H, D = q.shape
    N, P, S = int(frames), int(tokens_per_frame), int(special)
    if N * P != T or k.shape != q.shape or (v is not None and v.shape != q.shape):
        raise ValueError(f"q/k/v must be [B,{N}*{P},H,D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{None if v is None else tuple(v.shape)}")
    dev = q.device
    qp = torch.empty(B, H, N * (P - S), D, device=dev, dtype=torch.bfloat16)
    qs = torch.empty(B, H, N * S, D, device=dev, dtype=torch.bfloat16)
    ko = torch.empty(B, H, T, D, device=dev, dtype=torch.bfloat16)
    vo = None if v is None else torch.empty(B, H, T, D, device=dev, dtype=torch.bfloat16)
    keep, args = _layout_args(B, T, D, q_norm, k_norm, pos, rope_tables)
    vsrc = (None, 0, 0, 0) if v is None else _btht(v, "v")
    _lib.call("vasc_pack_qkv", *_btht(q, "q"), *_btht(k, "k"), *vsrc, B, H, N, P, S, D, *args,
              qp.data_ptr(), qs.data_ptr(), ko.data_ptr(), _ptr(vo), _stream())
    del keep
    return qp, (qs if S else None), ko, vo


def pack_global(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, frames: int, tokens_per_frame: int,
                special: int, *, q_norm=None, k_norm=None, pos: torch.Tensor | None = None,
                rope_tables: tuple[torch.Tensor, torch.Tensor] | None = None, innovation: bool = True,
                pooled_v: bool = False, q_scale: float = 1.0):
    """``pack_qkv`` with V packed straight into attention tiles and the
    block-mean pooling of the patch tokens in the same pass.

    Returns ``(q_patch, q_special, k, vt, pooled_q, pooled_k, innovation,
    pooled_v)``: ``q_patch`` / ``q_special`` / ``k`` as ``pack_qkv`` (bit
    for bit), ``vt`` as ``pack_v`` of the packed V, ``pooled_q`` / ``pooled_k``
    as ``pool_qkv(q_patch, k[:, :, :Np])``, ``innovation`` (or None) the pair
    innovation of the patch values' block means, ``pooled_v`` (or None) those
    means. With ``q_scale`` the queries are written as ``bf16(q * q_scale)``
    (``pooled_q`` stays that of the unscaled rows). Requires at least one
    patch token per frame.
    """
    B, T, H, D = q.shape
    N, P, S = int(frames), int(tokens_per_frame), int(special)
    if N * P != T or k.shape != q.shape or v.shape != q.shape:
        raise ValueError(f"q/k/v must be [B,{N}*{P},H,D], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if not 0 <= S < P:
        raise ValueError(f"frames of {P} tokens need at least one patch token (special={S})")
    dev = q.device
    n_patch = N * (P - S)
    kb = math.ceil(n_patch / BLOCK_K)
    bf = dict(device=dev, dtype=torch.bfloat16)
    qp = torch.empty(B, H, n_patch, D, **bf)
    qs = torch.empty(B, H, N * S, D, **bf)
    ko = torch.empty(B, H, T, D, **bf)
    vt = torch.empty(B, H, math.ceil(T / BLOCK_K), D, BLOCK_K, **bf)
    pq = torch.empty(B, H, math.ceil(n_patch / BLOCK_Q), D, **bf)
    pk = torch.empty(B, H, kb, D, **bf)
    pv = torch.empty(B, H, kb, D, **bf) if pooled_v else None
    inn = torch.empty(B, H, (kb + 1) // 2, device=dev, dtype=torch.float32) if innovation else None
    keep, args = _layout_args(B, T, D, q_norm, k_norm, pos, rope_tables)
    _lib.call("vasc_pack_global_scaled", *_btht(q, "q"), *_btht(k, "k"), *_btht(v, "v"), B, H, N, P, S, D, *args,
              qp.data_ptr(), qs.data_ptr(), ko.data_ptr(), vt.data_ptr(), pq.data_ptr(), pk.data_ptr(), _ptr(pv),
              _ptr(inn), float(q_scale), _stream())
    del keep
    return qp, (qs if S else None), ko, vt, pq, pk, inn, pv


def restore_tokens(x_patch: torch.Tensor, x_special: torch.Tensor | None, frames: int, tokens_per_frame: int,
                   special: int) -> torch.Tensor:
    """``[B,H,Np,D]`` + ``[B,H,Ns,D]`` -> frame-major ``[B,T,H*D]`` (bf16)."""
    x_patch = _bhtd(x_patch, "x_patch")
    B, H, n_patch, D = x_patch.shape
    N, P, S = int(frames), int(tokens_per_frame), int(special)
    if n_patch != N * (P - S):
        raise ValueError(f"x_patch holds {n_patch} tokens, expected {N * (P - S)}")
    xs = (None, 0, 0, 8)
    if S:
        if x_special is None or x_special.shape[2] != N * S:
            raise ValueError(f"x_special must hold {N * S} tokens")
        x_special = _bhtd(x_special, "x_special")
        xs = (x_special.data_ptr(), *x_special.stride()[:3])
    out = torch.empty(B, N * P, H * D, device=x_patch.device, dtype=torch.bfloat16)
    _lib.call("vasc_restore_tokens", x_patch.data_ptr(), *x_patch.stride()[:3], *xs, B, H, N, P, S, D,
              out.data_ptr(), _stream())
    return out


# ----------------------------------------------------------------- streaming
# A single query token's kernels take a few microseconds, so these wrappers
# count theirs: one look at each tensor, and no torch call that copies nothing.
_DTYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_ROWS = (torch.bfloat16, torch.float16, torch.float32)
_QUERIES = (torch.bfloat16, torch.float16)


def _launch(dev: int, name: str, *args) -> None:
    """``_lib.call`` on the current stream of GPU ``dev``."""
    if torch._C._cuda_getDevice() == dev:
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(dev))


def on_device(dev: int):
    """A context in which GPU ``dev`` is the current one."""
    return contextlib.nullcontext() if torch._C._cuda_getDevice() == dev else torch.cuda.device(dev)


def _gpu(t, name: str, dev: int = -1) -> int:
    """The GPU that holds ``t``; it has to be ``dev`` where that is given."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a GPU tensor (the HIP path has no CPU fallback)")
    at = t.get_device()
    if at != dev and dev >= 0:
        raise ValueError(f"{name} is on cuda:{at}, expected cuda:{dev}")
    return at


def _tangent(t: torch.Tensor) -> bool:
    """Whether ``t`` carries a forward-mode tangent (the level is -1 where nothing does)."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _inference(t: torch.Tensor, name: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: the block cache has no backward pass, "
                         "call it under torch.no_grad()")
    if _tangent(t):
        raise ValueError(f"{name} carries a forward-mode tangent: the block cache has no derivative")


def _rows8(t: torch.Tensor, name: str, dtypes: tuple) -> tuple:
    """(tensor, its address, strides) of ``[B,H,T,D]`` with unit stride on D and 16-byte aligned rows."""
    if t.dim() != 4:
        raise ValueError(f"{name} must be [B,H,T,D], got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    sb, sh, st, sd = t.stride()
    ptr = t.data_ptr()
    if sd != 1 or (sb | sh | st) & 7 or ptr & 15:
        t = t.contiguous()
        if t.data_ptr() & 15:  # contiguous, but a view that starts inside a row
            t = t.clone()
        _, H, T, D = t.shape
        if D & 7:
            raise ValueError(f"{name} has rows of {D} elements, expected a multiple of 8")
        ptr = t.data_ptr()
        sb, sh, st = H * T * D, T * D, D  # not the tensor's: those of dimensions of size 1 may be anything
    return t, ptr, sb, sh, st


def _int32(t: torch.Tensor, name: str) -> torch.Tensor:
    """``t`` as int32 (which is best kept so: others cost a launch or two); integers that it cannot hold become -1 or 2^31 - 1,
    which are out of range in the same sense."""
    if t.dtype is torch.int32:
        return t
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype is torch.bool:
        raise ValueError(f"{name} must hold integers, got {t.dtype}")
    if t.dtype.itemsize >= 4:
        t = t.to(torch.int64).clamp(-1, 2 ** 31 - 1)
    return t.to(torch.int32)


def _int_rows(t, name: str, B: int, dev: int):
    """``[B]`` int32, contiguous (None stays)."""
    if t is None or (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.shape == (B,)
                     and t.get_device() == dev and t.is_contiguous()):
        return t
    _gpu(t, name, dev)
    t = _int32(t, name)
    if t.shape != (B,):
        raise ValueError(f"{name} must hold {B} integers, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _page_table(t, B: int, dev: int) -> tuple:
    """(tensor, stride of a sequence, pages a sequence)."""
    if isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.get_device() == dev:
        shape, strides = t.shape, t.stride()
        if len(shape) == 2 and shape[0] == B and strides[1] == 1 and strides[0] >= shape[1] > 0:
            return t, strides[0] if B > 1 else shape[1], shape[1]
    _gpu(t, "page_table", dev)
    t = _int32(t, "page_table")
    if t.dim() != 2 or t.shape[0] != B or t.shape[1] == 0:
        raise ValueError(f"page_table must be [{B}, max_pages] integers, got {tuple(t.shape)}")
    mp = t.shape[1]
    sb, sp = t.stride()
    if (mp > 1 and sp != 1) or (B > 1 and sb < mp):
        t = t.contiguous()
        sb = mp
    return t, sb if B > 1 else mp, mp


def _rotary_out(x: torch.Tensor, D: int) -> torch.Tensor:
    """An output in the memory order of ``x`` (strides that fall as its do), D innermost."""
    out = torch.empty_like(x)
    return out if out.stride(3) == 1 or D == 1 else torch.empty(x.shape, device=x.device, dtype=x.dtype)


_NO_K = (None, 0, 0, 0, None, 0, 0, 0, 0)


def _rotary(q, k, pos, sections, inv_freq, inverse: bool) -> tuple:
    B, Hq, T, D = q.shape
    qsb, qsh, qst, qsd = q.stride()
    if qsd != 1:
        q = q.contiguous()
        qsb, qsh, qst, _ = q.stride()
    qo = _rotary_out(q, D)
    ko, kargs = None, _NO_K
    if k is not None:
        Hk = k.shape[1]
        ksb, ksh, kst, ksd = k.stride()
        if ksd != 1:
            k = k.contiguous()
            ksb, ksh, kst, _ = k.stride()
        ko = _rotary_out(k, D)
        if not Hk:
            k = None
        else:
            osb, osh, ost, _ = ko.stride()
            kargs = (k.data_ptr(), ksb, ksh, kst, ko.data_ptr(), osb, osh, ost, Hk)
    if B == 0 or T == 0 or (Hq == 0 and k is None):
        return qo, ko
    if Hq == 0:
        return qo, _rotary(k, None, pos, sections, inv_freq, inverse)[0]
    osb, osh, ost, _ = qo.stride()
    psb, pst, _ = pos.stride()
    sizes, axes, _ = _section_sizes(sections, D)
    _launch(q.get_device(), "vasc_rotary_axes", q.data_ptr(), qsb, qsh, qst, qo.data_ptr(), osb, osh, ost, Hq, *kargs,
            B, T, D, pos.data_ptr(), psb if pos.shape[0] > 1 else 0, pst, axes, sizes, inv_freq.data_ptr(),
            _DTYPE[q.dtype], inverse)
    return qo, ko


class _RotaryAxes(torch.autograd.Function):
    """A turn is orthogonal: its gradient is the opposite turn of the gradient, which is differentiable in turn. It is linear:
    its tangent is the same turn of the tangent."""

    @staticmethod
    def forward(ctx, q, k, pos, sections, inv_freq, inverse):
        ctx.save_for_backward(pos, inv_freq)
        if forward_ad._current_level >= 0:
            ctx.primals = q, k, pos, inv_freq
        ctx.sections, ctx.inverse = sections, inverse
        ctx.set_materialize_grads(False)
        return _rotary(q, k, pos, sections, inv_freq, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        if gq is None and gk is None:
            return None, None, None, None, None, None
        pos, inv_freq = ctx.saved_tensors
        turn = _RotaryAxes.apply if torch.is_grad_enabled() else _rotary  # grad mode: a second derivative is asked for
        if gq is None:
            return None, turn(gk, None, pos, ctx.sections, inv_freq, not ctx.inverse)[0], None, None, None, None
        return *turn(gq, gk, pos, ctx.sections, inv_freq, not ctx.inverse), None, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        q, k, pos, inv_freq = ctx.primals
        del ctx.primals
        tq = torch.zeros_like(q) if tq is None else tq
        tk = torch.zeros_like(k) if tk is None and k is not None else tk
        turn = _RotaryAxes.apply if torch.is_grad_enabled() else _rotary
        return turn(tq, tk, pos, ctx.sections, inv_freq, ctx.inverse)


def _one_graph(node, inputs=()) -> None:
    """Refuses a captured call on leaves that an eager call's live graph holds.

    Both graphs share a leaf's accumulation node, whose stream is the eager
    call's: the captured backward pass would wait for it from outside the
    capture, which ends the process. The mark goes with the node, so it is
    gone when the eager graph is. ``inputs``: the tensors of the node's first
    edges; an edge of a view of a leaf is followed to the leaf.
    """
    captured = torch.cuda.is_current_stream_capturing()
    for i, (leaf, _) in enumerate(node.next_functions):
        if leaf is None:
            continue
        if leaf.next_functions:
            base = inputs[i]._base if i < len(inputs) else None
            if base is None or not base.is_leaf:
                continue
            while leaf.next_functions:  # views have one input
                leaf = leaf.next_functions[0][0]
        if not captured:
            leaf.metadata["eager"] = True
        elif "eager" in leaf.metadata:
            raise ValueError("q or k is, or is a view of, a leaf of an eager graph that still lives: "
                             "drop that call's outputs before capturing")


@functools.lru_cache(maxsize=64)
def _section_sizes(sections: tuple, D: int):
    """(the checked sections of a head dimension as a C array, their number, their pairs)."""
    if not 1 <= len(sections) <= 4 or any(s <= 0 or s % 2 for s in sections) or sum(sections) > D:
        raise ValueError(f"sections {sections} must be 1 to 4 even sizes that sum to at most {D}")
    return (ctypes.c_int64 * len(sections))(*sections), len(sections), sum(sections) // 2


def rotary_axes(q: torch.Tensor, k: torch.Tensor | None, pos: torch.Tensor, sections, inv_freq: torch.Tensor):
    """Rotary embedding over several position axes, of q and k in one launch.

    q ``[B,Hq,T,D]``, k ``[B,Hk,T,D]`` or None, of one dtype (bf16, fp16 or
    fp32), any strides over B, H, T. Axis ``a`` of ``pos [B,T,A]`` (integers
    of 32 bits; ``[T,A]`` and ``[1,T,A]`` serve every sequence) turns the next
    ``sections[a]`` features: pair ``(j, j + sections[a]/2)`` by the angle
    ``pos * inv_freq``, whose float64 values ``[sum(sections)/2]`` hold the
    axes' frequencies one after another. Features past the sections pass
    through. Returns ``(q', k' or None)`` in the inputs' memory order;
    differentiable in q and k, backward and forward. Where q or k is a leaf or
    a view of one, a captured call is refused while an eager call's graph of
    that leaf lives, on whatever stream that was; eager graphs that other
    operators made of it, and leaves behind other operators, are not seen.
    """
    dev = _gpu(q, "q")
    dtype = q.dtype
    if q.dim() != 4 or dtype not in _DTYPE:
        raise ValueError(f"q must be [B,H,T,D] in bf16, fp16 or fp32, got {dtype} {tuple(q.shape)}")
    B, _, T, D = q.shape
    if k is not None:
        _gpu(k, "k", dev)
        kshape = k.shape
        if len(kshape) != 4 or k.dtype is not dtype or kshape[0] != B or kshape[2] != T or kshape[3] != D:
            raise ValueError(f"k must be [{B},H,{T},{D}] of {dtype}, got {k.dtype} {tuple(kshape)}")
    sections = tuple(sections)
    _, A, pairs = _section_sizes(sections, D)
    _gpu(pos, "pos", dev)
    if pos.dtype is not torch.int32:
        if pos.dtype.is_floating_point or pos.dtype is torch.bool:
            raise ValueError(f"pos must hold integers, got {pos.dtype}")
        pos = pos.to(torch.int32)
    pshape = pos.shape
    if len(pshape) == 2:
        pos = pos.unsqueeze(0)
        pshape = pos.shape
    if pshape != (B, T, A) and pshape != (1, T, A):
        raise ValueError(f"pos must be [{B} or 1, {T}, {A}], got {tuple(pshape)}")
    if A > 1 and pos.stride(2) != 1:
        pos = pos.contiguous()
    _gpu(inv_freq, "inv_freq", dev)
    if inv_freq.dtype is not torch.float64 or inv_freq.shape != (pairs,):
        raise ValueError(f"inv_freq must hold {pairs} float64 values, got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if not inv_freq.is_contiguous():
        inv_freq = inv_freq.contiguous()
    grad = torch.is_grad_enabled()
    if (grad and inv_freq.requires_grad) or _tangent(inv_freq):
        raise ValueError("inv_freq requires a gradient or carries a tangent: rotary_axes is differentiable in q and k only")
    grad = grad and (q.requires_grad or (k is not None and k.requires_grad))
    if grad or forward_ad._current_level >= 0:
        out = _RotaryAxes.apply(q, k, pos, sections, inv_freq, False)
        if grad:
            _one_graph(out[0].grad_fn, (q,) if k is None else (q, k))
        return out
    return _rotary(q, k, pos, sections, inv_freq, False)


def cache_write(cache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor,
                count: torch.Tensor | None = None) -> None:
    """Writes new tokens into a ``streaming.BlockCache``, in 8 bits.

    k, v ``[B,H,T,D]`` (bf16, fp16 or fp32, any strides over B, H, T): token
    ``t < count[b]`` (default T) of sequence b becomes its token
    ``start[b] + t``. ``page_table [B,max_pages]`` holds the sequences' pages
    (entries outside the cache: nothing is written there); no page may occur
    twice among the pages one call writes. Each (token, head) row is rounded
    to e4m3 values times a power of two, and every touched page's key mean is
    renewed over its tokens up to the last one written, so the tokens before
    ``start`` in its page must be there, and writing further back drops what
    came after. A token whose k or v row holds a value that is not finite is
    held as NaN in both. Nothing here waits for the GPU.
    """
    dev = _gpu(k, "k")
    _gpu(v, "v", dev)
    _inference(k, "k")
    _inference(v, "v")
    if cache.device_index != dev:
        raise ValueError(f"the cache is on cuda:{cache.device_index}, k on cuda:{dev}")
    k, *kargs = _rows8(k, "k", _ROWS)
    v, *vargs = _rows8(v, "v", _ROWS)
    B, H, T, D = shape = k.shape
    if shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k {k.dtype} {tuple(shape)} and v {v.dtype} {tuple(v.shape)} differ")
    if H != cache.heads or D != cache.head_dim:
        raise ValueError(f"the cache holds {cache.heads} heads of {cache.head_dim}, k has {H} of {D}")
    table, ts, mp = _page_table(page_table, B, dev)
    start, count = _int_rows(start, "start", B, dev), _int_rows(count, "count", B, dev)
    if start is None:
        raise ValueError("start is required")
    if B == 0 or T == 0:
        return
    _launch(dev, "vasc_cache_write", *kargs, *vargs, B, H, T, D,
            _DTYPE[k.dtype], table.data_ptr(), ts, mp, start.data_ptr(), _ptr(count), *cache.pointers,
            cache.mean_pointer, cache.pages)


def cache_read(cache, page_table: torch.Tensor, start: torch.Tensor, tokens: int, count: torch.Tensor | None = None,
               dtype: torch.dtype = torch.bfloat16) -> tuple:
    """``(k, v) [B,H,tokens,D]`` of the cache's tokens ``start[b]..`` in
    ``dtype`` (bf16: exactly what the cache holds). Rows from ``count[b]`` on
    (default ``tokens``) and rows that have no page are zero."""
    dev = _gpu(page_table, "page_table")
    if cache.device_index != dev:
        raise ValueError(f"the cache is on cuda:{cache.device_index}, page_table on cuda:{dev}")
    if dtype not in _DTYPE:
        raise ValueError(f"dtype must be bf16, fp16 or fp32, got {dtype}")
    B, H, D, tokens = page_table.shape[0], cache.heads, cache.head_dim, int(tokens)
    if tokens < 0:
        raise ValueError(f"tokens must not be negative, got {tokens}")
    table, ts, mp = _page_table(page_table, B, dev)
    start, count = _int_rows(start, "start", B, dev), _int_rows(count, "count", B, dev)
    if start is None:
        raise ValueError("start is required")
    k = torch.empty(B, H, tokens, D, device=table.device, dtype=dtype)
    v = torch.empty(B, H, tokens, D, device=table.device, dtype=dtype)
    if B and tokens:
        _launch(dev, "vasc_cache_read", *cache.pointers, cache.pages, table.data_ptr(), ts, mp, start.data_ptr(),
                _ptr(count), B, H, tokens, D, _DTYPE[dtype], k.data_ptr(), v.data_ptr())
    return k, v


def _cache_query(q, cache, page_table, lengths, q_count, block_q: int, dev: int) -> tuple:
    """(q, its shape, its C arguments, page table x 3, lengths, q_count), checked."""
    _inference(q, "q")
    if cache.device_index != dev:
        raise ValueError(f"the cache is on cuda:{cache.device_index}, q on cuda:{dev}")
    q, *args = _rows8(q, "q", _QUERIES)
    B, Hq, T, D = shape = q.shape
    H = cache.heads
    if D != cache.head_dim or Hq % H or Hq == 0:
        raise ValueError(f"q has {Hq} heads of {D}: expected a multiple of {H} heads of {cache.head_dim}")
    if not (1 <= block_q and block_q * (Hq // H) <= 128):
        raise ValueError(f"block_q {block_q} with {Hq // H} query heads a key head: a unit has 1 to 128 rows")
    lengths = _int_rows(lengths, "lengths", B, dev)
    if lengths is None:
        raise ValueError("lengths is required")
    return q, shape, args, *_page_table(page_table, B, dev), lengths, _int_rows(q_count, "q_count", B, dev)


def cache_select(q: torch.Tensor, cache, page_table: torch.Tensor, lengths: torch.Tensor, keep: int, *,
                 block_q: int = 1, sink: int = 1, recent: int = 1, causal: bool = False,
                 q_count: torch.Tensor | None = None, want_score: bool = False) -> tuple:
    """Pages that each unit of queries attends to, by a cheap score.

    A unit is ``block_q`` consecutive query tokens of the ``G = Hq / H`` query
    heads that share a key head (``block_q * G <= 128``); q ``[B,Hq,T,D]`` bf16
    or fp16. A page's score is the product of the unit's mean query and the
    page's mean key (both rounded to bf16, summed in float64). Listed are the
    first ``sink`` pages, the last ``recent``, and the ``keep`` of highest score
    among the others (equal scores in page order, NaN lowest). ``lengths[b]``:
    tokens of sequence b in the cache. With ``causal`` the ``q_count[b]``
    (default T) queries are its last tokens; a unit then sees the pages up to
    its last row's own, and ``recent`` counts back from its first row's own
    page (every page from there on is listed).

    Returns ``(index [B,H,U,W], count [B,H,U])`` int32, ``U = ceil(T / block_q)``:
    ascending logical pages, -1 behind them; ``W`` is the largest possible
    count. ``want_score`` adds the scores ``[B,H,U,max_pages]`` float32 (-inf
    for pages the unit does not see).
    """
    dev = _gpu(q, "q")
    block_q, keep, sink, recent, causal = int(block_q), int(keep), int(sink), int(recent), bool(causal)
    q, shape, qargs, table, ts, mp, lengths, q_count = _cache_query(q, cache, page_table, lengths, q_count, block_q, dev)
    if keep < 0 or sink < 0 or recent < 1:
        raise ValueError(f"keep {keep} and sink {sink} must not be negative, recent {recent} at least 1")
    B, Hq, T, D = shape
    H, U = cache.heads, -(-T // block_q)
    width = min(mp, sink + keep + recent + ((block_q + BLOCK_K - 2) // BLOCK_K if causal else 0))
    device = q.device
    index = torch.empty(B, H, U, width, device=device, dtype=torch.int32)
    count = torch.empty(B, H, U, device=device, dtype=torch.int32)
    score = torch.empty(B, H, U, mp, device=device, dtype=torch.float32)
    if B and T:
        _launch(dev, "vasc_cache_select", *qargs, B, Hq, H, T, D, _DTYPE[q.dtype], cache.mean_pointer, cache.pages,
                table.data_ptr(), ts, mp, lengths.data_ptr(), _ptr(q_count), block_q, sink, recent, keep, causal,
                score.data_ptr(), index.data_ptr(), width, count.data_ptr())
    return (index, count, score) if want_score else (index, count)


@functools.lru_cache(maxsize=256)
def _attn_workspace(*sizes: int) -> int:
    return _lib.fn("vasc_cache_attn_workspace_size")(*sizes)


def cache_attn(q: torch.Tensor, cache, page_table: torch.Tensor, lengths: torch.Tensor,
               index: torch.Tensor | None = None, count: torch.Tensor | None = None, *, block_q: int | None = None,
               causal: bool = False, q_count: torch.Tensor | None = None, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q ``[B,Hq,T,D]`` (bf16 or fp16) over the cache.

    ``index`` / ``count``: the lists of ``cache_select`` with the same
    ``block_q`` (ascending logical pages; an entry not above the one before it
    is skipped); without them every page is attended to. Keys at or past
    ``lengths[b]`` are not seen, nor, with ``causal``, those behind the row's
    own position ``lengths[b] - q_count[b] + t``. Rows that see no key, and
    rows from ``q_count[b]`` on, are zero; rows that see a NaN token, or whose
    query is not finite, are NaN. Softmax scale ``scale`` (default
    ``D ** -0.5``). Returns ``[B,Hq,T,D]`` of q's dtype, written to ``out``
    when given (unit stride over D).
    """
    dev = _gpu(q, "q")
    if (index is None) != (count is None):
        raise ValueError("index and count go together")
    if q.dim() != 4:
        raise ValueError(f"q must be [B,H,T,D], got {tuple(q.shape)}")
    if block_q is None:
        if index is not None and q.shape[2] > 1:
            raise ValueError("lists need the block_q they were made with")
        block_q = max(1, min(q.shape[2], 128 // max(1, q.shape[1] // cache.heads)))
    block_q = int(block_q)
    q, shape, qargs, table, ts, mp, lengths, q_count = _cache_query(q, cache, page_table, lengths, q_count, block_q, dev)
    B, Hq, T, D = shape
    H, width = cache.heads, 0
    if index is not None:
        U = -(-T // block_q)
        _gpu(index, "index", dev)
        _gpu(count, "count", dev)
        ishape = index.shape
        if len(ishape) != 4 or ishape[:3] != (B, H, U) or count.shape != (B, H, U):
            raise ValueError(f"index/count must be [{B},{H},{U},W]/[{B},{H},{U}], got {tuple(ishape)}/"
                             f"{tuple(count.shape)}")
        index, count = _int32(index, "index").contiguous(), _int32(count, "count").contiguous()
        width = ishape[3]
    if out is None:
        out = torch.empty(shape, device=q.device, dtype=q.dtype)
        osb, osh, ost = Hq * T * D, T * D, D
    else:
        _gpu(out, "out", dev)
        if out.shape != shape or out.dtype != q.dtype:
            raise ValueError(f"out must be {q.dtype} {tuple(shape)}, got {out.dtype} {tuple(out.shape)}")
        _inference(out, "out")
        osb, osh, ost, osd = (st if n > 1 else D for n, st in zip(shape, out.stride()))
        if not (osb and osh and ost):
            raise ValueError("out's rows overlap (an expanded tensor)")
        if osd != 1 or (osb | osh | ost) & 3 or out.data_ptr() & 7:
            raise ValueError("out needs unit stride over D and 8-byte aligned rows")
    if B == 0 or T == 0:
        return out
    if index is not None and width == 0:
        return out.zero_()
    size = _attn_workspace(B, Hq, H, T, D, block_q, mp, width)
    ws = torch.empty(size, device=q.device, dtype=torch.uint8) if size > 0 else None
    _launch(dev, "vasc_cache_attn", *qargs, out.data_ptr(), osb, osh, ost, B, Hq, H, T, D, _DTYPE[q.dtype],
            *cache.pointers, cache.pages, table.data_ptr(), ts, mp, lengths.data_ptr(), _ptr(q_count), block_q,
            _ptr(index), width, _ptr(count), bool(causal), D ** -0.5 if scale is None else scale, _ptr(ws), size)
    return out
