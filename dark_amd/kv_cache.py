"""Paged key / value cache: per-head norms and rotation, appending new tokens, attention of a chunk over the pages.

No counterpart in the reference, whose callers run with ``use_cache=False`` (configuration_dream.py:29-50) and recompute
the whole window in every denoise step.  With a cache a step recomputes only the positions that can still change
(``diffusion_generate(..., cache_interval=R)``), and windows are not limited to 128 positions.

A layer's cache is two tensors ``[n_pages, page_size, n_kv_heads, head_dim]`` (any strides with a contiguous last
dimension, the same for both); token ``j`` of a sequence lies in slot ``j % page_size`` of page
``block_table[b, j // page_size]``.  The functions enqueue on torch's current stream of the tensors' device, never
synchronise, and have no backward: a tensor that asks for gradients is refused while gradients are enabled.
"""
from __future__ import annotations

import struct
from typing import Optional, Sequence, Tuple

import torch

from . import _hip

_DTYPES = {torch.float32: _hip.DARK_F32, torch.bfloat16: _hip.DARK_BF16}
_KV = "2Q3q6i"                                    # dark_paged_kv
_NORM_ROPE = struct.Struct("=9Q8q6ifi")           # dark_qk_norm_rope_args
_APPEND = struct.Struct(f"={_KV}10Q8q3if")        # dark_kv_append_args
_ATTEND = struct.Struct(f"={_KV}9Q7q7if")         # dark_paged_attention_args


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _check(name: str, t: torch.Tensor, dev: torch.device, dtype: Optional[torch.dtype], dim: int) -> None:
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} has {t.dim()} dimensions, expected {dim}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} requires gradients: the cache's operators have no backward (use torch.no_grad())")


def _fits(t: torch.Tensor) -> bool:
    """16-byte pointer and strides, contiguous last dimension: what the kernels' vector accesses take."""
    if t.data_ptr() & 15 or t.stride(-1) != 1:
        return False
    es = t.element_size()
    return all(s * es % 16 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)


def _distinct(name: str, t: torch.Tensor) -> None:
    """Something is written through t: no two elements may share memory (expanded views)."""
    _need(all(s > 0 for s, n in zip(t.stride(), t.shape) if n > 1), f"{name}: an expanded tensor cannot be written")


def _rows(name: str, t: torch.Tensor, dev, dtype, T: int, HD: int) -> torch.Tensor:
    """A [T, heads, head_dim] input, copied only where its strides or its alignment do not fit."""
    _check(name, t, dev, dtype, 3)
    _need(t.shape[0] == T and t.shape[2] == HD, f"{name} is {tuple(t.shape)}, expected [{T}, heads, {HD}]")
    return t if _fits(t) else t.clone(memory_format=torch.contiguous_format)


def _out(name: str, t: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    if t is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    _check(name, t, like.device, like.dtype, 3)
    _need(t.shape == like.shape, f"{name} is {tuple(t.shape)}, expected {tuple(like.shape)}")
    _need(t.numel() == 0 or _fits(t), f"{name}: pointer and strides must be multiples of 16 bytes, the last dimension contiguous")
    _distinct(name, t)
    return t


def _vec(name: str, t: Optional[torch.Tensor], dev, dtype, n: int) -> int:
    if t is None:
        return 0
    _check(name, t, dev, dtype, 1)
    _need(t.shape[0] == n and t.is_contiguous(), f"{name} must be contiguous with {n} elements")
    return t.data_ptr()


def _tables(cos, sin, pos, dev, T: int, HD: int) -> Tuple[int, int, int, int]:
    if cos is None and sin is None:
        return 0, 0, 0, 0
    _need(cos is not None and sin is not None and pos is not None, "cos, sin and pos go together")
    _check("cos", cos, dev, torch.float32, 2)
    _check("sin", sin, dev, torch.float32, 2)
    _need(cos.shape == sin.shape and cos.shape[0] >= 1 and cos.shape[1] == HD // 2 and cos.is_contiguous() and sin.is_contiguous(),
          f"cos and sin must be contiguous [max_pos, {HD // 2}]")
    return cos.data_ptr(), sin.data_ptr(), _vec("pos", pos, dev, torch.int32, T), cos.shape[0]


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, dev, dtype):
    """The fields of dark_paged_kv."""
    _check("k_cache", k_cache, dev, dtype, 4)
    _check("v_cache", v_cache, dev, dtype, 4)
    _need(k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride(), "k_cache and v_cache must have the same shape and strides")
    n_pages, page, Hk, HD = k_cache.shape
    _need(page >= 1 and page & (page - 1) == 0, f"page size {page} must be a power of two")
    _need(k_cache.numel() == 0 or (_fits(k_cache) and _fits(v_cache)),
          "the cache's pointers and strides must be multiples of 16 bytes, the last dimension contiguous")
    _distinct("the cache", k_cache)
    ps, ss, hs, _ = k_cache.stride()
    # (a dimension of one has no stride of its own)
    return (k_cache.data_ptr(), v_cache.data_ptr(), ps if n_pages > 1 else 0, ss if page > 1 else 0, hs if Hk > 1 else 0,
            _DTYPES[dtype], n_pages, page, Hk, HD, 0)


def _ts_hs(t: torch.Tensor) -> Tuple[int, int]:
    a, b, _ = t.stride()
    return (a if t.shape[0] > 1 else 0), (b if t.shape[1] > 1 else 0)


def _begin(t: torch.Tensor) -> torch.device:
    if not t.is_cuda:
        raise RuntimeError("dark_amd runs on a HIP device only")
    if t.dtype not in _DTYPES:
        raise ValueError(f"dtype {t.dtype}: float32 and bfloat16 only")
    return t.device


def _call(fn, packed: bytes, dev: torch.device) -> None:
    if dev.index != torch.cuda.current_device():      # the library launches on the CURRENT device
        with torch.cuda.device(dev):
            _hip.check(fn(packed, _hip.stream_ptr(dev)))
    else:
        _hip.check(fn(packed, _hip.stream_ptr(dev)))


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], pos: Optional[torch.Tensor], eps: float = 1e-6,
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm over each head of ``q [T, n_heads, head_dim]`` and ``k [T, n_kv_heads, head_dim]`` (``weight [head_dim]``
    fp32, None = no norm), then the rotation by row ``pos[t]`` (int32, clamped) of the fp32 tables ``cos`` / ``sin
    [max_pos, head_dim/2]`` (both None = no rotation); fp32 inside, one rounding.  ``q_out`` / ``k_out`` may be ``q`` /
    ``k`` themselves.  Returns ``(q_out, k_out)``."""
    dev = _begin(q)
    T, Hq, HD = q.shape if q.dim() == 3 else (0, 0, 0)
    qi = _rows("q", q, dev, q.dtype, T, HD)
    ki = _rows("k", k, dev, q.dtype, T, HD)
    q_out, k_out = _out("q_out", q_out, q), _out("k_out", k_out, k)
    c, s, p, n = _tables(cos, sin, pos, dev, T, HD)
    _call(_hip.load().dark_qk_norm_rope,
          _NORM_ROPE.pack(qi.data_ptr(), ki.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                          _vec("q_weight", q_weight, dev, torch.float32, HD), _vec("k_weight", k_weight, dev, torch.float32, HD),
                          c, s, p, *_ts_hs(qi), *_ts_hs(ki), *_ts_hs(q_out), *_ts_hs(k_out),
                          _DTYPES[q.dtype], T, Hq, k.shape[1], HD, n, eps, 0), dev)
    return q_out, k_out


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
              cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None, *,
              q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
              k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Optional[torch.Tensor]:
    """Writes ``k`` (normed where ``k_weight`` is given, rotated where the tables are) and ``v`` ``[T, n_kv_heads,
    head_dim]`` of new tokens into the cache: token ``t`` into slot ``slots[t]`` (int64, ``page * page_size + slot``;
    a negative one, or one beyond the cache, is not stored).  The slots of one call must differ.  ``q`` is normed and
    rotated in the same pass into ``q_out`` (which may be ``q``), the return value."""
    dev = _begin(k)
    T, Hk, HD = k.shape if k.dim() == 3 else (0, 0, 0)
    kv = _cache(k_cache, v_cache, dev, k.dtype)
    _need(kv[8] == Hk and kv[9] == HD, f"k is {tuple(k.shape)}, the cache holds {kv[8]} heads of {kv[9]}")
    ki = _rows("k", k, dev, k.dtype, T, HD)
    vi = _rows("v", v, dev, k.dtype, T, HD)
    _need(v.shape == k.shape, f"v is {tuple(v.shape)}, expected {tuple(k.shape)}")
    qi, strides, Hq = None, (0, 0, 0, 0), 0
    if q is not None:
        qi = _rows("q", q, dev, k.dtype, T, HD)
        q_out = _out("q_out", q_out, q)
        strides, Hq = (*_ts_hs(qi), *_ts_hs(q_out)), q.shape[1]
    else:
        _need(q_out is None, "q_out without q")
    c, s, p, n = _tables(cos, sin, pos, dev, T, HD)
    _call(_hip.load().dark_kv_append,
          _APPEND.pack(*kv, 0 if qi is None else qi.data_ptr(), ki.data_ptr(), vi.data_ptr(), 0 if qi is None else q_out.data_ptr(),
                       _vec("q_weight", q_weight, dev, torch.float32, HD), _vec("k_weight", k_weight, dev, torch.float32, HD),
                       c, s, p, _vec("slots", slots, dev, torch.int64, T), *strides[:2], *_ts_hs(ki), *_ts_hs(vi), *strides[2:],
                       T, Hq, n, eps), dev)
    return q_out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_len: torch.Tensor, max_q: int, max_kv: int, *, q_index: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of new tokens ``q [T, n_heads, head_dim]`` over the cache (their own keys appended before).  Tokens
    ``cu_q[b] .. cu_q[b+1]-1`` (int32) belong to sequence ``b``, which has ``kv_len[b]`` (int32) keys in the pages
    ``block_table[b]`` (int32, an entry outside the cache leaves its keys out).  Left out are keys whose ``key_mask[b, j]``
    (uint8 or bool) is 0 and, with ``causal``, keys behind the token's own place ``q_index[t]`` (int32; default: the
    sequence's last places).  A token with no key left gets zeros (lse -inf).  ``max_q`` / ``max_kv``: the most new tokens /
    keys of a sequence.  ``scale`` defaults to ``head_dim ** -0.5``.  Returns ``out``, or ``(out, lse [T, n_heads] fp32)``."""
    dev = _begin(q)
    T, H, HD = q.shape if q.dim() == 3 else (0, 0, 0)
    kv = _cache(k_cache, v_cache, dev, q.dtype)
    qi = _rows("q", q, dev, q.dtype, T, HD)
    _need(kv[9] == HD and kv[8] >= 1 and H % kv[8] == 0, f"q is {tuple(q.shape)}, the cache holds {kv[8]} heads of {kv[9]}")
    _check("block_table", block_table, dev, torch.int32, 2)
    B, width = block_table.shape
    _need(width <= 1 or block_table.stride(1) == 1, "block_table rows must be contiguous")
    mask, mask_stride = 0, 0
    if key_mask is not None:
        _check("key_mask", key_mask, dev, None, 2)
        _need(key_mask.dtype in (torch.uint8, torch.bool), f"key_mask is {key_mask.dtype}, expected uint8 or bool")
        _need(key_mask.shape[0] == B and key_mask.shape[1] >= max_kv and (key_mask.shape[1] <= 1 or key_mask.stride(1) == 1),
              f"key_mask is {tuple(key_mask.shape)}, expected [{B}, >= {max_kv}] with contiguous rows")
        mask, mask_stride = key_mask.data_ptr(), key_mask.stride(0) if B > 1 else 0
    _need(max_q >= 0 and max_kv >= 0, f"max_q={max_q}, max_kv={max_kv}")
    if out is None:
        out = torch.empty((T, H, HD), dtype=q.dtype, device=dev)
    else:
        out = _out("out", out, q)
    lse = torch.empty((T, H), dtype=torch.float32, device=dev) if return_lse else None
    fields = [*kv, qi.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, block_table.data_ptr(),
              _vec("cu_q", cu_q, dev, torch.int32, B + 1), _vec("kv_len", kv_len, dev, torch.int32, B),
              _vec("q_index", q_index, dev, torch.int32, T), mask, 0, 0, *_ts_hs(qi), *_ts_hs(out),
              block_table.stride(0) if B > 1 else width, mask_stride, T, H, B, width, max_q, max_kv, int(bool(causal)),
              HD ** -0.5 if scale is None else scale]
    lib = _hip.load()
    packed = _ATTEND.pack(*fields)
    need = lib.dark_paged_attention_workspace_bytes(packed)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        fields[19], fields[20] = ws.data_ptr(), need
        packed = _ATTEND.pack(*fields)
    _call(lib.dark_paged_attention, packed, dev)
    return (out, lse) if return_lse else out
