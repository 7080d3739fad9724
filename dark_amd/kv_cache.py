"""Paged key / value cache: per-head norms and rotation, appending new tokens, attention of a chunk over the pages.

No counterpart in the reference, whose callers run with ``use_cache=False`` (configuration_dream.py:29-50) and recompute
the whole window in every denoise step.  With a cache a step recomputes only the positions that can still change
(``diffusion_generate(..., cache_interval=R)``), and windows are not limited to 128 positions.

A layer's cache is two tensors ``[n_pages, page_size, n_kv_heads, head_dim]`` (any strides with a contiguous last
dimension, the same for both); token ``j`` of a sequence lies in slot ``j % page_size`` of page
``block_table[b, j // page_size]``.  The functions enqueue on torch's current stream of the tensors' device, never
synchronise, and have no derivatives: a tensor that asks for gradients is refused while gradients are enabled, one with a
forward-mode tangent while those are.  What they write counts as written for autograd.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _hip

_DTYPES = {torch.float32: _hip.DARK_F32, torch.bfloat16: _hip.DARK_BF16}
_bind = None


def _ops():
    """The compiled binding (csrc/bind.cpp): checks operands, fills the argument structs of include/dark_hip.h."""
    global _bind
    if _bind is None:
        try:
            from . import _bind as mod
        except ImportError as e:
            raise ImportError(f"dark_amd/_bind.so cannot be loaded ({e}): build it with `make -C dark_amd/csrc`") from e
        lib = _hip.load()
        if getattr(mod, "ABI_VERSION", None) != _hip.ABI_VERSION:
            raise ImportError(f"dark_amd/_bind.so was built for ABI version {getattr(mod, 'ABI_VERSION', None)}, the library has "
                              f"{_hip.ABI_VERSION}: build it anew with `make -C dark_amd/csrc`")
        mod.init(_hip.DarkHipError, *(C.cast(getattr(lib, n), C.c_void_p).value for n in (
            "dark_qk_norm_rope", "dark_kv_append", "dark_paged_attention", "dark_paged_attention_workspace_bytes",
            "dark_hip_last_error")))
        _bind = mod
    return _bind


def _stream(t: torch.Tensor) -> int:
    """hipStream_t of torch's current stream on the tensor's device."""
    dev = t.get_device()
    return torch._C._cuda_getCurrentRawStream(dev) if dev >= 0 else 0


def _need(cond: bool, msg: str) -> None:
    if not cond:
        raise ValueError(msg)


def _refuse(name: str, t, dev: int, dtype, dim: int) -> None:
    """Returns if t is a tensor of this device, dtype and number of dimensions."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name} has {t.dim()} dimensions, expected {dim}")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor],
                 cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], pos: Optional[torch.Tensor], eps: float = 1e-6,
                 q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm over each head of ``q [T, n_heads, head_dim]`` and ``k [T, n_kv_heads, head_dim]`` (``weight [head_dim]``
    fp32, None = no norm), then the rotation by row ``pos[t]`` (int32, clamped) of the fp32 tables ``cos`` / ``sin
    [max_pos, head_dim/2]`` (both None = no rotation); fp32 inside, one rounding.  ``q_out`` / ``k_out`` may be ``q`` /
    ``k`` themselves.  Returns ``(q_out, k_out)``."""
    return (_bind or _ops()).qk_norm_rope(_stream(q), q, k, q_weight, k_weight, cos, sin, pos, eps, q_out, k_out)


def append_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
              cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None, *,
              q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
              k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> Optional[torch.Tensor]:
    """Writes ``k`` (normed where ``k_weight`` is given, rotated where the tables are) and ``v`` ``[T, n_kv_heads,
    head_dim]`` of new tokens into the cache: token ``t`` into slot ``slots[t]`` (int64, ``page * page_size + slot``;
    a negative one, or one beyond the cache, is not stored).  The slots of one call must differ.  ``q`` is normed and
    rotated in the same pass into ``q_out`` (which may be ``q``), the return value."""
    return (_bind or _ops()).append_kv(_stream(k), k, v, k_cache, v_cache, slots, cos, sin, pos, q, q_out, q_weight, k_weight, eps)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    cu_q: torch.Tensor, kv_len: torch.Tensor, max_q: int, max_kv: int, *, q_index: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, causal: bool = False, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of new tokens ``q [T, n_heads, head_dim]`` over the cache (their own keys appended before).  Tokens
    ``cu_q[b] .. cu_q[b+1]-1`` (int32) belong to sequence ``b``, which has ``kv_len[b]`` (int32) keys in the pages
    ``block_table[b]`` (int32, an entry outside the cache leaves its keys out).  Left out are keys whose ``key_mask[b, j]``
    (uint8 or bool) is 0 and, with ``causal``, keys behind the token's own place ``q_index[t]`` (int32; default: the
    sequence's last places).  A token with no key left gets zeros (lse -inf).  ``max_q`` / ``max_kv``: the most new tokens /
    keys of a sequence.  Tokens that belong to no sequence are not written; ``out`` must not overlap ``q``.  Scores and sums are
    fp32; in bf16 the softmax weights are rounded to bf16 for the product with the values.  ``scale`` defaults to
    ``head_dim ** -0.5``.  Returns ``out``, or ``(out, lse [T, n_heads] fp32)``."""
    return (_bind or _ops()).paged_attention(_stream(q), q, k_cache, v_cache, block_table, cu_q, kv_len, max_q, max_kv, q_index,
                                            key_mask, causal, scale, out, return_lse)


class PagedKVCache:
    """The pages of every layer of a model and who holds them.  ``k(l)`` / ``v(l)`` are layer ``l``'s ``[n_pages, page_size,
    n_kv_heads, head_dim]`` (a head's slots of a page lie together in memory: what the attention reads)."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, dtype: torch.dtype,
                 device) -> None:
        _need(dtype in _DTYPES, f"dtype {dtype}: float32 and bfloat16 only")
        _need(page_size >= 1 and page_size & (page_size - 1) == 0, f"page size {page_size} must be a power of two")
        _need(n_layers >= 0 and n_pages >= 0 and n_kv_heads >= 1 and head_dim >= 1, "negative size")
        self.n_layers, self.n_pages, self.page_size = n_layers, n_pages, page_size
        self.n_kv_heads, self.head_dim, self.dtype = n_kv_heads, head_dim, dtype
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self._k, self._v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        self._free = list(range(n_pages - 1, -1, -1))

    @property
    def device(self) -> torch.device:
        return self._k.device

    def k(self, layer: int) -> torch.Tensor:
        return self._k[layer].transpose(1, 2)

    def v(self, layer: int) -> torch.Tensor:
        return self._v[layer].transpose(1, 2)

    def pages_for(self, n_tokens: int) -> int:
        return -(-n_tokens // self.page_size)

    def allocate(self, n_tokens: int) -> list:
        """Page ids for ``n_tokens`` tokens of a sequence; MemoryError (nothing taken) if there are not enough."""
        n = self.pages_for(n_tokens)
        if n > len(self._free):
            raise MemoryError(f"{n} pages wanted, {len(self._free)} of {self.n_pages} free")
        out = [self._free.pop() for _ in range(n)]
        return out

    def free(self, pages) -> None:
        """Gives pages back; ValueError (nothing given back) if one of them is not held or named twice."""
        pages, gone = [int(p) for p in pages], set(self._free)
        for p in pages:
            _need(0 <= p < self.n_pages and p not in gone, f"page {p} is not held")
            gone.add(p)
        self._free.extend(pages)

    def slots(self, block_table: torch.Tensor, seq: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
        """Slot (int64) of token ``index[t]`` of sequence ``seq[t]``; -1 where the table names no page for it."""
        if block_table.numel() == 0:
            return torch.full(index.shape, -1, dtype=torch.int64, device=index.device)
        at, b = torch.div(index, self.page_size, rounding_mode="floor").long(), seq.long()
        inside = (at >= 0) & (at < block_table.shape[1]) & (b >= 0) & (b < block_table.shape[0])
        page = block_table[b.clamp(0, block_table.shape[0] - 1), at.clamp(0, block_table.shape[1] - 1)].long()
        return torch.where(inside & (page >= 0) & (page < self.n_pages), page * self.page_size + index % self.page_size, -1)

    def _fields(self):
        """dark_paged_kv of layer 0, elements between layers."""
        e = self._k.stride()
        return _hip.PagedKV(k=self._k.data_ptr(), v=self._v.data_ptr(), page_stride=e[1], slot_stride=e[3], head_stride=e[2],
                            dtype=_DTYPES[self.dtype], n_pages=self.n_pages, page_size=self.page_size,
                            n_kv_heads=self.n_kv_heads, head_dim=self.head_dim), e[0]


def forward_cached(model, cache: PagedKVCache, input_ids: torch.Tensor, seq: torch.Tensor, index: torch.Tensor,
                   block_table: torch.Tensor, cu_q: torch.Tensor, kv_len: torch.Tensor, max_q: int, max_kv: int, *,
                   position_ids: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None, causal: bool = False,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The body of a ``DreamModel_length`` for new tokens (``input_ids [T]`` int64, token ``t`` = place ``index[t]`` of sequence
    ``seq[t]``, the tokens of a sequence together as ``cu_q`` says) against ``cache``: their keys and values are written to
    their slots, every new token attends over all ``kv_len`` keys of its sequence (``causal``: up to its own place).
    ``position_ids [T]`` default to ``index``.  Rows of tokens that no sequence holds (padding behind ``cu_q[-1]``, ``seq`` -1) are
    undefined and reach no other row.  Returns the residual stream ``[T, hidden_size]`` (``out`` if given) for the LM
    head."""
    pk = model.packed()
    dev = pk.device
    T, B = input_ids.shape[0], kv_len.shape[0]
    if not isinstance(cache, PagedKVCache) or cache.device != dev or cache.dtype != pk.dtype:
        raise ValueError("the cache is not on the model's device or not of its dtype")
    cfg = model.config
    if cache.n_layers < cfg.num_hidden_layers or cache.n_kv_heads != cfg.num_attention_heads or cache.head_dim != cfg.head_dim:
        raise ValueError("the cache is not the model's: layers, heads or head_dim differ")
    if position_ids is None and max_kv > pk.max_pos:
        raise ValueError(f"max_kv={max_kv} exceeds the rotation tables ({pk.max_pos} rows: max_position_embeddings)")
    i32 = torch.int32
    for name, t, dt, n in (("input_ids", input_ids, torch.int64, T), ("seq", seq, None, T), ("index", index, i32, T),
                           ("cu_q", cu_q, i32, B + 1), ("kv_len", kv_len, i32, B), ("position_ids", position_ids, i32, T)):
        if t is not None:
            _refuse(name, t, dev.index, dt, 1)
            _need(t.shape[0] == n and t.is_contiguous(), f"{name} must be contiguous with {n} elements")
    _refuse("block_table", block_table, dev.index, i32, 2)
    _need(block_table.shape[0] == B and block_table.is_contiguous(), f"block_table must be contiguous with {B} rows")
    if key_mask is not None:
        _refuse("key_mask", key_mask, dev.index, torch.uint8, 2)
        _need(key_mask.shape[0] == B and key_mask.shape[1] >= max_kv and key_mask.is_contiguous(),
              f"key_mask must be contiguous [{B}, >= {max_kv}] uint8")
    hidden = torch.empty((T, cfg.hidden_size), dtype=pk.resid_dtype, device=dev) if out is None else out
    _refuse("out", hidden, dev.index, pk.resid_dtype, 2)
    _need(tuple(hidden.shape) == (T, cfg.hidden_size) and hidden.is_contiguous(), f"out must be contiguous [{T}, {cfg.hidden_size}]")
    if T == 0:
        return hidden
    lib = _hip.load()
    kv, layer_stride = cache._fields()
    with torch.cuda.device(dev):
        slots = cache.slots(block_table, seq, index)
        attn = _hip.PagedAttentionArgs(
            kv=kv, block_table=block_table.data_ptr(), cu_q=cu_q.data_ptr(), kv_len=kv_len.data_ptr(),
            q_index=index.data_ptr() if causal else None, key_mask=_hip.ptr(key_mask), table_stride=block_table.shape[1],
            mask_stride=0 if key_mask is None else key_mask.shape[1], n_tokens=T, n_heads=cfg.num_attention_heads, n_seqs=B,
            table_width=block_table.shape[1], max_q=max_q, max_kv=max_kv, causal=int(bool(causal)), scale=cfg.head_dim ** -0.5)
        tokens = _hip.CachedTokens(ids=input_ids.data_ptr(), pos=(index if position_ids is None else position_ids).data_ptr(),
                                   slots=slots.data_ptr(), layer_stride=layer_stride, attn=attn)
        need = lib.dark_forward_cached_workspace_bytes(pk.ref, tokens)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _hip.check(lib.dark_forward_cached(pk.ref, tokens, ws.data_ptr(), need, hidden.data_ptr(), _hip.stream_ptr(dev)))
    for t in (cache._k, cache._v, hidden):     # (autograd refuses to go back through what it saved of them before)
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)
    return hidden


class WindowCache:
    """Cached denoise steps of one batch of windows ``[B, N]`` (``diffusion_generate(..., cache_interval=R)``).

    Every R-th forward is a whole one: all positions are new tokens, their keys and values fill the cache.  The forwards
    between compute only the positions that may have changed since or that a sampler may read: the ones masked at the last
    whole forward and their left neighbours (the logit shift, generation_utils.py:496).  The other positions' keys and values
    stay those of that forward -- an approximation for bidirectional attention (they would change with the tokens committed
    meanwhile), exact for R = 1."""

    PAGE = 16

    def __init__(self, model, B: int, N: int, pos: Optional[torch.Tensor], key_mask: Optional[torch.Tensor], interval: int) -> None:
        cfg, dev = model.config, model.device
        self.model, self.B, self.N, self.interval = model, B, N, interval
        per = -(-N // self.PAGE)
        self.cache = PagedKVCache(cfg.num_hidden_layers, B * per, self.PAGE, cfg.num_attention_heads, cfg.head_dim,
                                  model.packed().dtype, dev)
        i32 = torch.int32
        self.table = torch.arange(B * per, dtype=i32, device=dev).view(B, per)
        self.kv_len = torch.full((B,), N, dtype=i32, device=dev)
        self.all_cu = torch.arange(0, B * N + 1, N, dtype=i32, device=dev)
        self.all_seq = torch.arange(B, device=dev).repeat_interleave(N)
        self.all_index = torch.arange(N, dtype=i32, device=dev).repeat(B)
        self.pos = None if pos is None else pos.reshape(-1)
        self.key_mask = key_mask
        self.rows = None          # flat positions the forwards between compute; None: a whole one is due
        self.done = 0             # forwards since the last whole one
        self.min_masked = 0       # fewest masks a row holds

    def expire(self) -> None:
        """The windows changed in a way the cache does not know of: the next forward is a whole one."""
        self.rows = None

    def committed(self, k: int) -> None:
        """k positions of every row were committed.  A row with fewer masks than k gets positions re-masked that were not
        (generation_utils.py:531-534): they may lie outside the rows computed, so a whole forward is due."""
        if k > self.min_masked:
            self.expire()
        self.min_masked -= k

    def forward(self, st, x: torch.Tensor, mask_id: int) -> None:
        """Leaves the residual stream of every position a sampler may read in ``st.hidden``."""
        st.rows_valid = False
        if self.rows is None or self.done + 1 >= self.interval:
            forward_cached(self.model, self.cache, x.view(-1), self.all_seq, self.all_index, self.table, self.all_cu, self.kv_len,
                           self.N, self.N, position_ids=self.pos, key_mask=self.key_mask, out=st.hidden)
            self.done = 0
            if self.interval > 1:
                self._choose(x == mask_id)
            return
        self.done += 1
        if self.rows.shape[0] > 0:
            hidden = forward_cached(self.model, self.cache, x.view(-1)[self.rows], self.seq, self.index, self.table, self.cu,
                                    self.kv_len, self.max_q, self.N, position_ids=self.rows_pos, key_mask=self.key_mask)
            st.hidden.index_copy_(0, self.rows, hidden)

    def _choose(self, masked: torch.Tensor) -> None:
        act = masked.clone()
        act[:, :-1] |= masked[:, 1:]
        n = act.sum(1)
        self.rows = act.view(-1).nonzero().flatten()
        self.min_masked, self.max_q = torch.stack([masked.sum(1).min(), n.max()]).tolist()
        self.cu = torch.zeros(self.B + 1, dtype=torch.int32, device=masked.device)
        self.cu[1:] = n.cumsum(0)
        self.seq, self.index = self.all_seq[self.rows], self.all_index[self.rows].contiguous()
        self.rows_pos = None if self.pos is None else self.pos[self.rows].contiguous()
