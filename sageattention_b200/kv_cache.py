"""Serving from a key/value cache held in 4 bits: what a server that generates tokens needs round :func:`sageattn_kvcache`.

A step of such a server, for requests that add one token or many:

    t = build_block_tables(lens, new_lens, block_table, free_pages, cache.page_size, num_tokens=T)
    q = qk_norm_rope_append(q, k, v, cache, t.slots, cos, sin, t.positions, q_weight=..., k_weight=...)
    o = sageattn_kvcache(q, cache, block_table, t.kv_lens, t.cu_seqlens_q, max_seqlen_q=..., max_seqlen_k=...)

Everything runs on the current stream of the tensors' device without synchronising, allocates through PyTorch and can be
captured into a CUDA graph.  The reference has no counterpart: its operators keep nothing between calls.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from .api import _as_bhnd_strides, _check_device, _on_device, _stream_ptr, _tensor_arg

_PAGE_SIZES = (16, 32, 64, 128)


def _require(cond, msg):
    if not cond:
        raise ValueError(msg)


def _check_bf16(*tensors):
    for t in tensors:
        if t.dtype != torch.bfloat16:
            raise AssertionError("TODO: support inputs other than bfloat16")     # as the other operators
        _require(t.stride(-1) == 1 or t.shape[-1] == 1, "the last dimension must be contiguous")


def _check_rows(*tensors):
    """16-byte vectors: aligned start, strides of whole vectors."""
    for t in tensors:
        _require(t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1),
                 "every row must start on a 16-byte boundary")


def _check_ids(name, t, dtype, shape, device):
    _require(t.dtype == dtype, f"{name} must be {dtype}")
    _require(tuple(t.shape) == tuple(shape), f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    _require(t.device == device, f"{name} must be on {device}")
    _require(t.is_contiguous(), f"{name} must be contiguous")


def _stored_dim(head_dim: int) -> int:
    return 64 if head_dim <= 64 else 128


class FP4KVCache:
    """Keys and values of one layer in pages of ``page_size`` tokens, in NVFP4: E2M1 codes with an E4M3 scale per 16 channels, 4.5 bits a
    value.

    ``data``: uint8 ``[num_pages, num_kv_heads, page_bytes]``, contiguous, on the GPU (:meth:`empty` allocates it; what is in it does not
    matter, since what was not written is never used).  A page can be copied, moved and shared as ``data[page]``.  Head dims up to
    128 that are a multiple of 8; they are stored as 64 or 128 channels.

    ``k_offset`` (optional bf16 ``[num_kv_heads, head_dim]``): keys are stored less this vector - the channel means of the layer's keys,
    calibrated beforehand, take the place of K smoothing (``sageattn4/api.py:184``), which would need all keys at once.  Softmax does
    not see it; :func:`sageattn_kvcache` puts it back into the log-sum-exp, :meth:`read` into the keys."""

    __slots__ = ("data", "num_pages", "num_kv_heads", "page_size", "head_dim", "k_offset", "device", "_struct", "_ref")

    def __init__(self, data: torch.Tensor, head_dim: int, page_size: int = 64, k_offset: Optional[torch.Tensor] = None):
        _require(page_size in _PAGE_SIZES, f"page_size must be one of {_PAGE_SIZES}")
        _require(0 < head_dim <= 128 and head_dim % 8 == 0, f"Unsupported head_dim: {head_dim} (a multiple of 8, at most 128)")
        _require(data.dtype == torch.uint8 and data.dim() == 3 and data.is_contiguous(), "data must be a contiguous uint8 tensor [num_pages, num_kv_heads, page_bytes]")
        pages, heads, nbytes = data.shape
        _require(nbytes == self.page_bytes(head_dim, page_size), f"pages of {page_size} tokens of head_dim {head_dim} take {self.page_bytes(head_dim, page_size)} bytes, not {nbytes}")
        _require(pages > 0 and heads > 0, "the cache must have pages and heads")
        _require(data.data_ptr() % 16 == 0, "data must start on a 16-byte boundary")
        if k_offset is not None:
            _check_bf16(k_offset)
            _check_ids("k_offset", k_offset, torch.bfloat16, (heads, head_dim), data.device)
            _require(k_offset.data_ptr() % 16 == 0, "k_offset must start on a 16-byte boundary")
        self.data, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim, self.k_offset = data, pages, heads, page_size, head_dim, k_offset
        self.device = data.device
        self._struct = _lib.KvCache(data.data_ptr(), pages, heads, page_size, head_dim, _stored_dim(head_dim),
                                    None if k_offset is None else k_offset.data_ptr())
        self._ref = C.pointer(self._struct)

    @staticmethod
    def page_bytes(head_dim: int, page_size: int) -> int:
        """Bytes of a page of one kv head: 9/16 per stored channel of a key and of a value."""
        return page_size * _stored_dim(head_dim) * 18 // 16

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, device="cuda",
              k_offset: Optional[torch.Tensor] = None) -> "FP4KVCache":
        _require(page_size in _PAGE_SIZES, f"page_size must be one of {_PAGE_SIZES}")
        _require(0 < head_dim <= 128 and head_dim % 8 == 0, f"Unsupported head_dim: {head_dim} (a multiple of 8, at most 128)")
        data = torch.empty((num_pages, num_kv_heads, cls.page_bytes(head_dim, page_size)), dtype=torch.uint8, device=device)
        return cls(data, head_dim, page_size, k_offset)

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Writes k, v (bf16 ``[T, num_kv_heads, head_dim]``) to the slots (int64 ``[T]``) ``page * page_size + place``.  Slots outside the cache
        (-1) are skipped; a slot named twice ends up with a mixture of its tokens."""
        T = self._check_tokens(k, v, slots)
        if T == 0:
            return
        a = _lib.KvTokensArgs()
        a.B, a.N, a.Hq, a.Hkv, a.D = 1, T, 0, self.num_kv_heads, self.head_dim
        a.k = _lib.Tensor(k.data_ptr(), 0, k.stride(1), k.stride(0))
        a.v = _lib.Tensor(v.data_ptr(), 0, v.stride(1), v.stride(0))
        a.cache, a.slots = self._ref, slots.data_ptr()
        with _on_device(self.device):
            _lib.check(_lib.load().sage3_kv_tokens(C.byref(a), _stream_ptr(self.device)), "sage3_kv_tokens")

    def read(self, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """The keys (with their offset) and values that the slots (int64 ``[T]``) stand for, bf16 ``[T, num_kv_heads, head_dim]``: for attention
        in higher precision over part of the cache, or to move tokens elsewhere.  Slots outside the cache give zeros."""
        _require(slots.dim() == 1, "slots must be [tokens]")
        _check_ids("slots", slots, torch.int64, slots.shape, self.device)
        _check_device(self.data)
        shape = (slots.shape[0], self.num_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        v = torch.empty(shape, dtype=torch.bfloat16, device=self.device)
        with _on_device(self.device):
            _lib.check(_lib.load().sage3_kv_read(self._ref, slots.data_ptr(), shape[0], k.data_ptr(), v.data_ptr(), _stream_ptr(self.device)), "sage3_kv_read")
        return k, v

    def _check_tokens(self, k, v, slots):
        _check_bf16(k, v)
        _require(k.dim() == 3 and k.shape == v.shape and k.shape[1:] == (self.num_kv_heads, self.head_dim),
                 f"k and v must be [tokens, {self.num_kv_heads}, {self.head_dim}]")
        _require(k.device == v.device == self.device, "k, v and the cache must be on one device")
        _check_ids("slots", slots, torch.int64, (k.shape[0],), self.device)
        _check_rows(k, v)
        _check_device(self.data)
        return k.shape[0]


@dataclass
class BlockTables:
    """What :func:`build_block_tables` gives: ``kv_lens`` int32 [B] (lengths after the step), ``cu_seqlens_q`` int32 [B+1], ``positions`` int32
    [num_tokens], ``slots`` int64 [num_tokens], ``pages_taken`` int32 [1]."""
    kv_lens: torch.Tensor
    cu_seqlens_q: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    pages_taken: torch.Tensor


def build_block_tables(lens_before: torch.Tensor, lens_new: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                       page_size: int, num_tokens: int) -> BlockTables:
    """Pages, positions and slots of a step, in one launch.

    ``lens_before``, ``lens_new``: int32 ``[B]`` (B <= 16384), the tokens that each request has in the cache and those that it adds.
    ``block_table``: int32 ``[B, columns]``, updated in place: entry j of a request is the page of its tokens ``j * page_size ...``; entries
    of pages that the step begins are taken from the front of ``free_pages`` (int32 ``[F]``), request by request.  ``num_tokens``: how many
    entries ``positions`` and ``slots`` get, the sum of ``lens_new`` or more (a padded batch); behind the last token slots are -1 and
    positions 0.  Nothing is read back: where the free pages or the columns do not suffice, table entries and slots are -1, and
    ``pages_taken`` says how many pages the step wanted."""
    _require(lens_before.dim() == 1 and lens_before.shape[0] > 0, "lens_before must be [requests]")
    B, dev = lens_before.shape[0], lens_before.device
    _require(B <= 16384, "at most 16384 requests")
    _require(page_size in _PAGE_SIZES, f"page_size must be one of {_PAGE_SIZES}")
    _require(0 <= num_tokens < 2 ** 31, "num_tokens must be a count")
    _check_ids("lens_before", lens_before, torch.int32, (B,), dev)
    _check_ids("lens_new", lens_new, torch.int32, (B,), dev)
    _require(free_pages.dim() == 1, "free_pages must be [pages]")
    _check_ids("free_pages", free_pages, torch.int32, free_pages.shape, dev)
    _check_table(block_table, B, dev)
    _check_device(lens_before)
    n = int(num_tokens)
    # one allocation for all of int32
    ints = torch.empty(2 * B + 2 + n, dtype=torch.int32, device=dev)
    kv_lens, cu, taken, positions = ints.split((B, B + 1, 1, n))
    slots = torch.empty(n, dtype=torch.int64, device=dev)
    a = _lib.KvTablesArgs(lens_before.data_ptr(), lens_new.data_ptr(), free_pages.data_ptr(), block_table.data_ptr(), block_table.stride(0), B,
                          block_table.shape[1], free_pages.shape[0], page_size, n, kv_lens.data_ptr(), cu.data_ptr(), positions.data_ptr(),
                          slots.data_ptr(), taken.data_ptr())
    with _on_device(dev):
        _lib.check(_lib.load().sage3_kv_block_tables(C.byref(a), _stream_ptr(dev)), "sage3_kv_block_tables")
    return BlockTables(kv_lens, cu, positions, slots, taken)


def _check_table(t, B, dev):
    _require(t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == B and t.shape[1] > 0, f"block_table must be int32 [{B}, columns]")
    _require(t.device == dev, f"block_table must be on {dev}")
    _require(t.stride(1) == 1 or t.shape[1] == 1, "the rows of block_table must be contiguous")
    _require(B == 1 or t.stride(0) >= t.shape[1], "the rows of block_table must not overlap")


def _norm_rope_args(q, k, cos, sin, positions, q_weight, k_weight, eps, adjacent_pairs, tensor_layout):
    """The argument struct of sage3_kv_tokens but for outputs and cache."""
    _check_bf16(q, k)
    _require(q.dim() == k.dim() and q.dim() in (3, 4), "q and k must be [tokens, heads, head_dim], or 4-D in tensor_layout")
    if q.dim() == 3:
        (N, Hq, D), (Nk, Hkv, Dk), B, Bk = q.shape, k.shape, 1, 1
        qs, ks = (0, q.stride(1), q.stride(0)), (0, k.stride(1), k.stride(0))
        where = (N,)
    else:
        B, Hq, N, D, *qs = _as_bhnd_strides(q, tensor_layout)
        Bk, Hkv, Nk, Dk, *ks = _as_bhnd_strides(k, tensor_layout)
        where = (B, N)
    _require((B, N, D) == (Bk, Nk, Dk), "q and k shapes do not match")
    _require(Hkv > 0, "k must have heads")
    _require(0 < D <= 128 and D % 8 == 0, f"Unsupported head_dim: {D} (a multiple of 8, at most 128)")
    _require(q.device == k.device, "q and k must be on one device")
    _check_rows(q, k)
    a = _lib.KvTokensArgs()
    a.B, a.N, a.Hq, a.Hkv, a.D = B, N, Hq, Hkv, D
    a.q, a.k = _lib.Tensor(q.data_ptr(), *qs), _lib.Tensor(k.data_ptr(), *ks)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _check_ids(name, w, torch.bfloat16, (D,), q.device)
            _require(w.data_ptr() % 16 == 0, f"{name} must start on a 16-byte boundary")
            setattr(a, name, w.data_ptr())
    _require(eps >= 0, "eps must not be negative")
    a.eps = float(eps)
    _require((cos is None) == (sin is None), "cos and sin go together")
    if cos is not None:
        _require(cos.dim() == 2 and cos.shape[0] > 0, "cos and sin must be [positions, rot_dim / 2]")
        rot = 2 * cos.shape[1]
        _require(0 < rot <= D and rot % 8 == 0, f"the rotated channels must be a multiple of 8, at most head_dim: {rot}")
        _check_ids("cos", cos, torch.float32, cos.shape, q.device)
        _check_ids("sin", sin, torch.float32, cos.shape, q.device)
        _require(cos.data_ptr() % 16 == 0 and sin.data_ptr() % 16 == 0, "cos and sin must start on a 16-byte boundary")
        a.cos, a.sin, a.places, a.rot_dim, a.adjacent_pairs = cos.data_ptr(), sin.data_ptr(), cos.shape[0], rot, int(bool(adjacent_pairs))
        if positions is not None:
            _require(positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64")
            _check_ids("positions", positions, positions.dtype, where, q.device)
            a.positions, a.positions_int64 = positions.data_ptr(), int(positions.dtype == torch.int64)
    _check_device(q)
    return a


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, adjacent_pairs: bool = False,
                 tensor_layout: str = "NHD", out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """Per-head RMS norm of queries and keys and the rotation by their positions, in one pass.

    q, k: bf16, ``[tokens, heads, head_dim]`` or 4-D in ``tensor_layout`` ("NHD" / "HND"), any strides over whole 16-byte vectors (a slice of
    a fused projection); head_dim a multiple of 8 up to 128.  ``q_weight``, ``k_weight`` (bf16 ``[head_dim]``): ``x * rsqrt(mean(x^2) + eps) *
    weight``, or no norm where None.  ``cos``, ``sin`` (fp32 ``[positions, rot_dim / 2]``): the first ``rot_dim`` channels are rotated, pairs being
    ``(i, i + rot_dim / 2)``, or ``(2i, 2i + 1)`` with ``adjacent_pairs``.  ``positions``: int32 or int64 ``[tokens]`` (``[batch, tokens]``), default
    0, 1, ... in each batch entry; one outside the table gives NaN.  All in fp32, rounded once.  ``out``: the two outputs, which may be q and
    k themselves."""
    a = _norm_rope_args(q, k, cos, sin, positions, q_weight, k_weight, eps, adjacent_pairs, tensor_layout)
    if out is None:
        out = torch.empty_like(q), torch.empty_like(k)
    for o, x, name in zip(out, (q, k), ("q_out", "k_out")):
        _check_bf16(o)
        _require(o.shape == x.shape and o.device == x.device, "outputs must have the shapes and device of q and k")
        _check_rows(o)
        s = (0, o.stride(1), o.stride(0)) if o.dim() == 3 else _as_bhnd_strides(o, tensor_layout)[4:]
        setattr(a, name, _lib.Tensor(o.data_ptr(), *s))
    if q.shape[0] and a.N:
        with _on_device(q.device):
            _lib.check(_lib.load().sage3_kv_tokens(C.byref(a), _stream_ptr(q.device)), "sage3_kv_tokens")
    return out[0], out[1]


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: FP4KVCache, slots: torch.Tensor,
                        cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                        positions: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, adjacent_pairs: bool = False,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`qk_norm_rope` of ``[tokens, heads, head_dim]`` tensors with the keys, and the values as they are, written straight to the cache
    (the same bits as :meth:`FP4KVCache.append` of its result).  Returns the queries."""
    _require(q.dim() == 3, "q must be [tokens, heads, head_dim]")
    a = _norm_rope_args(q, k, cos, sin, positions, q_weight, k_weight, eps, adjacent_pairs, "NHD")
    cache._check_tokens(k, v, slots)
    _require(q.device == cache.device, "q and the cache must be on one device")
    if out is None:
        out = torch.empty_like(q)
    _check_bf16(out)
    _require(out.shape == q.shape and out.device == q.device, "out must have the shape and device of q")
    _check_rows(out)
    a.q_out = _lib.Tensor(out.data_ptr(), 0, out.stride(1), out.stride(0))
    a.v = _lib.Tensor(v.data_ptr(), 0, v.stride(1), v.stride(0))
    a.cache, a.slots = cache._ref, slots.data_ptr()
    if a.N:
        with _on_device(q.device):
            _lib.check(_lib.load().sage3_kv_tokens(C.byref(a), _stream_ptr(q.device)), "sage3_kv_tokens")
    return out


def sageattn_kvcache(q: torch.Tensor, cache: FP4KVCache, block_table: torch.Tensor, kv_lens: torch.Tensor,
                     cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: int = 1, max_seqlen_k: Optional[int] = None,
                     is_causal: bool = True, sm_scale: Optional[float] = None, return_lse: bool = False,
                     out: Optional[torch.Tensor] = None):
    """Attention of new tokens over the 4-bit cache, their own keys (already appended) among the last ones.

    q: bf16 ``[tokens, Hq, head_dim]``, ``Hq`` a multiple of the cache's heads; sequence i has rows ``cu_seqlens_q[i] ... cu_seqlens_q[i+1]`` (int32
    ``[B+1]``), or row i alone where ``cu_seqlens_q`` is None.  ``kv_lens`` int32 ``[B]``: keys of each sequence, new ones included;
    ``block_table`` int32 ``[B, columns]``: their pages.  ``max_seqlen_q`` and ``max_seqlen_k`` (default: what the table can hold) must bound the
    lengths - they size grid and workspace; rows and keys beyond them are left out.  ``is_causal``: bottom-right aligned, the last row of
    a sequence sees all of its keys.

    Attention is over the values that the cache stands for, queries and softmax are not quantised.  Rows that see no key give zeros and an
    LSE of ``-inf``; keys of pages outside the cache (-1) are not seen; rows of q that belong to no sequence (a padded batch) are not
    touched in ``out`` (or are undefined in a new tensor).  Returns the output like q, and with ``return_lse`` the natural-log LSE fp32
    ``[tokens, Hq]`` of ``sm_scale * q.k``."""
    _check_bf16(q)
    _require(q.dim() == 3 and q.shape[2] == cache.head_dim, f"q must be [tokens, heads, {cache.head_dim}]")
    T, Hq, _ = q.shape
    _require(Hq > 0 and Hq % cache.num_kv_heads == 0, "num_qo_heads must be a multiple of num_kv_heads")
    dev = q.device
    _require(dev == cache.device, "q and the cache must be on one device")
    _require(kv_lens.dim() == 1 and kv_lens.shape[0] > 0, "kv_lens must be [sequences]")
    B = kv_lens.shape[0]
    _check_ids("kv_lens", kv_lens, torch.int32, (B,), dev)
    if cu_seqlens_q is not None:
        _check_ids("cu_seqlens_q", cu_seqlens_q, torch.int32, (B + 1,), dev)
        _require(max_seqlen_q > 0, "max_seqlen_q must be positive")
    else:
        _require(T >= B, "without cu_seqlens_q, q must have a row for each sequence")
        max_seqlen_q = 1
    _check_table(block_table, B, dev)
    room = block_table.shape[1] * cache.page_size
    max_seqlen_k = room if max_seqlen_k is None else min(int(max_seqlen_k), room)
    _require(max_seqlen_k > 0, "max_seqlen_k must be positive")
    _require(sm_scale is None or sm_scale > 0, "sm_scale must be positive")
    _check_rows(q)
    if out is None:
        out = torch.empty_like(q)
    _check_bf16(out)
    _require(out.shape == q.shape and out.device == dev, "out must have the shape and device of q")
    _check_rows(out)
    _check_device(q)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if T:
        lib = _lib.load()
        a = _lib.KvAttentionArgs(cache._ref, B, Hq, int(max_seqlen_q), int(max_seqlen_k), T, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(),
                                 out.stride(0), out.stride(1), None if lse is None else lse.data_ptr(),
                                 None if cu_seqlens_q is None else cu_seqlens_q.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(),
                                 block_table.stride(0), block_table.shape[1], int(bool(is_causal)), 0.0 if sm_scale is None else float(sm_scale))
        with _on_device(dev):
            n = C.c_size_t()
            _lib.check(lib.sage3_kv_attention_workspace(C.byref(a), C.byref(n)), "sage3_kv_attention_workspace")
            ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
            _lib.check(lib.sage3_kv_attention(C.byref(a), _stream_ptr(dev)), "sage3_kv_attention")
    return (out, lse) if return_lse else out
