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
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .api import _as_bhnd_strides, _check_device, _keep_plan, _on_device, _plans, _stream_ptr

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
    """16-byte vectors: strides of whole vectors (and an aligned start, which _check_aligned looks at in every call)."""
    for t in tensors:
        _require(all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1), "every row must start on a 16-byte boundary")


def _check_aligned(pointers, what):
    if pointers & 15:
        raise ValueError(f"{what} must start on a 16-byte boundary")


# What a call with given sizes and options needs is worked out once, as for the other operators (api.py): the checks and the argument struct
# but for its pointers.  A call looks its plan up by these, copies the struct and fills the pointers in.  Tensors of which only one
# shape, type and layout will do are not part of what a plan is found by, but looked at (_is) in every call; where one is not as it should
# be, the checks of the plan are run again to say so.  (Looking a tensor up costs 1.1 us, looking at it 0.45.)
class _Plan:
    __slots__ = ("device", "struct", "workspace", "rows", "where")


def _is(t, dtype, shape, device):
    return t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous()


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _check_ids(name, t, dtype, shape, device):
    _require(t.dtype == dtype, f"{name} must be {dtype}")
    _require(tuple(t.shape) == tuple(shape), f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    _require(t.device == device, f"{name} must be on {device}")
    _require(t.is_contiguous(), f"{name} must be contiguous")


def _stored_dim(head_dim: int) -> int:
    return 64 if head_dim <= 64 else 128


_b200 = set()


def _check_b200(device, tensor):
    """_check_device, asked once per device."""
    if device not in _b200:
        _check_device(tensor)
        _b200.add(device)


def _strides(x):
    """(stride_h, stride_n) of [tokens, heads, head_dim]; where there is but one, its stride says nothing"""
    n, h, _ = x.shape
    return x.stride(1) if h != 1 else 0, x.stride(0) if n != 1 else 0


def _strides4(x, tensor_layout):
    """(stride_b, stride_h, stride_n), likewise"""
    B, H, N, _, *strides = _as_bhnd_strides(x, tensor_layout)
    return [s if n != 1 else 0 for s, n in zip(strides, (B, H, N))]


def _check_numbers(**numbers):
    """A plan is found by these: a tensor would be found by its identity, whatever it has come to hold."""
    for name, x in numbers.items():
        _require(not isinstance(x, torch.Tensor), f"{name} must be a number, not a tensor")


def _run(fn, struct, device, where):
    if device.index == _current_device():           # (a tensor is on it, so CUDA is up)
        st = fn(C.byref(struct), _stream_ptr(device))
    else:
        with torch.cuda.device(device):
            st = fn(C.byref(struct), _stream_ptr(device))
    if st:
        _lib.check(st, where)


class FP4KVCache:
    """Keys and values of one layer in pages of ``page_size`` tokens, in NVFP4: E2M1 codes with an E4M3 scale per 16 channels, 4.5 bits a
    value.

    ``data``: uint8 ``[num_pages, num_kv_heads, page_bytes]``, contiguous, on the GPU (:meth:`empty` allocates it; what is in it does not
    matter, since what was not written is never used).  A page can be copied, moved and shared as ``data[page]``.  Head dims up to
    128 that are a multiple of 8; they are stored as 64 or 128 channels.

    ``k_offset`` (optional bf16 ``[num_kv_heads, head_dim]``): keys are stored less this vector - the channel means of the layer's keys,
    calibrated beforehand, take the place of K smoothing (``sageattn4/api.py:184``), which would need all keys at once.  Softmax does
    not see it; :func:`sageattn_kvcache` puts it back into the log-sum-exp, :meth:`read` into the keys."""

    __slots__ = ("_data", "num_pages", "num_kv_heads", "page_size", "head_dim", "_k_offset", "device", "_key", "_struct", "_ref")

    data = property(lambda self: self._data)                         # (the struct has their pointers: not to be exchanged)
    k_offset = property(lambda self: self._k_offset)

    def __init__(self, data: torch.Tensor, head_dim: int, page_size: int = 64, k_offset: Optional[torch.Tensor] = None):
        if page_size not in _PAGE_SIZES:
            raise ValueError(f"page_size must be one of {_PAGE_SIZES}")
        if not (0 < head_dim <= 128 and head_dim % 8 == 0):
            raise ValueError(f"Unsupported head_dim: {head_dim} (a multiple of 8, at most 128)")
        if data.dtype != torch.uint8 or data.dim() != 3 or not data.is_contiguous():
            raise ValueError("data must be a contiguous uint8 tensor [num_pages, num_kv_heads, page_bytes]")
        pages, heads, nbytes = data.shape
        if nbytes != self.page_bytes(head_dim, page_size):
            raise ValueError(f"pages of {page_size} tokens of head_dim {head_dim} take {self.page_bytes(head_dim, page_size)} bytes, not {nbytes}")
        if pages == 0 or heads == 0:
            raise ValueError("the cache must have pages and heads")
        pointer, device, offset = data.data_ptr(), data.device, None
        if k_offset is not None:
            if k_offset.dtype != torch.bfloat16 or k_offset.shape != (heads, head_dim) or k_offset.device != device or not k_offset.is_contiguous():
                raise ValueError(f"k_offset must be a contiguous bfloat16 tensor [{heads}, {head_dim}] on the device of data")
            offset = k_offset.data_ptr()
        if (pointer | (offset or 0)) & 15:
            raise ValueError("data and k_offset must start on a 16-byte boundary")
        self._data, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim, self._k_offset = data, pages, heads, page_size, head_dim, k_offset
        self.device = device
        self._key = (pages, heads, head_dim, page_size, device, offset is None)
        self._struct = _lib.KvCache(pointer, pages, heads, page_size, head_dim, 64 if head_dim <= 64 else 128, offset)
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
        (-1) are skipped; a slot named twice ends up with a mixture of its tokens.  A NaN makes its block of 16 channels NaN, infinities become
        the block's largest number."""
        key = ("kv_append", _sig(k), _sig(v), self._key)
        plan = _plans.get(key)
        if plan is None or not _is(slots, torch.int64, plan.rows, self.device):
            T = self._check_tokens(k, v, slots)
            plan = _Plan()
            a = plan.struct = _lib.KvTokensArgs()
            a.B, a.N, a.Hq, a.Hkv, a.D = 1, T, 0, self.num_kv_heads, self.head_dim
            a.k, a.v = _lib.Tensor(None, 0, *_strides(k)), _lib.Tensor(None, 0, *_strides(v))
            plan.rows = k.shape[:1]
            _keep_plan(key, plan)
        kp, vp = k.data_ptr(), v.data_ptr()
        _check_aligned(kp | vp, "k and v")
        a = _lib.KvTokensArgs.from_buffer_copy(plan.struct)
        a.k.ptr, a.v.ptr, a.cache, a.slots = kp, vp, self._ref, slots.data_ptr()
        if a.N:
            _run(_lib.load().sage3_kv_tokens, a, self.device, "sage3_kv_tokens")

    def read(self, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """The keys (with their offset) and values that the slots (int64 ``[T]``) stand for, bf16 ``[T, num_kv_heads, head_dim]``: for attention
        in higher precision over part of the cache, or to move tokens elsewhere.  Slots outside the cache give zeros."""
        T = slots.shape[0] if slots.dim() == 1 else -1
        if T < 0 or slots.dtype != torch.int64 or slots.device != self.device or not slots.is_contiguous():
            _require(T >= 0, "slots must be [tokens]")
            _check_ids("slots", slots, torch.int64, slots.shape, self.device)
        _require(T < 2 ** 31 - 64, "too many tokens for one call")
        dev = self.device
        _check_b200(dev, self.data)
        k = torch.empty((T, self.num_kv_heads, self.head_dim), dtype=torch.bfloat16, device=dev)
        v = torch.empty_like(k)
        with _on_device(dev):
            st = _lib.load().sage3_kv_read(self._ref, slots.data_ptr(), T, k.data_ptr(), v.data_ptr(), _stream_ptr(dev))
        if st:
            _lib.check(st, "sage3_kv_read")
        return k, v

    def _check_tokens(self, k, v, slots):
        _check_bf16(k, v)
        _require(k.dim() == 3 and k.shape == v.shape and k.shape[1:] == (self.num_kv_heads, self.head_dim),
                 f"k and v must be [tokens, {self.num_kv_heads}, {self.head_dim}]")
        _require(k.shape[0] < 2 ** 31 - 64, "too many tokens for one call")
        _require(k.device == v.device == self.device, "k, v and the cache must be on one device")
        _check_ids("slots", slots, torch.int64, (k.shape[0],), self.device)
        _check_rows(k, v)
        _check_device(self.data)
        return k.shape[0]


class BlockTables(NamedTuple):
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
    positions 0.  Sums of lengths stop at 2^31 - 1.  Nothing is read back: where the free pages or the columns do not suffice, table entries and slots are -1, and
    ``pages_taken`` says how many pages the step wanted."""
    # (the free pages and the tokens are other ones in every step: not part of the key)
    key = ("kv_tables", _sig(lens_before), block_table.shape, block_table.stride(), page_size)
    plan = _plans.get(key)
    if (plan is None or not _is(lens_new, torch.int32, plan.where, plan.device) or not _is(free_pages, torch.int32, free_pages.shape, plan.device) or
            free_pages.dim() != 1 or block_table.dtype is not torch.int32 or block_table.device != plan.device or
            type(num_tokens) is not int or not 0 <= num_tokens < 2 ** 31 or free_pages.shape[0] >= 2 ** 31):
        plan = _keep_plan(key, _plan_tables(lens_before, lens_new, block_table, free_pages, page_size, num_tokens))
    dev, a = plan.device, _lib.KvTablesArgs.from_buffer_copy(plan.struct)
    B, n = a.B, int(num_tokens)
    a.num_free, a.num_tokens = free_pages.shape[0], n
    # one allocation for all of int32
    ints = lens_new.new_empty(2 * B + 2 + n)
    kv_lens, cu, taken, positions = torch.split_with_sizes(ints, (B, B + 1, 1, n))
    slots = lens_new.new_empty(n, dtype=torch.int64)
    p = ints.data_ptr()
    a.lens_before, a.lens_new, a.free_pages, a.block_table = lens_before.data_ptr(), lens_new.data_ptr(), free_pages.data_ptr(), block_table.data_ptr()
    a.kv_lens, a.cu_seqlens_q, a.pages_taken, a.positions, a.slots = p, p + 4 * B, p + 8 * B + 4, p + 8 * B + 8, slots.data_ptr()
    _run(_lib.load().sage3_kv_block_tables, a, dev, "sage3_kv_block_tables")
    return BlockTables(kv_lens, cu, positions, slots, taken)


def _plan_tables(lens_before, lens_new, block_table, free_pages, page_size, num_tokens) -> _Plan:
    _check_numbers(page_size=page_size, num_tokens=num_tokens)
    _require(lens_before.dim() == 1 and lens_before.shape[0] > 0, "lens_before must be [requests]")
    B, dev = lens_before.shape[0], lens_before.device
    _require(B <= 16384, "at most 16384 requests")
    _require(page_size in _PAGE_SIZES, f"page_size must be one of {_PAGE_SIZES}")
    _require(0 <= num_tokens < 2 ** 31, "num_tokens must be a count")
    _check_ids("lens_before", lens_before, torch.int32, (B,), dev)
    _check_ids("lens_new", lens_new, torch.int32, (B,), dev)
    _require(free_pages.dim() == 1 and free_pages.shape[0] < 2 ** 31, "free_pages must be [pages]")
    _check_ids("free_pages", free_pages, torch.int32, free_pages.shape, dev)
    _check_table(block_table, B, dev)
    _check_device(lens_before)
    plan = _Plan()
    plan.device, plan.where = dev, lens_before.shape
    a = plan.struct = _lib.KvTablesArgs()
    a.row_stride, a.B, a.columns, a.page_size = max(block_table.stride(0), block_table.shape[1]), B, block_table.shape[1], page_size
    return plan


def _check_table(t, B, dev):
    _require(t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == B and 0 < t.shape[1] < 2 ** 31, f"block_table must be int32 [{B}, columns]")
    _require(t.device == dev, f"block_table must be on {dev}")
    _require(t.stride(1) == 1 or t.shape[1] == 1, "the rows of block_table must be contiguous")
    _require(B == 1 or t.stride(0) >= t.shape[1], "the rows of block_table must not overlap")


def _sig(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _norm_rope_plan(q, k, cos, sin, positions, q_weight, k_weight, eps, adjacent_pairs, tensor_layout) -> _Plan:
    """Checks, and the argument struct of sage3_kv_tokens but for pointers, outputs and cache."""
    _check_numbers(eps=eps, adjacent_pairs=adjacent_pairs)
    _check_bf16(q, k)
    _require(q.dim() == k.dim() and q.dim() in (3, 4), "q and k must be [tokens, heads, head_dim], or 4-D in tensor_layout")
    if q.dim() == 3:
        (N, Hq, D), (Nk, Hkv, Dk), B, Bk = q.shape, k.shape, 1, 1
        qs, ks = (0, *_strides(q)), (0, *_strides(k))
        where = (N,)
    else:
        B, Hq, N, D = _as_bhnd_strides(q, tensor_layout)[:4]
        Bk, Hkv, Nk, Dk = _as_bhnd_strides(k, tensor_layout)[:4]
        qs, ks = _strides4(q, tensor_layout), _strides4(k, tensor_layout)
        where = (B, N)
    _require((B, N, D) == (Bk, Nk, Dk), "q and k shapes do not match")
    _require(Hkv > 0, "k must have heads")
    _require(B * N < 2 ** 31 - 64, "too many tokens for one call")
    _require(0 < D <= 128 and D % 8 == 0, f"Unsupported head_dim: {D} (a multiple of 8, at most 128)")
    _require(q.device == k.device, "q and k must be on one device")
    _check_rows(q, k)
    plan = _Plan()
    plan.device, plan.where, plan.rows = q.device, torch.Size(where), torch.Size((D,))
    a = plan.struct = _lib.KvTokensArgs()
    a.B, a.N, a.Hq, a.Hkv, a.D = B, N, Hq, Hkv, D
    a.q, a.k = _lib.Tensor(None, *qs), _lib.Tensor(None, *ks)
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _check_ids(name, w, torch.bfloat16, (D,), q.device)
    _require(eps >= 0, "eps must not be negative")
    a.eps = float(eps)
    _require((cos is None) == (sin is None), "cos and sin go together")
    if cos is not None:
        _require(cos.dim() == 2 and cos.shape[0] > 0, "cos and sin must be [positions, rot_dim / 2]")
        rot = 2 * cos.shape[1]
        _require(0 < rot <= D and rot % 8 == 0, f"the rotated channels must be a multiple of 8, at most head_dim: {rot}")
        _check_ids("cos", cos, torch.float32, cos.shape, q.device)
        _check_ids("sin", sin, torch.float32, cos.shape, q.device)
        a.places, a.rot_dim, a.adjacent_pairs = cos.shape[0], rot, int(bool(adjacent_pairs))
        if positions is not None:
            _require(positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64")
            _check_ids("positions", positions, positions.dtype, where, q.device)
            a.positions_int64 = int(positions.dtype == torch.int64)
    _check_device(q)
    for x, name in ((q, "q_out"), (k, "k_out")):
        y = _rows(torch.empty_like(x, device="meta"), tensor_layout)
        y.ptr = None
        setattr(a, name, y)
    return plan


def _rows(x, tensor_layout):
    if x.dim() == 3:
        return _lib.Tensor(x.data_ptr(), 0, *_strides(x))
    return _lib.Tensor(x.data_ptr(), *_strides4(x, tensor_layout))


def _norm_rope_key(name, q, k, cos, positions, q_weight, k_weight, eps, adjacent_pairs, tensor_layout, *more):
    return (name, q.shape, q.stride(), q.dtype, q.device, k.shape, k.stride(), k.dtype, k.device, None if cos is None else cos.shape,
            None if cos is None or positions is None else positions.dtype, q_weight is None, k_weight is None, eps, adjacent_pairs, tensor_layout, more)


def _norm_rope_fits(plan, cos, sin, positions, q_weight, k_weight):
    """Whether the tensors that a plan is not found by are as it has them."""
    dev = plan.device
    if cos is None:
        if sin is not None:
            return False
    elif sin is None or not _is(cos, torch.float32, cos.shape, dev) or not _is(sin, torch.float32, cos.shape, dev):
        return False
    elif positions is not None and not _is(positions, positions.dtype, plan.where, dev):
        return False
    return ((q_weight is None or _is(q_weight, torch.bfloat16, plan.rows, dev)) and
            (k_weight is None or _is(k_weight, torch.bfloat16, plan.rows, dev)))


def _norm_rope_pointers(a, q, k, cos, sin, positions, q_weight, k_weight):
    a.q.ptr, a.k.ptr = qp, kp = q.data_ptr(), k.data_ptr()
    other = 0
    if q_weight is not None:
        a.q_weight = p = q_weight.data_ptr()
        other |= p
    if k_weight is not None:
        a.k_weight = p = k_weight.data_ptr()
        other |= p
    if cos is not None:
        a.cos, a.sin = cp, sp = cos.data_ptr(), sin.data_ptr()
        other |= cp | sp
        if positions is not None:
            a.positions = positions.data_ptr()
    if (qp | kp | other) & 15:
        _check_aligned(qp | kp, "q and k")
        _check_aligned(other, "weights, cos and sin")


def _check_out(o, x):
    _check_bf16(o)
    _require(o.shape == x.shape and o.device == x.device, "outputs must have the shapes and device of the inputs")
    end = 0                                                         # of the elements that the dimensions so far reach
    for step, n in sorted(zip(o.stride(), o.shape)):
        if n > 1:
            _require(step > end, "elements of an output must not lie on one another")
            end += step * (n - 1)
    _check_rows(o)
    _check_aligned(o.data_ptr(), "outputs")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                 positions: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, adjacent_pairs: bool = False,
                 tensor_layout: str = "NHD", out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None):
    """Per-head RMS norm of queries and keys and the rotation by their positions, in one pass.

    q, k: bf16, ``[tokens, heads, head_dim]`` or 4-D in ``tensor_layout`` ("NHD" / "HND"), any strides over whole 16-byte vectors (a slice of
    a fused projection); head_dim a multiple of 8 up to 128.  ``q_weight``, ``k_weight`` (bf16 ``[head_dim]``): ``x * rsqrt(mean(x^2) + eps) *
    weight``, or no norm where None.  ``cos``, ``sin`` (fp32 ``[positions, rot_dim / 2]``): the first ``rot_dim`` channels are rotated, pairs being
    ``(i, i + rot_dim / 2)``, or ``(2i, 2i + 1)`` with ``adjacent_pairs``.  ``positions``: int32 or int64 ``[tokens]`` (``[batch, tokens]``), default
    0, 1, ... in each batch entry; one outside the table gives NaN.  All in fp32, rounded once: a norm needs squares that fp32 holds (channels up
    to 1e18; a row beyond gives zeros or NaN).  ``out``: the two outputs, which may be q and
    k themselves (each its own); else they share no memory with them."""
    if out is not None:
        _check_out(out[0], q)
        _check_out(out[1], k)
    key = _norm_rope_key("qk_norm_rope", q, k, cos, positions, q_weight, k_weight, eps, adjacent_pairs, tensor_layout)
    plan = _plans.get(key)
    if plan is None or not _norm_rope_fits(plan, cos, sin, positions, q_weight, k_weight):
        plan = _keep_plan(key, _norm_rope_plan(q, k, cos, sin, positions, q_weight, k_weight, eps, adjacent_pairs, tensor_layout))
    a = _lib.KvTokensArgs.from_buffer_copy(plan.struct)
    _norm_rope_pointers(a, q, k, cos, sin, positions, q_weight, k_weight)
    if out is None:
        yq, yk = torch.empty_like(q), torch.empty_like(k)
        a.q_out.ptr, a.k_out.ptr = yq.data_ptr(), yk.data_ptr()      # (whose strides the plan has)
    else:
        yq, yk = out
        a.q_out, a.k_out = _rows(yq, tensor_layout), _rows(yk, tensor_layout)
    if a.B and a.N:
        _run(_lib.load().sage3_kv_tokens, a, plan.device, "sage3_kv_tokens")
    return yq, yk


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: FP4KVCache, slots: torch.Tensor,
                        cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                        positions: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                        k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, adjacent_pairs: bool = False,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`qk_norm_rope` of ``[tokens, heads, head_dim]`` tensors with the keys, and the values as they are, written straight to the cache
    (the same bits as :meth:`FP4KVCache.append` of its result).  Returns the queries; ``out``, for them, may be q itself."""
    if out is not None:
        _check_out(out, q)
    key = _norm_rope_key("qk_norm_rope_append", q, k, cos, positions, q_weight, k_weight, eps, adjacent_pairs, None, v.shape, v.stride(), v.dtype,
                         v.device, cache._key)
    plan = _plans.get(key)
    if plan is None or not _is(slots, torch.int64, plan.where, plan.device) or not _norm_rope_fits(plan, cos, sin, positions, q_weight, k_weight):
        _require(q.dim() == 3, "q must be [tokens, heads, head_dim]")
        plan = _norm_rope_plan(q, k, cos, sin, positions, q_weight, k_weight, eps, adjacent_pairs, "NHD")
        cache._check_tokens(k, v, slots)
        _require(q.device == cache.device, "q and the cache must be on one device")
        plan.struct.k_out = _lib.Tensor()                            # (keys go to the cache alone)
        plan.struct.v = _lib.Tensor(None, 0, *_strides(v))
        _keep_plan(key, plan)
    a = _lib.KvTokensArgs.from_buffer_copy(plan.struct)
    _norm_rope_pointers(a, q, k, cos, sin, positions, q_weight, k_weight)
    if out is None:
        out = torch.empty_like(q)
        a.q_out.ptr = out.data_ptr()
    else:
        a.q_out = _rows(out, "NHD")
    vp = v.data_ptr()
    if vp & 15:
        _check_aligned(vp, "v")
    a.v.ptr, a.cache, a.slots = vp, cache._ref, slots.data_ptr()
    if a.N:
        _run(_lib.load().sage3_kv_tokens, a, plan.device, "sage3_kv_tokens")
    return out


def sageattn_kvcache(q: torch.Tensor, cache: FP4KVCache, block_table: torch.Tensor, kv_lens: torch.Tensor,
                     cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: int = 1, max_seqlen_k: Optional[int] = None,
                     is_causal: bool = True, sm_scale: Optional[float] = None, return_lse: bool = False,
                     out: Optional[torch.Tensor] = None, check_status: bool = False):
    """Attention of new tokens over the 4-bit cache, their own keys (already appended) among the last ones.

    q: bf16 ``[tokens, Hq, head_dim]``, ``Hq`` a multiple of the cache's heads; sequence i has rows ``cu_seqlens_q[i] ... cu_seqlens_q[i+1]`` (int32
    ``[B+1]``), or row i alone where ``cu_seqlens_q`` is None.  ``kv_lens`` int32 ``[B]``: keys of each sequence, new ones included;
    ``block_table`` int32 ``[B, columns]``: their pages.  ``max_seqlen_q`` and ``max_seqlen_k`` (default: what the table can hold) must bound the
    lengths - they size grid and workspace; rows and keys beyond them, or beyond q and the table, are left out.  ``is_causal``: bottom-right
    aligned, the last row of a sequence sees all of its keys; the diagonal goes by the lengths as given, whatever is left out.

    Attention is over the values that the cache stands for, queries and softmax are not quantised.  Rows that see no key give zeros and an
    LSE of ``-inf``.  A row that sees a key or value with a NaN in it may be NaN altogether, others are not touched by it; scores (``sm_scale * q.k``)
    beyond 9e7 in size give NaN or zeros.  Keys of pages outside the cache (-1) are not seen.  Rows of q that belong to no sequence (a padded
    batch) are not touched in ``out``, or are undefined in a new tensor; ``out`` shares no memory with the inputs.  Returns the output like q, and
    with ``return_lse`` the natural-log LSE fp32 ``[tokens, Hq]`` of ``sm_scale * q.k``.  ``check_status`` waits for the kernels and raises where
    one of their bounded waits gave up.

    The longest request picks the kernel: where some bring many tokens and others one, two calls, each with its own rows, are faster."""
    if out is not None:
        _check_out(out, q)
    # (what the launch is made for goes by blocks of 128 keys: a plan lasts for as many steps)
    key = ("kvcache", q.shape, q.stride(), q.dtype, q.device, cache._key, block_table.shape, block_table.stride(), kv_lens.shape, cu_seqlens_q is None,
           max_seqlen_q, None if max_seqlen_k is None else -(-max_seqlen_k // 128), is_causal, sm_scale)
    plan = _plans.get(key)
    if (plan is None or not _is(kv_lens, torch.int32, kv_lens.shape, plan.device) or block_table.dtype is not torch.int32 or
            block_table.device != plan.device or not (cu_seqlens_q is None or _is(cu_seqlens_q, torch.int32, plan.where, plan.device))):
        plan = _keep_plan(key, _plan_attention(q, cache, block_table, kv_lens, cu_seqlens_q, max_seqlen_q, max_seqlen_k, is_causal, sm_scale))
    dev, a = plan.device, _lib.KvAttentionArgs.from_buffer_copy(plan.struct)
    if max_seqlen_k is not None:
        a.max_seqlen_k = min(int(max_seqlen_k), a.columns * cache.page_size)
    if out is None:
        out = torch.empty_like(q)                                    # (whose strides the plan has)
    else:
        a.out_stride_h, a.out_stride_n = _strides(out)
    lse = torch.empty(plan.rows, dtype=torch.float32, device=dev) if return_lse else None
    if a.total_q:
        qp = q.data_ptr()
        if qp & 15:
            _check_aligned(qp, "q")
        a.cache, a.q, a.out, a.kv_lens, a.block_table = cache._ref, qp, out.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr()
        if lse is not None:
            a.lse = lse.data_ptr()
        if cu_seqlens_q is not None:
            a.cu_seqlens_q = cu_seqlens_q.data_ptr()
        if plan.workspace:
            ws = cache.data.new_empty(plan.workspace)
            a.workspace = ws.data_ptr()
        status = torch.empty(1, dtype=torch.int32, device=dev) if check_status else None
        if status is not None:
            a.device_status = status.data_ptr()
        _run(_lib.load().sage3_kv_attention, a, dev, "sage3_kv_attention")
        if status is not None:
            with _on_device(dev):
                _lib.check(_lib.load().sage3_read_device_status(status.data_ptr(), _stream_ptr(dev), None), "attention kernel")
    return (out, lse) if return_lse else out


def _plan_attention(q, cache, block_table, kv_lens, cu_seqlens_q, max_seqlen_q, max_seqlen_k, is_causal, sm_scale) -> _Plan:
    _check_numbers(max_seqlen_q=max_seqlen_q, max_seqlen_k=max_seqlen_k, is_causal=is_causal, sm_scale=sm_scale)
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
    _require(max_seqlen_k <= 2 ** 30 and max_seqlen_q < 2 ** 30 and T < 2 ** 31 and B < 2 ** 31, "too many tokens for one call")
    _require(sm_scale is None or 0 < C.c_float(sm_scale).value < float("inf"), "sm_scale must be positive and finite in fp32")
    _check_rows(q)
    _check_device(q)
    plan = _Plan()
    plan.device, plan.rows, plan.where = dev, (T, Hq), torch.Size((B + 1,))
    a = plan.struct = _lib.KvAttentionArgs()
    a.B, a.Hq, a.max_seqlen_q, a.max_seqlen_k, a.total_q = B, Hq, int(max_seqlen_q), max_seqlen_k, T
    a.q_stride_h, a.q_stride_n = _strides(q)
    a.out_stride_h, a.out_stride_n = _strides(torch.empty_like(q, device="meta"))
    a.row_stride, a.columns, a.is_causal = block_table.stride(0), block_table.shape[1], int(bool(is_causal))
    a.sm_scale = 0.0 if sm_scale is None else float(sm_scale)
    # the size of the workspace goes by the sizes alone; a pointer says whether there are offsets
    a.cache, a.cu_seqlens_q = cache._ref, None if cu_seqlens_q is None else cu_seqlens_q.data_ptr()
    n = C.c_size_t()
    with _on_device(dev):
        _lib.check(_lib.load().sage3_kv_attention_workspace(C.byref(a), C.byref(n)), "sage3_kv_attention_workspace")
    a.cache, a.cu_seqlens_q = None, None
    plan.workspace = a.workspace_bytes = n.value
    return plan
