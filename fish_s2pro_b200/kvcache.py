"""Operators on a paged KV cache held in torch tensors (include/s2d_cache.h).

`PagedKvCache` is one layer's cache of a batch of sequences: pages of 64
positions from a pool, in the layout of the batched token loop, with a
page-table row per sequence.  `append` takes new tokens in (QK-norm, rotary
position, key and value rows into the pages), `attention` computes them over
a prefix shared by every sequence (read once for all of them) and their own
sequences, optionally adding up the attention weight that each slot receives,
and `evict` brings sequences down to a budget of slots by those weights.

A decode loop keeps two int32 tensors, `past` and the cache's `lengths`:

    cache.append(q, k, v, pos, past)       # lengths = past + 1
    out = cache.attention(q, prefix_pages=voice, prefix_len=n, weigh=True)
    cache.evict(budget, recent, past)      # past = min(lengths, budget)

Calls are enqueued on torch's current stream of the cache's device and return
without waiting; they can be captured into CUDA graphs.  One thread at a time
uses a PagedKvCache; workspaces come from torch's allocator, so calls on
several streams do not share one.  Lengths, past and q_start are read on the
device.  Errors in the arguments raise S2dError; what
only the device can see is kept in a status word that `check` reads.  The
operators have no backward pass.
"""
from __future__ import annotations

import ctypes
import math
import struct
import threading
from typing import Optional

from .s2d import S2dError, lib

_c = ctypes
_P = ctypes.POINTER
PAGE = 64  # S2D_CACHE_PAGE
S2D_EDEVICE = -6
BAD_PAGE, BAD_LENGTH, FULL, ABORTED = 1, 2, 4, 8  # bits of the status word


class _View(_c.Structure):
    _fields_ = [("k", _c.c_void_p), ("v", _c.c_void_p), ("page_stride", _c.c_int64), ("head_stride", _c.c_int64),
                ("page_table", _c.c_void_p), ("table_stride", _c.c_int64), ("lengths", _c.c_void_p),
                ("positions", _c.c_void_p), ("mass", _c.c_void_p), ("status", _c.c_void_p)] + \
               [(n, _c.c_int32) for n in ("n_seq", "kv_heads", "head_dim", "n_pages", "max_pages", "type", "device")]


class _Append(_c.Structure):
    _fields_ = [("q", _c.c_void_p), ("k", _c.c_void_p), ("v", _c.c_void_p), ("q_stride", _c.c_int64),
                ("k_stride", _c.c_int64), ("v_stride", _c.c_int64), ("q_out", _c.c_void_p),
                ("q_out_stride", _c.c_int64), ("q_norm", _c.c_void_p), ("k_norm", _c.c_void_p),
                ("pos", _c.c_void_p), ("past", _c.c_void_p), ("q_start", _c.c_void_p), ("tokens", _c.c_int32),
                ("heads", _c.c_int32), ("type", _c.c_int32), ("eps", _c.c_float), ("rope_base", _c.c_double)]


class _Attention(_c.Structure):
    _fields_ = [("q", _c.c_void_p), ("q_stride", _c.c_int64), ("out", _c.c_void_p), ("out_stride", _c.c_int64),
                ("lse", _c.c_void_p), ("q_start", _c.c_void_p), ("prefix_pages", _c.c_void_p),
                ("prefix_len", _c.c_int32), ("tokens", _c.c_int32), ("heads", _c.c_int32), ("type", _c.c_int32),
                ("weigh", _c.c_int32), ("scale", _c.c_float), ("workspace", _c.c_void_p),
                ("workspace_bytes", _c.c_size_t)]


class _Evict(_c.Structure):
    _fields_ = [("budget", _c.c_int32), ("recent", _c.c_int32), ("past", _c.c_void_p), ("workspace", _c.c_void_p),
                ("workspace_bytes", _c.c_size_t)]


def _bad(message: str) -> S2dError:
    return S2dError(-1, message)


def _packer(cls):
    """Packs a struct's fields, in their order and C's layout, into bytes: a tenth of the time of a ctypes.Structure."""
    codes = {_c.c_void_p: "P", _c.c_int32: "i", _c.c_int64: "q", _c.c_float: "f", _c.c_double: "d", _c.c_size_t: "N"}
    p = struct.Struct("@" + "".join(codes[t] for _, t in cls._fields_) + "0P")
    assert p.size == _c.sizeof(cls)

    def pack(*fields):
        try:
            return p.pack(*fields)
        except (struct.error, OverflowError) as e:
            raise _bad(f"an argument is out of range: {e}") from None
    return pack


_pack_append, _pack_attention, _pack_evict = _packer(_Append), _packer(_Attention), _packer(_Evict)

_i32 = _c.c_int32
_tail = [_c.c_char_p, _c.c_size_t]
# symbol -> (restype, argtypes); every function declared in include/s2d_cache.h.  Argument structs go in as packed bytes.
CACHE_SIGNATURES = {
    "s2d_cache_append": (_i32, [_P(_View), _c.c_void_p, _c.c_void_p] + _tail),
    "s2d_cache_attention_workspace": (_i32, [_P(_View), _c.c_void_p, _P(_c.c_size_t)] + _tail),
    "s2d_cache_attention": (_i32, [_P(_View), _c.c_void_p, _c.c_void_p] + _tail),
    "s2d_cache_evict_workspace": (_i32, [_P(_View), _c.c_void_p, _P(_c.c_size_t)] + _tail),
    "s2d_cache_evict": (_i32, [_P(_View), _c.c_void_p, _c.c_void_p] + _tail),
    "s2d_cache_status": (_i32, [_P(_View), _P(_i32), _c.c_void_p] + _tail),
}

_bound = None


def cache_lib() -> ctypes.CDLL:
    """libs2d.so with the paged-cache entry points typed."""
    global _bound
    if _bound is None:
        l = lib()
        for name, (res, args) in CACHE_SIGNATURES.items():
            fn = getattr(l, name)
            fn.restype = res
            fn.argtypes = args
        _bound = l
    return _bound


_words, _words_lock = {}, threading.Lock()  # device index -> (clear status words, how many of them are taken)


def _status_word(torch, device):
    """A status word that is clear whatever the current stream is at, as the cache may next be used on another one, and that no
    other cache has had, as a call of one that is gone may still be running.  Words are cleared in blocks, so that few caches
    wait for it."""
    with _words_lock:
        block, taken = _words.get(device.index, (None, 0))
        if block is None or taken == block.shape[0]:
            with torch.cuda.device(device):
                if torch.cuda.is_current_stream_capturing():
                    return torch.zeros(1, dtype=torch.int32, device=device)  # cleared by each replay
                stream = torch.cuda.Stream(device)
                with torch.cuda.stream(stream):
                    block, taken = torch.zeros(1024, dtype=torch.int32, device=device), 0
                stream.synchronize()
        _words[device.index] = block, taken + 1
        return block[taken:taken + 1]


class PagedKvCache:
    """One layer's paged cache over the caller's tensors, which it keeps and
    writes in place.

    k, v: [n_pages, kv_heads, 64, head_dim] f16 or bf16, head_dim 64 or 128;
    the last two dimensions contiguous, page and head strides free, the same
    for both (a layer's slice of a pool of every layer's pages will do).
    page_table: int32 [n_seq, max_pages], page ids of each sequence in order.
    lengths: int32 [n_seq], cached slots of each sequence.
    positions, mass: int32 and f32 [n_seq, kv_heads, max_pages * 64], the
    position and the accumulated attention weight of each slot; either may be
    left out where nothing evicts.  `weigh` needs mass, `evict` both."""

    def __init__(self, k, v, page_table, lengths, positions=None, mass=None):
        import torch
        self._torch, self._int32 = torch, torch.int32
        if k.dim() != 4 or k.shape[2] != PAGE or v.shape != k.shape or v.stride() != k.stride() or v.dtype != k.dtype:
            raise _bad("k and v must be alike, [n_pages, kv_heads, 64, head_dim]")
        if k.dtype not in (torch.float16, torch.bfloat16):
            raise _bad("the cache must be f16 or bf16")
        if k.stride(3) != 1 or k.stride(2) != k.shape[3]:
            raise _bad("the positions of a page must be contiguous rows")
        self.device = k.device
        if self.device.type != "cuda":
            raise _bad("the cache must be on a CUDA device")
        self._index = self.device.index
        # torch.cuda.current_stream(index).cuda_stream without the Stream object
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda index: torch.cuda.current_stream(index).cuda_stream)
        self.n_pages, self.kv_heads, _, self.head_dim = k.shape
        self.n_seq, self.max_pages = page_table.shape if page_table.dim() == 2 else (0, 0)
        self._ints("page_table", page_table, None)
        if page_table.dim() != 2 or page_table.stride(1) != 1:
            raise _bad("page_table must be [n_seq, max_pages] with contiguous rows")
        self._ints("lengths", lengths, (self.n_seq,))
        slots = (self.n_seq, self.kv_heads, self.max_pages * PAGE)
        if positions is not None:
            self._ints("positions", positions, slots)
        if mass is not None:
            self._dense("mass", mass, torch.float32, slots)
        if v.device != self.device:
            raise _bad("every buffer must be on the cache's device")
        for name, t in (("k", k), ("v", v), ("mass", mass)):
            if t is not None and t.requires_grad:
                self._no_grad(name)
        self.k, self.v, self.page_table, self.lengths, self.positions, self.mass = k, v, page_table, lengths, positions, mass
        self.dtype = k.dtype
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._types = {k.dtype: 1 if k.dtype == torch.float16 else 30}
        if k.dtype == torch.float16:
            self._types[torch.float32] = 0
        self._status = _status_word(torch, self.device)
        self._view = _View(
            k.data_ptr(), v.data_ptr(), k.stride(0) if self.n_pages > 1 else max(k.stride(0), self.kv_heads * PAGE * self.head_dim),
            k.stride(1) if self.kv_heads > 1 else PAGE * self.head_dim, page_table.data_ptr(),
            page_table.stride(0) if self.n_seq > 1 else self.max_pages, lengths.data_ptr(),
            positions.data_ptr() if positions is not None else None, mass.data_ptr() if mass is not None else None,
            self._status.data_ptr(), self.n_seq, self.kv_heads, self.head_dim, self.n_pages, self.max_pages,
            self._types[k.dtype], self.device.index)
        self._view_ref = _c.byref(self._view)
        self._err = _c.create_string_buffer(256)
        self._sizes = {}
        self._lib = cache_lib()

    def _dense(self, name, t, dtype, shape):
        if t.dtype != dtype or t.get_device() != self._index:
            raise _bad(f"{name} must be {dtype} on {self.device}")
        if shape is not None and (t.shape != shape or not t.is_contiguous()):
            raise _bad(f"{name} must be contiguous of shape {tuple(shape)}, got {tuple(t.shape)}")
        return t.data_ptr()

    def _ints(self, name, t, shape):
        return self._dense(name, t, self._int32, shape)

    def _rows(self, name, t, heads=None):
        """Token rows [tokens, heads, head_dim] with contiguous heads: (pointer, token stride)."""
        s = t.shape
        if len(s) != 3 or s[2] != self.head_dim or (heads is not None and s[1] != heads):
            raise _bad(f"{name} must be [tokens, {heads or 'heads'}, {self.head_dim}], got {tuple(s)}")
        step, st1, st2 = t.stride()
        if s[0] and (st2 != 1 or (st1 != s[2] and s[1] > 1)):
            raise _bad(f"the heads of a token of {name} must be contiguous")
        if t.get_device() != self._index:
            raise _bad(f"{name} must be on {self.device}")
        if t.requires_grad:
            self._no_grad(name)
        return t.data_ptr(), step if s[0] > 1 else s[1] * s[2]

    def _no_grad(self, name):
        if self._torch.is_grad_enabled():
            raise _bad(f"{name} requires a gradient: the cache operators have no backward pass")

    def _gain(self, name, t):
        if t.requires_grad:
            self._no_grad(name)
        return self._dense(name, t, self._torch.float32, (self.head_dim,))

    def _like_q(self, q, out):
        """The output for q, new if none is given: (tensor, pointer, token stride)."""
        if out is None:
            tokens, heads, d = q.shape
            out = q.new_empty_strided((tokens, heads, d), (heads * d, d, 1))
            return out, out.data_ptr(), heads * d
        if out.shape != q.shape or out.dtype != q.dtype:
            raise _bad("out must be like q")
        return (out, *self._rows("out", out))

    def _type(self, name, t):
        code = self._types.get(t.dtype)
        if code is None:
            raise _bad(f"{name} must be of the cache's type ({self.dtype})" +
                       (" or float32" if self.dtype == self._torch.float16 else ""))
        return code

    def _stream(self):
        return self._raw_stream(self._index)

    def _call(self, rc: int) -> None:
        if rc != 0:
            raise S2dError(rc, self._err.value.decode(errors="replace") or f"error {rc}")

    def _starts(self, q_start, tokens):
        if q_start is None:
            if tokens > self.n_seq:
                raise _bad(f"{tokens} tokens for {self.n_seq} sequences: give q_start")
            return 0
        return self._ints("q_start", q_start, (self.n_seq + 1,))

    def append(self, q, k, v, pos, past, *, q_start=None, q_norm=None, k_norm=None, eps: float = 1e-6,
               rope_base: float = 1_000_000.0, out=None):
        """Take new tokens in: q [tokens, heads, head_dim], k and v [tokens,
        kv_heads, head_dim], of the cache's type or f32 with an f16 cache.
        Queries and keys are normed per head (q_norm, k_norm: f32 [head_dim]
        gains; None leaves them as they are) and rotated by pos (int32
        [tokens]); keys and values go to the slots after past (int32 [n_seq]),
        with their positions and no mass, and lengths becomes past + tokens:
        neither past nor pos nor q_start may be the lengths tensor.  q_start:
        int32 [n_seq + 1], the sequences' first tokens in a packed batch; None:
        token i is sequence i's.
        Returns the queries, in `out` if given: q itself, or rows apart from
        those of q, k and v (slices of one packed tensor will do)."""
        tokens = q.shape[0] if q.dim() == 3 else 0
        ty = self._type("q", q)
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise _bad("q, k and v must have one type")
        qp, qs = self._rows("q", q)
        kp, ks = self._rows("k", k, self.kv_heads)
        vp, vs = self._rows("v", v, self.kv_heads)
        if k.shape[0] != tokens or v.shape[0] != tokens:
            raise _bad("q, k and v must have the same tokens")
        out, op, os_ = self._like_q(q, out)
        a = _pack_append(qp, kp, vp, qs, ks, vs, op, os_, 0 if q_norm is None else self._gain("q_norm", q_norm),
                         0 if k_norm is None else self._gain("k_norm", k_norm), self._ints("pos", pos, (tokens,)),
                         self._ints("past", past, (self.n_seq,)), self._starts(q_start, tokens), tokens, q.shape[1], ty, eps,
                         rope_base)
        self._call(self._lib.s2d_cache_append(self._view_ref, a, self._stream(), self._err, 256))
        return out

    def attention(self, q, *, q_start=None, prefix_pages=None, prefix_len: int = 0, scale: Optional[float] = None,
                  weigh: bool = False, out=None, return_lse: bool = False):
        """softmax(scale * q . k) v of each token over the shared prefix
        (prefix_pages: int32 page ids in the same pool, prefix_len positions)
        and the slots of its own sequence.  A sequence's tokens are its newest
        slots, and each sees the slots up to its own: call it after the append
        and before the next eviction.  weigh adds every own slot's softmax
        weight, summed over the tokens and the query heads of its KV head, to
        mass.  A token that sees nothing gives zeros.  Returns out, or (out,
        lse) with lse f32 [tokens, heads] the natural log of the sum of
        exponentials (-inf where a token sees nothing); rows past
        q_start[n_seq] are not written.  The rows of out, if given, lie apart
        from q's (slices of one packed tensor will do)."""
        ty = self._type("q", q)
        qp, qs = self._rows("q", q)
        tokens, heads = q.shape[0], q.shape[1]
        torch = self._torch
        out, op, os_ = self._like_q(q, out)
        lse = q.new_empty_strided((tokens, heads), (heads, 1), dtype=torch.float32) if return_lse else None
        prefix = 0
        if prefix_len:
            if prefix_pages is None or prefix_pages.dim() != 1 or prefix_len < 0 or prefix_pages.shape[0] * PAGE < prefix_len:
                raise _bad("prefix_pages must be int32 page ids that hold prefix_len positions")
            prefix = self._ints("prefix_pages", prefix_pages, prefix_pages.shape)
        fields = (qp, qs, op, os_, lse.data_ptr() if return_lse else 0, self._starts(q_start, tokens), prefix, prefix_len, tokens,
                  heads, ty, 1 if weigh else 0, self._scale if scale is None else scale)
        key = (tokens, heads, prefix_len, ty, weigh, q_start is None)
        need = self._sizes.get(key)
        if need is None:
            n = _c.c_size_t()
            self._call(self._lib.s2d_cache_attention_workspace(self._view_ref, _pack_attention(*fields, 0, 0), _c.byref(n), self._err, 256))
            if len(self._sizes) >= 256:
                self._sizes.clear()
            need = self._sizes[key] = n.value
        # from the caching allocator: stream-ordered, and a captured graph gets its own
        work = q.new_empty_strided((need,), (1,), dtype=torch.uint8) if need else None
        self._call(self._lib.s2d_cache_attention(self._view_ref, _pack_attention(*fields, work.data_ptr() if need else 0, need),
                                                 self._stream(), self._err, 256))
        return (out, lse) if return_lse else out

    def evict(self, budget: int, recent: int, past=None) -> None:
        """Keep `budget` slots of every (sequence, KV head) that has more:
        those of the last `recent` positions, then the heaviest by mass
        (equals: the lowest slot).  Kept rows at slots from budget on move
        into the freed ones before it, with their positions and mass.  past
        (int32 [n_seq], not the lengths tensor) receives min(length, budget),
        what the next append takes; lengths itself stays as it is."""
        to = 0 if past is None else self._ints("past", past, (self.n_seq,))
        key = budget
        need = self._sizes.get(key)
        if need is None:
            n = _c.c_size_t()
            self._call(self._lib.s2d_cache_evict_workspace(self._view_ref, _pack_evict(budget, recent, to, 0, 0), _c.byref(n), self._err, 256))
            if len(self._sizes) >= 256:
                self._sizes.clear()
            need = self._sizes[key] = n.value
        work = self.lengths.new_empty_strided((need,), (1,), dtype=self._torch.uint8) if need else None
        self._call(self._lib.s2d_cache_evict(self._view_ref, _pack_evict(budget, recent, to, work.data_ptr() if need else 0, need),
                                             self._stream(), self._err, 256))

    def check(self) -> None:
        """Wait for the current stream and raise S2dError if a call met a page
        id outside the pool, a length, past or q_start out of range, or a full
        sequence since the last check.  Not inside a capture."""
        bits = _c.c_int32()
        self._call(self._lib.s2d_cache_status(self._view_ref, _c.byref(bits), self._stream(), self._err, 256))
        if bits.value:
            what = [t for b, t in ((BAD_PAGE, "a page id outside the pool"), (BAD_LENGTH, "a length, past or q_start out of range"),
                                   (FULL, "a token past the last slot of its sequence"), (ABORTED, "a kernel gave up waiting")) if bits.value & b]
            raise S2dError(S2D_EDEVICE, "paged cache: " + ", ".join(what))
