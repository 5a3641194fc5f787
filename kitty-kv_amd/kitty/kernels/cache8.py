"""The 8-bit paged cache: written token by token or in chunks, read back, attended
over by one or many queries, by sequences that share prefixes, and cut down to the
tokens that got the most attention.

A layer that 2 bits cost too much (and that has no room for 16) keeps its keys
and values in e4m3 with one float32 scale per page, head and stream.  Unlike the
2-bit pages, whose tokens wait in 16-bit buffers until a page is full, tokens go
into their page as they come: the page's scale is a power of two that rises when
a larger token arrives, and its older codes are rounded again to the new scale.

Device tensors run the HIP kernels of csrc/cache8.hip, attend8*.hip, weigh8.hip and
evict8.hip, CPU tensors the torch code of ``kernels.cpu8``.  No call waits for the
GPU, reads a length on the host or keeps state of its own, so calls may be captured
into a graph and replayed with other lengths and tables in the same tensors.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Tuple, Union

import numpy as np
import torch

from .. import _hip
from . import cpu8
from .ops import _need, calls_followed

_SRC = {torch.float16: _hip.KITTY_SRC_F16, torch.bfloat16: _hip.KITTY_SRC_BF16, torch.float32: _hip.KITTY_SRC_F32}
_PAGE_TOKENS = (16, 32, 64, 128, 256)
# kitty_cache8_write_args / _read_args, kitty_cache8_attention_args, _shared_args, kitty_cache8_weights and
# kitty_cache8_evict_args as the C compiler lays them out (packing one takes a quarter of a ctypes structure's time)
_ROWS = struct.Struct("2P6qPq2P4i")
_ATTENTION = struct.Struct("3P6qPq2P7ifPN")
_SHARED = struct.Struct("3P6qPqPPq2P8ifPN")
_WEIGHTS = struct.Struct("P2qi")
_EVICT = struct.Struct("P2qPqPPq3P7iPN")


_FOLLOWED = "calls of the 8-bit cache cannot be traced, compiled or transformed"


def _sig(t: Optional[torch.Tensor]):
    """What the checks of a tensor depend on, but for its address."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _strides(t: torch.Tensor) -> Tuple[int, ...]:
    """Strides of the first three dimensions, 0 where a dimension has one entry."""
    return tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3]))


def _aligned16(t: torch.Tensor) -> bool:
    return all(s * t.element_size() % 16 == 0 for s in _strides(t))


def _given(t: torch.Tensor, name: str) -> torch.Tensor:
    """A tensor of values as a kernel may read it by pointer."""
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} needs a gradient and the 8-bit cache has no backward: call under torch.no_grad()")
    return t.resolve_neg() if t.is_neg() else t


def _into(t: torch.Tensor) -> None:
    """An output of the program's own: as torch's in-place writes."""
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("out needs a gradient and the 8-bit cache has no backward: call under torch.no_grad()")


_written = torch.autograd.graph.increment_version      # what torch's own writes do


def _span(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to behind its last."""
    return (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether no two rows (of contiguous elements, the last dimension) share memory."""
    dims, span = sorted((s, n) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1), t.shape[-1]
    if t.numel() == 0:
        return True
    nested = True
    for s, n in dims:
        nested = nested and s >= span
        span += (n - 1) * s
    if nested:
        return True
    starts = np.zeros(1, np.int64)      # rows laid between each other, or over
    for s, n in dims:
        starts = (starts[:, None] + s * np.arange(n)).ravel()
    return bool((np.diff(np.sort(starts)) >= t.shape[-1]).all())


class Cache8:
    """Pools of an 8-bit paged cache and the calls that work on them.

    key, value: (P, H, G, D) float8_e4m3fn (or uint8, the same bytes); scale:
    (P, H, 2) float32, of keys and of values.  G is 16, 32, 64, 128 or 256, D a
    multiple of 16 up to 256; pages and heads may lie at any 16-byte aligned
    strides.  Code c of a page stands for c * scale; pages written elsewhere may
    hold any finite scale from 2^-100 on.  One pool serves any number of sequences:
    ``block_table`` (B, W) int32 names each sequence's pages in order, and a page
    may stand in several tables (a shared prefix) as long as one sequence of a
    call writes to it.

    Lengths, tables and positions are int32 tensors on the pools' device, read
    by the kernels.  Page ids outside the pool are never followed: their tokens
    are not written, read as NaN and make the attention of rows that see them NaN.
    """

    def __init__(self, key: torch.Tensor, value: torch.Tensor, scale: torch.Tensor) -> None:
        for name, t in (("key", key), ("value", value)):
            _need(t.dtype in (torch.float8_e4m3fn, torch.uint8), f"{name} pool must be float8_e4m3fn or uint8")
            _need(t.dim() == 4 and t.shape == key.shape, "key and value pools must be (P, H, G, D) alike")
            _need(t.stride(3) == 1, f"{name} pool needs contiguous channels")
        P, H, G, D = key.shape
        _need(G in _PAGE_TOKENS, "pages must hold 16, 32, 64, 128 or 256 tokens")
        _need(H > 0 and D % 16 == 0 and D > 0, "head_dim must be a positive multiple of 16")
        if D > 256:
            raise NotImplementedError("the 8-bit cache is built for head_dim up to 256")
        _need(scale.dtype == torch.float32 and tuple(scale.shape) == (P, H, 2) and scale.stride(2) == 1,
              "scale must be float32 (P, H, 2) with the two streams next to each other")
        for name, t in (("key", key), ("value", value), ("scale", scale)):
            if t.requires_grad:
                raise RuntimeError(f"{name} needs a gradient and the 8-bit cache has no backward: detach it")
            _need(not t.is_neg(), f"{name} must not be a negated view")
        if value.device != key.device or scale.device != key.device:
            raise RuntimeError("key, value and scale must be on one device")
        self.key, self.value, self.scale = key, value, scale
        self.device = key.device
        self.num_pages, self.num_kv_heads, self.page_tokens, self.head_dim = P, H, G, D
        self._on_device = key.device.type == "cuda"
        if not self._on_device:
            if key.device.type != "cpu":
                raise RuntimeError(f"the 8-bit cache computes on ROCm devices and the CPU, not on {key.device}")
            return
        self._lib = _hip.load()
        self._index = key.device.index if key.device.index is not None else torch.cuda.current_device()
        self._c = _hip.Cache8(key.data_ptr(), value.data_ptr(), scale.data_ptr(), *_strides(key)[:2], key.stride(2),
                              *_strides(value)[:2], value.stride(2), *_strides(scale)[:2], P, H, D, G)
        self._ref = ctypes.byref(self._c)
        # what a call of these shapes, strides and types was found to need (the
        # checks of a signature run once; addresses are looked at in every call)
        self._known: dict = {}
        # a batch of none: what the library refuses of the pools, it refuses here
        _hip.check(self._lib.kitty_cache8_write(self._ref, _ROWS.pack(*[0] * 16), None))

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, head_dim: int, page_tokens: int = 128,
              device: Union[str, torch.device] = "cuda:0") -> "Cache8":
        """A cache with pools of its own, zeroed."""
        shape = (num_pages, num_kv_heads, page_tokens, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
        return cls(k, v, torch.ones(num_pages, num_kv_heads, 2, device=device))

    # ----------------------------------------------------------------- checks
    def _here(self, name: str, t: torch.Tensor) -> None:
        if t.device != self.device:
            raise RuntimeError(f"{name} is on {t.device}, the cache on {self.device}")

    def _i32(self, name: str, t: Optional[torch.Tensor], B: int, optional: bool = False) -> None:
        if t is None and optional:
            return
        _need(t is not None and t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == B and (B <= 1 or t.stride(0) == 1),
              f"{name} must be int32 ({B},)")
        self._here(name, t)

    def _check_table(self, t: torch.Tensor, B: int, name: str = "block_table") -> None:
        _need(t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == B and (t.shape[1] <= 1 or t.stride(1) == 1),
              f"{name} must be int32 ({B}, W) with contiguous rows")
        self._here(name, t)

    def _keep(self, sig, found):
        if len(self._known) >= 512:
            self._known.clear()
        self._known[sig] = found
        return found

    def _launch(self, fn, args: bytes) -> None:
        """`fn` on the current stream of the pools' device."""
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                rc = fn(self._ref, args, _hip.stream_ptr(self.device))
        else:
            rc = fn(self._ref, args, _hip.stream_ptr(self.device))
        if rc:
            _hip.check(rc)

    # The calls below run their checks once per signature (_known) and spend their time
    # on the host in tensor attributes, so they ask for each once.

    # ------------------------------------------------------------------ calls
    def write(self, key: torch.Tensor, value: torch.Tensor, block_table: torch.Tensor, start: torch.Tensor,
              lens: Optional[torch.Tensor] = None) -> None:
        """Rows t < lens[b] (all T where lens is None) of key and value (B, H, T, D)
        become tokens start[b] + t of sequence b.

        float16, bfloat16 or float32 at any strides.  A page's scale is the
        smallest power of two (2^-64 at least) with which its tokens stay within
        448; a page that holds tokens before start[b] keeps or raises its scale,
        and where it rises those tokens' codes are rounded again.  NaN and
        infinities become NaN.  Rows behind the last token keep their bytes.
        Tokens without a page (a negative start, a page number past the table, an
        id outside the pool) are dropped."""
        if calls_followed():
            raise NotImplementedError(_FOLLOWED)
        if key.requires_grad or value.requires_grad or key.is_neg() or value.is_neg():
            key, value = _given(key, "key"), _given(value, "value")
        sig = (key.shape, key.stride(), key.dtype, key.device, _sig(value), _sig(block_table), _sig(start), _sig(lens))
        found = self._known.get(sig) if self._on_device else None
        if found is None:
            _need(key.dim() == 4 and key.shape[1] == self.num_kv_heads and key.shape[3] == self.head_dim,
                  f"key must be (B, {self.num_kv_heads}, T, {self.head_dim})")
            _need(value.shape == key.shape and value.dtype == key.dtype, "value must have key's shape and dtype")
            _need(key.dtype in _SRC, "key and value must be float16, bfloat16 or float32")
            self._here("key", key)
            self._here("value", value)
            B, _, T, _ = key.shape
            self._check_table(block_table, B)
            self._i32("start", start, B)
            self._i32("lens", lens, B, optional=True)
            if key.stride(3) != 1 or value.stride(3) != 1:
                return self.write(key.contiguous(), value.contiguous(), block_table, start, lens)
            if B == 0 or T == 0:
                return
            if not self._on_device:
                cpu8.write(self.key, self.value, self.scale, key, value, block_table, start, lens)
                return
            found = self._keep(sig, ((*_strides(key), *_strides(value)), block_table.stride(0) if B > 1 else 0,
                                     (B, T, block_table.shape[1], _SRC[key.dtype])))
        strides, bt_stride, rest = found
        self._launch(self._lib.kitty_cache8_write, _ROWS.pack(
            key.data_ptr(), value.data_ptr(), *strides, block_table.data_ptr(), bt_stride, start.data_ptr(),
            0 if lens is None else lens.data_ptr(), *rest))

    def read(self, block_table: torch.Tensor, lens: torch.Tensor, tokens: int, start: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.float16,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(keys, values), each (B, H, tokens, D) of `dtype` (or the tensors of
        `out`): row t is token start[b] + t (start None: from 0) of sequence b,
        code * scale rounded once; 0 behind its lens[b] tokens, NaN where the
        token has no page.  The two tensors of `out` share no element."""
        if calls_followed():
            raise NotImplementedError(_FOLLOWED)
        tokens = int(tokens)
        if out is not None:
            _into(out[0])
            _into(out[1])
        sig = ("read", tokens, dtype, _sig(block_table), _sig(lens), _sig(start),
               None if out is None else (_sig(out[0]), _sig(out[1])))
        found = self._known.get(sig) if self._on_device else None
        if found is None:
            _need(tokens >= 0, "tokens must not be negative")
            _need(block_table.dim() == 2, "block_table must be int32 (B, W)")
            B = block_table.shape[0]
            self._check_table(block_table, B)
            self._i32("lens", lens, B)
            self._i32("start", start, B, optional=True)
            shape = (B, self.num_kv_heads, tokens, self.head_dim)
            if out is None:
                _need(dtype in _SRC, "dtype must be float16, bfloat16 or float32")
                k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
            else:
                k, v = out
                for t in out:
                    _need(tuple(t.shape) == shape and t.dtype == k.dtype and t.dtype in _SRC and t.stride(3) == 1,
                          f"out must be two {shape} tensors of one type with contiguous channels")
                    _need(_rows_apart(t), "out must not share memory between its rows")
                    self._here("out", t)
                _need(tokens == 0 or B == 0 or k.data_ptr() != v.data_ptr(), "out must not be the same memory twice")
                dtype = k.dtype
            if B == 0 or tokens == 0:
                return k, v
            if not self._on_device:      # its writes are torch's
                cpu8.read(self.key, self.value, self.scale, block_table, lens, start, (k, v))
                return k, v
            like = k.new_empty(1).expand(shape)      # what new outputs look like, of one element
            found = self._keep(sig, (like, _aligned16(k) and _aligned16(v), (*_strides(k), *_strides(v)),
                                     block_table.stride(0) if B > 1 else 0, (B, tokens, block_table.shape[1], _SRC[dtype])))
        like, aligned, strides, bt_stride, rest = found
        if out is None:
            k = torch.empty_like(like, memory_format=torch.contiguous_format)
            v = torch.empty_like(k)
        else:
            k, v = out
            kp, vp = k.data_ptr(), v.data_ptr()
            _need(kp != vp, "out must not be the same memory twice")
            if not aligned or kp % 16 or vp % 16 or k.is_neg() or v.is_neg():      # rows the kernel does not write in place
                for t, x in zip(out, self.read(block_table, lens, tokens, start, k.dtype)):
                    t.copy_(x)
                return k, v
            _written((k, v))
        self._launch(self._lib.kitty_cache8_read, _ROWS.pack(
            k.data_ptr(), v.data_ptr(), *strides, block_table.data_ptr(), bt_stride,
            0 if start is None else start.data_ptr(), lens.data_ptr(), *rest))
        return k, v

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
               q_lens: Optional[torch.Tensor] = None, causal: bool = True, sm_scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False, max_tokens: Optional[int] = None):
        """Softmax attention of q (B, Hq, T, D), float16 or bfloat16, over the
        lens[b] tokens each sequence has in the cache; T from one (a decode step)
        to a prompt's chunk.  Query head h reads KV head h // (Hq / H).

        causal: the q_lens[b] (T where None) queries of sequence b are its last
        tokens, written before the call, and each sees what precedes it and
        itself; otherwise every query sees every token (an encoder's states).
        Rows that see nothing, and rows past q_lens[b], are 0.  sm_scale defaults
        to D^-1/2.  Scores, softmax and sums are float32.  return_lse: also the
        rows' log of the sum of exp(score), float32 (B, Hq, T), -inf where a row
        sees nothing.  max_tokens: the largest lens[b] where the program knows it
        (default: what the table can hold); it only chooses how the work is split.
        out may be q, or lie in its memory in any way (a copy of q is then read)."""
        if calls_followed():
            raise NotImplementedError(_FOLLOWED)
        if q.requires_grad or q.is_neg():
            q = _given(q, "q")
        if out is not None:
            _into(out)
        causal, sm_scale = bool(causal), None if sm_scale is None else float(sm_scale)
        max_tokens = 0 if max_tokens is None else int(max_tokens)
        sig = (q.shape, q.stride(), q.dtype, q.device, _sig(block_table), _sig(lens), None if q_lens is None else _sig(q_lens),
               causal, sm_scale, None if out is None else _sig(out), max_tokens)
        found = self._known.get(sig) if self._on_device else None
        if found is None:
            _need(q.dim() == 4 and q.shape[3] == self.head_dim, f"q must be (B, Hq, T, {self.head_dim})")
            _need(q.dtype in (torch.float16, torch.bfloat16), "q must be float16 or bfloat16")
            self._here("q", q)
            B, Hq, T, D = q.shape
            _need(Hq > 0 and Hq % self.num_kv_heads == 0, f"q heads must be a positive multiple of {self.num_kv_heads}")
            self._check_table(block_table, B)
            self._i32("lens", lens, B)
            self._i32("q_lens", q_lens, B, optional=True)
            scale = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
            _need(0.0 < scale <= 1e30, "sm_scale must be positive and finite")
            _need(0 <= max_tokens < 1 << 31, "max_tokens must be in [0, 2^31)")
            if out is not None:
                _need(out.shape == q.shape and out.dtype == q.dtype and out.stride(3) == 1,
                      "out must have q's shape and dtype and contiguous channels")
                _need(_rows_apart(out), "out must not share memory between its rows")
                self._here("out", out)
            if B == 0 or T == 0 or not self._on_device:
                if out is None:
                    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
                lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device)
                if B and T:
                    cpu8.attend(self.key, self.value, self.scale, q, block_table, lens, q_lens, causal, scale, out, lse)
                return (out, lse) if return_lse else out
            in_place = q.stride(3) == 1 and _aligned16(q) and (out is None or _aligned16(out))
            # where the two lie in one piece of memory: their spans, and whether their rows are at the same places
            spans = None if out is None else (_span(q), _span(out), _strides(q) == _strides(out))
            o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
            W = block_table.shape[1]
            head = (*_strides(q), *_strides(o))
            rest = (B, Hq, T, W, max_tokens, causal,
                    _hip.KITTY_DTYPE_F16 if q.dtype == torch.float16 else _hip.KITTY_DTYPE_BF16, scale)
            bt_stride = block_table.stride(0) if B > 1 else 0
            size = ctypes.c_size_t(0)
            with torch.cuda.device(self._index):      # the plan is the pools' device's
                _hip.check(self._lib.kitty_cache8_attention_workspace_size(
                    self._ref, _ATTENTION.pack(0, 0, 0, *[0] * 6, 0, bt_stride, 0, 0, *rest, 0, 0), ctypes.byref(size)))
            found = self._keep(sig, (in_place, q.is_contiguous(), head, bt_stride, rest, size.value, spans))
        in_place, like_q, head, bt_stride, rest, need, spans = found
        qp = q.data_ptr()
        if out is not None:
            op = out.data_ptr()
            if op % 16 or out.is_neg() or (qp < op + spans[1] and op < qp + spans[0] and not (qp == op and spans[2])):
                in_place = False    # also: rows of out over other rows of q, which may be read after they are written
            else:
                _written(out)
        if not in_place or qp % 16:
            # rows the kernel does not read or write in place
            got = self.attend(q.clone(memory_format=torch.contiguous_format), block_table, lens, q_lens, causal, sm_scale,
                              None, return_lse, max_tokens)
            if out is None:
                return got
            out.copy_(got[0] if return_lse else got)
            return (out, got[1]) if return_lse else out
        if out is None:
            out = torch.empty_like(q) if like_q else torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
        # a workspace of the call's own, from torch's allocator on its stream: calls
        # on other streams and in captured graphs never share one
        ws = q.new_empty((need + 1) // 2) if need else None
        self._launch(self._lib.kitty_cache8_attention, _ATTENTION.pack(
            qp, out.data_ptr(), 0 if lse is None else lse.data_ptr(), *head, block_table.data_ptr(), bt_stride,
            lens.data_ptr(), 0 if q_lens is None else q_lens.data_ptr(), *rest, 0 if ws is None else ws.data_ptr(), need))
        return (out, lse) if return_lse else out

    def _check_queries(self, q: torch.Tensor, out: Optional[torch.Tensor], sm_scale: Optional[float]) -> float:
        """Checks of an attention's queries and output; its scale."""
        _need(q.dim() == 4 and q.shape[3] == self.head_dim, f"q must be (B, Hq, T, {self.head_dim})")
        _need(q.dtype in (torch.float16, torch.bfloat16), "q must be float16 or bfloat16")
        self._here("q", q)
        _need(q.shape[1] > 0 and q.shape[1] % self.num_kv_heads == 0,
              f"q heads must be a positive multiple of {self.num_kv_heads}")
        scale = 1.0 / math.sqrt(self.head_dim) if sm_scale is None else sm_scale
        _need(0.0 < scale <= 1e30, "sm_scale must be positive and finite")
        if out is not None:
            _need(out.shape == q.shape and out.dtype == q.dtype and out.stride(3) == 1,
                  "out must have q's shape and dtype and contiguous channels")
            _need(_rows_apart(out), "out must not share memory between its rows")
            self._here("out", out)
        return scale

    def attend_shared(self, q: torch.Tensor, prefix_table: torch.Tensor, prefix_lens: torch.Tensor, block_table: torch.Tensor,
                      lens: torch.Tensor, q_lens: Optional[torch.Tensor] = None, causal: bool = True,
                      sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """``attend`` for sequences that share prefixes (a system prompt, the samples of
        one prompt), which are read once for all of them.

        prefix_table (F, Wp) and prefix_lens (F,) name the prefixes, of any length; B is
        a multiple of F, and sequence b is prefix b // (B / F) followed by the lens[b]
        tokens of its own in the pages of block_table's row b (lens[b] may be 0; the first
        of them is row 0 of its first page).  causal: the q_lens[b] queries of sequence b
        are the last tokens of the two together; otherwise every query sees all of both.
        Results are ``attend``'s over the two in one table but for rounding; for bfloat16 and
        more than 64 rows of a prefix (its sequences' queries times the group's heads) that
        of the softmax weights is to 11 bits, a tenth of the output's own.  out may be q
        or lie in its memory in any way.  Parts of the rows take up to a gibibyte beside
        it; calls of more run in pieces."""
        if calls_followed():
            raise NotImplementedError(_FOLLOWED)
        if q.requires_grad or q.is_neg():
            q = _given(q, "q")
        if out is not None:
            _into(out)
        causal, sm_scale = bool(causal), None if sm_scale is None else float(sm_scale)
        sig = ("shared", q.shape, q.stride(), q.dtype, q.device, _sig(prefix_table), _sig(prefix_lens), _sig(block_table),
               _sig(lens), _sig(q_lens), causal, sm_scale, _sig(out))
        found = self._known.get(sig) if self._on_device else None
        if found is None:
            scale = self._check_queries(q, out, sm_scale)
            B, Hq, T, _ = q.shape
            _need(prefix_table.dim() == 2 and prefix_table.shape[0] > 0 and B % prefix_table.shape[0] == 0,
                  "prefix_table must be int32 (F, Wp), and the batch a multiple of F")
            F = prefix_table.shape[0]
            self._check_table(prefix_table, F, "prefix_table")
            self._i32("prefix_lens", prefix_lens, F)
            self._check_table(block_table, B)
            self._i32("lens", lens, B)
            self._i32("q_lens", q_lens, B, optional=True)
            if B == 0 or T == 0 or not self._on_device:
                o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
                lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device)
                if B and T:
                    cpu8.attend_shared(self.key, self.value, self.scale, q.contiguous(), prefix_table, prefix_lens, block_table, lens,
                                       q_lens, causal, scale, o, lse)
                return (o, lse) if return_lse else o
            in_place = q.stride(3) == 1 and _aligned16(q), out is None or _aligned16(out)
            o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
            # copies of rows that the kernel does not read or write in place are contiguous
            Hs, Ts = Hq * T * self.head_dim, T * self.head_dim
            packed = tuple(0 if n == 1 else s for n, s in zip((B, Hq, T), (Hs, Ts, self.head_dim)))
            head = (*(_strides(q) if in_place[0] else packed), *(_strides(o) if in_place[1] else packed))
            tables = prefix_table.stride(0) if F > 1 else 0, block_table.stride(0) if B > 1 else 0
            rest = (F, B, Hq, T, prefix_table.shape[1], block_table.shape[1], causal,
                    _hip.KITTY_DTYPE_F16 if q.dtype == torch.float16 else _hip.KITTY_DTYPE_BF16, scale)
            size = ctypes.c_size_t(0)
            with torch.cuda.device(self._index):      # the plan is the pools' device's
                _hip.check(self._lib.kitty_cache8_shared_attention_workspace_size(
                    self._ref, _SHARED.pack(0, 0, 0, *head, 0, tables[0], 0, 0, tables[1], 0, 0, *rest, 0, 0), ctypes.byref(size)))
            found = self._keep(sig, (in_place, q.is_contiguous(), packed, head, tables, rest, size.value,
                                     None if out is None else (_span(q), _span(out), _strides(q) == _strides(out))))
        (q_ok, out_ok), like_q, packed, head, tables, rest, need, spans = found
        qp, o = q.data_ptr(), out
        if out is None or not out_ok or out.data_ptr() % 16 or out.is_neg():
            o = torch.empty_like(q) if like_q else torch.empty(q.shape, dtype=q.dtype, device=q.device)
            if out is not None:
                head = (*head[:3], *packed)
        else:
            _written(out)
            op = out.data_ptr()
            # rows of out over other rows of q, which may be read after they are written
            q_ok = q_ok and not (qp < op + spans[1] and op < qp + spans[0] and not (qp == op and spans[2]))
        if not q_ok or qp % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            head = (*packed, *head[3:])
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
        ws = q.new_empty((need + 1) // 2) if need else None      # of the call's own, as attend's
        self._launch(self._lib.kitty_cache8_shared_attention, _SHARED.pack(
            q.data_ptr(), o.data_ptr(), 0 if lse is None else lse.data_ptr(), *head, prefix_table.data_ptr(), tables[0],
            prefix_lens.data_ptr(), block_table.data_ptr(), tables[1], lens.data_ptr(),
            0 if q_lens is None else q_lens.data_ptr(), *rest, 0 if ws is None else ws.data_ptr(), need))
        if out is not None and o is not out:
            out.copy_(o)
            o = out
        return (o, lse) if return_lse else o

    def _check_weights(self, weights: torch.Tensor, B: int) -> None:
        _need(weights.dtype == torch.float32 and weights.dim() == 3 and tuple(weights.shape[:2]) == (B, self.num_kv_heads)
              and (weights.shape[2] <= 1 or weights.stride(2) == 1),
              f"weights must be float32 ({B}, {self.num_kv_heads}, N) with contiguous tokens")
        self._here("weights", weights)
        _need(weights.shape[2] <= 1 << 30, "weights must be of at most 2^30 tokens")

    def attend_weighed(self, q: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor,
                       q_lens: Optional[torch.Tensor] = None, causal: bool = True, sm_scale: Optional[float] = None,
                       out: Optional[torch.Tensor] = None, return_lse: bool = False, max_tokens: Optional[int] = None):
        """``attend`` that also adds to weights[b, h, j] (B, H, N) float32, for the tokens
        j < lens[b], what token j of KV head h got: the softmax weights of the rows of the
        head's group, summed over the queries that see it.  ``evict`` goes by such sums.

        Weights behind lens[b], or of tokens that no query sees, stay as they are, and
        tokens from N on have none; a row whose softmax is NaN makes what it sees NaN.  To
        weigh the tokens by a prompt's last queries alone, pass those (they are causal to
        what the cache holds); the sums repeat bit for bit.  The other arguments are
        ``attend``'s."""
        if calls_followed():
            raise NotImplementedError(_FOLLOWED)
        if q.requires_grad or q.is_neg():
            q = _given(q, "q")
        if out is not None:
            _into(out)
        if weights.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("weights need a gradient and the 8-bit cache has no backward: call under torch.no_grad()")
        causal, sm_scale = bool(causal), None if sm_scale is None else float(sm_scale)
        max_tokens = 0 if max_tokens is None else int(max_tokens)
        sig = ("weighed", q.shape, q.stride(), q.dtype, q.device, _sig(block_table), _sig(lens), _sig(weights), _sig(q_lens),
               causal, sm_scale, _sig(out), max_tokens, weights.is_neg())
        found = self._known.get(sig) if self._on_device else None
        if found is None:
            scale = self._check_queries(q, out, sm_scale)
            B, Hq, T, _ = q.shape
            self._check_table(block_table, B)
            self._i32("lens", lens, B)
            self._i32("q_lens", q_lens, B, optional=True)
            self._check_weights(weights, B)
            _need(not weights.is_neg(), "weights must not be a negated view")
            _need(_rows_apart(weights), "weights must not share memory between sequences or heads")
            _need(0 <= max_tokens < 1 << 31, "max_tokens must be in [0, 2^31)")
            if B == 0 or T == 0 or not self._on_device:
                o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
                lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device)
                if B and T:
                    cpu8.attend(self.key, self.value, self.scale, q.contiguous(), block_table, lens, q_lens, causal, scale, o, lse,
                                weights)
                return (o, lse) if return_lse else o
            in_place = q.stride(3) == 1 and _aligned16(q), out is None or _aligned16(out)
            o = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else out
            # copies of rows that the kernel does not read or write in place are contiguous
            packed = tuple(0 if n == 1 else s for n, s in zip((B, Hq, T), (Hq * T * self.head_dim, T * self.head_dim, self.head_dim)))
            head = (*(_strides(q) if in_place[0] else packed), *(_strides(o) if in_place[1] else packed))
            rest = (B, Hq, T, block_table.shape[1], max_tokens, causal,
                    _hip.KITTY_DTYPE_F16 if q.dtype == torch.float16 else _hip.KITTY_DTYPE_BF16, scale)
            bt_stride = block_table.stride(0) if B > 1 else 0
            w = (*_strides(weights)[:2], weights.shape[2])
            size = ctypes.c_size_t(0)
            with torch.cuda.device(self._index):      # the plan is the pools' device's
                _hip.check(self._lib.kitty_cache8_weighed_attention_workspace_size(
                    self._ref, _ATTENTION.pack(0, 0, 0, *head, 0, bt_stride, 0, 0, *rest, 0, 0),
                    _WEIGHTS.pack(weights.data_ptr(), *w), ctypes.byref(size)))
            found = self._keep(sig, (in_place, q.is_contiguous(), packed, head, bt_stride, rest, w, size.value,
                                     None if out is None else (_span(q), _span(out))))
        (q_ok, out_ok), like_q, packed, head, bt_stride, rest, w, need, spans = found
        qp = q.data_ptr()
        o = out
        if out is None or not out_ok or out.data_ptr() % 16 or out.is_neg():
            o = torch.empty_like(q) if like_q else torch.empty(q.shape, dtype=q.dtype, device=q.device)
            if out is not None or not like_q:
                head = (*head[:3], *packed)
        else:
            _written(out)
            # the queries are read again after the output is written
            q_ok = q_ok and not (qp < out.data_ptr() + spans[1] and out.data_ptr() < qp + spans[0])
        if not q_ok or qp % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            qp = q.data_ptr()
            head = (*packed, *head[3:])
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
        ws = q.new_empty((need + 1) // 2)      # of the call's own, as attend's
        _written(weights)
        args = _ATTENTION.pack(qp, o.data_ptr(), 0 if lse is None else lse.data_ptr(), *head, block_table.data_ptr(), bt_stride,
                               lens.data_ptr(), 0 if q_lens is None else q_lens.data_ptr(), *rest, ws.data_ptr(), need)
        held = _WEIGHTS.pack(weights.data_ptr(), *w)
        fn = self._lib.kitty_cache8_weighed_attention
        self._launch(lambda ref, a, stream: fn(ref, a, held, stream), args)
        if out is not None and o is not out:
            out.copy_(o)
            o = out
        return (o, lse) if return_lse else o

    def evict(self, block_table: torch.Tensor, lens: torch.Tensor, weights: torch.Tensor, keep: int, first: int = 0,
              last: int = 0, into: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Cuts sequences of more than `keep` tokens down to that many by their weights
        (B, H, N), N at least the longest; (lengths (B,) int32, positions kept (B, H,
        min(keep, N)) int32, weights (B, H, N)), new tensors.

        Each KV head keeps tokens of its own: the first `first` (which many models lean
        on), the last `last`, and of those between the heaviest (of equal ones the
        earlier; NaN counts as heaviest).  The kept ones become tokens 0 .. of the
        sequence in their old order, in block_table's first pages, or in those of `into`
        (B, W') where given, which leaves the old pages as they are.  In place, sequences
        that are not cut keep their pages as they are.  Pages behind the new length are
        free to be used again, and attention over the new lengths goes on as before (keys
        keep the positions they were made with).  A page's scale is the largest of its
        tokens' former pages'; codes that had a smaller one are rounded again.  Positions
        behind the kept ones are -1, weights 0.

        A sequence comes back as -1 and as it was if its length is negative, or more than
        block_table or weights hold, or if a page that it would write is named once more by
        the call: `into` names pages that none of its sequences has, each once, and
        sequences that share pages they keep are cut into pages of their own."""
        if calls_followed():
            raise NotImplementedError(_FOLLOWED)
        if weights.requires_grad or weights.is_neg():
            weights = _given(weights, "weights")
        keep, first, last = int(keep), int(first), int(last)
        sig = ("evict", _sig(block_table), _sig(lens), _sig(weights), keep, first, last, _sig(into))
        found = self._known.get(sig) if self._on_device else None
        if found is None:
            _need(first >= 0 and last >= 0 and first + last <= keep < 1 << 31,
                  "first and last must not be negative, and keep at least both together and below 2^31")
            _need(block_table.dim() == 2, "block_table must be int32 (B, W)")
            B, W = block_table.shape
            self._check_table(block_table, B)
            self._i32("lens", lens, B)
            self._check_weights(weights, B)
            H, N = weights.shape[1:]
            K = min(keep, N)
            if into is not None:
                self._check_table(into, B, "into")
                _need(into.shape[1] * self.page_tokens >= min(K, W * self.page_tokens), f"into must have pages for {keep} tokens")
            strides = (*_strides(weights)[:2], block_table.stride(0) if B > 1 else 0,
                       0 if into is None or B <= 1 else into.stride(0))
            if B == 0 or not self._on_device:
                out = (torch.empty(B, dtype=torch.int32, device=self.device),
                       torch.empty(B, H, K, dtype=torch.int32, device=self.device),
                       torch.empty(B, H, N, device=self.device))
                if into is not None and into.data_ptr() == block_table.data_ptr() and strides[2] == strides[3]:
                    into = None
                if B:
                    cpu8.evict(self.key, self.value, self.scale, block_table, lens, weights, keep, first, last, into, *out)
                return out
            rest = (B, W, 0 if into is None else into.shape[1], N, keep, first, last)
            size = ctypes.c_size_t(0)
            _hip.check(self._lib.kitty_cache8_evict_workspace_size(
                self._ref, _EVICT.pack(0, 0, 0, 0, 0, 0, 0 if into is None else 16, 0, 0, 0, 0, *rest, 0, 0), ctypes.byref(size)))
            found = self._keep(sig, ((B, H, K), (B, H, N), strides, rest, size.value))
        kept_shape, shape, strides, rest, need = found
        if into is not None and into.data_ptr() == block_table.data_ptr() and strides[2] == strides[3]:
            return self.evict(block_table, lens, weights, keep, first, last)       # the same pages: in place
        out_lens = lens.new_empty(shape[0])
        kept, out_weights = lens.new_empty(kept_shape), weights.new_empty(shape)
        ws = lens.new_empty(need // 4) if need else None
        self._launch(self._lib.kitty_cache8_evict, _EVICT.pack(
            weights.data_ptr(), *strides[:2], block_table.data_ptr(), strides[2], lens.data_ptr(),
            0 if into is None else into.data_ptr(), strides[3], out_lens.data_ptr(), kept.data_ptr(), out_weights.data_ptr(),
            *rest, 0 if ws is None else ws.data_ptr(), need))
        return out_lens, kept, out_weights
