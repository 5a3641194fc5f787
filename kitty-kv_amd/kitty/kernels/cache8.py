"""The 8-bit paged cache: written token by token or in chunks, read back, and
attended over by one or many queries.

A layer that 2 bits cost too much (and that has no room for 16) keeps its keys
and values in e4m3 with one float32 scale per page, head and stream.  Unlike the
2-bit pages, whose tokens wait in 16-bit buffers until a page is full, tokens go
into their page as they come: the page's scale is a power of two that rises when
a larger token arrives, and its older codes are rounded again to the new scale.

Device tensors run the HIP kernels of csrc/cache8.hip and csrc/attend8*.hip, CPU
tensors the torch code of ``kernels.cpu8``.  No call waits for the GPU, reads a
length on the host or keeps state of its own, so calls may be captured into a
graph and replayed with other lengths and tables in the same tensors.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional, Tuple, Union

import torch

from .. import _hip
from . import cpu8
from .ops import _need, calls_followed

_SRC = {torch.float16: _hip.KITTY_SRC_F16, torch.bfloat16: _hip.KITTY_SRC_BF16, torch.float32: _hip.KITTY_SRC_F32}
_PAGE_TOKENS = (16, 32, 64, 128, 256)
# kitty_cache8_write_args / _read_args and kitty_cache8_attention_args as the C
# compiler lays them out (packing one takes a quarter of a ctypes structure's time)
_ROWS = struct.Struct("2P6qPq2P4i")
_ATTENTION = struct.Struct("3P6qPq2P7ifPN")


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

    def _check_table(self, t: torch.Tensor, B: int) -> None:
        _need(t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == B and (t.shape[1] <= 1 or t.stride(1) == 1),
              f"block_table must be int32 ({B}, W) with contiguous rows")
        self._here("block_table", t)

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
                    _need(torch._debug_has_internal_overlap(t) != 1, "out must not share memory between its rows")
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
                _need(torch._debug_has_internal_overlap(out) != 1, "out must not share memory between its rows")
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
