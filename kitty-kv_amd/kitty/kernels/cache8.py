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
from typing import Optional, Tuple, Union

import torch

from .. import _hip
from . import cpu8
from .ops import _need, calls_followed

_SRC = {torch.float16: _hip.KITTY_SRC_F16, torch.bfloat16: _hip.KITTY_SRC_BF16, torch.float32: _hip.KITTY_SRC_F32}
_PAGE_TOKENS = (16, 32, 64, 128, 256)


def _i32(t: Optional[torch.Tensor], B: int, name: str, dev: torch.device) -> int:
    """Address of an int32 (B,) tensor on the cache's device (0 for None)."""
    if t is None:
        return 0
    _need(t.dtype == torch.int32 and t.dim() == 1 and t.shape[0] == B and (B <= 1 or t.stride(0) == 1),
          f"{name} must be int32 ({B},)")
    if t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, the cache on {dev}")
    return t.data_ptr()


def _table(t: torch.Tensor, B: int, dev: torch.device) -> Tuple[int, int, int]:
    """(address, row stride, page numbers) of a block table."""
    _need(t.dtype == torch.int32 and t.dim() == 2 and t.shape[0] == B and (t.shape[1] <= 1 or t.stride(1) == 1),
          f"block_table must be int32 ({B}, W) with contiguous rows")
    if t.device != dev:
        raise RuntimeError(f"block_table is on {t.device}, the cache on {dev}")
    return t.data_ptr(), t.stride(0) if B > 1 else 0, t.shape[1]


def _plain(t: torch.Tensor, name: str, dev: torch.device) -> torch.Tensor:
    """`t` as a kernel may read it by pointer, channels next to each other."""
    if t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, the cache on {dev}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{name} needs a gradient and the 8-bit cache has no backward: call under torch.no_grad()")
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _strides(t: torch.Tensor) -> Tuple[int, ...]:
    """Strides of the first three dimensions, 0 where a dimension has one entry."""
    return tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3]))


def _rows16(t: torch.Tensor) -> Tuple[torch.Tensor, Tuple[int, ...]]:
    """A 16-bit tensor with 16-byte aligned rows (a copy if it has none), and its strides."""
    s = _strides(t)
    if s[0] % 8 or s[1] % 8 or s[2] % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s = _strides(t)
    return t, s


class Cache8:
    """Pools of an 8-bit paged cache and the calls that work on them.

    key, value: (P, H, G, D) float8_e4m3fn (or uint8, the same bytes); scale:
    (P, H, 2) float32, of keys and of values.  G is 16, 32, 64, 128 or 256, D a
    multiple of 16 up to 256; pages and heads may lie at any 16-byte aligned
    strides.  Code c of a page stands for c * scale; pages written elsewhere may
    hold any finite positive scale.  One pool serves any number of sequences:
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
        self._ws: dict = {}      # workspace bytes by the shapes they depend on
        # a batch of none: what the library refuses of the pools, it refuses here
        _hip.check(self._lib.kitty_cache8_write(self._ref, ctypes.byref(_hip.Cache8RowsArgs()), None))

    @classmethod
    def empty(cls, num_pages: int, num_kv_heads: int, head_dim: int, page_tokens: int = 128,
              device: Union[str, torch.device] = "cuda:0") -> "Cache8":
        """A cache with pools of its own, zeroed."""
        shape = (num_pages, num_kv_heads, page_tokens, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
        return cls(k, v, torch.ones(num_pages, num_kv_heads, 2, device=device))

    # ------------------------------------------------------------------ calls
    def _launch(self, fn, args) -> None:
        """`fn` on the current stream of the pools' device."""
        if torch._C._cuda_getDevice() != self._index:
            with torch.cuda.device(self._index):
                _hip.check(fn(self._ref, ctypes.byref(args), _hip.stream_ptr(self.device)))
        else:
            _hip.check(fn(self._ref, ctypes.byref(args), _hip.stream_ptr(self.device)))

    @staticmethod
    def _followed() -> None:
        if calls_followed():
            raise NotImplementedError("calls of the 8-bit cache cannot be traced, compiled or transformed")

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
        self._followed()
        _need(key.dim() == 4 and key.shape[1] == self.num_kv_heads and key.shape[3] == self.head_dim,
              f"key must be (B, {self.num_kv_heads}, T, {self.head_dim})")
        _need(value.shape == key.shape and value.dtype == key.dtype, "value must have key's shape and dtype")
        _need(key.dtype in _SRC, "key and value must be float16, bfloat16 or float32")
        B, _, T, _ = key.shape
        dev = self.device
        key, value = _plain(key, "key", dev), _plain(value, "value", dev)
        bt, bt_stride, W = _table(block_table, B, dev)
        _need(start is not None, "start must be given")
        start_p, lens_p = _i32(start, B, "start", dev), _i32(lens, B, "lens", dev)
        if B == 0 or T == 0:
            return
        if not self._on_device:
            cpu8.write(self.key, self.value, self.scale, key, value, block_table, start, lens)
            return
        self._launch(self._lib.kitty_cache8_write, _hip.Cache8RowsArgs(
            key.data_ptr(), value.data_ptr(), *_strides(key), *_strides(value), bt, bt_stride, start_p, lens_p, B, T, W,
            _SRC[key.dtype]))

    def read(self, block_table: torch.Tensor, lens: torch.Tensor, tokens: int, start: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.float16,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(keys, values), each (B, H, tokens, D) of `dtype` (or the tensors of
        `out`): row t is token start[b] + t (start None: from 0) of sequence b,
        code * scale rounded once; 0 behind its lens[b] tokens, NaN where the
        token has no page."""
        self._followed()
        tokens = int(tokens)
        _need(tokens >= 0, "tokens must not be negative")
        _need(block_table.dim() == 2, "block_table must be int32 (B, W)")
        B, dev = block_table.shape[0], self.device
        bt, bt_stride, W = _table(block_table, B, dev)
        _need(lens is not None, "lens must be given")
        lens_p, start_p = _i32(lens, B, "lens", dev), _i32(start, B, "start", dev)
        shape = (B, self.num_kv_heads, tokens, self.head_dim)
        if out is None:
            _need(dtype in _SRC, "dtype must be float16, bfloat16 or float32")
            out = (torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev))
        else:
            for t in out:
                _need(tuple(t.shape) == shape and t.dtype == out[0].dtype and t.dtype in _SRC and t.device == dev
                      and t.stride(3) == 1, f"out must be two {shape} tensors of one type with contiguous channels")
        k, v = out
        if B == 0 or tokens == 0:
            return k, v
        if not self._on_device:
            cpu8.read(self.key, self.value, self.scale, block_table, lens, start, (k, v))
        else:
            self._launch(self._lib.kitty_cache8_read, _hip.Cache8RowsArgs(
                k.data_ptr(), v.data_ptr(), *_strides(k), *_strides(v), bt, bt_stride, start_p, lens_p, B, tokens, W,
                _SRC[k.dtype]))
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
        (default: what the table can hold); it only chooses how the work is split."""
        self._followed()
        _need(q.dim() == 4 and q.shape[3] == self.head_dim, f"q must be (B, Hq, T, {self.head_dim})")
        _need(q.dtype in (torch.float16, torch.bfloat16), "q must be float16 or bfloat16")
        B, Hq, T, D = q.shape
        _need(Hq > 0 and Hq % self.num_kv_heads == 0, f"q heads must be a positive multiple of {self.num_kv_heads}")
        dev = self.device
        q = _plain(q, "q", dev)
        bt, bt_stride, W = _table(block_table, B, dev)
        _need(lens is not None, "lens must be given")
        lens_p, q_lens_p = _i32(lens, B, "lens", dev), _i32(q_lens, B, "q_lens", dev)
        scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
        _need(0.0 < scale <= 1e30, "sm_scale must be positive and finite")
        plan = 0 if max_tokens is None else int(max_tokens)
        _need(0 <= plan < 1 << 31, "max_tokens must be in [0, 2^31)")
        if out is None:
            out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=dev)
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == dev and out.stride(3) == 1,
              "out must have q's shape, dtype and device and contiguous channels")
        lse = torch.empty((B, Hq, T), dtype=torch.float32, device=dev) if return_lse else None
        if B and T:
            if not self._on_device:
                cpu8.attend(self.key, self.value, self.scale, q, block_table, lens, q_lens, bool(causal), scale, out,
                            torch.empty(B, Hq, T) if lse is None else lse)
            else:
                self._attend(q, out, lse, bt, bt_stride, W, lens_p, q_lens_p, plan, bool(causal), scale)
        return (out, lse) if return_lse else out

    def _attend(self, q: torch.Tensor, out: torch.Tensor, lse: Optional[torch.Tensor], bt: int, bt_stride: int, W: int,
                lens: int, q_lens: int, plan: int, causal: bool, scale: float) -> None:
        B, Hq, T, _ = q.shape
        q, qs = _rows16(q)
        o, os = out, _strides(out)
        if os[0] % 8 or os[1] % 8 or os[2] % 8 or o.data_ptr() % 16:
            o = torch.empty(out.shape, dtype=out.dtype, device=out.device)
            os = _strides(o)
        a = _hip.Cache8AttentionArgs(
            q.data_ptr(), o.data_ptr(), _hip.ptr(lse), *qs, *os, bt, bt_stride, lens, q_lens, B, Hq, T, W, plan,
            causal, _hip.KITTY_DTYPE_F16 if q.dtype == torch.float16 else _hip.KITTY_DTYPE_BF16, scale)
        shape = (B, Hq, T, W, plan)
        need = self._ws.get(shape)
        if need is None:
            size = ctypes.c_size_t(0)
            _hip.check(self._lib.kitty_cache8_attention_workspace_size(self._ref, ctypes.byref(a), ctypes.byref(size)))
            if len(self._ws) >= 256:
                self._ws.clear()
            need = self._ws[shape] = size.value
        # a workspace of the call's own, from torch's allocator on its stream: calls
        # on other streams and in captured graphs never share one
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        self._launch(self._lib.kitty_cache8_attention, a)
        if o is not out:
            out.copy_(o)
