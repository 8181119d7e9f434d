"""A key/value cache held in 4 bits, and the attention that reads it (shd_kv4_* of
include/shardlm_cuda.h, which states the format and the rules of visibility).

Against the f32 cache of the model loop (the reference's, crates/v2/server/src/routes/
secure_inference.rs:2452-2471) a position takes 5/32 of the memory. Rows are quantised as they are
written, straight from the K and V shares; queries may be limited to a sliding window, the first
`sinks` positions staying visible, and a cache smaller than its sequences is then used as a ring.

Device tensors in, device tensors out, asynchronous on torch's current stream, after the context's calls
on other streams (Context.bind_stream says what holds for graphs); errors that only the
device sees (a slot outside the cache, values that the format cannot hold) surface at Context.sync().
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import Kv4CacheC, check, lib
from .runtime import Context
from .sharing import SharingError

GROUP = 32
CHUNK = 16
_F32, _I32 = torch.float32, torch.int32
_INT_MAX = 0x7FFFFFFF


def _fits(**values: int) -> None:
    """Refuses what the C entries' 32-bit arguments would cut off."""
    for name, v in values.items():
        if not -_INT_MAX <= v <= _INT_MAX:
            raise SharingError(f"{name}: {v} does not fit 32 bits")


class Kv4Cache:
    """`slots` sequences of up to `capacity` rows (rounded up to a multiple of 16) of n_kv_heads heads."""

    def __init__(self, ctx: Context, slots: int, n_kv_heads: int, capacity: int, head_dim: int, sinks: int = 0):
        if slots <= 0 or n_kv_heads <= 0 or capacity <= 0:
            raise SharingError("a cache needs at least one slot, head and row")
        if head_dim not in (64, 128):
            raise SharingError("head_dim must be 64 or 128")
        capacity = -(-capacity // CHUNK) * CHUNK
        shape = (slots, n_kv_heads, capacity)
        codes = [ctx.empty(*shape, head_dim // 2, dtype=torch.uint8) for _ in range(2)]
        params = [ctx.empty(*shape, 2, head_dim // GROUP, dtype=torch.float16) for _ in range(2)]
        self._bind(ctx, codes[0], params[0], codes[1], params[1], sinks)

    @classmethod
    def from_tensors(cls, ctx: Context, k_codes: torch.Tensor, k_params: torch.Tensor, v_codes: torch.Tensor,
                     v_params: torch.Tensor, sinks: int = 0) -> "Kv4Cache":
        """A cache over tensors that the caller holds (uint8 codes and float16 params in the format's layout)."""
        self = cls.__new__(cls)
        self._bind(ctx, k_codes, k_params, v_codes, v_params, sinks)
        return self

    def _bind(self, ctx, k_codes, k_params, v_codes, v_params, sinks):
        if k_codes.dim() != 4:
            raise SharingError("ShapeMismatch: codes are [slots, n_kv_heads, capacity, head_dim / 2]")
        slots, heads, cap, half = k_codes.shape
        for t, shape, dtype in ((k_codes, (slots, heads, cap, half), torch.uint8),
                                (v_codes, (slots, heads, cap, half), torch.uint8),
                                (k_params, (slots, heads, cap, 2, half // 16), torch.float16),
                                (v_params, (slots, heads, cap, 2, half // 16), torch.float16)):
            if t.dtype != dtype or t.device != ctx.torch_device or not t.is_contiguous():
                raise SharingError(f"expected a contiguous {dtype} tensor on {ctx.torch_device}")
            if tuple(t.shape) != shape:
                raise SharingError(f"ShapeMismatch: expected {list(shape)}, got {list(t.shape)}")
        if half not in (32, 64):
            raise SharingError("head_dim must be 64 or 128")
        if cap % CHUNK or not 0 <= sinks < cap:
            raise SharingError("capacity must be a multiple of 16 and above the sinks")
        _fits(slots=slots, n_kv_heads=heads, capacity=cap)
        self.ctx, self._device = ctx, ctx.torch_device
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.slots, self.n_kv_heads, self.capacity, self.head_dim, self.sinks = slots, heads, cap, 2 * half, sinks
        self.kv_dim = heads * 2 * half
        self._c = Kv4CacheC(k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(), slots,
                            heads, cap, 2 * half, sinks)
        self._ref = C.byref(self._c)
        self._f32 = k_params.new_empty(0, dtype=_F32)  # new_empty of a tensor is the cheapest allocation

    @property
    def device_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_params, self.v_codes, self.v_params))

    # -- argument checks (a few microseconds a call: the smallest calls take not much longer) ----------
    def _plain(self, t: torch.Tensor, shape) -> bool:
        return (t.shape == shape and t.dtype is _F32 and t.device == self._device and t.is_contiguous()
                and not t.data_ptr() & 15)

    def _rows(self, t: torch.Tensor, width: int, name: str) -> torch.Tensor:
        """f32 [rows, width] on the cache's device whose rows the kernels can read: unit column stride,
        16-byte aligned rows (anything else is copied)."""
        shape = t.shape
        if t.dtype is not _F32 or t.device != self._device:
            raise SharingError(f"{name}: expected a float32 tensor on {self._device}")
        if len(shape) != 2 or shape[1] != width or shape[0] == 0:
            raise SharingError(f"ShapeMismatch: {name}: expected [rows, {width}], got {list(shape)}")
        ld, step = t.stride()
        if step != 1 or ld < width or ld % 4 or ld > 0x7FFFFFFF or t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    def _index(self, t: torch.Tensor, rows: int, name: str) -> int:
        """Address of `rows` device int32."""
        if t.dtype is not _I32 or t.device != self._device or not t.is_contiguous():
            raise SharingError(f"{name}: expected a contiguous int32 tensor on {self._device}")
        if t.numel() != rows:
            raise SharingError(f"ShapeMismatch: {name}: expected [{rows}], got {list(t.shape)}")
        return t.data_ptr()

    def _call(self, fn, *args) -> None:
        ctx = self.ctx
        ctx.bind_stream()
        rc = fn(ctx.ptr, self._ref, *args)
        if rc:
            check(rc, ctx.ptr)

    # -- writing and reading -------------------------------------------------------------------
    def _write(self, k_client, k_server, v_client, v_server, slot, pos, slot0, pos0, values):
        width, plain = self.kv_dim, self._plain
        kc, ks, vc, vs = k_client, k_server, v_client, v_server
        shape = kc.shape
        if len(shape) == 2 and shape[1] == width and shape[0] and plain(kc, shape) and plain(vc, shape) and (
                plain(ks, shape) and plain(vs, shape) if ks is not None and vs is not None else ks is vs):
            rows, ld = shape[0], width
        else:
            kc, vc = self._rows(kc, width, "k_client"), self._rows(vc, width, "v_client")
            if (ks is None) != (vs is None):
                raise SharingError("server shares are given for K and V or for neither")
            if ks is not None:
                ks, vs = self._rows(ks, width, "k_server"), self._rows(vs, width, "v_server")
            rows, ld = kc.shape[0], kc.stride(0)
            all_ = [x for x in (kc, vc, ks, vs) if x is not None]
            if any(x.shape[0] != rows for x in all_):
                raise SharingError("ShapeMismatch: K and V shares differ in rows")
            if rows == 1:
                ld = width
            elif any(x.stride(0) != ld for x in all_):
                kc, vc, ks, vs = (None if x is None else x.contiguous() for x in (kc, vc, ks, vs))
                ld = width
        if pos is not None:
            slot, pos = self._index(slot, rows, "slot"), self._index(pos, rows, "pos")
        k = v = None
        if values:
            k, v = self._f32.new_empty(rows, width), self._f32.new_empty(rows, width)
        self._call(lib().shd_kv4_write, kc.data_ptr(), None if ks is None else ks.data_ptr(), vc.data_ptr(),
                   None if vs is None else vs.data_ptr(), ld, slot, pos, slot0, pos0, rows,
                   k.data_ptr() if values else None, v.data_ptr() if values else None)
        return (k, v) if values else None

    def write(self, k_client, k_server, v_client, v_server, *, slot: torch.Tensor, pos: torch.Tensor, values: bool = False):
        """Quantise one row for each sequence: row m goes to position pos[m] of slot[m] (device int32;
        pos[m] < 0 skips the row). Server shares None: the client's hold the values. With `values`
        returns (K, V), f32 [M, kv_dim]: what the written rows stand for."""
        return self._write(k_client, k_server, v_client, v_server, slot, pos, 0, 0, values)

    def write_prompt(self, k_client, k_server, v_client, v_server, *, slot: int, pos0: int, values: bool = False):
        """Quantise consecutive positions pos0, pos0 + 1, .. of one slot."""
        _fits(slot=slot, pos0=pos0)
        return self._write(k_client, k_server, v_client, v_server, None, None, slot, pos0, values)

    def read(self, slot: int, pos0: int, n: int):
        """Positions [pos0, pos0 + n) of a slot as (K, V), f32 [n, kv_dim]."""
        if n <= 0:
            raise SharingError("read: n must be positive")
        _fits(slot=slot, pos0=pos0, n=n)
        k, v = self._f32.new_empty(n, self.kv_dim), self._f32.new_empty(n, self.kv_dim)
        self._call(lib().shd_kv4_read, slot, pos0, n, k.data_ptr(), v.data_ptr())
        return k, v

    # -- attention -----------------------------------------------------------------------------
    def _queries(self, q, mask):
        shape = q.shape
        if len(shape) != 2 or shape[1] % self.kv_dim:
            raise SharingError(f"ShapeMismatch: q: expected [rows, heads * {self.head_dim}] with heads a multiple of "
                               f"{self.n_kv_heads}, got {list(shape)}")
        rows, width = shape
        ldq = width
        if not (rows and self._plain(q, shape)):
            q = self._rows(q, width, "q")
            ldq = q.stride(0) if rows > 1 else width
        at = None
        if mask is not None:
            if not self._plain(mask, shape):
                mask = self._rows(mask, width, "mask").contiguous()
                if mask.shape[0] != rows:
                    raise SharingError("ShapeMismatch: mask and q differ in rows")
            at = mask.data_ptr()
        # the mask is returned too: it has to live until the call
        return q, ldq, rows, width, at, mask

    def attend(self, q: torch.Tensor, *, slot: torch.Tensor, pos: torch.Tensor, window: int = 0, mask: torch.Tensor | None = None):
        """One token for each sequence: q [M, heads * head_dim] reconstructed, row m at position pos[m] of
        slot[m] (device int32), whose K/V row is written. Output shares (attn - mask, mask), or (attn, 0)."""
        _fits(window=window)
        q, ldq, rows, width, mask_at, mask = self._queries(q, mask)
        c, s = self._f32.new_empty(rows, width), self._f32.new_empty(rows, width)
        self._call(lib().shd_kv4_attn_decode, q.data_ptr(), ldq, width // self.head_dim, self._index(slot, rows, "slot"),
                   self._index(pos, rows, "pos"), rows, window, mask_at, c.data_ptr(), s.data_ptr())
        return c, s

    def attend_prompt(self, q: torch.Tensor, *, slot: int, pos0: int, window: int = 0, mask: torch.Tensor | None = None):
        """Consecutive positions pos0, pos0 + 1, .. of one slot, all of whose K/V rows are written."""
        _fits(slot=slot, pos0=pos0, window=window)
        q, ldq, rows, width, mask_at, mask = self._queries(q, mask)
        c, s = self._f32.new_empty(rows, width), self._f32.new_empty(rows, width)
        self._call(lib().shd_kv4_attn_prefill, q.data_ptr(), ldq, width // self.head_dim, slot, pos0, rows, window, mask_at,
                   c.data_ptr(), s.data_ptr())
        return c, s
