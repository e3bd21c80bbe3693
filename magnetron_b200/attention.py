"""The operators between a layer's q/k/v projections and its output projection, over the C ABI: head norm with the rotation of
positions, the paged KV cache as it is written and read back, and the attention of new tokens over it.

    cache = KVCache(0, BFLOAT16, pages=4096, page_size=32, kv_heads=8, head_dim=128, bits=8)
    batch = KVBatch.from_lists(0, q_lens=[1, 1, 700], kv_lens=[900, 31, 700], tables=[[...], [...], [...]])
    qk_norm_rope(q, k, rope, q, k, q_weight=wq, k_weight=wk)
    kv_cache_write(cache, batch, k, v)
    out = paged_attention(q, cache, batch)

The objects here are headers: device pointers and sizes, made once and used for as many calls as their buffers live. They free
what they allocated themselves and nothing that they were given. The semantics are those of include/magnetron_b200.h.
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from . import KVBatchStruct, KVCacheStruct, MagB200Error, RopeStruct, Tensor, check, lib


class DeviceArray:
    """A host array copied to the device (block tables, lengths, positions, frequencies)."""

    def __init__(self, device: int, array: np.ndarray):
        array = np.ascontiguousarray(array)
        self.device, self.ptr, self.dtype, self.size = device, None, array.dtype, array.size
        p = C.c_void_p()
        check(lib().magb200_malloc(device, C.byref(p), max(array.nbytes, 1)))
        self.ptr = p.value
        self.update(array)

    def update(self, array: np.ndarray) -> None:
        """Other contents of the same type and at most the size that was allocated, in stream order."""
        array = np.ascontiguousarray(array)
        if array.dtype != self.dtype or array.size > self.size:
            raise ValueError(f"DeviceArray of {self.size} {self.dtype}: {array.size} {array.dtype} do not fit")
        check(lib().magb200_upload(self.device, self.ptr, array.ctypes.data, array.nbytes))

    def __del__(self):
        if self.ptr:
            try:
                lib().magb200_free(self.device, self.ptr)
            except Exception:
                pass


def _pointer(x, dtype, count: int, what: str):
    """The device pointer behind x. Of a DeviceArray the type and the size are known, so they are checked."""
    if not isinstance(x, DeviceArray):
        return x
    if x.dtype != dtype or x.size < count:
        raise ValueError(f"{what}: {count} {np.dtype(dtype)} expected, the array holds {x.size} {x.dtype}")
    return x.ptr


def _device_of(arrays):
    """The device of those that are DeviceArrays; None if none is."""
    devices = {x.device for x in arrays if isinstance(x, DeviceArray)}
    if len(devices) > 1:
        raise ValueError(f"arrays of the devices {sorted(devices)} in one header")
    return devices.pop() if devices else None


class KVCache:
    """A paged KV cache (magb200_kv_cache_t): K and V pools of [pages][kv_heads][page_size][head_dim], with bits=8 e4m3 codes and
    an exponent per row. Pools are allocated, uninitialised, unless device pointers are given."""

    def __init__(self, device: int, dtype: int, pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 16, *,
                 k: int | None = None, v: int | None = None, k_exp: int | None = None, v_exp: int | None = None):
        self.device, self._owned = device, []
        rows = pages * kv_heads * page_size
        size = rows * head_dim * bits // 8
        given = [k, v] + ([k_exp, v_exp] if bits == 8 else [])
        if any(p is None for p in given):
            if any(p is not None for p in given):
                raise ValueError("KVCache: either all pools are given or none")
            for i, n in enumerate([size, size] + [rows, rows] * (bits == 8)):
                p = C.c_void_p()
                check(lib().magb200_malloc(device, C.byref(p), n))
                self._owned.append(p.value)
                given[i] = p.value
        given += [None, None]
        self.struct = KVCacheStruct(given[0], given[1], given[2], given[3], pages, dtype, bits, page_size, kv_heads, head_dim, 0)
        self.header = C.byref(self.struct)
        self.scale = max(1, head_dim) ** -0.5

    def __del__(self):
        for p in self._owned:
            try:
                lib().magb200_free(self.device, p)
            except Exception:
                pass


class KVBatch:
    """The sequences of a call (magb200_kv_batch_t). `cu_q`, `kv_len` and `pages` are device pointers or DeviceArrays of int32;
    their contents may change between calls, `max_q` and `max_kv` bound them."""

    def __init__(self, batch: int, max_pages: int, *, cu_q, kv_len, pages, max_q: int = 0, max_kv: int = 0):
        self.arrays = (cu_q, kv_len, pages)
        self.device = _device_of(self.arrays)               # of arrays that are no plain pointers
        self.struct = KVBatchStruct(batch, max_pages, max_q, max_kv, _pointer(cu_q, np.int32, batch + 1, "cu_q"),
                                    _pointer(kv_len, np.int32, batch, "kv_len"), _pointer(pages, np.int32, batch * max_pages, "pages"))
        self.header = C.byref(self.struct)

    @classmethod
    def from_lists(cls, device: int, q_lens: Sequence[int], kv_lens: Sequence[int], tables: Sequence[Sequence[int]]) -> "KVBatch":
        if not len(q_lens) == len(kv_lens) == len(tables) > 0 or min(q_lens) < 0 or min(kv_lens) < 0:
            raise ValueError("KVBatch: a number of new tokens, a length and a table for each sequence")
        width = max([1] + [len(t) for t in tables])
        table = np.full((len(tables), width), -1, dtype=np.int32)
        for b, t in enumerate(tables):
            table[b, :len(t)] = t
        cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        return cls(len(q_lens), width, cu_q=DeviceArray(device, cu), kv_len=DeviceArray(device, np.asarray(kv_lens, dtype=np.int32)),
                   pages=DeviceArray(device, table), max_q=max(q_lens), max_kv=max(kv_lens))


class Rope:
    """Rotation of positions (magb200_rope_t): `positions` int32 per token, `inv_freq` float32 per pair, both on the device."""

    def __init__(self, positions, inv_freq, rotary_dim: int, *, interleaved: bool = False, factor: float = 1.0):
        self.arrays = (positions, inv_freq)
        self.device = _device_of(self.arrays)
        self.struct = RopeStruct(_pointer(positions, np.int32, 0, "positions"), _pointer(inv_freq, np.float32, rotary_dim // 2, "inv_freq"),
                                 rotary_dim, int(interleaved), factor, 0)
        self.header = C.byref(self.struct)
        self.tokens = positions.size if isinstance(positions, DeviceArray) else 1 << 62     # positions known to be there


# A decode step makes these calls once per layer and token, so they do nothing but pass headers on: the arguments' structs are made
# once, the functions are looked up once, and the status is compared here.
_bound = {}
_APART = "the tensors and arrays of a call lie on one device"


def _call(name: str, *args) -> None:
    f = _bound.get(name)
    if f is None:
        f = _bound[name] = getattr(lib(), name)
    code = f(*args)
    if code:
        raise MagB200Error(code, lib().magb200_last_error().decode(errors="replace"))


def qk_norm_rope(q: Tensor, k: Tensor | None, rope: Rope | None, q_out: Tensor | None = None, k_out: Tensor | None = None, *,
                 q_weight: Tensor | None = None, k_weight: Tensor | None = None, eps: float = 1e-6):
    """rotate(rmsnorm(x) * weight) of the heads of q and k; results go to q_out and k_out (new tensors unless given; may be q and k)."""
    if q_out is None:
        q_out = Tensor(q.device, q.dtype, q.shape)
    if k_out is None and k is not None:
        k_out = Tensor(k.device, k.dtype, k.shape)
    d = q.device
    if q_out.device != d or (k is not None and (k.device != d or k_out.device != d)) or (q_weight is not None and q_weight.device != d) or (
            k_weight is not None and k_weight.device != d) or (rope is not None and rope.device not in (None, d)):
        raise ValueError(_APART)
    if rope is not None and rope.tokens < q.shape[0]:
        raise ValueError(f"qk_norm_rope: {rope.tokens} positions for {q.shape[0]} tokens")
    _call("magb200_qk_norm_rope", d, q.header(), k and k.header(), q_weight and q_weight.header(), k_weight and k_weight.header(), eps,
          rope and rope.header, q_out.header(), k_out and k_out.header())
    return q_out, k_out


def kv_cache_write(cache: KVCache, batch: KVBatch, k: Tensor, v: Tensor) -> None:
    """Puts the rows of the batch's new tokens into the cache."""
    if not cache.device == k.device == v.device or batch.device not in (None, cache.device):
        raise ValueError(_APART)
    _call("magb200_kv_cache_write", cache.device, cache.header, batch.header, k.header(), v.header())


def kv_cache_read(cache: KVCache, batch: KVBatch, cu_kv, k: Tensor, v: Tensor) -> None:
    """Fills rows cu_kv[b] .. cu_kv[b + 1] - 1 of k and v with the first cached tokens of sequence b."""
    if not cache.device == k.device == v.device or batch.device not in (None, cache.device) or (
            isinstance(cu_kv, DeviceArray) and cu_kv.device != cache.device):
        raise ValueError(_APART)
    _call("magb200_kv_cache_read", cache.device, cache.header, batch.header, _pointer(cu_kv, np.int32, batch.struct.batch + 1, "cu_kv"), k.header(), v.header())


def paged_attention(q: Tensor, cache: KVCache, batch: KVBatch, out: Tensor | None = None, *, lse: Tensor | None = None,
                    scale: float | None = None, causal: bool = True, window: int = 0) -> Tensor:
    """softmax(scale * q K^T + mask) V of the batch's new tokens over their cached ones; scale is head_dim ** -0.5 unless given."""
    if out is None:
        out = Tensor(q.device, q.dtype, q.shape)
    if not cache.device == q.device == out.device or (lse is not None and lse.device != q.device) or batch.device not in (None, q.device):
        raise ValueError(_APART)
    _call("magb200_paged_attention", cache.device, q.header(), cache.header, batch.header, cache.scale if scale is None else scale, causal, window,
          out.header(), lse and lse.header())
    return out
