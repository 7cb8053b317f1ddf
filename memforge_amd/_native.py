"""ctypes binding of ``libmemforge_hip.so`` (the C ABI in ``include/memforge_hip.h``).

This module is the only place Python touches the device library. Every
function takes torch tensors that already live on the GPU, passes their data
pointers and element strides to the C entry point on torch's current stream,
and raises if the library is missing, a tensor is on the wrong device, or the
entry point returns an error status. There is no fallback path: the data path
runs on the MI355X or not at all.
"""

from __future__ import annotations

import ctypes
import threading
from collections import OrderedDict
from dataclasses import dataclass
from pathlib import Path
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

LIB_PATH = Path(__file__).resolve().with_name("libmemforge_hip.so")

MF_F32, MF_F16, MF_BF16 = 0, 1, 2
DTYPE_CODES = {torch.float32: MF_F32, torch.float16: MF_F16, torch.bfloat16: MF_BF16}

PLAN_ITEM_INTS = 12
PLAN_MERGE_INTS = 8
SLICE_INTS = 8
SLICE_MAX_TILES = 512
SLICE_MAX_SEGMENTS = 64
SLICE_MIN_TILES = 64
SLICE_WAVES_PER_CU = 4
# 16-key tiles one wave of a plan may cover (MF_MAX_ITEM_TILES in
# paged_attention.hip); a cooperative unit of four waves covers four times that
MAX_ITEM_TILES = 128
ENTRY_INTS = 6

PACK_TABLE_OVERFLOW = 1
PACK_NEGATIVE_POSITION = 2
PACK_DUPLICATE_SLOT = 4
PACK_BAD_ENTRY = 8
PACK_ROW_COUNT = 16
PACK_BLOCK_OUT_OF_POOL = 32

_c_int, _c_i64, _c_f32, _vp = ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p

_SIGNATURES = {
    "mf_version": (ctypes.c_char_p, []),
    "mf_last_hip_error": (_c_int, []),
    "mf_status_string": (ctypes.c_char_p, [_c_int]),
    "mf_kv_write": (_c_int, [_vp, _vp, _c_int, _c_i64, _c_i64, _vp, _c_i64, _vp, _vp, _c_int,
                             _c_i64, _c_i64, _c_i64, _c_int, _c_i64, _c_int, _c_int, _vp]),
    "mf_kv_gather": (_c_int, [_vp, _vp, _c_int, _c_i64, _c_i64, _c_i64, _c_int, _c_i64, _vp, _c_i64,
                              _vp, _vp, _c_int, _c_i64, _c_i64, _c_int, _c_int, _vp]),
    "mf_kv_copy_blocks": (_c_int, [_vp, _vp, _c_int, _c_int, _c_i64, _c_i64, _c_i64, _c_i64, _vp,
                                   _c_int, _vp]),
    "mf_ragged_pack": (_c_int, [_vp, _c_int, _vp, _c_i64, _vp, _c_i64, _c_int, _c_int, _c_i64, _vp,
                                _vp, _vp, _vp, _vp, _vp, _vp, _vp, _c_i64, _vp, _vp]),
    "mf_paged_attention": (_c_int, [
        _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _c_i64, _c_i64,
        _c_int, _vp, _c_i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _c_i64, _c_i64, _c_int, _c_int,
        _c_int, _c_f32, _vp, _c_i64, _c_i64, _vp, _c_i64, _vp, _c_i64, _vp, _vp]),
    "mf_paged_attention_counted": (_c_int, [
        _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _c_i64, _c_i64,
        _c_int, _vp, _c_i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _c_i64, _c_i64, _c_int, _c_int,
        _c_int, _c_f32, _vp, _c_i64, _c_i64, _vp, _c_i64, _vp, _vp, _c_i64, _vp]),
    "mf_paged_attention_kv_write": (_c_int, [
        _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _c_i64, _c_i64,
        _c_int, _vp, _c_i64, _vp, _vp, _vp, _vp, _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64,
        _c_int, _c_int, _c_int, _c_f32, _vp, _c_i64, _c_i64, _vp, _c_i64, _vp, _vp, _c_i64, _vp]),
    "mf_paged_attention_scored": (_c_int, [
        _vp, _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _c_i64, _c_i64,
        _c_int, _vp, _c_i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64,
        _c_int, _c_int, _c_int, _c_f32, _vp, _c_i64, _c_i64, _vp, _c_i64, _vp, _vp, _c_i64, _vp]),
    "mf_kv4_write": (_c_int, [_vp, _vp, _c_int, _c_i64, _c_i64, _vp, _c_i64, _vp, _vp]),
    "mf_kv4_gather": (_c_int, [_vp, _vp, _c_i64, _vp, _vp, _c_int, _c_i64, _c_i64, _vp]),
    "mf_paged_attention4": (_c_int, [
        _vp, _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _vp, _vp, _vp, _vp, _c_int,
        _c_f32, _vp, _c_i64, _c_i64, _vp, _c_i64, _vp, _vp, _c_i64, _vp]),
    "mf_paged_attention_noalloc": (_c_int, [
        _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _c_i64, _c_i64,
        _c_int, _vp, _c_i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _c_i64, _c_i64, _c_int, _c_int,
        _c_int, _c_f32, _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _vp]),
    "mf_attention_plan": (_c_int, [_c_int, _vp, _vp, _c_int, _c_int, _c_int, _c_int, _c_int,
                                   _vp, _c_i64, _vp, _c_i64, _vp]),
    "mf_attention_plan_device": (_c_int, [_c_int, _vp, _vp, _c_int, _c_int, _c_int, _c_int, _c_int,
                                          _vp, _c_i64, _vp, _c_i64, _vp]),
    "mf_attention_plan_merge_free": (_c_int, [_c_int, _vp, _vp, _c_int, _c_int, _c_int, _c_int, _c_int,
                                              _vp, _c_i64, _vp, _c_i64, _vp]),
    "mf_attention_plan4": (_c_int, [_c_int, _vp, _vp, _c_int, _c_int, _c_int, _c_int, _c_int,
                                    _vp, _c_i64, _vp, _c_i64, _vp]),
    "mf_attention_plan_slices": (_c_int, [_c_int, _vp, _vp, _c_int, _c_int, _c_int, _c_int, _c_int,
                                          _c_int, _vp, _c_i64, _vp, _c_i64, _vp]),
    "mf_paged_attention_slices": (_c_int, [
        _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _c_i64, _c_i64,
        _c_int, _vp, _c_i64, _vp, _vp, _vp, _c_int, _c_int, _c_int, _c_f32, _vp, _c_i64, _c_i64,
        _vp, _c_i64, _vp, _c_i64, _vp]),
    "mf_spec_verify_workspace_size": (_c_i64, [_c_int, _c_int]),
    "mf_spec_verify": (_c_int, [_c_int, _c_int, _c_int, _vp, _vp, _c_i64, _c_i64, _vp, _c_int,
                                _c_i64, _c_i64, _c_f32, _c_int, _vp, _vp, _c_i64, _vp, _vp, _vp,
                                _vp, _vp, _c_i64, _vp]),
    "mf_tables_extend": (_c_int, [_vp, _c_i64, _c_int, _vp, _vp, _vp, _c_i64, _vp, _vp, _c_int, _c_int, _c_i64,
                                  _vp, _c_i64, _c_int, _vp, _vp, _vp, _vp, _vp, _vp, _vp]),
    "mf_tables_truncate": (_c_int, [_vp, _c_i64, _c_int, _vp, _vp, _vp, _c_i64, _vp, _vp, _c_int, _c_int, _vp, _vp]),
    "mf_tree_accept": (_c_int, [_vp, _vp, _vp, _vp, _c_int, _c_i64, _c_int, _vp, _vp, _vp, _vp]),
    "mf_sample": (_c_int, [_vp, _c_int, _c_i64, _c_int, _c_int, _vp, _vp, _c_f32, _vp, _c_int, _vp, _c_f32, _vp,
                           _c_f32, _vp, _vp, _c_int, _vp, _c_i64, _vp]),
    "mf_sample_workspace_size": (_c_i64, [_c_int, _c_int, _c_int]),
    "mf_tree_plan_sizes": (_c_int, [_c_int, _c_i64, _c_int, _c_int, _c_int, _c_int, _c_int, _c_int, _vp, _vp]),
    "mf_tree_plan": (_c_int, [_vp, _vp, _vp, _c_int, _c_i64, _c_int, _c_i64, _c_int, _c_int, _c_int, _c_int, _c_int,
                              _vp, _c_i64, _vp, _vp]),
    "mf_tree_attention": (_c_int, [
        _vp, _c_i64, _c_i64, _vp, _c_i64, _c_i64, _c_int, _vp, _vp, _c_i64, _c_i64, _c_i64, _c_int, _c_i64, _vp, _c_i64,
        _vp, _vp, _c_i64, _c_i64, _c_int, _c_i64, _c_int, _c_int, _c_int, _c_int, _c_f32, _c_int, _vp, _c_i64, _vp,
        _c_i64, _vp]),
}

_LIB: Optional[ctypes.CDLL] = None


def exported_symbols() -> Tuple[str, ...]:
    return tuple(_SIGNATURES)


def lib() -> ctypes.CDLL:
    """The loaded device library; raises if it has not been built."""
    global _LIB
    if _LIB is None:
        if not LIB_PATH.exists():
            raise RuntimeError(
                f"{LIB_PATH.name} is not built; run `python -m memforge_amd._build` "
                "(memforge_amd has no CPU fallback)"
            )
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, (restype, argtypes) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = restype
            fn.argtypes = argtypes
        _LIB = handle
    return _LIB


class MemforgeHipError(RuntimeError):
    """A device entry point rejected its arguments or failed to launch."""


def _check(status: int, what: str) -> None:
    if status != 0:
        L = lib()
        msg = L.mf_status_string(status).decode()
        raise MemforgeHipError(f"{what}: {msg} (status {status}, hip error {L.mf_last_hip_error()})")


def _stream(device: Optional[torch.device] = None) -> int:
    """Raw handle of the current HIP stream of ``device`` (default: the current
    device) -- the stream torch's own kernels are queued on, also under
    ``torch.cuda.stream`` and graph capture. The raw query costs about 0.1 us
    against 3 us for building a ``torch.cuda.Stream`` object."""
    if device is None or device.index is None:
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())
    return torch._C._cuda_getCurrentRawStream(device.index)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def require_device(*tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError(
                f"memforge_amd runs on the GPU; got a tensor on {t.device} "
                "(there is no CPU path)"
            )


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return DTYPE_CODES[dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {dtype}; expected float32, float16 or bfloat16") from None


# --------------------------------------------------------------- pool views

@dataclass(frozen=True)
class PoolView:
    """One layer of a paged K or V pool as the C ABI addresses it."""

    k: torch.Tensor  # tensor whose data_ptr is the layer base
    v: torch.Tensor
    stride_block: int
    stride_slot: int
    stride_head: int
    block_size: int
    num_heads: int
    head_dim: int

    @property
    def num_blocks(self) -> int:
        return int(self.k.shape[0])

    @property
    def num_slots(self) -> int:
        """Token slots of the layer; the kernels skip slots outside [0, num_slots)."""
        return int(self.k.shape[0]) * self.block_size

    @staticmethod
    def from_bshd(k: torch.Tensor, v: torch.Tensor) -> "PoolView":
        """``(blocks, slots, heads, dim)`` -- one layer of PagedKVPool."""
        if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
            raise ValueError("K and V pools must share shape, strides and dtype")
        if k.stride(-1) != 1:
            raise ValueError("pool head_dim axis must be contiguous")
        n, bs, h, d = k.shape
        return PoolView(k, v, k.stride(0), k.stride(1), k.stride(2), bs, h, d)

    @staticmethod
    def from_bhsd(k: torch.Tensor, v: torch.Tensor) -> "PoolView":
        """``(blocks, heads, slots, dim)`` -- PagedKVCache's per-head layout."""
        if k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype:
            raise ValueError("K and V pools must share shape, strides and dtype")
        if k.stride(-1) != 1:
            raise ValueError("pool head_dim axis must be contiguous")
        n, h, bs, d = k.shape
        return PoolView(k, v, k.stride(0), k.stride(2), k.stride(1), bs, h, d)


class _Pool4Struct(ctypes.Structure):
    _fields_ = [("key_codes", _vp), ("key_scales", _vp), ("value_codes", _vp), ("value_scales", _vp),
                ("num_blocks", _c_i64), ("block_size", _c_int), ("num_heads", _c_int), ("head_dim", _c_int),
                ("dtype", _c_int)]


GROUP4 = 32  # elements of a 4-bit pool that share a scale
HEAD_DIMS4 = (32, 64, 128, 256)


class Pool4View:
    """One layer of a pool held in 4 bits (mf_pool4): int32 ``key_codes`` (blocks,
    heads, slots, head_dim / 8) and ``value_codes`` (blocks, heads, head_dim / 8,
    slots), uint8 ``key_scales`` (blocks, heads, slots, head_dim / 32) and
    ``value_scales`` (blocks, heads, head_dim / 32, slots), all contiguous.
    ``dtype`` is the type attention over it runs in."""

    def __init__(self, key_codes: torch.Tensor, key_scales: torch.Tensor, value_codes: torch.Tensor,
                 value_scales: torch.Tensor, dtype: torch.dtype):
        n, h, bs, words = key_codes.shape
        want = ((key_codes, torch.int32, (n, h, bs, words)), (key_scales, torch.uint8, (n, h, bs, words // 4)),
                (value_codes, torch.int32, (n, h, words, bs)), (value_scales, torch.uint8, (n, h, words // 4, bs)))
        for x, dt, shape in want:
            if x.dtype != dt or tuple(x.shape) != shape or not x.is_contiguous() or x.device != key_codes.device:
                raise ValueError(f"a 4-bit pool layer needs a contiguous {dt} tensor of {shape} on one device, got "
                                 f"{x.dtype} {tuple(x.shape)} on {x.device}")
        if 8 * words not in HEAD_DIMS4:
            raise ValueError(f"a 4-bit pool holds head_dims {HEAD_DIMS4}, got {8 * words}")
        if bs % 16 or bs > 512:
            raise ValueError(f"a 4-bit pool's block_size is a multiple of 16 up to 512, got {bs}")
        self.key_codes, self.key_scales = key_codes, key_scales
        self.value_codes, self.value_scales = value_codes, value_scales
        self.dtype = dtype
        self.num_blocks, self.num_heads, self.block_size, self.head_dim = n, h, bs, 8 * words
        self.device = key_codes.device
        self.struct = _Pool4Struct(_ptr(key_codes), _ptr(key_scales), _ptr(value_codes), _ptr(value_scales), n, bs, h,
                                   8 * words, dtype_code(dtype))
        self.address = ctypes.addressof(self.struct)

    @property
    def num_slots(self) -> int:
        return self.num_blocks * self.block_size


def kv_bits(pool) -> int:
    """4 for a pool object that holds its keys and values in 4 bits, 16 for any other
    (a caller's own class need not say)."""
    return getattr(pool, "kv_bits", 16)


def kv_dtype(pool) -> torch.dtype:
    """The type attention over a pool object runs in: its elements', or what a 4-bit one names."""
    return pool.spec.dtype if kv_bits(pool) == 4 else pool.key_pool.dtype


def kv_device(pool) -> torch.device:
    """Where a pool object's memory lies (its spec may name a kind of device alone)."""
    return (pool.key_codes if kv_bits(pool) == 4 else pool.key_pool).device


def same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Same shape and the same strides on every axis longer than one (the
    stride of a length-one axis is never used to address an element)."""
    return a.shape == b.shape and all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n > 1)


def _rows_ok(t: torch.Tensor, name: str) -> None:
    if t.dim() != 3:
        raise ValueError(f"{name} must be a (tokens, heads, head_dim) view, got {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} head_dim axis must be contiguous")


# ----------------------------------------------------------- KV write/gather

def kv_write(k_rows: torch.Tensor, v_rows: torch.Tensor, slots: torch.Tensor, pool: PoolView) -> None:
    """Scatter (T, H, D) rows into pool slots ``slots`` (int64, device)."""
    _rows_ok(k_rows, "k_rows")
    _rows_ok(v_rows, "v_rows")
    if not same_layout(k_rows, v_rows):
        v_rows = v_rows.contiguous()
        k_rows = k_rows.contiguous()
    require_device(k_rows, v_rows, slots, pool.k)
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    T, H, D = k_rows.shape
    if H != pool.num_heads or D != pool.head_dim or slots.numel() != T:
        raise ValueError(
            f"rows {tuple(k_rows.shape)} / {slots.numel()} slots do not match a pool of "
            f"{pool.num_heads} heads x {pool.head_dim}"
        )
    _check(lib().mf_kv_write(
        _ptr(k_rows), _ptr(v_rows), dtype_code(k_rows.dtype), k_rows.stride(0), k_rows.stride(1),
        _ptr(slots), T, _ptr(pool.k), _ptr(pool.v), dtype_code(pool.k.dtype),
        pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size, pool.num_slots, H, D,
        _stream(k_rows.device),
    ), "mf_kv_write")


def kv_gather(pool: PoolView, slots: torch.Tensor, k_rows: torch.Tensor, v_rows: torch.Tensor) -> None:
    """Copy pool slots ``slots`` into preallocated (T, H, D) rows."""
    _rows_ok(k_rows, "k_rows")
    _rows_ok(v_rows, "v_rows")
    if not same_layout(k_rows, v_rows):
        raise ValueError("k_rows and v_rows must share strides")
    require_device(k_rows, v_rows, slots, pool.k)
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    T, H, D = k_rows.shape
    _check(lib().mf_kv_gather(
        _ptr(pool.k), _ptr(pool.v), dtype_code(pool.k.dtype), pool.stride_block, pool.stride_slot,
        pool.stride_head, pool.block_size, pool.num_slots, _ptr(slots), T, _ptr(k_rows), _ptr(v_rows),
        dtype_code(k_rows.dtype), k_rows.stride(0), k_rows.stride(1), H, D, _stream(k_rows.device),
    ), "mf_kv_gather")


def _slots4(slots: torch.Tensor, pool: Pool4View) -> torch.Tensor:
    if slots.dtype != torch.int64 or not slots.is_contiguous():
        slots = slots.to(torch.int64).contiguous()
    if slots.get_device() != pool.device.index:
        raise ValueError(f"slots are on {slots.device}, the pool on {pool.device}")
    return slots


def _check_rows4(k: torch.Tensor, v: torch.Tensor, tokens: int, heads: int, dim: int, num_slots: int,
                 pool: Pool4View) -> None:
    if k.get_device() != pool.device.index or v.get_device() != pool.device.index:
        raise ValueError(f"rows are on {k.device} / {v.device}, the pool on {pool.device}")
    if k.shape != v.shape or k.dtype != v.dtype or tokens != num_slots or heads != pool.num_heads \
            or dim != pool.head_dim:
        raise ValueError(f"rows {tuple(k.shape)} / {tuple(v.shape)} of {k.dtype} / {v.dtype} and {num_slots} slots do "
                         f"not match a pool of {pool.num_heads} heads x {pool.head_dim}")


def kv4_write(k_rows: torch.Tensor, v_rows: torch.Tensor, slots: torch.Tensor, pool: Pool4View) -> None:
    """Round (T, H, D) rows to 4 bits into the pool slots ``slots`` (int64, device,
    distinct; a slot outside the pool skips its row)."""
    _rows_ok(k_rows, "k_rows")
    _rows_ok(v_rows, "v_rows")
    slots = _slots4(slots, pool)
    n = slots.numel()
    _check_rows4(k_rows, v_rows, *k_rows.shape, n, pool)
    if not same_layout(k_rows, v_rows):
        k_rows, v_rows = k_rows.contiguous(), v_rows.contiguous()
    _launch(pool.device, "mf_kv4_write", lib().mf_kv4_write, k_rows.data_ptr(), v_rows.data_ptr(),
            dtype_code(k_rows.dtype), k_rows.stride(0), k_rows.stride(1), slots.data_ptr(), n, pool.address)


def kv4_write_states(keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor, pool: Pool4View) -> None:
    """``kv4_write`` of a layer's ``(1, H, T, D)`` key and value states, as they are laid out."""
    if keys.dim() != 4 or keys.shape[0] != 1:
        raise ValueError(f"expected (1, heads, tokens, head_dim) states, got {tuple(keys.shape)}")
    if keys.stride() != values.stride() or keys.stride(3) != 1:
        return kv4_write(keys[0].permute(1, 0, 2).contiguous(), values[0].permute(1, 0, 2).contiguous(), slots, pool)
    slots = _slots4(slots, pool)
    n = slots.numel()
    _, h, tokens, d = keys.shape
    _check_rows4(keys, values, tokens, h, d, n, pool)
    _launch(pool.device, "mf_kv4_write", lib().mf_kv4_write, keys.data_ptr(), values.data_ptr(),
            dtype_code(keys.dtype), keys.stride(2), keys.stride(1), slots.data_ptr(), n, pool.address)


def kv4_gather(pool: Pool4View, slots: torch.Tensor, k_rows: torch.Tensor, v_rows: torch.Tensor) -> None:
    """The values that pool slots ``slots`` stand for, into preallocated (T, H, D) rows."""
    _rows_ok(k_rows, "k_rows")
    _rows_ok(v_rows, "v_rows")
    slots = _slots4(slots, pool)
    n = slots.numel()
    _check_rows4(k_rows, v_rows, *k_rows.shape, n, pool)
    if not same_layout(k_rows, v_rows):
        raise ValueError("k_rows and v_rows must share strides")
    _launch(pool.device, "mf_kv4_gather", lib().mf_kv4_gather, pool.address, slots.data_ptr(), n, k_rows.data_ptr(),
            v_rows.data_ptr(), dtype_code(k_rows.dtype), k_rows.stride(0), k_rows.stride(1))


def kv4_gather_states(pool: Pool4View, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of ``slots`` as new contiguous ``(1, H, T, D)`` keys and values in the pool's dtype."""
    slots = _slots4(slots, pool)
    n, h, d = slots.numel(), pool.num_heads, pool.head_dim
    k = torch.empty((1, h, n, d), dtype=pool.dtype, device=pool.device)
    v = torch.empty((1, h, n, d), dtype=pool.dtype, device=pool.device)
    _launch(pool.device, "mf_kv4_gather", lib().mf_kv4_gather, pool.address, slots.data_ptr(), n, k.data_ptr(),
            v.data_ptr(), dtype_code(pool.dtype), d, n * d)
    return k, v


def kv_copy_blocks(key_pool: torch.Tensor, value_pool: torch.Tensor,
                   pairs: Sequence[Tuple[int, int]]) -> None:
    """Copy block ``src`` to ``dst`` for every pair, in every layer of the
    ``(layers, blocks, slots, heads, dim)`` K and V pools (one launch per 32
    pairs; the pairs go in the kernel arguments)."""
    if key_pool.dim() != 5 or key_pool.shape != value_pool.shape:
        raise ValueError("block copy needs (layers, blocks, slots, heads, dim) K and V pools")
    if key_pool.stride() != value_pool.stride() or key_pool.dtype != value_pool.dtype:
        raise ValueError("K and V pools must share strides and dtype")
    L, N, bs, H, D = key_pool.shape
    if key_pool.stride()[2:] != (H * D, D, 1):
        raise ValueError("each block of a pool layer must be contiguous")
    require_device(key_pool, value_pool)
    flat = np.ascontiguousarray(np.asarray(list(pairs), dtype=np.int64).reshape(-1, 2))
    _check(lib().mf_kv_copy_blocks(
        _ptr(key_pool), _ptr(value_pool), dtype_code(key_pool.dtype), L, key_pool.stride(0),
        key_pool.stride(1), bs * H * D, N, flat.ctypes.data, flat.shape[0], _stream(key_pool.device),
    ), "mf_kv_copy_blocks")


# ------------------------------------------------------------------ uploads

def _layout(parts: Sequence[np.ndarray]) -> Tuple[List[np.ndarray], List[int], int]:
    """Contiguous copies of the parts, each part's int32-word offset (even, so
    int64 parts land on 8-byte boundaries) and the total word count."""
    arrs, offs, n = [], [], 0
    for p in parts:
        a = np.ascontiguousarray(p)
        if a.dtype not in (np.int32, np.int64):
            raise TypeError(f"upload takes int32/int64 arrays, got {a.dtype}")
        n = (n + 1) & ~1
        offs.append(n)
        n += a.size * a.itemsize // 4
        arrs.append(a)
    return arrs, offs, max(n, 2)


def _views(buf: torch.Tensor, arrs: Sequence[np.ndarray], offs: Sequence[int]) -> List[torch.Tensor]:
    out = []
    for a, o in zip(arrs, offs):
        t = buf[o:o + a.size * a.itemsize // 4]
        if a.dtype == np.int64:
            t = t.view(torch.int64)
        out.append(t.view(a.shape))
    return out


def _pack_host(parts: Sequence[np.ndarray], pinned: bool) -> Tuple[torch.Tensor, List[np.ndarray], List[int]]:
    """The parts packed into one int32 host tensor (pinned if asked), each on
    an 8-byte boundary: (tensor, contiguous parts, word offsets)."""
    arrs, offs, n = _layout(parts)
    host = torch.empty(n, dtype=torch.int32, pin_memory=pinned)
    h = host.numpy()
    for a, o in zip(arrs, offs):
        h[o:o + a.size * a.itemsize // 4] = a.reshape(-1).view(np.int32)
    return host, arrs, offs


def _refuse_capture(device: torch.device) -> None:
    """Uploads stage through a temporary pinned buffer that a captured copy
    would read again on every replay, after torch's host allocator has handed
    it out again; torch's pinned allocation is not permitted under capture
    anyway. Captured steps stage through buffers of their own
    (GraphedPagedDecoder, CountedPlan)."""
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise MemforgeHipError("host arrays cannot be uploaded under graph capture: stage them through "
                               "persistent buffers (GraphedPagedDecoder, CountedPlan) and capture those")


def upload_packed(parts: Sequence[np.ndarray], device) -> Tuple[torch.Tensor, List[int]]:
    """``upload`` without the per-part views: the device int32 buffer and each
    part's word offset in it (for callers that pass addresses to the C ABI)."""
    _refuse_capture(torch.device(device))
    host, _, offs = _pack_host(parts, True)
    buf = torch.empty(host.numel(), dtype=torch.int32, device=device)
    buf.copy_(host, non_blocking=True)
    return buf, offs


# upload_packed_cached: device buffers by their exact contents, device and
# stream, most recent last
_UPLOAD_CACHE: "OrderedDict[tuple, Tuple[torch.Tensor, List[int]]]" = OrderedDict()
UPLOAD_CACHE_SIZE = 64
UPLOAD_CACHE_MAX_WORDS = 1 << 18  # 1 MiB: at most 64 MiB of device memory held


def upload_packed_cached(parts: Sequence[np.ndarray], device) -> Tuple[torch.Tensor, List[int]]:
    """``upload_packed`` that hands back the buffer an earlier call made from
    the same bytes on the same device and stream (a model calling the
    attention operator once per layer sends the same tables, plan and
    positions for every layer of a step). The kernels only read these
    buffers, so sharing one between launches on its stream is safe; the key
    holds the stream, so no buffer is read on a stream its upload was not
    ordered before. Refused under graph capture, like every upload."""
    dev = torch.device(device)
    arrs, offs, words = _layout(parts)
    _refuse_capture(dev)  # a cached buffer could be evicted while a graph still replays
    if words > UPLOAD_CACHE_MAX_WORDS:  # a large launch amortises its own upload
        return upload_packed(arrs, dev)
    key = (dev.type, dev.index, _stream(dev) if dev.type == "cuda" else 0,
           tuple((a.dtype.str, a.shape) for a in arrs), b"".join(a.tobytes() for a in arrs))
    hit = _UPLOAD_CACHE.get(key)
    if hit is not None:
        _UPLOAD_CACHE.move_to_end(key)
        return hit
    made = upload_packed(arrs, dev)
    _UPLOAD_CACHE[key] = made
    if len(_UPLOAD_CACHE) > UPLOAD_CACHE_SIZE:
        _UPLOAD_CACHE.popitem(last=False)
    return made


def upload(parts: Sequence[np.ndarray], device) -> List[torch.Tensor]:
    """Move int32 / int64 host arrays to ``device`` with ONE host-to-device
    copy: they are packed into a pinned buffer (each part on an 8-byte
    boundary), copied asynchronously into a fresh device buffer on the current
    stream, and handed back as views with their own dtype and shape. The
    pinned buffer comes from torch's caching host allocator, which does not
    hand it out again before the copy has completed, so the host never waits
    for the GPU here."""
    dev = torch.device(device)
    _refuse_capture(dev)
    pinned = dev.type == "cuda"
    host, arrs, offs = _pack_host(parts, pinned)
    if not pinned:
        return _views(host.to(dev), arrs, offs)
    buf = torch.empty(host.numel(), dtype=torch.int32, device=dev)
    buf.copy_(host, non_blocking=True)
    return _views(buf, arrs, offs)


# ------------------------------------------------------------ scored attention

class _ScoringStruct(ctypes.Structure):
    _fields_ = [("softcap", _c_f32), ("slopes", _vp), ("first_keys", _vp), ("prefix_lens", _vp)]


@dataclass(frozen=True)
class Scoring:
    """What a model does to the scores of its attention (mf_scoring), for
    ``paged_attention`` and ``paged_attention_kv_write``:

    * ``softcap``: scores t become ``softcap * tanh(t / softcap)``; 0 for none.
    * ``slopes`` (fp32, one per query head): then ``slopes[h] * |position - key|``
      is subtracted.
    * ``first_keys`` (int32, one per sequence of the call): keys before it are not
      seen. A document mask runs every document's rows as a sequence of their own
      over the same block table.
    * ``prefix_lens`` (int32, one per sequence): keys before it are seen by every
      row, those after the row's position too (from ``first_keys`` on).

    A row that sees no key gets zeros, except in a sequence whose ``kv_lens`` entry is
    0: those rows are not in the plan and stay as they were. Plans for masked calls are made with the
    same ``first_keys`` and ``prefix_lens`` as host lists (``plan_attention``).
    Keys that no row of a sequence sees may hold anything; a value that is not
    finite reaches the rows of its sequence that do not see it too, as zero times
    it does in a product (a plain call's rows the same)."""

    softcap: float = 0.0
    slopes: Optional[torch.Tensor] = None
    first_keys: Optional[torch.Tensor] = None
    prefix_lens: Optional[torch.Tensor] = None

    def __post_init__(self):
        cap = 0.0 if self.softcap is None else float(self.softcap)
        held = ctypes.c_float(cap).value  # what the launch takes: a cap that vanishes there would be none
        if not 0.0 <= cap or not held < float("inf") or (cap > 0.0 and held == 0.0):
            raise ValueError(f"softcap must be finite and not negative in 32 bits, got {self.softcap}")
        object.__setattr__(self, "softcap", cap)

    @property
    def active(self) -> bool:
        return self.softcap > 0.0 or self.slopes is not None or self.first_keys is not None \
            or self.prefix_lens is not None

    def struct(self, num_q_heads: int, num_seqs: int, device: torch.device) -> _ScoringStruct:
        """The C structure, its tensors checked against the call."""
        for name, x, dt, n in (("slopes", self.slopes, torch.float32, num_q_heads),
                               ("first_keys", self.first_keys, torch.int32, num_seqs),
                               ("prefix_lens", self.prefix_lens, torch.int32, num_seqs)):
            if x is None:
                continue
            if x.dtype != dt or not x.is_contiguous() or x.numel() != n:
                raise TypeError(f"{name} must be a contiguous {dt} tensor of {n}, got {x.dtype} {tuple(x.shape)}")
            if x.device != device:
                raise ValueError(f"{name} is on {x.device}, the query on {device}")
        return _ScoringStruct(self.softcap, _ptr(self.slopes), _ptr(self.first_keys), _ptr(self.prefix_lens))


def _scored(scoring: Optional[Scoring]) -> Optional[Scoring]:
    return scoring if scoring is not None and scoring.active else None


# ---------------------------------------------------------------- attention

@dataclass
class AttentionPlan:
    """Work list for one mf_paged_attention call (valid for its dtype/head_dim)."""

    items: torch.Tensor      # int32 device, (n_items, PLAN_ITEM_INTS); slice plans: (n_slices + n_segments, SLICE_INTS)
    merges: torch.Tensor     # int32 device, (n_merges, PLAN_MERGE_INTS)
    n_narrow: int            # slice plans: slices
    n_wide: int              # slice plans: segments
    n_merges: int
    partials_floats: int
    items_host: np.ndarray
    merges_host: np.ndarray
    sliced: bool = False     # a decode slice plan (mf_attention_plan_slices)


def plan_attention_host(cu_seqlens: Sequence[int], kv_lens: Sequence[int], num_q_heads: int,
                        num_kv_heads: int, head_dim: int, dtype: torch.dtype,
                        partition_tiles: int = 0, num_cus: int = 0, merge_free: bool = False,
                        kv_bits: int = 16) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """mf_attention_plan on host arrays: (items [n, PLAN_ITEM_INTS], merges
    [m, PLAN_MERGE_INTS], counts [n_narrow, n_wide, n_merges, partials_floats]).
    With ``num_cus`` and no ``partition_tiles``, mf_attention_plan_device: the
    ranges cut for a GPU of that many compute units; with ``merge_free`` as well,
    mf_attention_plan_merge_free, which does not cut decode ranges for it; with
    ``kv_bits`` 4, mf_attention_plan4, which cuts them for a 4-bit pool."""
    cu = np.ascontiguousarray(np.asarray(cu_seqlens, dtype=np.int32))
    kv = np.ascontiguousarray(np.asarray(kv_lens, dtype=np.int32))
    B = kv.shape[0]
    if cu.shape[0] != B + 1:
        raise ValueError("cu_seqlens must have one more entry than kv_lens")
    counts = np.zeros(4, dtype=np.int64)
    L = lib()
    args = [B, cu.ctypes.data, kv.ctypes.data, num_q_heads, num_kv_heads, head_dim, dtype_code(dtype)]
    device = num_cus > 0 and partition_tiles <= 0
    plan = L.mf_attention_plan if not device else \
        L.mf_attention_plan_merge_free if merge_free else \
        L.mf_attention_plan4 if kv_bits == 4 else L.mf_attention_plan_device
    args.append(num_cus if device else partition_tiles)
    # One planner call when the plan fits the largest one seen so far (the
    # planner fills every row it reports); otherwise it reports the sizes and
    # a second call fills arrays of exactly that size.
    cap_items, cap_merges = _PLAN_CAPACITY
    items = np.empty((cap_items, PLAN_ITEM_INTS), dtype=np.int32)
    merges = np.empty((cap_merges, PLAN_MERGE_INTS), dtype=np.int32)
    st = plan(*args, items.ctypes.data, cap_items, merges.ctypes.data, cap_merges, counts.ctypes.data)
    if st == -3:  # MF_ERR_WORKSPACE: counts holds the sizes
        n_items, n_merges = int(counts[0] + counts[1]), int(counts[2])
        _PLAN_CAPACITY[0] = max(cap_items, min(n_items, 1 << 16))
        _PLAN_CAPACITY[1] = max(cap_merges, min(n_merges, 1 << 14))
        items = np.empty((max(n_items, 1), PLAN_ITEM_INTS), dtype=np.int32)
        merges = np.empty((max(n_merges, 1), PLAN_MERGE_INTS), dtype=np.int32)
        st = plan(*args, items.ctypes.data, n_items, merges.ctypes.data, n_merges, counts.ctypes.data)
    _check(st, "mf_attention_plan")
    n_items = int(counts[0] + counts[1])
    n_merges = int(counts[2])
    return items[:n_items], merges[:n_merges], counts


# host array sizes for a one-call plan, grown to the largest plan seen
_PLAN_CAPACITY = [256, 64]


def plan_upload_parts(items: np.ndarray, merges: np.ndarray) -> List[np.ndarray]:
    """The two arrays a plan puts on the device (at least one row each)."""
    return [items if items.shape[0] else np.zeros((1, PLAN_ITEM_INTS), np.int32),
            merges if merges.shape[0] else np.zeros((1, PLAN_MERGE_INTS), np.int32)]


def plan_from_parts(items: np.ndarray, merges: np.ndarray, counts: np.ndarray,
                    dev_items: torch.Tensor, dev_merges: torch.Tensor, sliced: bool = False) -> AttentionPlan:
    return AttentionPlan(dev_items, dev_merges, int(counts[0]), int(counts[1]), int(counts[2]),
                         int(counts[3]), items, merges, sliced)


def plan_slices_host(cu_seqlens: Sequence[int], kv_lens: Sequence[int], num_q_heads: int,
                     num_kv_heads: int, head_dim: int, dtype: torch.dtype, num_cus: int,
                     min_tiles: int = SLICE_MIN_TILES) -> Optional[Tuple[np.ndarray, np.ndarray, np.ndarray]]:
    """mf_attention_plan_slices on host arrays for a GPU of ``num_cus``
    compute units: (slices [n_slices + n_segments, SLICE_INTS], merges [m,
    PLAN_MERGE_INTS], counts [n_slices, n_segments, n_merges,
    partials_floats]), or None when the launch does not qualify (not a pure
    decode step, or fewer than ``min_tiles`` tiles per wave of one round)."""
    cu = np.ascontiguousarray(np.asarray(cu_seqlens, dtype=np.int32))
    kv = np.ascontiguousarray(np.asarray(kv_lens, dtype=np.int32))
    B = kv.shape[0]
    if cu.shape[0] != B + 1:
        raise ValueError("cu_seqlens must have one more entry than kv_lens")
    counts = np.zeros(4, dtype=np.int64)
    L = lib()
    args = (B, cu.ctypes.data, kv.ctypes.data, num_q_heads, num_kv_heads, head_dim, dtype_code(dtype),
            int(num_cus), int(min_tiles))
    st = L.mf_attention_plan_slices(*args, None, 0, None, 0, counts.ctypes.data)
    if st == -2:  # MF_ERR_UNSUPPORTED: not a decode step this plan form serves
        return None
    if st not in (0, -3):
        _check(st, "mf_attention_plan_slices")
    if counts[0] == 0:
        return None
    n_rec, n_merges = int(counts[0] + counts[1]), int(counts[2])
    slices = np.empty((n_rec, SLICE_INTS), dtype=np.int32)
    merges = np.empty((max(n_merges, 1), PLAN_MERGE_INTS), dtype=np.int32)
    _check(L.mf_attention_plan_slices(*args, slices.ctypes.data, n_rec, merges.ctypes.data, n_merges,
                                      counts.ctypes.data), "mf_attention_plan_slices")
    return slices, merges[:n_merges], counts


_DEVICE_CUS = {}


def device_cus(device) -> int:
    """Compute units of ``device`` (a slice plan's size is set by it)."""
    dev = torch.device(device)
    index = dev.index if dev.index is not None else torch.cuda.current_device()
    cus = _DEVICE_CUS.get(index)
    if cus is None:
        cus = _DEVICE_CUS[index] = torch.cuda.get_device_properties(index).multi_processor_count
    return cus


# plan_host results by their inputs, most recent last. The planners are pure
# functions of them, and a model that calls the attention operator once per
# layer asks for the same plan in every layer of a step. The arrays are handed
# out read-only, so no caller can change what a later hit returns.
_PLAN_CACHE: "OrderedDict[tuple, tuple]" = OrderedDict()
PLAN_CACHE_SIZE = 64


def _plan_from_first_keys(plan, cu_seqlens: Sequence[int], kv_lens: Sequence[int], first_keys: Sequence[int]):
    """``plan(kv_lens)``'s arrays for sequences whose keys before ``first_keys``
    no row sees: planned as contexts that begin at the first key's 16-key tile,
    then moved there. A sequence all of whose keys are hidden keeps its last
    tile, so that its rows are written (with zeros)."""
    kv = np.asarray(kv_lens, dtype=np.int64)
    tile = np.clip(np.asarray(first_keys, dtype=np.int64), 0, np.maximum(kv - 1, 0)) // 16
    items, merges, counts = plan((kv - 16 * tile).tolist())
    items = items.copy()
    live = items[:, 9] > 0
    at = tile[items[:, 0]] * live
    items[:, 4] += at.astype(np.int32)
    items[:, 5] += at.astype(np.int32)
    items[:, 10] += (16 * at).astype(np.int32)
    return items, merges, counts


def plan_host(cu_seqlens: Sequence[int], kv_lens: Sequence[int], num_q_heads: int, num_kv_heads: int,
              head_dim: int, dtype: torch.dtype, device=None, partition_tiles: int = 0,
              decode_slices: bool = False, first_keys: Optional[Sequence[int]] = None,
              prefix_lens: Optional[Sequence[int]] = None,
              kv_bits: int = 16) -> Tuple[np.ndarray, np.ndarray, np.ndarray, bool]:
    """Host plan arrays (items or slices, merges, counts) and whether they are
    a slice plan. With ``decode_slices`` (the caller's launch has 16-token
    blocks, no row map and no in-flight keys) a decode step large enough to
    fill the GPU on ``device`` more than once gets a slice plan; every other
    call, and an explicit ``partition_tiles``, the per-range plan.
    ``first_keys`` / ``prefix_lens`` (per sequence): the masks of a scored call
    (``Scoring``); tiles below a sequence's first key are not planned. ``kv_bits``:
    4 for a pool held in 4 bits."""
    on_gpu = partition_tiles <= 0 and device is not None and torch.device(device).type == "cuda"
    masked = first_keys is not None or prefix_lens is not None
    for name, x in (("first_keys", first_keys), ("prefix_lens", prefix_lens)):
        if x is not None and len(x) != len(kv_lens):
            raise ValueError(f"{len(x)} {name} for {len(kv_lens)} sequences")
    if prefix_lens is not None and not on_gpu and partition_tiles <= 0:
        raise ValueError("a plan for prefix_lens is made for a GPU device (or with partition_tiles): other plans leave "
                         "out tiles that only a prefix makes visible")
    slices = decode_slices and on_gpu and not masked and kv_bits == 16
    cus = device_cus(device) if on_gpu else 0
    firsts = None if first_keys is None else tuple(int(x) for x in first_keys)
    prefixes = None if prefix_lens is None else tuple(int(x) for x in prefix_lens)
    key = (tuple(int(x) for x in cu_seqlens), tuple(int(x) for x in kv_lens), num_q_heads, num_kv_heads,
           head_dim, dtype, partition_tiles, cus, slices, firsts, prefixes, kv_bits)
    hit = _PLAN_CACHE.get(key)
    if hit is not None:
        _PLAN_CACHE.move_to_end(key)
        return hit
    made = plan_slices_host(cu_seqlens, kv_lens, num_q_heads, num_kv_heads, head_dim, dtype, cus) if slices else None
    if made is not None:
        out = (*made, True)
    else:
        def plan(lens):
            return plan_attention_host(cu_seqlens, lens, num_q_heads, num_kv_heads, head_dim, dtype,
                                       partition_tiles, cus, kv_bits=kv_bits)

        out = (*(plan(kv_lens) if firsts is None else _plan_from_first_keys(plan, cu_seqlens, kv_lens, firsts)),
               False)
    for a in out[:3]:
        a.flags.writeable = False
    _PLAN_CACHE[key] = out
    if len(_PLAN_CACHE) > PLAN_CACHE_SIZE:
        _PLAN_CACHE.popitem(last=False)
    return out


def plan_attention(cu_seqlens: Sequence[int], kv_lens: Sequence[int], num_q_heads: int,
                   num_kv_heads: int, head_dim: int, dtype: torch.dtype, device,
                   partition_tiles: int = 0, decode_slices: bool = False,
                   first_keys: Optional[Sequence[int]] = None, prefix_lens: Optional[Sequence[int]] = None,
                   kv_bits: int = 16) -> AttentionPlan:
    """A plan for ``paged_attention`` (``plan_host``, then one upload)."""
    items, merges, counts, sliced = plan_host(cu_seqlens, kv_lens, num_q_heads, num_kv_heads, head_dim, dtype,
                                              device, partition_tiles, decode_slices, first_keys, prefix_lens,
                                              kv_bits)
    dev_items, dev_merges = upload(plan_upload_parts(items, merges), device)
    return plan_from_parts(items, merges, counts, dev_items, dev_merges, sliced)


class CountedPlan:
    """Fixed device buffers for a plan whose counts live in device memory
    (mf_paged_attention_counted): the shapes and addresses a captured HIP
    graph recorded stay valid while ``update`` swaps in each step's plan.

    Items hold ``cap_narrow`` narrow then ``cap_wide`` wide rows, each
    capacity rounded up to whole workgroups of four (the launch's grid, whose
    waves read their items before the live-count check); ``update`` raises if
    a plan does not fit. Host staging is pinned; each update waits for the
    previous one's copies before reusing it."""

    def __init__(self, cap_narrow: int, cap_wide: int, cap_merges: int, partials_floats: int, device):
        cap_narrow, cap_wide = -(-cap_narrow // 4) * 4, -(-cap_wide // 4) * 4
        self.cap_narrow, self.cap_wide, self.cap_merges = cap_narrow, cap_wide, cap_merges
        rows = max(cap_narrow + cap_wide, 1)
        self.items = torch.zeros((rows, PLAN_ITEM_INTS), dtype=torch.int32, device=device)
        self.merges = torch.zeros((max(cap_merges, 1), PLAN_MERGE_INTS), dtype=torch.int32, device=device)
        self.counts = torch.zeros(3, dtype=torch.int32, device=device)
        self.partials = torch.empty(max(partials_floats, 1), dtype=torch.float32, device=device)
        self._h_items = torch.zeros((rows, PLAN_ITEM_INTS), dtype=torch.int32).pin_memory()
        self._h_merges = torch.zeros((max(cap_merges, 1), PLAN_MERGE_INTS), dtype=torch.int32).pin_memory()
        self._h_counts = torch.zeros(3, dtype=torch.int32).pin_memory()
        self._copied = None

    def update(self, items: np.ndarray, merges: np.ndarray, counts: np.ndarray) -> None:
        n_narrow, n_wide, n_merges, floats = (int(x) for x in counts)
        if n_narrow > self.cap_narrow or n_wide > self.cap_wide or n_merges > self.cap_merges:
            raise ValueError(f"plan ({n_narrow}, {n_wide}, {n_merges}) exceeds the capacity "
                             f"({self.cap_narrow}, {self.cap_wide}, {self.cap_merges})")
        if floats > self.partials.numel():
            raise ValueError(f"plan needs {floats} partial floats, the buffer holds {self.partials.numel()}")
        if self._copied is not None:
            self._copied.synchronize()
        hi = self._h_items.numpy()
        hi[:n_narrow] = items[:n_narrow]
        hi[self.cap_narrow:self.cap_narrow + n_wide] = items[n_narrow:n_narrow + n_wide]
        if n_merges:
            self._h_merges.numpy()[:n_merges] = merges[:n_merges]
        self._h_counts.numpy()[:] = (n_narrow, n_wide, n_merges)
        self.items.copy_(self._h_items, non_blocking=True)
        if n_merges:
            self.merges[:n_merges].copy_(self._h_merges[:n_merges], non_blocking=True)
        self.counts.copy_(self._h_counts, non_blocking=True)
        self._copied = torch.cuda.Event()
        self._copied.record()


class Workspace(threading.local):
    """Grow-only scratch for split-K partials (fp32), merge arrival counters
    (int32, kept all-zero between calls by the kernels) and the rejection
    verify, one per (device, stream) so concurrent streams never share it; likewise the
    bins of split sampling rows (int64, kept all-zero).

    Every host thread has scratch of its own too (``threading.local``: each gets
    these dictionaries when it first comes here, and they end with it). A call may be
    several launches, the C entry points run without the interpreter's lock, and
    threads share a stream unless told otherwise, so another thread's launches
    can stand between those of one call.

    A call recorded into a graph gets memory of its own, which the graph's private
    pool holds: a shared buffer would be freed under the graph when a later call
    grows it, and shared with every other graph captured on the stream; one first
    made under capture would, kept here, be handed to eager calls though nothing
    has run yet. Captures that torch does not allocate a private pool for (begun
    by other means than torch.cuda.CUDAGraph) must hand in buffers of their own."""

    def __init__(self) -> None:
        self._partials = {}
        self._counters = {}
        self._verify = {}
        self._bins = {}

    def partials(self, floats: int, device) -> Optional[torch.Tensor]:
        if floats <= 0:
            return None
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(floats, dtype=torch.float32, device=device)
        dev = torch.device(device)
        key = (dev.index, _stream(dev))
        buf = self._partials.get(key)
        if buf is None or buf.numel() < floats:
            buf = torch.empty(max(floats, 1 << 16), dtype=torch.float32, device=device)
            self._partials[key] = buf
        return buf

    def verify(self, nbytes: int, device, stream: Optional[int] = None) -> torch.Tensor:
        """mf_spec_verify's scratch, kept between calls (``stream``: the raw
        handle of the device's current stream, when the caller has it)."""
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(nbytes, dtype=torch.uint8, device=device)
        dev = device if isinstance(device, torch.device) else torch.device(device)
        key = (dev.index, _stream(dev) if stream is None else stream)
        buf = self._verify.get(key)
        if buf is None or buf.numel() < nbytes:
            buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            self._verify[key] = buf
        return buf

    def counters(self, n: int, device) -> Optional[torch.Tensor]:
        if n <= 0:
            return None
        if torch.cuda.is_current_stream_capturing():  # zeroed by a kernel that the graph replays
            return torch.zeros(n, dtype=torch.int32, device=device)
        dev = torch.device(device)
        key = (dev.index, _stream(dev))
        buf = self._counters.get(key)
        if buf is None or buf.numel() < n:
            buf = torch.zeros(max(n, 1 << 12), dtype=torch.int32, device=device)
            self._counters[key] = buf
        return buf

    def bins(self, n: int, device) -> Optional[torch.Tensor]:
        """mf_sample's words for rows split over workgroups, all zero between calls like the counters."""
        if n <= 0:
            return None
        if torch.cuda.is_current_stream_capturing():
            return torch.zeros(n, dtype=torch.int64, device=device)
        key = (device.index, _stream(device))
        buf = self._bins.get(key)
        if buf is None or buf.numel() < n:
            buf = self._bins[key] = torch.zeros(n, dtype=torch.int64, device=device)
        return buf


_WORKSPACE = Workspace()


def paged_attention(q_rows: torch.Tensor, out_rows: torch.Tensor, pool: PoolView,
                    block_tables: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                    positions: torch.Tensor, plan: AttentionPlan, scale: float,
                    num_kv_heads: int, row_map: Optional[torch.Tensor] = None,
                    pool_lens: Optional[torch.Tensor] = None,
                    new_k_rows: Optional[torch.Tensor] = None,
                    new_v_rows: Optional[torch.Tensor] = None,
                    partials: Optional[torch.Tensor] = None,
                    counters: Optional[torch.Tensor] = None, fused_merge: bool = False,
                    scoring: Optional[Scoring] = None) -> None:
    """Varlen paged attention into ``out_rows`` ((rows, Hq, D) views, device).
    ``scoring``: capped, biased or masked scores (mf_paged_attention_scored;
    per-range plans, no fused merge). ``pool``: a layer of a 16- or 32-bit pool, or
    of one held in 4 bits (``Pool4View``; mf_paged_attention4, 16-bit queries,
    per-range plans made with ``kv_bits=4``, every key in the pool).

    Split-K partitions are merged by a separate merge kernel; with
    ``fused_merge`` the attention kernel merges them itself (the last partition
    of a group to finish, through arrival counters from the workspace unless
    given) -- correct, but slower on MI355X because every arriving partition
    must release its partials with an agent-scope fence."""
    _rows_ok(q_rows, "q_rows")
    _rows_ok(out_rows, "out_rows")
    if isinstance(pool, Pool4View):
        if pool_lens is not None or fused_merge:
            raise ValueError("a 4-bit pool takes no in-flight keys or fused merge")
        return _paged_attention4(scoring, q_rows, out_rows, pool, block_tables, cu_seqlens, kv_lens, positions, plan,
                                 scale, num_kv_heads, row_map, partials)
    require_device(q_rows, out_rows, pool.k, block_tables, cu_seqlens, kv_lens, positions)
    if q_rows.dtype != pool.k.dtype or out_rows.dtype != pool.k.dtype:
        raise TypeError("query, output and pool must share a dtype")
    for name, t, dt in (("block_tables", block_tables, torch.int32), ("cu_seqlens", cu_seqlens, torch.int32),
                        ("kv_lens", kv_lens, torch.int32), ("positions", positions, torch.int64)):
        if t.dtype != dt or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous {dt} tensor")
    Hq, D = q_rows.shape[1], q_rows.shape[2]
    if _scored(scoring) is not None:
        if fused_merge:
            raise ValueError("scored attention takes no fused merge")
        return _paged_attention_scored(scoring, q_rows, out_rows, pool, block_tables, cu_seqlens, kv_lens, positions,
                                       plan, scale, num_kv_heads, row_map, pool_lens, new_k_rows, new_v_rows,
                                       partials=partials)
    if isinstance(plan, CountedPlan):
        return _paged_attention_counted(q_rows, out_rows, pool, block_tables, cu_seqlens, kv_lens, positions,
                                        plan, scale, num_kv_heads, row_map, pool_lens, new_k_rows, new_v_rows)
    if partials is None:
        partials = _WORKSPACE.partials(plan.partials_floats, q_rows.device)
    if plan.sliced:
        if row_map is not None or pool_lens is not None or fused_merge:
            raise ValueError("a slice plan takes no row map, in-flight keys or fused merge")
        bt_stride = block_tables.shape[1] if block_tables.dim() == 2 else 0
        _check(lib().mf_paged_attention_slices(
            _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
            _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
            dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
            pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
            _ptr(block_tables), bt_stride, _ptr(cu_seqlens), _ptr(kv_lens), _ptr(positions),
            Hq, num_kv_heads, D, float(scale),
            _ptr(plan.items), plan.n_narrow, plan.n_wide, _ptr(plan.merges), plan.n_merges,
            _ptr(partials), partials.numel() if partials is not None else 0, _stream(q_rows.device),
        ), "mf_paged_attention_slices")
        return
    if fused_merge and counters is None:
        counters = _WORKSPACE.counters(plan.n_merges, q_rows.device)
    if not fused_merge:
        counters = None
    nk = new_k_rows if new_k_rows is not None else None
    nv = new_v_rows if new_v_rows is not None else None
    if pool_lens is not None:
        if nk is None or nv is None:
            raise ValueError("pool_lens needs the in-flight new_k_rows/new_v_rows")
        require_device(pool_lens, nk, nv)
        if not same_layout(nk, nv):
            raise ValueError("in-flight K and V rows must share strides")
    bt_stride = block_tables.shape[1] if block_tables.dim() == 2 else 0
    _check(lib().mf_paged_attention(
        _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
        _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
        dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
        pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
        _ptr(block_tables), bt_stride, _ptr(cu_seqlens), _ptr(kv_lens), _ptr(positions),
        _ptr(row_map), _ptr(pool_lens), _ptr(nk), _ptr(nv),
        nk.stride(0) if nk is not None else 0, nk.stride(1) if nk is not None else 0,
        Hq, num_kv_heads, D, float(scale),
        _ptr(plan.items), plan.n_narrow, plan.n_wide, _ptr(plan.merges), plan.n_merges,
        _ptr(partials), partials.numel() if partials is not None else 0, _ptr(counters), _stream(q_rows.device),
    ), "mf_paged_attention")


class _Plan:
    """A plan's launch arguments: counts or capacities, the live counts and the partials."""

    __slots__ = ("narrow", "wide", "merges", "counts", "partials")

    def __init__(self, plan, device, partials: Optional[torch.Tensor] = None):
        if isinstance(plan, CountedPlan):
            self.narrow, self.wide, self.merges = plan.cap_narrow, plan.cap_wide, plan.cap_merges
            self.counts, self.partials = plan.counts, plan.partials
            return
        if plan.sliced:
            raise ValueError("scored attention takes per-range plans (mf_attention_plan)")
        if plan.items.device != device:
            raise ValueError(f"the plan is on {plan.items.device}, the query on {device}")
        self.narrow, self.wide, self.merges = plan.n_narrow, plan.n_wide, plan.n_merges
        self.counts = None
        self.partials = partials if partials is not None else _WORKSPACE.partials(plan.partials_floats, device)
        if partials is not None and (partials.dtype != torch.float32 or not partials.is_contiguous()
                                     or partials.device != device or partials.numel() < plan.partials_floats):
            raise ValueError(f"the plan needs {plan.partials_floats} contiguous fp32 partials on {device}, got "
                             f"{partials.numel()} of {partials.dtype} on {partials.device}")


def _launch(device: torch.device, what: str, fn, *args) -> None:
    """``fn(*args, stream)`` on the device's current stream, with the device current."""
    if device.index == torch.cuda.current_device():
        status = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _stream(device))
    if status:
        _check(status, what)


def _index_tensors(q_rows: torch.Tensor, block_tables, cu_seqlens, kv_lens, positions, row_map=None,
                   pool_lens=None) -> None:
    index = q_rows.get_device()
    for name, t, dt in (("block_tables", block_tables, torch.int32), ("cu_seqlens", cu_seqlens, torch.int32),
                        ("kv_lens", kv_lens, torch.int32), ("positions", positions, torch.int64),
                        ("row_map", row_map, torch.int32), ("pool_lens", pool_lens, torch.int32)):
        if t is None:
            continue
        if t.dtype != dt or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous {dt} tensor")
        if t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, the query on {q_rows.device}")


def _paged_attention_scored(scoring: Scoring, q_rows, out_rows, pool, block_tables, cu_seqlens, kv_lens, positions,
                            plan, scale, num_kv_heads, row_map=None, pool_lens=None, nk=None, nv=None,
                            slot_mapping=None, partials=None) -> None:
    dev = q_rows.device
    if pool_lens is not None:
        if nk is None or nv is None:
            raise ValueError("pool_lens needs the in-flight new_k_rows/new_v_rows")
        if pool_lens.numel() != kv_lens.numel():
            raise ValueError(f"{pool_lens.numel()} pool_lens for {kv_lens.numel()} sequences")
        for name, x in (("new_k_rows", nk), ("new_v_rows", nv)):
            _rows_ok(x, name)
            if x.dtype != pool.k.dtype or x.shape[1:] != (pool.num_heads, pool.head_dim) or x.device != dev:
                raise ValueError(f"{name} must be rows of {pool.num_heads} heads x {pool.head_dim} in {pool.k.dtype} on "
                                 f"{dev}, got {tuple(x.shape)} in {x.dtype} on {x.device}")
        if not same_layout(nk, nv):
            raise ValueError("in-flight K and V rows must share strides")
    if out_rows.shape != q_rows.shape or q_rows.shape[1:] != (q_rows.shape[1], pool.head_dim) \
            or num_kv_heads != pool.num_heads:
        raise ValueError(f"query {tuple(q_rows.shape)}, output {tuple(out_rows.shape)} and {num_kv_heads} kv heads do "
                         f"not match a pool of {pool.num_heads} heads x {pool.head_dim}")
    if not dev == out_rows.device == pool.k.device:
        raise ValueError(f"query, output and pool must be on one device, the query is on {dev}")
    _index_tensors(q_rows, block_tables, cu_seqlens, kv_lens, positions, row_map, pool_lens)
    p = _Plan(plan, dev, partials)
    mods = scoring.struct(q_rows.shape[1], kv_lens.numel(), dev)
    bt_stride = block_tables.shape[1] if block_tables.dim() == 2 else 0
    _launch(
        dev, "mf_paged_attention_scored", lib().mf_paged_attention_scored,
        ctypes.addressof(mods), _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
        _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
        dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
        pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
        _ptr(block_tables), bt_stride, _ptr(cu_seqlens), _ptr(kv_lens), _ptr(positions),
        _ptr(row_map), _ptr(pool_lens), _ptr(nk), _ptr(nv),
        nk.stride(0) if nk is not None else 0, nk.stride(1) if nk is not None else 0,
        _ptr(slot_mapping), slot_mapping.numel() if slot_mapping is not None else 0, pool.num_slots,
        q_rows.shape[1], num_kv_heads, q_rows.shape[2], float(scale),
        _ptr(plan.items), p.narrow, p.wide, _ptr(plan.merges), p.merges, _ptr(p.counts),
        _ptr(p.partials), p.partials.numel() if p.partials is not None else 0)


def _check4(q_rows, out_rows, pool: Pool4View, num_kv_heads: int) -> None:
    require_device(q_rows, out_rows, pool.key_codes)
    if not q_rows.get_device() == out_rows.get_device() == pool.device.index:
        raise ValueError("query, output and pool must be on one device")
    if pool.dtype == torch.float32:
        raise TypeError("attention over a 4-bit pool runs in float16 or bfloat16; this pool's dtype is float32")
    if q_rows.dtype != pool.dtype or out_rows.dtype != pool.dtype:
        raise TypeError(f"query and output must be of the pool's dtype {pool.dtype}")
    if num_kv_heads != pool.num_heads or q_rows.shape[2] != pool.head_dim or out_rows.shape != q_rows.shape:
        raise ValueError(f"query {tuple(q_rows.shape)}, output {tuple(out_rows.shape)} and {num_kv_heads} kv heads do "
                         f"not match a pool of {pool.num_heads} heads x {pool.head_dim}")


def _paged_attention4(scoring, q_rows, out_rows, pool: Pool4View, block_tables, cu_seqlens, kv_lens, positions, plan,
                      scale, num_kv_heads, row_map=None, partials=None) -> None:
    _check4(q_rows, out_rows, pool, num_kv_heads)
    dev = q_rows.device
    _index_tensors(q_rows, block_tables, cu_seqlens, kv_lens, positions, row_map)
    p = _Plan(plan, dev, partials)
    scoring = _scored(scoring)
    mods = scoring.struct(q_rows.shape[1], kv_lens.numel(), dev) if scoring is not None else None
    _launch(
        dev, "mf_paged_attention4", lib().mf_paged_attention4,
        ctypes.addressof(mods) if mods is not None else None,
        q_rows.data_ptr(), q_rows.stride(0), q_rows.stride(1),
        out_rows.data_ptr(), out_rows.stride(0), out_rows.stride(1),
        dtype_code(q_rows.dtype), pool.address, block_tables.data_ptr(),
        block_tables.shape[1] if block_tables.dim() == 2 else 0,
        cu_seqlens.data_ptr(), kv_lens.data_ptr(), positions.data_ptr(), _ptr(row_map), q_rows.shape[1], float(scale),
        plan.items.data_ptr(), p.narrow, p.wide, plan.merges.data_ptr(), p.merges, _ptr(p.counts),
        _ptr(p.partials), p.partials.numel() if p.partials is not None else 0)


def paged_attention_kv_write(q_rows: torch.Tensor, out_rows: torch.Tensor, pool: PoolView,
                             block_tables: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                             positions: torch.Tensor, plan, scale: float, num_kv_heads: int,
                             new_k_rows: torch.Tensor, new_v_rows: torch.Tensor,
                             slot_mapping: torch.Tensor, scoring: Optional[Scoring] = None) -> None:
    """One launch for a packed step's KV write and its attention
    (mf_paged_attention_kv_write): rows ``new_k_rows``/``new_v_rows``
    ((rows, Hkv, D) views in the pool's dtype) go to the pool through
    ``slot_mapping`` (int64; slot -1 skips a row), and every sequence's keys
    from ``kv_lens[s] - q_len[s]`` on are read from those rows instead of the
    pool. Row cu_seqlens[s] + i must be sequence s's new token at position
    kv_lens[s] - q_len[s] + i. ``plan`` is an AttentionPlan or a CountedPlan
    (graph capture). Same pool contents and output as ``kv_write`` followed by
    ``paged_attention`` (with the same ``scoring``). Not for a pool held in 4 bits,
    whose rows are rounded before anything attends to them (``kv4_write``)."""
    if isinstance(pool, Pool4View):
        raise ValueError("a 4-bit pool takes no write in the attention launch: kv4_write, then paged_attention")
    _rows_ok(q_rows, "q_rows")
    _rows_ok(out_rows, "out_rows")
    _rows_ok(new_k_rows, "new_k_rows")
    _rows_ok(new_v_rows, "new_v_rows")
    require_device(q_rows, out_rows, pool.k, block_tables, cu_seqlens, kv_lens, positions, new_k_rows,
                   new_v_rows, slot_mapping)
    if q_rows.dtype != pool.k.dtype or out_rows.dtype != pool.k.dtype or new_k_rows.dtype != pool.k.dtype \
            or new_v_rows.dtype != pool.k.dtype:
        raise TypeError("query, output, new rows and pool must share a dtype")
    if not same_layout(new_k_rows, new_v_rows):
        raise ValueError("new K and V rows must share shape and strides")
    if slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous():
        raise TypeError("slot_mapping must be a contiguous int64 tensor")
    T, H, D = new_k_rows.shape
    if H != pool.num_heads or D != pool.head_dim or slot_mapping.numel() != T:
        raise ValueError(f"new rows {tuple(new_k_rows.shape)} / {slot_mapping.numel()} slots do not match a "
                         f"pool of {pool.num_heads} heads x {pool.head_dim}")
    if getattr(plan, "sliced", False):
        raise ValueError("a written-in-flight step takes per-range plans (mf_attention_plan)")
    bt_stride = block_tables.shape[1] if block_tables.dim() == 2 else 0
    if isinstance(plan, CountedPlan):
        n_narrow, n_wide, n_merges = plan.cap_narrow, plan.cap_wide, plan.cap_merges
        counts, partials = plan.counts, plan.partials
    else:
        n_narrow, n_wide, n_merges = plan.n_narrow, plan.n_wide, plan.n_merges
        counts, partials = None, _WORKSPACE.partials(plan.partials_floats, q_rows.device)
        # every item's rows (its sequence's first row and row count) must be
        # rows of the new K/V the launch reads in flight
        held = plan.items_host[: n_narrow + n_wide]
        if held.shape[0] and int((held[:, 8] + held[:, 9]).max()) > T:
            raise ValueError(f"the plan's sequences reach past the {T} new rows")
    if _scored(scoring) is not None:
        return _paged_attention_scored(scoring, q_rows, out_rows, pool, block_tables, cu_seqlens, kv_lens, positions,
                                       plan, scale, num_kv_heads, nk=new_k_rows, nv=new_v_rows,
                                       slot_mapping=slot_mapping)
    _check(lib().mf_paged_attention_kv_write(
        _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
        _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
        dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
        pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
        _ptr(block_tables), bt_stride, _ptr(cu_seqlens), _ptr(kv_lens), _ptr(positions),
        _ptr(new_k_rows), _ptr(new_v_rows), new_k_rows.stride(0), new_k_rows.stride(1),
        _ptr(slot_mapping), T, pool.num_slots,
        q_rows.shape[1], num_kv_heads, q_rows.shape[2], float(scale),
        _ptr(plan.items), n_narrow, n_wide, _ptr(plan.merges), n_merges, _ptr(counts),
        _ptr(partials), partials.numel() if partials is not None else 0, _stream(q_rows.device),
    ), "mf_paged_attention_kv_write")


# fp32 partials the no-allocation entry point holds per GPU (32 MiB)
NOALLOC_PARTIALS_FLOATS = 8 * 1024 * 1024


def plan_partials_reach(plan: AttentionPlan, head_dim: int) -> int:
    """fp32 partial floats up to the end of the highest partial slot a
    per-range plan's items or merge records name. The kernels take the slot
    numbers as given, so this (not a declared size) is what a buffer must
    hold."""
    stride = 16 * (max(32, head_dim) + 2)
    top = 0
    n_items = plan.n_narrow + plan.n_wide
    if n_items:
        it = np.asarray(plan.items_host[:n_items], dtype=np.int64)
        named = it[:, 6] >= 0
        if named.any():
            # an item writes slots pslot .. pslot + column tiles - 1
            top = max(top, int((it[named, 6] + np.maximum(it[named, 3], 1)).max()))
    if plan.n_merges:
        mg = np.asarray(plan.merges_host[:plan.n_merges], dtype=np.int64)
        # record: partitions mg[3] at slot mg[4] + p * mg[5]
        top = max(top, int((mg[:, 4] + (np.maximum(mg[:, 3], 1) - 1) * mg[:, 5] + 1).max()))
    return top * stride


def paged_attention_noalloc(q_rows: torch.Tensor, out_rows: torch.Tensor, pool: PoolView,
                            block_tables: torch.Tensor, cu_seqlens: torch.Tensor, kv_lens: torch.Tensor,
                            positions: torch.Tensor, plan: AttentionPlan, scale: float, num_kv_heads: int,
                            row_map: Optional[torch.Tensor] = None, pool_lens: Optional[torch.Tensor] = None,
                            new_k_rows: Optional[torch.Tensor] = None,
                            new_v_rows: Optional[torch.Tensor] = None) -> None:
    """``paged_attention`` through mf_paged_attention_noalloc: the split-K
    partials live in the library's own per-GPU array, so the call allocates
    nothing (neither here nor in the library). Plans needing more than
    NOALLOC_PARTIALS_FLOATS partial floats are refused."""
    if getattr(plan, "sliced", False):
        raise ValueError("the no-allocation entry point takes per-range plans (mf_attention_plan)")
    # The slots the plan's items and merge records name must lie inside the
    # library's array, whatever partials_floats declares: no kernel bounds a
    # slot against it.
    reach = max(plan_partials_reach(plan, q_rows.shape[2]), plan.partials_floats)
    if reach > NOALLOC_PARTIALS_FLOATS:
        raise MemforgeHipError(
            f"mf_paged_attention_noalloc: the plan's partial slots need {reach} floats, past the "
            f"{NOALLOC_PARTIALS_FLOATS} of the library's array (workspace too small)")
    _rows_ok(q_rows, "q_rows")
    _rows_ok(out_rows, "out_rows")
    require_device(q_rows, out_rows, pool.k, block_tables, cu_seqlens, kv_lens, positions)
    if q_rows.dtype != pool.k.dtype or out_rows.dtype != pool.k.dtype:
        raise TypeError("query, output and pool must share a dtype")
    nk, nv = new_k_rows, new_v_rows
    if pool_lens is not None:
        if nk is None or nv is None:
            raise ValueError("pool_lens needs the in-flight new_k_rows/new_v_rows")
        require_device(pool_lens, nk, nv)
        if not same_layout(nk, nv):
            raise ValueError("in-flight K and V rows must share strides")
    bt_stride = block_tables.shape[1] if block_tables.dim() == 2 else 0
    _check(lib().mf_paged_attention_noalloc(
        _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
        _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
        dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
        pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
        _ptr(block_tables), bt_stride, _ptr(cu_seqlens), _ptr(kv_lens), _ptr(positions),
        _ptr(row_map), _ptr(pool_lens), _ptr(nk), _ptr(nv),
        nk.stride(0) if nk is not None else 0, nk.stride(1) if nk is not None else 0,
        q_rows.shape[1], num_kv_heads, q_rows.shape[2], float(scale),
        _ptr(plan.items), plan.n_narrow, plan.n_wide, _ptr(plan.merges), plan.n_merges,
        plan.partials_floats, _stream(q_rows.device),
    ), "mf_paged_attention_noalloc")


def paged_attention_packed(q_rows: torch.Tensor, out_rows: torch.Tensor, pool: PoolView, buf: torch.Tensor,
                           offsets: Sequence[int], num_seqs: int, bt_stride: int, counts: np.ndarray,
                           scale: float, num_kv_heads: int, has_row_map: bool, has_pool_lens: bool,
                           new_k_rows: Optional[torch.Tensor] = None,
                           new_v_rows: Optional[torch.Tensor] = None, sliced: bool = False,
                           softcap: float = 0.0, slopes: Optional[torch.Tensor] = None,
                           has_first_keys: bool = False, has_prefix_lens: bool = False) -> None:
    """mf_paged_attention on index arrays that one ``upload`` placed in the
    device buffer ``buf`` at ``offsets`` (int32 words, as ``_layout`` gives
    them): the padded block tables, the plan's items, its merges, cu_seqlens
    followed by kv_lens (``num_seqs`` + 1 and ``num_seqs`` int32), the int64
    positions, then the row map, the pool lengths, the first keys and the prefix
    lengths (a scored call's masks, int32 per sequence) when present. The caller
    built all of them, so only the tensors it did not build (query, output,
    pool, in-flight rows) are checked, and the launch takes addresses inside
    ``buf`` instead of building a tensor view per array. ``sliced``: the plan
    is a slice plan (mf_paged_attention_slices; no row map or pool lengths)."""
    _rows_ok(q_rows, "q_rows")
    _rows_ok(out_rows, "out_rows")
    four = isinstance(pool, Pool4View)
    if four:
        _check4(q_rows, out_rows, pool, num_kv_heads)
        if has_pool_lens or sliced:
            raise ValueError("a 4-bit pool takes no in-flight keys or slice plans")
    else:
        require_device(q_rows, out_rows, pool.k, buf)
        if q_rows.dtype != pool.k.dtype or out_rows.dtype != pool.k.dtype:
            raise TypeError("query, output and pool must share a dtype")
    if buf.dtype != torch.int32 or not buf.is_contiguous():
        raise TypeError("buf must be a contiguous int32 tensor")
    nk, nv = new_k_rows, new_v_rows
    if has_pool_lens:
        if nk is None or nv is None:
            raise ValueError("pool_lens needs the in-flight new_k_rows/new_v_rows")
        require_device(nk, nv)
        if not same_layout(nk, nv):
            raise ValueError("in-flight K and V rows must share strides")
    dev = q_rows.device
    n_narrow, n_wide, n_merges, floats = (int(x) for x in counts)
    partials = _WORKSPACE.partials(floats, dev)
    addr = [buf.data_ptr() + 4 * o for o in offsets]
    if sliced:
        if has_row_map or has_pool_lens:
            raise ValueError("a slice plan takes no row map or in-flight keys")
        _check(lib().mf_paged_attention_slices(
            _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
            _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
            dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
            pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
            addr[0], bt_stride, addr[3], addr[3] + 4 * (num_seqs + 1), addr[4],
            q_rows.shape[1], num_kv_heads, q_rows.shape[2], float(scale),
            addr[1], n_narrow, n_wide, addr[2], n_merges,
            _ptr(partials), partials.numel() if partials is not None else 0, _stream(dev),
        ), "mf_paged_attention_slices")
        return
    row_map = addr[5] if has_row_map else None
    pool_lens = addr[5 + int(has_row_map)] if has_pool_lens else None
    mods = None
    if softcap or slopes is not None or has_first_keys or has_prefix_lens:
        at = 5 + int(has_row_map) + int(has_pool_lens)
        mods = Scoring(softcap, slopes).struct(q_rows.shape[1], num_seqs, dev)
        mods.first_keys = addr[at] if has_first_keys else None
        mods.prefix_lens = addr[at + int(has_first_keys)] if has_prefix_lens else None
    scored_at = ctypes.addressof(mods) if mods is not None else None
    if four:
        _launch(
            dev, "mf_paged_attention4", lib().mf_paged_attention4, scored_at,
            _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
            _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
            dtype_code(q_rows.dtype), pool.address, addr[0], bt_stride,
            addr[3], addr[3] + 4 * (num_seqs + 1), addr[4], row_map, q_rows.shape[1], float(scale),
            addr[1], n_narrow, n_wide, addr[2], n_merges, None,
            _ptr(partials), partials.numel() if partials is not None else 0)
        return
    if mods is not None:
        _launch(
            dev, "mf_paged_attention_scored", lib().mf_paged_attention_scored, scored_at,
            _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
            _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
            dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
            pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
            addr[0], bt_stride, addr[3], addr[3] + 4 * (num_seqs + 1), addr[4],
            row_map, pool_lens, _ptr(nk), _ptr(nv),
            nk.stride(0) if nk is not None else 0, nk.stride(1) if nk is not None else 0, None, 0, 0,
            q_rows.shape[1], num_kv_heads, q_rows.shape[2], float(scale),
            addr[1], n_narrow, n_wide, addr[2], n_merges, None,
            _ptr(partials), partials.numel() if partials is not None else 0)
        return
    _check(lib().mf_paged_attention(
        _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
        _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
        dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
        pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
        addr[0], bt_stride, addr[3], addr[3] + 4 * (num_seqs + 1), addr[4],
        row_map, pool_lens, _ptr(nk), _ptr(nv),
        nk.stride(0) if nk is not None else 0, nk.stride(1) if nk is not None else 0,
        q_rows.shape[1], num_kv_heads, q_rows.shape[2], float(scale),
        addr[1], n_narrow, n_wide, addr[2], n_merges,
        _ptr(partials), partials.numel() if partials is not None else 0, None, _stream(dev),
    ), "mf_paged_attention")


def _paged_attention_counted(q_rows, out_rows, pool, block_tables, cu_seqlens, kv_lens, positions,
                             plan: CountedPlan, scale, num_kv_heads, row_map, pool_lens, nk, nv) -> None:
    if pool_lens is not None:
        if nk is None or nv is None:
            raise ValueError("pool_lens needs the in-flight new_k_rows/new_v_rows")
        require_device(pool_lens, nk, nv)
    Hq, D = q_rows.shape[1], q_rows.shape[2]
    bt_stride = block_tables.shape[1] if block_tables.dim() == 2 else 0
    _check(lib().mf_paged_attention_counted(
        _ptr(q_rows), q_rows.stride(0), q_rows.stride(1),
        _ptr(out_rows), out_rows.stride(0), out_rows.stride(1),
        dtype_code(q_rows.dtype), _ptr(pool.k), _ptr(pool.v),
        pool.stride_block, pool.stride_slot, pool.stride_head, pool.block_size,
        _ptr(block_tables), bt_stride, _ptr(cu_seqlens), _ptr(kv_lens), _ptr(positions),
        _ptr(row_map), _ptr(pool_lens), _ptr(nk), _ptr(nv),
        nk.stride(0) if nk is not None else 0, nk.stride(1) if nk is not None else 0,
        Hq, num_kv_heads, D, float(scale),
        _ptr(plan.items), plan.cap_narrow, plan.cap_wide, _ptr(plan.merges), plan.cap_merges,
        _ptr(plan.counts), _ptr(plan.partials), plan.partials.numel(), _stream(q_rows.device),
    ), "mf_paged_attention_counted")


# -------------------------------------------------------------- ragged pack

@dataclass
class PackedStep:
    token_ids: torch.Tensor     # int64 [T]
    positions: torch.Tensor     # int64 [T]
    seq_slot: torch.Tensor      # int32 [T]
    slot_mapping: torch.Tensor  # int64 [T]
    cu_seqlens: torch.Tensor    # int32 [B+1]
    kv_lens: torch.Tensor       # int32 [B]
    block_tables: torch.Tensor  # int32 [B, max_blocks]
    status: torch.Tensor        # int32 [4]

    @classmethod
    def allocate(cls, total_tokens: int, num_entries: int, max_blocks: int, device) -> "PackedStep":
        return cls(
            token_ids=torch.empty(total_tokens, dtype=torch.int64, device=device),
            positions=torch.empty(total_tokens, dtype=torch.int64, device=device),
            seq_slot=torch.empty(total_tokens, dtype=torch.int32, device=device),
            slot_mapping=torch.empty(total_tokens, dtype=torch.int64, device=device),
            cu_seqlens=torch.empty(num_entries + 1, dtype=torch.int32, device=device),
            kv_lens=torch.empty(num_entries, dtype=torch.int32, device=device),
            block_tables=torch.empty((num_entries, max_blocks), dtype=torch.int32, device=device),
            status=torch.empty(4, dtype=torch.int32, device=device),
        )


def check_pack_entries(entries: np.ndarray, tables: np.ndarray, tokens_len: int, total_tokens: int,
                       num_blocks: Optional[int] = None) -> None:
    """Host check of ragged-pack descriptors before they go to the device:
    every field non-negative, every table run inside ``tables`` and every
    token run inside ``tokens_len``, the row count equal to the sum of q_len,
    and (with ``num_blocks``) every block id the runs name inside the pool.
    Raises ValueError / IndexError naming the first bad entry."""
    ent = np.asarray(entries, dtype=np.int64).reshape(-1, ENTRY_INTS)
    if ent.shape[0] == 0:
        if total_tokens:
            raise ValueError(f"{total_tokens} packed rows but no entries")
        return
    bad = np.flatnonzero((ent[:, [0, 2, 3, 4, 5]] < 0).any(axis=1)
                         | (ent[:, 3] + ent[:, 4] > len(tables))
                         | (ent[:, 5] + ent[:, 0] > tokens_len))
    if bad.size:
        e = int(bad[0])
        raise ValueError(f"ragged-pack entry {e} is malformed: {ent[e].tolist()} against "
                         f"{len(tables)} table ids and {tokens_len} tokens")
    rows = int(ent[:, 0].sum())
    if rows != total_tokens:
        raise ValueError(f"entries hold {rows} rows, the step declares {total_tokens}")
    if num_blocks is not None and len(tables):
        t = np.asarray(tables)
        lo, hi = int(t.min()), int(t.max())
        if lo < 0 or hi >= num_blocks:
            raise IndexError(f"block id {lo if lo < 0 else hi} is outside a pool of {num_blocks} blocks")


def ragged_pack(entries: torch.Tensor, tables: torch.Tensor, tokens: torch.Tensor,
                total_tokens: int, block_size: int, max_blocks: int,
                slot_bitmap: Optional[torch.Tensor] = None, num_slots: int = 0,
                out: Optional[PackedStep] = None) -> PackedStep:
    """Run mf_ragged_pack on device descriptors (int32 tensors already on the
    GPU), into ``out``'s buffers when given (they must be sized for
    ``total_tokens`` rows, ``entries.shape[0]`` entries and ``max_blocks``).
    The kernel bounds every load by ``tables.numel()`` / ``tokens.numel()``
    and, with ``num_slots``, every block id by the pool; host callers that
    built the descriptors check them first with ``check_pack_entries``."""
    require_device(entries, tables, tokens)
    if entries.dtype != torch.int32 or tables.dtype != torch.int32 or tokens.dtype != torch.int32:
        raise TypeError("ragged_pack takes int32 entries, tables and tokens")
    if not (entries.is_contiguous() and tables.is_contiguous() and tokens.is_contiguous()):
        raise ValueError("ragged_pack takes contiguous entries, tables and tokens")
    dev = entries.device
    B = entries.shape[0]
    if out is not None:
        if (out.token_ids.numel() != total_tokens or out.cu_seqlens.numel() != B + 1
                or tuple(out.block_tables.shape) != (B, max_blocks)):
            raise ValueError("preallocated pack buffers do not match the step")
    else:
        out = PackedStep.allocate(total_tokens, B, max_blocks, dev)
    _check(lib().mf_ragged_pack(
        _ptr(entries), B, _ptr(tables), tables.numel(), _ptr(tokens), tokens.numel(), block_size,
        max_blocks, total_tokens,
        _ptr(out.token_ids), _ptr(out.positions), _ptr(out.seq_slot), _ptr(out.slot_mapping),
        _ptr(out.cu_seqlens), _ptr(out.kv_lens), _ptr(out.block_tables), _ptr(slot_bitmap),
        num_slots, _ptr(out.status), _stream(),
    ), "mf_ragged_pack")
    return out


# --------------------------------------------------------- rejection verify

@dataclass
class VerifyResult:
    tokens: torch.Tensor        # int32 [B, K+1]
    is_draft: torch.Tensor      # uint8 [B, K+1]
    count: torch.Tensor         # int32 [B]
    num_accepted: torch.Tensor  # int32 [B]
    packed: Optional[torch.Tensor] = None  # the int32 buffer the four are views of, in the order of ``split``

    @staticmethod
    def split(packed: torch.Tensor, B: int, K: int) -> "VerifyResult":
        """The four results as views of a packed buffer (the device one, or its
        host copy: one transfer for all of them)."""
        n = B * (K + 1)
        return VerifyResult(
            tokens=packed[:n].view(B, K + 1),
            is_draft=packed[n + 2 * B:].view(torch.uint8)[:n].view(B, K + 1),
            count=packed[n:n + B],
            num_accepted=packed[n + B:n + 2 * B],
            packed=packed,
        )


_VERIFY_WS_BYTES = {}  # (rows, candidates) -> mf_spec_verify_workspace_size


def spec_verify(draft_tokens: torch.Tensor, draft_probs: torch.Tensor, target_logits: torch.Tensor,
                temperature: float, u_accept: torch.Tensor, exp_noise: torch.Tensor,
                target_is_probs: bool = False) -> VerifyResult:
    """Batched rejection sampling. Shapes: draft_tokens (B, K) int32,
    draft_probs (B, K, V) fp32, target_logits (B, K+1, >=V) -- or target
    probabilities (fp32) with ``target_is_probs`` --, u_accept (B, K) fp32,
    exp_noise (B, V) fp32."""
    require_device(draft_tokens, draft_probs, target_logits, u_accept, exp_noise)
    B, K = draft_tokens.shape
    V = draft_probs.shape[-1] if K > 0 else exp_noise.shape[-1]
    if target_logits.shape[0] != B or target_logits.shape[1] != K + 1 or target_logits.shape[2] < V:
        raise ValueError(f"target logits {tuple(target_logits.shape)} do not cover ({B}, {K + 1}, {V})")
    if target_logits.stride(-1) != 1 or draft_probs.stride(-1) != 1 or exp_noise.stride(-1) != 1:
        raise ValueError("vocabulary axes must be contiguous")
    if draft_tokens.dtype != torch.int32 or not draft_tokens.is_contiguous():
        draft_tokens = draft_tokens.to(torch.int32).contiguous()
    if u_accept.dtype != torch.float32 or not u_accept.is_contiguous():
        u_accept = u_accept.to(torch.float32).contiguous()
    dev = target_logits.device
    # one allocation for the four outputs (only the first count[b] entries of
    # each row are written); is_draft is bytes of its int32 tail. The kernels
    # are queued first and the views built after, so no view is made on the
    # way to the launch.
    n = B * (K + 1)
    out = torch.empty(n + 2 * B + (n + 3) // 4, dtype=torch.int32, device=dev)
    base = out.data_ptr()
    L = lib()
    ws_bytes = _VERIFY_WS_BYTES.get((B, K))
    if ws_bytes is None:
        ws_bytes = _VERIFY_WS_BYTES[(B, K)] = int(L.mf_spec_verify_workspace_size(B, K))
    stream = _stream(dev)
    ws = _WORKSPACE.verify(ws_bytes, dev, stream)
    _check(L.mf_spec_verify(
        B, K, V, draft_tokens.data_ptr(), draft_probs.data_ptr(),
        draft_probs.stride(0) if K > 0 else 0, draft_probs.stride(1) if K > 0 else 0,
        target_logits.data_ptr(), dtype_code(target_logits.dtype), target_logits.stride(0),
        target_logits.stride(1), float(temperature), int(bool(target_is_probs)), u_accept.data_ptr(),
        exp_noise.data_ptr(), exp_noise.stride(0), base, base + 4 * (n + 2 * B), base + 4 * n,
        base + 4 * (n + B), ws.data_ptr(), ws_bytes, stream,
    ), "mf_spec_verify")
    return VerifyResult.split(out, B, K)


def check_index(name: str, x: torch.Tensor, dtype: torch.dtype, device: torch.device, shape: Optional[tuple] = None) -> None:
    """An index tensor of a call: its type, its device, contiguous, and its shape when given."""
    if x.dtype is dtype and x.device == device and x.is_contiguous() and (shape is None or x.shape == shape):
        return
    if x.dtype != dtype or not x.is_contiguous():
        raise TypeError(f"{name} must be a contiguous {dtype} tensor, got {x.dtype} with strides {x.stride()}")
    if shape is not None and tuple(x.shape) != shape:
        raise ValueError(f"{name} must be of shape {shape}, got {tuple(x.shape)}")
    raise ValueError(f"{name} is on {x.device}, the call's other tensors on {device}")


# ---------------------------------------------------------------- sampling

SAMPLE_MAX_VOCAB = 1 << 20
_SAMPLE_WS_BYTES = {}  # (rows, vocab, compute units) -> mf_sample_workspace_size


def sample(logits: torch.Tensor, uniforms: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
           min_p=0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """mf_sample: (tokens int64, probs fp32), one per row of ``logits`` ((rows, vocab),
    the last axis contiguous). Settings are numbers, or tensors with one per row
    (fp32; top_k int32)."""
    require_device(logits, uniforms)
    if logits.dim() != 2 or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError(f"logits must be (rows, vocab) with a contiguous vocabulary axis, got {tuple(logits.shape)} "
                         f"with strides {logits.stride()}")
    rows, vocab = logits.shape
    if not 1 <= vocab <= SAMPLE_MAX_VOCAB:
        raise ValueError(f"a vocabulary holds 1 to {SAMPLE_MAX_VOCAB} tokens, got {vocab}")
    dev, code = logits.device, dtype_code(logits.dtype)
    check_index("uniforms", uniforms, torch.float32, dev, (rows,))
    settings = []
    for name, x, dt in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                        ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(x, torch.Tensor):
            require_device(x)
            check_index(name, x, dt, dev, (rows,))
            settings += [x.data_ptr(), 0]
        elif dt == torch.int32:
            settings += [None, min(int(x), SAMPLE_MAX_VOCAB) if x > 0 else 0]
        else:
            if x != x:
                raise ValueError(f"{name} must be a number, got {x}")
            settings += [None, float(x)]
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    probs = torch.empty(rows, dtype=torch.float32, device=dev)
    cus = device_cus(dev)
    shape = (rows, vocab, cus)
    nbytes = _SAMPLE_WS_BYTES.get(shape)
    if nbytes is None:
        if len(_SAMPLE_WS_BYTES) >= 4096:
            _SAMPLE_WS_BYTES.clear()
        nbytes = _SAMPLE_WS_BYTES[shape] = int(lib().mf_sample_workspace_size(*shape))
    ws = _WORKSPACE.bins(nbytes // 8, dev)
    _launch(dev, "mf_sample", lib().mf_sample, logits.data_ptr(), code, logits.stride(0), rows,
            vocab, uniforms.data_ptr(), *settings, tokens.data_ptr(), probs.data_ptr(), cus, _ptr(ws), nbytes)
    return tokens, probs


# ---------------------------------------------------- trees of drafted tokens

TREE_MAX_NODES = 1024


def tree_accept(tokens: torch.Tensor, targets: torch.Tensor, parents: torch.Tensor, cu_nodes: torch.Tensor,
                max_nodes: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """mf_tree_accept: (path int32 (B, max_nodes), tokens int64 (B, max_nodes), count int32 (B))."""
    require_device(tokens, targets, parents, cu_nodes)
    dev, rows, seqs = parents.device, parents.numel(), cu_nodes.numel() - 1
    shape = (rows,)
    check_index("parents", parents, torch.int32, dev, shape)
    check_index("tokens", tokens, torch.int64, dev, shape)
    check_index("targets", targets, torch.int64, dev, shape)
    check_index("cu_nodes", cu_nodes, torch.int32, dev, (seqs + 1,))
    if seqs < 0:
        raise ValueError("cu_nodes must have one more entry than sequences")
    if not 1 <= max_nodes <= TREE_MAX_NODES:
        raise ValueError(f"max_nodes must be 1 to {TREE_MAX_NODES}, got {max_nodes}")
    path = torch.empty((seqs, max_nodes), dtype=torch.int32, device=dev)
    out = torch.empty((seqs, max_nodes), dtype=torch.int64, device=dev)
    count = torch.empty(seqs, dtype=torch.int32, device=dev)
    _launch(dev, "mf_tree_accept", lib().mf_tree_accept, tokens.data_ptr(), targets.data_ptr(), parents.data_ptr(),
            cu_nodes.data_ptr(), seqs, rows, max_nodes, path.data_ptr(), out.data_ptr(), count.data_ptr())
    return path, out, count


TREE_HEAD_DIMS = (32, 64, 128, 256)
_TREE_SIZES = {}  # shape of a call -> mf_tree_plan_sizes


@dataclass
class TreePlan:
    """One step's trees as ``tree_attention`` reads them (mf_tree_plan)."""

    buffer: torch.Tensor      # int32
    positions: torch.Tensor   # int64 per row: context length + number of ancestors; 0: no node's row
    num_seqs: int
    num_rows: int
    max_nodes: int
    max_context: int
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    dtype: torch.dtype
    num_cus: int
    partials_floats: int
    device: torch.device


def tree_plan(parents: torch.Tensor, cu_nodes: torch.Tensor, context_lens: torch.Tensor, max_nodes: int, max_context: int,
              num_q_heads: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype) -> TreePlan:
    """mf_tree_plan into new buffers."""
    require_device(parents, cu_nodes, context_lens)
    dev, rows, seqs = parents.device, parents.numel(), context_lens.numel()
    check_index("parents", parents, torch.int32, dev, (rows,))
    check_index("cu_nodes", cu_nodes, torch.int32, dev, (seqs + 1,))
    check_index("context_lens", context_lens, torch.int32, dev, (seqs,))
    if not 1 <= max_nodes <= TREE_MAX_NODES:
        raise ValueError(f"max_nodes must be 1 to {TREE_MAX_NODES}, got {max_nodes}")
    if not 0 <= max_context <= 1 << 30:
        raise ValueError(f"max_context must be 0 to 2^30, got {max_context}")
    if num_kv_heads < 1 or num_q_heads < 1 or num_q_heads % num_kv_heads:
        raise ValueError(f"{num_q_heads} query heads is not a multiple of {num_kv_heads} kv heads")
    if head_dim not in TREE_HEAD_DIMS:
        raise ValueError(f"tree attention takes head_dims {TREE_HEAD_DIMS}, got {head_dim}")
    cus = device_cus(dev)
    shape = (seqs, rows, max_nodes, num_q_heads, num_kv_heads, head_dim, dtype_code(dtype), cus)
    sizes = _TREE_SIZES.get(shape)
    if sizes is None:
        got = np.zeros(2, dtype=np.int64)
        _check(lib().mf_tree_plan_sizes(*shape, got.ctypes.data, got.ctypes.data + 8), "mf_tree_plan_sizes")
        if len(_TREE_SIZES) >= 4096:
            _TREE_SIZES.clear()
        sizes = _TREE_SIZES[shape] = (int(got[0]), int(got[1]))
    buffer = torch.empty(sizes[0], dtype=torch.int32, device=dev)
    positions = torch.empty(rows, dtype=torch.int64, device=dev)
    _launch(dev, "mf_tree_plan", lib().mf_tree_plan, parents.data_ptr(), cu_nodes.data_ptr(), context_lens.data_ptr(),
            seqs, rows, max_nodes, max_context, num_q_heads, num_kv_heads, head_dim, shape[6], cus, buffer.data_ptr(),
            sizes[0], positions.data_ptr())
    return TreePlan(buffer, positions, seqs, rows, max_nodes, max_context, num_q_heads, num_kv_heads, head_dim, dtype, cus,
                    sizes[1], dev)


def _tree_rows(name: str, x: torch.Tensor, heads: int, plan: "TreePlan", rows: int, head: int) -> Tuple[int, int, int]:
    """(address, row stride, head stride) of a call's rows, whose axes ``rows`` and ``head`` are the rows and heads."""
    shape, stride = x.shape, x.stride()
    if shape[rows] != plan.num_rows or shape[head] != heads or shape[-1] != plan.head_dim or x.dtype is not plan.dtype \
            or x.device != plan.device:
        raise ValueError(f"{name} must be {plan.num_rows} rows of {heads} heads x {plan.head_dim} in {plan.dtype} on "
                         f"{plan.device}, got {tuple(shape)} in {x.dtype} on {x.device}")
    if stride[-1] != 1:
        raise ValueError(f"{name} head_dim axis must be contiguous")
    return x.data_ptr(), stride[rows] if shape[rows] > 1 else 0, stride[head] if heads > 1 else 0


def tree_attention_at(q: Tuple[int, int, int], out: Tuple[int, int, int], pool: Tuple[int, int, int, int, int, int, int],
                      block_tables: torch.Tensor, plan: "TreePlan", new_k: Tuple[int, int, int], new_v: int, scale: float,
                      partials: Optional[torch.Tensor] = None) -> None:
    """mf_tree_attention on addresses that the caller has checked: rows as ``_tree_rows`` gives them (``new_v`` laid out
    as ``new_k``), ``pool`` = (K address, V address, strides of blocks, slots and heads, block size, blocks)."""
    check_index("block_tables", block_tables, torch.int32, plan.device)
    shape = block_tables.shape
    if len(shape) != 2 or shape[0] != plan.num_seqs or shape[1] * pool[5] < plan.max_context:
        raise ValueError(f"block_tables {tuple(shape)} do not hold {plan.num_seqs} contexts of up to {plan.max_context} tokens "
                         f"in blocks of {pool[5]}")
    if not abs(scale) < float("inf"):
        raise ValueError(f"scale must be finite, got {scale}")
    if plan.num_rows == 0 or plan.num_seqs == 0:
        return
    dev = plan.device
    if partials is None:
        partials = _WORKSPACE.partials(plan.partials_floats, dev)
    elif partials.dtype != torch.float32 or not partials.is_contiguous() or partials.device != dev:
        raise ValueError(f"partials must be contiguous fp32 on {dev}, got {partials.dtype} on {partials.device}")
    # (tables of no columns have no address; no context reads them, and the entry point takes no null pointer)
    _launch(dev, "mf_tree_attention", lib().mf_tree_attention, *q, *out, DTYPE_CODES[plan.dtype], *pool,
            block_tables.data_ptr() if shape[1] else plan.buffer.data_ptr(), shape[1], new_k[0], new_v, new_k[1], new_k[2], plan.num_seqs, plan.num_rows,
            plan.max_nodes, plan.num_q_heads, plan.num_kv_heads, plan.head_dim, scale, plan.num_cus, plan.buffer.data_ptr(),
            plan.buffer.numel(), partials.data_ptr(), partials.numel())


def check_tree_pool(key_pool: torch.Tensor, num_heads: int, head_dim: int, plan: "TreePlan") -> None:
    if key_pool.dtype is not plan.dtype or num_heads != plan.num_kv_heads or head_dim != plan.head_dim \
            or key_pool.device != plan.device:
        raise ValueError(f"a pool of {num_heads} heads x {head_dim} in {key_pool.dtype} on {key_pool.device} does not match a "
                         f"plan for {plan.num_kv_heads} x {plan.head_dim} in {plan.dtype} on {plan.device}")


def tree_attention(q_rows: torch.Tensor, out_rows: torch.Tensor, pool: PoolView, block_tables: torch.Tensor, plan: TreePlan,
                   new_k_rows: torch.Tensor, new_v_rows: torch.Tensor, scale: float,
                   partials: Optional[torch.Tensor] = None) -> None:
    """mf_tree_attention into ``out_rows`` ((rows, Hq, D) views, device)."""
    require_device(q_rows, out_rows, pool.k, block_tables, new_k_rows, new_v_rows)
    for name, x in (("q_rows", q_rows), ("out_rows", out_rows), ("new_k_rows", new_k_rows), ("new_v_rows", new_v_rows)):
        _rows_ok(x, name)
    if not same_layout(new_k_rows, new_v_rows):
        new_k_rows, new_v_rows = new_k_rows.contiguous(), new_v_rows.contiguous()
    check_tree_pool(pool.k, pool.num_heads, pool.head_dim, plan)
    tree_attention_at(_tree_rows("q_rows", q_rows, plan.num_q_heads, plan, 0, 1),
                      _tree_rows("out_rows", out_rows, plan.num_q_heads, plan, 0, 1),
                      (pool.k.data_ptr(), pool.v.data_ptr(), pool.stride_block, pool.stride_slot, pool.stride_head,
                       pool.block_size, pool.num_blocks), block_tables, plan,
                      _tree_rows("new_k_rows", new_k_rows, plan.num_kv_heads, plan, 0, 1),
                      _tree_rows("new_v_rows", new_v_rows, plan.num_kv_heads, plan, 0, 1)[0], float(scale), partials)
