"""The ctypes binding of libbpt_b200.so (include/bpt_b200.h).

The library is loaded lazily, so importing the package never needs a GPU or the built library. A call that
reaches a kernel without the library raises: there is no CPU fallback anywhere in this package.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import struct
from pathlib import Path

import torch

LIB_PATH = Path(__file__).with_name("libbpt_b200.so")

OK, ERR_INVALID, ERR_UNSUPPORTED, ERR_ALIGNMENT, ERR_WORKSPACE, ERR_CUDA = range(6)
DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2
KV_FP8, KV_INT8, KV_F16, KV_BF16 = 1, 2, 3, 4
FLAG_PDL = 1
FLAG_KV_READY = 2

_DTYPES = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}

P, I64, I32, F32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float

# name -> argument types (the header's order)
SIGNATURES: dict[str, list] = {
    "bpt_abi_version": [],
    "bpt_last_error": [],
    "bpt_device_error": [],
    "bpt_w4a16_linear": [P, I64, P, P, P, P, I64, I64, I64, I64, I64, I32, P],
    "bpt_w4a16_gate_up_silu": [P, I64, P, P, P, P, I64, I64, I64, I64, I64, I32, P],
    "bpt_w4a16_kernel": [I64, I64, I64, I64, I32],
    "bpt_rms_norm_residual": [P, P, P, P, P, I64, I64, F32, I32, P],
    "bpt_qk_norm_rope_kv_write": [P, I64, I64, I64, I64, I64, P, P, P, P, F32, P, P, P, P, P, F32, F32, I64, I64, I32,
                                  P],
    "bpt_rope_kv_append": [ctypes.c_char_p],
    "bpt_rms_norm_int8": [P, I32, I64, P, I32, P, P, P, P, I64, I64, F32, I32, P],
    "bpt_w4a16_quantize": [P, I32, I64, I64, I64, P, P, P, P],
    "bpt_paged_decode_partials": [P, I32, I64, I64, P, P, I32, F32, F32, P, P, P, I64, P, I64, I64, I64, I64, I64, I64,
                                  I64, I64, F32, P, P, I32, P],
    "bpt_paged_attend_workspace_bytes": [I64, I64, I64, I64],
    "bpt_paged_attend": [P, I32, I64, I64, P, P, I32, F32, F32, P, P, P, I64, P, I64, I64, I64, I64, I64, I64, I64, I64,
                         F32, P, I32, P, I64, I32, P],
    "bpt_paged_attend_noalloc": [P, I32, I64, I64, P, P, I32, F32, F32, P, P, P, I64, P, I64, I64, I64, I64, I64, I64,
                                 I64, I64, F32, P, I32, I32, P],
    "bpt_paged_read_workspace_bytes": [I64, I64, I64, I32],
    "bpt_paged_read": [ctypes.c_char_p],
    "bpt_paged_prefill_workspace_bytes": [I64, I64, I64, I64, I64, I32, I64],
    "bpt_paged_prefill": [ctypes.c_char_p],
    "bpt_merge_partials": [P, P, I64, I64, I64, I64, P, I32, P],
    "bpt_kivi_decode_partials": [P, I32, I64, I64, I32, I32, P, P, P, P, P, P, P, I64, I64, I64, I64, I64, I64, I64,
                                 I64, I64, F32, P, P, P],
    "bpt_paged_kv_write": [P, P, I32, I64, I64, I64, I64, I64, I64, I64, P, P, P, P, I32, F32, F32, P, P, I64, I64, P],
    "bpt_kivi_quantize": [P, P, I32, I64, I64, I64, I64, I32, I64, P, P, P, P, P, P, I64, I64, I64, P],
}
RESTYPES = {"bpt_last_error": ctypes.c_char_p, "bpt_paged_attend_workspace_bytes": ctypes.c_int64,
            "bpt_paged_read_workspace_bytes": ctypes.c_int64, "bpt_paged_prefill_workspace_bytes": ctypes.c_int64}


class KernelLibraryMissing(RuntimeError):
    """libbpt_b200.so is not built (run bytes-per-token_b200/build.py)."""


@functools.cache
def lib() -> ctypes.CDLL:
    if not LIB_PATH.exists():
        raise KernelLibraryMissing(f"{LIB_PATH} is not built: run `python bytes-per-token_b200/build.py`")
    handle = ctypes.CDLL(str(LIB_PATH))
    for name, args in SIGNATURES.items():
        fn = getattr(handle, name)
        fn.argtypes = args
        fn.restype = RESTYPES.get(name, ctypes.c_int)
    return handle


class ArgStruct:
    """A function of the library that takes one struct of 8-byte fields (pointers P, integers q, doubles d), called with
    the fields' values in order; a pointer is an address, 0 for none. Packing 36 values takes 0.9 us, converting them one by
    one as ctypes arguments 8.6 us: more than the launch itself."""

    def __init__(self, name: str, fields: str):
        self.name = name
        self.fields = [f.split(":")[0] for f in fields.split()]
        self._pack = struct.Struct("@" + "".join(f.split(":")[1] for f in fields.split())).pack

    def __call__(self, *values) -> int:
        return getattr(lib(), self.name)(self._pack(*values))


rope_kv_append = ArgStruct(
    "bpt_rope_kv_append", (
        "q:P k:P v:P dtype:q q_stride_t:q q_stride_h:q k_stride_t:q k_stride_h:q v_stride_t:q v_stride_h:q T:q Hq:q "
        "Hkv:q D:q rotary:q positions:P cos:P sin:P table_rows:q interleaved:q q_norm:P k_norm:P eps:d q_out:P "
        "write_blocks:P write_offsets:P k_pool:P v_pool:P kind:q k_scale:d v_scale:d k_scales:P v_scales:P "
        "block_size:q num_blocks:q flags:q stream:P"))
paged_read = ArgStruct(
    "bpt_paged_read", (
        "q:P q_dtype:q q_stride_b:q q_stride_h:q k_pool:P v_pool:P kind:q k_scale:d v_scale:d k_scales:P v_scales:P "
        "block_table:P bt_stride:q bt_width:q lengths:P key_starts:P alibi_slopes:P softcap:d window:q B:q Hq:q Hkv:q "
        "D:q block_size:q num_blocks:q split:q n_splits:q tokens:q sm_scale:d out:P out_dtype:q out_partial:P lse_partial:P "
        "workspace:P workspace_bytes:q flags:q stream:P"))
paged_prefill = ArgStruct(
    "bpt_paged_prefill", (
        "q:P q_dtype:q q_stride_t:q q_stride_h:q k_pool:P v_pool:P kind:q k_scale:d v_scale:d k_scales:P v_scales:P "
        "block_table:P bt_stride:q bt_width:q cu_seqlens:P lengths:P positions:P key_starts:P prefix_lens:P "
        "alibi_slopes:P softcap:d window:q T:q B:q Hq:q Hkv:q D:q block_size:q num_blocks:q tokens:q sm_scale:d out:P "
        "workspace:P workspace_bytes:q flags:q stream:P"))


def check(status: int, what: str) -> None:
    """Turn a status code into the exception the reference would raise for the same mistake."""
    if status == OK:
        return
    message = lib().bpt_last_error().decode(errors="replace")
    if status == ERR_CUDA:
        raise RuntimeError(f"{what}: {message}")
    raise ValueError(f"{what}: {message}")


def dtype_code(t: torch.dtype) -> int:
    try:
        return _DTYPES[t]
    except KeyError:
        raise ValueError(f"unsupported dtype {t}") from None


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def addr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def stream_of(device: torch.device) -> int:
    """The handle of the device's current stream (what torch.cuda.current_stream(device).cuda_stream gives, without the
    Stream object: 0.2 us instead of 2)."""
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    """Every tensor on one CUDA device (that device is returned); anything else is a ValueError."""
    first = None
    index = -1
    for t in tensors:
        if t is None:
            continue
        if first is None:
            first, index = t, t.get_device()
            if index < 0 or not t.is_cuda:
                raise ValueError(f"expected CUDA tensors, got one on {t.device}: these kernels have no CPU path")
        elif t.get_device() != index:
            if not t.is_cuda:
                raise ValueError(f"expected CUDA tensors, got one on {t.device}: these kernels have no CPU path")
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    if first is None:
        raise ValueError("no tensor given")
    return first.device


_HERE = contextlib.nullcontext()


def on_device(device: torch.device):
    """A context in which `device` is the current one (kernels launch on the current device's streams only)."""
    if device.index is None or device.index == torch._C._cuda_getDevice():
        return _HERE
    return torch.cuda.device(device)


def as_int32(t: torch.Tensor) -> torch.Tensor:
    """A contiguous int32 copy of an integer tensor (itself where it is one already), out-of-range values saturated."""
    if t.dtype == torch.int32:
        return t if t.is_contiguous() else t.contiguous()
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise ValueError(f"expected whole numbers, got {t.dtype}")
    return t.clamp(-(2**31), 2**31 - 1).to(torch.int32).contiguous() if t.dtype == torch.int64 else t.to(torch.int32).contiguous()


def device_error() -> int:
    """Synchronize and return (and clear) the first device-side error code the kernels recorded."""
    return int(lib().bpt_device_error())
