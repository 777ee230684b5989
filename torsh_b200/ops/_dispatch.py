"""Shared helpers for the op wrappers: dtype codes, alignment checks, ctypes signatures."""
from __future__ import annotations

import ctypes
import struct

import torch

from .. import _native as nv

P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
_fns: dict = {}
_KERNEL_DTYPES = (torch.bfloat16, torch.float32)


def dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return 0
    if t.dtype == torch.float32:
        return 1
    raise TypeError(f"kernel supports bf16 / fp32, got {t.dtype}")


def kernel_ok(*tensors: torch.Tensor) -> bool:
    """True when every tensor is a CUDA bf16/fp32 tensor (the kernels' domain)."""
    for t in tensors:
        if t is not None and not (t.is_cuda and t.dtype in _KERNEL_DTYPES):
            return False
    return True


def aligned(t: torch.Tensor) -> torch.Tensor:
    """Contiguous and 16-byte aligned (copies only when needed)."""
    if not t.is_contiguous():
        t = t.contiguous()
    if t.data_ptr() % 16:
        t = t.clone()
    return t


def fn(name: str, argtypes):
    """Fetch a launcher from the CUDA library and set its signature once."""
    f = _fns.get(name)
    if f is None:
        f = getattr(nv.require_cuda(), name)
        f.restype = ctypes.c_int
        f.argtypes = argtypes
        _fns[name] = f
    return f


_KERNELS_PER_CALL = {"tb_flash_attn_bwd": 3, "tb_lamb_multi": 2, "tb_bn_fwd": 3, "tb_bn_bwd": 2, "tb_cache_attention": 2}


def call(name: str, argtypes, *args):
    rc = fn(name, argtypes)(*args)
    if rc != 0:
        nv.check(rc, name)
    nv.launch_count += _KERNELS_PER_CALL.get(name, 1)


class Record:
    """A launcher of the CUDA library that takes its arguments as one record of 8-byte fields (``q`` an integer or an address, ``d`` a
    double), packed in one call: 25 arguments through ``call`` cost 4 us of Python, the record 1. The launch goes to the device of
    ``index``, on that device's current stream, whichever device the caller is on."""

    def __init__(self, name: str, fields: str):
        self.name, self.pack, self.f, self.kernels = name, struct.Struct("=" + fields).pack, None, _KERNELS_PER_CALL.get(name, 1)

    def __call__(self, index: int, *fields) -> None:
        f = self.f
        if f is None:
            f = self.f = fn(self.name, [ctypes.c_char_p, P])
        d = torch._C._cuda_getDevice()
        if d != index:
            with torch.cuda.device(index):
                return self(index, *fields)
        if d != nv._bound_device:
            nv.stream_ptr()   # tells the library which device is current
        rc = f(self.pack(*fields), torch._C._cuda_getCurrentRawStream(d))
        if rc != 0:
            nv.check(rc, self.name)
        nv.launch_count += self.kernels
