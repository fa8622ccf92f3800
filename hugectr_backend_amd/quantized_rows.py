"""Embedding rows held in 8 or 4 bits on the GPU, addressed by slot: the hps_qrows_* entry points of libhps_amd.so (include/hps_amd.h) on
torch tensors.  The arithmetic is the HIP code in csrc/cache/qrows_kernels.hip; write() and read() are native calls
(csrc/python/torch_calls.cpp) that take the tensors apart and call the entry, torch holds the device buffers.
"""
from __future__ import annotations

import ctypes as C

from . import hps


def _invalid(msg: str):
    return hps.HpsError(hps.ERR_INVALID_ARG, msg)


_ELEM = {}


def elem_type(dtype) -> int:
    """HPS_TYPE_* of a torch dtype."""
    t = _ELEM.get(dtype)
    if t is None:
        import torch
        _ELEM.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
        t = _ELEM.get(dtype)
        if t is None:
            raise _invalid(f"fp32, fp16 or bf16 values expected, got {dtype}")
    return t


_CALLS = None


def calls():
    """The native calls on torch tensors (csrc/python/torch_calls.cpp): arguments checked, outputs allocated, the C entry called."""
    global _CALLS
    if _CALLS is None:
        import importlib.machinery
        import importlib.util

        import torch  # noqa: F401  (the module's symbols are torch's)
        path = hps._LIBPATH.with_name("hps_torch_calls.so")
        if not path.exists():
            raise ImportError(f"{path} is missing: build it with `python -m hugectr_backend_amd.build`")
        loader = importlib.machinery.ExtensionFileLoader("hps_torch_calls", str(path))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("hps_torch_calls", loader))
        loader.exec_module(module)
        module.set_error(hps.HpsError)
        _CALLS = module
    return _CALLS


class QuantizedRows:
    """`num_rows` rows of `dim` values in 8 (or 4) bits plus one fp32 scale per row, or per `group` consecutive values (16, 32, 64,
    128 or 256).  A value is held as the nearest multiple (ties to even) of scale = max|x| / 127 (7) of its group.  A group whose
    largest magnitude is below 2^-100 is held as zeros; one with a NaN or an infinity reads back as NaN.

    codes   [num_rows, row_bytes] int8 (8 bits) / uint8 (4 bits, two per byte, the first in the low half); rows padded to 4 bytes
    scales  [num_rows, groups] fp32
    A store of its own: which key has which slot is the caller's to keep; no session, cache or configuration of the parameter server
    fills it or reads from it.  Rows never written are zeros.  One write at a time per store (whatever the stream); reads beside reads are free, a read beside
    a write of the same slots is the caller's to order."""

    def __init__(self, num_rows: int, dim: int, bits: int = 8, group: int = 0, device: int = 0):
        import torch
        if hps.device_count() <= 0:
            raise hps.HpsError(hps.ERR_UNAVAILABLE, "quantised rows need a HIP device and none is visible; there is no CPU fallback")
        if num_rows < 0 or not 1 <= dim <= 16384 or bits not in (8, 4) or group not in (0, 16, 32, 64, 128, 256):
            raise _invalid(f"quantised rows: num_rows >= 0, dim 1..16384, bits 8 or 4, group 0, 16, 32, 64, 128 or 256 expected, got "
                           f"{num_rows}, {dim}, {bits}, {group}")
        self.num_rows, self.dim, self.bits, self.group, self.device = int(num_rows), int(dim), int(bits), int(group), int(device)
        dev = torch.device("cuda", self.device)
        self.codes = torch.zeros((num_rows, int(hps.LIB.hps_qrows_row_bytes(dim, bits))),
                                 dtype=torch.int8 if bits == 8 else torch.uint8, device=dev)
        self.scales = torch.zeros((num_rows, int(hps.LIB.hps_qrows_groups(dim, group))), dtype=torch.float32, device=dev)
        self._workspace = torch.zeros(int(hps.LIB.hps_qrows_workspace_bytes(num_rows)) // 4, dtype=torch.int32, device=dev)
        torch.cuda.current_stream(dev).synchronize()      # the store is ready for every stream from here on
        self._desc = hps.QRowsStore(self.codes.data_ptr(), self.scales.data_ptr(), self._workspace.data_ptr(), self.num_rows, self.dim,
                                    self.bits, self.group)
        self._desc_p = C.addressof(self._desc)
        self._write, self._read = calls().rows_write, calls().rows_read

    def write(self, rows, slots, held=None):
        """rows: CUDA fp32 / fp16 / bf16 [n, dim] (rows may be apart); slots: CUDA int64 [n]; a slot outside [0, num_rows) is
        skipped, of a slot named several times the last row stays.  held: None, or a tensor like `rows` (or `rows` itself) that takes
        the values the rows stand for once they are held — what read() gives from then on.  Returns `held`.  Runs on torch's
        current stream; may be captured."""
        return self._write(self._desc_p, self.device, self.dim, rows, slots, held)

    def read(self, slots, out=None, dtype=None, default_value: float = 0.0):
        """The rows at `slots` (CUDA int64 [n]) as fp32 (or `dtype`: fp16, bf16) [n, dim]; a slot outside [0, num_rows) reads as
        `default_value`.  Runs on torch's current stream; may be captured."""
        if out is not None and dtype is not None and out.dtype != dtype:
            raise _invalid(f"out: {dtype} asked for, got {out.dtype}")
        return self._read(self._desc_p, self.device, self.dim, slots, out, 0 if dtype is None else elem_type(dtype), default_value)
