"""Embedding rows held in 8 or 4 bits on the GPU, addressed by slot — a thin ctypes wrapper over the hps_qrows_* entry points of
libhps_amd.so (include/hps_amd.h).  The arithmetic is the HIP code in csrc/cache/qrows_kernels.hip; torch is used for device
buffers only.
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


def current_stream():
    """device -> hipStream_t of torch's current stream there (without the Stream object around it: 1 us of a 6-us call)."""
    import torch
    return torch._C._cuda_getCurrentRawStream


def row_stride(t, width: int, name: str, device: int) -> int:
    """Distance of the rows of a 2-D CUDA tensor on `device` whose values lie side by side, `width` of them per row."""
    if t.get_device() != device:
        raise _invalid(f"{name}: a tensor on cuda:{device} expected, got one on {t.device}")
    if t.dim() != 2 or t.shape[1] != width:
        raise _invalid(f"{name}: rows of {width} values expected, got shape {tuple(t.shape)}")
    rows, side = t.stride()
    if rows == width and side == 1:
        return width
    if width > 1 and side != 1:
        raise _invalid(f"{name}: the values of a row have to lie side by side")
    if t.shape[0] <= 1:
        return width
    if rows < width:
        raise _invalid(f"{name}: the rows overlap (stride {rows}, {width} values)")
    return rows


class QuantizedRows:
    """`num_rows` rows of `dim` values in 8 (or 4) bits plus one fp32 scale per row, or per `group` consecutive values (16, 32, 64,
    128 or 256).  A value is held as the nearest multiple (ties to even) of scale = max|x| / 127 (7) of its group.  A group whose
    largest magnitude is below 2^-100 is held as zeros; one with a NaN or an infinity reads back as NaN.

    codes   [num_rows, row_bytes] int8 (8 bits) / uint8 (4 bits, two per byte, the first in the low half); rows padded to 4 bytes
    scales  [num_rows, groups] fp32
    Rows never written are zeros.  One write at a time per store (whatever the stream); reads beside reads are free, a read beside
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
        self._slot_type, self._stream = torch.int64, current_stream()
        self._like = {}        # an empty tensor of every type read so far: new_empty of the same type is 0.5 us of a call less

    def _slots(self, slots) -> int:
        if slots.dtype != self._slot_type or slots.get_device() != self.device or slots.dim() != 1 or not slots.is_contiguous():
            raise _invalid(f"slots: a contiguous vector of int64 on cuda:{self.device} expected, got {slots.dtype} {tuple(slots.shape)} "
                           f"on {slots.device}")
        return slots.shape[0]

    def write(self, rows, slots, held=None):
        """rows: CUDA fp32 / fp16 / bf16 [n, dim] (rows may be apart); slots: CUDA int64 [n]; a slot outside [0, num_rows) is
        skipped, of a slot named several times the last row stays.  held: None, or a tensor like `rows` (or `rows` itself) that takes
        the values the rows stand for once they are held — what read() gives from then on.  Returns `held`.  Runs on torch's
        current stream; may be captured."""
        n = self._slots(slots)
        stride = row_stride(rows, self.dim, "rows", self.device)
        if rows.shape[0] != n:
            raise _invalid(f"write: {rows.shape[0]} rows for {n} slots")
        hp, hs = None, 0
        if held is not None:
            hs = row_stride(held, self.dim, "held", self.device)
            if held.dtype != rows.dtype or held.shape[0] != n:
                raise _invalid(f"held: {n} rows of {rows.dtype} expected, got {held.shape[0]} of {held.dtype}")
            hp = held.data_ptr()
        rc = hps.LIB.hps_qrows_write_device(self.device, self._desc_p, rows.data_ptr(), elem_type(rows.dtype), stride, slots.data_ptr(), n, hp,
                                            hs, self._stream(self.device))
        if rc:
            hps._check(rc)
        return held

    def read(self, slots, out=None, dtype=None, default_value: float = 0.0):
        """The rows at `slots` (CUDA int64 [n]) as fp32 (or `dtype`: fp16, bf16) [n, dim]; a slot outside [0, num_rows) reads as
        `default_value`.  Runs on torch's current stream; may be captured."""
        n = self._slots(slots)
        if out is None:
            like = self._like.get(dtype)
            if like is None:
                import torch
                elem_type(dtype or torch.float32)
                like = self._like[dtype] = torch.empty(0, dtype=dtype or torch.float32, device=self.codes.device)
            out, stride = like.new_empty(n, self.dim), self.dim
        else:
            if dtype is not None and out.dtype != dtype:
                raise _invalid(f"out: {dtype} asked for, got {out.dtype}")
            stride = row_stride(out, self.dim, "out", self.device)
            if out.shape[0] != n:
                raise _invalid(f"out: {n} rows expected, got {out.shape[0]}")
        rc = hps.LIB.hps_qrows_read_device(self.device, self._desc_p, slots.data_ptr(), n, default_value, out.data_ptr(),
                                           elem_type(out.dtype), stride, self._stream(self.device))
        if rc:
            hps._check(rc)
        return out
