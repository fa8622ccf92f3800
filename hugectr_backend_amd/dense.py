"""Host-side handle of the dense step behind a DLRM lookup (bottom MLP + dot interaction) — a thin ctypes
wrapper over the hps_dense_* entry points of libhps_amd.so (include/hps_amd.h) — and of the layers that come behind it:
LinearLayer, ExpertLayers (hps_linear_*) and group_rows (hps_group_rows_*), whose calls are native (csrc/python/torch_calls.cpp).  The arithmetic is the HIP/MFMA code in
csrc/dense/; torch is used for device buffers only.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import hps
from .quantized_rows import _invalid, calls, elem_type

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}


class DenseInteraction:
    """weights[l]: fp32 [K_l, dims[l]] (x @ W convention), biases[l]: fp32 [dims[l]]."""

    def __init__(self, weights, biases, num_tables: int, emb_dim: int, device: int = 0):
        ws = [np.ascontiguousarray(w, dtype=np.float32) for w in weights]
        bs = [np.ascontiguousarray(b, dtype=np.float32) for b in biases]
        if not ws or len(ws) != len(bs):
            raise hps.HpsError(hps.ERR_INVALID_ARG, "one weight matrix and one bias vector per layer")
        num_dense = ws[0].shape[0]
        k = num_dense
        for w, b in zip(ws, bs):
            if w.ndim != 2 or w.shape[0] != k or b.shape != (w.shape[1],):
                raise hps.HpsError(hps.ERR_INVALID_ARG, "layer shapes do not chain")
            k = w.shape[1]
        L = len(ws)
        dims = (C.c_uint32 * L)(*[w.shape[1] for w in ws])
        wp = (C.c_void_p * L)(*[w.ctypes.data for w in ws])
        bp = (C.c_void_p * L)(*[b.ctypes.data for b in bs])
        h = C.c_void_p()
        hps._check(hps.LIB.hps_dense_create(device, num_dense, L, dims, wp, bp, num_tables, emb_dim, C.byref(h)))
        self._h = h
        self.device = device
        self.num_dense = num_dense
        self.num_tables = num_tables
        self.emb_dim = emb_dim
        self.out_dim = int(hps.LIB.hps_dense_out_dim(h))
        self.out_stride = int(hps.LIB.hps_dense_out_stride(h))

    def forward(self, dense, embeddings, batch: int, out=None):
        """dense: CUDA fp32 [batch, num_dense]; embeddings: CUDA fp32, the lookup's OUTPUT0 (table-major
        [num_tables, batch, emb_dim], flat is fine).  Returns a CUDA fp16 tensor [batch, out_stride] (columns
        [0, out_dim) are the result, the rest zero padding).  Runs on torch's current stream."""
        import torch
        assert dense.is_cuda and embeddings.is_cuda and dense.dtype == torch.float32 and embeddings.dtype == torch.float32
        assert dense.is_contiguous() and embeddings.is_contiguous()
        assert dense.numel() == batch * self.num_dense and embeddings.numel() == self.num_tables * batch * self.emb_dim
        if out is None:
            out = torch.empty((batch, self.out_stride), dtype=torch.float16, device=dense.device)
        stream = torch.cuda.current_stream(dense.device).cuda_stream
        hps._check(hps.LIB.hps_dense_forward(self._h, dense.data_ptr(), embeddings.data_ptr(), batch, out.data_ptr(),
                                             C.c_void_p(stream)))
        return out

    def lookup_interact(self, session, keys, batch: int, dense, out=None):
        """Fused arrangement: `keys` CUDA int64 [num_tables * batch] (table-major, one key per table per sample)
        looked up through `session` (a LookupSession of a ps_direct_access model) and fed to the interaction from
        the cache slots / miss staging directly — no OUTPUT0.  Returns the same tensor as forward().  Blocking."""
        import torch
        assert keys.is_cuda and keys.dtype == torch.int64 and keys.is_contiguous() and keys.numel() == self.num_tables * batch
        assert dense.is_cuda and dense.dtype == torch.float32 and dense.is_contiguous() and dense.numel() == batch * self.num_dense
        if out is None:
            out = torch.empty((batch, self.out_stride), dtype=torch.float16, device=keys.device)
        torch.cuda.current_stream(keys.device).synchronize()      # the session works on its own stream
        hps._check(hps.LIB.hps_session_lookup_interact_device(session._h, self._h, keys.data_ptr(), batch, dense.data_ptr(),
                                                              out.data_ptr()))
        return out

    def close(self):
        if getattr(self, "_h", None):
            hps.LIB.hps_dense_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001
            pass


class ExpertLayers:
    """y = act(x W_e + b_e) * mul + residual for every expert e over its own run of rows, on the matrix cores: operands of `dtype`
    (fp16 or bf16), sums and everything behind them in fp32, one rounding at the end.

    weights: [num_experts, in_dim, out_dim] (x @ W convention), biases: None or [num_experts, out_dim]; numpy arrays or torch tensors,
    laid out for the kernels once, here: a copy of them that new weights do not reach (they take a new object).  activation: none, relu,
    gelu (with the error function), silu, sigmoid.  For serving: results carry no gradient."""

    def __init__(self, weights, biases=None, activation: str = "none", dtype="fp16", device: int = 0):
        import torch
        if hps.device_count() <= 0:
            raise hps.HpsError(hps.ERR_UNAVAILABLE, "dense layers need a HIP device and none is visible; there is no CPU fallback")
        dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}.get(dtype, dtype)
        if dtype not in (torch.float16, torch.bfloat16):
            raise _invalid(f"dense layers take fp16 or bf16 operands, got {dtype}")
        if activation not in ACTIVATIONS:
            raise _invalid(f"activation: one of {', '.join(ACTIVATIONS)} expected, got {activation!r}")
        dev = torch.device("cuda", int(device))
        w = torch.as_tensor(weights)
        if w.dim() != 3:
            raise _invalid(f"weights: [num_experts, in_dim, out_dim] expected, got shape {tuple(w.shape)}")
        if w.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            w = w.float()
        w = w.to(dev).resolve_neg().contiguous()
        b = None
        if biases is not None:
            b = torch.as_tensor(biases).to(device=dev, dtype=torch.float32).resolve_neg().contiguous()
            if tuple(b.shape) != (w.shape[0], w.shape[2]):
                raise _invalid(f"biases: [{w.shape[0]}, {w.shape[2]}] expected, got {tuple(b.shape)}")
        self.num_experts, self.in_dim, self.out_dim = (int(v) for v in w.shape)
        self.dtype, self.activation, self.device = dtype, activation, int(device)
        self._call, self._type = calls().linear_forward, elem_type(dtype)
        h = C.c_void_p()
        hps._check(hps.LIB.hps_linear_create(self.device, self.num_experts, self.in_dim, self.out_dim, elem_type(dtype),
                                             ACTIVATIONS[activation], w.data_ptr(), elem_type(w.dtype), b.data_ptr() if b is not None else None,
                                             1, torch.cuda.current_stream(dev).cuda_stream, C.byref(h)))
        self._h = h

    def forward(self, x, offsets, rows_in=None, rows_out=None, mul=None, residual=None, out=None, out_dtype=None):
        """x: CUDA `dtype` [x_rows, in_dim] (rows may be apart).  offsets: CUDA int32 [num_experts + 1]; expert e has the positions
        [offsets[e], offsets[e+1]) (clamped to the positions there are, read as their running maximum); None with one expert: all of
        them.  rows_in / rows_out: None or CUDA int32, one entry per position: the row of x it reads (outside x: zeros) and the row of
        out, mul and residual it has (outside out: not written; a row named twice holds, element by element, the result of either).
        Without them position p is row p.  group_rows() makes offsets and such an index from expert numbers.
        out: [rows, out_dim] of `dtype` or fp32; rows of no run stay as they were.  Without `out` a new tensor of `out_dtype` is
        returned, one row per position; rows of no run, and rows that rows_out does not name, are zero.
        mul, residual: None or `dtype`, rows like out's; either may be `out` itself (rows_out then names no row twice).
        Runs on torch's current stream; may be captured; calls may overlap."""
        return self._run(x, offsets, rows_in, rows_out, mul, residual, out, out_dtype)

    def _run(self, x, offsets, rows_in, rows_out, mul, residual, out, out_dtype):
        if out is not None and out_dtype is not None and out.dtype != out_dtype:
            raise _invalid(f"out: {out_dtype} asked for, got {out.dtype}")
        return self._call(self._h.value if self._h else 0, self.device, self._type, self.in_dim, self.out_dim, self.num_experts, x, offsets, rows_in,
                          rows_out, mul, residual, out, self._type if out_dtype is None else elem_type(out_dtype))

    def close(self):
        if getattr(self, "_h", None):
            hps.LIB.hps_linear_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001
            pass


class LinearLayer(ExpertLayers):
    """y = act(x W + b) * mul + residual: one layer over all rows.  weight: [in_dim, out_dim], bias: None or [out_dim]; the rest as in
    ExpertLayers."""

    def __init__(self, weight, bias=None, activation: str = "none", dtype="fp16", device: int = 0):
        super().__init__(weight[None], None if bias is None else bias[None], activation, dtype, device)

    def forward(self, x, mul=None, residual=None, out=None, out_dtype=None):
        """x: CUDA `dtype` [rows, in_dim]; out, mul, residual: [rows, out_dim] as in ExpertLayers.forward.  Runs on torch's current
        stream; may be captured; calls may overlap."""
        if out is not None and out.shape[0] != x.shape[0]:
            raise _invalid(f"out: {x.shape[0]} rows expected, got {out.shape[0]}")
        return self._run(x, None, None, None, mul, residual, out, out_dtype)


def group_rows(ids, num_experts: int):
    """(offsets, order) of a stable sort of the positions by expert number: ids CUDA int32 [n]; offsets int32 [num_experts + 1],
    order int32 [n]: expert e has the positions order[offsets[e] : offsets[e+1]] in ascending order; positions whose id is outside
    [0, num_experts) come behind the last run.  num_experts <= 1024.  Runs on torch's current stream; may be captured."""
    return calls().group_rows(ids, num_experts)
