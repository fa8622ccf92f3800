"""What the entries for quantised rows, dense layers and the grouping refuse, at the C boundary: every argument is checked before any
device is touched, so this runs without a GPU (the pointers are never followed)."""
import ctypes as C

import pytest

from hugectr_backend_amd import hps

L = hps.LIB
P = 0x10000           # some address; no check follows it
CODES, SCALES, WORK, SLOTS = (P + (k << 24) for k in range(1, 5))


def _store(**kw):
    return hps.QRowsStore(**{**dict(codes=CODES, scales=SCALES, workspace=WORK, num_rows=100, dim=16, bits=8, group=0), **kw})


def _msg():
    return L.hps_last_error().decode()


def _write(store, rows=P, type=0, stride=16, slots=SLOTS, n=4, held=None, held_stride=0):
    return L.hps_qrows_write_device(0, C.addressof(store) if store is not None else None, rows, type, stride, slots, n, held, held_stride, None)


def _read(store, slots=SLOTS, n=4, out=P, type=0, stride=16):
    return L.hps_qrows_read_device(0, C.addressof(store) if store is not None else None, slots, n, 0.0, out, type, stride, None)


def test_row_geometry():
    assert [L.hps_qrows_row_bytes(d, 8) for d in (1, 4, 5, 128)] == [4, 4, 8, 128]
    assert [L.hps_qrows_row_bytes(d, 4) for d in (1, 8, 9, 128)] == [4, 4, 8, 64]
    assert [L.hps_qrows_groups(100, g) for g in (0, 16, 64, 128)] == [1, 7, 2, 1]


@pytest.mark.parametrize("kw,word", [
    (dict(dim=0), "values per row"), (dict(dim=16385), "values per row"), (dict(bits=2), "8 or 4 bits"), (dict(bits=0), "8 or 4 bits"),
    (dict(group=17), "a scale per row"), (dict(group=512), "a scale per row"), (dict(codes=None), "null store"), (dict(scales=None), "null store"),
    (dict(codes=CODES + 2), "aligned"), (dict(scales=SCALES + 1), "aligned"),
])
def test_stores_that_cannot_be(kw, word):
    for call in (_write, _read):
        assert call(_store(**kw)) == hps.ERR_INVALID_ARG and word in _msg()


def test_write_and_read_arguments():
    s = _store()
    assert _write(None) == hps.ERR_INVALID_ARG and _read(None) == hps.ERR_INVALID_ARG
    assert _write(_store(workspace=None)) == hps.ERR_INVALID_ARG
    assert _write(_store(workspace=None, codes=None, scales=None, num_rows=0)) == hps.ERR_INVALID_ARG and "workspace" in _msg()   # (the list has a head of its own)
    assert _write(s, type=3) == hps.ERR_INVALID_ARG and "element type" in _msg()
    assert _read(s, type=-1) == hps.ERR_INVALID_ARG
    assert _write(s, rows=None) == hps.ERR_INVALID_ARG and _write(s, slots=None) == hps.ERR_INVALID_ARG
    assert _read(s, slots=None) == hps.ERR_INVALID_ARG and _read(s, out=None) == hps.ERR_INVALID_ARG
    assert _write(s, stride=15) == hps.ERR_INVALID_ARG and "closer together" in _msg()
    assert _read(s, stride=15) == hps.ERR_INVALID_ARG
    assert _write(s, held=P + (1 << 20), held_stride=3) == hps.ERR_INVALID_ARG
    assert _write(s, held=P + 64, held_stride=16) == hps.ERR_INVALID_ARG and "overlaps" in _msg()
    assert _write(s, held=P, held_stride=32) == hps.ERR_INVALID_ARG and "overlaps" in _msg()
    for kw in (dict(rows=P + 1), dict(rows=P + 2), dict(type=1, rows=P + 1), dict(slots=SLOTS + 4), dict(held=P + (1 << 20) + 2, held_stride=16)):
        assert _write(s, **kw) == hps.ERR_INVALID_ARG and "aligned" in _msg(), kw
    for kw in (dict(out=P + 2), dict(type=2, out=P + 1), dict(slots=SLOTS + 4)):
        assert _read(s, **kw) == hps.ERR_INVALID_ARG and "aligned" in _msg(), kw
    for kw in (dict(held=SLOTS - 64, held_stride=16), dict(rows=CODES + 64), dict(rows=SCALES - 4), dict(slots=WORK + 8),
               dict(held=CODES + 1596, held_stride=16), dict(rows=WORK + (2 * 100 + 65535) * 4)):
        assert _write(s, **kw) == hps.ERR_INVALID_ARG and "overlap" in _msg(), kw
    for kw in (dict(out=SLOTS + 28), dict(out=CODES - 252), dict(out=SCALES + 396), dict(out=P, n=1 << 30)):
        assert _read(s, **kw) == hps.ERR_INVALID_ARG and "overlap" in _msg(), kw
    assert _write(s, n=1 << 31) == hps.ERR_UNSUPPORTED and _read(s, n=1 << 31) == hps.ERR_UNSUPPORTED
    assert _write(s, rows=None, slots=None, n=0) == 0 and _read(s, slots=None, out=None, n=0) == 0


def _create(experts=1, k=16, n=16, type=1, act=0, weights=P, wtype=0, bias=None, on_device=1):
    h = C.c_void_p()
    return L.hps_linear_create(0, experts, k, n, type, act, weights, wtype, bias, on_device, None, C.byref(h))


def test_layers_that_cannot_be():
    for kw, word in ((dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(k=0), "widths"), (dict(n=0), "widths"),
                     (dict(k=(1 << 20) + 1), "widths"), (dict(type=0), "fp16 or bf16"), (dict(type=7), "element type"), (dict(wtype=9), "element type"),
                     (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(weights=None), "null weights"),
                     (dict(weights=P + 2), "aligned"), (dict(weights=P + 1, wtype=1), "aligned"), (dict(bias=P + 2), "aligned")):
        assert _create(**kw) == hps.ERR_INVALID_ARG and word in _msg(), kw
    assert _create(experts=1024, k=1 << 20, n=1 << 20) == hps.ERR_UNSUPPORTED
    assert L.hps_linear_create(0, 1, 16, 16, 1, 0, P, 0, None, 1, None, None) == hps.ERR_INVALID_ARG
    assert L.hps_linear_forward(None, None, None) == hps.ERR_INVALID_ARG
    L.hps_linear_destroy(None)


def test_grouping_arguments():
    call = lambda n=10, e=4, ids=P, off=CODES, order=SCALES, work=None: L.hps_group_rows_device(0, ids, n, e, off, order, work, None)  # noqa: E731
    assert call(e=0) == hps.ERR_INVALID_ARG and call(e=1025) == hps.ERR_INVALID_ARG and "1..1024" in _msg()
    assert call(n=1 << 31) == hps.ERR_UNSUPPORTED
    assert call(off=None) == hps.ERR_INVALID_ARG and call(ids=None) == hps.ERR_INVALID_ARG and call(order=None) == hps.ERR_INVALID_ARG
    assert L.hps_group_rows_workspace_bytes(10, 4) == 0 and L.hps_group_rows_workspace_bytes(100000, 4) > 0
    for kw in (dict(ids=P + 2), dict(off=CODES + 1), dict(order=SCALES + 2), dict(n=100000, work=WORK + 2)):
        assert call(**kw) == hps.ERR_INVALID_ARG and "aligned" in _msg(), kw
    for kw in (dict(order=P), dict(order=P + 36), dict(off=P - 16), dict(off=SCALES + 36), dict(n=100000, work=CODES), dict(n=100000, work=SCALES + 399996)):
        assert call(**kw) == hps.ERR_INVALID_ARG and "overlap" in _msg(), kw
    assert call(n=100000) == hps.ERR_INVALID_ARG      # needs its workspace


def test_without_a_device_every_call_says_so():
    if hps.device_count() > 0:
        pytest.skip("a HIP device is visible")
    import torch
    from hugectr_backend_amd.dense import LinearLayer, group_rows
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    s = _store()
    assert _write(s) == hps.ERR_UNAVAILABLE and _read(s) == hps.ERR_UNAVAILABLE and "no CPU fallback" in _msg()
    assert _create() == hps.ERR_UNAVAILABLE
    assert L.hps_group_rows_device(0, P, 10, 4, CODES, SCALES, None, None) == hps.ERR_UNAVAILABLE
    for make in (lambda: QuantizedRows(4, 4), lambda: LinearLayer(torch.zeros(4, 4))):
        with pytest.raises(hps.HpsError) as e:
            make()
        assert e.value.code == hps.ERR_UNAVAILABLE and "no CPU fallback" in e.value.msg
    with pytest.raises(hps.HpsError):
        group_rows(torch.zeros(4, dtype=torch.int32), 2)


@pytest.mark.gpu
def test_refusals_of_a_layer_and_of_the_wrappers():
    import numpy as np
    import torch
    from hugectr_backend_amd.dense import ExpertLayers, LinearLayer, group_rows
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    layer = LinearLayer(np.ones((8, 6), np.float32))
    experts = ExpertLayers(torch.ones(3, 8, 6), dtype="bf16")
    x, xb = torch.ones(5, 8, dtype=torch.float16, device="cuda"), torch.ones(5, 8, dtype=torch.bfloat16, device="cuda")
    off, idx = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    big = torch.zeros(5, 14, dtype=torch.float16, device="cuda")
    half = torch.zeros(5, 6, dtype=torch.float16, device="cuda")
    store = QuantizedRows(10, 8)
    rows, slots = torch.ones(5, 8, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda")
    bad = [
        lambda: LinearLayer(np.ones((8, 6), np.float32), dtype="fp32"), lambda: LinearLayer(np.ones((8, 6), np.float32), activation="tanh"),
        lambda: LinearLayer(np.ones((8, 6), np.float32), bias=np.ones(8, np.float32)), lambda: ExpertLayers(np.ones((8, 6), np.float32)),
        lambda: layer.forward(xb), lambda: layer.forward(x.cpu()), lambda: layer.forward(x[:, :7]), lambda: layer.forward(x.t()),
        lambda: layer.forward(x[:1].expand(5, 8)), lambda: layer.forward(x, out=torch.empty(4, 6, dtype=torch.float16, device="cuda")),
        lambda: layer.forward(x, out=torch.empty(5, 6, dtype=torch.bfloat16, device="cuda")),
        lambda: layer.forward(x, out=half, out_dtype=torch.float32),
        lambda: layer.forward(x, mul=half.float()), lambda: layer.forward(x, residual=half[:4]),
        lambda: layer.forward(big[:, :8], out=big[:, 8:]),                                   # interleaved: refused, the spans meet
        lambda: layer.forward(x, residual=big[:, :6], out=big[:, 1:7]),
        lambda: experts.forward(xb, off[:3]), lambda: experts.forward(xb, off.long()), lambda: experts.forward(xb, None),
        lambda: experts.forward(xb, off, rows_in=idx[:4], rows_out=idx), lambda: experts.forward(xb, off, rows_in=idx.float()),
        lambda: experts.forward(xb, off, rows_out=idx.cpu()),
        lambda: experts.forward(xb[:3], off, rows_out=idx),                                  # five positions, three rows
        lambda: group_rows(idx.long(), 3), lambda: group_rows(idx, 0), lambda: group_rows(idx, 1025), lambda: group_rows(idx.view(1, 5), 3),
        lambda: group_rows(torch.zeros(10, dtype=torch.int32, device="cuda")[::2], 3),
        lambda: store.write(rows.double(), slots), lambda: store.write(rows[:, :7], slots), lambda: store.write(rows, slots.int()),
        lambda: store.write(rows, slots[:4]), lambda: store.write(rows.cpu(), slots), lambda: store.write(rows, slots.cpu()),
        lambda: store.write(rows, slots, held=rows.half()), lambda: store.write(rows[:1].expand(5, 8), slots),
        lambda: store.read(slots.int()), lambda: store.read(slots, dtype=torch.float64), lambda: store.read(slots, out=rows[:4]),
        lambda: store.read(slots, out=rows, dtype=torch.float16),
        lambda: QuantizedRows(-1, 8), lambda: QuantizedRows(1, 0), lambda: QuantizedRows(1, 8, bits=5), lambda: QuantizedRows(1, 8, group=24),
    ]
    def odd(**kw):       # at the C boundary: pointers that torch does not make
        a = hps.LinearArgs(x.data_ptr(), 8, 5, half.data_ptr(), 6, 5, 1, 0)
        a.rows = 5
        for name, value in kw.items():
            setattr(a, name, value)
        hps._check(L.hps_linear_forward(layer._h, C.addressof(a), None))
    odd()
    bad += [lambda: odd(x=x.data_ptr() + 1), lambda: odd(out=half.data_ptr() + 1), lambda: odd(out_type=0, out=big.data_ptr() + 2),
            lambda: odd(mul=big.data_ptr() + 1, mul_stride=14), lambda: odd(residual=big.data_ptr() + 1, residual_stride=14),
            lambda: odd(rows_in=half.data_ptr() + 56), lambda: odd(rows_out=half.data_ptr()), lambda: odd(offsets=half.data_ptr() - 4),
            lambda: odd(rows_in=idx.data_ptr() + 2), lambda: odd(rows_out=idx.data_ptr() + 1), lambda: odd(offsets=off.data_ptr() + 2)]
    for k, f in enumerate(bad):
        with pytest.raises(hps.HpsError) as e:
            f()
        assert e.value.code == hps.ERR_INVALID_ARG, (k, e.value)
    for call in (lambda: L.hps_group_rows_device(99, idx.data_ptr(), 5, 3, off.data_ptr(), slots.data_ptr(), None, None),
                 lambda: L.hps_qrows_read_device(99, store._desc_p, slots.data_ptr(), 5, 0.0, rows.data_ptr(), 0, 8, None),
                 lambda: L.hps_qrows_write_device(-1, store._desc_p, rows.data_ptr(), 0, 8, slots.data_ptr(), 5, None, 0, None)):
        assert call() == hps.ERR_INVALID_ARG and "not visible" in _msg()
    torch.cuda.synchronize()
    assert layer.forward(x[:0]).shape == (0, 6) and experts.forward(xb[:0], off).shape == (0, 6)


def test_the_native_calls_on_torch_tensors():
    """What the module refuses by itself, as HpsError; what is not an argument at all stays Python's own error."""
    import torch
    from hugectr_backend_amd.quantized_rows import calls
    c, ids = calls(), torch.zeros(4, dtype=torch.int32)
    for f in (lambda: c.group_rows(ids, 2), lambda: c.group_rows(3, 2), lambda: c.group_rows(ids.to_sparse(), 2), lambda: c.group_rows(ids),
              lambda: c.rows_read(0, 0, 4, torch.zeros(3, dtype=torch.int64), None, 0, 0.0), lambda: c.rows_write(0, 0, 4, None, ids, None),
              lambda: c.linear_forward(0, 0, 1, 4, 4, 1, ids, None, None, None, None, None, None, 1)):
        with pytest.raises(hps.HpsError) as e:
            f()
        assert e.value.code == hps.ERR_INVALID_ARG and e.value.msg
    for f in (lambda: c.group_rows(torch.zeros(4, dtype=torch.int32), "two"), lambda: c.rows_read(None, 0, 4, ids, None, 0, 0.0)):
        with pytest.raises(TypeError):
            f()
