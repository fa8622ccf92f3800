"""How the operators behind the lookup (quantised rows, layers, experts, grouping) sit in a program: the thread's HIP error, outputs of their own."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


def _calls(torch):
    """Every entry once, outputs in hand (torch launches nothing meanwhile)."""
    from hugectr_backend_amd import hps
    from hugectr_backend_amd.dense import LinearLayer
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    layer = LinearLayer(torch.randn(64, 40, generator=g, device="cuda"))
    store = QuantizedRows(400000, 4)
    x, y = torch.randn(9, 64, generator=g, device="cuda").half(), torch.empty(9, 40, dtype=torch.float16, device="cuda")
    big, ybig = torch.randn(5000, 64, generator=g, device="cuda").half(), torch.empty(5000, 40, dtype=torch.float16, device="cuda")
    slots, rows, back = torch.arange(300000, device="cuda"), torch.randn(300000, 4, generator=g, device="cuda"), torch.empty(300000, 4, device="cuda")
    ids = torch.randint(0, 300, (100000,), generator=g, device="cuda").int()
    off, order = torch.empty(301, dtype=torch.int32, device="cuda"), torch.empty(100000, dtype=torch.int32, device="cuda")
    work = torch.empty(hps.LIB.hps_group_rows_workspace_bytes(100000, 300) // 4 + 1, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    return [lambda: layer.forward(x, out=y), lambda: layer.forward(big, out=ybig), lambda: store.write(rows[:5], slots[:5]),
            lambda: store.write(rows[:5000], slots[:5000]), lambda: store.write(rows, slots), lambda: store.read(slots, out=back),
            lambda: hps._check(hps.LIB.hps_group_rows_device(0, ids.data_ptr(), 1000, 300, off.data_ptr(), order.data_ptr(), work.data_ptr(), stream)),
            lambda: hps._check(hps.LIB.hps_group_rows_device(0, ids.data_ptr(), 100000, 300, off.data_ptr(), order.data_ptr(), work.data_ptr(), stream))]


def test_an_error_that_the_caller_has_yet_to_look_at_stays():
    """A HIP error of the caller's own (a device that is not there) is still pending behind every entry, and no entry takes it for its own."""
    import torch
    from hugectr_backend_amd import hps
    hip = hps.LIB                                   # (the runtime it is linked with)
    for k, call in enumerate(_calls(torch)):
        assert hip.hipGetLastError() == 0, k
        try:
            assert hip.hipSetDevice(9999) != 0
            left = hip.hipPeekAtLastError()
            call()
            assert left != 0 and hip.hipPeekAtLastError() == left, k
        finally:
            hip.hipGetLastError()
    torch.cuda.synchronize()


def test_an_entry_leaves_no_error_of_its_own():
    import torch
    from hugectr_backend_amd import hps
    torch.cuda.synchronize()
    hip, h = hps.LIB, C.c_void_p()
    assert hip.hipGetLastError() == 0
    rc = hip.hps_linear_create(0, 256, 1 << 20, 512, 1, 0, 0x10000, 0, None, 0, None, C.byref(h))      # 549 GB of weights: nothing is read
    assert rc == hps.ERR_INTERNAL and hip.hipPeekAtLastError() == 0
    rc = hip.hps_group_rows_device(99, 0x10000, 5, 3, 0x20000, 0x30000, None, None)                   # no such device
    assert rc == hps.ERR_INVALID_ARG and hip.hipPeekAtLastError() == 0


def _poisoned(torch, shape, dtype):
    """The next tensor of this size comes from memory full of NaN."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    t = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
    torch.cuda.synchronize()
    del t


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,k,n,e", [(1, 8, 8, 1), (7, 40, 33, 3), (300, 479, 256, 64), (600, 40, 48, 20), (2000, 33, 31, 5), (3000, 40, 1, 3), (30000, 24, 1, 2),
                                     (5000, 40, 72, 7), (9000, 64, 264, 3), (16384, 40, 136, 4), (40000, 40, 264, 4)])
def test_a_new_output_holds_nothing_that_was_there_before(m, k, n, e, dtype):
    """rows_out that names rows twice, rows outside the output, rows of no run: every row of a new tensor is a position's or zeros, never what lay
    in the memory.  (A permutation takes the same way and names them all.)"""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers, group_rows
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(m + n)
    x = torch.randn(m, k, generator=g, device="cuda").to(dt)
    w = (torch.randn(e, k, n, generator=g, device="cuda") / k ** 0.5).to(dt)
    layer = ExpertLayers(w, 0.3 * torch.randn(e, n, generator=g, device="cuda"), activation="sigmoid", dtype=dt)      # (no value of a run is zero)
    ids = torch.randint(-1, e, (m,), generator=g, device="cuda").int()
    offsets, order = group_rows(ids, e)
    some = torch.randint(-2, m + 2, (m,), generator=g, device="cuda").int()
    few = torch.full((m,), m // 2, dtype=torch.int32, device="cuda")                     # all positions name one row
    none = torch.full((m,), -1, dtype=torch.int32, device="cuda")
    low = torch.arange(m, device="cuda").int() // 2
    runs = torch.zeros(m, dtype=torch.bool, device="cuda")
    runs[: int(offsets[e])] = True
    for rows_out in (some, few, none, low, order):
        for out_t in (dt, torch.float32):
            filled = torch.full((m, n), 9.0, dtype=out_t, device="cuda")
            layer.forward(x, offsets, rows_in=order, rows_out=rows_out, out=filled)      # what the positions write, and nothing else
            _poisoned(torch, (m, n), out_t)
            got = layer.forward(x, offsets, rows_in=order, rows_out=rows_out, out_dtype=out_t)
            ok = (rows_out >= 0) & (rows_out < m)
            by_run = torch.zeros(m, dtype=torch.int64, device="cuda").index_add_(0, rows_out[ok & runs].long(), torch.ones_like(rows_out[ok & runs]).long())
            by_rest = torch.zeros(m, dtype=torch.int64, device="cuda").index_add_(0, rows_out[ok & ~runs].long(), torch.ones_like(rows_out[ok & ~runs]).long())
            assert not torch.isnan(got).any(), "memory that nobody wrote"
            assert (got[by_run == 0] == 0).all()
            one = (by_run == 1) & (by_rest == 0)
            assert torch.equal(got[one], filled[one]) and (filled[one] != 9).all()
            many = by_run > 0                        # element by element one of the positions' results, or a zero of a position of no run
            assert ((got[many] != 0) | (by_rest[many] > 0)[:, None]).all()
    alone = ExpertLayers(w[:1], activation="sigmoid", dtype=dt)                          # one layer without offsets
    _poisoned(torch, (m, n), dt)
    got = alone.forward(x, None, rows_out=some)
    named = torch.zeros(m + 4, dtype=torch.bool, device="cuda")
    named[some.long() + 2] = True
    assert not torch.isnan(got).any() and (got[~named[2: m + 2]] == 0).all() and (got[named[2: m + 2]] != 0).all()


def test_rows_that_nobody_names_need_a_row_per_position():
    import torch
    from hugectr_backend_amd import hps
    from hugectr_backend_amd.dense import LinearLayer
    layer = LinearLayer(torch.ones(8, 6))
    x, out = torch.ones(5, 8, dtype=torch.float16, device="cuda"), torch.ones(7, 6, dtype=torch.float16, device="cuda")
    names = torch.arange(5, device="cuda").int()
    torch.cuda.synchronize()

    def call(**kw):
        a = hps.LinearArgs(x.data_ptr(), 8, 5, out.data_ptr(), 6, 5, 1, 2)
        a.rows, a.rows_out = 5, names.data_ptr()
        for name, value in kw.items():
            setattr(a, name, value)
        return hps.LIB.hps_linear_forward(layer._h, C.addressof(a), None)
    assert call() == 0
    assert call(out_rows=7) == hps.ERR_INVALID_ARG and "names" in hps.LIB.hps_last_error().decode()
    torch.cuda.synchronize()
    assert (out[:5] == 8).all() and (out[5:] == 1).all()


def test_a_new_output_by_index_in_a_replayed_graph():
    import torch
    from hugectr_backend_amd.dense import ExpertLayers
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    for m, n in ((200, 40), (9000, 264)):
        x, w = torch.randn(m, 40, generator=g, device="cuda").half(), torch.randn(1, 40, n, generator=g, device="cuda")
        layer, names = ExpertLayers(w, activation="sigmoid"), torch.zeros(m, dtype=torch.int32, device="cuda")
        layer.forward(x, None, rows_out=names)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer.forward(x, None, rows_out=names)
        for _ in range(4):
            names.copy_(torch.randperm(m, generator=g, device="cuda").int() * 2 % (m + 50))
            got.fill_(float("nan"))
            graph.replay()
            want = layer.forward(x, None, rows_out=names, out=torch.zeros_like(got))
            torch.cuda.synchronize()
            once = torch.bincount(names.long().clamp(max=m), minlength=m + 1)[:m]
            assert not torch.isnan(got).any() and torch.equal(got[once < 2], want[once < 2]) and (got[once == 0] == 0).all()


def test_negated_views_are_not_read_as_what_lies_under_them():
    """torch.imag of a conjugate is a view whose memory holds the negated values."""
    import torch
    from hugectr_backend_amd import hps
    from hugectr_backend_amd.dense import ExpertLayers, LinearLayer, group_rows
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    z = torch.complex(torch.ones(6, 1), torch.full((6, 1), 2.0)).cuda()
    column = z.conj().imag                                       # [6, 1], stride 2
    assert column.is_neg() and (column == -2).all()
    store, slots = QuantizedRows(6, 1), torch.arange(6, device="cuda")
    x = torch.ones(6, 8, dtype=torch.float16, device="cuda")
    layer = LinearLayer(torch.eye(8))
    neg = torch._neg_view
    for call in (lambda: store.write(column, slots), lambda: store.write(column.resolve_neg(), slots, held=column), lambda: store.write(column.resolve_neg(), neg(slots)),
                 lambda: store.read(slots, out=column), lambda: layer.forward(neg(x)), lambda: layer.forward(x, mul=neg(x)),
                 lambda: layer.forward(x, residual=neg(x)), lambda: layer.forward(x, out=neg(x)), lambda: layer.forward(x, mul=torch._efficientzerotensor((6, 8), dtype=torch.float16, device="cuda")),
                 lambda: group_rows(neg(slots.int()), 3)):
        with pytest.raises(hps.HpsError, match="holds its values") as e:
            call()
        assert e.value.code == hps.ERR_INVALID_ARG
    store.write(column.resolve_neg(), slots)
    assert (store.read(slots) + 2).abs().max() <= 2.0 ** -22
    w, b = neg(2 * torch.eye(8, device="cuda")), neg(torch.ones(1, 8, device="cuda"))
    assert torch.equal(ExpertLayers(w[None], b).forward(x, torch.tensor([0, 6], dtype=torch.int32, device="cuda")), torch.full_like(x, -3))


@pytest.mark.parametrize("m", [2_200_003, 4097])
def test_a_new_output_of_many_rows(m):
    """More rows than sixteen blocks hold the names of; narrow rows, a name list that starts off 16 bytes."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    x = torch.randn(m, 4, generator=g, device="cuda").half()
    names = torch.randint(-1, m, (m + 1,), generator=g, device="cuda").int()[1:]
    for n in (1, 3):
        layer = ExpertLayers(torch.randn(1, 4, n, generator=g, device="cuda"), activation="sigmoid")
        _poisoned(torch, (m, n), torch.float16)
        got = layer.forward(x, None, rows_out=names)
        named = torch.zeros(m + 1, dtype=torch.bool, device="cuda")
        named[names.long() + 1] = True
        assert not torch.isnan(got).any() and (got[~named[1:]] == 0).all() and (got[named[1:]] != 0).all()
