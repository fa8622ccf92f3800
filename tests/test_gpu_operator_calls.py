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
