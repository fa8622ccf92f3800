"""Dense layers (csrc/dense/linear_kernels.hip) and the grouping of rows by expert (csrc/dense/group_rows.hip).

Layers are compared with y = act(x W + b) * mul + residual in 64 bits over the same (already rounded) operands.  The bound, value by
value, from the places that round:
  sum          K products of the operands are exact in fp32; adding them in any order and the bias costs at most (K + 2) 2^-24 of
               sum |x||w| + |b|; an activation passes it on at most 1.13-fold (the steepest slope of gelu; silu 1.1, the others 1)
  activation   none, relu: exact; gelu, silu, sigmoid: 2^-20 of max(1, |y|) (the error function is good to 1.5e-7 and about ten fp32
               operations follow; the exponential's argument is rounded, (|y| + 2) 2^-23 of e^-y)
  epilogue     the product with mul and the sum with residual: 2^-24 of each result
  output       half a step of its type, 2^-11 (fp16), 2^-8 (bf16), 2^-24 (fp32) of the value, 2^-25 below fp16's normal numbers
The grouping is compared for equality.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def _act64(y, act):
    import torch
    return {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * torch.special.ndtr(v),
            "silu": lambda v: v * torch.sigmoid(v), "sigmoid": torch.sigmoid}[act](y)


def _check(got, x, w, b, act, mul=None, residual=None):
    """got [m, n] against the 64-bit layer over x [m, k], w [k, n], b [n] or None; every bound as above."""
    import torch
    K = x.shape[1]
    x, w = x.double().cpu(), w.double().cpu()
    b = torch.zeros(w.shape[1], dtype=torch.float64) if b is None else b.double().cpu()
    s = x @ w + b
    off = (K + 2) * 2.0 ** -24 * (x.abs() @ w.abs() + b.abs())
    y = _act64(s, act)
    off = 1.13 * off
    if act not in ("none", "relu"):
        off = off + 2.0 ** -20 * s.abs().clamp(min=1)
    if mul is not None:
        m = mul.double().cpu()
        y, off = y * m, off * m.abs()
        off = off + 2.0 ** -24 * y.abs()
    if residual is not None:
        y = y + residual.double().cpu()
        off = off + 2.0 ** -24 * y.abs()
    half = HALF[str(got.dtype).split(".")[1]]
    off = off * (1 + half) + half * y.abs() + 2.0 ** -25
    bad = (got.double().cpu() - y).abs() > off
    assert not bad.any(), (int(bad.sum()), float(((got.double().cpu() - y).abs() / off).max()))


def _operands(torch, m, k, n, dt, seed, experts=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda").to(dt)
    w = (torch.randn(experts, k, n, generator=g, device="cuda") / math.sqrt(k)).to(dt)
    b = 0.3 * torch.randn(experts, n, generator=g, device="cuda")
    return x, w, b


SHAPES = [(1, 1, 1), (1, 1024, 1024), (2, 31, 33), (5, 8, 7), (16, 479, 64), (17, 33, 100), (33, 64, 257), (64, 100, 31), (65, 65, 65), (100, 512, 1),
          (128, 128, 128), (200, 127, 300), (257, 40, 8), (300, 1, 50), (511, 96, 129), (1000, 479, 256), (700, 300, 1)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_matches_64_bits(m, k, n, dtype):
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    dt = getattr(torch, dtype)
    x, w, b = _operands(torch, m, k, n, dt, m + 7 * k + 13 * n)
    layer = LinearLayer(w[0], b[0], dtype=dt)
    for out_t in (dt, torch.float32):
        got = layer.forward(x, out_dtype=out_t)
        assert got.dtype == out_t and got.shape == (m, n)
        _check(got, x, w[0], b[0], "none")
    layer.close()


@pytest.mark.parametrize("m,k,n", [(20000, 96, 512), (70000, 40, 264), (3000, 2000, 600)])
def test_linear_large_batches(m, k, n):
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    x, w, b = _operands(torch, m, k, n, torch.float16, m)
    got = LinearLayer(w[0], b[0], activation="relu").forward(x, out_dtype=torch.float32)
    pick = torch.cat((torch.arange(300), torch.arange(m // 2, m // 2 + 300), torch.arange(m - 300, m)))
    _check(got[pick.cuda()], x[pick.cuda()], w[0], b[0], "relu")
    # every other row: the same row alone (its sums run in another order: twice the sum's bound apart at most)
    alone = LinearLayer(w[0], b[0], activation="relu").forward(x[m - 50: m - 40].contiguous(), out_dtype=torch.float32)
    lim = 2 * (k + 2) * 2.0 ** -24 * (x[m - 50: m - 40].float().abs() @ w[0].float().abs() + b.abs()) + 2.0 ** -23
    assert ((got[m - 50: m - 40] - alone).abs() <= lim).all()


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("m", [3, 50, 300])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_activation_mul_and_residual(act, m, dtype):
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    dt = getattr(torch, dtype)
    k, n = 72, 90
    x, w, b = _operands(torch, m, k, n, dt, m)
    x = (3 * x.float()).to(dt)
    mul, res = _operands(torch, m, n, 2, dt, 2)[0], _operands(torch, m, n, 2, dt, 3)[0]
    layer = LinearLayer(w[0], b[0], activation=act, dtype=dt)
    for mm, rr in ((None, None), (mul, None), (None, res), (mul, res)):
        _check(layer.forward(x, mul=mm, residual=rr, out_dtype=torch.float32), x, w[0], b[0], act, mm, rr)
        _check(layer.forward(x, mul=mm, residual=rr), x, w[0], b[0], act, mm, rr)
    nobias = LinearLayer(w[0].float().cpu().numpy(), activation=act, dtype=dt)
    _check(nobias.forward(x), x, w[0], None, act)
    # in place over residual, and over mul
    r = res.clone()
    assert layer.forward(x, mul=mul, residual=r, out=r) is r
    assert torch.equal(r, layer.forward(x, mul=mul, residual=res))
    r = mul.clone()
    layer.forward(x, mul=r, residual=res, out=r)
    assert torch.equal(r, layer.forward(x, mul=mul, residual=res))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m", [5, 100, 400])
def test_every_width_below_and_beyond_eight(m, dtype):
    """K and N of every residue modulo 8 (the last values of a row are loaded and stored 4 + 2 + 1), in every kernel, with mul and
    residual, into both output types: the outputs between sentinels, the rows of x next to each other."""
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    dt = getattr(torch, dtype)
    for n in list(range(1, 17)) + [31, 39, 47, 61, 69, 77, 127, 131]:
        k = n if n < 17 else 2 * n
        x, w, b = _operands(torch, m, k, n, dt, n)
        mul, res = _operands(torch, m, n, 1, dt, n + 1)[0], _operands(torch, m, n, 1, dt, n + 2)[0]
        for act in ("relu", "silu"):
            layer = LinearLayer(w[0], b[0], activation=act, dtype=dt)
            for out_t in (dt, torch.float32):
                wide = torch.full((m, n + 3), 77.0, dtype=out_t, device="cuda")
                layer.forward(x, mul=mul, residual=res, out=wide[:, 1: 1 + n])
                _check(wide[:, 1: 1 + n], x, w[0], b[0], act, mul, res)
                assert (wide[:, 0] == 77).all() and (wide[:, 1 + n:] == 77).all()


def test_activations_far_out_stay_finite():
    """Sums of +-60000: no exponential overflows into a NaN."""
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    x = torch.tensor([[60000.0], [-60000.0], [88.0], [-88.0], [-104.0], [0.0], [-0.0]], dtype=torch.float16, device="cuda")
    w = torch.ones(1, 8, dtype=torch.float16)
    for act in ("none", "relu", "gelu", "silu", "sigmoid"):
        got = LinearLayer(w, activation=act).forward(x, out_dtype=torch.float32)
        assert torch.isfinite(got).all(), act
        _check(got, x, w, None, act)


@pytest.mark.parametrize("m", [3, 40, 300])
@pytest.mark.parametrize("pad_x,pad_o", [(1, 1), (8, 8), (3, 5), (0, 7)])
def test_strides_padding_and_neighbours(m, pad_x, pad_o):
    """Rows inside wider tensors whose other columns are NaN: none of it is read, none of it is written; a NaN row stays one row."""
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    k, n = 45, 37
    x, w, b = _operands(torch, m, k, n, torch.float16, 11 * m)
    wide = torch.full((m, k + pad_x + 2), float("nan"), dtype=torch.float16, device="cuda")
    xs = wide[:, 1: 1 + k]
    xs.copy_(x)
    res = torch.full((m + 1, n + pad_o + 2), float("nan"), dtype=torch.float16, device="cuda")
    rs = res[:m, 2: 2 + n]
    rs.copy_(torch.randn(m, n, device="cuda"))
    out = torch.full((m + 2, n + pad_o + 2), -7.0, dtype=torch.float16, device="cuda")
    layer = LinearLayer(w[0], b[0], activation="silu")
    layer.forward(xs, residual=rs, out=out[1: 1 + m, 1: 1 + n])
    _check(out[1: 1 + m, 1: 1 + n], x, w[0], b[0], "silu", None, rs)
    rest = out.clone()
    rest[1: 1 + m, 1: 1 + n] = -7.0
    assert (rest == -7.0).all()
    xs[m // 2] = float("nan")
    again = layer.forward(xs, residual=rs)
    lost = torch.isnan(again).any(1)
    assert int(lost.sum()) == 1 and bool(lost[m // 2]) and torch.isnan(again[m // 2]).all()
    keep = torch.arange(m, device="cuda") != m // 2
    assert torch.equal(again[keep], out[1: 1 + m, 1: 1 + n][keep])


def _group_ref(ids, e):
    to = np.where((ids >= 0) & (ids < e), ids, e)
    return np.concatenate(([0], np.cumsum(np.bincount(to, minlength=e + 1)[:e]))).astype(np.int32), np.argsort(to, kind="stable").astype(np.int32)


@pytest.mark.parametrize("n,e", [(0, 1), (0, 1024), (1, 1), (63, 2), (64, 3), (65, 7), (1000, 1), (1024, 16), (1025, 64), (5000, 1000), (8192, 1024), (8193, 5),
                                 (9000, 1024), (4096, 673), (4097, 673), (12288, 1023), (12289, 1023), (49152, 255), (49153, 255), (65536, 16), (65536, 1024), (65537, 700), (70001, 1024), (100000, 1), (3_000_000, 37)])
def test_group_rows_is_a_stable_sort(n, e):
    import torch
    from hugectr_backend_amd.dense import group_rows
    rng = np.random.default_rng(n + e)
    for kind in range(3):
        ids = rng.integers(0, e, n) if kind == 0 else rng.integers(-2, e + 2, n) if kind == 1 else np.minimum(rng.geometric(0.4, n) - 1, e)
        ids = ids.astype(np.int32)
        if kind == 1 and n > 1:
            ids[0], ids[-1] = np.iinfo(np.int32).min, np.iinfo(np.int32).max
        off, order = group_rows(torch.from_numpy(ids).cuda(), e)
        want = _group_ref(ids, e)
        assert np.array_equal(off.cpu().numpy(), want[0]) and np.array_equal(order.cpu().numpy(), want[1])


def _check_experts(got, x, w, b, act, offsets, order, residual=None, rest=0.0):
    """rows of got, in the rows of x, by each expert's run of `order`."""
    import torch
    seen = torch.zeros(got.shape[0], dtype=torch.bool)
    off = offsets.tolist()
    for e in range(len(off) - 1):
        rows = order[off[e]: off[e + 1]].long().cpu()
        seen[rows] = True
        if len(rows):
            at = rows.to(got.device)
            _check(got[at], x[at], w[e], b[e], act, None, None if residual is None else residual[at])
    assert (got.cpu()[~seen] == rest).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("m,e,k,n", [(1, 1, 16, 16), (1, 64, 33, 40), (10, 3, 64, 32), (100, 64, 100, 33), (300, 2, 64, 64), (300, 64, 479, 96), (700, 5, 40, 130),
                                     (2000, 130, 64, 48), (5000, 7, 72, 257), (3000, 1024, 16, 8)])
def test_experts_over_ragged_runs(m, e, k, n, dtype):
    """Unsorted rows through rows_in / rows_out, with ids of no expert: those rows come back as zeros, or stay as they were."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers, group_rows
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(m * e)
    x, w, b = _operands(torch, m, k, n, dt, m + e, experts=e)
    res = _operands(torch, m, n, 1, dt, 5)[0]
    layer = ExpertLayers(w, b, activation="silu", dtype=dt)
    for kind in range(3):
        ids = rng.integers(-1, e + 1, m) if kind == 0 else np.full(m, e - 1) if kind == 1 else np.minimum(rng.geometric(0.5, m) - 1, e)
        offsets, order = group_rows(torch.from_numpy(ids.astype(np.int32)).cuda(), e)
        got = layer.forward(x, offsets, rows_in=order, rows_out=order, residual=res, out_dtype=torch.float32)
        _check_experts(got, x, w, b, "silu", offsets, order, res)
        out = torch.full((m, n), 9.0, dtype=dt, device="cuda")
        layer.forward(x, offsets, rows_in=order, rows_out=order, residual=res, out=out)
        _check_experts(out, x, w, b, "silu", offsets, order, res, rest=9.0)
        xs = x[order.long()].contiguous()          # sorted rows, no index
        here = torch.arange(m, device="cuda", dtype=torch.int32)
        _check_experts(layer.forward(xs, offsets), xs, w, b, "silu", offsets, here)


def test_a_sequence_before_the_first_run_and_offsets_that_lie():
    """offsets[0] > 0, offsets beyond the rows, offsets that descend: clamped, read as their running maximum, never out of bounds."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers
    m, e, k, n = 400, 4, 24, 40
    x, w, b = _operands(torch, m, k, n, torch.float16, 1, experts=e)
    layer = ExpertLayers(w, b)
    here = torch.arange(m, device="cuda", dtype=torch.int32)
    for off in ([37, 100, 100, 333, 390], [-5, 20, 10, 399, 2 ** 31 - 1], [400, 0, 0, 0, 0], [0, 0, 0, 0, 0], [-2 ** 31, -1, -1, 5, 4], [10, 300, 40, 350, 2]):
        off_t = torch.tensor(off, dtype=torch.int32, device="cuda")
        real = torch.from_numpy(np.maximum.accumulate(np.clip(np.array(off, np.int64), 0, m)))
        _check_experts(layer.forward(x, off_t), x, w, b, "none", real, here)
        out = torch.full((m, n), 5.0, dtype=torch.float16, device="cuda")
        layer.forward(x, off_t, out=out)
        _check_experts(out, x, w, b, "none", real, here, rest=5.0)


def test_row_indexes_outside_their_tensors():
    """rows_in outside x reads zeros, rows_out outside out is not written; several positions may read one row."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers
    k, n, rows = 20, 24, 90
    x, w, b = _operands(torch, 10, k, n, torch.float16, 1, experts=2)
    layer = ExpertLayers(w, b)
    off = torch.tensor([0, 45, rows], dtype=torch.int32, device="cuda")
    rin = torch.arange(rows, device="cuda", dtype=torch.int32) % 13 - 1           # -1 .. 11: -1, 10 and 11 are outside
    rout = torch.arange(rows, device="cuda", dtype=torch.int32) - 5               # the first five are outside
    out = torch.full((80, n), 4.0, dtype=torch.float32, device="cuda")            # and the last five
    layer.forward(x, off, rows_in=rin, rows_out=rout, out=out)
    src = torch.zeros(rows, k, dtype=torch.float16, device="cuda")
    ok = (rin >= 0) & (rin < 10)
    src[ok] = x[rin[ok].long()]
    for e, (a, z) in enumerate(((0, 45), (45, rows))):
        p = torch.arange(a, z, device="cuda")
        p = p[(rout[p] >= 0) & (rout[p] < 80)]
        _check(out[rout[p].long()], src[p], w[e], b[e], "none")
    huge = torch.tensor([2 ** 31 - 1, -2 ** 31] * 45, dtype=torch.int32, device="cuda")
    zero = layer.forward(x, off, rows_in=huge)
    for e, (a, z) in enumerate(((0, 45), (45, rows))):
        assert torch.equal(zero[a:z], b[e].half().expand(z - a, n))
    layer.forward(x, off, rows_in=rin, rows_out=huge, out=out)                    # nothing at all is written


def test_a_row_that_no_run_has_is_never_read():
    import torch
    from hugectr_backend_amd.dense import ExpertLayers
    x, w, b = _operands(torch, 200, 32, 16, torch.bfloat16, 1, experts=3)
    x[150:] = float("nan")
    off = torch.tensor([0, 10, 10, 150], dtype=torch.int32, device="cuda")
    got = ExpertLayers(w, b, dtype="bf16").forward(x, off)
    assert torch.isfinite(got).all() and (got[150:] == 0).all()


def test_the_run_of_a_request():
    """A request as it is served: looked-up rows go into the narrow store, another request reads them, a layer, the grouping by domain
    and a tower per domain follow — eagerly, on another stream, and captured into a graph that is replayed with new inputs."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers, LinearLayer, group_rows
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    B, T, D, E, H, R = 500, 4, 32, 6, 72, 3000
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    store = QuantizedRows(R, D, bits=8)
    store.write(torch.randn(R, D, generator=g, device="cuda"), torch.arange(R, device="cuda"))
    _, w1, b1 = _operands(torch, 1, T * D, H, torch.float16, 3)
    _, w2, b2 = _operands(torch, 1, H, 1, torch.float16, 4, experts=E)
    layer, towers = LinearLayer(w1[0], b1[0], activation="relu"), ExpertLayers(w2, b2, activation="sigmoid")
    rows, into = torch.empty(64, D, device="cuda"), torch.empty(64, dtype=torch.int64, device="cuda")
    slots, ids = torch.empty(B * T, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")

    def serve():
        store.write(rows, into)
        x = store.read(slots, dtype=torch.float16).view(B, T * D)
        h = layer.forward(x)
        offsets, order = group_rows(ids, E)
        y = towers.forward(h, offsets, rows_in=order, rows_out=order, out_dtype=torch.float32)
        return x, h, offsets, order, y

    def request(k):
        rows.copy_(torch.randn(64, D, generator=g, device="cuda"))
        into.copy_(torch.randint(0, R, (64,), generator=g, device="cuda"))
        slots.copy_(torch.randint(0, R, (B * T,), generator=g, device="cuda"))
        ids.copy_(torch.randint(-1, E, (B,), generator=g, device="cuda"))

    def check(x, h, offsets, order, y):
        want = store.read(slots).view(B, T * D)
        assert torch.equal(x, want.half())
        _check(h, x, w1[0], b1[0], "relu")
        ref = _group_ref(ids.cpu().numpy(), E)
        assert np.array_equal(offsets.cpu().numpy(), ref[0]) and np.array_equal(order.cpu().numpy(), ref[1])
        _check_experts(y, h, w2, b2, "sigmoid", offsets, order)

    request(0)
    check(*serve())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = serve()
    torch.cuda.current_stream().wait_stream(side)
    check(*got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = serve()
    for k in range(4):
        request(k)
        graph.replay()
        check(*got)
        eager = serve()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), k


def test_two_streams_through_one_layer():
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    x, w, b = _operands(torch, 900, 256, 300, torch.float16, 1)
    layer = LinearLayer(w[0], b[0])
    want = layer.forward(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(layer.forward(x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


@pytest.mark.parametrize("rows", [7, 300, 3000])
def test_one_expert_without_offsets_takes_its_row_indexes(rows):
    import torch
    from hugectr_backend_amd.dense import ExpertLayers
    x, w, b = _operands(torch, 50, 40, 70, torch.float16, rows)
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    rin = torch.randint(0, 50, (rows,), generator=g, device="cuda", dtype=torch.int32)
    rout = torch.randperm(rows, generator=g, device="cuda").int()
    layer = ExpertLayers(w, b, activation="relu")
    _check(layer.forward(x, None, rows_in=rin), x[rin.long()], w[0], b[0], "relu")
    got = layer.forward(x, None, rows_in=rin, rows_out=rout)
    _check(got[rout.long()], x[rin.long()], w[0], b[0], "relu")
    _check(layer.forward(x, None), x, w[0], b[0], "relu")


def test_an_error_that_an_earlier_call_left_is_not_this_calls():
    """A layer that does not fit the card is an error of its own call alone."""
    import ctypes as C
    import torch
    from hugectr_backend_amd import hps
    from hugectr_backend_amd.dense import LinearLayer, group_rows
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    x, w, b = _operands(torch, 9, 64, 40, torch.float16, 1)
    layer, store = LinearLayer(w[0], b[0]), QuantizedRows(10, 4)
    slots = torch.arange(3, device="cuda")
    for call in (lambda: layer.forward(x), lambda: group_rows(slots.int(), 4), lambda: store.write(torch.ones(3, 4, device="cuda"), slots),
                 lambda: store.read(slots)):
        h = C.c_void_p()
        rc = hps.LIB.hps_linear_create(0, 256, 1 << 20, 512, 1, 0, 0x10000, 0, None, 0, None, C.byref(h))      # 549 GB of weights: nothing is read
        assert rc == hps.ERR_INTERNAL and "hipMalloc" in hps.LIB.hps_last_error().decode() and not h.value
        call()
    _check(layer.forward(x), x, w[0], b[0], "none")


@pytest.mark.parametrize("act", ["relu", "silu"])
@pytest.mark.parametrize("m,k,n,e", [(5, 70, 40, 3), (120, 64, 64, 4), (700, 96, 128, 3), (6000, 64, 520, 5), (9000, 40, 1030, 2)])
def test_towers_in_place_over_mul_and_residual(m, k, n, e, act):
    """The output is its own mul, its own residual, or both; rows in order and by index; every tile size."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers, group_rows
    x, w, b = _operands(torch, m, k, n, torch.float16, m, experts=e)
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    ids = torch.randint(-1, e, (m,), generator=g, device="cuda").int()
    offsets, order = group_rows(ids, e)
    layer = ExpertLayers(w, b, activation=act)
    off = offsets.tolist()
    for index in (order, None):
        for which in ("mul", "residual", "both"):
            was = torch.randn(m, n, generator=g, device="cuda").half()
            out = was.clone()
            layer.forward(x, offsets, rows_in=index, rows_out=index, mul=out if which != "residual" else None,
                          residual=out if which != "mul" else None, out=out)
            for q in range(e):
                rows = (order if index is not None else torch.arange(m, device="cuda"))[off[q]: off[q + 1]].long()
                if len(rows):
                    _check(out[rows], x[rows], w[q], b[q], act, was[rows] if which != "residual" else None, was[rows] if which != "mul" else None)
            rest = (order if index is not None else torch.arange(m, device="cuda"))[off[e]:].long()
            assert torch.equal(out[rest], was[rest])
