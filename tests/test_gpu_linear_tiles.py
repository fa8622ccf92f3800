"""Every kernel of the dense layers (csrc/dense/linear_kernels.hip) by itself: 16 and 32 rows x 32 columns, tiles of 64 x 64, 128 x 128 and 128 x 256, each
with rows on and off 16 bytes, K below and far beyond the buffers of a tile and of any residue, N off 8, every activation, mul and residual,
both types and both output types.  Which kernel a case runs is asked of the library, so that another rule cannot move the cases unseen.

Every output value is held against y = act(x W + b) * mul + residual in 64 bits over the same operands, within the bound of
tests/test_gpu_linear.py (its head derives it): (K + 2) 2^-24 of sum |x||w| + |b| passed on at most 1.13-fold by the activation; 2^-20 of
max(1, |sum|) for gelu, silu and sigmoid; 2^-24 of each result behind it; half a step of the output's type.
"""
import ctypes as C
import math

import pytest

pytestmark = pytest.mark.gpu

HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
# tile -> rows, columns; with experts: rows, experts, columns
TILES = {(16, 32): (100, 295), (32, 32): (400, 1003), (64, 64): (2000, 301), (128, 128): (7000, 300), (128, 256): (11000, 299)}
RUNS = {(16, 32): (150, 3, 100), (32, 32): (400, 3, 1003), (64, 64): (2000, 5, 301), (128, 128): (7000, 5, 300), (128, 256): (11000, 5, 299)}
EXACT = {(16, 32): (64, 256), (32, 32): (384, 1024), (64, 64): (2048, 320), (128, 128): (7168, 384), (128, 256): (10496, 512)}   # N on 32


def _act64(torch, y, act):
    return {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "gelu": lambda v: v * torch.special.ndtr(v),
            "silu": lambda v: v * torch.sigmoid(v), "sigmoid": torch.sigmoid}[act](y)


def _check(torch, got, x, w, b, act, mul=None, residual=None):
    """got [m, n] against x [m, k] double, w [k, n], b [n] or None: every value, on the device"""
    K = x.shape[1]
    x, w = x.double(), w.double()
    b = torch.zeros(w.shape[1], dtype=torch.float64, device="cuda") if b is None else b.double()
    s = x @ w + b
    off = 1.13 * (K + 2) * 2.0 ** -24 * (x.abs() @ w.abs() + b.abs())
    y = _act64(torch, s, act)
    if act not in ("none", "relu"):
        off = off + 2.0 ** -20 * s.abs().clamp(min=1)
    if mul is not None:
        y, off = y * mul.double(), off * mul.double().abs()
        off = off + 2.0 ** -24 * y.abs()
    if residual is not None:
        y = y + residual.double()
        off = off + 2.0 ** -24 * y.abs()
    half = HALF[str(got.dtype).split(".")[1]]
    off = off * (1 + half) + half * y.abs() + 2.0 ** -25
    bad = ~((got.double() - y).abs() <= off)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist())


def _tile(layer, rows, offsets=False):
    from hugectr_backend_amd import hps
    a, b = C.c_uint32(), C.c_uint32()
    hps._check(hps.LIB.hps_linear_tile(layer._h, rows, int(offsets), C.byref(a), C.byref(b)))
    return a.value, b.value


def _inside(torch, t, before, behind, fill=float("nan")):
    """t's values inside wider rows that are `fill` elsewhere: a view that starts `before` values into the row"""
    wide = torch.full((t.shape[0], t.shape[1] + before + behind), fill, dtype=t.dtype, device="cuda")
    view = wide[:, before: before + t.shape[1]]
    view.copy_(t)
    return wide, view


def _gen(torch, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# K, values before and behind x in its row: rows on 16 bytes (multiples of 8, or padded to them), and off
KS = [(64, 0, 0), (392, 0, 0), (520, 0, 8), (479, 0, 1), (45, 0, 3),
      (479, 0, 0), (393, 1, 1), (416, 1, 0), (1025, 0, 0), (385, 0, 2), (32, 1, 2), (64, 3, 6), (7, 0, 0), (33, 2, 0), (96, 0, 2), (128, 1, 1)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("k,before,behind", KS)
@pytest.mark.parametrize("tile", list(TILES))
def test_every_tile_with_rows_on_and_off_16_bytes(tile, k, before, behind, dtype):
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    dt = getattr(torch, dtype)
    m, n = TILES[tile]
    g = _gen(torch, k + n)
    _, x = _inside(torch, torch.randn(m, k, generator=g, device="cuda").to(dt), before, behind)
    w = (torch.randn(k, n, generator=g, device="cuda") / math.sqrt(k)).to(dt)
    b = 0.3 * torch.randn(n, generator=g, device="cuda")
    mul = _inside(torch, torch.randn(m, n, generator=g, device="cuda").to(dt), 1, 4)[1]
    res = _inside(torch, torch.randn(m, n, generator=g, device="cuda").to(dt), 0, 3)[1]
    layer = LinearLayer(w, b, activation="relu", dtype=dt)
    assert _tile(layer, m) == tile
    for out_t in (dt, torch.float32):
        for mm, rr in ((None, None), (mul, res), (mul, None), (None, res)):
            wide, out = _inside(torch, torch.zeros(m, n, dtype=out_t, device="cuda"), 1, 2, 77.0)
            layer.forward(x, mul=mm, residual=rr, out=out)
            _check(torch, out, x, w, b, "relu", mm, rr)
            assert (wide[:, 0] == 77).all() and (wide[:, 1 + n:] == 77).all()
            assert torch.equal(layer.forward(x, mul=mm, residual=rr, out_dtype=out_t), out)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("tile", list(TILES))
def test_every_activation_in_every_tile(tile, act, dtype):
    """N on 32 (none and relu leave straight from the accumulators) and off it (through LDS), with rows on and off 16 bytes."""
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    dt = getattr(torch, dtype)
    for (m, n), k in ((TILES[tile], 201), (EXACT[tile], 200), (EXACT[tile], 77)):
        g = _gen(torch, k + n)
        x = (3 * torch.randn(m, k, generator=g, device="cuda")).to(dt)
        w = (torch.randn(k, n, generator=g, device="cuda") / math.sqrt(k)).to(dt)
        b = 0.3 * torch.randn(n, generator=g, device="cuda")
        mul, res = (torch.randn(m, n, generator=g, device="cuda").to(dt) for _ in range(2))
        layer = LinearLayer(w, b, activation=act, dtype=dt)
        assert _tile(layer, m) == tile
        for out_t in (dt, torch.float32):
            for mm, rr in ((None, None), (mul, res), (None, res)):
                _check(torch, layer.forward(x, mul=mm, residual=rr, out_dtype=out_t), x, w, b, act, mm, rr)
        over = res.clone()
        assert torch.equal(layer.forward(x, mul=mul, residual=over, out=over), layer.forward(x, mul=mul, residual=res))
        over = mul.clone()
        assert torch.equal(layer.forward(x, mul=over, residual=over, out=over), layer.forward(x, mul=mul, residual=mul))
        _check(torch, LinearLayer(w, activation=act, dtype=dt).forward(x), x, w, None, act)


def _runs(torch, offsets, m):
    """(first, end) of every run: clamped, read as the running maximum"""
    ends, at = [], 0
    for v in offsets:
        at = max(at, min(max(v, 0), m))
        ends.append(at)
    return list(zip(ends[:-1], ends[1:]))


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("k,before,behind", [(72, 0, 0), (45, 0, 0), (425, 0, 0), (424, 3, 2)])
@pytest.mark.parametrize("tile", list(RUNS))
def test_runs_and_row_indexes_in_every_tile(tile, k, before, behind, dtype):
    """Offsets in order and offsets that lie, with rows in order, by a permutation, and by indexes that leave their tensors; mul and residual by the
    output's row; rows that nobody names stay as they were."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers
    dt = getattr(torch, dtype)
    m, e, n = RUNS[tile]
    g = _gen(torch, m + k)
    x_rows = m + 9
    _, x = _inside(torch, torch.randn(x_rows, k, generator=g, device="cuda").to(dt), before, behind)
    w = (torch.randn(e, k, n, generator=g, device="cuda") / math.sqrt(k)).to(dt)
    b = 0.3 * torch.randn(e, n, generator=g, device="cuda")
    out_rows = m + 5
    mul, res = (_inside(torch, torch.randn(out_rows, n, generator=g, device="cuda").to(dt), 1, 2)[1] for _ in range(2))
    perm = torch.randperm(m, generator=g, device="cuda").int()
    wild_in = torch.randint(-50, x_rows + 50, (m,), generator=g, device="cuda").int()
    wild_in[3], wild_in[m // 2] = 2 ** 31 - 1, -2 ** 31
    wild_out = (torch.randperm(out_rows + 60, generator=g, device="cuda")[:m] - 30).int()
    wild_out[wild_out < -28] = -2 ** 31
    honest = [0, m // 7, m // 7, m - m // 3] + [m - 3] * (e - 3)
    lying = [[m // 10, m // 2, m // 3, m + 7] + [2 ** 31 - 1] * (e - 3), [-5, m // 3, -2 ** 31, m // 2] + [m // 2 + 1] * (e - 3)]
    bits = [(honest, perm, perm), (honest, None, None), (lying[0], None, perm), (lying[1], wild_in, wild_out), (lying[0], wild_in, None)]
    for act, (off, rin, rout), ends in (("relu", bits[0], False), ("none", bits[1], True), ("silu", bits[2], True), ("gelu", bits[3], True),
                                        ("relu", bits[3], True), ("relu", bits[3], False), ("sigmoid", bits[4], False), ("none", bits[4], True)):
        layer = ExpertLayers(w, b, activation=act, dtype=dt)
        assert _tile(layer, m, True) == tile
        offsets = torch.tensor(off, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).int().cuda()
        src = torch.zeros(m, k, dtype=torch.float64, device="cuda")
        at = torch.arange(m, device="cuda") if rin is None else rin.long()
        there = (at >= 0) & (at < x_rows)
        src[there] = x[at[there]].double()
        to = torch.arange(m, device="cuda") if rout is None else rout.long()
        for out_t in (dt, torch.float32):
            out = torch.full((out_rows, n), 5.0, dtype=out_t, device="cuda")
            layer.forward(x if rin is not None else x[:m], offsets, rows_in=rin, rows_out=rout, mul=mul if ends else None, residual=res if ends else None, out=out)
            written = torch.zeros(out_rows, dtype=torch.bool, device="cuda")
            for q, (lo, hi) in enumerate(_runs(torch, off, m)):
                p = torch.arange(lo, hi, device="cuda")
                p = p[(to[p] >= 0) & (to[p] < out_rows)]
                if len(p):
                    r = to[p]
                    written[r] = True
                    _check(torch, out[r], src[p], w[q], b[q], act, mul[r] if ends else None, res[r] if ends else None)
            assert (out[~written] == 5).all()


@pytest.mark.parametrize("tile", list(TILES))
def test_a_row_that_is_not_finite_stays_one_row_in_every_tile(tile):
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    m, n = TILES[tile]
    for k in (96, 211):
        g = _gen(torch, k)
        x = torch.randn(m, k, generator=g, device="cuda").half()
        layer = LinearLayer(torch.randn(k, n, generator=g, device="cuda") / math.sqrt(k), activation="relu")
        want = layer.forward(x)
        bad = x.clone()
        rows = [0, m // 3, m - 1]
        for r, v, col in zip(rows, (float("nan"), float("inf"), float("-inf")), (k - 1, 0, k // 2)):
            bad[r, col] = v
        got = layer.forward(bad)
        keep = torch.ones(m, dtype=torch.bool, device="cuda")
        keep[rows] = False
        assert torch.equal(got[keep], want[keep])
        assert torch.isnan(got[rows[0]]).all() and not torch.isfinite(got[rows[1]]).all() and not torch.isfinite(got[rows[2]]).all()


def test_the_tile_of_a_call():
    import torch
    from hugectr_backend_amd import hps
    from hugectr_backend_amd.dense import LinearLayer
    layer = LinearLayer(torch.ones(8, 300))
    a = C.c_uint32()
    for args in ((None, 5, 0, C.byref(a), C.byref(a)), (layer._h, 0, 0, C.byref(a), C.byref(a)), (layer._h, 2 ** 31, 0, C.byref(a), C.byref(a)),
                 (layer._h, 5, 0, None, C.byref(a)), (layer._h, 5, 0, C.byref(a), None)):
        assert hps.LIB.hps_linear_tile(*args) == hps.ERR_INVALID_ARG
    assert _tile(layer, 1) == (16, 32) and _tile(layer, 2 ** 31 - 1) == (128, 256)


@pytest.mark.parametrize("m,n,k,before", [(30000, 299, 45, 1), (30000, 512, 72, 0), (140000, 61, 33, 0), (66000, 128, 100, 1)])
def test_streamed_outputs_anywhere(m, n, k, before):
    """Outputs of more than 32 MB leave past the caches: every row of them, at odd strides too, with what lies between the rows as it was."""
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    g = _gen(torch, m + k)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(k, n, generator=g, device="cuda") / math.sqrt(k)).bfloat16()
    res = torch.randn(m, n, generator=g, device="cuda").bfloat16()
    for act in ("relu", "silu"):
        layer = LinearLayer(w, activation=act, dtype="bf16")
        wide, out = _inside(torch, torch.zeros(m, n, device="cuda"), before, before + 2, 3.0)
        layer.forward(x, residual=res, out=out)
        _check(torch, out, x, w, None, act, None, res)
        assert (wide[:, :before] == 3).all() and (wide[:, before + n:] == 3).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("tile", list(TILES))
def test_gelu_holds_its_relative_precision_far_out(tile, dtype):
    """gelu(y) = y erfc(-y / sqrt 2) / 2 where it is next to nothing.  The sums are the inputs themselves (K = 1, W = 1), so what is left is the
    activation: the fit 1.1e-7 and a dozen fp32 operations (2^-20 together), the exponential's argument y^2 / 2 + 2, rounded a few times
    (2^-22 of it), and the output's half step."""
    import torch
    from hugectr_backend_amd.dense import LinearLayer
    dt = getattr(torch, dtype)
    m, n = TILES[tile]
    y = torch.linspace(-12, 12, m, device="cuda").to(dt)
    layer = LinearLayer(torch.ones(1, n), activation="gelu", dtype=dt)
    assert _tile(layer, m) == tile
    v = y.double()
    want = v * torch.special.erfc(-v / math.sqrt(2)) / 2
    for out_t in (dt, torch.float32):
        got = layer.forward(y[:, None], out_dtype=out_t).double()
        half = HALF[str(out_t).split(".")[1]]
        off = want.abs() * (2.0 ** -20 + (v * v / 2 + 2) * 2.0 ** -22 + half) + (2.0 ** -25 if out_t == torch.float16 else 2.0 ** -126)
        bad = ~((got - want[:, None]).abs() <= off[:, None])
        assert not bad.any(), (int(bad.sum()), v[bad.any(1)][:5].tolist())
