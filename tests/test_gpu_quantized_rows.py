"""Rows held in 8 or 4 bits (csrc/cache/qrows_kernels.hip) against the definition in 64 bits.

Codes and scales are compared for equality: scale = fp32(max|x| / L) is one correctly rounded division, and the code is the nearest
integer (ties to even) of the real quotient x / scale, which a 64-bit division of two 32-bit numbers decides without error (a quotient
of 24-bit significands that is not a half-integer is at least 2^-33 away from one, 2^-40 relative).  Values read back are code * scale,
one 32-bit product, rounded to the output's type: equal as well.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TINY = 2.0 ** -100


def _quantize(x, bits, group):
    """(codes int [n, dim], scales fp32 [n, groups]) of fp32 rows, by the definition."""
    n, dim = x.shape
    L = 127 if bits == 8 else 7
    step = dim if group == 0 or group >= dim else group
    codes, scales = np.zeros((n, dim), np.int64), []
    for a in range(0, dim, step):
        v = x[:, a: a + step].astype(np.float64)
        top = np.abs(v).max(1)
        with np.errstate(all="ignore"):
            s = (top / L).astype(np.float32)
            s[top < TINY] = 0
            s[~np.isfinite(top)] = np.nan
            q = np.clip(np.rint(v / s.astype(np.float64)[:, None]), -L, L)
        q[~(s > 0)] = 0
        codes[:, a: a + step] = q
        scales.append(s)
    return codes, np.stack(scales, 1)


def _values(codes, scales, group):
    dim = codes.shape[1]
    step = dim if group == 0 or group >= dim else group
    return codes.astype(np.float32) * np.repeat(scales, step, 1)[:, :dim]


def _unpacked(store):
    raw = store.codes.cpu().numpy()
    if store.bits == 8:
        return raw[:, : store.dim].astype(np.int64), raw[:, store.dim:]
    q = np.stack((raw & 15, raw >> 4), 2).reshape(raw.shape[0], -1).astype(np.int64)
    q = np.where(q > 7, q - 16, q)
    return q[:, : store.dim], q[:, store.dim:]


def _same(a, b):
    return np.array_equal(np.asarray(a), np.asarray(b), equal_nan=True)


def _rows(rng, n, dim):
    return (rng.standard_normal((n, dim)) * rng.uniform(0.01, 3, (n, 1))).astype(np.float32)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,dim,group", [
    (1, 1, 0), (3, 3, 0), (5, 8, 16), (65, 16, 0), (64, 17, 16), (33, 48, 32), (257, 100, 0), (100, 100, 32), (129, 128, 0), (70, 128, 64),
    (40, 200, 128), (21, 256, 256), (9, 500, 16), (12, 513, 256), (7, 1024, 0), (5, 2050, 64), (3, 4096, 0), (2, 5001, 0), (2, 16384, 256),
])
def test_write_and_read_are_exact(n, dim, group, dtype, bits):
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    rng = np.random.default_rng(n * 1000 + dim)
    dt = getattr(torch, dtype)
    R = 2 * n + 3
    rows = torch.from_numpy(_rows(rng, n, dim)).to(dt).cuda()
    x = rows.float().cpu().numpy()
    slots = rng.permutation(R)[:n].astype(np.int64)
    store = QuantizedRows(R, dim, bits=bits, group=group)
    held = store.write(rows, torch.from_numpy(slots).cuda(), held=torch.full_like(rows, 7))
    codes, scales = _quantize(x, bits, group)
    want_c, want_s = np.zeros((R, dim), np.int64), np.zeros((R, scales.shape[1]), np.float32)
    want_c[slots], want_s[slots] = codes, scales
    got_c, pad = _unpacked(store)
    assert _same(got_c, want_c) and not pad.any()
    assert _same(store.scales.cpu().numpy(), want_s)
    assert not store._workspace[: store.num_rows].any()          # the claims are clear again
    values = torch.from_numpy(_values(codes, scales, group))
    assert torch.equal(held.cpu(), values.to(dt))
    for out_t in (torch.float32, torch.float16, torch.bfloat16):
        got = store.read(torch.from_numpy(slots).cuda(), dtype=out_t).cpu()
        assert torch.equal(got, values.to(out_t)), out_t


@pytest.mark.parametrize("bits", [8, 4])
def test_ties_borders_and_special_values(bits):
    """Exact half-integers go to the even code, their neighbours to the nearer one; tiny groups are zeros, a NaN or an infinity makes
    its group (and no other) read as NaN; the largest finite values hold."""
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    L = 127 if bits == 8 else 7
    half = (np.arange(-2 * L, 2 * L + 1) / 2).astype(np.float32)
    rows = []
    for scale in (np.float32(0.125), np.float32(1), np.float32(3), np.float32(1e-3), np.float32(2.0 ** 100), np.float32(2.0 ** -90)):
        for shift in (0, 1, -1):
            v = half * scale
            v = np.nextafter(v, np.float32(np.inf if shift > 0 else -np.inf)).astype(np.float32) if shift else v
            v = np.resize(v, 512)
            v[0] = np.float32(L) * scale        # fixes the scale (its quotient by L rounds back to `scale` or next to it)
            rows.append(v)
    x = np.stack(rows)
    odd = np.zeros((10, 512), np.float32)
    odd[1] = 2.0 ** -101
    odd[2, 5] = 2.0 ** -100
    odd[3, 5] = 1e-45
    odd[4] = np.float32(3.4028235e38)
    odd[5, 17] = np.nan
    odd[6, 511] = np.inf
    odd[7, 0] = -np.inf
    odd[8, :16] = 1
    odd[8, 16:32] = np.nan
    odd[9] = -0.0
    x = np.concatenate((x, odd))
    for group in (0, 16, 256):
        store = QuantizedRows(len(x), 512, bits=bits, group=group)
        at = torch.arange(len(x), device="cuda")
        held = store.write(torch.from_numpy(x).cuda(), at, held=torch.empty(len(x), 512, device="cuda"))
        codes, scales = _quantize(x, bits, group)
        assert _same(_unpacked(store)[0], codes)
        assert _same(store.scales.cpu().numpy(), scales)
        want = _values(codes, scales, group)
        assert _same(store.read(at).cpu().numpy(), want) and _same(held.cpu().numpy(), want)
    assert np.isnan(want[len(x) - 5]).sum() == 256          # group 256: the NaN's own group alone


@pytest.mark.parametrize("n,dim,R", [(50, 16, 7), (300, 1, 2), (1000, 1, 400), (2000, 128, 300), (20000, 16, 9000), (26624, 16, 1000000), (40000, 1, 30000), (5000, 4, 700), (20000, 128, 3000), (270000, 8, 40000), (300000, 16, 5000000),
                                     (600000, 3, 10000000), (262144, 5, 3), (270000, 1100, 1000)])
def test_a_slot_named_again_keeps_its_last_row(n, dim, R):
    """Few rows, some, many; a few of the slots named twice (the last pass has a list of them), most of them (too many for the list)."""
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    rng = np.random.default_rng(n)
    x = _rows(rng, n, dim)
    slots = rng.integers(-3, R + 3, n).astype(np.int64)     # some outside the store: skipped
    slots[0], slots[1] = np.iinfo(np.int64).min, np.iinfo(np.int64).max
    store = QuantizedRows(R, dim)
    store.write(torch.from_numpy(_rows(rng, R, dim)).cuda(), torch.arange(R, device="cuda"))
    codes0, scales0 = _unpacked(store)[0], store.scales.cpu().numpy()
    codes, scales = _quantize(x, 8, 0)
    last = {s: i for i, s in enumerate(slots.tolist()) if 0 <= s < R}
    at, of = np.array(list(last)), np.array(list(last.values()))
    codes0[at], scales0[at] = codes[of], scales[of]
    held = store.write(torch.from_numpy(x).cuda(), torch.from_numpy(slots).cuda(), held=torch.empty(n, dim, device="cuda"))
    assert _same(_unpacked(store)[0], codes0) and _same(store.scales.cpu().numpy(), scales0)
    assert _same(held.cpu().numpy(), _values(codes, scales, 0))     # every row's, kept or not
    assert not store._workspace[: store.num_rows].any()          # the claims are clear again
    rows = torch.from_numpy(x).cuda()          # once more, in place and over what is there
    assert store.write(rows, torch.from_numpy(slots).cuda(), held=rows) is rows
    assert _same(rows.cpu().numpy(), _values(codes, scales, 0))
    assert _same(_unpacked(store)[0], codes0) and _same(store.scales.cpu().numpy(), scales0)
    got = store.read(torch.from_numpy(slots).cuda(), default_value=-2.5).cpu().numpy()
    inside = (slots >= 0) & (slots < R)
    assert _same(got[inside], _values(codes0, scales0, 0)[slots[inside]]) and (got[~inside] == -2.5).all()


@pytest.mark.parametrize("dtype,bits,group", [("float16", 8, 0), ("bfloat16", 4, 32), ("float32", 4, 16)])
@pytest.mark.parametrize("n,dim", [(900, 600), (1500, 2100), (3000, 600), (2600, 2100), (262145, 40)])
def test_a_slot_named_again_in_every_type(n, dim, dtype, bits, group):
    """Rows in registers and rows that are read twice, scales per group, in the three ways."""
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    rng = np.random.default_rng(n + dim)
    R = n // 3
    rows = torch.from_numpy(_rows(rng, n, dim)).to(getattr(torch, dtype)).cuda()
    x = rows.float().cpu().numpy()
    slots = rng.integers(-2, R + 2, n).astype(np.int64)
    store = QuantizedRows(R, dim, bits=bits, group=group)
    codes, scales = _quantize(x, bits, group)
    want_c, want_s = np.zeros((R, dim), np.int64), np.zeros((R, scales.shape[1]), np.float32)
    last = {s: i for i, s in enumerate(slots.tolist()) if 0 <= s < R}
    at, of = np.array(list(last)), np.array(list(last.values()))
    want_c[at], want_s[at] = codes[of], scales[of]
    values = torch.from_numpy(_values(codes, scales, group)).to(rows.dtype)
    for _ in range(2):                                   # the second time over what is there
        held = store.write(rows, torch.from_numpy(slots).cuda(), held=torch.empty_like(rows))
        assert torch.equal(held.cpu(), values)
        assert _same(_unpacked(store)[0], want_c) and _same(store.scales.cpu().numpy(), want_s)
    assert not store._workspace[: store.num_rows].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_strided_misaligned_and_in_place_rows(dtype):
    """Rows inside a wider tensor, starting anywhere; what lies between them stays as it was; held may be the rows themselves."""
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    dt = getattr(torch, dtype)
    rng = np.random.default_rng(5)
    n, dim = 37, 64
    for start, width in ((0, 80), (1, 80), (3, 67), (8, 72)):
        wide = torch.from_numpy(_rows(rng, n, width)).to(dt).cuda()
        rows = wide[:, start: start + dim] if start + dim <= width else wide[:, :dim]
        x = rows.float().cpu().numpy()
        before = wide.clone()
        store = QuantizedRows(n, dim, bits=4, group=32)
        at = torch.arange(n - 1, -1, -1, device="cuda")
        held = store.write(rows, at, held=rows)
        codes, scales = _quantize(x, 4, 32)
        want = torch.from_numpy(_values(codes, scales, 32)).to(dt).cuda()
        assert torch.equal(held, want) and _same(_unpacked(store)[0][::-1], codes)
        off = rows.storage_offset() % width
        before[:, off: off + dim] = want
        assert torch.equal(wide, before)
        out = torch.full((n, width), 3.0, dtype=dt, device="cuda")
        view = out[:, off: off + dim]
        store.read(at, out=view)
        keep = torch.full_like(out, 3.0)
        keep[:, off: off + dim] = want
        assert torch.equal(out, keep)


def test_nothing_to_do_and_an_empty_store():
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    store = QuantizedRows(4, 8)
    store.write(torch.empty(0, 8, device="cuda"), none)
    assert store.read(none).shape == (0, 8)
    empty = QuantizedRows(0, 8)
    slots = torch.tensor([0, -1, 5], device="cuda")
    held = empty.write(torch.ones(3, 8, device="cuda"), slots, held=torch.zeros(3, 8, device="cuda"))
    assert torch.equal(held, torch.ones_like(held)) or (held - 1).abs().max() <= 2.0 ** -23
    assert (empty.read(slots, default_value=1.5) == 1.5).all()
    for n in (3000, 300000):      # the ways of larger calls
        held = empty.write(torch.ones(n, 8, device="cuda"), torch.zeros(n, dtype=torch.int64, device="cuda"), held=torch.zeros(n, 8, device="cuda"))
        assert (held - 1).abs().max() <= 2.0 ** -23


def test_codes_beyond_4_gib():
    """The last rows of a store whose codes end beyond 2^32 bytes: places are computed in 64 bits."""
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    R, dim = 4_400_000, 1024
    store = QuantizedRows(R, dim)
    rng = np.random.default_rng(1)
    x = _rows(rng, 300, dim)
    slots = np.concatenate((np.arange(150), R - 1 - np.arange(150))).astype(np.int64)
    store.write(torch.from_numpy(x).cuda(), torch.from_numpy(slots).cuda())
    codes, scales = _quantize(x, 8, 0)
    assert _same(store.codes[torch.from_numpy(slots).cuda()].cpu().numpy(), codes)
    assert _same(store.read(torch.from_numpy(slots).cuda()).cpu().numpy(), _values(codes, scales, 0))
    assert int(torch.count_nonzero(store.scales)) == 300
    del store
    torch.cuda.empty_cache()


def test_streams_and_a_replayed_graph():
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    rng = np.random.default_rng(3)
    n, dim, R = 3000, 48, 4000
    rows, slots = torch.empty(n, dim, device="cuda"), torch.empty(n, dtype=torch.int64, device="cuda")
    store = QuantizedRows(R, dim, bits=4, group=16)
    plain = QuantizedRows(R, dim, bits=4, group=16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):      # warm, on a stream that is not the store's own
        store.write(rows.zero_(), slots.fill_(-1))
        store.read(slots)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        store.write(rows, slots)
        out = store.read(slots)
    for k in range(4):
        x = torch.from_numpy(_rows(rng, n, dim)).cuda()
        s = torch.from_numpy(rng.integers(-2, R, n).astype(np.int64)).cuda()
        rows.copy_(x)
        slots.copy_(s)
        g.replay()
        plain.write(x, s)              # eager work of the same kind between the replays
        want = plain.read(s)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(store.codes, plain.codes) and torch.equal(store.scales, plain.scales), k


@pytest.mark.parametrize("in_place", [False, True])
def test_more_rows_than_one_launch_holds(in_place):
    """2^24 rows are one launch; the rows at both sides of the border, and slots named at both sides of it."""
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    n, R = (1 << 24) + 1000, (1 << 24) - 500
    store = QuantizedRows(R, 1)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn(n, 1, generator=g, device="cuda").abs() + 0.5          # one value a row: code 127, scale x / 127
    slots = torch.arange(n, device="cuda") % R                             # the first 1,500 slots are named twice
    scale = (x.double() / 127).float()                                     # (torch divides fp32 by a number as a product with 1 / 127)
    want = scale[:R].clone()
    want[:1500] = scale[R:]
    rows = x.clone()
    held = store.write(rows, slots, held=rows if in_place else torch.empty_like(x))
    assert torch.equal(held, 127.0 * scale)
    assert torch.equal(store.scales, want) and (store.codes[:, 0] == 127).all()
    assert torch.equal(store.read(slots), 127.0 * want[slots])
