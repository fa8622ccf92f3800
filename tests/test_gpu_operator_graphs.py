"""Every way of a write and of the grouping inside a captured graph that is replayed with other inputs, one store written by all ways in turn, and
calls from several threads at once."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# rows of a call: one launch, claims, stamps (with few and with many slots named again)
WAYS = [(500, 300), (30000, 20000), (270000, 2000000), (270000, 60000)]


def _inputs(torch, g, n, R, dim):
    return torch.randn(n, dim, generator=g, device="cuda"), torch.randint(-2, R + 2, (n,), generator=g, device="cuda")


def _expected(torch, store, rows, slots):
    """codes and scales after the write: of a slot named again the last row (scale = fp32(max / 127), code = the quotient to the nearest, ties to even)"""
    R = store.num_rows
    ok = (slots >= 0) & (slots < R)
    last = torch.full((R,), -1, dtype=torch.int64, device="cuda")
    last.scatter_reduce_(0, slots[ok], torch.arange(len(slots), device="cuda")[ok], "amax")
    named = last >= 0
    codes, scales = store.codes.clone(), store.scales.clone()
    x = rows[last[named]].double()
    scale = (x.abs().amax(1) / 127.0).float()
    codes[named, : store.dim] = (x / scale.double()[:, None]).round().to(torch.int8)
    scales[named, 0] = scale
    return codes, scales


@pytest.mark.parametrize("n,R", WAYS)
def test_every_way_of_a_write_in_a_replayed_graph(n, R):
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    dim = 12
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    store = QuantizedRows(R, dim)
    rows, slots = _inputs(torch, g, n, R, dim)
    store.write(rows, slots)
    store.read(slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = store.write(rows, slots, held=torch.empty_like(rows))
        back = store.read(slots)
    for k in range(4):
        x, s = _inputs(torch, g, n, R, dim)
        rows.copy_(x)
        slots.copy_(s)
        want = _expected(torch, store, x, s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(store.codes, want[0]) and torch.equal(store.scales, want[1]), k
        ok = (s >= 0) & (s < R)
        assert torch.equal(back[ok], (store.codes[s[ok], :dim].float() * store.scales[s[ok]])) and (back[~ok] == 0).all()
        q = (x.double() / (x.double().abs().amax(1) / 127.0).float().double()[:, None]).round()
        assert torch.equal(held, (q * (x.double().abs().amax(1) / 127.0).float().double()[:, None]).float())
        x, s = _inputs(torch, g, 1000 * (k + 1), R, dim)       # eager work on the same store between the replays, by other ways
        want = _expected(torch, store, x, s)
        store.write(x, s)
        assert torch.equal(store.codes, want[0]) and torch.equal(store.scales, want[1]), k


def test_one_store_by_all_ways_in_turn():
    import torch
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    R, dim = 50000, 7
    store = QuantizedRows(R, dim)
    for k, n in enumerate((1, 2048, 2049, 262143, 262144, 300000, 5, 262144, 4000, 2048, 400000, 3000)):
        x, s = _inputs(torch, g, n, R, dim)
        if k % 3 == 2:
            s[: n // 2] = s[n // 2: 2 * (n // 2)]              # half of the rows name the others' slots
        want = _expected(torch, store, x, s)
        held = x.clone() if k % 2 else None
        store.write(held if k % 2 else x, s, held=held)        # (in place every other time)
        assert torch.equal(store.codes, want[0]) and torch.equal(store.scales, want[1]), (k, n)
        assert not store._workspace[:R].any()                   # no claim is left


@pytest.mark.parametrize("n,e", [(300, 64), (4096, 1024), (20000, 16), (65536, 1024), (200000, 37)])
def test_every_way_of_the_grouping_in_a_replayed_graph(n, e):
    import torch
    from hugectr_backend_amd.dense import group_rows
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    ids = torch.zeros(n, dtype=torch.int32, device="cuda")
    group_rows(ids, e)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = group_rows(ids, e)
        second = group_rows(ids, e)
    for _ in range(4):
        ids.copy_(torch.randint(-1, e + 1, (n,), generator=g, device="cuda"))
        graph.replay()
        eager = group_rows(ids, e)
        torch.cuda.synchronize()
        to = torch.where((ids >= 0) & (ids < e), ids, torch.full_like(ids, e)).long().cpu().numpy()
        order = np.argsort(to, kind="stable")
        offsets = np.concatenate(([0], np.cumsum(np.bincount(to, minlength=e + 1)[:e])))
        for got in (first, second, eager):
            assert np.array_equal(got[0].cpu().numpy(), offsets) and np.array_equal(got[1].cpu().numpy(), order)


def test_threads_call_at_once():
    """Four threads, a stream each, through one layer, one store (read) and the grouping: every result is what one thread gets."""
    import torch
    from hugectr_backend_amd.dense import ExpertLayers, group_rows
    from hugectr_backend_amd.quantized_rows import QuantizedRows
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    store = QuantizedRows(5000, 32)
    store.write(torch.randn(5000, 32, generator=g, device="cuda"), torch.arange(5000, device="cuda"))
    layer = ExpertLayers(torch.randn(5, 32, 72, generator=g, device="cuda") / 6, activation="silu")
    work = [(torch.randint(0, 5000, (m,), generator=g, device="cuda"), torch.randint(-1, 5, (m,), generator=g, device="cuda").int()) for m in (50, 700, 5000, 20000)]

    def run(slots, ids):
        x = store.read(slots, dtype=torch.float16)
        offsets, order = group_rows(ids, 5)
        return layer.forward(x, offsets, rows_in=order, rows_out=order)
    want = [run(*w) for w in work]
    torch.cuda.synchronize()
    bad = []

    def body(k):
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                for _ in range(50):
                    got = run(*work[k])
                    if not torch.equal(got, want[k]):
                        bad.append((k, "differs"))
        except Exception as e:  # noqa: BLE001
            bad.append((k, repr(e)))
    threads = [threading.Thread(target=body, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join(60) for t in threads]
    torch.cuda.synchronize()
    assert not bad and not any(t.is_alive() for t in threads), bad
