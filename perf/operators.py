"""Cases for the operators that serve what comes behind a lookup: rows kept in 8 or 4 bits (written and read back by slot), dense
layers with their epilogue, the same layers grouped by expert over ragged runs of rows, and the grouping of rows by expert.

Where ``own`` is false ``run`` computes an operator in plain torch operations (32 bits, 64 next to a rounding border); where it is
true it makes the calls that a program makes of hugectr_backend_amd.  ``exact`` is the definition in 64 bits, written apart.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
TINY = 2.0 ** -100   # a group of values whose largest magnitude is below this is held as zeros
DIMS = (1, 3, 8, 16, 17, 32, 48, 64, 100, 128, 200, 256, 500, 512, 1000, 1024)
ACTIVATIONS = ("none", "relu", "gelu", "silu", "sigmoid")


# ------------------------------------------------------------------------------------------------------------------ cases
def _write(name, n, dim, bits, group, type, echo, store):
    return {"name": name, "op": "write", "n": n, "dim": dim, "bits": bits, "group": group, "type": type, "echo": echo, "store": store}


def _read(name, n, dim, bits, group, type, store):
    return {"name": name, "op": "read", "n": n, "dim": dim, "bits": bits, "group": group, "type": type, "store": store}


def _linear(name, m, k, n, type, out, act, mul, residual, pad=0):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "type": type, "out": out, "act": act, "mul": mul, "residual": residual,
            "pad": pad}


def _experts(name, m, e, k, n, type, out, act, residual, sorted, skew, behind):
    return {"name": name, "op": "experts", "m": m, "e": e, "k": k, "n": n, "type": type, "out": out, "act": act, "residual": residual,
            "sorted": sorted, "skew": skew, "behind": behind}


def _group(name, m, e, skew, behind):
    return {"name": name, "op": "group", "m": m, "e": e, "skew": skew, "behind": behind}


def listed():
    return [
        # one whole Criteo request (65,536 samples x 26 tables, 128 floats a row) goes into the 8-bit store: filling it, refreshing it
        _write("write_criteo_request", 1703936, 128, 8, 0, "fp32", False, 4000000),
        # the wide rows of a Wide&Deep request (1,024 samples x 26 keys, 16 floats), held in 4 bits; the caller answers with the values
        # that later reads give
        _write("write_wide_and_deep_4bit", 26624, 16, 4, 0, "fp32", True, 1000000),
        # the few rows one small request missed, half precision, one scale per 32 values
        _write("write_missed_rows", 777, 200, 4, 32, "fp16", True, 100000),
        # a whole Criteo request is answered from the 8-bit store in the lookup's own type
        _read("read_criteo_request", 1703936, 128, 8, 0, "fp32", 4000000),
        # a 4,096-key request over 16-float rows (the smallest workload of the benchmark), 4 bits, half precision for a dense step
        _read("read_small_request_4bit", 4096, 16, 4, 0, "fp16", 1000000),
        # the first top layer of a 26-table DLRM: 128 + 351 interaction columns, rows 480 apart as the dense step writes them
        _linear("linear_dlrm_top", 65536, 479, 1024, "fp16", "fp16", "relu", False, False, 1),
        # one sample through a wide layer: only latency and the weights' bytes count
        _linear("linear_one_sample", 1, 1024, 1024, "fp16", "fp16", "relu", False, False),
        # a cross layer over 27 vectors of 128: x0 * (x W + b) + x
        _linear("linear_cross_layer", 16384, 3456, 3456, "bf16", "bf16", "none", True, True),
        # a tower per domain over a full batch in request order, a few domains with most of the samples
        _experts("experts_domains_batch", 65536, 16, 1024, 512, "fp16", "fp16", "relu", False, False, 0.5, False),
        # a small request over many experts: a handful of rows each, some none, sorted already, padding rows at the end
        _experts("experts_small_request", 300, 64, 479, 256, "bf16", "fp32", "silu", True, True, 0.5, True),
        # the grouping those calls need: a full batch, and a small request
        _group("group_batch", 65536, 16, 0.5, False),
        _group("group_small_request", 300, 64, 0.5, True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "read", "linear", "linear", "experts", "experts", "group"))
    if op in ("write", "read"):
        dim = rng.choice(DIMS)
        n = _log(rng, 1, max(1, 1703936 * 128 // max(dim, 128)))
        store = max(n + rng.randrange(1, 1000), min(4000000 * 128 // max(dim, 128), n * rng.randrange(1, 4)))
        bits, group, type = rng.choice((8, 4)), rng.choice((0, 0, 16, 32, 64, 128, 256)), rng.choice(tuple(TYPES))
        if op == "read":
            c = _read("", n, dim, bits, group, type, store)
        else:
            c = _write("", n, dim, bits, group, type, bits == 4 or rng.random() < 0.5, store)
    elif op == "linear":
        m, k, n = _log(rng, 1, 65536), _log(rng, 1, 3456), _log(rng, 1, 3456)
        while m * k * n > 16384 * 3456 * 3456 or m * (k + n) > 65536 * 2048:
            m = (m + 1) // 2
        type = rng.choice(("fp16", "bf16"))
        c = _linear("", m, k, n, type, rng.choice((type, "fp32")), rng.choice(ACTIVATIONS), rng.random() < 0.3, rng.random() < 0.3,
                    rng.choice((0, 0, 1, 8, 13)))
    elif op == "experts":
        m, e, k, n = _log(rng, 1, 65536), _log(rng, 1, 64), _log(rng, 8, 1024), _log(rng, 8, 512)
        type = rng.choice(("fp16", "bf16"))
        c = _experts("", m, e, k, n, type, rng.choice((type, "fp32")), rng.choice(ACTIVATIONS), rng.random() < 0.3, rng.random() < 0.5,
                     rng.choice((0.0, 0.5)), rng.random() < 0.3)
    else:
        c = _group("", _log(rng, 1, 65536), _log(rng, 1, 1024), rng.choice((0.0, 0.5, 1.0)), rng.random() < 0.3)
    del c["name"]
    return c


def work(c):
    op = c["op"]
    if op in ("write", "read"):
        n, d, size = c["n"], c["dim"], SIZE[c["type"]]
        held = n * (-(-d * c["bits"] // 8) + 4 * _groups(c))
        if op == "read":
            return {"bytes": n * 8 + held + n * d * size, "flops": n * d}
        return {"bytes": n * 8 + n * d * size * (2 if c["echo"] else 1) + held, "flops": 4 * n * d}
    if op == "linear":
        m, k, n, size = c["m"], c["k"], c["n"], SIZE[c["type"]]
        rows = m * k * size + m * n * (SIZE[c["out"]] + size * (int(c["mul"]) + int(c["residual"])))
        return {"bytes": rows + k * n * size + 4 * n, "flops": 2 * m * k * n}
    if op == "experts":
        m, k, n, size = c["m"], c["k"], c["n"], SIZE[c["type"]]
        rows = m * k * size + m * n * (SIZE[c["out"]] + size * int(c["residual"])) + (0 if c["sorted"] else 4 * m)
        return {"bytes": rows + min(c["e"], m) * (k * n * size + 4 * n) + 4 * (c["e"] + 1), "flops": 2 * m * k * n}
    return {"bytes": 8 * c["m"] + 4 * (c["e"] + 1), "flops": c["m"]}


# ------------------------------------------------------------------------------------------------------------------ inputs
def _groups(c):
    return -(-c["dim"] // c["group"]) if c["group"] else 1


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _rows(n, dim, type, g):
    # trained embedding rows: near zero, each row with a spread of its own
    spread = 0.02 + 0.2 * torch.rand(n, 1, generator=g, device=DEV)
    return (torch.randn(n, dim, generator=g, device=DEV) * spread).to(TYPES[type])


def _slots(n, store, g):
    # mostly distinct places in no order, now and then one twice, about one in a hundred a padding entry (-1)
    s = torch.randperm(store, generator=g, device=DEV)[:n].clone()
    r = torch.rand(n, generator=g, device=DEV)
    s = torch.where(r < 0.01, s.roll(1), s)
    return torch.where(r > 0.99, torch.full_like(s, -1), s)


def _ids(c, g):
    p = torch.arange(1, c["e"] + 1, device=DEV, dtype=torch.float64).pow(-c["skew"]).float()
    ids = torch.multinomial(p, c["m"], replacement=True, generator=g).to(torch.int32)
    if c["behind"]:
        ids = torch.where(torch.rand(c["m"], generator=g, device=DEV) < 0.05, torch.full_like(ids, -1), ids)
    return ids


def _data(c, seed):
    """The inputs alone, from the seed."""
    g, op = _gen(seed), c["op"]
    if op == "write":
        return {"rows": _rows(c["n"], c["dim"], c["type"], g), "slots": _slots(c["n"], c["store"], g)}
    if op == "read":
        return {"rows": _rows(c["store"], c["dim"], "fp32", g), "slots": _slots(c["n"], c["store"], g)}
    if op == "group":
        return {"ids": _ids(c, g)}
    t, e = TYPES[c["type"]], c.get("e", 1)
    m, k, n = c["m"], c["k"], c["n"]
    d = {"x": torch.randn(m, k + c.get("pad", 0), generator=g, device=DEV).to(t)[:, :k],
         "w": (torch.randn(e, k, n, generator=g, device=DEV) / math.sqrt(k)).to(t),
         "b": 0.1 * torch.randn(e, n, generator=g, device=DEV)}
    for name in ("mul", "residual"):
        d[name] = torch.randn(m, n, generator=g, device=DEV).to(t) if c.get(name) else None
    if op == "experts":
        ids = _ids(c, g)
        if c["sorted"]:
            ids = torch.where(ids < 0, torch.full_like(ids, e), ids).sort().values
        d["offsets"], d["order"] = _plain_group(ids, e)
        d["most"] = int((d["offsets"][1:] - d["offsets"][:-1]).max())
        if c["sorted"]:
            d["order"] = None
    return d


def prepare(c, seed):
    s = {"case": c, **_data(c, seed)}
    op = c["op"]
    if op == "write":
        if own:
            from hugectr_backend_amd.quantized_rows import QuantizedRows
            s["store"] = QuantizedRows(c["store"], c["dim"], bits=c["bits"], group=c["group"])
        else:   # one row more, where what is not kept goes
            s["codes"] = torch.zeros(c["store"] + 1, c["dim"], dtype=torch.int8, device=DEV)
            s["scales"] = torch.zeros(c["store"] + 1, _groups(c), device=DEV)
    elif op == "read":
        if own:
            from hugectr_backend_amd.quantized_rows import QuantizedRows
            s["store"] = QuantizedRows(c["store"], c["dim"], bits=c["bits"], group=c["group"])
            s["store"].write(s["rows"], torch.arange(c["store"], device=DEV))
        else:
            q, s["scales"] = _plain_quantize(s["rows"], c["bits"], c["group"])
            s["codes"] = _pack(q) if c["bits"] == 4 else q
        del s["rows"]
    elif own and op == "linear":
        from hugectr_backend_amd.dense import LinearLayer
        s["layer"] = LinearLayer(s.pop("w")[0], s.pop("b")[0], activation=c["act"], dtype=TYPES[c["type"]])
    elif own and op == "experts":
        from hugectr_backend_amd.dense import ExpertLayers
        s["layer"] = ExpertLayers(s.pop("w"), s.pop("b"), activation=c["act"], dtype=TYPES[c["type"]])
    return s


# ------------------------------------------------------------------------------------------------------------------ plain forms
def _by_group(rows, group):
    n, d = rows.shape
    g = group or d
    x = torch.nn.functional.pad(rows.float(), (0, -d % g))
    return x.view(n, -1, g)


def _plain_quantize(rows, bits, group):
    """codes [n, dim] int8, scales [n, groups]: scale = the group's largest magnitude / 127 (7) rounded to 32 bits,
    code = value / scale to the nearest, ties to even."""
    levels = 127.0 if bits == 8 else 7.0
    x = _by_group(rows, group)
    top = x.abs().amax(-1)
    scale = (top.double() / torch.full_like(top, levels, dtype=torch.float64)).float()
    scale = torch.where(top < TINY, torch.zeros_like(scale), scale)
    div = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    q = (x.double() / div[..., None]).round().clamp(-levels, levels)
    q = torch.where((scale > 0)[..., None], q, torch.zeros_like(q))
    return q.flatten(1)[:, : rows.shape[1]].to(torch.int8).contiguous(), scale


def _plain_values(q, scale, group, type):
    n, d = q.shape
    x = _by_group(q, group) * scale[..., None]
    return x.flatten(1)[:, :d].to(TYPES[type])


def _pack(q):
    q = torch.nn.functional.pad(q, (0, q.shape[1] % 2)).view(q.shape[0], -1, 2).to(torch.uint8)
    return (q[..., 0] & 15) | (q[..., 1] << 4)


def _unpack(p, d):
    q = torch.stack((p & 15, p >> 4), -1).flatten(1)[:, :d].to(torch.int8)
    return torch.where(q > 7, q - 16, q)


def _plain_write(s):
    c = s["case"]
    q, scale = _plain_quantize(s["rows"], c["bits"], c["group"])
    slots, n, store = s["slots"], c["n"], c["store"]
    # of a slot that is named twice the last row stays
    at = torch.arange(n, device=DEV)
    to = torch.where((slots >= 0) & (slots < store), slots, torch.full_like(slots, store))
    last = torch.full((store + 1,), -1, dtype=torch.int64, device=DEV).scatter_reduce(0, to, at, "amax")
    to = torch.where(last[to] == at, to, torch.full_like(to, store))
    s["codes"][to] = q
    s["scales"][to] = scale
    out = {"scales": s["scales"][:store]}
    if c["bits"] == 8:
        out["codes"] = s["codes"][:store]
    if c["echo"]:
        out["held"] = _plain_values(q, scale, c["group"], c["type"])
    return out


def _plain_read(s):
    c, slots = s["case"], s["slots"]
    inside = (slots >= 0) & (slots < c["store"])
    at = torch.where(inside, slots, torch.zeros_like(slots))
    q, scale = s["codes"][at], s["scales"][at]
    if c["bits"] == 4:
        q = _unpack(q, c["dim"])
    x = _plain_values(q, scale, c["group"], c["type"])
    return torch.where(inside[:, None], x, torch.zeros_like(x))


def _plain_act(y, act):
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-y))
    return y


def _plain_end(y, s):
    if s["mul"] is not None:
        y = y * s["mul"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(TYPES[s["case"]["out"]])


def _plain_linear(s):
    y = s["x"].float() @ s["w"][0].float() + s["b"]
    return _plain_end(_plain_act(y, s["case"]["act"]), s)


def _plain_experts(s):
    """Every expert's rows padded to the longest run, one batched product, and the rows back to where they belong."""
    c, x, off = s["case"], s["x"], s["offsets"].long()
    e, m, most = c["e"], c["m"], max(1, s["most"])
    j = torch.arange(most, device=DEV)
    at = torch.where(j < (off[1:] - off[:-1])[:, None], off[:-1, None] + j, torch.zeros_like(off[:-1, None]))
    src = at if s["order"] is None else s["order"].long()[at]
    y = torch.bmm(x[src.flatten()].float().view(e, most, c["k"]), s["w"].float()) + s["b"][:, None, :]
    y = _plain_act(y, c["act"]).flatten(0, 1)
    r = torch.arange(m, device=DEV)
    who = (r[:, None] >= off[1:]).sum(1)
    inside = who < e
    who = torch.where(inside, who, torch.zeros_like(who))
    y = y[torch.where(inside, who * most + r - off[who], torch.zeros_like(r))]
    if s["order"] is not None:
        back = torch.empty_like(r)
        back[s["order"].long()] = r
        y, inside = y[back], inside[back]
    y = _plain_end(y, s)
    return torch.where(inside[:, None], y, torch.zeros_like(y))


def _plain_group(ids, e):
    to = torch.where((ids >= 0) & (ids < e), ids, torch.full_like(ids, e)).long()
    counts = torch.zeros(e + 1, dtype=torch.int64, device=DEV).scatter_add(0, to, torch.ones_like(to))
    ends = counts[:e].cumsum(0)
    offsets = torch.cat((torch.zeros_like(ends[:1]), ends)).to(torch.int32)
    return offsets, torch.argsort(to, stable=True).to(torch.int32)


# ------------------------------------------------------------------------------------------------------------------ run
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "group":
            return _plain_group(s["ids"], c["e"])
        return {"write": _plain_write, "read": _plain_read, "linear": _plain_linear, "experts": _plain_experts}[op](s)
    if op == "write":
        store = s["store"]
        held = store.write(s["rows"], s["slots"], held=torch.empty_like(s["rows"]) if c["echo"] else None)
        out = {"scales": store.scales}
        if c["bits"] == 8:
            out["codes"] = store.codes[:, : c["dim"]]
        if c["echo"]:
            out["held"] = held
        return out
    if op == "read":
        return s["store"].read(s["slots"], dtype=TYPES[c["type"]])
    if op == "linear":
        return s["layer"].forward(s["x"], mul=s["mul"], residual=s["residual"], out_dtype=TYPES[c["out"]])
    if op == "experts":
        return s["layer"].forward(s["x"], s["offsets"], rows_in=s["order"], rows_out=s["order"], residual=s["residual"],
                                  out_dtype=TYPES[c["out"]])
    from hugectr_backend_amd.dense import group_rows
    return group_rows(s["ids"], c["e"])


# ------------------------------------------------------------------------------------------------------------------ exact
def _exact_codes(rows, c):
    """(code, scale of each value, scale of each group) of the definition, column blocks one after the other."""
    levels = 127 if c["bits"] == 8 else 7
    n, d = rows.shape
    step = c["group"] or d
    x = rows.double()
    code, wide, scales = torch.empty_like(x), torch.empty_like(x), []
    for a in range(0, d, step):
        part = x[:, a: a + step]
        top = part.abs().max(dim=1).values
        exact = top / levels
        held = exact.float().double()          # the scale is held in 32 bits by definition: codes are relative to that
        gone = top < TINY
        held[gone] = 0
        exact[gone] = 0
        safe = held.masked_fill(held == 0, 1)
        code[:, a: a + step] = torch.round(part / safe[:, None]).clamp_(-levels, levels)
        code[:, a: a + step][held == 0] = 0
        wide[:, a: a + step] = held[:, None]
        scales.append(exact)
    return code, wide, torch.stack(scales, 1)


def exact(c, seed):
    d, op = _data(c, seed), c["op"]
    if op == "group":
        return None
    if op == "write":
        code, wide, scale = _exact_codes(d["rows"], c)
        scales = torch.zeros(c["store"], scale.shape[1], dtype=torch.float64, device=DEV)
        slots = d["slots"].cpu().tolist()
        last = {}
        for i, slot in enumerate(slots):
            if 0 <= slot < c["store"]:
                last[slot] = i
        where = torch.tensor(list(last.keys()), dtype=torch.int64, device=DEV)
        scales[where] = scale[torch.tensor(list(last.values()), dtype=torch.int64, device=DEV)]
        out = {"scales": scales}
        if c["bits"] == 8:
            out["codes"] = None
        if c["echo"]:
            out["held"] = code * wide
        return out
    if op == "read":
        slots = d["slots"]
        inside = (slots >= 0) & (slots < c["store"])
        out = torch.zeros(c["n"], c["dim"], dtype=torch.float64, device=DEV)
        code, wide, _ = _exact_codes(d["rows"][slots[inside]], c)
        out[inside] = code * wide
        return out
    act = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "sigmoid": torch.sigmoid, "silu": lambda v: v * torch.sigmoid(v),
           "gelu": lambda v: v * torch.special.ndtr(v)}[c["act"]]
    x = d["x"].double()
    out = torch.zeros(c["m"], c["n"], dtype=torch.float64, device=DEV)
    runs = [(0, c["m"])]
    if op == "experts":
        ends = d["offsets"].tolist()
        runs = list(zip(ends[:-1], ends[1:]))
    for e, (a, b) in enumerate(runs):
        rows = torch.arange(a, b, device=DEV)
        if d.get("order") is not None:
            rows = d["order"].long()[a:b]
        y = act(x[rows] @ d["w"][e].double() + d["b"][e].double())
        if d["mul"] is not None:
            y = y * d["mul"][rows].double()
        if d["residual"] is not None:
            y = y + d["residual"][rows].double()
        out[rows] = y
    return out
