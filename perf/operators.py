"""Cases of the dense-layer operators: 8-bit rows, their matrix product, and matrix products grouped by expert.

They are the layers behind the pooled embedding of a ranking model (`RecomModel`): the pooled rows, one per sample, go
through a multi-layer perceptron of 1024, 256, 128 and 1 units, either one for all samples or one of several experts
chosen for each sample (a scenario, a market, a surface).  Row counts and widths are those of the benchmark
configurations (`recflex_b200/synth.py`): batches of 256, 4096, 16384 and 65536 samples; 480, 1924, 15608 and 24160
pooled units.  `run` computes an operator with elementary torch operations, or, with `own` set, with this package.
"""
import math

import torch

own = False

DEV = "cuda"
FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNITS = (480, 1924, 15608, 24160)  # pooled units of the benchmark configurations
LAYERS = (1024, 256, 128, 1)       # the perceptron of the end-to-end model
BATCH = 65536                      # the largest batch
MOST_FLOPS = 2 * 16384 * 15608 * 1024
MOST_BYTES = 3 * 16384 * 15608


# ---- cases -----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # pooled rows of one request, and of a whole batch, on their way into an 8-bit first layer
        {"name": "quantize one request", "op": "quantize", "rows": 1, "k": 15608, "dtype": "bf16"},
        {"name": "quantize cfg3 batch", "op": "quantize", "rows": 16384, "k": 15608, "dtype": "bf16"},
        # first layer for one request: latency, every weight read once
        {"name": "int8 one request", "op": "int8", "rows": 1, "k": 15608, "n": 1024, "act": "relu", "out": "bf16"},
        # first layer of an ordinary batch; 1924 units are no multiple of 16
        {"name": "int8 cfg2 batch", "op": "int8", "rows": 4096, "k": 1924, "n": 1024, "act": "relu", "out": "f16"},
        # first layer of the headline configuration's batch
        {"name": "int8 cfg3 batch", "op": "int8", "rows": 16384, "k": 15608, "n": 1024, "act": "relu", "out": "bf16"},
        # last layer: one unit, the scores of the largest batch in 32 bits
        {"name": "int8 scores", "op": "int8", "rows": 65536, "k": 128, "n": 1, "act": "sigmoid", "out": "f32"},
        # the samples of a small batch by scenario; a large batch with two experts a sample and padding
        {"name": "group small batch", "op": "group", "rows": 256, "groups": 8, "none": 0.0, "index": "i32"},
        {"name": "group large batch", "op": "group", "rows": 131072, "groups": 64, "none": 0.1, "index": "i64"},
        # first layer, a handful of requests over many experts: latency, only the experts hit are read
        {"name": "grouped few requests", "op": "grouped", "rows": 6, "groups": 16, "k": 1924, "n": 1024, "dtype": "bf16",
         "gather": True, "scatter": False, "act": "relu", "none": 0.0},
        # first layer of an ordinary batch, its rows taken in expert order by index
        {"name": "grouped cfg2 batch", "op": "grouped", "rows": 4096, "groups": 8, "k": 1924, "n": 1024, "dtype": "f16",
         "gather": True, "scatter": False, "act": "relu", "none": 0.0},
        # first layer of the headline configuration's batch
        {"name": "grouped cfg3 batch", "op": "grouped", "rows": 16384, "groups": 8, "k": 15608, "n": 1024, "dtype": "bf16",
         "gather": True, "scatter": False, "act": "relu", "none": 0.0},
        # second layer of the largest batch in 8 bits, back into the samples' own order
        {"name": "grouped int8 layer", "op": "grouped", "rows": 65536, "groups": 64, "k": 1024, "n": 256, "dtype": "i8",
         "gather": False, "scatter": True, "act": "none", "none": 0.05},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(("quantize", "int8", "int8", "group", "grouped", "grouped"))
    if op == "group":
        return {"op": op, "rows": _spread(rng, 1, 2 * BATCH), "groups": _spread(rng, 1, 256),
                "none": rng.choice((0.0, 0.0, 0.3)), "index": rng.choice(("i32", "i64"))}
    k = rng.choice(UNITS + LAYERS[:3]) if rng.random() < 0.4 else _spread(rng, 16, UNITS[-1])
    if op == "quantize":
        return {"op": op, "rows": _spread(rng, 1, min(BATCH, MOST_BYTES // (6 * k))), "k": k,
                "dtype": rng.choice(("f32", "bf16", "f16"))}
    n = rng.choice(LAYERS) if rng.random() < 0.5 else _spread(rng, 1, LAYERS[0])
    rows = _spread(rng, 1, min(BATCH, MOST_FLOPS // (2 * k * n)))
    if op == "int8":
        return {"op": op, "rows": rows, "k": k, "n": n, "act": rng.choice(("none", "relu", "sigmoid")),
                "out": rng.choice(("f32", "bf16", "f16"))}
    return {"op": op, "rows": rows, "groups": _spread(rng, 1, 64), "k": k, "n": n,
            "dtype": rng.choice(("bf16", "f16", "i8")), "gather": rng.random() < 0.5, "scatter": rng.random() < 0.5,
            "act": rng.choice(("none", "relu")), "none": rng.choice((0.0, 0.1))}


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _pitched(t, unit):
    """`t` [..., k] in storage whose rows start on 16-byte boundaries, as the layers keep their rows."""
    k = t.shape[-1]
    full = torch.zeros(t.shape[:-1] + ((k + unit - 1) // unit * unit,), dtype=t.dtype, device=t.device)
    full[..., :k] = t
    return full[..., :k]


def _pooled(rows, k, gen):
    """Pooled embedding rows: sums over bags of very different lengths, some features empty."""
    x = torch.randn(rows, k, generator=gen, device=DEV)
    bags = torch.rand(1, k, generator=gen, device=DEV)
    x *= 0.05 * torch.exp(2.0 * bags - 1.0)
    x *= torch.rand(1, k, generator=gen, device=DEV) > 0.1
    return x


def _codes(shape, gen):
    """8-bit values as a quantised normal vector of some thousand entries has them: about +-4 deviations over +-127."""
    return (torch.randn(shape, generator=gen, device=DEV) * 32.0).clamp_(-127, 127).round_().to(torch.int8)


def _experts(rows, groups, none, gen):
    """One expert a row, a few of them popular; -1 for rows of none (padding)."""
    share = torch.rand(groups, generator=gen, device=DEV) ** 3 + 0.02
    ids = torch.multinomial(share, rows, replacement=True, generator=gen)
    return torch.where(torch.rand(rows, generator=gen, device=DEV) < none, torch.full_like(ids, -1), ids)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    state = dict(case)
    rows, op = case["rows"], case["op"]
    if op == "quantize":
        state["x"] = _pooled(rows, case["k"], gen).to(FLOATS[case["dtype"]])
        return state
    if op == "group":
        state["ids"] = _experts(rows, case["groups"], case["none"], gen).to(
            torch.int32 if case["index"] == "i32" else torch.int64)
        return state
    k, n = case["k"], case["n"]
    if op == "int8":
        state["q"] = _pitched(_codes((rows, k), gen), 16)
        state["q_scale"] = torch.rand(rows, generator=gen, device=DEV) * 0.01 + 0.001
        state["w"] = _pitched(_codes((n, k), gen), 16)
        state["w_scale"] = (torch.rand(n, generator=gen, device=DEV) + 0.5) / (127.0 * math.sqrt(k))
        state["bias"] = (torch.rand(n, generator=gen, device=DEV) * 2 - 1) / math.sqrt(k)
        return state
    groups = case["groups"]
    ids = _experts(rows, groups, case["none"], gen)
    key = torch.where(ids < 0, torch.full_like(ids, groups), ids)
    state["order"] = torch.sort(key, stable=True).indices.to(torch.int32)
    counts = torch.stack([(key == g).sum() for g in range(groups)])
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device=DEV)
    offsets[1:] = counts.cumsum(0)
    state["offsets"] = offsets
    state["sizes"] = counts.tolist()  # the plain form's slices; the kernels read the offsets on the GPU
    if case["dtype"] == "i8":
        state["x"] = _pitched(_codes((rows, k), gen), 16)
        state["x_scale"] = torch.rand(rows, generator=gen, device=DEV) * 0.01 + 0.001
        state["w"] = _pitched(_codes((groups, n, k), gen), 16)
        state["w_scale"] = (torch.rand(groups, n, generator=gen, device=DEV) + 0.5) / (127.0 * math.sqrt(k))
    else:
        dtype = FLOATS[case["dtype"]]
        state["x"] = _pitched(_pooled(rows, k, gen).to(dtype), 8)
        w = torch.empty(groups, n, k, device=DEV).uniform_(-1.0 / math.sqrt(k), 1.0 / math.sqrt(k), generator=gen)
        state["w"] = _pitched(w.to(dtype), 8)
    state["bias"] = (torch.rand(groups, n, generator=gen, device=DEV) * 2 - 1) / math.sqrt(k)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------
def _act(y, act):
    return torch.relu(y) if act == "relu" else torch.sigmoid(y) if act == "sigmoid" else y


def _plain_quantize(s):
    x = s["x"].float()
    top = x.abs().amax(1)
    scale = top / torch.full_like(top, 127.0)
    # in 64 bits: which way a value next to the middle of two steps goes
    q = torch.round(s["x"].double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[:, None])
    return q.clamp(-127, 127).to(torch.int8), scale


def _plain_int8(s):
    y = torch.matmul(s["q"].float(), s["w"].float().t())
    y = y * (s["q_scale"][:, None] * s["w_scale"][None, :]) + s["bias"]
    return _act(y, s["act"]).to(FLOATS[s["out"]])


def _plain_group(s):
    ids, groups = s["ids"], s["groups"]
    key = torch.where((ids < 0) | (ids >= groups), torch.full_like(ids, groups), ids)
    keys, rows = torch.sort(key, stable=True)
    offsets = torch.searchsorted(keys, torch.arange(groups + 1, dtype=keys.dtype, device=keys.device))
    return rows.to(torch.int32), offsets.to(torch.int32)


def _plain_grouped(s):
    i8 = s["dtype"] == "i8"
    out = torch.zeros(s["rows"], s["n"], dtype=torch.bfloat16 if i8 else s["x"].dtype, device=DEV)
    order, at = s["order"].long(), 0
    for g, size in enumerate(s["sizes"]):  # one matrix product an expert, of that expert's rows alone
        if size:
            x = s["x"][order[at:at + size]] if s["gather"] else s["x"][at:at + size]
            y = torch.matmul(x.float(), s["w"][g].float().t())
            if i8:
                scale = s["x_scale"][order[at:at + size]] if s["gather"] else s["x_scale"][at:at + size]
                y = y * (scale[:, None] * s["w_scale"][g][None, :])
            y = _act(y + s["bias"][g], s["act"]).to(out.dtype)
            if s["scatter"]:
                out[order[at:at + size]] = y
            else:
                out[at:at + size] = y
        at += size
    return out


def run(state):
    op = state["op"]
    if own:
        from recflex_b200 import linear

        if op == "quantize":
            return linear.quantize_rows(state["x"])
        if op == "int8":
            return linear.int8_linear(state["q"], state["q_scale"], state["w"], state["w_scale"], bias=state["bias"],
                                      activation=state["act"], out_dtype=FLOATS[state["out"]])
        if op == "group":
            return linear.group_rows(state["ids"], state["groups"])
        order = state["order"]
        return linear.grouped_linear(state["x"], state["w"], state["offsets"], bias=state["bias"],
                                     activation=state["act"], in_rows=order if state["gather"] else None,
                                     out_rows=order if state["scatter"] else None, x_scale=state.get("x_scale"),
                                     weight_scale=state.get("w_scale"))
    return {"quantize": _plain_quantize, "int8": _plain_int8, "group": _plain_group, "grouped": _plain_grouped}[op](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    rows, op = case["rows"], case["op"]
    if op == "group":
        return {"bytes": rows * ((4 if case["index"] == "i32" else 8) + 4) + 4 * (case["groups"] + 1), "flops": 2 * rows}
    k = case["k"]
    if op == "quantize":
        return {"bytes": rows * (k * ((4 if case["dtype"] == "f32" else 2) + 1) + 4), "flops": 3 * rows * k}
    n = case["n"]
    if op == "int8":
        return {"bytes": rows * (k + 4 + n * (4 if case["out"] == "f32" else 2)) + n * (k + 8), "flops": 2 * rows * n * k}
    size = 1 if case["dtype"] == "i8" else 2
    hit = min(case["groups"], rows)  # a batch of few rows reads the experts that it hits
    fixed = case["groups"] * 4 + rows * 4 * (case["gather"] + case["scatter"])
    return {"bytes": rows * (k * size + 2 * n) + hit * n * (k * size + 4) + fixed, "flops": 2 * rows * n * k}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "group":
        member = [((s["ids"] == g).nonzero().flatten()) for g in range(case["groups"])]
        rest = ((s["ids"] < 0) | (s["ids"] >= case["groups"])).nonzero().flatten()
        ends = torch.tensor([0] + [len(m) for m in member], device=DEV).cumsum(0)
        return torch.cat(member + [rest]).to(torch.int32), ends.to(torch.int32)
    if op == "quantize":
        scale = s["x"].double().abs().max(dim=1).values / 127.0
        # the steps are those of the scale as it is held, in 32 bits
        step = scale.float().double()
        codes = (s["x"].double() / step.clamp(min=1e-300).unsqueeze(1)).round()
        return codes.clamp(min=-127, max=127).to(torch.int8), scale
    if op == "int8":
        y = torch.einsum("mk,nk->mn", s["q"].double() * s["q_scale"].double().unsqueeze(1),
                         s["w"].double() * s["w_scale"].double().unsqueeze(1)) + s["bias"].double()
    else:
        y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=DEV)
        place = torch.arange(case["rows"], device=DEV)
        source = s["order"].long() if case["gather"] else place
        target = s["order"].long() if case["scatter"] else place
        group_of = torch.searchsorted(s["offsets"][1:].contiguous().long(), place, right=True)
        for g in range(case["groups"]):
            mine = (group_of == g).nonzero().flatten()
            if len(mine):
                a, b = s["x"][source[mine]].double(), s["w"][g].double()
                if case["dtype"] == "i8":
                    a, b = a * s["x_scale"][source[mine]].double().unsqueeze(1), b * s["w_scale"][g].double().unsqueeze(1)
                z = torch.einsum("mk,nk->mn", a, b) + s["bias"][g].double()
                y[target[mine]] = z.clamp(min=0) if case["act"] == "relu" else z
        return y
    if case["act"] == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-y))
    return y.clamp(min=0) if case["act"] == "relu" else y
