"""The operators of this library that send each row of a batch to a weight of its own: rows sorted by expert and back,
the gradient of that, the experts' projections, and low-rank adapters beside a shared projection.

A case is one call of an operator as a serving or training program makes it. `op` says which:
  route     ids [T][k] -> the plan (order, position, offsets), the rows of x sorted by expert, and the experts' rows
            summed back per token with the router's weights
  grad      the gradient of both: of the experts' rows, the router's weights and x
  expert    x [T][K] quantized and projected by each row's expert (`rows` output rows of each of one or two weights that
            share the activation); `sorted`: x already lies in the plan's order, as a down projection finds it
  adapter   y + scale * B (A x), the adapter chosen per token, none for some
`mode` is the weight tier of an expert projection:
  token     int4 codes, FP16 scale per `group` (64 / 128), one activation scale per token
  block     int4 codes with zero points, `group` 32 / 64, one activation scale per (token, K32 block)
  w8        int8 codes, FP16 scale per K32, activation scales per K32 block
`drop` is the share of slots that carry no expert (rows whose expert lives on another GPU) or no adapter.
"""
import math

import torch

own = False

HIDDEN, INTER = 5120, 17408
BYTES = {"bf16": 2, "f32": 4}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _route(T, k, E, H, x, drop=0.0):
    return {"op": "route", "T": T, "k": k, "E": E, "H": H, "x": x, "drop": drop}


def _grad(T, k, E, H, x, drop=0.0):
    return {"op": "grad", "T": T, "k": k, "E": E, "H": H, "x": x, "drop": drop}


def _expert(T, k, E, K, rows, mode, group, x="bf16", out="bf16", in_order=False, drop=0.0):
    return {"op": "expert", "T": T, "k": k, "E": E, "K": K, "rows": rows, "mode": mode, "group": group, "x": x,
            "out": out, "sorted": in_order, "drop": drop}


def _adapter(T, n, r, K, M, x, y, seg="", drop=0.0):
    return {"op": "adapter", "T": T, "n": n, "r": r, "K": K, "M": M, "x": x, "y": y, "seg": seg, "drop": drop}


def listed():
    return [
        # a decode step of eight sequences through a router of 128 experts: latency
        dict(_route(8, 8, 128, HIDDEN, "bf16"), name="route_decode8"),
        # odd sizes throughout, a quarter of the experts on another GPU
        dict(_route(1777, 6, 61, 2049, "f32", 0.25), name="route_odd"),
        # a prefill chunk
        dict(_route(4096, 8, 128, HIDDEN, "bf16"), name="route_prefill"),
        # a training step's share of a batch, few large experts
        dict(_grad(4093, 2, 8, HIDDEN, "bf16"), name="grad_top2"),
        # the same of many small experts, in float32
        dict(_grad(1024, 8, 64, 2048, "f32", 0.1), name="grad_top8"),
        # one sequence: the down projections of its four experts, int4 with zero points
        dict(_expert(1, 4, 32, 1024, "5120", "block", 32, x="f32", out="f32", in_order=True),
             name="expert_down_decode1"),
        # a batch of 16 sequences: gate and up of up to 64 experts
        dict(_expert(16, 8, 64, HIDDEN, "1024,1024", "token", 128), name="expert_gate_up_decode16"),
        # a prompt of 300 tokens, int8 weights, half of the experts on another GPU
        dict(_expert(300, 6, 40, 2048, "1408", "w8", 32, out="f32", drop=0.5), name="expert_prompt300"),
        # a prefill chunk: gate and up of 64 experts
        dict(_expert(2048, 8, 64, HIDDEN, "1024,1024", "token", 128), name="expert_gate_up_prefill"),
        # eight requests, each with an adapter of its own, beside the attention output: latency
        dict(_adapter(8, 8, 16, HIDDEN, HIDDEN, "bf16", "bf16"), name="adapter_decode8"),
        # 61 requests over 24 adapters and none, beside the down projection with its float32 output
        dict(_adapter(61, 24, 64, INTER, HIDDEN, "f32", "f32", drop=0.2), name="adapter_decode61"),
        # six prompts of unequal length packed into one prefill, each with its adapter, beside gate
        dict(_adapter(3965, 6, 32, HIDDEN, INTER, "bf16", "bf16", seg="17,64,300,512,1024,2048"),
             name="adapter_packed"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["route", "grad", "expert", "adapter"])
    drop = rng.choice([0.0, 0.0, 0.1, 0.5])
    if op in ("route", "grad"):
        k, x = rng.choice([1, 2, 4, 6, 8]), rng.choice(["bf16", "f32"])
        H = spread(64, 5120)
        H = rng.choice([H, H // 8 * 8, H // 64 * 64])
        slots = 32768 // (2 if x == "f32" else 1) // (2 if op == "grad" else 1)
        return (_route if op == "route" else _grad)(spread(1, slots // max(k, 2)), k,
                                                     max(k, spread(4, 256)), H, x, drop)
    if op == "expert":
        k, E = rng.choice([1, 2, 4, 8]), rng.choice([8, 16, 32, 40, 64])
        mode, group = rng.choice([("token", 64), ("token", 128), ("block", 32), ("block", 64), ("w8", 32)])
        one = spread(64, 2048) // 16 * 16
        return _expert(spread(1, 2048), k, E, spread(512, 5120) // 128 * 128, rng.choice([str(one), "%d,%d" % (one, one)])
                       if one <= 1024 else str(one), mode, group, rng.choice(["bf16", "f32"]),
                       rng.choice(["bf16", "f32"]), rng.random() < 0.3, drop)
    K, M = spread(512, INTER) // 128 * 128, spread(512, INTER) // 16 * 16
    x, y = rng.choice(["bf16", "f32"]), rng.choice(["bf16", "f32"])
    T = spread(1, min(3965, int(3e8 / (K * BYTES[x] + 2 * M * BYTES[y]))))
    n = rng.choice([1, 3, 8, 24, 64])
    seg = ""
    if T > 256:
        cuts = sorted({rng.randrange(1, T) for _ in range(rng.randrange(0, 7))})
        seg = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [T]))
    return _adapter(T, n, rng.choice([8, 16, 24, 32, 64, 128]), K, M, x, y, seg, drop)


def _ids(case, gen, groups, k):
    """The k experts of each token, of uneven popularity, and the router's weights; -1 for a dropped slot."""
    T = case["T"]
    popular = torch.randn(groups, generator=gen, device="cuda") * 0.5
    score = popular + torch.randn(T, groups, generator=gen, device="cuda")
    top = score.topk(k, dim=1)
    ids = top.indices.to(torch.int32)
    weights = torch.softmax(top.values, dim=1)
    gone = torch.rand(T, k, generator=gen, device="cuda") < case["drop"]
    return torch.where(gone, torch.full_like(ids, -1), ids).contiguous(), weights


def _inputs(case, seed):
    """The seeded inputs of a case, as tensors on the GPU."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def normal(*shape, dtype="f32"):
        return torch.randn(*shape, generator=gen, device="cuda").to(TYPES[dtype])

    d = {}
    T = case["T"]
    if case["op"] in ("route", "grad"):
        k, H, x = case["k"], case["H"], case["x"]
        d["ids"], d["weights"] = _ids(case, gen, case["E"], k)
        d["rows"] = normal(T * k, H, dtype=x)
        if case["op"] == "route":
            d["x"] = normal(T, H, dtype=x)
        else:
            d["dy"], d["drows"] = normal(T, H, dtype=x), normal(T * k, H, dtype=x)
    elif case["op"] == "expert":
        k, E, K, group = case["k"], case["E"], case["K"], case["group"]
        d["ids"], _ = _ids(case, gen, E, k)
        d["x"] = normal(T * k if case["sorted"] else T, K, dtype=case["x"])
        d["codes"], d["scales"] = [], []
        for M in [int(m) for m in case["rows"].split(",")]:
            top = 128 if case["mode"] == "w8" else 8
            d["codes"].append(torch.randint(-top, top, (E * M, K), generator=gen, device="cuda", dtype=torch.int8))
            s = (torch.randn(E * M, K // group, generator=gen, device="cuda").abs() * (0.002 if top == 128 else 0.02))
            bits = s.to(torch.float16).view(torch.int16)
            if case["mode"] == "block":          # the low four bits hold the zero point
                zero = torch.randint(0, 16, bits.shape, generator=gen, device="cuda", dtype=torch.int16)
                bits = (bits & -16) | zero
            d["scales"].append(bits.contiguous())
    else:
        n, r, K, M = case["n"], case["r"], case["K"], case["M"]
        d["x"], d["y"] = normal(T, K, dtype=case["x"]), normal(T, M, dtype=case["y"])
        d["a"] = (normal(n, r, K) / math.sqrt(K)).to(torch.bfloat16)
        d["b"] = (normal(n, M, r) / math.sqrt(r)).to(torch.bfloat16)
        d["scale"] = torch.rand(n, generator=gen, device="cuda") * 2 + 0.25
        if case["seg"]:                          # packed prompts: one adapter each
            length = torch.tensor([int(s) for s in case["seg"].split(",")], device="cuda")
            pick = torch.randint(0, n, (len(length),), generator=gen, device="cuda")
            gone = torch.rand(len(length), generator=gen, device="cuda") < case["drop"]
            ids = torch.where(gone, torch.full_like(pick, -1), pick).repeat_interleave(length)
        else:
            ids = torch.randint(0, n, (T,), generator=gen, device="cuda")
            gone = torch.rand(T, generator=gen, device="cuda") < case["drop"]
            ids = torch.where(gone, torch.full_like(ids, -1), ids)
        d["ids"] = ids.to(torch.int32).view(T, 1).contiguous()
    return d


def _plan(ids, groups):
    """(offsets, order, position) of the slots sorted by group, those without one last."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat < 0) | (flat >= groups), groups, flat)
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(groups, device=key.device)).sum(0)
    offsets = torch.cat([torch.zeros_like(counts[:1]), counts.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    position = torch.where(key == groups, -1, place)
    return offsets.to(torch.int32), order.to(torch.int32), position.to(torch.int32).view_as(ids)


def prepare(case, seed):
    s = dict(case)
    s.update(_inputs(case, seed))
    T, k = case["T"], case.get("k", 1)
    groups = case["n"] if case["op"] == "adapter" else case["E"]
    s["groups"] = groups
    if case["op"] == "route":
        s["out"] = torch.zeros(T * k, case["H"], dtype=s["x"].dtype, device="cuda")
        return s
    # the step's plan, which its layers and its backward pass share
    s["plan"] = _plan(s["ids"], groups)
    # (the most rows of one expert; the plain form pads to it)
    s["most"] = int((s["plan"][0][1:] - s["plan"][0][:-1]).max())
    if case["op"] == "grad":
        s["out"] = torch.zeros(T * k, case["H"], dtype=s["rows"].dtype, device="cuda")
    elif case["op"] == "expert":
        s["outs"] = [torch.zeros(T * k, c.shape[0] // groups, dtype=TYPES[case["out"]], device="cuda") for c in s["codes"]]
        if own:                                  # the packed weights that a program keeps
            from knivesysl_xe_amd import _lib, ops
            if case["mode"] == "w8":
                s["packed"] = [ops.W4Weight.from_codes_s8(c, b) for c, b in zip(s["codes"], s["scales"])]
            else:
                enc = _lib.SCALE_FP16_ZP4 if case["mode"] == "block" else _lib.SCALE_FP16
                s["packed"] = [ops.W4Weight.from_codes(c, b, case["group"], enc) for c, b in zip(s["codes"], s["scales"])]
    else:
        s["out"] = torch.empty_like(s["y"])
    return s


def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from knivesysl_xe_amd import ops
    if s["op"] == "route":
        route = ops.route_rows(s["ids"], s["groups"])
        rows = ops.dispatch_rows(s["x"], route, out=s["out"])
        y = ops.combine_rows(s["rows"], route, s["weights"])
        return {"offsets": route.offsets, "order": route.order, "position": route.position, "rows": rows, "y": y}
    route = ops.RowRoute(s["T"], s.get("k", 1), s["groups"], *s["plan"])
    if s["op"] == "grad":
        drows, dweights = ops.combine_rows_backward(s["dy"], s["rows"], route, s["weights"], out=s["out"])
        return {"drows": drows, "dweights": dweights, "dx": ops.dispatch_rows_backward(s["drows"], route)}
    if s["op"] == "expert":
        a = ops.quantize_act(s["x"], 0 if s["mode"] == "token" else 32)
        return ops.expert_gemm_fanout(s["packed"], a, route, TYPES[s["out"]],
                                      sorted_rows=s["sorted"], outs=s["outs"])
    return ops.adapter_add(s["y"], s["x"], ops.Adapters(s["a"], s["b"], s["scale"]), route, out=s["out"])


def _summed(rows, position, weights, dtype):
    """sum_j weights[t, j] rows[position[t, j]], in 32 bits, rounded once."""
    at = position.long()
    picked = torch.where((at >= 0)[..., None], rows.float()[at.clamp(min=0)], 0.0)
    return (picked * weights[..., None]).sum(1).to(dtype)


def _codes(x, block):
    """The quantized values (codes times scale) of each row: absmax / 127 per row or per block of 32."""
    T, K = x.shape
    v = x.float().view(T, -1, block or K)
    top = v.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / torch.full_like(top, 127.0), torch.ones_like(top))
    return ((v / scale).round().clamp(-127, 127) * scale).view(T, K)


def _weights(codes, bits, group, mode):
    """The values of a weight's codes, in 32 bits."""
    rows, K = codes.shape
    c = codes.float().view(rows, -1, group)
    if mode == "block":
        zero = ((bits & 15) ^ 8) - 8
        return ((c - zero[..., None]) * (bits & -16).view(torch.float16).float()[..., None]).view(rows, K)
    return (c * bits.view(torch.float16).float()[..., None]).view(rows, K)


def _plain(s):
    T, k = s["T"], s.get("k", 1)
    if s["op"] == "route":
        offsets, order, position = _plan(s["ids"], s["groups"])
        live = torch.arange(T * k, device="cuda") < offsets[-1]
        rows = torch.where(live[:, None], s["x"][order.long() // k], s["out"])
        return {"offsets": offsets, "order": order, "position": position, "rows": rows,
                "y": _summed(s["rows"], position, s["weights"], s["rows"].dtype)}
    offsets, order, position = s["plan"]
    slot, at = order.long(), torch.arange(T * k, device="cuda")
    live = at < offsets[-1]
    token = slot // k
    if s["op"] == "grad":
        dy, dt = s["dy"].float(), s["rows"].dtype
        drows = torch.where(live[:, None], (s["weights"].reshape(-1)[slot][:, None] * dy[token]).to(dt), s["out"])
        dots = torch.zeros(T * k, device="cuda")
        dots[slot] = torch.where(live, (dy[token] * s["rows"].float()).sum(1), 0.0)
        ones = torch.ones_like(s["weights"])
        return {"drows": drows, "dweights": dots.view(T, k), "dx": _summed(s["drows"], position, ones, dt)}
    if s["op"] == "expert":
        # each expert's rows, padded to the most of one; the place behind them takes the rows without an expert
        most = max(s["most"], 1)
        group = (at[:, None] >= offsets[None, 1:]).sum(1).clamp(max=s["groups"] - 1)
        place = torch.where(live, group * most + at - offsets[group], s["groups"] * most)
        x = _codes(s["x"], 0 if s["mode"] == "token" else 32)
        padded = torch.zeros(s["groups"] * most + 1, s["K"], device="cuda")
        padded[place] = x if s["sorted"] else x[token]
        padded = padded[:-1].view(s["groups"], most, s["K"])
        ys = []
        for codes, bits, out in zip(s["codes"], s["scales"], s["outs"]):
            w = _weights(codes, bits, s["group"], s["mode"]).view(s["groups"], -1, s["K"]).transpose(1, 2).contiguous()
            y = torch.bmm(padded, w).view(s["groups"] * most, -1)[place.clamp(max=s["groups"] * most - 1)]
            ys.append(torch.where(live[:, None], y.to(out.dtype), out))
        return ys
    # adapters: x through all of them, what is not its own masked out
    n, r = s["n"], s["r"]
    low = s["x"].float() @ s["a"].float().view(n * r, -1).t()
    mine = s["ids"] == torch.arange(n, device="cuda")
    low = torch.where(mine[..., None], low.view(-1, n, r) * s["scale"][:, None], 0.0).view(-1, n * r)
    return (s["y"].float() + low @ s["b"].float().transpose(1, 2).reshape(n * r, -1)).to(s["y"].dtype)


def _touched(groups, slots, drop):
    """Groups that have a row, expected for slots spread evenly."""
    return groups * (1.0 - (1.0 - 1.0 / groups) ** max(1.0, slots * (1 - drop)))


def work(case):
    T, drop = case["T"], case["drop"]
    if case["op"] in ("route", "grad"):
        N, H, b = T * case["k"], case["H"], BYTES[case["x"]]
        live = N * (1 - drop)
        if case["op"] == "route":
            return {"bytes": 16 * N + 4 * case["E"] + b * H * (2 * T + 2 * live), "flops": 2 * live * H}
        return {"bytes": 12 * N + b * H * (2 * T + 3 * live), "flops": 4 * live * H}
    if case["op"] == "expert":
        N, K = T * case["k"] * (1 - drop), case["K"]
        M = sum(int(m) for m in case["rows"].split(","))
        code = (1.0 if case["mode"] == "w8" else 0.5) + 2.0 / case["group"]
        return {"bytes": _touched(case["E"], T * case["k"], drop) * M * K * code +
                (N if case["sorted"] else T) * K * BYTES[case["x"]] + N * M * BYTES[case["out"]], "flops": 2 * N * M * K}
    K, M, r = case["K"], case["M"], case["r"]
    used = _touched(case["n"], len(case["seg"].split(",")) if case["seg"] else T, drop)
    live = T * (1 - drop)
    return {"bytes": 2 * used * r * (K + M) + live * K * BYTES[case["x"]] + 2 * T * M * BYTES[case["y"]],
            "flops": 2 * live * r * (K + M)}


def exact(case, seed):
    d = _inputs(case, seed)
    T, k = case["T"], case.get("k", 1)
    groups = case["n"] if case["op"] == "adapter" else case["E"]
    ids = d["ids"].cpu().reshape(-1).tolist()
    members = [[] for _ in range(groups)]
    for slot, e in enumerate(ids):
        if 0 <= e < groups:
            members[e].append(slot)
    line = [slot for m in members for slot in m]                 # slots with a group, in sorted order
    slots = torch.tensor(line, dtype=torch.long, device="cuda")
    n = len(line)
    if case["op"] in ("route", "grad"):
        H = case["H"]
        w = d["weights"].double().reshape(-1)[slots]
        if case["op"] == "route":
            rows = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
            rows[:n] = d["x"].double()[slots // k]
            y = torch.zeros(T, H, dtype=torch.float64, device="cuda")
            y.index_add_(0, slots // k, d["rows"][:n].double() * w[:, None])
            return {"offsets": None, "order": None, "position": None, "rows": rows, "y": y}
        drows = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
        drows[:n] = d["dy"].double()[slots // k] * w[:, None]
        dots = torch.zeros(T * k, dtype=torch.float64, device="cuda")
        dots[slots] = torch.linalg.vecdot(d["dy"].double()[slots // k], d["rows"][:n].double())
        dx = torch.zeros(T, H, dtype=torch.float64, device="cuda")
        dx.index_add_(0, slots // k, d["drows"][:n].double())
        return {"drows": drows, "dweights": dots.view(T, k), "dx": dx}
    if case["op"] == "expert":
        K, group = case["K"], case["group"]
        # the codes are defined in float32 (scale absmax / 127, quotients rounded to the nearest even)
        x, span = d["x"].float(), K if case["mode"] == "token" else 32
        parts = x.reshape(-1, span)
        scale = parts.abs().max(1).values.div(torch.tensor(127.0, device="cuda").expand(parts.shape[0]))
        scale[scale == 0] = 1.0
        q = torch.round(parts.div(scale[:, None])).clamp(-127, 127).double().mul(scale.double()[:, None]).reshape(-1, K)
        ys = []
        for codes, bits in zip(d["codes"], d["scales"]):
            M = codes.shape[0] // groups
            y = torch.zeros(T * k, M, dtype=torch.float64, device="cuda")
            p = 0
            for e, m in enumerate(members):
                if not m:
                    continue
                c = codes[e * M:(e + 1) * M].double()
                b = bits[e * M:(e + 1) * M]
                if case["mode"] == "block":
                    z = (b & 15).double()
                    c = c - torch.where(z > 7, z - 16, z).repeat_interleave(group, 1)
                    b = b & ~15
                c = c * b.view(torch.float16).double().repeat_interleave(group, 1)
                which = torch.arange(p, p + len(m), device="cuda") if case["sorted"] else torch.tensor(m, device="cuda") // k
                y[p:p + len(m)] = q[which] @ c.t().contiguous()
                p += len(m)
            ys.append(y)
        return ys
    out = d["y"].double()
    for e, m in enumerate(members):
        if m:
            at = torch.tensor(m, device="cuda")
            low = d["x"][at].double() @ d["a"][e].double().t().contiguous()
            out[at] += d["scale"][e].double() * (low @ d["b"][e].double().t().contiguous())
    return out
