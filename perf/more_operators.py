"""Products with weights in 8-bit floating point (e4m3, a scale for each block of 128 x 128), for one weight and by expert,
and their gradients.

A case is one call of an operator as a serving or training program makes it. `op` says which:
  gemm      x [T][K] quantized (a scale for each row and block of 128 columns) and projected by one or two weights that
            share it, of `rows` output rows each
  expert    the same by each row's expert, of k for each token; `sorted`: x already lies in the plan's order, as a down
            projection finds it
  grad      a training step's gradients of one projection, dense or (E > 0) by expert: of x, from the quantized dy and
            the transposed weight, and of the weight, from the rows of dy and x as they are
`drop` is the share of slots that carry no expert (rows whose expert lives on another GPU).
"""
import math

import torch

own = False

HIDDEN, INTER = 5120, 17408
BYTES = {"bf16": 2, "f32": 4}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 128


def _gemm(T, K, rows, x="bf16", out="bf16"):
    return {"op": "gemm", "T": T, "K": K, "rows": rows, "x": x, "out": out}


def _expert(T, k, E, K, rows, x="bf16", out="bf16", in_order=False, drop=0.0):
    return {"op": "expert", "T": T, "k": k, "E": E, "K": K, "rows": rows, "x": x, "out": out, "sorted": in_order,
            "drop": drop}


def _grad(T, k, E, K, rows, out="f32", drop=0.0):
    return {"op": "grad", "T": T, "k": k, "E": E, "K": K, "rows": rows, "out": out, "drop": drop}


def listed():
    return [
        # one sequence: a square projection, float32 in and out: latency
        dict(_gemm(1, 4096, "4096", "f32", "f32"), name="gemm_decode1"),
        # a decode step of eight sequences: gate and up
        dict(_gemm(8, HIDDEN, "%d,%d" % (INTER, INTER)), name="gemm_gate_up_decode8"),
        # a short prompt, odd throughout: the last blocks of both sides are not whole
        dict(_gemm(97, 1456, "2064", "f32", "f32"), name="gemm_odd97"),
        # a prompt of 512 tokens through the down projection
        dict(_gemm(512, INTER, "%d" % HIDDEN), name="gemm_down512"),
        # six prompts packed into one prefill: gate and up
        dict(_gemm(3965, HIDDEN, "%d,%d" % (INTER, INTER)), name="gemm_gate_up_packed"),
        # one sequence: the down projections of its four experts
        dict(_expert(1, 4, 32, 1024, "5120", "f32", "f32", in_order=True), name="expert_down_decode1"),
        # a decode step of 16 sequences: gate and up of up to 64 experts
        dict(_expert(16, 8, 64, HIDDEN, "1024,1024"), name="expert_gate_up_decode16"),
        # a prompt of 300 tokens, half of the experts on another GPU
        dict(_expert(300, 6, 40, 2048, "1408", out="f32", drop=0.5), name="expert_prompt300"),
        # a prefill chunk: gate and up of 64 experts
        dict(_expert(2048, 8, 64, HIDDEN, "1024,1024"), name="expert_gate_up_prefill"),
        # a training step's share of a batch through a square projection
        dict(_grad(2048, 1, 0, HIDDEN, "%d" % HIDDEN), name="grad_dense2048"),
        # the same by expert: two experts a token
        dict(_grad(4093, 2, 16, 2048, "1024", "bf16"), name="grad_top2"),
        # a small one, odd throughout, a quarter of the experts on another GPU: latency
        dict(_grad(150, 3, 5, 336, "208", "f32", 0.25), name="grad_odd150"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def size(lo, hi):                            # rows and columns come in multiples of 16, mostly of 128
        step = rng.choice([128, 128, 128, 16])
        return max(step, spread(lo, hi) // step * step)

    op = rng.choice(["gemm", "expert", "grad"])
    drop = rng.choice([0.0, 0.0, 0.1, 0.5])
    x, out = rng.choice(["bf16", "f32"]), rng.choice(["bf16", "f32"])
    if op == "gemm":
        K, M = size(256, INTER), size(256, INTER)
        rows = rng.choice(["%d" % M, "%d,%d" % (M, M)]) if M <= 8192 else "%d" % M
        return _gemm(spread(1, 3965), K, rows, x, out)
    if op == "expert":
        k, E = rng.choice([1, 2, 4, 8]), rng.choice([8, 16, 32, 40, 64])
        K, M = size(256, 5120), size(64, 2048)
        rows = rng.choice(["%d" % M, "%d,%d" % (M, M)]) if M <= 1024 else "%d" % M
        return _expert(spread(1, 2048), k, E, K, rows, x, out, rng.random() < 0.3, drop)
    if rng.random() < 0.4:
        return _grad(spread(1, 4096), 1, 0, size(128, 5120), "%d" % size(128, 5120), out)
    k, E = rng.choice([1, 2, 4]), rng.choice([4, 8, 16, 32])
    return _grad(spread(1, 8192 // k), k, E, size(128, 2048), "%d" % size(128, 2048), out, drop)


def _ids(case, gen):
    """The k experts of each token, of uneven popularity; -1 for a dropped slot."""
    T, k, E = case["T"], case["k"], case["E"]
    popular = torch.randn(E, generator=gen, device="cuda") * 0.5
    ids = (popular + torch.randn(T, E, generator=gen, device="cuda")).topk(k, dim=1).indices.to(torch.int32)
    gone = torch.rand(T, k, generator=gen, device="cuda") < case["drop"]
    return torch.where(gone, torch.full_like(ids, -1), ids).contiguous()


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _weight(E, M, K, gen):
    """e4m3 codes [E][M][K] of normal weights and the scale of each 128 x 128 block."""
    mb, kb = _blocks(M), _blocks(K)
    codes = torch.empty(E, M, K, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(E, mb, kb, device="cuda")
    for e in range(E):
        w = torch.randn(M, K, generator=gen, device="cuda") / math.sqrt(K)
        padded = torch.zeros(mb * BLOCK, kb * BLOCK, device="cuda")
        padded[:M, :K] = w
        scales[e] = padded.view(mb, BLOCK, kb, BLOCK).abs().amax((1, 3)) / 448.0
        codes[e] = (w / scales[e].repeat_interleave(BLOCK, 0)[:M].repeat_interleave(BLOCK, 1)[:, :K]).to(codes.dtype)
    return codes, scales


def _inputs(case, seed):
    """The seeded inputs of a case, as tensors on the GPU."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def normal(*shape, dtype="bf16"):
        return torch.randn(*shape, generator=gen, device="cuda").to(TYPES[dtype])

    d = {}
    T, K, k, E = case["T"], case["K"], case.get("k", 1), case.get("E", 0)
    if E:
        d["ids"] = _ids(case, gen)
    rows = [int(m) for m in case["rows"].split(",")]
    if case["op"] == "grad":
        d["x"], d["dy"] = normal(T * k, K), normal(T * k, rows[0])
    else:
        d["x"] = normal(T * k if case.get("sorted") else T, K, dtype=case["x"])
    d["weights"] = [_weight(max(E, 1), m, K, gen) for m in rows]
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
    T, k, E, K = case["T"], case.get("k", 1), case.get("E", 0), case["K"]
    rows = [int(m) for m in case["rows"].split(",")]
    if E:
        # the step's plan, which its layers and its backward pass share
        s["plan"] = _plan(s["ids"], E)
        # (the most rows of one expert; the plain form pads to it)
        s["most"] = int((s["plan"][0][1:] - s["plan"][0][:-1]).max())
    N = T * k
    if case["op"] == "grad":
        s["dx"] = torch.zeros(N, K, dtype=s["x"].dtype, device="cuda")
    else:
        s["outs"] = [torch.zeros(N, m, dtype=TYPES[case["out"]], device="cuda") for m in rows]
    if own:                                      # the packed weights that a program keeps
        from knivesysl_xe_amd import ops
        s["packed"] = [ops.F8Weight.from_codes(c if E else c[0], b if E else b[0]) for c, b in s["weights"]]
        if case["op"] == "grad":
            s["packed"] = [w.transposed() for w in s["packed"]]
    return s


def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from knivesysl_xe_amd import ops
    E = s.get("E", 0)
    route = ops.RowRoute(s["T"], s["k"], E, *s["plan"]) if E else None
    if s["op"] == "gemm":
        return ops.gemm_f8_fanout(s["packed"], s["x"], TYPES[s["out"]], outs=s["outs"])
    if s["op"] == "expert":
        return ops.expert_gemm_f8_fanout(s["packed"], s["x"], route, TYPES[s["out"]], sorted_rows=s["sorted"],
                                         outs=s["outs"])
    dtype = TYPES[s["out"]]
    if E:
        dx = ops.expert_gemm_f8(s["packed"][0], s["dy"], route, s["dx"].dtype, sorted_rows=True, out=s["dx"])
        return {"dx": dx, "dw": ops.expert_grad_weight(s["dy"], s["x"], route, dtype)}
    dx = ops.gemm_f8(s["packed"][0], s["dy"], s["dx"].dtype, out=s["dx"])
    return {"dx": dx, "dw": ops.grad_weight(s["dy"], s["x"], dtype)}


def _quantized(x):
    """The values (codes times scale) of the rows' e4m3 codes, a scale for each row and block of 128 columns."""
    T, K = x.shape
    kb = _blocks(K)
    v = torch.zeros(T, kb * BLOCK, device=x.device)
    v[:, :K] = x.float()
    v = v.view(T, kb, BLOCK)
    top = v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    most = torch.full_like(top, 448.0)
    return ((v * (most / top)).to(torch.float8_e4m3fn).float() * (top / most)).view(T, -1)[:, :K]


def _values(codes, scales):
    """The values of a weight's codes, in 32 bits: [E][M][K]."""
    M, K = codes.shape[1:]
    w = codes.float()
    return w * scales.repeat_interleave(BLOCK, 1)[:, :M].repeat_interleave(BLOCK, 2)[:, :, :K]


def _spread(s, rows, place, E, most):
    """Sorted rows, padded to the most of one expert: [E][most][columns]."""
    padded = torch.zeros(E * most + 1, rows.shape[1], device="cuda")
    padded[place] = rows
    return padded[:-1].view(E, most, -1)


def _plain(s):
    E, T, k = s.get("E", 0), s["T"], s.get("k", 1)
    if not E:
        if s["op"] == "gemm":
            x = _quantized(s["x"])
            return [(x @ _values(c, b)[0].t()).to(o.dtype) for (c, b), o in zip(s["weights"], s["outs"])]
        w = _values(*s["weights"][0])[0]
        dw = s["dy"].float().t() @ s["x"].float()
        return {"dx": (_quantized(s["dy"]) @ w).to(s["x"].dtype), "dw": dw.to(TYPES[s["out"]])}
    offsets, order, _ = s["plan"]
    at = torch.arange(T * k, device="cuda")
    live = at < offsets[-1]
    # each expert's rows, padded to the most of one; the place behind them takes the rows without an expert
    most = max(s["most"], 1)
    group = (at[:, None] >= offsets[None, 1:]).sum(1).clamp(max=E - 1)
    place = torch.where(live, group * most + at - offsets[group], E * most)
    back = place.clamp(max=E * most - 1)
    if s["op"] == "expert":
        x = _quantized(s["x"])
        padded = _spread(s, x if s["sorted"] else x[order.long() // k], place, E, most)
        ys = []
        for (c, b), out in zip(s["weights"], s["outs"]):
            y = torch.bmm(padded, _values(c, b).transpose(1, 2).contiguous()).view(E * most, -1)[back]
            ys.append(torch.where(live[:, None], y.to(out.dtype), out))
        return ys
    w = _values(*s["weights"][0])
    dx = torch.bmm(_spread(s, _quantized(s["dy"]), place, E, most), w).view(E * most, -1)[back]
    dy = _spread(s, s["dy"].float(), place, E, most).transpose(1, 2).contiguous()
    dw = torch.bmm(dy, _spread(s, s["x"].float(), place, E, most))
    return {"dx": torch.where(live[:, None], dx.to(s["x"].dtype), s["dx"]), "dw": dw.to(TYPES[s["out"]])}


def _touched(groups, slots, drop):
    """Groups that have a row, expected for slots spread evenly."""
    return groups * (1.0 - (1.0 - 1.0 / groups) ** max(1.0, slots * (1 - drop)))


def work(case):
    T, K, k, E, drop = case["T"], case["K"], case.get("k", 1), case.get("E", 0), case.get("drop", 0.0)
    M = sum(int(m) for m in case["rows"].split(","))
    N = T * k * (1 - drop)
    weight = (_touched(E, T * k, drop) if E else 1) * M * K * (1 + 4.0 / BLOCK ** 2)
    if case["op"] == "grad":
        return {"bytes": weight + 2 * N * (2 * K + M) + max(E, 1) * M * K * BYTES[case["out"]], "flops": 4 * N * M * K}
    read = T * k if case.get("sorted") else T
    return {"bytes": weight + read * K * BYTES[case["x"]] + N * M * BYTES[case["out"]], "flops": 2 * N * M * K}


def exact(case, seed):
    d = _inputs(case, seed)
    T, K, k, E = case["T"], case["K"], case.get("k", 1), case.get("E", 0)
    N = T * k

    def codes_of(rows):
        # the codes are defined in float32: scale max / 448, products with 448 / max rounded to the nearest e4m3
        out = torch.zeros(rows.shape, dtype=torch.float64, device="cuda")
        for j in range(0, rows.shape[1], BLOCK):
            part = rows[:, j:j + BLOCK].float()
            top = torch.maximum(part.abs().max(1).values, torch.tensor(2.0 ** -100, device="cuda"))
            up = torch.tensor(448.0, device="cuda").expand_as(top).div(top)
            down = top.div(torch.tensor(448.0, device="cuda").expand_as(top))
            out[:, j:j + BLOCK] = part.mul(up[:, None]).to(torch.float8_e4m3fn).double() * down.double()[:, None]
        return out

    def weight_of(pair, e):
        codes, scales = pair[0][e].double(), pair[1][e].double()
        for i in range(scales.shape[0]):
            for j in range(scales.shape[1]):
                codes[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= scales[i, j]
        return codes

    # the rows of each expert: the sorted place of its first, and their slots
    if E:
        flat = d["ids"].cpu().reshape(-1).tolist()
        members = [[] for _ in range(E)]
        for slot, e in enumerate(flat):
            if 0 <= e < E:
                members[e].append(slot)
    else:
        members = [list(range(N))]
    runs, p = [], 0
    for m in members:
        runs.append((p, torch.tensor(m, dtype=torch.long, device="cuda")))
        p += len(m)
    if case["op"] == "grad":
        dx = torch.zeros(N, K, dtype=torch.float64, device="cuda")
        dw = torch.zeros(max(E, 1), int(case["rows"]), K, dtype=torch.float64, device="cuda")
        back = codes_of(d["dy"])
        for e, (p, m) in enumerate(runs):
            at = slice(p, p + len(m))
            if len(m):
                dx[at] = back[at] @ weight_of(d["weights"][0], e)
                dw[e] = d["dy"][at].double().t().contiguous() @ d["x"][at].double()
        return {"dx": dx, "dw": dw if E else dw[0]}
    x = codes_of(d["x"])
    ys = []
    for pair in d["weights"]:
        y = torch.zeros(N, pair[0].shape[1], dtype=torch.float64, device="cuda")
        for e, (p, m) in enumerate(runs):
            if len(m):
                rows = x if not E else x[p:p + len(m)] if case["sorted"] else x[m // k]
                y[p:p + len(m)] = rows @ weight_of(pair, e).t().contiguous()
        ys.append(y)
    return ys
