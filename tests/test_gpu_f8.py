"""The 8-bit floating tier on the GPU against 64-bit references: quantizer, weight layouts, products dense and by
expert, at the sizes and masks where they can go wrong."""
import pytest
import torch

from knivesysl_xe_amd import ops
from f8_ref import (BF16, F32, F8, blocks, bound, exact_rows, exact_weight, expand, gen, members, normal_weight, quantized,
                          row_values, weight_values)

pytestmark = pytest.mark.gpu


# ---- quantizer -------------------------------------------------------------

def codes_of(a):
    return a.q.view(F8)[:, :a.K]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K", [(1, 16), (1, 128), (3, 144), (17, 1456), (300, 5120), (2048, 2048), (5, 17408)])
def test_quantizer_bits(T, K, dtype):
    x = (torch.randn(T, K, generator=gen(T + K), device="cuda") * 3).to(dtype)
    x[0, :16] = 0.0
    a = ops.quantize_act_f8(x)
    q, s = quantized(x)
    assert torch.equal(a.scale, s)
    assert torch.equal(codes_of(a).view(torch.uint8), q.view(torch.uint8))
    assert not a.q[:, K:].any()                              # columns past K are zero codes


def test_quantizer_rounds_every_bf16_as_torch_does():
    bits = torch.arange(0, 0x7F80, dtype=torch.int32, device="cuda").to(torch.int16)     # every finite bf16 >= 0
    v = bits.view(BF16)
    x = torch.stack([v, -v], 1).reshape(-1)
    x = x[torch.randperm(x.numel(), generator=gen(1), device="cuda")][: x.numel() // 128 * 128].view(-1, 128).contiguous()
    x = torch.cat([x, torch.sort(v.view(-1, 128), 1).values])
    a = ops.quantize_act_f8(x)
    q, s = quantized(x)
    assert torch.equal(a.scale, s)
    assert torch.equal(codes_of(a).view(torch.uint8), q.view(torch.uint8))


def test_quantizer_of_zeros_and_small_blocks():
    x = torch.zeros(4, 256, device="cuda")
    x[1, 5] = 2.0 ** -110                                    # below the floor: a code of zero
    x[2, 130] = 2.0 ** -100
    a = ops.quantize_act_f8(x)
    assert torch.isfinite(a.scale).all() and (a.scale > 0).all()
    assert torch.equal(codes_of(a).view(torch.uint8), quantized(x)[0].view(torch.uint8))
    assert codes_of(a)[2, 130].float() == 448.0


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("T,dtype", [(4, F32), (4, BF16), (300, F32), (300, BF16)])
def test_rows_that_are_not_finite_make_their_outputs_nan_alone(bad, T, dtype):
    codes, scales = normal_weight(1, 160, 256, 3)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = torch.randn(T, 256, generator=gen(5), device="cuda").to(dtype)
    clean = ops.gemm_f8(w, x, dtype)
    x[2, 200] = bad
    y = ops.gemm_f8(w, x, dtype)
    assert y[2].isnan().all()
    keep = torch.arange(T, device="cuda") != 2
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K", [(1, 16), (3, 1456), (129, 1024)])
def test_silu_mul_quantizer(T, K, dtype):
    g = (torch.randn(T, K, generator=gen(1), device="cuda") * 2).to(dtype)
    u = torch.randn(T, K, generator=gen(2), device="cuda").to(dtype)
    hidden, a = ops.silu_mul_quant_f8(g, u)
    want = g.double() / (1 + torch.exp(-g.double())) * u.double()
    # exp of at most |g| < 16 off by a few units, 1 + e, the quotient and the product: four roundings and exp's 2^-21
    assert ((hidden.double() - want).abs() <= want.abs() * 2.0 ** -20).all()
    # (its values are quantized by the rule: the values it wrote give the same codes)
    q, s = quantized(hidden)
    assert torch.equal(a.scale, s) and torch.equal(codes_of(a).view(torch.uint8), q.view(torch.uint8))
    none, b = ops.silu_mul_quant_f8(g, u, keep_hidden=False)
    assert none is None and torch.equal(b.q, a.q) and torch.equal(b.scale, a.scale)


# ---- weights ---------------------------------------------------------------

@pytest.mark.parametrize("groups,M,K", [(1, 16, 16), (1, 128, 128), (3, 208, 336), (2, 144, 1024), (1, 5120, 2048)])
def test_weights_pack_unpack_transpose(groups, M, K):
    bits = torch.randint(0, 256, (groups, M, K), generator=gen(M + K), device="cuda", dtype=torch.uint8)
    scales = torch.rand(groups, blocks(M), blocks(K), generator=gen(7), device="cuda") + 0.5
    w = ops.F8Weight.from_codes(bits, scales)
    codes, s = w.unpack()
    assert torch.equal(codes.view(torch.uint8), bits) and torch.equal(s, scales)
    t, ts = w.transposed().unpack()
    assert torch.equal(t.view(torch.uint8), bits.transpose(1, 2)) and torch.equal(ts, scales.transpose(1, 2))
    back = w.transposed().transposed()
    assert torch.equal(back.codes, w.codes) and torch.equal(back.scales, w.scales)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("groups,M,K", [(1, 16, 16), (2, 208, 336), (1, 1024, 768)])
def test_weights_quantized(groups, M, K, dtype):
    w = torch.randn(groups, M, K, generator=gen(M), device="cuda").to(dtype)
    w[0, :16, :16] = 0.0
    got = ops.F8Weight.quantize(w)
    padded = torch.zeros(groups, blocks(M) * 128, blocks(K) * 128, device="cuda")
    padded[:, :M, :K] = w.float()
    top = padded.view(groups, blocks(M), 128, blocks(K), 128).abs().amax((2, 4)).clamp(min=2.0 ** -100)
    assert torch.equal(got.scales, top / torch.full_like(top, 448.0))
    codes = (w.float() * expand(torch.full_like(top, 448.0) / top, M, K)).to(F8)
    assert torch.equal(got.unpack()[0].view(torch.uint8), codes.view(torch.uint8))
    again = ops.F8Weight.quantize(w.neg(), out=got)
    assert again is got and torch.equal(got.unpack()[0].float(), -codes.float())


# ---- products --------------------------------------------------------------

SIZES = [(1, 16, 16), (1, 4096, 1024), (2, 144, 128), (7, 1456, 2064), (16, 5120, 256), (17, 128, 144), (31, 640, 1040),
         (33, 272, 528), (64, 384, 320), (65, 2048, 16), (129, 16, 2064), (257, 1152, 272), (300, 5120, 640), (515, 400, 912)]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,K,M", SIZES)
def test_product_exactly(T, K, M, out):
    codes, scales = exact_weight(1, M, K, T + M)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    for dtype in (F32, BF16):
        x = exact_rows(T, K, K, dtype)
        want = (x.double() @ weight_values(codes, scales)[0].t().contiguous()).to(out)
        assert torch.equal(ops.gemm_f8(w, x, out), want)
        assert torch.equal(ops.gemm_f8(w, ops.quantize_act_f8(x), out), want)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,K,M", [(1, 5120, 512), (16, 2048, 1040), (40, 1456, 272), (200, 4096, 384), (700, 640, 2064)])
def test_product_of_normal_values(T, K, M, out):
    codes, scales = normal_weight(1, M, K, T + M)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = torch.randn(T, K, generator=gen(K), device="cuda")
    xv, wv = row_values(x), weight_values(codes, scales)[0]
    want = xv @ wv.t().contiguous()
    y = ops.gemm_f8(w, x, out)
    assert ((y.double() - want).abs() <= bound(xv, wv, want, out, False)).all()
    residual = torch.randn(T, M, generator=gen(9), device="cuda")
    z = ops.gemm_f8(w, x, out, residual=residual)
    # (one more addition, rounded to float32 before the output's rounding)
    want = want + residual.double()
    assert ((z.double() - want).abs() <= bound(xv, wv, want, out, False) + want.abs() * 2.0 ** -23).all()


def test_the_matrix_cores_cut_stays_within_its_bound():
    # one large product among seven small ones of each eight columns: the worst of the cut that bf16 outputs allow
    T, K, M = 256, 512, 256
    codes = torch.full((M, K), 1.125, device="cuda")
    codes[:, ::8] = 448.0
    x = torch.full((T, K), 1.875, device="cuda")
    x[:, ::8] = 448.0
    x[:, ::16] = -448.0                                      # the large products cancel
    w = ops.F8Weight.from_codes(codes.to(F8), torch.ones(blocks(M), blocks(K), device="cuda"))
    xv, wv = row_values(x), codes.double()
    want = xv @ wv.t().contiguous()
    for out in (F32, BF16):
        assert ((ops.gemm_f8(w, x, out).double() - want).abs() <= bound(xv, wv, want, out, False)).all()


def test_fanout_gives_each_weights_product():
    for T in (1, 9, 40, 300):
        ws = [ops.F8Weight.from_codes(*[t[0] for t in exact_weight(1, M, 656, M)]) for M in (272, 16, 1040, 128)]
        x = exact_rows(T, 656, T)
        for out in (F32, BF16):
            ys = ops.gemm_f8_fanout(ws, x, out)
            for w, y in zip(ws, ys):
                assert torch.equal(y, ops.gemm_f8(w, x, out))


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,K,Ms", [(1100, 144, (16400,)), (2600, 16, (4112, 4240)), (1025, 528, (8192, 8208)), (70000, 128, (272,))])
def test_products_of_more_tiles_than_work_groups(T, K, Ms, out):
    # (a work-group takes several tiles, one after another, of either weight)
    cs = [exact_weight(1, M, K, M) for M in Ms]
    ws = [ops.F8Weight.from_codes(c[0], s[0]) for c, s in cs]
    x = exact_rows(T, K, T)
    for y, c in zip(ops.gemm_f8_fanout(ws, x, out), cs):
        want = torch.empty_like(y)
        wt = weight_values(*c)[0].t().contiguous()
        for t in range(0, T, 8192):
            want[t:t + 8192] = (x[t:t + 8192].double() @ wt).to(out)
        assert torch.equal(y, want)


def test_products_of_no_rows():
    codes, scales = normal_weight(1, 64, 128, 1)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    assert ops.gemm_f8(w, torch.empty(0, 128, device="cuda")).shape == (0, 64)
    assert ops.quantize_act_f8(torch.empty(0, 128, device="cuda")).q.shape == (0, 128)
    route = ops.route_rows(torch.empty(0, 2, dtype=torch.int32, device="cuda"), 1)
    assert ops.expert_gemm_f8(w, torch.empty(0, 128, device="cuda"), route).shape == (0, 64)


# ---- by expert -------------------------------------------------------------

def ids_of(T, k, E, drop, seed, skew=0.0):
    g = gen(seed)
    score = torch.randn(T, E, generator=g, device="cuda") + skew * torch.randn(E, generator=g, device="cuda")
    ids = score.topk(k, 1).indices.to(torch.int32)
    gone = torch.rand(T, k, generator=g, device="cuda") < drop
    return torch.where(gone, -1, ids).to(torch.int32).contiguous()


EXPERTS = [(1, 1, 1, 128, 16, 0.0), (1, 4, 32, 1024, 272, 0.0), (16, 8, 64, 640, 144, 0.0), (5, 2, 3, 144, 128, 1.0),
           (40, 2, 5, 336, 208, 0.3), (300, 6, 40, 256, 320, 0.5), (500, 4, 4, 528, 272, 0.1), (700, 2, 70, 128, 144, 0.0),
           (1024, 8, 8, 384, 512, 0.0)]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,k,E,K,M,drop", EXPERTS)
def test_expert_product_exactly(T, k, E, K, M, drop, out):
    codes, scales = exact_weight(E, M, K, T + M)
    w = ops.F8Weight.from_codes(codes, scales)
    wv = weight_values(codes, scales)
    ids = ids_of(T, k, E, drop, T, skew=1.0)
    route = ops.route_rows(ids, E)
    rows = members(ids, E)
    line = torch.tensor([s for m in rows for s in m], dtype=torch.long, device="cuda")
    for in_order in (False, True):
        x = exact_rows(T * k if in_order else T, K, K, BF16 if in_order else F32)
        want = torch.full((T * k, M), -7.0, dtype=out, device="cuda")
        p = 0
        for e, m in enumerate(rows):
            if m:
                xe = x[p:p + len(m)] if in_order else x[line[p:p + len(m)] // k]
                want[p:p + len(m)] = (xe.double() @ wv[e].t().contiguous()).to(out)
                p += len(m)
        y = torch.full((T * k, M), -7.0, dtype=out, device="cuda")
        # (rows behind the last expert's stay as they were)
        assert ops.expert_gemm_f8(w, x, route, out, sorted_rows=in_order, out=y) is y
        assert torch.equal(y, want)
        y.fill_(-7.0)
        ops.expert_gemm_f8(w, ops.quantize_act_f8(x), route, out, sorted_rows=in_order, out=y)
        assert torch.equal(y, want)


def test_one_expert_takes_all_rows_and_a_token_names_it_twice():
    codes, scales = exact_weight(6, 144, 256, 1)
    w = ops.F8Weight.from_codes(codes, scales)
    ids = torch.full((130, 2), 4, dtype=torch.int64, device="cuda")
    route = ops.route_rows(ids, 6)
    x = exact_rows(130, 256, 2)
    y = ops.expert_gemm_f8(w, x, route)
    want = (x.double() @ weight_values(codes, scales)[4].t().contiguous()).float().repeat_interleave(2, 0)
    assert torch.equal(y, want)


def test_expert_fanout_gives_each_weights_product():
    E, K = 9, 400
    ws = [ops.F8Weight.from_codes(*exact_weight(E, M, K, M)) for M in (272, 144)]
    for T, k in ((3, 2), (200, 4)):
        route = ops.route_rows(ids_of(T, k, E, 0.2, T), E)
        x = exact_rows(T, K, T)
        for out in (F32, BF16):
            a = [torch.zeros(T * k, w.M, dtype=out, device="cuda") for w in ws]
            ops.expert_gemm_f8_fanout(ws, x, route, out, outs=a)
            for w, y in zip(ws, a):
                assert torch.equal(y, ops.expert_gemm_f8(w, x, route, out, out=torch.zeros_like(y)))


# ---- streams, graphs -------------------------------------------------------

@pytest.mark.parametrize("T", [4, 200])
def test_products_replay_from_a_graph(T):
    E, K, M, k = 8, 384, 272, 2
    codes, scales = normal_weight(E, M, K, 1)
    w = ops.F8Weight.from_codes(codes, scales)
    one = ops.F8Weight.from_codes(codes[0], scales[0])
    x = torch.randn(T, K, generator=gen(1), device="cuda")
    ids = ids_of(T, k, E, 0.2, 3)
    out = torch.zeros(T * k, M, dtype=BF16, device="cuda")
    dense = torch.zeros(T, M, device="cuda")

    def step():
        route = ops.route_rows(ids, E)
        ops.expert_gemm_f8(w, x, route, BF16, out=out)
        ops.gemm_f8(one, x, out=dense)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(torch.randn(T, K, generator=gen(10 + i), device="cuda"))
        ids.copy_(ids_of(T, k, E, 0.2, 20 + i))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, got_dense = out.clone(), dense.clone()
        out.zero_()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(got_dense, dense)


def test_products_on_two_streams_at_once():
    codes, scales = normal_weight(1, 1024, 2048, 1)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    xs = [torch.randn(200, 2048, generator=gen(i), device="cuda") for i in range(2)]
    want = [ops.gemm_f8(w, x, BF16) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.gemm_f8(w, xs[i], BF16))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


# ---- the experts' MLP, as it is used ---------------------------------------

@pytest.mark.parametrize("T", [3, 150])
def test_an_experts_mlp(T):
    E, k, H, I = 6, 2, 384, 272
    cs = [normal_weight(E, *s, i) for i, s in enumerate([(I, H), (I, H), (H, I)])]
    gate, up, down = [ops.F8Weight.from_codes(*c) for c in cs]
    gv, uv, dv = [weight_values(*c) for c in cs]
    x = torch.randn(T, H, generator=gen(1), device="cuda")
    ids = ids_of(T, k, E, 0.2, 2)
    weights = torch.rand(T, k, generator=gen(3), device="cuda")
    route = ops.route_rows(ids, E)
    g, u = [torch.zeros(T * k, I, device="cuda") for _ in range(2)]
    ops.expert_gemm_f8_fanout([gate, up], x, route, outs=[g, u])
    hidden, h = ops.silu_mul_quant_f8(g, u)
    rows = ops.expert_gemm_f8(down, h, route, sorted_rows=True)
    y = ops.combine_rows(rows, route, weights)
    # each step from what the one before wrote, in 64 bits
    at, xv, hv = route.position.long(), row_values(x), row_values(hidden)
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for t in range(T):
        for j in range(k):
            e, p = int(ids[t, j]), int(at[t, j])
            if e < 0:
                continue
            for got, v in ((g, gv), (u, uv)):
                exact = v[e] @ xv[t]
                assert ((got[p].double() - exact).abs() <= bound(xv[t:t + 1], v[e], exact, F32, True)[0]).all()
            want[t] += weights[t, j].double() * (dv[e] @ hv[p])
            size[t] += weights[t, j].double() * (dv[e].abs() @ hv[p].abs())
    # the down product's bound (3 blocks: 138 additions), then a product and a sum of two in float32
    assert ((y.double() - want).abs() <= size * (145 * 2.0 ** -23)).all()
