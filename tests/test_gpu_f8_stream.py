"""Every instance of the 8-bit floating tier's kernel for few rows (f8_shapes.py: the shapes that reach them) against 64-bit
references: rows as codes and as values of both types, residuals, a replayed graph."""
import pytest
import torch

import f8_shapes as shapes
from knivesysl_xe_amd import ops
from f8_ref import BF16, F32, bound, exact_rows, exact_weight, gen, normal_weight, plan_of, row_values, weight_values
from test_gpu_f8 import ids_of
from test_gpu_f8_tiles import BAD, _card, each_expert, packed  # noqa: F401 (_card: the fixture)

pytestmark = pytest.mark.gpu

DENSE = [(T, K, Ms) for table in shapes.STREAM.values() for T, k, E, K, Ms in table if not E]
GROUPED = [(T, k, E, K, Ms) for table in shapes.STREAM.values() for T, k, E, K, Ms in table if E]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,K,Ms", DENSE)
def test_dense_products_exactly(T, K, Ms, out):
    cs = [exact_weight(1, M, K, T + M) for M in Ms]
    ws = [packed(*c) for c in cs]
    for dtype in (F32, BF16):
        x = exact_rows(T, K, K, dtype)
        wants = [x.double() @ weight_values(*c)[0].t().contiguous() for c in cs]
        for rows in (x, ops.quantize_act_f8(x)):
            assert all(torch.equal(y, want.to(out)) for y, want in zip(ops.gemm_f8_fanout(ws, rows, out), wants))
    # (whole numbers below 2^10: every sum stays exact in float32)
    r = torch.randint(-1000, 1000, (T, Ms[0]), generator=gen(1), device="cuda").float()
    want = (wants[0] + r.double()).to(F32)
    assert torch.equal(ops.gemm_f8(ws[0], x, out, residual=r), want.to(out))
    assert ops.gemm_f8(ws[0], x, residual=r, out=r) is r and torch.equal(r, want)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,k,E,K,Ms", GROUPED)
def test_grouped_products_exactly(T, k, E, K, Ms, out):
    cs = [exact_weight(E, M, K, T + M) for M in Ms]
    ws = [packed(*c, E) for c in cs]
    for drop, skew in ((0.0, 0.0), (0.3, 1.0)):
        route = plan_of(ids_of(T, k, E, drop, T, skew), E)
        line = route.order.long()
        for dtype, in_order in ((F32, False), (BF16, False), (F32, True), (BF16, True)):
            x = exact_rows(T * k if in_order else T, K, K, dtype)
            wants = [torch.full((T * k, M), -7.0, dtype=out, device="cuda") for M in Ms]
            for want, c in zip(wants, cs):
                wv = weight_values(*c)

                def fill(e, a, b):
                    want[a:b] = ((x[a:b] if in_order else x[line[a:b] // k]).double() @ wv[e].t().contiguous()).to(out)

                each_expert(route.offsets, fill)
            for rows in (x, ops.quantize_act_f8(x)):
                # (rows behind the last expert's stay as they were)
                ys = [torch.full_like(want, -7.0) for want in wants]
                ops.expert_gemm_f8_fanout(ws, rows, route, out, sorted_rows=in_order, outs=ys)
                assert all(torch.equal(y, want) for y, want in zip(ys, wants)), (drop, dtype, in_order)


@pytest.mark.parametrize("T,K,Ms", DENSE)
def test_dense_products_of_normal_values_are_exact_ones(T, K, Ms):
    # few rows: exact products and FP32 sums in either output type
    M = Ms[0]
    codes, scales = normal_weight(1, M, K, T + M)
    w, x = packed(codes, scales), torch.randn(T, K, generator=gen(K), device="cuda")
    xv, wv = row_values(x), weight_values(codes, scales)[0]
    want = xv @ wv.t().contiguous()
    for out in (F32, BF16):
        assert ((ops.gemm_f8(w, x, out).double() - want).abs() <= bound(xv, wv, want, out, True)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,Ms", [c for c in DENSE if c[0] > 1])
def test_rows_that_are_not_finite_stay_alone(T, K, Ms, dtype):
    w = packed(*normal_weight(1, Ms[0], K, 3))
    x = torch.randn(T, K, generator=gen(5), device="cuda").to(dtype)
    clean = ops.gemm_f8(w, x)
    rows = sorted({0, T // 2, T - 1})
    for i, t in enumerate(rows):
        x[t, (i * 97 + 5) % K] = BAD[i % 3]
    y = ops.gemm_f8(w, x)
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[rows] = False
    assert y[rows].isnan().all() and torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("T,k,E,K,Ms", GROUPED)
def test_grouped_products_replay_from_a_graph(T, k, E, K, Ms):
    w = packed(*normal_weight(E, Ms[0], K, 1), E)
    x = torch.randn(T, K, generator=gen(1), device="cuda")
    ids = ids_of(T, k, E, 0.2, 3)
    y = torch.zeros(T * k, Ms[0], device="cuda")

    def step(to):
        return ops.expert_gemm_f8(w, x, ops.route_rows(ids, E), out=to)

    step(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(y)
    for i in range(4):
        x.copy_(torch.randn(T, K, generator=gen(10 + i), device="cuda"))
        ids.copy_(ids_of(T, k, E, 0.2 * i, 20 + i, skew=1.0 * i))
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, step(torch.zeros_like(y))), i
