"""The 8-bit floating tier and the weights' gradient at the limits of their sizes: 2^22 columns or weight rows, the smallest
weights under many rows, plans that leave every row out or have none."""
import pytest
import torch

import f8_shapes as shapes
from knivesysl_xe_amd import ops
from f8_ref import BF16, F32, blocks, exact_rows, exact_weight, gen, plan_of, weight_values
from test_gpu_f8 import ids_of
from test_gpu_f8_edges import needs
from test_gpu_grad_weight import whole

pytestmark = pytest.mark.gpu
MOST = 1 << 22


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("T,K", [(3, MOST // 2), (2, MOST), (40, MOST), (260, MOST), (260, MOST - 16)])
def test_products_of_the_most_columns(T, K):
    # (few rows, values quantized by the product and by a launch of their own; tiles)
    needs(60)
    M = 32 if T > 16 else 16
    codes, scales = exact_weight(1, M, K, T)
    # codes in 100 blocks, the first and the last among them, so that every sum stays exact (f8_shapes: 118 do)
    kb = blocks(K)
    some = torch.zeros(kb, dtype=torch.bool, device="cuda")
    some[torch.randperm(kb, generator=gen(3), device="cuda")[:98]] = True
    some[0] = some[-1] = True
    codes = torch.where(some.repeat_interleave(128)[:K], codes.float(), torch.zeros((), device="cuda")).to(codes.dtype)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    wt = weight_values(codes, scales)[0].t().contiguous()
    for dtype in (F32, BF16):
        x = exact_rows(T, K, 5, dtype)
        want = x.double() @ wt
        q = ops.quantize_act_f8(x)
        for out in (F32, BF16):
            assert torch.equal(ops.gemm_f8(w, x, out), want.to(out))
            assert torch.equal(ops.gemm_f8(w, q, out), want.to(out))
        del x, q


@pytest.mark.parametrize("T", [2, 40, 260])
def test_products_of_the_most_weight_rows(T):
    needs(60)
    K = 16
    codes, scales = exact_weight(1, MOST, K, T)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = exact_rows(T, K, 5)
    want = x.double() @ weight_values(codes, scales)[0].t().contiguous()
    for out in (F32, BF16):
        assert torch.equal(ops.gemm_f8(w, x, out), want.to(out))
    # the transposed weight has the most columns
    t = w.transposed()
    assert torch.equal(t.unpack()[0].view(torch.uint8), codes.view(torch.uint8).transpose(1, 2)) and (t.M, t.K) == (K, MOST)
    assert torch.equal(t.transposed().codes, w.codes)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T", [600_000, 2_000_003])
def test_the_smallest_weight_under_many_rows(T, out):
    codes, scales = exact_weight(1, 16, 16, 1)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = exact_rows(T, 16, 2)
    want = (x.double() @ weight_values(codes, scales)[0].t().contiguous()).to(out)
    assert torch.equal(ops.gemm_f8(w, x, out), want)


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("N,M,K", [(300, MOST, 16), (300, 16, MOST), (1, MOST, 16), (33, 16, MOST - 16)])
def test_gradients_of_the_most_rows_and_columns(N, M, K, out):
    needs(30)
    dy, x = whole(N, M, 1), whole(N, K, 2)
    want = dy.double().t().contiguous() @ x.double()
    assert torch.equal(ops.grad_weight(dy, x, out), want.to(out))
    add = torch.randint(-50, 50, (M, K), generator=gen(3), device="cuda").to(out)
    assert torch.equal(ops.grad_weight(dy, x, out, add=add), (want + add.double()).to(out))


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,k,E,K,Ms", [c for table in shapes.GROUPED.values() for c in table])
def test_plans_that_leave_every_row_out(T, k, E, K, Ms, out):
    w = ops.F8Weight.from_codes(*exact_weight(E, Ms[0], K, 1))
    route = plan_of(torch.full((T, k), -1, dtype=torch.int32, device="cuda"), E)
    y = torch.full((T * k, Ms[0]), -7.0, dtype=out, device="cuda")
    ops.expert_gemm_f8(w, exact_rows(T, K, 1), route, out, out=y)
    assert (y == -7.0).all()
    nan = torch.full((T * k, Ms[0]), float("nan"), dtype=BF16, device="cuda")
    rows = torch.full((T * k, K), float("nan"), dtype=BF16, device="cuda")
    assert not ops.expert_grad_weight(nan, rows, route, out).any()


@pytest.mark.parametrize("out", [F32, BF16])
def test_plans_without_rows(out):
    E, M, K = 5, 144, 272
    route = plan_of(torch.empty(0, 3, dtype=torch.int32, device="cuda"), E)
    w = ops.F8Weight.from_codes(*exact_weight(E, M, K, 1))
    x = torch.empty(0, K, device="cuda")
    assert ops.expert_gemm_f8(w, x, route, out).shape == (0, M)
    dy, rows = [torch.empty(0, n, dtype=BF16, device="cuda") for n in (M, K)]
    assert not ops.expert_grad_weight(dy, rows, route, out).any()
    add = torch.randint(-50, 50, (E, M, K), generator=gen(3), device="cuda").to(out)
    assert torch.equal(ops.expert_grad_weight(dy, rows, route, out, add=add), add)


@pytest.mark.parametrize("E,skew", [(64, 0.0), (64, 50.0)])
def test_rows_that_gather_in_one_expert(E, skew):
    # 1,024 slots over 64 experts: few rows of each, or (50.0) nearly all of one
    T, K, M = 1024, 400, 272
    codes, scales = exact_weight(E, M, K, 1)
    w, wv = ops.F8Weight.from_codes(codes, scales), weight_values(codes, scales)
    route = plan_of(ids_of(T, 1, E, 0.0, 3, skew), E)
    x = exact_rows(T, K, 2)
    at = route.offsets.tolist()
    for out in (F32, BF16):
        y = ops.expert_gemm_f8(w, x, route, out)
        for e in range(E):
            rows = x[route.order[at[e]:at[e + 1]].long()]
            assert torch.equal(y[at[e]:at[e + 1]], (rows.double() @ wv[e].t().contiguous()).to(out)), e
