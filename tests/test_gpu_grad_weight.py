"""Gradients of the 8-bit floating tier's projections: of the weight (grad_weight, expert_grad_weight) and of the input (the
transposed weight), against 64-bit references and differences."""
import pytest
import torch

from knivesysl_xe_amd import ops
from f8_ref import BF16, F32, exact_rows, exact_weight, gen, members, weight_values
from test_gpu_f8 import ids_of

pytestmark = pytest.mark.gpu


def whole(N, C, seed):
    """BF16 rows of small whole numbers: products and sums are exact in float32 in any order."""
    return torch.randint(-9, 10, (N, C), generator=gen(seed), device="cuda").to(BF16)


SIZES = [(0, 64, 32), (1, 16, 16), (1, 128, 5120), (7, 48, 144), (31, 272, 64), (32, 128, 128), (33, 208, 336), (150, 1040, 80),
         (513, 256, 256), (1000, 640, 1456), (4096, 144, 272), (16384, 16, 48), (2048, 2064, 4224)]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("N,M,K", SIZES)
def test_dense_gradient_exactly(N, M, K, out):
    dy, x = whole(N, M, 1), whole(N, K, 2)
    want = (dy.double().t().contiguous() @ x.double())
    assert torch.equal(ops.grad_weight(dy, x, out), want.to(out))
    add = torch.randint(-50, 50, (M, K), generator=gen(3), device="cuda").to(out)
    both = (want + add.double()).to(out)
    assert torch.equal(ops.grad_weight(dy, x, out, add=add), both)
    assert ops.grad_weight(dy, x, out, add=add, out=add) is add and torch.equal(add, both)


@pytest.mark.parametrize("N,M,K", [(777, 272, 400), (3000, 80, 144), (20000, 32, 64)])
def test_dense_gradient_of_normal_values(N, M, K):
    dy, x = [torch.randn(N, c, generator=gen(c), device="cuda").to(BF16) for c in (M, K)]
    want = dy.double().t().contiguous() @ x.double()
    size = dy.double().abs().t().contiguous() @ x.double().abs()
    got = ops.grad_weight(dy, x)
    # exact products; N additions in float32, each off by at most 2^-23 of the sum of magnitudes
    assert ((got.double() - want).abs() <= size * (N * 2.0 ** -23)).all()
    # (and in practice by the square root of that)
    assert (got.double() - want).norm() <= 2.0 ** -20 * want.norm()


GROUPS = [(1, 1, 1, 16, 16, 0.0), (5, 2, 3, 48, 144, 1.0), (40, 2, 5, 208, 336, 0.25), (300, 4, 40, 144, 272, 0.5),
          (700, 2, 70, 64, 16, 0.0), (2000, 1, 2, 272, 128, 0.0), (1024, 4, 8, 528, 640, 0.1)]


@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,k,E,M,K,drop", GROUPS)
def test_expert_gradient_exactly(T, k, E, M, K, drop, out):
    N = T * k
    dy, x = whole(N, M, 1), whole(N, K, 2)
    ids = ids_of(T, k, E, drop, T, skew=1.0)
    route = ops.route_rows(ids, E)
    end = int(route.offsets[-1])
    dy[end:], x[end:] = float("nan"), float("inf")           # rows behind the last expert's are left out
    want = torch.zeros(E, M, K, dtype=torch.float64, device="cuda")
    p = 0
    for e, m in enumerate(members(ids, E)):
        want[e] = dy[p:p + len(m)].double().t().contiguous() @ x[p:p + len(m)].double()
        p += len(m)
    assert torch.equal(ops.expert_grad_weight(dy, x, route, out), want.to(out))
    add = torch.randint(-50, 50, (E, M, K), generator=gen(3), device="cuda").to(out)
    assert torch.equal(ops.expert_grad_weight(dy, x, route, out, add=add), (want + add.double()).to(out))


def test_a_row_that_is_not_finite_stays_in_its_group():
    dy, x = whole(90, 48, 1), whole(90, 80, 2)
    ids = torch.arange(90, device="cuda").to(torch.int32) // 30          # sorted places 30 to 59 are group 1's
    route = ops.route_rows(ids, 3)
    clean = ops.expert_grad_weight(dy, x, route)
    dy[59, 3], x[59, 7] = float("inf"), float("nan")
    got = ops.expert_grad_weight(dy, x, route)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2])
    assert got[1, 3].isnan().any() and got[1, :, 7].isnan().all()


@pytest.mark.parametrize("T,K,M", [(3, 144, 64), (40, 272, 160), (200, 384, 512)])
def test_gradients_against_differences(T, K, M):
    # y = W x is linear in both, and the inputs are such that y, its gradients and the sums are exact: the loss <dy, y>
    # moves by dx[t][k] when x[t][k] moves by one, and by dw[m][k] when w[m][k] does
    codes, scales = exact_weight(1, M, K, 1)
    scales.fill_(1.0)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = exact_rows(T, K, 2)
    x = torch.where(x.abs() < 100, x.sign() * x.abs().clamp(max=14).floor(), x)
    x[:, ::128] = 448.0                                      # scale 1 everywhere
    dy = torch.randint(-14, 15, (T, M), generator=gen(4), device="cuda").float()
    dy[:, ::128] = 448.0
    dx = ops.gemm_f8(w.transposed(), dy)
    dw = ops.grad_weight(dy.to(BF16), x.to(BF16))
    assert torch.equal(dx.double(), dy.double() @ weight_values(codes, scales)[0])
    assert torch.equal(dw.double(), dy.double().t().contiguous() @ x.double())

    def loss(weight, rows):
        return (dy.double() * ops.gemm_f8(weight, rows).double()).sum()

    base = loss(w, x)
    for i in range(6):
        t, k, m = (7 * i) % T, (13 * i + 1) % K, (11 * i + 1) % M
        if k % 128 == 0:
            k += 1
        moved = x.clone()
        moved[t, k] += 1.0
        assert loss(w, moved) - base == dx[t, k]
        c = codes[0].float()
        step = 1.0 if c[m, k] < 15 else -1.0
        c[m, k] += step
        assert loss(ops.F8Weight.from_codes(c.to(codes.dtype), scales[0]), x) - base == step * dw[m, k]


def test_an_experts_training_step():
    # dispatch, project, and the gradients back to x and to the weights
    E, k, T, K, M = 5, 2, 60, 256, 208
    codes, scales = exact_weight(E, M, K, 1)
    w, wv = ops.F8Weight.from_codes(codes, scales), weight_values(codes, scales)
    ids = ids_of(T, k, E, 0.2, 2)
    route = ops.route_rows(ids, E)
    x = whole(T, K, 3)
    x[:, ::128] = 448.0
    dys = whole(T * k, M, 4)
    dys[:, ::128] = 448.0
    xs = ops.dispatch_rows(x, route)
    dxs = ops.expert_gemm_f8(w.transposed(), dys, route, F32, sorted_rows=True)
    dx = ops.dispatch_rows_backward(dxs, route)
    dw = ops.expert_grad_weight(dys, xs, route)
    want, want_dw, p = torch.zeros(T, K, dtype=torch.float64, device="cuda"), torch.zeros_like(wv), 0
    for e, m in enumerate(members(ids, E)):
        for s in m:
            want[s // k] += dys[p].double() @ wv[e]
            want_dw[e] += torch.outer(dys[p].double(), x[s // k].double())
            p += 1
    assert torch.equal(dx.double(), want) and torch.equal(dw.double(), want_dw)


def test_gradients_replay_from_a_graph():
    E, T, k, M, K = 4, 96, 2, 144, 80
    ids = ids_of(T, k, E, 0.2, 1)
    dy, x = whole(T * k, M, 1), whole(T * k, K, 2)
    long_dy, long_x = whole(9000, 32, 3), whole(9000, 48, 4)             # (a split sum)
    dw, long_dw = torch.zeros(E, M, K, device="cuda"), torch.zeros(32, 48, device="cuda")

    def step():
        route = ops.route_rows(ids, E)
        ops.expert_grad_weight(dy, x, route, out=dw)
        ops.grad_weight(long_dy, long_x, out=long_dw)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        ids.copy_(ids_of(T, k, E, 0.2, 20 + i))
        dy.copy_(whole(T * k, M, 30 + i))
        long_dy.copy_(whole(9000, 32, 40 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = dw.clone(), long_dw.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got[0], dw) and torch.equal(got[1], long_dw)
        assert torch.equal(long_dw.double(), long_dy.double().t().contiguous() @ long_x.double())
