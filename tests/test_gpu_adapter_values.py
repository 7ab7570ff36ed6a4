"""Infinities among the weights of low-rank adapters (csrc/kxw4_adapter.hip): an
output is the infinity or NaN that the definition gives in 64 bits, and those
that no infinity reaches keep their bits. Rows without an adapter are y, bit for
bit."""
import numpy as np
import pytest
import torch

from knivesysl_xe_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF = float("inf")


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# both in one launch; two launches, B's rows a lane each and four lanes each, a
# long A, one token tile and two; B in registers, 1 to 4 chunks of r
SIZES = [(8, 3, 16, 256, 64), (5, 2, 32, 128, 1040), (7, 2, 8, 5248, 48), (61, 3, 64, 512, 80), (20, 2, 256, 128, 48),
         (300, 4, 24, 640, 96), (1600, 3, 24, 4096, 48), (1600, 3, 128, 4096, 48), (1250, 3, 16, 128, 16016),
         (1250, 3, 40, 128, 16016), (1250, 3, 128, 256, 16016), (4300, 5, 32, 128, 4656)]


def place(v):
    """0 finite, 1 infinity, -1 its negative, 2 NaN."""
    return torch.where(torch.isnan(v), 2, torch.where(torch.isinf(v), torch.sign(v), 0.0)).to(torch.int8)


@pytest.mark.parametrize("T,n,r,K,M", SIZES)
@pytest.mark.parametrize("x_t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("y_t", [torch.float32, torch.bfloat16])
def test_infinite_weights(T, n, r, K, M, x_t, y_t):
    rng = np.random.default_rng(T + r + M)

    def values(*shape):
        return torch.from_numpy(rng.integers(-2, 3, shape).astype(np.float32))

    # small whole numbers, so that low holds zeros and values of one BF16 part;
    # x of odd tokens in all 24 bits
    a, b = values(n, r, K).bfloat16(), values(n, M, r).bfloat16()
    x = values(T, K)
    x[1::2] *= 1 + 2.0 ** -20 * torch.from_numpy(rng.integers(0, 8, (len(x[1::2]), K)).astype(np.float32))
    x[:, 3] = torch.tensor([1.0, -2.0, 0.0, 1.0 + 2.0 ** -22])[torch.arange(T) % 4]
    x = x.to(x_t)
    y = values(T, M).to(y_t)
    ids = torch.arange(T, dtype=torch.int32) % (n + 1) - 1
    route = ops.route_rows(ids.to(DEV), n)
    scale = torch.tensor([0.5, 2.0, -1.0, 1.0, 0.25][:n])
    add = lambda a, b: ops.adapter_add(y.to(DEV), x.to(DEV), ops.Adapters(a.to(DEV), b.to(DEV), scale.to(DEV)), route).cpu()
    plain = add(a, b)
    assert torch.isfinite(plain).all()

    # B: outputs m of adapter 0's tokens, in the first and the last column of r
    spots = [(0, 0), (7, r - 1), (M - 1, r // 2), (M // 2, 0), (17, r - 1)]
    b2 = b.clone()
    for i, (m, j) in enumerate(spots):
        b2[0, m, j] = INF if i % 2 else -INF
    got = add(a, b2)
    mine = torch.nonzero(ids == 0).flatten()
    low = x[mine].double() @ a[0].double().t() * scale[0].double()
    rows = torch.tensor([m for m, _ in spots])
    want = y[mine][:, rows].double() + low @ b2[0, rows].double().t()
    assert torch.equal(place(got[mine][:, rows]), place(want))
    got[mine[:, None], rows] = plain[mine[:, None], rows]
    assert torch.equal(got, plain)

    # A: low of adapter 1's tokens, or of half of them not a number
    for k in (3, K - 1):
        a2 = a.clone()
        a2[1, 0, k] = INF
        a2[1, r - 1, k] = -INF
        got = add(a2, b)
        mine = torch.nonzero(ids == 1).flatten()
        cols = torch.unique(torch.cat([torch.arange(0, M, max(1, M // 64)), torch.tensor([M - 1])]))
        low = x[mine].double() @ a2[1].double().t() * scale[1].double()
        want = y[mine][:, cols].double() + low @ b[1, cols].double().t()
        assert torch.equal(place(got[mine][:, cols]), place(want))
        got[mine] = plain[mine]
        assert torch.equal(got, plain)


def test_infinite_weights_and_inputs_and_padding():
    # an infinite x times an infinite weight; NaN in rows without an adapter
    T, r, K, M = 9, 8, 128, 32
    a, b = torch.ones(2, r, K).bfloat16(), torch.ones(2, M, r).bfloat16()
    a[0, :, 5] = INF
    x, y = torch.ones(T, K), torch.zeros(T, M)
    x[1, 5], x[2, 5], x[4] = INF, -INF, float("nan")
    ids = torch.tensor([0, 0, 0, 1, -1, 0, 1, 2, 0], dtype=torch.int32)
    got = ops.adapter_add(y.to(DEV), x.to(DEV), ops.Adapters(a.to(DEV), b.to(DEV), torch.ones(2, device=DEV)),
                          ops.route_rows(ids.to(DEV), 2)).cpu()
    assert (got[[0, 1, 5, 8]] == INF).all() and (got[2] == -INF).all()
    assert (got[[3, 6]] == r * K).all() and (got[[4, 7]] == 0).all()


@pytest.mark.parametrize("T,n,r,K,M", SIZES)
@pytest.mark.parametrize("y_t", [torch.float32, torch.bfloat16])
def test_rows_without_an_adapter_are_copied(T, n, r, K, M, y_t):
    # any bit patterns: zeros of both signs, NaNs of every kind
    bits = torch.int32 if y_t is torch.float32 else torch.int16
    gen = torch.Generator(device=DEV)
    gen.manual_seed(T)
    y = torch.zeros(T, M, dtype=bits, device=DEV)
    y.random_(-(1 << (8 * y.element_size() - 1)), (1 << (8 * y.element_size() - 1)) - 1, generator=gen)
    y[:, ::3] = -(1 << (8 * y.element_size() - 1))                       # -0
    y[:, 1::7] = 0x7F800001 if y_t is torch.float32 else 0x7F81
    x = torch.randn(T, K, generator=gen, device=DEV)
    ad = ops.Adapters(torch.randn(n, r, K, generator=gen, device=DEV).bfloat16(),
                      torch.randn(n, M, r, generator=gen, device=DEV).bfloat16(), torch.ones(n, device=DEV))
    ids = torch.randint(-1, n + 1, (T,), generator=gen, device=DEV)
    none = (ids < 0) | (ids >= n)
    none[0], ids[0] = True, -1
    got = ops.adapter_add(y.view(y_t), x, ad, ops.route_rows(ids, n))
    assert torch.equal(got.view(bits)[none], y[none])
