"""Low-rank adapters (csrc/kxw4_adapter.hip) on inputs whose every product and
sum fits float32: the outputs have to equal the definition's, rounded once. A
bound on rounding grows with K and r until it hides a dropped step or a wrong
adapter; here one is seen at any length, which the first test shows without a
GPU."""
import numpy as np
import pytest
import torch

from knivesysl_xe_amd import ops

DEV = "cuda:0"


def weights(gen, n, r, K, M, device="cpu"):
    """A in -2..2, eight columns of each row of B 1 or -1, every column in one row at least, scales of 1 and 2."""
    a = torch.randint(-2, 3, (n, r, K), generator=gen, device=device, dtype=torch.int8).bfloat16()
    b = (1 - 2 * torch.randint(0, 2, (n, M, r), generator=gen, device=device, dtype=torch.int8)).bfloat16()
    assert 8 * M >= r
    first = 8 * torch.arange(M, device=device)[:, None]
    b *= (torch.arange(r, device=device) - first) % r < 8
    return a, b, torch.tensor([1.0, 2.0, -1.0, -2.0], device=device)[torch.arange(n, device=device) % 4]


def inputs(gen, T, K, M, x_t, y_t):
    """Small whole numbers; three of a float32 row's x of 17 bits, which make three BF16 parts."""
    x = torch.randint(-4, 5, (T, K), generator=gen).float()
    if x_t is torch.float32:
        x.scatter_(1, torch.randint(0, K, (T, 3), generator=gen), 65793.0)
    return x.to(x_t), torch.randint(-100, 101, (T, M), generator=gen).to(y_t)


def expected(y, x, a, b, scale, ids):
    """The definition in float64, after a check that float32 holds every partial sum."""
    want = y.double()
    for e in range(len(a)):
        at = torch.nonzero(ids == e).flatten()
        if not len(at):
            continue
        A, B, X = a[e].double(), b[e].double(), x[at].double()
        low = X @ A.t()
        assert (X.abs() @ A.abs().t()).max() < 2 ** 24
        assert ((low.abs() @ B.abs().t()) * scale[e].abs().double() + 100).max() < 2 ** 24
        want[at] += scale[e].double() * (low @ B.t())
    return want.float().to(y.dtype)


SIZES = [(1, 1, 8, 128, 16), (8, 8, 16, 5120, 512), (17, 3, 24, 384, 80), (13, 2, 32, 2560, 1040),
         # two launches
         (61, 24, 64, 2048, 512), (5, 2, 200, 17408, 64), (7, 2, 256, 17408, 144), (300, 4, 256, 384, 96),
         (40, 3, 16, 17408, 272), (129, 200, 40, 256, 48), (2003, 1, 128, 5120, 16), (1600, 40, 56, 4224, 32),
         (1537, 3, 24, 4096, 48), (1900, 6, 16, 8192, 64), (1600, 3, 136, 4096, 48), (1600, 2, 256, 5120, 32),
         # B in registers, one token tile and two
         (1250, 3, 16, 17408, 16016), (1250, 3, 40, 640, 16016), (1250, 2, 128, 5120, 16016), (4300, 6, 32, 2048, 4656),
         (4300, 3, 64, 256, 4656), (5000, 60, 24, 512, 4000)]


def case(T, n, r, K, M, x_t, y_t):
    gen = torch.Generator()
    gen.manual_seed(T * r + K)
    a, b, scale = weights(gen, n, r, K, M)
    x, y = inputs(gen, T, K, M, x_t, y_t)
    ids = torch.randint(-1, n, (T,), generator=gen, dtype=torch.int32)
    ids[0], ids[-1] = n - 1, 0
    return x, y, a, b, scale, ids


@pytest.mark.parametrize("T,n,r,K,M", [s for s in SIZES if s[0] * s[4] < 300000])
def test_mistakes_are_seen(T, n, r, K, M):
    x, y, a, b, scale, ids = case(T, n, r, K, M, torch.float32, torch.float32)
    want = expected(y, x, a, b, scale, ids)

    def planted(x=x, a=a, b=b, scale=scale):
        return expected(y, x, a, b, scale, ids)

    def without(t, *at):
        t = t.clone()
        t[at] = 0
        return t

    wrong = {"no update": y, "last 32 columns of x": planted(x=without(x, slice(None), slice(K - 32, K))),
             "first 32 columns of x": planted(x=without(x, slice(None), slice(0, 32))),
             "last row of A": planted(a=without(a, slice(None), r - 1)), "scale": planted(scale=scale * 2),
             "x of one part": planted(x=x.bfloat16().float())}
    if n > 1:
        wrong["the next adapter"] = planted(a=a.roll(1, 0), b=b.roll(1, 0))
    for what, got in wrong.items():
        for e in torch.unique(ids[(ids >= 0) & (ids < n)]).tolist():
            assert not torch.equal(got[ids == e], want[ids == e]), (what, e)


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,K,M", SIZES)
@pytest.mark.parametrize("x_t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("y_t", [torch.float32, torch.bfloat16])
def test_equals_the_definition(T, n, r, K, M, x_t, y_t):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    x, y, a, b, scale, ids = case(T, n, r, K, M, x_t, y_t)
    got = ops.adapter_add(y.to(DEV), x.to(DEV), ops.Adapters(a.to(DEV), b.to(DEV), scale.to(DEV)),
                          ops.route_rows(ids.to(DEV), n))
    assert torch.equal(got.cpu(), expected(y, x, a, b, scale, ids))


@pytest.mark.gpu
def test_adapters_past_two_to_the_31_elements_exactly():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    n, r, K, M, T = 600, 256, 17408, 17408, 40               # 2.7e9 elements of a and of b
    gen = torch.Generator(device=DEV)
    gen.manual_seed(2)
    a, b, scale = weights(gen, n, r, K, M, DEV)
    x, y = inputs(torch.Generator().manual_seed(3), T, K, M, torch.float32, torch.float32)
    used = [0, 300, 598, 599]
    ids = torch.tensor([599, 0, 598, 300, -1] * 8, dtype=torch.int32)
    got = ops.adapter_add(y.to(DEV), x.to(DEV), ops.Adapters(a, b, scale), ops.route_rows(ids.to(DEV), n))
    local = torch.tensor([used.index(i) if i in used else -1 for i in ids.tolist()])
    assert torch.equal(got.cpu(), expected(y, x, a[used].cpu(), b[used].cpu(), scale[used].cpu(), local))
