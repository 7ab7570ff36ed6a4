"""Calls of so many tokens that their work takes more threads
than the 2^32 of one launch. All values are whole numbers or powers of two that
every step holds exactly, so outputs are compared bit for bit."""
import pytest
import torch

from knivesysl_xe_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def whole(gen, *shape, dtype=torch.bfloat16):
    """Whole numbers from -8 to 8."""
    t = torch.empty(shape, dtype=torch.int8, device=DEV)
    return t.random_(-8, 9, generator=gen).to(dtype)


@pytest.mark.parametrize("T,k", [((1 << 24) + 777, 1), ((1 << 23) + 5, 5)])
def test_gradients_of_many_tokens(T, k):
    # one 256-thread work-group for each token and four choices
    gen = torch.Generator(device=DEV)
    gen.manual_seed(T)
    H, groups = 8, 3
    ids = torch.randint(-1, groups, (T, k), generator=gen, device=DEV, dtype=torch.int32)
    r = ops.route_rows(ids, groups)
    rows, dy = whole(gen, T * k, H), whole(gen, T, H)
    w = torch.exp2(whole(gen, T, k, dtype=torch.float32))
    out = torch.full((T * k, H), 77.0, dtype=torch.bfloat16, device=DEV)
    drows, dw = ops.combine_rows_backward(dy, rows, r, w, out=out)
    live = int(r.offsets[-1])
    slot = r.order[:live].long()
    assert torch.equal(drows[:live], (w.view(-1)[slot][:, None] * dy[slot // k].float()).bfloat16())
    assert (drows[live:] == 77).all()
    want = torch.zeros(T * k, device=DEV)
    want[slot] = (dy[slot // k].float() * rows[:live].float()).sum(1)
    assert torch.equal(dw, want.view(T, k))


def test_dispatch_and_combine_of_many_tokens():
    # 33 pieces of 16 bytes a row: a 64-thread work-group for each token
    T, H, groups, step = (1 << 26) + 777, 264, 5, 1 << 20
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1)
    r = ops.route_rows(torch.randint(0, groups, (T,), generator=gen, device=DEV, dtype=torch.int32), groups)
    x = torch.empty(T, H, dtype=torch.bfloat16, device=DEV)              # 35 GB, positive and finite
    x.view(torch.int16).random_(0, 0x3F80, generator=gen)
    rows = torch.zeros_like(x)
    ops.dispatch_rows(x, r, out=rows)
    y = torch.zeros_like(x)
    ops.combine_rows(rows, r, out=y)
    for t in range(0, T, step):
        assert torch.equal(rows[r.position[t:t + step, 0].long()], x[t:t + step]), t
        assert torch.equal(y[t:t + step], x[t:t + step]), t


def test_adapters_of_many_tokens():
    # 32 tokens a work-group of 1,024 threads in the first of the two launches
    T, K, M, r, n, step = (1 << 27) + 777, 128, 16, 8, 3, 1 << 20
    gen = torch.Generator(device=DEV)
    gen.manual_seed(2)
    ids = torch.randint(-1, n, (T,), generator=gen, device=DEV, dtype=torch.int32)
    x = torch.empty(T, K, dtype=torch.bfloat16, device=DEV)              # 34 GB of 1 and -1
    x.view(torch.int16).random_(0, 2, generator=gen).mul_(-0x8000).add_(0x3F80)
    a, b, y = whole(gen, n, r, K), whole(gen, n, M, r), whole(gen, T, M, dtype=torch.float32)
    scale = torch.tensor([0.5, 2.0, -1.0], device=DEV)
    got = ops.adapter_add(y, x, ops.Adapters(a, b, scale), ops.route_rows(ids, n))
    # (|update| <= 2 * 8 * 8 * 8 * 128 = 2^17 in halves: exact)
    both = (b.double() @ a.double()) * scale.double()[:, None, None]
    for t in range(0, T, step):
        want = y[t:t + step].double()
        for e in range(n):
            at = ids[t:t + step] == e
            want[at] += x[t:t + step][at].double() @ both[e].t()
        assert torch.equal(got[t:t + step].double(), want), t
