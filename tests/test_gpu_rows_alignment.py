"""Row calls (csrc/kxw4_rows.hip) at every alignment of their type: the same bits
as on aligned buffers, sums of weights' gradients among them, since the pieces of
a row go by its length alone. And their rounding to bfloat16, over every float32."""
import numpy as np
import pytest
import torch

from knivesysl_xe_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def shifted(t, by):
    """A copy of t that starts `by` elements into its memory."""
    base = torch.empty(t.numel() + by, dtype=t.dtype, device=DEV)
    out = base[by:].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 == by * t.element_size() % 16
    return out


@pytest.mark.parametrize("T,k,H", [(21, 2, 64), (9, 3, 5), (14, 5, 130), (7, 1, 1003), (6, 4, 2049), (5, 9, 4352)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_bits_at_any_alignment(T, k, H, dtype):
    rng = np.random.default_rng(H)
    groups = 4
    r = ops.route_rows(torch.from_numpy(rng.integers(-1, groups, (T, k)).astype(np.int32)).to(DEV), groups)

    def normal(*shape):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(DEV)

    x, rows, dy, w = normal(T, H).to(dtype), normal(T * k, H).to(dtype), normal(T, H), normal(T, k)

    def calls(by):
        def out(t):
            return shifted(torch.full_like(t, 7.0), by)
        a, b, c, d = (shifted(t, by) for t in (x, rows, dy, w))
        return (ops.dispatch_rows(a, r, out=out(rows)), ops.combine_rows(b, r, d, out=out(x)), ops.combine_rows(b, r, out=out(dy)),
                *ops.combine_rows_backward(c, b, r, d, out=out(rows)), *ops.combine_rows_backward(a, b, r, d, out=out(rows)))

    want = calls(0)
    for by in range(1, 16 // x.element_size()):
        for i, (got, ref) in enumerate(zip(calls(by), want)):
            assert torch.equal(got, ref), (by, i)


def test_all_float32_patterns_round_to_the_nearest_bfloat16():
    T, H = 1 << 19, 512
    r = ops.route_rows(torch.zeros(T, dtype=torch.int32, device=DEV), 1)
    low = torch.arange(T * H, dtype=torch.int32, device=DEV).view(T, H)
    for i in range(16):
        x = (low + ((i - 8) << 28)).view(torch.float32)
        y, want = ops.combine_rows(x, r, dtype=torch.bfloat16), x.bfloat16()
        # (1 * x + 0: a zero of either sign is +0)
        same = (y.view(torch.int16) == want.view(torch.int16)) | ((y == 0) & (want == 0))
        assert (same | (torch.isnan(x) & torch.isnan(y))).all(), i
