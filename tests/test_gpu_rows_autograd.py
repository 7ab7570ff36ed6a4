"""Row and adapter calls on tensors that require grad: refused where the
gradient would be lost, and used in a torch.autograd.Function as a training
program does, against the gradients of the same sums in float64."""
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


class Rows(torch.autograd.Function):
    """y = sum_j w[t, j] f[expert of (t, j)] x[t], f a factor per expert."""

    @staticmethod
    def forward(ctx, x, w, f, route):
        place = torch.arange(route.T * route.k, device=x.device)
        e = torch.bucketize(place, route.offsets[1:].long(), right=True).clamp(max=route.groups - 1)
        rows = ops.dispatch_rows(x, route, out=torch.zeros(route.T * route.k, x.shape[1], device=x.device))
        hidden = rows * f[e][:, None]
        ctx.save_for_backward(w, f, rows, hidden, e)
        ctx.route = route
        return ops.combine_rows(hidden, route, w)

    @staticmethod
    def backward(ctx, dy):
        w, f, rows, hidden, e = ctx.saved_tensors
        dhidden, dw = ops.combine_rows_backward(dy.contiguous(), hidden, ctx.route, w, out=torch.zeros_like(rows))
        df = torch.zeros_like(f).index_add_(0, e, (dhidden * rows).sum(1))
        return ops.dispatch_rows_backward(dhidden * f[e][:, None], ctx.route), dw, df, None


def test_in_an_autograd_function():
    rng = np.random.default_rng(3)
    T, k, groups, H = 33, 3, 7, 48
    ids = torch.from_numpy(rng.integers(-1, groups, (T, k)).astype(np.int64))

    def leaf(*shape):
        return torch.from_numpy(rng.standard_normal(shape)).float().to(DEV).requires_grad_()

    x, w, f = leaf(T, H), leaf(T, k), leaf(groups)
    dy = torch.from_numpy(rng.standard_normal((T, H))).float().to(DEV)
    y = Rows.apply(x, w, f, ops.route_rows(ids.to(DEV), groups))
    y.backward(dy)
    live = (ids >= 0).double()

    def sums(*leaves):
        x, w, f, dy = (t.detach().cpu().double() for t in leaves)
        for t in (x, w, f):
            t.requires_grad_()
        y = (w * live * f[ids.clamp(min=0)]).sum(1, keepdim=True) * x
        y.backward(dy)
        return y.detach(), x.grad, w.grad, f.grad

    # a sum of n terms of three products each is off by at most (n + 4) 2^-24
    # times the terms' magnitudes; the longest chains, of a factor's gradient,
    # add H terms and then T k sums
    off = (H + T * k + 4) * 2.0 ** -24
    want, size = sums(x, w, f, dy), sums(x.abs(), w.abs(), f.abs(), dy.abs())
    for got, ref, most in zip((y, x.grad, w.grad, f.grad), want, size):
        assert ((got.detach().cpu().double() - ref).abs() <= off * most + 1e-30).all()


def test_gradients_are_not_lost_without_a_word():
    T, k, H = 4, 2, 16
    r = ops.route_rows(torch.zeros(T, k, dtype=torch.int32, device=DEV), 3)
    one = ops.route_rows(torch.zeros(T, dtype=torch.int32, device=DEV), 3)
    x, rows, w = torch.ones(T, H, device=DEV), torch.ones(T * k, H, device=DEV), torch.ones(T, k, device=DEV)
    parts = {"y": torch.ones(T, 32, device=DEV), "x": torch.ones(T, 128, device=DEV),
             "a": torch.ones(3, 8, 128, device=DEV).bfloat16(), "b": torch.ones(3, 32, 8, device=DEV).bfloat16(),
             "scale": torch.ones(3, device=DEV)}

    def leaf(t):
        return t.clone().requires_grad_()

    def adapter(y, x, a, b, scale):
        return ops.adapter_add(y, x, ops.Adapters(a, b, scale), one)

    calls = [("dispatch_rows", lambda: ops.dispatch_rows(leaf(x), r)),
             ("combine_rows", lambda: ops.combine_rows(leaf(rows), r)),
             ("combine_rows", lambda: ops.combine_rows(rows, r, leaf(w))),
             ("combine_rows", lambda: ops.dispatch_rows_backward(leaf(rows), r)),
             ("combine_rows_backward", lambda: ops.combine_rows_backward(leaf(x), rows, r, w)),
             ("combine_rows_backward", lambda: ops.combine_rows_backward(x, leaf(rows), r, w)),
             ("combine_rows_backward", lambda: ops.combine_rows_backward(x, rows, r, leaf(w))),
             ("dispatch_rows", lambda: ops.dispatch_rows(x, r, out=leaf(rows))),
             ("combine_rows", lambda: ops.combine_rows(rows, r, out=leaf(x)))]
    calls += [("adapter_add", lambda n=n: adapter(**{**parts, n: leaf(parts[n])})) for n in parts]
    for name, call in calls:
        with pytest.raises(ValueError, match=f"{name} records no gradient"):
            call()
        with torch.no_grad():
            call()
        with torch.inference_mode():
            call()
