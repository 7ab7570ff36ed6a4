"""Calls that record no gradient refuse tensors whose gradient or tangent they would lose: tensors that require grad, and dual
tensors of forward-mode differentiation."""
import pytest
import torch
from torch.autograd import forward_ad

from knivesysl_xe_amd import ops
from f8_ref import BF16, F32, exact_weight, gen, plan_of

pytestmark = pytest.mark.gpu
T, K, M, E, k = 12, 128, 32, 3, 2


def rand(*shape, dtype=F32):
    return torch.randn(*shape, generator=gen(sum(shape)), device="cuda").to(dtype)


def calls():
    """name -> (the floating tensors of a call, the call on them)"""
    codes, scales = exact_weight(E, M, K, 1)
    one = ops.F8Weight.from_codes(codes[0], scales[0])
    many = ops.F8Weight.from_codes(codes, scales)
    route = plan_of(torch.arange(T * k, device="cuda", dtype=torch.int32).view(T, k) % E, E)
    x, rows, y = rand(T, K), rand(T * k, K), rand(T, M)
    adapters = [rand(2, 16, K, dtype=BF16), rand(2, M, 16, dtype=BF16), rand(2)]
    which = ops.route_rows(torch.zeros(T, 1, device="cuda", dtype=torch.int32), 2)
    return {
        "dispatch_rows": ([x], lambda x: ops.dispatch_rows(x, route)),
        "combine_rows": ([rows, rand(T, k)], lambda rows, w: ops.combine_rows(rows, route, w)),
        "combine_rows_backward": ([x, rows, rand(T, k)], lambda dy, rows, w: ops.combine_rows_backward(dy, rows, route, w)),
        "adapter_add": ([y, x, *adapters], lambda y, x, a, b, s: ops.adapter_add(y, x, ops.Adapters(a, b, s), which)),
        "F8Weight.from_codes": ([scales[0]], lambda s: ops.F8Weight.from_codes(codes[0], s)),
        "F8Weight.quantize": ([rand(M, K)], ops.F8Weight.quantize),
        "quantize_act_f8": ([x], ops.quantize_act_f8),
        "silu_mul_quant_f8": ([x, rand(T, K)], ops.silu_mul_quant_f8),
        "gemm_f8": ([x, y], lambda x, r: ops.gemm_f8(one, x, residual=r)),
        "expert_gemm_f8": ([x], lambda x: ops.expert_gemm_f8(many, x, route)),
        "grad_weight": ([rand(T, M, dtype=BF16), x.to(BF16), rand(M, K)], lambda dy, x, add: ops.grad_weight(dy, x, add=add)),
        "expert_grad_weight": ([rand(T * k, M, dtype=BF16), rows.to(BF16)], lambda dy, x: ops.expert_grad_weight(dy, x, route)),
    }


NAMES = ("dispatch_rows", "combine_rows", "combine_rows_backward", "adapter_add", "F8Weight.from_codes", "F8Weight.quantize",
         "quantize_act_f8", "silu_mul_quant_f8", "gemm_f8", "expert_gemm_f8", "grad_weight", "expert_grad_weight")


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    tensors, call = calls()[name]
    for i in range(len(tensors)):
        with forward_ad.dual_level():
            call(*tensors)                                   # (no dual tensor: nothing to lose)
            some = list(tensors)
            some[i] = forward_ad.make_dual(some[i], torch.ones_like(some[i]))
            with pytest.raises(ValueError, match="tangent"):
                call(*some)
        call(*tensors)


@pytest.mark.parametrize("name", NAMES)
def test_gradients_are_refused(name):
    tensors, call = calls()[name]
    for i in range(len(tensors)):
        some = [t.clone() for t in tensors]
        some[i].requires_grad_()
        with pytest.raises(ValueError, match="records no gradient"):
            call(*some)
        with torch.no_grad():
            call(*some)


def test_a_function_with_a_jvp_of_its_own_may_call():
    codes, scales = exact_weight(1, M, K, 1)
    w = ops.F8Weight.from_codes(codes[0], scales[0])

    class Project(torch.autograd.Function):
        @staticmethod
        def forward(x):
            return ops.gemm_f8(w, x)

        @staticmethod
        def setup_context(ctx, inputs, output):
            pass

        @staticmethod
        def jvp(ctx, dx):
            return torch.full((T, M), 2.0, device="cuda")

    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(Project.apply(forward_ad.make_dual(rand(T, K), rand(T, K))))
        assert torch.equal(y.primal, ops.gemm_f8(w, rand(T, K))) and (y.tangent == 2.0).all()
