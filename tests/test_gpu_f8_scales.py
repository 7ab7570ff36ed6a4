"""Scales of 8-bit floating weights and rows that require grad: calls that would lose their gradient refuse them."""
import pytest
import torch

from knivesysl_xe_amd import ops
from f8_ref import exact_rows, exact_weight, plan_of

pytestmark = pytest.mark.gpu
T, K, M, E = 12, 128, 32, 3


def test_scales_that_require_grad_are_refused():
    codes, scales = exact_weight(E, M, K, 1)
    x = exact_rows(T, K, 1)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    w.scales.requires_grad_()
    a = ops.quantize_act_f8(x)
    for call in (lambda: ops.gemm_f8(w, x), lambda: ops.gemm_f8_fanout([ops.F8Weight.from_codes(codes[1], scales[1]), w], a),
                 w.transposed):
        with pytest.raises(ValueError, match="records no gradient"):
            call()
        with torch.no_grad():
            call()
    many = ops.F8Weight.from_codes(codes, scales)
    route = plan_of(torch.zeros(T, 1, device="cuda", dtype=torch.int32), E)
    many.scales.requires_grad_()
    with pytest.raises(ValueError, match="records no gradient"):
        ops.expert_gemm_f8(many, x, route)
    a.scale.requires_grad_()
    w.scales.requires_grad_(False)
    with pytest.raises(ValueError, match="records no gradient"):
        ops.gemm_f8(w, a)
    with pytest.raises(ValueError, match="records no gradient"):
        ops.quantize_act_f8(x, out=a)                        # (written to in place)
    with torch.no_grad():
        ops.gemm_f8(w, ops.quantize_act_f8(x, out=a))
