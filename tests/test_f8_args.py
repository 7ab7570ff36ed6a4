"""Refusals of the 8-bit floating tier and of the weights' gradient, before any launch (no GPU needed): the C ABI's codes
on addresses that no call reads, and the torch front end on CPU tensors."""
import ctypes as C

import pytest
import torch

from knivesysl_xe_amd import _lib, ops

BIG = 1 << 22
AT = 4096                                                    # an aligned address that nothing reads


def W(M=256, K=512, groups=1, codes=AT, scales=AT):
    return _lib.WeightF8(groups, M, K, codes, scales)


def A(T=8, K=512, x_dtype=0, q=2 * AT, scale=AT, x=None):
    return _lib.ActF8(T, K, x_dtype, q, scale, x)


def R(T=8, k=1, groups=4, at=AT):
    return _lib.Route(T, k, groups, at, at, at)


def array(ws):
    return (C.POINTER(_lib.WeightF8) * len(ws))(*[C.pointer(w) if w is not None else None for w in ws])


def gemm(ws=None, ys=None, a=None, dtype=0, residual=None, ws_at=16 * AT, count=None):
    ws = [W()] if ws is None else ws
    ys = [4 * AT + 65536 * i for i in range(len(ws))] if ys is None else ys
    return _lib.lib().kxw4_gemm_f8(array(ws), (C.c_void_p * len(ys))(*ys), len(ws) if count is None else count,
                                   C.byref(A() if a is None else a), dtype, residual, ws_at, None)


def expert(w=None, a=None, r=None, in_order=0, dtype=0, ws_at=16 * AT):
    w = W(groups=4) if w is None else w
    return _lib.lib().kxw4_expert_gemm_f8(array([w]), (C.c_void_p * 1)(4 * AT), 1, C.byref(A() if a is None else a),
                                          C.byref(R() if r is None else r), in_order, dtype, ws_at, None)


def test_product_refusals():
    arg, shape, prep = _lib.EARG, _lib.ESHAPE, _lib.EPREP
    for bad in (dict(M=250), dict(K=500), dict(M=0), dict(K=0), dict(M=BIG + 16), dict(K=BIG + 16), dict(M=-16)):
        a = A(K=bad.get("K", 512))
        assert gemm([W(**bad)], a=a) == shape, bad
    assert gemm([W(codes=None)]) == arg and gemm([W(scales=None)]) == arg
    assert gemm([W(codes=AT + 8)]) == arg and gemm([W(scales=AT + 2)]) == arg
    assert gemm([W(groups=2)]) == shape                       # a stack of experts is not one projection
    assert gemm([W(), W(K=640)]) == shape and gemm([W()], a=A(K=640)) == shape
    assert gemm([W()] * 5, count=5) == arg and gemm(count=0) == arg and gemm([None]) == arg
    assert gemm(dtype=2) == shape and gemm(a=A(T=-1)) == shape
    assert gemm(a=A(scale=None)) == prep and gemm(a=A(q=None, x=None)) == prep
    assert gemm(a=A(q=None, x=2 * AT, x_dtype=3)) == shape
    assert gemm(a=A(q=AT + 8)) == arg and gemm(a=A(q=None, x=AT + 4)) == arg
    assert gemm(ys=[0]) == arg and gemm(ys=[AT + 8]) == arg
    assert gemm([W(), W()], ys=[4 * AT, 4 * AT]) == arg       # one output for two weights
    assert gemm(ys=[2 * AT]) == arg                           # the rows' codes
    assert gemm(a=A(q=None, x=4 * AT)) == arg                 # the rows' values
    assert gemm([W(), W()], residual=AT) == arg and gemm(residual=AT + 4) == arg
    assert gemm(residual=4 * AT, dtype=1) == arg              # a BF16 output over its residual
    assert gemm(a=A(T=0, q=None, scale=None)) == 0            # no rows: nothing is read or launched
    assert _lib.lib().kxw4_gemm_f8(None, None, 1, C.byref(A()), 0, None, None, None) == arg
    assert _lib.lib().kxw4_gemm_f8(array([W()]), (C.c_void_p * 1)(AT), 1, None, 0, None, None, None) == arg


def test_rows_of_values_ask_for_scratch():
    L = _lib.lib()
    a, w = A(T=1000, q=None, scale=None, x=2 * AT), W(M=1024)
    assert L.kxw4_gemm_f8_workspace(array([w]), 1, C.byref(a), 0) >= 1000 * 512 + 4 * 1000 * 4
    assert gemm([w], a=a, ws_at=None) == _lib.EARG and gemm([w], a=a, ws_at=AT + 8) == _lib.EARG
    # (a short launch quantizes by itself)
    assert L.kxw4_gemm_f8_workspace(array([W()]), 1, C.byref(a), 0) == 0
    assert L.kxw4_gemm_f8_workspace(array([W()]), 1, C.byref(A(T=0)), 0) == 0
    e = W(M=1024, groups=4)
    assert L.kxw4_expert_gemm_f8_workspace(array([e]), 1, C.byref(a), C.byref(R(T=1000)), 0, 0) >= 1000 * 512
    assert expert(w=e, a=a, r=R(T=1000), ws_at=None) == _lib.EARG


def test_expert_product_refusals():
    arg, shape, prep = _lib.EARG, _lib.ESHAPE, _lib.EPREP
    assert expert(w=W(groups=3)) == shape                     # not the plan's groups
    assert expert(r=R(groups=1025)) == shape and expert(r=R(k=0)) == shape and expert(r=R(T=-1)) == shape
    assert expert(r=R(at=None)) == prep
    assert expert(a=A(T=9)) == shape and expert(r=R(k=2), in_order=1) == shape
    assert expert(a=A(T=0), r=R(T=0, at=None)) == 0
    # 32-bit offsets of the rows' codes
    big = A(T=1 << 20, K=2048)
    assert expert(w=W(groups=4, K=2048), a=big, r=R(T=1 << 20)) == shape
    L = _lib.lib()
    assert L.kxw4_expert_gemm_f8(array([W(groups=4)]), (C.c_void_p * 1)(4 * AT), 1, C.byref(A()), None, 0, 0, None, None) == arg


def test_layout_refusals():
    L, arg, shape = _lib.lib(), _lib.EARG, _lib.ESHAPE
    assert L.kxw4_f8_code_bytes(3, 208, 336) == 3 * 208 * 384 and L.kxw4_f8_code_bytes(1, 200, 128) == 0
    assert L.kxw4_pack_weight_f8(None, 1, 16, 16, AT, None) == arg and L.kxw4_pack_weight_f8(AT, 1, 16, 16, AT, None) == arg
    assert L.kxw4_pack_weight_f8(AT, 1, 24, 16, 2 * AT, None) == shape and L.kxw4_pack_weight_f8(AT, 0, 16, 16, 2 * AT, None) == shape
    w = W()
    assert L.kxw4_unpack_weight_f8(C.byref(w), None, None) == arg and L.kxw4_unpack_weight_f8(None, AT, None) == arg
    assert L.kxw4_transpose_weight_f8(C.byref(w), AT, 2 * AT, None) == arg       # codes over themselves
    assert L.kxw4_transpose_weight_f8(C.byref(w), 2 * AT, AT, None) == arg
    assert L.kxw4_quantize_weight_f8(AT, 5, 1, 16, 16, 2 * AT, 3 * AT, None) == shape
    assert L.kxw4_quantize_weight_f8(AT + 4, 0, 1, 16, 16, 2 * AT, 3 * AT, None) == arg
    assert L.kxw4_quantize_act_f8(AT, 0, 4, 100, 2 * AT, 3 * AT, None) == shape
    assert L.kxw4_quantize_act_f8(AT, 0, -1, 128, 2 * AT, 3 * AT, None) == shape
    assert L.kxw4_quantize_act_f8(AT, 0, 4, 128, AT, 3 * AT, None) == arg
    assert L.kxw4_quantize_act_f8(None, 0, 0, 128, None, None, None) == 0
    # more rows and blocks than one launch takes
    assert L.kxw4_quantize_act_f8(AT, 0, 1 << 30, 1024, 2 * AT, 3 * AT, None) == shape
    assert L.kxw4_silu_mul_quant_f8(AT, AT, 2 * AT, 0, 4, 128, 3 * AT, 4 * AT, None) == arg
    assert L.kxw4_silu_mul_quant_f8(None, AT, None, 0, 4, 128, 3 * AT, 4 * AT, None) == arg
    assert L.kxw4_silu_mul_quant_f8(None, AT, 2 * AT, 0, 4, 120, 3 * AT, 4 * AT, None) == shape


def test_gradient_refusals():
    L, arg, shape = _lib.lib(), _lib.EARG, _lib.ESHAPE

    def grad(dy=AT, x=2 * AT, N=64, M=256, K=128, r=None, add=None, dw=3 * AT, dtype=0, at=16 * AT):
        return L.kxw4_grad_weight(dy, x, N, M, K, None if r is None else C.byref(r), add, dw, dtype, at, None)

    assert grad(M=100) == shape and grad(K=8) == shape and grad(N=-1) == shape and grad(dtype=2) == shape
    assert grad(M=BIG + 16) == shape
    assert grad(dy=None) == arg and grad(x=None) == arg and grad(dw=None) == arg
    assert grad(dy=AT + 8) == arg and grad(dw=3 * AT + 4) == arg and grad(add=AT + 4) == arg
    assert grad(dw=AT) == arg and grad(dw=2 * AT) == arg
    assert grad(r=R(T=63)) == shape and grad(r=R(T=64, groups=0)) == shape and grad(r=R(T=64, at=None)) == _lib.EPREP


def test_front_end_refuses_cpu_tensors_and_wrong_sizes():
    w = ops.F8Weight(1, 16, 128, torch.zeros(16 * 128, dtype=torch.uint8), torch.zeros(1, 1, 1))
    with pytest.raises(ValueError, match="weights must be on the GPU"):
        ops.gemm_f8(w, torch.zeros(2, 128))
    with pytest.raises(ValueError, match="one to four weights"):
        ops.gemm_f8_fanout([], torch.zeros(2, 128))
    with pytest.raises(ValueError, match="codes must be on the GPU"):
        ops.F8Weight.from_codes(torch.zeros(16, 128, dtype=torch.uint8), torch.zeros(1, 1))
    with pytest.raises(ValueError, match="w must be on the GPU"):
        ops.F8Weight.quantize(torch.zeros(16, 128))
    with pytest.raises(ValueError, match="x must be on the GPU"):
        ops.quantize_act_f8(torch.zeros(2, 128))
    with pytest.raises(ValueError, match="gate must be on the GPU"):
        ops.silu_mul_quant_f8(torch.zeros(2, 128), torch.zeros(2, 128))
    with pytest.raises(ValueError, match="dy must be on the GPU"):
        ops.grad_weight(torch.zeros(2, 16), torch.zeros(2, 16))
    for bad in ((0, 16, 16), (1025, 16, 16), (1, 20, 16), (1, 16, 8), (1, BIG + 16, 16)):
        with pytest.raises(ValueError, match="multiples of 16"):
            ops.F8Weight.empty(*bad, device="cpu")
    with pytest.raises(ValueError, match="multiple of 16"):
        ops._f8_rows(2, 100, "cpu", None)
    with pytest.raises(ValueError, match="out does not match"):
        ops._f8_rows(2, 128, "cpu", ops.QuantActF8.empty(3, 128, "cpu"))
    short = ops.QuantActF8(4, 256, torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(4, 2))
    with pytest.raises(ValueError, match="activation scales"):
        ops._check_act_f8(short, torch.device("cpu"))


def test_a_copied_weight_is_checked_anew():
    import copy
    w = ops.F8Weight.empty(2, 16, 144, device="cpu")
    assert w.codes.numel() == 2 * 16 * 256 and tuple(w.scales.shape) == (2, 1, 2)
    w.__dict__["_made"] = ("cpu", w.at(), w.c())
    c = copy.deepcopy(w)
    assert c._made is None and (c.groups, c.M, c.K) == (2, 16, 144)
