"""Refusals of the row routing, expert and adapter calls: argument checks of
the C ABI and of the torch front end, made before any HIP call."""
import ctypes as C

import pytest
import torch

from knivesysl_xe_amd import _lib, ops

P = C.c_void_p(64)
OTHER = C.c_void_p(128)                                     # an output beside the inputs at P


def R(T=8, k=2, groups=4, offsets=64, order=64, position=64):
    return _lib.Route(T, k, groups, offsets, order, position)


def W(M=256, K=1024, group=128, enc=0, codes=64, scales=64):
    return _lib.Weight(M, K, group, enc, codes, scales)


def A(T=8, K=1024, block=0, q=64, scale=64, s=64):
    return _lib.Act(T, K, block, q, scale, s)


def D(n=4, r=16, K=1024, M=256, a=64, b=64, scale=64):
    return _lib.AdapterSet(n, r, K, M, a, b, scale)


def test_route_refuses_bad_plans():
    f = _lib.lib().kxw4_route_rows
    assert f(P, 0, None, None, None) == _lib.EARG
    assert f(None, 0, C.byref(R()), None, None) == _lib.EARG
    for missing in ("offsets", "order", "position"):
        assert f(P, 0, C.byref(R(**{missing: None})), None, None) == _lib.EARG
    for bad in (dict(T=-1), dict(k=0), dict(groups=0), dict(groups=1025), dict(T=1 << 30, k=2)):
        assert f(P, 0, C.byref(R(**bad)), None, None) == _lib.ESHAPE
    # a large plan needs its scratch
    assert f(P, 0, C.byref(R(T=1 << 20)), None, None) == _lib.EARG


def test_route_workspace_sizes():
    size = _lib.lib().kxw4_route_workspace
    assert size(8, 2, 4) == 0 and size(8192, 1, 4) == 0 and size(0, 1, 4) == 0
    assert size(8193, 1, 4) == (8193 + 2047) // 2048 * 5 * 4
    assert size(1 << 20, 8, 128) == 256 * 129 * 4
    assert size(8, 2, 0) == 0 and size(-1, 2, 4) == 0 and size(1 << 30, 2, 4) == 0


def test_row_calls_refuse_bad_arguments():
    L = _lib.lib()

    def dispatch(x=P, dtype=0, H=64, r=R(), rows=OTHER):
        return L.kxw4_dispatch_rows(x, dtype, H, None if r is None else C.byref(r), rows, None)

    def combine(rows=P, rt=0, H=64, w=P, r=R(), y=OTHER, yt=0):
        return L.kxw4_combine_rows(rows, rt, H, w, None if r is None else C.byref(r), y, yt, None)

    def backward(dy=P, dt=0, rows=P, rt=0, H=64, w=P, r=R(), drows=OTHER, dw=P):
        return L.kxw4_combine_rows_backward(dy, dt, rows, rt, H, w, None if r is None else C.byref(r), drows, dw, None)

    for call in (dispatch, combine, backward):
        assert call(r=None) == _lib.EARG
        assert call(r=R(offsets=None)) == call(r=R(order=None)) == call(r=R(position=None)) == _lib.EPREP
        assert call(r=R(k=0)) == call(r=R(T=-3)) == call(r=R(groups=2000)) == _lib.ESHAPE
        assert call(H=0) == call(H=-8) == _lib.ESHAPE
        # no tokens: nothing to read or write, whatever the pointers
        assert call(r=R(T=0, offsets=None, order=None, position=None)) == 0
    assert dispatch(dtype=2) == combine(rt=2) == combine(yt=-1) == backward(dt=3) == backward(rt=3) == _lib.ESHAPE
    odd = C.c_void_p(65)
    assert dispatch(x=None) == dispatch(rows=None) == dispatch(x=odd) == dispatch(rows=odd) == _lib.EARG
    assert combine(rows=None) == combine(y=None) == combine(rows=odd) == combine(y=odd) == combine(w=odd) == _lib.EARG
    for name in ("dy", "rows", "w", "drows", "dw"):
        assert backward(**{name: None}) == backward(**{name: odd}) == _lib.EARG
    # an output in the place of an input
    assert dispatch(rows=P) == combine(y=P) == backward(drows=P) == _lib.EARG
    assert backward(rows=C.c_void_p(256), drows=C.c_void_p(256)) == _lib.EARG
    assert backward(drows=C.c_void_p(256), dw=P, w=P) == _lib.EARG


def test_expert_gemm_refuses_bad_arguments():
    f = _lib.lib().kxw4_expert_gemm

    def call(ws=(W(),), a=A(), r=R(), in_order=0, dtype=0, y=64, count=None):
        arr = (C.POINTER(_lib.Weight) * len(ws))(*[C.pointer(w) for w in ws])
        ys = (C.c_void_p * len(ws))(*[y] * len(ws))
        return f(arr, ys, len(ws) if count is None else count, None if a is None else C.byref(a),
                 None if r is None else C.byref(r), in_order, dtype, None)

    assert f(None, None, 1, C.byref(A()), C.byref(R()), 0, 0, None) == _lib.EARG
    assert call(count=0) == call(count=5) == call(a=None) == call(r=None) == call(y=None) == _lib.EARG
    assert call(ws=(W(codes=None),)) == _lib.EARG
    assert call(r=R(order=None)) == _lib.EPREP
    assert call(a=A(q=None)) == call(a=A(scale=None)) == _lib.EPREP
    # rows that the groups do not divide into 16-row slices, mixed weights
    assert call(r=R(groups=3)) == call(ws=(W(M=32),)) == _lib.ESHAPE
    assert call(ws=(W(), W(K=2048))) == call(ws=(W(), W(group=64))) == _lib.ESHAPE
    # activation rows: T, or T * k in sorted order
    assert call(a=A(T=16)) == call(in_order=1) == call(a=A(K=512)) == call(a=A(block=16)) == call(dtype=4) == _lib.ESHAPE
    # offsets past 31 bits
    assert call(a=A(T=1 << 22), r=R(T=1 << 22)) == _lib.ESHAPE
    # tiers that are not built for experts
    assert call(ws=(W(group=32),)) == call(ws=(W(enc=1),)) == call(a=A(block=32)) == _lib.ETIER
    assert call(ws=(W(group=128, enc=1),), a=A(block=32)) == call(ws=(W(group=16, enc=1),), a=A(block=32)) == _lib.ETIER
    assert call(ws=(W(group=32, enc=2),)) == _lib.ETIER                  # W8 has K32 activation blocks
    # one output for two weights, buffers off their alignment
    assert call(ws=(W(), W())) == call(y=72) == _lib.EARG
    assert call(a=A(q=72)) == call(a=A(scale=66)) == call(ws=(W(codes=72),)) == call(ws=(W(scales=72),)) == _lib.EARG
    assert call(ws=(W(group=32, enc=1),), a=A(block=32, scale=68)) == _lib.EARG
    assert call(r=R(T=0, offsets=None, order=None, position=None), a=A(T=0, q=None, scale=None), y=None) == 0


def test_expert_gemm_refuses_grids_past_two_to_the_32_threads():
    # W8 strips of 32 places x 64 rows: 2^25 slots x 2,048 rows come to 2^25
    # work-groups of 256 threads, of which a launch would leave none
    f = _lib.lib().kxw4_expert_gemm
    for rows in (2048, 1 << 14):
        w = W(M=8 * rows, K=1024, group=32, enc=2)
        arr, ys = (C.POINTER(_lib.Weight) * 1)(C.pointer(w)), (C.c_void_p * 1)(64)
        a, r = A(T=1 << 20, block=32), R(T=1 << 20, k=32, groups=8)
        assert f(arr, ys, 1, C.byref(a), C.byref(r), 0, 0, None) == _lib.ESHAPE


def test_adapter_add_refuses_bad_arguments():
    L = _lib.lib()

    def call(y=P, yt=1, x=OTHER, xt=1, ad=D(), r=R(k=1), out=P, ws=P):
        return L.kxw4_adapter_add(y, yt, x, xt, None if ad is None else C.byref(ad), None if r is None else C.byref(r),
                                  out, ws, None)

    assert call(ad=None) == call(r=None) == _lib.EARG
    assert call(r=R()) == call(r=R(k=1, groups=5)) == _lib.ESHAPE        # k = 2; another number of adapters
    for bad in (dict(r=0), dict(r=12), dict(r=264), dict(K=1000), dict(K=0), dict(M=250), dict(M=0)):
        assert call(ad=D(**bad)) == _lib.ESHAPE
    assert call(yt=2) == call(xt=2) == _lib.ESHAPE
    odd = C.c_void_p(72)
    for name in ("y", "x", "out", "ws"):
        assert call(ad=D(r=64), **{name: None}) == call(ad=D(r=64), **{name: odd}) == _lib.EARG
    for name in ("a", "b", "scale"):
        assert call(ad=D(**{name: None})) == _lib.EARG
    assert call(out=OTHER) == _lib.EARG                                  # out in the place of x
    assert call(ad=D(a=72)) == call(ad=D(b=72)) == call(ad=D(scale=66)) == _lib.EARG
    assert call(r=R(T=0, k=1, offsets=None, order=None, position=None), y=None, x=None, out=None, ws=None) == 0
    size = L.kxw4_adapter_workspace
    assert size(None, 8) == 0 and size(C.byref(D()), 0) == 0
    # two launches keep the low rows of every part between them, one nothing
    assert size(C.byref(D(r=64)), 8) % (8 * 64 * 4) == 0 and size(C.byref(D(r=64)), 8) >= 8 * 64 * 4
    assert size(C.byref(D()), 8) == 0 and size(C.byref(D(K=17408)), 8) > 0


def test_front_end_refuses_host_tensors():
    x = torch.zeros(4, 64)
    r = ops.RowRoute.empty(4, 2, 8, "cpu")
    with pytest.raises(ValueError, match="ids must be on the GPU"):
        ops.route_rows(torch.zeros(4, 2, dtype=torch.int32), 8)
    with pytest.raises(ValueError, match="x must be on the GPU"):
        ops.dispatch_rows(x, r)
    with pytest.raises(ValueError, match="rows must be on the GPU"):
        ops.combine_rows(x, r)
    with pytest.raises(ValueError, match="rows must be on the GPU"):
        ops.combine_rows_backward(x, x, r, torch.zeros(4, 2))
    with pytest.raises(ValueError, match="y must be on the GPU"):
        ops.adapter_add(x, x, None, r)
    with pytest.raises(ValueError, match="must be a torch.Tensor"):
        ops.route_rows([[1, 2]], 8)
    w = ops.W4Weight(64, 128, 128, 0, torch.zeros(64 * 64, dtype=torch.uint8), torch.zeros(64, dtype=torch.int16))
    with pytest.raises(ValueError, match="one to four weights, got 0"):
        ops.expert_gemm_fanout([], ops.QuantAct.empty(4, 128, 0, "cpu"), r)
    with pytest.raises(ValueError, match="one to four weights, got 5"):
        ops.expert_gemm_fanout([w] * 5, ops.QuantAct.empty(4, 128, 0, "cpu"), r)
    with pytest.raises(ValueError, match="weights must be on the GPU"):
        ops.expert_gemm(w, ops.QuantAct.empty(4, 128, 0, "cpu"), r)


def test_route_buffers_are_checked():
    r = ops.RowRoute.empty(4, 2, 8, "cpu")
    assert ops._check_route(r, torch.device("cpu")) is r
    with pytest.raises(ValueError, match="must be a RowRoute"):
        ops._check_route(None, torch.device("cpu"))
    with pytest.raises(ValueError, match="groups 0"):
        ops._check_route(ops.RowRoute(4, 2, 0, r.offsets, r.order, r.position), torch.device("cpu"))
    short = ops.RowRoute(4, 2, 9, r.offsets, r.order, r.position)
    with pytest.raises(ValueError, match="route offsets must have shape"):
        ops._check_route(short, torch.device("cpu"))
    wide = ops.RowRoute(4, 2, 8, r.offsets, r.order.long(), r.position)
    with pytest.raises(ValueError, match="route order must be torch.int32"):
        ops._check_route(wide, torch.device("cpu"))
    flat = ops.RowRoute(4, 2, 8, r.offsets, r.order, r.position.view(-1))
    with pytest.raises(ValueError, match="route position must have shape"):
        ops._check_route(flat, torch.device("cpu"))


def test_a_plan_is_checked_once_and_copied_whole():
    import copy
    import dataclasses
    import pickle
    cpu = torch.device("cpu")
    r = ops.RowRoute.empty(4, 2, 8, "cpu")
    ref = ops._plan(r, cpu)
    assert ops._plan(r, cpu) is ref
    with pytest.raises(ValueError, match="must be on"):
        ops._plan(r, torch.device("meta"))
    for name in ("T", "offsets"):
        with pytest.raises(dataclasses.FrozenInstanceError):
            setattr(r, name, getattr(r, name))
    for other in (copy.deepcopy(r), pickle.loads(pickle.dumps(r)), dataclasses.replace(r, order=r.order.clone())):
        assert ops._plan(other, cpu) is not ref
        c = ops._plan(other, cpu)._obj
        assert (c.T, c.k, c.groups, c.order) == (4, 2, 8, other.order.data_ptr()) and c.order != ref._obj.order
    with pytest.raises(ValueError, match="route order must have shape"):
        ops._plan(dataclasses.replace(r, order=r.order[:3]), cpu)


def test_a_checked_plan_follows_its_tensors():
    # a plan whose tensors were given other memory is checked anew
    cpu = torch.device("cpu")

    def checked():
        r = ops.RowRoute.empty(4, 2, 8, "cpu")
        ops._plan(r, cpu)
        return r

    for name in ("offsets", "order", "position"):
        size = getattr(checked(), name).shape
        for move in (lambda t: t.set_(torch.empty(size, dtype=torch.int32)),
                     lambda t: setattr(t, "data", torch.empty(size, dtype=torch.int32))):
            r = checked()
            move(getattr(r, name))
            assert getattr(ops._plan(r, cpu)._obj, name) == getattr(r, name).data_ptr()
        r = checked()
        getattr(r, name).resize_(4096)
        with pytest.raises(ValueError, match=f"route {name} must have shape"):
            ops._plan(r, cpu)
        r = checked()
        getattr(r, name).data = torch.empty(size, dtype=torch.int64)
        with pytest.raises(ValueError, match=f"route {name} must be torch.int32"):
            ops._plan(r, cpu)
        # memory that was given back: no address is left, which the C calls refuse
        r = checked()
        getattr(r, name).untyped_storage().resize_(0)
        assert not getattr(ops._plan(r, cpu)._obj, name)


def test_a_call_runs_on_its_tensors_device(monkeypatch):
    # the current device is 0; a call for device 1 makes that current around
    # the launch and takes its stream, and a failure names the function
    import contextlib
    seen, current = [], [0]

    @contextlib.contextmanager
    def device(i):
        before, current[0] = current[0], i
        yield
        current[0] = before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setitem(ops._FUNCTIONS, "call", lambda *args: seen.append((current[0], args)) or 0)
    monkeypatch.setitem(ops._FUNCTIONS, "fails", lambda *args: -2)
    ops._launch("call", torch.device("cuda:0"), 5)
    ops._launch("call", torch.device("cuda:1"), 6)
    assert seen == [(0, (5, 100)), (1, (6, 101))] and current == [0]
    with pytest.raises(_lib.KxError, match="fails"):
        ops._launch("fails", torch.device("cuda:1"))


def test_adapter_scratch_is_that_of_the_tensors_device(monkeypatch):
    # (two launches or one go by the CUs of the current device)
    import contextlib
    current = [0]

    @contextlib.contextmanager
    def device(i):
        before, current[0] = current[0], i
        yield
        current[0] = before

    class Library:
        @staticmethod
        def kxw4_adapter_workspace(ad, T):
            a = ad._obj
            return 1000 * current[0] + T + a.n + a.r + a.K + a.M

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(ops, "lib", lambda: Library)
    ops._adapter_bytes.cache_clear()
    for i in (0, 3, 0):
        assert ops._adapter_bytes(i, 2, 16, 128, 32, 5) == 1000 * i + 183 and current == [0]
    ops._adapter_bytes.cache_clear()


def test_sizes_past_32_bits_are_refused(monkeypatch):
    # (tensors without memory; a call that went on would reach the launch)
    monkeypatch.setattr(ops, "_gpu", lambda t, name: t.device)
    monkeypatch.setattr(ops, "_launch", lambda *args: pytest.fail("launched"))
    monkeypatch.setattr(ops, "_adapter_bytes", lambda *args: 0)
    meta = torch.device("meta")

    def empty(*shape, dtype=torch.float32):
        return torch.empty(shape, dtype=dtype, device=meta)

    for shape in ((1 << 32,), ((1 << 30) + 1, 1), (2, 1 << 32), (1 << 32, 2), (0, 1 << 32)):
        with pytest.raises(ValueError, match="up to 2\\^30 slots"):
            ops.route_rows(empty(*shape, dtype=torch.int32), 4)
    H = (1 << 32) + 64
    r = ops.RowRoute.empty(2, 1, 4, meta)
    for call in (lambda: ops.dispatch_rows(empty(2, H), r), lambda: ops.combine_rows(empty(2, H), r),
                 lambda: ops.combine_rows_backward(empty(2, H), empty(2, H), r, empty(2, 1))):
        with pytest.raises(ValueError, match="up to 2\\^28 elements"):
            call()
    for K, M in ((H, 64), (128, H)):
        ad = ops.Adapters(empty(4, 8, K, dtype=torch.bfloat16), empty(4, M, 8, dtype=torch.bfloat16), empty(4))
        with pytest.raises(ValueError, match="past 31 bits"):
            ops.adapter_add(empty(2, M), empty(2, K), ad, r)
