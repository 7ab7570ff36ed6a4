"""Rows sorted by the group each slot names, and back (csrc/kxw4_rows.hip):
the plan against a stable sort in numpy, exactly; dispatch bit for bit; the
weighted sums and their gradient against float64.

Tolerances. A sum of n FP32 terms in any order is off by at most n 2^-24 times
the sum of the terms' magnitudes (to first order; products inside an fma are
exact); the output's own rounding adds half a step of its type: 2^-24 relative
for float32, 2^-8 for bfloat16."""
import numpy as np
import pytest
import torch

from knivesysl_xe_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def plan_of(ids, groups):
    """(offsets, order, position) by numpy's stable sort."""
    flat = ids.reshape(-1).astype(np.int64)
    key = np.where((flat < 0) | (flat >= groups), groups, flat)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(groups + 1))
    position = np.full(flat.size, -1)
    live = offsets[groups]
    position[order[:live]] = np.arange(live)
    return offsets, order, position.reshape(ids.shape)


def make_ids(rng, T, k, groups, drop=0.2, dtype=np.int32):
    ids = rng.integers(0, groups, (T, k))
    ids = np.where(rng.random((T, k)) < drop, rng.choice([-1, groups, groups + 7, -5]), ids)
    return ids.astype(dtype)


def route(ids, groups):
    return ops.route_rows(torch.from_numpy(ids).to(DEV), groups)


def check_plan(r, ids, groups, what=""):
    offsets, order, position = plan_of(ids, groups)
    assert np.array_equal(r.offsets.cpu().numpy(), offsets), what
    assert np.array_equal(r.order.cpu().numpy(), order), what
    assert np.array_equal(r.position.cpu().numpy(), position), what


@pytest.mark.parametrize("T,k,groups", [
    (1, 1, 1), (1, 8, 8), (3, 1, 1024), (7, 2, 3), (64, 1, 64), (63, 1, 63), (65, 1, 65), (511, 1, 5), (513, 3, 127),
    (2048, 8, 128), (2049, 8, 128), (4096, 4, 256), (4097, 4, 255), (16384, 1, 1), (16385, 1, 2), (9001, 6, 61),
    (131073, 8, 64), (40000, 2, 1024)])
@pytest.mark.parametrize("wide", [False, True])
def test_plan_is_the_stable_sort(T, k, groups, wide):
    rng = np.random.default_rng(T + groups)
    ids = make_ids(rng, T, k, groups, dtype=np.int64 if wide else np.int32)
    check_plan(route(ids, groups), ids, groups)


@pytest.mark.parametrize("T", [1, 70, 5000, 20000])
def test_plan_of_one_group_of_none_and_sorted_ids(T):
    for ids in (np.full((T, 2), 3), np.full((T, 2), -1), np.arange(2 * T).reshape(T, 2) % 16,
                np.sort(np.arange(2 * T) % 16).reshape(T, 2)):
        ids = ids.astype(np.int32)
        check_plan(route(ids, 16), ids, 16)


def test_plan_of_far_ids_and_no_tokens():
    # 64-bit ids that are valid once cut to 32 bits name no group
    ids = np.array([[1 << 32, 2], [(1 << 33) + 1, -(1 << 40)], [0, 3]], np.int64)
    check_plan(route(ids, 4), ids, 4)
    for shape in ((0, 3), (0,)):
        r = ops.route_rows(torch.empty(shape, dtype=torch.int32, device=DEV), 9)
        assert r.offsets.cpu().tolist() == [0] * 10 and r.order.numel() == 0
        x = torch.empty(0, 40, device=DEV)
        assert ops.dispatch_rows(x, r).shape == (0, 40)
        assert ops.combine_rows(x, r).shape == (0, 40)
        d, dw = ops.combine_rows_backward(x, x, r, torch.empty(0, r.k, device=DEV))
        assert d.shape == (0, 40) and dw.shape == (0, r.k)


def test_plan_buffers_are_reused():
    rng = np.random.default_rng(5)
    r = ops.RowRoute.empty(300, 4, 32, DEV)
    for _ in range(3):
        ids = make_ids(rng, 300, 4, 32)
        assert ops.route_rows(torch.from_numpy(ids).to(DEV), 32, out=r) is r
        check_plan(r, ids, 32)


SHAPES = [(1, 1, 4, 8), (1, 8, 8, 5120), (5, 3, 7, 1), (13, 2, 4, 64), (64, 8, 16, 2048), (301, 6, 61, 2049),
          (77, 5, 9, 130), (33, 4, 8, 17408), (257, 1, 8, 1000), (40, 13, 16, 24)]


@pytest.mark.parametrize("T,k,groups,H", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dispatch_copies_rows_and_leaves_the_rest(T, k, groups, H, dtype):
    rng = np.random.default_rng(T * H)
    ids = make_ids(rng, T, k, groups)
    r = route(ids, groups)
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(DEV).to(dtype)
    out = torch.full((T * k, H), 7.0, device=DEV, dtype=dtype)
    assert ops.dispatch_rows(x, r, out=out) is out
    offsets, order, _ = plan_of(ids, groups)
    live = offsets[groups]
    want = torch.full((T * k, H), 7.0, dtype=dtype)
    want[:live] = x.cpu()[order[:live] // k]
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("T,k,groups,H", SHAPES)
@pytest.mark.parametrize("rows_t,y_t", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                        (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_combine_and_its_gradient(T, k, groups, H, rows_t, y_t):
    rng = np.random.default_rng(T * H + 1)
    ids = make_ids(rng, T, k, groups)
    r = route(ids, groups)
    offsets, order, position = plan_of(ids, groups)
    live = offsets[groups]
    rows = torch.from_numpy(rng.standard_normal((T * k, H)).astype(np.float32)).to(rows_t)
    rows[live:] = float("nan")                               # rows of no slot are not read
    weights = torch.from_numpy(rng.random((T, k)).astype(np.float32))
    dy = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(y_t)
    on = torch.from_numpy(position >= 0)
    picked = rows.double()[torch.from_numpy(position).clamp(min=0)]
    picked = torch.where(on[..., None], picked, torch.zeros(()).double())          # [T][k][H]

    for w in (weights, None):
        terms = picked * (w.double()[..., None] if w is not None else 1.0)
        want, size = terms.sum(1), terms.abs().sum(1)
        y = ops.combine_rows(rows.to(DEV), r, None if w is None else w.to(DEV), dtype=y_t)
        assert y.dtype is y_t and y.shape == (T, H)
        off = (y.cpu().double() - want).abs()
        assert (off <= k * 2.0 ** -24 * size + HALF[y_t] * want.abs() * 1.01 + 1e-40).all()

    out = torch.full((T * k, H), 5.0, device=DEV, dtype=rows_t)
    drows, dw = ops.combine_rows_backward(dy.to(DEV), rows.to(DEV), r, weights.to(DEV), out=out)
    assert drows is out
    slot = torch.from_numpy(order[:live])
    want = weights.double().reshape(-1)[slot][:, None] * dy.double()[slot // k]
    got = drows.cpu().double()
    # (one FP32 product, then the rounding to rows' type)
    assert ((got[:live] - want).abs() <= (HALF[rows_t] + 2.0 ** -24) * 1.01 * want.abs() + 1e-40).all()
    assert (got[live:] == 5.0).all()
    terms = picked * dy.double()[:, None, :]
    off = (dw.cpu().double() - terms.sum(2)).abs()
    assert (off <= H * 2.0 ** -24 * terms.abs().sum(2) + 1e-40).all()
    assert (dw.cpu()[~on] == 0).all()


def test_gradients_against_differences():
    # combine is linear in rows and in weights: a difference of two calls is
    # the gradient's inner product with the step
    rng = np.random.default_rng(3)
    T, k, groups, H = 19, 3, 5, 48
    ids = make_ids(rng, T, k, groups)
    r = route(ids, groups)

    def normal(*shape):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(DEV)

    rows, w, dy, x = normal(T * k, H), normal(T, k), normal(T, H), normal(T, H)
    srows, sw, sx = normal(T * k, H), normal(T, k), normal(T, H)
    n = int(r.offsets[-1])
    drows, dw = ops.combine_rows_backward(dy, rows, r, w)

    def loss(a, b):
        return (ops.combine_rows(a, r, b).double() * dy.double()).sum()

    # (each side sums T*H <= 912 products of values of order 1: 1e-3 holds
    # 912 * 10 * 2^-24 = 5e-4 of rounding)
    assert abs((loss(rows + srows, w) - loss(rows, w)) - (drows[:n].double() * srows[:n].double()).sum()) < 1e-3
    assert abs((loss(rows, w + sw) - loss(rows, w)) - (dw.double() * sw.double()).sum()) < 1e-3
    g = normal(T * k, H)
    dx = ops.dispatch_rows_backward(g, r)
    moved = ops.dispatch_rows(sx, r)
    assert abs((moved[:n].double() * g[:n].double()).sum() - (dx.double() * sx.double()).sum()) < 1e-3


def test_unaligned_rows_take_narrower_pieces():
    rng = np.random.default_rng(4)
    T, k, groups, H = 21, 2, 4, 64
    ids = make_ids(rng, T, k, groups)
    r = route(ids, groups)
    flat = torch.from_numpy(rng.standard_normal(T * k * H + 3).astype(np.float32)).to(DEV)
    for dtype in (torch.float32, torch.bfloat16):
        base = flat.to(dtype)
        for shift in (1, 2, 3):
            rows = base[shift:shift + T * k * H].view(T * k, H)
            x = base[shift:shift + T * H].view(T, H)
            assert torch.equal(ops.combine_rows(rows, r), ops.combine_rows(rows.clone(), r))
            live = int(r.offsets[-1])
            assert torch.equal(ops.dispatch_rows(x, r)[:live], ops.dispatch_rows(x.clone(), r)[:live])
            w = torch.rand(T, k, device=DEV)
            got, want = ops.combine_rows_backward(x, rows, r, w), ops.combine_rows_backward(x.clone(), rows.clone(), r, w)
            assert torch.equal(got[0][:live], want[0][:live])
            # (the two walk the row in different strides: two sums of 64 terms)
            assert ((got[1] - want[1]).abs() <= 2 * H * 2.0 ** -24 * 64 * 16).all()


def test_infinities_and_nan_stay_where_they_are():
    ids = np.array([[0, 1], [1, -1]], np.int32)
    r = route(ids, 2)
    rows = torch.tensor([[1.0, float("inf"), 2.0], [3.0, 1.0, float("nan")], [float("-inf"), 4.0, 5.0]], device=DEV)
    rows = torch.cat([rows, torch.full((1, 3), float("nan"), device=DEV)])
    for dtype in (torch.float32, torch.bfloat16):
        y = ops.combine_rows(rows.to(dtype), r, torch.ones(2, 2, device=DEV)).float().cpu()
        assert y[0, 0] == 4 and y[0, 1] == float("inf") and torch.isnan(y[0, 2])
        assert y[1].tolist() == [float("-inf"), 4.0, 5.0]
    # NaNs of low mantissa bits only are not rounded to infinity
    quiet = torch.full((4, 8), 0x7F800001, dtype=torch.int32, device=DEV).view(torch.float32)
    assert torch.isnan(ops.combine_rows(quiet, r, dtype=torch.bfloat16)).all()


def test_another_stream_and_a_captured_step():
    rng = np.random.default_rng(6)
    T, k, groups, H = 37, 4, 16, 256
    ids = torch.empty(T, k, dtype=torch.int32, device=DEV)
    x = torch.empty(T, H, device=DEV)
    w = torch.empty(T, k, device=DEV)

    def fill():
        ids.copy_(torch.from_numpy(make_ids(rng, T, k, groups)))
        x.copy_(torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)))
        w.copy_(torch.from_numpy(rng.random((T, k)).astype(np.float32)))

    def step():
        r = ops.route_rows(ids, groups)
        rows = ops.dispatch_rows(x, r, out=torch.zeros(T * k, H, device=DEV))
        y = ops.combine_rows(rows, r, w)
        return r.offsets, r.order, r.position, rows, y, *ops.combine_rows_backward(y, rows, r, w, out=torch.zeros_like(rows))

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.synchronize()
    for _ in range(4):
        fill()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(held, step()):
            assert torch.equal(got, want)
        torch.cuda.synchronize()


def test_rows_past_two_to_the_31_elements():
    T, k, groups, H = 66000, 8, 37, 4160                     # 2.2e9 elements of rows
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1)
    ids = torch.randint(-1, groups, (T, k), generator=gen, device=DEV, dtype=torch.int32)
    r = ops.route_rows(ids, groups)
    check_plan(r, ids.cpu().numpy(), groups)
    x = torch.randn(T, H, generator=gen, device=DEV, dtype=torch.bfloat16)
    w = torch.rand(T, k, generator=gen, device=DEV)
    rows = ops.dispatch_rows(x, r)
    live = int(r.offsets[-1])
    at = torch.cat([torch.arange(100), torch.randint(0, live, (300,)), torch.arange(live - 100, live)]).to(DEV)
    assert torch.equal(rows[at], x[r.order[at].long() // k])
    y = ops.combine_rows(rows, r, w, dtype=torch.float32)
    tokens = torch.cat([torch.arange(50), torch.arange(T - 50, T)]).to(DEV)
    # every row of a token is its own x: y = x times the sum of its weights
    want = x[tokens].double() * torch.where(r.position[tokens] >= 0, w[tokens], 0.0).double().sum(1, keepdim=True)
    assert ((y[tokens].double() - want).abs() <= (k + 1) * 2.0 ** -24 * k * x[tokens].double().abs()).all()
    drows, dw = ops.combine_rows_backward(x, rows, r, w)
    slot = r.order[at].long()
    assert torch.equal(drows[at], (w.reshape(-1)[slot][:, None] * x[slot // k].float()).bfloat16())
    norm = (x[tokens].double() ** 2).sum(1, keepdim=True)
    off = (dw[tokens].double() - torch.where(r.position[tokens] >= 0, norm, 0.0)).abs()
    assert (off <= H * 2.0 ** -24 * norm).all()


def test_calls_at_once_on_two_streams():
    # the same inputs and plans, each call with scratch of its own
    rng = np.random.default_rng(7)
    T, k, groups, H = 20000, 2, 100, 320
    ids = [torch.from_numpy(make_ids(rng, T, k, groups)).to(DEV) for _ in range(2)]
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(DEV)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                r = ops.route_rows(ids[i], groups)
                rows = ops.dispatch_rows(x, r, out=torch.zeros(T * k, H, device=DEV))
                got[i].append((r, rows, ops.combine_rows(rows, r)))
    torch.cuda.synchronize()
    for i in range(2):
        check_plan(got[i][0][0], ids[i].cpu().numpy(), groups)
        for r, rows, y in got[i]:
            assert torch.equal(r.order, got[i][0][0].order) and torch.equal(rows, got[i][0][1])
            assert torch.equal(y, got[i][0][2])


def test_every_float32_pattern_rounds_to_the_nearest_bfloat16():
    # random bit patterns (subnormals, ties, infinities and NaNs among them);
    # one choice without weights: y = 1 * x + 0
    rng = np.random.default_rng(12)
    bits = rng.integers(0, 1 << 32, (4096, 512), dtype=np.uint64).astype(np.uint32)
    bits[0] = np.arange(512, dtype=np.uint32) << 7           # subnormals
    bits[1] |= 0x7F000000                                    # large ones, infinities, NaNs
    bits[2] = (bits[2] & 0xFFFF0000) | 0x8000                # ties
    x = torch.from_numpy(bits.view(np.float32)).to(DEV)
    r = ops.route_rows(torch.arange(4096, device=DEV) % 7, 7)
    y = ops.combine_rows(ops.dispatch_rows(x, r), r, dtype=torch.bfloat16)
    want = x.bfloat16()
    assert ((y == want) | (torch.isnan(y) & torch.isnan(want))).all()


def test_plans_passed_as_out_are_checked():
    import dataclasses
    ids = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="must be a RowRoute"):
        ops.route_rows(ids, 8, out=(4, 2, 8))
    with pytest.raises(ValueError, match="does not match"):
        ops.route_rows(ids, 8, out=ops.RowRoute.empty(4, 2, 9))
    r = ops.RowRoute.empty(4, 2, 8)
    with pytest.raises(ValueError, match="route position must be torch.int32"):
        ops.route_rows(ids, 8, out=dataclasses.replace(r, position=r.position.float()))
    with pytest.raises(ValueError, match="must be on the GPU|must be on cuda"):
        ops.route_rows(ids, 8, out=ops.RowRoute.empty(4, 2, 8, "cpu"))
