"""Low-rank adapters of many requests (csrc/kxw4_adapter.hip) against float64.

Tolerance. Products are exact. Each of the two sums takes at most 3 n FP32
additions for n terms (three parts of an FP32 value), each off by at most a
whole step 2^-23 of the running sum whatever the rounding of the matrix
instruction, plus one product with the scale and, in `low`, at most 32 + 4
partial sums. So with L = |A| |x|, `low` is off by (3 K + 37) 2^-23 L, and the
update by scale |B| times that, plus (3 r + 1) 2^-23 scale |B| |low|; adding y
rounds to half a step of the output's type."""
import numpy as np
import pytest
import torch

from knivesysl_xe_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
STEP = 2.0 ** -23


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def normal(rng, *shape, dtype=torch.float32):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)


def make(rng, n, r, K, M):
    a = (normal(rng, n, r, K) / K ** 0.5).to(torch.bfloat16)
    b = (normal(rng, n, M, r) / r ** 0.5).to(torch.bfloat16)
    return ops.Adapters(a.to(DEV), b.to(DEV), torch.from_numpy(rng.random(n).astype(np.float32) * 2).to(DEV))


def pick(rng, T, n, drop=0.2):
    ids = rng.integers(0, n, T)
    return np.where(rng.random(T) < drop, rng.choice([-1, n, n + 3]), ids).astype(np.int32)


def check(got, y, x, ad, ids):
    """`got` against y + scale B (A x) in float64, within the derived bound."""
    n, r, K = ad.a.shape
    A, B, scale = ad.a.double().cpu(), ad.b.double().cpu(), ad.scale.double().cpu()
    g, x64, y64 = got.double().cpu(), x.double().cpu(), y.double().cpu()
    for e in range(-1, n):
        at = torch.from_numpy(np.flatnonzero(ids == e if e >= 0 else (ids < 0) | (ids >= n)))
        if e < 0:
            assert torch.equal(got.cpu()[at], y.cpu()[at])
            continue
        if not len(at):
            continue
        xe = x64[at]
        low = xe @ A[e].t()
        want = y64[at] + scale[e] * (low @ B[e].t())
        off_low = (3 * K + 37) * STEP * (xe.abs() @ A[e].abs().t())
        off = scale[e] * (off_low @ B[e].abs().t() + (3 * r + 1) * STEP * (low.abs() @ B[e].abs().t()))
        off = off * 1.01 + HALF[got.dtype] * 1.01 * want.abs() + 1e-30
        bad = (g[at] - want).abs() > off
        assert not bad.any(), (e, len(at), int(bad.sum()), float((g[at] - want).abs().max()))


@pytest.mark.parametrize("T,n,r,K,M", [
    (1, 1, 8, 128, 16), (1, 5, 16, 1024, 64), (8, 8, 16, 5120, 5120), (13, 3, 24, 384, 80), (16, 1, 32, 256, 256),
    (17, 1, 32, 256, 272), (61, 24, 64, 2048, 512), (64, 64, 16, 640, 112), (65, 2, 8, 128, 1040), (100, 3, 128, 512, 144),
    (129, 200, 40, 256, 48), (300, 4, 256, 384, 96), (1000, 6, 16, 256, 1008), (70, 1024, 8, 128, 32), (5, 2, 200, 17408, 64),
    # many tokens, of few outputs
    (1536, 24, 16, 128, 1040), (1537, 1, 8, 256, 16), (2100, 6, 40, 256, 528), (1601, 3, 128, 384, 80), (3000, 2, 72, 128, 144),
    (1600, 3, 136, 128, 48), (1600, 30, 32, 128, 48),
    # with long rows of A
    (1537, 3, 24, 4096, 48), (1600, 40, 56, 4224, 32), (2003, 1, 128, 5120, 16)])
@pytest.mark.parametrize("x_t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("y_t", [torch.float32, torch.bfloat16])
def test_against_float64(T, n, r, K, M, x_t, y_t):
    rng = np.random.default_rng(T * r + M)
    ad = make(rng, n, r, K, M)
    ids = pick(rng, T, n)
    route = ops.route_rows(torch.from_numpy(ids).to(DEV), n)
    x, y = normal(rng, T, K, dtype=x_t).to(DEV), normal(rng, T, M, dtype=y_t).to(DEV)
    keep = y.clone()
    got = ops.adapter_add(y, x, ad, route)
    assert got.dtype is y_t and got.data_ptr() != y.data_ptr() and torch.equal(y, keep)
    check(got, y, x, ad, ids)
    # in place: the same bits, and rows without an adapter left alone
    assert ops.adapter_add(y, x, ad, route, out=y) is y
    assert torch.equal(y, got)


# 20 million outputs: B's rows in registers, one token tile for each CU and more
@pytest.mark.parametrize("T,n,r,K,M", [
    (1024, 16, 16, 128, 19536), (1025, 1, 8, 256, 19520), (1600, 24, 24, 128, 12512), (2100, 6, 40, 256, 9536),
    (1601, 3, 128, 384, 12512), (3000, 2, 72, 128, 6672), (4200, 3, 16, 128, 4768), (4300, 60, 24, 384, 4656),
    (5003, 40, 64, 256, 4000), (4500, 1, 128, 640, 4448)])
@pytest.mark.parametrize("x_t,y_t", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                     (torch.bfloat16, torch.bfloat16)])
def test_many_outputs(T, n, r, K, M, x_t, y_t):
    # (the first, the last and every 29th column against float64)
    rng = np.random.default_rng(T)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(T)
    a = torch.randn(n, r, K, generator=gen, device=DEV) / K ** 0.5
    b = torch.randn(n, M, r, generator=gen, device=DEV) / r ** 0.5
    ad = ops.Adapters(a.bfloat16(), b.bfloat16(), torch.rand(n, generator=gen, device=DEV) * 2)
    cols = torch.cat([torch.arange(130), torch.arange(130, M - 130, 29), torch.arange(M - 130, M)]).to(DEV)
    part = ops.Adapters(ad.a, ad.b[:, cols].contiguous(), ad.scale)
    for ids in (pick(rng, T, n), np.sort(pick(rng, T, n))[::-1], np.full(T, n - 1)):
        ids = np.ascontiguousarray(ids).astype(np.int32)
        x = torch.randn(T, K, generator=gen, device=DEV).to(x_t)
        y = torch.randn(T, M, generator=gen, device=DEV).to(y_t)
        route = ops.route_rows(torch.from_numpy(ids).to(DEV), n)
        got = ops.adapter_add(y, x, ad, route)
        check(got[:, cols], y[:, cols], x, part, ids)
        assert torch.equal(ops.adapter_add(y, x, ad, route, out=y), got)


@pytest.mark.parametrize("T", [3, 90, 700])
def test_one_adapter_for_all_none_for_all_and_packed_prompts(T):
    rng = np.random.default_rng(T)
    ad = make(rng, 6, 16, 512, 320)
    x, y = normal(rng, T, 512).to(DEV), normal(rng, T, 320).to(DEV)
    for ids in (np.full(T, 4), np.full(T, -1), np.sort(rng.integers(0, 6, T)), np.sort(rng.integers(0, 6, T))[::-1]):
        ids = np.ascontiguousarray(ids).astype(np.int32)
        check(ops.adapter_add(y, x, ad, ops.route_rows(torch.from_numpy(ids).to(DEV), 6)), y, x, ad, ids)


def test_large_and_small_values_and_infinities():
    rng = np.random.default_rng(9)
    ad = make(rng, 2, 16, 128, 32)
    ids = np.array([0, 1, 0, 1, -1], np.int32)
    route = ops.route_rows(torch.from_numpy(ids).to(DEV), 2)
    x = normal(rng, 5, 128).to(DEV)
    x[0] *= 1e30
    x[1] *= 1e-30
    y = normal(rng, 5, 32).to(DEV)
    check(ops.adapter_add(y, x, ad, route), y, x, ad, ids)
    # an infinity or NaN in x reaches the outputs of its own token only
    for bad in (float("inf"), float("nan")):
        z = x.clone()
        z[0] = 1.0
        z[1] = 1.0
        z[2, 5] = bad
        z[4, 0] = bad                                        # a token without an adapter
        got = ops.adapter_add(y, z, ad, route)
        assert not torch.isfinite(got[2]).any()
        want = ops.adapter_add(y, torch.where(torch.isfinite(z), z, 0.0), ad, route)
        for t in (0, 1, 3, 4):
            assert torch.equal(got[t], want[t])
    # a NaN of low mantissa bits only stays a NaN
    z = x.clone()
    z[3] = torch.full((128,), 0x7F800001, dtype=torch.int32, device=DEV).view(torch.float32)
    assert torch.isnan(ops.adapter_add(y, z, ad, route)[3]).all()


def test_beside_a_projection_captured():
    # quantize -> gemm -> adapters in place, as a decode step replays it
    rng = np.random.default_rng(11)
    T, n, K, M = 24, 5, 512, 256
    codes = torch.from_numpy(rng.integers(-8, 8, (M, K)).astype(np.int8)).to(DEV)
    bits = torch.from_numpy((np.abs(rng.standard_normal((M, K // 128))) * 0.02).astype(np.float16).view(np.int16)).to(DEV)
    w = ops.W4Weight.from_codes(codes, bits, 128, _lib.SCALE_FP16)
    ad = make(rng, n, 32, K, M)
    ids = torch.empty(T, dtype=torch.int32, device=DEV)
    x = torch.empty(T, K, dtype=torch.bfloat16, device=DEV)

    def fill():
        now = pick(rng, T, n)
        ids.copy_(torch.from_numpy(now))
        x.copy_(normal(rng, T, K, dtype=torch.bfloat16))
        return now

    def step():
        y = ops.gemm(w, ops.quantize_act(x, 0), torch.bfloat16)
        return ops.adapter_add(y, x, ad, ops.route_rows(ids, n), out=y)

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    for _ in range(4):
        now = fill()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, step())
        y = ops.gemm(w, ops.quantize_act(x, 0), torch.bfloat16)
        check(held, y, x, ad, now)
        torch.cuda.synchronize()


def test_front_end_refuses_mismatched_buffers():
    rng = np.random.default_rng(1)
    ad = make(rng, 3, 16, 256, 64)
    x, y = torch.zeros(4, 256, device=DEV), torch.zeros(4, 64, device=DEV)
    r = ops.route_rows(torch.zeros(4, dtype=torch.int32, device=DEV), 3)
    with pytest.raises(ValueError, match="y must have shape"):
        ops.adapter_add(torch.zeros(4, 80, device=DEV), x, ad, r)
    with pytest.raises(ValueError, match="x must have shape"):
        ops.adapter_add(y, x[:3].contiguous(), ad, r)
    with pytest.raises(ValueError, match="out must be torch.float32"):
        ops.adapter_add(y, x, ad, r, out=y.bfloat16())
    with pytest.raises(ValueError, match="4 groups and k 1 for 3 adapters"):
        ops.adapter_add(y, x, ad, ops.route_rows(torch.zeros(4, dtype=torch.int32, device=DEV), 4))
    # (a b of 128 rows asks for 128 columns of y)
    with pytest.raises(ValueError, match="y must have shape"):
        ops.adapter_add(y, x, ops.Adapters(ad.a, ad.b.view(3, 128, 8), ad.scale), r)
    with pytest.raises(ValueError, match="adapters.b must have shape"):
        ops.adapter_add(y, x, ops.Adapters(ad.a, ad.b[:2].contiguous(), ad.scale), r)
    with pytest.raises(_lib.KxError):
        ops.adapter_add(torch.zeros(4, 40, device=DEV), x, make(rng, 3, 16, 256, 40), r)
    assert ops.adapter_add(y[:0], x[:0], ad, ops.route_rows(torch.zeros(0, dtype=torch.int32, device=DEV), 3)).shape == (0, 64)


@pytest.mark.parametrize("T,n,r,K,M", [(8, 8, 16, 1024, 512), (61, 24, 64, 2048, 512), (2000, 3, 32, 512, 528),
                                       (2000, 3, 32, 512, 10000)])
def test_the_same_bits_every_time_two_streams_and_two_graphs(T, n, r, K, M):
    rng = np.random.default_rng(T)
    ad = make(rng, n, r, K, M)
    route = ops.route_rows(torch.from_numpy(pick(rng, T, n)).to(DEV), n)
    x = [normal(rng, T, K).to(DEV) for _ in range(2)]
    y = normal(rng, T, M).to(DEV)
    want = [ops.adapter_add(y, x[i], ad, route) for i in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, ops.adapter_add(y, x[i], ad, route)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in got)
    # two captured steps replayed side by side: each has scratch of its own
    graphs, outs = [], []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ops.adapter_add(y, x[i], ad, route))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_adapters_past_two_to_the_31_elements():
    n, r, K, M, T = 600, 256, 17408, 17408, 40               # 2.7e9 elements of a and of b
    gen = torch.Generator(device=DEV)
    gen.manual_seed(2)
    a = torch.randn(n, r, K, generator=gen, device=DEV, dtype=torch.bfloat16) / K ** 0.5
    b = torch.randn(n, M, r, generator=gen, device=DEV, dtype=torch.bfloat16) / r ** 0.5
    ad = ops.Adapters(a, b, torch.rand(n, generator=gen, device=DEV) + 0.5)
    ids = torch.tensor([599, 0, 598, 300, -1] * 8, dtype=torch.int32, device=DEV)
    x = torch.randn(T, K, generator=gen, device=DEV)
    y = torch.randn(T, M, generator=gen, device=DEV)
    got = ops.adapter_add(y, x, ad, ops.route_rows(ids, n))
    part = ops.Adapters(a[[0, 300, 598, 599]], b[[0, 300, 598, 599]], ad.scale[[0, 300, 598, 599]])
    local = np.array([{599: 3, 0: 0, 598: 2, 300: 1, -1: -1}[i] for i in ids.tolist()])
    check(got, y, x, part, local)
