"""Projections by expert (kxw4_expert_gemm) against float64 and, bit for bit,
against kxw4_gemm on each expert's own weight.

Tolerance against float64: the int32 unit partials are exact; an output is a
chain of one FP32 update per unit (K / group, or K / 32 with K32 blocks, where
the product of the two scales rounds once more), a sum over at most 16 splits
and one product with the token's scale. So it is off by at most (2 units + 18)
2^-24 times the sum of the units' magnitudes, and half a step of the output's
type."""
import numpy as np
import pytest
import torch

from knivesysl_xe_amd import _lib, ops
from test_gpu_rows import make_ids, plan_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
# group, activation block, scale encoding
MODES = {"token128": (128, 0, _lib.SCALE_FP16), "token64": (64, 0, _lib.SCALE_FP16),
         "block32": (32, 32, _lib.SCALE_FP16_ZP4), "block64": (64, 32, _lib.SCALE_FP16_ZP4),
         "w8": (32, 32, _lib.SCALE_W8)}


@pytest.fixture(autouse=True, scope="module")
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def weight(rng, mode, M, K):
    """(packed weight, its values [M][K / unit][unit] in float64)."""
    group, block, enc = MODES[mode]
    lim = (-128, 128) if mode == "w8" else (-8, 8)
    codes = rng.integers(*lim, (M, K)).astype(np.int8)
    bits = (np.abs(rng.standard_normal((M, K // group))) * 0.02).astype(np.float16).view(np.uint16)
    zero = np.zeros(bits.shape)
    if enc == _lib.SCALE_FP16_ZP4:
        z = rng.integers(-8, 8, bits.shape)
        bits = ((bits & 0xFFF0) | (z & 0xF)).astype(np.uint16)
        zero = z.astype(np.float64)
    scale = (bits & 0xFFF0 if enc == _lib.SCALE_FP16_ZP4 else bits).astype(np.uint16).view(np.float16).astype(np.float64)
    value = (codes.reshape(M, -1, group) - zero[..., None]) * scale[..., None]
    c, b = torch.from_numpy(codes).to(DEV), torch.from_numpy(bits.view(np.int16)).to(DEV)
    w = ops.W4Weight.from_codes_s8(c, b) if mode == "w8" else ops.W4Weight.from_codes(c, b, group, enc)
    return w, value.reshape(M, K)


def slice_of(w, e, groups):
    """Expert e's rows as a weight of their own."""
    n = w.codes.numel() // groups
    m = w.scales.numel() // groups
    return ops.W4Weight(w.M // groups, w.K, w.group, w.scale_enc, w.codes[e * n:(e + 1) * n].clone(),
                        w.scales[e * m:(e + 1) * m].clone())


def act_values(a):
    q = ops.act_codes_natural(a).double()
    s = a.scale.double()
    s = s[:, None] if a.block == 0 else s.repeat_interleave(32, 1)
    return (q * s).cpu().numpy()


def rows_of(a, at):
    return ops.QuantAct(len(at), a.K, a.block, a.q[at].contiguous(), a.scale[at].contiguous(), a.sum[at].contiguous())


def run(rng, mode, T, k, groups, K, Ms, dtype, in_order, ids=None):
    group, block, _ = MODES[mode]
    if ids is None:
        ids = make_ids(rng, T, k, groups)
    offsets, order, _ = plan_of(ids, groups)
    live = offsets[groups]
    N = T * k
    x = rng.standard_normal((N if in_order else T, K)).astype(np.float32)
    x[0] = 0.0
    a = ops.quantize_act(torch.from_numpy(x).to(DEV), block)
    ws = [weight(rng, mode, groups * M, K) for M in Ms]
    r = ops.route_rows(torch.from_numpy(ids).to(DEV), groups)
    outs = [torch.full((N, M), 3.0, dtype=dtype, device=DEV) for M in Ms]
    ys = ops.expert_gemm_fanout([w for w, _ in ws], a, r, dtype, sorted_rows=in_order, outs=outs)
    torch.cuda.synchronize()
    av = act_values(a)
    unit = 32 if block else group
    source = np.arange(N) if in_order else order // k
    for (w, value), y, M in zip(ws, ys, Ms):
        got = y.double().cpu().numpy()
        assert (got[live:] == 3.0).all()
        for e in range(groups):
            p = np.arange(offsets[e], offsets[e + 1])
            if not len(p):
                continue
            xe = av[source[p]].reshape(len(p), -1, unit)
            we = value[e * M:(e + 1) * M].reshape(M, -1, unit)
            part = np.matmul(xe.transpose(1, 0, 2), we.transpose(1, 2, 0))          # [units][rows][M]
            want, size = part.sum(0), np.abs(part).sum(0)
            tol = (2 * part.shape[0] + 18) * 2.0 ** -24 * size + HALF[dtype] * 1.01 * np.abs(want) + 1e-40
            bad = np.abs(got[p] - want) > tol
            assert not bad.any(), (e, len(p), int(bad.sum()), float(np.abs(got[p] - want).max()))
    return ws, a, r, ys, offsets, source


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("T,k,groups,K,Ms,in_order", [
    (1, 1, 1, 128, [16], False), (1, 1, 3, 256, [48, 16], True), (1, 8, 64, 1024, [64], False),
    (2, 4, 8, 384, [80], True), (7, 2, 5, 640, [16, 16, 32, 16], False), (16, 8, 16, 512, [112, 112], False),
    (33, 3, 4, 1152, [64], False), (90, 4, 40, 256, [144], True), (130, 6, 3, 384, [96], False),
    (1000, 2, 8, 256, [80], False), (70, 2, 200, 256, [32], False), (40, 1, 1024, 128, [16], True)])
def test_projections_of_every_tier(mode, T, k, groups, K, Ms, in_order):
    rng = np.random.default_rng(T * K + groups)
    run(rng, mode, T, k, groups, K, Ms, torch.float32, in_order)


@pytest.mark.parametrize("mode", ["token128", "token64", "block64", "w8"])
@pytest.mark.parametrize("T,groups,K,M", [(3, 4, 1024, 64), (37, 4, 5120, 32), (300, 2, 1024, 128), (1500, 3, 512, 272)])
def test_bfloat16_outputs(mode, T, groups, K, M):
    rng = np.random.default_rng(T + K)
    run(rng, mode, T, 2, groups, K, [M], torch.bfloat16, False)


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("T,groups,K,M", [(6, 4, 2048, 32), (50, 4, 1024, 64), (400, 3, 512, 80), (1200, 2, 384, 144)])
def test_a_row_has_the_bits_of_its_experts_own_projection(mode, T, groups, K, M):
    rng = np.random.default_rng(T * M)
    ws, a, r, (y,), offsets, source = run(rng, mode, T, 2, groups, K, [M], torch.float32, False)
    w = ws[0][0]
    same = []
    for splits in (1, 2, 4, 8, 16):
        equal = True
        for e in range(groups):
            p = np.arange(offsets[e], offsets[e + 1])
            own = ops.gemm(slice_of(w, e, groups), rows_of(a, torch.from_numpy(source[p]).to(DEV)), forced_splits=splits)
            equal = equal and torch.equal(own, y[offsets[e]:offsets[e + 1]])
        same.append(equal)
    assert any(same)


@pytest.mark.parametrize("mode,T,groups,K,Ms", [
    ("token128", 700, 40, 384, [144, 272]), ("token64", 700, 40, 384, [144, 272]),       # tiles of 32 places x 128 rows
    ("token128", 2100, 8, 256, [512, 496]), ("token64", 2100, 8, 256, [512, 496]),       # 64 x 256
    ("token128", 4150, 16, 128, [1040, 1040]), ("token64", 4150, 16, 128, [1040, 1040]),  # group 128: 128 x 256
    ("block32", 1600, 24, 256, [704, 688]), ("block64", 1600, 24, 256, [704, 688]),      # K32 blocks: 64 x 128
    ("block32", 3100, 100, 128, [512]),
])
def test_large_tiles(mode, T, groups, K, Ms):
    # uneven experts: some with no rows, one row, and most of them; the bits of
    # each expert's own projection in one split
    rng = np.random.default_rng(T)
    ids = make_ids(rng, T, 2, groups, 0.05)
    ids[ids == 1] = 0
    ids[ids == 2] = 0
    ids[T // 2, 1] = 2
    ws, a, r, ys, offsets, source = run(rng, mode, T, 2, groups, K, Ms, torch.float32, False, ids)
    for (w, _), y in zip(ws, ys):
        for e in range(groups):
            p = np.arange(offsets[e], offsets[e + 1])
            if not len(p):
                continue
            own = ops.gemm(slice_of(w, e, groups), rows_of(a, torch.from_numpy(source[p]).to(DEV)), forced_splits=1)
            assert torch.equal(own, y[offsets[e]:offsets[e + 1]]), e
    run(rng, mode, T, 2, groups, K, Ms, torch.bfloat16, True, ids)


@pytest.mark.parametrize("T", [9, 200, 2500])
def test_all_rows_to_one_expert_and_to_none(T):
    rng = np.random.default_rng(T)
    for e in (0, 6, 15):
        run(rng, "token128", T, 1, 16, 256, [48], torch.float32, False, np.full((T, 1), e, np.int32))
    # the same expert twice by one token, and no expert at all
    run(rng, "block32", T, 2, 16, 256, [48], torch.float32, False, np.full((T, 2), 3, np.int32))
    run(rng, "token64", T, 2, 16, 256, [48], torch.float32, False, np.full((T, 2), -1, np.int32))


def test_wide_k_and_many_rows():
    rng = np.random.default_rng(1)
    run(rng, "token128", 5, 2, 3, 17408, [32], torch.float32, False)
    run(rng, "block32", 3, 2, 2, 17408, [16], torch.float32, True)
    run(rng, "w8", 20, 2, 4, 5120, [1408], torch.bfloat16, False)


def test_an_expert_block_runs_together():
    # router -> gate and up -> SiLU -> down -> weighted sum, as a layer does,
    # eager and captured, against float64 on the library's own hidden codes
    rng = np.random.default_rng(8)
    T, k, groups, H, inner = 29, 4, 12, 512, 256
    gate, vg = weight(rng, "token128", groups * inner, H)
    up, vu = weight(rng, "token128", groups * inner, H)
    down, vd = weight(rng, "token128", groups * H, inner)
    ids = torch.empty(T, k, dtype=torch.int32, device=DEV)
    x = torch.empty(T, H, device=DEV)
    w = torch.empty(T, k, device=DEV)

    def fill():
        ids.copy_(torch.from_numpy(make_ids(rng, T, k, groups)))
        x.copy_(torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)))
        w.copy_(torch.from_numpy(rng.random((T, k)).astype(np.float32)))

    def layer():
        r = ops.route_rows(ids, groups)
        a = ops.quantize_act(x, 0)
        g, u = (torch.zeros(T * k, inner, device=DEV) for _ in range(2))
        ops.expert_gemm_fanout([gate, up], a, r, outs=[g, u])
        hidden, ha = ops.silu_mul_quant(g, u, 0)
        rows = ops.expert_gemm(down, ha, r, sorted_rows=True)
        return ops.combine_rows(rows, r, w), g, u, rows, r, a, ha

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = layer()[0]
    for _ in range(3):
        fill()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        y, g, u, rows, r, a, ha = layer()
        assert torch.equal(held, y)
        torch.cuda.synchronize()
    offsets, order, position = plan_of(ids.cpu().numpy(), groups)
    live = offsets[groups]
    av, hv = act_values(a), act_values(ha)
    want = np.zeros((T, H))
    for e in range(groups):
        for p in range(offsets[e], offsets[e + 1]):
            t, j = divmod(int(order[p]), k)
            xe = av[t]
            # (K / 128 = 4 units and fewer than 16 splits: see the tolerance above)
            for got, value in ((g, vg), (u, vu)):
                we = value[e * inner:(e + 1) * inner]
                size = np.abs(we.reshape(inner, -1, 128) * xe.reshape(1, -1, 128)).sum((1, 2))
                assert (np.abs(got[p].cpu().numpy() - we @ xe) <= 26 * 2.0 ** -24 * size).all()
            want[t] += float(w[t, j]) * (vd[e * H:(e + 1) * H] @ hv[p])
    big = np.abs(want).max()
    # (the sums above and k = 4 weighted terms: 2^-24 times a few dozen, with
    # the units' magnitudes at most ~20 times an output of the largest size)
    assert np.abs(y.cpu().numpy() - want).max() <= 30 * 20 * 2.0 ** -24 * big
    assert live < T * k


def test_another_stream():
    rng = np.random.default_rng(2)
    w, _ = weight(rng, "token128", 4 * 64, 512)
    ids = make_ids(rng, 50, 2, 4)
    x = torch.from_numpy(rng.standard_normal((50, 512)).astype(np.float32)).to(DEV)
    r = ops.route_rows(torch.from_numpy(ids).to(DEV), 4)
    a = ops.quantize_act(x, 0)
    want = ops.expert_gemm(w, a, r, out=torch.zeros(100, 64, device=DEV))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = torch.zeros(100, 64, device=DEV)
        got = ops.expert_gemm(w, a, ops.route_rows(torch.from_numpy(ids).to(DEV), 4), out=out)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("mode", ["token128", "block32"])
def test_weights_past_two_to_the_31_codes(mode):
    # the last experts' codes and scales lie past 32-bit offsets
    group, block, enc = MODES[mode]
    groups, M, K, T = 70, 2048, 17408, 9                     # 2.5e9 codes
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    codes = torch.randint(0, 256, (groups * M * K // 2,), generator=gen, device=DEV, dtype=torch.uint8)
    scales = (torch.rand(groups * M * (K // group), generator=gen, device=DEV) * 0.02).half().view(torch.int16)
    w = ops.W4Weight(groups * M, K, group, enc, codes, scales)
    ids = torch.tensor([0, 69, 68, 61, 69, 35, 60, 69, 1], dtype=torch.int32, device=DEV)
    r = ops.route_rows(ids, groups)
    a = ops.quantize_act(torch.randn(T, K, generator=gen, device=DEV), block)
    y = ops.expert_gemm(w, a, r)
    for e in (0, 60, 61, 68, 69):
        p0, p1 = int(r.offsets[e]), int(r.offsets[e + 1])
        tokens = r.order[p0:p1].long()
        own = [ops.gemm(slice_of(w, e, groups), rows_of(a, tokens), forced_splits=s) for s in (1, 2, 4, 8)]
        assert any(torch.equal(o, y[p0:p1]) for o in own), e


@pytest.mark.parametrize("mode,T,groups,K,M", [("token128", 40, 8, 1024, 64), ("w8", 300, 5, 512, 80),
                                               ("token64", 1500, 6, 256, 1040), ("block64", 1700, 24, 128, 1408)])
def test_the_same_bits_every_time_and_two_streams_at_once(mode, T, groups, K, M):
    rng = np.random.default_rng(T)
    group, block, _ = MODES[mode]
    w, _ = weight(rng, mode, groups * M, K)
    ids = torch.from_numpy(make_ids(rng, T, 2, groups)).to(DEV)
    a = ops.quantize_act(torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).to(DEV), block)
    r = ops.route_rows(ids, groups)
    want = ops.expert_gemm(w, a, r, out=torch.zeros(2 * T, M, device=DEV))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.expert_gemm(w, a, r, out=torch.zeros(2 * T, M, device=DEV)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


@pytest.mark.parametrize("mode", ["token128", "block32", "w8"])
def test_no_tokens(mode):
    rng = np.random.default_rng(4)
    w, _ = weight(rng, mode, 4 * 32, 256)
    r = ops.route_rows(torch.zeros(0, 3, dtype=torch.int64, device=DEV), 4)
    assert r.offsets.tolist() == [0] * 5
    a = ops.QuantAct.empty(0, 256, MODES[mode][1], DEV)
    assert ops.expert_gemm(w, a, r).shape == ops.expert_gemm(w, a, r, sorted_rows=True).shape == (0, 32)
