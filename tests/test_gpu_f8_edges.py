"""The 8-bit floating tier and the weights' gradient at their edges: outputs over their residual, two calls at once, two
captured graphs, tensors of another stream, hundreds of groups, and sizes whose offsets pass 32 bits."""
import pytest
import torch

from knivesysl_xe_amd import ops
from f8_ref import BF16, F32, exact_rows, exact_weight, gen, members, weight_values
from test_gpu_f8 import ids_of
from test_gpu_grad_weight import whole

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def needs(gb):
    if torch.cuda.mem_get_info()[0] < gb * 1e9:
        pytest.skip(f"needs {gb} GB of the GPU's memory")


# (stream kernel; large tiles; sums split over the columns; tiles of 256 rows)
@pytest.mark.parametrize("T,K,M", [(3, 272, 144), (200, 400, 528), (256, 8192, 512), (1100, 144, 16400)])
def test_an_output_may_be_its_residual(T, K, M):
    codes, scales = exact_weight(1, M, K, T)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = exact_rows(T, K, K)
    # (whole numbers below 2^10: every sum stays exact in float32)
    y = torch.randint(-1000, 1000, (T, M), generator=gen(1), device="cuda").float()
    product = x.double() @ weight_values(codes, scales)[0].t().contiguous()
    want = product + y.double()
    assert torch.equal(ops.gemm_f8(w, x, BF16, residual=y), want.to(F32).to(BF16))
    assert ops.gemm_f8(w, x, residual=y, out=y) is y
    assert torch.equal(y, want.float())


def test_residuals_that_are_refused():
    w = ops.F8Weight.from_codes(*[t[0] for t in exact_weight(1, 32, 128, 1)])
    x = exact_rows(4, 128, 1)
    r = torch.zeros(4, 32, device="cuda")
    with pytest.raises(ValueError, match="residual must have shape"):
        ops.gemm_f8(w, x, residual=r[:3])
    with pytest.raises(ValueError, match="records no gradient"):
        ops.gemm_f8(w, x, residual=r.clone().requires_grad_())
    with pytest.raises(ValueError, match="residual must be torch.float32"):
        ops.gemm_f8(w, x, residual=r.to(BF16))
    codes, scales = [t[0] for t in exact_weight(1, 32, 128, 1)]
    with pytest.raises(ValueError, match="records no gradient"):
        ops.F8Weight.from_codes(codes, scales.clone().requires_grad_())


def test_gradients_on_two_streams_at_once():
    # (a split sum, whose parts lie in a workspace)
    a = [(whole(9000, 64, i), whole(9000, 80, 9 + i)) for i in range(2)]
    want = [ops.grad_weight(*p) for p in a]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in a]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.grad_weight(*a[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_two_graphs_replayed_at_once_share_no_workspace():
    codes, scales = exact_weight(1, 512, 8192, 1)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    xs = [exact_rows(256, 8192, i) for i in range(2)]
    dys = [whole(9000, 64, 20 + i) for i in range(2)]
    rows = whole(9000, 80, 30)
    ys = [torch.zeros(256, 512, device="cuda") for _ in xs]
    dws = [torch.zeros(64, 80, device="cuda") for _ in xs]

    def step(i):
        ops.gemm_f8(w, xs[i], out=ys[i])                      # (quantized rows and parts of sums in the workspace)
        ops.grad_weight(dys[i], rows, out=dws[i])

    for i in range(2):
        step(i)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in xs]
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            step(i)
    streams = [torch.cuda.Stream() for _ in xs]
    for n in range(4):
        for i in range(2):
            xs[i].copy_(exact_rows(256, 8192, 40 + 2 * n + i))
            dys[i].copy_(whole(9000, 64, 60 + 2 * n + i))
            ys[i].zero_()
            dws[i].zero_()
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            got, got_dw = ys[i].clone(), dws[i].clone()
            step(i)
            torch.cuda.synchronize()
            assert torch.equal(got, ys[i]) and torch.equal(got_dw, dws[i])


def test_a_gradient_over_itself_in_a_graph():
    # accumulation: each replay adds to what the last one left
    dy, x = whole(300, 144, 1), whole(300, 272, 2)
    long_dy, long_x = whole(9000, 64, 3), whole(9000, 80, 4)
    dw, long_dw = torch.zeros(144, 272, device="cuda"), torch.zeros(64, 80, device="cuda")

    def step():
        ops.grad_weight(dy, x, add=dw, out=dw)
        ops.grad_weight(long_dy, long_x, add=long_dw, out=long_dw)

    step()
    torch.cuda.synchronize()
    one = [dw.clone(), long_dw.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    dw.zero_()
    long_dw.zero_()
    for n in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        # (whole numbers: sums of 9,000 products below 2^7, four times over, stay below 2^24)
        assert torch.equal(dw, one[0] * n) and torch.equal(long_dw, one[1] * n)


def test_tensors_of_another_stream():
    codes, scales = exact_weight(4, 144, 256, 3)
    w, t = ops.F8Weight.from_codes(codes, scales), ops.F8Weight.from_codes(codes, scales).transposed()
    ids = ids_of(90, 2, 4, 0.1, 5)
    x = exact_rows(90, 256, 1)
    route = ops.route_rows(ids, 4)
    end = int(route.offsets[-1])
    want = ops.expert_gemm_f8(w, x, route)[:end].clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        r = ops.route_rows(ids, 4)
        y = ops.expert_gemm_f8(w, x, r)
        q = ops.quantize_act_f8(y[:end].contiguous())
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y[:end], want)
    assert torch.equal(q.q, ops.quantize_act_f8(want).q)
    assert t.M == 256 and t.K == 144


# ---- many groups -----------------------------------------------------------

@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("T,k,E,K,M,skew", [(3000, 4, 65, 144, 272, 0.0), (2500, 2, 1024, 128, 16, 2.0), (6000, 3, 300, 16, 144, 3.0),
                                            (9000, 4, 130, 128, 272, 0.5)])
def test_products_and_gradients_of_many_groups(T, k, E, K, M, skew, out):
    codes, scales = exact_weight(E, M, K, T)
    w = ops.F8Weight.from_codes(codes, scales)
    ids = ids_of(T, k, E, 0.1, 7, skew)
    route = ops.route_rows(ids, E)
    end = int(route.offsets[-1])
    x = exact_rows(T * k, K, 1)
    y = ops.expert_gemm_f8(w, x, route, out, sorted_rows=True)
    dy, rows = whole(T * k, M, 2), whole(T * k, K, 3)
    dw = ops.expert_grad_weight(dy, rows, route, out)
    offsets = route.offsets.tolist()
    wv = weight_values(codes, scales)
    for e in range(E):
        a, b = offsets[e], offsets[e + 1]
        assert torch.equal(dw[e], (dy[a:b].double().t().contiguous() @ rows[a:b].double()).to(out)), e
        if a < b:
            assert torch.equal(y[a:b], (x[a:b].double() @ wv[e].t().contiguous()).to(out)), e
    assert end == offsets[E]


# ---- offsets past 32 bits ---------------------------------------------------

def test_weights_past_32_bits():
    # 70 experts of 67 MB: the last ones' codes lie past 2^32
    E, M, K = 70, 4096, 16384
    needs(30)
    codes = torch.zeros(E, M, K, dtype=torch.uint8, device="cuda")
    scales = torch.ones(E, M // 128, K // 128, device="cuda")
    some, _ = exact_weight(2, M, K, 1)
    codes[66:68] = some.view(torch.uint8)
    w = ops.F8Weight.from_codes(codes, scales)
    assert torch.equal(w.unpack()[0][66:68].view(torch.uint8), codes[66:68])
    back = w.transposed().transposed()
    assert torch.equal(back.codes.view(E, -1)[66:68], w.codes.view(E, -1)[66:68])
    del back
    wv = some.double()
    for T in (8, 200):                                        # (weights' stream, large tiles)
        ids = torch.full((T, 1), 66, dtype=torch.int32, device="cuda")
        ids[T // 2:] = 67
        route = ops.route_rows(ids, E)
        x = exact_rows(T, K, T)
        for out in (F32, BF16):
            y = ops.expert_gemm_f8(w, x, route, out)
            want = torch.cat([x[:T // 2].double() @ wv[0].t().contiguous(), x[T // 2:].double() @ wv[1].t().contiguous()])
            assert torch.equal(y, want.to(out)), (T, out)


@pytest.mark.parametrize("out", [F32, BF16])
def test_rows_and_outputs_past_32_bits(out):
    # 4.6e9 codes of rows, then 2.3e9 outputs
    needs(60)
    T, K = 280_001, 16384
    codes, scales = exact_weight(1, 32, K, 1)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = torch.zeros(T, K, dtype=BF16, device="cuda")
    x[-300:] = exact_rows(300, K, 2, BF16)
    y = ops.gemm_f8(w, x, out)
    want = x[-300:].double() @ weight_values(codes, scales)[0].t().contiguous()
    assert torch.equal(y[-300:], want.to(out)) and not y[:-300].any()
    del x, y
    T, K, M = 70_001, 128, 33_008
    codes, scales = exact_weight(1, M, K, 3)
    w = ops.F8Weight.from_codes(codes[0], scales[0])
    x = exact_rows(T, K, 4, BF16)
    y = ops.gemm_f8(w, x, out)
    wv = weight_values(codes, scales)[0].t().contiguous()
    for a in (0, 35_000, T - 700):
        assert torch.equal(y[a:a + 700], (x[a:a + 700].double() @ wv).to(out))


@pytest.mark.parametrize("out", [F32, BF16])
def test_gradients_past_32_bits(out):
    # rows of 2.5e9 values: the last group's lie past 2^31 elements
    needs(80)
    N, M, K = 150_000, 16_400, 48
    dy = torch.zeros(N, M, dtype=BF16, device="cuda")
    dy[-400:] = whole(400, M, 1)
    x = whole(N, K, 2)
    ids = torch.zeros(N, 1, dtype=torch.int32, device="cuda")
    ids[-400:] = 2
    dw = ops.expert_grad_weight(dy, x, ops.route_rows(ids, 3), out)
    assert not dw[:2].any()
    want = dy[-400:].double().t().contiguous() @ x[-400:].double()
    assert torch.equal(dw[2], want.to(out))
    assert torch.equal(ops.grad_weight(dy, x, out), want.to(out))
    del dy, dw
    # 4.3e9 gradients: the last group's lie past 2^32
    E, M, K = 65, 8192, 8192
    dy, x = whole(E * 3, M, 3), whole(E * 3, K, 4)
    ids = torch.arange(E, device="cuda", dtype=torch.int32).repeat_interleave(3).view(-1, 1).contiguous()
    dw = ops.expert_grad_weight(dy, x, ops.route_rows(ids, E), out)
    for e in (0, 33, 64):
        want = dy[3 * e:3 * e + 3].float().t().contiguous() @ x[3 * e:3 * e + 3].float()
        assert torch.equal(dw[e], want.to(out)), e


def test_weight_blocks_of_more_threads_than_a_launch():
    # 33.5 million blocks of 256 threads
    needs(160)
    E, M, K = 1024, 16, 1 << 22
    codes = torch.empty(E, M, K, dtype=torch.uint8, device="cuda")
    some = torch.randint(0, 127, (3, M, K), generator=gen(1), device="cuda", dtype=torch.uint8)
    codes[0], codes[600], codes[-1] = some[0], some[1], some[2]
    w = ops.F8Weight(E, M, K, torch.empty(E * M * K, dtype=torch.uint8, device="cuda"), torch.ones(E, 1, K // 128, device="cuda"))
    ops._launch("kxw4_pack_weight_f8", w.codes.device, codes.data_ptr(), E, M, K, w.codes.data_ptr())
    for i, e in enumerate((0, 600, E - 1)):
        one = ops.F8Weight.from_codes(some[i], torch.ones(1, K // 128, device="cuda"))
        assert torch.equal(w.codes.view(E, -1)[e], one.codes), e
