"""64-bit references and inputs of the tests of the 8-bit floating tier."""
import torch

from knivesysl_xe_amd import ops

BF16, F32 = torch.bfloat16, torch.float32
F8 = torch.float8_e4m3fn


def blocks(n):
    return (n + 127) // 128


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def expand(scales, M, K):
    """[..][MB][KB] -> [..][M][K]"""
    return scales.repeat_interleave(128, -2)[..., :M, :].repeat_interleave(128, -1)[..., :K]


def weight_values(codes, scales):
    M, K = codes.shape[-2:]
    return codes.double() * expand(scales, M, K).double()


def quantized(x):
    """(codes [T][K] float8, scales [KB][T]) by the rule, in float32."""
    T, K = x.shape
    kb = blocks(K)
    v = torch.zeros(T, kb * 128, device=x.device)
    v[:, :K] = x.float()
    v = v.view(T, kb, 128)
    top = v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    q = (v * (torch.full_like(top, 448.0) / top)).to(F8)
    return q.view(T, -1)[:, :K], (top / torch.full_like(top, 448.0)).squeeze(-1).t().contiguous()


def row_values(x):
    q, s = quantized(x)
    return q.double() * s.t().repeat_interleave(128, 1)[:, :x.shape[1]].double()


def exact_weight(groups, M, K, seed):
    """Codes that are small whole numbers and scales that are powers of two: with exact_rows every product, partial sum and
    scaled sum is a multiple of 1/4 below 2^22, so any order of float32 sums gives it exactly, and so does a matrix core
    that cuts products to 2^-13 of the largest near them (products below 2^13, multiples of 1)."""
    g = gen(seed)
    codes = torch.randint(-15, 16, (groups, M, K), generator=g, device="cuda").float().to(F8)
    scales = 2.0 ** torch.randint(-1, 1, (groups, blocks(M), blocks(K)), generator=g, device="cuda").float()
    return codes, scales


def exact_rows(T, K, seed, dtype=F32):
    """Rows whose quantization is exact with scale 1 or 1/2: the first column of each block is the block's largest, 448
    times the scale; the others are whole multiples of the scale."""
    g = gen(seed)
    x = torch.randint(-15, 16, (T, K), generator=g, device="cuda").float()
    x[:, ::128] = 448.0
    s = 2.0 ** torch.randint(-1, 1, (T, blocks(K)), generator=g, device="cuda").float()
    return (x * s.repeat_interleave(128, 1)[:, :K]).to(dtype)


def normal_weight(groups, M, K, seed):
    g = gen(seed)
    w = torch.randn(groups, M, K, generator=g, device="cuda") * K ** -0.5
    scales = torch.empty(groups, blocks(M), blocks(K), device="cuda")
    padded = torch.zeros(groups, blocks(M) * 128, blocks(K) * 128, device="cuda")
    padded[:, :M, :K] = w
    scales[:] = padded.view(groups, blocks(M), 128, blocks(K), 128).abs().amax((2, 4)) / 448.0
    return (w / expand(scales, M, K)).to(F8), scales


def bound(x_values, w_values, y, out, few):
    """How far an output may be from its value y: FP32 sums of exact products (128 of a block and its block sums, each
    addition off by at most 2^-23 of the sum of magnitudes, the combined scale by 2^-24), the matrix core's cut with bf16
    outputs and many rows (eight products of a group, each by less than 2^-13 of the largest: 2^-10 of their sum), and
    the output's rounding, 2^-8 (bf16) or 2^-24 of the value."""
    size = x_values.abs() @ w_values.abs().transpose(-1, -2).contiguous()
    kb = blocks(x_values.shape[-1])
    b = size * ((128 + 2 * kb + 4) * 2.0 ** -23)
    if out is BF16 and not few:
        b = b + size * 2.0 ** -10
    return b + (y.abs() + b) * (2.0 ** -8 if out is BF16 else 2.0 ** -24)


def plan_of(ids, groups):
    return ops.route_rows(ids, groups)


def members(ids, groups):
    """The slots of each group in order, from the ids."""
    flat = ids.cpu().reshape(-1).tolist()
    return [[s for s, e in enumerate(flat) if e == g] for g in range(groups)]
