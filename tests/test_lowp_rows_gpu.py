"""GPU tests of 4-bit linear layers whose rows carry their own global scales.

The restatement quantises row by row with 2^e, e the smallest with which the
row's largest magnitude is at most 2688 x 2^e, and multiplies in 64 bits; the
bound is that of the other linear layers: (K / 64 + 66) 2^-23 of sum |a w| for
the tensor core's float32 sums, scale and bias, 2^-8 of the result for its
rounding to bf16, and for GELU 2^-14 more with a slope of 1.13."""
import math

import pytest
import torch

import _lowp_reference as ref
from wan_dit import lowp
from wan_dit._ops import CudaOps

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(cuda_device):
    lowp._load()
    yield
    from in_context_sparse_attention import device_status
    device_status()


def row_scale(row):
    top = float(row.abs().max())
    if top == 0 or not math.isfinite(top):
        return 1.0
    m, e = math.frexp(top / 2688)
    return 2.0 ** max(min(e - (m == 0.5), 90), -90)


def restated(x):
    """The values that x has in nvfp4 with a scale for each row."""
    return torch.cat([ref.fp4_quantize(x[r:r + 1], "nvfp4", row_scale(x[r]))[2] for r in range(x.shape[0])])


def weight(N, K, seed=0):
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(seed + N + K)) * K ** -0.5
    return lowp.fp4_quantize(w.cuda(), "nvfp4", 2.0 ** -9), ref.fp4_quantize(w, "nvfp4", 2.0 ** -9)[2].cuda()


def spread_rows(M, K, dtype, seed=1):
    g = torch.Generator().manual_seed(seed + M + K)
    return (torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-40, 30, (M, 1), generator=g).float())).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K,act", [
    (1, 640, 5120, None), (1, 16, 1, None), (9, 520, 768, "gelu_tanh"), (3, 40, 8192, None),       # few rows, joined
    (33, 200, 1030, None), (64, 257, 300, "gelu_tanh"),
    (70, 300, 900, None), (70, 40, 4096, "gelu_tanh"), (300, 513, 1041, None), (513, 600, 257, "gelu_tanh"),
    (4200, 72, 530, None)])                                                                        # whole rows a warp
def test_rows_of_any_magnitude_keep_their_bits(M, N, K, act, dtype):
    x = spread_rows(M, K, dtype)
    wq, wv = weight(N, K)
    b = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    for bias in (None, b):
        got = lowp.fp4_linear(x.cuda(), wq, None if bias is None else bias.cuda(), act, row_scales=True).double()
        xv = restated(x).cuda()
        s, mass = xv @ wv.T, xv.abs() @ wv.abs().T
        if bias is not None:
            s, mass = s + bias.cuda().double(), mass + bias.cuda().double().abs()
        tol = (K / 64 + 66) * 2.0 ** -23 * mass
        if act:
            s, tol = ref.gelu_tanh(s), 1.13 * tol
        tol = tol + s.abs() * (2.0 ** -8 + 2.0 ** -14) + 1e-30
        assert bool(((got - s).abs() <= tol).all()), float(((got - s).abs() / tol).max())


@pytest.mark.parametrize("M", [1, 40, 300, 4200])
def test_a_power_of_two_passes_through(M):
    x = torch.randn(M, 512, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).cuda()
    for fmt in ("nvfp4", "mxfp4"):
        w = CudaOps.fp4_weight(torch.randn(96, 512, generator=torch.Generator().manual_seed(5)).cuda(), fmt)
        y = lowp.fp4_linear(x, w, row_scales=True)
        assert bool(y.any(dim=1).all())
        for e in (-10, -40, 20):
            assert torch.equal(lowp.fp4_linear(x * 2.0 ** e, w, row_scales=True), y * 2.0 ** e)
        if fmt == "mxfp4":
            assert torch.equal(y, lowp.fp4_linear(x, w))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_the_model_keeps_small_attention_and_gelu_outputs(fmt):
    """Rows of 2^-10, which scale 1 makes zero in nvfp4, give 2^-10 of the result in every layer whose input no
    norm brings to order one."""
    from wan_dit import WanDiT, WanDiTConfig
    model = WanDiT(WanDiTConfig(dim=256, ffn_dim=512, num_heads=2, num_layers=1, freq_dim=32, text_dim=64, text_len=80,
                                in_dim=4, out_dim=4, linear_format=fmt), seed=0)
    blk = model.blocks[0]
    for w, b in (("w_o", "b_o"), ("wc_o", "bc_o"), ("w2", "b2"), ("wc_kv", "bc_kv")):
        assert not bool(getattr(blk, b).any())
        x = torch.randn(100, blk.fp4[w].shape[1], generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
        y = model._linear(blk, w, b, x)
        assert bool(y.any(dim=1).all()) and torch.equal(model._linear(blk, w, b, x * 2.0 ** -10), y * 2.0 ** -10)
    x = torch.randn(100, 512, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda() * 2.0 ** -10
    res = torch.zeros(100, 256, device="cuda")
    model._linear_residual_(blk, "w2", "b2", res, x, None, 100)
    assert torch.equal(res, model._linear(blk, "w2", "b2", x).float())


def test_row_scales_are_those_of_the_kernel():
    x = torch.cat([spread_rows(50, 64, torch.float32), torch.zeros(1, 64), torch.full((1, 64), 2688.0),
                   torch.full((1, 64), 2688.002), torch.full((1, 64), 1e-38), torch.full((1, 64), 3e38),
                   torch.full((1, 64), math.inf)])
    g = lowp.fp4_row_scales(x)
    assert g.flatten().tolist() == [row_scale(r) for r in x]
    assert g[50:].flatten().tolist() == [1.0, 1.0, 2.0, 2.0 ** -90, 2.0 ** 90, 1.0]


@pytest.mark.parametrize("M", [12, 200])
def test_special_rows(M):
    K, N = 300, 130
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(2))
    clean = x.clone()
    wq, wv = weight(N, K)
    base = lowp.fp4_linear(clean.cuda(), wq, row_scales=True)
    x[0] = 0.0
    x[1, 40], x[2, 40], x[3, 299] = math.nan, math.inf, -math.inf
    x[4] *= 2.0 ** -120                        # beyond the scales' range: zeros
    x[5] *= 2.0 ** 110                         # saturates
    x[6, 17] = 2688.0                          # just in range of scale 1, and just above it
    x[7, 17] = 2688.002
    x[8] *= 2.0 ** -100
    y = lowp.fp4_linear(x.cuda(), wq, row_scales=True)
    assert not bool(y[0].any()) and bool(torch.isnan(y[1:4]).all()) and not bool(y[4].any())
    assert torch.equal(y[9:], base[9:])
    xv = restated(x[5:9]).cuda()
    s, mass = xv @ wv.T, xv.abs() @ wv.abs().T
    tol = (K / 64 + 66) * 2.0 ** -23 * mass + s.abs() * (2.0 ** -8 + 2.0 ** -14) + 1e-38
    assert bool(((y[5:9].double() - s).abs() <= tol).all())


@pytest.mark.parametrize("M", [5, 300])
def test_strided_rows_and_replays(M):
    wide = spread_rows(M, 700, torch.bfloat16).cuda()
    w, _ = weight(64, 300)
    for x in (wide[:, 3:303], wide[:, 16:316], wide[:, ::2][:, :300], wide[:1, :300].expand(M, 300)):
        assert torch.equal(lowp.fp4_linear(x, w, row_scales=True), lowp.fp4_linear(x.contiguous(), w, row_scales=True))
    assert lowp.fp4_linear(wide[:0, :300], w, row_scales=True).shape == (0, 64)
    static = wide[:, :300].contiguous()
    lowp.fp4_linear(static, w, row_scales=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lowp.fp4_linear(static, w, row_scales=True)
    for x in (wide[:, 300:600], wide[:, 3:303].flip(0) * 2.0 ** -20):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, lowp.fp4_linear(static.clone(), w, row_scales=True))


def test_workspace_is_checked_and_not_overrun():
    lib = lowp._load()
    M, N, K = 70, 40, 4096
    x = spread_rows(M, K, torch.bfloat16).cuda()
    w, _ = weight(N, K)
    want = lowp.fp4_linear(x, w, row_scales=True)
    size = lib.icsa_fp4_linear_scaled_rows_workspace_size(0, M, N, K)
    assert size == lib.icsa_fp4_linear_rows_workspace_size(0, M, N, K) + 512   # 280 bytes of row scales
    ws = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((M + 2, 48), 7.0, dtype=torch.bfloat16, device="cuda")

    def call(ptr, n):
        return lib.icsa_fp4_linear_scaled_rows(0, x.data_ptr(), 0, K, w.data.data_ptr(), w.scales.data_ptr(),
                                               w.global_scale, None, 0, out.data_ptr(), 48, M, N, K, ptr, n,
                                               torch.cuda.current_stream().cuda_stream)
    assert call(None, size) == 4 and call(ws.data_ptr(), size - 1) == 4 and call(ws.data_ptr() + 16, size) == 1
    assert call(ws.data_ptr(), size) == 0
    assert torch.equal(out[:M, :N], want)
    assert bool((out[M:] == 7).all()) and bool((out[:, N:] == 7).all()) and bool((ws[size:] == 0xFF).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt,g", [("nvfp4", 1.0), ("nvfp4", 2.0 ** -9), ("nvfp4", 0.37), ("mxfp4", 1.0)])
def test_negative_zeros_and_tiny_negatives_keep_their_sign(fmt, g, dtype):
    """The code of -0 is that of the float32 quotient, -0 (GELU and ReLU give such elements)."""
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(200, 512, generator=gen)
    x = torch.where(torch.rand(200, 512, generator=gen) < 0.3, -0.0, x)
    x[:, 7] = -1e-30
    x = x.to(dtype)
    code, sb, _ = ref.fp4_quantize(x, fmt, g)
    t = lowp.fp4_quantize(x.cuda(), fmt, g)
    assert torch.equal(t.scales.flatten().cpu(), ref.fp4_scale_bytes(sb, 200, 512, fmt))
    assert torch.equal(t.data.cpu(), ref.fp4_data_bytes(code, 512))
