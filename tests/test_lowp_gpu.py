"""GPU tests of the low-precision operators against their restatement in 64
bits (tests/_lowp_reference.py).

Quantised storage is compared byte for byte: codes and scales are roundings
of float32 quotients (or of exact power-of-two scalings), which both sides
round the same way.  Dequantised values are single products, equal as well.

Linear layers: the result is one rounding to bf16 (at most 2^-8 of the value)
of a float32 sum; the tensor core adds K / 64 partial sums of 64 products, so
with S = sum |a w| the sum is off by at most (K / 64 + 64) 2^-23 S, bias and
global scale by 2^-23 more each; GELU has slope at most 1.13 and its float32
evaluation (exponential of an argument up to 2^8) an error of 2^-14 of the
value.

Attention: one rounding to bf16 (2^-8 of the value), the probabilities' 16-bit
roundings (f16, 2^-11, in the kernel for few rows; bf16, 2^-8, in the others)
weighted with sum p |v|, and an error of the scores' float32 evaluation of
(|s| + 1) 2^-20 in the exponent, which moves p by as much."""
import math

import pytest
import torch

import _lowp_reference as ref
from wan_dit import lowp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(cuda_device):
    lowp._load()
    yield
    from in_context_sparse_attention import device_status
    device_status()


def rows(n, K, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + 7 * n + K)
    x = torch.randn(n, K, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))
    return x.to(dtype)


def assert_fp4_equal(t, x, fmt, g=1.0):
    n, K = x.shape
    code, sb, val = ref.fp4_quantize(x, fmt, g)
    assert torch.equal(t.scales.flatten().cpu(), ref.fp4_scale_bytes(sb, n, K, fmt))
    assert torch.equal(t.data.cpu(), ref.fp4_data_bytes(code, K))
    for dt in (torch.float32, torch.bfloat16):
        got, want = lowp.fp4_dequantize(t, dt).cpu(), val.to(torch.float32).to(dt)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


# --------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("fmt,g", [("nvfp4", 1.0), ("nvfp4", 2.0 ** -6), ("nvfp4", 0.0371), ("mxfp4", 1.0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,K", [(1, 1), (1, 16), (3, 47), (5, 512), (33, 130), (128, 256), (129, 257), (130, 520),
                                 (7, 5120), (260, 1027)])
def test_quantisation_gives_the_defined_bytes(fmt, g, dtype, n, K):
    x = rows(n, K, dtype)
    assert_fp4_equal(lowp.fp4_quantize(x.cuda(), fmt, g), x, fmt, g)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantisation_of_zeros_ties_extremes_and_non_finite_blocks(fmt):
    x = torch.zeros(20, 96)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    x[1, :8], x[1, 8:16] = ties, -ties
    x[2, :8] = ties * 2.0 ** -20                # nvfp4: the scale rounds to zero or a subnormal
    x[3, :8] = ties * 2.0 ** -140               # subnormal float32
    x[4, :8] = ties * 2.0 ** 100                # nvfp4: above 448 x 6, saturates
    x[5, 40] = math.nan
    x[6, 40] = math.inf
    x[7, 40] = -math.inf
    x[8, 95], x[8, 94] = 3.3e38, -3.3e38
    x[9, 0] = 2.0 ** -126
    x[10, :] = -0.0
    x[11, 33], x[11, 34] = 1.0, 2.0 ** -149
    x[12:] = torch.randn(8, 96, generator=torch.Generator().manual_seed(5)) * 1e-9
    for g in ((1.0, 2.0 ** -30, 2.0 ** -60, 2.0 ** 60, 1e-37) if fmt == "nvfp4" else (1.0,)):
        assert_fp4_equal(lowp.fp4_quantize(x.cuda(), fmt, g), x, fmt, g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantisation_takes_strided_and_unaligned_rows(dtype):
    base = rows(9, 700, dtype).cuda()
    for x in (base[:, 3:270], base[:, 16:528], base[::2, :64], base[:, 1:2], base.t()[:40], base[2:3, 5:69],
              base[:1].expand(4, 700)):
        assert_fp4_equal(lowp.fp4_quantize(x, "nvfp4"), x.cpu(), "nvfp4")
    empty = lowp.fp4_quantize(base[:0], "mxfp4")
    assert empty.shape == (0, 700) and lowp.fp4_dequantize(empty).shape == (0, 700)


def test_rows_behind_the_last_and_columns_behind_K_are_zero_bytes():
    x = rows(5, 300, torch.bfloat16).cuda()
    lib = lowp._load()
    data = torch.full((5 * 160 + 64,), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((lib.icsa_fp4_scale_bytes(0, 5, 300) + 64,), 0xEE, dtype=torch.uint8, device="cuda")
    assert lib.icsa_fp4_quantize(x.data_ptr(), 0, 300, 5, 300, 0, 1.0, data.data_ptr(), scales.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream) == 0
    code, sb, _ = ref.fp4_quantize(x.cpu(), "nvfp4")
    assert torch.equal(data[:800].view(5, 160).cpu(), ref.fp4_data_bytes(code, 300))
    assert torch.equal(scales[:-64].cpu(), ref.fp4_scale_bytes(sb, 5, 300, "nvfp4"))
    assert bool((data[800:] == 0xEE).all()) and bool((scales[-64:] == 0xEE).all())


# --------------------------------------------------------------------------- linear layers
def linear_case(M, N, K, fmt, bias, act, seed=0, g_x=1.0):
    gen = torch.Generator().manual_seed(seed + M + 3 * N + 5 * K)
    x = torch.randn(M, K, generator=gen).to(torch.bfloat16)
    w = (torch.randn(N, K, generator=gen) * K ** -0.5).to(torch.bfloat16)
    b = torch.randn(N, generator=gen).to(torch.bfloat16) if bias else None
    g_w = 2.0 ** -9 if fmt == "nvfp4" else 1.0
    _, _, xv = ref.fp4_quantize(x, fmt, g_x)
    _, _, wv = ref.fp4_quantize(w, fmt, g_w)
    xv, wv = xv.cuda(), wv.cuda()               # float64 products
    s = xv @ wv.T
    mass = xv.abs() @ wv.abs().T
    if bias:
        s = s + b.cuda().double()
        mass = mass + b.cuda().double().abs()
    tol = (K / 64 + 66) * 2.0 ** -23 * mass
    if act == "gelu_tanh":
        s, tol = ref.gelu_tanh(s), 1.13 * tol
    tol = tol + s.abs() * (2.0 ** -8 + 2.0 ** -14) + 1e-30
    wq = lowp.fp4_quantize(w.cuda(), fmt, g_w)
    return x.cuda(), wq, (b.cuda() if bias else None), s, tol


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M,N,K,bias,act", [
    (1, 1, 1, True, None), (1, 640, 5120, True, None), (2, 257, 47, False, "gelu_tanh"), (3, 16, 256, True, None),
    (5, 256, 1000, False, None), (8, 1000, 4097, True, "gelu_tanh"), (9, 520, 768, True, None),
    (17, 100, 300, True, None), (63, 256, 513, False, None), (128, 128, 128, False, None),
    (129, 260, 257, True, "gelu_tanh"), (255, 513, 640, True, None), (257, 255, 16, False, None),
    (300, 2056, 1040, True, "gelu_tanh"), (513, 5120, 320, True, None), (1031, 3000, 2000, False, None),
    (4000, 7001, 512, True, "gelu_tanh")])
def test_linear_layer(fmt, M, N, K, bias, act):
    x, w, b, want, tol = linear_case(M, N, K, fmt, bias, act)
    got = lowp.fp4_linear(x, w, b, act)
    assert got.shape == (M, N) and got.dtype == torch.bfloat16
    d = (got.double() - want).abs()
    print(f"linear {fmt} {M}x{N}x{K}: worst error {float((d / tol).max()):.3f} of its bound")
    assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M,N,K,bias,act", [
    (1, 30001, 1030, True, None), (1, 128, 65536, False, None), (16, 19001, 520, True, "gelu_tanh"),
    (17, 129, 8192, True, None), (32, 3000, 256, False, None), (33, 40000, 300, True, None),
    (64, 2560, 5120, True, "gelu_tanh"), (65, 2560, 5120, True, "gelu_tanh"),
    (1, 20000, 5120, False, None), (5, 19001, 5300, True, "gelu_tanh"), (40, 19001, 5300, True, None)])
def test_linear_layer_of_few_rows(fmt, M, N, K, bias, act):
    """Tiles cut between CTAs at every kind of boundary: many tiles, one tile, whole tiles."""
    test_linear_layer(fmt, M, N, K, bias, act)


def test_linear_layer_of_a_quantised_input_and_of_float32_rows():
    x, w, b, want, tol = linear_case(70, 300, 900, "nvfp4", True, None, g_x=2.0 ** -3)
    t = lowp.fp4_quantize(x, "nvfp4", 2.0 ** -3)
    got = lowp.fp4_linear(t, w, b)
    assert bool(((got.double() - want).abs() <= tol).all())
    x, w, b, want, tol = linear_case(70, 300, 900, "mxfp4", True, None)
    assert torch.equal(lowp.fp4_linear(x, w, b), lowp.fp4_linear(x.float(), w, b))
    wide = torch.cat([x, x], dim=1)[:, 900:]                   # rows of a wider tensor
    assert torch.equal(lowp.fp4_linear(wide, w, b), lowp.fp4_linear(x, w, b))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("M", [4, 400])
def test_non_finite_inputs_stay_in_their_row_and_column(fmt, M):
    x, w, b, want, tol = linear_case(M, 384, 512, fmt, True, None)
    clean = lowp.fp4_linear(x, w, b)
    x = x.clone()
    x[1, 100], x[3, 511] = math.nan, math.inf
    wf = lowp.fp4_dequantize(w, torch.float32)
    wf[7, 300] = -math.inf
    wf[250, 0] = math.nan
    got = lowp.fp4_linear(x, lowp.fp4_quantize(wf, fmt, w.global_scale), b)
    bad = torch.zeros(M, 384, dtype=torch.bool, device="cuda")
    bad[1], bad[3], bad[:, 7], bad[:, 250] = True, True, True, True
    assert bool(torch.isnan(got)[bad].all())
    assert torch.equal(got[~bad], clean[~bad])


def test_linear_layer_refuses_mixed_formats_and_devices():
    x, w, b, _, _ = linear_case(4, 32, 64, "nvfp4", True, None)
    for call in (lambda: lowp.fp4_linear(lowp.fp4_quantize(x, "mxfp4"), w), lambda: lowp.fp4_linear(x.cpu(), w),
                 lambda: lowp.fp4_linear(x, w, b.cpu()), lambda: lowp.fp4_linear(x, w, b.float()),
                 lambda: lowp.fp4_linear(x.half(), w), lambda: lowp.fp4_linear(x[:, :63], w)):
        with pytest.raises(ValueError):
            call()
    assert lowp.fp4_linear(x[:0], w, b).shape == (0, 32)


@pytest.mark.parametrize("M,K", [(3, 8192), (70, 4096)])
def test_linear_layer_checks_its_workspace_and_leaves_what_is_behind_its_rows(M, K):
    lib = lowp._load()
    x, w, b, want, tol = linear_case(M, 40, K, "nvfp4", True, None)
    a = lowp.fp4_quantize(x, "nvfp4")
    size = lib.icsa_fp4_linear_workspace_size(M, 40, K)
    assert size > 0                                              # few tiles: K is split
    out = torch.full((M + 2, 48), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device="cuda")

    def call(ws_ptr, nbytes):
        return lib.icsa_fp4_linear(0, a.data.data_ptr(), a.scales.data_ptr(), 1.0, w.data.data_ptr(),
                                   w.scales.data_ptr(), w.global_scale, b.data_ptr(), 0, out.data_ptr(), 48, M, 40,
                                   K, ws_ptr, nbytes, torch.cuda.current_stream().cuda_stream)
    assert call(None, size) == 4 and call(ws.data_ptr(), size - 1) == 4 and call(ws.data_ptr() + 16, size) == 1
    assert call(ws.data_ptr(), size) == 0
    assert bool(((out[:M, :40].double() - want).abs() <= tol).all())
    assert bool((out[M:] == 7).all()) and bool((out[:, 40:] == 7).all()) and bool((ws[size:] == 0xFF).all())


# --------------------------------------------------------------------------- cache
def kv_rows(B, L, H, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + B + 3 * L + 5 * H + D)
    k = torch.randn(B, L, H, D, generator=g) * torch.exp(torch.randn(1, L, H, 1, generator=g))
    v = torch.randn(B, L, H, D, generator=g) * torch.exp(0.3 * torch.randn(1, L, 1, 1, generator=g))
    return k.to(dtype), v.to(dtype)


def assert_cache_equal(c, k, v, lengths=None):
    kc, ks, kval = ref.kv8_quantize(k, lengths)
    vc, vs, vval = ref.kv8_quantize(v, lengths)
    for got, want in ((c.k_scale, ks), (c.v_scale, vs)):
        assert torch.equal(got.cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))
    assert torch.equal(c.k.view(torch.uint8).cpu(), kc)
    assert torch.equal(c.v.view(torch.uint8).cpu().transpose(-1, -2), vc)
    for dt in (torch.bfloat16, torch.float32):
        for got, want in zip(lowp.kv8_dequantize(c, dt), (kval, vval)):
            assert got.dtype == dt and torch.equal(got.double().cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,L,H,D,lengths", [(1, 1, 1, 64, None), (2, 63, 3, 128, None), (1, 64, 2, 64, [64]),
                                             (3, 65, 2, 128, [65, 0, 1]), (2, 200, 5, 64, [128, 129]),
                                             (2, 331, 1, 128, [400, -3])])
def test_cache_holds_the_defined_bytes(dtype, B, L, H, D, lengths):
    k, v = kv_rows(B, L, H, D, dtype)
    n = None
    if lengths is not None:
        n = torch.tensor(lengths, dtype=torch.int32)
        for b, m in enumerate(lengths):                          # what is behind a length is not read
            k[b, max(m, 0):], v[b, max(m, 0):] = math.nan, math.inf
        n = n.cuda()
    assert_cache_equal(lowp.kv8_quantize(k.cuda(), v.cuda(), n), k, v, lengths)


def test_cache_of_special_values():
    k, v = kv_rows(1, 64 * 9, 2, 64, torch.float32)
    k[0, 0:64] = 0.0
    k[0, 64:128, 0], v[0, 64:128, 0] = 0.0, 0.0
    k[0, 70, 0, 3], v[0, 70, 0, 3] = 448.0, 448.001
    k[0, 130, 1, 0], v[0, 140, 0, 5] = math.nan, -math.inf
    k[0, 192:256] *= 1e-33
    v[0, 192:256] *= 1e34                                        # above 448 x 2^96: saturates
    v[0, 256:320] *= 2.0 ** -120
    k[0, 330, 0, 1] = 2.0 ** -149
    k[0, 400, 1, 7] = 3.4e38
    assert_cache_equal(lowp.kv8_quantize(k.cuda(), v.cuda()), k, v)


def test_cache_takes_strided_keys_and_values():
    B, L, H, D = 2, 100, 3, 64
    kv = torch.randn(B * L, 2 * H * D + 5, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    k, v = kv[:, :H * D].unflatten(0, (B, L)).unflatten(2, (H, D)), kv[:, H * D:2 * H * D].unflatten(0, (B, L)).unflatten(2, (H, D))
    assert_cache_equal(lowp.kv8_quantize(k, v), k.cpu(), v.cpu())
    kt = torch.randn(B, H, L, D, generator=torch.Generator().manual_seed(4)).cuda().transpose(1, 2)
    assert_cache_equal(lowp.kv8_quantize(kt, kt), kt.cpu(), kt.cpu())
    ke = kt[:1].expand(B, L, H, D)                               # one sequence for the whole batch
    assert_cache_equal(lowp.kv8_quantize(ke, ke), ke.cpu(), ke.cpu())
    kd = torch.randn(B, L, D, H, generator=torch.Generator().manual_seed(4)).cuda().transpose(2, 3)
    assert_cache_equal(lowp.kv8_quantize(kd, kd), kd.cpu(), kd.cpu())


# --------------------------------------------------------------------------- attention
def check_attention(q, cache, lengths=None, k=None, v=None):
    got = lowp.kv8_attention(q.cuda(), cache)
    if k is None:
        k, v = (t.double().cpu() for t in lowp.kv8_dequantize(cache, torch.float32))
    want, mass, big = ref.attention(q, k, v, lengths)
    assert got.shape == q.shape and got.dtype == torch.bfloat16
    # Below 2^-14 a probability in fp16 is off by up to 2^-25, not 2^-11 of itself.  The kernels' p is
    # 2^(x - m) of the codes, x = score + log2(S_j) with S_j a value block's scale, m an x that occurs: that
    # key adds 1 / S to the row sum, so the sum is at least 1 / max(S), and the quotient is off by at most
    # 2^-25 sum_j |code_j| max(S).  (It shows where the key that takes almost all of a row has a value of 0.)
    scale = cache.v_scale.double().cpu().nan_to_num(0.0).repeat_interleave(64, 2)[:, :, :k.shape[1]].transpose(1, 2)
    valid = torch.tensor([k.shape[1]] * k.shape[0] if lengths is None else list(lengths)).clamp(0, k.shape[1])
    valid = (torch.arange(k.shape[1])[None] < valid[:, None])[..., None]
    code = torch.where(valid[..., None], v.nan_to_num(0.0).abs() / scale.clamp_min(2.0 ** -126)[..., None], 0.0)
    tiny = code.sum(1) * (scale * valid).amax(1)[..., None] * 2.0 ** -25
    tiny = tiny[:, None].repeat_interleave(q.shape[2] // k.shape[2], 2)
    few = q.shape[1] * (q.shape[2] // k.shape[2]) <= 48
    tol = want.abs() * 2.0 ** -8 + mass * ((2.0 ** -11 if few else 2.0 ** -8) + (big + 1) * 2.0 ** -20) + tiny + 1e-30
    d = (got.double().cpu() - want).abs()
    print(f"attention {tuple(q.shape)}: worst error {float((d / tol).max()):.3f} of its bound, scores to {big:.1f}")
    assert bool((d <= tol).all()), float((d / tol).max())
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Lq,Lk,H,group,lengths", [
    (1, 1, 1, 1, 1, None), (2, 1, 63, 3, 1, None), (1, 1, 65, 2, 4, [64]), (3, 2, 129, 2, 1, [129, 0, 1]),
    (2, 8, 200, 2, 1, [131, 200]), (4, 9, 331, 4, 4, [331, 280, 10, 0]), (1, 3, 4000, 1, 3, None),
    (2, 1, 9000, 2, 1, [8000, 77]), (1, 32, 500, 1, 1, None),
    (1, 33, 100, 2, 1, None), (2, 16, 70, 1, 4, [0, 70]), (3, 77, 331, 2, 2, [331, 0, 130]), (1, 64, 64, 3, 1, None),
    (2, 65, 1, 1, 2, None), (2, 300, 1000, 2, 1, [1000, 63]), (1, 257, 128, 2, 1, [127]),
    # bf16 copies with shared heads and an empty sequence; rounds cut between clusters, groups that
    # no box of queries holds; more sequences than a launch takes; many splits
    (3, 700, 900, 2, 3, [0, 900, 65]), (1, 60, 9000, 2, 1, [8777]), (2, 20, 5000, 3, 5, [4999, 129]),
    (1, 130, 6000, 1, 3, None), (130, 49, 70, 1, 1, list(range(-30, 100))), (129, 51, 1100, 1, 1, None),
    (1, 1, 32000, 1, 2, None), (2, 9, 3000, 40, 1, [3000, 1]), (2, 16, 700, 40, 1, None), (1, 37, 5000, 8, 1, [4990]),
    (1, 5, 6000, 16, 5, None),
    # SM pairs: one step, shared heads, an odd number of tiles, rounds cut between clusters; then the bf16 copy
    (2, 300, 100, 16, 1, [100, 37]), (2, 40, 120, 4, 8, None), (4, 100, 331, 8, 3, [331, 0, 5, 331]),
    (3, 70, 500, 16, 5, None), (2, 700, 331, 16, 1, [331, 200]), (1, 512, 8000, 8, 1, [7900]),
    (1, 150, 8000, 8, 3, None), (1, 700, 8000, 8, 1, [7777]), (1, 4096, 2000, 8, 1, [1990])])
def test_attention_over_the_cache(D, B, Lq, Lk, H, group, lengths):
    k, v = kv_rows(B, Lk, H, D, torch.bfloat16)
    q = torch.randn(B, Lq, H * group, D, generator=torch.Generator().manual_seed(Lq + Lk)).to(torch.bfloat16)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cache = lowp.kv8_quantize(k.cuda(), v.cuda(), n)
    got = check_attention(q, cache, lengths)
    for b, m in enumerate(lengths or []):
        if m <= 0:
            assert not bool(got[b].any())


@pytest.mark.parametrize("Lq,H", [(1, 2), (40, 2), (300, 16)])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_ignores_what_the_cache_holds_behind_a_length(Lq, H, D):
    lengths = [70, 0, 128]
    k, v = kv_rows(3, 192, H, D, torch.bfloat16)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    q = torch.randn(3, Lq, H, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    cache = lowp.kv8_quantize(k.cuda(), v.cuda(), n)
    clean = check_attention(q, cache, lengths)
    for b, m in enumerate(lengths):
        for i in range(3):
            t = max(0, min(64, m - 64 * i))
            cache.k.view(torch.uint8)[b, :, i, t:], cache.v.view(torch.uint8)[b, :, i, :, t:] = 0x7F, 0xFF
            if t == 0:
                cache.k_scale[b, :, i], cache.v_scale[b, :, i] = math.nan, math.inf
    assert torch.equal(lowp.kv8_attention(q.cuda(), cache), clean)
    kd, vd = lowp.kv8_dequantize(cache)
    assert bool(torch.isfinite(kd).all()) and bool(torch.isfinite(vd).all())


@pytest.mark.parametrize("Lq,H", [(2, 2), (50, 2), (300, 16), (300, 80)])
def test_attention_with_peaked_scores_and_unequal_scales(Lq, H):
    """Scores to several hundred, and value blocks whose scales differ by 2^40."""
    B, L, D = 1, 400, 128
    k, v = kv_rows(B, L, H, D, torch.float32)
    k = k * 6
    v = v * torch.exp2(torch.tensor([0.0, -20.0, 20.0, 3.0, -3.0, 0.0, 10.0]).repeat_interleave(64)[:L])[None, :, None, None]
    q = (torch.randn(B, Lq, H, D, generator=torch.Generator().manual_seed(2)) * 4).to(torch.bfloat16)
    check_attention(q, lowp.kv8_quantize(k.cuda(), v.cuda()))


def test_attention_of_tiny_and_huge_queries():
    k, v = kv_rows(1, 100, 1, 64, torch.bfloat16)
    cache = lowp.kv8_quantize(k.cuda(), v.cuda())
    q = torch.randn(1, 6, 1, 64, generator=torch.Generator().manual_seed(2))
    q[0, 0] = 0.0
    q[0, 1] *= 1e-38
    q[0, 2] *= 1e-20
    q[0, 3, 0, 1:] *= 1e-9
    q = q.to(torch.bfloat16)
    check_attention(q, cache)
    huge = (q * 1e4).to(torch.bfloat16)
    got = lowp.kv8_attention(huge.cuda(), cache)                 # one key takes all of the probability
    kd, vd = (t.double().cpu() for t in lowp.kv8_dequantize(cache, torch.float32))
    best = (huge[0, 4:, 0].double() @ kd[0, :, 0].T).argmax(-1)
    assert torch.equal(got[0, 4:, 0].cpu(), vd[0, best, 0].to(torch.bfloat16))


@pytest.mark.parametrize("Lq,H", [(3, 2), (100, 2), (300, 16)])
def test_non_finite_values_reach_the_rows_that_read_them(Lq, H):
    k, v = kv_rows(2, 130, H, 64, torch.bfloat16)
    q = torch.randn(2, Lq, H, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    clean = lowp.kv8_attention(q.cuda(), lowp.kv8_quantize(k.cuda(), v.cuda()))
    k[0, 10, 0, 3], v[1, 129, 1, 0] = math.nan, math.inf
    q[0, 1, 1, 5] = math.nan
    got = lowp.kv8_attention(q.cuda(), lowp.kv8_quantize(k.cuda(), v.cuda()))
    bad = torch.zeros(2, Lq, H, dtype=torch.bool, device="cuda")
    bad[0, :, 0], bad[1, :, 1], bad[0, 1, 1] = True, True, True
    assert bool(torch.isnan(got)[bad].all()) and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("Lq,H", [(1, 3), (5, 3), (90, 3), (300, 16)])
def test_attention_takes_strided_queries(Lq, H):
    B, D = 2, 64
    k, v = kv_rows(B, 150, H, D, torch.bfloat16)
    cache = lowp.kv8_quantize(k.cuda(), v.cuda())
    wide = torch.randn(B * Lq, 2 * H * D + 8, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    for q in (wide[:, :H * D].view(B, Lq, H, D) if Lq == 1 else wide[:, :H * D].unflatten(0, (B, Lq)).unflatten(2, (H, D)),
              wide[:, 8:8 + H * D].unflatten(0, (B, Lq)).unflatten(2, (H, D)),
              wide[:, 3:3 + H * D].unflatten(0, (B, Lq)).unflatten(2, (H, D)),
              torch.randn(B, H, Lq, D, device="cuda").to(torch.bfloat16).transpose(1, 2),
              wide[:1, :H * D].unflatten(0, (1, 1)).unflatten(2, (H, D)).expand(B, Lq, H, D)):
        assert torch.equal(lowp.kv8_attention(q, cache), lowp.kv8_attention(q.contiguous(), cache))
    assert lowp.kv8_attention(wide[:0, :H * D].view(0, 1, H, D).new_zeros(B, 0, H, D), cache).shape == (B, 0, H, D)


def test_strided_heads_over_a_long_cache_are_copied_by_python_and_refused_by_c():
    import ctypes
    k, v = kv_rows(1, 5000, 2, 128, torch.bfloat16)
    cache = lowp.kv8_quantize(k.cuda(), v.cuda())
    q = torch.randn(1, 2, 4000, 128, device="cuda").to(torch.bfloat16).transpose(1, 2)
    want = lowp.kv8_attention(q.contiguous(), cache)
    assert torch.equal(lowp.kv8_attention(q, cache), want)
    lib, desc = lowp._load(), cache._desc()
    size = lib.icsa_kv8_attention_workspace_size(ctypes.byref(desc), 4000, 2)
    ws, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros_like(want)
    assert lib.icsa_kv8_attention(ctypes.byref(desc), q.data_ptr(), (ctypes.c_int64 * 3)(0, 128, 4000 * 128),
                                  out.data_ptr(), 4000, 2, ws.data_ptr(), size,
                                  torch.cuda.current_stream().cuda_stream) == 2
    assert not bool(out.any())


def test_attention_refuses_other_shapes_and_devices():
    k, v = kv_rows(2, 64, 2, 64, torch.bfloat16)
    cache = lowp.kv8_quantize(k.cuda(), v.cuda())
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: lowp.kv8_attention(q[:, :, :3], cache), lambda: lowp.kv8_attention(q[:1], cache),
                 lambda: lowp.kv8_attention(q.float(), cache), lambda: lowp.kv8_attention(q[..., :32], cache),
                 lambda: lowp.kv8_attention(q.cpu(), cache), lambda: lowp.kv8_quantize(k.cuda(), v),
                 lambda: lowp.kv8_quantize(k.cuda(), v.cuda(), torch.tensor([1, 2])),
                 lambda: lowp.kv8_quantize(k.cuda()[..., :32], v.cuda()[..., :32]),
                 lambda: lowp.kv8_quantize(k.cuda()[:, :0], v.cuda()[:, :0])):
        with pytest.raises(ValueError):
            call()


def test_attention_checks_its_workspace():
    import ctypes
    lib = lowp._load()
    k, v = kv_rows(1, 5000, 1, 64, torch.bfloat16)
    cache = lowp.kv8_quantize(k.cuda(), v.cuda())
    for Lq in (2, 80):
        q = torch.randn(1, Lq, 1, 64, device="cuda").to(torch.bfloat16)
        want = lowp.kv8_attention(q, cache)
        desc = cache._desc()
        size = lib.icsa_kv8_attention_workspace_size(ctypes.byref(desc), Lq, 1)
        assert size > 0
        ws = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device="cuda")
        out = torch.full((Lq + 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        strides = (ctypes.c_int64 * 3)(Lq * 64, 64, 64)

        def call(p, n):
            return lib.icsa_kv8_attention(ctypes.byref(desc), q.data_ptr(), strides, out.data_ptr(), Lq, 1, p, n,
                                          torch.cuda.current_stream().cuda_stream)
        assert call(None, size) == 4 and call(ws.data_ptr(), size - 1) == 4 and call(ws.data_ptr() + 16, size) == 1
        assert call(ws.data_ptr(), size) == 0
        assert torch.equal(out[:Lq].view(want.shape), want)
        assert bool((out[Lq:] == 7).all()) and bool((ws[size:] == 0xFF).all())


# --------------------------------------------------------------------------- streams, graphs, devices
def together(x, w1, b1, w2, k, v, n, q):
    """A feed-forward pair and a cross-attention, as a block runs them."""
    h = lowp.fp4_linear(lowp.fp4_linear(x, w1, b1, "gelu_tanh"), w2)
    cache = lowp.kv8_quantize(k, v, n)
    return h, lowp.kv8_attention(q, cache), lowp.kv8_attention(q[:, :1], cache)


def together_inputs(seed, M=70):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, 384, generator=g).to(torch.bfloat16).cuda()
    k, v = (torch.randn(2, 150, 2, 128, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(2, M, 2, 128, generator=g).to(torch.bfloat16).cuda()
    return x, k, v, torch.tensor([150, 90], dtype=torch.int32).cuda(), q


def together_weights():
    g = torch.Generator().manual_seed(11)
    w1 = lowp.fp4_quantize((torch.randn(512, 384, generator=g) / 20).cuda(), "nvfp4", 2.0 ** -9)
    w2 = lowp.fp4_quantize((torch.randn(384, 512, generator=g) / 20).cuda(), "nvfp4", 2.0 ** -9)
    return w1, torch.randn(512, generator=g).to(torch.bfloat16).cuda(), w2


def test_a_run_of_the_operators_is_captured_replayed_and_repeatable():
    w1, b1, w2 = together_weights()
    static = together_inputs(0)

    def run(x, k, v, n, q):
        return together(x, w1, b1, w2, k, v, n, q)
    want = [run(*together_inputs(s)) for s in (0, 1, 2)]
    again = run(*together_inputs(1))
    assert all(torch.equal(a, b) for a, b in zip(want[1], again))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run(*static)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]          # two graphs of the same calls
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(run(*static))
    for s in (1, 2, 0):
        for dst, src in zip(static, together_inputs(s)):
            dst.copy_(src)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want[s]))


def test_second_kernels_in_two_graphs_and_on_two_streams():
    """Products split along K, tiles and rounds cut between CTAs: every call launches a kernel that
    joins partial results from its workspace."""
    g = torch.Generator().manual_seed(4)
    w = lowp.fp4_quantize((torch.randn(300, 4096, generator=g) / 64).cuda(), "nvfp4", 2.0 ** -9)
    long = lowp.fp4_quantize((torch.randn(300, 16384, generator=g) / 64).cuda(), "nvfp4", 2.0 ** -9)
    k, v = kv_rows(1, 9000, 2, 128, torch.bfloat16)
    cache = lowp.kv8_quantize(k.cuda(), v.cuda())
    k, v = kv_rows(1, 8000, 8, 128, torch.bfloat16)
    cache8 = lowp.kv8_quantize(k.cuda(), v.cuda())

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        return [torch.randn(n, m, generator=g).to(torch.bfloat16).cuda() for n, m in ((9, 16384), (70, 4096))] + [
            torch.randn(1, n, h, 128, generator=g).to(torch.bfloat16).cuda() for n, h in ((1, 2), (60, 2), (512, 8))]

    def run(x9, x70, q1, q60, q512):
        return (lowp.fp4_linear(x9, long), lowp.fp4_linear(x70, w), lowp.kv8_attention(q1, cache),
                lowp.kv8_attention(q60, cache), lowp.kv8_attention(q512, cache8))
    want = [run(*inputs(s)) for s in (0, 1, 2)]
    static = inputs(0)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(run(*static))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in (1, 2):
        for dst, src in zip(static, inputs(s)):
            dst.copy_(src)
        torch.cuda.synchronize()
        for _ in range(3):
            for gr, st in zip(graphs, streams):                  # both at once
                with torch.cuda.stream(st):
                    gr.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want[s]))


@pytest.mark.parametrize("Lq,H,L", [(2, 2, 9000), (300, 16, 200), (512, 8, 8000), (700, 2, 900)])
def test_lengths_may_change_between_replays(Lq, H, L):
    """The few-row kernel, SM pairs with and without a join, the bf16 copy."""
    k, v = kv_rows(2, L, H, 128, torch.bfloat16)
    k, v = k.cuda(), v.cuda()
    q = torch.randn(2, Lq, H, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    n = torch.tensor([L, L // 3], dtype=torch.int32, device="cuda")

    def run():
        cache = lowp.kv8_quantize(k, v, n)
        return lowp.kv8_attention(q, cache), *lowp.kv8_dequantize(cache)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for lengths in ([L // 2, 0], [1, L], [0, 0], [L, L]):
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))
        assert all(not bool(out[0][b].any()) for b in range(2) if lengths[b] == 0)


def test_calls_on_two_streams_at_once():
    w1, b1, w2 = together_weights()
    inputs = [together_inputs(s, 200) for s in range(2)]
    want = [together(x, w1, b1, w2, k, v, n, q) for x, k, v, n, q in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                x, k, v, n, q = inputs[i]
                got[i] = together(x, w1, b1, w2, k, v, n, q)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))


def test_tensors_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    dev = torch.device("cuda", 1)
    x, k, v, n, q = (t.to(dev) for t in together_inputs(0))
    w1, b1, w2 = together_weights()
    want = together(*together_inputs(0)[:1], w1, b1, w2, *together_inputs(0)[1:])
    move = lambda t: lowp.Fp4Tensor(t.data.to(dev), t.scales.to(dev), t.shape, t.fmt, t.global_scale)  # noqa: E731
    got = together(x, move(w1), b1.to(dev), move(w2), k, v, n, q)
    assert all(g.device == dev and torch.equal(g.cpu(), w.cpu()) for g, w in zip(got, want))


# --------------------------------------------------------------------------- large tensors
def test_offsets_beyond_32_bits_in_4_bit_tensors():
    rows, K = 262144 + 3, 16400                                  # 4.3e9 elements
    x = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
    x[:-200] = 1.0
    x[-200:] = torch.randn(200, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    t = lowp.fp4_quantize(x, "nvfp4")
    n = rows - 128 * 2023                                        # enough rows for the same order of sums
    tail = lowp.fp4_quantize(x[-n:], "nvfp4")
    assert torch.equal(t.data[-n:], tail.data) and torch.equal(t.scales[2023:], tail.scales)
    del x
    out = lowp.fp4_dequantize(t)
    # a block of ones: scale e4m3(1 / 6) = 11 / 64, code e2m1(64 / 11) = 6
    assert torch.equal(out[-n:], lowp.fp4_dequantize(tail)) and bool((out[:300] == 66 / 64).all())
    del out
    w = lowp.fp4_quantize(torch.randn(8208, K, generator=torch.Generator().manual_seed(2)).cuda(), "nvfp4", 2.0 ** -7)
    y = lowp.fp4_linear(t, w)                                    # 2.15e9 outputs
    assert torch.equal(y[-n:], lowp.fp4_linear(tail, w)) and torch.equal(y[7], y[100000])


@pytest.mark.parametrize("Lq", [1, 64])
def test_offsets_beyond_32_bits_in_the_cache(Lq):
    L, D = (1 << 25) + 70, 128                                   # 4.3e9 elements
    k = torch.zeros(1, L, 1, D, dtype=torch.bfloat16, device="cuda")
    last = torch.randn(70, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    k[0, -70:, 0] = last * 64
    cache = lowp.kv8_quantize(k, k)
    del k
    tail = lowp.kv8_quantize(last.view(1, 70, 1, D) * 64, last.view(1, 70, 1, D) * 64)
    for a, b in ((cache.k, tail.k), (cache.v, tail.v)):
        assert torch.equal(a[0, 0, -2:].view(torch.uint8), b[0, 0].view(torch.uint8))
    assert torch.equal(cache.k_scale[0, 0, -2:], tail.k_scale[0, 0]) and bool((cache.v_scale[0, 0, :-2] == 1).all())
    # only the last 70 keys and values are not zero: every key before them has score 0
    q = (torch.randn(1, Lq, 1, D, generator=torch.Generator().manual_seed(2)) / 16).to(torch.bfloat16).cuda()
    got = lowp.kv8_attention(q, cache)[0, :, 0].double()
    kd, vd = (x[0, :, 0].double() for x in lowp.kv8_dequantize(tail, torch.float32))
    s = q[0, :, 0].double() @ kd.T / math.sqrt(D)
    top = s.amax(1, keepdim=True).clamp_min(0)
    p = torch.exp(s - top)
    total = p.sum(1, keepdim=True) + (L - 70) * torch.exp(-top)
    want, mass = p @ vd / total, p @ vd.abs() / total
    # a row sum of up to 4096 steps one behind the other, each rounded by 2^-24
    tol = want.abs() * 2.0 ** -8 + mass * (2.0 ** -11 + (float(s.abs().max()) + 1) * 2.0 ** -20 + 2.0 ** -12)
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


# --------------------------------------------------------------------------- in the model
TINY = dict(dim=256, ffn_dim=512, num_heads=2, num_layers=2, freq_dim=32, text_dim=64, text_len=80, in_dim=4,
            out_dim=4)


def tiny(seq=False):
    g = torch.Generator().manual_seed(3)
    latent = torch.randn(4, 4, 16, 32, generator=g).cuda()
    context = torch.randn(2, 80, 64, generator=g).cuda()
    return latent, 0.8 * latent + 0.1, context, 2 * 4 * 8 * 16


def stepped(model, context, **kw):
    latent, source, _, seq = tiny()
    return model.denoise_step(latent, source, 500.0, 1.0, 0.9, context, seq, **kw) - latent


def test_model_with_an_8_bit_text_cache_follows_the_one_without():
    """The cache rounds keys and values to e4m3 (2^-4 of a value), the rest of the step is the same."""
    from wan_dit import WanDiT, WanDiTConfig
    model = WanDiT(WanDiTConfig(**TINY), seed=0)
    _, _, context, _ = tiny()
    base = stepped(model, context)
    cache = model.text_cache(context)
    assert len(cache) == 2 and cache[0].L == 80
    got = stepped(model, None, text_cache=cache)
    assert torch.equal(got, stepped(model, None, text_cache=cache))
    rel = float((got - base).norm() / base.norm())
    print(f"8-bit text cache: step differs by {rel:.2e}")
    assert 0 < rel <= 2.0 ** -4
    # a prompt's valid length is what the attention reads
    n = torch.tensor([80, 33], dtype=torch.int32, device="cuda")
    short = model.text_cache(context, n)
    garbage = context.clone()
    garbage[1, 33:] = 1e3
    assert torch.equal(stepped(model, None, text_cache=short),
                       stepped(model, None, text_cache=model.text_cache(garbage, n)))
    with pytest.raises(ValueError):
        stepped(model, None, text_cache=cache[:1])


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_model_with_4_bit_layers_follows_its_dequantised_weights(fmt):
    """The 4-bit model against the bf16 model whose weights and layer inputs
    are the dequantised ones: the two differ by the order of float32 sums and
    by bf16 roundings, but a quantised activation may step (2^-2 of a value)
    where they differ, so the outputs agree on the whole."""
    from wan_dit import WanDiT, WanDiTConfig
    from wan_dit._ops import CudaOps

    class Rounded(CudaOps):
        @staticmethod
        def fp4_weight(w, f):
            return lowp.fp4_dequantize(CudaOps.fp4_weight(w, f), torch.bfloat16)

        @staticmethod
        def fp4_linear(x, w, b=None, activation=None):
            xv = lowp.fp4_dequantize(lowp.fp4_quantize(x, fmt), torch.float32)
            y = xv @ w.float().t()
            y = y if b is None else y + b.float()
            return (torch.nn.functional.gelu(y, approximate="tanh") if activation else y).to(torch.bfloat16)
    _, _, context, _ = tiny()
    cfg = WanDiTConfig(**TINY, linear_format=fmt)
    model = WanDiT(cfg, seed=0)
    assert model.blocks[0].w1 is None and model.blocks[0].fp4["w1"].fmt == fmt
    got = stepped(model, context)
    want = stepped(WanDiT(cfg, seed=0, ops=Rounded()), context)
    bf16 = stepped(WanDiT(WanDiTConfig(**TINY), seed=0), context)
    near, far = float((got - want).norm() / want.norm()), float((got - bf16).norm() / bf16.norm())
    print(f"{fmt} model: {near:.2e} from its restatement, {far:.2e} from bf16")
    assert bool(torch.isfinite(got).all()) and near <= 3e-2 and far <= 0.5
    # with the cache as well
    both = stepped(model, None, text_cache=model.text_cache(context))
    assert bool(torch.isfinite(both).all()) and float((both - got).norm() / got.norm()) <= 2.0 ** -3
