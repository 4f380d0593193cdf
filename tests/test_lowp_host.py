"""CPU checks of the low-precision operators: the storage containers, the
refusals of the Python functions and of the C ABI (before any launch), and
the 64-bit restatement that the GPU tests compare with."""
import ctypes
import math

import pytest
import torch

import _lowp_reference as ref
from wan_dit import lowp
from wan_dit import Fp4Tensor, Kv8Cache, WanDiT, WanDiTConfig

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4


def test_nearest_code_ties_go_to_the_even_code():
    a = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2500001, 4.9999, 7.0, 0.0])
    assert ref.nearest_code(a, ref.E2M1).tolist() == [0, 2, 2, 4, 4, 6, 6, 1, 6, 7, 0]
    t = ref.e4m3_table()
    assert t[-1] == 448 and t[1] == 2.0 ** -9 and len(t) == 127
    x = torch.randn(1000).abs() * 100
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).long()
    assert torch.equal(ref.nearest_code(x, t), want)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 47), (128, 256), (129, 257), (700, 5120)])
def test_storage_sizes_agree_between_python_and_c(fmt, rows, K):
    lib = lowp._load()
    data, scales = lowp.fp4_storage(rows, K, fmt)
    assert math.prod(data) == lib.icsa_fp4_data_bytes(rows, K)
    assert math.prod(scales) == lib.icsa_fp4_scale_bytes(lowp.FP4_FORMATS[fmt], rows, K)
    # every scale has a byte of its own
    blocks = -(-K // lowp.FP4_BLOCK[fmt])
    sb = torch.ones(rows, blocks, dtype=torch.uint8)
    assert int(ref.fp4_scale_bytes(sb, rows, K, fmt).sum()) == rows * blocks


def test_containers_check_their_tensors():
    data, scales = (torch.zeros(s, dtype=torch.uint8) for s in lowp.fp4_storage(3, 47, "nvfp4"))
    t = Fp4Tensor(data, scales, (3, 47), "nvfp4", 0.5)
    assert t.shape == (3, 47)
    for bad in (dict(shape=(4, 47)), dict(fmt="fp4"), dict(fmt="mxfp4"), dict(global_scale=0.0),
                dict(global_scale=math.inf), dict(global_scale=math.nan), dict(data=data.int()),
                dict(data=torch.zeros(24, 3, dtype=torch.uint8).t()), dict(shape=(3, 0))):
        with pytest.raises(ValueError):
            Fp4Tensor(**{**dict(data=data, scales=scales, shape=(3, 47), fmt="nvfp4", global_scale=1.0), **bad})
    k = torch.zeros(2, 3, 2, 64, 128).to(torch.float8_e4m3fn)
    v = torch.zeros(2, 3, 2, 128, 64).to(torch.float8_e4m3fn)
    s = torch.ones(2, 3, 2)
    n = torch.tensor([5, 70], dtype=torch.int32)
    Kv8Cache(k, v, s, s, 100, n)
    for bad in (dict(L=64), dict(L=129), dict(L=0), dict(v=k), dict(k_scale=s.double()), dict(v_scale=s[:1]),
                dict(lengths=n.long()), dict(lengths=n[:1]), dict(k=k.float())):
        with pytest.raises(ValueError):
            Kv8Cache(**{**dict(k=k, v=v, k_scale=s, v_scale=s, L=100, lengths=n), **bad})


def test_global_scale_is_the_smallest_power_of_two_in_range():
    for top in (1e-30, 0.02, 2688.0, 2689.0, 1.0, 3e38):
        g = lowp.fp4_global_scale(torch.tensor([[-top, 0.0]]))
        assert math.frexp(g)[0] == 0.5
        t32 = float(torch.tensor(top))
        assert t32 <= g * 2688 * (1 + 1e-12) or g == 2.0 ** 100
        assert t32 > g / 2 * 2688 or g == 2.0 ** -100
    assert lowp.fp4_global_scale(torch.zeros(2, 3)) == 1.0
    with pytest.raises(ValueError):
        lowp.fp4_global_scale(torch.tensor([math.nan]))


def test_python_functions_refuse_what_they_cannot_take():
    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    data, scales = (torch.zeros(s, dtype=torch.uint8) for s in lowp.fp4_storage(8, 32, "nvfp4"))
    w = Fp4Tensor(data, scales, (8, 32), "nvfp4")
    kv = torch.zeros(1, 5, 2, 128, dtype=torch.bfloat16)
    cache = Kv8Cache(torch.zeros(1, 2, 1, 64, 128).to(torch.float8_e4m3fn),
                     torch.zeros(1, 2, 1, 128, 64).to(torch.float8_e4m3fn), torch.ones(1, 2, 1), torch.ones(1, 2, 1), 5)
    for call in (lambda: lowp.fp4_quantize(x), lambda: lowp.fp4_quantize(x, "fp4"),
                 lambda: lowp.fp4_quantize(x, "mxfp4", 2.0), lambda: lowp.fp4_quantize(x, "nvfp4", -1.0),
                 lambda: lowp.fp4_dequantize(w), lambda: lowp.fp4_dequantize(w, torch.float16),
                 lambda: lowp.fp4_linear(x, w), lambda: lowp.fp4_linear(x, w, activation="relu"),
                 lambda: lowp.fp4_linear(x, x), lambda: lowp.fp4_linear(x[:, :16], w),
                 lambda: lowp.fp4_linear(x, w, torch.zeros(8)),
                 lambda: lowp.kv8_quantize(kv, kv), lambda: lowp.kv8_dequantize(cache),
                 lambda: lowp.kv8_attention(kv, cache)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        WanDiT(WanDiTConfig(dim=256, num_heads=2, num_layers=0, linear_format="fp8"), device="cpu", ops=object())


def test_c_abi_refuses_before_any_launch():
    lib = lowp._load()
    e = lambda: lib.icsa_last_error()  # noqa: E731
    assert lib.icsa_fp4_quantize(16, 0, 31, 4, 32, 0, 1.0, 16, 128, None) == INVALID and b"ldx" in e()
    assert lib.icsa_fp4_quantize(16, 0, 32, 4, 32, 2, 1.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(16, 5, 32, 4, 32, 0, 1.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(16, 0, 32, -1, 32, 0, 1.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(16, 0, 32, 4, 0, 0, 1.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(16, 0, 32, 4, 32, 0, 0.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(16, 0, 32, 4, 32, 1, 2.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(16, 0, 32, 4, 32, 0, 1.0, 8, 128, None) == INVALID and b"aligned" in e()
    assert lib.icsa_fp4_quantize(16, 0, 32, 4, 32, 0, 1.0, 16, 64, None) == INVALID
    assert lib.icsa_fp4_quantize(17, 0, 32, 4, 32, 0, 1.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(None, 0, 32, 4, 32, 0, 1.0, 16, 128, None) == INVALID
    assert lib.icsa_fp4_quantize(16, 0, 1 << 30, 4, 1 << 30, 0, 1.0, 16, 128, None) == UNSUPPORTED
    assert lib.icsa_fp4_quantize(None, 0, 32, 0, 32, 0, 1.0, None, None, None) == 0           # no rows: nothing to do
    assert lib.icsa_fp4_dequantize(16, 128, 4, 32, 0, 1.0, 16, 0, 31, None) == INVALID
    assert lib.icsa_fp4_dequantize(16, 128, 4, 32, 0, 1.0, 2, 1, 32, None) == INVALID
    assert lib.icsa_fp4_dequantize(16, None, 4, 32, 0, 1.0, 16, 1, 32, None) == INVALID

    def linear(fmt=0, a=16, sa=128, ga=1.0, w=16, sw=128, gw=1.0, bias=None, act=0, out=16, ldo=8, M=4, N=8, K=32):
        return lib.icsa_fp4_linear(fmt, a, sa, ga, w, sw, gw, bias, act, out, ldo, M, N, K, None, 0, None)
    for bad in (dict(fmt=7), dict(a=None), dict(sa=64), dict(w=8), dict(sw=None), dict(ga=-1.0), dict(gw=math.nan),
                dict(bias=3), dict(act=2), dict(out=None), dict(out=1), dict(ldo=7), dict(M=-1), dict(N=0), dict(K=0),
                dict(fmt=1, ga=0.5)):
        assert linear(**bad) == INVALID, bad
    assert linear(M=1 << 28) == UNSUPPORTED
    assert linear(M=0, a=None, out=None) == 0

    def rows(fmt=0, x=16, dt=0, ldx=32, w=16, sw=128, gw=1.0, bias=None, act=0, out=16, ldo=8, M=4, N=8, K=32, ws=256,
             size=1 << 20):
        return lib.icsa_fp4_linear_rows(fmt, x, dt, ldx, w, sw, gw, bias, act, out, ldo, M, N, K, ws, size, None)
    for bad in (dict(fmt=7), dict(w=8), dict(sw=None), dict(gw=-1.0), dict(bias=3), dict(act=2), dict(out=None),
                dict(ldo=7), dict(M=-1), dict(N=0), dict(K=0), dict(ws=128)):
        assert rows(**bad) == INVALID, bad
    assert rows(ws=None) == WORKSPACE and rows(size=100) == WORKSPACE
    assert rows(M=0, x=None, out=None, ws=None, size=0) == 0

    strides = (ctypes.c_int64 * 3)(0, 256, 128)
    odd = (ctypes.c_int64 * 3)(0, 257, 128)
    neg = (ctypes.c_int64 * 3)(0, -256, 128)

    def desc(**kw):
        d = dict(B=1, H=2, L=5, D=128, k=16, v=16, k_scale=16, v_scale=16, lengths=None)
        return ctypes.byref(lowp._Kv8Desc(*{**d, **kw}.values()))
    for bad, code in ((dict(B=0), INVALID), (dict(H=0), INVALID), (dict(L=0), INVALID), (dict(D=96), UNSUPPORTED),
                      (dict(k=None), INVALID), (dict(v_scale=None), INVALID), (dict(v=8), INVALID),
                      (dict(lengths=2), INVALID), (dict(B=40000, H=2), UNSUPPORTED), (dict(L=1 << 31 - 1), INVALID)):
        if bad == dict(L=1 << 31 - 1):
            bad, code = dict(L=(1 << 31) - 1), UNSUPPORTED
        assert lib.icsa_kv8_quantize(desc(**bad), 16, 16, 0, strides, strides, None) == code, bad
        assert lib.icsa_kv8_attention(desc(**bad), 16, strides, 16, 1, 2, None, 0, None) == code, bad
    assert lib.icsa_kv8_quantize(None, 16, 16, 0, strides, strides, None) == INVALID
    assert lib.icsa_kv8_quantize(desc(), None, 16, 0, strides, strides, None) == INVALID
    assert lib.icsa_kv8_quantize(desc(), 16, 16, 3, strides, strides, None) == INVALID
    assert lib.icsa_kv8_quantize(desc(), 16, 18, 1, strides, strides, None) == INVALID
    assert lib.icsa_kv8_quantize(desc(), 16, 16, 0, strides, neg, None) == INVALID
    assert lib.icsa_kv8_dequantize(desc(), 8, 16, 0, None) == INVALID
    assert lib.icsa_kv8_dequantize(desc(), 16, 16, 9, None) == INVALID
    assert lib.icsa_kv8_dequantize(desc(), None, None, 0, None) == 0
    for args in ((None, strides, 16, 1, 2), (16, None, 16, 1, 2), (16, strides, None, 1, 2), (8, strides, 16, 1, 2),
                 (16, strides, 24, 1, 2), (16, odd, 16, 1, 2), (16, neg, 16, 1, 2), (16, strides, 16, 0, 2),
                 (16, strides, 16, 1, 3), (16, strides, 16, 1, 0)):
        assert lib.icsa_kv8_attention(desc(), *args, None, 0, None) == INVALID, args
    assert lib.icsa_kv8_attention_workspace_size(desc(D=32), 1, 2) == 0


def test_restated_cache_uses_the_smallest_scale_that_fits():
    x = torch.zeros(1, 130, 1, 64)
    x[0, 0, 0, 0], x[0, 64, 0, 3], x[0, 129, 0, 5] = 448.0, -449.0, 1e-35
    codes, scales, values = ref.kv8_quantize(x)
    assert scales.flatten().tolist() == [1.0, 2.0, 2.0 ** -96]
    assert values[0, 0, 0, 0] == 448 and values[0, 64, 0, 3] == -448 and values[0, 129, 0, 5] == 0
    assert int(codes[0, 0, 0, 0, 0]) == 0x7E
