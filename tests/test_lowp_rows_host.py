"""CPU checks of the 4-bit linear layer on rows with their own scales: refusals, before any launch."""
import math

import pytest
import torch

from wan_dit import Fp4Tensor, Kv8Cache, lowp

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4


def test_row_scales_are_for_rows_that_are_to_be_quantised():
    data, scales = (torch.zeros(s, dtype=torch.uint8) for s in lowp.fp4_storage(8, 32, "nvfp4"))
    w = Fp4Tensor(data, scales, (8, 32), "nvfp4")
    with pytest.raises(ValueError, match="row_scales"):
        lowp.fp4_linear(w, w, row_scales=True)
    with pytest.raises(ValueError, match="CUDA"):
        lowp.fp4_linear(torch.zeros(4, 32), w, row_scales=True)


@pytest.mark.parametrize("fmt", [0, 1])
def test_c_abi_refuses_before_any_launch(fmt):
    lib = lowp._load()

    def rows(fmt=fmt, x=16, dt=0, ldx=32, w=16, sw=128, gw=1.0, bias=None, act=0, out=16, ldo=8, M=4, N=8, K=32, ws=256,
             size=1 << 20):
        return lib.icsa_fp4_linear_scaled_rows(fmt, x, dt, ldx, w, sw, gw, bias, act, out, ldo, M, N, K, ws, size, None)
    for bad in (dict(fmt=7), dict(w=8), dict(sw=None), dict(gw=-1.0), dict(gw=math.nan), dict(bias=3), dict(act=2),
                dict(out=None), dict(ldo=7), dict(M=-1), dict(N=0), dict(K=0), dict(ws=128)):
        assert rows(**bad) == INVALID, bad
    need = 256 + lib.icsa_fp4_scale_bytes(fmt, 4, 32) + 256
    assert rows(ws=None) == WORKSPACE and rows(size=need - 1) == WORKSPACE
    assert rows(M=1 << 28) == UNSUPPORTED
    assert rows(M=0, x=None, out=None, ws=None, size=0) == 0
    assert lib.icsa_fp4_linear_scaled_rows_workspace_size(fmt, 0, 8, 32) == 0
    assert lib.icsa_fp4_linear_scaled_rows_workspace_size(7, 4, 8, 32) == 0


def test_global_scales_whose_product_leaves_float_are_refused():
    """alpha = a_global_scale w_global_scale is one float: beyond its range it would be an infinity or zero."""
    lib = lowp._load()

    def linear(ga, gw):
        return lib.icsa_fp4_linear(0, 16, 128, ga, 16, 128, gw, None, 0, 16, 8, 0, 8, 32, None, 0, None)
    for ga, gw in ((1e-30, 1e-30), (1e30, 1e30), (2.0 ** -100, 2.0 ** -50), (1e-22, 1e-22)):
        assert linear(ga, gw) == INVALID and b"product" in lib.icsa_last_error()
    for ga, gw in ((1e-30, 1e30), (2.0 ** -60, 2.0 ** -60), (2.0 ** 60, 2.0 ** 60), (1.0, 1e-38),
                   (2.0 ** -70, 2.0 ** -70)):                    # (small, but exact)
        assert linear(ga, gw) == 0                               # no rows: nothing to launch
    # a scale that is no float
    data, scales = (torch.zeros(s, dtype=torch.uint8) for s in lowp.fp4_storage(8, 32, "nvfp4"))
    for g in (1e-60, 1e60):
        with pytest.raises(ValueError, match="global scale"):
            Fp4Tensor(data, scales, (8, 32), "nvfp4", g)


def test_inputs_that_require_a_gradient_are_refused_where_gradients_are_enabled():
    data, scales = (torch.zeros(s, dtype=torch.uint8) for s in lowp.fp4_storage(8, 32, "nvfp4"))
    w = Fp4Tensor(data, scales, (8, 32), "nvfp4")
    x, bias = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(8, dtype=torch.bfloat16)
    cache = Kv8Cache(torch.zeros(1, 2, 1, 64, 128).to(torch.float8_e4m3fn),
                     torch.zeros(1, 2, 1, 128, 64).to(torch.float8_e4m3fn), torch.ones(1, 2, 1), torch.ones(1, 2, 1), 5)
    q = torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16)

    def leaf(t):
        return t.clone().requires_grad_()
    calls = (lambda: lowp.fp4_linear(leaf(x), w), lambda: lowp.fp4_linear(x, w, leaf(bias)),
             lambda: lowp.fp4_linear(w, w, leaf(bias)), lambda: lowp.kv8_attention(leaf(q), cache))
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):      # as without one: tensors on the CPU
            call()


def test_strided_workspace_size_refuses_what_the_attention_refuses():
    import ctypes
    lib = lowp._load()
    for bad in (dict(D=32), dict(B=0), dict(L=0)):
        d = {**dict(B=1, H=2, L=5, D=128), **bad}
        assert lib.icsa_kv8_attention_strided_workspace_size(ctypes.byref(lowp._Kv8Desc(*d.values())), 1, 2) == 0
    assert lib.icsa_kv8_attention_strided_workspace_size(ctypes.byref(lowp._Kv8Desc(1, 2, 5, 128)), 1, 3) == 0
