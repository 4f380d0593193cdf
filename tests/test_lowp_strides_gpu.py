"""GPU tests of the attention over an 8-bit cache for queries of other layouts than rows: the kernels of a few
queries and of SM pairs take any strides as they are, the copy of a long cache takes rows."""
import ctypes

import pytest
import torch

from wan_dit import lowp

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _device(cuda_device):
    lowp._load()
    yield
    from in_context_sparse_attention import device_status
    device_status()


def case(B, Lq, L, H, group, D):
    g = torch.Generator().manual_seed(Lq + L + D)
    k, v = (torch.randn(B, L, H, D, generator=g).cuda() for _ in range(2))
    q = torch.randn(B, Lq, H * group, D, generator=g).to(torch.bfloat16).cuda()
    return q, lowp.kv8_quantize(k, v)


def layouts(q):
    """The same queries in other strides."""
    B, Lq, H, D = q.shape
    yield q.transpose(1, 2).contiguous().transpose(1, 2)                      # heads outside
    yield q.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)              # tokens outside
    yield torch.cat([q, q, q], 2)[:, :, H:2 * H]                              # rows of a wider tensor
    yield torch.cat([q, q], 3)[..., D:]                                       # wider heads
    yield torch.cat([q, q[:, :1]], 1)[:, :Lq]                                 # gaps between batch elements


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Lq,L,H,group", [(2, 1, 300, 4, 1), (2, 5, 3000, 2, 3), (1, 16, 700, 40, 1),
                                            (2, 300, 450, 40, 1), (4, 150, 331, 16, 2), (1, 512, 8000, 8, 1),
                                            (2, 100, 331, 16, 5)])
def test_queries_of_any_strides_are_read_as_they_are(B, Lq, L, H, group, D):
    q, cache = case(B, Lq, L, H, group, D)
    want = lowp.kv8_attention(q, cache)
    for x in layouts(q):
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats()["allocation.all.allocated"]
        got = lowp.kv8_attention(x, cache)
        # the output, and a workspace where there is one: no copy of the queries
        assert torch.cuda.memory_stats()["allocation.all.allocated"] - before <= 2 - (lowp._attention_workspace(
            0, B, H, L, D, Lq, H * group) == 0)
        assert torch.equal(got, want)
    one = q[:, :1].expand(B, Lq, H * group, D)                                # one token for all
    assert torch.equal(lowp.kv8_attention(one, cache), lowp.kv8_attention(one.contiguous(), cache))


@pytest.mark.parametrize("D", [64, 128])
def test_strided_queries_over_a_long_cache_take_the_pair_kernel_in_its_workspace(D):
    lib = lowp._load()
    q, cache = case(1, 4096, 2000, 8, 1, D)
    desc = cache._desc()
    plain = lib.icsa_kv8_attention_workspace_size(ctypes.byref(desc), 4096, 8)
    size = lib.icsa_kv8_attention_strided_workspace_size(ctypes.byref(desc), 4096, 8)
    assert size != plain
    want = lowp.kv8_attention(q, cache)
    for x in layouts(q):
        assert torch.equal(lowp.kv8_attention(x, cache), want)                # Python copies the queries here
    x = q.transpose(1, 2).contiguous().transpose(1, 2)
    ws = torch.full((max(size, plain) + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(want)

    def call(n):
        return lib.icsa_kv8_attention(ctypes.byref(desc), x.data_ptr(), (ctypes.c_int64 * 3)(0, *x.stride()[1:3]),
                                      out.data_ptr(), 4096, 8, ws.data_ptr(), n,
                                      torch.cuda.current_stream().cuda_stream)
    assert call(size - 1) == 2 and b"strided_workspace_size" in lib.icsa_last_error() and not bool(out.any())
    assert call(size) == 0
    # two kernels of the same rounding: each is off by 2^-11 of sum p |v| and 2^-8 of the result, and more in the sums
    p = torch.softmax(torch.einsum("bqhd,bkhd->bhqk", q.float(), lowp.kv8_dequantize(cache, torch.float32)[0])
                      / D ** 0.5, -1)
    mass = torch.einsum("bhqk,bkhd->bqhd", p, lowp.kv8_dequantize(cache, torch.float32)[1].abs())
    d = (out.float() - want.float()).abs()
    assert bool((d <= 2 * (mass * 2.0 ** -10 + want.float().abs() * 2.0 ** -8)).all())
    assert bool((ws[max(size, plain):] == 0xFF).all())
