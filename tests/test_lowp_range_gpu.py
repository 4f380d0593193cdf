"""GPU tests of the low-precision operators where magnitudes lie far apart:
value blocks of unequal scales in the attention over an 8-bit cache.

Bound of an attention result, with p the probabilities of the row, v the
values that the cache holds and "mass" = sum p |v|:
  * one rounding to bf16: 2^-8 of the result;
  * the probabilities' rounding.  In f16 2^-11 of each, and for those below
    2^-14 of the row's largest 2^-25 of that one: 2^-11 mass + 2^-25 max(p)
    sum |v|.  In bf16, on the copy of a head whose scales lie more than 2^22
    apart, 2^-8 mass;
  * scores: float32 sums of D products, 16 to an instruction, with sa the
    largest sum |q k| / sqrt(D): at most (16 + D / 16) 2^-23 sa < 2^-18 sa,
    and 2^-18 for the exponential; p moves by as much of itself;
  * sums over L keys, 16 to an instruction: (L / 16 + 64) 2^-23 of the mass.
No term knows a block's scale: what a block of large values holds may not
cost the others bits."""
import ctypes
import math

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


# --------------------------------------------------------------------------- attention
def on_copy(cache, Lq, Hq):
    """Whether the call runs on a bf16 copy of the cache: told by its workspace."""
    B, H, _, _, D = cache.k.shape
    size = lowp._load().icsa_kv8_attention_workspace_size(ctypes.byref(cache._desc()), Lq, Hq)
    return size == 2 * (-(-B * cache.L * H * D * 2 // 256) * 256) + -(-B * H * 4 // 256) * 256


def check(q, cache, copy=None):
    """kv8_attention within the bound above; returns the worst error as a share of it."""
    B, Lq, Hq, D = q.shape
    got = lowp.kv8_attention(q, cache)
    k, v = (t.double() for t in lowp.kv8_dequantize(cache, torch.float32))
    L, H = k.shape[1:3]
    if copy is not None:
        assert on_copy(cache, Lq, Hq) == copy
    copied = on_copy(cache, Lq, Hq)
    worst = 0.0
    for b in range(B):
        n = L if cache.lengths is None else min(max(int(cache.lengths[b]), 0), L)
        if n == 0:
            assert not bool(got[b].any())
            continue
        for h in range(Hq):
            kk, vv, qq = k[b, :n, h * H // Hq], v[b, :n, h * H // Hq], q[b, :, h].double()
            sa = float((qq.abs() @ kk.abs().T).max()) / math.sqrt(D)
            p = torch.softmax(qq @ kk.T / math.sqrt(D), -1)
            want, mass = p @ vv, p @ vv.abs()
            e = torch.log2(cache.v_scale[b, h * H // Hq, :-(-n // 64)])
            bits = 8 if copied and float(e.max() - e.min()) > 22 else 11
            tol = (want.abs() * 2.0 ** -8 + mass * (2.0 ** -bits + (sa + 1) * 2.0 ** -18 + (n / 16 + 64) * 2.0 ** -23)
                   + 1e-38)
            if bits == 11:
                tol = tol + 2.0 ** -25 * p.amax(-1, keepdim=True) * vv.abs().sum(0)
            d = (got[b, :, h].double() - want).abs()
            assert bool((d <= tol).all()), (b, h, float((d / tol).max()))
            worst = max(worst, float((d / tol).max()))
    print(f"attention {tuple(q.shape)} over {L}: worst error {worst:.3f} of its bound")
    return got


# One line per path: batch, queries, keys, heads, query heads per cache head, whether it runs on the copy (at D = 128).
PATHS = {"few rows": (2, 2, 500, 2, 1, False), "few rows, shared heads": (2, 9, 331, 2, 4, False),
         "few rows, splits": (1, 3, 9000, 2, 1, False), "two groups": (2, 16, 700, 40, 1, False),
         "whole rounds": (2, 300, 450, 40, 1, False), "one tile": (2, 200, 450, 16, 1, False),
         "whole rounds, two tiles": (2, 700, 331, 16, 1, False),
         "cut rounds": (1, 512, 8000, 8, 1, False), "cut rounds, shared heads": (1, 150, 8000, 8, 3, False),
         "copy": (1, 4096, 2000, 8, 1, True)}

# exponents of the 64-token blocks' values, repeated over the cache; None: a block of zeros
PATTERNS = {"zeros beside 2^-10": [None, -10], "zeros beside 2^-20": [-20, None, -20], "zeros beside 2^-40": [None, -40],
            "zeros first, then 2^-90": [None] + [-90] * 200, "steps within a pair": [0, -9, 3, -6, 0, 8],
            "far steps": [0, -20, 20, 3, -3, 0, 10, -60], "falling": [-3 * i for i in range(200)],
            "rising": [3 * i - 60 for i in range(40)], "one large": [30] + [0] * 200}


def pattern_rows(L, exps):
    e = [exps[i % len(exps)] for i in range(-(-L // 64))]
    s = torch.tensor([0.0 if x is None else 2.0 ** max(min(x, 90), -90) for x in e], dtype=torch.float64)
    return s.repeat_interleave(64)[:L]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pattern", list(PATTERNS))
@pytest.mark.parametrize("path", list(PATHS))
def test_value_blocks_of_unequal_scales_cost_no_bits(path, pattern, D):
    B, Lq, L, H, group, copy = PATHS[path]
    g = torch.Generator().manual_seed(L + D)
    k, v = (torch.randn(B, L, H, D, generator=g) for _ in range(2))
    v = (v.double() * pattern_rows(L, PATTERNS[pattern])[None, :, None, None]).float()
    q = torch.randn(B, Lq, H * group, D, generator=g).to(torch.bfloat16).cuda()
    check(q, lowp.kv8_quantize(k.cuda(), v.cuda()), copy if D == 128 else None)


@pytest.mark.parametrize("path", ["few rows", "few rows, splits", "whole rounds", "cut rounds", "copy"])
def test_a_row_sees_its_own_key_beside_large_values_of_others(path):
    """Each row's probability lies on one key whose values are 2^-30 of what the other blocks hold; and an
    outlier that no row looks at sets a block's scale, its other values being zero."""
    B, Lq, L, H, _, copy = PATHS[path]
    D = 128
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(B, L, H, D, generator=g) for _ in range(2))
    own = torch.arange(Lq) * 37 % (L // 64) * 64 + 5          # a key in some block, the same for several rows
    v[:, own] *= 2.0 ** -30
    k = k * 0.01
    k[:, own] = torch.randn(1, 1, H, D, generator=g) * 8
    q = (k[:, own] * 0.5).to(torch.bfloat16).cuda()           # score about 8 * 4 * sqrt(128)
    check(q, lowp.kv8_quantize(k.cuda(), v.cuda()), copy)
    v = torch.randn(B, L, H, D, generator=g) * 2.0 ** -24
    v[:, 128:192] = 0.0
    v[:, 150] = 1.0
    k[:, 150] = -q[0, 0].float().cpu()                         # (score far below every other)
    check(q, lowp.kv8_quantize(k.cuda(), v.cuda()), copy)


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("D", [64, 128])
def test_probabilities_keep_the_bits_of_their_path(path, D):
    """Ordinary values and ragged lengths, at the bound of the path that was taken."""
    _, Lq, L, H, group, _ = PATHS[path]
    g = torch.Generator().manual_seed(L)
    k, v = (torch.randn(3, L, H, D, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn(3, Lq, H * group, D, generator=g).to(torch.bfloat16).cuda()
    n = torch.tensor([L, 0, L - 77], dtype=torch.int32, device="cuda")
    check(q, lowp.kv8_quantize(k, v, n))


@pytest.mark.parametrize("D", [64, 128])
def test_copied_heads_of_both_kinds(D):
    """Heads whose scales lie near together and far apart, shared by query heads, with lengths that leave the far
    blocks of one sequence out; then blocks exactly 22 and 23 binades apart, and a block with a NaN."""
    g = torch.Generator().manual_seed(9)
    B, Lq, L, H, group = 2, 4096, 2000, 4, 2
    k, v = (torch.randn(B, L, H, D, generator=g) for _ in range(2))
    v[:, :1024, 1] *= 2.0 ** -30
    v[:, 1024:, 2] *= 2.0 ** 40
    v[:, 64:128, 3] = 0.0
    q = torch.randn(B, Lq, H * group, D, generator=g).to(torch.bfloat16).cuda()
    n = torch.tensor([L, 1000], dtype=torch.int32, device="cuda")
    check(q, lowp.kv8_quantize(k.cuda(), v.cuda(), n), True)
    v = torch.randn(B, L, H, D, generator=g).clamp(-3, 3)
    v[:, ::64] = 3.0                                            # the same scale in every block
    v[:, 640:704, 0] *= 2.0 ** -22
    v[:, 640:704, 1] *= 2.0 ** -23
    cache = lowp.kv8_quantize(k.cuda(), v.cuda(), n)
    for h, apart in ((0, 22), (1, 23), (2, 0)):
        e = torch.log2(cache.v_scale[0, h])
        assert float(e.max() - e.min()) == apart
    clean = check(q, cache, True)
    v[0, 700, 2, 5] = math.nan
    bad = lowp.kv8_attention(q, lowp.kv8_quantize(k.cuda(), v.cuda(), n))
    assert bool(torch.isnan(bad[0, :, 4:6]).all())
    rest = torch.ones(B, H * group, dtype=torch.bool)
    rest[0, 4:6] = False
    assert all(torch.equal(bad[b, :, h], clean[b, :, h]) for b in range(B) for h in range(H * group) if rest[b, h])


def test_a_replayed_call_follows_scales_that_change():
    """Which steps are taken in two parts is read from the cache on the device."""
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 450, 40, 128, generator=g).cuda() for _ in range(2))
    q = torch.randn(2, 300, 40, 128, generator=g).to(torch.bfloat16).cuda()
    lowp.kv8_attention(q, lowp.kv8_quantize(k, v))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lowp.kv8_attention(q, lowp.kv8_quantize(k, v))
    base = v.clone()
    for pattern in ("far steps", "one large", "zeros beside 2^-20"):
        v.copy_(base * pattern_rows(450, PATTERNS[pattern]).float().cuda()[None, :, None, None])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check(q, lowp.kv8_quantize(k, v)))
