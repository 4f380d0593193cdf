"""The low-precision operators (include/icsa_lowp.h) restated in 64 bits on the
CPU: quantisation by nearest-value search over the format's tables, storage by
explicit indices, linear layers and attention as float64 sums."""
import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def e4m3_table():
    """Non-negative finite e4m3 values by code (0 .. 0x7e)."""
    out = []
    for c in range(0x7F):
        e, m = c >> 3, c & 7
        out.append(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return out


def nearest_code(a, table):
    """Index of the table value nearest to each a >= 0, ties to the even index, the last where a is beyond."""
    t = torch.tensor(table, dtype=torch.float64)
    mid = (t[1:] + t[:-1]) / 2
    a = a.double().contiguous()
    up = torch.searchsorted(mid, a, right=False)          # mid[i] < a counted: ties stay below
    tie = (up < len(mid)) & (mid[up.clamp(max=len(mid) - 1)] == a)
    return torch.where(tie & (up % 2 == 1), up + 1, up)


def fp4_quantize(x, fmt, g=1.0):
    """(codes uint8 [rows, K'], scale bytes uint8 [rows, blocks], values f64 [rows, K]); K' = K padded to the block.
    Quotients are those of float32 division, which the formats' definition names."""
    n = 16 if fmt == "nvfp4" else 32
    rows, K = x.shape
    b = torch.nn.functional.pad(x.float().cpu(), (0, -K % n)).view(rows, -1, n)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    safe = torch.where(bad, 0.0, top)
    g32 = torch.tensor(g, dtype=torch.float32)
    if fmt == "nvfp4":
        sb = nearest_code(safe / (torch.tensor(6.0) * g32), e4m3_table())
        d = torch.tensor(e4m3_table())[sb].float() * g32
        sb = torch.where(bad, 0x7F, sb)
    else:
        e = (torch.frexp(safe.double())[1] - 3).clamp(-127, 127)
        e = torch.where(safe == 0, -127, e)
        d = torch.ldexp(torch.ones_like(safe, dtype=torch.float64), e)
        sb = torch.where(bad, 0xFF, e + 127)
    dd = d.unsqueeze(-1)
    q = torch.where(dd > 0, (b.double() / dd if fmt == "mxfp4" else (b / dd).double()), 0.0)
    q = torch.where(bad.unsqueeze(-1), 0.0, q)
    code = nearest_code(q.abs(), E2M1)
    val = torch.tensor(E2M1, dtype=torch.float64)[code] * dd.double() * torch.where(torch.signbit(b), -1.0, 1.0)
    val = torch.where(bad.unsqueeze(-1), math.nan, val)
    code = torch.where((dd > 0) & ~bad.unsqueeze(-1), code + 8 * torch.signbit(b), 0)   # code 0 where there is no step
    return code.view(rows, -1).to(torch.uint8), sb.to(torch.uint8), val.reshape(rows, -1)[:, :K]


def fp4_scale_bytes(sb, rows, K, fmt):
    """The scale buffer, byte by byte, from [rows, blocks] scale bytes."""
    atoms = 4 if fmt == "nvfp4" else 2
    k_tiles = -(-K // 256)
    buf = torch.zeros(-(-rows // 128) * k_tiles * atoms * 512, dtype=torch.uint8)
    r = torch.arange(rows)[:, None]
    c = torch.arange(sb.shape[1])[None]
    at = ((r // 128) * k_tiles * atoms + c // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + c % 4
    buf[at.expand(rows, sb.shape[1]).reshape(-1)] = sb.reshape(-1)
    return buf


def fp4_data_bytes(code, K):
    """[rows, K' / 2] packed codes, K' = K rounded up to 32."""
    kp = -(-K // 32) * 32
    full = torch.zeros(code.shape[0], kp, dtype=torch.uint8)
    full[:, :K] = code[:, :K]
    return full[:, 0::2] | (full[:, 1::2] << 4)


def gelu_tanh(y):
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def kv8_quantize(x, lengths=None):
    """(codes uint8 [B, H, nb, 64, D], scales f32 [B, H, nb], values f64 [B, L, H, D])."""
    B, L, H, D = x.shape
    nb = -(-L // 64)
    x = x.float().cpu()
    codes = torch.zeros(B, H, nb, 64, D, dtype=torch.uint8)
    scales = torch.ones(B, H, nb)
    values = torch.zeros(B, L, H, D, dtype=torch.float64)
    table = e4m3_table()
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        for i in range(-(-n // 64)):
            part = x[b, 64 * i:min(64 * i + 64, n)]                  # [t, H, D]
            for h in range(H):
                p = part[:, h]
                if not torch.isfinite(p).all():
                    scales[b, h, i] = math.nan
                    values[b, 64 * i:64 * i + p.shape[0], h] = math.nan
                    continue
                top = float(p.abs().max())
                e = 0
                if top > 0:
                    e = math.frexp(top / 448)[1]
                    if 448 * 2.0 ** (e - 1) >= top:
                        e -= 1
                    e = min(max(e, -96), 96)
                q = p.double() * 2.0 ** -e
                c = nearest_code(q.abs(), table)
                scales[b, h, i] = 2.0 ** e
                codes[b, h, i, :p.shape[0]] = (c + 128 * torch.signbit(p)).to(torch.uint8)
                values[b, 64 * i:64 * i + p.shape[0], h] = (torch.tensor(table, dtype=torch.float64)[c] * 2.0 ** e
                                                            * torch.where(torch.signbit(p), -1.0, 1.0))
    return codes, scales, values


def attention(q, k, v, lengths=None):
    """(softmax(q k^T / sqrt D) v, sum of p |v|, largest |score|) in f64; k, v f64 [B, L, H, D]."""
    B, Lq, Hq, D = q.shape
    H = k.shape[2]
    out = torch.zeros(B, Lq, Hq, D, dtype=torch.float64)
    mass = torch.zeros_like(out)
    big = 0.0
    for b in range(B):
        n = k.shape[1] if lengths is None else min(max(int(lengths[b]), 0), k.shape[1])
        if n == 0:
            continue
        for h in range(Hq):
            hk = h // (Hq // H)
            s = q[b, :, h].double().cpu() @ k[b, :n, hk].T / math.sqrt(D)
            p = torch.softmax(s, -1)
            out[b, :, h] = p @ v[b, :n, hk]
            mass[b, :, h] = p @ v[b, :n, hk].abs()
            big = max(big, float(s.abs().nan_to_num(0.0).max()))
    return out, mass, big
