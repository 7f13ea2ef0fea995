"""Plain 64-bit statements of the serving operators, for their tests: no code of the package, no fused torch calls."""
import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def e4m3_table():
    v = []
    for code in range(128):
        e, m = code >> 3, code & 7
        v.append(math.nan if code == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return torch.tensor(v + [-x for x in v], dtype=torch.float64)


def e2m1_table():
    return torch.tensor(E2M1 + [-x for x in E2M1], dtype=torch.float64)


def scale_table():
    return torch.tensor([2.0 ** (b - 127) for b in range(255)] + [math.nan], dtype=torch.float64)


def decode(codes, scale, fp4):
    """Values (..., d) in 64 bits of packed codes (..., bytes) and scale bytes (..., d / 32)."""
    codes, scale = codes.cpu(), scale.cpu()
    if fp4:
        v = e2m1_table()[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()]
    else:
        v = e4m3_table()[codes.long()]
    return v * scale_table()[scale.long()].repeat_interleave(32, -1)


def quantise_block(x, fp4):
    """(values, scale byte) of one block of 32 floats, by search: the smallest power of two at which nothing saturates,
    then for each element the nearest value of the format, ties to the even code."""
    x = [float(v) for v in x]
    if not all(math.isfinite(v) for v in x):
        return [math.nan] * 32, 255
    grid = E2M1 if fp4 else e4m3_table()[:127].tolist()
    byte = 0
    while byte < (252 if fp4 else 246) and max(abs(v) for v in x) > grid[-1] * 2.0 ** (byte - 127):
        byte += 1
    out = []
    for v in x:
        a = min(abs(v) * 2.0 ** (127 - byte), grid[-1])
        best = min(range(len(grid)), key=lambda c: (abs(grid[c] - a), c & 1))
        out.append(math.copysign(grid[best] * 2.0 ** (byte - 127), v))
    return out, byte


def attention(q, prefix_k, prefix_v, own_k, own_v, scale):
    """q (batch, tokens, heads, d), prefix (kv_heads, n, d), own: one (kv_heads, n_b, d) a sequence, all float64.
    Returns o, lse, and per output element what the error bound needs: sum of w |v|, sum of |v|, largest sum |q||k|."""
    batch, tokens, heads, d = q.shape
    o, lse = torch.zeros_like(q), torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=q.device)
    wv, vsum, qk = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(lse)
    kv = prefix_k.shape[0]
    g = heads // kv
    for b in range(batch):
        for j in range(tokens):
            n = max(0, own_k[b].shape[1] - (tokens - 1 - j))
            k = torch.cat([prefix_k, own_k[b][:, :n]], 1)
            v = torch.cat([prefix_v, own_v[b][:, :n]], 1)
            if k.shape[1] == 0:
                continue
            qq = q[b, j].view(kv, g, d)
            x = torch.matmul(qq, k.transpose(1, 2)) * scale
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - top)
            total = p.sum(-1, keepdim=True)
            w = p / total
            o[b, j] = torch.matmul(w, v).view(heads, d)
            lse[b, j] = (torch.log(total) + top).view(heads)
            wv[b, j] = torch.matmul(w, v.abs()).view(heads, d)
            vsum[b, j] = v.abs().sum(1).repeat_interleave(g, 0)
            qk[b, j] = (torch.matmul(qq.abs(), k.abs().transpose(1, 2)).amax(-1) * abs(scale)).view(heads)
    return o, lse, wv, vsum, qk


def attention_bounds(dtype, o, wv, vsum, qk, keys, mx=False):
    """Error bounds of (o, lse), derived: with u = 2^-22 for every fp32 operation in a chain (tensor-core sums may truncate)
      logit: at most 24 sums of products of total magnitude qk -> 24 u qk, twice that in exp, u each for exp2 and scaling;
      weights: rounded to `dtype` once, eps / 2, below float16's normal range 2^-25 absolute (their maximum is 1);
      sums: keys / 16 + 48 fp32 additions; V: below float16's normal range 2^-25 absolute; output: one more rounding.
    Over an MX cache (mx) the weights are float16 for either `dtype`: relative 2^-11, which eps / 2 covers, and below 2^-14,
    where float16's places are 2^-24 apart, 2^-25 absolute; the weights being at most 1 and their sum at least 1, that is
    2^-25 |v| a key, at most 2^-25 vsum."""
    half = torch.finfo(dtype).eps / 2
    u = 2.0 ** -22
    logit = (24 * qk + 8) * u
    chain = (keys / 16 + 48) * u
    rel = half + 2 * logit[..., None] + 2 * chain
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return rel * wv + (2.0 ** -25 if mx else tiny) * vsum + 2 * tiny + half * o.abs() + 1e-30, logit + chain + u * 8


def w4_weights(w, scale, zero, group):
    """(n, k) float64 weights and their magnitude bound |code - 8| s + |8 - zero| s."""
    w, scale = w.cpu(), scale.cpu()
    codes = torch.stack([w & 15, w >> 4], -1).flatten(-2)
    if scale.dtype == torch.uint8:
        v = e2m1_table()[codes.long()] * scale_table()[scale.long()].repeat_interleave(group, -1)
        return v, v.abs()
    s = scale.double().repeat_interleave(group, -1)
    z = zero.cpu().double().repeat_interleave(group, -1) if zero is not None else torch.full_like(s, 8.0)
    c = codes.double()
    return s * (c - z), s.abs() * ((c - 8).abs() + (8 - z).abs())


def w4_bound(dtype, out_dtype, x, mag, y, k):
    """Error bound of w4_matvec: fp32 sums, 2^-22 for each of at most k / 32 + 32 additions on a path, of terms whose
    magnitudes sum to |x| mag^T; one rounding to the output's type."""
    chain = (k / 32 + 32) * 2.0 ** -22
    tiny = 2.0 ** -25 if out_dtype == torch.float16 else 0.0
    return chain * (x.double().cpu().abs() @ mag.t()) + torch.finfo(out_dtype).eps / 2 * y.abs() + tiny + 1e-30
