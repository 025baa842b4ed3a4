"""The paged 8-bit KV cache operators in 64 bits, for the tests: written from the
definitions in include/yk.h, one token and one head at a time."""
import math

import torch

PAGE, BIAS, EMIN, EMAX = 16, 127, -60, 60


def decode(codes: torch.Tensor, byte: torch.Tensor) -> torch.Tensor:
    """codes [..., 16, dh] uint8, byte [...]: the values the cells stand for, float64."""
    e = byte.to(torch.float64).sub(BIAS).clamp(EMIN, EMAX)
    return codes.view(torch.float8_e4m3fn).to(torch.float64) * (2.0 ** e)[..., None, None]


def encode(x: torch.Tensor, e: int) -> torch.Tensor:
    """float64 values to codes at exponent e: nearest even, saturating."""
    return (x * 2.0 ** -e).clamp(-448, 448).to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)


def cover(amax: float) -> int:
    if amax == 0:
        return EMIN
    e = math.ceil(math.log2(amax / 448.0))
    while amax > 448.0 * 2.0 ** e:
        e += 1
    while amax <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return max(EMIN, min(EMAX, e))


def normed(x, gain, eps):
    if gain is None:
        return x
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + eps) * gain.to(torch.float64)


def rotated(x, rope):
    """x [T, heads, dh], rope [T, dh / 2, 2]."""
    if rope is None:
        return x
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = rope[:, None, :, 0].to(torch.float64), rope[:, None, :, 1].to(torch.float64)
    y = torch.empty_like(x)
    y[..., 0::2] = a * c - b * s
    y[..., 1::2] = a * s + b * c
    return y


def attention(q, pool, scales, layer, starts, ctx, tables, window=0, scale=0.0, cap=0.0):
    """(out, weight, spread, floor) in float64: weight = sum_j softmax_j |V_j| per element, spread =
    the largest sum_d |q_d K_jd| * scale of a row, floor = the largest softmax_j * (scale of j's V
    block) of a row times sum_j |code of V_j|, for error bounds.  Rows outside the batch are NaN
    in out."""
    T, H, dh = q.shape
    G = pool.shape[3]
    sc = scale or dh ** -0.5
    out = torch.full((T, H, dh), math.nan, dtype=torch.float64)
    weight, spread, floor = torch.zeros_like(out), torch.zeros(T, H, dtype=torch.float64), torch.zeros_like(out)
    q = q.cpu().to(torch.float64)
    for b in range(len(ctx)):
        n = starts[b + 1] - starts[b]
        pages = (ctx[b] + PAGE - 1) // PAGE
        ids = [int(i) for i in tables[b][:pages]]
        if ids:
            kv = decode(pool[ids, layer].cpu(), scales[ids, layer].cpu())  # [pages, 2, G, 16, dh]
            kv = kv.permute(1, 2, 0, 3, 4).reshape(2, G, -1, dh)
            unit = 2.0 ** scales[ids, layer, 1].cpu().double().sub(BIAS).clamp(EMIN, EMAX)  # [pages, G]
            unit = unit.T.repeat_interleave(PAGE, 1)
        for i in range(n):
            t, p = starts[b] + i, ctx[b] - n + i
            lo = max(0, p - window + 1) if window > 0 else 0
            for h in range(H):
                if p < 0:
                    out[t, h] = 0.0
                    continue
                K, V = kv[0, h * G // H, lo:p + 1], kv[1, h * G // H, lo:p + 1]
                x = (K @ q[t, h]) * sc
                spread[t, h] = (K.abs() @ q[t, h].abs()).max() * sc
                if cap > 0:
                    x = cap * torch.tanh(x / cap)
                w = torch.softmax(x, 0)
                out[t, h] = w @ V
                weight[t, h] = w @ V.abs()
                u = unit[h * G // H, lo:p + 1]
                floor[t, h] = (w * u).max() * (V.abs() / u[:, None]).sum(0)
    return out, weight, spread, floor


def attention_bound(out, weight, spread, floor, dh, dtype):
    """How far a result may be from attention()'s, element by element.

    Scores: an fp32 dot product of dh products, scaled, in the log2 domain: relative error of the
    sum of magnitudes at most (dh + 8) * 2^-23 (2^-23 rather than 2^-24 a step: the matrix
    instruction may truncate), so a weight is off by a factor exp(+-d), d = spread * (dh + 8) * 2^-23,
    numerator and denominator each.  Weights: rounded to 11 bits (bf16 results) or to 22 (fp32), half
    a step each, 2^-11 and 2^-22; exp2 and the sums: 2^-20 together.  The result: half a step of its type.
    f16 ends at 2^-24: a weight times its V block's scale is held as f16 with the row's largest at 2^3 or
    above (fp32 queries: 2^7), so it is also off by half of 2^-24, 2^-28 (2^-32) of that largest; that error
    meets |code of V_j|, which gives floor * 2^-28 (2^-32) over all keys (it counts where a dimension's V is
    zero for every key of weight)."""
    d = spread[..., None] * (dh + 8) * 2.0 ** -23
    w = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22
    half = torch.finfo(dtype).eps / 2
    return out.abs() * half + weight * (1 + half) * (2 * torch.expm1(d) + w + 2.0 ** -20) + floor * (2.0 ** -28 if dtype == torch.bfloat16 else 2.0 ** -32) + 1e-30
