"""Plain 64-bit implementations of the prompt-side operators and the 8-bit cache, and the bounds their kernels keep."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}  # half the smallest number


def rotate(x, positions, inv, factor, r, layout):
    """x [B, H, T, D], positions [B, T], inv [r/2] radians per position; 64 bits."""
    ang = positions.double()[:, None, :, None] * inv
    c, s = torch.cos(ang) * factor, torch.sin(ang) * factor
    y = x.double().clone()
    if layout == "half":
        a, b = x[..., : r // 2].double(), x[..., r // 2: r].double()
        y[..., : r // 2], y[..., r // 2: r] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:r:2].double(), x[..., 1:r:2].double()
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    return y


def rotate_bound(x, y, factor, r, layout, positions, inv):
    """Half a step of the output plus the 32-bit work: sine and cosine (times the factor) to half a step, 2^-25 of the
    factor and a little; a product rounded to half a step and the sum of the two: in all at most 1.6 * 2^-24, within
    2^-23 of |x1| + |x2|, times the factor.  The angles themselves are 64-bit products: the formula's is rounded once
    (2^-53 of its size), the kernel's three times (the pair's turns, their table entry, the product): together within
    2^-51 of position * frequency, which counts from position 2^20 on."""
    pair = x.double().abs().clone()
    far = 2.0 ** -51 * positions.double().abs()[:, None, :, None] * inv
    if layout == "half":
        s = (pair[..., : r // 2] + pair[..., r // 2: r]) * (2.0 ** -23 + far)
        pair[..., : r // 2], pair[..., r // 2: r] = s, s
    else:
        s = (pair[..., 0:r:2] + pair[..., 1:r:2]) * (2.0 ** -23 + far)
        pair[..., 0:r:2], pair[..., 1:r:2] = s, s
    pair[..., r:] = 0.0
    return HALF[x.dtype] * y.abs() + factor * pair + TINY[x.dtype]


def attend(q, k, v, scaling, limits):
    """q [n, D], k / v [m, D] in 64 bits; row i sees keys 0 .. limits[i] - 1 and nothing of the others.  Returns the
    result and sum p |v| / sum p; rows that see nothing are zero."""
    n, m = q.shape[0], k.shape[0]
    seen = torch.arange(m, device=q.device)[None, :] < limits[:, None]
    out = torch.zeros(n, q.shape[1], dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    for i in range(n):
        w = int(limits[i])
        if w > 0:
            s = (k[:w] @ q[i]) * scaling
            p = torch.softmax(s, 0)
            out[i] = p @ v[:w]
            mag[i] = p @ v[:w].abs()
    del seen
    return out, mag


def attend_fast(q, k, v, scaling, limits):
    """As attend, for finite inputs, all rows at once."""
    m = k.shape[0]
    if m == 0:
        z = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        return z, z.clone()
    seen = torch.arange(m, device=q.device)[None, :] < limits[:, None]
    s = (q @ k.T) * scaling
    s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    p = torch.where(limits[:, None] > 0, p, torch.zeros_like(p))
    return p @ v, p @ v.abs()


def logit_error(q, k, scaling):
    """Largest error of a logit (natural units): 128 products summed in 32 bits, truncated at worst (2^-23 each), plus the
    scale's and the exponential's own steps (2^-22 of the logit's size)."""
    if k.shape[0] == 0:
        return 0.0
    size = (q.abs() @ k.abs().T).max().item() * abs(scaling)
    return (128 * 2.0 ** -23 + 2.0 ** -21) * size + 2.0 ** -21


def attention_bound(out, mag, dtype, weight_half, delta):
    """Half a step of the output, half a step of each weight, and what a logit's error does to weights and sum."""
    return HALF[dtype] * out.abs() + (weight_half + 2.0 * delta + 2.0 ** -18) * mag + TINY[dtype] + 1e-7 * mag


def hold(x):
    """Whole blocks [..., n, 128] (n a multiple of 32) as the 8-bit cache holds them: codes and scales."""
    *lead, n, d = x.shape
    y = x.double().reshape(*lead, n // 32, 32, d)
    top = y.abs().amax(dim=(-2, -1))
    t = y * 127.0 / torch.where(top > 0, top, torch.ones_like(top))[..., None, None]
    codes = torch.sign(t) * torch.floor(t.abs() + 0.5)
    scale = torch.where(top > 0, top.float() / 127.0, torch.ones_like(top).float())
    return codes, scale


def held_values(x, dtype):
    codes, scale = hold(x)
    return (codes.float() * scale[..., None, None]).reshape(x.shape).to(dtype)


def read_records(layer, lengths):
    """Decode the cache's whole blocks from the documented record layout: per row (k codes, k scales, v codes, v scales)
    with codes [H, n, 128] as float64."""
    out = []
    pages, table = layer.pages.cpu(), layer.page_table.cpu()
    piece = torch.arange(256)
    i, hf, g, t = piece >> 6, (piece >> 5) & 1, (piece >> 2) & 7, piece & 3
    k_tok, k_ch = 8 * (g // 2) + 2 * i + g % 2, 64 * hf + 16 * t
    v_tok, v_ch = 8 * t, 16 * (piece >> 5) + g
    for b, n in enumerate(lengths):
        H, nb = layer.H_KV, n // 32
        kc, vc = torch.zeros(H, nb, 32, 128, dtype=torch.float64), torch.zeros(H, nb, 32, 128, dtype=torch.float64)
        ks, vs = torch.zeros(H, nb), torch.zeros(H, nb)
        for j in range(nb):
            rec = pages[table[b, j // 4], :, j % 4]                              # [H, 8208]
            code = rec[:, :8192].view(torch.int8).to(torch.float64)
            kp, vp = code[:, :4096].reshape(H, 256, 16), code[:, 4096:].reshape(H, 256, 16)
            for e in range(16):
                kc[:, j, k_tok, k_ch + e] = kp[:, :, e]
                vc[:, j, v_tok + e % 8, v_ch + 8 * (e // 8)] = vp[:, :, e]
            sc = rec[:, 8192:8200].contiguous().view(torch.float32)
            ks[:, j], vs[:, j] = sc[:, 0], sc[:, 1]
        out.append((kc.reshape(H, nb * 32, 128), ks, vc.reshape(H, nb * 32, 128), vs))
    return out
