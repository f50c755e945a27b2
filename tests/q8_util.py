"""Plain forms of the 8-bit operators in 64 bits, on the CPU, and the tolerances that their tests use."""
import math

import torch

E4M3, I8 = torch.float8_e4m3fn, torch.int8
MOST = {E4M3: 448.0, I8: 127.0}
BLOCK = 32


def nearest(t, codes):
    """Values of the codes nearest to t (f64), ties to the even code; NaN stays NaN."""
    if codes is I8:
        return t.round()
    _, e = torch.frexp(t)
    step = torch.pow(2.0, (e - 1).clamp(min=-6).double() - 3)
    return ((t / step).round() * step).clamp(-448.0, 448.0)


def quantize(x, residual=None, norm=False, relu_squared=False, eps=0.0, codes=I8):
    """(h, code values, scale) of rows, f64 but for h, which has x's type."""
    h = x
    if residual is not None:
        h = (x.double() + residual.double()).to(x.dtype)
    d = h.double()
    if relu_squared:                             # (the kernel squares in f32)
        d = torch.where(d <= 0, torch.zeros_like(d), (d * d).float().double())
    top = d.abs().amax(-1)
    fine = torch.isfinite(d).all(-1)
    inv = 1.0 / torch.sqrt((d * d).mean(-1) + eps) if norm else torch.ones_like(top)
    scale = torch.where(top == 0, torch.zeros_like(top), top * inv / MOST[codes])
    q = nearest(d * MOST[codes] / torch.where(top > 0, top, torch.ones_like(top))[..., None], codes)
    return h, torch.where(fine[..., None], q, torch.zeros_like(q)), torch.where(fine, scale, torch.full_like(scale, math.nan))


def scale_tolerance(C):
    """Relative error of a row's scale: the sum of squares is a chain of at most C / 32 + 10 additions, under a root, and six more roundings."""
    return ((C / 32 + 10) / 2 + 6) * 2.0 ** -24


def append(codes, scales, new, start, count):
    """cache_q8_append on code values (f64, [B,H,cap,D]) and f32 scales; new of any float type.  In place."""
    for b in range(codes.shape[0]):
        a, e = int(start[b]), int(start[b]) + int(count[b])
        for i in range(a // BLOCK, -(-e // BLOCK)) if e > a else ():
            lo, hi = max(a, i * BLOCK), min(e, (i + 1) * BLOCK)
            for h in range(codes.shape[1]):
                rows = new[b, h, lo - a:hi - a].double()
                rows = torch.where(torch.isfinite(rows), rows, torch.full_like(rows, math.nan))
                scale = torch.nan_to_num(rows).abs().max().float() * torch.tensor(1 / 448, dtype=torch.float32)
                if i * BLOCK < a:
                    was = scales[b, h, i].clone()
                    if scale > was:
                        codes[b, h, i * BLOCK:lo] = nearest(codes[b, h, i * BLOCK:lo] * was.double() / scale.double(), E4M3)
                    scale = torch.maximum(scale, was)
                codes[b, h, lo:hi] = nearest(rows / (scale.double() if scale > 0 else 1.0), E4M3)
                scales[b, h, i] = scale


def decode(q, k, ks, v, vs, lengths, scale, causal=True):
    """(o, lse) in f64 and how far an f32 computation of each may be off, from code values and scales."""
    q = q.double()
    B, H, Tq, D = q.shape
    G = H // k.shape[1]
    o, lse = torch.zeros_like(q), torch.full((B, H, Tq), -math.inf, dtype=torch.float64)
    err_o, err_l = torch.zeros_like(lse), torch.zeros_like(lse)
    for b in range(B):
        n = int(lengths[b])
        of = torch.arange(n) // BLOCK
        for h in range(H):
            kk = k[b, h // G, :n].double() * ks[b, h // G].double()[of][:, None]
            vv = v[b, h // G, :n].double() * vs[b, h // G].double()[of][:, None]
            for i in range(Tq):
                m = n - (Tq - 1 - i) if causal else n
                if m <= 0:
                    continue
                s = kk[:m] @ q[b, h, i] * scale
                lse[b, h, i] = torch.logsumexp(s, 0)
                o[b, h, i] = torch.softmax(s, 0) @ vv[:m]
                # A score is a sum of D products, off by 2^-23 (a truncated addition) of their sizes each, and takes a few roundings more; a weight
                # is off by twice the scores' error, its own two f16 parts and exp2 (2^-21); sums over the keys, in the order of a warp's walk,
                # by 2^-23 for every addition.
                # (a NaN among the operands is no size: what it reaches is NaN on both sides)
                ds = (D + 16) * 2.0 ** -23 * float((torch.nan_to_num(kk[:m]).abs() @ torch.nan_to_num(q[b, h, i]).abs()).max()) * abs(scale)
                sums = (m / 8 + 64) * 2.0 ** -23
                err_o[b, h, i] = float(torch.nan_to_num(vv[:m]).abs().max()) * (2 * ds + 2.0 ** -21 + sums)
                err_l[b, h, i] = ds + sums + 2.0 ** -22 * abs(float(torch.nan_to_num(lse[b, h, i])))
    return o, lse, err_o, err_l


def half_step(t, dtype):
    """Half a step of dtype at the values t."""
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).tiny
    return t.abs() * (eps / 2) + tiny * eps / 2
