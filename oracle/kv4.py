"""64-bit numpy form of the 4-bit KV cache and of the attention over it (tests only).

The cache is [kv head][block of 32 positions]; a block is K codes | K parameters | V codes | V parameters."""
import numpy as np


def quantise(x):
    """x [..., head_dim] f32 -> (codes uint8 [..., ng, 32], m [..., ng], d [..., ng]) with m, d f64 on the f16 grid."""
    g = np.asarray(x, np.float64).reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)

    def spacing(a):
        return np.ldexp(1.0, np.maximum(np.frexp(a)[1] - 11, -24))
    lo = np.maximum(g.min(-1), -65504.0)
    m = np.minimum(np.floor(lo / spacing(lo)) * spacing(lo), 65504.0) + 0.0
    d = np.maximum(g.max(-1) - m, 0.0) / 15
    d = np.minimum(np.ceil(d / spacing(d)) * spacing(d), 65504.0)
    code = np.clip(np.rint((g - m[..., None]) / np.where(d > 0, d, 1.0)[..., None]), 0, 15)
    code = np.where((d > 0)[..., None], code, 0)
    return code.astype(np.uint8), np.where(bad, np.nan, m), np.where(bad, 0.0, d)


def values(x):
    """What rows x stand for once they are in the cache (f32, one rounding)."""
    c, m, d = quantise(x)
    return (m[..., None] + d[..., None] * c).astype(np.float32).reshape(x.shape)


def nbytes(max_seq, n_kv, hd):
    return n_kv * ((max_seq + 31) // 32) * 40 * hd


def store(cache, k, v, pos0, max_seq):
    """Write rows k, v [n, n_kv, hd] into the bytes of a cache, one position at a time, by address."""
    n, n_kv, hd = k.shape
    ng, nb = hd // 32, (max_seq + 31) // 32
    for values_side, x in ((False, k), (True, v)):
        c, m, d = quantise(x)
        par = np.concatenate((m, d), -1).astype(np.float16)
        if np.isnan(m).any():
            par.view(np.uint16)[np.isnan(par)] = 0x7FFF
        for t in range(n):
            pos = pos0 + t
            for h in range(n_kv):
                blk = (h * nb + pos // 32) * 40 * hd + (20 * hd if values_side else 0)
                row = blk + (pos % 32) * (hd // 2)
                if values_side:   # 16-bit word r * ng + g: dims 32 g + 4 r + i
                    nib = c[t, h].reshape(ng, 8, 4).transpose(1, 0, 2).reshape(-1)
                else:             # 32-bit word t * ng + g: dims 32 g + 8 t + i
                    nib = c[t, h].reshape(ng, 4, 8).transpose(1, 0, 2).reshape(-1)
                cache[row:row + hd // 2] = nib[0::2] | (nib[1::2] << 4)
                at = blk + 16 * hd + (pos % 32) * 4 * ng
                cache[at:at + 4 * ng] = par[t, h].view(np.uint8)
    return cache


def attention(q, k, v, pos0, window, scale, sinks):
    """q [n, n_heads, hd] at positions pos0 .., k / v [S, n_kv, hd] (the cache's values): (out f64, bound f64).

    The bound is that of an f32 evaluation: a score of hd products has an error of at most (hd + 16) 2^-23 of
    sum |q_i k_i| scale (products, sums, and 2^-22 for an operand split into two 11-bit parts), a weight exp(s) twice
    the largest of these plus 2^-21 relative (argument times log2 e, exponential), a sum of n terms n 2^-24, and the
    weights and values enter numerator and denominator: |error| <= sum p |v| * (2 e_s * 2 + (n + 32) 2^-22)."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, nh, hd = q.shape
    G = nh // k.shape[1]
    out, bound = np.zeros((n, nh, hd)), np.zeros((n, nh, hd))
    for t in range(n):
        p = pos0 + t
        lo = max(0, p + 1 - window) if window > 0 else 0
        for h in range(nh):
            kk, vv = k[lo:p + 1, h // G], v[lo:p + 1, h // G]
            s = kk @ q[t, h] * scale
            e_s = (np.abs(kk) @ np.abs(q[t, h])).max() * scale * (hd + 16) * 2.0 ** -23
            top = max(s.max(), float(sinks[h])) if sinks is not None else s.max()
            e = np.exp(s - top)
            den = e.sum() + (np.exp(float(sinks[h]) - top) if sinks is not None else 0.0)
            out[t, h] = e @ vv / den
            bound[t, h] = (e @ np.abs(vv)) / den * (4 * e_s + (p + 1 - lo + 32) * 2.0 ** -22) + 1e-30
    return out, bound
