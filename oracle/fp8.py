"""8-bit floating point (e4m3) with block scales, in float64: the activation quantiser, the block-scaled product and the
routed experts on such tables, with a bound on how far an fp32 evaluation of each may be off."""
import ml_dtypes
import numpy as np

E4M3 = ml_dtypes.float8_e4m3fn
GROUP = 128
LEAST = 448.0 * 2.0 ** -100


def group_scales(x):
    """x [N, K] -> [N, ceil(K / 128)]: the least power of two s >= 2^-100 with max|x| <= 448 s; NaN beside inf / NaN."""
    N, K = x.shape
    out = np.empty((N, -(-K // GROUP)))
    for b in range(out.shape[1]):
        top = np.abs(x[:, GROUP * b:GROUP * (b + 1)]).max(axis=1)
        bad = ~np.isfinite(top)
        t = np.maximum(np.where(bad, 1.0, top), LEAST)
        m, e = np.frexp(t / 448.0)                       # t / 448 = m 2^e, m in [0.5, 1)
        s = np.ldexp(1.0, np.where(m == 0.5, e - 1, e))
        s = np.where(448.0 * s / 2 >= t, s / 2, s)       # t / 448 is rounded: settle the border exactly
        out[:, b] = np.where(bad, np.nan, np.where(448.0 * s < t, s * 2, s))
    return out


def spread(s, K):
    return np.repeat(s, GROUP, axis=-1)[..., :K]


def codes(x, s):
    """e4m3(x / s) as float64 values."""
    with np.errstate(invalid="ignore"):
        return (x / spread(s, x.shape[1])).astype(np.float32).astype(E4M3).astype(np.float64)


def quantized(x):
    """The values that x stands for after quantisation."""
    s = group_scales(x)
    return codes(x, s) * spread(s, x.shape[1])


def weights(q, s):
    """Codes [rows, K] (any float type) and block scales -> float64 [rows, K]."""
    q, s = np.asarray(q, np.float64), np.asarray(s, np.float64)
    return q * spread(np.repeat(s, GROUP, axis=0)[:q.shape[0]], q.shape[1])


def sum_bound(K):
    """Relative bound on an fp32 sum of K block-scaled products, against the sum of their magnitudes. A block's 128
    products are exact; its 128 additions are off by at most 2^-23 each (truncated to 24 bits), the product of the two
    scales and the multiply-add into the running sum by 2^-24 each, once per block; partial sums of up to 64 ranges of
    blocks are joined by as many additions."""
    kb = -(-K // GROUP)
    return 128 * 2.0 ** -23 + (3 * kb + 64) * 2.0 ** -24


def linear(q, s, x, half_eps):
    """(y, bound): y = quantized(x) W^T and how far an output rounded at half_eps (eps / 2 of its type) may be off."""
    xv, w = quantized(x), weights(q, s)
    y = xv @ w.T
    off = sum_bound(x.shape[1]) * (np.abs(xv) @ np.abs(w).T)
    return y, off + half_eps * (np.abs(y) + off)


def swiglu(g, u, limit):
    g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    return g / (1 + np.exp(-g)) * u


def experts(gate, up, down, x, idx, w, limit, half_eps):
    """(y, bound) of the routed experts: tables as [(codes, scales)] per expert. The bound follows the sums' errors through
    SwiGLU to the codes of h: a value within its error of a rounding border may fall on either side."""
    N, k = idx.shape
    H = x.shape[1]
    y, bound = np.zeros((N, H)), np.zeros((N, H))
    xv = quantized(x)
    mag = np.zeros((N, H))
    for e in np.unique(idx[idx >= 0]):
        t, j = np.nonzero(idx == e)
        wg, wu, wd = weights(*gate[e]), weights(*up[e]), weights(*down[e])
        a, b = xv[t] @ wg.T, xv[t] @ wu.T
        ea, eb = (sum_bound(H) * (np.abs(xv[t]) @ np.abs(m).T) for m in (wg, wu))
        h = swiglu(a, b, limit)
        # |d silu| <= 1.1, |silu| <= |a|; expf, the division and the products: 8 steps of 2^-23
        eh = 1.1 * ea * (np.minimum(np.abs(b), limit) + eb) + (np.abs(np.minimum(a, limit)) + ea) * eb + 2.0 ** -20 * np.abs(h)
        lo, hi = np.abs(h) - eh, np.abs(h) + eh
        s = group_scales(h)
        hq = codes(h, s) * spread(s, h.shape[1])
        step = np.zeros_like(h)
        for sc in (s, group_scales(hi), group_scales(np.maximum(lo, 0))):
            for v in (np.maximum(lo, 0), hi):
                v = np.minimum(v, 448.0 * spread(sc, h.shape[1]))
                step = np.maximum(step, np.abs(codes(v, sc) * spread(sc, h.shape[1]) - np.abs(hq)))
        o = hq @ wd.T
        eo = step @ np.abs(wd).T + sum_bound(h.shape[1]) * ((np.abs(hq) + step) @ np.abs(wd).T)
        np.add.at(y, t, w[t, j][:, None] * o)
        np.add.at(bound, t, np.abs(w[t, j])[:, None] * eo)
        np.add.at(mag, t, np.abs(w[t, j])[:, None] * np.abs(o))
    bound += k * 2.0 ** -23 * mag
    return y, bound + half_eps * (np.abs(y) + bound)
