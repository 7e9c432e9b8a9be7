"""64-bit restatements of the operators behind the collectives, in numpy, with the
bounds their 32-bit kernels are held to.  u(t) is half a rounding step of a type
relative to the value; E = 2^-24 is fp32's."""
import numpy as np

from flagcx_amd import _native as N
from flagcx_amd import kernels as K

E = 2.0 ** -24
U = {N.DT_BF16: 2.0 ** -8, N.DT_FP16: 2.0 ** -11, N.DT_FP32: 2.0 ** -24}
SMALLEST = {N.DT_BF16: 2.0 ** -133, N.DT_FP16: 2.0 ** -24, N.DT_FP32: 2.0 ** -149}     # subnormal step


def codes_to_f64(a, dtype):
    if dtype == N.DT_E4M3:
        return E4M3[a]
    if dtype == N.DT_BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if dtype == N.DT_FP16:
        return a.view(np.float16).astype(np.float64)
    return a.astype(np.float64)


def _e4m3_table():
    c = np.arange(256)
    s, e, m = c >> 7, (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9.0)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(s == 1, -v, v)


E4M3 = _e4m3_table()


def to_e4m3(x):
    """Nearest codes of |x| <= 448 (ties to even codes)."""
    pos = E4M3[:127]
    mid = (pos[1:] + pos[:-1]) / 2
    a = np.abs(x)
    lo = np.searchsorted(mid, a, side="left")                # a == mid[i] -> i, the lower code
    tie = (lo < 126) & (a == mid[np.minimum(lo, 125)]) & (lo % 2 == 1)
    return (lo + tie + 128 * (np.signbit(x))).astype(np.uint8)


def normal(dtype, shape, seed, std=1.0):
    n = int(np.prod(shape))
    return K.synth(max(n, 1), dtype, K.SYNTH_NORMAL, 0.0, std, seed)[:n].reshape(shape)


def rounding(y, dtype):
    return U[dtype] * np.abs(y) + SMALLEST[dtype]


# ---------------------------------------------------------------- norm

def norm(ins, residual, weight, eps):
    """s, y, sum of magnitudes, 1/rms; all in 64 bits."""
    s, mag = np.zeros_like(ins[0]), np.zeros_like(ins[0])
    for x in list(ins) + ([residual] if residual is not None else []):
        s, mag = s + x, mag + np.abs(x)
    r = 1 / np.sqrt(np.mean(s * s, axis=1, keepdims=True) + eps)
    return s, s * r * (1.0 if weight is None else weight), mag, r


def norm_bounds(s, y, mag, r, weight, terms):
    """|error| of total and y before their rounding.  s: `terms` - 1 additions, each off by E of a partial sum <= mag.
    r: the squares' sum adds C / threads + 16 nonnegative terms per step (at most 64 roundings for the widths tested
    here), ds moves it by at most |ds| / |s| in the 2-norm; sqrt, division, mean and eps add four more.  y: two products."""
    ds = terms * E * mag
    norm_s = np.sqrt(np.sum(s * s, axis=1, keepdims=True))
    dr = 70 * E + np.sqrt(np.sum(ds * ds, axis=1, keepdims=True)) / np.maximum(norm_s, 1e-300)
    w = 1.0 if weight is None else np.abs(weight)
    return ds, ds * r * w + np.abs(y) * (dr + 4 * E)


def norm_grad(dy, x, weight, dtotal, eps):
    w = 1.0 if weight is None else weight
    r = 1 / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + eps)
    g = dy * w
    m = np.mean(g * x, axis=1, keepdims=True)
    dx = r * g - x * r ** 3 * m + (0 if dtotal is None else dtotal)
    dw = np.sum(dy * x * r, axis=0)
    # bounds: r is off by 70 E (above); m by 70 E of the mean magnitude; a handful of roundings per product
    dm = 70 * E * np.mean(np.abs(g * x), axis=1, keepdims=True)
    bx = (r * np.abs(g) + np.abs(x) * r ** 3 * np.abs(m)) * 220 * E + np.abs(x) * r ** 3 * dm + 4 * E * np.abs(dx)
    if dtotal is not None:
        bx = bx + 4 * E * np.abs(dtotal)
    # dweight: each term is off by 80 E; rows / 256 + 1 additions in a workgroup (long rows: / 64), 3 over its wavefronts,
    # 8 + 32 where the workgroups' sums are joined: under 120 at the sizes tested here
    bw = 200 * E * np.sum(np.abs(dy * x * r), axis=0)
    return dx, dw, bx, bw


# ------------------------------------------------------------- products

def clamp_offsets(offsets, rows):
    o = np.clip(np.asarray(offsets, np.int64), 0, rows)
    return [(int(a), int(max(a, b))) for a, b in zip(o, o[1:])]


def product(x, w, offsets, nk):
    """y and the bound's sum of magnitudes; rows outside every expert are NaN in y."""
    n = w.shape[1] if nk else w.shape[2]
    y, mag = np.full((x.shape[0], n), np.nan), np.zeros((x.shape[0], n))
    for e, (a, b) in enumerate(clamp_offsets(offsets, x.shape[0])):
        we = w[e].T if nk else w[e]
        y[a:b], mag[a:b] = x[a:b] @ we, np.abs(x[a:b]) @ np.abs(we)
    return y, mag


def product_dw(dy, x, offsets):
    segs = clamp_offsets(offsets, x.shape[0])
    dw = np.zeros((len(segs), dy.shape[1], x.shape[1]))
    mag = np.zeros_like(dw)
    for e, (a, b) in enumerate(segs):
        dw[e], mag[e] = dy[a:b].T @ x[a:b], np.abs(dy[a:b]).T @ np.abs(x[a:b])
    return dw, mag


def sum_bound(terms, mag):
    """A chain of `terms` fp32 additions in any order; the matrix cores may truncate where a sum would round."""
    return (terms + 8) * 2 * E * mag


def within(got, want, t, bound):
    """got is want, off by `bound` at most, rounded to type t.  fp16 ends at 65504: what rounds to 65520 or more is an
    infinity of want's sign."""
    fine = np.abs(got - want) <= rounding(want, t) * 1.01 + bound
    if t == N.DT_FP16:
        fine |= (np.abs(want) + bound >= 65520) & (got == np.copysign(np.inf, want))
    return bool(fine.all())
