"""Products grouped by expert against the 64-bit restatement."""
import ctypes as C

import numpy as np
import pytest

from flagcx_amd import _native as N
from flagcx_amd import kernels as K
from tests import model_ref as R
from tests.util import DevBufs

pytestmark = pytest.mark.gpu

NAN16 = {N.DT_BF16: 0x7fc0, N.DT_FP16: 0x7e00}


def ragged(rows, experts, rng, empty=0.2):
    """Ascending offsets with empty experts, a gap in front and one behind."""
    inner = np.sort(rng.integers(0, rows + 1, experts + 1))
    for e in range(1, experts + 1):
        if rng.random() < empty:
            inner[e] = inner[e - 1]
    return inner.astype(np.int32)


def with_ld(a, ld, fill):
    out = np.full(a.shape[:-1] + (ld,), fill, a.dtype)
    out[..., :a.shape[-1]] = a
    return out


def run(dev, dtype, rows, n, k, offsets, *, nk=True, out32=False, pad=0, shift=0, seed=0, stream=None):
    experts = 1 if offsets is None else len(offsets) - 1
    x, w = R.normal(dtype, (rows, k), seed), R.normal(dtype, (experts, n, k) if nk else (experts, k, n), seed + 1)
    segs = offsets if offsets is not None else [0, rows]
    inside = np.zeros(rows, bool)
    for a, b in R.clamp_offsets(segs, rows):
        inside[a:b] = True
    x[~inside] = NAN16[dtype]                                # rows of nobody must not reach any result
    odt = np.float32 if out32 else np.uint16
    ldx, ldw, ldy = k + pad, w.shape[2] + pad, n + pad
    st = dict(x=ldx, w=ldw, y=ldy, expert_w=w.shape[1] * ldw + pad) if pad else None
    wbuf = with_ld(w, ldw, NAN16[dtype]).reshape(experts, -1)
    if pad:
        wbuf = np.concatenate([wbuf, np.full((experts, pad), NAN16[dtype], np.uint16)], axis=1)
    fill = odt(9)
    with DevBufs(dev) as b:
        dx = b.put(with_ld(x, ldx, NAN16[dtype]), pad_before=2 * shift)
        dw = b.put(wbuf, pad_before=2 * shift)
        do = b.put(np.ascontiguousarray(offsets)) if offsets is not None else None
        dy = b.put(np.full((rows, ldy), fill, odt), pad_before=shift * odt().itemsize)
        N.check(K.expert_product(dy, dx, dw, do, experts, rows, n, k, dtype, out_dtype=N.DT_FP32 if out32 else None,
                                 layout=K.W_NK if nk else K.W_KN, strides=st, stream=stream), "fx_expert_product")
        dev.sync()
        y = dev.to_host(dy, rows * ldy, odt).reshape(rows, ldy)
    assert (y[:, n:] == fill).all() and (y[~inside] == fill).all(), "rows and columns of nobody stay as they were"
    want, mag = R.product(R.codes_to_f64(x, dtype), R.codes_to_f64(w, dtype), segs, nk)
    t = N.DT_FP32 if out32 else dtype
    got = R.codes_to_f64(y[inside, :n], t)
    want, mag = want[inside], mag[inside]
    assert (np.abs(got - want) <= R.rounding(want, t) * 1.01 + R.sum_bound(k, mag)).all()
    return y


@pytest.mark.parametrize("name,dtype", [("bf16", N.DT_BF16), ("fp16", N.DT_FP16)])
@pytest.mark.parametrize("nk", [True, False])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 17, 5), (16, 64, 64), (17, 128, 72), (65, 100, 200), (130, 257, 136), (300, 520, 1000)])
def test_plain_products(dev, name, dtype, nk, rows, n, k):
    print(name, nk, rows, n, k, flush=True)
    run(dev, dtype, rows, n, k, None, nk=nk, seed=rows)
    run(dev, dtype, rows, n, k, None, nk=nk, out32=True, seed=rows)


@pytest.mark.parametrize("nk", [True, False])
@pytest.mark.parametrize("rows,experts,n,k", [(5, 3, 64, 64), (40, 8, 128, 256), (200, 5, 264, 328), (700, 13, 200, 96), (500, 70, 64, 128),
                                              (90, 200, 32, 64), (1100, 3, 300, 520)])
def test_ragged_products(dev, nk, rows, experts, n, k):
    rng = np.random.default_rng(rows)
    for dtype in (N.DT_BF16, N.DT_FP16):
        o = ragged(rows, experts, rng)
        print(nk, rows, experts, n, k, o.tolist()[:20], flush=True)
        run(dev, dtype, rows, n, k, o, nk=nk, out32=dtype == N.DT_FP16, seed=rows)


@pytest.mark.parametrize("nk", [True, False])
@pytest.mark.parametrize("rows,experts,n,k", [(40, 1, 520, 1096), (100, 1, 2056, 264), (250, 1, 3080, 136), (600, 1, 1032, 72),
                                              (1000, 20, 1288, 264), (1900, 32, 2056, 136), (4000, 30, 1032, 72)])
def test_sizes_between_few_rows_and_full_tiles(dev, nk, rows, experts, n, k):
    """Where the tile's shape depends on how many tiles there are."""
    rng = np.random.default_rng(n)
    for t in (N.DT_BF16, N.DT_FP16):
        for out32 in (False, True):
            run(dev, t, rows, n, k, None if experts == 1 else ragged(rows, experts, rng), nk=nk, out32=out32, seed=k)


@pytest.mark.parametrize("nk", [True, False])
def test_strides_and_alignment(dev, nk):
    rng = np.random.default_rng(3)
    for pad, shift in ((1, 0), (8, 0), (0, 1), (3, 1), (8, 4)):
        for rows, n, k in ((50, 72, 136), (260, 136, 264), (33, 129, 65)):
            print(nk, pad, shift, rows, n, k, flush=True)
            run(dev, N.DT_BF16, rows, n, k, ragged(rows, 4, rng), nk=nk, pad=pad, shift=shift, seed=pad)


@pytest.mark.parametrize("nk", [True, False])
def test_large_products(dev, nk):
    """Sizes that fill the chip: aligned operands (with an odd tail of the reduction, ragged rows and a partial last
    column tile) and unaligned ones."""
    rng = np.random.default_rng(8)
    for rows, experts, n, k, pad in ((3200, 1, 4160, 200, 0), (3300, 7, 4168, 136, 8), (3100, 40, 4104, 64, 0), (3300, 7, 4168, 136, 1)):
        o = None if experts == 1 else ragged(rows, experts, rng)
        print(nk, rows, experts, n, k, pad, flush=True)
        run(dev, N.DT_BF16, rows, n, k, o, nk=nk, pad=pad, seed=k, out32=pad == 8)


def test_no_reduction_gives_zeros(dev):
    with DevBufs(dev) as b:
        y = b.put(np.full((5, 7), 3, np.uint16))
        o = b.put(np.array([0, 2, 4], np.int32))
        N.check(K.expert_product(y, None, None, o, 2, 5, 7, 0, N.DT_BF16))
        dev.sync()
        got = dev.to_host(y, 35, np.uint16).reshape(5, 7)
    assert not got[:4].any() and (got[4] == 3).all()


@pytest.mark.parametrize("offsets", [[-5, 3, 9, 400], [0, 30, 10, 40], [50, 40, 30, 20], [400, 400, 400, 400], [-9, -8, -7, -6]])
def test_bad_offsets_touch_nothing_outside(dev, offsets):
    """Clamped to the rows; a descending pair is an empty expert.  Rows claimed twice get either answer, so only the
    guards around y and the finiteness of what lies inside are checked."""
    rows, n, k = 40, 72, 64
    x, w = R.normal(N.DT_BF16, (rows, k), 1), R.normal(N.DT_BF16, (3, n, k), 2)
    guard = np.full((64, n), 9, np.uint16)
    with DevBufs(dev) as b:
        dx, dw, do = b.put(x), b.put(w), b.put(np.array(offsets, np.int32))
        base = b.put(np.concatenate([guard, np.full((rows, n), 9, np.uint16), guard]))
        dy, ddw = base + guard.nbytes, b.alloc(3 * n * k * 4)
        N.check(K.expert_product(dy, dx, dw, do, 3, rows, n, k, N.DT_BF16))
        N.check(K.expert_product_dw(ddw, dy, dx, do, 3, rows, n, k, N.DT_BF16, out_dtype=N.DT_FP32))
        dev.sync()
        y = dev.to_host(base, (rows + 128) * n, np.uint16).reshape(-1, n)
        dwv = dev.to_host(ddw, 3 * n * k, np.float32)
    assert (y[:64] == 9).all() and (y[-64:] == 9).all() and np.isfinite(dwv).all()


def run_dw(dev, dtype, rows, n, k, offsets, *, out32=False, pad=0, shift=0, seed=0):
    experts = 1 if offsets is None else len(offsets) - 1
    dy, x = R.normal(dtype, (rows, n), seed), R.normal(dtype, (rows, k), seed + 1)
    segs = offsets if offsets is not None else [0, rows]
    inside = np.zeros(rows, bool)
    for a, b in R.clamp_offsets(segs, rows):
        inside[a:b] = True
    dy[~inside] = NAN16[dtype]
    x[~inside] = NAN16[dtype]
    odt, t = (np.float32, N.DT_FP32) if out32 else (np.uint16, dtype)
    fill = odt(9)
    st = dict(dy=n + pad, x=k + pad, dw=k + pad, expert_dw=n * (k + pad) + pad) if pad else None
    with DevBufs(dev) as b:
        ddy = b.put(with_ld(dy, n + pad, NAN16[dtype]), pad_before=2 * shift)
        dx = b.put(with_ld(x, k + pad, NAN16[dtype]), pad_before=2 * shift)
        do = b.put(np.ascontiguousarray(offsets)) if offsets is not None else None
        per = n * (k + pad) + pad
        ddw = b.put(np.full(experts * per + 64, fill, odt), pad_before=shift * odt().itemsize)
        N.check(K.expert_product_dw(ddw, ddy, dx, do, experts, rows, n, k, dtype, out_dtype=t, strides=st), "fx_expert_product_dw")
        dev.sync()
        dw = dev.to_host(ddw, experts * per + 64, odt)
    assert (dw[experts * per:] == fill).all()
    dw = dw[:experts * per].reshape(experts, per)
    assert (dw[:, n * (k + pad):] == fill).all()
    dw = dw[:, :n * (k + pad)].reshape(experts, n, k + pad)
    assert (dw[:, :, k:] == fill).all()
    want, mag = R.product_dw(R.codes_to_f64(dy, dtype), R.codes_to_f64(x, dtype), segs)
    assert (np.abs(R.codes_to_f64(dw[:, :, :k], t) - want) <= R.rounding(want, t) * 1.01 + R.sum_bound(rows, mag)).all()


@pytest.mark.parametrize("rows,experts,n,k", [(1, 1, 1, 1), (9, 2, 17, 5), (64, 1, 64, 64), (200, 5, 136, 264), (700, 13, 200, 96),
                                              (90, 70, 32, 64), (1100, 3, 300, 520)])
def test_weight_gradients(dev, rows, experts, n, k):
    rng = np.random.default_rng(rows)
    for dtype in (N.DT_BF16, N.DT_FP16):
        o = ragged(rows, experts, rng)
        print(dtype, rows, experts, n, k, o.tolist()[:20], flush=True)
        run_dw(dev, dtype, rows, n, k, o, seed=rows)
        run_dw(dev, dtype, rows, n, k, o, out32=True, seed=rows)
    run_dw(dev, N.DT_BF16, rows, n, k, None, seed=rows)


def test_weight_gradient_strides_and_alignment(dev):
    rng = np.random.default_rng(3)
    for pad, shift in ((1, 0), (8, 0), (0, 1), (3, 1), (8, 4)):
        for rows, n, k in ((50, 72, 136), (260, 136, 264), (33, 129, 65)):
            print(pad, shift, rows, n, k, flush=True)
            run_dw(dev, N.DT_BF16, rows, n, k, ragged(rows, 4, rng), pad=pad, shift=shift, seed=pad)


def test_large_weight_gradients(dev):
    rng = np.random.default_rng(8)
    for rows, experts, n, k, pad in ((300, 1, 4104, 4096, 0), (500, 4, 2080, 2056, 8), (200, 4, 2080, 2056, 1)):
        print(rows, experts, n, k, pad, flush=True)
        run_dw(dev, N.DT_FP16, rows, n, k, None if experts == 1 else ragged(rows, experts, rng), pad=pad, seed=k, out32=pad == 8)


@pytest.mark.parametrize("experts", [1, 2, 4, 8])
def test_weight_gradients_of_middling_sizes(dev, experts):
    rng = np.random.default_rng(experts)
    for t in (N.DT_BF16, N.DT_FP16):
        for out32 in (False, True):
            run_dw(dev, t, 300, 1032, 1032, ragged(300, experts, rng), out32=out32, seed=experts)


def test_few_rows_of_many_columns(dev):
    """A workgroup for every 32 columns fills the chip: one expert's rows, and a row each of many experts."""
    rng = np.random.default_rng(1)
    for rows, experts, n, k in ((1, 1, 8200, 136), (16, 1, 8200, 1000), (13, 1, 8201, 65), (40, 40, 520, 264), (100, 64, 264, 72)):
        o = None if experts == 1 else ragged(rows, experts, rng)
        print(rows, experts, n, k, flush=True)
        for t in (N.DT_BF16, N.DT_FP16):
            for out32 in (False, True):
                run(dev, t, rows, n, k, o, seed=k, out32=out32)
        for out in (N.DT_BF16, N.DT_FP16, N.DT_FP32):
            run8(dev, rows, n, k, o, out, seed=k)
    for rows, n, k in ((28, 1000, 520), (60, 1000, 520)):
        run(dev, N.DT_BF16, rows, n, k, None, seed=k, out32=True)
        run8(dev, rows, n, k, None, N.DT_BF16, seed=k)


def test_large_products_in_32_bits(dev):
    for nk in (True, False):
        run(dev, N.DT_BF16, 3200, 4160, 200, None, nk=nk, out32=True, seed=1)
        run(dev, N.DT_FP16, 3300, 4168, 136, None, nk=nk, out32=True, seed=2, pad=8)
        run(dev, N.DT_FP16, 3300, 4168, 136, None, nk=nk, seed=3)
    for t in (N.DT_BF16, N.DT_FP16):
        for out32 in (False, True):
            run(dev, t, 200, 263, 135, None, out32=out32, seed=4)      # nothing aligned


def test_weight_gradient_without_rows_is_zero(dev):
    with DevBufs(dev) as b:
        dw, o = b.put(np.full((2, 5, 7), 3, np.uint16)), b.put(np.zeros(3, np.int32))
        N.check(K.expert_product_dw(dw, None, None, o, 2, 0, 5, 7, N.DT_BF16))
        dev.sync()
        assert not dev.to_host(dw, 70, np.uint16).any()


# ------------------------------------------------------------------- e4m3

def run8(dev, rows, n, k, offsets, out, *, pad=0, shift=0, seed=0, codes=None):
    experts = 1 if offsets is None else len(offsets) - 1
    rng = np.random.default_rng(seed)
    kg, ng = -(-k // 128), -(-n // 128)
    make = codes or (lambda s: R.to_e4m3(np.clip(rng.standard_normal(s) * 120, -448, 448)))
    x, w = make((rows, k)), make((experts, n, k))
    xs = np.exp2(rng.uniform(-9, 1, (rows, kg))).astype(np.float32)
    ws = np.exp2(rng.uniform(-12, -4, (experts, ng, kg))).astype(np.float32)
    segs = offsets if offsets is not None else [0, rows]
    inside = np.zeros(rows, bool)
    for a, b in R.clamp_offsets(segs, rows):
        inside[a:b] = True
    x[~inside] = 0x7f
    xs[~inside] = np.nan
    odt = np.float32 if out == N.DT_FP32 else np.uint16
    fill = odt(9)
    ldx, ldy = k + pad, n + pad
    st = dict(x=ldx, w=ldx, y=ldy, expert_w=n * ldx + pad, xscale=kg + (pad > 0), wscale=kg + (pad > 0),
              expert_wscale=ng * (kg + (pad > 0)) + pad) if pad else None
    wbuf = with_ld(w, ldx, 0x7f).reshape(experts, -1)
    wsbuf = with_ld(ws, kg + (pad > 0), np.nan).reshape(experts, -1)
    if pad:
        wbuf = np.concatenate([wbuf, np.full((experts, pad), 0x7f, np.uint8)], axis=1)
        wsbuf = np.concatenate([wsbuf, np.full((experts, pad), np.nan, np.float32)], axis=1)
    with DevBufs(dev) as b:
        dx, dw = b.put(with_ld(x, ldx, 0x7f), pad_before=shift), b.put(wbuf, pad_before=shift)
        dxs, dws = b.put(with_ld(xs, kg + (pad > 0), np.nan)), b.put(wsbuf)
        do = b.put(np.ascontiguousarray(offsets)) if offsets is not None else None
        dy = b.put(np.full((rows, ldy), fill, odt), pad_before=shift * odt().itemsize)
        N.check(K.expert_product_e4m3(dy, dx, dxs, dw, dws, do, experts, rows, n, k, out, strides=st), "fx_expert_product_e4m3")
        dev.sync()
        y = dev.to_host(dy, rows * ldy, odt).reshape(rows, ldy)
    assert (y[:, n:] == fill).all() and (y[~inside] == fill).all()
    fx = R.E4M3[x] * np.repeat(xs.astype(np.float64), 128, axis=1)[:, :k]
    fw = R.E4M3[w] * np.repeat(np.repeat(ws.astype(np.float64), 128, axis=2)[:, :, :k], 128, axis=1)[:, :n]
    want, mag = R.product(fx, fw, segs, True)
    want, mag = want[inside], mag[inside]
    got = R.codes_to_f64(y[inside, :n], out)
    # fp32 results: sums as in fp32.  16-bit ones: the 8-bit matrix instructions' own error per group of 128.
    group = 0 if out == N.DT_FP32 else 2.0 ** -12
    assert R.within(got, want, out, R.sum_bound(min(k, 128) + kg + 4, mag) + group * mag)


@pytest.mark.parametrize("out", [N.DT_BF16, N.DT_FP16, N.DT_FP32])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 17, 5), (16, 64, 128), (17, 128, 144), (33, 500, 400), (65, 100, 200), (130, 257, 272),
                                      (300, 520, 1000)])
def test_e4m3_plain_products(dev, out, rows, n, k):
    print(out, rows, n, k, flush=True)
    run8(dev, rows, n, k, None, out, seed=rows)


@pytest.mark.parametrize("rows,experts,n,k", [(5, 3, 64, 64), (40, 8, 128, 256), (200, 5, 264, 336), (700, 13, 200, 96), (90, 200, 32, 64),
                                              (1100, 3, 300, 520)])
def test_e4m3_ragged_products(dev, rows, experts, n, k):
    rng = np.random.default_rng(rows)
    for out in (N.DT_BF16, N.DT_FP32):
        o = ragged(rows, experts, rng)
        print(out, rows, experts, n, k, o.tolist()[:20], flush=True)
        run8(dev, rows, n, k, o, out, seed=rows)


@pytest.mark.parametrize("rows,experts,n,k", [(40, 1, 528, 1104), (100, 1, 2064, 272), (250, 1, 3088, 144), (600, 1, 1040, 80),
                                              (1000, 20, 1296, 272), (1900, 32, 2064, 144), (4000, 30, 1040, 272)])
def test_e4m3_sizes_between_few_rows_and_full_tiles(dev, rows, experts, n, k):
    rng = np.random.default_rng(n)
    for out in (N.DT_BF16, N.DT_FP16, N.DT_FP32):
        run8(dev, rows, n, k, None if experts == 1 else ragged(rows, experts, rng), out, seed=k)


def test_e4m3_strides_and_alignment(dev):
    rng = np.random.default_rng(3)
    for pad, shift in ((1, 0), (16, 0), (0, 1), (3, 1), (16, 16)):
        for rows, n, k in ((50, 72, 144), (260, 136, 272), (33, 129, 65)):
            print(pad, shift, rows, n, k, flush=True)
            run8(dev, rows, n, k, ragged(rows, 4, rng), N.DT_BF16, pad=pad, shift=shift, seed=pad)
            run8(dev, rows, n, k, ragged(rows, 4, rng), N.DT_FP32, pad=pad, shift=shift, seed=pad)


@pytest.mark.parametrize("out", [N.DT_BF16, N.DT_FP16, N.DT_FP32])
def test_e4m3_large_products(dev, out):
    rng = np.random.default_rng(8)
    for rows, experts, n, k, pad in ((3200, 1, 4160, 400, 0), (3300, 7, 4176, 272, 16), (3100, 40, 4112, 128, 0), (3300, 7, 4176, 272, 1)):
        o = None if experts == 1 else ragged(rows, experts, rng)
        print(out, rows, experts, n, k, pad, flush=True)
        run8(dev, rows, n, k, o, out, pad=pad, seed=k)


# ------------------------------------------------------------------- graph

hip = C.CDLL("libamdhip64.so.7")
hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
hip.hipGraphExecDestroy.argtypes = [C.c_void_p]
hip.hipGraphDestroy.argtypes = [C.c_void_p]


@pytest.mark.parametrize("rows,n,k", [(24, 96, 160), (600, 320, 512)])
def test_products_replay_in_a_graph_with_new_routing(dev, rows, n, k):
    """The captured calls read the offsets when they execute: every replay has other rows per expert."""
    experts, t = 6, N.DT_BF16
    stream = dev.stream_create()
    raw = dev.raw_stream(stream)
    rng = np.random.default_rng(1)
    with DevBufs(dev) as b:
        w = R.normal(t, (experts, n, k), 9)
        dw, dx, do = b.put(w), b.alloc(rows * k * 2), b.alloc(64)
        dy, dg = b.alloc(rows * n * 2), b.alloc(experts * n * k * 4)
        graph, gexec = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(raw, 0) == 0
        try:
            N.check(K.expert_product(dy, dx, dw, do, experts, rows, n, k, t, stream=raw))
            N.check(K.expert_product_dw(dg, dy, dx, do, experts, rows, n, k, t, out_dtype=N.DT_FP32, stream=raw))
        finally:
            assert hip.hipStreamEndCapture(raw, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
        for rep in range(4):
            o = ragged(rows, experts, rng)
            dev.upload(dx, R.normal(t, (rows, k), rep))
            dev.upload(do, o)
            dev.memset(dy, 0, rows * n * 2)
            dev.sync()
            assert hip.hipGraphLaunch(gexec, raw) == 0
            dev.stream_sync(stream)
            got = dev.to_host(dy, rows * n, np.uint16), dev.to_host(dg, experts * n * k, np.uint32)
            dev.memset(dy, 0, rows * n * 2)
            N.check(K.expert_product(dy, dx, dw, do, experts, rows, n, k, t))
            N.check(K.expert_product_dw(dg, dy, dx, do, experts, rows, n, k, t, out_dtype=N.DT_FP32))
            dev.sync()
            assert np.array_equal(got[0], dev.to_host(dy, rows * n, np.uint16))
            assert np.array_equal(got[1], dev.to_host(dg, experts * n * k, np.uint32))
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
    dev.stream_destroy(stream)


@pytest.mark.parametrize("rows", [20, 1500])
def test_weights_and_rows_far_apart(dev, rows):
    """Offsets beyond 32 bits: experts 2.4 GB apart, and rows so far apart that the direct loads' offsets do not reach."""
    n, k, experts, t = 264, 136, 3, N.DT_BF16
    far = 1_200_000_000
    x, w = R.normal(t, (rows, k), 1), R.normal(t, (experts, n, k), 2)
    o = np.array([0, rows // 4, rows // 2, rows], np.int32)
    want, mag = R.product(R.codes_to_f64(x, t), R.codes_to_f64(w, t), o, True)
    with DevBufs(dev) as b:
        dx, do, dy = b.put(x), b.put(o), b.alloc(rows * n * 2)
        dw = b.alloc((far * (experts - 1) + n * k) * 2)
        for e in range(experts):
            dev.upload(dw + 2 * far * e, np.ascontiguousarray(w[e]))
        st = dict(x=k, w=k, y=n, expert_w=far)
        N.check(K.expert_product(dy, dx, dw, do, experts, rows, n, k, t, strides=st))
        dev.sync()
        got = R.codes_to_f64(dev.to_host(dy, rows * n, np.uint16).reshape(rows, n), t)
        assert (np.abs(got - want) <= R.rounding(want, t) * 1.01 + R.sum_bound(k, mag)).all()
        dev.free(b.ptrs.pop())
        ld = (5 << 30) // 2 // rows // 8 * 8                           # rows of x spread over 5 GB
        dfar, dw2 = b.alloc(rows * ld * 2), b.put(w)
        for r in range(rows):
            dev.upload(dfar + r * ld * 2, np.ascontiguousarray(x[r]))
        st = dict(x=ld, w=k, y=n, expert_w=n * k)
        N.check(K.expert_product(dy, dfar, dw2, do, experts, rows, n, k, t, strides=st))
        dev.sync()
        got = R.codes_to_f64(dev.to_host(dy, rows * n, np.uint16).reshape(rows, n), t)
        assert (np.abs(got - want) <= R.rounding(want, t) * 1.01 + R.sum_bound(k, mag)).all()
        # the weights' gradient walks the same far rows
        dyv = R.normal(t, (rows, n), 5)
        ddy, ddw = b.put(dyv), b.alloc(experts * n * k * 4)
        st = dict(dy=n, x=ld, dw=k, expert_dw=n * k)
        N.check(K.expert_product_dw(ddw, ddy, dfar, do, experts, rows, n, k, t, out_dtype=N.DT_FP32, strides=st))
        dev.sync()
        gw = dev.to_host(ddw, experts * n * k, np.float32).reshape(experts, n, k).astype(np.float64)
    want, mag = R.product_dw(R.codes_to_f64(dyv, t), R.codes_to_f64(x, t), o)
    assert (np.abs(gw - want) <= R.rounding(want, N.DT_FP32) * 1.01 + R.sum_bound(rows, mag)).all()


def test_products_on_two_streams_at_once(dev):
    rows, n, k, experts, t = 900, 520, 264, 5, N.DT_BF16
    rng = np.random.default_rng(4)
    streams = [dev.stream_create() for _ in range(2)]
    with DevBufs(dev) as b:
        sets = []
        for i in range(2):
            sets.append((b.alloc(rows * n * 2), b.put(R.normal(t, (rows, k), i)), b.put(R.normal(t, (experts, n, k), 7 + i)),
                         b.put(ragged(rows, experts, rng)), b.alloc(experts * n * k * 2)))
            dev.memset(sets[-1][0], 0, rows * n * 2)
        dev.sync()

        def call(s, raw):
            N.check(K.expert_product(s[0], s[1], s[2], s[3], experts, rows, n, k, t, stream=raw))
            N.check(K.expert_product_dw(s[4], s[0], s[1], s[3], experts, rows, n, k, t, stream=raw))
        read = lambda s: (dev.to_host(s[0], rows * n, np.uint16), dev.to_host(s[4], experts * n * k, np.uint16))  # noqa: E731
        alone = []
        for s in sets:
            call(s, None)
            dev.sync()
            alone.append(read(s))
        for _ in range(10):
            for s, st in zip(sets, streams):
                call(s, dev.raw_stream(st))
        dev.sync()
        for s, a in zip(sets, alone):
            got = read(s)
            assert np.array_equal(got[0], a[0]) and np.array_equal(got[1], a[1])
    for st in streams:
        dev.stream_destroy(st)


@pytest.mark.parametrize("rest", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255])
def test_last_tiles_of_every_length(dev, rest):
    """Experts whose last tile has `rest` rows, in the smallest and the largest tile shapes."""
    o = np.cumsum([0, 256 + rest, rest, 0, 512, rest]).astype(np.int32)
    for n, k in ((200, 72), (4104, 128)):
        run(dev, N.DT_BF16, int(o[-1]) + 3, n, k, o, seed=rest)
        run(dev, N.DT_FP16, int(o[-1]) + 3, n, k, o, seed=rest, nk=False)
        run8(dev, int(o[-1]) + 3, n // 16 * 16, k // 16 * 16, o, N.DT_BF16, seed=rest)


@pytest.mark.parametrize("rests", [(1, 64, 130, 200), (63, 65, 129, 193), (255, 192, 128, 16)])
def test_last_tiles_among_many_large_ones(dev, rests):
    o = np.cumsum([0, 2048 + rests[0], 1536 + rests[1], 0, rests[2], 4096 + rests[3]]).astype(np.int32)
    rows = int(o[-1]) + 5
    for nk in (True, False):
        run(dev, N.DT_BF16, rows, 4168, 136, o, nk=nk, seed=rests[0])
    run8(dev, rows, 4176, 272, o, N.DT_BF16, seed=rests[0])
    run8(dev, rows, 4176, 144, o, N.DT_FP32, seed=rests[0])


def test_e4m3_long_reduction_in_large_tiles(dev):
    """Long enough for the lines that are touched ahead, with and without a partial slab at the end."""
    for k in (1024, 1040, 2064):
        run8(dev, 3200, 4160, k, None, N.DT_BF16, seed=k)
        run8(dev, 4500, 4160, k, np.array([0, 2100, 4400], np.int32), N.DT_BF16, seed=k)


def test_infinities_and_nan_stay_in_their_rows(dev):
    """A row with a NaN or an infinity spoils its own results alone, also where its tile's other rows belong to another
    expert; a weight with one spoils its own column."""
    for rows, n, k in ((40, 136, 264), (700, 264, 136)):
        x, w = R.normal(N.DT_BF16, (rows, k), 1), R.normal(N.DT_BF16, (2, n, k), 2)
        x[rows // 2, 3], x[rows // 2 + 1, k - 1] = 0x7fc0, 0x7f80
        w[1, 7, k - 1] = 0x7fc0
        o = np.array([0, rows // 2 + 1, rows], np.int32)
        with DevBufs(dev) as b:
            dx, dw, do, dy = b.put(x), b.put(w), b.put(o), b.alloc(rows * n * 4)
            N.check(K.expert_product(dy, dx, dw, do, 2, rows, n, k, N.DT_BF16, out_dtype=N.DT_FP32))
            dev.sync()
            y = dev.to_host(dy, rows * n, np.float32).reshape(rows, n)
        assert np.isnan(y[rows // 2]).all() and not np.isfinite(y[rows // 2 + 1]).any()
        assert np.isnan(y[rows // 2 + 1:, 7]).all()
        rest = np.delete(y, [rows // 2, rows // 2 + 1], axis=0)
        assert np.isfinite(rest[:rows // 2]).all() and np.isfinite(np.delete(rest, 7, axis=1)).all()


@pytest.mark.parametrize("nk", [True, False])
@pytest.mark.parametrize("rows,n,k", [(8, 136, 264), (300, 264, 136), (301, 261, 133)])
def test_fp16_subnormals_keep_their_values(dev, nk, rows, n, k):
    """Rows of nothing but subnormal values: the products are those of the values, not of zeros."""
    rng = np.random.default_rng(rows)
    x = (rng.integers(1, 0x400, (rows, k)) | rng.integers(0, 2, (rows, k)) << 15).astype(np.uint16)
    w = R.normal(N.DT_FP16, (1, n, k) if nk else (1, k, n), 5)
    with DevBufs(dev) as b:
        dx, dw, dy = b.put(x), b.put(w), b.alloc(rows * n * 4)
        N.check(K.expert_product(dy, dx, dw, None, 1, rows, n, k, N.DT_FP16, out_dtype=N.DT_FP32, layout=K.W_NK if nk else K.W_KN))
        dev.sync()
        y = dev.to_host(dy, rows * n, np.float32).reshape(rows, n).astype(np.float64)
    want, mag = R.product(R.codes_to_f64(x, N.DT_FP16), R.codes_to_f64(w, N.DT_FP16), [0, rows], nk)
    assert (np.abs(y - want) <= R.rounding(want, N.DT_FP32) * 1.01 + R.sum_bound(k, mag)).all()


@pytest.mark.parametrize("rest", [1, 2, 3, 5, 7, 8, 9, 11, 15, 16, 17, 31, 33, 63])
def test_reductions_and_widths_of_every_remainder(dev, rest):
    """What is left behind whole chunks and whole slabs, on rows that start at any byte: few rows, small and large tiles."""
    rng = np.random.default_rng(rest)
    n, k = 128 + rest, 192 + rest
    for nk in (True, False):
        run(dev, N.DT_BF16, 21, n, k, ragged(21, 3, rng), nk=nk, seed=rest)
        run(dev, N.DT_FP16, 500, n, k, ragged(500, 3, rng), nk=nk, out32=True, seed=rest)
        run(dev, N.DT_FP16, 150, rest, rest, None, nk=nk, seed=rest)
    run_dw(dev, N.DT_BF16, 300, n, k, ragged(300, 3, rng), seed=rest)
    run_dw(dev, N.DT_FP16, 60 + rest, rest, n, ragged(60 + rest, 2, rng), out32=True, seed=rest)
    run8(dev, 21, n, k, ragged(21, 3, rng), N.DT_BF16, seed=rest)
    run8(dev, 500, n, k, ragged(500, 3, rng), N.DT_FP16, seed=rest)
    run8(dev, 500, n, k, ragged(500, 3, rng), N.DT_FP32, shift=rest % 4, pad=rest % 5, seed=rest)
    run8(dev, 150, rest, rest, None, N.DT_BF16, seed=rest)


def test_large_products_of_odd_sizes(dev):
    """Enough rows for tiles of 128 at sizes that no vector divides."""
    rng = np.random.default_rng(9)
    for rows, n, k in ((4500, 2057, 141), (4501, 2061, 322)):
        for nk in (True, False):
            for t in (N.DT_BF16, N.DT_FP16):
                run(dev, t, rows, n, k, ragged(rows, 3, rng), nk=nk, out32=rows % 2 == 0, seed=n)
                run(dev, t, rows, n, k, None, nk=nk, out32=rows % 2 == 1, seed=n)
        for out in (N.DT_BF16, N.DT_FP16, N.DT_FP32):
            run8(dev, rows, n, k, ragged(rows, 3, rng), out, seed=n)
    for t in (N.DT_BF16, N.DT_FP16):
        for out32 in (False, True):
            run_dw(dev, t, 1501, 1029, 2053, ragged(1501, 12, rng), out32=out32, seed=3)


@pytest.mark.parametrize("nk", [True, False])
def test_rows_of_less_than_a_chunk_and_few_rows_at_any_byte(dev, nk):
    rng = np.random.default_rng(4)
    for t in (N.DT_BF16, N.DT_FP16):
        for out32 in (False, True):
            run(dev, t, 150, 5, 7, None, nk=nk, out32=out32, seed=1)
            run(dev, t, 31, 205, 203, ragged(31, 1, rng), nk=nk, out32=out32, seed=2)
            run(dev, t, 20, 205, 203, None, nk=nk, out32=out32, pad=1, shift=1, seed=3)
            run_dw(dev, t, 150, 5, 70, ragged(150, 3, rng), out32=out32, seed=4)
    for out in (N.DT_BF16, N.DT_FP16, N.DT_FP32):
        run8(dev, 150, 70, 13, None, out, seed=5)
        run8(dev, 50, 205, 203, None, out, seed=6)
        run8(dev, 18, 205, 403, ragged(18, 1, rng), out, pad=1, shift=3, seed=7)


def cancelling(rng, shape):
    """e4m3 codes in which every run of eight columns holds two large values of opposite sign and six small ones, at random
    places; used on both sides, the large products of a run cancel."""
    rows, k = int(np.prod(shape[:-1])), shape[-1]
    c = rng.integers(0x01, 0x40, (rows, -(-k // 8), 8)).astype(np.uint8)
    big = rng.integers(0x70, 0x7f, (rows, c.shape[1]))
    c[:, :, 2], c[:, :, 5] = big, big
    return c.reshape(rows, -1)[:, :k].reshape(shape)


def just_below(side, shape):
    """Runs of one product 256 * 256 and seven of 2 * 3.75, just below the eighth that the cut keeps."""
    c = np.full(shape, 0x47 if side else 0x40, np.uint8)
    c[..., ::8] = 0x78
    return c


def cut_products(x, w):
    """Sums over whole rows of k columns as the 8-bit matrix instructions form them, in 64 bits but for the cut, and the
    magnitudes that the documented bound is taken of.  x [rows, k], w [n, k]: codes."""
    field = lambda c: np.where(c & 0x78, ((c >> 3) & 15).astype(int) - 7, -6)  # noqa: E731
    lifted = lambda c: np.where(c & 0x7f, np.maximum(np.abs(R.E4M3[c]), 2.0 ** -6), 0.0)  # noqa: E731
    got, mag = np.zeros((x.shape[0], w.shape[0])), np.zeros((x.shape[0], w.shape[0]))
    for c in range(0, x.shape[1], 8):
        xs, ws = x[:, None, c:c + 8], w[None, :, c:c + 8]
        p = R.E4M3[xs] * R.E4M3[ws]
        e = np.where(p != 0, field(xs) + field(ws), -99).max(axis=2, keepdims=True)
        u = 2.0 ** (e - 13.0)
        got += (np.trunc(p / u) * u).sum(axis=2)
        mag += (lifted(xs) * lifted(ws)).max(axis=2)
    return got, mag


@pytest.mark.parametrize("out", [N.DT_BF16, N.DT_FP16, N.DT_FP32])
@pytest.mark.parametrize("kind", ["cancelling", "below", "any"])
@pytest.mark.parametrize("rows,n,k", [(70, 64, 128), (200, 200, 256), (700, 72, 141), (300, 520, 13), (5000, 40, 384), (2100, 272, 128)])
def test_e4m3_sums_are_cut_as_documented(dev, out, kind, rows, n, k):
    """One scale of 1, so that the result is the sum itself.  16-bit results: off the exact sum by less than 2^-10 of each
    run's largest product (a run of eight loses less than 2^(e-13) of each of its eight products at most, and the largest
    lifted one is at least 2^e); and what the cut leaves is summed as in fp32.  fp32 results: no cut."""
    rng = np.random.default_rng(rows)
    some = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    make = {"cancelling": lambda side, s: cancelling(rng, s), "below": just_below, "any": lambda side, s: rng.choice(some, s)}[kind]
    x, w = make(0, (rows, k)), make(1, (n, k))
    if kind == "cancelling":
        x[:, 5::8] |= 0x80                                   # + and - in the pair
    kg, ng = -(-k // 128), -(-n // 128)
    odt = np.float32 if out == N.DT_FP32 else np.uint16
    with DevBufs(dev) as b:
        dx, dw, dy = b.put(x), b.put(w), b.alloc(rows * n * 4)
        ones = b.put(np.ones(max(rows, ng) * kg, np.float32))
        N.check(K.expert_product_e4m3(dy, dx, ones, dw, ones, None, 1, rows, n, k, out))
        dev.sync()
        got = R.codes_to_f64(dev.to_host(dy, rows * n, odt).reshape(rows, n), out)
    want = R.E4M3[x] @ R.E4M3[w].T
    mag = np.abs(R.E4M3[x]) @ np.abs(R.E4M3[w]).T
    sums = R.sum_bound(min(k, 128) + kg + 4, mag)
    if out == N.DT_FP32:
        assert R.within(got, want, out, sums)
        return
    cut, largest = cut_products(x, w)
    assert (np.abs(cut - want) <= 2.0 ** -10 * largest).all()
    assert R.within(got, want, out, sums + 2.0 ** -10 * largest)
    assert R.within(got, cut, out, sums)
    if kind == "cancelling" and k % 8 == 0:                  # every pair is whole: what the documentation warns of
        assert (np.abs(cut - want) > np.abs(want) / 4).any()
    if kind == "below":
        assert (np.abs(cut - want) > 2.0 ** -11 * mag).all()


def test_many_experts_that_claim_all_rows_touch_nothing_outside(dev):
    """Boundaries 0, rows, 0, rows, ... of 131072 experts: their tiles, counted, are 2^30, and 2^32 in four columns of tiles.
    All experts share one matrix, so a row is right or left alone."""
    rows, n, k, experts = 1 << 20, 8, 8, 1 << 17
    x, w = R.normal(N.DT_BF16, (rows, k), 1), R.normal(N.DT_BF16, (1, k, n), 2)
    o = np.zeros(experts + 1, np.int32)
    o[1::2] = rows
    guard = np.full((256, n), 9, np.uint16)
    with DevBufs(dev) as b:
        dx, dw, do = b.put(x), b.put(w), b.put(o)
        base = b.put(np.concatenate([guard, np.full((rows, n), 9, np.uint16), guard]))
        st = dict(x=k, w=n, y=n, expert_w=0)
        N.check(K.expert_product(base + guard.nbytes, dx, dw, do, experts, rows, n, k, N.DT_BF16, layout=K.W_KN, strides=st))
        dev.sync()
        y = dev.to_host(base, (rows + 512) * n, np.uint16).reshape(-1, n)
    assert (y[:256] == 9).all() and (y[-256:] == 9).all()
    y = y[256:-256]
    done = ~(y == 9).all(axis=1)
    want, mag = R.product(R.codes_to_f64(x, N.DT_BF16), R.codes_to_f64(w, N.DT_BF16), [0, rows], False)
    bad = np.abs(R.codes_to_f64(y, N.DT_BF16) - want) > R.rounding(want, N.DT_BF16) * 1.01 + R.sum_bound(k, mag)
    assert done.any() and not bad[done].any()


def test_more_columns_than_one_launch_takes(dev):
    """4096 experts with a row each share one matrix of so many columns that the call goes through them in two launches;
    likewise the weights' gradient of a million experts, most of them without rows."""
    experts, k = 4096, 16
    x, o = R.normal(N.DT_BF16, (experts, k), 1), np.arange(experts + 1, dtype=np.int32)
    for n, fp8 in ((62500, False), (123500, True)):
        some = np.unique(np.concatenate([np.arange(0, n, 97), np.arange(61300, 61900), np.arange(n - 600, n)]))
        kw = dict(x=k, w=k, y=n, expert_w=0)
        with DevBufs(dev) as b:
            dy, do = b.alloc(experts * n * 2), b.put(o)
            if fp8:
                rng = np.random.default_rng(2)
                x8, w = (R.to_e4m3(np.clip(rng.standard_normal(s) * 120, -448, 448)) for s in ((experts, k), (n, k)))
                xs, ws = np.exp2(rng.uniform(-9, 1, (experts, 1))).astype(np.float32), np.exp2(rng.uniform(-12, -4, (-(-n // 128), 1))).astype(np.float32)
                st = dict(kw, xscale=1, wscale=1, expert_wscale=0)
                N.check(K.expert_product_e4m3(dy, b.put(x8), b.put(xs), b.put(w), b.put(ws), do, experts, experts, n, k, N.DT_BF16, strides=st))
                fx, fw = R.E4M3[x8] * xs, (R.E4M3[w] * np.repeat(ws.astype(np.float64), 128, axis=0)[:n])[some]
            else:
                w = R.normal(N.DT_BF16, (n, k), 2)
                N.check(K.expert_product(dy, b.put(x), b.put(w), do, experts, experts, n, k, N.DT_BF16, strides=kw))
                fx, fw = R.codes_to_f64(x, N.DT_BF16), R.codes_to_f64(w[some], N.DT_BF16)
            dev.sync()
            y = dev.to_host(dy, experts * n, np.uint16).reshape(experts, n)[:, some]
        want, mag = fx @ fw.T, np.abs(fx) @ np.abs(fw).T
        assert (np.abs(R.codes_to_f64(y, N.DT_BF16) - want) <= R.rounding(want, N.DT_BF16) * 1.01 + R.sum_bound(k + 8, mag)).all(), fp8
    experts, rows, k = 1 << 20, 300, 2000                    # one column of dy: 2000 dw values an expert
    dy, x = R.normal(N.DT_BF16, (rows, 1), 3), R.normal(N.DT_BF16, (rows, k), 4)
    at = np.sort(np.random.default_rng(5).choice(experts, rows // 2, replace=False))         # the experts of two rows each
    o = np.zeros(experts + 1, np.int32)
    o[at + 1] = 2
    o = np.cumsum(o).astype(np.int32)
    f = lambda a: R.codes_to_f64(a, N.DT_BF16)  # noqa: E731
    with DevBufs(dev) as b:
        dw = b.alloc(experts * k * 2)
        N.check(K.expert_product_dw(dw, b.put(dy), b.put(x), b.put(o), experts, rows, 1, k, N.DT_BF16))
        dev.sync()
        for i, e in enumerate(at):
            got = f(dev.to_host(dw + int(e) * k * 2, k, np.uint16))
            a, d = f(x[2 * i:2 * i + 2]), f(dy[2 * i:2 * i + 2])
            want, mag = (d * a).sum(axis=0), np.abs(d * a).sum(axis=0)
            assert (np.abs(got - want) <= R.rounding(want, N.DT_BF16) * 1.01 + R.sum_bound(2, mag)).all(), e
        for e in (0, 1, 77777, experts - 1):
            if e not in at:
                assert not dev.to_host(dw + e * k * 2, k, np.uint16).any()


@pytest.mark.parametrize("out", [N.DT_BF16, N.DT_FP32])
@pytest.mark.parametrize("rows,n,k,offsets", [(330, 208, 8320, [0, 90, 200, 330]), (330, 208, 16400, [0, 90, 200, 330]), (130, 1040, 8336, None),
                                              (1600, 1040, 8320, [0, 520, 1090, 1600]), (1600, 1040, 16400, [0, 520, 1090, 1600]),
                                              (4400, 1040, 8336, [0, 2150, 4400]), (300, 200, 8325, [0, 100, 300]),
                                              (40, 200, 16400, [0, 10, 25, 40]), (12, 200, 8325, [0, 5, 12])])
def test_e4m3_reductions_of_many_blocks(dev, out, rows, n, k, offsets):
    """More than 64 groups of 128 (a wavefront holds 64 blocks' scales at a time), walked from another slab for each expert
    and around the end, with a partial last group."""
    print(out, rows, n, k, flush=True)
    run8(dev, rows, n, k, None if offsets is None else np.array(offsets, np.int32), out, seed=k)


@pytest.mark.parametrize("rows,n,k,offsets", [(2600, 4160, 8336, [0, 1200, 2600]), (4400, 2080, 8336, [0, 2150, 4400])])
def test_e4m3_reductions_of_many_blocks_in_the_largest_tiles(dev, rows, n, k, offsets):
    run8(dev, rows, n, k, np.array(offsets, np.int32), N.DT_BF16, seed=k)
