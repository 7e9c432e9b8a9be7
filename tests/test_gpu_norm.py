"""fx_reduce_norm and its gradients against the 64-bit restatement."""
import ctypes as C

import numpy as np
import pytest

from flagcx_amd import _native as N
from flagcx_amd import kernels as K
from tests import model_ref as R
from tests.util import DevBufs

pytestmark = pytest.mark.gpu

EPS = 1e-6
TYPES = {"bf16": N.DT_BF16, "fp16": N.DT_FP16, "fp32": N.DT_FP32}


def padded(codes, ld, fill):
    """Rows of `ld` elements whose tails hold a pattern."""
    out = np.full((codes.shape[0], ld), fill, codes.dtype)
    out[:, :codes.shape[1]] = codes
    return out


def run_norm(dev, dtype, rows, cols, k, *, residual=True, weight="same", quant=False, pad=0, shift=0, alias=None, seed=0, edit=None):
    """Runs the call and checks every output; returns the raw outputs."""
    es, wd = N.DTYPE_SIZE[dtype], N.DT_FP32 if weight == "fp32" else dtype
    ins = [R.normal(dtype, (rows, cols), seed + p) for p in range(k)]
    res = R.normal(dtype, (rows, cols), seed + 77, 3.0) if residual else None
    w = R.normal(wd, (cols,), seed + 99) if weight else None
    if edit:
        edit(ins)
    ld, groups = cols + pad, -(-cols // 128)
    lds = groups + (pad > 0)
    st = dict(in_=ld, residual=ld, total=ld, out=ld, scale=lds) if pad else None
    fill = np.array([0x4b4b4b4b], np.uint32).view(ins[0].dtype)[0]
    with DevBufs(dev) as b:
        put = lambda a: b.put(padded(a, ld, fill), pad_before=shift * a.itemsize)  # noqa: E731
        dins, dres = [put(a) for a in ins], put(res) if residual else None
        dw = b.put(w, pad_before=shift * w.itemsize) if w is not None else None
        dtot = put(np.full((rows, cols), fill, ins[0].dtype))
        oes = 1 if quant else es
        odt = np.uint8 if quant else ins[0].dtype
        ofill = np.uint8(0x4b) if quant else fill
        dout = b.put(np.full((rows, ld), ofill, odt), pad_before=shift * oes)
        dsc = b.put(np.full((rows, lds), -7.0, np.float32)) if quant else None
        if alias == "total=residual":
            dtot = dres
        elif alias == "total=in":
            dtot = dins[-1]
        elif alias == "out=in":
            dout = dins[0]
        N.check(K.reduce_norm(dout, dins, dw, rows, cols, dtype, eps=EPS, residual=dres, total=dtot, scale=dsc,
                              out_dtype=N.DT_E4M3 if quant else None, weight_dtype=wd, strides=st), "fx_reduce_norm")
        dev.sync()
        total = dev.to_host(dtot, rows * ld, N.NP_DTYPE[dtype]).reshape(rows, ld)
        out = dev.to_host(dout, rows * ld, odt).reshape(rows, ld)
        scale = dev.to_host(dsc, rows * lds, np.float32).reshape(rows, lds) if quant else None
    if pad:
        assert (total[:, cols:] == fill).all() and (out[:, cols:] == (fill if alias == "out=in" else ofill)).all()
        assert scale is None or (scale[:, groups:] == -7.0).all()
    total, out = total[:, :cols], out[:, :cols]
    f = [R.codes_to_f64(a, dtype) for a in ins]
    fr = R.codes_to_f64(res, dtype) if residual else None
    fw = R.codes_to_f64(w, wd) if w is not None else None
    s, y, mag, r = R.norm(f, fr, fw, EPS)
    ds, dy = R.norm_bounds(s, y, mag, r, fw, k + residual)
    fine = np.isfinite(s).all(axis=1)
    err = np.abs(R.codes_to_f64(total, dtype) - s)
    assert (err[fine] <= (R.rounding(s, dtype) * 1.01 + ds)[fine]).all(), "total"
    if not quant:
        err = np.abs(R.codes_to_f64(out, dtype) - y)
        assert (err[fine] <= (R.rounding(y, dtype) * 1.01 + dy)[fine]).all(), "out"
    else:
        sc = scale[:, :groups].astype(np.float64)
        for g in range(groups):
            c = slice(g * 128, (g + 1) * 128)
            amax = np.abs(y[:, c]).max(axis=1)
            want = np.maximum(amax / 448, 2.0 ** -126)
            assert (np.abs(sc[:, g] - want) <= 4 * R.E * want + dy[:, c].max(axis=1) / 448)[fine].all(), "scale"
            # e4m3: half a step of the value, 2^-4, or half the subnormal step 2^-9, times the scale
            got = R.E4M3[out[:, c]] * sc[:, g:g + 1]
            tol = np.maximum(2.0 ** -4 * np.abs(y[:, c]) * 1.001, 2.0 ** -10 * sc[:, g:g + 1] * 1.001) + 2 * dy[:, c] + 8 * R.E * np.abs(y[:, c])
            assert (np.abs(got - y[:, c]) <= tol)[fine].all(), "out"
            top = np.abs(R.E4M3[out[:, c]]).max(axis=1)
            assert (((top == 448) | (amax < 448 * 2.0 ** -126)) | ~fine).all(), "the largest of a group is 448"
    return total, out, scale


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [1, 7, 8, 127, 128, 129, 500, 512, 513, 1000, 1025, 2048, 2049, 4100, 8192, 8200, 16385, 32768, 32769, 40003])
def test_norm_widths(dev, name, cols):
    print(name, cols, flush=True)
    run_norm(dev, TYPES[name], 5, cols, 2, seed=cols)
    run_norm(dev, TYPES[name], 3, cols, 3, quant=True, seed=cols, residual=False)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 7, 8, 9, 17, 64])
@pytest.mark.parametrize("cols", [300, 1500, 5000, 33000])
def test_norm_inputs(dev, k, cols):
    print(k, cols, flush=True)
    run_norm(dev, N.DT_BF16, 9, cols, k, seed=k)
    run_norm(dev, N.DT_FP16, 2, cols, k, residual=False, weight=None, seed=k, quant=k % 2 == 0)


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 255, 256, 257, 1030])
def test_norm_rows(dev, rows):
    run_norm(dev, N.DT_BF16, rows, 640, 2, seed=rows, quant=True)
    run_norm(dev, N.DT_FP32, rows, 1536, 2, seed=rows)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("weight", ["same", "fp32", None])
def test_norm_strides_and_alignment(dev, name, quant, weight):
    for cols, pad, shift in ((200, 3, 1), (1000, 5, 3), (4096, 7, 1), (33001, 9, 1)):
        print(name, quant, weight, cols, flush=True)
        run_norm(dev, TYPES[name], 4, cols, 2, quant=quant, weight=weight, pad=pad, shift=shift, seed=cols)


@pytest.mark.parametrize("alias", ["total=residual", "total=in", "out=in"])
@pytest.mark.parametrize("cols", [3, 100, 515, 2000, 2052, 9000, 35000, 32772, 40963])
def test_norm_in_place(dev, alias, cols):
    run_norm(dev, N.DT_BF16, 6, cols, 3, alias=alias, seed=cols)
    run_norm(dev, N.DT_FP32, 2, cols, 2, alias=alias, seed=cols, pad=4)


def test_norm_zeros_infinities_and_nan(dev):
    """A row of zeros gives zeros and the smallest scale; a NaN or an infinity stays in its row, and in a row with an
    infinity only the groups that hold it are NaN (everything else is a finite value times zero)."""
    rows, cols = 6, 400
    x = np.zeros((rows, cols), np.float32)
    x[1] = np.linspace(-3, 3, cols)
    x[2] = 1
    x[2, 5] = np.nan
    x[3] = 2
    x[3, 390] = np.inf
    x[4] = 1e-38
    x[5] = -0.0
    with DevBufs(dev) as b:
        dx, do, ds, dq = b.put(x), b.alloc(x.nbytes), b.alloc(rows * 4 * 4), b.alloc(rows * cols)
        N.check(K.reduce_norm(do, [dx], None, rows, cols, N.DT_FP32, eps=EPS))
        N.check(K.reduce_norm(dq, [dx], None, rows, cols, N.DT_FP32, eps=EPS, out_dtype=N.DT_E4M3, scale=ds))
        dev.sync()
        y = dev.to_host(do, rows * cols, np.float32).reshape(rows, cols)
        q = dev.to_host(dq, rows * cols, np.uint8).reshape(rows, cols)
        s = dev.to_host(ds, rows * 4, np.float32).reshape(rows, 4)
    assert not y[0].any() and not (q[0] & 0x7f).any() and (s[0] == np.float32(2.0 ** -126)).all()
    assert np.isfinite(y[1]).all() and np.isfinite(s[1]).all()
    assert np.isnan(y[2]).all() and np.isnan(s[2]).all() and (q[2] & 0x7f == 0x7f).all()
    assert np.isnan(y[3, 390]) and not np.delete(y[3], 390).any()
    assert np.isnan(s[3, 3]) and (q[3, 384:] & 0x7f == 0x7f).all()
    assert (s[3, :3] == np.float32(2.0 ** -126)).all() and not (q[3, :384] & 0x7f).any()
    assert np.allclose(y[4], 1e-38 * 1e3, rtol=1e-5, atol=0)
    assert not y[5].any() and np.signbit(y[5]).all()                # -0 is not turned into +0


def run_grad(dev, dtype, rows, cols, *, dtotal=True, weight="same", pad=0, shift=0, alias=None, seed=0, want=("dx", "dweight")):
    wd = N.DT_FP32 if weight == "fp32" else dtype
    x, dy = R.normal(dtype, (rows, cols), seed, 2.0), R.normal(dtype, (rows, cols), seed + 1)
    dt = R.normal(dtype, (rows, cols), seed + 2) if dtotal else None
    w = R.normal(wd, (cols,), seed + 3) if weight else None
    ld = cols + pad
    st = dict(dy=ld, x=ld, dtotal=ld, dx=ld) if pad else None
    fill = np.array([0x4b4b4b4b], np.uint32).view(x.dtype)[0]
    need = K.reduce_norm_grad_workspace(rows, cols)
    with DevBufs(dev) as b:
        put = lambda a: b.put(padded(a, ld, fill), pad_before=shift * a.itemsize)  # noqa: E731
        ddy, dxx, ddt = put(dy), put(x), put(dt) if dtotal else None
        dw = b.put(w, pad_before=shift * w.itemsize) if w is not None else None
        ddx = {"dy": ddy, "dtotal": ddt}.get(alias) or put(np.full((rows, cols), fill, x.dtype))
        ddw = b.put(np.full(cols, 3, N.NP_DTYPE[wd]), pad_before=shift * N.DTYPE_SIZE[wd])
        ws = b.put(np.full(need + 64, 0xEE, np.uint8))
        N.check(K.reduce_norm_grad(ddx if "dx" in want else None, ddw if "dweight" in want else None, ddy, dxx, dw, rows, cols, dtype,
                                   ws, need, eps=EPS, dtotal=ddt, weight_dtype=wd, strides=st), "fx_reduce_norm_grad")
        dev.sync()
        gdx = dev.to_host(ddx, rows * ld, N.NP_DTYPE[dtype]).reshape(rows, ld)
        gdw = dev.to_host(ddw, cols, N.NP_DTYPE[wd])
        tail = dev.to_host(ws, need + 64, np.uint8)[need:]
    assert (tail == 0xEE).all(), "the workspace ends where it should"
    f = lambda a, t=dtype: None if a is None else R.codes_to_f64(a, t)  # noqa: E731
    edx, edw, bx, bw = R.norm_grad(f(dy), f(x), f(w, wd), f(dt), EPS)
    if "dx" in want:
        assert (gdx[:, cols:] == fill).all()
        assert (np.abs(f(gdx[:, :cols]) - edx) <= R.rounding(edx, dtype) * 1.01 + bx).all(), "dx"
    else:
        assert (gdx == fill).all()
    if "dweight" in want:
        assert (np.abs(f(gdw, wd) - edw) <= R.rounding(edw, wd) * 1.01 + bw).all(), "dweight"
    else:
        assert (f(gdw, wd) == f(np.full(1, 3, N.NP_DTYPE[wd]), wd)).all()
    return gdx, gdw


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [1, 9, 128, 511, 1000, 1030, 2047, 4096, 4099, 8200, 16384, 17000, 33000])
def test_norm_gradient_widths(dev, name, cols):
    print(name, cols, flush=True)
    run_grad(dev, TYPES[name], 7, cols, seed=cols)
    run_grad(dev, TYPES[name], 70, cols, seed=cols, dtotal=False, weight="fp32")


@pytest.mark.parametrize("rows", [1, 2, 5, 511, 513, 2000])
def test_norm_gradient_rows(dev, rows):
    for cols in (96, 1025):
        run_grad(dev, N.DT_BF16, rows, cols, seed=rows)
        run_grad(dev, N.DT_FP32, rows, cols, seed=rows, weight=None)


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [3, 200, 516, 3000, 4099, 16381, 32772, 33010])
def test_norm_gradient_strides_aliases_and_parts(dev, name, cols):
    t = TYPES[name]
    run_grad(dev, t, 6, cols, pad=3, shift=1, seed=cols)
    for alias in ("dy", "dtotal"):
        run_grad(dev, t, 6, cols, alias=alias, seed=cols)
    run_grad(dev, t, 6, cols, want=("dx",), seed=cols)
    run_grad(dev, t, 6, cols, want=("dweight",), seed=cols)


def test_norm_gradient_without_rows_clears_dweight(dev):
    with DevBufs(dev) as b:
        dw = b.put(np.full(300, 5.0, np.float32))
        N.check(K.reduce_norm_grad(None, dw, None, None, None, 0, 300, N.DT_FP32, None, 0, eps=EPS))
        dev.sync()
        assert not dev.to_host(dw, 300, np.float32).any()


def test_norm_gradient_twice_gives_the_same_bits(dev):
    a = run_grad(dev, N.DT_BF16, 1500, 1000, seed=4)
    b = run_grad(dev, N.DT_BF16, 1500, 1000, seed=4)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


hip = C.CDLL("libamdhip64.so.7")
hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
hip.hipGraphExecDestroy.argtypes = [C.c_void_p]
hip.hipGraphDestroy.argtypes = [C.c_void_p]


def test_norm_and_gradients_replay_in_a_graph(dev):
    rows, cols, t = 40, 1100, N.DT_BF16
    stream = dev.stream_create()
    raw = dev.raw_stream(stream)
    need = K.reduce_norm_grad_workspace(rows, cols)
    with DevBufs(dev) as b:
        din = [b.alloc(rows * cols * 2) for _ in range(3)]
        dres, dy, dwt, tot, out, dx, dwg = (b.alloc(rows * cols * 2) for _ in range(7))
        ws = b.alloc(need)
        w = R.normal(t, (cols,), 1)
        dev.upload(dwt, w)
        graph, gexec = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(raw, 0) == 0
        try:
            N.check(K.reduce_norm(out, din, dwt, rows, cols, t, eps=EPS, residual=dres, total=tot, stream=raw))
            N.check(K.reduce_norm_grad(dx, dwg, dy, tot, dwt, rows, cols, t, ws, need, eps=EPS, dtotal=out, stream=raw))
        finally:
            assert hip.hipStreamEndCapture(raw, C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
        for rep in range(4):
            for p, d in enumerate(din + [dres, dy]):
                dev.upload(d, R.normal(t, (rows, cols), 50 * rep + p))
            for d in (tot, out, dx, dwg):
                dev.memset(d, 0xEE, cols * 2)
            dev.sync()
            assert hip.hipGraphLaunch(gexec, raw) == 0
            dev.stream_sync(stream)
            got = [dev.to_host(d, n, np.uint16) for d, n in ((tot, rows * cols), (out, rows * cols), (dx, rows * cols), (dwg, cols))]
            N.check(K.reduce_norm(out, din, dwt, rows, cols, t, eps=EPS, residual=dres, total=tot))
            N.check(K.reduce_norm_grad(dx, dwg, dy, tot, dwt, rows, cols, t, ws, need, eps=EPS, dtotal=out))
            dev.sync()
            eager = [dev.to_host(d, n, np.uint16) for d, n in ((tot, rows * cols), (out, rows * cols), (dx, rows * cols), (dwg, cols))]
            for g, e in zip(got, eager):
                assert np.array_equal(g, e), rep
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)
    dev.stream_destroy(stream)


def test_norm_rows_far_apart_and_many(dev):
    """Offsets beyond 32 bits: rows 16 MiB apart (4.8 GB from first to last), and more rows than one launch takes."""
    rows, cols, ld = 300, 640, 8 << 20
    x = R.normal(N.DT_BF16, (rows, cols), 3)
    with DevBufs(dev) as b:
        dx, dt = b.alloc(rows * ld * 2), b.alloc(rows * ld * 2)
        for r in (0, 1, 150, rows - 1):
            dev.upload(dx + r * ld * 2, np.ascontiguousarray(x[r]))
        st = dict(in_=ld, residual=ld, total=ld, out=ld, scale=5)
        N.check(K.reduce_norm(dt, [dx], None, rows, cols, N.DT_BF16, eps=EPS, strides=st))
        dev.sync()
        for r in (0, 1, 150, rows - 1):
            f = R.codes_to_f64(x[r:r + 1], N.DT_BF16)
            s, y, mag, q = R.norm([f], None, None, EPS)
            got = R.codes_to_f64(dev.to_host(dt + r * ld * 2, cols, np.uint16), N.DT_BF16)
            assert (np.abs(got - y[0]) <= R.rounding(y[0], N.DT_BF16) * 1.01 + R.norm_bounds(s, y, mag, q, None, 1)[1][0]).all(), r
    rows, cols = (1 << 22) + 1003, 8
    x = R.normal(N.DT_BF16, (rows, cols), 4)
    with DevBufs(dev) as b:
        dx, dt = b.put(x), b.alloc(rows * cols * 2)
        N.check(K.reduce_norm(dt, [dx], None, rows, cols, N.DT_BF16, eps=EPS))
        dev.sync()
        got = R.codes_to_f64(dev.to_host(dt, rows * cols, np.uint16).reshape(rows, cols)[-3000:], N.DT_BF16)
    s, y, mag, q = R.norm([R.codes_to_f64(x[-3000:], N.DT_BF16)], None, None, EPS)
    assert (np.abs(got - y) <= R.rounding(y, N.DT_BF16) * 1.01 + R.norm_bounds(s, y, mag, q, None, 1)[1]).all()


def test_norm_gradients_on_two_streams_with_a_workspace_each(dev):
    rows, cols, t = 700, 2000, N.DT_BF16
    need = K.reduce_norm_grad_workspace(rows, cols)
    streams = [dev.stream_create() for _ in range(2)]
    with DevBufs(dev) as b:
        sets = []
        for i in range(2):
            x, dy, w = R.normal(t, (rows, cols), 10 + i), R.normal(t, (rows, cols), 20 + i), R.normal(t, (cols,), 30 + i)
            sets.append((b.put(x), b.put(dy), b.put(w), b.alloc(rows * cols * 2), b.alloc(cols * 2), b.alloc(need)))
        dev.sync()
        call = lambda s, raw: N.check(K.reduce_norm_grad(s[3], s[4], s[1], s[0], s[2], rows, cols, t, s[5], need, eps=EPS, stream=raw))  # noqa: E731
        read = lambda s: (dev.to_host(s[3], rows * cols, np.uint16), dev.to_host(s[4], cols, np.uint16))  # noqa: E731
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


@pytest.mark.parametrize("rows,most,cols,widest", [(256, 300, 8192, 8192), (256, 257, 5003, 5003), (512, 512, 16384, 16385),
                                                   (1000, 1029, 700, 700), (64, 70, 20000, 33000), (3, 5000, 100, 40000)])
def test_norm_gradients_in_the_workspace_of_a_larger_call(dev, rows, most, cols, widest):
    t, need = N.DT_BF16, K.reduce_norm_grad_workspace(most, widest)
    x, dy, w = R.normal(t, (rows, cols), 1, 2.0), R.normal(t, (rows, cols), 2), R.normal(t, (cols,), 3)
    with DevBufs(dev) as b:
        ws = b.put(np.full(need + 64, 0xEE, np.uint8))
        dx, dw = b.alloc(rows * cols * 2), b.alloc(cols * 2)
        N.check(K.reduce_norm_grad(dx, dw, b.put(dy), b.put(x), b.put(w), rows, cols, t, ws, need, eps=EPS), "fx_reduce_norm_grad")
        dev.sync()
        gx = R.codes_to_f64(dev.to_host(dx, rows * cols, np.uint16).reshape(rows, cols), t)
        gw = R.codes_to_f64(dev.to_host(dw, cols, np.uint16), t)
        assert (dev.to_host(ws, need + 64, np.uint8)[need:] == 0xEE).all()
    f = lambda a: R.codes_to_f64(a, t)  # noqa: E731
    edx, edw, bx, bw = R.norm_grad(f(dy), f(x), f(w), None, EPS)
    assert (np.abs(gx - edx) <= R.rounding(edx, t) * 1.01 + bx).all() and (np.abs(gw - edw) <= R.rounding(edw, t) * 1.01 + bw).all()


# Rows enough for results of more than 32 MiB (streamed), in each way that a row is held: one or two octets to a lane of a
# wavefront, two or four to a lane of a workgroup.
@pytest.mark.parametrize("name,rows,cols", [("bf16", 23000, 500), ("fp16", 12000, 1000), ("bf16", 2900, 4003), ("bf16", 1400, 8192),
                                            ("fp16", 700, 16500), ("fp32", 450, 16000), ("fp32", 300, 32001)])
def test_norm_of_large_calls(dev, name, rows, cols):
    print(name, rows, cols, flush=True)
    t = TYPES[name]
    assert rows * cols * (N.DTYPE_SIZE[t] + 1) > 32 << 20
    run_norm(dev, t, rows, cols, 2, quant=True, seed=cols)
    run_norm(dev, t, rows, cols, 1, seed=cols, alias="total=residual")


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", [5003, 8192, 8200, 16384])
def test_norm_gradients_of_several_rows_a_workgroup(dev, name, cols):
    """Wide rows, more of them than workgroups: the next row loaded ahead or not, the sums of two rows in turn."""
    print(name, cols, flush=True)
    run_grad(dev, TYPES[name], 600, cols, seed=cols)


# More than 128 MiB read and written (streamed), in each way that a row is held.
@pytest.mark.parametrize("name,rows,cols,alias", [("bf16", 34000, 500, None), ("fp16", 17500, 1000, "dy"), ("bf16", 4200, 4096, "dtotal"),
                                                  ("bf16", 2200, 8000, "dy"), ("fp16", 1100, 16000, "dtotal"), ("fp32", 530, 16384, "dy"),
                                                  ("fp32", 4300, 2001, None)])
def test_norm_gradients_of_large_calls(dev, name, rows, cols, alias):
    print(name, rows, cols, alias, flush=True)
    t = TYPES[name]
    assert rows * cols * N.DTYPE_SIZE[t] * 4 > 128 << 20
    run_grad(dev, t, rows, cols, alias=alias, seed=cols)
