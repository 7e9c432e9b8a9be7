"""The operators behind the collectives without a GPU: what they refuse, what they
accept as nothing to do, and the gradients' formulas against differences."""
import argparse
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

from flagcx_amd import _native as N
from flagcx_amd import kernels as K
from flagcx_amd import perf
from tests import model_ref as R

P = 0x1000
OK, BAD, NOT = N.SUCCESS, N.INVALID_ARGUMENT, N.NOT_SUPPORTED


def norm(**kw):
    a = dict(out=P, ins=[P, P], weight=P, rows=4, cols=256, dtype=N.DT_BF16, eps=1e-6, residual=P, total=2 * P)
    a.update(kw)
    return K.reduce_norm(**a)


def test_norm_refusals():
    assert norm(dtype=N.DT_FP64) == NOT and norm(dtype=N.DT_INT32) == NOT and norm(dtype=N.DT_E4M3) == NOT
    assert norm(dtype=10) == BAD and norm(dtype=-1) == BAD and norm(out_dtype=11) == BAD and norm(weight_dtype=77) == BAD
    assert norm(out_dtype=N.DT_FP16) == NOT and norm(weight_dtype=N.DT_FP16) == NOT and norm(out_dtype=N.DT_FP32) == NOT
    assert norm(ins=[]) == BAD and norm(ins=[P] * 65) == BAD and norm(ins=[P, None]) == BAD and norm(ins=[P + 1, P]) == BAD
    assert norm(out=None) == BAD and norm(out=P + 1) == BAD and norm(total=P + 1) == BAD and norm(residual=P + 1) == BAD
    assert norm(weight=P + 1) == BAD and norm(weight=P + 2, weight_dtype=N.DT_FP32) == BAD
    assert norm(eps=-1.0) == BAD and norm(eps=float("nan")) == BAD
    assert norm(out_dtype=N.DT_E4M3) == BAD                       # no scale
    assert norm(scale=P) == BAD                                   # a scale nobody writes
    assert norm(out_dtype=N.DT_E4M3, scale=P + 2) == BAD
    wide = dict(in_=256, residual=256, total=256, out=256, scale=2)
    for name in ("in_", "residual", "total", "out"):
        assert norm(strides={**wide, name: 255}) == BAD
    assert norm(out_dtype=N.DT_E4M3, scale=P, strides={**wide, "scale": 1}) == BAD
    assert norm(rows=1 << 31) == BAD and norm(cols=1 << 31) == BAD
    assert norm(rows=0, out=None, ins=[None]) == OK and norm(cols=0, out=None) == OK
    assert norm(total=P, out=P) == BAD and norm(total=P, out=P, ins=[P]) == BAD   # one buffer for two results


def grad(**kw):
    a = dict(dx=P, dweight=P, dy=P, x=P, weight=P, rows=4, cols=256, dtype=N.DT_BF16, workspace=P, workspace_bytes=1 << 20,
             eps=1e-6, dtotal=P)
    a.update(kw)
    return K.reduce_norm_grad(**a)


def test_norm_gradient_refusals():
    assert grad(dtype=N.DT_INT8) == NOT and grad(dtype=99) == BAD and grad(weight_dtype=N.DT_FP16) == NOT
    assert grad(dy=None) == BAD and grad(x=P + 1) == BAD and grad(dx=P + 1) == BAD and grad(dtotal=P + 1) == BAD
    assert grad(weight=P + 1) == BAD and grad(dweight=P + 1) == BAD and grad(eps=-1e-9) == BAD
    need = K.reduce_norm_grad_workspace(4, 256)
    assert need > 0 and grad(workspace=None) == BAD and grad(workspace_bytes=need - 1) == BAD and grad(workspace=P + 8) == BAD
    rows = dict(dy=256, x=256, dtotal=256, dx=256)
    for name in rows:
        assert grad(strides={**rows, name: 255}) == BAD
    assert grad(rows=1 << 31) == BAD and grad(cols=(1 << 28) + 1, strides=None, workspace_bytes=1 << 50) == BAD
    assert K.reduce_norm_grad_workspace(1, (1 << 28) + 1) == 0 and K.reduce_norm_grad_workspace(1, 1 << 28) > 0
    assert grad(dx=None, dweight=None, dy=None) == OK and grad(cols=0) == OK
    assert grad(rows=0, dweight=None, dy=None, x=None) == OK
    assert K.reduce_norm_grad_workspace(0, 256) == 0 and K.reduce_norm_grad_workspace(5, 0) == 0


def test_norm_gradient_workspace_of_the_largest_call_serves_all():
    """Never less for more rows or columns, and a call of fewer rows accepts what was sized for more."""
    rows = list(range(1, 530)) + [700, 1023, 1024, 1025, 1029, 4095, 4096, 4097, 100000]
    cols = [1, 31, 32, 33, 500, 1023, 1024, 1025, 1056, 4096, 8192, 8200, 16352, 16383, 16384, 16385, 16416, 17000, 40000, 65537]
    need = [[K.reduce_norm_grad_workspace(r, c) for c in cols] for r in rows]
    for a, b in zip(need, need[1:]):
        assert all(x <= y for x, y in zip(a, b))
    for a in need:
        assert all(x <= y for x, y in zip(a, a[1:]))
    for r, c, most in ((256, 8192, 300), (256, 8192, 257), (1, 16384, 2), (512, 16384, 512), (1000, 700, 1029)):
        have = K.reduce_norm_grad_workspace(most, c + (c == 16384))
        assert have >= K.reduce_norm_grad_workspace(r, c)
    assert grad(rows=256, cols=8192, workspace_bytes=256 * 8192 * 4 - 1) == BAD        # what the call itself uses


def product(**kw):
    a = dict(y=P, x=P, w=P, offsets=P, experts=4, rows=64, n=128, k=256, dtype=N.DT_BF16)
    a.update(kw)
    return K.expert_product(**a)


def test_product_refusals():
    assert product(dtype=N.DT_FP32) == NOT and product(dtype=N.DT_E4M3) == NOT and product(dtype=10) == BAD
    assert product(out_dtype=N.DT_FP16) == NOT and product(out_dtype=-1) == BAD and product(layout=2) == BAD
    assert product(offsets=None) == BAD and product(offsets=P + 2) == BAD
    assert product(y=None) == BAD and product(x=None) == BAD and product(w=P + 1) == BAD
    assert product(y=P + 2, out_dtype=N.DT_FP32) == BAD
    st = dict(x=256, w=256, y=128, expert_w=128 * 256)
    for name, v in (("x", 255), ("w", 255), ("y", 127)):
        assert product(strides={**st, name: v}) == BAD
    assert product(layout=K.W_KN, strides={**st, "w": 127}) == BAD
    assert product(rows=1 << 31) == BAD and product(n=1 << 31) == BAD and product(k=1 << 31) == BAD
    assert product(rows=0, y=None, x=None) == OK and product(n=0, y=None) == OK and product(experts=0, y=None) == OK


def test_products_of_millions_of_experts_are_refused():
    """Row tiles that need 2^32 threads by themselves: 512, 512 and four times 256 threads an expert."""
    assert product(experts=1 << 24, rows=1 << 24) == NOT
    assert K.expert_product_dw(P, P, P, P, 1 << 24, 64, 128, 256, N.DT_BF16) == NOT
    assert K.expert_product_e4m3(P, P, P, P, P, P, 1 << 23, 1 << 23, 128, 300, N.DT_BF16) == NOT


def test_product_dw_refusals():
    def dw(**kw):
        a = dict(dw=P, dy=P, x=P, offsets=P, experts=4, rows=64, n=128, k=256, dtype=N.DT_FP16)
        a.update(kw)
        return K.expert_product_dw(**a)
    assert dw(dtype=N.DT_FP32) == NOT and dw(out_dtype=N.DT_BF16) == NOT and dw(dtype=12) == BAD
    assert dw(offsets=None) == BAD and dw(dw=None) == BAD and dw(dy=None) == BAD and dw(x=P + 1) == BAD
    st = dict(dy=128, x=256, dw=256, expert_dw=128 * 256)
    for name, v in (("dy", 127), ("x", 255), ("dw", 255)):
        assert dw(strides={**st, name: v}) == BAD
    assert dw(rows=1 << 31) == BAD
    assert dw(experts=0, dw=None) == OK and dw(n=0, dw=None) == OK and dw(k=0, dw=None) == OK


def test_product_e4m3_refusals():
    def e(**kw):
        a = dict(y=P, x=P, xscale=P, w=P, wscale=P, offsets=P, experts=4, rows=64, n=128, k=300, out_dtype=N.DT_BF16)
        a.update(kw)
        return K.expert_product_e4m3(**a)
    assert e(out_dtype=N.DT_E4M3) == NOT and e(out_dtype=N.DT_INT8) == NOT and e(out_dtype=50) == BAD
    assert e(offsets=None) == BAD and e(y=P + 1) == BAD and e(x=None) == BAD and e(w=None) == BAD
    assert e(xscale=None) == BAD and e(wscale=P + 2) == BAD
    st = dict(x=300, w=300, y=128, expert_w=128 * 300, xscale=3, wscale=3, expert_wscale=3)
    for name, v in (("x", 299), ("w", 299), ("y", 127), ("xscale", 2), ("wscale", 2)):
        assert e(strides={**st, name: v}) == BAD
    assert e(rows=0, y=None) == OK and e(n=0, y=None) == OK


def test_norm_gradient_formula_against_differences():
    rng = np.random.default_rng(5)
    x, w, c, ct = (rng.standard_normal(s) for s in ((3, 17), (17,), (3, 17), (3, 17)))
    eps = 1e-3
    f = lambda x, w: float(np.sum(c * R.norm([x], None, w, eps)[1]) + np.sum(ct * x))  # noqa: E731
    dx, dw, _, _ = R.norm_grad(c, x, w, ct, eps)
    h = 1e-6
    for r, q in ((0, 0), (1, 8), (2, 16)):
        d = np.zeros_like(x)
        d[r, q] = h
        assert abs((f(x + d, w) - f(x - d, w)) / (2 * h) - dx[r, q]) < 1e-7
    for q in (0, 9):
        d = np.zeros_like(w)
        d[q] = h
        assert abs((f(x, w + d) - f(x, w - d)) / (2 * h) - dw[q]) < 1e-7


def test_product_gradient_formula_against_differences():
    rng = np.random.default_rng(6)
    x, w, c, o = rng.standard_normal((7, 5)), rng.standard_normal((3, 4, 5)), rng.standard_normal((7, 4)), [0, 3, 3, 6]
    f = lambda x, w: float(np.nansum(c * R.product(x, w, o, True)[0]))  # noqa: E731
    dx, dw = R.product(c, w, o, False)[0], R.product_dw(c, x, o)[0]
    h = 1e-6
    for at in ((0, 1), (5, 4)):
        d = np.zeros_like(x)
        d[at] = h
        assert abs((f(x + d, w) - f(x - d, w)) / (2 * h) - dx[at]) < 1e-7
    for at in ((0, 0, 0), (1, 2, 2), (2, 3, 4)):
        d = np.zeros_like(w)
        d[at] = h
        assert abs((f(x, w + d) - f(x, w - d)) / (2 * h) - dw[at]) < 1e-7
    assert not dw[1].any() and np.isnan(dx[6]).all()


def test_e4m3_table():
    assert R.E4M3[0x7e] == 448 and R.E4M3[1] == 2.0 ** -9 and R.E4M3[0x38] == 1 and np.isnan(R.E4M3[0xff])
    codes = np.array([c for c in range(256) if c & 127 != 127], np.uint8)
    assert np.array_equal(R.to_e4m3(R.E4M3[codes]), codes)
    assert R.to_e4m3(np.array([1.0625]))[0] == 0x38 and R.to_e4m3(np.array([1.1875]))[0] == 0x3a       # ties to even


def test_header_is_plain_c(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("no gcc")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "client.c"
    src.write_text(r'''
#include <stddef.h>
#include "flagcx_amd/fx_model.h"
int main(void) {
  size_t need = fx_reduce_norm_grad_workspace(3, 100);
  if (need < 100 * sizeof(float)) return 1;
  if (fx_reduce_norm(NULL, NULL, NULL, NULL, 1, NULL, NULL, 1, 1, NULL, flagcxBfloat16, flagcxBfloat16, flagcxBfloat16, 1e-6f, NULL) != flagcxInvalidArgument) return 2;
  if (fx_expert_product(NULL, NULL, NULL, NULL, 1, 0, 8, 8, FX_WEIGHT_NK, NULL, flagcxFloat16, flagcxFloat32, NULL) != flagcxSuccess) return 3;
  return 0;
}
''')
    exe, libdir = tmp_path / "client", os.path.join(root, "flagcx_amd", "lib")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-pedantic", f"-I{root}/include", str(src), "-o", str(exe),
                    f"-L{libdir}", "-lflagcx-kernels-mi355x", f"-Wl,-rpath,{libdir}", "-Wl,-rpath,/opt/rocm/lib"], check=True)
    subprocess.run([str(exe)], check=True)


def test_assembly_names_the_registers_it_uses():
    """m0 holds the LDS address of a load into LDS: it is an operand of every such statement and is written by none, so that
    the compiler never takes it to hold something else."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flagcx_amd", "csrc")
    loads = 0
    for name in sorted(os.listdir(csrc)):
        if name.endswith((".hip", ".hpp")):
            for text in re.findall(r"asm volatile\((.*?)\);", open(os.path.join(csrc, name)).read(), re.S):
                code, operands = text.split("::", 1) if "::" in text else (text, "")
                assert not re.search(r"\bm0\b", code), (name, text)
                if re.search(r"buffer_load\w* .*\blds\b", code):
                    loads += 1
                    assert '"{m0}"' in operands, (name, text)
    assert loads >= 3


def test_stride_blocks_match_the_header():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "flagcx_amd", "fx_model.h")).read(), flags=re.S)
    for name, cls in (("fxNormStrides", N.NormStrides), ("fxNormGradStrides", N.NormGradStrides), ("fxProductStrides", N.ProductStrides),
                      ("fxProductDwStrides", N.ProductDwStrides), ("fxProductE4m3Strides", N.ProductE4m3Strides)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        fields = re.findall(r"\w+", body.replace("size_t", ""))
        assert [f.rstrip("_") for f, _ in cls._fields_] == fields, name


class Buffers:
    """Stands in for a device: hands out address ranges and answers how much of one is left behind an address."""

    def __init__(self):
        self.at, self.sizes = 1 << 20, {}

    def malloc(self, n):
        p = self.at
        self.sizes[p] = n
        self.at += (n + (1 << 20)) & ~0xfff
        return p

    def upload(self, p, a):
        assert a.nbytes <= self.left(p)

    def to_device(self, a):
        return self.malloc(a.nbytes)

    def left(self, p):
        return next((base + n - p for base, n in self.sizes.items() if base <= p <= base + n), 0)


@pytest.mark.parametrize("cols", [1, 7, 129, 640])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_norm_command_allocates_what_the_calls_write(monkeypatch, capsys, cols, dtype):
    dev, es = Buffers(), 2 if dtype == "bf16" else 4

    class Timer:
        raw = None

        def __init__(self, dev):
            pass

        def both(self, fn, cold):
            fn()
            return 1.0, None

    def forward(out, ins, weight, rows, cols, dt, *, eps, residual, total, stream, scale=None, out_dtype=None):
        n = rows * cols * es
        assert all(dev.left(p) >= n for p in (*ins, residual, total)) and dev.left(weight) >= cols * es
        assert dev.left(out) >= (rows * cols if scale else n)
        assert scale is None or dev.left(scale) >= 4 * rows * -(-cols // 128)
        return OK

    def backward(dx, dw, dy, x, weight, rows, cols, dt, ws, nbytes, *, eps, dtotal, stream):
        assert all(dev.left(p) >= rows * cols * es for p in (dx, dy, x, dtotal)) and dev.left(dw) >= cols * es
        assert dev.left(ws) >= nbytes >= K.reduce_norm_grad_workspace(rows, cols)
        return OK
    monkeypatch.setattr(perf, "Timer", Timer)
    monkeypatch.setattr(perf.K, "reduce_norm", forward)
    monkeypatch.setattr(perf.K, "reduce_norm_grad", backward)
    perf.run_norm(dev, argparse.Namespace(dtype=dtype, k=2, cols=cols, min="3", max="729", factor=3, cold=False))
    assert capsys.readouterr().out.count("GB/s") == 18
