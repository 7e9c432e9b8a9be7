"""The operators behind the collectives as a layer uses them, over simulated ranks:
the ranks' partial results are summed, normed and handed on in 8 bits, the rows go to
their experts' ranks through an all-to-all-v, are multiplied there, come back, and the
sum goes into the next norm; then the gradients the other way.  Every step is held to
its own bound, from what the step before it left on the GPU."""
import numpy as np
import pytest

from flagcx_amd import _native as N
from flagcx_amd import kernels as K
from flagcx_amd import sim as S
from tests import model_ref as R
from tests.util import DevBufs

pytestmark = pytest.mark.gpu

EPS = 1e-5


def quantised_blocks(w):
    """[n, k] as e4m3 with a scale per 128 x 128."""
    n, k = w.shape
    s = np.zeros((-(-n // 128), -(-k // 128)), np.float32)
    q = np.zeros((n, k), np.uint8)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            part = w[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128]
            s[i, j] = np.abs(part).max() / 448
            q[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128] = R.to_e4m3(np.clip(part / np.float64(s[i, j]), -448, 448))
    return q, s


def test_norm_dispatch_experts_and_back(dev):
    ranks, tokens, h, t = 4, 97, 640, N.DT_BF16
    groups = h // 128
    rng = np.random.default_rng(2)
    stream = dev.stream_create()
    raw = dev.raw_stream(stream)
    with DevBufs(dev) as b, S.SimGroup(ranks) as g:
        # tensor parallel: every rank's partial result, the residual, the norm in 8 bits
        parts = [R.normal(t, (tokens, h), 10 + r) for r in range(ranks)]
        res, w = R.normal(t, (tokens, h), 5, 2.0), R.normal(t, (h,), 6)
        dparts, dres, dwt = [b.put(p) for p in parts], b.put(res), b.put(w)
        dtot, dq, dsc = b.alloc(tokens * h * 2), b.alloc(tokens * h), b.alloc(tokens * groups * 4)
        N.check(K.reduce_norm(dq, dparts, dwt, tokens, h, t, eps=EPS, residual=dres, total=dtot, scale=dsc, out_dtype=N.DT_E4M3,
                              stream=raw))
        dev.stream_sync(stream)
        q, sc = dev.to_host(dq, tokens * h, np.uint8).reshape(tokens, h), dev.to_host(dsc, tokens * groups, np.float32).reshape(tokens, groups)
        f = [R.codes_to_f64(p, t) for p in parts]
        s, y, mag, r = R.norm(f, R.codes_to_f64(res, t), R.codes_to_f64(w, t), EPS)
        dy = R.norm_bounds(s, y, mag, r, R.codes_to_f64(w, t), ranks + 1)[1]
        rows8 = R.E4M3[q] * np.repeat(sc.astype(np.float64), 128, axis=1)
        assert (np.abs(rows8 - y) <= np.maximum(2.0 ** -4 * np.abs(y) * 1.001, 2.0 ** -10 * np.repeat(sc, 128, axis=1) * 1.001)
                + 2 * dy + 8 * R.E * np.abs(y)).all()

        # expert parallel: token i lives on rank i % ranks and goes to rank owner[i]; codes and scales travel as they are
        owner = rng.integers(0, ranks, tokens)
        owner[owner == 2] = 3                                              # rank 2's expert gets nothing
        order = [[i for d in range(ranks) for i in range(tokens) if i % ranks == src and owner[i] == d] for src in range(ranks)]
        counts = np.array([[sum(1 for i in order[src] if owner[i] == d) for d in range(ranks)] for src in range(ranks)])
        excl = lambda c: np.concatenate([[0], np.cumsum(c)[:-1]])  # noqa: E731
        got = counts.sum(axis=0)
        at = [[i for src in range(ranks) for i in order[src] if owner[i] == d] for d in range(ranks)]     # rows as they arrive
        dsend = [b.put(np.concatenate([q[order[src]].ravel(), np.zeros(16, np.uint8)])) for src in range(ranks)]
        dssend = [b.put(np.concatenate([sc[order[src]].ravel(), np.zeros(4, np.float32)])) for src in range(ranks)]
        drecv = [b.alloc(int(got[d]) * h + 64) for d in range(ranks)]
        dsrecv = [b.alloc(int(got[d]) * groups * 4 + 64) for d in range(ranks)]
        for bufs, recvs, per, dt in ((dsend, drecv, h, N.DT_UINT8), (dssend, dsrecv, groups, N.DT_FP32)):
            N.check(g.all_to_allv(bufs, counts * per, [excl(c) * per for c in counts], recvs, counts.T * per,
                                  [excl(c) * per for c in counts.T], dt, stream))
        n = 384
        ws = [quantised_blocks(rng.standard_normal((n, h)) / np.sqrt(h)) for _ in range(ranks)]
        dy8 = []
        for d in range(ranks):
            dw, dws, do = b.put(ws[d][0]), b.put(ws[d][1]), b.put(np.array([0, got[d]], np.int32))
            dy8.append(b.alloc(int(got[d]) * n * 2 + 64))
            N.check(K.expert_product_e4m3(dy8[d], drecv[d], dsrecv[d], dw, dws, do, 1, int(got[d]), n, h, t, stream=raw))
        # and back to where the tokens live
        dback = [b.alloc(len(order[src]) * n * 2 + 64) for src in range(ranks)]
        N.check(g.all_to_allv(dy8, counts.T * n, [excl(c) * n for c in counts.T], dback, counts * n, [excl(c) * n for c in counts], t, stream))
        dev.stream_sync(stream)
        expert = np.full((tokens, n), np.nan)
        for src in range(ranks):
            back = dev.to_host(dback[src], len(order[src]) * n, np.uint16).reshape(-1, n)
            expert[order[src]] = R.codes_to_f64(back, t)
        for d in range(ranks):
            if got[d]:
                fw = R.E4M3[ws[d][0]] * np.repeat(np.repeat(ws[d][1].astype(np.float64), 128, 0), 128, 1)[:n, :h]
                x = rows8[at[d]]
                want, m = x @ fw.T, np.abs(x) @ np.abs(fw).T
                assert R.within(expert[at[d]], want, t, R.sum_bound(128 + groups + 4, m) + 2.0 ** -12 * m), d

        # the same expert in bf16, with its gradients: rows of all tokens sorted by expert
        idx = np.concatenate([np.where(owner == d)[0] for d in range(ranks)])
        o = np.concatenate([[0], np.cumsum(got)]).astype(np.int32)
        xs, wb = R.normal(t, (tokens, h), 60), R.normal(t, (ranks, n, h), 61, 0.05)
        xs = xs[idx]
        dx, dwb, do, dyb = b.put(xs), b.put(wb), b.put(o), b.alloc(tokens * n * 2)
        N.check(K.expert_product(dyb, dx, dwb, do, ranks, tokens, n, h, t, stream=raw))
        dnext, dnw = b.alloc(tokens * n * 2), b.put(R.normal(t, (n,), 62))
        N.check(K.reduce_norm(dnext, [dyb], dnw, tokens, n, t, eps=EPS, stream=raw))
        grad = R.normal(t, (tokens, n), 63)
        need = K.reduce_norm_grad_workspace(tokens, n)
        dgr, dgy, dgw, space = b.put(grad), b.alloc(tokens * n * 2), b.alloc(n * 2), b.alloc(need)
        N.check(K.reduce_norm_grad(dgy, dgw, dgr, dyb, dnw, tokens, n, t, space, need, eps=EPS, stream=raw))
        dgx, ddw = b.alloc(tokens * h * 2), b.alloc(ranks * n * h * 4)
        N.check(K.expert_product(dgx, dgy, dwb, do, ranks, tokens, h, n, t, layout=K.W_KN, stream=raw))
        N.check(K.expert_product_dw(ddw, dgy, dx, do, ranks, tokens, n, h, t, out_dtype=N.DT_FP32, stream=raw))
        dev.stream_sync(stream)
        host = lambda p, *shape: R.codes_to_f64(dev.to_host(p, int(np.prod(shape)), np.uint16).reshape(shape), t)  # noqa: E731
        yb, gy = host(dyb, tokens, n), host(dgy, tokens, n)
        fx, fw = R.codes_to_f64(xs, t), R.codes_to_f64(wb, t)
        want, m = R.product(fx, fw, o, True)
        assert R.within(yb, want, t, R.sum_bound(h, m))
        nw = R.codes_to_f64(R.normal(t, (n,), 62), t)
        s, y, mag, r = R.norm([yb], None, nw, EPS)
        assert R.within(host(dnext, tokens, n), y, t, R.norm_bounds(s, y, mag, r, nw, 1)[1])
        ex, ew, bx, bw = R.norm_grad(R.codes_to_f64(grad, t), yb, nw, None, EPS)
        assert R.within(gy, ex, t, bx) and R.within(host(dgw, n), ew, t, bw)
        want, m = R.product(gy, fw, o, False)
        assert R.within(host(dgx, tokens, h), want, t, R.sum_bound(n, m))
        want, m = R.product_dw(gy, fx, o)
        gw = dev.to_host(ddw, ranks * n * h, np.float32).reshape(ranks, n, h).astype(np.float64)
        assert R.within(gw, want, N.DT_FP32, R.sum_bound(tokens, m)) and not gw[2].any()
    dev.stream_destroy(stream)
