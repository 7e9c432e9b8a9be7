"""Cases, plain forms and exact values of the operators that stand behind this library's collectives in a model:

* ``norm``      the sum of k ranks' partial results, the residual's addition and the root-mean-square norm behind a
                tensor-parallel all-reduce; the norm leaves in the inputs' type or as e4m3 with a scale per 128 columns
* ``normgrad``  its gradients
* ``experts``   matrix products grouped by expert over the ragged rows that an all-to-all delivers
* ``expertgrad`` the gradients of those
* ``block``     the product of e4m3 operands with a scale per 128 columns (activations) and per 128 x 128 (weights),
                plain or grouped by expert

``run`` computes them with elementary torch operations, or, where ``own`` is true, with the library's entry points.
"""
import math

import torch

own = False

GROUP = 128            # columns that share a scale
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TINY = 2.0 ** -126     # the smallest scale
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one generated token behind an all-reduce of eight ranks' partial results; latency counts
        {"name": "norm token", "op": "norm", "rows": 1, "cols": 8192, "k": 8, "type": "bf16", "out": "e4m3", "residual": True},
        # a decoding batch between two layers
        {"name": "norm batch", "op": "norm", "rows": 256, "cols": 5120, "k": 2, "type": "bf16", "out": "same", "residual": True},
        # a long prompt whose norm is handed on in 8 bits
        {"name": "norm prompt", "op": "norm", "rows": 16384, "cols": 8192, "k": 2, "type": "bf16", "out": "e4m3", "residual": True},
        # a training step's backward pass through one norm
        {"name": "normgrad step", "op": "normgrad", "rows": 8192, "cols": 4096, "type": "bf16", "dtotal": True},
        # an odd width and a ragged number of rows, as a narrow tensor-parallel slice leaves them
        {"name": "normgrad odd", "op": "normgrad", "rows": 777, "cols": 5003, "type": "fp16", "dtotal": False},
        # one token sent to eight experts of 64
        {"name": "experts token", "op": "experts", "tokens": 1, "top": 8, "experts": 64, "n": 2048, "k": 4096, "type": "bf16",
         "out": "same", "spare": 8},
        # a ragged batch of odd sizes
        {"name": "experts odd", "op": "experts", "tokens": 765, "top": 2, "experts": 13, "n": 776, "k": 1000, "type": "fp16",
         "out": "fp32", "spare": 0},
        # a prompt's tokens after the all-to-all
        {"name": "experts prompt", "op": "experts", "tokens": 8192, "top": 2, "experts": 16, "n": 4096, "k": 4096, "type": "bf16",
         "out": "same", "spare": 512},
        # a training step's backward pass through the same experts
        {"name": "expertgrad step", "op": "expertgrad", "tokens": 8192, "top": 2, "experts": 16, "n": 2048, "k": 4096,
         "type": "bf16", "spare": 512},
        # a decoding batch through a dense projection held in 8 bits
        {"name": "block batch", "op": "block", "tokens": 16, "top": 1, "experts": 1, "n": 8192, "k": 8192, "out": "bf16"},
        # a prompt through it
        {"name": "block prompt", "op": "block", "tokens": 8192, "top": 1, "experts": 1, "n": 8192, "k": 8192, "out": "bf16"},
        # experts held in 8 bits behind an all-to-all that moved the rows in 8 bits
        {"name": "block experts", "op": "block", "tokens": 4096, "top": 2, "experts": 32, "n": 4096, "k": 4096, "out": "bf16"},
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["norm", "normgrad", "experts", "expertgrad", "block"])
    while True:
        if op == "norm":
            case = {"op": op, "rows": spread(1, 16384), "cols": spread(128, 16384), "k": rng.randint(1, 8),
                    "type": rng.choice(["bf16", "fp16", "fp32"]), "out": rng.choice(["same", "e4m3"]),
                    "residual": rng.random() < 0.7}
            fits = work(case)["bytes"] <= 1.2e9
        elif op == "normgrad":
            case = {"op": op, "rows": spread(1, 16384), "cols": spread(128, 16384), "type": rng.choice(["bf16", "fp16", "fp32"]),
                    "dtotal": rng.random() < 0.5}
            fits = work(case)["bytes"] <= 1.2e9
        else:
            experts = 1 if op == "block" and rng.random() < 0.5 else spread(4, 64)
            case = {"op": op, "tokens": spread(1, 8192), "top": 1 if experts == 1 else rng.randint(1, min(8, experts)),
                    "experts": experts, "n": spread(128, 8192), "k": spread(128, 8192)}
            if rng.random() < 0.7:      # most widths are multiples of 64
                case["n"], case["k"] = max(1, case["n"] // 64) * 64, max(1, case["k"] // 64) * 64
            if op != "block":
                case["type"] = rng.choice(["bf16", "fp16"])
                case["spare"] = rng.choice([0, spread(1, 512)])
            if op != "expertgrad":
                case["out"] = rng.choice(["bf16", "fp32"] if op == "block" else ["same", "fp32"])
            fits = (experts * case["n"] * case["k"] <= 1 << 29 and case["tokens"] * case["top"] <= 32768
                    and case["tokens"] * case["top"] * case["n"] * case["k"] * (2 if op == "expertgrad" else 1) <= 1 << 38)
        if fits:
            return case


def work(case):
    if case["op"] == "norm":
        r, c, es = case["rows"], case["cols"], TYPES[case["type"]].itemsize
        out = r * c + 4 * r * -(-c // GROUP) if case["out"] == "e4m3" else r * c * es
        return {"bytes": r * c * es * (case["k"] + 1 + bool(case["residual"])) + out + c * es, "flops": r * c * (case["k"] + 6)}
    if case["op"] == "normgrad":
        r, c, es = case["rows"], case["cols"], TYPES[case["type"]].itemsize
        return {"bytes": r * c * es * (3 + bool(case["dtotal"])) + 2 * c * es, "flops": 10 * r * c}
    t, e, n, k = case["tokens"] * case["top"], case["experts"], case["n"], case["k"]
    reached = e * (1 - (1 - case["top"] / e) ** case["tokens"])      # experts that get a row, with even routing
    if case["op"] == "experts":
        out = 4 if case["out"] == "fp32" else 2
        return {"bytes": 2 * reached * n * k + 2 * t * k + out * t * n, "flops": 2 * t * n * k}
    if case["op"] == "expertgrad":     # reads w, x, dy, writes dx and every expert's dw
        return {"bytes": 2 * reached * n * k + 2 * e * n * k + 2 * t * (2 * k + n), "flops": 4 * t * n * k}
    out = 4 if case["out"] == "fp32" else 2
    return {"bytes": reached * n * k + t * k + 4 * t * -(-k // GROUP) + out * t * n, "flops": 2 * t * n * k}


# ---------------------------------------------------------------------------------------------------------- inputs

def _quantised(x, rows, cols):
    """x [..., a, b] as e4m3 with one fp32 scale for each rows x cols block."""
    a, b = x.shape[-2:]
    pad = torch.nn.functional.pad(x, (0, -b % cols, 0, -a % rows))
    blocks = pad.unflatten(-1, (-1, cols)).unflatten(-3, (-1, rows))                # [..., A, rows, B, cols]
    scale = (blocks.abs().amax(dim=(-1, -3)) / E4M3_MAX).clamp(min=TINY)
    q = (blocks / scale[..., :, None, :, None]).to(E4M3)
    return q.flatten(-4, -3).flatten(-2, -1)[..., :a, :b].contiguous(), scale.contiguous()


def _routed(case, gen):
    """Offsets of the experts' rows, as routing of `tokens` tokens to their `top` best experts gives them, and the
    longest list as the host knows it."""
    e = case["experts"]
    liking = torch.randn(case["tokens"], e, device="cuda", generator=gen) + 0.5 * torch.randn(e, device="cuda", generator=gen)
    counts = torch.bincount(liking.topk(case["top"], dim=1).indices.flatten(), minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, int(counts.max())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    s = {"case": dict(case)}
    if case["op"] in ("norm", "normgrad"):
        r, c, t = case["rows"], case["cols"], TYPES[case["type"]]
        s["weight"] = (1 + 0.1 * rand(c)).to(t)
        loud = 1 + 20 * (torch.rand(c, device="cuda", generator=gen) < 0.002)         # a few columns are far larger
        if case["op"] == "norm":
            s["parts"] = torch.empty(case["k"], r, c, device="cuda", dtype=t)
            for p in s["parts"]:
                p.copy_(rand(r, c))
            s["residual"] = (rand(r, c) * loud).to(t) if case["residual"] else None
            s["total"] = torch.empty(r, c, device="cuda", dtype=t)
            s["out"] = torch.empty(r, c, device="cuda", dtype=E4M3 if case["out"] == "e4m3" else t)
            s["scale"] = torch.empty(r, -(-c // GROUP), device="cuda") if case["out"] == "e4m3" else None
        else:
            s["x"], s["dy"] = (rand(r, c) * loud).to(t), rand(r, c).to(t)
            s["dtotal"] = rand(r, c).to(t) if case["dtotal"] else None
            s["dx"], s["dweight"] = torch.empty_like(s["x"]), torch.empty_like(s["weight"])
        return s
    e, n, k = case["experts"], case["n"], case["k"]
    s["offsets"], s["longest"] = _routed(case, gen)
    rows = case["tokens"] * case["top"] + case.get("spare", 0)
    if case["op"] == "block":
        s["x"], s["xscale"] = _quantised(rand(rows, k), 1, GROUP)
        s["w"], s["wscale"] = (torch.empty(e, n, k, device="cuda", dtype=E4M3),
                               torch.empty(e, -(-n // GROUP), -(-k // GROUP), device="cuda"))
        for i in range(e):
            s["w"][i], s["wscale"][i] = _quantised(rand(n, k) / math.sqrt(k), GROUP, GROUP)
        s["y"] = torch.zeros(rows, n, device="cuda", dtype=TYPES[case["out"]])
        return s
    t = TYPES[case["type"]]
    s["x"], s["w"] = rand(rows, k).to(t), torch.empty(e, n, k, device="cuda", dtype=t)
    for w in s["w"]:
        w.copy_(rand(n, k) / math.sqrt(k))
    if case["op"] == "experts":
        s["y"] = torch.zeros(rows, n, device="cuda", dtype=torch.float32 if case["out"] == "fp32" else t)
    else:
        s["dy"] = rand(rows, n).to(t)
        s["dx"], s["dw"] = torch.zeros_like(s["x"]), torch.empty_like(s["w"])
    return s


# ----------------------------------------------------------------------------------------------------- one pass

def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _plain_norm(s):
    total = s["parts"].float().sum(0)
    if s["residual"] is not None:
        total = total + s["residual"].float()
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    total = total.to(s["total"].dtype)
    if s["scale"] is None:
        return {"total": total, "out": y.to(s["out"].dtype)}
    c = y.shape[1]
    y = torch.nn.functional.pad(y, (0, -c % GROUP)).unflatten(-1, (-1, GROUP))
    scale = (y.abs().amax(-1) / E4M3_MAX).clamp(min=TINY)
    return {"total": total, "out": (y / scale[..., None]).to(E4M3).flatten(-2)[:, :c].contiguous(), "scale": scale}


def _plain_normgrad(s):
    x, dy, w = s["x"].float(), s["dy"].float(), s["weight"].float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    xh, g = x * r, dy * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdim=True))
    if s["dtotal"] is not None:
        dx = dx + s["dtotal"].float()
    return {"dx": dx.to(s["dx"].dtype), "dweight": (dy * xh).sum(0).to(s["dweight"].dtype)}


def _padded(s, x):
    """Rows [rows, c] as [experts, longest, c] in 32 bits, with zeros behind each expert's last."""
    o = s["offsets"].long()
    at = o[:-1, None] + torch.arange(s["longest"], device="cuda")
    live = at < o[1:, None]
    return torch.where(live[..., None], x.float()[at.clamp(max=x.shape[0] - 1)], torch.zeros((), device="cuda"))


def _unpadded(s, y, dtype):
    """The inverse, for y [experts, longest, c]; rows behind the last expert's stay zero."""
    o = s["offsets"].long()
    row = torch.arange(s["x"].shape[0], device="cuda")
    e = torch.searchsorted(o[1:], row, right=True).clamp(max=o.numel() - 2)
    y = y[e, (row - o[e]).clamp(max=s["longest"] - 1)]
    return torch.where((row < o[-1])[:, None], y, torch.zeros((), device="cuda")).to(dtype)


def _plain_experts(s):
    y = torch.bmm(s["w"].float(), _padded(s, s["x"]).transpose(1, 2).contiguous())       # [experts, n, longest]
    return {"y": _unpadded(s, y.transpose(1, 2), s["y"].dtype)}


def _plain_expertgrad(s):
    dy = _padded(s, s["dy"])
    dx = torch.bmm(dy, s["w"].float())
    dw = torch.bmm(dy.transpose(1, 2).contiguous(), _padded(s, s["x"]))
    return {"dx": _unpadded(s, dx, s["dx"].dtype), "dw": dw.to(s["dw"].dtype)}


def _plain_block(s):
    n, k = s["w"].shape[1:]
    x = s["x"].float() * s["xscale"].repeat_interleave(GROUP, 1)[:, :k]
    w = s["w"].float() * s["wscale"].repeat_interleave(GROUP, 2)[:, :, :k].repeat_interleave(GROUP, 1)[:, :n]
    if w.shape[0] == 1:
        return {"y": (x @ w[0].t()).to(s["y"].dtype)}
    y = torch.bmm(w, _padded(s, x).transpose(1, 2).contiguous())
    return {"y": _unpadded(s, y.transpose(1, 2), s["y"].dtype)}


_plain = {"norm": _plain_norm, "normgrad": _plain_normgrad, "experts": _plain_experts, "expertgrad": _plain_expertgrad,
          "block": _plain_block}


def _code(t):
    from flagcx_amd import comm
    return comm.dtype_code(t.dtype)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_norm(s):
    from flagcx_amd import _native as N
    from flagcx_amd import kernels as K
    r, c = s["total"].shape
    at = s["parts"].data_ptr()
    step = r * c * s["parts"].element_size()
    N.check(K.reduce_norm(s["out"].data_ptr(), [at + p * step for p in range(s["parts"].shape[0])], s["weight"].data_ptr(), r, c,
                          _code(s["total"]), eps=EPS, residual=s["residual"].data_ptr() if s["residual"] is not None else None,
                          total=s["total"].data_ptr(), scale=s["scale"].data_ptr() if s["scale"] is not None else None,
                          out_dtype=N.DT_E4M3 if s["scale"] is not None else None, stream=_stream()), "fx_reduce_norm")
    return {"total": s["total"], "out": s["out"], "scale": s["scale"]}


def _own_normgrad(s):
    from flagcx_amd import _native as N
    from flagcx_amd import kernels as K
    r, c = s["x"].shape
    if "space" not in s:      # the workspace that a training program keeps from step to step
        s["space"] = torch.empty(K.reduce_norm_grad_workspace(r, c), device="cuda", dtype=torch.uint8)
    N.check(K.reduce_norm_grad(s["dx"].data_ptr(), s["dweight"].data_ptr(), s["dy"].data_ptr(), s["x"].data_ptr(),
                               s["weight"].data_ptr(), r, c, _code(s["x"]), s["space"].data_ptr(), s["space"].numel(), eps=EPS,
                               dtotal=s["dtotal"].data_ptr() if s["dtotal"] is not None else None, stream=_stream()),
            "fx_reduce_norm_grad")
    return {"dx": s["dx"], "dweight": s["dweight"]}


def _own_experts(s):
    from flagcx_amd import _native as N
    from flagcx_amd import kernels as K
    e, n, k = s["w"].shape
    N.check(K.expert_product(s["y"].data_ptr(), s["x"].data_ptr(), s["w"].data_ptr(), s["offsets"].data_ptr(), e, s["x"].shape[0],
                             n, k, _code(s["x"]), out_dtype=_code(s["y"]), stream=_stream()), "fx_expert_product")
    return {"y": s["y"]}


def _own_expertgrad(s):
    from flagcx_amd import _native as N
    from flagcx_amd import kernels as K
    e, n, k = s["w"].shape
    rows, t, o, stream = s["x"].shape[0], _code(s["x"]), s["offsets"].data_ptr(), _stream()
    # dx = dy w: the reduction runs over n, and w is held with its k columns contiguous
    N.check(K.expert_product(s["dx"].data_ptr(), s["dy"].data_ptr(), s["w"].data_ptr(), o, e, rows, k, n, t, layout=K.W_KN,
                             stream=stream), "fx_expert_product")
    N.check(K.expert_product_dw(s["dw"].data_ptr(), s["dy"].data_ptr(), s["x"].data_ptr(), o, e, rows, n, k, t, stream=stream),
            "fx_expert_product_dw")
    return {"dx": s["dx"], "dw": s["dw"]}


def _own_block(s):
    from flagcx_amd import _native as N
    from flagcx_amd import kernels as K
    e, n, k = s["w"].shape
    N.check(K.expert_product_e4m3(s["y"].data_ptr(), s["x"].data_ptr(), s["xscale"].data_ptr(), s["w"].data_ptr(),
                                  s["wscale"].data_ptr(), s["offsets"].data_ptr() if e > 1 else None, e, s["x"].shape[0], n, k,
                                  _code(s["y"]), stream=_stream()), "fx_expert_product_e4m3")
    return {"y": s["y"]}


_own = {"norm": _own_norm, "normgrad": _own_normgrad, "experts": _own_experts, "expertgrad": _own_expertgrad, "block": _own_block}


# --------------------------------------------------------------------------------------------- values in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        total = torch.zeros(case["rows"], case["cols"], device="cuda", dtype=torch.float64)
        for p in s["parts"]:
            total += p
        if s["residual"] is not None:
            total += s["residual"]
        y = total / torch.sqrt(torch.sum(total * total, 1, keepdim=True) / case["cols"] + EPS) * s["weight"].double()
        if s["scale"] is None:
            return {"total": total, "out": y}
        scale, q = torch.empty(s["scale"].shape, device="cuda", dtype=torch.float64), torch.empty_like(y)
        for g in range(scale.shape[1]):
            part = y[:, g * GROUP:(g + 1) * GROUP]
            scale[:, g] = torch.clamp(part.abs().max(1).values / E4M3_MAX, min=TINY)
            q[:, g * GROUP:(g + 1) * GROUP] = part / scale[:, g:g + 1]
        return {"total": total, "out": q.to(E4M3).double(), "scale": scale}
    if case["op"] == "normgrad":
        x, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
        m = x.shape[1]
        d = torch.sqrt(torch.sum(x * x, 1, keepdim=True) / m + EPS)
        g = dy * w
        dx = g / d - x * (torch.sum(g * x, 1, keepdim=True) / (m * d ** 3))
        if s["dtotal"] is not None:
            dx += s["dtotal"]
        return {"dx": dx, "dweight": torch.sum(dy * (x / d), 0)}
    at = s["offsets"].tolist()
    if case["op"] == "expertgrad":
        dx, dw = torch.zeros(s["dx"].shape, device="cuda", dtype=torch.float64), torch.zeros(s["dw"].shape, device="cuda", dtype=torch.float64)
        for e, (a, b) in enumerate(zip(at, at[1:])):
            if b > a:
                dy = s["dy"][a:b].double()
                dx[a:b] = dy @ s["w"][e].double()
                dw[e] = dy.t().contiguous() @ s["x"][a:b].double()
        return {"dx": dx, "dw": dw}
    y = torch.zeros(s["y"].shape, device="cuda", dtype=torch.float64)
    for e, (a, b) in enumerate(zip(at, at[1:])):
        x, w = s["x"][a:b].double(), s["w"][e].double()
        if case["op"] == "block":
            for g in range(s["xscale"].shape[1]):
                x[:, g * GROUP:(g + 1) * GROUP] *= s["xscale"][a:b, g:g + 1]
                for h in range(s["wscale"].shape[1]):
                    w[h * GROUP:(h + 1) * GROUP, g * GROUP:(g + 1) * GROUP] *= s["wscale"][e, h, g]
        if b > a:
            y[a:b] = x @ w.t()
    return {"y": y}
