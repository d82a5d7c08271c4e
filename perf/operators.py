"""Performance cases of the products with epilogues and of the grouped products.

Five operators of the GEMM library and their plain forms:

  fused      C = act(A*B + bias) + residual, with Z = A*B + bias kept for the backward pass
  gradient   C = (A*B) .* act'(Z) and the bias gradient, the column sums of C
  grouped    rows [offsets[e], offsets[e+1]) of A times the matrix of expert e, same epilogues
  wgrad      C_e = A_e^T * B_e, the weight gradients of the experts (ragged contraction)
  backward   dZ = dY .* act'(Z) and the bias gradient, where no product precedes

`own` false: elementary torch operations in 32 bits; `own` true: the library's calls.
"""
import math

import torch

own = False

TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ELEM = {"f16": 2, "bf16": 2, "f32": 4}
GELU_C0 = 2.0 * math.sqrt(2.0 / math.pi)
GELU_C1 = 0.044715 * GELU_C0


def listed():
    return [
        # one decoding step of 16 sequences through an output projection, weights stored N x K
        dict(name="fused decode 16", kind="fused", m=16, n=8192, k=8192, dt="bf16", out="bf16", act="none", bias=True, residual=True, preact=False, lb=1),
        # a short prompt through a small layer with sizes that no tile divides, f32 output
        dict(name="fused ragged f32", kind="fused", m=333, n=1000, k=2056, dt="f16", out="f32", act="gelu", bias=True, residual=True, preact=False, lb=0),
        # training forward of the wide projection, keeping Z
        dict(name="fused train large", kind="fused", m=8192, n=28672, k=8192, dt="bf16", out="bf16", act="gelu_tanh", bias=True, residual=False, preact=True, lb=1),
        # backward of a block: gradient of the hidden layer through the second projection
        dict(name="gradient train", kind="gradient", m=4096, n=5120, k=5120, dt="bf16", out="bf16", act="gelu_tanh", bias=True, lb=0),
        # the same for a small layer, ragged sizes
        dict(name="gradient ragged", kind="gradient", m=129, n=520, k=1032, dt="f16", out="f16", act="silu", bias=True, lb=1),
        # one decoding step over experts: four rows an expert, every expert's weights are read
        dict(name="grouped decode", kind="grouped", m=64, n=14336, k=4096, e=16, dt="bf16", out="bf16", act="silu", bias=False, preact=False, grad=False, lb=1),
        # training forward over experts, keeping Z
        dict(name="grouped train", kind="grouped", m=16384, n=4096, k=2048, e=32, dt="bf16", out="bf16", act="silu", bias=True, preact=True, grad=False, lb=0),
        # backward over experts: gradient of the hidden layer, bias gradients per expert
        dict(name="grouped gradient", kind="grouped", m=8191, n=2048, k=4096, e=16, dt="bf16", out="bf16", act="gelu_tanh", bias=True, preact=False, grad=True, lb=1),
        # weight gradients of the experts in f32, as an optimizer with f32 state takes them
        dict(name="wgrad train f32", kind="wgrad", m=16384, n=4096, k=2048, e=32, dt="bf16", out="f32", lc=0),
        # small experts with few rows each
        dict(name="wgrad small", kind="wgrad", m=1000, n=1024, k=512, e=8, dt="f16", out="f16", lc=1),
        # backward through the activation of the wide layer
        dict(name="backward large", kind="backward", m=8192, n=28672, dt="bf16", act="gelu", bias=True),
        # the same for a small one
        dict(name="backward small", kind="backward", m=333, n=1000, dt="f32", act="silu", bias=True),
    ]


def _log(rng, lo, hi, step=1):
    v = int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))
    return max(lo, min(hi, v)) // step * step or step


def draw(rng):
    kind = rng.choice(["fused", "fused", "gradient", "grouped", "grouped", "wgrad", "backward"])
    dt = rng.choice(["bf16", "bf16", "f16"])
    out = rng.choice([dt, dt, "f32"])
    act = rng.choice(["none", "relu", "silu", "gelu_tanh", "gelu"])
    # most layers are multiples of 64 wide, some of 8, a few of nothing
    step = rng.choice([64, 64, 64, 8, 8, 1])
    top = 8192 if step > 1 else 2048
    n, k, m = _log(rng, 256, top, step), _log(rng, 256, top, step), _log(rng, 1, top)
    flag = lambda: rng.random() < 0.5  # noqa: E731
    if kind == "fused":
        return dict(kind=kind, m=m, n=n, k=k, dt=dt, out=out, act=act, bias=flag(), residual=flag(), preact=flag(), lb=rng.randrange(2))
    if kind == "gradient":
        return dict(kind=kind, m=m, n=n, k=k, dt=dt, out=out, act=act, bias=flag(), lb=rng.randrange(2))
    if kind == "backward":
        return dict(kind=kind, m=m, n=n, dt=out, act=act, bias=flag())
    e = _log(rng, 2, 64 if step > 1 else 16)
    n, k = min(n, 4096), min(k, 4096)
    if kind == "wgrad":
        return dict(kind=kind, m=m, n=n, k=k, e=e, dt=dt, out=out, lc=rng.randrange(2))
    grad = flag()
    return dict(kind=kind, m=m, n=n, k=k, e=e, dt=dt, out=out, act=act, bias=flag(), preact=flag() and not grad, grad=grad, lb=rng.randrange(2))


def _counts(m, e, seed):
    """Rows per expert: a skewed routing in which one expert gets none."""
    g = torch.Generator().manual_seed(seed)
    p = torch.exp(0.7 * torch.randn(e, generator=g))
    p[int(torch.randint(e, (1,), generator=g))] = 0.0
    return torch.bincount(torch.multinomial(p, m, replacement=True, generator=g), minlength=e)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, n, kind = case["m"], case["n"], case["kind"]
    dt, out = TORCH[case["dt"]], TORCH[case.get("out", case["dt"])]

    def rnd(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    s = {"case": case}
    e = case.get("e", 0)
    if e:
        counts = _counts(m, e, seed)
        ends = torch.cumsum(counts, 0)
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int32).cuda()
        s["counts"] = counts.tolist()
        # where each row stands when every expert has room for the largest group (the plain form's layout)
        owner = torch.repeat_interleave(torch.arange(e), counts)
        s["room"] = int(counts.max())
        s["place"] = (owner * s["room"] + torch.arange(m) - (ends - counts)[owner]).cuda()
        s["owner"] = owner.cuda()
    if kind == "backward":
        s["dy"], s["z"] = rnd(m, n), rnd(m, n)
        s["dz"] = torch.empty(m, n, device="cuda", dtype=dt)
        s["bias_grad"] = torch.empty(n, device="cuda") if case["bias"] else None
    elif kind == "wgrad":
        k = case["k"]
        s["a"], s["b"] = rnd(m, k), rnd(m, n)
        s["c"] = torch.empty((e, n, k) if case["lc"] else (e, k, n), device="cuda", dtype=out)
    else:
        k = case["k"]
        grad = kind == "gradient" or case.get("grad", False)
        lead = (e,) if e else ()
        s["a"] = rnd(m, k)
        s["w"] = rnd(*lead, *((n, k) if case["lb"] else (k, n)), scale=k ** -0.5)
        s["c"] = torch.empty(m, n, device="cuda", dtype=out)
        s["bias"] = rnd(*lead, n, scale=0.1, dtype=out) if case["bias"] and not grad else None
        s["residual"] = rnd(m, n, dtype=out) if case.get("residual") else None
        s["z"] = rnd(m, n, dtype=out) if grad else torch.empty(m, n, device="cuda", dtype=out) if case["preact"] else None
        s["bias_grad"] = torch.empty(*lead, n, device="cuda") if grad and case["bias"] else None
    if own:
        import rocm_wmma_gemm_b200 as g
        s["loader"] = g.loader()
    return s


def _act(x, act):
    if act == "relu":
        return x * (x > 0)
    if act == "silu":
        return x / (1 + torch.exp(-x))
    if act == "gelu_tanh":
        return x / (1 + torch.exp(-x * (GELU_C0 + GELU_C1 * x * x)))
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x


def _act_grad(x, act):
    if act == "relu":
        return (x > 0).to(x.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    if act == "gelu_tanh":
        s = 1 / (1 + torch.exp(-x * (GELU_C0 + GELU_C1 * x * x)))
        return s * (1 + x * (1 - s) * (GELU_C0 + 3 * GELU_C1 * x * x))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (0.5 / math.pi) ** 0.5
    return torch.ones_like(x)


def _spread(s, x):
    """Rows sorted by expert -> [experts, room, width], zero where an expert has fewer rows."""
    e = s["case"]["e"]
    return x.new_zeros(e * s["room"], x.shape[1]).index_copy_(0, s["place"], x).view(e, s["room"], x.shape[1])


def _plain(s):
    c = s["case"]
    kind, out = c["kind"], TORCH[c.get("out", c["dt"])]
    if kind == "backward":
        dz = s["dy"].float() * _act_grad(s["z"].float(), c["act"])
        return [dz.to(out)] + ([dz.sum(0)] if c["bias"] else [])
    if kind == "wgrad":
        a, b = _spread(s, s["a"].float()), _spread(s, s["b"].float())
        return (torch.matmul(b.transpose(1, 2), a) if c["lc"] else torch.matmul(a.transpose(1, 2), b)).to(out)
    w = s["w"].float()
    w = w.transpose(-1, -2) if c["lb"] else w
    if kind == "grouped":
        x = torch.matmul(_spread(s, s["a"].float()), w).view(-1, c["n"])[s["place"]]
        bias = s["bias"].float()[s["owner"]] if s["bias"] is not None else None
    else:
        x = torch.matmul(s["a"].float(), w)
        bias = s["bias"].float() if s["bias"] is not None else None
    if kind == "gradient" or c.get("grad"):
        x = x * _act_grad(s["z"].float(), c["act"])
        if s["bias_grad"] is None:
            return [x.to(out)]
        return [x.to(out), torch.zeros_like(s["bias_grad"]).index_add_(0, s["owner"], x) if kind == "grouped" else x.sum(0)]
    z = x + bias if bias is not None else x
    y = _act(z, c["act"])
    y = y + s["residual"].float() if s["residual"] is not None else y
    return [y.to(out), z.to(out)] if s["z"] is not None else [y.to(out)]


def _own(s):
    c, L = s["case"], s["loader"]
    kind, m, n = c["kind"], c["m"], c["n"]
    if kind == "backward":
        L.activation_backward(s["dz"], s["dy"], s["z"], m, n, activation=c["act"], bias_grad=s["bias_grad"])
        return [s["dz"], s["bias_grad"]] if c["bias"] else [s["dz"]]
    if kind == "wgrad":
        L.gemm_grouped_wgrad(s["c"], s["a"], s["b"], s["offsets"], m, c["k"], n, c["e"], layout_c=c["lc"])
        return s["c"]
    grad = kind == "gradient" or c.get("grad", False)
    extra = dict(activation=c["act"], bias=s["bias"], residual=s["residual"], preact=s["z"], gradient=grad, bias_grad=s["bias_grad"])
    if kind == "grouped":
        L.gemm_grouped(s["c"], s["a"], s["w"], s["offsets"], m, n, c["k"], c["e"], layout_b=c["lb"], **extra)
    else:
        L.gemm_fused(s["c"], s["a"], s["w"], m, n, c["k"], layout_b=c["lb"], **extra)
    if grad:
        return [s["c"], s["bias_grad"]] if s["bias_grad"] is not None else [s["c"]]
    return [s["c"], s["z"]] if s["z"] is not None else [s["c"]]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    m, n, kind = case["m"], case["n"], case["kind"]
    i, o = ELEM[case["dt"]], ELEM[case.get("out", case["dt"])]
    bias_grad = 4 * n * max(1, case.get("e", 1)) if case.get("bias") else 0
    if kind == "backward":
        return {"bytes": 3 * m * n * i + bias_grad, "flops": 0}
    k = case["k"]
    if kind == "wgrad":
        return {"bytes": m * (n + k) * i + case["e"] * n * k * o, "flops": 2 * m * n * k}
    grad = kind == "gradient" or case.get("grad", False)
    weights = min(case["e"] - 1, m) if "e" in case else 1  # one expert gets no rows
    matrices = 1 + (1 if grad or case.get("preact") else 0) + (1 if case.get("residual") else 0)
    vector = bias_grad if grad else (weights * n * o if case["bias"] else 0)
    return {"bytes": (m * k + weights * n * k) * i + matrices * m * n * o + vector, "flops": 2 * m * n * k}


def _exact_act(x, act):
    """Activation and derivative in 64 bits."""
    if act == "relu":
        return torch.clamp(x, min=0), torch.where(x > 0, 1.0, 0.0).double()
    if act == "silu":
        s = torch.sigmoid(x)
        return x * s, s + x * s * (1 - s)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-x / math.sqrt(2))
        return x * p, p + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    return x, torch.ones_like(x)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "backward":
        dz = s["dy"].double() * _exact_act(s["z"].double(), case["act"])[1]
        return [dz, dz.sum(0)] if case["bias"] else [dz]
    starts = [sum(s["counts"][:e]) for e in range(case["e"] + 1)] if "e" in case else [0, case["m"]]
    spans = list(zip(starts[:-1], starts[1:]))
    if kind == "wgrad":
        c = torch.stack([s["a"][p:q].double().T @ s["b"][p:q].double() for p, q in spans])
        return c.transpose(1, 2).contiguous() if case["lc"] else c
    grad = kind == "gradient" or case.get("grad", False)
    ys, zs, sums = [], [], []
    for e, (p, q) in enumerate(spans):
        w = (s["w"][e] if "e" in case else s["w"]).double()
        x = s["a"][p:q].double() @ (w.T if case["lb"] else w)
        if grad:
            y = x * _exact_act(s["z"][p:q].double(), case["act"])[1]
            sums.append(y.sum(0))
        else:
            if s["bias"] is not None:
                x = x + (s["bias"][e] if "e" in case else s["bias"]).double()
            y = _exact_act(x, case["act"])[0]
            if s["residual"] is not None:
                y = y + s["residual"][p:q].double()
        ys.append(y)
        zs.append(x)
    y = torch.cat(ys)
    if grad:
        if s["bias_grad"] is None:
            return [y]
        return [y, torch.stack(sums) if "e" in case else sums[0]]
    return [y, torch.cat(zs)] if s["z"] is not None else [y]
