"""Measured cases of the W8A8 feed-forward operators.

Four groups, each with a plain form (elementary torch operations in 32 bits, rounded once at the end) and the calls
that a user makes of the operator module:

  linear   y  = act(a_deq w_deq^T + bias) + residual, and its gradient through the frozen int8 weight
  gated    h  = act(g) * u with [g, u] = a_deq w13_deq^T + bias, and its gradient
  norm     layer norm with the residual add in front, and its gradient with those of weight and bias
  block    add_layernorm_quant -> gated -> per_token_quant_int8 -> linear with bias and residual

a_deq = a * sa[row], w_deq = w * sb[channel]; a and w are int8 codes.  The gradients are those of the dequantised
activations (the quantiser is passed straight through); the int8 weight itself has none.
"""
import math

import torch

own = False

EPS = 1e-6
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through the down projection of the dense FFN: weight streaming, latency counts
        dict(name="linear decode", op="linear", M=1, N=7168, K=18432, act="none", bias=True, residual=True, wide=False),
        # a prefill chunk through the same projection: bias and residual stream beside a full tensor-core load
        dict(name="linear prefill", op="linear", M=2048, N=7168, K=18432, act="none", bias=True, residual=True, wide=True),
        # fine-tuning step of a biased GELU projection over a frozen int8 weight
        dict(name="linear backward", op="linear_bwd", M=2048, N=4096, K=7168, act="gelu", bias=True, wide=False),
        # a decode batch through the gate/up projections of a shared expert
        dict(name="gated decode", op="gated", M=16, I=2048, K=7168, act="silu", bias=False),
        # a prefill chunk through the gate/up projections of the dense FFN
        dict(name="gated prefill", op="gated", M=2048, I=18432, K=7168, act="silu", bias=False),
        # fine-tuning step of the shared expert's first half
        dict(name="gated backward", op="gated_bwd", M=4096, I=2048, K=7168, act="silu", bias=False, wide=False),
        # the same with nothing a multiple of a tile: a packed batch of ragged prompts, biased GEGLU
        dict(name="gated backward ragged", op="gated_bwd", M=333, I=1001, K=1040, act="gelu_tanh", bias=True, wide=True),
        # the norm in front of a projection, a prefill chunk
        dict(name="norm prefill", op="norm", M=8192, K=7168, add=True),
        # the norm of a few tokens with a width that is no multiple of a vector
        dict(name="norm few odd", op="norm", M=7, K=1001, add=False),
        # its gradient over a training batch, weight and bias gradients summed over all tokens
        dict(name="norm backward", op="norm_bwd", M=8192, K=7168, add=True),
        # the whole block, eight tokens of a decode step
        dict(name="block decode", op="block", M=8, I=2048, K=7168, act="silu"),
        # the whole block, a prefill chunk
        dict(name="block prefill", op="block", M=2048, I=4096, K=7168, act="silu"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_bwd", "gated", "gated", "gated_bwd", "norm", "norm_bwd", "block"])
    if op in ("norm", "norm_bwd"):
        M, K = _log(rng, 1, 16384), _log(rng, 16, 16384)
        if rng.random() < 0.6:
            K = max(8, K // 8 * 8)
        while M * K > 8192 * 7168:
            M = max(1, M // 2)
        return dict(op=op, M=M, K=K, add=rng.random() < 0.6)
    M, N, K = _log(rng, 1, 4096), _log(rng, 48, 18432), max(1, _log(rng, 64, 18432) // 16) * 16
    if rng.random() < 0.6:
        N = max(8, N // 8 * 8)
    width = 1 if op in ("linear", "linear_bwd") else 2
    passes = 1 if op in ("linear", "gated") else 2
    while passes * width * M * N * K > 2048 * 36864 * 7168:
        M = max(1, M // 2)
    act = rng.choice(ACTS) if op in ("linear", "linear_bwd") else rng.choice(("silu", "gelu", "gelu_tanh", "relu"))
    if op == "linear":
        return dict(op=op, M=M, N=N, K=K, act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5, wide=rng.random() < 0.3)
    if op == "linear_bwd":
        return dict(op=op, M=M, N=N, K=K, act=act, bias=rng.random() < 0.5, wide=rng.random() < 0.3)
    if op == "gated":
        return dict(op=op, M=M, I=N, K=K, act=act, bias=rng.random() < 0.3)
    if op == "gated_bwd":
        return dict(op=op, M=M, I=N, K=K, act=act, bias=rng.random() < 0.3, wide=rng.random() < 0.3)
    return dict(op=op, M=M, I=max(16, N // 16 * 16), K=K, act=act)  # the hidden rows feed a GEMM: 16-byte rows


# ---- inputs ------------------------------------------------------------------------------------------------------
class _Maker:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float32)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.g, device="cuda", dtype=torch.float32) * (hi - lo) + lo

    def bf16(self, *shape, scale=1.0):
        return (self.normal(*shape) * scale).to(torch.bfloat16)

    def tokens(self, m, k):
        """Activations as the quantiser leaves them: int8 codes with the row's largest at 127, fp32 [m, 1] scales."""
        x = self.normal(m, k)
        x = torch.where(torch.rand((m, k), generator=self.g, device="cuda") < 0.01, x * 4.0, x)
        amax = x.abs().amax(1, keepdim=True).clamp_min(1e-10)
        return torch.round(x * (127.0 / amax)).to(torch.int8), amax / 127.0

    def weight(self, n, k):
        """int8 weight of about normal codes, channel scales that give projections of unit size."""
        w = (torch.randn((n, k), generator=self.g, device="cuda", dtype=torch.float16) * 36.0).clamp_(-127, 127)
        return w.round_().to(torch.int8), self.uniform(0.5, 1.5, n) / (36.0 * math.sqrt(k))

    def rows(self, m, n, wide):
        """bf16 [m, n], dense or a column slab of a wider buffer."""
        return self.bf16(m, n + 24)[:, :n] if wide else self.bf16(m, n)


def prepare(case, seed):
    mk, op = _Maker(seed), case["op"]
    s = dict(case)
    if op in ("linear", "linear_bwd", "gated", "gated_bwd"):
        n = case["N"] if op.startswith("linear") else 2 * case["I"]
        s["a"], s["sa"] = mk.tokens(case["M"], case["K"])
        s["w"], s["sw"] = mk.weight(n, case["K"])
        s["b"] = mk.bf16(n, scale=0.5) if case["bias"] else None
        if op == "linear":
            s["r"] = mk.rows(case["M"], n, case["wide"]) if case["residual"] else None
        elif op.endswith("bwd"):
            s["dy"] = mk.rows(case["M"], n if op == "linear_bwd" else case["I"], case["wide"])
    elif op in ("norm", "norm_bwd"):
        m, k = case["M"], case["K"]
        s["x"] = mk.normal(m, k).mul_(mk.uniform(0.5, 2.0, m, 1)).add_(mk.uniform(-1.0, 1.0, m, 1)).to(torch.bfloat16)
        s["gamma"], s["beta"] = mk.uniform(0.5, 1.5, k).to(torch.bfloat16), mk.bf16(k, scale=0.1)
        s["other"] = mk.bf16(m, k) if case["add"] else None  # the residual in front, or the gradient that arrives past the norm
        if op == "norm_bwd":
            s["dy"] = mk.bf16(m, k)
            x = s["x"].double()  # the statistics that the forward pass hands on
            s["mean"] = x.mean(1).float()
            s["rstd"] = (x.var(1, unbiased=False) + EPS).rsqrt().float()
    else:
        m, i, k = case["M"], case["I"], case["K"]
        s["x"], s["res"] = mk.bf16(m, k), mk.bf16(m, k)
        s["gamma"], s["beta"] = mk.uniform(0.5, 1.5, k).to(torch.bfloat16), mk.bf16(k, scale=0.1)
        s["w13"], s["s13"] = mk.weight(2 * i, k)
        s["w2"], s["s2"] = mk.weight(k, i)
        s["b2"] = mk.bf16(k, scale=0.1)
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z * _sigmoid(z)
    if act == "gelu":
        return z * (0.5 + 0.5 * torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return z * _sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
    return z


def _dact(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        p = _sigmoid(z)
        return p * (1.0 + z * (1.0 - p))
    if act == "gelu":
        return 0.5 + 0.5 * torch.erf(z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = 2.0 * math.sqrt(2.0 / math.pi)
        p = _sigmoid(c * (z + 0.044715 * z * z * z))
        return p + z * p * (1.0 - p) * c * (1.0 + 3.0 * 0.044715 * z * z)
    return torch.ones_like(z)


def _project(a, sa, w, sw, b):
    z = (a.float() @ w.float().T) * sa.reshape(-1, 1) * sw
    return z if b is None else z + b.float()


def _norm(x, gamma, beta):
    x = x.float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    return d * rstd * gamma.float() + beta.float(), mean.reshape(-1), rstd.reshape(-1)


def _quantise(y):
    amax = y.float().abs().amax(1, keepdim=True).clamp_min(1e-10)
    return torch.round(y.float() * (127.0 / amax)), amax / 127.0


def _plain(s):
    op = s["op"]
    if op == "linear":
        y = _act(_project(s["a"], s["sa"], s["w"], s["sw"], s["b"]), s["act"])
        return (y if s["r"] is None else y + s["r"].float()).to(torch.bfloat16)
    if op == "linear_bwd":
        dz = s["dy"].float()
        if s["act"] != "none":
            dz = dz * _dact(_project(s["a"], s["sa"], s["w"], s["sw"], s["b"]), s["act"])
        dx = ((dz * s["sw"]) @ s["w"].float()).to(torch.bfloat16)
        return [dx] if s["b"] is None else [dx, dz.sum(0)]
    if op == "gated":
        z = _project(s["a"], s["sa"], s["w"], s["sw"], s["b"])
        return (_act(z[:, : s["I"]], s["act"]) * z[:, s["I"]:]).to(torch.bfloat16)
    if op == "gated_bwd":
        z, dh = _project(s["a"], s["sa"], s["w"], s["sw"], s["b"]), s["dy"].float()
        g, u = z[:, : s["I"]], z[:, s["I"]:]
        dz = torch.cat([dh * u * _dact(g, s["act"]), dh * _act(g, s["act"])], 1)
        dx = ((dz * s["sw"]) @ s["w"].float()).to(torch.bfloat16)
        return [dx] if s["b"] is None else [dx, dz.sum(0)]
    if op == "norm":
        if s["other"] is None:
            y, mean, rstd = _norm(s["x"], s["gamma"], s["beta"])
            return [y.to(torch.bfloat16), mean, rstd]
        s["other"].copy_(s["other"].float() + s["x"].float())  # the residual is updated in place
        y, mean, rstd = _norm(s["other"], s["gamma"], s["beta"])
        return [y.to(torch.bfloat16), mean, rstd, s["other"]]
    if op == "norm_bwd":
        dy, rstd = s["dy"].float(), s["rstd"].reshape(-1, 1)
        xhat = (s["x"].float() - s["mean"].reshape(-1, 1)) * rstd
        t = dy * s["gamma"].float()
        dx = (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True)) * rstd
        if s["other"] is not None:
            dx = dx + s["other"].float()
        return [dx.to(torch.bfloat16), (dy * xhat).double().sum(0).float(), dy.double().sum(0).float()]
    s["res"].copy_(s["res"].float() + s["x"].float())
    q, sq = _quantise(_norm(s["res"], s["gamma"], s["beta"])[0])
    z = _project(q, sq, s["w13"], s["s13"], None)
    h = (_act(z[:, : s["I"]], s["act"]) * z[:, s["I"]:]).to(torch.bfloat16)
    q, sq = _quantise(h)
    out = _project(q, sq, s["w2"], s["s2"], s["b2"]) + s["res"].float()
    return [out.to(torch.bfloat16), s["res"]]


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _own(s):
    from bw1000_dsv4_kernels_b200 import dsv4_native_ext as ext
    op = s["op"]
    if op == "linear":
        return ext.w8a8_linear(s["a"], s["w"], s["sa"], s["sw"], s["b"], s["act"], s["r"])
    if op == "linear_bwd":
        dx, db = ext.w8a8_linear_backward(s["dy"], s["a"], s["w"], s["sa"], s["sw"], s["b"], s["act"])
        return [dx] if s["b"] is None else [dx, db]
    if op == "gated":
        return ext.w8a8_gated(s["a"], s["w"], s["sa"], s["sw"], s["b"], s["act"])
    if op == "gated_bwd":
        dx, db = ext.w8a8_gated_backward(s["dy"], s["a"], s["w"], s["sa"], s["sw"], s["b"], s["act"])
        return [dx] if s["b"] is None else [dx, db]
    if op == "norm":
        if s["other"] is None:
            return list(ext.layernorm(s["x"], s["gamma"], s["beta"], EPS))
        return list(ext.add_layernorm(s["other"], s["x"], s["gamma"], s["beta"], EPS)) + [s["other"]]
    if op == "norm_bwd":
        return list(ext.layernorm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"], s["other"]))
    q, sq, _, _ = ext.add_layernorm_quant(s["res"], s["x"], s["gamma"], s["beta"], EPS)
    h = ext.w8a8_gated(q, s["w13"], sq, s["s13"], None, s["act"])
    q, sq = ext.per_token_quant_int8(h)
    return [ext.w8a8_linear(q, s["w2"], sq, s["s2"], s["b2"], "none", s["res"]), s["res"]]


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    if op in ("norm", "norm_bwd"):
        add = 1 if case["add"] else 0
        if op == "norm":  # x in, y out; the residual in and out; gamma, beta; two statistics a row
            return {"bytes": 4 * M * K + add * 4 * M * K + 4 * K + 8 * M, "flops": 8 * M * K}
        return {"bytes": 6 * M * K + add * 2 * M * K + 8 * M + 2 * K + 8 * K, "flops": 14 * M * K}
    if op == "block":
        I = case["I"]
        return {"bytes": 3 * I * K + 4 * (2 * I + K) + 6 * K + 6 * M * K + 2 * M * K, "flops": 6 * M * I * K}
    n = case["N"] if op.startswith("linear") else 2 * case["I"]
    read = n * K + 4 * n + (2 * n if case["bias"] else 0)
    if op == "linear":
        return {"bytes": read + M * K + 4 * M + 2 * M * n * (2 if case["residual"] else 1), "flops": 2 * M * n * K}
    if op == "gated":
        return {"bytes": read + M * K + 4 * M + 2 * M * case["I"], "flops": 2 * M * n * K}
    again = case["act"] != "none"  # the projection has to be computed again for the activation's derivative
    out = 2 * M * K + (4 * n if case["bias"] else 0)
    grad = 2 * M * (n if op == "linear_bwd" else case["I"])
    return {"bytes": read + grad + out + (M * K + 4 * M if again else 0), "flops": (4 if again else 2) * M * n * K}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------
def _act64(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z * (z > 0)
    if act == "silu":
        return z / (1.0 + (-z).exp())
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))


def _codes64(v):
    top = torch.clamp(v.abs().max(1, keepdim=True).values, min=1e-10)
    return torch.round(v * 127.0 / top) * (top / 127.0)


def _ln64(x, gamma, beta):
    mean = x.sum(1, keepdim=True) / x.shape[1]
    var = (x * x).sum(1, keepdim=True) / x.shape[1] - mean * mean
    rstd = (var + EPS) ** -0.5
    return (x - mean) * rstd * gamma + beta, mean[:, 0], rstd[:, 0]


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "norm":
        x = s["x"].double()
        if s["other"] is None:
            return list(_ln64(x, s["gamma"].double(), s["beta"].double()))
        r = (s["other"].double() + x).to(torch.bfloat16).double()  # the residual as it is stored is what is normalised
        return list(_ln64(r, s["gamma"].double(), s["beta"].double())) + [r]
    if op == "norm_bwd":
        x, g = s["x"].double().requires_grad_(), s["gamma"].double().requires_grad_()
        b = torch.zeros_like(g).requires_grad_()
        dx, dg, db = torch.autograd.grad(_ln64(x, g, b)[0], (x, g, b), s["dy"].double())
        return [dx if s["other"] is None else dx + s["other"].double(), dg, db]
    if op == "block":
        r = (s["res"].double() + s["x"].double()).to(torch.bfloat16).double()
        y = _codes64(_ln64(r, s["gamma"].double(), s["beta"].double())[0])
        z = y @ (s["w13"].double() * s["s13"].double()[:, None]).T
        h = (_act64(z[:, : case["I"]], case["act"]) * z[:, case["I"]:]).to(torch.bfloat16).double()
        return [_codes64(h) @ (s["w2"].double() * s["s2"].double()[:, None]).T + s["b2"].double() + r, r]
    x = s["a"].double() * s["sa"].double().reshape(-1, 1)
    w = s["w"].double() * s["sw"].double()[:, None]
    b = torch.zeros(w.shape[0], dtype=torch.float64, device="cuda") if s["b"] is None else s["b"].double()
    grad = op.endswith("bwd")
    if grad:
        x.requires_grad_()
        b.requires_grad_()
    z = x @ w.T + b
    if op.startswith("linear"):
        y = _act64(z, case["act"])
        if not grad:
            return y if s["r"] is None else y + s["r"].double()
    else:
        y = _act64(z[:, : case["I"]], case["act"]) * z[:, case["I"]:]
        if not grad:
            return y
    dx, db = torch.autograd.grad(y, (x, b), s["dy"].double())
    return [dx] if s["b"] is None else [dx, db]
