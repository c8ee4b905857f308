"""64-bit restatements of the fused linear, gated projection and layer norm with their gradients, written out by hand
(no autograd), and the inputs that their tests share.  tests/test_ffn_cpu.py pins them against differences."""
import math

import torch

from tests import workloads as wl

ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
GATED_ACTS = ("silu", "gelu", "gelu_tanh", "relu")
U32 = 2.0 ** -24   # half a step of fp32, relative
UBF = 2.0 ** -8    # half a step of bf16, relative


def act(z, name):
    if name == "relu":
        return z * (z > 0)
    if name == "gelu":
        return 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def dact(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1.0 + th) + 0.5 * z * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = torch.sigmoid(z)
        return p + z * p * (1.0 - p)
    return torch.ones_like(z)


def project(a, sa, w, sw, b):
    """z and the magnitude that its fp32 rounding errors scale with"""
    acc = a.double() @ w.double().T   # exact: |acc| < 2^53
    z = acc * sa.double().reshape(-1, 1) * sw.double()
    size = z.abs()
    if b is not None:
        z = z + b.double()
        size = size + b.double().abs()
    return z, size


def linear(a, sa, w, sw, b=None, name="none", r=None):
    z, size = project(a, sa, w, sw, b)
    y = act(z, name)
    return y if r is None else y + r.double(), size


def linear_backward(dy, a, sa, w, sw, b=None, name="none"):
    """dx, db, and the fp32 gradient rows scaled by sw (dz * sw)"""
    z, _ = project(a, sa, w, sw, b)
    dz = dy.double() * dact(z, name)
    t = dz * sw.double()
    return t @ w.double(), dz.sum(0), t, dz


def gated(a, sa, w, sw, b=None, name="silu"):
    z, size = project(a, sa, w, sw, b)
    i = w.shape[0] // 2
    return act(z[:, :i], name) * z[:, i:], (size[:, :i], size[:, i:], z[:, :i], z[:, i:])


def gated_backward(dh, a, sa, w, sw, b=None, name="silu"):
    z, _ = project(a, sa, w, sw, b)
    i = w.shape[0] // 2
    g, u, dh = z[:, :i], z[:, i:], dh.double()
    dz = torch.cat([dh * u * dact(g, name), dh * act(g, name)], 1)
    t = dz * sw.double()
    return t @ w.double(), dz.sum(0), t, dz


def layernorm(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return d * rstd * w.double() + b.double(), mean.squeeze(-1), rstd.squeeze(-1)


def layernorm_backward(dy, x, mean, rstd, w, dres=None):
    dy, x, rstd = dy.double(), x.double(), rstd.double().unsqueeze(-1)
    xh = (x - mean.double().unsqueeze(-1)) * rstd
    t = dy * w.double()
    dx = rstd * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True))
    if dres is not None:
        dx = dx + dres.double()
    return dx, (dy * xh).sum(0), dy.sum(0)


def tokens(m, k, seed):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    return a, torch.rand((m, 1), generator=g) * 0.02 + 0.005


def weight(n, k, seed):
    """codes in -127..127 and scales that give projections of about unit size for tokens() above"""
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    return w, (torch.rand(n, generator=g) + 0.5) / (73.0 * 73.0 * 0.015 * math.sqrt(k))


def bf16(shape, seed, scale=1.0):
    return (wl.randn_bf16(shape, seed=seed).float() * scale).to(torch.bfloat16)
