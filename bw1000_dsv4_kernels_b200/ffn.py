"""W8A8 feed-forward blocks on top of the operator module: dense FFNs and the shared expert of an MoE layer.

    W8A8GatedFFN   per_token_quant_int8 -> w8a8_gated -> per_token_quant_int8 -> w8a8_linear (+ bias, + residual)
    W8A8FFN        the same with a plain activation: w8a8_linear (bias, act) in place of w8a8_gated
    NormFFN        add_layernorm_quant in front of either, the normalised residual added to its output

Four launches a forward (the norm writes the first codes itself).  The reference leaves these blocks to its engine
(DSV4_OPERATOR_ANALYSIS.md:37-49).

Training with the int8 weights frozen: `forward(..., keep=True)` returns what `backward` needs, which is the int8 codes
and scales that the GEMMs read anyway (a quarter of what fp32 activations take), and `backward` returns the gradient of
the input and those of the biases and of the norm.  The quantisers are passed straight through; the int8 weights have no
gradient.  Nothing here is an autograd function: the calls are explicit and can be captured into a CUDA graph.
"""
from dataclasses import dataclass
from typing import Optional

import torch


def _ext():
    import bw1000_dsv4_kernels_b200 as pkg
    return pkg.dsv4_native_ext


@dataclass
class FFNSaved:
    """What one forward leaves for its backward pass."""
    q: torch.Tensor       # int8 [M, H], codes of the input
    s: torch.Tensor       # fp32 [M, 1]
    h_q: torch.Tensor     # int8 [M, I], codes of the hidden rows
    h_s: torch.Tensor


@dataclass
class FFNGrads:
    dx: torch.Tensor                      # bf16 [M, H]
    db1: Optional[torch.Tensor]           # fp32, bias of the first projection (gated: gate and up)
    db2: Optional[torch.Tensor]           # fp32 [H]


class W8A8FFN:
    """act(x w1^T + b1) w2^T + b2 [+ residual].  w1 int8 [I, H], w2 int8 [H, I], scales fp32 per row, biases bf16."""

    def __init__(self, w1, s1, w2, s2, b1=None, b2=None, act: str = "gelu"):
        self.w1, self.s1, self.w2, self.s2, self.b1, self.b2, self.act = w1, s1, w2, s2, b1, b2, act
        if w1.shape[0] != self.hidden_rows() or w2.shape[0] != w1.shape[1]:
            raise ValueError(f"{type(self).__name__}: w1 {tuple(w1.shape)} and w2 {tuple(w2.shape)} do not belong together")

    def hidden_rows(self) -> int:
        """rows of the first weight for the width that the second one takes"""
        return self.w2.shape[1]

    def _hidden(self, q, s):
        return _ext().w8a8_linear(q, self.w1, s, self.s1, self.b1, self.act)

    def _hidden_backward(self, dh, saved):
        return _ext().w8a8_linear_backward(dh, saved.q, self.w1, saved.s, self.s1, self.b1, self.act)

    def forward_codes(self, q, s, residual=None, keep: bool = False):
        """Input as int8 codes and scales (of a quantising norm): bf16 [M, H], and FFNSaved with `keep`."""
        ext = _ext()
        h_q, h_s = ext.per_token_quant_int8(self._hidden(q, s))
        out = ext.w8a8_linear(h_q, self.w2, h_s, self.s2, self.b2, "none", residual)
        return (out, FFNSaved(q, s, h_q, h_s)) if keep else out

    def forward(self, x, residual=None, keep: bool = False):
        """x bf16 [M, H] -> bf16 [M, H], plus `residual` (bf16 [M, H], rows may be strided)."""
        q, s = _ext().per_token_quant_int8(x)
        return self.forward_codes(q, s, residual, keep)

    def backward(self, dout, saved: FFNSaved) -> FFNGrads:
        """dout bf16 [M, H]: gradients of the input and of the biases.  That of the residual is dout itself."""
        dh, db2 = _ext().w8a8_linear_backward(dout, saved.h_q, self.w2, saved.h_s, self.s2, self.b2, "none")
        dx, db1 = self._hidden_backward(dh, saved)
        return FFNGrads(dx, db1, db2)


class W8A8GatedFFN(W8A8FFN):
    """(act(x wg^T + bg) * (x wu^T + bu)) w2^T + b2 [+ residual].  w13 int8 [2 I, H], the gate rows first."""

    def __init__(self, w13, s13, w2, s2, b13=None, b2=None, act: str = "silu"):
        super().__init__(w13, s13, w2, s2, b13, b2, act)

    def hidden_rows(self) -> int:
        return 2 * self.w2.shape[1]

    def _hidden(self, q, s):
        return _ext().w8a8_gated(q, self.w1, s, self.s1, self.b1, self.act)

    def _hidden_backward(self, dh, saved):
        return _ext().w8a8_gated_backward(dh, saved.q, self.w1, saved.s, self.s1, self.b1, self.act)


@dataclass
class NormFFNSaved:
    ffn: FFNSaved
    res: torch.Tensor     # the updated residual: must not change before the backward pass has run
    mean: torch.Tensor
    rstd: torch.Tensor


@dataclass
class NormFFNGrads:
    dx: torch.Tensor      # of the block's input and equally of the residual that it was added to
    dgamma: torch.Tensor  # fp32 [H]
    dbeta: torch.Tensor
    db1: Optional[torch.Tensor]
    db2: Optional[torch.Tensor]


class NormFFN:
    """res <- res + x;  out = res + ffn(layernorm(res)): the second half of a pre-norm transformer layer."""

    def __init__(self, gamma, beta, ffn: W8A8FFN, eps: float = 1e-6):
        self.gamma, self.beta, self.ffn, self.eps = gamma, beta, ffn, eps

    def forward(self, res, x, keep: bool = False):
        """res bf16 [M, H] is updated in place; -> bf16 [M, H], and NormFFNSaved with `keep`."""
        q, s, mean, rstd = _ext().add_layernorm_quant(res, x, self.gamma, self.beta, self.eps)
        if not keep:
            return self.ffn.forward_codes(q, s, res)
        out, saved = self.ffn.forward_codes(q, s, res, keep=True)
        return out, NormFFNSaved(saved, res, mean, rstd)

    def backward(self, dout, saved: NormFFNSaved) -> NormFFNGrads:
        """dout bf16 [M, H], dense (it is also the gradient that reaches the residual past the norm)."""
        g = self.ffn.backward(dout, saved.ffn)
        dx, dgamma, dbeta = _ext().layernorm_backward(g.dx, saved.res, saved.mean, saved.rstd, self.gamma, dout)
        return NormFFNGrads(dx, dgamma, dbeta, g.db1, g.db2)
