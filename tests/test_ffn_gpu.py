"""The feed-forward blocks end to end: every stage of a forward re-derived in 64 bits from the codes that the stage in
front of it produced, and the whole backward chain from the saved codes.

Tolerances: a stage's output is off by half a bf16 step (2^-8 of each element, 2^-9 in the 2-norm where mantissas are
spread) plus fp32 terms far below that; the backward chain rounds to bf16 after each of its products, so its 2-norm error
is at most the number of roundings times 2^-8."""
import pytest
import torch

from bw1000_dsv4_kernels_b200 import ffn, moe
from oracle import cpu as oracle
from tests import ffn_reference as ref
from tests import workloads as wl

pytestmark = pytest.mark.gpu


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def rel(got, want):
    return float((got.detach().cpu().double() - want).norm() / want.norm())


def make(m, h, i, gated, bias, act):
    (w1, s1), (w2, s2) = ref.weight(2 * i if gated else i, h, 1), ref.weight(h, i, 2)
    # hidden rows are of about unit size: the same scale for the second weight as tokens() of unit size would get
    s1, s2 = s1 * 0.6, s2 * 1.0
    b1, b2 = (ref.bf16((w1.shape[0],), 3, 0.3), ref.bf16((h,), 4, 0.3)) if bias else (None, None)
    cls = ffn.W8A8GatedFFN if gated else ffn.W8A8FFN
    return (w1, s1, w2, s2, b1, b2), cls(*cuda(w1, s1, w2, s2, b1, b2), act)


@pytest.mark.parametrize("m,h,i", [(1, 256, 128), (37, 400, 272), (200, 512, 384), (600, 784, 528)])
@pytest.mark.parametrize("gated,bias,act", [(True, False, "silu"), (True, True, "gelu_tanh"), (False, True, "gelu")])
def test_norm_ffn_forward_and_backward(ext, m, h, i, gated, bias, act):
    (w1, s1, w2, s2, b1, b2), layer = make(m, h, i, gated, bias, act)
    gamma, beta = wl.gamma_bf16(h, seed=5), ref.bf16((h,), 6, 0.2)
    block = ffn.NormFFN(gamma.cuda(), beta.cuda(), layer, 1e-6)
    res, x, dout = ref.bf16((m, h), 7), ref.bf16((m, h), 8), ref.bf16((m, h), 9)
    res_d = res.cuda()
    out, saved = block.forward(res_d, x.cuda(), keep=True)
    assert torch.equal(block.forward(res.cuda(), x.cuda()).view(torch.int16), out.view(torch.int16))

    a = (res.float() + x.float()).to(torch.bfloat16)
    assert torch.equal(res_d.cpu().view(torch.int16), a.view(torch.int16))
    y64, mean64, rstd64 = ref.layernorm(a, gamma, beta, 1e-6)
    q, s, h_q, h_s = (t.cpu() for t in (saved.ffn.q, saved.ffn.s, saved.ffn.h_q, saved.ffn.h_s))
    assert ((q.double() * s.double() - y64).abs() <= 0.501 * s.double()).all()
    h64 = (ref.gated(q, s, w1, s1, b1, act) if gated else ref.linear(q, s, w1, s1, b1, act))[0]
    half = h_s.double() / 2 * 1.01
    assert ((h_q.double() * h_s.double() - h64).abs() <= half + ref.UBF * h64.abs() + 1e-6).all()
    out64 = ref.linear(h_q, h_s, w2, s2, b2, "none", a)[0]
    assert rel(out, out64) <= 2.0 ** -8

    g = block.backward(dout.cuda(), saved)
    dh64, db2, _, _ = ref.linear_backward(dout, h_q, h_s, w2, s2, b2, "none")
    back = ref.gated_backward if gated else ref.linear_backward
    dy64, db1, _, _ = back(dh64, q, s, w1, s1, b1, act)
    dx64, dgamma, dbeta = ref.layernorm_backward(dy64, a, mean64, rstd64, gamma, dout)
    assert rel(g.dx, dx64) <= 3 * ref.UBF
    assert rel(g.dgamma, dgamma) <= 2 * ref.UBF and rel(g.dbeta, dbeta) <= 2 * ref.UBF
    if bias:
        assert rel(g.db2, db2) <= 1e-6 and rel(g.db1, db1) <= ref.UBF
    else:
        assert g.db1 is None and g.db2 is None


def test_block_is_captured_with_its_backward(ext):
    m, h, i = 130, 512, 256
    _, layer = make(m, h, i, True, True, "silu")
    block = ffn.NormFFN(wl.gamma_bf16(h, seed=5).cuda(), ref.bf16((h,), 6).cuda(), layer)
    res0, x, dout = (ref.bf16((m, h), k).cuda() for k in (7, 8, 9))

    def step(res):
        out, saved = block.forward(res, x, keep=True)
        return out, block.backward(dout, saved)
    want_out, want = step(res0.clone())
    torch.cuda.synchronize()
    res = res0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, g = step(res)
    for _ in range(3):
        res.copy_(res0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want_out)
        for name in ("dx", "dgamma", "dbeta", "db1", "db2"):
            assert torch.equal(getattr(g, name), getattr(want, name)), name


def test_moe_layer_with_a_shared_expert(ext):
    t, e, topk, h, i = 40, 8, 2, 256, 128
    w13, w2 = wl.int8_weights((e, 2 * i, h), seed=1), wl.int8_weights((e, h, i), seed=2)
    s13, s2 = wl.channel_scales((e, 2 * i), seed=3), wl.channel_scales((e, h), seed=4)
    args, shared = make(t, h, i, True, False, "silu")
    x = ref.bf16((t, h), 5)
    ids, w = moe.route(torch.randn(t, e).cuda(), topk)
    plain = moe.W8A8MoE(*cuda(w13, s13, w2, s2), e).forward(x.cuda(), ids, w)
    both = moe.W8A8MoE(*cuda(w13, s13, w2, s2), e, shared=shared).forward(x.cuda(), ids, w)
    # the shared expert alone, from the same codes, on top of the routed rows
    q, s = oracle.per_token_quant_int8(x)
    h_q, h_s = ext.per_token_quant_int8(ext.w8a8_gated(*cuda(q, args[0], s, args[1])))
    want = ref.linear(h_q.cpu(), h_s.cpu(), args[2], args[3], None, "none", plain.cpu())[0]
    assert rel(both, want) <= 2.0 ** -8
    assert torch.equal(both, shared.forward(x.cuda(), residual=plain))
