"""The fused W8A8 linear and the gated projection against 64 bits on the CPU, at sizes that reach every kernel behind them
(weight streaming for up to 16, 32, 64, 128 and 256 tokens, the same by CTA pairs, tiles of CTA pairs) and end inside their
tiles.

Tolerances: the integer sum is exact; its conversion, two products and the bias add round once each (4 * 2^-24 of
|acc*sa*sb| + |bias|), the activations have slopes of at most 1.13 and are off by 2^-18 of their value where the fast
exponential enters (argument up to 40 at 2^-23 each), the residual add rounds once, and the output is off by half a
bf16 step (2^-8)."""
import pytest
import torch

from tests import ffn_reference as ref
from tests import workloads as wl

pytestmark = pytest.mark.gpu
U = ref.U32


def close(got, want, slack):
    err = (got.cpu().double() - want).abs()
    assert (err <= ref.UBF * (want.abs() + slack) + slack).all(), float((err - ref.UBF * want.abs() - slack).max())


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


SHAPES = [(1, 8, 16), (1, 257, 144), (5, 40, 48), (16, 384, 2064), (17, 127, 128), (33, 1000, 272), (64, 129, 1040),
          (100, 320, 256), (128, 100, 528), (129, 255, 160), (200, 256, 2064), (256, 1001, 144), (257, 8, 64), (300, 1000, 400),
          (300, 7700, 144), (513, 5129, 272), (1100, 2304, 1040),
          # K split over pairs, one block of tokens and several; few tokens by tiles; rows of a few elements
          (140, 600, 6160), (200, 100, 5520), (300, 260, 7200), (600, 1000, 5520), (70, 900, 528), (80, 20000, 144),
          (128, 19001, 272), (900, 3, 144), (400, 1, 32), (270, 5, 6000)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_without_extras_has_the_bits_of_the_plain_gemm(ext, m, n, k):
    (a, sa), (w, sw) = ref.tokens(m, k, 1), ref.weight(n, k, 2)
    a, sa, w, sw = cuda(a, sa, w, sw)
    assert torch.equal(ext.w8a8_linear(a, w, sa, sw).view(torch.int16), ext.w8a8_gemm(a, w, sa, sw).view(torch.int16))


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("act,bias,residual", [("none", True, True), ("gelu", True, False), ("silu", False, True),
                                               ("gelu_tanh", True, True), ("relu", True, False)])
def test_linear(ext, m, n, k, act, bias, residual):
    (a, sa), (w, sw) = ref.tokens(m, k, m + n), ref.weight(n, k, k)
    b = ref.bf16((n,), 3) if bias else None
    r = ref.bf16((m, n + 5), 4)[:, 2:2 + n] if residual else None   # rows at odd addresses
    y64, size = ref.linear(a, sa, w, sw, b, act, r)
    ad, sad, wd, swd, bd = cuda(a, sa, w, sw, b)
    rd = None
    if residual:
        rd = torch.zeros((m, n + 5), dtype=torch.bfloat16, device="cuda")[:, 2:2 + n]
        rd.copy_(r)
    y = ext.w8a8_linear(ad, wd, sad, swd, bd, act, rd)
    assert y.dtype == torch.bfloat16 and y.shape == (m, n)
    slack = 1.13 * 4 * U * size + 2.0 ** -18 * size + 1e-9
    if residual:
        slack = slack + U * (size + r.double().abs())
        yc = ext.w8a8_linear(ad, wd, sad, swd, bd, act, rd.contiguous())   # 16-byte rows where n allows them: the same bits
        assert torch.equal(y.view(torch.int16), yc.view(torch.int16))
    close(y, y64, slack)


def gated_slack(size_g, size_u, g, u, act):
    ag = ref.act(g, act).abs()
    err_g = 1.13 * 4 * U * size_g + 2.0 ** -18 * size_g + 1e-9
    err_u = 4 * U * size_u
    return err_g * (u.abs() + err_u) + ag * err_u + U * ag * u.abs()


@pytest.mark.parametrize("m,i,k", SHAPES)
@pytest.mark.parametrize("act,bias", [("silu", False), ("silu", True), ("gelu", False), ("gelu_tanh", True), ("relu", True)])
def test_gated(ext, m, i, k, act, bias):
    i = max(1, i // 2)
    (a, sa), (w, sw) = ref.tokens(m, k, m + i), ref.weight(2 * i, k, k)
    b = ref.bf16((2 * i,), 3) if bias else None
    h64, (size_g, size_u, g, u) = ref.gated(a, sa, w, sw, b, act)
    h = ext.w8a8_gated(*cuda(a, w, sa, sw, b), act)
    assert h.dtype == torch.bfloat16 and h.shape == (m, i)
    close(h, h64, gated_slack(size_g, size_u, g, u, act))


@pytest.mark.parametrize("m", [1, 3, 40, 150, 400])
def test_gates_and_ups_are_not_swapped_and_stay_with_their_outputs(ext, m):
    """gate rows that give large positive sums act as identity under relu; each up row has one code of its own"""
    i, k = 300, 320
    a = torch.ones((m, k), dtype=torch.int8)
    w = torch.zeros((2 * i, k), dtype=torch.int8)
    w[:i, 0] = 1                               # every gate is 1
    w[i:, 1] = (torch.arange(i) % 127).to(torch.int8)
    one = torch.ones((m, 1))
    h = ext.w8a8_gated(a.cuda(), w.cuda(), one.cuda(), torch.ones(2 * i).cuda(), None, "relu")
    assert torch.equal(h.cpu().float(), (torch.arange(i) % 127).float().expand(m, -1))


def test_large_scales_and_special_values_pass_through(ext):
    (a, sa), (w, sw) = ref.tokens(40, 128, 1), ref.weight(96, 128, 2)
    b = torch.zeros(96)
    b[3], b[5], b[7] = float("inf"), float("-inf"), float("nan")
    b = b.to(torch.bfloat16)
    for act in ref.ACTS:
        y = ext.w8a8_linear(*cuda(a, w, sa, sw, b), act).cpu().float()
        assert (y[:, 3] == float("inf")).all() and y[:, 7].isnan().all()
        if act in ("none", "relu"):
            assert (y[:, 5] == (0.0 if act == "relu" else float("-inf"))).all()
        rest = [j for j in range(96) if j not in (3, 5, 7)]
        assert y[:, rest].isfinite().all()
    huge = ext.w8a8_linear(a.cuda(), w.cuda(), (sa * 1e6).cuda(), sw.cuda(), None, "silu").cpu().double()
    z = ref.project(a, sa * 1e6, w, sw, None)[0]
    assert ((huge - torch.clamp(z, min=0)).abs() <= 2.0 ** -8 * z.abs() + 1.0).all()


def tail_arguments(lo, hi):
    """every fourth bf16 number from -hi to hi with magnitudes from lo on"""
    bits = torch.arange(0, 0x7F80, 4, dtype=torch.int32)
    v = (bits << 16).view(torch.float32)
    v = v[(v >= lo) & (v <= hi)]
    return torch.cat([-v.flip(0), v])


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_activations_keep_their_digits_far_from_zero(ext, act):
    """the value itself to bf16, also where it is tiny: z is the bias, the weight is zero.  Relative error of the value:
    the exponential's argument is at most 88 with four roundings of 2^-24, which is 2^-15.6 of the exponential; the reciprocal
    and the polynomial add less than 2^-19."""
    z = tail_arguments(2.0 ** -20, {"gelu": 12.0, "gelu_tanh": 9.0, "silu": 80.0}[act])
    n = z.numel()
    b = z.to(torch.bfloat16).cuda()
    for m in (1, 300):   # weight streaming and tiles
        a, w = torch.zeros((m, 16), dtype=torch.int8, device="cuda"), torch.zeros((n, 16), dtype=torch.int8, device="cuda")
        y = ext.w8a8_linear(a, w, torch.ones((m, 1), device="cuda"), torch.ones(n, device="cuda"), b, act)
        zd = z.double()
        if act == "gelu_tanh":   # 1 + tanh loses every digit far below zero
            want = zd * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (zd + 0.044715 * zd ** 3))
        else:
            want = ref.act(zd, act)
        err = (y.cpu().double() - want).abs()
        bad = err > (ref.UBF + 1.01 * 2.0 ** -15) * want.abs()
        assert not bad.any(), (z[bad[0]][:5], (err / want.abs())[0].max())


def test_residual_rows_of_a_broadcast_or_wrong_shape_are_refused(ext):
    (a, sa), (w, sw) = ref.tokens(4, 64, 1), ref.weight(32, 64, 2)
    a, sa, w, sw = cuda(a, sa, w, sw)
    r = torch.zeros((4, 32), dtype=torch.bfloat16, device="cuda")
    for bad in (r[:3], r[:, :31], r[0].expand(4, 32), r.float(), r.cpu(), r.t().contiguous().t()):
        with pytest.raises(RuntimeError):
            ext.w8a8_linear(a, w, sa, sw, None, "none", bad)
    for bad in ("swish", "SILU", ""):
        with pytest.raises(RuntimeError, match="activation"):
            ext.w8a8_linear(a, w, sa, sw, None, bad)
    with pytest.raises(RuntimeError, match="activation"):
        ext.w8a8_gated(a, w, sa, sw, None, "none")
    with pytest.raises(RuntimeError, match="up rows"):
        ext.w8a8_gated(a, w[:31].contiguous(), sa, sw[:31].contiguous())
    with pytest.raises(RuntimeError, match="bias"):
        ext.w8a8_gated(a, w, sa, sw, torch.zeros(16, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(RuntimeError, match="multiple of 16"):
        ext.w8a8_linear(a[:, :40].contiguous(), w[:, :40].contiguous(), sa, sw)


def test_empty_batches(ext):
    (a, sa), (w, sw) = ref.tokens(1, 64, 1), ref.weight(32, 64, 2)
    a, sa, w, sw = cuda(a[:0], sa[:0], w, sw)
    assert ext.w8a8_linear(a, w, sa, sw).shape == (0, 32) and ext.w8a8_gated(a, w, sa, sw).shape == (0, 16)


def test_residual_in_place_through_the_c_abi(ext):
    """the output may be the residual's own array"""
    import ctypes
    import bw1000_dsv4_kernels_b200 as pkg
    lib = pkg.c_abi()
    p, ll = (lambda t: ctypes.c_void_p(t.data_ptr())), ctypes.c_longlong
    for m, n, k in ((3, 200, 256), (40, 333, 144), (150, 600, 160), (600, 2600, 144), (300, 90, 144)):
        (a, sa), (w, sw) = ref.tokens(m, k, 5), ref.weight(n, k, 6)
        a, sa, w, sw = cuda(a, sa, w, sw)
        r = ref.bf16((m, n), 7).cuda()
        want = ext.w8a8_linear(a, w, sa, sw, None, "gelu", r)
        rc = lib.launch_w8a8_linear(p(a), p(w), p(sa), p(sw), None, 2, p(r), ll(n), p(r), ll(n), m, n, k,
                                    ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0 and torch.equal(r.view(torch.int16), want.view(torch.int16))


def test_rows_and_columns_around_the_output_stay_as_they_were(ext):
    import ctypes
    import bw1000_dsv4_kernels_b200 as pkg
    lib = pkg.c_abi()
    p, ll = (lambda t: ctypes.c_void_p(t.data_ptr())), ctypes.c_longlong
    for m, n, k in ((3, 200, 256), (40, 333, 144), (150, 600, 160), (600, 2600, 144), (300, 90, 144)):
        (a, sa), (w, sw) = ref.tokens(m, k, 5), ref.weight(2 * n, k, 6)
        a, sa, w, sw = cuda(a, sa, w, sw)
        st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        buf = torch.full((m + 2, n + 8), 9.0, dtype=torch.bfloat16, device="cuda")
        out = buf[1:m + 1, :n]
        assert lib.launch_w8a8_gated(p(a), p(w), p(sa), p(sw), None, 4, ctypes.c_void_p(out.data_ptr()), ll(n + 8), m, n, k, st) == 0
        assert torch.equal(out.contiguous().view(torch.int16), ext.w8a8_gated(a, w, sa, sw).view(torch.int16))
        assert (buf[0] == 9).all() and (buf[m + 1] == 9).all() and (buf[:, n:] == 9).all()
        buf.fill_(9.0)
        assert lib.launch_w8a8_linear(p(a), p(w), p(sa), p(sw), None, 4, None, ll(0), ctypes.c_void_p(out.data_ptr()), ll(n + 8), m, n, k, st) == 0
        assert (buf[0] == 9).all() and (buf[m + 1] == 9).all() and (buf[:, n:] == 9).all()


@pytest.mark.parametrize("m", [2, 60, 200, 400])
def test_captured_replays_and_overlap_with_the_kernel_before(ext, m):
    i, k = 192, 512
    (w13, s13), (w2, s2) = ref.weight(2 * i, k, 1), ref.weight(k, i, 2)
    w13, s13, w2, s2 = cuda(w13, s13, w2, s2)
    gamma, beta = wl.gamma_bf16(k, seed=3).cuda(), ref.bf16((k,), 4).cuda()
    x, res = ref.bf16((m, k), 5).cuda(), ref.bf16((m, k), 6).cuda()

    def block(res):
        q, s, _, _ = ext.add_layernorm_quant(res, x, gamma, beta, 1e-6)
        h = ext.w8a8_gated(q, w13, s, s13)
        q, s = ext.per_token_quant_int8(h)
        return ext.w8a8_linear(q, w2, s, s2, beta, "none", res)
    want = block(res.clone())
    torch.cuda.synchronize()
    for overlap in (False, True):
        ext.set_overlap_previous_kernel(overlap)
        try:
            static = res.clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = block(static)
        finally:
            ext.set_overlap_previous_kernel(False)
        for _ in range(3):
            static.copy_(res)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y.view(torch.int16), want.view(torch.int16))
    assert ext.device_status() == 0
