"""Layer norm, forward and backward, against 64 bits on the CPU.

Tolerances: an output in bf16 is off by half a step (2^-8 relative) plus what the fp32 arithmetic in front of it is off.
A row's sum takes at most SEQ sequential fp32 additions (elements of one thread, then the exchange), so the mean is off
by SEQ * 2^-24 * mean|a|, a deviation by that and its own rounding, and rstd by about SEQ * 2^-24 relative."""
import pytest
import torch

from tests import ffn_reference as ref
from tests import workloads as wl

pytestmark = pytest.mark.gpu
EPS = 1e-6
U = ref.U32


def seq(k):
    """sequential fp32 operations of one row sum, with slack for the divisions and products around it"""
    return 40 + (0 if k <= 16384 else k // 1024)


def rows(m, k, seed, mean=0.0):
    x = wl.randn_bf16((m, k), seed=seed).float()
    x = x * torch.linspace(0.25, 4.0, m).unsqueeze(1) + mean
    return x.to(torch.bfloat16)


def weights(k, seed):
    return wl.gamma_bf16(k, seed=seed), ref.bf16((k,), seed + 1, 0.2)


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 16), (2, 255), (33, 256), (7, 1001), (9, 1000), (4, 2047), (3, 4096), (3, 4104),
          (2, 4099), (65, 7168), (2, 8192), (2, 8200), (2, 8193), (1, 16384), (2, 16383), (2, 16392), (1, 20001), (1000, 40),
          (300, 128), (40, 520), (400, 1001), (1300, 1003), (700, 2066), (333, 4097), (5, 65), (2, 71)]


def y_slack(a, mean, rstd, w, b, k):
    return U * seq(k) * (a.double().abs().amax(1, keepdim=True) * 2 * rstd[:, None] * w.double().abs() * 2 + b.double().abs())


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("add", [False, True])
def test_layernorm(ext, m, k, add):
    x, (w, b) = rows(m, k, 1), weights(k, 2)
    a = x
    if add:
        res = rows(m, k, 3)
        a = (res.float() + x.float()).to(torch.bfloat16)
        res_d = res.cuda()
        y, mean, rstd = ext.add_layernorm(res_d, x.cuda(), w.cuda(), b.cuda(), EPS)
        assert torch.equal(res_d.cpu().view(torch.int16), a.view(torch.int16))
    else:
        y, mean, rstd = ext.layernorm(x.cuda(), w.cuda(), b.cuda(), EPS)
    y64, mean64, rstd64 = ref.layernorm(a, w, b, EPS)
    assert y.dtype == torch.bfloat16 and y.shape == x.shape and mean.shape == (m,) and rstd.shape == (m,)
    big = a.double().abs().amax(1)
    assert ((mean.cpu().double() - mean64).abs() <= U * seq(k) * big).all()
    # relative: the deviations' own rounding, plus the mean's error, which enters squared
    var_err = 2 * seq(k) * U + (U * seq(k) * big * rstd64) ** 2 + 4 * U * seq(k) * big * rstd64
    assert ((rstd.cpu().double() / rstd64 - 1).abs() <= var_err).all()
    slack = y_slack(a, mean64, rstd64, w, b, k) + var_err[:, None] * y64.abs() * 2 + var_err[:, None] * b.double().abs()
    assert ((y.cpu().double() - y64).abs() <= ref.UBF * (y64.abs() + slack) + slack).all()


@pytest.mark.parametrize("mean", [0.0, 300.0])
def test_rows_with_a_large_mean_keep_their_variance(ext, mean):
    x, (w, b) = rows(6, 2048, 5, mean), weights(2048, 6)
    _, m, rstd = ext.layernorm(x.cuda(), w.cuda(), b.cuda(), EPS)
    _, m64, rstd64 = ref.layernorm(x, w, b, EPS)
    assert ((rstd.cpu().double() / rstd64 - 1).abs() <= U * 200).all()
    assert ((m.cpu().double() / m64 - 1).abs() <= U * 60).all() or mean == 0.0


def test_constant_rows_have_the_bias_as_output(ext):
    x = torch.full((3, 512), 2.5, dtype=torch.bfloat16)   # the row sums are exact, so the deviations are zero
    w, b = weights(512, 7)
    y, mean, rstd = ext.layernorm(x.cuda(), w.cuda(), b.cuda(), EPS)
    assert torch.equal(y.cpu(), b.expand(3, -1)) and (mean.cpu() == 2.5).all()
    assert ((rstd.cpu().double() * EPS ** 0.5 - 1).abs() <= 8 * U).all()


@pytest.mark.parametrize("m,k", [(1, 8), (3, 7), (9, 1000), (7, 1001), (5, 7168), (2, 16392), (1, 20001), (1300, 1003),
                                 (700, 2066), (4, 8195)])
@pytest.mark.parametrize("add", [False, True])
def test_layernorm_quant_codes_and_scales(ext, m, k, add):
    x, (w, b) = rows(m, k, 11), weights(k, 12)
    a = x
    if add:
        res = rows(m, k, 13)
        a = (res.float() + x.float()).to(torch.bfloat16)
        res_d = res.cuda()
        q, s, mean, rstd = ext.add_layernorm_quant(res_d, x.cuda(), w.cuda(), b.cuda(), EPS)
        assert torch.equal(res_d.cpu().view(torch.int16), a.view(torch.int16))
        y2, mean2, rstd2 = ext.add_layernorm(res.cuda(), x.cuda(), w.cuda(), b.cuda(), EPS)
    else:
        q, s, mean, rstd = ext.layernorm_quant(x.cuda(), w.cuda(), b.cuda(), EPS)
        y2, mean2, rstd2 = ext.layernorm(x.cuda(), w.cuda(), b.cuda(), EPS)
    assert torch.equal(mean, mean2) and torch.equal(rstd, rstd2)
    assert q.dtype == torch.int8 and q.shape == x.shape and s.shape == (m, 1)
    y64, mean64, rstd64 = ref.layernorm(a, w, b, EPS)
    big = a.double().abs().amax(1)
    var_err = 2 * seq(k) * U + 4 * U * seq(k) * big * rstd64
    err = y_slack(a, mean64, rstd64, w, b, k) + var_err[:, None] * (y64.abs() + b.double().abs()) * 2
    top = y64.abs().amax(1, keepdim=True).clamp_min(1e-10)
    assert ((s.cpu().double() * 127 - top).abs() <= err.amax(1, keepdim=True) + 2 * U * top).all()
    # a code is the nearest integer to y * 127 / top, with the errors of y, of top and of two roundings
    exact = y64 * 127 / top
    slack = err * 127 / top + exact.abs() * (err.amax(1, keepdim=True) / top + 4 * U)
    assert ((q.cpu().double() - exact).abs() <= 0.5 + slack).all()


@pytest.mark.parametrize("m,k", SHAPES + [(700, 7168), (2000, 24)])
@pytest.mark.parametrize("add", [False, True])
def test_layernorm_backward(ext, m, k, add):
    x, (w, b) = rows(m, k, 21), weights(k, 22)
    dy, dres = wl.randn_bf16((m, k), seed=23), wl.randn_bf16((m, k), seed=24) if add else None
    _, mean, rstd = ref.layernorm(x, w, b, EPS)
    mean, rstd = mean.float(), rstd.float()
    dx, dw, db = ext.layernorm_backward(dy.cuda(), x.cuda(), mean.cuda(), rstd.cuda(), w.cuda(), dres.cuda() if add else None)
    dx64, dw64, db64 = ref.layernorm_backward(dy, x, mean, rstd, w, dres)
    assert dx.dtype == torch.bfloat16 and dw.dtype == db.dtype == torch.float32
    xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    t = dy.double() * w.double()
    size = rstd.double()[:, None] * (t.abs() + t.abs().mean(1, keepdim=True) + xh.abs() * (t * xh).abs().mean(1, keepdim=True))
    slack = U * 2 * seq(k) * size
    if add:
        slack = slack + U * dres.double().abs()
    assert ((dx.cpu().double() - dx64).abs() <= ref.UBF * (dx64.abs() + slack) + slack).all()
    # a column: each row's product is off by three roundings, and the sum takes at most M additions
    adds = U * (min(m, 400) + 8)
    assert ((dw.cpu().double() - dw64).abs() <= adds * (dy.double() * xh).abs().sum(0) + 1e-30).all()
    assert ((db.cpu().double() - db64).abs() <= adds * dy.double().abs().sum(0) + 1e-30).all()


def test_backward_matches_differences_of_the_forward(ext):
    """directional derivative of sum(y * dy) through the kernel's own dx, dw, db, against central differences in 64 bits"""
    m, k = 5, 96
    x, (w, b) = rows(m, k, 31), weights(k, 32)
    dy, v = wl.randn_bf16((m, k), seed=33), torch.randn(m, k, dtype=torch.float64)
    vw, vb = torch.randn(k, dtype=torch.float64), torch.randn(k, dtype=torch.float64)
    _, mean, rstd = ext.layernorm(x.cuda(), w.cuda(), b.cuda(), EPS)
    dx, dw, db = (t.cpu().double() for t in ext.layernorm_backward(dy.cuda(), x.cuda(), mean, rstd, w.cuda()))
    h = 1e-5

    def f(t):
        return (ref.layernorm(x.double() + t * v, w.double() + t * vw, b.double() + t * vb, EPS)[0] * dy.double()).sum()
    slope = (f(h) - f(-h)) / (2 * h)
    got = (dx * v).sum() + (dw * vw).sum() + (db * vb).sum()
    # dx is rounded to bf16 once; the differences are off by about h^2
    assert (got - slope).abs() <= ref.UBF * (dx * v).abs().sum() + 1e-6 * slope.abs() + 1e-6


def test_two_runs_give_the_same_bits(ext):
    x, (w, b) = rows(500, 1000, 41).cuda(), (t.cuda() for t in weights(1000, 42))
    dy = wl.randn_bf16((500, 1000), seed=43).cuda()
    _, mean, rstd = ext.layernorm(x, w, b, EPS)
    first = ext.layernorm_backward(dy, x, mean, rstd, w)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, ext.layernorm_backward(dy, x, mean, rstd, w)))


def test_empty_batches(ext):
    w, b = (t.cuda() for t in weights(64, 51))
    x = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    y, mean, rstd = ext.layernorm(x, w, b, EPS)
    assert y.shape == (0, 64) and mean.shape == rstd.shape == (0,)
    q, s, _, _ = ext.add_layernorm_quant(x.clone(), x, w, b, EPS)
    assert q.shape == (0, 64) and s.shape == (0, 1)
    dx, dw, db = ext.layernorm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_unaligned_views_and_leading_dimensions(ext):
    w, b = weights(256, 61)
    buf = rows(1, 12 * 256 + 3, 62).flatten()
    x = buf[3:].view(3, 4, 256)     # 6 bytes past an aligned address
    y, mean, rstd = ext.layernorm(x.cuda(), w.cuda(), b.cuda(), EPS)
    moved = torch.empty(12 * 256 + 3, dtype=torch.bfloat16, device="cuda")
    moved.copy_(buf)
    y2, mean2, rstd2 = ext.layernorm(moved[3:].view(3, 4, 256), w.cuda(), b.cuda(), EPS)
    y64, mean64, rstd64 = ref.layernorm(x.reshape(12, 256), w, b, EPS)
    for yy in (y, y2):
        assert yy.shape == (3, 4, 256)
        assert ((yy.cpu().double().view(12, 256) - y64).abs() <= ref.UBF * y64.abs() + 2e-5).all()
    assert mean2.shape == (12,) and ((rstd2.cpu().double() / rstd64 - 1).abs() <= 200 * U).all()


def test_other_stream_and_captured_replay(ext):
    m, k = 40, 1024
    w, b = (t.cuda() for t in weights(k, 71))
    x, dy = rows(m, k, 72).cuda(), wl.randn_bf16((m, k), seed=73).cuda()
    _, mean, rstd = ext.layernorm(x, w, b, EPS)
    want = ext.layernorm_backward(dy, x, mean, rstd, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for _ in range(20):   # workspaces of calls in flight on another stream are not handed to this one
        outs.append(ext.layernorm_backward_stream(dy, x, mean, rstd, w, None, side.cuda_stream))
        torch.full((4096, 256), float("nan"), device="cuda")
    side.synchronize()
    assert all(torch.equal(p, q) for o in outs for p, q in zip(want, o))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, mean2, rstd2 = ext.layernorm(x, w, b, EPS)
        grads = ext.layernorm_backward(dy, x, mean2, rstd2, w)
    for seed in (75, 76):
        x.copy_(rows(m, k, seed))
        dy.copy_(wl.randn_bf16((m, k), seed=seed + 10))
        graph.replay()
        eager = ext.layernorm(x, w, b, EPS)
        want = ext.layernorm_backward(dy, x, eager[1], eager[2], w)
        torch.cuda.synchronize()
        assert torch.equal(y, eager[0]) and all(torch.equal(p, q) for p, q in zip(want, grads))


@pytest.mark.parametrize("m,k", [(12, 1), (12, 33), (12, 64), (600, 2048), (12, 4104), (3, 16392)])
def test_a_row_with_nan_or_infinity_keeps_it(ext, m, k):
    """statistics, bf16 rows and scales of such rows are not finite, and no other row notices"""
    x, (w, b) = rows(m, k, 1), weights(k, 2)
    clean = x.clone()
    x[1, k // 2], x[2, 0] = float("nan"), float("inf")
    y, mean, rstd = ext.layernorm(*(t.cuda() for t in (x, w, b)), EPS)
    q, s, _, _ = ext.layernorm_quant(*(t.cuda() for t in (x, w, b)), EPS)
    y0 = ext.layernorm(*(t.cuda() for t in (clean, w, b)), EPS)[0]
    q0, s0, _, _ = ext.layernorm_quant(*(t.cuda() for t in (clean, w, b)), EPS)
    fine = [r for r in range(m) if r not in (1, 2)]
    for t in (y[1:3], rstd[1:3], s[1:3]):
        assert t.isnan().all()
    assert torch.equal(y[fine], y0[fine]) and torch.equal(q[fine], q0[fine]) and torch.equal(s[fine], s0[fine])
    b[k - 1] = float("nan")
    assert ext.layernorm_quant(*(t.cuda() for t in (clean, w, b)), EPS)[1].isnan().all()


def view_at(t, offset):
    """the same values on the device, `offset` elements into a buffer whose elements around them are NaN"""
    if t is None:
        return None
    buf = torch.full((t.numel() + 32,), float("nan"), dtype=t.dtype, device="cuda")
    v = buf[offset:offset + t.numel()].view(t.shape)
    v.copy_(t)
    return v


def check_forward(a, w, b, k, y, mean, rstd):
    y64, mean64, rstd64 = ref.layernorm(a, w, b, EPS)
    big = a.double().abs().amax(1)
    assert ((mean.cpu().double() - mean64).abs() <= U * seq(k) * big).all()
    var_err = 2 * seq(k) * U + (U * seq(k) * big * rstd64) ** 2 + 4 * U * seq(k) * big * rstd64
    assert ((rstd.cpu().double() / rstd64 - 1).abs() <= var_err).all()
    slack = y_slack(a, mean64, rstd64, w, b, k) + var_err[:, None] * (2 * y64.abs() + b.double().abs())
    assert ((y.cpu().double() - y64).abs() <= ref.UBF * (y64.abs() + slack) + slack).all()


def check_codes(a, w, b, k, q, s):
    y64, mean64, rstd64 = ref.layernorm(a, w, b, EPS)
    big = a.double().abs().amax(1)
    var_err = 2 * seq(k) * U + 4 * U * seq(k) * big * rstd64
    err = y_slack(a, mean64, rstd64, w, b, k) + var_err[:, None] * (y64.abs() + b.double().abs()) * 2
    top = y64.abs().amax(1, keepdim=True).clamp_min(1e-10)
    assert ((s.cpu().double() * 127 - top).abs() <= err.amax(1, keepdim=True) + 2 * U * top).all()
    exact = y64 * 127 / top
    slack = err * 127 / top + exact.abs() * (err.amax(1, keepdim=True) / top + 4 * U)
    assert ((q.cpu().double() - exact).abs() <= 0.5 + slack).all()


def check_backward(dy, x, mean, rstd, w, dres, k, dx, dw, db):
    m = x.shape[0]
    dx64, dw64, db64 = ref.layernorm_backward(dy, x, mean, rstd, w, dres)
    xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    t = dy.double() * w.double()
    size = rstd.double()[:, None] * (t.abs() + t.abs().mean(1, keepdim=True) + xh.abs() * (t * xh).abs().mean(1, keepdim=True))
    slack = U * 2 * seq(k) * size + (0 if dres is None else U * dres.double().abs())
    assert ((dx.cpu().double() - dx64).abs() <= ref.UBF * (dx64.abs() + slack) + slack).all()
    adds = U * (min(m, 400) + 8)
    assert ((dw.cpu().double() - dw64).abs() <= adds * (dy.double() * xh).abs().sum(0) + 1e-30).all()
    assert ((db.cpu().double() - db64).abs() <= adds * dy.double().abs().sum(0) + 1e-30).all()


# arrays at offsets of their own: x, residual (or the gradient past the norm), output side (dy), weight, bias
OFFSETS = [(0, 0, 0, 0, 0), (2, 2, 2, 0, 0), (1, 1, 1, 0, 0), (2, 0, 4, 2, 6), (1, 2, 3, 0, 1), (8, 5, 0, 8, 8)]


@pytest.mark.parametrize("m,k", [(3, 4098), (2, 8190), (3, 8191), (2, 8192), (2, 12290), (2, 16383), (2, 16384), (300, 4098),
                                 (5, 61), (700, 65), (40, 16386)])
@pytest.mark.parametrize("offsets", OFFSETS)
@pytest.mark.parametrize("add", [False, True])
def test_forward_of_arrays_at_any_offset(ext, m, k, offsets, add):
    ox, orr, _, ow, ob = offsets
    x, (w, b) = rows(m, k, 81), weights(k, 82)
    res = rows(m, k, 83) if add else None
    a = (res.float() + x.float()).to(torch.bfloat16) if add else x
    xd, wd, bd = view_at(x, ox), view_at(w, ow), view_at(b, ob)
    if add:
        res_d = view_at(res, orr)
        y, mean, rstd = ext.add_layernorm(res_d, xd, wd, bd, EPS)
        assert torch.equal(res_d.cpu().view(torch.int16), a.view(torch.int16))
        around = res_d._base
        assert around[:orr].isnan().all() and around[orr + m * k:].isnan().all()
        res_d.copy_(res)
        q, s, mean2, rstd2 = ext.add_layernorm_quant(res_d, xd, wd, bd, EPS)
        assert torch.equal(res_d.cpu().view(torch.int16), a.view(torch.int16))
    else:
        y, mean, rstd = ext.layernorm(xd, wd, bd, EPS)
        q, s, mean2, rstd2 = ext.layernorm_quant(xd, wd, bd, EPS)
    check_forward(a, w, b, k, y, mean, rstd)
    check_forward(a, w, b, k, y, mean2, rstd2)
    check_codes(a, w, b, k, q, s)


@pytest.mark.parametrize("m,k", [(3, 7170), (2, 7176), (2, 8190), (3, 8191), (1, 8184), (2, 8194), (3, 16382), (2, 16383), (400, 7170),
                                 (300, 8191), (330, 8190), (160, 16382), (700, 12289), (5, 61), (900, 65), (300, 4098)])
@pytest.mark.parametrize("offsets", OFFSETS)
@pytest.mark.parametrize("add", [False, True])
def test_backward_of_arrays_at_any_offset(ext, m, k, offsets, add):
    ox, orr, oy, ow, _ = offsets
    x, (w, b) = rows(m, k, 91), weights(k, 92)
    dy, dres = wl.randn_bf16((m, k), seed=93), wl.randn_bf16((m, k), seed=94) if add else None
    _, mean, rstd = ref.layernorm(x, w, b, EPS)
    mean, rstd = mean.float(), rstd.float()
    dx, dw, db = ext.layernorm_backward(view_at(dy, oy), view_at(x, ox), mean.cuda(), rstd.cuda(), view_at(w, ow), view_at(dres, orr))
    check_backward(dy, x, mean, rstd, w, dres, k, dx, dw, db)


@pytest.mark.parametrize("m,k,off", [(5, 4104, 4), (3, 8190, 1), (4, 8191, 3), (2, 12290, 2), (3, 16383, 5), (300, 1000, 7), (40, 7170, 2)])
def test_outputs_at_any_offset_through_the_c_abi(ext, m, k, off):
    """torch's own outputs are always aligned; a C caller's need not be.  Nothing around them is written."""
    import ctypes
    import bw1000_dsv4_kernels_b200 as pkg
    lib = pkg.c_abi()
    p = lambda t: ctypes.c_void_p(t.data_ptr())   # noqa: E731
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    x, (w, b) = rows(m, k, 101), weights(k, 102)
    xd, wd, bd = x.cuda(), w.cuda(), b.cuda()
    mean, rstd, s = (torch.empty(m, device="cuda") for _ in range(3))
    y = view_at(torch.zeros((m, k), dtype=torch.bfloat16), off)
    eps = ctypes.c_float(EPS)
    assert lib.launch_layernorm(None, p(xd), p(wd), p(bd), p(y), p(mean), p(rstd), m, k, eps, st) == 0
    check_forward(x, w, b, k, y, mean, rstd)
    assert y._base[:off].isnan().all() and y._base[off + m * k:].isnan().all()
    codes = torch.full((m * k + 64,), 99, dtype=torch.int8, device="cuda")
    q = codes[off:off + m * k].view(m, k)
    assert lib.launch_layernorm_quant(None, p(xd), p(wd), p(bd), p(q), p(s), p(mean), p(rstd), m, k, eps, st) == 0
    check_codes(x, w, b, k, q, s.unsqueeze(1))
    assert (codes[:off] == 99).all() and (codes[off + m * k:] == 99).all()
    dy = wl.randn_bf16((m, k), seed=103)
    _, mean64, rstd64 = ref.layernorm(x, w, b, EPS)
    mean, rstd = mean64.float(), rstd64.float()
    dx, dw, db = view_at(torch.zeros((m, k), dtype=torch.bfloat16), off), torch.empty(k, device="cuda"), torch.empty(k, device="cuda")
    lib.dsv4_layernorm_backward_workspace.restype = ctypes.c_int64
    size = lib.dsv4_layernorm_backward_workspace(m, k)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    md, rd, yd = mean.cuda(), rstd.cuda(), dy.cuda()
    assert lib.launch_layernorm_backward(p(yd), p(xd), p(md), p(rd), p(wd), None, p(dx), p(dw), p(db), p(ws),
                                         ctypes.c_longlong(size), m, k, st) == 0
    check_backward(dy, x, mean, rstd, w, None, k, dx, dw, db)
    assert dx._base[:off].isnan().all() and dx._base[off + m * k:].isnan().all()
