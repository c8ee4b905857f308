"""Gradients of the fused W8A8 linear and of the gated projection against 64 bits on the CPU.

Tolerances.  dz: the recomputed z is off by 4 * 2^-24 of its size, slopes of at most 1.13 (their own slope at most 1.2)
and the fast exponential's 2^-18 make that 2^-17 of the terms' magnitude at most.  dx: every row of t = dz * sb is in
fixed point with a step of top / 32639, off by half of it, so a sum of N terms is off by at most
(step / 2) * sum |W[n, k]|, plus dz's own error times |W|, plus the two conversions, plus half a bf16 step of the
result.  GELU's normal distribution function comes from a published polynomial that is off by 0.75e-7 (2^-23.6) at most,
which is CDF * |z| <= 2^-23 |z| in the activation.  dbias: dz's error, and the fp32 additions of a column (rows of a block, then the blocks' slices)."""
import pytest
import torch

from tests import ffn_reference as ref
from tests import workloads as wl

pytestmark = pytest.mark.gpu
U = ref.U32
DZ = 2.0 ** -17


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def check_dx(dx, dx64, t, t_err, w):
    step = t.abs().amax(1, keepdim=True).clamp_min(1e-30) / 32639
    wsum = w.double().abs().sum(0, keepdim=True)
    slack = step / 2 * 1.01 * wsum + t_err @ w.double().abs() + 4 * U * (t.abs() @ w.double().abs())
    err = (dx.cpu().double() - dx64).abs()
    assert (err <= ref.UBF * (dx64.abs() + slack) + slack).all(), float((err - ref.UBF * dx64.abs() - slack).max())
    # the fixed point is worth more than bf16: the rounding of the result dominates
    if dx64.abs().max() > 0:
        assert err.norm() <= 4e-3 * dx64.norm()


def check_db(db, db64, dz, dz_err):
    m = dz.shape[0]
    slack = dz_err.sum(0) + U * (40 + m // 16) * dz.abs().sum(0) + 1e-30
    assert db.dtype == torch.float32 and ((db.cpu().double() - db64).abs() <= slack).all()


SHAPES = [(1, 8, 16), (3, 40, 48), (17, 127, 128), (64, 128, 144), (100, 257, 272), (129, 320, 1040), (256, 256, 256),
          (257, 1000, 400), (300, 129, 2064), (513, 600, 528), (700, 2305, 784),
          # sums split over clusters for 16, 32, 64 and 128 rows and several blocks of them; rows of a few elements
          (1, 2000, 2064), (16, 1500, 1040), (30, 4000, 144), (40, 3000, 528), (128, 4100, 400), (300, 2600, 400),
          (200, 300, 6160), (500, 3, 400), (260, 1, 48), (83, 5000, 96), (50, 2600, 256)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("act,bias", [("none", False), ("none", True), ("gelu", True), ("silu", False), ("gelu_tanh", True),
                                      ("relu", True)])
def test_linear_backward(ext, m, n, k, act, bias):
    (a, sa), (w, sw) = ref.tokens(m, k, m), ref.weight(n, k, n)
    b = ref.bf16((n,), 3) if bias else None
    dy = ref.bf16((m, n + 3), 4)[:, 1:n + 1]
    dx64, db64, t, dz = ref.linear_backward(dy, a, sa, w, sw, b, act)
    dyd = torch.zeros((m, n + 3), dtype=torch.bfloat16, device="cuda")[:, 1:n + 1]   # strided rows at odd addresses
    dyd.copy_(dy)
    ad, wd, sad, swd, bd = cuda(a, w, sa, sw, b)
    dx, db = ext.w8a8_linear_backward(dyd, ad, wd, sad, swd, bd, act)
    assert dx.dtype == torch.bfloat16 and dx.shape == (m, k)
    z, size = ref.project(a, sa, w, sw, b)
    dz_err = (dy.double().abs() * (DZ + 1.2 * 4 * U * size)) if act != "none" else torch.zeros_like(dz)
    if act == "relu":   # where z is within its rounding of zero the kernel may take either side
        dz_err = torch.where(z.abs() <= 4 * U * size, dy.double().abs(), 0 * dz)
    check_dx(dx, dx64, t, dz_err * sw.double(), w)
    assert (db is None) == (not bias)
    if bias:
        check_db(db, db64, dz, dz_err)
    dx2, db2 = ext.w8a8_linear_backward(dyd.contiguous(), ad, wd, sad, swd, bd, act)   # aligned rows: the same bits
    assert torch.equal(dx.view(torch.int16), dx2.view(torch.int16)) and (not bias or torch.equal(db, db2))


@pytest.mark.parametrize("m,i,k", SHAPES)
@pytest.mark.parametrize("act,bias", [("silu", False), ("silu", True), ("gelu", False), ("gelu_tanh", True), ("relu", False)])
def test_gated_backward(ext, m, i, k, act, bias):
    i = max(1, i // 2)
    (a, sa), (w, sw) = ref.tokens(m, k, m), ref.weight(2 * i, k, i)
    b = ref.bf16((2 * i,), 3) if bias else None
    dh = ref.bf16((m, i), 4)
    dx64, db64, t, dz = ref.gated_backward(dh, a, sa, w, sw, b, act)
    dx, db = ext.w8a8_gated_backward(dh.cuda(), *cuda(a, w, sa, sw, b), act)
    z, size = ref.project(a, sa, w, sw, b)
    g, u, size_g, size_u = z[:, :i], z[:, i:], size[:, :i], size[:, i:]
    d = dh.double().abs()
    err_g = d * u.abs() * (DZ + 1.2 * 4 * U * size_g) + d * 1.13 * 4 * U * size_u
    err_u = d * (DZ * (ref.act(g, act).abs() + 1e-6) + 1.13 * 4 * U * size_g + 2.0 ** -23 * g.abs())
    if act == "relu":
        near = g.abs() <= 4 * U * size_g
        err_g = torch.where(near, d * u.abs() * 1.01, d * 1.13 * 4 * U * size_u + U * d * u.abs())
    err = torch.cat([err_g, err_u], 1) + 4 * U * dz.abs()
    check_dx(dx, dx64, t, err * sw.double(), w)
    assert (db is None) == (not bias)
    if bias:
        check_db(db, db64, dz, err)


def test_the_gradient_product_takes_every_weight_row_and_column(ext):
    """unit scales and gradients of small integers, then one row of the weight per row of the result"""
    m, n, k = 300, 640, 432
    g = torch.Generator().manual_seed(1)
    dy = torch.randint(-8, 9, (m, n), generator=g).float()
    dy[:, 0] = 8.0
    dy = dy.to(torch.bfloat16)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    (a, sa) = ref.tokens(m, k, 2)
    dx, _ = ext.w8a8_linear_backward(dy.cuda(), a.cuda(), w.cuda(), sa.cuda(), torch.ones(n).cuda())
    want = dy.double() @ w.double()
    step = 8.0 / 32639
    bound = step / 2 * w.double().abs().sum(0)
    assert ((dx.cpu().double() - want).abs() <= ref.UBF * (want.abs() + bound) + bound).all()
    # one row of the weight at a time comes back as itself
    one = torch.zeros((m, n), dtype=torch.bfloat16)
    one[torch.arange(m), torch.arange(m) % n] = 1.0
    dx, _ = ext.w8a8_linear_backward(one.cuda(), a.cuda(), w.cuda(), sa.cuda(), torch.ones(n).cuda())
    assert ((dx.cpu().double() - w[torch.arange(m) % n].double()).abs() <= 127 * 2.0 ** -15).all()


def test_rows_are_scaled_by_themselves(ext):
    """rows of very different size, rows of zeros, and rows with a NaN or an infinity do not touch one another"""
    m, n, k = 12, 96, 64
    (a, sa), (w, sw) = ref.tokens(m, k, 1), ref.weight(n, k, 2)
    dy = ref.bf16((m, n), 3).float() * (10.0 ** torch.arange(-24, 24, 4).float()).unsqueeze(1)
    dy[5] = 0.0
    dy[7, 11] = float("nan")
    dy[8, 12] = float("inf")
    dy = dy.to(torch.bfloat16)
    for act in ("none", "silu"):
        dx, db = ext.w8a8_linear_backward(dy.cuda(), *cuda(a, w, sa, sw, torch.zeros(n, dtype=torch.bfloat16)), act)
        dx = dx.cpu().double()
        assert (dx[5] == 0).all() and dx[7].isnan().all() and not dx[8].isfinite().any()
        fine = [r for r in range(m) if r not in (5, 7, 8)]
        want = ref.linear_backward(dy[fine], a[fine], sa[fine], w, sw, None, act)[0]
        assert ((dx[fine] - want).norm(dim=1) <= 4e-3 * want.norm(dim=1)).all()
        assert db.cpu()[11].isnan() and not db.cpu()[12].isfinite()


def outlier_rows(m, n, w, seed):
    """gradients of unit size with one element of 3000 in some rows, where the weight has a row of zeros: nothing of the
    outlier reaches dx"""
    w = w.clone()
    w[5 % n] = 0
    dy = ref.bf16((m, n), seed).float()
    some = torch.arange(m) % 3 == 1
    dy[some, 5 % n] = 3000.0
    return dy.to(torch.bfloat16), w, some


def check_dx_by_typical_size(dx, dx64, t, t_err, w):
    """Half a step of the fixed point: two digits, or three where the typical size (the square of the mean root, every root
    within 6 %) is below top / 256; either way at most 2^-8 of the typical size, or 2^-24 of top where that is more.  The
    latter is what fp32 sums lose wherever the outlier meets a code that is not zero."""
    top = t.abs().amax(1, keepdim=True)
    typical = 1.06 ** 2 * t.abs().sqrt().mean(1, keepdim=True) ** 2
    half_step = torch.maximum(torch.minimum(top * 2.0 ** -16, typical * 2.0 ** -8), top * 2.0 ** -24) * 1.01
    wsum = w.double().abs()
    slack = half_step * wsum.sum(0, keepdim=True) + (t_err + 4 * U * t.abs()) @ wsum
    err = (dx.cpu().double() - dx64).abs()
    assert (err <= ref.UBF * (dx64.abs() + slack) + slack).all(), float((err - ref.UBF * dx64.abs() - slack).max())
    # in the 2-norm of a row: half a bf16 step, and twice the root mean square of the fixed point's error, which is uniform
    # and independent from element to element (a third of half a step's square, times the codes' squares)
    spread = half_step.squeeze(1) / 3 ** 0.5 * w.double().norm() + ((t_err + 4 * U * t.abs()) @ wsum).norm(dim=1)
    assert (err.norm(dim=1) <= ref.UBF * dx64.norm(dim=1) + 2 * spread).all()


@pytest.mark.parametrize("m,n,k", [(3, 600, 256), (14, 400, 528), (30, 700, 272), (64, 520, 400), (128, 4100, 400), (200, 300, 6160),
                                   (300, 2600, 400), (257, 1000, 400), (700, 2305, 784), (1030, 400, 512), (5, 40, 48)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_rows_with_outliers_are_as_exact_as_the_others(ext, m, n, k, act):
    """dx against the magnitudes that really enter it, as everywhere else, and the rows without outliers bit for bit what they
    are without those neighbours"""
    (a, sa), (w, sw) = ref.tokens(m, k, m), ref.weight(n, k, n)
    dy, w, some = outlier_rows(m, n, w, 4)
    b = torch.zeros(n, dtype=torch.bfloat16)
    if act != "none":
        b[5 % n] = 4.0   # the weight row of zeros: z is the bias, whose slope is about one
    dx64, db64, t, dz = ref.linear_backward(dy, a, sa, w, sw, b, act)
    dx, db = ext.w8a8_linear_backward(dy.cuda(), *cuda(a, w, sa, sw, b), act)
    _, size = ref.project(a, sa, w, sw, b)
    dz_err = dy.double().abs() * (DZ + 1.2 * 4 * U * size) if act != "none" else torch.zeros_like(dz)
    check_db(db, db64, dz, dz_err)
    check_dx_by_typical_size(dx, dx64, t, dz_err * sw.double(), w)
    assert ((dx.cpu().double() - dx64).norm(dim=1) <= 4e-3 * dx64.norm(dim=1)).all()
    calm = torch.where(some[:, None], torch.zeros_like(dy), dy)
    dx2, _ = ext.w8a8_linear_backward(calm.cuda(), *cuda(a, w, sa, sw, b), act)
    assert torch.equal(dx2.cpu()[~some].view(torch.int16), dx.cpu()[~some].view(torch.int16))


@pytest.mark.parametrize("m", [9, 120, 400])
def test_outliers_of_every_size_stay_within_the_bound(ext, m):
    """one and several outliers per row, from three times to 10^6 times the rest, on both sides of the rule"""
    n, k = 1100, 400
    (a, sa), (w, sw) = ref.tokens(m, k, m), ref.weight(n, k, n)
    w[5], w[600], w[1099] = 0, 0, 0
    dy = ref.bf16((m, n), 4).float()
    size = 10.0 ** (0.5 + 5.5 * torch.arange(m) / m)
    dy[:, 5] = size
    dy[::2, 600], dy[::3, 1099] = size[::2], -size[::3]
    dy = dy.to(torch.bfloat16)
    dx64, _, t, dz = ref.linear_backward(dy, a, sa, w, sw)
    dx, _ = ext.w8a8_linear_backward(dy.cuda(), *cuda(a, w, sa, sw))
    check_dx_by_typical_size(dx, dx64, t, torch.zeros_like(dz), w)


@pytest.mark.parametrize("m,i,k", [(20, 300, 272), (300, 700, 528), (700, 1100, 784)])
def test_gated_rows_with_outliers(ext, m, i, k):
    """an outlier in the incoming gradient, whose gate and up rows of the weight are zero"""
    (a, sa), (w, sw) = ref.tokens(m, k, m), ref.weight(2 * i, k, i)
    w[7], w[i + 7] = 0, 0
    b = torch.zeros(2 * i, dtype=torch.bfloat16)
    b[7], b[i + 7] = 2.0, 1.0
    dh = ref.bf16((m, i), 4).float()
    dh[::2, 7] = 30000.0
    dh = dh.to(torch.bfloat16)
    dx64, db64, t, dz = ref.gated_backward(dh, a, sa, w, sw, b, "silu")
    dx, db = ext.w8a8_gated_backward(dh.cuda(), *cuda(a, w, sa, sw, b), "silu")
    z, size = ref.project(a, sa, w, sw, b)
    g, u, size_g, size_u, d = z[:, :i], z[:, i:], size[:, :i], size[:, i:], dh.double().abs()
    err_g = d * u.abs() * (DZ + 1.2 * 4 * U * size_g) + d * 1.13 * 4 * U * size_u
    err_u = d * (DZ * (ref.act(g, "silu").abs() + 1e-6) + 1.13 * 4 * U * size_g)
    check_dx_by_typical_size(dx, dx64, t, (torch.cat([err_g, err_u], 1) + 4 * U * dz.abs()) * sw.double(), w)
    again = ext.w8a8_gated_backward(dh.cuda(), *cuda(a, w, sa, sw, b), "silu")
    assert torch.equal(again[0].view(torch.int16), dx.view(torch.int16)) and torch.equal(again[1], db)


def test_every_row_wide_at_many_tiles(ext):
    """more tiles than pairs of CTAs, wide and calm blocks of rows in turn, captured and replayed"""
    m, n, k = 5200, 520, 1808
    (w, sw) = ref.weight(n, k, 2)
    w[5] = 0
    (a, sa) = ref.tokens(m, k, 3)
    dy = ref.bf16((m, n), 4).float()
    wide = (torch.arange(m) // 700) % 2 == 0
    dy[wide, 5] = 3000.0
    dy = dy.to(torch.bfloat16)
    ad, wd, sad, swd, dyd = cuda(a, w, sa, sw, dy)
    dx, _ = ext.w8a8_linear_backward(dyd, ad, wd, sad, swd)
    want = ref.linear_backward(dy, a, sa, w, sw)[0]
    assert ((dx.cpu().double() - want).norm(dim=1) <= 4e-3 * want.norm(dim=1)).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = ext.w8a8_linear_backward(dyd, ad, wd, sad, swd)
    for flip in (True, False):
        dyd.copy_(dy.flip(0) if flip else dy)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), ext.w8a8_linear_backward(dyd, ad, wd, sad, swd)[0].view(torch.int16))
    assert torch.equal(out.view(torch.int16), dx.view(torch.int16)) and ext.device_status() == 0


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_slopes_keep_their_digits_far_from_zero(ext, act):
    """act'(z) of one element per row, to bf16 of its two terms' magnitude: z is the bias, dx the element's digits times 127.
    Each term has the relative error of the exponential, 2^-15.6 (arguments up to 88, four roundings), and less than 2^-19
    beside it."""
    hi = {"gelu": 9.0, "gelu_tanh": 9.0, "silu": 60.0}[act]
    bits = torch.arange(0, 0x7F80, 8, dtype=torch.int32)
    v = (bits << 16).view(torch.float32)
    v = v[(v >= 2.0 ** -20) & (v <= hi)]
    z = torch.cat([-v.flip(0), v])
    z = torch.cat([z, torch.zeros(-z.numel() % 16)])
    n = z.numel()
    zd = z.double()
    if act == "gelu":
        terms = (0.5 * torch.erfc(-zd / 2 ** 0.5), zd * torch.exp(-0.5 * zd * zd) / (2 * torch.pi) ** 0.5)
    else:
        c = 2 * (2 / torch.pi) ** 0.5
        arg, slope = (zd, 1.0) if act == "silu" else (c * (zd + 0.044715 * zd ** 3), c * (1 + 3 * 0.044715 * zd * zd))
        p = torch.sigmoid(arg)
        terms = (p, zd * p * torch.sigmoid(-arg) * slope)
    want, size = sum(terms), sum(t.abs() for t in terms)
    w = torch.diag(torch.full((n,), 127, dtype=torch.int8)).cuda()
    one = torch.ones(n, device="cuda")
    for rows in (range(0, n, n // 40), range(n)):   # weight streaming and tiles
        rows = torch.tensor(list(rows))
        m = rows.numel()
        dy = torch.zeros((m, n), dtype=torch.bfloat16)
        dy[torch.arange(m), rows] = 1.0
        a = torch.zeros((m, n), dtype=torch.int8)
        dx, _ = ext.w8a8_linear_backward(dy.cuda(), a.cuda(), w, one[:m].contiguous(), one, z.to(torch.bfloat16).cuda(), act)
        got = dx.cpu().double()[torch.arange(m), rows] / 127
        err = (got - want[rows]).abs()
        assert (err <= ref.UBF * want[rows].abs() + 1.01 * 2.0 ** -15 * size[rows]).all(), float((err / size[rows]).max())


def test_directional_difference_of_the_forward(ext):
    """dx and dbias of the kernels against central differences of the 64-bit forward, in the dequantised activations"""
    m, i, k, h = 9, 40, 96, 1e-5
    (a, sa), (w, sw) = ref.tokens(m, k, 1), ref.weight(2 * i, k, 2)
    b, dh = ref.bf16((2 * i,), 3), ref.bf16((m, i), 4)
    x, wd = a.double() * sa.double(), w.double() * sw.double()[:, None]
    v, vb = torch.randn(m, k, dtype=torch.float64), torch.randn(2 * i, dtype=torch.float64)
    for act in ref.GATED_ACTS[:3]:
        def f(t):
            z = (x + t * v) @ wd.T + b.double() + t * vb
            return (ref.act(z[:, :i], act) * z[:, i:] * dh.double()).sum()
        dx, db = ext.w8a8_gated_backward(dh.cuda(), *cuda(a, w, sa, sw, b), act)
        got = (dx.cpu().double() * v).sum() + (db.cpu().double() * vb).sum()
        assert (got - (f(h) - f(-h)) / (2 * h)).abs() <= 2 * ref.UBF * (dx.cpu().double() * v).abs().sum() + 1e-4


def test_empty_batches_and_refusals(ext):
    (a, sa), (w, sw) = ref.tokens(4, 64, 1), ref.weight(32, 64, 2)
    a, sa, w, sw = cuda(a, sa, w, sw)
    b = torch.zeros(32, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros((4, 32), dtype=torch.bfloat16, device="cuda")
    dx, db = ext.w8a8_linear_backward(dy[:0], a[:0], w, sa[:0], sw, b, "gelu")
    assert dx.shape == (0, 64) and (db == 0).all() and db.shape == (32,)
    dx, db = ext.w8a8_linear_backward(dy, a, w, sa, sw, b, "none")
    assert (dx == 0).all() and (db == 0).all()
    for bad in (dy[:, :16], dy[:3], dy.float(), dy.cpu(), dy[0].expand(4, 32)):
        with pytest.raises(RuntimeError):
            ext.w8a8_linear_backward(bad, a, w, sa, sw)
    with pytest.raises(RuntimeError):
        ext.w8a8_gated_backward(dy, a, w, sa, sw)            # [4, 16] wanted
    with pytest.raises(RuntimeError, match="activation"):
        ext.w8a8_gated_backward(dy[:, :16], a, w, sa, sw, None, "none")


def test_more_rows_than_a_grid_dimension_of_row_blocks(ext):
    """2.1 million rows: 65536 blocks of 32"""
    m, n, k = 65536 * 32 + 5, 16, 16
    (w, sw) = ref.weight(n, k, 2)
    g = torch.Generator(device="cuda").manual_seed(1)
    a = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    sa = torch.rand((m, 1), generator=g, device="cuda") * 0.02
    dy = torch.randn((m, n), generator=g, device="cuda").to(torch.bfloat16)
    b = ref.bf16((n,), 3)
    dx, db = ext.w8a8_linear_backward(dy, a, *(t.cuda() for t in (w,)), sa, sw.cuda(), b.cuda(), "silu")
    pick = torch.tensor([0, 1, 31, 32, 65535 * 32 - 1, 65535 * 32, 65536 * 32 - 1, 65536 * 32, m - 1])
    want = ref.linear_backward(dy.cpu()[pick], a.cpu()[pick], sa.cpu()[pick], w, sw, b, "silu")[0]
    assert ((dx.cpu()[pick].double() - want).norm(dim=1) <= 4e-3 * want.norm(dim=1)).all()
    dz = (dy.double() * ref.dact((a.double() @ w.cuda().double().T) * sa.double() * sw.cuda().double() + b.cuda().double(), "silu"))
    # 65537 block sums in sixteen chains of at most 4097 additions, 32 rows each
    assert ((db.double() - dz.sum(0)).abs() <= U * (4097 + 60) * dz.abs().sum(0)).all()


@pytest.mark.parametrize("m,i,k", [(200, 136, 272), (16, 700, 528), (700, 136, 272)])
def test_two_runs_other_streams_and_captured_replays(ext, m, i, k):
    (a, sa), (w, sw) = ref.tokens(m, k, 1), ref.weight(2 * i, k, 2)
    b = ref.bf16((2 * i,), 3)
    a, sa, w, sw, b = cuda(a, sa, w, sw, b)
    dh = ref.bf16((m, i), 4).cuda()
    want = ext.w8a8_gated_backward(dh, a, w, sa, sw, b)
    again = ext.w8a8_gated_backward(dh, a, w, sa, sw, b)
    assert all(torch.equal(p, q) for p, q in zip(want, again))
    torch.cuda.synchronize()
    side, outs = torch.cuda.Stream(), []
    for _ in range(10):
        outs.append(ext.w8a8_gated_backward_stream(dh, a, w, sa, sw, b, "silu", side.cuda_stream))
        torch.full((8 << 20,), 77, dtype=torch.uint8, device="cuda")   # would land in a workspace freed to this stream
    side.synchronize()
    assert all(torch.equal(p, q) for o in outs for p, q in zip(want, o))
    graphs = []
    for _ in range(2):   # two graphs alive at once, replayed alternately
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ext.w8a8_gated_backward(dh, a, w, sa, sw, b)
            lin = ext.w8a8_linear_backward(dh, a, w[:i], sa, sw[:i], b[:i], "none")
        graphs.append((graph, out, lin))
    for seed in (11, 12, 13):
        dh.copy_(ref.bf16((m, i), seed))
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = ext.w8a8_gated_backward(dh, a, w, sa, sw, b)
        lin64 = ext.w8a8_linear_backward(dh, a, w[:i], sa, sw[:i], b[:i], "none")
        for _, out, lin in graphs:
            assert all(torch.equal(p, q) for p, q in zip(want, out))
            assert all(torch.equal(p, q) for p, q in zip(lin64, lin))
    assert ext.device_status() == 0
