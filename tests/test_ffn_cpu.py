"""What can be checked of the feed-forward operators without a GPU: the 64-bit formulas that the GPU tests compare with
(against differences and autograd), the arithmetic of the gradient digits, argument checks, and the blocks' wiring."""
import ctypes

import pytest
import torch

import bw1000_dsv4_kernels_b200 as pkg
from bw1000_dsv4_kernels_b200 import ffn
from tests import ffn_reference as ref


@pytest.mark.parametrize("name", ref.ACTS)
def test_activation_slopes_match_differences(name):
    z = torch.linspace(-6, 6, 241, dtype=torch.float64) + 0.0123
    h = 1e-6
    assert ((ref.act(z + h, name) - ref.act(z - h, name)) / (2 * h) - ref.dact(z, name)).abs().max() < 1e-8


@pytest.mark.parametrize("name", ref.GATED_ACTS)
def test_gated_and_linear_gradients_match_autograd(name):
    (a, sa), (w, sw) = ref.tokens(5, 16, 1), ref.weight(12, 16, 2)
    b, dh, dy = ref.bf16((12,), 3), ref.bf16((5, 6), 4), ref.bf16((5, 12), 5)
    x = (a.double() * sa.double()).requires_grad_()
    bb = b.double().requires_grad_()
    z = x @ (w.double() * sw.double()[:, None]).T + bb
    gx, gb = torch.autograd.grad((ref.act(z[:, :6], name) * z[:, 6:] * dh.double()).sum(), (x, bb), retain_graph=True)
    dx, db, _, _ = ref.gated_backward(dh, a, sa, w, sw, b, name)
    assert (dx - gx).abs().max() < 1e-12 and (db - gb).abs().max() < 1e-12
    gx, gb = torch.autograd.grad((ref.act(z, name) * dy.double()).sum(), (x, bb))
    dx, db, _, _ = ref.linear_backward(dy, a, sa, w, sw, b, name)
    assert (dx - gx).abs().max() < 1e-12 and (db - gb).abs().max() < 1e-12


def test_layernorm_gradients_match_differences():
    x, w, b, dy = (torch.randn(4, 9, dtype=torch.float64) for _ in range(4))
    w, b = w[0], b[0]
    _, mean, rstd = ref.layernorm(x, w, b, 1e-6)
    dx, dw, db = ref.layernorm_backward(dy, x, mean, rstd, w)
    for (v, vw, vb) in [(torch.randn(4, 9, dtype=torch.float64), torch.randn(9, dtype=torch.float64),
                         torch.randn(9, dtype=torch.float64)) for _ in range(3)]:
        def f(t):
            return (ref.layernorm(x + t * v, w + t * vw, b + t * vb, 1e-6)[0] * dy).sum()
        slope = (f(1e-6) - f(-1e-6)) / 2e-6
        assert abs(float((dx * v).sum() + (dw * vw).sum() + (db * vb).sum() - slope)) < 1e-6


def test_every_digit_pair_is_int8_and_gives_its_value_back():
    v = torch.arange(-32639, 32640)
    hi = (v + 128) >> 8
    lo = v - (hi << 8)
    assert hi.min() >= -127 and hi.max() <= 127 and lo.min() >= -128 and lo.max() <= 127
    assert torch.equal(256 * hi + lo, v)
    # the largest sums of either digit stay below 2^31 for the most weight rows that the entry points take
    assert 131071 * 128 * 128 < 2 ** 31


def test_three_digits_are_the_bytes_of_a_shifted_sum():
    """w = 65536 hi + 256 mid + lo with signed digits: the bytes of w + 0x8080 are hi, mid + 128 and lo + 128 (mod 256)"""
    top = 32639 * 256
    w = torch.cat([torch.arange(-32639, 32640) * 256, torch.arange(-top - 2, top + 3, 61), torch.tensor([-top - 2, top + 2])])
    s = w + 0x8080
    signed = lambda b: torch.where(b >= 128, b - 256, b)   # noqa: E731
    hi, mid, lo = signed((s >> 16) & 255), signed(((s >> 8) & 255) ^ 128), signed((s & 255) ^ 128)
    assert torch.equal(65536 * hi + 256 * mid + lo, w)
    assert hi.abs().max() <= 127 and (lo[:2 * 32639 + 1] == 0).all()


def test_c_abi_refuses_before_it_touches_a_device():
    lib = pkg.c_abi()
    lib.dsv4_last_error.restype = ctypes.c_char_p
    lib.dsv4_w8a8_backward_workspace.restype = ctypes.c_int64
    lib.dsv4_layernorm_backward_workspace.restype = ctypes.c_int64
    null, one, odd = ctypes.c_void_p(0), ctypes.c_void_p(16), ctypes.c_void_p(24)
    ll, f = ctypes.c_longlong, ctypes.c_float
    err = lambda: lib.dsv4_last_error()   # noqa: E731
    linear = lambda **k: lib.launch_w8a8_linear(*[k.get(n, d) for n, d in (   # noqa: E731
        ("A", one), ("B", one), ("sa", one), ("sb", one), ("bias", null), ("act", 0), ("res", null), ("ldr", ll(0)),
        ("C", one), ("ldc", ll(8)), ("M", 4), ("N", 8), ("K", 32), ("st", null))])
    assert linear(M=0) == 0 and linear(N=0) == 0
    for bad, word in ((dict(act=5), b"activation"), (dict(act=-1), b"activation"), (dict(res=one, ldr=ll(7)), b"stride"),
                      (dict(K=24), b"multiple of 16"), (dict(K=0), b"positive"), (dict(A=odd), b"aligned"),
                      (dict(C=null), b"null"), (dict(sb=null), b"null"), (dict(ldc=ll(4)), b"ldc"), (dict(M=-1), b"negative")):
        assert linear(**bad) == 1 and word in err(), (bad, err())
    gated = lambda **k: lib.launch_w8a8_gated(*[k.get(n, d) for n, d in (   # noqa: E731
        ("A", one), ("B", one), ("sa", one), ("sb", one), ("bias", null), ("act", 4), ("C", one), ("ldc", ll(8)), ("M", 4),
        ("I", 8), ("K", 32), ("st", null))])
    assert gated(M=0) == 0
    for bad, word in ((dict(act=0), b"activation"), (dict(I=2 ** 30), b"int32"), (dict(K=8), b"multiple of 16")):
        assert gated(**bad) == 1 and word in err()
    size = lib.dsv4_w8a8_backward_workspace(4, 8, 0, 2, 1)
    assert size > 2 * 4 * 16 + 4 * 4 * 8 and lib.dsv4_w8a8_backward_workspace(0, 8, 0, 2, 1) == 0
    back = lambda **k: lib.launch_w8a8_linear_backward(*[k.get(n, d) for n, d in (   # noqa: E731
        ("dy", one), ("ldy", ll(8)), ("A", one), ("B", one), ("sa", one), ("sb", one), ("bias", null), ("act", 2), ("dx", one),
        ("db", one), ("ws", one), ("bytes", ll(size)), ("M", 4), ("N", 8), ("K", 32), ("st", null))])
    for bad, word in ((dict(act=9), b"activation"), (dict(ldy=ll(7)), b"stride"), (dict(K=40), b"multiple of 16"),
                      (dict(N=131072, ldy=ll(131072)), b"131071"), (dict(bytes=ll(size - 1)), b"workspace"), (dict(ws=odd), b"workspace"),
                      (dict(ws=null), b"null"), (dict(A=null), b"null"), (dict(dx=null), b"null"), (dict(B=odd), b"aligned"),
                      (dict(M=-2), b"negative")):
        assert back(**bad) == 1 and word in err(), (bad, err())
    norm = lambda **k: lib.launch_layernorm(*[k.get(n, d) for n, d in (   # noqa: E731
        ("res", null), ("x", one), ("w", one), ("b", one), ("y", one), ("mean", one), ("rstd", one), ("M", 4), ("N", 8),
        ("eps", f(1e-6)), ("st", null))])
    assert norm(M=0) == 0
    for bad in (dict(x=null), dict(w=null), dict(b=null), dict(y=null), dict(mean=null), dict(rstd=null), dict(N=0), dict(M=-1)):
        assert norm(**bad) == 1
    size = lib.dsv4_layernorm_backward_workspace(4, 8)
    assert size == 4 * 2 * 8 * 4 and lib.dsv4_layernorm_backward_workspace(4, 0) == 0
    nback = lambda **k: lib.launch_layernorm_backward(*[k.get(n, d) for n, d in (   # noqa: E731
        ("dy", one), ("x", one), ("mean", one), ("rstd", one), ("w", one), ("dres", null), ("dx", one), ("dw", one), ("db", one),
        ("ws", one), ("bytes", ll(size)), ("M", 4), ("N", 8), ("st", null))])
    for bad in (dict(dy=null), dict(ws=null), dict(bytes=ll(size - 1)), dict(dw=null), dict(N=0), dict(N=-1)):
        assert nback(**bad) == 1


def test_layernorm_backward_refuses_a_workspace_that_its_stores_do_not_fit():
    """shares of the column sums are stored eight bytes at a time, so four-byte alignment is not enough"""
    lib = pkg.c_abi()
    lib.dsv4_last_error.restype = ctypes.c_char_p
    lib.dsv4_layernorm_backward_workspace.restype = ctypes.c_int64
    one, null = ctypes.c_void_p(16), ctypes.c_void_p(0)
    size = lib.dsv4_layernorm_backward_workspace(4, 8)

    for offset in (1, 2, 4, 8, 12):
        rc = lib.launch_layernorm_backward(one, one, one, one, one, null, one, one, one, ctypes.c_void_p(4096 + offset),
                                           ctypes.c_longlong(size), 4, 8, null)
        assert rc == 1 and b"16-byte aligned" in lib.dsv4_last_error(), (offset, rc, lib.dsv4_last_error())


def test_operators_refuse_cpu_tensors():
    ext = pkg.dsv4_native_ext
    (a, sa), (w, sw) = ref.tokens(2, 16, 1), ref.weight(4, 16, 2)
    x, v = ref.bf16((2, 16), 3), ref.bf16((16,), 4)
    for call in (lambda: ext.w8a8_linear(a, w, sa, sw), lambda: ext.w8a8_gated(a, w, sa, sw),
                 lambda: ext.w8a8_linear_backward(x, a, w, sa, sw), lambda: ext.w8a8_gated_backward(x, a, w, sa, sw),
                 lambda: ext.layernorm(x, v, v, 1e-6), lambda: ext.add_layernorm(x, x, v, v, 1e-6),
                 lambda: ext.layernorm_quant(x, v, v, 1e-6), lambda: ext.add_layernorm_quant(x, x, v, v, 1e-6),
                 lambda: ext.layernorm_backward(x, x, sa, sa, v)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for name in ("w8a8_linear", "w8a8_linear_backward", "w8a8_gated", "w8a8_gated_backward", "layernorm", "add_layernorm",
                 "layernorm_quant", "add_layernorm_quant", "layernorm_backward"):
        assert hasattr(ext, name + "_stream")


def test_blocks_refuse_weights_that_do_not_belong_together():
    (w1, s1), (w2, s2) = ref.weight(32, 64, 1), ref.weight(64, 32, 2)
    ffn.W8A8FFN(w1, s1, w2, s2)
    ffn.W8A8GatedFFN(w1, s1, w2[:, :16].contiguous(), s2)
    with pytest.raises(ValueError):
        ffn.W8A8GatedFFN(w1, s1, w2, s2)
    with pytest.raises(ValueError):
        ffn.W8A8FFN(w1, s1, w2[:48], s2[:48])
