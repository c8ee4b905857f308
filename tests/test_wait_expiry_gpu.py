"""The give-up path of the GEMM kernels' bounded waits, exercised without a fault or a hang: a
test hook of the library launches the real kernel with its tile producer switched off and a wait
limit of one millisecond, so every consumer wait of the launch runs out.  The kernel has to record
the wait site, leave through its normal teardown and return; the next ordinary launch reports the
failure once; and a GEMM after that is correct, which also shows that tensor memory was freed
(its allocation would not return otherwise)."""
import ctypes
import time

import pytest
import torch

from oracle import cpu as oracle
from tests import workloads as wl

pytestmark = pytest.mark.gpu

DSV4_ERR_DEVICE_WAIT = 4
WAIT_SITES = {101, 102, 103, 104}


def _operands(m, n, k, seed):
    return (wl.int8_weights((m, k), seed=seed), wl.int8_weights((n, k), seed=seed + 1),
            wl.channel_scales((m,), seed=seed + 2), wl.channel_scales((n,), seed=seed + 3))


@pytest.mark.parametrize("m,n,k,grouped", [
    (2048, 2560, 256, False),   # CTA-pair kernel (80 tiles)
    (300, 512, 256, False),     # one CTA per tile, dense
    (300, 256, 256, True),      # one CTA per tile, grouped over two expert segments
])
def test_bounded_waits_give_up_and_report(cabi, m, n, k, grouped):
    lib = cabi.lib()
    assert cabi.device_status() == 0
    A, B, sa, sb = _operands(m, n, k, seed=m + n)
    Ad, sad = A.cuda(), sa.cuda()
    if grouped:
        off = torch.tensor([0, 130, m], dtype=torch.int32, device="cuda")
        Bd = torch.stack([B, wl.int8_weights((n, k), seed=99)]).cuda()
        sbd = torch.stack([sb, wl.channel_scales((n,), seed=98)]).cuda()
        off_p, e = ctypes.c_void_p(off.data_ptr()), 2
    else:
        Bd, sbd, off_p, e = B.cuda(), sb.cuda(), ctypes.c_void_p(0), 1
    C = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: ctypes.c_void_p(t.data_ptr())

    torch.cuda.synchronize()
    t0 = time.perf_counter()
    rc = lib.dsv4_test_gemm_wait_expiry(p(Ad), p(Bd), p(sad), p(sbd), p(C), m, n, k, off_p, e,
                                        ctypes.c_ulonglong(1_000_000), stream)
    assert rc == 0, cabi.last_error()
    torch.cuda.synchronize()                       # the kernel returns by itself
    assert time.perf_counter() - t0 < 5.0
    assert (C == 7.0).all(), "a launch without operand loads must not write its output"

    # the next ordinary launch on the device refuses once, with the wait site in its message ...
    C2 = torch.empty((m, n), dtype=torch.bfloat16, device="cuda")
    rc = lib.launch_w8a8_gemm(p(Ad), p(B.cuda()), p(sad), p(sb.cuda()), p(C2), m, n, k, stream)
    assert rc == DSV4_ERR_DEVICE_WAIT
    assert "bounded wait" in cabi.last_error()
    # ... the status word holds the site until it is read, and is clear afterwards
    assert cabi.device_status() in WAIT_SITES
    assert cabi.device_status() == 0
    # ... and the device is fine: tensor memory was released and the same kernels give the oracle's bits
    got = cabi.w8a8_gemm(Ad, B.cuda(), sad, sb.cuda())
    torch.cuda.synchronize()
    ref = oracle.w8a8_gemm(A, B, sa, sb)
    assert torch.equal(got.cpu().view(torch.int16), ref.view(torch.int16))
    assert cabi.device_status() == 0


def _refused_once_and_clear(cabi, launch):
    """the next launch on the device refuses once, and the status word holds the site until it is read"""
    assert launch() == DSV4_ERR_DEVICE_WAIT and "bounded wait" in cabi.last_error()
    assert cabi.device_status() in WAIT_SITES
    assert cabi.device_status() == 0
    assert launch() == 0, cabi.last_error()
    torch.cuda.synchronize()
    assert cabi.device_status() == 0


@pytest.mark.parametrize("act", [0, 2, 4])
def test_fused_epilogue_gives_up_and_reports(cabi, ext, act):
    m, n, k = 700, 5200, 256   # tiles of CTA pairs, more of them than pairs
    lib = cabi.lib()
    A, B, sa, sb = (t.cuda() for t in _operands(m, n, k, seed=act))
    C = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: ctypes.c_void_p(t.data_ptr())   # noqa: E731
    rc = lib.dsv4_test_linear_wait_expiry(p(A), p(B), p(sa), p(sb), act, p(C), m, n, k, ctypes.c_ulonglong(1_000_000), stream)
    assert rc == 0, cabi.last_error()
    torch.cuda.synchronize()
    assert (C == 7.0).all(), "a launch without operand loads must not write its output"
    _refused_once_and_clear(cabi, lambda: lib.launch_w8a8_linear(
        p(A), p(B), p(sa), p(sb), None, act, None, ctypes.c_longlong(0), p(C), ctypes.c_longlong(n), m, n, k, stream))
    want = ext.w8a8_linear(A, B, sa, sb, None, ("none", "relu", "gelu", "gelu_tanh", "silu")[act])
    assert torch.equal(C.view(torch.int16), want.view(torch.int16)) and not (C == 7.0).all()


@pytest.mark.parametrize("m,n,k,many", [(2048, 640, 2560, True), (16, 2048, 512, False), (100, 4096, 512, False)])
def test_gradient_product_gives_up_and_reports(cabi, ext, m, n, k, many):
    lib = cabi.lib()
    _, W, _, sb = (t.cuda() for t in _operands(m, n, k, seed=m))
    A, sa = torch.zeros((m, k), dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda")
    dy = wl.randn_bf16((m, n), seed=5).cuda()
    want = ext.w8a8_linear_backward(dy, A, W, sa, sb)[0]
    lib.dsv4_w8a8_backward_workspace.restype = ctypes.c_int64
    size = lib.dsv4_w8a8_backward_workspace(m, n, 0, 0, 0)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    dx = torch.full((m, k), 7.0, dtype=torch.bfloat16, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p, ll = (lambda t: ctypes.c_void_p(t.data_ptr())), ctypes.c_longlong
    rc = lib.dsv4_test_backward_wait_expiry(p(dy), p(W), p(sb), p(dx), p(ws), ll(size), m, n, k, ctypes.c_ulonglong(1_000_000), stream)
    assert rc == 0, cabi.last_error()
    torch.cuda.synchronize()
    if many:
        assert (dx == 7.0).all(), "a launch without operand loads must not write its output"
    # no GEMM is part of this backward pass: it has to look for itself
    _refused_once_and_clear(cabi, lambda: lib.launch_w8a8_linear_backward(
        p(dy), ll(n), p(A), p(W), p(sa), p(sb), None, 0, p(dx), None, p(ws), ll(size), m, n, k, stream))
    assert torch.equal(dx.view(torch.int16), want.view(torch.int16))


_FIRST_CALL = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import bw1000_dsv4_kernels_b200 as pkg
ext = pkg.dsv4_native_ext
g = torch.Generator(device="cuda").manual_seed(1)
m, n, k = 40, 320, 256
dy = torch.randn((m, n), generator=g, device="cuda").to(torch.bfloat16)
w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
a, sa, sb = torch.zeros((m, k), dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"), torch.rand(n, generator=g, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    dx, _ = ext.w8a8_linear_backward(dy, a, w, sa, sb)
    y = ext.w8a8_linear(a, w, sa, sb)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(dx, ext.w8a8_linear_backward(dy, a, w, sa, sb)[0]) and (y == 0).all() and ext.device_status() == 0
print("captured")
"""


def test_the_first_call_of_a_process_can_be_captured():
    """the host mirror of the status word is set up on the first call, without disturbing a capture"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", _FIRST_CALL, root], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]
