"""GPU: single-tile products of 8-bit codes through TMA + tcgen05, in the operand arrangements that the attention over
8-bit blocks uses.  Products of two codes are exact, and so are the sums here up to fp32's rounding."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", [6, 7])
def test_umma_f8_tile(lib, mode):
    g = torch.Generator().manual_seed(mode)
    if mode == 6:
        a = torch.randn(128, 128, generator=g).mul(16).to(torch.float8_e4m3fn)
        b = torch.randn(32, 128, generator=g).to(torch.float8_e4m3fn)
        ref = a.double() @ b.double().t()
        size = a.double().abs() @ b.double().abs().t()
    else:
        a = torch.randn(128, 128, generator=g).mul(16).to(torch.float8_e4m3fn)     # At: (K rows, M)
        b = torch.randn(128, 32, generator=g).exp().to(torch.float8_e5m2)          # Bt: (K rows, N)
        ref = a.double().t() @ b.double()
        size = a.double().abs().t() @ b.double().abs()
    d = torch.full((128, 32), float("nan"), device="cuda")
    status = torch.zeros(4, dtype=torch.int32, device="cuda")
    a_d, b_d = a.cuda(), b.cuda()
    fn = lib.ifv2_selftest_umma
    fn.argtypes = [ctypes.c_int] + [ctypes.c_void_p] * 5
    fn.restype = ctypes.c_int
    rc = fn(mode, a_d.data_ptr(), b_d.data_ptr(), d.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.ifv2_last_error()
    torch.cuda.synchronize()
    assert int(status[0]) == 0, f"bounded wait ran out at site {int(status[0])}"
    # 128 sums of exact products: at most 128 half-steps of 2^-24 of the sum of magnitudes
    assert bool(((d.cpu().double() - ref).abs() <= 128 * 2.0 ** -24 * size).all()), float(((d.cpu().double() - ref).abs() / size).max())
