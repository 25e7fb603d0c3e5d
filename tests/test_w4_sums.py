"""Products with 4-bit weights whose every term, (code - zero) * element, and whose sums of any of them are whole numbers below 2^23, a bit less than fp32 holds: whatever
the order, the sum in fp32 is exact, and the result is that sum times a power of two, with beta C, rounded once.  It has to be equal: what a kernel makes of the codes may not
cost the sums any of fp32's bits.  In numbers that stand for more than code - zero -- the code and 128, say, whose columns' sums then come off -- the sums pass 2^24."""
import ctypes

import numpy as np
import pytest
import torch

import gemm_mmbo_amd as G
import w4_reference as R
from gemm_mmbo_amd import api

F16, BF16 = G.F16, G.BF16
UNIT = {F16: 2.0 ** -8, BF16: 1.0}                  # alpha or the scales: fp16 ends at 65504


ELEMENTS = {"many": (4, 64, 1.0), "few": (32, 256, 2.0 ** -14)}      # every how many-th is large, 128 to 255 of what, the others' unit (fp16: the smallest normal number)


def _problem(dtype, m, n, k, group, zeros, elements="many"):
    """Weights of scale 1, columns whose runs of 128 have one sign and large elements among small odd ones, and the exact products, in units."""
    g = torch.Generator().manual_seed(m + n + k + group)
    w = R.Weight(g, dtype, m, k, group, zeros)
    w.scales[:] = 1.0
    every, step, unit = ELEMENTS[elements]
    b = torch.randint(0, 8, (n, k), generator=g) * 2 + 1
    b[:, ::every] = torch.randint(128, 256, b[:, ::every].shape, generator=g) * step    # 8 bits: exact in bf16
    b[:, (torch.arange(k) // 128) % 2 == 1] *= -1
    value = w.parts()[0]
    assert (np.abs(b.numpy()) @ np.abs(value).T).max() < 2 ** 23
    held = (b * unit).to(R.TORCH[dtype])
    assert torch.equal(held.double(), b.double() * unit)
    return w, held, b.double().numpy() @ value.T


def _rounded(v, dtype):
    assert np.array_equal(torch.from_numpy(v).float().double().numpy(), v)              # (exact in fp32: the type's rounding is the only one)
    return torch.from_numpy(v).to(R.TORCH[dtype]).double().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n", [1, 3, 16, 32, 40, 150])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("elements", ["many", "few"])
def test_sums_that_fp32_holds_are_exact(elements, dtype, n, zeros, group):
    """C takes off what the type has of the result, and the lowest bits remain."""
    for m, k in ((200, 256), (33, 201), (130, 64)):
        w, b, exact = _problem(dtype, m, n, k, group, zeros, elements)
        c = torch.from_numpy(-UNIT[dtype] * exact).to(R.TORCH[dtype])
        want = _rounded(UNIT[dtype] * exact + c.double().numpy(), dtype)
        q, s, z, db, dc = w.q.cuda(), w.scales.cuda(), None if w.zeros is None else w.zeros.cuda(), b.cuda(), c.cuda()
        torch.cuda.synchronize()
        G.gemm_w4(dtype, m, n, k, group, UNIT[dtype] / ELEMENTS[elements][2], q, w.ldq, s, w.lds, z, w.lds, db, k, 1.0, dc, m)
        torch.cuda.synchronize()
        off = dc.cpu().double().numpy() - want
        assert not off.any(), f"{m} x {n} x {k}: {np.mean(off != 0):.2g} of all, by up to {np.abs(off).max() / UNIT[dtype]} of {np.abs(exact).max()}"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel", [0, 1, 2, 3])
@pytest.mark.parametrize("elements", ["many", "few"])
def test_sums_that_fp32_holds_are_exact_in_every_kernel(elements, dtype, kernel):
    """Each of the kernels that a call with more than 32 columns may be given."""
    f = api.lib().mmbo_internal_gemm_w4
    f.argtypes = [ctypes.c_int, ctypes.c_int] + [ctypes.c_size_t] * 4 + [ctypes.c_void_p] * 6
    for group, zeros in ((32, True), (64, False), (128, True)):
        m, n, k = 170, 140, 250
        w, b, exact = _problem(dtype, m, n, k, group, zeros, elements)
        w.scales[:] = UNIT[dtype] / ELEMENTS[elements][2]
        want = _rounded(UNIT[dtype] * exact, dtype)
        q, s, z, db = w.q.cuda(), w.scales.cuda(), w.zeros.cuda() if zeros else None, b.cuda()
        dc = torch.full((n, m), float("nan"), dtype=R.TORCH[dtype], device="cuda")
        torch.cuda.synchronize()
        assert f(kernel, dtype, m, n, k, group, q.data_ptr(), s.data_ptr(), z.data_ptr() if zeros else None, db.data_ptr(), dc.data_ptr(), None) == 0
        torch.cuda.synchronize()
        off = dc.cpu().double().numpy() - want
        assert not off.any(), f"groups of {group}: {np.mean(off != 0):.2g} of all, by up to {np.abs(off).max() / UNIT[dtype]}"


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 3, 16, 32, 40, 150])
@pytest.mark.parametrize("zeros", [False, True])
def test_bf16_elements_up_to_2_to_the_114(n, zeros):
    """Sums of 128 places stay below 127 * 128 * 2^114 < 2^128.  With elements near that, codes near their zero points and small scales: results far below fp32's end."""
    m, k, group = 40, 384, 128
    g = torch.Generator().manual_seed(n)
    w = R.Weight(g, BF16, m, k, group, zeros)
    w.scales[:] = 2.0 ** -10
    code = torch.randint(7, 11, (m, k), generator=g)
    if zeros:
        w.zeros[:] = torch.randint(6, 12, w.zeros.shape, generator=g, dtype=torch.uint8)
        w.zeros[::5] = 127                                          # (the farthest: every term has one sign)
    w.q = (code[:, ::2] + 16 * code[:, 1::2]).to(torch.uint8)
    b = (torch.randint(240, 256, (n, k), generator=g) * 2.0 ** 106).bfloat16()              # just below 2^114
    exact, bound = R.gemm(BF16, w, b, 1.0, 0.0, None)
    q, s, z, db = w.q.cuda(), w.scales.cuda(), w.zeros.cuda() if zeros else None, b.cuda()
    dc = torch.empty((n, m), dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    G.gemm_w4(BF16, m, n, k, group, 1.0, q, w.ldq, s, w.lds, z, w.lds, db, k, 0.0, dc, m)
    torch.cuda.synchronize()
    got = dc.cpu().double().numpy()
    assert np.isfinite(got).all() and (np.abs(got - exact) <= bound).all()
