"""Work-groups that take several units one behind the other, in the configurations of the largest weights, and zero points of a whole byte: against the definition in
64 bits, within the bounds of w4_reference.py."""
import copy
import ctypes

import numpy as np
import pytest
import torch

import gemm_mmbo_amd as G
import w4_reference as R
from gemm_mmbo_amd import api
from test_moe import Problem, _check

F16, BF16 = G.F16, G.BF16


def _gemm_on_gpu(dtype, w, b, alpha, beta, c):
    """w4_reference.gemm for large weights: in 64 bits on the GPU, device tensors."""
    def spread(v):
        return v.double().repeat_interleave(w.group, 1)[:, :w.k]

    q = w.q.cuda()
    code, s = torch.stack((q & 15, q >> 4), -1).flatten(-2)[:, :w.k].double(), spread(w.scales.cuda())
    z = spread(w.zeros.cuda()) if w.zeros is not None else 8.0
    b = b.cuda().double()
    exact = alpha * (b @ ((code - z) * s).t().contiguous()) + beta * c.cuda().double()
    off = abs(alpha) * (R.depth(w.k) + 4) * 2 * R.U * (b.abs() @ ((code + z + 256) * s).t().contiguous()) + 4 * R.U * exact.abs() + 2 * R.U * abs(beta) * c.cuda().double().abs()
    return exact, off + R.half_step(dtype) * (exact.abs() + off) + R.smallest(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 3, 16, 32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_several_units_to_a_work_group(dtype, n, zeros, group):
    """Two tiles of rows to a unit (from 8192 rows on), 1101 units for at most 512 work-groups, the last of 13 rows; k of 16 whole blocks, and of 16 and 35 places."""
    m = 32 * 1100 + 13
    for k in (2048, 2083):
        g = torch.Generator().manual_seed(n + k + group)
        w = R.Weight(g, dtype, m, k, group, zeros)
        b = torch.randn((n, k), generator=g).to(R.TORCH[dtype])
        c = torch.randn((n, m), generator=g).to(R.TORCH[dtype])
        exact, bound = _gemm_on_gpu(dtype, w, b, -0.5, 0.75, c)
        out = c.cuda()
        q, s, z, db = w.q.cuda(), w.scales.cuda(), w.zeros.cuda() if zeros else None, b.cuda()
        torch.cuda.synchronize()
        G.gemm_w4(dtype, m, n, k, group, -0.5, q, w.ldq, s, w.lds, z, w.lds, db, k, 0.75, out, m)
        torch.cuda.synchronize()
        worst = ((out.double() - exact).abs() / bound).max().item()
        assert worst <= 1.0, f"k {k}: {worst:.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("tokens", [3, 20])
def test_several_units_of_a_layer_to_a_work_group(dtype, group, tokens):
    """63 tiles of h for 12 jobs and more, at most 512 work-groups; several blocks of k to a wavefront in both products, the last one cut."""
    _check(Problem(dtype, tokens, 1403, 1001, 16, 4, group, zeros=True))


def _byte_zeros(w, g):
    """(w with zero points of all 8 bits, of which the low seven count; w as it counts)."""
    w.zeros[:] = torch.randint(0, 256, w.zeros.shape, generator=g, dtype=torch.uint8)
    counts = copy.copy(w)
    counts.zeros = w.zeros & 127
    return counts


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 4, 16, 32, "16 rows", "32 rows", "64 x 64", "256 x 128"])
def test_zero_points_of_a_byte(dtype, group, n):
    """Codes far from their zero points, up to 127, with the eighth bit set or not: every kernel, and weights taken back from 4 bits."""
    m, k = 90, 333
    kernel = ["16 rows", "32 rows", "64 x 64", "256 x 128"].index(n) if isinstance(n, str) else None
    n = 50 if kernel is not None else n
    g = torch.Generator().manual_seed(group + n)
    w = R.Weight(g, dtype, m, k, group, True)
    counts = _byte_zeros(w, g)
    b = torch.randn((n, k), generator=g).to(R.TORCH[dtype])
    exact, bound = R.gemm(dtype, counts, b, 1.0, 0.0, None)
    q, s, z, db = w.q.cuda(), w.scales.cuda(), w.zeros.cuda(), b.cuda()
    out = torch.empty((n, m), dtype=b.dtype, device="cuda")
    back = torch.empty((m, k), dtype=b.dtype, device="cuda")
    torch.cuda.synchronize()
    if kernel is None:
        G.gemm_w4(dtype, m, n, k, group, 1.0, q, w.ldq, s, w.lds, z, w.lds, db, k, 0.0, out, m)
    else:
        f = api.lib().mmbo_internal_gemm_w4
        f.argtypes = [ctypes.c_int, ctypes.c_int] + [ctypes.c_size_t] * 4 + [ctypes.c_void_p] * 6
        assert f(kernel, dtype, m, n, k, group, q.data_ptr(), s.data_ptr(), z.data_ptr(), db.data_ptr(), out.data_ptr(), None) == 0
    G.w4_dequantize(dtype, m, k, group, q, w.ldq, s, w.lds, z, w.lds, back, k)
    torch.cuda.synchronize()
    assert (np.abs(out.cpu().double().numpy() - exact) <= bound).all()
    value = counts.parts()[0]                                       # (a whole number of 8 bits times a scale of 11: exact in fp32)
    assert torch.equal(back.cpu(), torch.from_numpy(value).float().to(b.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 4, 20])
def test_zero_points_of_a_byte_in_a_layer(dtype, group, tokens):
    p = Problem(dtype, tokens, 150, 70, 5, 2, group, zeros=True)
    g = torch.Generator().manual_seed(tokens)
    for w in (p.gate_up, p.down):
        w.scales *= 0.125                                           # (weights of the size of other tests')
    counts = copy.copy(p)
    counts.gate_up, counts.down = _byte_zeros(p.gate_up, g), _byte_zeros(p.down, g)
    exact, bound, ids, _ = counts.exact()
    y, got_ids, _ = p.run()
    assert np.array_equal(got_ids, ids) and (np.abs(y.double().numpy() - exact) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,m,n,k", [(F16, 2 ** 22 + 37, 1, 40), (BF16, 2 ** 22 + 37, 3, 40), (F16, 2 ** 22 + 5, 40, 32), (BF16, 20, 2 ** 16 + 19, 70), (F16, 300, 2 ** 16 + 1, 33)])
def test_more_rows_or_columns_than_one_launch_takes(dtype, m, n, k):
    g = torch.Generator().manual_seed(n)
    w = R.Weight(g, dtype, m, k, 32, True)
    b = torch.randn((n, k), generator=g).to(R.TORCH[dtype])
    c = torch.randn((n, m + 1), generator=g).to(R.TORCH[dtype])
    exact, bound = _gemm_on_gpu(dtype, w, b, 0.5, -1.0, c[:, :m])
    out = c.cuda()
    q, s, z, db = w.q.cuda(), w.scales.cuda(), w.zeros.cuda(), b.cuda()
    torch.cuda.synchronize()
    G.gemm_w4(dtype, m, n, k, 32, 0.5, q, w.ldq, s, w.lds, z, w.lds, db, k, -1.0, out, m + 1)
    torch.cuda.synchronize()
    worst = ((out[:, :m].double() - exact).abs() / bound).max().item()
    assert worst <= 1.0 and torch.equal(out[:, m].cpu(), c[:, m]), f"{worst:.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("tokens", [64, 130])
def test_most_pairs_and_jobs(group, tokens):
    """2048 pairs to 64 tokens, of 512 experts: the largest table, beside the fewest wavefronts."""
    for dtype in (F16, BF16):
        _check(Problem(dtype, tokens, 40, 24, G.MOE_MAX_EXPERTS, G.MOE_MAX_TOP_K, group, zeros=True))
