"""Products with 4-bit weights and their format: refusals (no GPU), and on the GPU every result against the definition in 64 bits, within bounds that rounding
allows (w4_reference.py)."""
import ctypes

import numpy as np
import pytest
import torch

import gemm_mmbo_amd as G
import w4_reference as R
from gemm_mmbo_amd import api

F32, F16, F64, BF16 = G.F32, G.F16, G.F64, G.BF16


def _gemm_status(dtype=F16, m=4, n=2, k=64, group=32, alpha=True, Q=16, ldq=64, scales=16, lds=2, zeros=None, ldz=0, B=16, ldb=64, beta=True, C=16, ldc=4):
    one = ctypes.c_float(1.0)
    p = ctypes.byref(one)
    return api.lib().mmbo_gemm_w4(dtype, m, n, k, group, p if alpha else None, Q, ldq, scales, lds, zeros, ldz, B, ldb, p if beta else None, C, ldc, None)


def _quantize_status(w_dtype=F16, dtype=F16, m=4, k=64, group=32, W=16, ldw=64, Q=16, ldq=64, scales=16, lds=2, zeros=None, ldz=0):
    return api.lib().mmbo_w4_quantize(w_dtype, dtype, m, k, group, W, ldw, Q, ldq, scales, lds, zeros, ldz, None)


def _dequantize_status(dtype=F16, m=4, k=64, group=32, Q=16, ldq=64, scales=16, lds=2, zeros=None, ldz=0, W=16, ldw=64):
    return api.lib().mmbo_w4_dequantize(dtype, m, k, group, Q, ldq, scales, lds, zeros, ldz, W, ldw, None)


WEIGHT_REFUSALS = [(dict(group=0), 3), (dict(group=16), 3), (dict(group=33), 3), (dict(group=2 ** 31), 3), (dict(ldq=63), 3), (dict(ldq=62), 3), (dict(ldq=2 ** 31), 3),
                   (dict(lds=1), 3), (dict(zeros=16, ldz=1), 3), (dict(m=2 ** 31), 3), (dict(k=2 ** 31), 3), (dict(dtype=F32), 1), (dict(dtype=F64), 1), (dict(dtype=7), 1),
                   (dict(Q=None), 4), (dict(scales=None), 4)]


@pytest.mark.parametrize("call", [_gemm_status, _quantize_status, _dequantize_status])
@pytest.mark.parametrize("change,status", WEIGHT_REFUSALS)
def test_weights_that_are_refused(call, change, status):
    assert call(**change) == status


@pytest.mark.parametrize("change,status", [(dict(n=2 ** 31), 3), (dict(ldb=63), 3), (dict(ldc=3), 3), (dict(ldb=2 ** 31), 3), (dict(ldc=2 ** 31), 3), (dict(alpha=False), 4),
                                           (dict(beta=False), 4), (dict(B=None), 4), (dict(C=None), 4)])
def test_products_that_are_refused(change, status):
    assert _gemm_status(**change) == status


def test_conversions_that_are_refused():
    assert _quantize_status(w_dtype=F64) == 1 and _quantize_status(w_dtype=9) == 1
    assert _quantize_status(ldw=63) == 3 and _dequantize_status(ldw=63) == 3
    assert _quantize_status(W=None) == 4 and _dequantize_status(W=None) == 4
    with pytest.raises(G.MmboError) as e:
        G.w4_quantize(F16, F16, 4, 64, 48, 16, 64, 16, 64, 16, 2)
    assert e.value.status == 3


def test_empty_calls_touch_nothing():
    assert _gemm_status(m=0, Q=None, C=None) == 0 and _gemm_status(n=0, B=None, C=None) == 0
    assert _quantize_status(m=0, W=None) == 0 and _quantize_status(k=0, W=None, Q=None) == 0 and _dequantize_status(k=0, W=None) == 0


def test_bf16_stays_with_the_calls_that_name_it():
    one = ctypes.c_float(1.0)
    assert api.lib().mmbo_gemm(BF16, 0, 0, 4, 4, 4, ctypes.byref(one), 16, 4, 16, 4, ctypes.byref(one), 16, 4, -1, None) == 1


# ---- on the GPU

def _run_gemm(dtype, w, b, c, alpha, beta, m, n, stream=None):
    """b [n, ldb], c [n, ldc] host tensors; the result as a host tensor."""
    q, s, z = w.q.cuda(), w.scales.cuda(), None if w.zeros is None else w.zeros.cuda()
    db, dc = b.cuda(), c.cuda()
    torch.cuda.synchronize()
    G.gemm_w4(dtype, m, n, w.k, w.group, alpha, q, w.ldq, s, w.lds, z, w.lds, db, b.shape[1], beta, dc, c.shape[1], stream)
    torch.cuda.synchronize()
    return dc.cpu()


def _close(got, exact, bound, label=""):
    got = got.double().numpy()
    fine = np.isfinite(exact)
    worst = np.max(np.abs(got - exact)[fine] / bound[fine]) if fine.any() else 0.0
    assert np.isfinite(got[fine]).all() and worst <= 1.0, f"{label}: {worst:.3g} of the bound"


def _problem(dtype, m, n, k, group, zeros=False, alpha=1.0, beta=0.0, pad=0, seed=0):
    g = torch.Generator().manual_seed(1000 * m + 10 * n + k + seed)
    w = R.Weight(g, dtype, m, k, group, zeros, pad_bytes=pad, pad_groups=pad)
    b = torch.randn((n, k + pad), generator=g).to(R.TORCH[dtype])
    c = torch.randn((n, m + pad), generator=g).to(R.TORCH[dtype]) if beta else torch.full((n, m + pad), float("nan"), dtype=R.TORCH[dtype])
    if pad:
        c[:, m:] = -7.0
    return w, b, c


def _check_gemm(dtype, m, n, k, group, zeros=False, alpha=1.0, beta=0.0, pad=0):
    w, b, c = _problem(dtype, m, n, k, group, zeros, alpha, beta, pad)
    got = _run_gemm(dtype, w, b, c, alpha, beta, m, n)
    exact, bound = R.gemm(dtype, w, b[:, :k], alpha, beta, c[:, :m])
    _close(got[:, :m], exact, bound, f"{m}x{n}x{k}")
    assert bool((got[:, m:] == -7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k,group", [
    (16, 1, 128, 128), (1, 1, 1, 32), (17, 1, 31, 32), (15, 2, 33, 32), (33, 1, 127, 64), (64, 3, 129, 32), (65, 15, 160, 96), (130, 16, 257, 128),
    (48, 17, 512, 64), (31, 32, 1000, 128), (100, 33, 384, 256), (80, 64, 515, 32), (129, 65, 300, 64), (257, 130, 1003, 128), (19, 7, 2048, 2048),
    (40, 1, 4100, 128), (16, 5, 8192, 4096), (300, 200, 640, 32)])
def test_products_against_the_definition(dtype, m, n, k, group):
    _check_gemm(dtype, m, n, k, group)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [1, 2, 9, 16, 24, 48, 64, 77, 144])
@pytest.mark.parametrize("pad", [0, 1, 5])
def test_products_with_zeros_scalars_and_rows_inside_larger_arrays(dtype, n, pad):
    _check_gemm(dtype, 77, n, 451, 32, zeros=True, alpha=-0.75, beta=0.5, pad=pad)
    _check_gemm(dtype, 50, n, 256, 128, zeros=True, alpha=1.25, beta=1.0, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kernel", [0, 1, 2, 3])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_every_kernel_for_many_columns(dtype, kernel, group):
    """Each of the kernels that a call with more than 32 columns may be given, on sizes that the pick gives to others too."""
    f = api.lib().mmbo_internal_gemm_w4
    f.argtypes = [ctypes.c_int, ctypes.c_int] + [ctypes.c_size_t] * 4 + [ctypes.c_void_p] * 6
    for m, n, k, zeros in ((300, 150, 384, True), (256, 128, 1024, False), (17, 33, 95, True), (70, 260, 640, True), (513, 40, 1003, False), (64, 64, 32, True)):
        w, b, c = _problem(dtype, m, n, k, group, zeros)
        q, s, z = w.q.cuda(), w.scales.cuda(), w.zeros.cuda() if zeros else None
        db, dc = b.cuda(), c.cuda()
        torch.cuda.synchronize()
        assert f(kernel, dtype, m, n, k, group, q.data_ptr(), s.data_ptr(), z.data_ptr() if zeros else None, db.data_ptr(), dc.data_ptr(), None) == 0
        torch.cuda.synchronize()
        exact, bound = R.gemm(dtype, w, b, 1.0, 0.0, c)
        _close(dc.cpu(), exact, bound, f"{m}x{n}x{k}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_no_k_gives_beta_c(dtype):
    for beta in (0.0, 0.5):
        w, b, c = _problem(dtype, 20, 3, 0, 32, beta=beta, pad=1)                # (a leading dimension is 1 at least)
        got = _run_gemm(dtype, w, b, c, 1.0, beta, 20, 3)
        want = beta * c[:, :20].double() if beta else torch.zeros((3, 20), dtype=torch.float64)
        assert torch.equal(got[:, :20].double(), want.to(R.TORCH[dtype]).double())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [2, 16, 40, 130])
def test_a_column_of_infinities_or_nan_reaches_no_other(dtype, n):
    w, b, c = _problem(dtype, 70, n, 300, 32, zeros=True)
    exact, bound = R.gemm(dtype, w, b, 1.0, 0.0, c)
    for bad in (float("nan"), float("inf"), -float("inf")):
        broken = b.clone()
        broken[n // 2, 299] = bad
        got = _run_gemm(dtype, w, broken, c, 1.0, 0.0, 70, n)
        others = [j for j in range(n) if j != n // 2]
        _close(got[others], exact[others], bound[others])
        hit = (R.codes_of(w.q, 300)[:, 299] != w.zeros[:, 9].double().numpy())
        assert not np.isfinite(got[n // 2].double().numpy()[hit]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n", [(F16, 1), (BF16, 20), (F16, 100)])
def test_bytes_behind_the_operands_are_not_used(dtype, n):
    """Rows of codes, columns of B and scales that end where the array ends: what lies behind (NaN) reaches nothing."""
    m, k, group = 37, 77, 32
    w, b, c = _problem(dtype, m, n, k, group)
    exact, bound = R.gemm(dtype, w, b, 1.0, 0.0, c)
    t = R.TORCH[dtype]
    q = torch.full((w.q.numel() + 64,), 255, dtype=torch.uint8)
    q[:w.q.numel()] = w.q.flatten()
    q[(torch.arange(m) + 1) * w.q.shape[1] - 1] |= 0xF0            # the unused half of a row's last byte
    nan_b, nan_s = torch.full((b.numel() + 64,), float("nan"), dtype=t), torch.full((w.scales.numel() + 64,), float("nan"), dtype=t)
    nan_b[:b.numel()], nan_s[:w.scales.numel()] = b.flatten(), w.scales.flatten()
    dc = c.cuda()
    G.gemm_w4(dtype, m, n, k, group, 1.0, q.cuda(), w.ldq, nan_s.cuda(), w.lds, None, 0, nan_b.cuda(), k, 0.0, dc, m)
    torch.cuda.synchronize()
    _close(dc.cpu(), exact, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n", [(F16, 1), (BF16, 33), (F16, 96)])
def test_offsets_past_32_bits(dtype, n):
    """Rows of codes a GiB apart and columns of C two GiB apart."""
    m, k, group = 6, 100, 32
    w, b, c = _problem(dtype, m, n, k, group)
    row = 2 ** 30 - 2
    far = torch.empty(row * (m - 1) + 64, dtype=torch.uint8, device="cuda")
    for i in range(m):
        far[i * row:i * row + 50] = w.q[i, :50].cuda()
    dc = c.cuda()
    torch.cuda.synchronize()
    G.gemm_w4(dtype, m, n, k, group, 1.0, far, 2 * row, w.scales.cuda(), w.lds, None, 0, b.cuda(), k, 0.0, dc, m)
    torch.cuda.synchronize()
    exact, bound = R.gemm(dtype, w, b, 1.0, 0.0, c)
    _close(dc.cpu(), exact, bound)
    del far
    if n > 1:
        n = 4
        col = 2 ** 30 + 3
        out = torch.empty(col * (n - 1) + 64, dtype=R.TORCH[dtype], device="cuda")
        G.gemm_w4(dtype, m, n, k, group, 1.0, w.q.cuda(), w.ldq, w.scales.cuda(), w.lds, None, 0, b.cuda(), k, 0.0, out, col)
        torch.cuda.synchronize()
        for j in range(n):
            _close(out[j * col:j * col + m].cpu()[None], exact[j:j + 1], bound[j:j + 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n", [(F16, 1), (BF16, 16), (BF16, 64), (F16, 200)])
def test_products_in_a_graph_and_on_two_streams(dtype, n):
    m, k, group = 96, 640, 64
    w, b, c = _problem(dtype, m, n, k, group, zeros=True)
    q, s, z = w.q.cuda(), w.scales.cuda(), w.zeros.cuda()
    db, dc = b.cuda(), c.cuda()

    def call(out, stream):
        G.gemm_w4(dtype, m, n, k, group, 1.0, q, w.ldq, s, w.lds, z, w.lds, db, k, 0.0, out, m, stream)

    call(dc, None)
    torch.cuda.synchronize()
    first = dc.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(dc, torch.cuda.current_stream())
    g = torch.Generator().manual_seed(5)
    for _ in range(3):
        db.copy_(torch.randn((n, k), generator=g).to(b.dtype))
        want = torch.empty_like(dc)
        call(want, torch.cuda.current_stream())
        dc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dc, want)
    db.copy_(b)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.empty_like(dc), torch.empty_like(dc)]
    torch.cuda.synchronize()
    for _ in range(4):
        for st, out in zip(streams, outs):
            call(out, st)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)


def _quantized(w, w_dtype, dtype, group, zeros, pad=0):
    m, k = w.shape
    groups = -(-k // group)
    dw = torch.full((m, k + pad), float("nan"), dtype=w.dtype)
    dw[:, :k] = w
    dw = dw.cuda()
    q = torch.full((m, (k + 1) // 2 + pad), 0xA5, dtype=torch.uint8, device="cuda")
    s = torch.full((m, groups + pad), 9.0, dtype=R.TORCH[dtype], device="cuda")
    z = torch.full((m, groups + pad), 77, dtype=torch.uint8, device="cuda") if zeros else None
    G.w4_quantize(w_dtype, dtype, m, k, group, dw, k + pad, q, 2 * q.shape[1], s, groups + pad, z, groups + pad)
    back = torch.full((m, k + pad), -7.0, dtype=R.TORCH[dtype], device="cuda")
    G.w4_dequantize(dtype, m, k, group, q, 2 * q.shape[1], s, groups + pad, z, groups + pad, back, k + pad)
    torch.cuda.synchronize()
    return q.cpu(), s.cpu(), None if z is None else z.cpu(), back.cpu()


def _check_quantized(w, w_dtype, dtype, group, zeros, pad=0):
    m, k = w.shape
    groups = -(-k // group)
    q, s, z, back = _quantized(w, w_dtype, dtype, group, zeros, pad)
    codes, scales, zs = R.quantize(w, dtype, group, zeros)
    assert torch.equal(s[:, :groups], scales) and bool((s[:, groups:] == 9.0).all())
    if zeros:
        assert np.array_equal(z[:, :groups].numpy(), zs) and bool((z[:, groups:] == 77).all())
    assert np.array_equal(R.codes_of(q, k), codes)
    used = (k + 1) // 2
    assert bool((q[:, used:] == 0xA5).all())
    if k % 2:
        assert bool((q[:, used - 1] >> 4 == 0).all())
    spread = np.repeat(scales.double().numpy(), group, 1)[:, :k]
    zero = np.repeat(zs, group, 1)[:, :k] if zeros else 8.0
    want = torch.from_numpy(((codes - zero) * spread).astype(np.float32)).to(R.TORCH[dtype])     # (15 bits: exact in fp32)
    assert torch.equal(back[:, :k], want) and bool((back[:, k:] == -7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("w_dtype,dtype", [(F16, F16), (BF16, BF16), (F32, F16), (F32, BF16), (F16, BF16), (BF16, F16)])
@pytest.mark.parametrize("zeros", [False, True])
def test_codes_are_those_of_the_definition(w_dtype, dtype, zeros):
    g = torch.Generator().manual_seed(3)
    for m, k, group, pad in ((1, 1, 32, 0), (7, 31, 32, 1), (33, 128, 64, 0), (20, 451, 96, 3), (5, 1000, 128, 0), (3, 300, 4096, 5), (300, 515, 32, 0)):
        w = (torch.randn((m, k), generator=g) * 0.3 + (0.2 if zeros else 0)).to(R.TORCH[w_dtype])
        _check_quantized(w, w_dtype, dtype, group, zeros, pad)


@pytest.mark.gpu
@pytest.mark.parametrize("w_dtype", [F32, F16, BF16])
@pytest.mark.parametrize("zeros", [False, True])
def test_codes_on_borders_and_of_extreme_weights(w_dtype, zeros):
    """Values half way between two codes, groups of zeros, the largest and smallest numbers, infinities and NaN."""
    t = R.TORCH[w_dtype]
    rows = [torch.arange(-15, 17).float() / 2,                                  # scale 15 / 14 or 1: many halves with zeros
            torch.zeros(32), torch.full((32,), 7.0), torch.full((32,), -7.0), (torch.arange(32).float() - 14) * 0.5,
            torch.full((32,), torch.finfo(t).max), torch.full((32,), -torch.finfo(t).max), torch.full((32,), torch.finfo(t).smallest_normal),
            torch.full((32,), torch.finfo(t).smallest_normal * torch.finfo(t).eps)]
    odd = torch.linspace(-3, 3, 32)
    for bad in (float("inf"), -float("inf"), float("nan")):
        v = odd.clone()
        v[5] = bad
        rows.append(v)
    rows.append(torch.full((32,), float("nan")))
    half = torch.linspace(-7, 7, 29)                                            # scale 1: every other value half way
    rows.append(torch.cat((half, half[:3])))
    w = torch.stack(rows).to(t)
    for dtype in (F16, BF16):
        _check_quantized(w, w_dtype, dtype, 32, zeros)
        _check_quantized(w.repeat(1, 3)[:, :75], w_dtype, dtype, 32, zeros)


@pytest.mark.gpu
def test_rounding_to_four_bits_and_multiplying():
    """The three calls as a program uses them: weights to 4 bits, a product with them, and the same product with what they became."""
    g = torch.Generator().manual_seed(8)
    m, n, k, group = 200, 12, 700, 64
    for dtype in (F16, BF16):
        w = (torch.randn((m, k), generator=g) / k ** 0.5).to(R.TORCH[dtype])
        b = torch.randn((n, k), generator=g).to(R.TORCH[dtype])
        for zeros in (False, True):
            q, s, z, back = _quantized(w, dtype, dtype, group, zeros)
            held = object.__new__(R.Weight)
            held.__dict__.update(k=k, group=group, groups=s.shape[1], q=q, scales=s, zeros=z, ldq=2 * q.shape[1], lds=s.shape[1])
            got = _run_gemm(dtype, held, b, torch.zeros((n, m), dtype=b.dtype), 1.0, 0.0, m, n)
            exact, bound = R.gemm(dtype, held, b, 1.0, 0.0, None)
            _close(got, exact, bound)
            # and near the product of the weights themselves: a code is off by half a scale at most, a scale by its rounding
            plain = b.double() @ w.double().t()
            step = torch.from_numpy(np.repeat(s.double().numpy(), group, 1)[:, :k])
            room = b.double().abs() @ (step * (0.5 + 8 * 2 * R.half_step(dtype))).t()
            assert bool(((got.double() - plain).abs() <= room + torch.from_numpy(bound)).all())
