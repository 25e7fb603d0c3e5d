"""What the mixture-of-experts layer holds between its two products: h = silu(gate) * up has fp32's range and its 24 bits, whatever the layer's type."""
import numpy as np
import pytest
import torch

import gemm_mmbo_amd as G
import w4_reference as R

F16, BF16 = G.F16, G.BF16
U = R.U


class Layer:
    """One expert, with weights given as whole numbers times a power of two: in 16 bits, or in 4 (whole numbers -8 .. 7)."""

    def __init__(self, dtype, group, gate_up, gate_up_unit, down, down_unit):
        self.dtype, self.group = dtype, group
        self.inner, self.hidden = down.shape[1], down.shape[0]
        t = R.TORCH[dtype]

        def matrix(v, unit):
            rows, k = v.shape
            if not group:
                w = (v * unit).to(t)
                assert torch.equal(w.double(), v.double() * unit)
                return G.moe_matrix(w.cuda(), k, rows * k)
            code = torch.zeros((rows, (k + 1) // 2 * 2), dtype=torch.uint8)
            code[:, :k] = (v + 8).to(torch.uint8)
            groups = -(-k // group)
            scales = torch.full((rows, groups), unit, dtype=t)
            assert bool((scales.double() == unit).all())
            return G.moe_matrix((code[:, ::2] + 16 * code[:, 1::2]).to(torch.uint8).cuda(), code.shape[1], rows * code.shape[1], scales.cuda(), groups, rows * groups)

        self.w1, self.w2 = gate_up.double().numpy() * gate_up_unit, down.double().numpy() * down_unit
        self.layer = G.moe_layer(dtype, self.hidden, self.inner, 1, 1, torch.zeros(self.hidden, dtype=t, device="cuda"), self.hidden, matrix(gate_up, gate_up_unit),
                                 matrix(down, down_unit), group=group)

    def run(self, x, alpha=1.0):
        t = x.shape[0]
        dx, y = x.cuda(), torch.full((t, self.hidden), float("nan"), dtype=x.dtype, device="cuda")
        ws = torch.full((G.moe_workspace_bytes(self.layer, t),), 0xEE, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        G.moe(self.layer, t, alpha, dx, self.hidden, 0.0, y, self.hidden, ws, ws.numel())
        torch.cuda.synchronize()
        return y.cpu().double().numpy()

    def exact(self, x, alpha=1.0):
        """(value, bound, h): sums in fp32 of depth R.depth, h rounded as fp32 alone -- exp, the quotient and two products: 16 U -- and one rounding to the type."""
        x64 = x.double().numpy()
        gu, terms = x64 @ self.w1.T, (R.depth(self.hidden) + 4) * 2 * U * (np.abs(x64) @ np.abs(self.w1).T)
        g, u, dg, du = gu[:, :self.inner], gu[:, self.inner:], terms[:, :self.inner], terms[:, self.inner:]
        with np.errstate(over="ignore"):
            silu = g / (1 + np.exp(-g))
        h = silu * u
        dh = 1.1 * dg * np.abs(u) + np.abs(silu) * du + 1.1 * dg * du + 16 * U * np.abs(h)
        # (4-bit weights: a term is a code and a zero point of up to 15 and 8 units, of which up to 8 remain)
        size = np.abs(self.w2) + (23 * np.abs(self.w2).max() / 7 if self.group else 0)
        y = alpha * (h @ self.w2.T)
        off = abs(alpha) * (dh @ np.abs(self.w2).T + (R.depth(self.inner) + 4) * 2 * U * ((np.abs(h) + dh) @ size.T)) + 4 * U * np.abs(y)
        return y, off + R.half_step(self.dtype) * (np.abs(y) + off) + R.smallest(self.dtype), h


def _whole(g, rows, k):
    return torch.randint(-7, 8, (rows, k), generator=g)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("tokens", [1, 4, 7, 20])
@pytest.mark.parametrize("size", ["past fp16", "far past fp16", "small", "smaller than fp16"])
def test_h_of_any_size_in_fp16(size, tokens, group):
    """h of 1e5, 1e10, 1e-6 and 1e-9 at most, and down weights (alpha) that bring y back into range."""
    hidden, inner = 128, 72
    g = torch.Generator().manual_seed(tokens)
    #                        x     gate, up    down        alpha
    x_unit, up_unit, down_unit, alpha = {"past fp16": (1.0, 2.0 ** 2, 2.0 ** -14, 1.0), "far past fp16": (2.0 ** 6, 2.0 ** 5, 2.0 ** -14, 2.0 ** -18),
                                         "small": (2.0 ** -4, 2.0 ** -11, 2.0 ** 11, 1.0), "smaller than fp16": (2.0 ** -7, 2.0 ** -14, 2.0 ** 12, 2.0 ** 12)}[size]
    layer = Layer(F16, group, _whole(g, 2 * inner, hidden), up_unit, _whole(g, hidden, inner), down_unit)
    x = (torch.randn((tokens, hidden), generator=g) * x_unit).half()
    y, bound, h = layer.exact(x, alpha)
    assert {"past fp16": 1e5, "far past fp16": 1e9}.get(size, 0) < np.abs(h).max() < {"small": 1e-4, "smaller than fp16": 1e-7}.get(size, 1e12)
    assert np.median(np.abs(y)) > 0.01 and np.abs(y).max() < 60000
    got = layer.run(x, alpha)
    worst = np.max(np.abs(got - y) / bound)
    assert np.isfinite(got).all() and worst <= 1.0, f"{worst:.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 3, 8, 21])
def test_h_has_the_bits_of_fp32(dtype, group, tokens):
    """In each 32 elements of h a pair with the same gate, whose ups differ by 2^-15 to 2^-11 of themselves, the others 0, and a row of down that takes one from the other.
    Gate and up are exact: few bits each.  The same gate has the same silu s (16 U off); each h is s * up, rounded (U); and what comes behind is exact where h is: the
    two are less than 2^24 of h's last places apart, a code or a zero point times 8 of its bits has 12, and of either only these two are summed.  So y is off by
    2 U |h| + 16 U |y| and its own rounding."""
    hidden, pairs = 48, 12
    g = torch.Generator().manual_seed(tokens + group)
    gate_up = torch.zeros((2 * 32 * pairs, hidden), dtype=torch.int64)
    down = torch.zeros((hidden, 32 * pairs), dtype=torch.int64)
    first = torch.arange(pairs) * 32 + torch.randint(0, 16, (pairs,), generator=g)
    second = torch.arange(pairs) * 32 + torch.randint(16, 32, (pairs,), generator=g)
    gate, up, apart = (torch.randint(1, 8, (pairs,), generator=g) * (torch.randint(0, 2, (pairs,), generator=g) * 2 - 1) for _ in range(3))
    for place in (first, second):
        gate_up[place, 0] = gate
        gate_up[32 * pairs + place, 0] = up
    gate_up[32 * pairs + second, 1] = apart
    down[torch.arange(pairs), first] = 1
    down[torch.arange(pairs), second] = -1
    layer = Layer(dtype, group, gate_up, 0.25, down, 1.0)
    x = torch.zeros((tokens, hidden))
    x[:, 0] = torch.randint(128, 256, (tokens,), generator=g) / 128.0
    x[:, 1] = 2.0 ** -12
    x = x.to(R.TORCH[dtype])
    y, _, h = layer.exact(x)
    room = 16 * U * np.abs(y)
    room[:, :pairs] += 2 * U * np.maximum(np.abs(h[:, first]), np.abs(h[:, second]))
    got = layer.run(x)
    worst = np.max(np.abs(got - y) / (room + R.half_step(dtype) * (np.abs(y) + room) + R.smallest(dtype)))
    assert worst <= 1.0, f"{worst:.3g} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("tokens", [1, 6, 30])
def test_an_infinite_h_reaches_no_other_token(tokens, group):
    """Past fp32: bf16 elements of 1e25 on both sides of the product."""
    hidden, inner = 64, 40
    g = torch.Generator().manual_seed(4)
    layer = Layer(BF16, group, _whole(g, 2 * inner, hidden), 0.25, _whole(g, hidden, inner), 0.125)
    x = torch.randn((tokens, hidden), generator=g)
    x[tokens // 2] *= 1e25
    x = x.bfloat16()
    got = layer.run(x)
    others = [t for t in range(tokens) if t != tokens // 2]
    y, bound, _ = layer.exact(x)
    assert not np.isfinite(got[tokens // 2]).any()
    assert (np.abs(got - y)[others] <= bound[others]).all()
