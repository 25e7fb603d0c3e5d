"""The mixture-of-experts layer: refusals (no GPU), and on the GPU the selection and the output against the definition in 64 bits, within bounds that rounding
allows (w4_reference.py)."""
import ctypes

import numpy as np
import pytest
import torch

import gemm_mmbo_amd as G
import w4_reference as R
from gemm_mmbo_amd import api

F32, F16, F64, BF16 = G.F32, G.F16, G.F64, G.BF16


def _layer(group=0, gate_up=None, down=None, **change):
    h, i = change.get("hidden", 64), change.get("inner", 32)
    w4 = group != 0
    gate_up = gate_up or G.moe_matrix(16, h, 2 * i * h, 16 if w4 else None, 64 if w4 else 0)
    down = down or G.moe_matrix(16, i, h * i, 16 if w4 else None, 64 if w4 else 0)
    args = dict(dtype=F16, hidden=64, inner=32, experts=4, top_k=2, router=16, ld_router=64)
    args.update(change)
    return G.moe_layer(gate_up=gate_up, down=down, group=group, **args)


def _status(layer, tokens=2, x=16, ldx=64, y=16, ldy=64, workspace=16, nbytes=1 << 20, alpha=True, beta=True):
    one = ctypes.c_float(1.0)
    p = ctypes.byref(one)
    return api.lib().mmbo_moe(ctypes.byref(layer) if layer is not None else None, tokens, p if alpha else None, x, ldx, p if beta else None, y, ldy, None, None,
                              workspace, nbytes, None)


@pytest.mark.parametrize("layer,status", [
    (dict(dtype=F32), 1), (dict(dtype=F64), 1), (dict(dtype=F16, router_dtype=BF16), 1), (dict(scoring=2), 2), (dict(hidden=0), 3), (dict(inner=0), 3), (dict(hidden=65537, ld_router=65537), 3), (dict(inner=65537), 3),
    (dict(experts=0), 3), (dict(experts=G.MOE_MAX_EXPERTS + 1), 3), (dict(top_k=0), 3), (dict(top_k=5), 3), (dict(experts=64, top_k=G.MOE_MAX_TOP_K + 1), 3),
    (dict(group=16), 3), (dict(group=2 ** 31), 3), (dict(ld_router=63), 3), (dict(gate_up=G.moe_matrix(16, 63, 1 << 20)), 3), (dict(down=G.moe_matrix(16, 31, 1 << 20)), 3),
    (dict(down=G.moe_matrix(16, 32, -64)), 3), (dict(group=32, gate_up=G.moe_matrix(16, 64, 1 << 20, 16, 1)), 3), (dict(group=32, gate_up=G.moe_matrix(16, 65, 1 << 20, 16, 2)), 3),
    (dict(group=32, down=G.moe_matrix(16, 32, 1023, 16, 1)), 3), (dict(group=32, down=G.moe_matrix(16, 32, 1024, 16, 1, -1)), 3),
    (dict(group=32, down=G.moe_matrix(16, 32, 1024, 16, 1, 64, 16, 0)), 3), (dict(group=32, down=G.moe_matrix(16, 32, 1024, 16, 1, 64, 16, 1, -2)), 3)])
def test_layers_that_are_refused(layer, status):
    made = _layer(**layer)
    assert _status(made) == status
    assert api.lib().mmbo_moe_workspace_bytes(ctypes.byref(made), 1) == 0
    with pytest.raises(G.MmboError):
        G.moe_workspace_bytes(made, 1)


def test_calls_that_are_refused():
    layer = _layer()
    assert _status(None) == 4
    assert _status(layer, alpha=False) == 4 and _status(layer, beta=False) == 4
    assert _status(layer, tokens=G.MOE_MAX_TOKENS + 1) == 3 and _status(layer, ldx=63) == 3 and _status(layer, ldy=63) == 3
    assert _status(layer, x=None) == 4 and _status(layer, y=None) == 4 and _status(layer, workspace=None) == 4
    assert _status(_layer(router=None)) == 4 and _status(_layer(gate_up=G.moe_matrix(None, 64, 4096))) == 4
    assert _status(_layer(group=32, down=G.moe_matrix(16, 32, 2048, None, 1))) == 4
    need = G.moe_workspace_bytes(layer, 2)
    assert need > 0 and _status(layer, nbytes=need - 1) == 8 and _status(layer, workspace=24) == 8
    assert G.moe_workspace_bytes(layer, G.MOE_MAX_TOKENS) >= need
    with pytest.raises(G.MmboError):
        G.moe_workspace_bytes(layer, G.MOE_MAX_TOKENS + 1)
    assert _status(layer, tokens=0, x=None, y=None, workspace=None) == 0


@pytest.mark.parametrize("change", [dict(hidden=2048, ld_router=2048), dict(experts=32, top_k=32), dict(hidden=16, ld_router=64, experts=512, top_k=32)])
def test_a_workspace_serves_fewer_tokens_too(change):
    h = change.get("hidden", 64)
    layer = _layer(gate_up=G.moe_matrix(16, h, 64 * h), down=G.moe_matrix(16, 32, 32 * h), **change)
    sizes = [G.moe_workspace_bytes(layer, t) for t in range(G.MOE_MAX_TOKENS + 1)]
    assert sizes == sorted(sizes) and all(n % 16 == 0 for n in sizes)


# ---- on the GPU

class Problem:
    def __init__(self, dtype, tokens, hidden, inner, experts, top_k, group=0, zeros=False, sigmoid=False, renormalize=True, bias=False, router32=False, alpha=1.0,
                 beta=0.0, pad=0, seed=0):
        self.__dict__.update(dtype=dtype, tokens=tokens, hidden=hidden, inner=inner, experts=experts, top_k=top_k, group=group, sigmoid=sigmoid,
                             renormalize=renormalize, router32=router32, alpha=alpha, beta=beta, pad=pad)
        g = torch.Generator().manual_seed(7 * tokens + hidden + 3 * inner + experts + seed)
        t = R.TORCH[dtype]
        self.x = torch.randn((tokens, hidden + pad), generator=g).to(t)
        self.y = torch.randn((tokens, hidden + pad), generator=g).to(t) if beta else torch.full((tokens, hidden + pad), float("nan"), dtype=t)
        if pad:
            self.y[:, hidden:] = -7.0
        self.router = (torch.randn((experts, hidden), generator=g) / hidden ** 0.5).to(torch.float32 if router32 else t)
        self.bias = torch.randn((experts,), generator=g) * 0.1 if bias else None
        if group:
            self.gate_up = R.Weight(g, dtype, 2 * inner, hidden, group, zeros, pad, pad, (experts,), 0.2 / hidden ** 0.5)
            self.down = R.Weight(g, dtype, hidden, inner, group, zeros, pad, pad, (experts,), 0.2 / inner ** 0.5)
        else:
            self.gate_up = (torch.randn((experts, 2 * inner, hidden + pad), generator=g) / hidden ** 0.5).to(t)
            self.down = (torch.randn((experts, hidden, inner + pad), generator=g) / inner ** 0.5).to(t)

    def matrix(self, w):
        if self.group:
            z = None if w.zeros is None else w.zeros.cuda()
            per = w.scales.shape[1] * w.lds
            return G.moe_matrix(w.q.cuda(), w.ldq, w.q.shape[1] * w.ldq, w.scales.cuda(), w.lds, per, z, w.lds, per)
        return G.moe_matrix(w.cuda(), w.shape[2], w.shape[1] * w.shape[2])

    def layer(self):
        return G.moe_layer(self.dtype, self.hidden, self.inner, self.experts, self.top_k, self.router.cuda(), self.hidden, self.matrix(self.gate_up),
                           self.matrix(self.down), group=self.group, bias=None if self.bias is None else self.bias.cuda(),
                           scoring=G.MOE_SIGMOID if self.sigmoid else G.MOE_SOFTMAX, renormalize=self.renormalize, router_dtype=F32 if self.router32 else None)

    def exact(self):
        cut = (lambda w, k: w) if self.group else (lambda w, k: w[..., :k])
        return R.moe(self.dtype, self.x[:, :self.hidden], self.router, cut(self.gate_up, self.hidden), cut(self.down, self.inner), self.inner, self.top_k,
                     self.sigmoid, self.renormalize, self.bias, self.alpha, self.beta, self.y[:, :self.hidden])

    def run(self, layer=None, x=None):
        layer = layer or self.layer()
        x, y = (self.x if x is None else x).cuda(), self.y.cuda()
        ids = torch.full((self.tokens, self.top_k), -1, dtype=torch.int32, device="cuda")
        weights = torch.full((self.tokens, self.top_k), -1.0, device="cuda")
        ws = torch.full((G.moe_workspace_bytes(layer, self.tokens),), 0xEE, dtype=torch.uint8, device="cuda")       # (no contents are expected)
        torch.cuda.synchronize()
        G.moe(layer, self.tokens, self.alpha, x, x.shape[1], self.beta, y, y.shape[1], ws, ws.numel(), ids, weights)
        torch.cuda.synchronize()
        return y.cpu(), ids.cpu().numpy(), weights.cpu().double().numpy()


def _check(p):
    y, ids, weights = p.run()
    exact, bound, want_ids, want_weights = p.exact()
    assert np.array_equal(ids, want_ids)
    # in 64 bits, rounded once to fp32
    assert np.allclose(weights, want_weights, rtol=2 * R.U, atol=1e-40)
    got = y[:, :p.hidden].double().numpy()
    worst = np.max(np.abs(got - exact) / bound)
    assert np.isfinite(got).all() and worst <= 1.0, f"{worst:.3g} of the bound"
    assert bool((y[:, p.hidden:] == -7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [0, 32, 128])
@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [
    (1, 64, 32, 4, 2), (1, 1, 1, 1, 1), (2, 33, 17, 3, 3), (1, 256, 128, 64, 8), (3, 130, 70, 5, 1), (16, 128, 96, 8, 2), (17, 200, 48, 6, 4), (40, 96, 160, 3, 2),
    (70, 64, 40, 2, 2), (5, 515, 261, 40, 6), (33, 160, 64, 128, 8)])
def test_layers_against_the_definition(dtype, group, tokens, hidden, inner, experts, top_k):
    _check(Problem(dtype, tokens, hidden, inner, experts, top_k, group))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("sigmoid,renormalize,bias", [(False, False, False), (False, True, True), (True, True, True), (True, False, False), (True, False, True)])
def test_scores_bias_scalars_zeros_and_rows_inside_larger_arrays(dtype, group, sigmoid, renormalize, bias):
    for tokens, pad in ((1, 0), (6, 3), (20, 1)):
        _check(Problem(dtype, tokens, 100, 60, 12, 3, group, zeros=True, sigmoid=sigmoid, renormalize=renormalize, bias=bias, router32=pad == 3, alpha=-0.5,
                       beta=0.75, pad=pad))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens", [1, 9])
@pytest.mark.parametrize("zeros", ["gate_up", "down"])
def test_zero_points_of_one_matrix_alone(dtype, tokens, zeros):
    p = Problem(dtype, tokens, 96, 64, 6, 2, group=32, zeros=True)
    other = Problem(dtype, tokens, 96, 64, 6, 2, group=32, seed=1)
    setattr(p, *(("down", other.down) if zeros == "gate_up" else ("gate_up", other.gate_up)))
    _check(p)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, 32])
def test_the_largest_counts(group):
    _check(Problem(BF16, G.MOE_MAX_TOKENS, 48, 32, 16, 4, group))
    _check(Problem(F16, 3, 64, 32, G.MOE_MAX_EXPERTS, G.MOE_MAX_TOP_K, group))
    _check(Problem(BF16, 100, 32, 16, G.MOE_MAX_EXPERTS, 4, group))


@pytest.mark.gpu
@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("tokens,experts,top_k", [(5, 16, 2), (8, G.MOE_MAX_EXPERTS, G.MOE_MAX_TOP_K), (9, G.MOE_MAX_EXPERTS, G.MOE_MAX_TOP_K), (8, 1, 1), (8, 4, 1),
                                                  (7, 65, 3), (64, 128, 2), (65, 128, 4), (64, 128, 5)])
def test_where_the_selection_and_the_jobs_change_their_form(group, tokens, experts, top_k):
    """Up to 8 tokens and more; jobs of four columns (up to two pairs to an expert) and of sixteen."""
    _check(Problem(BF16, tokens, 72, 40, experts, top_k, group))
    _check(Problem(F16, tokens, 136, 24, experts, top_k, group, zeros=True, sigmoid=True, beta=0.5, pad=8))


@pytest.mark.gpu
def test_one_workspace_for_calls_one_behind_the_other():
    """Layers of different sizes and numbers of tokens over the same memory, as a program's layers share it: eager, and captured into one graph."""
    problems = [Problem(F16, t, h, i, e, k, group) for t, h, i, e, k, group in
                ((40, 96, 64, 8, 2, 0), (1, 160, 48, 32, 4, 32), (8, 64, 32, 64, 8, 0), (9, 64, 32, 64, 8, 64), (70, 80, 24, 5, 3, 0))]
    layers = [p.layer() for p in problems]
    nbytes = max(G.moe_workspace_bytes(layer, p.tokens) for layer, p in zip(layers, problems))
    ws = torch.full((nbytes,), 0xEE, dtype=torch.uint8, device="cuda")
    xs, ys = [p.x.cuda() for p in problems], [torch.empty((p.tokens, p.hidden), dtype=torch.float16, device="cuda") for p in problems]

    def calls(stream):
        for p, layer, x, y in zip(problems, layers, xs, ys):
            G.moe(layer, p.tokens, 1.0, x, p.hidden, 0.0, y, p.hidden, ws, nbytes, stream=stream)

    alone = [p.run()[0] for p in problems]
    for _ in range(2):
        calls(None)
        torch.cuda.synchronize()
        assert all(torch.equal(y.cpu(), a) for y, a in zip(ys, alone))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream())
    for _ in range(3):
        for y in ys:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y.cpu(), a) for y, a in zip(ys, alone))
        ws.fill_(0xFF)


@pytest.mark.gpu
def test_ties_go_to_the_lower_expert():
    p = Problem(F16, 9, 64, 32, 96, 6)
    p.router[:] = p.router[0]                       # every expert the same logit
    p.router[70] = p.router[0] * 2                  # one above or below
    y, ids, weights = p.run()
    _, _, want, want_weights = p.exact()
    assert np.array_equal(ids, want) and np.allclose(weights, want_weights, rtol=2 * R.U)
    assert set(ids[ids != 70]) <= set(range(6))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,group", [(F16, 0), (BF16, 0), (BF16, 32), (F16, 32)])
def test_a_token_of_nan_or_infinities_reaches_no_other(dtype, group):
    p = Problem(dtype, 20, 96, 64, 8, 2, group)
    exact, bound, want_ids, want_weights = p.exact()
    layer = p.layer()
    for bad in (float("nan"), float("inf")):
        x = p.x.clone()
        x[11, 5] = bad
        y, ids, weights = p.run(layer, x)
        others = [t for t in range(20) if t != 11]
        assert np.array_equal(ids[others], want_ids[others])
        assert (np.abs(y[others].double().numpy() - exact[others]) <= bound[others]).all()
        assert not torch.isfinite(y[11]).any()
        assert len(set(ids[11])) == 2 and ids[11].min() >= 0 and ids[11].max() < 8


@pytest.mark.gpu
@pytest.mark.parametrize("sigmoid", [False, True])
def test_logits_far_apart(sigmoid):
    """Scores that are 0 in any format but the largest: weights stay numbers."""
    p = Problem(F16, 4, 64, 32, 6, 3, sigmoid=sigmoid, router32=True)
    p.router *= 4000
    if sigmoid:
        p.router[:] = -p.x[0, :64].float() * 100    # token 0: every score is 0
    y, ids, weights = p.run()
    exact, bound, want_ids, want_weights = p.exact()
    assert np.array_equal(ids, want_ids) and np.isfinite(weights).all() and np.allclose(weights, want_weights, rtol=2 * R.U, atol=1e-38)
    assert (np.abs(y.double().numpy() - exact) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,group,tokens", [(BF16, 0, 1), (F16, 64, 1), (BF16, 64, 24), (F16, 0, 24)])
def test_layers_in_a_graph_and_on_two_streams(dtype, group, tokens):
    p = Problem(dtype, tokens, 192, 96, 16, 4, group)
    layer = p.layer()
    nbytes = G.moe_workspace_bytes(layer, tokens)
    x = p.x.cuda()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ws = [torch.full((nbytes,), 0xEE, dtype=torch.uint8, device="cuda") for _ in range(3)]
    ys = [torch.empty((tokens, 192), dtype=x.dtype, device="cuda") for _ in range(3)]

    def call(which, stream):
        G.moe(layer, tokens, 1.0, x, 192, 0.0, ys[which], 192, ws[which], nbytes, stream=stream)

    call(2, None)
    torch.cuda.synchronize()
    first = ys[2].clone()
    for _ in range(5):
        for k, st in enumerate(streams):
            call(k, st)
    torch.cuda.synchronize()
    assert torch.equal(ys[0], first) and torch.equal(ys[1], first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(2, torch.cuda.current_stream())
    g = torch.Generator().manual_seed(9)
    for _ in range(4):
        x.copy_(torch.randn((tokens, 192), generator=g).to(x.dtype))
        call(0, torch.cuda.current_stream())
        ys[2].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys[0], ys[2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_one_expert_for_all_is_two_products(dtype):
    """A layer of one 4-bit expert beside gemm_w4 on the same weights: the calls as a program mixes them."""
    p = Problem(dtype, 12, 128, 64, 1, 1, 32)
    y, ids, weights = p.run()
    assert (ids == 0).all() and (weights == 1.0).all()
    x, t = p.x.cuda(), R.TORCH[dtype]
    gu = torch.empty((12, 128), dtype=t, device="cuda")
    out = torch.empty((12, 128), dtype=t, device="cuda")
    up, down = p.gate_up, p.down
    G.gemm_w4(dtype, 128, 12, 128, 32, 1.0, up.q[0].cuda(), up.ldq, up.scales[0].cuda(), up.lds, None, 0, x, 128, 0.0, gu, 128)
    h = (torch.nn.functional.silu(gu[:, :64].float()) * gu[:, 64:].float()).to(t)
    G.gemm_w4(dtype, 128, 12, 64, 32, 1.0, down.q[0].cuda(), down.ldq, down.scales[0].cuda(), down.lds, None, 0, h, 64, 0.0, out, 128)
    torch.cuda.synchronize()
    # between the two: gate, up, h and the output each rounded to the type (silu' < 1.1)
    g64, e = p.exact(), R.half_step(dtype)
    w1, w2 = up.parts()[0][0], down.parts()[0][0]
    gu64 = p.x.double().numpy() @ w1.T
    room = (3 * e * 1.1 * np.abs(gu64[:, :64]) * np.abs(gu64[:, 64:])) @ np.abs(w2).T
    assert (np.abs(out.cpu().double().numpy() - y.double().numpy()) <= 1.05 * room + 2 * g64[1]).all()
