"""An expert whose row of the router is NaN: it comes behind all others, and what its NaN does to the others' scores is what the header says."""
import copy

import numpy as np
import pytest
import torch

import gemm_mmbo_amd as G
import w4_reference as R
from test_moe import Problem

F16, BF16 = G.F16, G.BF16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens", [1, 8, 9, 70])
@pytest.mark.parametrize("experts", [6, 70, 200])
def test_it_comes_behind_all_others(dtype, tokens, experts):
    for sigmoid, renormalize in ((False, True), (True, True), (True, False), (False, False)):
        p = Problem(dtype, tokens, 96, 40, experts, 4, sigmoid=sigmoid, renormalize=renormalize)
        p.router[2] = float("nan")
        y, ids, weights = p.run()
        without = copy.copy(p)                                      # the same layer with an expert that no token takes in its place
        without.router = p.router.clone()
        without.router[2] = 0
        logits = p.x[:, :96].double().numpy() @ without.router.double().numpy().T
        logits[:, 2] = -np.inf
        want_ids, want = R.select(logits, 4, sigmoid, renormalize, None)
        assert np.array_equal(ids, want_ids) and (ids != 2).all()
        if renormalize or sigmoid:
            assert np.allclose(weights, want, rtol=2 * R.U, atol=1e-40) and bool(torch.isfinite(y).all())
        else:
            assert np.isnan(weights).all() and bool(torch.isnan(y).all())


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 9])
def test_it_is_taken_when_there_is_no_other(tokens):
    p = Problem(F16, tokens, 96, 40, 5, 5)
    p.router[1] = float("nan")
    y, ids, weights = p.run()
    assert (ids[:, 4] == 1).all() and (np.sort(ids, 1) == np.arange(5)).all() and np.isnan(weights).all() and bool(torch.isnan(y).all())
