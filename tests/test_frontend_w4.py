"""gemm_w4 and moe of the CPython module (csrc/frontend.cc) beside the Python functions they stand in for, form by form.  No call of these reaches a device: they
end at a size of zero or at an argument check."""
import inspect

import numpy as np
import pytest

import gemm_mmbo_amd as G
from gemm_mmbo_amd import api
from test_frontend import Broken, Stream, Tensor, _result

W4 = [1, 0, 5, 64, 32, 1.0, Tensor(), 64, Tensor(), 2, None, 0, Tensor(), 64, 0.0, Tensor(), 5]
MOE = [None, 0, 1.0, Tensor(), 64, 0.0, Tensor(), 64, Tensor(), 4096]
CHANGES = {
    3: [{}, {0: 0}, {0: 3}, {0: 7}, {0: "1"}, {1: -1}, {1: 4}, {1: np.int64(0)}, {1: 4.0}, {2: 2 ** 70}, {4: 33}, {4: None}, {5: 1}, {5: "x"}, {5: None}, {6: None, 1: 4}, {6: Broken()},
        {7: 63}, {8: object()}, {9: 1}, {10: Tensor()}, {10: Tensor(), 11: 2}, {12: 0, 1: 4}, {13: 63}, {14: 10 ** 400}, {15: None, 1: 4}, {16: 0}],
    4: [{}, {0: 3}, {0: "layer"}, {1: -1}, {1: 4, 8: None}, {1: 4, 9: 16}, {1: 600}, {1: "a"}, {2: None}, {3: Broken()}, {4: 63}, {5: 1}, {6: None, 1: 2}, {7: 0}, {8: 24, 1: 1}, {9: None}]}
TAILS = {3: [(), (None,), (0,), (Stream(),), (object(),), (None, 3)],
         4: [(), (None,), (None, None), (None, None, None), (Tensor(), Tensor(), Stream()), (object(),), (None, None, object()), (None, None, None, 1)]}


@pytest.mark.skipif(api._frontend is None, reason="the module is not built")
@pytest.mark.parametrize("which", [3, 4])
def test_every_form_of_a_call_gives_what_the_python_function_gives(which):
    ours, python = (G.gemm_w4, G.moe)[which - 3], api._PYTHON_FRONT_ENDS[which]
    assert ours is not python and inspect.signature(ours) == inspect.signature(python) and ours.__name__ == python.__name__
    assert inspect.getdoc(ours) == inspect.getdoc(python)
    layer = G.moe_layer(G.F16, 64, 32, 4, 2, 16, 64, G.moe_matrix(16, 64, 4096), G.moe_matrix(16, 32, 2048))
    names, taken = list(inspect.signature(python).parameters), set()
    for change in CHANGES[which]:
        for tail in TAILS[which]:
            args = list(W4 if which == 3 else [layer] + MOE[1:])
            for i, v in change.items():
                args[i] = v
            full = args + list(tail)
            forms = [(full, {})] + [(full[:cut], dict(zip(names[cut:], full[cut:]))) for cut in (3, 0) if len(full) <= len(names)]
            for a, kw in forms + [(args[:-1], {})]:
                got, want = _result(ours, a, kw), _result(python, a, kw)
                assert got == want, (a, kw, got, want)
                taken.add(want if want is None else want[0])
    assert {None, G.MmboError, TypeError} <= taken
