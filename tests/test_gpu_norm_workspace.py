"""Layer norm's backward for dx alone, which has no sums over rows to keep."""
import numpy as np
import pytest

import aetcnn
from aetcnn import ACH_EWORKSPACE, BF16, F16, F32
from test_gpu_checkpoint import activations
from test_gpu_layernorm import Backward, parameters
from test_gpu_logits import Rows

pytestmark = pytest.mark.gpu


class Nothing:
    ptr = None


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n", [(1, 40), (700, 10), (600, 1000), (5, 9001), (300, 16384)])
def test_without_a_workspace(gpu, rows, n, kind):
    rng = np.random.default_rng(n)
    x, (s, _) = Rows(activations(rng, rows, n), kind), parameters(rng, n)
    for from_kept in (False, True):
        g = Backward(gpu, Rows(rng.standard_normal((rows, n)), kind), (x, 1e-5), s, from_kept,
                     outputs=("dx",))
        g.ws, g.nb = Nothing, 0
        g.call()
        g.check()


def test_rows_in_parts_need_one(gpu):
    """for the sums of the parts"""
    rng = np.random.default_rng(1)
    x = Rows(activations(rng, 3, 16385), F32)
    g = Backward(gpu, Rows(rng.standard_normal((3, 16385)), F32), (x, 1e-5), None, outputs=("dx",))
    ws, g.ws, g.nb = g.ws, Nothing, 0
    with pytest.raises(aetcnn.HipError) as e:
        g.call()
    assert f"code {ACH_EWORKSPACE}" in str(e.value)
    assert np.isnan(g.dx.read()).all()
    g.ws, g.nb = ws, gpu.ach_layernorm_bwd_workspace(g.desc)
    g.call()
    g.check()
