"""Linear layers beside test_gpu_linear.py: calls in place, and every size of tile with every epilogue at sizes that are no multiple of it."""
import numpy as np
import pytest

from test_gpu_attention import from_bf16, to_bf16
from test_gpu_linear import GELU, NONE, RELU, SILU

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2049, 70001])
@pytest.mark.parametrize("a", [NONE, RELU, SILU, GELU])
def test_activation_gradient_in_place(br, a, n):
    """dpre may be dy: the same bits as into another tensor, at whole and broken groups of eight."""
    rng = np.random.default_rng(n)
    pre, dy = to_bf16(3 * rng.standard_normal(n)), to_bf16(rng.standard_normal(n))
    D = br.DevArray.from_numpy
    out, g, p = br.DevArray(n, np.uint16), D(dy), D(pre)
    br.check(br.lib.mi355_act_bwd_bf16_dev(out.ptr, g.ptr, p.ptr, 0.25, a, n))
    br.check(br.lib.mi355_act_bwd_bf16_dev(g.ptr, g.ptr, p.ptr, 0.25, a, n))
    assert np.array_equal(g.numpy(), out.numpy()) and np.all(np.isfinite(from_bf16(out.numpy())))
