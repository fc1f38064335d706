"""GPU check of embedding rows times zero: the zeros have the scale's sign, in either order of
the calls."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from ends_ref import host, ints, tensor
from rew_amd import ops as O


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_scale_of_either_zero(gpu, dtype):
    w, wh = tensor([[1.0, -2.0, 3.0, -0.5]], dtype)
    for scale in (0.0, -0.0, 0.0):
        np.testing.assert_array_equal(np.signbit(host(O.embedding(w, ints([0]), scale))),
                                      np.signbit(wh * scale))
