"""GPU checks of rmsNorm rows whose 16-byte chunks fill whole waves, 1 to 8 times.

Tolerances: float32 <= 1e-5 relative; bf16 half a step of the result (2^-8) beside it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from rew_amd import eager as E
from rew_amd import nn
from rew_amd import ops as O
from rew_amd.eager import DType


@pytest.mark.parametrize("rows", [1, 60, 257])
@pytest.mark.parametrize("n", [256, 512, 768, 1024, 1280, 1536, 2560])
@pytest.mark.parametrize("bf16", [False, True])
def test_rmsnorm_widths(gpu, oracle, rows, n, bf16):
    x = oracle.normal_f32(oracle.init_key(n + rows), rows * n).reshape(rows, n)
    g = oracle.normal_f32(oracle.fold_in(oracle.init_key(5), n), n, 1.0, 0.1)
    if bf16:
        x = oracle.round_bf16(x)
        t = O.astype(E.fromHost(x, DType.BFLOAT16), DType.FLOAT32)
        got = E.toHostF32(O.astype(nn.rmsNorm(t, E.fromHost(g), 1e-5), DType.BFLOAT16))
    else:
        got = E.toHostF32(nn.rmsNorm(E.fromHost(x), E.fromHost(g), 1e-5))
    want = oracle.rmsnorm_rows(x, g, 1e-5)
    np.testing.assert_allclose(got, want, rtol=2.0 ** -8 + 1e-5 if bf16 else 1e-5, atol=1e-6)
