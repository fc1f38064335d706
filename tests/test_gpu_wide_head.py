"""GPU check of the cross entropy of a head as wide as it may be: the aligned copy of a piece of
its weight is more than 2^32 runs of 16 bytes."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import ends_ref as R
from ends_ref import ints, tensor
from rew_amd import _lib
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType


def test_weight_of_2_21_rows(gpu):
    """The first, a middle and the last row of the weight hold values, the others zeros, and x is
    one everywhere: the logits are the sums of three rows.  A 64 GiB weight and as much working
    memory."""
    H, V = 2 ** 21, 16385
    hip = C.CDLL("libamdhip64.so")
    _lib.load().rew_mi355x_shutdown(E.context())  # (frees the cached blocks)
    free, total = C.c_size_t(), C.c_size_t()
    assert hip.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    if free.value < 160 << 30:
        pytest.skip("less than 160 GiB of device memory is free")
    r = np.random.default_rng(0)
    w = E.empty(DType.BFLOAT16, (H, V))
    E.sync()
    at = E.devicePtr(w)
    assert hip.hipMemset(C.c_void_p(at), 0, C.c_size_t(2 * H * V)) == 0
    rows = r.integers(-8, 9, (3, V)) / 4.0  # (exact in bfloat16, as are their sums in float32)
    for row, v in zip((0, H // 2 + 1, H - 1), rows):
        bits = np.ascontiguousarray(E.f32_to_bf16_bits(v.astype(np.float32)))
        assert hip.hipMemcpy(C.c_void_p(at + 2 * row * V), bits.ctypes.data_as(C.c_void_p),
                             C.c_size_t(2 * V), 1) == 0
    assert hip.hipDeviceSynchronize() == 0
    x = tensor(np.ones((2, H)), "bfloat16")[0]
    t = [V - 1, 77]
    loss, lse = O.linearCrossEntropy(x, w, ints(t), withLse=True)
    for got, (want, bound) in zip((loss, lse), R.cross_entropy(np.ones((2, 3)), rows, t)):
        R.check(got, want, bound)
    del w, x, loss, lse, got
    _lib.load().rew_mi355x_shutdown(E.context())
