"""GPU check: the library itself refuses the cross entropy of 2^30 tokens."""
import pytest

pytestmark = pytest.mark.gpu

from rew_amd import eager as E
from rew_amd.eager import DType, EagerError


def test_library_refusals(gpu):
    T = 2 ** 30
    x, w, t = (E.empty(DType.BFLOAT16, (T, 1)), E.empty(DType.BFLOAT16, (1, 7)),
               E.empty(DType.INT32, (T,)))
    f = E.empty(DType.FLOAT32, (T,))
    for op, ins, attrs in (("linearCrossEntropy", [x, w, t], [("stats", "true")]),
                           ("linearCrossEntropyGrad", [x, w, t, f, f], [])):
        with pytest.raises(EagerError, match="2\\^30 tokens"):
            E.dispatchEager(op, ins, [("tied", "false"), *attrs])
