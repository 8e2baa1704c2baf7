"""What the residual block's operators make of single values: activations on
their own, NaN and infinities through them, and rows of nothing."""
import math

import numpy as np
import pytest

from tests import blockops as bo
from tests import blockplan as bp
from tests.blockops import ACTS, F16, F32, NP, U32
from tests.test_gpu_block import within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    L = bo.lib()
    L.thvm_hip_shutdown()
    assert L.thvm_hip_init() == 0
    yield L
    L.thvm_hip_shutdown()


# ---- rows of nothing ----

@pytest.mark.parametrize("dt", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 700])
def test_statistics_of_empty_rows(hip, rows, dt):
    """The mean of no values is 0 / 0, and so is what stands on it."""
    y, mean, rstd = bo.run_layer_norm(hip, np.zeros((rows, 0), NP[dt]), None, None, 1e-5, dt)
    with bo.Bufs(hip) as b:
        m, r = b.put(np.ones(rows, np.float32)), b.put(np.ones(rows, np.float32))
        x = b.put(np.zeros((rows, 0), NP[dt]))
        assert hip.thvm_hip_layer_norm(b.out((rows, 0), NP[dt]), m, r, x, 0, 0, rows, 0, 1e-5, dt) == 0
        assert np.isnan(b.get(m)).all() and np.isnan(b.get(r)).all()
