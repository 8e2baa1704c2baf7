"""The launches of the residual block's calls (tests/blockplan.py)."""
import pytest

from tests import blockplan as bp
from tests.blockops import F16, F32


@pytest.mark.parametrize("rows,cols,dtype", [(2 ** 32 - 1, 1, F16), (2 ** 32 - 1, 600, F32), (2 ** 32 - 2 ** 25 + 1, 3, F32), (2 ** 25 + 1, 64, F16),
                                             (2 ** 23 + 5, 4096, F16), (7, 64, F32)], ids=str)
def test_layer_norm_takes_each_row_once(rows, cols, dtype):
    """Rows up to the last that 32 bits count."""
    done = 0
    for v in bp.launches("thvm_hip_layer_norm", 1, 0, 0, 2, 0, 0, rows, cols, 1e-5, dtype):
        assert v.first == (2 << 44) + done * cols * (2 if dtype == F16 else 4) and v.gx * v.bx < 1 << 32
        done += v.rows
    assert done == rows
