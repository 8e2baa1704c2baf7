"""The launches of the residual block's calls (tests/blockplan.py)."""
import re

import pytest

from tests import blockplan as bp
from tests import test_gpu_block, test_gpu_block_kernels, test_gpu_block_paths
from tests.blockops import F16, F32
from tinyhvm_amd import build


@pytest.mark.parametrize("rows,cols,dtype", [(2 ** 32 - 1, 1, F16), (2 ** 32 - 1, 600, F32), (2 ** 32 - 2 ** 25 + 1, 3, F32), (2 ** 25 + 1, 64, F16),
                                             (2 ** 23 + 5, 4096, F16), (7, 64, F32)], ids=str)
def test_layer_norm_takes_each_row_once(rows, cols, dtype):
    """Rows up to the last that 32 bits count."""
    done = 0
    for v in bp.launches("thvm_hip_layer_norm", 1, 0, 0, 2, 0, 0, rows, cols, 1e-5, dtype):
        assert v.first == (2 << 44) + done * cols * (2 if dtype == F16 else 4) and v.gx * v.bx < 1 << 32
        done += v.rows
    assert done == rows


def test_a_gpu_test_reaches_each_kernel():
    """The kernels that the library holds for the block, and those that the
    sizes of the GPU tests launch, are the same."""
    with open(build.LIB_PATH, "rb") as f:
        held = {v.decode() for v in re.findall(rb"(thvm_(?:ln|lnb|gemm|ns|few\d+n?|direct|pack|sum_parts|muon)_[A-Za-z0-9_]+)\.kd", f.read())}
    t, paths, kernels = test_gpu_block, test_gpu_block_paths, test_gpu_block_kernels
    run = set()
    for dt in (F32, F16):
        for shape in t.LINEAR + paths.LIES + paths.PACKED + paths.FEW + [v[0] for v in kernels.DIRECT] + [v[0] for v in kernels.LAYERS if v[1] == dt]:
            run.update(bp.linear(*shape, dt))
        for shape in t.LINEAR + [v[0] for v in kernels.GRADS]:
            run.update(bp.linear_grad(*shape, dt))
        for rows, cols in t.LN + [(600, 4096), (515, 4099), (4100, 1000), (4099, 1999), (1500, 1000), (1025, 500), (511, 4096), (3, 30001)]:
            run.update(bp.names("thvm_hip_layer_norm", 1, 2, 3, 4, 5, 6, rows, cols, 1e-5, dt))
        for rows, cols in t.LN + [(2500, 96), (1999, 1000)]:
            run.update(bp.names("thvm_hip_layer_norm_grad", 1, 2, 3, 4, 5, 6, 7, 8, 9, rows, cols, dt))
        for shape in t.MUON + [(12, 1104, 1104), (16, 1232, 1232), (2, 1500, 700)]:
            run.update(bp.muon_step(*shape, dt))
    assert held and run == held
