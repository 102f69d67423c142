"""GPU tests of the norms of 8-bit checkpoints at the edges of their kernels."""
import pytest

from test_act8_gpu import check_norm, check_norm_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("cols", [20, 999, 1001, 3990, 8189])
@pytest.mark.parametrize("rows", [3, 16, 70])
def test_norm_grad_of_few_rows_whose_last_columns_fill_no_run(pkg, dtype, cols, rows):
    """Aligned rows, a width that is no multiple of 16 (nor of 4): the threads of the last warp take different branches
    before the barrier of the cluster that adds the partial sums."""
    pad = -cols % 16
    check_norm(pkg, rows, cols, dtype, rows, cpad=pad, ypad=pad)
    check_norm_grad(pkg, rows, cols, dtype, rows, cpad=pad, pad=pad, dpad=pad, accumulate=rows == 16)
