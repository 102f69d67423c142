"""GPU tests of the norms of 8-bit checkpoints at the edges of their kernels."""
import pytest
import torch

import operator_oracle as Q
from test_act8_gpu import check_norm, check_norm_grad, held, norm_case

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


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [1024, 300])
def test_matrices_beside_each_other_in_one_buffer(pkg, dtype, cols):
    """dy, dresidual and dx as parts of the rows of one buffer: what separate buffers give, bit for bit."""
    rows = 50
    x, w, dy, dres = norm_case(rows, cols, dtype, 3)
    cb, sb, _ = held(pkg, x)
    wb, ws = w.cuda(), torch.empty(pkg.act8_rmsnorm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    apart = [dy.cuda(), dres.cuda(), torch.empty_like(dy).cuda()]
    one = torch.stack([dy, dres, torch.zeros_like(dy)], 1).cuda()
    results = []
    for parts, stride in ((apart, cols), ([one[:, k] for k in range(3)], 3 * cols)):
        dw = torch.empty(cols, device="cuda")
        pkg.act8_rmsnorm_grad(cb.ptr, sb.ptr, rows, cols, wb.data_ptr(), pkg.F32, 1e-6, parts[0].data_ptr(), Q.kind(pkg, dtype), parts[2].data_ptr(),
                              dw.data_ptr(), ws.data_ptr(), ws.numel(), parts[1].data_ptr(), cb.stride, stride, stride, stride)
        torch.cuda.synchronize()
        results.append((parts[2].clone(), dw))
    assert all(torch.equal(p, q) for p, q in zip(*results))
    assert torch.equal(one[:, 0].cpu(), dy) and torch.equal(one[:, 1].cpu(), dres)
