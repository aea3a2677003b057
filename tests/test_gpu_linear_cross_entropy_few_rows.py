"""functional.linear_cross_entropy in training below 256 rows: the weight's gradient from the
128-row tiles themselves, and through f32 sums of columns of the vocabulary at a time where its
sizes or its address suit no 16-byte stores.  References and bounds are those of
test_gpu_linear_cross_entropy.py."""
import math

import pytest
import torch

from tests import row_ref as R
from tests.test_gpu_linear_cross_entropy import DT, _check, _normal, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dt,n,V,C", [("bf16", 128, 16384, 1024), ("bf16", 40, 1032, 264), ("bf16", 200, 72, 40),
                                      ("f32", 40, 20003, 4100), ("bf16", 33, 20003, 4100), ("bf16", 7, 20000, 4104)])
def test_training(dt, n, V, C, tied):
    x, w = _normal((n, C), DT[dt], n), _normal((C, V), DT[dt], V, 2.0 / math.sqrt(C))
    t = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(n))
    t[0], t[n - 1] = -1, V - 1
    for a in (0.0, 0.1):
        _check(x, w, t, a, _normal((n,), torch.float32, V) / n, tied)


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_gradient_at_any_address(offset, rows):
    """dw of the C entry between guards, `offset` elements behind an aligned address."""
    from pratchya_amd import _lib
    lib = _lib.load()
    n, C, V = 100, 4096, 4096
    x, w = _normal((n, C), torch.bfloat16, 1), _normal((C, V), torch.bfloat16, 2, 2.0 / math.sqrt(C))
    t, g = torch.arange(n) * 31 % V, _normal((n,), torch.float32, 3)
    want, bound = reference(x, w, t, 0.0, g)
    xd, wd, td, gd = x.cuda(), (w.t().contiguous() if rows else w).cuda(), t.cuda(), g.cuda()
    ld = C if rows else V
    size = lib.pratchya_linear_cross_entropy_workspace_bytes

    def space(*back):
        return torch.empty(size(xd.data_ptr(), C, wd.data_ptr(), ld, 1, rows, n, C, V, *back), dtype=torch.uint8, device="cuda")
    loss, stats = torch.empty(n, device="cuda"), torch.empty((n, 2), device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    ws = space(0, 0)
    assert lib.pratchya_linear_cross_entropy(xd.data_ptr(), C, wd.data_ptr(), ld, 1, rows, td.data_ptr(), n, C, V, 0.0,
                                             loss.data_ptr(), stats.data_ptr(), ws.data_ptr(), ws.numel(), stream) == _lib.OK
    ws, out = space(0, 1), torch.full((C * V + 32,), 7.0, dtype=torch.bfloat16, device="cuda")
    assert lib.pratchya_linear_cross_entropy_bwd(xd.data_ptr(), C, wd.data_ptr(), ld, 1, rows, td.data_ptr(), stats.data_ptr(),
                                                 gd.data_ptr(), n, C, V, 0.0, None, out.data_ptr() + 2 * offset, ws.data_ptr(),
                                                 ws.numel(), stream) == _lib.OK
    torch.cuda.synchronize()
    dw = out[offset:offset + C * V].view(wd.shape)
    R.close(dw.t() if rows else dw, want[2], bound[2], "dw")
    assert bool((out[:offset] == 7).all()) and bool((out[offset + C * V:] == 7).all())


@pytest.mark.parametrize("n,V,C,ld,tied", [(64, 20032, 64, 131072, True), (40, 1024, 64, 30000000, False)])
def test_weight_inside_a_wider_array(n, V, C, ld, tied):
    """Rows so far apart that a whole piece of them lies beyond 32-bit offsets."""
    from pratchya_amd import functional as F
    x, w = _normal((n, C), torch.bfloat16, 1), _normal((C, V), torch.bfloat16, 2, 0.2)
    t, g = torch.arange(n) * 17 % V, _normal((n,), torch.float32, 3)
    wide = torch.empty((V if tied else C, ld), dtype=torch.bfloat16, device="cuda")
    view = wide[:, :C if tied else V]
    view.copy_(w.t() if tied else w)
    view = view.detach().requires_grad_(True)
    xd = x.cuda().requires_grad_(True)
    y = F.linear_cross_entropy(xd, view.t() if tied else view, t.cuda())
    dx, dw = torch.autograd.grad(y, (xd, view), g.cuda())
    want, bound = reference(x, w, t, 0.0, g)
    R.close(y, want[0], bound[0], "loss")
    R.close(dx, want[1], bound[1], "dx")
    R.close(dw.t() if tied else dw, want[2], bound[2], "dw")


def test_rows_beyond_31_bits():
    """From 256 rows on, of a table and of x so far apart that the tiles take copies of them."""
    from pratchya_amd import functional as F
    n, V, C = 300, 512, 256
    x, w = _normal((n, C), torch.bfloat16, 1), _normal((C, V), torch.bfloat16, 2, 0.2)
    t, g = torch.arange(n) * 17 % V, _normal((n,), torch.float32, 3)
    want, bound = reference(x, w, t, 0.0, g)
    for wide_x in (False, True):
        apart = torch.empty((n if wide_x else V, 1 << 22), dtype=torch.bfloat16, device="cuda")
        view = apart[:, :C]
        view.copy_(x if wide_x else w.t())
        view = view.detach().requires_grad_(True)
        other = (w.t().contiguous() if wide_x else x).cuda().requires_grad_(True)
        xd, table = (view, other) if wide_x else (other, view)
        y = F.linear_cross_entropy(xd, table.t(), t.cuda())
        dx, dw = torch.autograd.grad(y, (xd, table), g.cuda())
        R.close(y, want[0], bound[0], "loss")
        R.close(dx, want[1], bound[1], "dx")
        R.close(dw.t(), want[2], bound[2], "dw")
