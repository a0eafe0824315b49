"""Layer norm and orthogonalised updates where an earlier form of them went wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("rows,cols,dtype,shift,launches", [(3, 4096, torch.bfloat16, 0, 1), (4000, 64, torch.float32, 0, 2), (3, 8193, torch.float32, 0, 3),
                                                            (700, 16384, torch.bfloat16, 0, 2), (700, 16384, torch.bfloat16, 1, 3),
                                                            (700, 16384, torch.float32, 0, 3)])
def test_layer_norm_backward_counts_its_launches(rows, cols, dtype, shift, launches):
    from parallelkernelbench_b200 import _native as nv
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    buf = torch.randn(rows * cols + shift, device="cuda", generator=_gen(1)).to(dtype)
    x = buf[shift:].view(rows, cols)
    _, mean, rstd = layer_norm_fwd(x)
    before = nv.launches()
    layer_norm_bwd(x, None, x, mean, rstd)
    assert nv.launches() - before == launches
