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


# every form of the forward: teams with wide and single accesses, the ring at each of its widths, the ring of rows that start anywhere, rows in passes
MEAN_SHAPES = [(5, 1000), (5, 1001), (2, 4097), (3, 7168), (9, 520), (9, 40), (2400, 1032), (1185, 4000), (400, 7168), (303, 12288), (1300, 1101), (700, 4097),
               (310, 7169), (3, 9000), (2, 16400)]
U = 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", MEAN_SHAPES)
def test_layer_norm_of_constant_rows(rows, cols, dtype):
    """Every difference from the first mean is the same small multiple of a step of fp32, so their sum, its quotient and what they leave are exact: the
    mean is the constant, the deviation is eps alone, and the result is the bias."""
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    values = torch.tensor([1e5, 99840.0, -1000.0, 0.1, 1e3, -3e4, 123.456, 7e-3], device="cuda").to(dtype)
    x = values[torch.arange(rows, device="cuda") % len(values)][:, None].expand(rows, cols).contiguous()
    beta = torch.randn(cols, device="cuda", generator=_gen(3))
    y, mean, rstd = layer_norm_fwd(x, None, beta)
    assert torch.equal(y, beta.to(dtype).expand(rows, cols))
    assert torch.equal(mean, x[:, 0].float())
    assert ((rstd.double() * 1e-5 ** 0.5 - 1).abs() <= 2.0 ** -21).all()
    dy = torch.randn(rows, cols, device="cuda", generator=_gen(4)).to(dtype)
    dx, dgamma, _ = layer_norm_bwd(x, None, dy, mean, rstd)
    assert not dgamma.any()
    want = rstd.double()[:, None] * (dy.double() - dy.double().mean(1, keepdim=True))
    slack = rstd.double()[:, None] * ((cols / 512 + 64) * U * dy.double().abs().mean(1, keepdim=True) + 4 * U * dy.double().abs())
    assert ((dx.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 1.01 * slack).all()


@pytest.mark.parametrize("center", [1e3, -3e4, 1e5])
@pytest.mark.parametrize("rows,cols", MEAN_SHAPES)
def test_layer_norm_of_nearly_constant_rows(rows, cols, center):
    """Rows a few steps of fp32 wide. With K = cols / 512 + 64 terms on the way of a sum, the first mean m0 is off by K U |x|; x - m0 is exact (the two
    are within a factor of two of one another); its mean is then off by e = K U (mean|x - mean| + K U |x|) and is all that separates the result
    from (x - mean) rstd, besides the variance's K U, halved by the root, and a few roundings of the result."""
    from parallelkernelbench_b200.ops import layer_norm_fwd

    g = _gen(cols)
    x = center + 0.02 * torch.randn(rows, cols, device="cuda", generator=g)
    y, mean, rstd = layer_norm_fwd(x)
    xd = x.double()
    m = xd.mean(1, keepdim=True)
    d = xd - m
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
    k = cols / 512 + 64
    e = k * U * (d.abs().mean(1, keepdim=True) + k * U * xd.abs().mean(1, keepdim=True))
    assert ((mean.double()[:, None] - m).abs() <= U * m.abs() + e).all()
    assert ((rstd.double()[:, None] - r).abs() <= r * (k * U + (e * r) ** 2)).all()
    assert ((y.double() - d * r).abs() <= e * r + (k * U + (e * r) ** 2) * (d * r).abs() + 4 * U * (d * r).abs()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spread", [0.1, 0.3])
def test_layer_norm_of_millions_of_columns(spread, dtype):
    """A sum's error must not grow with the width: rows one constant distance above and below their mean, whose squares round the same way in every
    addition. 32 terms are added in fp32, the runs in 64 bits, and 512 threads by a tree of 9: K = 32 + 9 + 1 roundings of 2^-24, taken as 64."""
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    cols, k = (1 << 22) + 3, 64
    sign = 1.0 - 2.0 * (torch.arange(cols, device="cuda") % 2)
    x = torch.stack([1.0 + spread * sign, torch.full_like(sign, spread), spread * sign.flip(0) - 0.7]).to(dtype)
    dy = torch.stack([sign * spread + 0.01, torch.full_like(sign, 0.3), torch.randn(cols, device="cuda", generator=_gen(9))]).to(dtype)
    y, mean, rstd = layer_norm_fwd(x, None, None, 1e-5)
    xd, half = x.double(), torch.finfo(dtype).eps / 2
    m = xd.mean(1, keepdim=True)
    d = xd - m
    r = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
    e = k * U * (d.abs().mean(1, keepdim=True) + k * U * xd.abs().mean(1, keepdim=True))
    assert ((mean.double()[:, None] - m).abs() <= U * m.abs() + e).all()
    assert ((rstd.double()[:, None] - r).abs() <= r * (k * U + (e * r) ** 2)).all()
    e_x = e * r + (k * U + (e * r) ** 2) * (d * r).abs() + 4 * U * (d * r).abs()
    assert ((y.double() - d * r).abs() <= half * (d * r).abs() + e_x * (1 + half)).all()
    dx, _, dbeta = layer_norm_bwd(x, None, dy, mean, rstd)
    xh, g = (xd - mean.double()[:, None]) * rstd.double()[:, None], dy.double()
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    want = rstd.double()[:, None] * (g - c1 - xh * c2)
    slack = rstd.double()[:, None] * (k * U * (g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True)) + 8 * U * (g.abs() + (xh * c2).abs()))
    assert ((dx.double() - want).abs() <= half * want.abs() + slack * (1 + half)).all()
    assert ((dbeta.double() - g.sum(0)).abs() <= 4 * U * g.abs().sum(0)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1300, 4096), (1300, 4097), (2401, 1032), (301, 16384), (700, 333), (3, 9000)])
def test_layer_norm_bad_rows_stay_alone(rows, cols, dtype):
    """Rows that share their barriers and shuffles with others: NaN and infinities reach nobody else, nor the rows' own statistics of other rows."""
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    g = _gen(rows + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    dy = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    good = layer_norm_fwd(x)
    want = layer_norm_bwd(x, None, dy, *good[1:])[0]
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for i, (r, c, v) in enumerate([(0, 0, float("nan")), (rows // 2, cols - 1, float("inf")), (rows - 1, cols // 2, float("-inf"))]):
        x[r, c] = v
        bad[r] = True
    y, mean, rstd = layer_norm_fwd(x)
    dx = layer_norm_bwd(x, None, dy, mean, rstd)[0]
    for got, before in ((y, good[0]), (mean, good[1]), (rstd, good[2]), (dx, want)):
        assert torch.equal(got[~bad], before[~bad])
    assert torch.isnan(y[bad]).all() and torch.isnan(dx[bad]).all()


def test_first_calls_inside_a_capture():
    """A process whose first calls are captured: what the library asks the device for once must not end the capture."""
    code = """
import torch
from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd, muon_step, newton_schulz
from parallelkernelbench_b200.ops.moe import permute_tokens, sort_by_expert
t = lambda *s: torch.randn(*s, device="cuda")
u, v, w, x = t(3, 64, 900), t(333, 700), t(4, 600, 900), t(1300, 4096)
idx = torch.randint(0, 16, (9000, 2), device="cuda", dtype=torch.int32)
p, m = t(333, 700), t(333, 700)
def run():
    y, mean, rstd = layer_norm_fwd(x)
    srt = sort_by_expert(idx, 16)
    return [newton_schulz(u), newton_schulz(v), newton_schulz(w), y, *layer_norm_bwd(x, None, y, mean, rstd), srt.slots, permute_tokens(idx.float(), srt)]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = run()
    muon_step(p, m, v, lr=0.0)
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run()))
print("the same")
"""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]
