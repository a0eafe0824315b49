"""Layer norm against its definition in 64 bits.

Bounds: u = 2^-24 is half a step of fp32. A row's sum runs over at most cols / 512 + 16 values per thread, 5 steps of a warp and 16 warps, so
it is off by at most K u times the sum of the absolute values with K = cols / 512 + 37 (taken as K = cols / 512 + 64, which leaves room for
the squares' and the inverse root's own roundings). A result is rounded once to its type: eps / 2 of its value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(rows, cols, dtype, param, offset=0.5):
    g = _gen(rows * 7 + cols)
    x = (torch.randn(rows, cols, device="cuda", generator=g) * 2 + offset).to(dtype)
    dy = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    gamma = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(param)
    beta = (0.3 * torch.randn(cols, device="cuda", generator=g)).to(param)
    return x, dy, gamma, beta


def _check(x, dy, gamma, beta, eps, got, stats=None, grads=None):
    xd = x.double().reshape(-1, x.shape[-1])
    cols, half = xd.shape[1], torch.finfo(x.dtype).eps / 2
    gd = torch.ones(cols, device="cuda", dtype=torch.float64) if gamma is None else gamma.double()
    bd = torch.zeros(cols, device="cuda", dtype=torch.float64) if beta is None else beta.double()
    k = cols / 512 + 64
    mean = xd.mean(1, keepdim=True)
    var = ((xd - mean) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (xd - mean) * rstd
    e_mean = k * U * xd.abs().mean(1, keepdim=True)
    # d(xhat): the mean's error, the variance's (relative k u, halved by the root; the mean's error enters it squared) and a few roundings
    e_x = e_mean * rstd * (1 + e_mean * rstd * xhat.abs()) + k * U * xhat.abs() + 2 * U
    y = xhat * gd + bd
    err = (got.double().reshape(xd.shape) - y).abs()
    assert (err <= half * y.abs() + (e_x * gd.abs() + 2 * U * (bd.abs() + y.abs())) * (1 + half)).all(), err.max()
    if stats is not None:
        m, r = (s.double().reshape(-1, 1) for s in stats)
        assert ((m - mean).abs() <= e_mean + U * mean.abs()).all()
        assert ((r - rstd).abs() <= rstd * (k * U + (e_mean * rstd) ** 2)).all()
    if grads is not None:
        dyd = dy.double().reshape(xd.shape)
        dx, dgamma, dbeta = (t.double() for t in grads)
        g = dyd * gd
        c1, c2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
        a1, a2 = g.abs().mean(1, keepdim=True), (g * xhat).abs().mean(1, keepdim=True)
        want = rstd * (g - c1 - xhat * c2)
        e_c2 = k * U * a2 + (g.abs() * e_x).mean(1, keepdim=True)
        e_dx = rstd * (4 * U * g.abs() + k * U * a1 + xhat.abs() * e_c2 + e_x * c2.abs()) + k * U * want.abs() + 4 * U * rstd * (xhat * c2).abs()
        err = (dx.reshape(xd.shape) - want).abs()
        assert (err <= half * want.abs() + e_dx * (1 + half)).all(), err.max()
        n = xd.shape[0] + 16                  # a sum of that many terms, in any order
        assert ((dgamma - (dyd * xhat).sum(0)).abs() <= (n * U * (dyd * xhat).abs() + dyd.abs() * e_x).sum(0) * (1 + n * U)).all()
        assert ((dbeta - dyd.sum(0)).abs() <= n * U * dyd.abs().sum(0)).all()


# one column, one access, the ends of a team's reach (32, 64, 128, 256, 512 threads of 16 values) and one more, rows that start at odd
# addresses, rows beyond the teams, more rows than the grid takes at a time
SHAPES = [(1, 1), (3, 2), (1, 4096), (3, 7), (5, 8), (7, 512), (7, 513), (9, 520), (9, 1024), (2, 1032), (33, 2048), (3, 2056), (17, 4096), (5, 4097),
          (5, 4104), (3, 8192), (2, 8193), (3, 8200), (2, 20001), (300, 8200), (2500, 64), (1333, 1001), (9001, 33),
          # the last rows that a cluster's launch takes backward, and one more, at every team's width; a few hundred wide rows
          (1024, 500), (1025, 500), (512, 1000), (513, 1000), (257, 2048), (129, 4096), (400, 4104), (129, 8192),
          # many wide rows (the ring): every width class, the last row of a round and one more, a row that is no multiple of a thread's access
          (2400, 1032), (1185, 2048), (1400, 2056), (1184, 4096), (1185, 4096), (3000, 4104), (600, 8192), (700, 8200), (301, 16384), (400, 16392),
          # the same of rows that start anywhere
          (2400, 1025), (1300, 2047), (1400, 2049), (1301, 4095), (700, 4097), (400, 8191), (330, 8193), (310, 9001), (307, 12280), (303, 12290), (300, 16383)]


@pytest.mark.parametrize("dtype,param", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32),
                                         (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward_and_backward(rows, cols, dtype, param):
    from parallelkernelbench_b200.ops import layer_norm, layer_norm_bwd, layer_norm_fwd

    x, dy, gamma, beta = _inputs(rows, cols, dtype, param)
    y, mean, rstd = layer_norm_fwd(x, gamma, beta, 1e-5)
    grads = layer_norm_bwd(x, gamma, dy, mean, rstd)
    assert y.dtype == dtype and mean.shape == (rows,) and grads[1].dtype == torch.float32
    _check(x, dy, gamma, beta, 1e-5, y, (mean, rstd), grads)
    assert torch.equal(layer_norm(x, gamma, beta, 1e-5), y)
    for a, b in zip(grads, layer_norm_bwd(x, gamma, dy, mean, rstd)):
        assert torch.equal(a, b)              # the same bits again


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_without_gain_and_bias(dtype):
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    x, dy, gamma, beta = _inputs(40, 264, dtype, torch.float32)
    for g, b in ((None, None), (gamma, None), (None, beta)):
        y, mean, rstd = layer_norm_fwd(x, g, b)
        _check(x, dy, g, b, 1e-5, y, (mean, rstd), layer_norm_bwd(x, g, dy, mean, rstd))


@pytest.mark.parametrize("cols", [96, 1000, 9000])
def test_rows_far_from_zero(cols):
    """A common offset of 1000 times the spread: the variance must not be a difference of two large numbers."""
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    x, dy, gamma, beta = _inputs(11, cols, torch.float32, torch.float32, offset=2000.0)
    y, mean, rstd = layer_norm_fwd(x, gamma, beta)
    _check(x, dy, gamma, beta, 1e-5, y, (mean, rstd), layer_norm_bwd(x, gamma, dy, mean, rstd))


def test_constant_rows():
    from parallelkernelbench_b200.ops import layer_norm, layer_norm_fwd

    x = torch.full((4, 256), 3.0, device="cuda")
    y, mean, rstd = layer_norm_fwd(x)
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(mean, torch.full((4,), 3.0, device="cuda"))
    assert torch.isfinite(rstd).all()
    assert torch.equal(layer_norm(torch.full((3, 1), 7.5, device="cuda"), None, torch.full((1,), 2.0, device="cuda")), torch.full((3, 1), 2.0, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_backward_of_large_constant_rows(dtype):
    """xhat is zero although mean * rstd leaves fp32: so dx = rstd (g - mean(g)), with the sum of the mean's error. Team form, then the rings."""
    from parallelkernelbench_b200.ops import layer_norm_bwd

    for rows, cols in ((5, 1101), (1300, 1101), (1300, 1104), (700, 5000), (700, 5001)):
        _, dy, gamma, _ = _inputs(rows, cols, dtype, torch.float32)
        x = torch.full_like(dy, 2.0 ** 110)
        mean, rstd = torch.full((rows,), 2.0 ** 110, device="cuda"), torch.full((rows,), 2.0 ** 20, device="cuda")
        dx, dgamma, dbeta = (t.double() for t in layer_norm_bwd(x, gamma, dy, mean, rstd))
        g = dy.double() * gamma.double()
        want = 2.0 ** 20 * (g - g.mean(1, keepdim=True))
        slack = 2.0 ** 20 * ((cols / 512 + 64) * U * g.abs().mean(1, keepdim=True) + 4 * U * g.abs())
        half = torch.finfo(dtype).eps / 2
        assert ((dx - want).abs() <= half * want.abs() + slack * (1 + half)).all()
        assert not dgamma.any()
        assert ((dbeta - dy.double().sum(0)).abs() <= (rows + 16) * U * dy.double().abs().sum(0)).all()


def test_a_bad_row_stays_alone():
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    x, dy, gamma, beta = _inputs(6, 1024, torch.float32, torch.float32)
    good = layer_norm_fwd(x, gamma, beta)[0]
    x[2, 5], x[4, 0] = float("nan"), float("inf")
    y, mean, rstd = layer_norm_fwd(x, gamma, beta)
    dx = layer_norm_bwd(x, gamma, dy, mean, rstd)[0]
    for r in range(6):
        assert torch.isnan(y[r]).any() == (r in (2, 4)) and torch.isnan(dx[r]).any() == (r in (2, 4))
        if r not in (2, 4):
            assert torch.equal(y[r], good[r])


# views: off the 16-byte boundary, rows apart, more dimensions, the inner dimension not contiguous, one row for all
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("view", ["offset", "pitch", "odd_pitch", "dims", "transposed", "expanded"])
def test_layouts(view, dtype):
    _layouts(view, dtype, 24)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("view", ["offset", "pitch", "odd_pitch", "expanded", "odd_expanded", "overlapping"])
def test_layouts_of_many_wide_rows(view, dtype):
    """The first and last rows' ends are what copies of whole 16-byte pieces must not reach across."""
    _layouts(view, dtype, 1300, 4)


def _layouts(view, dtype, rows, times=1):
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    n = 512 * times
    x, dy, gamma, beta = _inputs(rows, n + 8, dtype, torch.float32)

    def lay(t):
        if view == "offset":
            return t.reshape(-1)[1:1 + (rows - 1) * n].view(rows - 1, n)
        if view == "pitch":
            return t[:, :n]
        if view == "odd_pitch":
            return torch.nn.functional.pad(t, (0, 1))[:, :n]
        if view == "dims":
            return t[:, :n].reshape(2, 3, 4, n)
        if view == "transposed":
            return t[:, :n].t().contiguous().t()
        if view == "odd_expanded":
            return t[:1, 1:n + 1].expand(rows, n)
        if view == "overlapping":
            return t.reshape(-1)[3:].as_strided((rows, n), (5, 1), t.storage_offset() + 3)
        return t[:1, :n].expand(rows, n)

    xv, dyv, g, b = lay(x), lay(dy), gamma[:n], beta[:n]
    before = (x.clone(), dy.clone())
    y, mean, rstd = layer_norm_fwd(xv, g, b)
    assert y.shape == xv.shape and mean.shape == xv.shape[:-1]
    _check(xv, dyv, g, b, 1e-5, y, (mean, rstd), layer_norm_bwd(xv, g, dyv, mean, rstd))
    # gain and bias off the 16-byte boundary
    y, mean, rstd = layer_norm_fwd(xv, gamma[1:n + 1], beta[1:n + 1])
    _check(xv, dyv, gamma[1:n + 1], beta[1:n + 1], 1e-5, y, (mean, rstd), layer_norm_bwd(xv, gamma[1:n + 1], dyv, mean, rstd))
    assert torch.equal(x, before[0]) and torch.equal(dy, before[1])


def test_no_rows():
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    x = torch.empty(0, 48, device="cuda")
    y, mean, rstd = layer_norm_fwd(x)
    dx, dg, db = layer_norm_bwd(x, None, x, mean, rstd)
    assert y.shape == (0, 48) and mean.shape == (0,) and dx.shape == (0, 48)
    assert torch.equal(dg, torch.zeros(48, device="cuda")) and torch.equal(db, torch.zeros(48, device="cuda"))


def test_gradient_against_differences():
    from parallelkernelbench_b200.ops import layer_norm, layer_norm_bwd, layer_norm_fwd

    x, dy, gamma, beta = _inputs(3, 40, torch.float32, torch.float32)
    _, mean, rstd = layer_norm_fwd(x, gamma, beta)
    dx, dgamma, dbeta = layer_norm_bwd(x, gamma, dy, mean, rstd)
    for t, grad in ((x, dx), (gamma, dgamma), (beta, dbeta)):
        d = torch.randn(t.shape, device="cuda", generator=_gen(5))
        h = 2.0 ** -6
        up = (layer_norm(*(v + h * d if v is t else v for v in (x, gamma, beta))).double() * dy.double()).sum()
        down = (layer_norm(*(v - h * d if v is t else v for v in (x, gamma, beta))).double() * dy.double()).sum()
        # the central difference of 120 outputs of at most 5: each is known to 2^-20, divided by 2h, plus h^2 / 6 times a third derivative
        # that is under 2^6 for rows of unit spread
        assert abs((up - down) / (2 * h) - (grad.double() * d.double()).sum()) <= 120 * 5 * 2.0 ** -20 / h + h * h * 2 ** 6


def test_streams_and_graphs():
    from parallelkernelbench_b200.ops import layer_norm_bwd, layer_norm_fwd

    x, dy, gamma, beta = _inputs(64, 768, torch.bfloat16, torch.float32)

    def both():
        y, mean, rstd = layer_norm_fwd(x, gamma, beta)
        return (y, mean, rstd, *layer_norm_bwd(x, gamma, dy, mean, rstd))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both()
        graphs.append((g, out))
    for t in (x, dy):
        t.mul_(-0.5)
    for g, _ in graphs:
        g.replay()
    want2 = both()
    torch.cuda.synchronize()
    for k in range(6):
        assert torch.equal(got[k], want[k])
        assert torch.equal(graphs[0][1][k], want2[k]) and torch.equal(graphs[1][1][k], want2[k])
