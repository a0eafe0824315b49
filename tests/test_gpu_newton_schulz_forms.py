"""Every form of the Newton-Schulz products, wide and tall, within bounds that a wrong product, edge or remainder does not meet (newton_schulz_bounds).

An optimiser step of scale -1 on a weight of zeros, without momentum and decay, leaves the fp32 result itself: nothing hides behind the rounding to bf16."""
import math

import pytest
import torch
from newton_schulz_bounds import CUBIC, FAST, allowed, distances, emulated, exact, matrix, within

pytestmark = pytest.mark.gpu

# by the rules of the kernels: up to 128 x 4096 in one launch, by one CTA or by clusters of 2 to 16 that share it in whole and in part; then tiles of 128 x 128,
# each on a cluster of 16, 8, 4, 2 or 1, while they fit the GPU at once; then tiles of CTA pairs: only the update's at first, the symmetric products' from about
# 2100 on or in a batch. Sides on and off the multiples of 8, 64, 128 and 256.
ONE_LAUNCH = [(1, 7), (16, 16), (33, 65), (65, 33), (128, 128), (100, 300), (128, 1024), (1024, 128), (64, 2048), (2048, 40), (3, 120, 250), (9, 500, 72),
              (128, 4096), (4095, 127)]
SPLIT = [(129, 130), (130, 129), (70, 4097), (4097, 70), (333, 1000), (1000, 333), (256, 512), (3, 200, 264), (3, 264, 200), (513, 700), (700, 513), (1024, 1024)]
PAIRS = [(1411, 1700), (1700, 1411), (1536, 2048), (2048, 1536), (4, 1101, 1413), (4, 1413, 1101), (4, 1280, 1536), (4, 1536, 1280), (2305, 2401), (2401, 2305)]


def _plain(u, steps, coefficients=FAST):
    """The result in fp32."""
    from parallelkernelbench_b200.ops import muon_step

    p, m = torch.zeros(u.shape, device="cuda"), torch.zeros(u.shape, device="cuda")
    muon_step(p, m, u, lr=1.0, momentum=0.0, nesterov=False, scale=-1.0, steps=steps, coefficients=coefficients)
    assert torch.equal(m, u.float())
    return p


def _hold(got, u, coefficients):
    for g, v in zip(got.reshape(-1, *got.shape[-2:]), u.reshape(-1, *u.shape[-2:])):
        want, bounds = allowed(v, coefficients)
        d = distances(g, want)
        assert all(a <= b for a, b in zip(d, bounds)), (d, bounds)


@pytest.mark.parametrize("kind,steps", [("rank", 1), ("rank", 2), ("low", 2), ("noise", 5), ("low", 5), ("rank", 5)])
@pytest.mark.parametrize("shape", ONE_LAUNCH + SPLIT + PAIRS)
def test_every_form(shape, kind, steps):
    from parallelkernelbench_b200.ops import newton_schulz

    u = matrix(shape, kind, "cuda")
    got = _plain(u, steps)
    _hold(got, u, (FAST,) * steps)
    # the same sums, rounded once
    assert torch.equal(newton_schulz(u, steps=steps), got.to(torch.bfloat16))


@pytest.mark.parametrize("shape,kind,steps", [((m, n), kind, steps) for m, n in ((1411, 1700), (1700, 1411), (2305, 2401))
                                              for kind, steps in (("rank", 1), ("rank", 5), ("low", 5), ("noise", 5)) if m < 2048 or steps == 5])
def test_bounds_bind_at_large_sides(shape, kind, steps):
    """As on the CPU for the smaller ones, without a launch of the kernels. (One step of a rank of four at 2305: twice the emulation's error, most of
    it the sums', is 1.06e-4, as much as bf16 products are off. Five steps tell them apart there.)"""
    u = matrix(shape, kind, "cuda")
    co = (FAST,) * steps
    want, bounds = allowed(u, co)
    assert bounds[0] <= 5e-3
    assert not within(emulated(u, co, dtype=torch.bfloat16), want, bounds)
    assert not within(torch.zeros_like(want), want, bounds)
    assert not within(exact(u, co[:-1] + ((FAST[0], FAST[1], 0.0),)), want, bounds)
    for cut in (lambda t: t[-1].zero_(), lambda t: t[:, -1].zero_(), lambda t: t[:128].zero_(), lambda t: t[:, -256:].zero_()):
        bad = want.clone()
        cut(bad)
        assert not within(bad, want, bounds)


@pytest.mark.parametrize("shape", [(100, 300), (24, 40), (300, 520), (1000, 333), (1411, 1700), (4, 1101, 1413)])
def test_other_coefficients_in_every_form(shape):
    u = matrix(shape, "low", "cuda", seed=1)
    _hold(_plain(u, 8, CUBIC), u, (CUBIC,) * 8)
    per_step = (FAST, (2.0, -1.5, 0.5), CUBIC)
    _hold(_plain(u, 3, per_step), u, per_step)


@pytest.mark.parametrize("shape", [(24, 40), (128, 4096), (333, 1000), (1000, 333), (1411, 1700), (1700, 1411), (4, 1101, 1413), (4, 1413, 1101)])
@pytest.mark.parametrize("nesterov,dtype,offset", [(True, torch.bfloat16, 0), (False, torch.float32, 1), (True, torch.float32, 3)])
def test_the_whole_step(shape, nesterov, dtype, offset):
    """Momentum, combination, decay and copy around the products. The result o of the combination u alone is held to its bounds above; here
    p' = decay p - lr scale o to a rounding of each term, and 1e-4 of the update for values of u that 64 bits round the other way."""
    from parallelkernelbench_b200.ops import muon_step

    n = math.prod(shape)

    def at(t):
        buf = torch.empty(n + offset, dtype=t.dtype, device="cuda")
        buf[offset:].copy_(t.reshape(-1))
        return buf[offset:].view(shape)

    p, m = at(matrix(shape, "noise", "cuda", seed=2) * 0.02), at(matrix(shape, "low", "cuda", seed=3) * 1e-3)
    grad, copy = at((matrix(shape, "noise", "cuda", seed=4) * 1e-3).to(dtype)), at(torch.zeros(shape, device="cuda", dtype=torch.bfloat16))
    p0, m0 = p.double(), m.double()
    lr, mu, decay, scale = 0.05, torch.tensor(0.9).item(), 0.1, 0.2 * math.sqrt(max(shape[-2:]))      # (the kernels take fp32 factors)
    muon_step(p, m, grad, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, p_bf16=copy)
    m1 = mu * m0 + grad.double()
    assert ((m.double() - m1).abs() <= 2.0 ** -23 * (mu * m0.abs() + m1.abs())).all()
    u = (grad.double() + mu * m.double()).float() if nesterov else m.clone()
    o = _plain(u, 5).double()
    want = p0 * (1 - lr * decay) - lr * scale * o
    assert (p.double() - want).norm() <= 2.0 ** -22 * (p0.norm() + lr * scale * o.norm()) + 1e-4 * lr * scale * o.norm()
    assert torch.equal(copy, p.to(torch.bfloat16))


@pytest.mark.parametrize("batch,rows,cols", [(7, 100, 2000), (8, 100, 2000), (15, 64, 1000), (16, 64, 1000), (34, 1000, 64), (75, 64, 500), (149, 60, 250), (8, 90, 4000)])
def test_batches_around_what_is_resident(batch, rows, cols):
    """As many clusters of 16, 8, 4 and 2 as a GPU holds at once, and one more, which waits or takes smaller ones."""
    u = matrix((batch, rows, cols), "noise", "cuda")
    got = _plain(u, 5)
    for i in (0, batch // 2, batch - 1):
        _hold(got[i], u[i], (FAST,) * 5)
