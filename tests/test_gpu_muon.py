"""Newton-Schulz products and the step around them against their definition in 64 bits.

Bound. A step is f(s) = a s + b s^3 + c s^5 of the singular values. To first order an error E of X grows by at most L = max |f'| over the
singular values reached (the divided differences of an odd polynomial are bounded by its derivative), and a step adds, with h = 2^-11 for a
rounding to fp16 (half a step relative to the value; the iterate itself stays in fp32, so its own rounding to fp16 enters only the products):
  A from rounded factors and rounded itself:  dA <= 2 h |X|_2 |X|_F + h |A|_F
  B rounded, from A:                          dB <= (|b| + 2 |c| |A|_2) dA + h |B|_F
  X' = a X + B X:                             dX <= dB |X|_2 + |B|_2 h |X|_F
all in the Frobenius norm, with the norms of the 64-bit iterates, 10 % for second order, the fp32 sums (K 2^-24 with K below 2^12, half
of h at most for the sizes here) and subnormal fp16 entries (2^-25 each, over at most 2^21 of them: below 1e-4). The result is rounded to bf16: 2^-8 of it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
FAST = (3.4445, -4.7750, 2.0315)
CUBIC = (1.5, -0.5, 0.0)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _exact(u, steps=5, coefficients=FAST, eps=1e-7):
    """(X, bound on the Frobenius norm of its error) of one matrix in 64 bits."""
    x = u.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.mT
    per = coefficients if isinstance(coefficients[0], tuple) else (coefficients,) * steps
    h, err = 1.5 * 2.0 ** -11, 2.0 ** -22
    for a, b, c in per:
        gram = x @ x.mT
        poly = b * gram + c * (gram @ gram)
        sv = torch.linalg.eigvalsh(gram).clamp(min=0).sqrt()
        top = sv.max().item()
        s = torch.linspace(0, top * 1.05, 1024, dtype=torch.float64)
        lip = (a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max().item()
        xf = x.norm().item()
        da = 2 * h * top * xf + h * gram.norm().item()
        db = (abs(b) + 2 * abs(c) * top ** 2) * da + h * poly.norm().item()
        err = 1.1 * (lip * err + db * top + torch.linalg.matrix_norm(poly, 2).item() * h * xf) + 1e-4
        x = a * x + poly @ x
    return (x.mT if tall else x), err


def _matrix(shape, kind, seed=0):
    g = _gen(seed + shape[-1])
    m, n = shape[-2:]
    if kind == "noise":
        return torch.randn(*shape, device="cuda", generator=g)
    r = max(1, min(m, n) // 16)
    low = torch.randn(*shape[:-1], r, device="cuda", generator=g) @ torch.randn(*shape[:-2], r, n, device="cuda", generator=g)
    return low + 0.02 * torch.randn(*shape, device="cuda", generator=g)


def _check(out, u, **kw):
    want, err = _exact(u, **kw)
    diff = (out.double() - want).norm().item()
    assert diff <= err + 2.0 ** -8 * want.norm().item(), (diff, err)
    return diff / max(want.norm().item(), 1e-30)


# one value, rows and columns of one, slices of the one-launch form (a side of up to 128, the longer up to 4096) that end anywhere, the first
# sizes beyond it, the edges of tiles (256) and of a CTA's half (128), odd sides, wide and tall, a long inner extent
SHAPES = [(1, 1), (1, 5), (5, 1), (7, 3), (16, 16), (3, 2000), (64, 2048), (2048, 40), (128, 128), (129, 127), (33, 65), (128, 4096), (3001, 96), (70, 4097),
          (4100, 128), (129, 300), (1, 5000), (5000, 1), (3, 16001), (9000, 17), (256, 256), (257, 255), (333, 1000), (1000, 333),
          (512, 1024), (640, 512), (1025, 513)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["noise", "low"])
@pytest.mark.parametrize("shape", SHAPES)
def test_newton_schulz(shape, kind, dtype):
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix(shape, kind).to(dtype)
    out = newton_schulz(u)
    assert out.dtype == torch.bfloat16 and out.shape == u.shape
    _check(out, u)
    assert torch.equal(newton_schulz(u), out)


@pytest.mark.parametrize("coefficients,steps", [(CUBIC, 8), (FAST, 1), ((FAST, CUBIC, CUBIC), 3), ([list(FAST), list(CUBIC)], 2)])
def test_other_coefficients(coefficients, steps):
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix((300, 520), "noise")
    out = newton_schulz(u, steps=steps, coefficients=coefficients)
    _check(out, u, steps=steps, coefficients=tuple(map(tuple, coefficients)) if isinstance(coefficients[0], (list, tuple)) else coefficients)


@pytest.mark.parametrize("shape", [(4, 100, 300), (2, 3, 260, 72), (5, 1, 9)])
def test_batches_are_matrices_of_their_own(shape):
    """Each matrix of a batch comes out as it does alone, whatever stands beside it: zeros, infinities, NaN."""
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix(shape, "noise").to(torch.bfloat16)
    flat = u.view(-1, *shape[-2:])
    flat[1] = 0
    flat[2, 0, 0] = float("inf")
    flat[3, -1, -1] = float("nan")
    out = newton_schulz(u).view_as(flat)
    for i in range(flat.shape[0]):
        if i in (2, 3):
            assert torch.isnan(out[i]).any()
        else:
            assert torch.equal(out[i], newton_schulz(flat[i]))
    assert torch.equal(out[1], torch.zeros_like(out[1]))


@pytest.mark.parametrize("shape", [(4, 200, 300), (4, 513, 257), (4, 40, 4100), (2, 2, 4099, 33), (4, 1300, 1290)])
def test_a_bad_matrix_stays_alone(shape):
    """The same batch with and without bad neighbours: bit for bit the same for the others. (Alone a matrix may be split in another way.)"""
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix(shape, "noise").to(torch.bfloat16)
    flat = u.view(-1, *shape[-2:])
    clean = newton_schulz(u).view_as(flat)
    flat[1] = 0
    flat[2, 0, 0] = float("inf")
    flat[3, -1, -1] = float("nan")
    out = newton_schulz(u).view_as(flat)
    assert torch.equal(out[0], clean[0]) and torch.equal(out[1], torch.zeros_like(out[1]))
    assert torch.isnan(out[2]).any() and torch.isnan(out[3]).any()
    _check(out[0], flat[0])


@pytest.mark.parametrize("batch,rows,cols", [(7, 64, 512), (40, 100, 72), (70, 12, 1000), (3, 1500, 90)])
def test_many_small_matrices(batch, rows, cols):
    """However many CTAs share a matrix, and whether or not all matrices are resident at once."""
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix((batch, rows, cols), "noise").to(torch.bfloat16)
    out = newton_schulz(u)
    for i in (0, 1, batch // 2, batch - 1):
        _check(out[i], u[i])


def test_more_steps_than_one_launch_takes():
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix((24, 40), "noise")
    for steps in (16, 17):
        _check(newton_schulz(u, steps=steps, coefficients=CUBIC), u, steps=steps, coefficients=CUBIC)


@pytest.mark.parametrize("factor", [1e-30, 1e-12, 1e25])
def test_scale_of_the_input(factor):
    """|u| may be far from one: its square does not fit fp32 for the outer two. eps counts against |u| itself."""
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix((96, 160), "noise") * factor
    _check(newton_schulz(u, eps=0.0), u, eps=0.0)
    _check(newton_schulz(u), u)


@pytest.mark.parametrize("shape", [(96, 160), (9, 1000), (200, 264)])
@pytest.mark.parametrize("eps", [0.0, 1e-300, 1e-7])
def test_zeros_stay_zero(shape, eps):
    from parallelkernelbench_b200.ops import newton_schulz

    out = newton_schulz(torch.zeros(shape, device="cuda"), eps=eps)
    assert torch.equal(out, torch.zeros_like(out))


def test_layouts():
    from parallelkernelbench_b200.ops import newton_schulz

    u = _matrix((200, 264), "noise")
    for v in (u.t(), u[:, :256], u[:, 1:258], u.reshape(-1)[1:1 + 199 * 264].view(199, 264), u[:1].expand(200, 264)):
        _check(newton_schulz(v), v)
        _check(newton_schulz(v.to(torch.bfloat16)), v.to(torch.bfloat16))


def test_nothing():
    from parallelkernelbench_b200.ops import muon_step, newton_schulz

    for shape in ((0, 4), (4, 0), (0, 3, 5)):
        t = torch.empty(shape, device="cuda")
        assert newton_schulz(t).shape == shape
        muon_step(t, t.clone(), t, lr=0.1)


def _step(shape, dtype, nesterov, decay, copy, offset=0):
    g = _gen(shape[-1] + offset)

    def at(t):        # a tensor that starts `offset` elements after an aligned address
        buf = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")
        v = buf[offset:].view(t.shape)
        v.copy_(t)
        return v

    p = at(torch.randn(*shape, device="cuda", generator=g) * 0.02)
    m = at(_matrix(shape, "low", 1) * 1e-3)
    grad = at((_matrix(shape, "noise", 2) * 1e-3).to(dtype))
    pb = at(torch.zeros(shape, device="cuda", dtype=torch.bfloat16)) if copy else None
    return p, m, grad, pb


@pytest.mark.parametrize("shape", [(40, 72), (72, 40), (300, 130), (257, 512), (3, 128, 256), (1, 9), (2, 200, 333), (4200, 24), (1700, 1411)])
@pytest.mark.parametrize("dtype,nesterov,decay,copy,offset", [(torch.bfloat16, True, 0.1, True, 0), (torch.float32, False, 0.0, False, 0),
                                                              (torch.bfloat16, False, 0.1, True, 1), (torch.float32, True, 0.1, False, 3)])
def test_muon_step(shape, dtype, nesterov, decay, copy, offset):
    from parallelkernelbench_b200.ops import muon_step

    p, m, grad, pb = _step(shape, dtype, nesterov, decay, copy, offset)
    p0, m0, g0 = p.double().clone(), m.double().clone(), grad.clone()
    lr, mu = 0.02, 0.9
    for _ in range(2):
        want_m = mu * m0 + g0.double()
        muon_step(p, m, grad, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=decay, p_bf16=pb)
        assert torch.equal(grad, g0)
        assert ((m.double() - want_m).abs() <= 2.0 ** -23 * (m0.abs() * mu + want_m.abs())).all()
        u = g0.double() + mu * want_m if nesterov else want_m
        scale = 0.2 * math.sqrt(max(shape[-2:]))
        flat = lambda t: t.reshape(-1, *shape[-2:])  # noqa: E731
        for i, ui in enumerate(flat(u)):
            o, err = _exact(ui)
            want = flat(p0)[i] * (1 - lr * decay) - lr * scale * o
            assert (flat(p)[i].double() - want).norm() <= lr * scale * err + 2.0 ** -22 * (want.norm() + lr * scale * o.norm())
        if pb is not None:
            assert torch.equal(pb, p.to(torch.bfloat16))
        p0, m0 = p.double().clone(), m.double().clone()


def test_scale_is_taken():
    from parallelkernelbench_b200.ops import muon_step, newton_schulz

    p, m, grad, _ = _step((64, 96), torch.float32, True, 0.0, False)
    m.zero_()
    before = p.clone()
    muon_step(p, m, grad, lr=0.5, momentum=0.0, scale=3.0)
    o = newton_schulz(grad).double()
    assert torch.equal(m, grad)
    assert ((before.double() - p.double()) / 1.5 - o).abs().max() <= 2.0 ** -8 * o.abs().max() + 2.0 ** -22


def test_streams_and_graphs():
    from parallelkernelbench_b200.ops import muon_step, newton_schulz

    u = _matrix((2, 300, 520), "noise").to(torch.bfloat16)
    want = newton_schulz(u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = newton_schulz(u)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    p, m, grad, pb = _step((130, 264), torch.bfloat16, True, 0.1, True)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = newton_schulz(u)
            muon_step(p, m, grad, lr=0.01, weight_decay=0.1, p_bf16=pb)
        graphs.append((g, out))
    u.copy_(u.flip(-1).clone())
    q, n = p.clone(), m.clone()
    for g, _ in graphs:
        g.replay()
    for _ in range(2):
        muon_step(q, n, grad, lr=0.01, weight_decay=0.1)
    torch.cuda.synchronize()
    want = newton_schulz(u)
    for _, out in graphs:
        assert torch.equal(out, want)
    assert torch.equal(p, q) and torch.equal(m, n) and torch.equal(pb, p.to(torch.bfloat16))
