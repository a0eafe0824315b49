"""What the Newton-Schulz tests compare with and how much they allow.

The kernels round at known places: the iterate M = k X is fp32 (k a power of two near the root of the longer side), the products take fp16 copies of X, of
A = X X^T and of B = b A + c A^2, and their sums run in fp32. ``emulated`` rounds at the same places, in 64 bits otherwise. Its distance from ``exact`` is
the error that the choice of types causes. The kernels' own is not the same number: a sum that ends a bit off turns some roundings to fp16 the
other way, and after a few steps their roundings are independent of the emulation's; but it is of the same size, and twice that is allowed
(three times in the worst row and column). Against bf16 products (eight times as coarse), a step too few, a row or a column that is missing or a
result of zeros that is binding; tests/test_cpu_newton_schulz_bounds.py shows each.

The sums have to be part of the emulation. Each of K products is added to a running sum of 24 bits whose rest the tensor cores cut off: up to 2^-23 of
the sum each time, always toward zero. In the directions of a matrix that is nothing beside fp16's 2^-11, but in those in which the matrix has nothing it is
all there is, and every further step multiplies it by a = 3.4445, four steps by 140. With K = 2400 the additions of one product alone leave noise of
2^-23 sqrt(K / 12) = 1.7e-6, 2.4e-4 four steps later, and the cut's mean of K / 2 halves of a last bit as much again, where the fp16 roundings of a
matrix of four singular values leave 1.3e-4. (An emulation without the sums allowed 2.5e-4 there, one that rounds them to nearest 3.4e-4, and
kernels that are right were 4.7e-4 off.)"""
import math

import torch

FAST = (3.4445, -4.7750, 2.0315)
CUBIC = (1.5, -0.5, 0.0)
# what fp32 sums and the fp32 iterate leave where the products add next to nothing: a few times 2^-24 of every value, at most this
FLOOR = 2.0 ** -20


def matrix(shape, kind, device="cpu", seed=0):
    """fp32. noise: all singular values of one size; low: a few directions over noise; rank: four singular values of 0.3 to 0.7, on which the products
    weigh from the first step on."""
    g = torch.Generator().manual_seed(1000 * seed + 7 * shape[-2] + shape[-1])
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    lead, (m, n) = shape[:-2], shape[-2:]
    if kind == "noise":
        u = r(*shape)
    elif kind == "low":
        d = max(1, min(m, n) // 16)
        u = r(*lead, m, d) @ r(*lead, d, n) + 0.02 * r(*shape)
    else:
        d = min(4, m, n)
        u = (torch.linalg.qr(r(*lead, m, d))[0] * torch.tensor([0.7, 0.5, 0.4, 0.3], dtype=torch.float64)[:d]) @ torch.linalg.qr(r(*lead, n, d))[0].mT
    return u.float().to(device)


def one_launch(shape):
    """Matrices that stay on the chip for the whole call; they keep B as two fp16 numbers."""
    return min(shape[-2:]) <= 128 and max(shape[-2:]) <= 4096


def _sums(x, y):
    """x @ y of values that fp16 or bf16 hold: every product added to a running sum that keeps the 24 bits of fp32, the rest cut off."""
    acc = torch.zeros(x.shape[0], y.shape[1], dtype=torch.float64, device=x.device)
    bits = acc.view(torch.int64)
    for i in range(x.shape[1]):
        acc.addr_(x[:, i], y[i])
        bits.bitwise_and_(-(1 << 29))            # 53 bits to 24
    return acc


def _iterate(u, coefficients, eps, dtype, head_and_rest):
    x = u.double()
    x = x / (x.norm() + eps)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.mT
    k = 2.0 ** round(math.log2(max(x.shape)) / 2)
    for a, b, c in coefficients:
        if dtype is None:
            gram = x @ x.mT
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        else:
            cut = lambda t: t.float().to(dtype).double()  # noqa: E731
            x16 = cut(x.float().double() * k) / k
            gram = cut(_sums(x16, x16.mT))
            poly = b * gram + c * _sums(gram, gram)
            poly16 = cut(poly)
            move = _sums(poly16, x16)
            if head_and_rest:
                move = move + _sums(cut(poly - poly16), x16)
            x = (a * x + move).float().double()
    return x.mT if tall else x


def exact(u, coefficients, eps=1e-7):
    return _iterate(u, coefficients, eps, None, False)


def emulated(u, coefficients, eps=1e-7, dtype=torch.float16):
    return _iterate(u, coefficients, eps, dtype, one_launch(u.shape))


def allowed(u, coefficients, eps=1e-7):
    """(exact, what its distance may be: of the whole, of the worst row, of the worst column, each relative to its share of the result's norm)."""
    want = exact(u, coefficients, eps)
    d = distances(emulated(u, coefficients, eps), want)
    return want, tuple(factor * v + FLOOR for factor, v in zip((2, 3, 3), d))


def distances(got, want):
    """Of one matrix: Frobenius norm of the difference relative to the result's; the largest row's and column's, relative to those of a result
    whose rows (columns) are all alike."""
    d, norm = got.double() - want, max(want.norm().item(), 1e-30)
    rows, cols = want.shape
    return (d.norm().item() / norm, d.norm(dim=1).max().item() * math.sqrt(rows) / norm, d.norm(dim=0).max().item() * math.sqrt(cols) / norm)


def within(got, want, bounds):
    return all(v <= b for v, b in zip(distances(got, want), bounds))      # (NaN is not)
