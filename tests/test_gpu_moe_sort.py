"""Tokens sorted by expert and back against their definitions: whole numbers exactly, sums in 64 bits.

Bounds: u = 2^-24 is half a step of fp32; a sum of k products is off by at most (k + 1) u times the sum of their absolute values, a dot product
over a row of H by (H / 256 + 32) u (a thread adds at most H / 256 + 8 products, then 5 steps of a warp and 8 warps); a result is rounded
once to its type, eps / 2 of its value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _sort_ref(idx, experts):
    flat = idx.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    kept = int((key < experts).sum())
    offsets = torch.cat([key.new_zeros(1), torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0)])
    slots = torch.full_like(flat, -1)
    slots[order[:kept]] = torch.arange(kept, device=flat.device)
    order[kept:] = -1
    return offsets.int(), order.int(), slots.int(), kept


def _indices(tokens, k, experts, kind):
    g = _gen(tokens * 31 + k * 7 + experts)
    if kind == "distinct":
        return torch.rand(tokens, experts, device="cuda", generator=g).topk(min(k, experts), -1).indices.int().contiguous()
    idx = torch.randint(0, experts, (tokens, k), device="cuda", generator=g, dtype=torch.int32)
    if kind == "one":
        idx.fill_(experts - 1)
    elif kind == "none":
        idx.fill_(-1)
    elif kind == "dropped":
        idx[torch.rand(tokens, k, device="cuda", generator=g) < 0.4] = -1
        idx[::3] = experts                                   # tokens without any expert, named by a value that is none
        idx[1::7, 0] = -2 ** 31
        idx[2::7, 0] = 2 ** 31 - 1
    return idx


# one assignment; the last of a warp's round and one more; many experts; the end of the one-CTA form (8192 assignments) and one more; a size
# whose runs end inside a round; more assignments than one pass of every warp
@pytest.mark.parametrize("tokens,k,experts", [(1, 1, 1), (1, 8, 256), (4, 8, 64), (11, 3, 7), (33, 1, 1024), (500, 8, 1000), (1024, 8, 256), (8193, 1, 5),
                                              (5000, 2, 16), (8192, 8, 256), (40001, 3, 128)])
@pytest.mark.parametrize("kind", ["any", "distinct", "one", "none", "dropped"])
def test_sort(tokens, k, experts, kind):
    from parallelkernelbench_b200.ops.moe import sort_by_expert

    idx = _indices(tokens, k, experts, kind)
    srt = sort_by_expert(idx, experts)
    offsets, order, slots, _ = _sort_ref(idx, experts)
    assert torch.equal(srt.offsets, offsets) and torch.equal(srt.order, order) and torch.equal(srt.slots, slots)
    assert srt.offsets.dtype == srt.order.dtype == srt.slots.dtype == torch.int32


def _case(tokens, k, experts, hidden, dtype, kind):
    g = _gen(tokens + hidden)
    idx = _indices(tokens, k, experts, kind)
    k = idx.shape[1]
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    return idx, r(tokens, hidden), r(tokens * k, hidden), r(tokens, hidden), r(tokens * k, hidden), torch.rand(tokens, k, device="cuda", generator=g)


def _refs(idx, experts, x, y, dout, dxp, gates):
    offsets, order, slots, kept = _sort_ref(idx, experts)
    t, k = idx.shape
    tok = order[:kept].long() // k
    gate = gates.double().reshape(-1)[order[:kept].long()][:, None]
    xp, dy = torch.zeros_like(dxp), torch.zeros_like(y, dtype=torch.float64)
    xp[:kept] = x[tok]
    dy[:kept] = gate * dout.double()[tok]
    zero = torch.zeros(t, x.shape[1], device="cuda", dtype=torch.float64)
    yk = y[:kept].double()
    out, out_abs = zero.index_add(0, tok, gate * yk), zero.index_add(0, tok, (gate * yk).abs())
    dx, dx_abs = zero.index_add(0, tok, dxp[:kept].double()), zero.index_add(0, tok, dxp[:kept].double().abs())
    dg, dg_abs = (torch.zeros(t * k, device="cuda", dtype=torch.float64) for _ in range(2))
    prod = yk * dout.double()[tok]
    dg[order[:kept].long()], dg_abs[order[:kept].long()] = prod.sum(1), prod.abs().sum(1)
    return xp, (out, out_abs), (dx, dx_abs), dy, (dg.view(t, k), dg_abs.view(t, k)), kept


def _check(idx, experts, x, y, dout, dxp, gates):
    from parallelkernelbench_b200.ops.moe import permute_tokens, permute_tokens_bwd, sort_by_expert, unpermute_tokens, unpermute_tokens_bwd

    srt = sort_by_expert(idx, experts)
    k, h, half = idx.shape[1], x.shape[1], torch.finfo(x.dtype).eps / 2
    xp_r, (out_r, out_a), (dx_r, dx_a), dy_r, (dg_r, dg_a), kept = _refs(idx, experts, x, y, dout, dxp, gates)
    # rows behind the last expert's hold whatever was there before: they must not be read
    yy, gg = y.clone(), dxp.clone()
    yy[kept:], gg[kept:] = float("nan"), float("nan")
    assert torch.equal(permute_tokens(x, srt), xp_r)
    out, dx = unpermute_tokens(yy, srt, gates), permute_tokens_bwd(gg, srt)
    dy, dg = unpermute_tokens_bwd(dout, yy, srt, gates)
    assert out.dtype == dx.dtype == dy.dtype == x.dtype and dg.dtype == torch.float32
    for got, want, mag in ((out, out_r, out_a), (dx, dx_r, dx_a)):
        assert ((got.double() - want).abs() <= half * want.abs() + (k + 1) * U * mag * (1 + half)).all()
    assert ((dy.double() - dy_r).abs() <= half * dy_r.abs()).all()
    assert ((dg.double() - dg_r).abs() <= (h / 256 + 32) * U * dg_a).all()
    again = unpermute_tokens_bwd(dout, yy, srt, gates)
    assert torch.equal(again[0], dy) and torch.equal(again[1], dg) and torch.equal(unpermute_tokens(yy, srt, gates), out)


# widths: one value, one access, a team's reach and one access more, several pieces per row, odd ones (single values per access)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,k,experts,hidden", [(1, 1, 1, 1), (1, 8, 256, 7168), (3, 2, 4, 8), (37, 4, 9, 100), (64, 2, 8, 1024), (50, 8, 16, 1001),
                                                     (19, 9, 32, 264), (5, 17, 40, 4104), (2, 3, 5, 16392), (4, 2, 6, 5001), (3000, 3, 64, 72)])
@pytest.mark.parametrize("kind", ["any", "dropped"])
def test_rows(tokens, k, experts, hidden, dtype, kind):
    _check(*(lambda c: (c[0], experts, *c[1:]))(_case(tokens, k, experts, hidden, dtype, kind)))


@pytest.mark.parametrize("kind", ["none", "one"])
def test_all_dropped_and_all_to_one(kind):
    _check(*(lambda c: (c[0], 12, *c[1:]))(_case(130, 3, 12, 136, torch.bfloat16, kind)))


# the same expert twice in a token's list gives it two rows
def test_the_same_expert_twice():
    idx = torch.tensor([[3, 3], [3, 1], [0, 0]], device="cuda", dtype=torch.int32)
    _check(idx, 4, *_case(3, 2, 4, 64, torch.float32, "any")[1:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts(dtype):
    """Rows apart, off the 16-byte boundary, columns not contiguous, the same row for all."""
    idx, x, y, dout, dxp, gates = _case(40, 4, 8, 264, dtype, "dropped")
    wide = lambda t: torch.nn.functional.pad(t, (0, 3))  # noqa: E731
    _check(idx, 8, wide(x)[:, :264], wide(y)[:, :264], wide(dout)[:, :264], wide(dxp)[:, :264], gates)
    _check(idx, 8, *(t[:, :256] for t in (x, y, dout, dxp)), gates)
    _check(idx, 8, *(t[:, 1:257] for t in (x, y, dout, dxp)), gates)
    _check(idx, 8, *(t.t().contiguous().t() for t in (x, y, dout, dxp)), gates.t().contiguous().t())
    _check(idx.t().contiguous().t(), 8, x[:1].expand(40, 264), y, dout[:1].expand(40, 264), dxp, gates)


def test_no_tokens():
    from parallelkernelbench_b200.ops.moe import permute_tokens, permute_tokens_bwd, sort_by_expert, unpermute_tokens, unpermute_tokens_bwd

    for shape in ((0, 2), (3, 0)):
        t, k = shape
        srt = sort_by_expert(torch.empty(shape, dtype=torch.int32, device="cuda"), 6)
        assert torch.equal(srt.offsets, torch.zeros(7, dtype=torch.int32, device="cuda")) and srt.order.numel() == 0
        x, y, g = torch.ones(t, 16, device="cuda"), torch.empty(0, 16, device="cuda"), torch.empty(shape, device="cuda")
        assert permute_tokens(x, srt).shape == (0, 16)
        for got in (unpermute_tokens(y, srt, g), permute_tokens_bwd(y, srt)):
            assert torch.equal(got, torch.zeros(t, 16, device="cuda"))
        dy, dg = unpermute_tokens_bwd(x, y, srt, g)
        assert dy.shape == (0, 16) and dg.shape == shape


def test_unweighted_is_weights_of_one():
    from parallelkernelbench_b200.ops.moe import sort_by_expert, unpermute_tokens

    idx, _, y, _, _, gates = _case(30, 5, 8, 320, torch.bfloat16, "dropped")
    srt = sort_by_expert(idx, 8)
    assert torch.equal(unpermute_tokens(y, srt), unpermute_tokens(y, srt, torch.ones_like(gates)))


def test_streams_and_graphs():
    from parallelkernelbench_b200.ops.moe import permute_tokens, permute_tokens_bwd, sort_by_expert, unpermute_tokens, unpermute_tokens_bwd

    idx, x, y, dout, dxp, gates = _case(3000, 4, 32, 256, torch.bfloat16, "dropped")

    def everything():
        srt = sort_by_expert(idx, 32)
        return (srt.offsets, srt.order, srt.slots, permute_tokens(x, srt), unpermute_tokens(y, srt, gates), permute_tokens_bwd(dxp, srt),
                *unpermute_tokens_bwd(dout, y, srt, gates))

    want = everything()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = everything()
        graphs.append((g, out))
    idx.copy_(idx.flip(0).clone())
    x.neg_()
    for g, _ in graphs:
        g.replay()
    want2 = everything()
    torch.cuda.synchronize()
    for a, b, c, d, e in zip(got, want, graphs[0][1], graphs[1][1], want2):
        assert torch.equal(a, b) and torch.equal(c, e) and torch.equal(d, e)
