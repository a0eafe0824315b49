"""The operators of a MoE layer's training step together, as a program uses them: layer norm, router, sort, experts' products, the way home, all
gradients, and the weights' orthogonalised update.

The reference is autograd in 64 bits on the same routing. Every bf16 tensor on the way is off by at most 2^-8 of itself (2-norm); a linear map by
random weights, a gather or a weighted sum carries a relative error on unchanged in the 2-norm up to its spread, for which a factor of two is
left. The number of roundings on the way to each result is given with it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8


def _setup(tokens, hidden, experts, top_k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return {"x": r(tokens, hidden).to(torch.bfloat16), "gamma": 1 + 0.1 * r(hidden), "beta": 0.1 * r(hidden),
            "router": (r(experts, hidden) / math.sqrt(hidden)).to(torch.bfloat16),
            "w": (r(experts, hidden, hidden) / math.sqrt(hidden)).to(torch.bfloat16), "dout": r(tokens, hidden).to(torch.bfloat16)}


def _forward(s, top_k):
    from parallelkernelbench_b200.ops import gemm_bf16, layer_norm_fwd
    from parallelkernelbench_b200.ops.moe import grouped_gemm, permute_tokens, route_topk, sort_by_expert, unpermute_tokens

    h, mean, rstd = layer_norm_fwd(s["x"], s["gamma"], s["beta"])
    logits = gemm_bf16(h, s["router"], out_dtype=torch.float32)
    gates, idx, _ = route_topk(logits, None, top_k)
    srt = sort_by_expert(idx, s["router"].shape[0])
    hp = permute_tokens(h, srt)
    yp = grouped_gemm(hp, s["w"], srt.offsets)
    return h, mean, rstd, gates, idx, srt, hp, yp, unpermute_tokens(yp, srt, gates)


def _backward(s, saved):
    from parallelkernelbench_b200.ops import layer_norm_bwd
    from parallelkernelbench_b200.ops.moe import grouped_gemm, permute_tokens_bwd, unpermute_tokens_bwd

    h, mean, rstd, gates, idx, srt, hp, yp, _ = saved
    dyp, dgates = unpermute_tokens_bwd(s["dout"], yp, srt, gates)
    dhp = grouped_gemm(dyp, s["w"].transpose(1, 2).contiguous(), srt.offsets)
    dh = permute_tokens_bwd(dhp, srt)
    dx, dgamma, dbeta = layer_norm_bwd(s["x"], s["gamma"], dh, mean, rstd)
    return dyp, dgates, dx, dgamma, dbeta


def _weight_gradients(saved, dyp, experts):
    from parallelkernelbench_b200.ops import gemm_bf16_tn

    srt, hp = saved[5], saved[6]
    dw = torch.zeros(experts, dyp.shape[1], hp.shape[1], device="cuda", dtype=torch.bfloat16)
    off = srt.offsets.tolist()
    for e in range(experts):
        if off[e + 1] > off[e]:
            gemm_bf16_tn(dyp[off[e]:off[e + 1]], hp[off[e]:off[e + 1]], out=dw[e])
    return dw


def _near(got, want, roundings):
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel <= 2 * roundings * HALF, rel


@pytest.mark.parametrize("tokens,hidden,experts,top_k", [(300, 256, 8, 2), (1000, 512, 16, 4), (7, 128, 32, 3)])
def test_a_training_step(tokens, hidden, experts, top_k):
    from parallelkernelbench_b200.ops import muon_step

    s = _setup(tokens, hidden, experts, top_k)
    saved = _forward(s, top_k)
    gates, idx, srt, out = saved[3], saved[4], saved[5], saved[8]
    assert int(srt.offsets[-1]) == tokens * top_k
    dyp, dgates, dx, dgamma, dbeta = _backward(s, saved)
    dw = _weight_gradients(saved, dyp, experts)

    x, gamma, beta, w, gd = (t.double().requires_grad_() for t in (s["x"], s["gamma"], s["beta"], s["w"], gates))
    h = torch.nn.functional.layer_norm(x, (hidden,), gamma, beta, 1e-5)
    y = torch.stack([torch.einsum("th,toh->to", h, w[idx[:, j].long()]) for j in range(top_k)], 1)
    ref = (y * gd[:, :, None]).sum(1)
    ref.backward(s["dout"].double())
    _near(out, ref, 3)                  # h, the experts' outputs, the result
    _near(dgates, gd.grad, 2)           # h, the experts' outputs
    _near(dw, w.grad, 3)                # h, dy, the result
    _near(dx, x.grad, 4)                # dy, dhp, dh, the result
    _near(dgamma, gamma.grad, 3)
    _near(dbeta, beta.grad, 3)

    master, m, copy = s["w"].float(), torch.zeros(s["w"].shape, device="cuda"), s["w"].clone()
    before = master.clone()
    muon_step(master, m, dw, lr=0.01, weight_decay=0.1, p_bf16=copy)
    # the first step's nesterov combination is (1 + momentum) times the gradient; in 64 bits, with the bound of the products' own tests. (A
    # gradient of a few tokens has few directions: rounding the combination to bf16 first would add noise to all others, which five steps
    # lift by up to 3.4445^5 = 485 times.)
    from test_gpu_muon import _exact

    scale = 0.01 * 0.2 * math.sqrt(hidden)
    for e in range(experts):
        o, err = _exact(dw[e].double() * 1.95)
        want = before[e].double() * (1 - 0.001) - scale * o
        assert (master[e].double() - want).norm() <= scale * err + 2.0 ** -22 * (want.norm() + scale * o.norm())
    assert torch.equal(copy, master.to(torch.bfloat16)) and torch.equal(m, dw.float())
    used = (srt.offsets[1:] > srt.offsets[:-1])
    assert (master[~used] == before[~used] * (1 - 0.001)).all()        # experts without tokens only decay


def test_a_captured_step_replays():
    """Forward and backward of a layer in one graph, replayed on other tokens, beside another graph of the same shapes."""
    s = _setup(600, 256, 8, 2)

    def step():
        saved = _forward(s, 2)
        return (saved[8], *_backward(s, saved))

    step()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    s["x"].copy_(s["x"].flip(0).clone() * 0.5)
    s["dout"].neg_()
    for g, _ in graphs:
        g.replay()
    want = step()
    torch.cuda.synchronize()
    for _, out in graphs:
        for a, b in zip(out, want):
            assert torch.equal(a, b)
