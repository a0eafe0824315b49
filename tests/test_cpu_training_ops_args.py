"""Refusals of the layer-norm, expert-sort and orthogonalisation entry points: before any launch, so without a GPU."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(4096)
LL, D, F = ctypes.c_longlong, ctypes.c_double, ctypes.c_float


def _refused(rc):
    from parallelkernelbench_b200 import _native as nv

    return rc != 0 and b"bad argument" in nv.cuda_lib().pkb_last_error()


def test_layer_norm_wrappers():
    from parallelkernelbench_b200.ops import layer_norm, layer_norm_bwd, layer_norm_fwd

    x = torch.zeros(4, 8)
    g = torch.ones(8)
    with pytest.raises(TypeError):
        layer_norm(x.half())
    with pytest.raises(TypeError):
        layer_norm(x.long())
    with pytest.raises(ValueError, match="column"):
        layer_norm(torch.zeros(()))
    with pytest.raises(ValueError, match="column"):
        layer_norm(torch.zeros(3, 0))
    for bad in (g[:7], g.half(), torch.ones(16)[::2], g.double()):
        with pytest.raises(ValueError, match="gamma"):
            layer_norm(x, bad)
        with pytest.raises(ValueError, match="beta"):
            layer_norm_fwd(x, g, bad)
    with pytest.raises(TypeError, match="same dtype"):
        layer_norm(x, g, g.to(torch.bfloat16))
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, g, g, -1e-5)
    with pytest.raises(ValueError, match="eps"):
        layer_norm(x, g, g, float("nan"))
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(x, g, g)
    mean, rstd = torch.zeros(4), torch.ones(4)
    for dy in (x.to(torch.bfloat16), x[:3], x.view(2, 2, 8)):
        with pytest.raises(ValueError, match="dy"):
            layer_norm_bwd(x, g, dy, mean, rstd)
    for bad in (mean[:3], mean.double(), torch.zeros(8)[::2]):
        with pytest.raises(ValueError, match="mean"):
            layer_norm_bwd(x, g, x, bad, rstd)
        with pytest.raises(ValueError, match="rstd"):
            layer_norm_bwd(x, g, x, mean, bad)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm_bwd(x, g, x, mean, rstd)


def test_widths_beyond_32_bits():
    """A width is a 32-bit number in the kernels: one that does not fit is refused, not cut off."""
    from parallelkernelbench_b200.ops import layer_norm, layer_norm_bwd
    from parallelkernelbench_b200.ops.moe import ExpertSort, permute_tokens, unpermute_tokens, unpermute_tokens_bwd

    for cols in ((1 << 30) + 1, (1 << 32) + 8):
        x = torch.zeros(1, 1).expand(1, cols)
        with pytest.raises(ValueError, match="column"):
            layer_norm(x)
        with pytest.raises(ValueError, match="column"):
            layer_norm_bwd(x, None, x, torch.zeros(1), torch.zeros(1))
        srt = ExpertSort(torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1, 1)
        for call in (lambda: permute_tokens(x, srt), lambda: unpermute_tokens(x, srt), lambda: unpermute_tokens_bwd(x, x, srt, torch.ones(1, 1))):
            with pytest.raises(ValueError, match="column"):
                call()


def test_expert_sort_wrappers():
    from parallelkernelbench_b200.ops.moe import (ExpertSort, permute_tokens, permute_tokens_bwd, sort_by_expert, unpermute_tokens,
                                                  unpermute_tokens_bwd)

    idx = torch.zeros(4, 2, dtype=torch.int32)
    for bad in (idx.long(), idx.view(-1), idx.float()):
        with pytest.raises(TypeError):
            sort_by_expert(bad, 4)
    for experts in (0, -1, 1025):
        with pytest.raises(ValueError, match="experts"):
            sort_by_expert(idx, experts)
    with pytest.raises(ValueError, match="2\\^31"):
        sort_by_expert(torch.zeros(1, 1, dtype=torch.int32).expand(1 << 16, 1 << 15), 4)
    with pytest.raises(ValueError, match="CUDA"):
        sort_by_expert(idx, 4)
    i32 = torch.zeros(9, dtype=torch.int32)
    srt = ExpertSort(i32[:5], i32[:8], i32[:8], 4, 2)
    x, y, gates = torch.zeros(4, 16), torch.zeros(8, 16), torch.zeros(4, 2)
    with pytest.raises(TypeError):
        permute_tokens(x.half(), srt)
    for bad in (x[:3], x[0], torch.zeros(4, 0), y):
        with pytest.raises(ValueError, match="rows"):
            permute_tokens(bad, srt)
    for bad in (x, torch.zeros(9, 16)):
        with pytest.raises(ValueError, match="rows"):
            unpermute_tokens(bad, srt, gates)
        with pytest.raises(ValueError, match="rows"):
            permute_tokens_bwd(bad, srt)
    for bad in (srt._replace(slots=i32[:7]), srt._replace(slots=i32[:8].long()), srt._replace(offsets=i32[:0]), srt._replace(offsets=i32.long()),
                srt._replace(slots=torch.zeros(16, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError, match="of the sort"):
            permute_tokens(x, bad)
    with pytest.raises(ValueError, match="CUDA"):
        permute_tokens(x, srt)
    meta = ExpertSort(*(t.to("meta") for t in srt[:3]), 4, 2)
    with pytest.raises(ValueError, match="CUDA"):
        unpermute_tokens(y.to("meta"), meta)
    with pytest.raises(ValueError, match="width"):
        _with_device(unpermute_tokens_bwd, x[:, :8], y, srt, gates)
    with pytest.raises(ValueError, match="width"):
        _with_device(unpermute_tokens_bwd, x.to(torch.bfloat16), y, srt, gates)
    for bad in (gates.half(), gates[:, :1], gates[:3], gates.view(-1)):
        with pytest.raises(ValueError, match="gates"):
            _with_device(unpermute_tokens, y, srt, bad)


def _with_device(f, *args):
    """Past the device check, which CPU tensors do not pass: the argument checks behind it."""
    from parallelkernelbench_b200.ops import moe

    real = moe._sort_arg
    moe._sort_arg = lambda srt, like: srt.tokens * srt.top_k
    try:
        return f(*args)
    finally:
        moe._sort_arg = real


def test_orthogonalisation_wrappers():
    from parallelkernelbench_b200.ops import muon_step, newton_schulz

    g = torch.zeros(4, 6)
    with pytest.raises(TypeError):
        newton_schulz(g.half())
    with pytest.raises(ValueError, match="matrices"):
        newton_schulz(g[0])
    with pytest.raises(ValueError, match="step"):
        newton_schulz(g, steps=0)
    with pytest.raises(ValueError, match="eps"):
        newton_schulz(g, eps=-1.0)
    for bad in ((1.0, 2.0), (), ((1.5, -0.5, 0.0), (1.5, -0.5, 0.0)), ((1.5, -0.5),) * 5):
        with pytest.raises(ValueError, match="coefficients"):
            newton_schulz(g, coefficients=bad)
    with pytest.raises(ValueError, match="finite"):
        newton_schulz(g, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(ValueError, match="range"):
        newton_schulz(g, coefficients=(8.0, 0.0, 0.0), steps=8)
    with pytest.raises(ValueError, match="65535"):
        newton_schulz(torch.zeros(1, 1, 1).expand(65536, 1, 1))
    with pytest.raises(ValueError, match="sides"):
        newton_schulz(torch.zeros(1, 1).expand(1 << 24, 1))
    with pytest.raises(ValueError, match="CUDA"):
        newton_schulz(g)
    p, m = torch.zeros(4, 6), torch.zeros(4, 6)
    for bad in (p.to(torch.bfloat16), torch.zeros(6, 4).t()):
        with pytest.raises(TypeError, match="p must"):
            muon_step(bad, m, g, lr=0.1)
        with pytest.raises(TypeError, match="m must"):
            muon_step(p, bad, g, lr=0.1)
    with pytest.raises(TypeError, match="g must"):
        muon_step(p, m, g.half(), lr=0.1)
    for args in ((p, m, g[:3]), (p, torch.zeros(4, 7), g), (p[0], m[0], g[0])):
        with pytest.raises(ValueError, match="one shape"):
            muon_step(*args, lr=0.1)
    for bad in (p, p.to(torch.bfloat16)[:3], torch.zeros(6, 4, dtype=torch.bfloat16).t()):
        with pytest.raises(ValueError, match="p_bf16"):
            muon_step(p, m, g, lr=0.1, p_bf16=bad)
    for args in ((p, p, g), (p, m, m), (p, m, p)):
        with pytest.raises(ValueError, match="different"):
            muon_step(*args, lr=0.1)
    with pytest.raises(ValueError, match="step"):
        muon_step(p, m, g, lr=0.1, steps=0)
    with pytest.raises(ValueError, match="CUDA"):
        muon_step(p, m, g, lr=0.1)


def test_native_entry_points():
    """Error codes and messages, not launches; addresses that nothing reads stand in for the tensors."""
    from parallelkernelbench_b200 import _native as nv

    lib = nv.cuda_lib()
    one = F(1e-5)
    calls = {
        "forward without rows": lambda: lib.pkb_layer_norm_fwd(P, LL(8), P, P, 0, P, P, P, LL(0), 8, one, 0, None),
        "forward without columns": lambda: lib.pkb_layer_norm_fwd(P, LL(8), P, P, 0, P, P, P, LL(1), 0, one, 0, None),
        "forward with half of the statistics": lambda: lib.pkb_layer_norm_fwd(P, LL(8), P, P, 0, P, P, None, LL(1), 8, one, 0, None),
        "forward of an unknown type": lambda: lib.pkb_layer_norm_fwd(P, LL(8), P, P, 0, P, P, P, LL(1), 8, one, 2, None),
        "backward without scratch": lambda: lib.pkb_layer_norm_bwd(P, LL(8), P, LL(8), P, 0, P, P, P, P, P, None, LL(1 << 20), 8, 0, None),
        "backward without a result": lambda: lib.pkb_layer_norm_bwd(P, LL(8), P, LL(8), P, 0, P, P, P, P, None, P, LL(1), 8, 0, None),
        "backward of an unknown type": lambda: lib.pkb_layer_norm_bwd(P, LL(8), P, LL(8), P, 0, P, P, P, P, P, P, LL(1), 8, 3, None),
        "sort of nothing": lambda: lib.pkb_moe_sort(P, LL(0), 4, P, P, P, None),
        "sort of too many": lambda: lib.pkb_moe_sort(P, LL(1 << 31), 4, P, P, P, None),
        "sort by too many experts": lambda: lib.pkb_moe_sort(P, LL(8), 1025, P, P, P, None),
        "permute without tokens": lambda: lib.pkb_moe_permute(P, LL(8), P, P, P, LL(0), 2, 8, 0, None),
        "permute of too many assignments": lambda: lib.pkb_moe_permute(P, LL(8), P, P, P, LL(1 << 30), 2, 8, 0, None),
        "unpermute of an unknown type": lambda: lib.pkb_moe_unpermute(P, LL(8), P, P, P, LL(4), 2, 8, 7, None),
        "unpermute without columns": lambda: lib.pkb_moe_unpermute(P, LL(8), P, P, P, LL(4), 2, 0, 0, None),
        "gradient without weights": lambda: lib.pkb_moe_unpermute_bwd(P, LL(8), P, LL(8), P, None, P, P, P, LL(4), 2, 8, 0, None),
        "no matrices": lambda: lib.pkb_newton_schulz(P, 0, None, F(0), 0, LL(0), 4, 4, P, 5, D(0), P, None, F(0), F(0), None, P, None),
        "too many matrices": lambda: lib.pkb_newton_schulz(P, 0, None, F(0), 0, LL(65536), 4, 4, P, 5, D(0), P, None, F(0), F(0), None, P, None),
        "no steps": lambda: lib.pkb_newton_schulz(P, 0, None, F(0), 0, LL(1), 4, 4, P, 0, D(0), P, None, F(0), F(0), None, P, None),
        "two results": lambda: lib.pkb_newton_schulz(P, 0, None, F(0), 0, LL(1), 4, 4, P, 5, D(0), P, P, F(0), F(0), None, P, None),
        "no result": lambda: lib.pkb_newton_schulz(P, 0, None, F(0), 0, LL(1), 4, 4, P, 5, D(0), None, None, F(0), F(0), None, P, None),
    }
    for what, call in calls.items():
        assert _refused(call()), (what, lib.pkb_last_error())
    lib.pkb_newton_schulz_scratch.restype = LL
    size = lambda b, r, c, steps=5: lib.pkb_newton_schulz_scratch(LL(b), r, c, steps, None)  # noqa: E731
    assert size(0, 4, 4) == size(1, 0, 4) == 0
    assert size(1, 16, 16) == 0                                     # one CTA keeps all
    assert size(1, 128, 4096) == 16 * 65536 + 32768 and size(1, 4096, 128) == size(1, 128, 4096)
    assert size(1, 300, 300) >= 300 * 304 * 8 and size(3, 300, 300) >= 3 * size(1, 300, 300) - 4096
    assert lib.pkb_layer_norm_bwd_partials(LL(0), 8, 0) == 0 and lib.pkb_layer_norm_bwd_partials(LL(1), 8, 0) == 0 and lib.pkb_layer_norm_bwd_partials(LL(1 << 20), 8, 0) > 0
