"""What the layer-norm and orthogonalisation entry points decide on the host before any launch, so without a GPU."""
import ctypes

import pytest

LL = ctypes.c_longlong


def _blocks(rows, cols, dtype, aligned, sms):
    from parallelkernelbench_b200 import _native as nv

    return nv.cuda_lib().pkb_layer_norm_bwd_blocks(LL(rows), cols, dtype, aligned, sms)


@pytest.mark.parametrize("sms", [1, 16, 36, 60, 64, 132, 148, 160])
def test_backward_without_scratch_writes_none(sms):
    """A backward that is told to bring no scratch (one launch of a cluster) must not take a form that writes partial sums, whatever the alignment and
    however few SMs there are: on 60 of them 128 rows of 8192 columns are also enough rows for the ring."""
    for dtype in (0, 1):
        for cols in (1, 64, 512, 513, 1024, 1025, 1032, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16392):
            team_rows = 1 if cols > 4096 else 256 // (32 if cols <= 512 else 64 if cols <= 1024 else 128 if cols <= 2048 else 256)
            most = 8 * 16 * team_rows
            for rows in {1, 2, 2 * sms, 2 * sms + 1, 4 * sms + 1, 8 * sms + 1, most - 1, most, most + 1, 5000}:
                both = [_blocks(rows, cols, dtype, aligned, sms) for aligned in (0, 1)]
                if cols <= 8192 and rows <= most:
                    assert both == [0, 0], (rows, cols, dtype, both)
                else:
                    assert min(both) >= 1, (rows, cols, dtype, both)


def test_scratch_holds_what_either_alignment_writes():
    from parallelkernelbench_b200 import _native as nv

    for dtype in (0, 1):
        for cols in (33, 1001, 1032, 4096, 8192, 9001, 16384, 20001):
            for rows in (1, 100, 257, 600, 1300, 2400, 9001):
                told = nv.cuda_lib().pkb_layer_norm_bwd_partials(LL(rows), cols, dtype)
                assert told == max(_blocks(rows, cols, dtype, aligned, 0) for aligned in (0, 1)) <= 4 * 160
    assert _blocks(0, 8, 0, 1, 0) == _blocks(8, 0, 0, 1, 0) == 0


def test_launches_of_the_backward():
    """One launch of a cluster, two with the weights' sums, three where a row goes in passes."""
    from parallelkernelbench_b200 import _native as nv

    def launches(rows, cols, dtype, aligned):
        return nv.cuda_lib().pkb_layer_norm_bwd_launches(LL(rows), cols, dtype, aligned, 148)

    assert launches(4, 4096, 0, 1) == launches(4, 4097, 1, 0) == 1
    assert launches(4000, 64, 0, 1) == launches(8192, 4096, 0, 1) == launches(8192, 4097, 1, 0) == launches(400, 16384, 0, 1) == 2
    assert launches(3, 8193, 0, 0) == launches(400, 16384, 0, 0) == launches(400, 16384, 1, 1) == launches(4, 20000, 0, 1) == 3
    assert launches(0, 8, 0, 1) == launches(8, 0, 0, 1) == 0


@pytest.mark.parametrize("batch,rows,cols", [(65535, 1, 65537), (65535, 65537, 1), (64, 1 << 17, 1 << 17)])
def test_too_many_tiles_are_refused_before_anything_changes(batch, rows, cols):
    """The refusal comes before the first launch, which updates the momentum: here, where no launch can succeed, it is still the answer."""
    from parallelkernelbench_b200 import _native as nv

    p = ctypes.c_void_p(4096)
    coeff = (ctypes.c_float * 3)(1.5, -0.5, 0.0)
    f, d = ctypes.c_float, ctypes.c_double
    lib = nv.cuda_lib()
    rc = lib.pkb_newton_schulz(p, 0, p, f(0.9), 1, LL(batch), rows, cols, coeff, 1, d(1e-7), None, p, f(1), f(1), None, p, None)
    assert rc != 0 and b"too many tiles" in lib.pkb_last_error(), lib.pkb_last_error()


def test_coefficients_that_shrink_the_iterate_are_refused():
    """Two steps of (0, 1, 1) on 1101 x 1413 of noise leave singular values of 1e-5 and less: as fp16 entries they are zero, and so was the result."""
    import torch

    from parallelkernelbench_b200.ops import muon_step, newton_schulz

    g = torch.zeros(4, 6)
    for bad, steps in (((0.0, 1.0, 1.0), 1), ((0.0, 1.0, 1.0), 2), ((0.01, 1.0, 0.0), 1), ((0.2, 1.0, 0.0), 3), (((1.5, -0.5, 0.0), (0.0, 1.0, 0.0), (2.0, 0.0, 0.0)), 3)):
        with pytest.raises(ValueError, match="shrink"):
            newton_schulz(g, coefficients=bad, steps=steps)
        with pytest.raises(ValueError, match="shrink"):
            muon_step(g, g.clone(), g.clone(), lr=0.1, coefficients=bad, steps=steps)
    # what comes through ends at the next check, as a tensor on the CPU
    for good, steps in (((3.4445, -4.7750, 2.0315), 5), ((1.5, -0.5, 0.0), 16), ((2.0, -1.5, 0.5), 8), ((0.5, 0.5, 0.0), 6), (((-1.5, 0.5, 0.0), (2.0, -1.0, 0.0)), 2)):
        with pytest.raises(ValueError, match="CUDA"):
            newton_schulz(g, coefficients=good, steps=steps)


def test_tensors_of_a_step_do_not_overlap():
    """Weight, momentum, gradient and copy are written or read while others are written: not only the same tensor but any shared byte is refused."""
    import torch

    from parallelkernelbench_b200.ops import muon_step

    buf = torch.zeros(200)
    at = lambda i, n=24: buf[i:i + n].view(4, 6)  # noqa: E731
    half = torch.zeros(400, dtype=torch.bfloat16)
    g = torch.zeros(4, 6)
    cases = [(at(0), at(23), g, None), (at(0), at(30), at(40), None), (at(10), at(60), at(12, 24), None), (at(10), at(60), buf[50:].as_strided((4, 6), (20, 1)), None),
             (at(0), at(30), g, buf[:12].view(torch.bfloat16).view(4, 6)), (at(0), at(30), half[:24].view(4, 6), half[20:44].view(4, 6))]
    for p, m, grad, copy in cases:
        with pytest.raises(ValueError, match="different"):
            muon_step(p, m, grad, lr=0.1, p_bf16=copy)
    # side by side they end at the next check, as tensors on the CPU
    for p, m, grad, copy in ((at(0), at(24), at(48), None), (at(48), at(0), buf[72:].as_strided((4, 6), (1, 4)), buf[100:112].view(torch.bfloat16).view(4, 6)),
                             (at(0), at(24), g[:1].expand(4, 6), half[:24].view(4, 6))):
        with pytest.raises(ValueError, match="CUDA"):
            muon_step(p, m, grad, lr=0.1, p_bf16=copy)
