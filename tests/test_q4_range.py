"""The range of a 4-bit weight's scales and what a product refuses, without a GPU."""
import pytest
import torch

from burn_lm_b200 import kernels as K


def test_scales_outside_the_range_are_refused():
    v = torch.randint(-8, 8, (16, 64), generator=torch.Generator().manual_seed(1), dtype=torch.int8)
    for s in (2.0 ** -110, 2.0 ** 80, -2.0 ** 80, 0.0, -1.5 * 2.0 ** -110):
        w = K.pack_q4(v, torch.full((16, 1), s), 64)
        assert torch.equal(K.q4_values(w).double(), v.double() * s)
    for s in (2.0 ** -111, -2.0 ** -130, 1.0625 * 2.0 ** 80, -2.0 ** 100, 2.0 ** -149):
        with pytest.raises(K.KernelError, match="pack_q4: scales are"):
            K.pack_q4(v, torch.full((16, 1), s), 64)


def test_weights_too_large_or_small():
    w = torch.zeros(16, 64)
    w[3, 5], w[4, 6] = 2.0 ** 83, -2.0 ** -107
    got = K.q4_values(K.quantize_q4(w, 64)).double()
    assert torch.equal(got, w.double().where(w != 0, torch.zeros(())))
    w[4, 6] = -2.0 ** -109
    assert (K.q4_values(K.quantize_q4(w, 64))[4] == 0).all()
    for big in (2.0 ** 84, -2.0 ** 84, 3.3e38):
        w[3, 5] = big
        with pytest.raises(K.KernelError, match="beyond 2.83"):
            K.quantize_q4(w, 64)


def test_results_whose_rows_overlap_are_refused():
    w = K.pack_q4(torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 1), 64)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    for out in (torch.zeros(1, 16).expand(3, 16), torch.zeros(64).as_strided((3, 16), (8, 1))):
        for end in (dict(out=out), dict(add_into=out)):
            with pytest.raises(K.KernelError, match="rows of the result overlap"):
                K.product_q4(w, x, **end)
    with pytest.raises(K.KernelError, match="CUDA device"):      # (a single row overlaps nothing)
        K.product_q4(w, x[:1], out=torch.zeros(64).as_strided((1, 16), (8, 1)))
