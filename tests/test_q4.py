"""Weights in 4 bits on the CPU: rounding, packing, what is refused."""
import pytest
import torch

from burn_lm_b200 import kernels as K


def rows(m, k, seed=0):
    return torch.randn((m, k), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


@pytest.mark.parametrize("group", K.Q4_GROUPS)
@pytest.mark.parametrize("m,k", [(1, 1), (16, 64), (17, 65), (40, 320), (5, 1000), (4200, 64)])
def test_packed_and_read_back(m, k, group):
    g = torch.Generator().manual_seed(m + k)
    values = torch.randint(-8, 8, (m, k), generator=g, dtype=torch.int8)
    scales = torch.randint(16, 32, (m, -(-k // group)), generator=g).float() * 2.0 ** -9
    scales[0, 0] = 0
    w = K.pack_q4(values, scales, group)
    got = K.q4_values(w)
    want = values.double() * scales.double().repeat_interleave(group, dim=1)[:, :k]
    assert got.dtype == torch.bfloat16 and torch.equal(got.double(), want)      # a scale times a whole number is a bfloat16 number


@pytest.mark.parametrize("group", K.Q4_GROUPS)
def test_rounding(group):
    """Every number is the nearest of its group's sixteen; the largest one is -8 steps, up to the scale's own rounding."""
    w = rows(50, 1000, 3)
    got = K.q4_values(K.quantize_q4(w, group)).double()
    for g in range(-(-1000 // group)):
        x, y = w[:, g * group: (g + 1) * group].double(), got[:, g * group: (g + 1) * group]
        top = x.gather(1, x.abs().argmax(dim=1, keepdim=True))
        step = K._five_bits((top / -8).float()).double()
        assert ((step - top / -8).abs() <= 2.0 ** -5 * (top / 8).abs()).all()
        want = torch.round(x / step).clamp(-8, 7) * step
        # (the negative of two that are equally large is the largest)
        tie = (x.amax(dim=1) == -x.amin(dim=1))
        assert torch.equal(y[~tie], want[~tie])


def test_special_groups():
    w = torch.zeros(2, 128)
    w[0, 0], w[0, 1] = 4.0, -4.0
    w[1, 64] = 1e-37
    got = K.q4_values(K.quantize_q4(w, 64))
    assert got[0, 1] == -4.0 and got[0, 0] == 3.5 and (got[1] == 0).all() and (got[0, 2:] == 0).all()
    for bad in (float("nan"), float("inf")):
        w[0, 5] = bad
        with pytest.raises(K.KernelError, match="infinity or a NaN"):
            K.quantize_q4(w, 64)


def test_five_bits():
    x = torch.tensor([1.0, 1.0625, 1.03125, 1.09375, 31.0, 33.0, 35.0, -0.3, 0.0])
    assert torch.equal(K._five_bits(x)[:7], torch.tensor([1.0, 1.0625, 1.0, 1.125, 31.0, 32.0, 36.0])) and K._five_bits(x)[8] == 0
    assert (K._five_bits(x)[7] + 0.3).abs() <= 0.3 * 2.0 ** -5


def test_refusals():
    v, s = torch.zeros(16, 64, dtype=torch.int8), torch.ones(16, 1)
    for bad in (dict(values=v + 8), dict(values=v - 9), dict(values=v.float()), dict(scales=torch.ones(16, 2)), dict(scales=s * 1.03), dict(group=16),
                dict(scales=s * float("inf"))):
        a = dict(values=v, scales=s, group=64)
        a.update(bad)
        with pytest.raises(K.KernelError, match="pack_q4"):
            K.pack_q4(**a)
    for bad in (dict(w=rows(4, 64).to(torch.float16)), dict(w=rows(4, 64)[0]), dict(w=rows(4, 64), group=63)):
        with pytest.raises(K.KernelError, match="quantize_q4"):
            K.quantize_q4(**bad)
    w, x = K.pack_q4(v, s, 64), rows(3, 64)
    good = torch.zeros(3, 16, dtype=torch.bfloat16)
    for bad in (dict(x=x.float(), out=good), dict(x=rows(3, 72), out=good), dict(x=rows(64, 3).t(), out=good), dict(x=x), dict(x=x, out=good.half()),
                dict(x=x, out=good[:2]), dict(x=x, out=good, swiglu=True), dict(x=x, add_into=good), dict(x=x, out=good, add_into=good.float()),
                dict(x=x, out=torch.zeros(16, 3, dtype=torch.bfloat16).t())):
        with pytest.raises(K.KernelError, match="product_q4"):
            K.product_q4(w, **bad)
    with pytest.raises(K.KernelError, match="product_q4"):
        K.product_q4(K.pack_q4(torch.zeros(24, 64, dtype=torch.int8), torch.ones(24, 1), 64), x, out=torch.zeros(3, 12, dtype=torch.bfloat16), swiglu=True)
    with pytest.raises(K.KernelError, match="CUDA device"):
        K.product_q4(w, x, out=good)
