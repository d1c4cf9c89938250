"""Products with 4-bit weights: tokens that are no numbers, scales at the ends of their range, long rows."""
import pytest
import torch

from test_gpu_q4 import BF16, DEV, F32, K, check, tokens, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 8, 9, 40])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k", [(64, 192), (200, 72), (48, 4160)])
def test_tokens_that_are_no_numbers(m, k, group, n):
    """An infinite place gives every row the infinity of its weight's sign there, or no number where the weight is zero or infinities of both
    signs meet, whatever the number of tokens; the other tokens' results are untouched."""
    w, dense = weight(m, k, group)
    x = tokens(n, k, 1)
    inf = float("inf")
    x[0, 5] = inf
    if n > 1:
        x[1, k - 1], x[1, 33] = -inf, -inf
    if n > 2:
        x[3, 64], x[4, k // 2], x[4, k // 2 + 1], x[6, 0] = -inf, inf, inf, float("nan")
    want = torch.stack([(row * dense).sum(dim=1) for row in x.double()])
    for dtype in (BF16, F32):
        out = torch.full((n, m), 3.0, dtype=dtype, device=DEV)
        K().product_q4(w, x, out=out)
        odd = ~torch.isfinite(x).all(dim=1)
        assert torch.equal(out[odd].double().nan_to_num(nan=7.0), want[odd].nan_to_num(nan=7.0))
        check(out[~odd], x[~odd], dense, k)
    if m % 16 == 0:
        gated = torch.full((n, m // 2), 3.0, dtype=F32, device=DEV)
        K().product_q4(w, x, out=gated, swiglu=True)
        both = want.view(n, -1, 2, 8)
        act = (both[:, :, 0] / (1 + torch.exp(-both[:, :, 0])) * both[:, :, 1]).reshape(n, -1)
        assert torch.equal(gated[odd].double().nan_to_num(nan=7.0), act[odd].nan_to_num(nan=7.0))


@pytest.mark.parametrize("n", [1, 8, 9, 40])
@pytest.mark.parametrize("exponent", [-110, 80])
def test_scales_at_the_ends_of_their_range(exponent, n):
    k_ = K()
    m, k, group = 48, 512, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    values = torch.randint(-8, 8, (m, k), device=DEV, generator=g, dtype=torch.int8)
    scales = torch.full((m, k // group), 2.0 ** exponent, device=DEV)
    scales[::3] *= -1
    w = k_.pack_q4(values, scales, group)
    dense = values.double() * scales.double().repeat_interleave(group, dim=1)
    assert torch.equal(k_.q4_values(w).double(), dense)
    x = (tokens(n, k, 2).float() * (2.0 ** -20 if exponent > 0 else 2.0 ** 20)).to(BF16)
    out = torch.empty((n, m), dtype=F32, device=DEV)
    k_.product_q4(w, x, out=out)
    # (a scale that is a power of two changes exponents only)
    check(out.double().mul(2.0 ** -exponent).float(), x, dense * 2.0 ** -exponent, k)


@pytest.mark.parametrize("n", [1, 3, 8, 9])
@pytest.mark.parametrize("m,k", [(40, 14336), (40, 14400), (200, 16384), (64, 16392), (40, 20000)])
def test_long_rows(m, k, n):
    """Rows of K cut over clusters of seven and eight blocks, and longer ones, which the other kernel takes."""
    k_ = K()
    w, dense = weight(m, k, 64)
    x = tokens(n, k, n)
    out = torch.full((n, m), float("nan"), dtype=F32, device=DEV)
    k_.product_q4(w, x, out=out)
    check(out, x, dense, k)
    if m % 16 == 0:
        gated = torch.full((n, m // 2), float("nan"), dtype=BF16, device=DEV)
        k_.product_q4(w, x, out=gated, swiglu=True)
        check(gated, x, dense, k, gated=True)
    k_.check_status(torch.device("cuda:0"))


@pytest.mark.parametrize("n", [2, 8, 9, 40, 300])
def test_the_same_row_many_times(n):
    """A broadcast token, and rows that overlap: read as what they are."""
    k_ = K()
    m, k = 48, 512
    w, dense = weight(m, k, 64)
    x = tokens(1, k, 3).expand(n, k)
    out = torch.full((n, m), float("nan"), dtype=F32, device=DEV)
    k_.product_q4(w, x, out=out)
    check(out, x, dense, k)
    assert (out == out[0]).all()
    x = tokens(1, k + 8 * n, 4)[0].as_strided((n, k), (8, 1))
    k_.product_q4(w, x, out=out)
    check(out, x, dense, k)
