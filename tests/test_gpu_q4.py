"""Products with 4-bit weights against the same product in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def K():
    from burn_lm_b200 import kernels
    return kernels


def weight(m, k, group, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + m + k)
    values = torch.randint(-8, 8, (m, k), device=DEV, generator=g, dtype=torch.int8)
    scales = torch.randint(16, 32, (m, -(-k // group)), device=DEV, generator=g).float() * 2.0 ** -11
    scales *= torch.randint(0, 2, scales.shape, device=DEV, generator=g) * 2 - 1
    return K().pack_q4(values, scales, group), values.double() * scales.double().repeat_interleave(group, dim=1)[:, :k]


def tokens(n, k, seed=0):
    return torch.randn((n, k), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(BF16)


def check(got, x, dense, k, extra=None, gated=False):
    """The products of whole numbers and bfloat16 tokens are exact; up to K of them and the groups' sums are added in 32 bits, the tensor
    cores cutting their sums off: a unit of 2^-23 of the sum of magnitudes each at most, of which a twentieth is ample for the random
    walk of K of them beyond the first few hundred."""
    size = x.double().abs() @ dense.abs().t()
    want = x.double() @ dense.t()
    off = size * 2.0 ** -23 * (16 + k / 20)
    if gated:
        n = want.shape[0]
        w, o = want.view(n, -1, 2, 8), off.view(n, -1, 2, 8)
        gate, up = w[:, :, 0], w[:, :, 1]
        act = gate * torch.sigmoid(gate)
        # silu's slope is at most 1.1; the exponential and the division are good to 2^-20 of the result
        off = (1.1 * o[:, :, 0] * up.abs() + act.abs() * o[:, :, 1] + 2.0 ** -20 * (act * up).abs()).reshape(n, -1)
        want = (act * up).reshape(n, -1)
    if extra is not None:
        want = want + extra.double()
        off = off + 2.0 ** -24 * want.abs()
    half = torch.finfo(got.dtype).eps / 2
    bound = off * (1 + half) + half * want.abs() + 1e-30
    err = (got.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())


SIZES = [(16, 64), (40, 64), (64, 256), (17, 72), (200, 192), (77, 1000), (2048, 2048), (520, 4160), (1000, 8192), (16, 14336), (300, 65), (33, 7)]


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 16, 17, 33, 64, 100, 129, 300])
@pytest.mark.parametrize("m,k", SIZES)
def test_products(m, k, n):
    k_ = K()
    group = k_.Q4_GROUPS[(m + k + n) % 3]
    w, dense = weight(m, k, group)
    x = tokens(n, k, n)
    for dtype in (BF16, F32):
        out = torch.full((n, m), float("nan"), dtype=dtype, device=DEV)
        k_.product_q4(w, x, out=out)
        check(out, x, dense, k)
    stream = torch.randn((n, m), device=DEV)
    y = stream.clone()
    k_.product_q4(w, x, add_into=y)
    check(y, x, dense, k, extra=stream)


@pytest.mark.parametrize("n", [1, 5, 16, 40, 200])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,k", [(16, 64), (48, 128), (4096, 512), (1024, 1000)])
def test_gated(m, k, group, n):
    w, dense = weight(m, k, group)
    x = tokens(n, k, n)
    for dtype in (BF16, F32):
        out = torch.full((n, m // 2), float("nan"), dtype=dtype, device=DEV)
        K().product_q4(w, x, out=out, swiglu=True)
        check(out, x, dense, k, gated=True)


@pytest.mark.parametrize("n", [3, 40, 150])
def test_column_ranges_and_odd_rows(n):
    """x and the results as column ranges of wider tensors, whose other columns stay as they are; rows that begin anywhere."""
    k_ = K()
    m, k = 72, 256
    w, dense = weight(m, k, 64)
    for shift in (0, 8, 3):
        wide = tokens(n, k + 40, n)
        x = wide[:, shift: shift + k]
        out = torch.full((n, m + 30), 9.0, dtype=BF16, device=DEV)
        k_.product_q4(w, x, out=out[:, 7: 7 + m])
        check(out[:, 7: 7 + m], x, dense, k)
        assert (out[:, :7] == 9).all() and (out[:, 7 + m:] == 9).all()
        stream = torch.full((n, m + 30), 9.0, device=DEV)
        k_.product_q4(w, x, add_into=stream[:, 5: 5 + m])
        check(stream[:, 5: 5 + m], x, dense, k, extra=torch.full((n, m), 9.0, device=DEV))
        assert (stream[:, :5] == 9).all() and (stream[:, 5 + m:] == 9).all()


@pytest.mark.parametrize("n", [2, 40, 140])
def test_infinities_stay_in_their_row(n):
    w, dense = weight(64, 192, 64)
    x = tokens(n, 192, 1)
    x[1, 5] = float("inf")
    out = torch.empty((n, 64), dtype=BF16, device=DEV)
    K().product_q4(w, x, out=out)
    rest = [i for i in range(n) if i != 1]
    assert not torch.isfinite(out[1]).all() and torch.isfinite(out[rest]).all()
    check(out[rest], x[rest], dense, 192)


@pytest.mark.parametrize("n", [1, 16, 200])
def test_captured_and_on_another_stream(n):
    k_ = K()
    w, dense = weight(256, 512, 128)
    x, out = tokens(n, 512), torch.empty((n, 256), dtype=F32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k_.product_q4(w, x, out=out)
    side.synchronize()
    check(out, x, dense, 512)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        k_.product_q4(w, x, out=out)
    x.copy_(tokens(n, 512, 9))
    out.fill_(float("nan"))
    g.replay()
    check(out, x, dense, 512)
    first = out.clone()
    g.replay()
    assert torch.equal(first, out)          # sums in one fixed order


def test_quantized_on_the_device():
    k_ = K()
    w = torch.randn((520, 1000), device=DEV).to(BF16)
    here, there = k_.quantize_q4(w, 64), k_.quantize_q4(w.cpu(), 64)
    assert torch.equal(here.packed.cpu(), there.packed)
    assert torch.equal(k_.q4_values(here).cpu(), k_.q4_values(there))
    x = tokens(5, 1000)
    out = torch.empty((5, 520), dtype=F32, device=DEV)
    k_.product_q4(here, x, out=out)
    check(out, x, k_.q4_values(here).double(), 1000)


@pytest.mark.parametrize("n,over", [(40, 5), (100, 1), (200, 3), (300, 70)])
def test_a_grid_with_a_few_blocks_over(n, over):
    """Some blocks more than the SMs hold at once, whose last run as a launch of their own: alone, before a product that reads the result,
    and captured with it; each end."""
    k_ = K()
    blocks = torch.cuda.get_device_properties(0).multi_processor_count * (2 if n <= 128 else 1)
    m, k = -(-(blocks + over) // -(-n // 256)) * 128 - 24, 520
    w, dense = weight(m, k, 64)
    after, after_dense = weight(64, 512, 32)
    x = tokens(n, k, n)
    out, last = torch.empty((n, m), dtype=BF16, device=DEV), torch.empty((n, 64), dtype=F32, device=DEV)
    def both():
        k_.product_q4(w, x, out=out)
        k_.product_q4(after, out[:, m - 512:], out=last)
    for run in range(3):
        if run == 1:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                both()
        x.copy_(tokens(n, k, n + run))
        out.fill_(float("nan"))
        both() if run == 0 else g.replay()
        check(out, x, dense, k)
        check(last, out[:, m - 512:], after_dense, 512)
    stream = torch.randn((n, m), device=DEV)
    y = stream.clone()
    k_.product_q4(w, x, add_into=y)
    check(y, x, dense, k, extra=stream)
    gated = torch.empty((n, (m - m % 16) // 2), dtype=BF16, device=DEV)
    rows = w.first_rows(m - m % 16)
    k_.product_q4(rows, x, out=gated, swiglu=True)
    check(gated, x, dense[: m - m % 16], k, gated=True)
    k_.check_status(torch.device("cuda:0"))
