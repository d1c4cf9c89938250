"""Attention over a cache line in 8 bits where its numbers are far from 1, or none."""
import numpy as np
import pytest
import torch

from test_gpu_q8 import BF16, F32, Batch, K

pytestmark = pytest.mark.gpu


def sized(b, n, size):
    """Rows of a step whose values are about `size`."""
    x = b.rows(n).view(n, -1, b.dim)
    x[:, b.heads + b.n_kv:] *= size
    return x.view(n, -1)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("pages,own", [(1e-20, 1e-20), (1e-8, 1e-8), (1e8, 1e8), (1e20, 1e20), (1e30, 1e30), (1.0, 1e-8), (1e-8, 1.0), (0.0, 1.0), (1.0, 0.0)])
def test_single_tokens_with_values_of_any_size(pages, own, dim):
    """The rows of the own block and the pages weigh what they are worth, whatever the size of either's values."""
    b = Batch(3, 16, 2, dim, BF16, 768, seed=dim)
    b.append([(0, 576), (1, 300), (2, 64)], qkv=sized(b, 940, pages), check=False)
    b.append([(0, 20), (1, 2), (2, 40)], qkv=sized(b, 62, own), check=False)
    for _ in range(2):
        step, out, old = b.append([(0, 1), (1, 1), (2, 1)], qkv=sized(b, 3, own), check=False)
        b.attend([(0, 1), (1, 1), (2, 1)], step, out, old)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("times", [1.0, 2.5, 12.0])
@pytest.mark.parametrize("single", [True, False])
def test_a_tall_key_without_a_value(dim, times, single):
    """A key of the own block far above all others, whose value is zero: what is left is the others', however small."""
    heads, n_kv = 8, 2
    b = Batch(1, heads, n_kv, dim, BF16, 700, seed=3)
    b.append([(0, 576)], rot=0, check=False)
    query = b.rows(1)
    tall = b.rows(5)
    rows = tall.view(5, -1, dim)
    rows[1, heads: heads + n_kv] = times * query.view(1, -1, dim)[0, [0, heads // n_kv]]
    rows[1, heads + n_kv:] = 0
    rows[1:, :heads] = query.view(1, -1, dim)[0, [0] * (heads // n_kv) + [heads // n_kv] * (heads // n_kv)]
    b.append([(0, 5)], qkv=tall, rot=0, check=False)
    qkv = query if single else torch.cat([query, b.rows(2)])
    qkv.view(len(qkv), -1, dim)[0, :heads] = rows[1, :heads]
    step, out, old = b.append([(0, len(qkv))], qkv=qkv, rot=0, check=False)
    b.attend([(0, len(qkv))], step, out, old)


@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_a_cached_key_that_is_none(dim, bad):
    """A complete block with an infinite key reads as no number to every head of its kv head, and the other kv head is untouched."""
    outs = []
    for with_it in (False, True):
        b = Batch(8, 32, 2, dim, BF16, 400, seed=1)
        rows = b.rows(8 * 330)
        if with_it:
            rows.view(8, 330, -1, dim)[:, 100, 32, 3] = bad
        b.append([(s, 330) for s in range(8)], qkv=rows, rot=0, check=False)
        step, out, old = b.append([(s, 1) for s in range(8)], rot=0, check=False)
        outs.append(b.attend([(s, 1) for s in range(8)], step, out, old, check=False).view(8, 2, 16, dim))
    assert torch.isnan(outs[1][:, 0]).all() and torch.equal(outs[1][:, 1], outs[0][:, 1])


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 64, BF16), (6, 1, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32)])
@pytest.mark.parametrize("size", [1e-20, 1e-12, 1e-8, 1e8, 1e20, 1e25])
def test_portions_with_values_of_any_size(heads, n_kv, dim, dtype, size):
    """Whole prompts, and portions whose walk several blocks share."""
    b = Batch(2, heads, n_kv, dim, dtype, 1500, seed=dim)
    for entries in ([(0, 300), (1, 70)], [(0, 1000)], [(0, 40), (1, 5)]):
        step, out, old = b.append(entries, qkv=sized(b, sum(n for _, n in entries), size), check=False)
        b.attend(entries, step, out, old)
    K().check_status(torch.device("cuda:0"))


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 64, BF16), (8, 2, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32)])
@pytest.mark.parametrize("pages,own", [(1e-12, 1.0), (1.0, 1e-12), (1e12, 1.0), (1.0, 1e12), (0.0, 1.0), (1.0, 0.0)])
def test_portions_with_pages_of_unlike_sizes(heads, n_kv, dim, dtype, pages, own):
    """Pages and own block, and pages beside one another, whose values are of very different sizes."""
    b = Batch(1, heads, n_kv, dim, dtype, 1500, seed=dim)
    b.append([(0, 448)], qkv=sized(b, 448, pages), check=False)
    b.append([(0, 448)], qkv=sized(b, 448, own), check=False)
    step, out, old = b.append([(0, 90)], qkv=sized(b, 90, own), check=False)
    b.attend([(0, 90)], step, out, old)


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 1, 64, BF16), (8, 1, 128, BF16), (8, 1, 80, BF16), (8, 1, 64, F32), (6, 1, 128, F32)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_an_infinite_key_of_the_own_block(heads, n_kv, dim, dtype, bad):
    """Rows that see an infinite key: no numbers where its score is plus infinity, the others' result where it is minus infinity.
    The block with it, once it is in 8 bits, reads as none of them numbers."""
    b = Batch(1, heads, n_kv, dim, dtype, 256, seed=6)
    qkv = b.rows(130)
    qkv.view(130, -1, dim)[100, heads, 5] = bad
    step, out, old = b.append([(0, 130)], qkv=qkv, rot=0, check=False)
    got = b.attend([(0, 130)], step, out, old, check=False).view(130, heads, dim).double().cpu().numpy()
    q = out.view(130, -1, dim)[:, :heads].double().cpu().numpy()
    rows = b.line.rows[0].copy()
    b.line.rows[0] = rows[:128]
    with np.errstate(invalid="ignore"):
        want, weight, _ = b.line.attend(0, q[:128], 0, b.scale)
    finite = rows[:128].copy()
    finite[100, 0, 0, 5] = 0
    b.line.rows[0] = finite
    _, _, reach = b.line.attend(0, q[:128], 0, b.scale)
    # as for finite numbers: rounded scores and sums, in bfloat16 a rounded probability and result
    relative = (dim + 8) * 2.0 ** -24 * 2 * reach + 2.0 ** -21 + 80 * 2.0 ** -24
    half = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    seen_up = np.sign(bad) * q[100:128, :, 5] > 0
    assert np.isnan(want[100:][seen_up]).all() and np.isfinite(want[100:][~seen_up]).all() and seen_up.any() and not seen_up.all()
    assert np.isnan(got[100:128][seen_up]).all()
    there = np.isfinite(want)
    bound = np.broadcast_to(weight * (2 * relative + (half if dtype == BF16 else 0.0)) + half * np.abs(want) + 1e-30, want.shape)
    assert (np.abs(got[:128][there] - want[there]) <= bound[there]).all()
    assert np.isnan(got[128:]).all()


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 64, BF16), (6, 1, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32)])
@pytest.mark.parametrize("keys", [1e-17, 1e-8, 1e8, 1e17])
def test_keys_of_any_size(heads, n_kv, dim, dtype, keys):
    """Keys far from 1 against queries as far on the other side: prompts, portions and single tokens."""
    def rows(b, n):
        x = b.rows(n).view(n, -1, dim)
        x[:, :heads] /= keys
        x[:, heads: heads + n_kv] *= keys
        return x.view(n, -1)
    b = Batch(2, heads, n_kv, dim, dtype, 1000, seed=dim)
    for entries in ([(0, 700), (1, 70)], [(0, 40), (1, 5)], [(0, 1), (1, 1)]):
        step, out, old = b.append(entries, qkv=rows(b, sum(n for _, n in entries)), check=False)
        b.attend(entries, step, out, old)


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 64, BF16), (8, 2, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32)])
@pytest.mark.parametrize("window", [0, 100])
def test_scores_times_zero(heads, n_kv, dim, dtype, window):
    """The mean of the values that a query sees."""
    b = Batch(2, heads, n_kv, dim, dtype, 600, seed=dim)
    b.scale = 0.0
    for entries in ([(0, 300), (1, 70)], [(0, 40), (1, 5)], [(0, 1), (1, 1)]):
        b.go(entries, window=window)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("every", [2, 3, 4, 5])
def test_pages_that_are_none_between_others(dim, every):
    """Every second to fifth page of a long walk outside the pool: each place of the ring holds a page, none, and a page again."""
    from q8_reference import PAGE, Line
    b = Batch(1, 8, 2, dim, BF16, 2200, seed=every)
    b.append([(0, 2048)], rot=0, check=False)
    b.table[0, :32:every] = -1
    kept = [i for i in range(2048) if i // PAGE % every]
    line = Line(1, 2, dim)
    line.append(0, b.line.rows[0][kept])
    b.line = line
    for new in (70, 1):
        step, out, old = b.append([(0, new)], rot=0, check=False)
        o = b.attend([(0, new)], step, out, old, check=False)
        step.start_pos = step.start_pos.cpu() - (2048 - len(kept))
        b.check_attention([(0, new)], step, out, o, 0)
    K().check_status(torch.device("cuda:0"))


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 64, BF16), (8, 2, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("size", [1.0, 1e-12])
@pytest.mark.parametrize("where", [0, 20, 33])
def test_a_value_that_is_none_beside_single_tokens(heads, n_kv, dim, dtype, bad, size, where):
    """One lane of one value of the own block, in the tail or the token's own: that lane shows it, the others are what they are without it."""
    b = Batch(1, heads, n_kv, dim, dtype, 500, seed=dim)
    b.append([(0, 384)], qkv=sized(b, 384, size), rot=0, check=False)
    own, last = sized(b, 33, size), sized(b, 1, size)
    rows = own.view(33, -1, dim)[where] if where < 33 else last.view(-1, dim)
    rows[heads + n_kv, 5] = bad
    b.append([(0, 33)], qkv=own, rot=0, check=False)
    step, out, old = b.append([(0, 1)], qkv=last, rot=0, check=False)
    o = b.attend([(0, 1)], step, out, old, check=False).view(heads, dim)
    mine = o[: heads // n_kv, 5].clone()
    assert torch.isnan(mine).all() if bad != bad else (mine == bad).all()
    # without it: its lane taken out on both sides
    b.line.rows[0][384 + where, 1, 0, 5] = 0
    for h in range(heads // n_kv):
        o[h, 5] = 0
    b.line.rows[0][:, 1, 0, 5] = 0
    b.check_attention([(0, 1)], step, out, o.view(1, -1), 0)



@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 64, BF16), (8, 2, 128, BF16), (4, 2, 80, BF16), (4, 2, 64, F32), (4, 2, 128, F32)])
@pytest.mark.parametrize("cuts", [(130,), (90, 40), (100, 1, 1, 28)])
def test_a_key_that_is_none_in_the_own_block(heads, n_kv, dim, dtype, cuts):
    """A NaN among a key's lanes: every later query of its heads has no result, the others and those before are untouched by it."""
    outs = []
    for with_it in (False, True):
        b = Batch(1, heads, n_kv, dim, dtype, 256, seed=6)
        qkv, parts, at = b.rows(130), [], 0
        if with_it:
            qkv.view(130, -1, dim)[95, heads, 3] = float("nan")
        for n in cuts:
            step, out, old = b.append([(0, n)], qkv=qkv[at: at + n].clone(), rot=0, check=False)
            parts.append(b.attend([(0, n)], step, out, old, check=False))
            at += n
        outs.append(torch.cat(parts).view(130, n_kv, heads // n_kv, dim))
    assert torch.isnan(outs[1][95:, 0]).all()
    assert torch.equal(outs[1][:95], outs[0][:95]) and torch.equal(outs[1][:, 1], outs[0][:, 1])
