"""A cache line in 8 bits: the append with its rotation, and attention over it, against plain numpy in 64 bits."""
import numpy as np
import pytest
import torch

from q8_reference import PAGE, Line, in_eight, rotate

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def K():
    from burn_lm_b200 import kernels
    return kernels


def make_step(lengths, starts, slots, padding=0, max_q_len=None):
    from burn_lm_b200.engine.engine import Workspace
    from burn_lm_b200.parts.base import StepContext
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return StepContext(
        n_tokens=cu[-1] + padding, n_seqs=len(lengths), max_q_len=max_q_len or max(lengths), max_kv_len=max(s + n for s, n in zip(starts, lengths)),
        tokens=i32([0] * (cu[-1] + padding)), token_seq=i32([s for s, n in enumerate(lengths) for _ in range(n)] + [-1] * padding),
        token_pos=i32([s + t for s, n in zip(starts, lengths) for t in range(n)] + [0] * padding), cu_seqlens=i32(cu), slot_of_seq=i32(slots),
        start_pos=i32(starts), want_rows=None, n_want=0, workspace=Workspace(torch.device(DEV)))


class Batch:
    """Sequences on the device with a reference beside them.  Unused memory is filled with NaN (tails) and scales of NaN (pages)."""

    def __init__(self, n_slots, heads, n_kv, dim, dtype, room, seed=0, scale=None):
        k = K()
        self.heads, self.n_kv, self.dim, self.dtype = heads, n_kv, dim, dtype
        each = -(-room // PAGE)
        self.pool, self.scales = k.q8_pool(n_slots * each + 3, n_kv, dim, DEV)
        self.pool.fill_(-77)
        self.scales.fill_(float("nan"))
        order = torch.randperm(n_slots * each + 3, generator=torch.Generator().manual_seed(seed))[: n_slots * each]
        self.table = order.to(torch.int32).view(n_slots, each).to(DEV)
        self.tail = torch.full((n_slots, 2, n_kv, PAGE, dim), float("nan"), dtype=dtype, device=DEV)
        self.line = Line(n_slots, n_kv, dim)
        self.length = [0] * n_slots
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.scale = scale or dim ** -0.5
        self.freq = lambda rot: torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=DEV)

    def rows(self, n):
        x = torch.randn((n, self.heads + 2 * self.n_kv, self.dim), device=DEV, generator=self.g)
        x[:, self.heads: self.heads + self.n_kv, :: max(1, self.dim // 4)] *= 4.0        # a few lanes of the keys are larger
        return x.to(self.dtype).view(n, -1)

    def append(self, entries, qkv=None, rot=None, pairs=0, padding=0, table=None, turn_scale=1.0, in_place=False, max_q_len=None, check=True):
        """entries: [(slot, new tokens)].  Runs the append, checks everything it wrote, and brings the reference up to date."""
        k = K()
        lengths, slots = [n for _, n in entries], [s for s, _ in entries]
        starts = [self.length[s] for s in slots]
        rot = self.dim if rot is None else rot
        step = make_step(lengths, starts, slots, padding, max_q_len)
        n = sum(lengths)
        qkv = self.rows(n + padding) if qkv is None else qkv
        given = qkv.clone()
        out = qkv if in_place else torch.full_like(qkv, 7.0)
        tail = self.tail.clone()
        freq = self.freq(rot) if rot else None
        old = k.rope_append_q8(qkv, out, step, self.pool, self.scales, self.tail, self.table, freq, rot, pairs, self.heads, self.n_kv, self.dim,
                               table=table, turn_scale=turn_scale)
        rows = out.view(n + padding, -1, self.dim)
        stored = rows[:n, self.heads:].float().cpu().numpy().reshape(n, 2, self.n_kv, self.dim)
        at = 0
        for (slot, new), start in zip(entries, starts):
            self.line.append(slot, stored[at: at + new])
            self.length[slot] += new
            at += new
        if check:
            assert torch.equal(rows[n:], (given if in_place else torch.full_like(given, 7.0)).view(n + padding, -1, self.dim)[n:])
            want = given.view(n + padding, -1, self.dim)[:n].double().cpu().numpy()
            pos = np.concatenate([np.arange(s, s + m) for s, m in zip(starts, lengths)]).astype(np.float64)
            turned = rotate(want[:, : self.heads + self.n_kv], pos, freq.cpu().numpy() if rot else None, rot, pairs, turn_scale)
            # cosine and sine are rounded to 32 bits and times turn_scale, two products and their sum rounded: five roundings of
            # 2^-24 each of at most |x| + |y|; then one to the type
            size = np.abs(want[:, : self.heads + self.n_kv]).max(axis=2, keepdims=True) * 2 * abs(turn_scale)
            half = torch.finfo(self.dtype).eps / 2
            got = rows[:n, : self.heads + self.n_kv].double().cpu().numpy()
            assert (np.abs(got - turned) <= 5 * 2.0 ** -24 * size + half * (np.abs(turned) + 2.0 ** -20 * size)).all()
            assert torch.equal(rows[:n, self.heads + self.n_kv:], given.view(n + padding, -1, self.dim)[:n, self.heads + self.n_kv:])
            self.check_line(entries, starts, tail, old)
        return step, out, old

    def check_line(self, entries, starts, tail, old):
        k = K()
        new_tail = self.tail.float().cpu().numpy()
        was = tail.float().cpu().numpy()
        touched = set()
        for i, ((slot, new), start) in enumerate(zip(entries, starts)):
            end = start + new
            for b in range(start // PAGE, end // PAGE):
                page = self.table[slot, b: b + 1]
                whole, scales = self.line.block(slot, b)
                assert np.array_equal(self.scales[page.long()][0].cpu().numpy(), scales)
                got = k.q8_values(self.pool, self.scales, page, self.dim, F32)[0].cpu().numpy()
                assert np.array_equal(got, whole * scales.T[:, :, None, None])
                touched.add(int(page))
            first = (start if end // PAGE == start // PAGE else end // PAGE * PAGE) % PAGE
            want = was[slot].copy()
            if end % PAGE:
                rows = self.line.rows[slot][end - end % PAGE + first: end]
                want[:, :, first: end % PAGE] = rows.transpose(1, 2, 0, 3)
            assert np.array_equal(new_tail[slot], want, equal_nan=True)
            if old is not None and start % PAGE:
                found = self.line.rows[slot][start - start % PAGE: start].transpose(1, 2, 0, 3)
                assert np.array_equal(old[i, :, :, : start % PAGE].float().cpu().numpy(), found)
        for slot in range(len(was)):
            if slot not in [s for s, _ in entries]:
                assert np.array_equal(new_tail[slot], was[slot], equal_nan=True)
        # pages that no sequence holds are untouched
        loose = sorted(set(range(self.pool.shape[0])) - set(self.table.flatten().tolist()))
        assert (self.pool[loose][:, :, :-16] == -77).all() and torch.isnan(self.scales[loose]).all()

    def attend(self, entries, step, out, old, window=0, padding=0, check=True):
        n = out.shape[0]
        o = torch.full((n, self.heads * self.dim), 5.0, dtype=self.dtype, device=DEV)
        if old is not None:
            # what the append did not write is nobody's: it must not matter
            for i, s in enumerate(step.start_pos.tolist()):
                old[i, :, :, s % PAGE:] = float("nan")
        K().attention_q8(out, step, self.pool, self.scales, self.tail, old, self.table, o, self.heads, self.n_kv, self.dim, self.scale, window=window)
        if check:
            self.check_attention(entries, step, out, o, window)
        return o

    def check_attention(self, entries, step, out, o, window):
        at = 0
        for (slot, new), start in zip(entries, step.start_pos.tolist()):
            q = out[at: at + new].view(new, -1, self.dim)[:, : self.heads].double().cpu().numpy()
            want, weight, reach = self.line.attend(slot, q, start, self.scale, window)
            got = o[at: at + new].view(new, self.heads, self.dim).double().cpu().numpy()
            assert not np.isnan(got).any()
            # A score is off by (D + 8) roundings of 2^-24 of its |q||k| and by its conversion to base 2; exp2 by 2^-22; sums of up to
            # start + new numbers in 32 bits.  bfloat16: a probability (times a scale) and the result are rounded to 8 bits.
            keys = start + new
            relative = (self.dim + 8) * 2.0 ** -24 * 2 * reach + 2.0 ** -21 + (64 + keys / 8) * 2.0 ** -24
            half = 2.0 ** -8 if self.dtype == BF16 else 2.0 ** -24
            bound = weight * (2 * relative + (half if self.dtype == BF16 else 0.0)) + half * np.abs(want) + 1e-30
            assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
            at += new
        assert (o[at:] == 5.0).all()                     # rows of no sequence are left as they are

    def go(self, entries, window=0, **more):
        step, out, old = self.append(entries, **more)
        return self.attend(entries, step, out, old, window, more.get("padding", 0))


HEADS = [(4, 2, 16), (6, 1, 48), (8, 8, 64), (8, 2, 64), (16, 1, 128), (12, 4, 80), (5, 1, 128), (2, 1, 256)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,n_kv,dim", HEADS)
def test_prompts_and_tokens(heads, n_kv, dim, dtype):
    """Prompts that end inside a block, at its end and after one token, then tokens one by one over a block's end, then a portion."""
    b = Batch(4, heads, n_kv, dim, dtype, 320, seed=heads + dim)
    b.go([(0, 62), (2, 64), (1, 1), (3, 130)])
    for _ in range(3):
        b.go([(1, 1), (0, 1), (3, 1)])
    b.go([(0, 5), (1, 1), (3, 70)])
    b.go([(2, 1), (1, 1)])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_portion_fills_the_block_it_found_and_begins_the_next(dtype):
    """The rows found in the tail are needed after the tail has taken the next block's."""
    b = Batch(2, 8, 2, 64, dtype, 512, seed=3)
    b.go([(0, 40), (1, 63)])
    b.go([(0, 100), (1, 66)])        # 140: two blocks filled, 12 rows of the third; 129: one row
    b.go([(0, 30), (1, 1)])
    b.go([(0, 200), (1, 63)])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rot,pairs", [(64, 1), (64, 2), (0, 0), (32, 0), (32, 2), (20, 0), (20, 1), (2, 0), (6, 1)])
def test_rotations(rot, pairs, dtype):
    b = Batch(2, 4, 2, 64, dtype, 256, seed=rot)
    b.go([(0, 70), (1, 3)], rot=rot, pairs=pairs, turn_scale=1.25)
    for _ in range(2):
        b.go([(0, 1), (1, 1)], rot=rot, pairs=pairs, turn_scale=1.25)


def test_tables_and_places():
    """Angles from a table that ends inside the step, and q|k|v rotated in place."""
    for in_place in (False, True):
        b = Batch(2, 8, 2, 64, BF16, 256, seed=5)
        table = K().rope_table(b.freq(64), 50)
        b.go([(0, 70), (1, 20)], table=table, in_place=in_place)
        b.go([(0, 1), (1, 1)], table=table, in_place=in_place)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [1, 5, 64, 65, 100])
def test_windows(window, dtype):
    b = Batch(2, 8, 2, 64, dtype, 512, seed=window)
    b.go([(0, 150), (1, 64)], window=window)
    for _ in range(2):
        b.go([(0, 1), (1, 1)], window=window)
    b.go([(0, 60), (1, 90)], window=window)


def test_rows_of_no_sequence():
    b = Batch(2, 8, 2, 64, BF16, 256, seed=8)
    b.go([(0, 70), (1, 3)], padding=23)
    b.go([(0, 9), (1, 1)], padding=1)


def test_a_step_bound_longer_than_its_runs():
    """A captured step's longest run is rounded up, and its last sequences are empty."""
    k = K()
    b = Batch(2, 8, 2, 64, BF16, 256, seed=9)
    step, out, old = b.append([(0, 70), (1, 3)], max_q_len=256)
    b.attend([(0, 70), (1, 3)], step, out, old)
    step, out, old = b.append([(0, 1), (1, 1)], max_q_len=128)
    b.attend([(0, 1), (1, 1)], step, out, old)
    step = make_step([1, 1], b.length, [0, 1])
    step.n_seqs = 3
    step.cu_seqlens = torch.tensor([0, 1, 2, 2], dtype=torch.int32, device=DEV)
    step.slot_of_seq = torch.tensor([0, 1, 1], dtype=torch.int32, device=DEV)
    step.start_pos = torch.tensor(b.length + [b.length[1]], dtype=torch.int32, device=DEV)
    qkv = b.rows(2)
    out = torch.empty_like(qkv)
    k.rope_append_q8(qkv, out, step, b.pool, b.scales, b.tail, b.table, b.freq(64), 64, 0, 8, 2, 64)
    b.line.append(0, out[:1].view(1, -1, 64)[:, 8:].float().cpu().numpy().reshape(1, 2, 2, 64))
    b.line.append(1, out[1:].view(1, -1, 64)[:, 8:].float().cpu().numpy().reshape(1, 2, 2, 64))
    o = torch.full((2, 8 * 64), 5.0, dtype=BF16, device=DEV)
    k.attention_q8(out, step, b.pool, b.scales, b.tail, None, b.table, o, 8, 2, 64, 0.125)
    step.start_pos = step.start_pos[:2]
    b.check_attention([(0, 1), (1, 1)], step, out, o, 0)


@pytest.mark.parametrize("value", [0.0, 1e-30, 3e38])
def test_blocks_of_extreme_numbers(value):
    """A block of zeros has scale 0 and reads as zeros; tiny and huge blocks keep their 8 bits."""
    b = Batch(1, 2, 1, 64, F32, 256, seed=1, scale=1e-30)
    qkv = b.rows(130)
    qkv[:, 128:] = value * torch.sign(qkv[:, 128:])
    qkv[:64, 2 * 64 + 64:] *= 0.5
    step, out, old = b.append([(0, 130)], qkv=qkv, rot=0)
    if value < 1:
        b.attend([(0, 130)], step, out, old)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_numbers_that_are_none(bad):
    """A NaN or an infinity spoils its own block of its own head and leaves the others alone."""
    k = K()
    b = Batch(2, 4, 2, 64, BF16, 256, seed=2)
    qkv = b.rows(200)
    qkv.view(200, 8, 64)[70, 4, 3] = bad                 # a key of head 0, block 1 of the first sequence
    step = make_step([130, 70], [0, 0], [0, 1])
    out = torch.empty_like(qkv)
    k.rope_append_q8(qkv, out, step, b.pool, b.scales, b.tail, b.table, None, 0, 0, 4, 2, 64)
    vals = k.q8_values(b.pool, b.scales, b.table[:, :2].reshape(-1).contiguous(), 64)[:3]
    assert not torch.isfinite(vals[1, 0, 0]).any()
    assert torch.isfinite(vals[0]).all() and torch.isfinite(vals[2]).all() and torch.isfinite(vals[1, 1]).all() and torch.isfinite(vals[1, 0, 1]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_cuts_do_not_matter(dtype):
    """The same tokens in one step, in portions and one by one: the same pages and, up to rounding, the same attention."""
    n, heads, n_kv, dim = 150, 8, 2, 64
    rows = None
    results = []
    for cut in ([150], [1] * 150, [40, 100, 10], [64, 64, 22], [2] * 75, [63, 1, 1, 85]):
        b = Batch(1, heads, n_kv, dim, dtype, 256, seed=4)
        rows = b.rows(n) if rows is None else rows
        outs, at = [], 0
        for m in cut:
            step, out, old = b.append([(0, m)], qkv=rows[at: at + m].clone(), check=False)
            outs.append(b.attend([(0, m)], step, out, old, check=False))
            at += m
        pages = K().q8_values(b.pool, b.scales, b.table[0, :2].contiguous(), dim)
        results.append((torch.cat(outs).float(), pages, b.tail[:, :, :, : n % PAGE].clone()))
    for o, pages, tail in results[1:]:
        assert torch.equal(pages, results[0][1]) and torch.equal(tail, results[0][2])
        # two roundings of a probability and of the result each
        torch.testing.assert_close(o, results[0][0], rtol=4 * torch.finfo(dtype).eps, atol=4 * torch.finfo(dtype).eps if dtype == BF16 else 1e-5)


def test_a_token_run_twice_and_one_forgotten():
    """A step of one token a sequence may be run again, with the same token or with another, at a block's end too."""
    for n in (20, 62, 63, 64):
        b = Batch(1, 8, 2, 64, BF16, 256, seed=n)
        b.go([(0, n)])
        at = b.length[0]
        qkv, other = b.rows(1), b.rows(1)
        step = make_step([1], [at], [0])
        out = torch.empty_like(qkv)
        for x in (qkv, other):
            K().rope_append_q8(x, out, step, b.pool, b.scales, b.tail, b.table, b.freq(64), 64, 0, 8, 2, 64)
        step, out, old = b.append([(0, 1)], qkv=qkv, check=False)
        first = b.attend([(0, 1)], step, out, old)
        assert torch.equal(first, b.attend([(0, 1)], step, out, old))
        b.go([(0, 1)])


def test_long_cache():
    """One sequence far beyond the tables, pages in no order, offsets of the pool beyond 2^31 bytes."""
    k = K()
    heads, n_kv, dim = 4, 2, 128
    line = k.q8_line_bytes(dim)
    n_pages = (1 << 31) // (n_kv * line) + 40
    pool, scales = k.q8_pool(n_pages, n_kv, dim, DEV)
    b = Batch(1, heads, n_kv, dim, BF16, 256, seed=11)
    b.pool, b.scales = pool, scales
    b.table = torch.tensor([[n_pages - 1, 5, n_pages - 3, 0]], dtype=torch.int32, device=DEV)
    def values_are_right():
        for i in range(b.length[0] // PAGE):
            whole, s = b.line.block(0, i)
            got = k.q8_values(pool, scales, b.table[0, i: i + 1].contiguous(), dim)[0].cpu().numpy()
            assert np.array_equal(got, whole * s.T[:, :, None, None])
    for n in (190, 1, 1, 1):
        step, out, old = b.append([(0, n)], check=False)
        b.attend([(0, n)], step, out, old)
    values_are_right()


def test_on_another_stream_and_captured():
    """Captured and replayed with other tokens and lengths; two graphs alive at once; on a stream of its own."""
    k = K()
    b = Batch(2, 8, 2, 64, BF16, 512, seed=12)
    b.go([(0, 100), (1, 61)])
    step = make_step([1, 1], b.length, [0, 1])
    step.max_kv_len = 512
    qkv = b.rows(2)
    graphs = []
    for _ in range(2):
        out, o = torch.empty_like(qkv), torch.empty((2, 8 * 64), dtype=BF16, device=DEV)
        def both():
            k.rope_append_q8(qkv, out, step, b.pool, b.scales, b.tail, b.table, freq, 64, 0, 8, 2, 64)
            k.attention_q8(out, step, b.pool, b.scales, b.tail, None, b.table, o, 8, 2, 64, 0.125)
        freq = b.freq(64)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            both()
        graphs.append((g, out, o))
    for i in range(6):
        g, out, o = graphs[i % 2]
        qkv.copy_(b.rows(2))
        step.start_pos.copy_(torch.tensor(b.length, dtype=torch.int32))
        g.replay()
        for s in range(2):
            b.line.append(s, out[s: s + 1].view(1, -1, 64)[:, 8:].float().cpu().numpy().reshape(1, 2, 2, 64))
        o.view(2, 8, 64)
        b.check_attention([(0, 1), (1, 1)], step, out, o, 0)
        b.length = [n + 1 for n in b.length]


def test_written_pages_are_read_back():
    k = K()
    for dim in (16, 48, 64, 80, 128, 256):
        pool, scales = k.q8_pool(5, 3, dim, DEV)
        g = torch.Generator(device=DEV).manual_seed(dim)
        keys, values = (torch.randint(-127, 128, (2, 3, PAGE, dim), device=DEV, generator=g).to(torch.int8) for _ in range(2))
        ks, vs = (torch.rand((2, 3), device=DEV, generator=g) for _ in range(2))
        pages = torch.tensor([4, 1], dtype=torch.int32, device=DEV)
        k.q8_write(pool, scales, pages, keys, ks, values, vs)
        got = k.q8_values(pool, scales, torch.tensor([1, 4, 9, -1], dtype=torch.int32, device=DEV), dim)
        want = torch.stack([keys * ks[:, :, None, None], values * vs[:, :, None, None]], dim=1).float()
        assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[0]) and (got[2:] == 0).all()
        cpu = k.q8_pool(5, 3, dim, "cpu")
        k.q8_write(*cpu, pages.cpu(), keys.cpu(), ks.cpu(), values.cpu(), vs.cpu())
        assert torch.equal(cpu[0], pool.cpu()) and torch.equal(cpu[1], scales.cpu())


def test_the_definition_is_the_reference():
    """The oracle itself: a block of known numbers."""
    whole, scale = in_eight(np.array([[127.0, -63.5], [0.5, 1.5]], np.float32))
    assert scale == 1.0 and np.array_equal(whole, [[127, -64], [0, 2]])


@pytest.mark.parametrize("heads,n_kv,dim", [(32, 8, 64), (8, 8, 64), (24, 8, 128), (16, 2, 64), (12, 1, 64), (9, 1, 128), (32, 2, 128), (7, 1, 64)])
@pytest.mark.parametrize("lengths,window", [((1500,), 0), ((700, 3, 64), 0), ((1, 63, 128, 129, 640), 0), ((1500, 90), 200), ((1300,), 1100), ((70,) * 40, 0)])
def test_single_tokens_of_long_and_short_sequences(heads, n_kv, dim, lengths, window):
    """Sequences of unequal lengths in one step: shares of one sequence, none of another; groups of up to 16 query heads; over a
    block's end."""
    if len(lengths) > 8 and heads > 12:
        heads, n_kv = 8, 4
    b = Batch(len(lengths), heads, n_kv, dim, BF16, max(lengths) + 8, seed=heads + len(lengths))
    b.append([(s, n) for s, n in enumerate(lengths)], check=False)
    for i in range(2):
        step, out, old = b.append([(s, 1) for s in range(len(lengths))], check=False)
        if i == 1:
            step.max_kv_len = 4 * max(lengths)           # a bound, as a captured step has
        b.attend([(s, 1) for s in range(len(lengths))], step, out, old, window)
    K().check_status(torch.device("cuda:0"))


def test_one_key_towers():
    """One key far above hundreds, in each block and at the borders of the warps' shares: single tokens and a portion."""
    heads, n_kv, dim = 8, 2, 64
    for where in (0, 15, 16, 63, 64, 200, 383, 384, 400, 401):
        b = Batch(1, heads, n_kv, dim, BF16, 512, seed=where)
        qkv = b.rows(401)
        rows = qkv.view(401, -1, dim)
        rows[:, heads: heads + n_kv] *= 0.25
        query = b.rows(1)
        if where < 401:
            rows[where, heads: heads + n_kv] = query.view(1, -1, dim)[0, [0, 4]]
        b.append([(0, 401)], qkv=qkv, rot=0, check=False)
        step, out, old = b.append([(0, 1)], qkv=query, rot=0, check=False)
        b.attend([(0, 1)], step, out, old)


def test_a_page_that_is_none():
    """A table that names a page outside the pool: its keys are not seen, by either kernel, and nothing is read or written there."""
    k = K()
    for dtype, dim in ((F32, 64), (BF16, 64), (BF16, 128)):
        b = Batch(1, 8, 2, dim, dtype, 256, seed=2)
        b.append([(0, 190)], check=False)
        pool = b.pool.clone()
        b.table[0, 1] = -1 if dim == 64 else b.pool.shape[0]
        step, out, old = b.append([(0, 1)], check=False)
        o = torch.empty((1, 8 * dim), dtype=dtype, device=DEV)
        k.attention_q8(out, step, b.pool, b.scales, b.tail, None, b.table, o, 8, 2, dim, b.scale)
        # the reference with those keys taken out: out of reach of a softmax
        line = Line(1, 2, dim)
        line.append(0, np.concatenate([b.line.rows[0][:64], b.line.rows[0][128:]]))
        want, _, _ = line.attend(0, out.view(1, -1, dim)[:, :8].double().cpu().numpy(), 126, b.scale)
        assert np.abs(o.view(1, 8, dim).double().cpu().numpy() - want).max() < 0.03
        b.table[0, 2] = -5                               # the block that fills up next has no page: nothing is stored
        for _ in range(2):
            b.append([(0, 1)], check=False)
        assert torch.equal(b.pool, pool)


@pytest.mark.parametrize("heads,n_kv,dim", [(8, 8, 64), (4, 2, 64), (6, 2, 128), (8, 2, 128), (5, 1, 64), (8, 1, 128), (12, 1, 64)])
@pytest.mark.parametrize("window", [0, 100, 64, 1])
def test_portions_of_any_group(heads, n_kv, dim, window):
    """Portions of unequal lengths, from anywhere in a block, with one to twelve query heads a kv head."""
    b = Batch(3, heads, n_kv, dim, BF16, 640, seed=heads + dim + window)
    b.go([(0, 300), (1, 65), (2, 2)], window=window)
    b.go([(0, 17), (1, 130), (2, 1)], window=window, padding=3)
    b.go([(0, 3), (2, 61)], window=window)
    b.go([(0, 64), (1, 2), (2, 200)], window=window)
    K().check_status(torch.device("cuda:0"))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_later_tokens_that_are_no_numbers(dim, bad):
    """A NaN or an infinity in a later key or value of the same block does not reach the queries before it; the rows that see it show it."""
    k = K()
    for which in (0, 1):                                 # in a key, in a value
        b = Batch(1, 4, 1, dim, BF16, 256, seed=6)
        qkv = b.rows(130)
        clean = qkv.clone()
        qkv.view(130, 6, dim)[100, 4 + which, 5] = bad
        outs = []
        for rows in (clean, qkv):
            b = Batch(1, 4, 1, dim, BF16, 256, seed=6)
            step, out, old = b.append([(0, 130)], qkv=rows.clone(), rot=0, check=False)
            outs.append(b.attend([(0, 130)], step, out, old, check=False).view(130, 4, dim))
        assert torch.equal(outs[0][:100], outs[1][:100]) and torch.isfinite(outs[1][:100]).all()
        if which == 0:
            assert not torch.isfinite(outs[1][100:]).any() or bad == float("inf")
        else:
            assert not torch.isfinite(outs[1][100:128, :, 5]).any()
            others = [i for i in range(dim) if i != 5]
            assert torch.equal(outs[1][100:128][:, :, others], outs[0][100:128][:, :, others])
        assert not torch.isfinite(outs[1][128:]).all()   # the block with it reads as none of them numbers


def test_a_page_of_nan_outside_a_window():
    """A window's edge lies in a page whose scales are NaN: the rows that see none of it are untouched by it."""
    b = Batch(1, 4, 1, 64, BF16, 512, seed=7)
    b.append([(0, 64)], check=False)
    page = int(b.table[0, 0])
    step, out, old = b.append([(0, 130)], check=False)
    good = b.attend([(0, 130)], step, out, old, window=40)
    b.scales[page] = float("nan")
    bad = b.attend([(0, 130)], step, out, old, window=40, check=False)
    # positions 64 + t see keys from 64 + t - 39 on: those of the first page while t < 39
    assert not torch.isfinite(bad[:39]).any() and torch.equal(bad[39:], good[39:])


def test_long_portions():
    b = Batch(2, 8, 2, 128, BF16, 3000, seed=13)
    b.append([(0, 1800), (1, 70)], check=False)
    step, out, old = b.append([(0, 90), (1, 300)], check=False)
    b.attend([(0, 90), (1, 300)], step, out, old)
    K().check_status(torch.device("cuda:0"))


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 64, BF16), (8, 2, 128, BF16), (6, 2, 128, BF16), (12, 1, 64, BF16), (4, 2, 80, BF16), (8, 2, 64, F32),
                                                  (3, 1, 128, F32), (2, 1, 256, F32), (6, 3, 16, F32)])
@pytest.mark.parametrize("window", [0, 700, 70])
def test_portions_behind_long_contexts(heads, n_kv, dim, dtype, window):
    """Few new tokens on many pages, whose walk several blocks share: some of them with no page at all, sequences of unequal lengths."""
    b = Batch(3, heads, n_kv, dim, dtype, 1800, seed=heads + dim + window)
    b.append([(0, 1500), (1, 330), (2, 60)], check=False)
    b.go([(0, 70), (1, 2), (2, 9)], window=window, padding=2)
    b.go([(0, 2)], window=window)
    b.go([(1, 40), (0, 1), (2, 3)], window=window)
    K().check_status(torch.device("cuda:0"))


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (80, BF16), (64, F32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_later_values_that_are_no_numbers_behind_a_long_context(dim, dtype, bad):
    """As above, where the rows that see such a value and those that do not meet from several blocks."""
    outs = []
    for with_it in (False, True):
        b = Batch(1, 4, 1, dim, dtype, 1300, seed=6)
        b.append([(0, 1200)], rot=0, check=False)
        qkv = b.rows(70)
        if with_it:
            qkv.view(70, 6, dim)[10, 5, 5] = bad         # position 1,210, of the block of 1,152 .. 1,215
        step, out, old = b.append([(0, 70)], qkv=qkv, rot=0, check=False)
        outs.append(b.attend([(0, 70)], step, out, old, check=False).view(70, 4, dim))
    others = [i for i in range(dim) if i != 5]
    assert torch.equal(outs[0][:10], outs[1][:10]) and torch.isfinite(outs[1][:10]).all()
    assert torch.equal(outs[0][10:16][:, :, others], outs[1][10:16][:, :, others])
    assert torch.isnan(outs[1][10:16, :, 5]).all() if bad != bad else (outs[1][10:16, :, 5] == bad).all()
    assert not torch.isfinite(outs[1][16:]).all(dim=2).any()          # the block with it reads as none of them numbers


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (48, BF16), (64, F32)])
@pytest.mark.parametrize("gone", [(0,), (3, 4), (9,), tuple(range(10))])
def test_pages_that_are_none_in_a_portions_walk(dim, dtype, gone):
    """Pages outside the pool, at a walk's beginning, inside and at its end, or all of them: their keys are not seen."""
    b = Batch(1, 8, 2, dim, dtype, 800, seed=2)
    b.append([(0, 640)], rot=0, check=False)
    for page in gone:
        b.table[0, page] = -1 if page % 2 else b.pool.shape[0]
    step, out, old = b.append([(0, 64)], rot=0, check=False)
    o = b.attend([(0, 64)], step, out, old, check=False)
    line = Line(1, 2, dim)
    kept = [i for i in range(704) if i // PAGE not in gone]
    line.append(0, np.asarray(b.line.rows[0])[kept])
    b.line = line
    step.start_pos = torch.tensor([640 - PAGE * len(gone)], dtype=torch.int32)
    b.check_attention([(0, 64)], step, out, o, 0)


def test_a_portion_captured_and_two_graphs_at_once():
    """A portion's append and attention in two graphs that are replayed in turns, behind a long context."""
    k = K()
    b = Batch(2, 8, 2, 128, BF16, 1400, seed=21)
    b.append([(0, 1100), (1, 900)], check=False)
    step = make_step([40, 40], b.length, [0, 1])
    freq = b.freq(128)
    graphs = []
    for i in range(2):
        qkv = b.rows(80)
        out, o = torch.empty_like(qkv), torch.empty((80, 8 * 128), dtype=BF16, device=DEV)
        tail = b.tail.clone()
        def both():
            b.tail.copy_(tail)
            old = k.rope_append_q8(qkv, out, step, b.pool, b.scales, b.tail, b.table, freq, 128, 0, 8, 2, 128)
            k.attention_q8(out, step, b.pool, b.scales, b.tail, old, b.table, o, 8, 2, 128, b.scale)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        plain = o.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            both()
        graphs.append((g, qkv, out, o, plain))
    for i in (0, 1, 0, 1, 1):
        g, qkv, out, o, plain = graphs[i]
        o.fill_(float("nan"))
        g.replay()
        assert torch.equal(o, plain)
    k.check_status(torch.device("cuda:0"))


@pytest.mark.parametrize("which", [0, 1])
def test_the_largest_floats(which):
    """Keys and values next to the largest float32 number, which no bfloat16 number reaches: later ones do not reach the queries before."""
    outs = []
    for with_it in (False, True):
        b = Batch(1, 4, 1, 64, F32, 256, seed=6, scale=1e-3)
        qkv = b.rows(90)
        if with_it:
            qkv.view(90, 6, 64)[70, 4 + which, 5] = torch.finfo(F32).max if which else 3.39e38
        step, out, old = b.append([(0, 90)], qkv=qkv, rot=0, check=False)
        outs.append(b.attend([(0, 90)], step, out, old, check=False).view(90, 4, 64))
    assert torch.equal(outs[0][:70], outs[1][:70]) and torch.isfinite(outs[1][:70]).all()
    if which == 1:
        assert torch.isfinite(outs[1][70:]).all() and (outs[1][70:, :, 5] > 1e30).all()


@pytest.mark.parametrize("heads,n_kv,dim,dtype", [(8, 2, 128, BF16), (4, 2, 80, BF16), (4, 1, 64, F32)])
def test_a_prompt_beside_many_single_tokens(heads, n_kv, dim, dtype):
    """More than 32 sequences of very unequal lengths in one step, some of them empty, the long one in the middle."""
    b = Batch(40, heads, n_kv, dim, dtype, 300, seed=dim)
    b.append([(s, 1 + 7 * s % 90) for s in range(40)], check=False)
    entries = [(s, 150 if s == 37 else 2 if s == 3 else 65 if s == 20 else 1) for s in range(40) if s % 5 != 4]
    b.go(entries, padding=3)
    K().check_status(torch.device("cuda:0"))
