"""What is timed of a model held in fewer bits: keys and values in 8 bits with a scale for every block of 64 positions and head,
and weights in 4 bits with a scale for every group along K.

Three operators, each through the call a decoder layer makes:

  append    rotate a step's queries and keys by their positions and append keys and values to the paged cache: the rows of a
            block that the step completes are stored in 8 bits, those of a block still unfinished unrounded, in the sequence's
            tail.  Scale of a block's keys (values) of one head: largest magnitude of its 64 x D numbers / 127.
  attend    causal grouped-query attention over that cache: a query sees the blocks before its own in 8 bits and the keys of
            its own block unrounded.
  product   x W^T with W = scale[row, k // group] * (a whole number of -8 .. 7), plain, added into a float32 stream, or gated
            (tiles of 8 gate rows followed by the 8 up rows of the same outputs).

A case's "lengths" are the new tokens of every sequence ("1x8": eight sequences of one token), "cached" the positions every
sequence holds before the step, give or take a few so that the batch is ragged.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
DEV = "cuda"
THETA = 500000.0


def listed():
    return [
        # eight chats that decode, one layer of the 1B decoder: the smallest call; one sequence fills a block
        dict(name="append_decode8", kind="append", heads=32, kv=8, dim=64, lengths="1x8", cached=1003, dtype="bfloat16"),
        # a full batch decoding with heads of 128 (the 8B decoder's layer)
        dict(name="append_decode64", kind="append", heads=32, kv=8, dim=128, lengths="1x64", cached=2011, dtype="bfloat16"),
        # a packed batch of unequal prompts
        dict(name="append_prompts", kind="append", heads=32, kv=8, dim=64, lengths="1000,611,37,400", cached=0, dtype="bfloat16"),
        # eight chats of about 2,000 tokens, heads of 128
        dict(name="attend_decode8", kind="attend", heads=32, kv=8, dim=128, lengths="1x8", cached=2000, window=0, dtype="bfloat16"),
        # a full batch of about 1,100 tokens each, heads of 64
        dict(name="attend_decode64", kind="attend", heads=32, kv=8, dim=64, lengths="1x64", cached=1087, window=0, dtype="bfloat16"),
        # one sequence with a long document behind it
        dict(name="attend_long", kind="attend", heads=32, kv=8, dim=128, lengths="1", cached=32005, window=0, dtype="bfloat16"),
        # a long prompt
        dict(name="attend_prompt", kind="attend", heads=32, kv=8, dim=128, lengths="2048", cached=0, window=0, dtype="bfloat16"),
        # portions of prompts in the middle of a conversation, in the 32-bit path
        dict(name="attend_float32", kind="attend", heads=32, kv=8, dim=64, lengths="100,37", cached=700, window=0, dtype="float32"),
        # one token through the 1B decoder's gate and up weights
        dict(name="product_gated1", kind="product", tokens=1, out=16384, inner=2048, group=64, end="gated"),
        # eight tokens through the 8B decoder's q|k|v weight
        dict(name="product_qkv8", kind="product", tokens=8, out=6144, inner=4096, group=128, end="store"),
        # sixteen tokens through its down weight, added into the residual stream
        dict(name="product_down16", kind="product", tokens=16, out=4096, inner=14336, group=64, end="add"),
        # a prompt through its gate and up weights
        dict(name="product_prompt", kind="product", tokens=512, out=28672, inner=4096, group=64, end="gated"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "product", "product"])
    if kind == "product":
        end = rng.choice(["store", "add", "gated"])
        out, inner = _log(rng, 500, 14000), _log(rng, 500, 14336)
        if rng.random() < 0.7:
            inner = -(-inner // 64) * 64
        if end == "gated":
            out = -(-out // 16) * 16
        tokens = min(_log(rng, 1, 600), max(1, 59_000_000_000 // (out * inner)))
        return dict(kind=kind, tokens=tokens, out=out, inner=inner, group=rng.choice([32, 64, 128]), end=end)
    heads, kv = rng.choice([(32, 8), (32, 8), (24, 8), (16, 16), (8, 1), (12, 4), (20, 4)])
    dim = rng.choice([64, 128, 64, 128, 80])
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    if rng.random() < 0.6:
        seqs = _log(rng, 1, 64)
        lengths, cached = "1x%d" % seqs, _log(rng, 1, min(16000, 100000 // seqs))
    else:
        seqs = rng.randint(1, 4)
        lengths = ",".join(str(_log(rng, 2, (1400 if dtype == "bfloat16" else 300) // seqs)) for _ in range(seqs))
        cached = rng.choice([0, _log(rng, 1, 1200)])
    case = dict(kind=kind, heads=heads, kv=kv, dim=dim, lengths=lengths, cached=cached, dtype=dtype)
    if kind == "attend":
        case["window"] = rng.choice([0, 0, 0, _log(rng, 20, 2000)])
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------------
def _lengths(case):
    text = case["lengths"]
    if "x" in text:
        n, times = text.split("x")
        return [int(n)] * int(times)
    return [int(n) for n in text.split(",")]


def _starts(case):
    """Positions cached before the step: about `cached` each, ragged; the fourth of every 32 sequences is about to fill a block."""
    c, n = case["cached"], len(_lengths(case))
    starts = [0 if c == 0 else max(1, c + (s * 20) % 83 - min(41, 20 * (n - 1))) for s in range(n)]
    return [s // PAGE * PAGE + PAGE - 1 if i % 32 == 3 and s else s for i, s in enumerate(starts)]


def _dtype(case):
    return torch.float32 if case["dtype"] == "float32" else torch.bfloat16


class _Draws:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 7919 + 5)

    def normal(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=DEV).normal_(generator=self.g)

    def uniform(self, lo, hi, *shape):
        return torch.empty(shape, dtype=torch.float32, device=DEV).uniform_(lo, hi, generator=self.g)


def _frequencies(dim):
    return torch.tensor([THETA ** (-2.0 * i / dim) for i in range(dim // 2)], dtype=torch.float64, device=DEV)


def _in_eight(x):
    """x [blocks, 64, kv, D] as (int8 of the same shape, float32 scales [blocks, kv]): the rule of the cache."""
    x = x.float()
    scale = x.abs().amax(dim=(1, 3)) / 127.0
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.round(x / safe[:, None, :, None]).clamp(-127, 127).to(torch.int8), scale


def _pages(case):
    """How many pages every sequence holds after the step, and which ones: in a shuffled order."""
    each = [-(-(s + n) // PAGE) for s, n in zip(_starts(case), _lengths(case))]
    order = np.random.RandomState(sum(each) + len(each)).permutation(sum(each))
    table = np.zeros((len(each), max(each)), dtype=np.int32)
    at = 0
    for s, e in enumerate(each):
        table[s, :e] = order[at: at + e]
        at += e
    return table, sum(each)


def _step(case):
    from burn_lm_b200.engine.engine import Workspace
    from burn_lm_b200.parts.base import StepContext
    lens, starts = _lengths(case), _starts(case)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return StepContext(
        n_tokens=cu[-1], n_seqs=len(lens), max_q_len=max(lens), max_kv_len=max(s + n for s, n in zip(starts, lens)),
        tokens=i32([0] * cu[-1]), token_seq=i32([s for s, n in enumerate(lens) for _ in range(n)]),
        token_pos=i32([s + t for s, n in zip(starts, lens) for t in range(n)]), cu_seqlens=i32(cu),
        slot_of_seq=i32(list(range(len(lens)))), start_pos=i32(starts), want_rows=None, n_want=0, workspace=Workspace(torch.device(DEV)))


def prepare(case, seed):
    d = _Draws(seed)
    if case["kind"] == "product":
        m, k, group = case["out"], case["inner"], case["group"]
        groups = -(-k // group)
        values = torch.empty((m, k), dtype=torch.float32, device=DEV).normal_(generator=d.g).mul_(3.0).round_().clamp_(-8, 7).to(torch.int8)
        # scales as a weight's quantising leaves them: about 1 / (3 sqrt(K)), five significant bits
        mantissa = torch.round(d.uniform(16.0, 31.0, m, groups))
        scales = (mantissa * 2.0 ** math.floor(math.log2(k ** -0.5 / 60.0))).to(torch.bfloat16)
        state = dict(case=case, values=values, scales=scales, x=d.normal(case["tokens"], k).to(torch.bfloat16))
        if case["end"] == "add":
            state["stream"] = d.normal(case["tokens"], m)
        if own:
            from burn_lm_b200 import kernels as K
            state["weight"] = K.pack_q4(values, scales, group)
        return state
    dt, kv, dim = _dtype(case), case["kv"], case["dim"]
    lens, starts = _lengths(case), _starts(case)
    n, width = sum(lens), (case["heads"] + 2 * kv) * dim
    # keys have a few lanes that are several times as large as the others
    lane = torch.ones(dim, device=DEV)
    lane[torch.randperm(dim, generator=d.g, device=DEV)[: max(1, dim // 16)]] = 5.0
    table, n_pages = _pages(case)
    state = dict(case=case, freq=_frequencies(dim), table=torch.from_numpy(table).to(DEV))
    rows = d.normal(n, case["heads"] + 2 * kv, dim)
    rows[:, case["heads"]: case["heads"] + kv] *= lane
    if case["kind"] == "append":
        state["qkv"] = rows.view(n, width).to(dt)
        state["tail0"] = (d.normal(len(lens), 2, kv, PAGE, dim) * lane).to(dt)
        state["tail"] = state["tail0"].clone()
        state["done"] = [(s, b) for s in range(len(lens)) for b in range(starts[s] // PAGE, (starts[s] + lens[s]) // PAGE)]
        if own:
            from burn_lm_b200 import kernels as K
            state["step"] = _step(case)
            state["pool"], state["scales"] = K.q8_pool(n_pages, kv, dim, DEV)
            state["done_pages"] = torch.tensor([int(table[s, b]) for s, b in state["done"]], dtype=torch.int32, device=DEV)
            state["turns"] = K.rope_table(state["freq"], max(s + t for s, t in zip(starts, lens)))
        return state
    # attend: every sequence's keys and values, the blocks that are complete after the step in 8 bits, the step's own rows and the
    # rows of the block it found unfinished as they are
    state["rotated"] = rows.view(n, width).to(dt)
    state["tail"] = torch.zeros((len(lens), 2, kv, PAGE, dim), dtype=dt, device=DEV)
    state["blocks"] = []
    at = 0
    for s, (start, new) in enumerate(zip(starts, lens)):
        k = (d.normal(start + new, kv, dim) * lane * 0.8).to(dt)
        v = d.normal(start + new, kv, dim).to(dt)
        step_rows = state["rotated"][at: at + new].view(new, -1, dim)
        k[start:], v[start:] = step_rows[:, case["heads"]: case["heads"] + kv], step_rows[:, case["heads"] + kv:]
        first = start // PAGE * PAGE
        # (a step of one token a sequence has left its own row in the tail as well, unless it completed the block)
        last = start if (start + new) % PAGE == 0 or max(lens) > 1 else start + new
        state["tail"][s, 0, :, : last - first] = k[first:last].transpose(0, 1)
        state["tail"][s, 1, :, : last - first] = v[first:last].transpose(0, 1)
        full = (start + new) // PAGE
        cut = lambda x: x[: full * PAGE].view(full, PAGE, kv, dim)  # noqa: E731
        state["blocks"].append(_in_eight(cut(k)) + _in_eight(cut(v)))
        at += new
    if own:
        from burn_lm_b200 import kernels as K
        state["step"] = _step(case)
        state["pool"], state["scales"] = K.q8_pool(n_pages, kv, dim, DEV)
        for s, (k8, ks, v8, vs) in enumerate(state["blocks"]):
            K.q8_write(state["pool"], state["scales"], state["table"][s, : k8.shape[0]], k8.transpose(1, 2), ks, v8.transpose(1, 2), vs)
        state["old"] = state["tail"] if max(lens) > 1 else None
    return state


# ---- the operators -------------------------------------------------------------------------------------------------------
def run(state):
    return {"append": _append, "attend": _attend, "product": _product}[state["case"]["kind"]](state)


def _append(state):
    c = state["case"]
    if max(_lengths(c)) > 1 and c["cached"]:
        state["tail"].copy_(state["tail0"])             # the rows a portion finds; it may write the next block's over them
    if own:
        from burn_lm_b200 import kernels as K
        out = torch.empty_like(state["qkv"])
        K.rope_append_q8(state["qkv"], out, state["step"], state["pool"], state["scales"], state["tail"], state["table"], state["freq"],
                         c["dim"], K.PAIRS_HALVES, c["heads"], c["kv"], c["dim"], table=state["turns"])
        got = dict(rotated=out, tail=state["tail"])
        if state["done"]:
            got["cached"] = K.q8_values(state["pool"], state["scales"], state["done_pages"], c["dim"], out.dtype)
            got["scales"] = state["scales"][state["done_pages"]]
        return got
    heads, kv, dim, dt = c["heads"], c["kv"], c["dim"], _dtype(c)
    lens, starts = _lengths(c), _starts(c)
    pos = torch.tensor([s + t for s, n in zip(starts, lens) for t in range(n)], dtype=torch.float64, device=DEV)
    angle = pos[:, None] * state["freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = state["qkv"].view(len(pos), heads + 2 * kv, dim).float()
    a, b = x[:, : heads + kv, : dim // 2], x[:, : heads + kv, dim // 2:]
    out = torch.cat([torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2), x[:, heads + kv:]], dim=1).to(dt)
    keys, values, tail = out[:, heads: heads + kv], out[:, heads + kv:], state["tail"]
    got = dict(rotated=out.view(len(pos), -1), tail=tail)
    done_k, done_v, at = [], [], 0
    for s, (start, n) in enumerate(zip(starts, lens)):
        first, had, full = start // PAGE, start % PAGE, (start + n) // PAGE
        k = torch.cat([tail[s, 0, :, :had].transpose(0, 1), keys[at: at + n]])
        v = torch.cat([tail[s, 1, :, :had].transpose(0, 1), values[at: at + n]])
        cut = (full - first) * PAGE
        done_k.append(k[:cut].view(-1, PAGE, kv, dim))
        done_v.append(v[:cut].view(-1, PAGE, kv, dim))
        new = max(cut, had)             # the rows of the unfinished block that this step brings
        tail[s, 0, :, new - cut: len(k) - cut] = k[new:].transpose(0, 1)
        tail[s, 1, :, new - cut: len(v) - cut] = v[new:].transpose(0, 1)
        at += n
    if state["done"]:
        k8, ks = _in_eight(torch.cat(done_k))
        v8, vs = _in_eight(torch.cat(done_v))
        both = torch.stack([k8 * ks[:, None, :, None], v8 * vs[:, None, :, None]], dim=1)      # [blocks, 2, 64, kv, D]
        got["cached"], got["scales"] = both.transpose(2, 3).contiguous().to(dt), torch.stack([ks, vs], dim=2)
    return got


def _attend(state):
    c = state["case"]
    heads, kv, dim, dt = c["heads"], c["kv"], c["dim"], _dtype(c)
    n = state["rotated"].shape[0]
    out = torch.empty((n, heads * dim), dtype=dt, device=DEV)
    if own:
        from burn_lm_b200 import kernels as K
        K.attention_q8(state["rotated"], state["step"], state["pool"], state["scales"], state["tail"], state["old"], state["table"], out,
                       heads, kv, dim, dim ** -0.5, window=c["window"])
        return out
    rows, at, group = state["rotated"].view(n, -1, dim), 0, heads // kv
    for s, (start, new) in enumerate(zip(_starts(c), _lengths(c))):
        k8, ks, v8, vs = state["blocks"][s]
        had, first, length = start % PAGE, start // PAGE * PAGE, start + new
        mine = rows[at: at + new]
        exact = [torch.cat([state["tail"][s, i, :, :had].transpose(0, 1), mine[:, heads + i * kv: heads + (i + 1) * kv]]).float() for i in range(2)]
        cached = [torch.zeros((length, kv, dim), device=DEV) for _ in range(2)]
        cached[0][: k8.shape[0] * PAGE] = (k8 * ks[:, None, :, None]).view(-1, kv, dim)
        cached[1][: k8.shape[0] * PAGE] = (v8 * vs[:, None, :, None]).view(-1, kv, dim)
        i, j = torch.arange(start, length, device=DEV)[:, None], torch.arange(length, device=DEV)[None, :]
        inside = i // PAGE == j // PAGE
        seen = (j <= i) & ((j > i - c["window"]) if c["window"] else True)
        for h in range(kv):
            q = mine[:, h * group: (h + 1) * group].float().transpose(0, 1)                     # [group, new, D]
            scores = q @ cached[0][:, h].t()
            scores[:, :, first:] = torch.where(inside[:, first:], q @ exact[0][:, h].t(), scores[:, :, first:])
            scores = torch.where(seen, scores * dim ** -0.5, torch.full((), -math.inf, device=DEV))
            w = torch.exp(scores - scores.amax(dim=2, keepdim=True))
            w = w / w.sum(dim=2, keepdim=True)
            o = (w * ~inside) @ cached[1][:, h] + (w * inside)[:, :, first:] @ exact[1][:, h]
            out[at: at + new].view(new, heads, dim)[:, h * group: (h + 1) * group] = o.transpose(0, 1).to(dt)
        at += new
    return out


def _product(state):
    c, x = state["case"], state["x"]
    if own:
        from burn_lm_b200 import kernels as K
        if c["end"] == "add":
            stream = state["stream"].clone()
            K.product_q4(state["weight"], x, add_into=stream)
            return stream
        out = torch.empty((x.shape[0], c["out"] // (2 if c["end"] == "gated" else 1)), dtype=torch.bfloat16, device=DEV)
        K.product_q4(state["weight"], x, out=out, swiglu=c["end"] == "gated")
        return out
    scales = state["scales"].float().repeat_interleave(c["group"], dim=1)[:, : c["inner"]]
    y = x.float() @ (state["values"] * scales).t()
    if c["end"] == "add":
        return state["stream"] + y
    if c["end"] == "gated":
        y = y.view(x.shape[0], -1, 2, 8)
        gate, up = y[:, :, 0], y[:, :, 1]
        y = (gate / (1.0 + torch.exp(-gate)) * up).reshape(x.shape[0], -1)
    return y.to(torch.bfloat16)


# ---- what they cannot do without -----------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "product":
        n, m, k = case["tokens"], case["out"], case["inner"]
        ends = {"store": 2 * n * m, "gated": n * m, "add": 8 * n * m}[case["end"]]
        return {"bytes": m * k / 2 + 2 * m * -(-k // case["group"]) + 2 * n * k + ends, "flops": 2 * n * m * k}
    heads, kv, dim, e = case["heads"], case["kv"], case["dim"], 4 if case["dtype"] == "float32" else 2
    lens, starts = _lengths(case), _starts(case)
    n, line = sum(lens), 2 * kv * dim
    if case["kind"] == "append":
        total = 2 * n * (heads + 2 * kv) * dim * e
        for s, new in zip(starts, lens):
            blocks, had = (s + new) // PAGE - s // PAGE, s % PAGE
            total += blocks * (PAGE * line + 8 * kv) + (had * line * e if blocks else 0)      # what it completes, the rows found for it
            total += ((s + new) % PAGE if blocks else new) * line * e                         # what goes to the tail
        return {"bytes": total, "flops": 6 * n * (heads + kv) * dim // 2}
    total, flops, window = 2 * n * heads * dim * e, 0, case["window"]
    for s, new in zip(starts, lens):
        low = max(0, s - window + 1) if window else 0
        total += (s // PAGE - low // PAGE) * (PAGE * line + 8 * kv) + (s % PAGE + new) * line * e
        pairs = sum(min(s + t + 1, window) if window else s + t + 1 for t in range(new))
        flops += 4 * heads * dim * pairs
    return {"bytes": total, "flops": flops}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "product":
        n, m, k, group = case["tokens"], case["out"], case["inner"], case["group"]
        y = torch.zeros((n, m), dtype=torch.float64, device=DEV)
        for g in range(-(-k // group)):                 # group after group: whole numbers first, then the group's scale
            part = state["x"][:, g * group: (g + 1) * group].double() @ state["values"][:, g * group: (g + 1) * group].double().t()
            y += part * state["scales"][:, g].double()
        if case["end"] == "add":
            return y + state["stream"].double()
        if case["end"] == "gated":
            tiles = y.view(n, m // 16, 16)
            return (tiles[:, :, :8] * torch.sigmoid(tiles[:, :, :8]) * tiles[:, :, 8:]).reshape(n, m // 2)
        return y
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    lens, starts = _lengths(case), _starts(case)
    group, at = heads // kv, 0
    if case["kind"] == "append":
        x = state["qkv"].double().view(-1, heads + 2 * kv, dim)
        pos = torch.cat([torch.arange(s, s + n, device=DEV) for s, n in zip(starts, lens)]).double()
        pairs = torch.view_as_complex(torch.stack([x[..., : dim // 2], x[..., dim // 2:]], dim=-1).contiguous())
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.outer(pos, state["freq"]))
        turned = torch.view_as_real(pairs * turn[:, None])
        x = torch.where((torch.arange(heads + 2 * kv, device=DEV) < heads + kv)[:, None], torch.cat([turned[..., 0], turned[..., 1]], dim=-1), x)
        tail, cached, scales = state["tail0"].double(), [], []
        stored = x.to(_dtype(case)).double()            # what the cache is made of: the rows in the compute type
        for s, (start, n) in enumerate(zip(starts, lens)):
            had = start % PAGE
            now = stored[at: at + n, heads:].view(n, 2, kv, dim)
            rows = torch.cat([state["tail0"][s].double().permute(2, 0, 1, 3)[:had], now])        # [positions, 2, kv, D]
            while len(rows) >= PAGE:
                block = rows[:PAGE].permute(1, 2, 0, 3)
                scale = block.abs().amax(dim=(2, 3), keepdim=True) / 127
                cached.append(torch.round(block / scale.clamp(min=1e-300)) * scale)
                scales.append(scale[:, :, 0, 0].t())
                rows, had = rows[PAGE:], 0
            tail[s, :, :, had: len(rows)] = rows[had:].permute(1, 2, 0, 3)
            at += n
        got = dict(rotated=x.view(len(pos), -1), tail=tail)
        if cached:
            got["cached"], got["scales"] = torch.stack(cached), torch.stack(scales)
        return got
    out = torch.empty((sum(lens), heads, dim), dtype=torch.float64, device=DEV)
    for s, (start, n) in enumerate(zip(starts, lens)):
        k8, ks, v8, vs = (t.double() for t in state["blocks"][s])
        k_all, v_all = (k8 * ks[:, None, :, None]).reshape(-1, kv, dim), (v8 * vs[:, None, :, None]).reshape(-1, kv, dim)
        mine = state["rotated"][at: at + n].double().view(n, -1, dim)
        first = start - start % PAGE
        found = state["tail"][s].double()[:, :, : start - first].permute(2, 0, 1, 3)
        near = torch.cat([found, mine[:, heads:].view(n, 2, kv, dim)])                             # unrounded, from position `first` on
        for begin in range(first, start + n, PAGE):     # the queries of one block: what they see is one stretch of keys
            lo, hi = max(begin, start), min(begin + PAGE, start + n)
            low = max(0, lo - case["window"] + 1) if case["window"] else 0
            low = min(low, begin)
            block = near[begin - first: hi - first]
            k = torch.cat([k_all[low:begin], block[:, 0]])
            v = torch.cat([v_all[low:begin], block[:, 1]])
            q = mine[lo - start: hi - start, :heads].view(hi - lo, kv, group, dim)
            scores = torch.einsum("qhgd,khd->hgqk", q, k) / math.sqrt(dim)
            away = torch.arange(lo, hi, device=DEV)[:, None] - torch.arange(low, hi, device=DEV)[None, :]
            hidden = (away < 0) | ((away >= case["window"]) if case["window"] else False)
            weights = torch.softmax(scores.masked_fill(hidden, -math.inf), dim=-1)
            out[at + lo - start: at + hi - start] = torch.einsum("hgqk,khd->qhgd", weights, v).reshape(hi - lo, heads, dim)
        at += n
    return out.view(sum(lens), -1)
