"""What the functions of a cache line in 8 bits refuse, without a GPU: every check comes before the first launch."""
import types

import pytest
import torch

from burn_lm_b200 import kernels as K


def arguments(**change):
    n, heads, kv, dim, pages, slots = 3, 4, 2, 32, 5, 2
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    pool, scales = K.q8_pool(pages, kv, dim, "cpu")
    a = dict(qkv=torch.zeros(n, (heads + 2 * kv) * dim), pool=pool, scales=scales, tail=torch.zeros(slots, 2, kv, 64, dim),
             table=torch.zeros(slots, 4, dtype=torch.int32), freq=torch.ones(dim // 2, dtype=torch.float64), rot=dim, turns=None, out=None,
             old=torch.zeros(2, 2, kv, 64, dim), o=torch.zeros(n, heads * dim), window=0, heads=heads, kv=kv, dim=dim,
             step=types.SimpleNamespace(cu_seqlens=i32([0, 2, 3]), slot_of_seq=i32([0, 1]), start_pos=i32([0, 5]), n_seqs=2, max_q_len=2, max_kv_len=6))
    a.update(change)
    if a["out"] is None:
        a["out"] = torch.empty_like(a["qkv"])
    return types.SimpleNamespace(**a)


def append(a):
    return K.rope_append_q8(a.qkv, a.out, a.step, a.pool, a.scales, a.tail, a.table, a.freq, a.rot, 0, a.heads, a.kv, a.dim, table=a.turns)


def attend(a):
    return K.attention_q8(a.out, a.step, a.pool, a.scales, a.tail, a.old, a.table, a.o, a.heads, a.kv, a.dim, 1.0, window=a.window)


BAD_LINE = [dict(pool=torch.zeros(5, 2, 64 * 60, dtype=torch.int8)), dict(pool=torch.zeros(5, 2, 64 * 64)), dict(scales=torch.zeros(5, 2)),
            dict(scales=torch.zeros(4, 2, 2)), dict(scales=torch.zeros(5, 2, 2, dtype=torch.float64)), dict(tail=torch.zeros(2, 2, 2, 63, 32)),
            dict(tail=torch.zeros(2, 2, 2, 64, 32, dtype=torch.bfloat16)), dict(tail=torch.zeros(3, 2, 2, 64, 32)),
            dict(table=torch.zeros(2, 4, dtype=torch.int64)), dict(kv=1), dict(dim=16), dict(heads=5)]


@pytest.mark.parametrize("change", BAD_LINE + [dict(out=torch.zeros(3, 250)), dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)),
                                               dict(freq=torch.ones(16)), dict(freq=torch.ones(15, dtype=torch.float64)), dict(freq=None),
                                               dict(turns=torch.zeros(9, 16, 2, dtype=torch.float64)), dict(turns=torch.zeros(9, 15, 2))])
def test_the_append_refuses(change):
    with pytest.raises(K.KernelError, match="rope_append_q8"):
        append(arguments(**change))


@pytest.mark.parametrize("change", BAD_LINE + [dict(old=None), dict(old=torch.zeros(1, 2, 2, 64, 32)), dict(o=torch.zeros(3, 64)),
                                               dict(o=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(window=-1)])
def test_attention_refuses(change):
    with pytest.raises(K.KernelError, match="attention_q8"):
        attend(arguments(**change))


def test_cpu_tensors_are_refused():
    a = arguments()
    for f in (append, attend):
        with pytest.raises(K.KernelError, match="CUDA device"):
            f(a)
    with pytest.raises(K.KernelError, match="CUDA device"):
        K.q8_values(a.pool, a.scales, torch.zeros(1, dtype=torch.int32), a.dim)


@pytest.mark.parametrize("dim", [8, 17, 24, 272])
def test_head_sizes(dim):
    with pytest.raises(K.KernelError, match="multiples of 16"):
        K.q8_pool(1, 1, dim, "cpu")


def test_places_of_values_are_a_permutation():
    for dim in (16, 48, 64, 80, 128, 256):
        at = K._q8_value_places(dim, torch.device("cpu")).reshape(-1)
        assert at.unique().numel() == 64 * dim and int(at.max()) < K.q8_line_bytes(dim) - 64 * dim


def test_writing_refuses():
    pool, scales = K.q8_pool(3, 2, 32, "cpu")
    eight, s = torch.zeros(2, 2, 64, 32, dtype=torch.int8), torch.zeros(2, 2)
    pages = torch.tensor([0, 2])
    K.q8_write(pool, scales, pages, eight, s, eight, s)
    before = pool.clone()
    K.q8_write(pool, scales, pages[:0], eight[:0], s[:0], eight[:0], s[:0])     # no block at all
    assert torch.equal(pool, before)
    for bad in (dict(keys=eight.float()), dict(values=eight[:1]), dict(ks=s[:1]), dict(pages=pages[:1])):
        a = dict(pages=pages, keys=eight, ks=s, values=eight, vs=s)
        a.update(bad)
        with pytest.raises(K.KernelError, match="q8_write"):
            K.q8_write(pool, scales, a["pages"], a["keys"], a["ks"], a["values"], a["vs"])
