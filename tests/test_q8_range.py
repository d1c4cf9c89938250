"""What the functions of a cache line in 8 bits refuse beside shapes and types, without a GPU."""
import types

import pytest
import torch

from burn_lm_b200 import kernels as K
from test_q8 import arguments


class On:
    """A tensor on a device, as far as an address is asked for."""

    def __init__(self, device, contiguous=True):
        self.device, self.contiguous = device, contiguous

    def get_device(self):
        return self.device

    def is_contiguous(self):
        return self.contiguous

    def data_ptr(self):
        return 64 + self.device


def test_a_steps_tensors_lie_on_the_current_device(monkeypatch):
    """Kernels run on the current device's stream: a step on another one is refused, as the other tensors are."""
    monkeypatch.setattr(K, "_current_device", lambda: 1)
    step = lambda *t: types.SimpleNamespace(cu_seqlens=t[0], slot_of_seq=t[1], start_pos=t[2])  # noqa: E731
    assert K._step_ptrs("attention_q8", step(On(1), On(1), On(1))) == (65, 65, 65)
    for bad in ((On(0), On(0), On(0)), (On(1), On(0), On(1)), (On(1), On(1), On(0)), (On(1), On(1), On(1, False)), (On(-1), On(-1), On(-1))):
        with pytest.raises(K.KernelError, match="attention_q8: a step's tensors"):
            K._step_ptrs("attention_q8", step(*bad))


@pytest.mark.parametrize("scale", [-0.125, -1e-30, float("nan"), float("inf")])
def test_scales_of_scores_that_are_refused(scale):
    """The portions' kernel seeks the largest score before it multiplies: a negative scale would make it the smallest."""
    a = arguments()
    with pytest.raises(K.KernelError, match="attention_q8: scores times"):
        K.attention_q8(a.out, a.step, a.pool, a.scales, a.tail, a.old, a.table, a.o, a.heads, a.kv, a.dim, scale)
    for fine in (0.0, 1.0):
        with pytest.raises(K.KernelError, match="CUDA device"):
            K.attention_q8(a.out, a.step, a.pool, a.scales, a.tail, a.old, a.table, a.o, a.heads, a.kv, a.dim, fine)


def test_writing_refuses_scales_below_zero_and_pages_of_another_pool():
    """A block with a negative scale would be taken for a page that is none, and its keys left out; page -1 would be the pool's last."""
    pool, scales = K.q8_pool(3, 2, 32, "cpu")
    eight, s, pages = torch.ones(2, 2, 64, 32, dtype=torch.int8), torch.ones(2, 2), torch.tensor([0, 2])
    before = pool.clone()
    down = s.clone()
    down[1, 0] = -1.0
    for ks, vs in ((down, s), (s, down)):
        with pytest.raises(K.KernelError, match="below zero"):
            K.q8_write(pool, scales, pages, eight, ks, eight, vs)
    for wrong in ([-1, 0], [0, 3]):
        with pytest.raises(K.KernelError, match="numbers below 3"):
            K.q8_write(pool, scales, torch.tensor(wrong), eight, s, eight, s)
    assert torch.equal(pool, before)
    for fine in (s * 0, s * float("inf"), s * float("nan")):
        K.q8_write(pool, scales, pages, eight, fine, eight, s)


@pytest.mark.parametrize("heads,kv", [(0, 2), (-2, 2), (5, 2), (2, 0), (1, 2)])
@pytest.mark.parametrize("dtype,dim,new", [(1, 64, 1), (1, 128, 5), (0, 64, 1), (1, 80, 7)])
def test_numbers_of_heads_at_the_entry(heads, kv, dtype, dim, new):
    """The entries refuse what cannot be planned (with no head at all, a division by zero ended the process); no pointer is looked at."""
    with pytest.raises(K.KernelError, match="attention_q8: .* heads do not divide"):
        K._call("attention_q8", "blm_attention_q8", 0, 0, 0, 1, dtype, 0, 4, 0, 0, 0, 0, new, 1, heads, kv, dim, 1, 0, 0.125, new, 64, 0, 1, 0, 0)
    with pytest.raises(K.KernelError, match="rope_append_q8: .* heads do not divide"):
        K._call("attention_q8", "blm_rope_append_q8", 0, 0, dtype, 0, 0, 0, 0, 4, 0, 0, 0, 0, 0, 1.0, 0, 0, 0, new, 1, new, heads, kv, dim, 1, 0)
    assert K._ask("attention_q8", "blm_attention_q8_splits", dtype, 1, new, 5000, heads, kv, dim, 0) >= 1
