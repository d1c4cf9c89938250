"""A model with its cache in 8 bits or its weights in 4 bits: what is accepted and refused, and the cache's bookkeeping, without a GPU."""
import types

import pytest
import torch

from burn_lm_b200 import kernels as K
from burn_lm_b200 import preset
from burn_lm_b200.cache import Cache, CacheError
from burn_lm_b200.model import Model, make_runtime, plan_of
from burn_lm_b200.parts.base import CacheNeed
from burn_lm_b200.plan import ScheduleEntry
from tiny import TINY_D


def model(config, **kw):
    _, typed, plan = plan_of(config)
    return Model(plan, make_runtime(kw.pop("dtype", "bfloat16"), "cpu", **kw), typed)


def test_what_a_model_keeps():
    m = model(TINY_D, cache="int8")
    need = m.cache_needs()[0]
    assert need.bits == 8 and (need.n_kv_heads, need.head_dim) == (2, 64)
    assert "attention_q8" in m.kernel_modules() and "attention" not in m.kernel_modules()
    assert "gemm_q4" in model(TINY_D, weights="int4").kernel_modules()
    assert model(TINY_D).cache_needs()[0].bits == 0 and "gemm_q4" not in model(TINY_D).kernel_modules()


@pytest.mark.parametrize("name", ["fobilorn_tiny", "nufolix_tiny", "ridopel_tiny", "marinex_tiny", "tomalix_tiny", "samusun_tiny"])
def test_mixers_that_keep_their_cache_in_the_compute_dtype(name):
    with pytest.raises(ValueError, match="cache in 8 bits"):
        model(preset(name), cache="int8")


def test_refused_runtimes():
    for kw in (dict(cache="int4"), dict(weights="int8"), dict(cache=8)):
        with pytest.raises(ValueError, match="one of"):
            make_runtime("bfloat16", "cpu", **kw)
    with pytest.raises(ValueError, match="bfloat16 compute"):
        make_runtime("float32", "cpu", weights="int4")
    assert make_runtime("float32", "cpu", cache="int8").exact


def test_a_run_that_reads_anothers_line():
    import dataclasses
    _, typed, plan = plan_of(TINY_D)
    plan = dataclasses.replace(plan, schedule=(ScheduleEntry(0), ScheduleEntry(1, cache_of=0)))
    Model(plan, make_runtime("bfloat16", "cpu"), typed)
    with pytest.raises(ValueError, match="reads the cache line"):
        Model(plan, make_runtime("bfloat16", "cpu", cache="int8"), typed)


def test_lines_of_a_cache():
    need = CacheNeed("kv", n_kv_heads=2, head_dim=64, bits=8)
    schedule = [ScheduleEntry(0), ScheduleEntry(1)]
    c = Cache([need, need], schedule, 300, 3, 256, torch.bfloat16, torch.device("cpu"))
    v0, v1 = c.view(0), c.view(1)
    assert v0.pool.dtype == torch.int8 and tuple(v0.pool.shape) == (5, 2, K.q8_line_bytes(64)) and tuple(v0.tail.shape) == (3, 2, 2, 64, 64)
    assert v0.tail.dtype == torch.bfloat16 and v0.pool.data_ptr() != v1.pool.data_ptr() and v0.tail.data_ptr() != v1.tail.data_ptr()
    K._q8_line("view", v0.pool, v0.scales, 2, 64)
    assert c.bytes() == 2 * (5 * 2 * K.q8_line_bytes(64) + 3 * 2 * 2 * 64 * 64 * 2)
    slot = c.acquire()
    c.reserve([(slot, 130)])
    assert c.free_pages == 2
    c.release(slot)
    assert c.free_pages == 5
    for bad in (dict(bits=4), dict(bits=8, value_dim=32), dict(bits=8, keep_first=4), dict(bits=8, chunk=64)):
        with pytest.raises(CacheError, match="bits"):
            Cache([CacheNeed("kv", n_kv_heads=2, head_dim=64, **bad)], [ScheduleEntry(0)], 64, 1, 64, torch.bfloat16, torch.device("cpu"))


def test_a_window_gives_pages_back():
    c = Cache([CacheNeed("kv", n_kv_heads=1, head_dim=16, bits=8, window=70)], [ScheduleEntry(0)], 640, 1, 640, torch.float32, torch.device("cpu"))
    slot = c.acquire()
    for n in (200, 201, 400):
        c.reserve([(slot, n)])
        c.set_length(slot, n)
    c.reserve([(slot, 401)])
    assert c.free_pages == 10 - (7 - (400 - 70 + 1) // 64)


def test_linear_in_four_bits():
    from burn_lm_b200.parts.linear import Linear
    w = torch.randn(64, 96, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    lin = Linear(w)
    want = K.q4_values(K.quantize_q4(w, 64))
    lin.to_4bit()
    assert lin.weight is None and torch.equal(K.q4_values(lin.q4), want) and (lin.out_features, lin.in_features) == (64, 96)
    first = lin.first_rows(32)
    assert torch.equal(K.q4_values(first.q4), want[:32]) and first is lin.first_rows(32) and first.out_features == 32
    with pytest.raises(K.KernelError, match="tiles of 16"):
        lin.first_rows(20)
    with pytest.raises(ValueError, match="bfloat16"):
        Linear(w.float()).to_4bit()
    plain = Linear(w)
    assert plain.first_rows(20).weight.data_ptr() == w.data_ptr() and tuple(plain.first_rows(20).weight.shape) == (20, 96)


def test_the_command_line_passes_it_on(monkeypatch):
    from burn_lm_b200 import cli
    seen = []
    monkeypatch.setattr(cli.api, "load", lambda folder, **kw: (seen.append(kw), types.SimpleNamespace())[1])
    monkeypatch.setattr(cli, "_answer", lambda *a: 0)
    for flags, want in (([], {}), (["--cache", "int8"], {"cache": "int8"}), (["--weights", "int4", "--cache", "int8"], {"cache": "int8", "weights": "int4"})):
        args = cli.build_parser().parse_args(["run", "folder", *flags, "1 2"])
        cli._load(args)
        assert {k: v for k, v in seen[-1].items() if k in ("cache", "weights")} == want
    with pytest.raises(SystemExit):
        cli.build_parser().parse_args(["run", "folder", "--cache", "int4", "1 2"])
