"""Whole models with their cache in 8 bits and their weights in 4 bits, against the plain implementation given the same."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from plain import llama_plain as plain
from q8_reference import Line
from tiny import MORE_CONFIGS, make_folder, random_tokens, row_error

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def engine(folder, dtype="bfloat16", max_tokens=2048, **kw):
    from burn_lm_b200 import Engine
    return Engine.from_folder(folder, dtype=dtype, max_tokens=max_tokens, max_seqs=4, **kw)


def in_four_bits(tensors):
    """The tensors with the layers' weights rounded to 4 bits, as the model rounds them."""
    from burn_lm_b200 import kernels as K
    out = dict(tensors)
    for name, w in tensors.items():
        if name.endswith("_proj.weight"):
            out[name] = K.q4_values(K.quantize_q4(torch.from_numpy(w).to(torch.bfloat16), 64)).double().numpy()
    return out


def forward(cfg, tensors, tokens, dtype):
    """plain.forward with the keys and values of blocks before a query's own in 8 bits, of rows rounded to `dtype`."""
    cfg = plain.complete_config(cfg)
    inv = plain.model_inverse_frequencies(cfg)
    heads, kv, dim, eps = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], cfg["rms_norm_eps"]
    n = len(tokens)
    h = plain.embedding(tensors["model.embed_tokens.weight"], tokens)
    for layer in range(cfg["num_hidden_layers"]):
        lw = plain.layer_weights(tensors, layer)
        x = plain.rms_norm(h, lw["input_layernorm"], eps)
        q, k, v = ((x @ lw[w].T).reshape(n, -1, dim) for w in ("q_proj", "k_proj", "v_proj"))
        q, k = (plain.rope_apply(t.transpose(1, 0, 2), np.arange(n), inv, "half").transpose(1, 0, 2) for t in (q, k))
        line = Line(1, kv, dim)
        stored = torch.from_numpy(np.stack([k, v], axis=1)).to(dtype).float().numpy()
        line.append(0, stored)
        o, _, _ = line.attend(0, q, 0, dim ** -0.5)
        h = h + o.reshape(n, heads * dim) @ lw["o_proj"].T
        h = h + plain.feed_forward(plain.rms_norm(h, lw["post_attention_layernorm"], eps), lw["gate_proj"], lw["up_proj"], lw["down_proj"])
    h = plain.rms_norm(h, tensors["model.norm.weight"], eps)
    return h @ (tensors["model.embed_tokens.weight"] if cfg["tie_word_embeddings"] else tensors["lm_head.weight"]).T


def logits_of(eng, tokens, cuts):
    from burn_lm_b200 import StepEntry
    slot, at, out = eng.acquire(), 0, []
    for n in cuts:
        out.append(eng.step([StepEntry(slot, tokens[at: at + n], list(range(n)))]).float().cpu().numpy().copy())
        at += n
    eng.verify()
    eng.release(slot)
    return np.concatenate(out)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["tiny_c", "tiny_d", "tiny_e", "tiny_f"])
def test_logits_with_a_cache_in_8_bits(tmp_path, name, dtype):
    folder = make_folder(tmp_path, name, seed=3, dtype="bfloat16")
    cfg, tensors = plain.read_model_folder(folder)
    tokens = random_tokens(5, 200, cfg["vocab_size"])
    want, exact = forward(cfg, tensors, tokens, getattr(torch, dtype)), plain.forward(cfg, tensors, tokens)
    eng = engine(folder, dtype, cache="int8")
    for cuts in ([200], [130, 1, 1, 1, 67], [60] + [1] * 12 + [128]):
        got = logits_of(eng, tokens, cuts)
        err = row_error(got, want)
        # float32: a number near a border between two of its block's 255 values may fall to the other side (one in some thousands)
        assert err.max() < (5e-3 if dtype == "float32" else 4e-2)
        if dtype == "float32":                   # what the 8 bits change is there, and it is not what is left
            assert np.median(err[64:]) < 0.2 * np.median(row_error(exact, want)[64:])


@pytest.mark.parametrize("name", ["tiny_c", "tiny_d", "tiny_e"])
def test_logits_with_weights_in_4_bits(tmp_path, name):
    folder = make_folder(tmp_path, name, seed=3, dtype="bfloat16")
    cfg, tensors = plain.read_model_folder(folder)
    tokens = random_tokens(6, 150, cfg["vocab_size"])
    want = plain.forward(cfg, in_four_bits(tensors), tokens)
    eng = engine(folder, weights="int4")
    for cuts in ([150], [100, 1, 1, 20, 28], [4] * 37 + [2]):
        assert row_error(logits_of(eng, tokens, cuts), want).max() < 4e-2


def test_both_together_generate(tmp_path):
    """Greedy generation of a batch of unequal prompts through the captured steps, the device-side loop and steps enqueued ahead:
    every token is the plain implementation's or a near tie with it."""
    import burn_lm_b200 as blm
    folder = make_folder(tmp_path, "tiny_d", seed=4, dtype="bfloat16")
    cfg, tensors = plain.read_model_folder(folder)
    four = in_four_bits(tensors)
    prompts = [random_tokens(n, length, cfg["vocab_size"]) for n, length in enumerate([5, 62, 130])]
    outs = []
    for ahead in (False, True):
        lm = blm.load(folder, max_seq_len=256, max_batch=3, cache="int8", weights="int4", decode_ahead=ahead)
        outs.append(lm.generate(prompts, sample_len=70, ignore_stop=True).tokens)
        drawn = lm.generate(prompts, sample_len=9, temperature=0.8, seed=3, ignore_stop=True).tokens
        assert all(len(t) == 9 for t in drawn)
        lm.engine.verify()
    assert outs[0] == outs[1]
    for p, out in zip(prompts, outs[0]):
        logits = forward(cfg, four, p + out, torch.bfloat16)[len(p) - 1: -1]
        near = logits.max(axis=1) - logits[np.arange(len(out)), out]
        assert (near <= 6e-2 * np.abs(logits).max(axis=1)).all()


def test_device_side_loop_matches_steps(tmp_path):
    """decode_run over a block's end: the same tokens as step by step (its first step is run twice before it is captured)."""
    folder = make_folder(tmp_path, "tiny_e", seed=2, dtype="bfloat16")
    from burn_lm_b200 import StepEntry
    eng = engine(folder, cache="int8", weights="int4")
    prompts = [random_tokens(7, 60, 640), random_tokens(8, 120, 640)]
    runs = []
    for device_side in (True, False):
        slots = [eng.acquire() for _ in prompts]
        logits = eng.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)])
        tokens = logits.argmax(dim=1).tolist()
        if device_side:
            runs.append(eng.decode_run(slots, tokens, 12).tolist())
        else:
            got = []
            for _ in range(12):
                tokens = eng.step([StepEntry(s, [t], [0]) for s, t in zip(slots, tokens)]).argmax(dim=1).tolist()
                got.append(tokens)
            runs.append(got)
        for s in slots:
            eng.release(s)
    assert runs[0] == runs[1]
    eng.verify()


def test_a_windowed_model_in_8_bits(tmp_path):
    """Attention over a window of 70 keys: pages before it go back and are used again, by another sequence."""
    import dataclasses
    from burn_lm_b200 import Engine, StepEntry
    from burn_lm_b200.model import Model, make_runtime, plan_of
    from burn_lm_b200.weights.loader import load_tensors
    folder = make_folder(tmp_path, "tiny_d", seed=5, dtype="bfloat16")
    cfg, tensors = plain.read_model_folder(folder)
    results = []
    for cache in ("compute", "int8"):
        _, typed, plan = plan_of(cfg)
        layers = []
        for lp in plan.layers:
            parts = [dataclasses.replace(p, plan=dataclasses.replace(p.plan, spec=dataclasses.replace(p.plan.spec, window=70))) if p.name == "mixer" else p
                     for p in lp.parts]
            layers.append(dataclasses.replace(lp, parts=type(lp.parts)(parts)))
        plan = dataclasses.replace(plan, layers=type(plan.layers)(layers))
        m = Model(plan, make_runtime("bfloat16", "cuda", cache), typed)
        m.bind(load_tensors(folder, m.tensor_specs(), torch.bfloat16, torch.device("cuda"), plan.ignorable_tensors, plan.duplicate_tensors))
        eng = Engine(m, max_tokens=64 * 8, max_seqs=2)
        tokens = random_tokens(3, 400, cfg["vocab_size"])
        slot, out = eng.acquire(), []
        for at in range(0, 400, 50):
            if at == 200:
                other = eng.acquire()
                eng.step([StepEntry(other, random_tokens(9, 100, cfg["vocab_size"]), [0])])
                eng.release(other)
            out.append(eng.step([StepEntry(slot, tokens[at: at + 50], list(range(50)))]).float().cpu().numpy().copy())
        eng.verify()
        results.append(np.concatenate(out))
    assert row_error(results[1], results[0]).max() < 6e-2


def test_command_line_and_replay(tmp_path):
    folder = make_folder(tmp_path, "tiny_d", seed=1, dtype="bfloat16")
    run = lambda *a, **k: subprocess.run([sys.executable, *a], cwd=ROOT, capture_output=True, text=True, timeout=300, **k)
    r = run(os.path.join("bin", "burn-lm"), "run", folder, "--cache", "int8", "--weights", "int4", "--sample-len", "5", "--no-stats", "5 17 3")
    assert r.returncode == 0 and len(r.stdout.split()) >= 1, r.stderr
    steps = '{"step": 0, "entries": [{"id": "a", "tokens": [5, 17, 3, 9], "want": [3]}], "end": []}\n'
    out = str(tmp_path / "o")
    r = run(os.path.join("bin", "trace_run"), "--model", folder, "--dtype", "bfloat16", "--out", out, "--max-tokens", "64", "--cache", "int8", "--weights",
            "int4", input=steps)
    assert r.returncode == 0 and "done 0" in r.stdout, r.stderr
    cfg, tensors = plain.read_model_folder(folder)
    got = np.fromfile(os.path.join(out, "0.f32"), dtype="<f4")[None]
    assert row_error(got, forward(cfg, in_four_bits(tensors), [5, 17, 3, 9], torch.bfloat16)[-1:]).max() < 4e-2
