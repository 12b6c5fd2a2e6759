"""The engine with weights in 8 bits and the cache in 4: the whole path against a plain float64 model that rounds weights, activations, keys and
values by the formats' rules, prompts against tokens one by one, batches, windows, generation, the guard words.

Tolerance.  Rounding is a step: where the engine's bfloat16 activations and the plain model's float64 differ by 2^-9, a few per cent of the codes land one
step away, and how far that moves the logits depends on the model.  So each test lets the plain model say it: the same plain model is run with its
activations rounded to bfloat16 at the engine's places, and the engine may be twice as far from the float64 one as that is (two paths that
round in other orders), and 0.02 more, in the 2-norm over all logits.  A wrong mask, position, page or scale shows as 0.5 and above."""
import numpy as np
import pytest
import torch

import plain_llama
from helpers import random_requests, run_trace, tail_trace, whole_trace, batched_trace
from plain_lowbit import product8, rounded4

pytestmark = pytest.mark.gpu


def config(name):
    from exl3_server_b200 import LlamaConfig
    if name == "64":
        return LlamaConfig(hidden_size=144, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=208,
                           vocab_size=301, tie_word_embeddings=True, rope_theta=100000.0, rms_norm_eps=1e-5, scale_emb=2.0, scale_depth=1.0,
                           dim_model_base=72, max_position_embeddings=4096, sliding_window=80, layer_types=["full_attention", "sliding_attention"])
    return LlamaConfig(hidden_size=208, num_hidden_layers=2, num_attention_heads=6, num_key_value_heads=2, head_dim=128, intermediate_size=272,
                       vocab_size=331, tie_word_embeddings=False, rope_theta=500000.0, rms_norm_eps=2e-5, max_position_embeddings=4096)


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    from exl3_server_b200 import write_random_model
    root = tmp_path_factory.mktemp("lowbit")
    return {n: write_random_model(config(n), str(root / n), seed=77, std=0.08, norm_std=0.1, dtype=torch.bfloat16) for n in ("64", "128")}


def off(a, b):
    return float(np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b))


class Plain:
    """The plain model's logits, and how far an engine may be from them."""

    def __init__(self, folder, ids, weights, cache):
        self.logits = plain_logits(folder, ids, weights, cache)
        self.bound = 0.02 + 2 * off(plain_logits(folder, ids, weights, cache, True), self.logits)
        assert self.bound < 0.35, "the bound has to stay below what a fault shows"

    def check(self, got, rows=slice(None)):
        assert off(got, self.logits[rows]) <= self.bound, (off(got, self.logits[rows]), self.bound)


def plain_logits(folder, ids, weights, cache, narrow=False):
    """plain_llama with the formats' rounding put where the engine has it: the fused matrices as the engine fuses them.  ``narrow``: activations
    rounded to bfloat16 where the engine keeps them so."""
    n16 = (lambda x: x.bfloat16().double()) if narrow else (lambda x: x)
    from exl3_server_b200.ops import kernels as K
    m = plain_llama.PlainModel(folder)
    fused = {}

    def linear8(x, key, parts):
        if key not in fused:
            fused[key] = K.fp8_quantize_weight(torch.cat([m.w[p] for p in parts]).bfloat16())
        return product8(x.bfloat16(), *fused[key])

    def layer(h, w, i, c):
        p = f"model.layers.{i}."
        a, f, L, d = p + "self_attn.", p + "mlp.", h.shape[0], c["head_dim"]
        r = n16(plain_llama.rms_norm(h, w[p + "input_layernorm.weight"], c["eps"]))
        names = [a + n + "_proj.weight" for n in "qkv"]
        qkv = linear8(r, a, names) if weights else torch.cat([r @ w[n].T for n in names], 1)
        q, k, v = n16(qkv).split([w[n].shape[0] for n in names], dim=1)
        q, k, v = (x.reshape(L, -1, d).transpose(0, 1) for x in (q, k, v))
        pos = torch.arange(L)
        q, k = plain_llama.rope(q, pos, c["theta"]), plain_llama.rope(k, pos, c["theta"])
        if cache:
            k, v = rounded4(k), rounded4(v)
        o = n16(plain_llama.attention(n16(q), k, v, c["windows"][i]).transpose(0, 1).reshape(L, -1))
        h = h + n16(linear8(o, a + "o", [a + "o_proj.weight"]) if weights else o @ w[a + "o_proj.weight"].T) * c["rho"]
        r = n16(plain_llama.rms_norm(h, w[p + "post_attention_layernorm.weight"], c["eps"]))
        if weights:
            if f not in fused:
                g, u = w[f + "gate_proj.weight"], w[f + "up_proj.weight"]
                n = g.shape[0] // 8
                fused[f] = K.fp8_quantize_weight(torch.stack([g.view(n, 8, -1), u.view(n, 8, -1)], 1).reshape(2 * g.shape[0], -1).bfloat16())
            y = linear8(n16(product8(r.bfloat16(), *fused[f], gated=True)), f + "d", [f + "down_proj.weight"])
        else:
            y = plain_llama.swiglu(r, *(w[f + n + "_proj.weight"] for n in ("gate", "up", "down")))
        return h + n16(y) * c["rho"]

    keep, plain_llama.layer = plain_llama.layer, layer
    try:
        return m.logits(ids).numpy()
    finally:
        plain_llama.layer = keep


def engine(folder, weights, cache, max_tokens=4096):
    from exl3_server_b200 import Engine
    return Engine.from_folder(folder, dtype="bfloat16", max_tokens=max_tokens, weight_type="fp8" if weights else None, cache_type="int4" if cache else None)


@pytest.mark.parametrize("name", ["64", "128"])
@pytest.mark.parametrize("weights,cache", [(True, False), (False, True), (True, True)])
def test_prompts_and_single_tokens(folders, name, weights, cache):
    toks = random_requests(301, [230], seed=5)["r0"]
    want = Plain(folders[name], toks, weights, cache)
    eng = engine(folders[name], weights, cache)
    whole = run_trace(eng, whole_trace({"r0": toks}))["r0"]
    tail = run_trace(eng, tail_trace({"r0": toks}, tail=90))["r0"]
    want.check(whole)
    want.check(tail)
    eng.check_kernels()


@pytest.mark.parametrize("name", ["64", "128"])
def test_batches(folders, name):
    reqs = random_requests(301, [3, 70, 129, 40, 1], seed=6)
    want = {r: Plain(folders[name], t, True, True) for r, t in reqs.items()}
    eng = engine(folders[name], True, True)
    got = run_trace(eng, batched_trace(reqs, [["r0", "r1", "r2"], ["r3", "r4"]], {"r0": 1, "r1": 33, "r2": 100, "r3": 40, "r4": 1}))
    for r in reqs:
        want[r].check(got[r])
    eng.check_kernels()


def test_prompts_cut_into_steps_and_taken_back(folders):
    """A prompt in portions; a sequence rewound into the middle of a page and gone on with."""
    from exl3_server_b200 import StepEntry
    toks = random_requests(301, [300], seed=7)["r0"]
    want = Plain(folders["128"], toks, True, True)
    eng = engine(folders["128"], True, True)
    slot, got, at = eng.open(), [], 0
    for n in (7, 1, 130, 2, 60, 100):
        got.append(eng.step([StepEntry(slot, toks[at:at + n], "all")]).float().cpu().numpy())
        at += n
    want.check(np.concatenate(got))
    eng.truncate(slot, 203)
    again = eng.step([StepEntry(slot, toks[203:260], "all")]).float().cpu().numpy()
    want.check(again, slice(203, 260))
    eng.close(slot)
    eng.cache.check()
    eng.check_kernels()


def test_generation_and_bytes(folders):
    from exl3_server_b200 import Engine, GenerateOptions
    eng = engine(folders["64"], True, True)
    full = Engine.from_folder(folders["64"], dtype="bfloat16", max_tokens=4096)
    res = eng.generate([[5, 9, 17, 200], [3] * 90, [1]], GenerateOptions(max_tokens=70, ignore_eos=True))
    assert [len(r.tokens) for r in res] == [70, 70, 70] and all(0 <= t < 301 for r in res for t in r.tokens)
    alone = eng.generate([[3] * 90], GenerateOptions(max_tokens=70, ignore_eos=True))
    assert len(alone[0].tokens) == 70
    g4, g16 = eng.cache.groups[0], full.cache.groups[0]
    assert g4.k.dtype == torch.uint8 and g4.bytes_per_token(2) * 16 == g16.bytes_per_token(2) * 5
    assert g4.k.numel() * 16 == (g16.k.numel() + g16.v.numel()) * 2 * 5
    assert eng.model.weight_bytes() < 0.62 * full.model.weight_bytes() + eng.model.head.read_bytes()
    assert abs(eng._body_params - full._body_params) <= 0.01 * full._body_params
    eng.check_kernels()
    eng.cache.groups[0]._k_store[3] = 7                                  # a write before the pool
    with pytest.raises(Exception):
        eng.cache.check_guards()


def test_command_line(folders, capsys):
    from exl3_server_b200.cli import main
    assert main(["--model", folders["64"], "-p", "1,15,27", "--max-tokens", "8", "--ignore-eos", "--weight-type", "fp8", "--cache-type", "int4", "--quiet"]) == 0
    assert len(capsys.readouterr().out.strip().split(",")) == 8
