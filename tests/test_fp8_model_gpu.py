"""The 8-bit operators together, as the engine runs them: every call that a generation makes is checked against its plain form on the
call's own data, and a folder that holds 8-bit weights gives what the same weights quantised as they are loaded give."""

from __future__ import annotations

import json
import os

import pytest
import torch
from safetensors.torch import load_file, save_file

import plain_fp8 as pf
from conftest import TINY_PAGE, random_ids
from plain_fp8 import EPS32, FP8, groups

pytestmark = pytest.mark.gpu


def engine(folder, dtype, name="F", **kw):
    from acvram_b200 import Engine
    args = dict(max_batch_size=4, max_model_len=256, page_size=TINY_PAGE[name], num_pages=64, token_budget=64)
    args.update(kw)
    return Engine(folder, dtype, **args)


def generate(eng, prompts, n=8, **kw):
    from acvram_b200 import SamplingParams
    return eng.generate_batch(prompts, SamplingParams(temperature=0.0, max_tokens=n, ignore_eos=True, **kw))


def prompts_of(eng, lengths=(5, 17, 33)):
    return [random_ids(eng.model.plan.vocab_size, n, 100 + n) for n in lengths]


def near(off, bound, what):
    off, bound = off.double(), bound.double()
    assert bool((off <= bound).all()), (what, float((off / bound).max()))


def checked(ops, counts):
    """The four operators with a check of what each call gave."""
    def quantize(x, values, scales, block_rows=1):
        out = ops["quantize_fp8"](x, values, scales, block_rows)
        q, s = pf.quantize(x.cpu().float(), block_rows)
        assert torch.equal(scales.cpu(), s) and torch.equal(values.cpu().float(), q.float())
        counts["quantize"] += 1
        return out

    def linear(x, xs, w, ws, out, static_weights=False):
        ops["linear_fp8"](x, xs, w, ws, out, static_weights)
        assert static_weights
        y, error = pf.product(x.cpu(), xs.cpu(), w.cpu(), ws.cpu())
        near((out.cpu().double() - y).abs(), error + pf.half_step(y.abs() + error, out.dtype), "product")
        counts["linear"] += 1
        return out

    def gated(x, xs, g, gs, u, us, out, so, static_weights=False):
        ops["linear_fp8_swiglu"](x, xs, g, gs, u, us, out, so, static_weights)
        assert static_weights
        yg, eg = pf.product(x.cpu(), xs.cpu(), g.cpu(), gs.cpu())
        yu, eu = pf.product(x.cpu(), xs.cpu(), u.cpu(), us.cpu())
        h = yg * torch.sigmoid(yg) * yu
        error = 1.1 * eg * (yu.abs() + eu) + (yg * torch.sigmoid(yg)).abs() * eu + h.abs() * 16 * EPS32
        near((pf.values(out, so, 1) - h).abs(), pf.quantized_error(h, so, error), "gated product")
        counts["gated"] += 1
        return out, so

    def norms(x, delta, out, scales=None, *, residual_scale=1.0, weight=None, eps=0.0, static_weights=False):
        assert static_weights
        before, d = x.cpu().double(), None if delta is None else delta.cpu().double()
        ops["add_gated_norms"](x, delta, out, scales, residual_scale=residual_scale, weight=weight, eps=eps, static_weights=static_weights)
        kept = x.cpu().double()
        want = before if d is None else before + residual_scale * d
        near((kept - want).abs(), want.abs() * 2 * EPS32 + pf.half_step(want * (1 + EPS32), x.dtype), "stream")
        h = kept / torch.sqrt(kept.square().mean(1, keepdim=True) + eps) * weight.cpu().double()
        near((pf.values(out, scales, 1) - h).abs(), pf.quantized_error(h, scales, h.abs() * 50 * EPS32), "norm")
        counts["norms"] += 1
        return out

    return {"quantize_fp8": quantize, "linear_fp8": linear, "linear_fp8_swiglu": gated, "add_gated_norms": norms}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["D", "E", "F"])
def test_every_call_of_a_generation_is_the_operators(tiny_folders, monkeypatch, name, dtype):
    """Prompts of several lengths and decoding, without graphs; heads whose projections stack (F) and do not (D, E), a width of 100 (E)."""
    from acvram_b200.kernels import ops
    eng = engine(tiny_folders[name], dtype, name, enable_cuda_graphs=False, weights="fp8")
    counts = dict.fromkeys(("quantize", "linear", "gated", "norms"), 0)
    names = ("quantize_fp8", "linear_fp8", "linear_fp8_swiglu", "add_gated_norms")
    for n, f in checked({n: getattr(ops, n) for n in names}, counts).items():
        monkeypatch.setattr(ops, n, f)
    out = generate(eng, prompts_of(eng), 4)
    assert all(len(o) == 4 for o in out)
    layers = len(eng.model.blocks)
    steps = counts["gated"] // layers
    assert steps >= 4 and counts["gated"] == steps * layers and counts["norms"] == 2 * steps * layers
    assert counts["quantize"] == steps * layers
    assert counts["linear"] == steps * layers * (2 + len(eng.model.blocks[0].mixer.qkv.matrices))


@pytest.mark.parametrize("name", ["E", "F"])
def test_weights_stored_in_8_bits(tiny_folders, tmp_path, name):
    tensors = load_file(os.path.join(tiny_folders[name], "model.safetensors"))
    stored = {}
    for key, t in tensors.items():
        if key.endswith("_proj.weight"):
            stored[key], stored[key + "_scale_inv"] = pf.quantize(t.float(), 128)
        else:
            stored[key] = t
    save_file({k: v.contiguous() for k, v in stored.items()}, str(tmp_path / "model.safetensors"), metadata={"format": "pt"})
    cfg = json.load(open(os.path.join(tiny_folders[name], "config.json")))
    cfg["quantization_config"] = {"quant_method": "fp8", "fmt": "e4m3", "activation_scheme": "dynamic", "weight_block_size": [128, 128]}
    (tmp_path / "config.json").write_text(json.dumps(cfg))
    a, b = engine(str(tmp_path), "float32", name), engine(tiny_folders[name], "float32", name, weights="fp8")
    assert a.config == b.config and a.config.weights_fp8
    for x, y in zip(a.model.blocks, b.model.blocks):
        for p, q in zip(x.mixer.qkv.matrices + x.feed_forward.down.matrices, y.mixer.qkv.matrices + y.feed_forward.down.matrices):
            assert torch.equal(p[0].view(torch.uint8), q[0].view(torch.uint8)) and torch.equal(p[1], q[1])
    prompts = prompts_of(a)
    assert generate(a, prompts) == generate(b, prompts)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_give_the_same_tokens(tiny_folders, dtype):
    plain = engine(tiny_folders["F"], dtype, enable_cuda_graphs=False, weights="fp8")
    graphs = engine(tiny_folders["F"], dtype, weights="fp8")
    prompts = prompts_of(plain)
    assert generate(plain, prompts, 24) == generate(graphs, prompts, 24)


def test_logits_are_near_those_of_more_bits(tiny_folders):
    """Weights and activations are rounded to four bits of significand, each value off by at most 2^-4 of itself and by a third of that in
    the root of the mean square (an error spread evenly over a step): a sum of many of each is off by 2^-4 / sqrt(3) * sqrt(2), 5 % of its
    size, and two layers of several such sums stay under four times that."""
    from acvram_b200 import SamplingParams
    rows = []
    for weights in (None, "fp8"):
        eng = engine(tiny_folders["F"], "float32", weights=weights)
        got = []
        forward = eng.model.forward
        eng.model.forward = lambda ctx, storage: got.append(forward(ctx, storage)) or got[-1]
        eng.generate_batch([random_ids(eng.model.plan.vocab_size, 40, 7)], SamplingParams(temperature=0.0, max_tokens=1, ignore_eos=True))
        rows.append(got[0].double())
    assert float((rows[1] - rows[0]).norm() / rows[0].norm()) < 0.2


def test_random_weights_and_their_bytes(tiny_folders):
    from conftest import tiny_config
    eng = engine(tiny_config("F"), "bfloat16", random_weights=True, seed=5, weights="fp8")
    cfg = eng.config
    assert cfg.weights_fp8
    matrices = cfg.hidden_size * (cfg.q_size + 2 * cfg.kv_size) + cfg.q_size * cfg.hidden_size + 3 * cfg.hidden_size * cfg.intermediate_size
    block = eng.model.blocks[0]
    assert matrices < block.mixer.weight_bytes() + block.feed_forward.weight_bytes() < 1.05 * matrices
    assert generate(eng, prompts_of(eng), 4) == generate(engine(tiny_folders["F"], "bfloat16", weights="fp8"), prompts_of(eng), 4)
