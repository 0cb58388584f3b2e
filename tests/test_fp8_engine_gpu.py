"""Layers in 8-bit floats through the engine: the same steps against a plain 64-bit decoder that rounds where the layers do.

Both sides round the same values, but not to the last bit of the same float32 numbers: once in some 10^5 elements a value stands so
near the middle between two steps that they land on different ones, and that row, and what attends to it, is off by what one step of
one element makes (an eighth of the element at most, of 64 and more that a sum has).  Rows without such an element agree as the float32
engine's do (2e-5 of the largest logit in its own tests, where a plain layer has as many operations).  So in float32 the median row is
held to 1e-4, and every row to 0.2, which a wrong scale or another row's values pass at once; and the median error has to be a tenth
at most of what the rounding itself makes.  In bfloat16 the activations in front of every rounding carry bfloat16's own error, 2^-9
and more of a value, and where that moves a value over the middle between two steps (about 3 % of them, each by 2^-3) the product's
terms differ: 2 % of a term on average, and as much of a sum of such terms with either sign; eight projections in a row make 6 %, and of
the largest logit, four times a typical one, the largest difference of a row is about as much.  Twice that, 0.12, is allowed to the
median row, and 0.4 to all."""

import contextlib
import io
import json

import numpy as np
import pytest
import torch

import plain_qwen2 as plain
import replay_plans as plans
from test_int8_engine_gpu import errors, run_plan, tokens_of

pytestmark = pytest.mark.gpu


def rounded(v, rows=1):
    """v with each block of ``rows`` x 128 as what its 8-bit values stand for, the steps found in float32, as the operator defines them."""
    n, k = v.shape[-2], v.shape[-1]
    padded = v.new_zeros(-(-n // rows) * rows, -(-k // 128) * 128)
    padded[:n, :k] = v
    tiles = padded.reshape(-1, rows, padded.shape[1] // 128, 128)
    t32 = tiles.to(torch.float32)
    top = t32.abs().amax(dim=(1, 3), keepdim=True)
    inverse = torch.where(top > 0, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
    q = (t32 * inverse).to(torch.float8_e4m3fn).to(torch.float64)
    return (q * (tiles.abs().amax(dim=(1, 3), keepdim=True) / 448)).reshape(padded.shape)[:n, :k]


def plain_logits(folder, requests, dtype, fp8=True):
    config, weights = plain.read_model_folder(folder, torch.float64)
    if dtype == "bfloat16":
        weights = {k: v.to(torch.bfloat16).to(torch.float64) if v.dim() == 2 else v for k, v in weights.items()}
    s = plain.sizes(config)
    r = rounded if fp8 else (lambda v: v)
    if fp8:
        for i in range(s["layers"]):
            names = [f"model.layers.{i}.self_attn.{p}_proj.weight" for p in "qkv"]
            stacked = rounded(torch.cat([weights[n] for n in names]), 128)  # (one matrix, whose blocks do not end where q, k and v do)
            for n, part in zip(names, stacked.split([weights[n].shape[0] for n in names])):
                weights[n] = part
            for n in (f"model.layers.{i}.{p}.weight" for p in ("self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")):
                weights[n] = rounded(weights[n], 128)

    def linear(x, name):
        y = r(x) @ weights[f"{name}.weight"].T
        bias = weights.get(f"{name}.bias")
        return y if bias is None else y + bias

    def logits(ids):
        n = len(ids)
        x = weights["model.embed_tokens.weight"][torch.tensor(ids)]
        cos, sin = plain.rotary_tables(torch.arange(n), s["head_dim"], s["theta"], torch.float64)
        for i in range(s["layers"]):
            at = f"model.layers.{i}"
            h = plain.rms_norm(x, weights[f"{at}.input_layernorm.weight"], s["eps"])
            q, k, v = (linear(h, f"{at}.self_attn.{p}_proj").view(n, -1, s["head_dim"]) for p in "qkv")
            q, k = plain.apply_rotary(q, cos, sin), plain.apply_rotary(k, cos, sin)
            x = x + linear(plain.causal_attention(q, k, v, s["head_dim"] ** -0.5), f"{at}.self_attn.o_proj")
            h = plain.rms_norm(x, weights[f"{at}.post_attention_layernorm.weight"], s["eps"])
            gate = linear(h, f"{at}.mlp.gate_proj")
            x = x + linear(gate * torch.sigmoid(gate) * linear(h, f"{at}.mlp.up_proj"), f"{at}.mlp.down_proj")
        x = plain.rms_norm(x, weights["model.norm.weight"], s["eps"])
        return (x @ weights.get("lm_head.weight", weights["model.embed_tokens.weight"]).T).numpy()
    return {rid: logits(ids) for rid, ids in requests.items()}


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_logits_are_those_of_the_plain_decoder_that_rounds_alike(model_folders, name, dtype):
    from slipstream_b200.engine.runner import ModelRunner

    folder, config, page = model_folders[name]
    requests = tokens_of(config)
    want = plain_logits(folder, requests, dtype)
    made = np.median(errors({k: list(v) for k, v in plain_logits(folder, requests, dtype, fp8=False).items()}, want))
    runner = ModelRunner(folder, dtype=dtype, page_size=page, num_pages=256 // page, max_num_seqs=4, quantization="fp8")
    for what, steps in (("whole", plans.whole(requests)), ("tail one by one", plans.tail_one_by_one(requests)),
                        ("changing portions", plans.changing_portions(requests)), ("mixed", plans.mixed(requests, 256, page, seed=5))):
        err = errors(plans.collect(steps, run_plan(runner, steps)), want)
        assert np.median(err) <= (1e-4 if dtype == "float32" else 0.12), (what, np.median(err))
        assert err.max() <= (0.2 if dtype == "float32" else 0.4), (what, err.max())
        if dtype == "float32":
            assert np.median(err) <= 0.1 * made, (what, np.median(err), made)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_steps_replayed_from_graphs(model_folders, dtype):
    """Decode steps and steps with prompt portions, captured (padded to their buckets) and kernel by kernel, with the same plans."""
    from slipstream_b200.engine.runner import ModelRunner

    folder, config, page = model_folders["B"]
    requests = tokens_of(config)
    results = []
    for captured in (False, True):
        runner = ModelRunner(folder, dtype=dtype, page_size=page, num_pages=256 // page, max_num_seqs=4, quantization="fp8", use_cuda_graphs=captured)
        runner.mixed_graph_after = 0
        steps = plans.tail_one_by_one(requests)
        results.append(plans.collect(steps, run_plan(runner, steps)))
        assert bool(runner._graphs) == captured
    for rid in requests:
        a, b = (np.stack(r[rid]) for r in results)
        # (a captured step is padded to its bucket, whose number of tokens may have another plan: K in other slices adds in another order)
        assert np.abs(a - b).max() <= 0.2 * np.abs(a).max() and np.median(np.abs(a - b).max(axis=1)) <= (1e-4 if dtype == "float32" else 0.12) * np.abs(a).max()


def test_generation_through_the_engine(model_folders):
    """Greedy tokens of several requests, twice, and through the command line with their log probabilities."""
    from slipstream_b200 import LLM, SamplingParams
    from slipstream_b200.entrypoints.cli import main

    folder, config, page = model_folders["A"]
    prompts = [ids[:20 + 3 * i] for i, ids in enumerate(tokens_of(config).values()) if len(ids) > 40]
    params = SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True, logprobs=2, prompt_logprobs=0)
    llm = LLM(folder, dtype="bfloat16", block_size=page, num_gpu_blocks=128, max_num_seqs=8, quantization="fp8")
    first = llm.generate(prompt_token_ids=prompts, sampling_params=params)
    assert all(len(o.output_token_ids) == len(o.logprobs) == 12 for o in first)
    again = llm.generate(prompt_token_ids=prompts, sampling_params=params)
    assert [o.output_token_ids for o in again] == [o.output_token_ids for o in first]
    alone = llm.generate(prompt_token_ids=[prompts[0]], sampling_params=params)[0]
    out = io.StringIO()
    with contextlib.redirect_stdout(out):
        assert main(["--model", folder, "--dtype", "bfloat16", "--quantization", "fp8", "--block-size", str(page), "--num-gpu-blocks", "128",
                     "--max-num-seqs", "8", "--prompt-ids", ",".join(map(str, prompts[0])), "--max-tokens", "12", "--temperature", "0",
                     "--ignore-eos", "--logprobs", "2", "--prompt-logprobs", "0"]) == 0
    line = json.loads(out.getvalue())
    assert line["output_token_ids"] == alone.output_token_ids
    assert [t["logprob"] for t in line["logprobs"]] == [t.logprob for t in alone.logprobs]
    assert line["prompt_logprobs"][0] is None and len(line["prompt_logprobs"]) == len(prompts[0])


def test_what_rounding_costs_is_told_by_log_probabilities(model_folders):
    """The same text under the float32 model and under its fp8 form: the mean log probability of its tokens differs by no more than the
    logits do (|log p - log p'| <= 2 max |z - z'| for any row)."""
    from slipstream_b200 import LLM, SamplingParams

    folder, config, page = model_folders["A"]
    text = tokens_of(config)["r2"]
    params = SamplingParams(max_tokens=1, temperature=0.0, prompt_logprobs=0)
    told = {}
    for quantization in (None, "fp8"):
        llm = LLM(folder, dtype="float32", block_size=page, num_gpu_blocks=128, max_num_seqs=4, quantization=quantization)
        told[quantization] = np.array([t.logprob for t in llm.generate(prompt_token_ids=[text], sampling_params=params)[0].prompt_logprobs[1:]])
    plainly = plain_logits(folder, {"t": text}, "float32", fp8=False)["t"], plain_logits(folder, {"t": text}, "float32")["t"]
    bound = 2 * np.abs(plainly[0] - plainly[1]).max(axis=1)[:-1]
    assert np.all(np.abs(told[None] - told["fp8"]) <= bound + 2e-2 * np.abs(plainly[0]).max())


def test_parts_refuse_what_they_cannot_run():
    from slipstream_b200 import ops
    from slipstream_b200.parts import Fp8RMSNorm, Fp8SwiGLUFeedForward, Runtime

    runtime = Runtime(torch.device("cuda:0"), torch.bfloat16)
    norm = Fp8RMSNorm("n", 32, 1e-6)
    norm.bind({"n.weight": torch.ones(32, device="cuda:0")}, runtime)
    stream = torch.randn(3, 32, device="cuda:0")
    assert isinstance(norm.add_norm(stream, None), ops.Fp8Rows)
    with pytest.raises(ValueError):
        norm.add_norm(stream, None, rows=torch.zeros(1, dtype=torch.int32, device="cuda:0"))
    with pytest.raises(ValueError):
        Fp8SwiGLUFeedForward("f", 32, 64, limit=7.0).bind({}, runtime)
