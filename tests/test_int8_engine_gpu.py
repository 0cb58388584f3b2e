"""Layers in 8 bits through the engine: the same steps against a plain 64-bit decoder that rounds where the layers do.

Both sides round the same values, but not to the last bit of the same float32 numbers: once in some 10^5 elements a value stands so
near the middle between two steps that they land on different ones, and that row, and what attends to it, is off by what one step of
one element makes.  Rows without such an element agree as the float32 engine's do (2e-5 of the largest logit in its own tests, where
a plain layer has as many operations).  So in float32 the median row is held to 1e-4, and every row to 0.1, which a wrong scale, a
missing rounding or another row's values pass at once; and the median error has to be a tenth at most of what the rounding itself
makes.  In bfloat16 the activations in front of every rounding carry bfloat16's own error (3e-2 of the largest logit in the
engine's tests without 8 bits), which moves many elements by a step (1 / 127 of the row's largest, against 2^-9 of the element): 6e-2
for the median row, 0.2 for all."""

import numpy as np
import pytest
import torch

import plain_qwen2 as plain
import replay_plans as plans

pytestmark = pytest.mark.gpu

LENGTHS = {"r0": 70, "r1": 45, "r2": 97, "r3": 33, "r4": 64, "r5": 21}


def tokens_of(config, lengths=LENGTHS):
    return {rid: [int(t) for t in torch.randint(0, config.vocab_size, (n,), generator=torch.Generator().manual_seed(300 + i))]
            for i, (rid, n) in enumerate(lengths.items())}


def rounded(v):
    """Rows of v as what their 8-bit values stand for.  The steps are found in float32, as the operator defines them: weights that
    are stored in bfloat16 have elements of exactly half their row's largest, which stand in the middle between two steps, and which
    of the two it is depends on the rounding of 127 / a."""
    v32 = v.to(torch.float32)
    top = v32.abs().amax(dim=-1, keepdim=True)
    steps = torch.where(top > 0, (v32 * (torch.full_like(top, 127.0) / top)).round(), torch.zeros_like(v32))
    return steps.to(torch.float64) * (v.abs().amax(dim=-1, keepdim=True) / 127)


def plain_logits(folder, requests, dtype, int8=True):
    config, weights = plain.read_model_folder(folder, torch.float64)
    if dtype == "bfloat16":
        weights = {k: v.to(torch.bfloat16).to(torch.float64) if v.dim() == 2 else v for k, v in weights.items()}
    s, r = plain.sizes(config), rounded if int8 else (lambda v: v)
    weights = {k: r(v) if "proj.weight" in k else v for k, v in weights.items()}

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


def run_plan(runner, steps):
    from slipstream_b200.engine.runner import StepEntry

    outs = []
    for step in steps:
        outs.append(runner.step([StepEntry(e["id"], e["tokens"], e["want"]) for e in step["entries"]]).cpu().numpy())
        for rid in step["end"]:
            runner.release(rid)
    runner.check()
    return outs


def errors(rows, want):
    """Of every row: its largest difference over the largest logit of its request."""
    return np.concatenate([np.abs(np.stack(rows[rid]) - ref).max(axis=1) / np.abs(ref).max() for rid, ref in want.items()])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_logits_are_those_of_the_plain_decoder_that_rounds_alike(model_folders, name, dtype):
    from slipstream_b200.engine.runner import ModelRunner

    folder, config, page = model_folders[name]
    requests = tokens_of(config)
    want = plain_logits(folder, requests, dtype)
    made = np.median(errors({k: list(v) for k, v in plain_logits(folder, requests, dtype, int8=False).items()}, want))
    runner = ModelRunner(folder, dtype=dtype, page_size=page, num_pages=256 // page, max_num_seqs=4, quantization="int8")
    plain_runner = ModelRunner(folder, dtype=dtype, page_size=page, num_pages=8, max_num_seqs=1)
    norms = sum(p.weight_bytes() for p in runner.model.parts() if "norm" in getattr(p, "name", ""))
    kept = runner.model.lm_head.weight_bytes() + norms
    assert runner.weight_bytes_per_step() - kept < 0.7 * (plain_runner.weight_bytes_per_step() - kept)
    for what, steps in (("whole", plans.whole(requests)), ("tail one by one", plans.tail_one_by_one(requests)),
                        ("changing portions", plans.changing_portions(requests)), ("mixed", plans.mixed(requests, 256, page, seed=5))):
        err = errors(plans.collect(steps, run_plan(runner, steps)), want)
        assert np.median(err) <= (1e-4 if dtype == "float32" else 6e-2), (what, np.median(err))
        assert err.max() <= (0.1 if dtype == "float32" else 0.2), (what, err.max())
        if dtype == "float32":
            assert np.median(err) <= 0.1 * made, (what, np.median(err), made)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_steps_replayed_from_graphs_give_the_same_bits(model_folders, dtype):
    """Decode steps and steps with prompt portions, captured (padded to their buckets) and kernel by kernel."""
    from slipstream_b200.engine.runner import ModelRunner

    folder, config, page = model_folders["B"]
    requests = tokens_of(config)
    results = []
    for captured in (False, True):
        runner = ModelRunner(folder, dtype=dtype, page_size=page, num_pages=256 // page, max_num_seqs=4, quantization="int8",
                             use_cuda_graphs=captured)
        runner.mixed_graph_after = 0
        assert runner.use_cuda_graphs == captured
        steps = plans.tail_one_by_one(requests)
        results.append(plans.collect(steps, run_plan(runner, steps)))
        steps = plans.mixed(requests, 256, page, seed=7)
        results[-1] = (results[-1], plans.collect(steps, run_plan(runner, steps)))
        assert bool(runner._graphs) == captured
    for a, b in zip(*results):
        for rid in requests:
            assert np.array_equal(np.stack(a[rid]), np.stack(b[rid])), rid


def test_generation_through_the_engine(model_folders):
    """Greedy tokens of several requests, together and alone, and those of the command line."""
    import contextlib
    import io
    import json

    from slipstream_b200 import LLM, SamplingParams
    from slipstream_b200.entrypoints.cli import main

    folder, config, page = model_folders["A"]
    prompts = [ids[:20 + 3 * i] for i, ids in enumerate(tokens_of(config).values()) if len(ids) > 40]
    params = SamplingParams(max_tokens=12, temperature=0.0, ignore_eos=True)
    llm = LLM(folder, dtype="bfloat16", block_size=page, num_gpu_blocks=128, max_num_seqs=8, quantization="int8")
    together = [o.output_token_ids for o in llm.generate(prompt_token_ids=prompts, sampling_params=params)]
    assert all(len(t) == 12 for t in together)
    alone = [llm.generate(prompt_token_ids=[p], sampling_params=params)[0].output_token_ids for p in prompts]
    again = [o.output_token_ids for o in llm.generate(prompt_token_ids=prompts, sampling_params=params)]
    assert again == together
    assert sum(a == b for a, b in zip(alone, together)) >= len(prompts) - 1  # (other attention kernels may break a near tie)
    out = io.StringIO()
    with contextlib.redirect_stdout(out):
        assert main(["--model", folder, "--dtype", "bfloat16", "--quantization", "int8", "--block-size", str(page), "--num-gpu-blocks", "128",
                     "--max-num-seqs", "8", "--prompt-ids", ",".join(map(str, prompts[0])), "--max-tokens", "12", "--temperature", "0",
                     "--ignore-eos"]) == 0
    assert json.loads(out.getvalue())["output_token_ids"] == alone[0]


def test_parts_refuse_what_they_cannot_run():
    from slipstream_b200 import ops
    from slipstream_b200.parts import Int8RMSNorm, Int8SwiGLUFeedForward, Runtime

    runtime = Runtime(torch.device("cuda:0"), torch.bfloat16)
    norm = Int8RMSNorm("n", 32, 1e-6)
    norm.bind({"n.weight": torch.ones(32, device="cuda:0")}, runtime)
    stream = torch.randn(3, 32, device="cuda:0")
    assert isinstance(norm.add_norm(stream, None), ops.Int8Rows)
    with pytest.raises(ValueError):
        norm.add_norm(stream, None, rows=torch.zeros(1, dtype=torch.int32, device="cuda:0"))
    with pytest.raises(ValueError):
        Int8SwiGLUFeedForward("f", 32, 64, limit=7.0).bind({}, runtime)
