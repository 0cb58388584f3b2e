"""Log probabilities through the engine, against the log softmax in 64 bits of the engine's own logits of the whole text.

Two cuts of a request give logits that agree to 1e-4 of the largest in float32 (20 float32 sums of a few hundred terms one behind
another, 2^-24 each, with room).  A difference d of the logits moves a log probability by 2 d at most; beside that stands the operator's
own error, below 1e-5 at these sizes."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def log_softmax(z):
    z = torch.from_numpy(np.asarray(z, dtype=np.float64))
    return torch.log_softmax(z, dim=-1).numpy()


def engine_of(folder, page, **more):
    from slipstream_b200 import LLM

    options = dict(dtype="float32", block_size=page, num_gpu_blocks=256, max_num_seqs=8)
    return LLM(folder, **{**options, **more})


def logits_of(llm, ids):
    """The engine's own logits of every place (a runner of the same model, whole)."""
    from slipstream_b200.engine.runner import StepEntry

    runner = llm.engine.runner
    out = runner.step([StepEntry("whole", ids, list(range(len(ids))))]).cpu().numpy()
    runner.release("whole")
    return out


def check(told, rows, tokens, n):
    """``told`` against rows of logits: each row's distribution, of which the token is one.  The engine's logits of two cuts of a
    request agree to 1e-4 of the largest in float32."""
    assert len(told) == len(rows) == len(tokens)
    if not len(rows):  # (a prompt of one token)
        return
    lp = log_softmax(rows)
    off = 2e-4 * np.abs(rows).max() + 1e-5
    for t, row, z, token in zip(told, lp, rows, tokens):
        assert t.token_id == token and abs(t.logprob - row[token]) <= off
        p = np.exp(row)
        assert abs(t.entropy + (p * row).sum()) <= off * (1 + np.abs(row).max())
        # ranks and alternatives, but for logits that stand nearer to one another than they are known
        slack = 1e-4 * np.abs(rows).max()
        assert (z > z[token] + slack).sum() + 1 <= t.rank <= (z >= z[token] - slack).sum()
        assert len(t.alternatives) == n
        for place, (token_id, logprob) in enumerate(t.alternatives):
            assert abs(logprob - row[token_id]) <= off and z[token_id] >= np.sort(z)[::-1][place] - slack


def prompts_of(config, lengths, seed=900):
    return [[int(t) for t in torch.randint(0, config.vocab_size, (n,), generator=torch.Generator().manual_seed(seed + i))] for i, n in enumerate(lengths)]


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("chunk", [256, 7])
def test_of_prompts_and_outputs(model_folders, name, chunk):
    """Several requests with different wishes in one batch, whole and in portions; their tokens are those without any wish."""
    from slipstream_b200 import SamplingParams

    folder, config, page = model_folders[name]
    llm = engine_of(folder, page, prefill_chunk_size=chunk)
    prompts = prompts_of(config, (1, 2, 9, 30, 41))
    wishes = [(2, 0), (None, 3), (0, None), (None, None), (5, 5)]
    params = [SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True, logprobs=a, prompt_logprobs=b) for a, b in wishes]
    outs = llm.generate(prompt_token_ids=prompts, sampling_params=params)
    without = llm.generate(prompt_token_ids=prompts, sampling_params=SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True))
    for out, plain_out, (a, b), ids in zip(outs, without, wishes, prompts):
        assert out.output_token_ids == plain_out.output_token_ids and plain_out.logprobs is None and plain_out.prompt_logprobs is None
        whole = ids + out.output_token_ids
        rows = logits_of(llm, whole)
        assert (out.logprobs is None) == (a is None) and (out.prompt_logprobs is None) == (b is None)
        if a is not None:
            assert len(out.logprobs) == 6
            check(out.logprobs, rows[len(ids) - 1:-1], out.output_token_ids, a)
        if b is not None:
            assert out.prompt_logprobs[0] is None and len(out.prompt_logprobs) == len(ids)
            check(out.prompt_logprobs[1:], rows[: len(ids) - 1], ids[1:], b)


def test_behind_the_host_and_ahead_of_it(model_folders):
    """Steps that run ahead of the host tell the same as steps that do not, sampled tokens too; a stop token ends both lists alike."""
    from slipstream_b200 import SamplingParams

    folder, config, page = model_folders["A"]
    prompts = prompts_of(config, (12, 20, 5))
    results = []
    for ahead in (True, False):
        llm = engine_of(folder, page)
        llm.engine.run_ahead = ahead
        params = [SamplingParams(max_tokens=20, temperature=0.9, seed=3 + i, ignore_eos=True, logprobs=4, stop_token_ids=tuple(range(0, 40, 4))) for i in range(3)]
        results.append(llm.generate(prompt_token_ids=prompts, sampling_params=params))
    for a, b in zip(*results):
        assert a.output_token_ids == b.output_token_ids and len(a.logprobs) == len(a.output_token_ids) == len(b.logprobs)
        assert [t.token_id for t in a.logprobs] == a.output_token_ids
        for x, y in zip(a.logprobs, b.logprobs):
            assert abs(x.logprob - y.logprob) <= 1e-3 and x.rank == y.rank


def test_after_a_preemption(model_folders):
    """A pool so small that requests are preempted and replayed: every token is told of once."""
    from slipstream_b200 import SamplingParams

    folder, config, page = model_folders["A"]
    prompts = prompts_of(config, (30, 30, 30, 30))
    params = SamplingParams(max_tokens=24, temperature=0.0, ignore_eos=True, logprobs=1, prompt_logprobs=1)
    small = engine_of(folder, page, num_gpu_blocks=120 // page, max_num_seqs=4, prefill_chunk_size=8)
    outs = small.generate(prompt_token_ids=prompts, sampling_params=params)
    assert small.engine.scheduler.preemptions > 0
    big = engine_of(folder, page)
    for out, ids in zip(outs, prompts):
        assert len(out.logprobs) == len(out.output_token_ids) == 24 and len(out.prompt_logprobs) == 30
        rows = logits_of(big, ids + out.output_token_ids)
        check(out.prompt_logprobs[1:], rows[:29], ids[1:], 1)
        check(out.logprobs, rows[29:-1], out.output_token_ids, 1)


def test_wishes_that_are_refused(model_folders):
    from slipstream_b200 import SamplingParams

    for bad in (-1, 65):
        with pytest.raises(ValueError, match="logprobs"):
            SamplingParams(logprobs=bad)
        with pytest.raises(ValueError, match="prompt_logprobs"):
            SamplingParams(prompt_logprobs=bad)
    from slipstream_b200 import ops
    from slipstream_b200.config.sampling_params import MAX_TOP_LOGPROBS

    assert ops.MAX_TOP_LOGPROBS == MAX_TOP_LOGPROBS
