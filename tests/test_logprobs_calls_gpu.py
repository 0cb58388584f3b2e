"""Log probabilities by the engine's calls that return token ids."""

import pytest

from test_logprobs_engine_gpu import engine_of, prompts_of

pytestmark = pytest.mark.gpu


def test_generate_generate_batch_and_stream(model_folders):
    """They return tokens; what else the requests asked for is there as `LLM.generate` tells it."""
    from slipstream_b200 import Request, SamplingParams

    folder, config, page = model_folders["A"]
    llm = engine_of(folder, page)
    prompts = prompts_of(config, (12, 7, 20))
    wishes = [(2, None), (None, 1), (None, None)]
    params = [SamplingParams(max_tokens=5, temperature=0.0, ignore_eos=True, logprobs=a, prompt_logprobs=b) for a, b in wishes]
    told = llm.generate(prompt_token_ids=prompts, sampling_params=params)

    def same(got, want):
        assert (got is None) == (want is None)
        for a, b in zip(got or [], want or [], strict=True):
            assert (a is None) == (b is None)
            # (steps of other batches may sum in another order)
            assert a is None or (a.token_id == b.token_id and abs(a.logprob - b.logprob) < 1e-3 and len(a.alternatives) == len(b.alternatives))

    requests = [Request(f"r{i}", None, ids, p) for i, (ids, p) in enumerate(zip(prompts, params))]
    engine = llm.engine
    assert engine.generate_batch(requests) == [t.output_token_ids for t in told]
    for got, prompt_got, t in zip(engine.last_logprobs, engine.last_prompt_logprobs, told, strict=True):
        same(got, t.logprobs)
        same(prompt_got, t.prompt_logprobs)
    for request, t in zip(requests, told):
        assert engine.generate(request) == t.output_token_ids
        same(engine.last_logprobs[0], t.logprobs)
        same(engine.last_prompt_logprobs[0], t.prompt_logprobs)
        for i, token in enumerate(engine.stream(request)):
            assert token == t.output_token_ids[i]
            assert t.logprobs is None or len(engine.last_logprobs[0]) > i
        same(engine.last_logprobs[0], t.logprobs)
        same(engine.last_prompt_logprobs[0], t.prompt_logprobs)
