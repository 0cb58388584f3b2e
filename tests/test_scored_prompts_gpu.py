"""Memory of steps that score prompts."""

import pytest
import torch

pytestmark = pytest.mark.gpu

VOCABULARY = 151936


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    from slipstream_b200.config.model_config import Qwen2Config
    from slipstream_b200.weights.random_init import write_random_model

    path = tmp_path_factory.mktemp("wide_vocabulary")
    write_random_model(Qwen2Config(vocab_size=VOCABULARY, hidden_size=64, num_hidden_layers=1, max_position_embeddings=512, torch_dtype="bfloat16",
                                   intermediate_size=128, num_attention_heads=2, num_key_value_heads=1, head_dim=32, rms_norm_eps=1e-6,
                                   rope_theta=10000.0, tie_word_embeddings=True), path, seed=4)
    return str(path)


def prompts():
    return [torch.randint(0, VOCABULARY, (250 + i,), generator=torch.Generator().manual_seed(i)).tolist() for i in range(32)]


def scored(llm):
    from slipstream_b200 import SamplingParams

    return llm.generate(prompt_token_ids=prompts(), sampling_params=SamplingParams(max_tokens=2, temperature=0.0, ignore_eos=True, logprobs=0, prompt_logprobs=1))


def test_logits_of_a_step_are_bounded(folder):
    """8,192 tokens of 32 prompts fit the budget of one step: their logits, 5 GB, are never there at once.  (1,024 scored rows and 32 rows
    that are sampled from, twice: 0.66 GB; what else a step of this model holds is far below 0.2 GB.)"""
    from slipstream_b200 import LLM

    llm = LLM(folder, dtype="bfloat16", num_gpu_blocks=1024, max_num_seqs=32, max_num_batched_tokens=8192, prefill_chunk_size=512, use_cuda_graphs=False)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    outs = scored(llm)
    assert torch.cuda.max_memory_allocated() - before < (1024 + 2 * 32) * VOCABULARY * 4 + 2 * 10 ** 8
    for out, ids in zip(outs, prompts()):
        assert [t.token_id for t in out.prompt_logprobs[1:]] == ids[1:] and len(out.logprobs) == 2


def test_logits_of_captured_steps_are_bounded(folder):
    """Captured steps with logits per token keep no more than they may all together; the others run kernel by kernel, with the same results."""
    from slipstream_b200 import LLM
    from slipstream_b200.engine.graphs import MixedGraph

    llm = LLM(folder, dtype="bfloat16", num_gpu_blocks=1024, max_num_seqs=32, prefill_chunk_size=64)
    runner = llm.engine.runner
    first = scored(llm)
    runner.mixed_graph_after = 0
    for limit in (10 ** 9, 1):
        runner._mixed_graphs.clear()
        runner.max_graph_logits_bytes = limit
        outs = scored(llm)
        kept = [g for g in runner._mixed_graphs.values() if isinstance(g, MixedGraph) and g.n_logits > g.n_requests]
        assert sum(g.logits.numel() * 4 for g in kept) <= limit and (limit == 1 or kept)
        for a, b in zip(outs, first):
            assert a.output_token_ids == b.output_token_ids
            # (a step padded to its bucket may sum in another order: bfloat16 logits of this model are off by less than 0.1)
            assert all(abs(x.logprob - y.logprob) < 0.2 for x, y in zip(a.prompt_logprobs[1:], b.prompt_logprobs[1:]))


def test_replayed_steps_are_scored_where_their_logits_lie(folder):
    """A replayed step hands the engine a view of its logits; who calls the runner gets a copy unless it says otherwise."""
    from slipstream_b200 import LLM
    from slipstream_b200.engine.context import StepEntry
    from slipstream_b200.engine.graphs import MixedGraph

    llm = LLM(folder, dtype="bfloat16", num_gpu_blocks=1024, max_num_seqs=32, prefill_chunk_size=64)
    runner = llm.engine.runner
    runner.mixed_graph_after = 0
    step, seen = runner.step, []
    runner.step = lambda entries, **more: seen.append(step(entries, **more)) or seen[-1]
    first = scored(llm)
    own = {g.logits.data_ptr() for g in runner._mixed_graphs.values() if isinstance(g, MixedGraph)}
    assert own & {t.data_ptr() for t in seen}
    runner.step = step
    results = {}
    for keep in (True, False):
        entries = [StepEntry(f"r{keep}", prompts()[0][:64], list(range(64)))]
        results[keep] = runner.step(entries, keep=keep)
        runner.release(f"r{keep}")
    graphs = [g for g in runner._mixed_graphs.values() if isinstance(g, MixedGraph)]
    assert results[True].data_ptr() not in {g.logits.data_ptr() for g in graphs}
    assert results[False].data_ptr() in {g.logits.data_ptr() for g in graphs} and torch.equal(results[True], results[False])
    assert all(a.output_token_ids == b.output_token_ids for a, b in zip(first, scored(llm)))
