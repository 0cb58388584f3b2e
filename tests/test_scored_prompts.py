"""How many prompt tokens a step scores, on the host."""

import random

import pytest

from slipstream_b200.cache import CacheManager, GroupLayout
from slipstream_b200.config.engine_config import SchedulerConfig
from slipstream_b200.config.sampling_params import SamplingParams
from slipstream_b200.engine.scheduler import MAX_SCORED_TOKENS, Scheduler, Sequence
from slipstream_b200.parts.base import CacheSpec


def sequence(i, n, wish, max_new=2):
    return Sequence(seq_id=i, prompt_token_ids=list(range(n)), sampling_params=SamplingParams(max_tokens=max_new, prompt_logprobs=wish), arrival_ts=float(i),
                    max_new_tokens=max_new)


def run(lengths, wishes, chunk, budget=8192, max_steps=2000):
    """Steps until everything is done: of each the takes, and the tokens scored."""
    cache = CacheManager([GroupLayout(CacheSpec(2, 16, None), 2)], 8192, 16, 64, 16384)
    sched = Scheduler(SchedulerConfig(max_num_seqs=64, max_num_batched_tokens=budget, prefill_chunk_size=chunk or 1, enable_chunked_prefill=bool(chunk)), cache)
    seqs = [sequence(i, n, w) for i, (n, w) in enumerate(zip(lengths, wishes))]
    for s in seqs:
        sched.add_seq(s)
    steps = []
    while sched.has_work():
        assert len(steps) < max_steps
        plan = sched.schedule()
        assert plan.scheduled
        scored = 0
        for item in plan.scheduled:
            places = item.seq.places_to_score(item.take)
            scored += len(places)
            item.seq.prompt_logprobs += [item.seq.num_computed_tokens + p + 1 for p in places]
        for item in plan.scheduled:
            ends = item.samples
            item.seq.num_computed_tokens += item.take
            cache.commit(item.seq.seq_id, item.take)
            if ends:
                item.seq.output_token_ids.append(1)
                if item.seq.num_output_tokens == item.seq.max_new_tokens:
                    sched.finish(item.seq)
        steps.append(([(i.seq.seq_id, i.take) for i in plan.scheduled], scored))
    return seqs, steps


@pytest.mark.parametrize("chunk", [256, 7, 0, 4096])
def test_a_step_scores_a_bounded_number_of_tokens(chunk):
    lengths = [600, 1, 2, 5000, 1024, 1025, 1026, 257, 300, 8000, 90, 600] + [256] * 20
    wishes = [None if i % 5 == 3 else i % 4 for i in range(len(lengths))]
    if chunk == 7:
        lengths = [n // 10 + 1 for n in lengths]
    seqs, steps = run(lengths, wishes, chunk)
    assert all(scored <= MAX_SCORED_TOKENS for _, scored in steps)
    for s, n, w in zip(seqs, lengths, wishes):  # every token behind the first is scored once, in order
        assert s.prompt_logprobs[1:] == ([] if w is None else list(range(1, n))) and s.num_output_tokens == 2


def test_prompts_that_are_not_scored_are_cut_as_ever():
    lengths = [600, 5000, 1025, 8000] + [256] * 20
    _, steps = run(lengths, [None] * len(lengths), 4096)
    assert steps[0][0][:3] == [(0, 600), (1, 4096), (2, 1025)] and sum(t for _, t in steps[0][0]) == 8192
    # and one that is scored beside them is cut alone; another waits for the rows of the next steps, who asks for none does not
    _, steps = run([5000, 3000, 100, 10], [0, None, 3, None], 8192)
    assert steps[0] == ([(0, MAX_SCORED_TOKENS), (1, 3000), (3, 10)], MAX_SCORED_TOKENS)
    assert steps[4][0] == [(0, 5000 - 4 * MAX_SCORED_TOKENS), (2, 100)]


def test_the_part_of_a_portion_that_scores_so_many():
    rng = random.Random(3)
    for _ in range(2000):
        n = rng.randint(1, 40)
        s = sequence(0, n, rng.choice([0, 2, None]))
        s.output_token_ids = [1] * rng.randint(0, 5)
        s.num_computed_tokens = rng.randint(0, s.num_tokens - 1)
        s.prompt_logprobs = [None] * rng.randint(1, n)
        take, limit = rng.randint(1, s.num_tokens - s.num_computed_tokens), rng.randint(0, 12)
        fits = [t for t in range(take + 1) if len(s.places_to_score(t)) <= limit]
        assert s.take_scoring(take, limit) == max(fits)


def test_bytes_for_pages():
    """The logits of scored prompts come off the pages only where the rest would not hold them."""
    from slipstream_b200.engine.runner import page_bytes

    gb = 10 ** 9
    assert page_bytes(170 * gb, 0.9, 7 * gb) == int(170 * gb * 0.9 * 0.9)
    assert page_bytes(170 * gb, 1.0, 7 * gb) == int(170 * gb * 0.9) - 7 * gb
    assert page_bytes(20 * gb, 0.9, 2 * gb) == 16 * gb
    assert page_bytes(gb, 0.9, 2 * gb) == int(0.9 * gb) - gb // 4


@pytest.mark.parametrize("name", ["logprobs", "prompt_logprobs"])
def test_alternatives_are_whole_numbers(name):
    """A number that is none would otherwise be found out in the middle of a step, beside other requests."""
    import numpy as np

    for bad in (1.5, 2.0, True, "3", float("nan"), -1, 65):
        with pytest.raises(ValueError, match=name):
            SamplingParams(**{name: bad})
    for good in (None, 0, 64, np.int64(5)):
        assert getattr(SamplingParams(**{name: good}), name) == good
