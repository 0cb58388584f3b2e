"""8-bit layers on the host: their options, who takes them, the products' plans and the layout of stacked weights."""

import pytest
import torch

from slipstream_b200.config.engine_config import EngineConfig, ModelOptions
from slipstream_b200.config.model_config import ConfigError, Qwen2Config
from slipstream_b200.ops.int8 import RUN, int8_plan, stack_gate_up
from slipstream_b200.registry import architectures, resolve_architecture


def test_the_option_is_read_and_refused():
    assert ModelOptions("m").quantization is None and ModelOptions("m", quantization="int8").quantization == "int8"
    assert EngineConfig.for_model("m", quantization="int8").model.quantization == "int8"
    with pytest.raises(ValueError, match="quantization"):
        ModelOptions("m", quantization="int4")


def test_architectures_say_which_quantizations_they_have():
    config = Qwen2Config(vocab_size=64, hidden_size=64, num_hidden_layers=2, max_position_embeddings=64, torch_dtype="bfloat16",
                         intermediate_size=96, num_attention_heads=4, num_key_value_heads=2, head_dim=16, rms_norm_eps=1e-6,
                         rope_theta=1e4, tie_word_embeddings=True)
    qwen2 = resolve_architecture({"architectures": ["Qwen2ForCausalLM"]})
    plain, int8 = qwen2.build_model(config), qwen2.build_model(config, "int8")
    assert [s.name for s in plain.weight_specs()] == [s.name for s in int8.weight_specs()]
    assert type(int8.blocks[0].mixer).__name__ == "Int8PagedAttention" and type(plain.blocks[0].mixer).__name__ == "PagedAttention"
    assert type(int8.final_norm).__name__ == "RMSNorm"
    with pytest.raises(ConfigError, match="int4"):
        qwen2.build_model(config, "int4")
    for name in architectures():
        if name != "Qwen2ForCausalLM":
            with pytest.raises(ConfigError, match="quantization"):
                resolve_architecture({"architectures": [name]}).build_model(None, "int8")


RESIDENT = ((148, 74, 45, 33, 26, 22, 15, 15), (296, 148, 93, 71, 56, 45, 37, 33))


@pytest.mark.parametrize("resident", [None, RESIDENT, ((1,) * 8, (1,) * 8)])
@pytest.mark.parametrize("sms", [1, 2, 80, 148])
def test_plans_are_forms_that_the_kernels_have(sms, resident):
    for gated in (False, True):
        for tokens in (1, 2, 15, 16, 17, 100, 255, 256, 257, 640, 641, 5000, 100000):
            for features, k in ((128, 1), (128, 17), (256, 128), (1152, 896), (4608, 3584), (3584, 18944), (37888, 3584), (128, 131071)):
                many, tile, slices, per, steps = int8_plan(tokens, features, k, sms, gated, resident)
                assert steps in (1, 2)
                if many:
                    assert tile % 32 == 0 and 32 <= tile <= 256 and tokens > 64 and (not gated or tile % 128 == 0)
                else:
                    assert tile % 16 == 0 and 16 <= tile <= 256 and 1 <= slices <= min(8, -(-k // 128)) and per in (1, 2) and tokens <= 640
                    # what the kernel keeps in shared memory: two stages of the ring, and its share of the sums
                    rest = 2560 + (-(-tile // slices) * 512 if slices > 1 else 0)
                    assert 2 * steps * (128 + tile) * 128 + rest <= 232448


def test_plans_of_more_features_than_a_grid_has_rows_for_their_tiles():
    """The kernel for few tokens has its tiles of 128 features along grid.y: up to 65,535 of them."""
    for tokens in (1, 64, 65, 640, 700):
        for gated in (False, True):
            assert tokens > 64 or int8_plan(tokens, 65535 * 128, 16, 148, gated, RESIDENT)[0] == 0
            many, tile, slices, per, steps = int8_plan(tokens, 65535 * 128 + (128 if gated else 1), 16, 148, gated, RESIDENT)
            assert many == 1 and tile % (128 if gated else 32) == 0 and steps in (1, 2)


def test_plans_do_not_change_within_a_step_of_tokens():
    for tokens in (1, 17, 300, 1000):
        step = 16 if tokens <= 640 else 256
        upto = -(-tokens // step) * step
        assert int8_plan(tokens, 4608, 3584, 148, False, RESIDENT) == int8_plan(upto, 4608, 3584, 148, False, RESIDENT)


def test_decode_plans_cut_k_where_tiles_are_few():
    """The o, q/k/v and gate/up projections of the 7B layer sizes: K in slices where there are fewer tiles than multiprocessors."""
    for tokens in (1, 8, 16):
        for features, gated in ((3584, False), (4608, False), (37888, True)):
            many, tile, slices, per, steps = int8_plan(tokens, features, 3584, 148, gated, RESIDENT)
            assert (many, tile) == (0, 16) and (slices > 1) == (features < 37888) and features // 128 * slices <= 2 * 148


def test_stacked_gate_and_up_rows():
    for rows in (1, 63, 64, 65, 200):
        gate, up = torch.randn(rows, 3), torch.randn(rows, 3)
        stacked = stack_gate_up(gate, up)
        runs = stacked.reshape(-1, 2, RUN, 3)
        assert torch.equal(runs[:, 0].reshape(-1, 3)[:rows], gate) and torch.equal(runs[:, 1].reshape(-1, 3)[:rows], up)
        assert not runs[:, 0].reshape(-1, 3)[rows:].any() and not runs[:, 1].reshape(-1, 3)[rows:].any()
    assert stack_gate_up(torch.ones(5), torch.zeros(5)).shape == (128,)
