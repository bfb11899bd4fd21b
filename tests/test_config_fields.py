"""The options of the engine by position: those of a later feature stand behind the ones that were there."""

from dataclasses import fields

from atma_amd.engine import Config

EARLIER = ["model", "kvcache_block_size", "gpu_memory_utilization", "max_num_seqs", "max_num_batched_tokens", "max_model_len",
           "enforce_eager", "fp8_mlp", "strict_weights", "eos", "num_kvcache_blocks", "init_std", "seed", "hf_config"]


def test_options_by_position():
    assert [f.name for f in fields(Config)][:len(EARLIER)] == EARLIER
    c = Config("path", 256, 0.9, 16, 1024, 512, True, False, True, 7)
    assert c.strict_weights is True and c.eos == 7 and c.fp4_weights is False
    assert Config(fp4_weights=True).fp4_weights is True
