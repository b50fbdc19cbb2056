"""``disable_cascade_attn=False`` on an engine that cannot share prefixes is no silent no-op."""
import logging

import pytest

from vllm_ascend_b200 import LLM


@pytest.mark.parametrize("model,kw,said", [
    ("tiny-qwen", {}, False), ("tiny-qwen", {"disable_cascade_attn": False}, False), ("tiny-gdn", {}, False),
    ("tiny-gdn", {"disable_cascade_attn": False}, True), ("tiny-deepseek-sparse", {"disable_cascade_attn": False}, True),
    ("tiny-qwen", {"disable_cascade_attn": False, "enable_lora": True}, True),
    ("tiny-qwen", {"disable_cascade_attn": False, "speculative_config": {"method": "ngram", "num_speculative_tokens": 2}}, True)])
def test_engines_that_cannot_share_say_so(caplog, model, kw, said):
    logger = logging.getLogger("vllm_ascend_b200")
    logger.addHandler(caplog.handler)
    try:
        LLM(model, device="cpu", max_model_len=64, max_num_seqs=2, **kw)
        assert any("disable_cascade_attn" in r.getMessage() for r in caplog.records) is said
    finally:
        logger.removeHandler(caplog.handler)
