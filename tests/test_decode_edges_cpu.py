"""The answering path without a GPU where its calls meet their limits: refusals, pages copied onto themselves, temperatures without end, answers of
trainers that hold more than text."""
import math

import pytest
import torch

from surogate_b200 import ops
from test_decode_cpu import _cache, _trainer


def test_attention_refuses_caps_and_scales_that_fp32_cannot_hold():
    kv, table = _cache()
    q, n = torch.randn(3, 4, 8), torch.tensor([64, 0, 17], dtype=torch.int32)
    for kw in (dict(softcap=1e300), dict(softcap=1e38), dict(softcap=1e-300), dict(softcap=1e-38), dict(softcap=math.inf), dict(softcap=math.nan), dict(softmax_scale=1e300),
               dict(softmax_scale=math.inf), dict(softmax_scale=math.nan)):
        with pytest.raises(RuntimeError):
            ops.paged_attention(q, kv, table, n, **kw)
    assert torch.isfinite(ops.paged_attention(q, kv, table, n, softcap=2.0 ** 64, softmax_scale=-1.0)).all()


# ---------------------------------------------------------------------------------------------- answers
def test_generate_refuses_prompt_tokens_outside_the_vocabulary(tmp_path):
    tr = _trainer(tmp_path, "qwen3")
    V = tr.model.vocab_size
    for bad in (-1, V, 2 ** 31 - 1, 2 ** 40):
        with pytest.raises(ValueError, match="vocabulary"):
            tr.generate([[1, 2], [3, bad, 4]], max_new_tokens=2)
    assert len(tr.generate([[0, V - 1]], max_new_tokens=2)[0][0].tokens) == 2 and tr.store.grads_enabled
