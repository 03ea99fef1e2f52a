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


def test_recipes_keep_their_state_over_inference():
    """What passes between training steps measure, and the copies of weights that they make, are gone afterwards, after an error too."""
    from types import SimpleNamespace

    from surogate_b200.recipes.base import Recipe
    from surogate_b200.recipes.fp8_hybrid import FP8HybridRecipe

    with Recipe().inference():
        pass
    for grouped in (False, True):
        r = FP8HybridRecipe(SimpleNamespace(n_layers=2), torch.device("cpu"))
        r.amax_cur.uniform_(), r.scale.uniform_(), r.scale_inv.uniform_()
        r.weight_cache[(0, "qkv")] = "kept"
        if grouped:
            r._gstate(torch.device("cpu"))["amax"].uniform_()
            r.expert_weight_cache[(1, "experts_down")] = "kept too"
        kept = [t.clone() for t in (r.amax_cur, r.scale, r.scale_inv)]
        same = [r.amax_cur, r.scale, r.scale_inv]
        g = {k: v.clone() for k, v in r._gstate(torch.device("cpu")).items() if torch.is_tensor(v)} if grouped else None
        try:
            with r.inference():
                assert r.apart
                for t in same:
                    t.add_(1.0)
                r.weight_cache[(0, "out")] = r.expert_weight_cache[(0, "experts_down")] = "new"
                st = r._gstate(torch.device("cpu"))
                for k in ("scale", "inv", "amax"):
                    st[k].add_(2.0)
                raise KeyError
        except KeyError:
            pass
        assert not r.apart and all(a is b and torch.equal(a, k) for a, b, k in zip((r.amax_cur, r.scale, r.scale_inv), same, kept))
        assert r.weight_cache == {(0, "qkv"): "kept"} and r.expert_weight_cache == ({(1, "experts_down"): "kept too"} if grouped else {})
        assert all(torch.equal(r._g_state[k], v) for k, v in g.items()) if grouped else not hasattr(r, "_g_state")


def test_generate_refuses_visual_inputs(tmp_path):
    """They were left out without a word."""
    tr = _trainer(tmp_path, "qwen3")
    tr.set_visual_inputs(mrope_position_ids=torch.zeros(3, 1, 2, dtype=torch.int32))
    with pytest.raises(NotImplementedError, match="visual"):
        tr.generate([[1, 2]], max_new_tokens=2)
    tr.set_visual_inputs()
    assert len(tr.generate([[1, 2]], max_new_tokens=2)[0][0].tokens) == 2


def test_chat_without_a_positive_temperature_is_greedy(tmp_path):
    """As the helper always was: temperatures that are not above 0 are greedy, no room means no tokens."""
    from surogate_b200.cli.chat import generate

    tr = _trainer(tmp_path, "qwen3")
    want = generate(tr, None, [1, 2, 3], max_new_tokens=4)
    assert len(want) == 4 and all(generate(tr, None, [1, 2, 3], max_new_tokens=4, temperature=t) == want for t in (-1.0, math.nan))
    assert generate(tr, None, [1, 2, 3], max_new_tokens=-1) == []


def test_copying_pages_refuses_scales_of_other_caches():
    kv = torch.zeros(2, 4, 2, 1, 16, 8)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    good = torch.ones(kv.shape[:5])
    for bad in (good.double(), good[:1], good[:, :3], good[:, :, :1], good.expand(2, 4, 2, 2, 16), good[..., :8], good[0]):
        with pytest.raises(RuntimeError):
            ops.kv_copy_pages(kv.to(torch.float8_e4m3fn), i32(0), i32(1), bad)
    ops.kv_copy_pages(kv.to(torch.float8_e4m3fn), i32(0), i32(1), good)


def test_sampling_at_a_temperature_without_end():
    """All tokens weigh the same, those of -inf and NaN nothing; of infinite logits only those count."""
    x = torch.tensor([[0.0, -math.inf, 3.0, math.nan, 1.0]]).expand(6, 5)
    u = torch.tensor([0.0, 0.3, 0.34, 0.66, 0.67, 0.999])
    for t in (math.inf, torch.full((6,), math.inf)):
        tok, lp = ops.sample_tokens(x, u, temperature=t)
        assert tok.tolist() == [0, 0, 2, 2, 4, 4]
        assert torch.allclose(lp, torch.log_softmax(torch.tensor([0.0, -math.inf, 3.0, -math.inf, 1.0]), 0)[tok.long()])
    assert ops.sample_tokens(torch.tensor([[1.0, math.inf, math.inf]]), torch.tensor([0.6]), temperature=math.inf)[0].tolist() == [2]


@pytest.mark.parametrize("name", ["qwen3", "llama"])
def test_generate_on_an_8_bit_cache_follows_the_logits(tmp_path, name):
    """Rounding keys (of scores with a spread of about 1) and values to e4m3, 0.026 of an element in rms, costs 0.04 of an attention output, and 0.06 of the
    hidden state after two layers: that share of the logits' spread in the mean, six times it at most."""
    import numpy as np

    tr = _trainer(tmp_path, name)
    g = np.random.default_rng(5)
    prompts = [g.integers(0, 320, n).tolist() for n in (9, 16, 18)]
    errs = []
    for p, cs in zip(prompts, tr.generate(prompts, max_new_tokens=6, seed=2, page_size=16, cache_dtype=torch.float8_e4m3fn)):
        lg = tr.logits(np.asarray([p + cs[0].tokens], np.int32))[0].double()[len(p) - 1:-1]
        lp = torch.log_softmax(lg, -1).gather(1, torch.tensor(cs[0].tokens)[:, None])[:, 0]
        errs.append((lp - torch.tensor(cs[0].logprobs)).abs() / lg.std(-1))
    errs = torch.cat(errs)
    assert 0 < errs.mean() <= 0.06 and errs.max() <= 0.36
