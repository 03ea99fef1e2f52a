"""The answering path without a GPU: the PyTorch forms of its operators, the books of the paged cache, refusals, and ``Trainer.generate``
against the logits of a full pass over every architecture."""
import math
import os

import numpy as np
import pytest
import torch

from surogate_b200 import ops
from surogate_b200.dsl.compiler import load_hf_config
from surogate_b200.ops import PagedKVCache
from surogate_b200.ops.paged_kv import quantize_e4m3
from surogate_b200.runtime import generation
from surogate_b200.runtime.trainer import Trainer, TrainerConfig
from test_hf_parity_cpu import _cases

CASES = dict(_cases())
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------- operators
def _cache(B=3, width=4, P=16, Hkv=2, D=8, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = B * width + 2
    return torch.randn(n, 2, Hkv, P, D, generator=g).to(dtype), torch.randperm(n, generator=g)[:B * width].view(B, width).to(torch.int32)


@pytest.mark.parametrize("window,softcap,sinks", [(0, 0.0, False), (5, 0.0, False), (0, 3.0, True), (20, 2.0, True)])
def test_paged_attention_is_attention_over_the_gathered_rows(window, softcap, sinks):
    kv, table = _cache()
    q = torch.randn(3, 4, 8, generator=torch.Generator().manual_seed(1))
    sk = torch.tensor([0.5, -2.0, 9.0, 0.0]) if sinks else None
    n = torch.tensor([64, 0, 17], dtype=torch.int32)
    got, lse = ops.paged_attention(q, kv, table, n, window=window, softcap=softcap, sinks=sk, return_lse=True)
    for b, x in enumerate(n.tolist()):
        for h in range(4):
            s, vals = [], []
            for j in range(max(0, x - window) if window else 0, x):
                k, v = kv[table[b, j // 16], :, h // 2, j % 16].double()
                t = float(q[b, h].double() @ k) / math.sqrt(8)
                s.append(softcap * math.tanh(t / softcap) if softcap else t)
                vals.append(v)
            if not s:
                assert (got[b, h] == 0).all() and lse[b, h] == -math.inf
                continue
            e = torch.tensor(s, dtype=torch.float64).exp()
            want = (e[:, None] * torch.stack(vals)).sum(0) / (e.sum() + (math.exp(float(sk[h])) if sinks else 0.0))
            assert torch.allclose(got[b, h].double(), want, atol=1e-5) and abs(float(lse[b, h]) - math.log(e.sum())) < 1e-5


def test_append_copy_and_quantised_caches():
    kv, table = _cache()
    k, v = torch.randn(3, 5, 2, 8), torch.randn(3, 5, 2, 8)
    start, count = torch.tensor([0, 14, 60], dtype=torch.int32), torch.tensor([5, 5, 3], dtype=torch.int32)
    before = kv.clone()
    ops.kv_append(kv, k, v, table, start, count)
    assert torch.equal(kv[table[1, 0], 0, :, 15], k[1, 1]) and torch.equal(kv[table[1, 1], 1, :, 2], v[1, 4]) and torch.equal(kv[table[2, 3], 1, :, 14], v[2, 2])
    assert int((kv != before).any(-1).sum()) == 2 * 2 * 13                  # 13 tokens, no other place
    q8, scales = torch.zeros(kv.shape).to(E4M3), torch.ones(kv.shape[:4])
    ops.kv_append(q8, k, v, table, start, count, scales)
    back = q8[table[1, 0], 0, :, 15].float() * scales[table[1, 0], 0, :, 15, None]
    assert ((back - k[1, 1]).abs() <= 2.0 ** -4 * k[1, 1].abs() + 2.0 ** -10 * scales[table[1, 0], 0, :, 15, None]).all()   # half a step; of a subnormal value 2^-10
    assert quantize_e4m3(torch.zeros(2, 8))[1].tolist() == [1.0, 1.0]
    layers, ls = torch.stack([kv, kv + 1]), torch.rand(2, *kv.shape[:4])
    want, ws = layers.clone(), ls.clone()
    want[:, [3, 5]], ws[:, [3, 5]] = layers[:, [0, 0]], ls[:, [0, 0]]
    ops.kv_copy_pages(layers, torch.tensor([0, 0], dtype=torch.int32), torch.tensor([3, 5], dtype=torch.int32), ls)
    assert torch.equal(layers, want) and torch.equal(ls, ws)


def test_refusals():
    kv, table = _cache()
    q, n = torch.randn(3, 4, 8), torch.tensor([64, 0, 17], dtype=torch.int32)
    k = torch.randn(3, 2, 2, 8)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    bad = table.clone()
    bad[0, 2] = kv.shape[0]
    for call in [lambda: ops.paged_attention(q[:, :3], kv, table, n), lambda: ops.paged_attention(q[..., :4], kv, table, n), lambda: ops.paged_attention(q, kv[0], table, n),
                 lambda: ops.paged_attention(q, kv, table, i32(65, 0, 0)), lambda: ops.paged_attention(q, kv, table, i32(-1, 0, 0)), lambda: ops.paged_attention(q, kv, bad, n),
                 lambda: ops.paged_attention(q, kv, table, n, window=-1), lambda: ops.paged_attention(q, kv, table, n, scales=torch.ones(kv.shape[:4])),
                 lambda: ops.kv_append(kv, k, k[:, :1], table, i32(0, 0, 0)), lambda: ops.kv_append(kv, k.double(), k.double(), table, i32(0, 0, 0)),
                 lambda: ops.kv_append(kv, k, k, table, i32(0, 63, 0)), lambda: ops.kv_append(kv, k, k, bad, i32(32, 0, 0)), lambda: ops.kv_append(kv, k, k, table, i32(0, -1, 0)),
                 lambda: ops.kv_append(kv.to(E4M3), k, k, table, i32(0, 0, 0)), lambda: ops.kv_copy_pages(kv, i32(0), i32(1)),
                 lambda: ops.kv_copy_pages(kv[None], i32(0, 1), i32(2, 2)), lambda: ops.kv_copy_pages(kv[None], i32(0, 1), i32(1, 2)), lambda: ops.kv_copy_pages(kv[None], i32(0), i32(99)),
                 lambda: ops.kv_copy_pages(kv[None], i32(0), i32(1, 2)), lambda: ops.kv_copy_pages(kv[None].to(E4M3), i32(0), i32(1)),
                 lambda: ops.sample_tokens(torch.zeros(1, 0), torch.zeros(1)), lambda: ops.sample_tokens(q[0].double(), torch.zeros(4)), lambda: ops.sample_tokens(q[0], torch.zeros(3)),
                 lambda: ops.sample_tokens(q[0], torch.zeros(4), temperature=-1.0), lambda: ops.sample_tokens(q[0], torch.zeros(4), top_k=torch.ones(4))]:
        with pytest.raises(RuntimeError):
            call()


def test_sample_tokens_by_hand():
    """Probabilities 0.5, 0.25, 0.125, 0.125 at indices 2, 0, 3, 1."""
    x = torch.log(torch.tensor([[0.25, 0.125, 0.5, 0.125]]))
    draw = lambda u, **kw: int(ops.sample_tokens(x, torch.tensor([u]), **kw)[0])  # noqa: E731
    assert [draw(u) for u in (0.0, 0.24, 0.26, 0.37, 0.38, 0.87, 0.88, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert draw(0.999, temperature=0.0) == 2 and draw(0.999, top_k=1) == 2
    assert [draw(u, top_k=2) for u in (0.0, 0.33, 0.34, 0.99)] == [0, 0, 2, 2]
    assert [draw(u, top_k=3) for u in (0.28, 0.29, 0.42, 0.43)] == [0, 1, 1, 2]       # of the two equal ones the lower index stays
    assert [draw(u, top_p=0.6) for u in (0.0, 0.34)] == [0, 2] and draw(0.0, top_p=0.5) == 2 and draw(0.0, top_p=0.0) == 2
    assert draw(0.0, min_p=0.6) == 2 and draw(0.0, min_p=0.4) == 0 and draw(0.34, min_p=0.4) == 2
    assert [draw(u, temperature=0.5) for u in (0.17, 0.19)] == [0, 1]                 # weights 1/4, 1/16, 1, 1/16
    tok, lp = ops.sample_tokens(x.expand(3, 4), torch.tensor([0.1, 0.5, 0.9]), temperature=0.3, top_p=0.9)
    assert torch.allclose(lp, x[0, tok.long()], atol=1e-6)
    empty = torch.tensor([[-math.inf, math.nan], [0.0, -math.inf]])
    tok, lp = ops.sample_tokens(empty, torch.tensor([0.5, 0.999]))
    assert tok.tolist() == [-1, 0] and lp.tolist() == [-math.inf, 0.0]


# ---------------------------------------------------------------------------------------------- the books
def test_cache_books():
    c = PagedKVCache(2, 10, 16, 1, 8, 6, dtype=torch.float32)
    c.reserve({0: 20, 1: 16})
    assert c.pages(0) == [0, 1] and c.pages(1) == [2] and c.free_pages == 7 and c.length(0) == 20
    c.kv[:, 0], c.kv[:, 1] = 5.0, 7.0
    c.fork(0, [2, 3])
    assert c.pages(2) == c.pages(3) == [0, 1] and c.free_pages == 7
    c.reserve({2: 1})                                                      # its last page is shared and partly filled: copied
    assert c.pages(2) == [0, 3] and c.pages(3) == [0, 1] and bool((c.kv[:, 3] == 7).all())
    c.reserve({0: 1, 3: 1})                                                # the one that goes last keeps the page
    assert c.pages(0) == [0, 4] and c.pages(3) == [0, 1] and bool((c.kv[:, 4] == 7).all())
    with pytest.raises(RuntimeError, match="full"):
        c.reserve({0: 100})
    assert c.length(0) == 21 and c.free_pages == 5
    with pytest.raises(ValueError):
        c.fork(0, [1])
    with pytest.raises(ValueError):
        c.fork(0, [4, 4])
    with pytest.raises(ValueError):
        c.reserve({6: 1})
    c.free(0)
    c.free(1)
    assert c.free_pages == 7 and c.sequences() == [2, 3]
    c.kv[:, 3] = 9.0
    assert c.compact() == 1 and c.pages(2) == [0, 2] and c.pages(3) == [0, 1] and bool((c.kv[:, 2] == 9).all()) and c.compact() == 0
    assert c.table([3, 2], tokens=40).tolist() == [[0, 1, -1], [0, 2, -1]]
    c.truncate(2, 16)
    assert c.pages(2) == [0] and c.free_pages == 8
    c.free(2)
    c.free(3)
    assert c.free_pages == 10
    c.reserve({0: 0})
    assert c.pages(0) == [] and c.table([0]).tolist() == [[-1]]
    q8 = PagedKVCache(1, 4, 16, 1, 8, 2, dtype=E4M3)
    k = torch.randn(1, 3, 1, 8)
    q8.reserve({0: 3})
    q8.append(0, k, k, q8.table([0]), torch.zeros(1, dtype=torch.int32))
    q8.fork(0, [1])
    q8.reserve({1: 1})                                                     # its own copy of the page, with the scales
    assert torch.equal(q8.kv[0, q8.pages(1)[0], :, :, :3].float(), q8.kv[0, 0, :, :, :3].float()) and torch.equal(q8.scales[0, q8.pages(1)[0]], q8.scales[0, 0])
    assert q8.pages(1) != q8.pages(0)
    for bad in (dict(page_size=8), dict(page_size=0), dict(num_pages=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(n_layers=1, num_pages=4, page_size=16, num_kv_heads=1, head_dim=8, max_seqs=1), **bad})


def test_cache_of_a_full_page_is_shared_without_a_copy():
    c = PagedKVCache(1, 4, 16, 1, 8, 3, dtype=torch.float32)
    c.reserve({0: 16})
    c.fork(0, [1, 2])
    c.reserve({0: 1, 1: 1, 2: 1})
    assert c.pages(0)[0] == c.pages(1)[0] == c.pages(2)[0] and c.free_pages == 0
    assert len({c.pages(s)[1] for s in range(3)}) == 3


# ---------------------------------------------------------------------------------------------- answers
def _trainer(tmp_path, name):
    CASES[name].save_pretrained(os.path.join(tmp_path, name))
    tr = Trainer(TrainerConfig(model=load_hf_config(os.path.join(tmp_path, name)), batch_size=1, seq_len=24, zero_level=0), device=torch.device("cpu"))
    tr.init_weights(seed=0)
    return tr


def _check_greedy(tr, prompts, outs):
    for p, cs in zip(prompts, outs):
        for c in cs:
            lg = tr.logits(np.asarray([list(p) + c.tokens], np.int32))[0].double()
            for i, t in enumerate(c.tokens):
                row = lg[len(p) - 1 + i]
                assert row[t] >= row.max() - 1e-3 and abs(float(torch.log_softmax(row, -1)[t]) - c.logprobs[i]) < 1e-3


@pytest.mark.parametrize("name", list(CASES))
def test_generate_follows_the_logits_of_full_passes(tmp_path, name):
    """Greedy answers of prompts of several lengths are the largest logits of a pass over the whole row, on the cache where there is one."""
    tr = _trainer(tmp_path, name)
    cached = generation.cache_layout(tr.cm, torch.device("cpu"))
    assert (cached is not None) == (name in ("qwen3", "qwen3-untied", "qwen2", "llama", "mistral", "qwen3-moe", "gpt-oss"))
    g = np.random.default_rng(1)
    prompts = [g.integers(0, 320, n).tolist() for n in (1, 16, 21)]
    outs = tr.generate(prompts, max_new_tokens=6, temperature=0.0, page_size=16, prompt_rows=2)
    assert all(len(c.tokens) == len(c.logprobs) == 6 and c.finish_reason == "length" for cs in outs for c in cs)
    _check_greedy(tr, prompts, outs)


def test_generate_samples_the_same_with_and_without_the_cache(tmp_path, monkeypatch):
    """Several completions of each prompt: the same draws on the cache as by full passes, independent of which neighbours end, and of how many
    prompts share a pass."""
    tr = _trainer(tmp_path, "qwen3")
    g = np.random.default_rng(2)
    prompts = [g.integers(0, 320, n).tolist() for n in (5, 32, 17)]
    kw = dict(n=3, max_new_tokens=20, temperature=1.0, top_p=0.95, top_k=100, min_p=0.001, seed=7, page_size=16)
    a = tr.generate(prompts, **kw)
    assert len({tuple(c.tokens) for cs in a for c in cs}) == 9
    stop = a[1][1].tokens[4]
    b = tr.generate(prompts, eos_id=stop, prompt_rows=1, **kw)
    for x, y in zip((c for cs in a for c in cs), (c for cs in b for c in cs)):
        cut = x.tokens[:x.tokens.index(stop) + 1] if stop in x.tokens else x.tokens
        assert y.tokens == cut and (y.finish_reason == "stop") == (stop in x.tokens)
    monkeypatch.setattr(generation, "cache_layout", lambda cm, device: None)
    c = tr.generate(prompts, **kw)
    assert [x.tokens for cs in a for x in cs] == [x.tokens for cs in c for x in cs]
    assert np.allclose([x.logprobs for cs in a for x in cs], [x.logprobs for cs in c for x in cs], atol=1e-3)
    row = np.asarray([prompts[2] + a[2][0].tokens], np.int32)
    lp = tr.token_logprobs(row[:, :-1], row[:, 1:])[0, len(prompts[2]) - 1:]
    assert np.allclose(lp, a[2][0].logprobs, atol=1e-3)


def test_generate_refusals_and_ends(tmp_path):
    tr = _trainer(tmp_path, "qwen3")
    assert tr.generate([]) == [] and tr.generate([[1]], max_new_tokens=0)[0][0].tokens == []
    for bad in (dict(n=0), dict(max_new_tokens=-1), dict(prompt_rows=0)):
        with pytest.raises(ValueError):
            tr.generate([[1, 2]], **bad)
    with pytest.raises(ValueError):
        tr.generate([[]])
    with pytest.raises(ValueError):
        _trainer(tmp_path, "lfm2").generate([[1]], cache_dtype=torch.float32)
    assert tr.store.grads_enabled
    # an 8-bit cache: other values, the same kind of answer
    out = tr.generate([[3, 4, 5]], max_new_tokens=4, temperature=0.0, cache_dtype=E4M3)
    assert len(out[0][0].tokens) == 4
