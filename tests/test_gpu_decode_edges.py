"""The kernels of the answering path where formulas meet the ends of their types: numbers that are not finite, caps of scores, values of zero,
pages copied onto themselves, calls captured into graphs.  Tolerances as in ``test_gpu_decode``, or stated at the test."""
import math
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_decode import BF16, DEV, E4M3, FP16, FP32, _attention64, _check_attention, _check_sample, _model, _no_errors, _ops, _problem

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- attention: numbers that are not finite
def _check_not_finite(q, kv, table, n, **kw):
    """Outputs are not finite where the definition's are not (of an infinite value NaN may come out: its weight has two terms, of two signs), the
    log-sum-exp is what the definition gives, and where the definition is finite the two agree to what their types hold."""
    got, lse = _ops().paged_attention(q, kv, table, n, return_lse=True, **kw)
    _no_errors()
    want, wlse, mag, big = _attention64(q, kv, table, n, q.shape[-1] ** -0.5, **kw)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), (torch.isfinite(got) != torch.isfinite(want)).nonzero()[:5].tolist()
    assert torch.isnan(got)[torch.isnan(want)].all()
    for odd in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(odd(lse), odd(wlse)), (odd.__name__, lse, wlse)
    fin = torch.isfinite(want)
    # (half a step of the output, and the weights' and scores' errors: the widest of the types', e4m3's, over all)
    bound = torch.finfo(q.dtype).eps / 2 * want.abs() + (2.0 ** -11 + 2.0 ** -17 * (1 + big.unsqueeze(-1).nan_to_num(0, 0, 0))) * mag.nan_to_num(0, 0, 0) * 1.01 + 2.0 ** -24
    assert ((got.double() - want).abs()[fin] <= bound[fin]).all()
    fin = torch.isfinite(wlse)
    assert ((lse.double() - wlse)[fin].abs() <= 2.0 ** -17 * (1 + wlse[fin].abs() + big[fin].nan_to_num(0, 0, 0))).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, E4M3])
@pytest.mark.parametrize("longest", [300, 1000, 3000])
@pytest.mark.parametrize("sinks", [False, True])
def test_paged_attention_scores_that_are_not_finite(dtype, longest, sinks):
    """NaN and infinities in a query, in one key, in all keys of a row, and over the keys of single warps: rows that stay whole, few and many, and rows
    that are split and joined.  A row without keys stays zeros."""
    for B in (3, 90):
        lengths = [longest, 0, 20] + [longest // 2 + 5 * i for i in range(B - 3)]
        lengths = [min(x, longest) for x in lengths]
        q, kv, table, n, s = _problem(B, 4, 2, 64, 16, lengths, dtype, seed=longest + B)
        kw = dict(scales=s, sinks=torch.linspace(-3.0, 3.0, 4, device=DEV) if sinks else None)
        for value in (math.nan, math.inf):
            x = q.clone()
            x[0, 1, 7] = value
            if value != value:
                x[2] = value
                x[2, 3] = q[2, 3]
            if dtype != E4M3 or value != value:                          # (infinite elements and 8-bit zeros: NaN scores in both)
                _check_not_finite(x, kv, table, n, **kw)
        page = table[0].long()
        bad = [math.nan] if dtype == E4M3 else [math.nan, math.inf, -math.inf]
        for value in bad:
            for keys in ([5], [longest - 1], range(longest), [j for j in range(longest) if j // 16 % 4 == 1], [j for j in range(longest) if j // 16 % 4 != 1], range(64)):
                dirty = kv.clone()
                j = torch.tensor(list(keys), device=DEV)
                dirty[page[j // 16], 0, 0, j % 16, 3] = torch.full((), value, device=DEV).to(dtype)
                _check_not_finite(q, dirty, table, n, **kw)
        # one value, and a whole row of values
        dirty = kv.clone()
        dirty[page[0], 1, 1, 9, 11] = torch.full((), bad[-1], device=DEV).to(dtype)
        dirty[page[1], 1, 0, 2] = torch.full((), math.nan, device=DEV).to(dtype)
        _check_not_finite(q, dirty, table, n, **kw)


def test_paged_attention_of_scores_that_are_all_minus_infinity():
    """Without a sink 0 / 0, with one the sink takes all; the log-sum-exp is -inf."""
    for longest in (40, 2500):
        q, kv, table, n, _ = _problem(2, 4, 2, 64, 16, [longest, 30], BF16)
        q[0] = q[0].abs()
        kv[table[0].long(), 0, :, :, 5] = -math.inf
        _check_not_finite(q, kv, table, n)
        _check_not_finite(q, kv, table, n, sinks=torch.zeros(4, device=DEV))
        out, lse = _ops().paged_attention(q, kv, table, n, sinks=torch.zeros(4, device=DEV), return_lse=True)
        assert (out[0] == 0).all() and (lse[0] == -math.inf).all() and torch.isfinite(out[1]).all()


def test_paged_attention_of_value_scales_that_are_not_finite():
    """A value scale of NaN, or of infinity, makes the row's outputs NaN; its log-sum-exp, which no value enters, stays."""
    for longest in (300, 3000):
        for value in (math.nan, math.inf):
            q, kv, table, n, s = _problem(3, 4, 2, 64, 16, [longest, 0, 20], E4M3, seed=longest)
            s[table[0, 1].long(), 1, 0, 5] = value
            _check_not_finite(q, kv, table, n, scales=s)


def test_paged_attention_of_zero_values():
    """Tokens whose values are all zero have the scale 1, far above the others' 1e-4; where they have the highest scores, the weights of the others keep
    their bits: errors as in ``test_gpu_decode``.  One such token, every third, the first ones only, and all of a row."""
    for dtype in (E4M3, BF16, FP16):
        for longest in (200, 2100):
            for zero in ([0], [longest // 2], range(0, longest, 3), range(70), range(longest)):
                q, kv, table, n, s = _problem(2, 4, 2, 64, 16, [longest, longest // 3], dtype, seed=longest)
                j = torch.tensor(list(zero), device=DEV)
                page, place = table[0].long()[j // 16], j % 16
                # their scores, q . k / 8: 14 (base 2) for the first half of them, 50 for the second
                score = torch.where(torch.arange(len(j), device=DEV) < (len(j) + 1) // 2, 14.0, 50.0) * math.log(2)
                q[:, :, 0] = 8.0
                kv[page, :, :, place] = torch.zeros((), device=DEV).to(dtype)
                if dtype == E4M3:
                    kv[page, 0, :, place, 0] = torch.full((), 256.0, device=DEV).to(dtype)
                    s[:, 1] = 0.05 / 448
                    s[page, 0, :, place] = (score / 256)[:, None].expand(-1, 2)
                    s[page, 1, :, place] = 1.0
                else:
                    kv[page, 0, :, place, 0] = score[:, None].to(dtype).expand(-1, 2)
                _check_attention(q, kv, table, n, scales=s)


@pytest.mark.parametrize("dtype", [BF16, FP16, E4M3])
@pytest.mark.parametrize("Hq,Hkv", [(18, 1), (40, 2)])
def test_paged_attention_of_long_rows_with_heads_of_256_in_groups(dtype, Hq, Hkv):
    """More than eight query heads a key head of 256 elements: groups of eight, each over all of a row's pieces."""
    q, kv, table, n, s = _problem(4, Hq, Hkv, 256, 16, [5003, 0, 33, 9001], dtype, seed=Hq)
    _check_attention(q, kv, table, n, scales=s)
    _check_attention(q, kv, table, n, scales=s, window=3000, softcap=30.0, sinks=torch.linspace(-3.0, 3.0, Hq, device=DEV))


# ---------------------------------------------------------------------------------------------- attention: caps of the scores
@pytest.mark.parametrize("cap", [1e-3, 0.5, 5.0, 30.0, 50.0, 1e3, 1e4, 1e6, 1e12])
@pytest.mark.parametrize("spread", [1e-3, 0.05, 2.0, 30.0])
def test_paged_attention_cap_keeps_small_scores(cap, spread):
    """Capped scores keep the relative accuracy of fp32.  Scores come out of fp32 sums of 64 products (some 2^-20 of the largest one, over
    ``test_gpu_decode``'s 2^-19 with the rest); the cap adds 2^-20 of a score, and the log-sum-exp a rounding of its own.  Errors of the
    log-sum-exp are held without what the cap's size could excuse: 2^-19 of the largest score, 2^-20 of the result and 2^-22."""
    for longest in (300, 2500):
        q, kv, table, n, _ = _problem(3, 4, 2, 64, 16, [longest, 1, 77], FP16, seed=int(spread * 1000))
        q = (q.float() * spread / 2).half()
        _check_attention(q, kv, table, n, softcap=cap)
        _, lse = _ops().paged_attention(q, kv, table, n, softcap=cap, return_lse=True)
        _, want, _, big = _attention64(q, kv, table, n, 0.125, softcap=cap)
        assert ((lse.double() - want).abs() <= 2.0 ** -19 * big + 2.0 ** -20 * want.abs() + 2.0 ** -22).all()


def test_paged_attention_refuses_caps_and_scales_that_fp32_cannot_hold():
    q, kv, table, n, _ = _problem(2, 4, 2, 64, 16, [20, 20], BF16)
    for kw in (dict(softcap=1e300), dict(softcap=1e38), dict(softcap=1e-300), dict(softcap=1e-38), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(softmax_scale=1e300),
               dict(softmax_scale=float("inf"))):
        with pytest.raises(RuntimeError):
            _ops().paged_attention(q, kv, table, n, **kw)
    _no_errors()


# ---------------------------------------------------------------------------------------------- pages
def test_kv_copy_pages_onto_themselves():
    """A pair of one page leaves it as it is, and other pairs may read it; what breaks the rules does so here as on the CPU."""
    kv = torch.randn(2, 8, 2, 2, 16, 64, device=DEV).bfloat16()
    for src, dst in [((1, 1), (1, 4)), ((2, 1, 2, 2), (3, 4, 2, 5)), ((1, 0), (1, 1)), ((0, 1), (1, 1)), ((6,), (6,)), ((1, 1), (1, 1))]:
        pairs = [torch.tensor(x, dtype=torch.int32) for x in (src, dst)]
        got, want = kv.clone(), kv.cpu()
        _ops().kv_copy_pages(got, *(x.to(DEV) for x in pairs))
        try:
            _ops().kv_copy_pages(want, *pairs)
            word = 0
        except RuntimeError:
            word = 9
        torch.cuda.synchronize()
        assert int(_ops().ext().read_error_flag(True)) == word and torch.equal(got.cpu(), want), (src, dst)


def test_kv_copy_pages_refuses_scales_of_other_caches():
    kv = torch.zeros(2, 4, 2, 1, 16, 64, device=DEV).to(E4M3)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    good = torch.ones(kv.shape[:5], device=DEV)
    for bad in (good.double(), good.half(), good[:1], good[:, :3], good[:, :, :1].contiguous(), good.expand(2, 4, 2, 2, 16).contiguous(), good[..., :8].contiguous(), good[0], good.cpu()):
        with pytest.raises(RuntimeError):
            _ops().kv_copy_pages(kv, i32(0), i32(1), bad)
    _ops().kv_copy_pages(kv, i32(0), i32(1), good)
    _no_errors()


# ---------------------------------------------------------------------------------------------- drawing
@pytest.mark.parametrize("V", [5, 700, 40000])
def test_sample_tokens_at_a_temperature_without_end(V):
    """All tokens weigh the same, those of -inf and NaN nothing; of infinite logits only those count."""
    x = torch.randn(6, V, generator=torch.Generator().manual_seed(V)).to(DEV)
    x[:, 1::3], x[2, 0], x[5, 2:] = -math.inf, math.nan, math.inf
    u = torch.tensor([0.0, 0.3, 0.34, 0.66, 0.67, 0.999], device=DEV)
    for kw in ({}, dict(top_k=3), dict(top_p=0.4), dict(min_p=0.5)):
        _check_sample(x, u, temperature=math.inf, **kw)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("V", [7, 3000, 151936])
def test_sample_tokens_log_probabilities_near_zero(V, dtype):
    """A token that is almost sure: its log-probability is -log(1 + z), z the sum of the others, and keeps z's accuracy however small z is.  The weight of a
    logit 14 below: exponents of base 2 round by 2^-20 there, 2^-20.5 of the weight, the constant log2(e) by 2^-22, the exponential by 2^-22; sums and the
    logarithm add 2^-22: 2^-19 in all, of the result.  Without filters at T = 1 z is a sum of multiples of 2^-44, each off by up to 2^-45."""
    B = 24
    g = torch.Generator().manual_seed(V)
    x = torch.randn(B, V, generator=g) * 2.5
    margin = torch.linspace(0.25, 14.0, B)
    second, top = torch.arange(B) % (V - 1), V - 1
    x[::2] = -math.inf                                                  # every other row: one token beside it, margin below
    x[torch.arange(B), second] = torch.where(torch.arange(B) % 2 == 0, 1.5, x[torch.arange(B), second])
    x[:, top] = x[:, :top].max(1).values + margin
    x = x.to(dtype).to(DEV)
    u = torch.linspace(0.0, 0.999, B).to(DEV)
    lf = x.double()
    for kw in (dict(temperature=0.0), dict(top_k=3), dict(top_p=0.95), dict(min_p=1e-6, temperature=0.8), dict(temperature=1.3), {}):
        tok, lp = _ops().sample_tokens(x, u, **kw)
        _check_sample(x, u, **kw)
        t = tok.long()[:, None]
        rest = torch.exp(lf - lf.max(1, keepdim=True).values)
        rest[torch.arange(B), lf.argmax(1)] = 0.0
        want = (lf.gather(1, t) - lf.max(1, keepdim=True).values)[:, 0] - torch.log1p(rest.sum(1))
        bound = 2.0 ** -19 * want.abs() + (V * 2.0 ** -45 if kw == {} else 0.0)
        assert ((lp.double() - want).abs() <= bound).all(), (kw, ((lp.double() - want).abs() / bound).max())


# ---------------------------------------------------------------------------------------------- graphs
def _captured(f):
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = f()
    return graph, out


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_append_and_copy_in_a_graph(dtype):
    """A replay writes what its inputs hold at its time: other keys, starts, counts and pairs of pages than at the capture; nothing else is touched."""
    g = torch.Generator().manual_seed(0)
    L, n, H, P, D, B, T = 2, 20, 2, 16, 64, 3, 9
    kv = torch.randn(L, n, 2, H, P, D, generator=g).to(DEV).to(dtype)
    s = torch.rand(L, n, 2, H, P, generator=g).to(DEV) if dtype == E4M3 else None
    part = lambda x, layer: None if x is None else x[layer]  # noqa: E731
    table = torch.randperm(n, generator=g)[:6].view(3, 2).to(torch.int32).to(DEV)
    k, v = (torch.randn(B, T, H, D, generator=g).to(DEV).bfloat16() for _ in range(2))
    start, count = torch.zeros(B, dtype=torch.int32, device=DEV), torch.full((B,), T, dtype=torch.int32, device=DEV)
    rest = [p for p in range(n) if p not in table.flatten().tolist()]
    src, dst = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (rest[:3], rest[3:6]))

    def step():
        _ops().kv_append(kv[1], k, v, table, start, count, part(s, 1))
        _ops().kv_copy_pages(kv, src, dst, s)

    graph, _ = _captured(step)
    for i in range(3):
        k.copy_(torch.randn(k.shape, generator=g)), v.copy_(torch.randn(v.shape, generator=g))
        start.copy_(torch.tensor([0, 5 + i, 20], dtype=torch.int32)), count.copy_(torch.tensor([T, i, 0], dtype=torch.int32))
        dst.copy_(torch.tensor(rest[3 + i:6 + i], dtype=torch.int32))
        kept, ks = kv.clone(), None if s is None else s.clone()
        graph.replay()
        torch.cuda.synchronize()
        got, gs = kv.clone(), None if s is None else s.clone()
        kv.copy_(kept)
        if s is not None:
            s.copy_(ks)
        step()
        assert torch.equal(got.view(torch.uint8), kv.view(torch.uint8)) and (s is None or torch.equal(gs, s))
        assert not torch.equal(got.view(torch.uint8), kept.view(torch.uint8))
    _no_errors()


def test_errors_outlive_the_replay_of_a_graph_that_was_the_first_call():
    """In a process whose first call of all is captured: the error word is not part of the graph, whose replay would clear it."""
    code = """if True:
        import torch
        from surogate_b200 import ops
        q, kv = torch.zeros(1, 2, 64, device="cuda").bfloat16(), torch.zeros(2, 2, 1, 16, 64, device="cuda").bfloat16()
        table, n = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_attention(q, kv, table, n)
        torch.cuda.synchronize()
        assert ops.ext().read_error_flag(True) == 0
        ops.paged_attention(q, kv, table + 2, n)
        graph.replay()
        torch.cuda.synchronize()
        assert ops.ext().read_error_flag(True) == 8
        graph.replay()
        torch.cuda.synchronize()
        assert ops.ext().read_error_flag(True) == 0 and (out == 0).all()
    """
    done = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=200)
    assert done.returncode == 0, done.stderr[-2000:]


def test_a_decode_step_in_graphs_of_one_memory_pool():
    """Append, attention and draw captured together, twice, in one pool: the two replayed in turn give what eager calls give, whose workspaces are their own."""
    g = torch.Generator().manual_seed(3)
    B, Hq, H, D, P, V = 4, 8, 2, 64, 16, 5000
    kv = torch.zeros(200 * B, 2, H, P, D, device=DEV).bfloat16()
    table = torch.randperm(200 * B, generator=g).view(B, 200).to(torch.int32).to(DEV)
    head = torch.randn(Hq * D, V, generator=g).to(DEV).bfloat16() * 0.05
    _ops().kv_append(kv, *(torch.randn(B, 2990, H, D, generator=g).to(DEV).bfloat16() for _ in range(2)), table, torch.zeros(B, dtype=torch.int32, device=DEV))
    ins = [[torch.zeros(B, 1, H, D, device=DEV).bfloat16(), torch.zeros(B, 1, H, D, device=DEV).bfloat16(), torch.zeros(B, Hq, D, device=DEV).bfloat16(),
            torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B, device=DEV)] for _ in range(2)]

    def step(k, v, q, start, u):
        _ops().kv_append(kv, k, v, table, start)
        att = _ops().paged_attention(q, kv, table, start + 1)
        return (att,) + _ops().sample_tokens(att.reshape(B, -1) @ head, u, top_p=0.9, top_k=200)

    pool, graphs = torch.cuda.graph_pool_handle(), []
    for x in ins:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, pool=pool):
            graphs.append((graph, step(*x)))
    for t in range(6):
        x, (graph, out) = ins[t % 2], graphs[t % 2]
        for y in x[:3] + x[4:]:
            y.copy_(torch.randn(y.shape, generator=g).abs() % 1 if y.dtype == FP32 else torch.randn(y.shape, generator=g))
        x[3].copy_(torch.tensor([2990 + t, 10 + t, 1500, t], dtype=torch.int32))
        graph.replay()
        got = [y.clone() for y in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step(*x)))
    torch.cuda.synchronize()
    _no_errors()


# ---------------------------------------------------------------------------------------------- answers
def _trainer(kind="qwen3", **kw):
    from surogate_b200.runtime.trainer import Trainer, TrainerConfig

    tr = Trainer(TrainerConfig(**{**dict(model=_model(kind), batch_size=2, seq_len=256), **kw}), device=torch.device("cuda:0"))
    tr.init_weights(seed=0)
    return tr


def test_generate_raises_what_its_kernels_report(monkeypatch):
    """A page number outside the cache, which the kernels leave out and report, ends ``generate`` with that error, and none is left for the next call."""
    tr, table = _trainer(), _ops().PagedKVCache.table
    kw = dict(max_new_tokens=3, temperature=0.0)
    want = tr.generate([[5, 6, 7]], **kw)[0][0].tokens

    def wrong(self, seqs, tokens=0):
        t = table(self, seqs, tokens)
        t[0, 0] = self.num_pages
        return t

    with monkeypatch.context() as m:
        m.setattr(_ops().PagedKVCache, "table", wrong)
        with pytest.raises(RuntimeError, match="paged key/value cache"):
            tr.generate([[5, 6, 7]], **kw)
    _no_errors()
    assert tr.store.grads_enabled and tr.generate([[5, 6, 7]], **kw)[0][0].tokens == want


def test_generate_refuses_prompt_tokens_outside_the_vocabulary_before_any_launch():
    tr = _trainer()
    for bad in (-1, 4096):
        before = _ops().ext().launch_count()
        with pytest.raises(ValueError):
            tr.generate([[5, bad]], max_new_tokens=2)
        assert _ops().ext().launch_count() == before
    _no_errors()


@pytest.mark.parametrize("kind,recipe", [("qwen3", "fp8_hybrid"), ("moe", "fp8_hybrid"), ("qwen3", "nvfp4"), ("moe", "nvfp4")])
def test_generate_leaves_the_recipes_scales_alone(kind, recipe):
    """Answers before the first training step, between steps, and twice with one seed: the recipe's scales, abs-max values and copies of weights are what they
    were, bit for bit, and the same call gives the same answers."""
    import numpy as np

    tr = _trainer(kind, recipe=recipe)
    r = tr.recipe
    tensors = lambda: {n: getattr(r, n).clone() for n in ("amax_hist", "amax_cur", "scale", "scale_inv") if hasattr(r, n)}  # noqa: E731
    grouped = lambda: {k: v.clone() for k, v in (r.__dict__.get("_g_state") or {}).items() if torch.is_tensor(v)}  # noqa: E731
    g = np.random.default_rng(0)
    for step in range(3):
        before, gb, calls, copies = tensors(), grouped(), getattr(r, "calls", 0), set(r.expert_weight_cache)
        small = tr.generate([[5], list(range(140))], n=2, max_new_tokens=6, top_k=50, seed=1)
        tr.generate([list(range(900, 930))], max_new_tokens=3, seed=9)
        again = tr.generate([[5], list(range(140))], n=2, max_new_tokens=6, top_k=50, seed=1)
        if kind == "qwen3":                                              # (experts add up their tokens in no fixed order)
            assert [(c.tokens, c.logprobs) for cs in small for c in cs] == [(c.tokens, c.logprobs) for cs in again for c in cs]
        after, ga = tensors(), grouped()
        assert all(torch.equal(before[k], after[k]) for k in before) and set(gb) == set(ga) and all(torch.equal(gb[k], ga[k]) for k in gb)
        assert getattr(r, "calls", 0) == calls and set(r.expert_weight_cache) == copies
        tokens = g.integers(0, 4096, (2, 257)).astype(np.int32)
        tr.step(tokens[:, :-1], tokens[:, 1:])
    _no_errors()


@pytest.mark.parametrize("recipe,cache_dtype,mean,most", [("fp8_hybrid", None, 0.1, 0.3), ("nvfp4", None, 0.2, 1.2), ("bf16", E4M3, 0.06, 0.2)])
def test_generate_in_low_precision_agrees_with_scoring(recipe, cache_dtype, mean, most):
    """Log-probabilities of the answers against ``token_logprobs`` of the finished rows, whose tensors are quantised by other scales.  Rounding to e4m3 is 0.026
    (rms) of an element, so two passes differ by 0.037 in each of the eight products of two layers: 0.1 of the hidden state, 0.05 on logits of spread
    0.5, at most twice that in the mean and six times over all.  E2m1 in blocks rounds by 0.1: four times as much.  An e4m3 cache errs by 0.026 in
    keys (of the scores, whose spread is 1) and in values: 0.06 of the hidden state after two layers, 0.03 on the logits.  The same tokens behind
    other prompts are further away than the mean's bound, so wrong places, pages or scales would be."""
    import numpy as np

    tr = _trainer(recipe=recipe, batch_size=4)
    g = np.random.default_rng(0)
    prompts = [g.integers(0, 4096, n).tolist() for n in (100, 128, 213, 129)]
    outs = tr.generate(prompts, max_new_tokens=40, seed=3, page_size=32, cache_dtype=cache_dtype)

    def errors(prompts):
        rows = np.zeros((4, 256), np.int32)
        for i, p in enumerate(prompts):
            rows[i, :len(p) + 40] = p + outs[i][0].tokens
        lp = tr.token_logprobs(rows, np.roll(rows, -1, axis=1)).cpu()
        return torch.stack([(lp[i, len(p) - 1:len(p) + 39] - torch.tensor(outs[i][0].logprobs)).abs() for i, p in enumerate(prompts)])

    err = errors(prompts)
    assert err.mean() <= mean and err.max() <= most, (err.mean(), err.max())
    assert errors([[(t + 1) % 4096 for t in p] for p in prompts]).mean(1).min() > mean
    _no_errors()
