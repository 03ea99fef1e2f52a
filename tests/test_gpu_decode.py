"""The kernels of the answering path against plain forms in fp64: paged cache, attention over it, drawing of tokens.

Tolerances.  An attention output is rounded once to q's type, half a step of it, relative to the value; before that the weights carry 16 bits
(bf16 cache: two bf16 terms), 22 (fp16) or 11 (e4m3 cache: one fp16 term), and exponentials, sums and products are fp32 with errors of some
2^-21.  A weight's error changes an output by that share of sum p |v|, so outputs are held to
    |error| <= step(type) / 2 * |out| + (weight step + 2^-19) * sum p |v|,
and the log-sum-exp to 2^-19 * (1 + |lse|) + 2^-19 * the largest |score| (fp32 scores).  e4m3 scores see a query whose fp16 form is 2^-12 off at
most where it is not exact (bf16 queries are exact down to 2^-15 of the largest element of a row, and 2^-25 of it below)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, FP16, FP32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def _ops():
    from surogate_b200 import ops

    return ops


def _no_errors():
    _ops().check_device_errors()


def _error_word():
    torch.cuda.synchronize()
    return int(_ops().ext().read_error_flag(True))


def _pages(B, per_row, extra=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = B * per_row + extra
    return n, torch.randperm(n, generator=g)[:B * per_row].view(B, per_row).to(torch.int32).to(DEV)


def _attention64(q, kv, table, lengths, scale, window=0, softcap=0.0, sinks=None, scales=None):
    """(out, lse, sum p |v|, largest |score|) in fp64."""
    B, Hq, D = q.shape
    Hkv, P = kv.shape[2], kv.shape[3]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    mag, lse, big = out.clone(), torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device), torch.zeros(B, Hq, dtype=torch.float64, device=q.device)
    for b in range(B):
        n = int(lengths[b])
        a = max(0, n - window) if window else 0
        if n <= a:
            continue
        j = torch.arange(a, n, device=q.device)
        x = kv[table[b].long()[j // P], :, :, j % P].double()           # [n - a, 2, Hkv, D]
        if scales is not None:
            x = x * scales[table[b].long()[j // P], :, :, j % P].double().unsqueeze(-1)
        for h in range(Hq):
            k, v = x[:, 0, h // (Hq // Hkv)], x[:, 1, h // (Hq // Hkv)]
            s = (k @ q[b, h].double()) * scale
            if softcap:
                s = torch.tanh(s / softcap) * softcap
            lse[b, h] = torch.logsumexp(s, 0)
            big[b, h] = s.abs().max()
            total = lse[b, h] if sinks is None else torch.logaddexp(lse[b, h], sinks[h].double())
            p = torch.exp(s - total)
            out[b, h], mag[b, h] = p @ v, p @ v.abs()
    return out, lse, mag, big


def _check_attention(q, kv, table, lengths, **kw):
    got, lse = _ops().paged_attention(q, kv, table, lengths, return_lse=True, **kw)
    torch.cuda.synchronize()
    _no_errors()
    scale = kw.pop("softmax_scale", None) or q.shape[-1] ** -0.5
    want, wlse, mag, big = _attention64(q, kv, table, lengths, scale, **kw)
    weight = {BF16: 2.0 ** -16, FP16: 2.0 ** -21, E4M3: 2.0 ** -11}[kv.dtype]
    err = (got.double() - want).abs()
    step = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).tiny * step                             # half a step of the subnormal values
    bound = step * want.abs() + (weight + 2.0 ** -19 * (1 + big.unsqueeze(-1))) * mag * (1 + step) + tiny
    if kv.dtype == E4M3 and q.dtype == BF16:
        bound = bound + 2.0 ** -17 * (1 + big.unsqueeze(-1)) * mag     # elements of a query far below its largest
    assert got.dtype == q.dtype and (err <= bound).all(), (err / bound).max().item()
    fin = torch.isfinite(wlse)
    assert torch.equal(fin, torch.isfinite(lse)) and (lse[~fin] == -math.inf).all() and (got[~fin] == 0).all()
    lerr = (lse.double() - wlse)[fin].abs()
    lbound = (2.0 ** -19 * (1 + wlse.abs() + big) + (2.0 ** -17 * (1 + big) if kv.dtype == E4M3 else 0))[fin]
    assert (lerr <= lbound).all(), (lerr / lbound).max().item()


def _problem(B, Hq, Hkv, D, P, lengths, dtype, seed=0, width=None):
    g = torch.Generator().manual_seed(seed)
    per_row = width or max(1, (max(lengths) + P - 1) // P)
    n, table = _pages(B, per_row, seed=seed)
    qt = BF16 if dtype == E4M3 else dtype
    q = torch.randn(B, Hq, D, generator=g).to(DEV).mul(2).to(qt)
    kv = torch.randn(n, 2, Hkv, P, D, generator=g).to(DEV)
    scales = None
    if dtype == E4M3:
        from surogate_b200.ops.paged_kv import quantize_e4m3

        kv, scales = quantize_e4m3(kv * torch.rand(n, 2, Hkv, P, 1, generator=g).to(DEV) * 3)
    else:
        kv = kv.to(dtype)
    return q, kv, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), scales


# ---------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [BF16, FP16, E4M3])
@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (32, 8, 128), (8, 8, 64), (14, 2, 64), (64, 4, 128), (12, 2, 256), (20, 1, 128), (40, 1, 64), (18, 1, 256), (300, 2, 64), (7, 7, 128)])
def test_paged_attention_heads(dtype, Hq, Hkv, D):
    q, kv, table, n, s = _problem(3, Hq, Hkv, D, 16, [1, 77, 1030], dtype, seed=Hq + D)
    _check_attention(q, kv, table, n, scales=s)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
@pytest.mark.parametrize("P", [16, 32, 48, 64, 80, 128, 256])
def test_paged_attention_lengths(dtype, P):
    """Empty rows, one token, ends on and beside tile and page borders, few and many tiles (one launch, and pieces that are joined)."""
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 255, 256, 300, 2, 0]
    q, kv, table, n, s = _problem(len(lengths), 4, 2, 64, P, lengths, dtype, seed=P)
    _check_attention(q, kv, table, n, scales=s)
    lengths = [0, 1, 4097, 0, 513, 6000, 33, 0]                          # (rows that may be longer than 1024 keys are split)
    q, kv, table, n, s = _problem(len(lengths), 8, 2, 128, P, lengths, dtype, seed=P + 1)
    _check_attention(q, kv, table, n, scales=s)


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 32, 2), (256, 4, 1)])
@pytest.mark.parametrize("B", [1, 3, 180])
@pytest.mark.parametrize("capacity", [16, 1024, 1040])
def test_paged_attention_short_rows(B, D, Hq, Hkv, capacity):
    """Few and many short rows, on both sides of the capacity up to which rows stay whole, with and without a window."""
    lengths = [(i * 37) % (capacity + 1) if i else capacity for i in range(B)]
    q, kv, table, n, s = _problem(B, Hq, Hkv, D, 16, lengths, BF16, seed=B, width=capacity // 16)
    _check_attention(q, kv, table, n)
    _check_attention(q, kv, table, n, window=70)


@pytest.mark.parametrize("B,Hkv", [(1, 1), (1, 8), (2, 3), (300, 2), (1000, 1)])
def test_paged_attention_many_rows_and_one(B, Hkv):
    """One long row spread over all blocks; many rows, more than a block's threads, most of them short or empty."""
    g = torch.Generator().manual_seed(B)
    lengths = [20011] if B == 1 else [int(x) for x in torch.randint(0, 700, (B,), generator=g)]
    lengths = [0 if i % 7 == 3 else x for i, x in enumerate(lengths)]
    q, kv, table, n, s = _problem(B, 2 * Hkv, Hkv, 64, 32, lengths, BF16, seed=B)
    _check_attention(q, kv, table, n)


@pytest.mark.parametrize("window", [1, 2, 64, 65, 100, 1000, 5000])
@pytest.mark.parametrize("sinks,softcap", [(False, 0.0), (True, 0.0), (False, 20.0), (True, 5.0)])
def test_paged_attention_window_sinks_softcap(window, sinks, softcap):
    for dtype in (BF16, FP16, E4M3):
        q, kv, table, n, s = _problem(5, 8, 2, 64, 16, [1, 64, 0, 1500, 3001], dtype, seed=window)
        sk = torch.linspace(-30.0, 40.0, 8, device=DEV) if sinks else None
        _check_attention(q, kv, table, n, window=window, softcap=softcap, sinks=sk, scales=s)


def test_paged_attention_strides_and_alignment():
    """q as part of packed projections, at an odd offset (copied), and caches laid out in other orders."""
    q, kv, table, n, _ = _problem(4, 8, 2, 64, 16, [100, 700, 33, 0], BF16)
    packed = torch.randn(4, 12, 64, device=DEV).bfloat16()
    packed[:, :8] = q
    odd = torch.zeros(4 * 8 * 64 + 1, device=DEV).bfloat16()[1:].view(4, 8, 64)
    odd.copy_(q)
    want = _ops().paged_attention(q, kv, table, n)
    for x in (packed[:, :8], odd, q.transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(_ops().paged_attention(x, kv, table, n), want)
    # [pages, page size, 2, heads, dim] in memory; and pages that lie apart
    other = kv.permute(0, 3, 1, 2, 4).contiguous().permute(0, 2, 3, 1, 4)
    apart = torch.zeros(kv.shape[0], 2, 2, 2, 16, 64, device=DEV).bfloat16()
    apart[:, 1] = kv
    wide = torch.full((4, table.shape[1] + 5), -7, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    for c in (other, apart[:, 1]):
        assert torch.equal(_ops().paged_attention(q, c, table, n), want)
    assert torch.equal(_ops().paged_attention(q, kv, wide[:, :table.shape[1]], n), want)
    _check_attention(q, kv, wide, n)                                     # page numbers behind a row's last page are not looked at
    _no_errors()


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_paged_attention_ignores_what_is_not_there(dtype):
    """NaN and infinities behind a row's end, before its window and in pages of nobody do not reach the output."""
    q, kv, table, n, s = _problem(3, 4, 2, 64, 32, [70, 1, 1000], dtype)
    want = _ops().paged_attention(q, kv, table, n, window=900, scales=s)
    dirty, ds = kv.clone(), None if s is None else s.clone()
    bad = torch.full((), float("nan"), device=DEV).to(dtype)
    owned = torch.zeros(kv.shape[0], kv.shape[3], dtype=torch.bool, device=DEV)
    for b, x in enumerate([70, 1, 1000]):
        for j in range(max(0, x - 900), x):
            owned[table[b, j // 32].long(), j % 32] = True
    page, place = (~owned).nonzero(as_tuple=True)
    dirty[page, :, :, place] = bad
    if ds is not None:
        ds[page, :, :, place] = float("nan")
    else:
        dirty[page[::2], :, :, place[::2]] = float("inf")
    assert torch.equal(_ops().paged_attention(q, dirty, table, n, window=900, scales=ds), want)
    _no_errors()


def test_paged_attention_extreme_scores():
    """Scores of thousands, one key that takes all, equal keys; a first key whose score is far above the rest, and far below."""
    q, kv, table, n, _ = _problem(2, 8, 2, 64, 16, [900, 600], BF16)
    kv[:, 0] *= 40
    _check_attention(q, kv, table, n)
    kv[:, 0] = 1.0
    _check_attention(q, kv, table, n)
    first = table[:, 0].long()
    kv[first, 0, :, 0] = (q.view(2, 2, 4, 64)[:, :, 0] * 30).to(BF16)
    _check_attention(q, kv, table, n)
    kv[first, 0, :, 0] *= -1
    _check_attention(q, kv, table, n)


def test_paged_attention_e4m3_scales():
    """Scales of 2^-60 to 2^40 beside one another, rows of zeros, fp16 queries."""
    q, kv, table, n, s = _problem(2, 8, 2, 128, 16, [900, 40], E4M3)
    s[:, 1] *= torch.exp2(torch.randint(-60, 40, s[:, 1].shape, device=DEV).float())
    _check_attention(q, kv, table, n, scales=s)
    _check_attention(q.half(), kv, table, n, scales=torch.ones_like(s) * 0.01)
    kv.copy_(torch.zeros_like(kv))
    s.fill_(1.0)
    _check_attention(q, kv, table, n, scales=s)


def test_paged_attention_is_repeatable_and_runs_on_other_streams():
    q, kv, table, n, _ = _problem(6, 16, 4, 128, 16, [5000, 1, 3000, 0, 17, 9000], BF16)
    want = _ops().paged_attention(q, kv, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [_ops().paged_attention(q, kv, table, n) for _ in range(3)]
    mine = [_ops().paged_attention(q, kv, table, n) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in outs + mine)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _ops().paged_attention(q, kv, table, n)
    for lengths in ([5000, 1, 3000, 0, 17, 9000], [10, 2000, 0, 0, 8999, 31]):   # a replay sees the lengths of its time
        n.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _ops().paged_attention(q, kv, table, n))
    _no_errors()


def test_paged_attention_reports_bad_pages_and_lengths():
    """A page number outside the cache is left out and reported, so is a length beyond the row's pages; nothing else changes."""
    q, kv, table, n, _ = _problem(3, 4, 2, 64, 16, [64, 64, 64], BF16)
    good = _ops().paged_attention(q, kv, table, n)
    for bad in (-1, kv.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[1, 1] = bad
        got = _ops().paged_attention(q, kv, t, n)
        assert _error_word() == 8
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2]) and torch.isfinite(got).all()
    for bad in (65, 2 ** 31 - 1, -1):
        m = n.clone()
        m[1] = bad
        got = _ops().paged_attention(q, kv, table, m)
        assert _error_word() == 8
        assert torch.equal(got[0], good[0]) and torch.equal(got[1], good[1] if bad > 0 else torch.zeros_like(good[1]))


def test_paged_attention_refusals():
    q, kv, table, n, _ = _problem(2, 4, 2, 64, 16, [20, 20], BF16)
    att = _ops().paged_attention
    for args in [(q.half(), kv, table, n), (q.float(), kv.float(), table, n), (q[:, :3], kv, table, n), (q, kv[..., :32], table, n), (q, kv[:, :, :, :8], table, n),
                 (q, kv, table.long(), n), (q, kv, table[:1], n), (q, kv, table, n.long()), (q, kv, table, n[:1]), (q, kv.cpu(), table.cpu(), n.cpu()), (q.cpu(), kv, table, n),
                 (q, kv, table.cpu(), n), (q, kv[0], table, n), (q, kv.transpose(3, 4), table, n), (q, kv.to(E4M3), table, n)]:
        with pytest.raises(RuntimeError):
            att(*args)
    for kw in [dict(window=-1), dict(softcap=-1.0), dict(sinks=torch.zeros(3, device=DEV)), dict(scales=torch.ones(kv.shape[:4], device=DEV)), dict(softmax_scale=float("nan"))]:
        with pytest.raises(RuntimeError):
            att(q, kv, table, n, **kw)
    assert att(q[:0], kv, table[:0], n[:0]).shape == (0, 4, 64)
    _no_errors()


# ---------------------------------------------------------------------------------------------- append, pages
def test_pages_beyond_32_bit_offsets():
    """A cache of 2^32 elements and more: new tokens, copies and attention at its far end."""
    n, Hkv, P, D, T = 33000, 8, 64, 128, 70
    kv = torch.empty(n, 2, Hkv, P, D, dtype=BF16, device=DEV)
    assert kv.numel() > 2 ** 32
    table = torch.tensor([[n - 1, 5], [n - 4, n - 2]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, T, Hkv, D, generator=g).to(BF16).to(DEV) for _ in range(2))
    start, lengths = torch.zeros(2, dtype=torch.int32, device=DEV), torch.full((2,), T, dtype=torch.int32, device=DEV)
    _ops().kv_append(kv, k, v, table, start)
    for b in range(2):
        for t in (0, 63, 64, T - 1):
            assert torch.equal(kv[table[b, t // P], 0, :, t % P], k[b, t]) and torch.equal(kv[table[b, t // P], 1, :, t % P], v[b, t])
    q = torch.randn(2, 2 * Hkv, D, generator=g).to(BF16).to(DEV)
    _check_attention(q, kv, table, lengths)
    _ops().kv_copy_pages(kv[None], torch.tensor([n - 1, n - 2], dtype=torch.int32, device=DEV), torch.tensor([n - 3, 7], dtype=torch.int32, device=DEV))
    assert torch.equal(kv[n - 3, :, :, :], kv[n - 1]) and torch.equal(kv[7, :, :, :6], kv[n - 2, :, :, :6])
    _check_attention(q, kv, torch.tensor([[n - 3, 5], [n - 4, 7]], dtype=torch.int32, device=DEV), lengths)


@pytest.mark.parametrize("dtype,D,Hkv", [(BF16, 128, 8), (FP16, 64, 1), (FP32, 128, 3), (BF16, 256, 2), (BF16, 80, 3), (FP16, 8, 5)])
@pytest.mark.parametrize("T", [1, 2, 37])
def test_kv_append(dtype, D, Hkv, T):
    """Against the definition: places written as given, all others as they were, padding left out."""
    from surogate_b200.ops.paged_kv import kv_append_reference

    B, P = 5, 16
    g = torch.Generator().manual_seed(T + D)
    n, table = _pages(B, 6, seed=T)
    kv = torch.randn(n, 2, Hkv, P, D, generator=g).to(dtype).to(DEV)
    qkv = torch.randn(B, T, 4 * Hkv, D, generator=g).to(dtype).to(DEV)
    start = torch.tensor([0, 15, 16, 40, 3], dtype=torch.int32, device=DEV)
    for count in (None, torch.tensor([0, T, 1, max(1, T - 1), 0], dtype=torch.int32, device=DEV)):
        want = kv.clone()
        kv_append_reference(want, qkv[:, :, 2 * Hkv:3 * Hkv], qkv[:, :, 3 * Hkv:], table, start, count)
        got = kv.clone()
        _ops().kv_append(got, qkv[:, :, 2 * Hkv:3 * Hkv], qkv[:, :, 3 * Hkv:], table, start, count)
        assert torch.equal(got, want)
    _no_errors()


@pytest.mark.parametrize("src", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [16, 64, 80, 128, 256])
def test_kv_append_e4m3(src, D):
    """The quantised values are those of the definition, bit for bit, and the scales one fp32 division of it; a row of zeros, very small and very large rows."""
    from surogate_b200.ops.paged_kv import kv_append_reference

    B, T, P, Hkv = 3, 7, 32, 2
    g = torch.Generator().manual_seed(D)
    n, table = _pages(B, 2)
    k = torch.randn(B, T, Hkv, D, generator=g).to(DEV)
    k[0, 0], k[0, 1], k[1, 2] = 0.0, k[0, 1] * 1e-6, k[1, 2] * 1e4
    k, v = k.to(src), torch.randn(B, T, Hkv, D, generator=g).to(src).to(DEV)
    start = torch.tensor([0, 30, 5], dtype=torch.int32, device=DEV)
    got, gs = torch.zeros(n, 2, Hkv, P, D, device=DEV).to(E4M3), torch.ones(n, 2, Hkv, P, device=DEV)
    want, ws = got.clone(), gs.clone()
    kv_append_reference(want, k, v, table, start, None, ws)
    _ops().kv_append(got, k, v, table, start, None, gs)
    assert torch.equal(gs, ws) and torch.equal(got.view(torch.uint8), want.view(torch.uint8))
    _no_errors()


def test_kv_append_e4m3_ends_of_the_range():
    """fp32 rows of the largest numbers, of the smallest, of zeros of both signs, and with infinities (finite neighbours become zeros, they NaN)."""
    from surogate_b200.ops.paged_kv import kv_append_reference

    T, D, P = 12, 64, 16
    n, table = _pages(1, 1)
    k = torch.randn(1, T, 1, D, generator=torch.Generator().manual_seed(2)).to(DEV)
    for t, scale in enumerate((3.0e38 / 6, 1e30, 1e-30, 1e-37, 1e-40, 1e-44)):
        k[0, t] *= scale
    k[0, 6] = torch.where(k[0, 6] > 0, 0.0, -0.0)
    k[0, 7, :, ::3] = -0.0
    k[0, 8, :, 5] = float("inf")
    k[0, 9, :, 6] = -float("inf")
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    got, gs = torch.zeros(n, 2, 1, P, D, device=DEV).to(E4M3), torch.ones(n, 2, 1, P, device=DEV)
    want, ws = got.clone(), gs.clone()
    kv_append_reference(want, k, -k, table, start, None, ws)
    _ops().kv_append(got, k, -k, table, start, None, gs)
    assert torch.equal(gs, ws)
    a, b = got.view(torch.uint8), want.view(torch.uint8)
    nan = (b & 0x7f) == 0x7f                                           # a NaN's sign means nothing
    assert torch.equal((a & 0x7f) == 0x7f, nan) and torch.equal(a[~nan], b[~nan])
    _no_errors()


def test_kv_append_odd_sources_and_bad_places():
    B, T, P, Hkv, D = 3, 4, 16, 2, 64
    n, table = _pages(B, 2)
    k = torch.randn(B * T * Hkv * D + 1, device=DEV).bfloat16()[1:].view(B, T, Hkv, D)     # not 16-byte aligned
    v = torch.randn(T, B, D, Hkv, device=DEV).bfloat16().permute(1, 0, 3, 2)               # elements not contiguous
    start = torch.tensor([0, 3, 14], dtype=torch.int32, device=DEV)
    a, b = torch.zeros(n, 2, Hkv, P, D, device=DEV).bfloat16(), torch.zeros(n, 2, Hkv, P, D, device=DEV).bfloat16()
    _ops().kv_append(a, k, v, table, start)
    _ops().kv_append(b, k.clone(), v.contiguous(), table, start)
    assert torch.equal(a, b) and a.abs().sum() > 0
    # the same places in a cache with another order of its dimensions
    c = torch.zeros(n, P, 2, Hkv, D, device=DEV).bfloat16().permute(0, 2, 3, 1, 4)
    _ops().kv_append(c, k, v, table, start)
    assert torch.equal(c, a)
    _no_errors()
    # a start beyond the row, a negative one, pages of nobody: reported, and only those tokens are missing
    for s, t in ((torch.tensor([0, 30, 14]), table), (torch.tensor([0, -2, 14]), table)):
        d = torch.zeros_like(a)
        _ops().kv_append(d, k, v, t, s.to(torch.int32).to(DEV))
        assert _error_word() == 8
        assert torch.equal(d[table[0].long()], a[table[0].long()])
    bad = table.clone()
    bad[1] = n
    d = torch.zeros_like(a)
    _ops().kv_append(d, k, v, bad, start)
    assert _error_word() == 8 and d[table[1].long()].abs().sum() == 0 and torch.equal(d[table[2].long()], a[table[2].long()])


def test_kv_append_refusals():
    n, table = _pages(2, 2)
    kv = torch.zeros(n, 2, 2, 16, 64, device=DEV).bfloat16()
    k = torch.zeros(2, 3, 2, 64, device=DEV).bfloat16()
    start = torch.zeros(2, dtype=torch.int32, device=DEV)
    for args in [(kv, k, k.half(), table, start), (kv, k.half(), k.half(), table, start), (kv, k[:, :2], k, table, start), (kv, k[..., :32], k[..., :32], table, start),
                 (kv[:, :1], k, k, table, start), (kv[:, :, :, :8], k, k, table, start), (kv, k, k, table.long(), start), (kv, k, k, table, start.long()),
                 (kv, k, k, table[:1], start), (kv, k, k, table, start[:1]), (kv.to(E4M3), k, k, table, start), (kv, k.cpu(), k.cpu(), table, start)]:
        with pytest.raises(RuntimeError):
            _ops().kv_append(*args)
    with pytest.raises(RuntimeError):
        _ops().kv_append(kv, k, k, table, start, None, torch.ones(kv.shape[:4], device=DEV))
    _ops().kv_append(kv, k[:0], k[:0], table[:0], start[:0])
    _ops().kv_append(kv, k[:, :0], k[:, :0], table, start)
    _no_errors()


@pytest.mark.parametrize("L,n,P,dtype", [(1, 1, 16, BF16), (3, 5, 16, FP16), (2, 40, 48, FP32), (5, 300, 16, E4M3), (36, 7, 64, BF16)])
def test_kv_copy_pages(L, n, P, dtype):
    pages = 2 * n + 3
    g = torch.Generator().manual_seed(n)
    kv = torch.randn(L, pages, 2, 2, P, 64, generator=g).to(DEV).to(dtype)
    scales = torch.rand(L, pages, 2, 2, P, generator=g).to(DEV) if dtype == E4M3 else None
    order = torch.randperm(pages, generator=g).to(torch.int32).to(DEV)
    src, dst = order[:n].contiguous(), order[n:2 * n].contiguous()
    if n > 4:
        src[1] = src[0]                                                 # one page forked twice
    want, ws = kv.clone(), None if scales is None else scales.clone()
    bits = lambda t: t.view(torch.uint8)  # noqa: E731
    bits(want)[:, dst.long()] = bits(kv)[:, src.long()]
    if ws is not None:
        ws[:, dst.long()] = scales[:, src.long()]
    _ops().kv_copy_pages(kv, src, dst, scales)
    assert torch.equal(bits(kv), bits(want)) and (ws is None or torch.equal(scales, ws))
    _no_errors()


def test_kv_copy_pages_reports_what_breaks_the_rules():
    kv = torch.randn(2, 8, 2, 2, 16, 64, device=DEV).bfloat16()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for src, dst, word, done in [((0, 1), (2, 2), 9, ()), ((0, 1, 3), (1, 4, 5), 9, ((1, 4), (3, 5))), ((0, 1), (8, 3), 8, ((1, 3),)), ((-1, 1), (2, 3), 8, ((1, 3),)),
                                 ((2, 1), (2, 3), 0, ((1, 3),))]:
        x, want = kv.clone(), kv.clone()
        for a, b in done:
            want[:, b] = kv[:, a]
        _ops().kv_copy_pages(x, i32(*src), i32(*dst))
        assert _error_word() == word and torch.equal(x, want), (src, dst)
    for args in [(kv[0], i32(0), i32(1)), (kv, i32(0), i32(1, 2)), (kv, i32(0).long(), i32(1)), (kv.transpose(2, 3), i32(0), i32(1)), (kv, i32(0).cpu(), i32(1).cpu()), (kv.to(E4M3), i32(0), i32(1))]:
        with pytest.raises(RuntimeError):
            _ops().kv_copy_pages(*args)
    _ops().kv_copy_pages(kv, i32(), i32())
    _no_errors()


# ---------------------------------------------------------------------------------------------- drawing
def _logits(B, V, dtype, seed=0, sigma=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, V, generator=g) * sigma).to(dtype).to(DEV)


def _check_sample(logits, u, **kw):
    """Tokens equal to the definition's in fp64; the log-probability within fp32's errors (2^-20 of the largest term, one rounding)."""
    from surogate_b200.ops.sampling import _each, sample_tokens_reference

    B = logits.shape[0]
    tok, lp = _ops().sample_tokens(logits, u, **kw)
    f = lambda name, d, t=FP32: _each(kw.get(name, d), B, t, DEV)  # noqa: E731
    want, wlp = sample_tokens_reference(logits, u, f("temperature", 1.0), f("top_k", 0, torch.int32), f("top_p", 1.0), f("min_p", 0.0))
    torch.cuda.synchronize()
    assert tok.dtype == torch.int32 and torch.equal(tok, want), (tok != want).nonzero().flatten().tolist()
    fin = torch.isfinite(wlp)
    assert torch.equal(lp[~fin], wlp[~fin])
    assert ((lp - wlp)[fin].abs() <= 2.0 ** -20 * (8 + wlp[fin].abs())).all()
    _no_errors()


def _uniform(B, seed=0):
    return torch.rand(B, generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("V", [1, 2, 7, 31, 513, 4096, 32001, 128256, 151936])
def test_sample_tokens(dtype, V):
    B = 24
    x, u = _logits(B, V, dtype, seed=V), _uniform(B, V)
    for kw in [{}, dict(temperature=0.0), dict(temperature=0.7, top_k=20, top_p=0.8, min_p=0.01), dict(top_p=0.9), dict(top_k=1), dict(top_k=5), dict(top_k=1000, top_p=0.95),
               dict(min_p=0.1), dict(min_p=1.0), dict(temperature=2.0, top_p=0.3), dict(top_k=V), dict(top_p=1.0, min_p=0.0), dict(temperature=1e-3), dict(temperature=50.0, top_p=0.999)]:
        _check_sample(x, u, **kw)


@pytest.mark.parametrize("B", [1, 2, 150, 700])
def test_sample_tokens_parameters_of_rows(B):
    V = 5003
    r = torch.arange(B, device=DEV)
    x, u = _logits(B, V, FP32, seed=B), _uniform(B, B)
    _check_sample(x, u, temperature=torch.where(r % 3 == 0, 0.0, 0.5 + (r % 5) / 4.0), top_k=torch.where(r % 2 == 0, 40, 0).to(torch.int32),
                  top_p=torch.where(r % 4 == 1, 0.7, 1.0), min_p=torch.where(r % 5 == 2, 0.05, 0.0))


@pytest.mark.parametrize("V", [700, 40000])
@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_sample_tokens_ties(V, dtype):
    """All logits equal; a few levels only; the cut inside a run of equal logits, longer than any list."""
    B = 12
    u = torch.linspace(0, 0.999999, B).to(DEV)
    flat = torch.zeros(B, V, device=DEV).to(dtype)
    levels = (torch.randint(0, 4, (B, V), generator=torch.Generator().manual_seed(V)).float() * 0.5).to(dtype).to(DEV)
    signed = torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0).expand(B, V).to(dtype).contiguous()
    for x in (flat, levels, signed):
        for kw in [{}, dict(temperature=0.0), dict(top_k=1), dict(top_k=600), dict(top_k=V - 1), dict(top_p=0.5), dict(top_p=0.25, top_k=100), dict(top_p=0.999), dict(min_p=0.6),
                   dict(min_p=0.3, top_p=0.37)]:
            _check_sample(x, u, **kw)


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("V", [300, 30011, 151936])
@pytest.mark.parametrize("sigma", [0.05, 1.0, 4.0])
def test_sample_tokens_top_p_alone(sigma, V, dtype):
    """From rows that are almost flat to peaked ones; in half of them a few tokens stand out; shares from one token to all but the lightest."""
    B = 6
    x = _logits(B, V, FP32, seed=V, sigma=sigma)
    x[::2, 7::V // 3] += 9.0
    x, u = x.to(dtype), _uniform(B, V)
    for temperature in (0.3, 1.0, 1.7, 8.0):
        for top_p in (1e-6, 0.05, 0.5, 0.9, 0.99, 0.999999):
            _check_sample(x, u, temperature=temperature, top_p=top_p)


def test_sample_tokens_crowded_bins():
    """Logits crowded at two places, so that bins have to be divided again and again, down to neighbouring fp32 values."""
    B, V = 6, 30000
    g = torch.Generator().manual_seed(1)
    base = torch.rand(B, V, generator=g) * 1e-3
    step = torch.nextafter(torch.tensor(1.0), torch.tensor(2.0)) - 1.0
    near = 1.0 + torch.randint(0, 3, (B, V), generator=g).float() * step
    far = torch.where(torch.rand(B, V, generator=g) < 0.5, near, base - 20.0)
    u = _uniform(B)
    for x in (base, near, far):
        for kw in [dict(top_k=3000), dict(top_k=V // 2), dict(top_p=0.4), dict(top_k=20000, top_p=0.9), dict(temperature=0.05, top_p=0.5)]:
            _check_sample(x.to(DEV), u, **kw)


def test_sample_tokens_masked_and_empty_rows():
    V = 9000
    x = _logits(8, V, FP32)
    lowest = torch.finfo(FP32).min
    x[0] = -float("inf")
    x[1] = float("nan")
    x[2, 1:] = -float("inf")
    x[3, :8000] = lowest
    x[4] = lowest
    x[5, 17] = float("inf")
    x[5, 4000] = float("inf")
    x[6, ::2] = float("nan")
    x[7, 5:] = -float("inf")
    u = torch.tensor([0.3, 0.3, 0.9, 0.5, 0.5, 0.7, 0.5, 0.99], device=DEV)
    for kw in [{}, dict(temperature=0.0), dict(top_k=3), dict(top_p=0.9), dict(min_p=0.2), dict(top_k=100, top_p=0.5, temperature=0.6), dict(top_k=8999, temperature=3.0)]:
        _check_sample(x, u, **kw)
    tok, lp = _ops().sample_tokens(x, u)
    assert tok[:2].tolist() == [-1, -1] and (lp[:2] == -float("inf")).all() and tok[2] == 0 and tok[5] in (17, 4000)


def test_sample_tokens_parameters_at_their_ends():
    x = _logits(5, 2000, FP32)
    u = torch.tensor([0.0, 1.0, 0.9999999, float("nan"), -1.0], device=DEV)
    for kw in [{}, dict(top_p=0.0), dict(top_p=-1.0), dict(min_p=2.0), dict(top_k=-3), dict(top_k=10 ** 9), dict(top_p=float("nan")), dict(temperature=1e-30), dict(top_p=1e-9)]:
        _check_sample(x, torch.nan_to_num(u, nan=0.0), **kw)
        _ops().sample_tokens(x, u, **kw)
    _no_errors()


def test_sample_tokens_layouts_streams_and_graphs():
    B, V = 7, 33333
    big = _logits(B, V + 5, BF16)
    u = _uniform(B)
    for x in (big[:, 3:V], big[:, :V - 1], big[::2, 1:], big.t().contiguous().t()):
        _check_sample(x, _uniform(x.shape[0]), top_p=0.8)
    x = _logits(B, V, FP32)
    want = _ops().sample_tokens(x, u, top_k=50, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = _ops().sample_tokens(x, u, top_k=50, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b = _ops().sample_tokens(x, u, top_k=50, top_p=0.9)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for y in (a, b) for p, q in zip(y, want))
    u.copy_(_uniform(B, 5))
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(b, _ops().sample_tokens(x, u, top_k=50, top_p=0.9)))


@pytest.mark.parametrize("V", [900001])
def test_sample_tokens_vocabulary_beyond_shared_memory(V):
    for dtype in (FP32, BF16):
        x = _logits(2, V, dtype)
        for kw in [{}, dict(top_p=0.5), dict(top_k=1000)]:
            _check_sample(x, _uniform(2), **kw)


@pytest.mark.parametrize("B,V", [(1, 2 ** 20 - 1), (100000, 40), (3000, 1)])
def test_sample_tokens_largest_and_most_rows(B, V):
    g = torch.Generator(device=DEV).manual_seed(V)
    x, u = torch.randn(B, V, generator=g, device=DEV) * 3, torch.rand(B, generator=g, device=DEV)
    tok, lp = _ops().sample_tokens(x, u, top_p=0.8)
    rows = torch.arange(0, B, max(1, B // 50), device=DEV)
    _check_sample(x[rows].contiguous(), u[rows], top_p=0.8)
    assert torch.equal(_ops().sample_tokens(x[rows].contiguous(), u[rows], top_p=0.8)[0], tok[rows])
    _check_sample(x[rows].contiguous(), u[rows], temperature=0.9, top_k=7)


def test_sample_tokens_rows_far_apart():
    """Rows whose offsets pass 2^31 elements, one row of the tensor used twice, and calls on two streams at once."""
    V, far = 30000, 2 ** 30 + 8
    x = torch.as_strided(torch.empty(2 * far + V, device=DEV), (3, V), (far, 1))
    x.copy_(_logits(3, V, FP32, seed=4))
    u = _uniform(3, 4)
    _check_sample(x, u, top_p=0.9)
    _check_sample(x[2:].expand(5, V), _uniform(5), temperature=0.8, top_k=30)
    y, v = _logits(200, V, BF16, seed=5), _uniform(200, 5)
    want = _ops().sample_tokens(x, u, top_p=0.7), _ops().sample_tokens(y, v, top_p=0.7)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        got = []
        for s, (a, b) in zip(streams, ((x, u), (y, v))):
            with torch.cuda.stream(s):
                got.append(_ops().sample_tokens(a, b, top_p=0.7))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for w, g in zip(want, got) for p, q in zip(w, g))
    _no_errors()


def test_sample_tokens_follows_the_distribution():
    """50000 draws of 40 tokens: counts within six standard deviations of the softmax's."""
    n, V = 50000, 40
    x = _logits(1, V, FP32, sigma=1.5).expand(n, V).contiguous()
    tok, _ = _ops().sample_tokens(x, _uniform(n))
    p = torch.softmax(x[0].double(), 0)
    assert ((torch.bincount(tok.long(), minlength=V) - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt() + 1).all()


def test_sample_tokens_refusals():
    x, u = _logits(3, 100, FP32), _uniform(3)
    for args, kw in [((x.double(), u), {}), ((x, u.double()), {}), ((x, u[:2]), {}), ((x[0], u), {}), ((x, u), dict(temperature=-1.0)), ((x, u), dict(temperature=float("nan"))),
                     ((x, u), dict(temperature=torch.ones(2, device=DEV))), ((x, u), dict(top_k=torch.ones(3, device=DEV))), ((x, u), dict(top_p=torch.ones(3))), ((x[:, :0], u), {}), ((torch.zeros(1, 1 << 20, device=DEV), u[:1]), {}),
                     ((x, u.cpu()), {})]:
        with pytest.raises(RuntimeError):
            _ops().sample_tokens(*args, **kw)
    assert _ops().sample_tokens(x[:0], u[:0])[0].shape == (0,)


# ---------------------------------------------------------------------------------------------- a run of them together
def _model(kind):
    if kind == "qwen3":
        return dict(architecture="Qwen3ForCausalLM", vocab_size=4096, d_model=512, n_layers=2, num_query_heads=4, num_kv_heads=2, head_size=128, d_ff=1536, tie_word_embeddings=True)
    if kind == "llama":
        return dict(architecture="LlamaForCausalLM", vocab_size=4096, d_model=512, n_layers=2, num_query_heads=8, num_kv_heads=2, head_size=64, d_ff=1536)
    if kind == "moe":
        return dict(architecture="Qwen3MoeForCausalLM", vocab_size=4096, d_model=512, n_layers=2, num_query_heads=4, num_kv_heads=2, head_size=128, num_experts=8,
                    num_experts_per_tok=2, moe_d_ff=256)
    return dict(architectures=["GptOssForCausalLM"], model_type="gpt_oss", vocab_size=4096, hidden_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                head_dim=64, intermediate_size=256, num_local_experts=4, num_experts_per_tok=2, sliding_window=32, max_position_embeddings=4096, rms_norm_eps=1e-5,
                rope_theta=150000.0, layer_types=["sliding_attention", "full_attention"], tie_word_embeddings=False)


@pytest.mark.parametrize("kind", ["qwen3", "llama", "moe", "gpt_oss"])
def test_generate_agrees_with_scoring(kind):
    """``Trainer.generate`` on the cache against ``token_logprobs`` of the finished rows.  Two bf16 passes over two layers: some sixteen
    independent roundings of 2^-9 leave 1 % on the hidden state, so 0.005 on logits of spread 0.5; six times that, and half a step (2^-8) of bf16
    logits below 2 on the scoring side, stay below 0.05.  Routed experts may be chosen differently for single tokens; there the mean is held."""
    import numpy as np

    from surogate_b200.runtime import generation
    from surogate_b200.runtime.trainer import Trainer, TrainerConfig

    tr = Trainer(TrainerConfig(model=_model(kind), batch_size=4, seq_len=256, recipe="bf16"), device=torch.device("cuda:0"))
    tr.init_weights(seed=0)
    assert generation.cache_layout(tr.cm, tr.device) is not None
    g = np.random.default_rng(0)
    prompts = [g.integers(0, 4096, n).tolist() for n in (1, 100, 128, 213)]
    before = _ops().ext().launch_count()
    outs = tr.generate(prompts, n=3, max_new_tokens=40, temperature=1.0, top_p=0.9, seed=3, page_size=32, prompt_rows=3)
    assert _ops().ext().launch_count() > before + 40 * 2 * 3
    _no_errors()
    for p, cs in zip(prompts, outs):
        assert len({tuple(c.tokens) for c in cs}) == 3
        rows = np.zeros((3, 256), np.int32)
        for i, c in enumerate(cs):
            rows[i, :len(p) + 40] = p + c.tokens
        tgt = np.roll(rows, -1, axis=1)
        want = tr.token_logprobs(np.vstack([rows, rows[:1]]), np.vstack([tgt, tgt[:1]]))[:3, len(p) - 1:len(p) + 39].cpu()
        err = (torch.tensor([c.logprobs for c in cs]) - want).abs()
        assert (err.max() if kind in ("qwen3", "llama") else err.mean()) < 0.05, err.max()
    again = tr.generate(prompts, n=3, max_new_tokens=40, temperature=1.0, top_p=0.9, seed=3, page_size=32, prompt_rows=3)
    if kind in ("qwen3", "llama"):
        assert [c.tokens for cs in again for c in cs] == [c.tokens for cs in outs for c in cs]
    small = tr.generate(prompts[:2], n=2, max_new_tokens=8, temperature=0.0, cache_dtype=E4M3)
    assert all(len(c.tokens) == 8 and all(math.isfinite(x) for x in c.logprobs) for cs in small for c in cs)
    _no_errors()


@pytest.mark.parametrize("recipe", ["fp8_hybrid", "nvfp4"])
def test_generate_under_low_precision_recipes(recipe):
    """Single tokens and padded prompts run through the recipes' products; the answers are tokens with finite log-probabilities."""
    from surogate_b200.runtime.trainer import Trainer, TrainerConfig

    tr = Trainer(TrainerConfig(model=_model("qwen3"), batch_size=2, seq_len=256, recipe=recipe), device=torch.device("cuda:0"))
    tr.init_weights(seed=0)
    outs = tr.generate([[5], list(range(140))], n=2, max_new_tokens=12, top_k=50, seed=1)
    assert all(len(c.tokens) == 12 and all(math.isfinite(x) and x <= 0 for x in c.logprobs) for cs in outs for c in cs)
    _no_errors()


def test_generate_with_fp32_activations_runs_whole_passes():
    from surogate_b200.runtime.trainer import Trainer, TrainerConfig

    tr = Trainer(TrainerConfig(model=_model("qwen3"), batch_size=2, seq_len=256, param_dtype="fp32", grad_dtype="fp32", backend="ref"), device=torch.device("cuda:0"))
    tr.init_weights(seed=0)
    assert len(tr.generate([[5, 6]], max_new_tokens=3, temperature=0.0)[0][0].tokens) == 3
    with pytest.raises(ValueError):
        tr.generate([[5, 6]], cache_dtype=FP32)


def test_decode_step_of_a_forked_group_on_one_cache():
    """Append, fork, diverge, compact, attend: one prompt's three completions on two layers of an e4m3 cache against caches that were never shared."""
    L, H, D, P = 2, 2, 64, 16
    g = torch.Generator().manual_seed(0)
    shared, alone = (_ops().PagedKVCache(L, 40, P, H, D, 4, dtype=E4M3, device=DEV) for _ in range(2))
    prompt = torch.randn(L, 2, 1, 21, H, D, generator=g).to(DEV).bfloat16()
    new = torch.randn(30, L, 2, 3, 1, H, D, generator=g).to(DEV).bfloat16()
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    shared.reserve({0: 21})
    for s in range(3):
        alone.reserve({s: 21})
    for layer in range(L):
        shared.append(layer, prompt[layer, 0], prompt[layer, 1], shared.table([0]), zero)
        for s in range(3):
            alone.append(layer, prompt[layer, 0], prompt[layer, 1], alone.table([s]), zero)
    shared.fork(0, [1, 2])
    q = torch.randn(3, 4, D, generator=g).to(DEV).bfloat16()
    for t in range(30):
        start = torch.full((3,), 21 + t, dtype=torch.int32, device=DEV)
        for c in (shared, alone):
            c.reserve({0: 1, 1: 1, 2: 1})
            for layer in range(L):
                c.append(layer, new[t, layer, 0], new[t, layer, 1], c.table([0, 1, 2]), start)
        if t == 15:
            shared.fork(2, [3])
            shared.free(2)
            shared.fork(3, [2])
            shared.free(3)
            shared.compact()
        for layer in range(L):
            a, b = (c.attend(layer, q, c.table([0, 1, 2]), start + 1) for c in (shared, alone))
            assert torch.equal(a, b)
    assert shared.free_pages > alone.free_pages
    _no_errors()
