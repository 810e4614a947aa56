"""Paged attention in 16-bit types: what the float32 probabilities lose on
their way through the tensor cores, and values that are not finite."""
import pytest
import torch

import serving_reference as R
from walsh_research_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = [torch.float16, torch.bfloat16]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def attend(q, k, v, pos0, window=0, sinks=0):
    """As serving_reference.attend with a bound in which each probability is
    held by two terms of q's type: off by half a step of a half step relative,
    and in float16, whose smallest step is 2^-24, by 2^-25 of the largest."""
    dt, hd, L = q.dtype, q.shape[-1], k.shape[0]
    half = torch.finfo(dt).eps / 2
    q, k, v = (t.double() for t in (q, k, v))
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    i, j = pos0 + torch.arange(q.shape[0], device=q.device)[:, None], torch.arange(L, device=q.device)[None]
    see = j <= i
    if window:
        see = see & ((j > i - window) | (j < sinks))
    scale = hd ** -0.5
    s = torch.einsum("thd,jhd->htj", q, k) * scale
    s_abs = torch.einsum("thd,jhd->htj", q.abs(), k.abs()).masked_fill(~see, 0.0).amax(-1) * scale
    p = torch.exp(s - s.masked_fill(~see, float("-inf")).amax(-1, keepdim=True)).masked_fill(~see, 0.0)
    l = p.sum(-1, keepdim=True)
    o = torch.einsum("htj,jhd->thd", p / l, v)
    a = torch.einsum("htj,jhd->thd", p / l, v.abs())
    seen = torch.einsum("htj,jhd->thd", see.double().expand_as(p) / l, v.abs())
    # scores: hd products summed in float32, good exponentials; sums over the keys in at least 16 parts
    d = 2 * (2.0 ** -24 * (hd + 4) * s_abs + 2.0 ** -22) + 2 * (L / 16 + 64) * 2.0 ** -24
    least = 2.0 ** -25 if dt is torch.float16 else 0.0
    return o, half * o.abs() + (half * half + d.t()[..., None]) * a + least * seen + torch.finfo(dt).tiny * torch.finfo(dt).eps


def close(got, want, bound):
    got = got.double()
    assert not torch.isnan(got).any()
    d = (got - want).abs()
    assert (d <= bound).all(), f"{int((d > bound).sum())} of {d.numel()} off, worst {float((d / bound).max()):.3g} bounds"


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hk,hd", [(32, 32, 16), (4, 2, 32), (8, 1, 64), (6, 2, 128), (20, 1, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 3)])
def test_prefill_keeps_probabilities_in_two_terms(dtype, hq, hk, hd, window, sinks):
    g = gen(hd + hq)
    new, past = [200, 70], [0, 150]
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [a + b for a, b in zip(new, past)], hk, 16, hd, dtype))
    q = (1.5 * torch.randn(sum(new), hq, hd, generator=g)).to(dtype).to(DEV)
    off = torch.tensor([0] + new).cumsum(0).int().to(DEV)
    out = ops.paged_prefill_attention(q, off, kp, vp, table, kl, window=window, sinks=sinks)
    at = 0
    for b, t in enumerate(new):
        k, v = (R.gather_keys(p, table[b], past[b] + t) for p in (kp, vp))
        close(out[at:at + t], *attend(q[at:at + t], k, v, past[b], window, sinks))
        at += t


@pytest.mark.parametrize("dtype", HALF + [torch.float32])
@pytest.mark.parametrize("hq,hk,hd", [(32, 32, 16), (4, 2, 32), (8, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 3)])
def test_prefill_with_rounded_probabilities(dtype, hq, hk, hd, window, sinks):
    """serving_reference.attend's bound counts one rounding of each probability; float32 has none."""
    g = gen(hd + hq)
    new, past = [200, 70], [0, 150]
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [a + b for a, b in zip(new, past)], hk, 16, hd, dtype))
    q = (1.5 * torch.randn(sum(new), hq, hd, generator=g)).to(dtype).to(DEV)
    off = torch.tensor([0] + new).cumsum(0).int().to(DEV)
    out = ops.paged_prefill_attention(q, off, kp, vp, table, kl, window=window, sinks=sinks, rounded=True)
    if dtype is torch.float32:
        assert torch.equal(out, ops.paged_prefill_attention(q, off, kp, vp, table, kl, window=window, sinks=sinks))
    at = 0
    for b, t in enumerate(new):
        k, v = (R.gather_keys(p, table[b], past[b] + t) for p in (kp, vp))
        close(out[at:at + t], *R.attend(q[at:at + t], k, v, past[b], window, sinks))
        at += t


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("hq,hk,hd", [(8, 8, 16), (8, 1, 64), (9, 1, 16), (16, 1, 32), (24, 2, 64), (40, 2, 128)])
def test_decode_keeps_probabilities_in_two_terms(dtype, hq, hk, hd):
    g = gen(hd + hq)
    lens = [700, 33, 1, 2500]
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, lens, hk, 16, hd, dtype))
    q = (1.5 * torch.randn(len(lens), hq, hd, generator=g)).to(dtype).to(DEV)
    for window, sinks in ((0, 0), (300, 2)):
        out = ops.paged_attention(q, kp, vp, table, kl, window=window, sinks=sinks)
        for b, n in enumerate(lens):
            k, v = (R.gather_keys(p, table[b], n) for p in (kp, vp))
            close(out[b:b + 1], *attend(q[b:b + 1], k, v, n - 1, window, sinks))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_limits_past_31_bits_see_everything(dtype):
    g = gen(4)
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [50, 7], 2, 16, 32, dtype))
    q = torch.randn(2, 4, 32, generator=g).to(dtype).to(DEV)
    off = torch.arange(3, dtype=torch.int32, device=DEV)
    want = ops.paged_attention(q, kp, vp, table, kl), ops.paged_prefill_attention(q, off, kp, vp, table, kl)
    for kw in (dict(window=2 ** 31 - 1), dict(window=2 ** 40), dict(window=3, sinks=2 ** 31), dict(window=2 ** 31, sinks=2 ** 33)):
        assert torch.equal(ops.paged_attention(q, kp, vp, table, kl, max_len=2 ** 40, **kw), want[0])
        assert torch.equal(ops.paged_prefill_attention(q, off, kp, vp, table, kl, **kw), want[1])


def test_positions_past_32_bits_are_reported_whatever_the_slots_type():
    n, h, hd, page = 4, 2, 16, 4
    x = torch.ones(n, h, hd, dtype=torch.float16, device=DEV)
    t = torch.ones(3, hd // 2, device=DEV)
    pos = torch.tensor([0, 2 ** 32 + 1, 2, -2 ** 32], device=DEV)
    for slots in (torch.tensor([0, 1, 2, 3], dtype=i, device=DEV) for i in (torch.int32, torch.int64)):
        kp = torch.zeros(1, h, page, hd, dtype=torch.float16, device=DEV)
        vp = torch.zeros_like(kp)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        q = ops.paged_append(x, x, x, kp, vp, slots, positions=pos, rope=(t, t * 0), err=err)
        assert int(err) == -9
        for y in (q, kp[0].transpose(0, 1), vp[0].transpose(0, 1)):
            assert (y[[0, 2]] == 1).all() and not y[[1, 3]].any()
    # and slots past 32 bits beside int32 positions
    err.zero_()
    slots = torch.tensor([0, 2 ** 32 + 1, 2, 3], device=DEV)
    ops.paged_append(None, x, 2 * x, kp, vp, slots, positions=torch.zeros(n, dtype=torch.int32, device=DEV), rope=(t, t * 0), err=err)
    assert int(err) == -9 and (vp[0, :, [0, 2, 3]] == 2).all() and not vp[0, :, 1].any()


def test_prefill_bound_of_zero_still_computes_the_spans():
    """max_q only sizes the grid; a bound that is too small is not an empty call."""
    g = gen(6)
    for dtype in (torch.float16, torch.float32):
        kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [90, 7], 2, 16, 32, dtype))
        q = torch.randn(97, 4, 32, generator=g).to(dtype).to(DEV)
        off = torch.tensor([0, 90, 97], dtype=torch.int32, device=DEV)
        out = torch.full_like(q, 7.0)
        want = ops.paged_prefill_attention(q, off, kp, vp, table, kl)
        assert torch.equal(ops.paged_prefill_attention(q, off, kp, vp, table, kl, max_q=0, out=out), want)


@pytest.mark.parametrize("dtype", HALF + [torch.float32])
@pytest.mark.parametrize("hq,hk,hd", [(4, 2, 16), (8, 1, 64), (2, 2, 128)])
def test_attention_in_place_with_hidden_values_that_are_not_finite(dtype, hq, hk, hd):
    """out may be q: rows computed again (hidden NaN and infinities) read their queries as they were."""
    g = gen(7)
    n = 90
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [n], hk, 16, hd, dtype))
    for j, x in ((40, float("nan")), (77, float("inf")), (89, float("nan"))):
        vp[int(table[0, j // 16]), :, j % 16] = x
    q = torch.randn(n, hq, hd, generator=g).to(dtype).to(DEV)
    off = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    want = ops.paged_prefill_attention(q, off, kp, vp, table, kl, window=20, sinks=2)
    mine = q.clone()
    assert ops.paged_prefill_attention(mine, off, kp, vp, table, kl, window=20, sinks=2, out=mine) is mine
    assert torch.equal(mine.nan_to_num(9.0), want.nan_to_num(9.0)) and torch.isfinite(want[:40].float()).all()
    one = q[:1].clone()
    want = ops.paged_attention(one, kp, vp, table, kl, window=12)
    assert torch.equal(ops.paged_attention(one, kp, vp, table, kl, window=12, out=one).nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", HALF + [torch.float32])
@pytest.mark.parametrize("hq,hk,hd", [(1, 1, 16), (8, 1, 64), (16, 1, 32), (20, 1, 128), (8, 2, 128)])
@pytest.mark.parametrize("n", [40, 3000])
def test_decode_infinite_values_of_tiny_probability(dtype, hq, hk, hd, n):
    """A value that is infinite reaches its channel although its probability,
    e^-25, is nothing in float16; other channels stay as they are."""
    g = gen(n + hd)
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [n, 30], hk, 16, hd, dtype))
    kp.zero_()
    j = n // 2 + 3
    page, row = int(table[0, j // 16]), j % 16
    kp[page, :, row, 0] = -25
    vp[page, :, row, 0], vp[page, :, row, 3] = float("inf"), float("-inf")
    q = torch.zeros(2, hq, hd, dtype=dtype, device=DEV)
    q[:, :, 0] = 1
    out = ops.paged_attention(q, kp, vp, table, kl, scale=1.0)
    assert (out[0, :, 0] == float("inf")).all() and (out[0, :, 3] == float("-inf")).all()
    v = R.gather_keys(vp, table[0], n).double()
    v[j] = 0                                               # e^-25 of it
    want = (v.sum(0) / (n - 1)).repeat_interleave(hq // hk, 0)
    a = (v.abs().sum(0) / (n - 1)).repeat_interleave(hq // hk, 0)
    # equal probabilities: exact in any type; float32 sums of n values in at least
    # 16 parts, the division, and one rounding of the result; e^-25 of a value below 6
    rest = [c for c in range(hd) if c not in (0, 3)]
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2 * (n / 16 + 64) * 2.0 ** -24 * a + 1e-10
    assert ((out[0].double() - want).abs() <= bound)[:, rest].all()
    assert torch.isfinite(out[1].float()).all()
