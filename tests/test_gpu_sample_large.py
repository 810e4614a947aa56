"""Token sampling of batches of large vocabularies: every layout of a row over
CTAs, against the definition in float64."""
from fractions import Fraction

import numpy as np
import pytest
import torch

import serving_reference as R
from walsh_research_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def expect(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(ids, sure): the draws of the definition in float64, and which of them
    do not hang on sums closer than 1e-9 of the row's mass (weights are float64
    exponentials of relative error 1e-15; sums of 2^18 of them, 2^18 2^-53)."""
    z = logits.double()
    V = z.shape[1]
    w = torch.exp((z - z.amax(1, keepdim=True)) / temperature)
    order = torch.argsort(z, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    if 0 < top_k < V:
        ws[:, top_k:] = 0
    sure = torch.ones(len(z), dtype=torch.bool, device=z.device)
    if top_p < 1:
        before, total = ws.cumsum(1) - ws, ws.sum(1, keepdim=True)
        keep = before < top_p * total
        keep[:, 0] = True
        sure &= ((before - top_p * total).abs() > 1e-9 * total).all(1)
        ws = ws * keep
    if min_p > 0:
        sure &= ((ws - min_p).abs() > 1e-12).all(1)
        ws = ws * (ws >= min_p)
    kept = torch.zeros_like(w).scatter_(1, order, ws)
    run = kept.cumsum(1)
    t = u.double()[:, None] * run[:, -1:]
    ids = (run <= t).sum(1)
    near = torch.stack((run.gather(1, ids[:, None].clamp_max(V - 1))[:, 0], run.gather(1, (ids[:, None] - 1).clamp_min(0))[:, 0]))
    sure &= ((near - t[:, 0]).abs() > 1e-9 * run[:, -1]).all(0) | ((ids == 0) & (near[0] - t[:, 0] > 1e-9 * run[:, -1]))
    return ids, sure, torch.log(kept.gather(1, ids[:, None].clamp_max(V - 1))[:, 0] / run[:, -1])


def check(logits, u, **kw):
    want, sure, lp = expect(logits, u, **kw)
    assert sure.float().mean() > 0.9
    for _ in range(2):
        ids = ops.sample_tokens(logits, u, **kw)
        assert torch.equal(ids[sure], want[sure]), (int((ids[sure] != want[sure]).sum()), int(sure.sum()))
        ids, logp = ops.sample_tokens(logits, u, want_logprob=True, **kw)
        assert torch.equal(ids[sure], want[sure])
        # rounded once to float32; the weight itself good to 2^-45 of the largest
        bound = 2.0 ** -23 * lp.abs() + 2.0 ** -44 * torch.exp((-lp).clamp_max(30.0))
        assert ((logp.double() - lp).abs() <= bound)[sure].all()


def rand(rows, vocab, seed, dtype=torch.float32, spread=2.0, pad=0):
    """Rows ``vocab + pad`` apart, starting ``pad`` elements into their memory."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    z = (spread * torch.randn(rows, vocab + pad, generator=g, device=DEV)).to(dtype)[:, pad:]
    return z, torch.rand(rows, generator=g, device=DEV)


WAYS = [dict(), dict(min_p=0.001), dict(top_p=0.9), dict(top_p=0.97, min_p=0.0005, temperature=1.5), dict(top_k=600),
        dict(top_k=40, top_p=0.9)]


@pytest.mark.parametrize("kw", WAYS, ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 70000), (18, 33000), (19, 50257), (36, 20000), (37, 40000), (73, 50257),
                                        (74, 9000), (100, 50257), (147, 9000), (60, 8200)])
def test_rows_on_clusters_of_every_size(rows, vocab, kw):
    for seed in range(3):
        check(*rand(rows, vocab, seed + rows), **kw)


@pytest.mark.parametrize("kw", WAYS, ids=str)
@pytest.mark.parametrize("rows,vocab,dtype,pad", [
    (150, 65537, torch.float32, 0), (150, 65536, torch.float32, 1), (150, 65534, torch.float32, 3),
    (150, 128256, torch.float32, 0), (100, 151936, torch.float32, 0), (150, 151936, torch.bfloat16, 0),
    (150, 131066, torch.float16, 7), (148, 1 << 18, torch.float32, 1), (148, 1 << 18, torch.bfloat16, 0),
    (80, 1 << 18, torch.float16, 3), (40, 1 << 18, torch.float32, 3)])
def test_many_rows_of_large_vocabularies(rows, vocab, dtype, pad, kw):
    """Parts of up to 129 steps per warp, also of rows that start off a 16-byte boundary."""
    check(*rand(rows, vocab, vocab + rows, dtype, pad=pad), **kw)


@pytest.mark.parametrize("rows", [1, 150])
@pytest.mark.parametrize("step", [1e-3, 1e-6])
def test_top_p_within_a_hair_of_a_token(rows, step):
    """top_p a relative 1.5e-11 to either side of the mass before a token, which
    60000 equal tokens behind the border decide.  Weights are multiples of 2^-44
    of the largest, so the reach is good to 60300 * 2^-45 of a mass of over 340:
    5e-12.  u draws the last token that stays (its share is over 2^-9, u is 1 -
    2^-24)."""
    z = torch.cat((-step * torch.arange(300), torch.full((60000,), -9.49 * 0.6931472)))
    w = [int(x) for x in np.rint(np.exp(z.double().numpy()) * 2.0 ** 60)]
    logits = z.to(DEV).expand(rows, -1)
    u = torch.full((rows,), 1 - 2.0 ** -24, device=DEV)
    for r in (2, 40, 111, 250, 299):
        p = float(Fraction(sum(w[:r]), sum(w)))
        for side, last in ((1 - 1.5e-11, r - 1), (1 + 1.5e-11, r)):
            assert R.sample_row(z.double().numpy(), 1 - 2.0 ** -24, top_p=p * side)[0] == last
            ids = ops.sample_tokens(logits, u, top_p=p * side)
            assert (ids == last).all(), (r, side > 1, ids[0].item())


@pytest.mark.parametrize("t", [float("inf"), 3e38, 1.2e38, 2e37, 1e-45])
@pytest.mark.parametrize("kw", [dict(), dict(top_p=0.8), dict(min_p=0.2), dict(top_k=600, top_p=0.9)], ids=str)
def test_temperatures_and_differences_at_the_ends_of_float32(t, kw):
    """Differences of logits past float32's range, or of its smallest steps, and
    temperatures that still weigh them: +-3e38 at 1.2e38 is a weight of e^-5."""
    g = torch.Generator().manual_seed(21)
    if t > 1:
        z = 3e38 * (2 * torch.rand(24, 700, generator=g) - 1)
    else:
        z = torch.randint(0, 6, (24, 700), generator=g).float() * 2.0 ** -149
    u = torch.rand(24, generator=g)
    ids = ops.sample_tokens(z.to(DEV), u.to(DEV), temperature=t, **kw).tolist()
    want = [R.sample_row(z[r].double().numpy(), float(u[r]), t, kw.get("top_k", 0), kw.get("top_p", 1.0),
                         kw.get("min_p", 0.0))[0] for r in range(24)]
    assert ids == want
