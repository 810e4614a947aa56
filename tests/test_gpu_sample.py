"""Token sampling against the definition in float64: ids equal, log
probabilities to float32 rounding."""
import numpy as np
import pytest
import torch

import serving_reference as R
from walsh_research_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    ids, logp = ops.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                                  want_logprob=True)
    assert torch.equal(ids, ops.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p))
    z, un = logits.double().cpu().numpy(), u.double().cpu().numpy()

    def at(x, r):
        return x[r].item() if isinstance(x, torch.Tensor) else x

    for r in range(len(z)):
        i, lp = R.sample_row(z[r], un[r], at(temperature, r), at(top_k, r), at(top_p, r), at(min_p, r))
        assert int(ids[r]) == i, (r, int(ids[r]), i)
        got = float(logp[r])
        # rounded once to float32 (2^-24 relative), the weight itself good to 2^-45 of the largest
        assert (got != got and lp != lp) or abs(got - lp) <= 2.0 ** -23 * abs(lp) + 2.0 ** -44 * np.exp(-max(lp, -30.0)), (r, got, lp)


def rand(rows, vocab, seed, dtype=torch.float32, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn(rows, vocab, generator=g)).to(dtype).to(DEV), torch.rand(rows, generator=g).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 37), (4, 1000), (7, 4096), (3, 50257), (1, 130001)])
@pytest.mark.parametrize("kw", [dict(), dict(top_k=1), dict(top_k=5), dict(top_k=300, temperature=0.7), dict(top_p=0.9),
                                dict(top_p=0.5, min_p=0.05), dict(min_p=0.1, temperature=1.4),
                                dict(top_k=50, top_p=0.95, min_p=0.01, temperature=0.8), dict(temperature=0.0),
                                dict(top_p=0.99, temperature=3.0)], ids=str)
def test_draws(dtype, rows, vocab, kw):
    check(*rand(rows, vocab, rows * vocab, dtype), **kw)


def test_batch_of_256():
    check(*rand(256, 5000, 2), top_p=0.9, min_p=0.02)


def test_one_value_per_row():
    logits, u = rand(64, 3001, 3)
    g = torch.Generator().manual_seed(4)
    t = (2 * torch.rand(64, generator=g)).to(DEV)
    t[5], t[6] = 0.0, -1.0
    k = torch.randint(-1, 80, (64,), generator=g, dtype=torch.int32).to(DEV)
    k[9] = 10 ** 6
    p = (0.3 + torch.rand(64, generator=g)).to(DEV)
    p[10] = 0.0
    m = (0.2 * torch.rand(64, generator=g)).to(DEV)
    m[11], m[12] = 5.0, -1.0
    check(logits, u, t, k, p, m)
    check(logits, u, 0.9, k, 0.8, m)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=7), dict(top_p=0.6), dict(top_k=100, top_p=0.35), dict(min_p=0.5),
                                dict(temperature=0.0), dict(top_k=2999, top_p=0.999)], ids=str)
def test_ties_go_to_the_lowest_index(kw):
    """All equal; few distinct values; coarse 16-bit values; +0 and -0."""
    u = torch.tensor([0.0, 0.2, 0.5, 0.77, 0.9999], device=DEV)
    check(torch.zeros(5, 3000, device=DEV), u, **kw)
    z = torch.arange(3000, device=DEV).remainder(4).float().expand(5, -1)
    check(z, u, **kw)
    check(rand(5, 3000, 8, torch.bfloat16, 1.0)[0], u, **kw)
    check(torch.where(torch.arange(3000, device=DEV) % 2 == 0, 0.0, -0.0).expand(5, -1), u, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.9), dict(top_p=0.9, top_k=700, temperature=0.5)], ids=str)
def test_masked_and_nonfinite_logits(kw):
    logits, u = rand(8, 2000, 5)
    logits[0, 100:] = float("-inf")
    logits[1, :] = float("-inf")
    logits[2, 17] = float("inf")
    logits[2, 1700] = float("inf")
    logits[3, ::3] = float("nan")
    logits[4, 5:] = torch.finfo(torch.float32).min
    logits[5, :] = torch.finfo(torch.float32).min
    logits[6, :] = float("nan")
    logits[7, :1999] = float("-inf")
    check(logits, u, **kw)


def test_ends_of_the_uniform_range():
    logits, _ = rand(6, 500, 6)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, float("nan")], device=DEV)
    check(logits, u)
    check(logits, u, top_k=10)


@pytest.mark.parametrize("t", [1e-30, 1e-45, 1e30, float("inf"), 0.02])
def test_extreme_temperatures(t):
    logits, u = rand(3, 700, 7)
    check(logits, u, temperature=t)
    check(logits, u, temperature=t, top_p=0.7)
    check(logits, u, temperature=t, top_k=600)


def test_wide_spread_and_the_largest_vocabulary():
    check(*rand(2, 1 << 18, 9), top_p=0.95)
    check(*rand(2, 1 << 18, 10, spread=0.001), top_k=100000, top_p=0.5)
    check(*rand(2, 9000, 11, spread=300.0), top_k=4000, top_p=0.9999)
    check(*rand(2, 9000, 12, spread=1e30), top_k=4000)


@pytest.mark.parametrize("kw", [dict(top_p=0.95), dict(top_p=0.5, min_p=0.01), dict(top_p=0.9, temperature=30.0)], ids=str)
def test_many_tokens_at_a_top_p_border(kw):
    """Far more equal or nearly equal logits at the border than are ranked one by one."""
    check(*rand(3, 100001, 15, torch.bfloat16), **kw)
    logits, u = rand(3, 20000, 16)
    check((logits * 4).round() / 4, u, **kw)
    check(logits * 1e-4, u, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [700, 1023, 1025, 1500, 2049, 3333, 4097, 9000])
@pytest.mark.parametrize("top_k", [33, 300, 512, 513])
def test_top_k_of_rows_of_all_sizes(dtype, vocab, top_k):
    check(*rand(3, vocab, vocab + top_k, dtype), top_k=top_k, top_p=0.97)


@pytest.mark.parametrize("rows,vocab", [(150, 3000), (150, 40000), (40, 20000)])
def test_parts_held_or_read_again(rows, vocab):
    """One CTA per row or several, with and without room to hold the row."""
    check(*rand(rows, vocab, 17), top_p=0.9, min_p=0.01)
    check(*rand(rows, vocab, 18, torch.float16), top_k=40, top_p=0.9)
    logits, u = rand(rows, vocab, 19)
    logits[::7, 5] = float("inf")
    logits[1::7, ::2] = float("nan")
    check(logits, u, temperature=0.7)
    check(logits, u, top_p=0.8)


def test_rows_of_a_wider_matrix():
    big, u = rand(9, 1100, 13)
    check(big[::2, 3:1003], u[:5].contiguous(), top_p=0.8)
    check(big[:, 1:2], u)
    assert ops.sample_tokens(big[:0], u[:0]).shape == (0,)


def test_captured_draws_read_new_uniforms():
    logits, u = rand(4, 3000, 14)
    ops.sample_tokens(logits, u, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids = ops.sample_tokens(logits, u, top_p=0.9)
    for s in range(3):
        u.copy_(rand(4, 3, 20 + s)[1])
        graph.replay()
        assert torch.equal(ids, ops.sample_tokens(logits, u, top_p=0.9))
