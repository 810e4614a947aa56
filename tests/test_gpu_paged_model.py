"""mHCWalsh over the paged cache: against the dense cache and the oracle,
sequences of different lengths together, joined and retired, windows, and
generate_batch."""
import numpy as np
import pytest
import torch

import cases
from oracle import walsh_oracle as O
from test_gpu_generate import _oracle_greedy

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _model(name="model_h512", dtype=torch.float32, **over):
    from walsh_research_b200.model import WalshConfig, mHCWalsh
    cfg, n, _, sd = cases.model_inputs(name)
    cfg = dict(cfg, block_size=64, **over)
    m = mHCWalsh(WalshConfig(**cfg), n_streams=n)
    m.load_state_dict({k: torch.from_numpy(np.array(v)) for k, v in sd.items()}, strict=False)
    m = m.to(DEV).eval()
    m.compute_dtype = dtype
    return cfg, n, sd, m


def _cache(m, cfg, page=16, **kw):
    from walsh_research_b200 import _lib
    from walsh_research_b200.model import PagedKVCache
    H = cfg["n_head"]
    return PagedKVCache(cfg["n_layer"], kw.pop("n_pages", 64), page, H, cfg["n_embd"] // H, DEV,
                        dtype=_lib.inner_dtype(m._act_dtype()), max_seqs=8, max_seq_len=128, **kw)


def _ids(cfg, *shape, seed=0):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, cfg["vocab_size"], shape)).to(DEV)


# the paged and the dense attention kernels add in different orders: float32
# logits agree to the model's own parity bound (1e-4 of the largest logit),
# 16-bit ones to its absolute one (2e-2)
def _near(a, b, dtype):
    if dtype == torch.float32:
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
    else:
        assert float((a - b).abs().max()) <= 2e-2


@pytest.mark.parametrize("name", ["model_h512", "model_o512"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [1, 5, 16])
def test_paged_steps_match_the_dense_cache(name, dtype, page):
    from walsh_research_b200 import _lib
    from walsh_research_b200.model import KVCache
    cfg, n, sd, m = _model(name, dtype)
    H = cfg["n_head"]
    dense = KVCache(cfg["n_layer"], 64, H, cfg["n_embd"] // H, DEV, dtype=_lib.inner_dtype(m._act_dtype()), batch_size=3)
    cache = _cache(m, cfg, page, n_pages=256)
    batch = cache.select(cache.add(3))
    with torch.no_grad():
        for i, T in enumerate((9, 1, 1, 6, 1)):
            ids = _ids(cfg, 3, T, seed=i)
            a, _ = m(ids, kv_cache=dense, start_pos=dense.cached_len)
            b, _ = m(ids, kv_cache=batch)
            dense.increment(T)
            batch.increment(T)
            _near(b, a, dtype)
    cache.check()
    assert cache.lengths(batch.ids) == [18] * 3


def test_sequences_of_different_lengths_decode_together_like_the_oracle():
    cfg, n, sd, m = _model()
    prompts = [_ids(cfg, t, seed=t) for t in (3, 12, 7, 12)]
    out = m.generate_batch(prompts, 5, top_k=1, page_size=4)
    for p, o in zip(prompts, out):
        assert torch.equal(o[:p.numel()], p)
        assert np.array_equal(o.cpu().numpy(), _oracle_greedy(cfg, n, sd, p.cpu().numpy(), 5, True))


def test_sequences_join_and_retire_without_touching_the_others():
    """A sequence decoded alone gives what it gives among others that come and go."""
    cfg, n, sd, m = _model()
    cache = _cache(m, cfg, 4)
    p = [_ids(cfg, 1, t, seed=40 + t) for t in (5, 9, 6)]
    steps = [_ids(cfg, 1, 1, seed=60 + i) for i in range(6)]
    with torch.no_grad():
        alone = []
        s = cache.select(cache.add())
        m(p[0], kv_cache=s)
        s.increment(5)
        for t in steps:
            alone.append(m(t, kv_cache=s)[0])
            s.increment()
        cache.remove(s.ids)
        a = cache.add()
        m(p[0], kv_cache=cache.select(a))
        cache.select(a).increment(5)
        b = cache.add()
        m(p[1], kv_cache=cache.select(b))
        cache.select(b).increment(9)
        together = []
        live = a + b
        for i, t in enumerate(steps):
            if i == 2:
                cache.remove(b)
                live = a
            if i == 4:
                c = cache.add()
                m(p[2], kv_cache=cache.select(c))
                cache.select(c).increment(6)
                live = c + a
            batch = cache.select(live)
            out, _ = m(t.expand(len(live), 1), kv_cache=batch)
            batch.increment()
            together.append(out[live.index(a[0])])
    cache.check()
    for x, y in zip(alone, together):
        _near(y, x[0], torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(8, 0), (5, 3)])
def test_window_steps_match_one_pass_under_the_window(dtype, window, sinks):
    """Without channel modulation (which averages over a call's tokens) a prompt
    in one call, in parts and token by token are the same model; pages behind
    the window are given back on the way."""
    cfg, n, sd, m = _model("model_h512", dtype, use_channel_mod=False)
    ids = _ids(cfg, 2, 40, seed=9)
    whole, parts, full = (_cache(m, cfg, 4, n_pages=40, window=w, sinks=s) for w, s in ((window, sinks), (window, sinks), (0, 0)))
    with torch.no_grad():
        a, _ = m(ids, kv_cache=whole.select(whole.add(2)))
        c, _ = m(ids, kv_cache=full.select(full.add(2)))
        batch = parts.select(parts.add(2))
        for lo, hi in [(0, 17), (17, 30)] + [(i, i + 1) for i in range(30, 40)]:
            b, _ = m(ids[:, lo:hi], kv_cache=batch)
            batch.increment(hi - lo)
    _near(b, a, dtype)
    assert float((a - c).abs().max()) > 1e-3       # the window is felt
    assert parts.free_pages >= 40 - 2 * (-(-sinks // 4) + -(-window // 4) + 1)
    parts.check()


def test_a_window_of_the_whole_length_changes_nothing():
    cfg, n, sd, m = _model()
    prompts = [_ids(cfg, t, seed=t) for t in (4, 11)]
    a = m.generate_batch(prompts, 6, top_k=1)
    b = m.generate_batch(prompts, 6, top_k=1, window=64, sinks=2, page_size=3)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_generate_batch_draws_stops_and_ends():
    cfg, n, sd, m = _model()
    prompts = [_ids(cfg, t, seed=t) for t in (5, 62, 64, 5)]
    g = torch.Generator(device=DEV)
    a = m.generate_batch(prompts, 7, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01, generator=g.manual_seed(3))
    b = m.generate_batch(prompts, 7, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01, generator=g.manual_seed(3))
    c = m.generate_batch(prompts, 7, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01, generator=g.manual_seed(4))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and not all(torch.equal(x, y) for x, y in zip(a, c))
    # up to 64 tokens are cached; the last drawn one is not
    assert [x.numel() for x in a] == [12, 65, 65, 12]
    stop = int(a[0][6])
    d = m.generate_batch(prompts, 7, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01, generator=g.manual_seed(3),
                         stop_token=stop)
    first = a[0][5:].tolist().index(stop)
    assert torch.equal(d[0], a[0][:5 + first + 1])
    assert m.generate_batch([], 3) == [] and torch.equal(m.generate_batch(prompts[:1], 0)[0], prompts[0])


def test_generate_batch_returns_long_prompts_whole():
    """Only the last max_seq_len ids are read, but all of them come back."""
    cfg, n, sd, m = _model()
    long, short = _ids(cfg, 90, seed=1), _ids(cfg, 6, seed=2)
    a = m.generate_batch([long, short], 3, top_k=1, max_seq_len=32)
    b = m.generate_batch([long[-32:], short], 3, top_k=1, max_seq_len=32)
    assert torch.equal(a[0][:90], long) and torch.equal(a[0][90:], b[0][32:]) and a[0].numel() == 91
    assert torch.equal(a[1], b[1]) and a[1].numel() == 9


def test_generate_with_top_p_follows_sample_tokens():
    from walsh_research_b200 import _lib, ops
    from walsh_research_b200.model import KVCache
    cfg, n, sd, m = _model()
    idx = _ids(cfg, 2, 9, seed=6)
    g = torch.Generator(device=DEV)
    got = m.generate(idx, 5, temperature=0.8, top_k=50, top_p=0.9, min_p=0.02, generator=g.manual_seed(11))
    g.manual_seed(11)
    H = cfg["n_head"]
    kv = KVCache(cfg["n_layer"], 64, H, cfg["n_embd"] // H, DEV, dtype=_lib.inner_dtype(m._act_dtype()), batch_size=2)
    seq, new = idx, idx
    with torch.no_grad():
        for _ in range(5):
            z, _ = m(new, kv_cache=kv, start_pos=kv.cached_len)
            kv.increment(new.shape[1])
            new = ops.sample_tokens(z[:, -1], torch.rand(2, device=DEV, generator=g), temperature=0.8, top_k=50, top_p=0.9,
                                    min_p=0.02)[:, None]
            seq = torch.cat((seq, new), 1)
    assert torch.equal(got, seq)


def test_refusals():
    cfg, n, sd, m = _model()
    cache = _cache(m, cfg, 16)
    batch = cache.select(cache.add(2))
    with torch.no_grad():
        with pytest.raises(ValueError, match="2 sequences"):
            m(_ids(cfg, 3, 1), kv_cache=batch)
        with pytest.raises(ValueError, match="start_pos"):
            m(_ids(cfg, 2, 1), kv_cache=batch, start_pos=4)
        with pytest.raises(ValueError, match="per sequence"):
            m(_ids(cfg, 2, 129), kv_cache=batch)
        m.compute_dtype = torch.bfloat16
        with pytest.raises(ValueError, match="float32"):
            m(_ids(cfg, 2, 1), kv_cache=batch)
        m.compute_dtype = torch.float32
        for kw in (dict(max_seq_len=0), dict(max_seq_len=10 ** 6)):
            with pytest.raises(ValueError):
                m.generate_batch([_ids(cfg, 3)], 2, **kw)
        with pytest.raises(ValueError):
            m.generate_batch([_ids(cfg, 3)[:0]], 2)
