"""Paged append, paged decode attention and paged prefill attention against
float64 forms: types, head layouts, lengths from nothing to long, pages that
end anywhere, windows, strides, and what the calls leave alone."""
import pytest
import torch

import serving_reference as R
from walsh_research_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LAYOUTS = [(32, 32, 16), (4, 2, 32), (8, 1, 64), (6, 2, 128), (20, 1, 16)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, want, bound):
    got = got.double()
    assert not torch.isnan(got).any()
    d = (got - want).abs()
    bad = d > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((d / bound.clamp_min(1e-300)).max()):.3g} bounds"


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,hd", LAYOUTS)
@pytest.mark.parametrize("norm,rope,n,page", [(False, False, 1, 16), (False, True, 37, 7), (True, True, 130, 16),
                                              (True, False, 5, 1)])
def test_append(dtype, hq, hk, hd, norm, rope, n, page):
    g = gen(n * hd + hq)
    qkv = torch.randn(n, hq + 2 * hk, hd, generator=g).to(dtype).to(DEV)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    pages = -(-n // page) + 3
    kp = torch.randn(pages, hk, page, hd, generator=g).to(dtype).to(DEV)
    vp = torch.randn(pages, hk, page, hd, generator=g).to(dtype).to(DEV)
    slots = torch.randperm(pages * page, generator=g)[:n].to(DEV)
    slots[n // 2] = -1                                     # padding
    pos = torch.randint(0, 50, (n,), generator=g).to(DEV)
    cos, sin = torch.randn(50, hd // 2, generator=g).to(DEV), torch.randn(50, hd // 2, generator=g).to(DEV)
    qn, kn = (1 + 0.2 * torch.randn(hd, generator=g)).to(DEV), (1 + 0.2 * torch.randn(hd, generator=g)).to(DEV)
    k0, v0 = kp.clone(), vp.clone()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    idx = torch.int32 if n % 2 else torch.int64
    out = ops.paged_append(q, k, v, kp, vp, slots.to(idx), positions=pos.to(idx) if rope else None,
                           rope=(cos, sin) if rope else None, q_norm=qn if norm else None, k_norm=kn if norm else None,
                           eps=1e-5, err=err)
    assert int(err) == 0
    c, s = (cos[pos], sin[pos]) if rope else (None, None)
    wq, bq = R.rotate(q, qn if norm else None, c, s, 1e-5)
    wk, bk = R.rotate(k, kn if norm else None, c, s, 1e-5)
    close(out, wq, bq)
    put = slots >= 0
    page_id, row = slots[put] // page, slots[put] % page
    close(kp[page_id, :, row], wk[put], bk[put])
    assert torch.equal(vp[page_id, :, row], v[put])
    if not norm and not rope:
        assert torch.equal(out, q) and torch.equal(kp[page_id, :, row], k[put])
    k0[page_id, :, row], v0[page_id, :, row] = kp[page_id, :, row], vp[page_id, :, row]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)     # nothing else was touched


def test_append_without_queries_head_major_and_pages_of_another_order():
    """k, v as head-major views, pages laid out [page, slot, head, hd]."""
    g = gen(3)
    n, hk, hd, page = 19, 4, 32, 8
    k = torch.randn(hk, n, hd, generator=g).half().to(DEV).transpose(0, 1)
    v = torch.randn(hk, n, hd, generator=g).half().to(DEV).transpose(0, 1)
    pool = torch.zeros(2, 5, page, hk, hd, dtype=torch.float16, device=DEV)
    kp, vp = pool[0].transpose(1, 2), pool[1].transpose(1, 2)
    slots = torch.arange(n, device=DEV) + 4
    assert ops.paged_append(None, k, v, kp, vp, slots) is None
    flat = pool.flatten(1, 2)
    assert torch.equal(flat[0, 4:4 + n], k) and torch.equal(flat[1, 4:4 + n], v)
    assert not flat[:, :4].any() and not flat[:, 4 + n:].any()


def test_append_out_of_range_is_reported_and_skipped():
    n, h, hd, page = 6, 2, 16, 4
    x = torch.ones(n, h, hd, dtype=torch.float16, device=DEV)
    kp = torch.zeros(2, h, page, hd, dtype=torch.float16, device=DEV)
    vp = torch.zeros_like(kp)
    t = torch.ones(3, hd // 2, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    slots = torch.tensor([0, 8, 1 << 40, 3, 4, -5], device=DEV)
    pos = torch.tensor([0, 1, 2, 3, -1, 2], device=DEV)
    q = ops.paged_append(x, x, x, kp, vp, slots, positions=pos, rope=(t, t * 0), err=err)
    assert int(err) == -9
    assert (q[[0, 1, 2, 5]] == 1).all() and not q[3].any() and not q[4].any()
    stored = torch.zeros(8, dtype=torch.bool)
    stored[0] = True
    assert torch.equal(kp.transpose(1, 2).flatten(0, 1).any(-1).any(-1).cpu(), stored)
    assert torch.equal(vp.transpose(1, 2).flatten(0, 1).any(-1).any(-1).cpu(), stored)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", [False, True])
def test_append_rows_on_16_byte_boundaries_only(dtype, norm):
    """Rows, tables and pages that start 16 but not 32 bytes into their memory; an odd start is copied first."""
    g = gen(17)
    n, h, hd, page, e = 21, 3, 32, 4, 16 // torch.tensor([], dtype=dtype).element_size()
    for shift in (e, 1):
        flat = torch.randn(n * (3 * h * hd + e) + shift, generator=g).to(dtype).to(DEV)
        x = flat[shift:].view(n, 3 * h * hd + e)[:, :3 * h * hd].unflatten(1, (3, h, hd))
        q, k, v = x[:, 0], x[:, 1], x[:, 2]
        pool = torch.zeros(2, 8 * h * page * (hd + e) + e, dtype=dtype, device=DEV)
        kp, vp = (t[e:].view(8, h, page, hd + e)[..., :hd] for t in pool)
        slots = torch.randperm(8 * page, generator=g)[:n].to(DEV)
        pos = torch.arange(n, device=DEV)
        tab = torch.randn(2 * n * hd // 2 + 2, generator=g).to(DEV)
        cos, sin = tab[1:1 + n * hd // 2].view(n, hd // 2), tab[1 + n * hd // 2:1 + n * hd].view(n, hd // 2)
        w = (1 + torch.rand(hd, generator=g)).to(DEV) if norm else None
        out = ops.paged_append(q, k, v, kp, vp, slots, positions=pos, rope=(cos, sin), q_norm=w, k_norm=w)
        wq, bq = R.rotate(q, w, cos, sin)
        wk, bk = R.rotate(k, w, cos, sin)
        close(out, wq, bq)
        close(kp[slots // page, :, slots % page], wk, bk)
        assert torch.equal(vp[slots // page, :, slots % page], v)
        assert int((pool != 0).sum()) == int((kp != 0).sum()) + int((vp != 0).sum())


def test_append_of_nothing():
    kp = torch.zeros(1, 2, 4, 16, device=DEV)
    x = torch.zeros(0, 2, 16, device=DEV)
    assert ops.paged_append(x, x, x, kp, kp.clone(), torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 2, 16)


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------

def run_decode(dtype, hq, hk, hd, lens, page, window=0, sinks=0, scale=None, max_len=None, seed=0, spread=1.5, **kw):
    g = gen(seed)
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, lens, hk, page, hd, dtype, **kw))
    q = (spread * torch.randn(len(lens), hq, hd, generator=g)).to(dtype).to(DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    o = ops.paged_attention(q, kp, vp, table, kl, max_len=max_len, window=window, sinks=sinks, scale=scale, err=err)
    assert int(err) == 0
    for b, n in enumerate(lens):
        k, v = R.gather_keys(kp, table[b], n), R.gather_keys(vp, table[b], n)
        want, bound = R.attend(q[b:b + 1], k, v, n - 1, window, sinks, scale)
        close(o[b:b + 1], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,hd", LAYOUTS)
@pytest.mark.parametrize("lens,page,window,sinks", [
    ([1], 16, 0, 0), ([0, 1, 2, 15, 16, 17, 0], 16, 0, 0), ([333, 64, 65, 7], 24, 0, 0),
    ([1, 5, 6, 7, 200, 131], 5, 6, 2), ([100, 33, 1, 0], 64, 1, 0), ([90, 91, 92, 500], 16, 90, 3)])
def test_decode(dtype, hq, hk, hd, lens, page, window, sinks):
    run_decode(dtype, hq, hk, hd, lens, page, window, sinks, seed=len(lens) + page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,hd,lens", [(2, 2, 16, [5000, 1, 300]), (8, 1, 128, [3001, 0]), (1, 1, 64, [20011]),
                                           (32, 2, 32, [2500])])
def test_decode_long_caches_are_split_and_joined(dtype, hq, hk, hd, lens):
    run_decode(dtype, hq, hk, hd, lens, 16)
    run_decode(dtype, hq, hk, hd, lens, 48, window=2222, sinks=5)


def test_decode_many_sequences():
    lens = [(i * 37) % 300 for i in range(400)]
    run_decode(torch.float16, 4, 4, 16, lens, 16)
    run_decode(torch.bfloat16, 8, 2, 32, lens, 32, window=100, sinks=1)


@pytest.mark.parametrize("max_len", [0, 1, 40, 100000])
def test_decode_max_len_only_decides_how_the_work_is_cut(max_len):
    run_decode(torch.float16, 2, 2, 16, [700, 3, 0, 1500], 16, max_len=max_len)
    run_decode(torch.float32, 4, 2, 64, [700, 3, 0, 1500], 16, max_len=max_len, window=650, sinks=2)


@pytest.mark.parametrize("scale", [1.0, 0.01])
def test_decode_scale_and_sharp_scores(scale):
    run_decode(torch.float32, 4, 4, 64, [77, 300], 16, scale=scale, spread=6.0)
    run_decode(torch.float16, 4, 4, 16, [77, 300], 16, scale=scale, spread=6.0)


def test_decode_reads_strided_queries_pages_and_tables():
    g = gen(9)
    lens, hq, hk, hd, page = [45, 130], 4, 2, 32, 8
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, lens, hk, page, hd, torch.float16, cols_extra=3))
    q = torch.randn(hq, len(lens), hd, generator=g).half().to(DEV)
    want = ops.paged_attention(q.transpose(0, 1).contiguous(), kp, vp, table, kl)
    pool = torch.stack([kp.transpose(1, 2), vp.transpose(1, 2)], 1).contiguous()       # [page, 2, slot, head, hd]
    wide = torch.full((len(lens), 2, table.shape[1]), 1 << 30, dtype=torch.int32, device=DEV)
    wide[:, 0] = table
    got = ops.paged_attention(q.transpose(0, 1), pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2), wide[:, 0], kl)
    assert torch.equal(got, want)


def test_decode_dense_cache_is_one_page_per_sequence():
    """ops.attention's cache [B, H, ctx, hd] as B pages of ctx slots."""
    g = gen(10)
    B, H, ctx, hd, n = 3, 32, 96, 16, 77
    kc, vc = (torch.randn(B, H, ctx, hd, generator=g).half().to(DEV) for _ in range(2))
    q = torch.randn(B, H, 1, hd, generator=g).half().to(DEV)
    table = torch.arange(B, dtype=torch.int32, device=DEV)[:, None]
    kl = torch.full((B,), n, dtype=torch.int32, device=DEV)
    got = ops.paged_attention(q[:, :, 0], kc, vc, table, kl)
    dense = ops.attention(q, kc, vc, n - 1)[:, 0]
    for b in range(B):
        want, bound = R.attend(q[b].transpose(0, 1), kc[b, :, :n].transpose(0, 1), vc[b, :, :n].transpose(0, 1), n - 1)
        close(got[b:b + 1], want, bound)
        close(dense[b:b + 1], want, bound)


def test_decode_bad_page_ids_and_lengths_are_reported():
    g = gen(11)
    lens, h, hd, page = [50, 40, 30], 2, 32, 16
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, lens, h, page, hd, torch.float16))
    q = torch.randn(3, h, hd, generator=g).half().to(DEV)
    table[0, 1] = kp.shape[0]                              # one past the pool
    table[1, 0] = -3
    kl[2] = table.shape[1] * page + 1                      # longer than the table: clamped, unowned slots are NaN
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for dt in (torch.float16, torch.float32):
        err.zero_()
        o = ops.paged_attention(q.to(dt), kp.to(dt), vp.to(dt), table, kl, err=err)
        assert int(err) == -9
        for b, (lo, hi) in enumerate([(16, 32), (0, 16)]):
            tr = table[b].clone()
            tr[tr < 0] = 0
            tr[tr >= kp.shape[0]] = 0
            k, v = R.gather_keys(kp.to(dt), tr, lens[b]), R.gather_keys(vp.to(dt), tr, lens[b])
            hide = torch.zeros(lens[b], dtype=torch.bool, device=DEV)
            hide[lo:hi] = True
            k[hide] = v[hide] = 0
            want, bound = R.attend(q[b:b + 1].to(dt), k, v, lens[b] - 1, hide=hide)
            close(o[b:b + 1], want, bound)
    err.zero_()
    kl[2] = -1
    table[0, 1] = table[1, 0] = 0
    o = ops.paged_attention(q, kp, vp, table, kl, err=err)
    assert int(err) == -9 and not o[2].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_decode_nonfinite_values_stay_where_they_are_seen(dtype):
    """-inf scores weigh nothing, a row of them alone gives zeros, and a NaN
    reaches its own row only."""
    h, hd, page = 2, 16, 8
    kp = torch.zeros(4, h, page, hd, dtype=dtype, device=DEV)
    vp = torch.ones_like(kp)
    table = torch.arange(4, dtype=torch.int32, device=DEV)[:, None]
    kl = torch.full((4,), 8, dtype=torch.int32, device=DEV)
    q = torch.zeros(4, h, hd, dtype=dtype, device=DEV)
    q[:, :, 0] = 1
    kp[1, :, 3, 0] = float("-inf")
    vp[1, :, 3] = 5
    kp[2, :, :, 0] = float("-inf")
    kp[3, :, 2, 0] = float("nan")
    o = ops.paged_attention(q, kp, vp, table, kl)
    assert (o[0] == 1).all() and (o[1] == 1).all() and (o[2] == 0).all() and torch.isnan(o[3]).all()
    off = torch.arange(5, dtype=torch.int32, device=DEV)
    o = ops.paged_prefill_attention(q, off, kp, vp, table, kl)
    assert (o[0] == 1).all() and (o[1] == 1).all() and (o[2] == 0).all() and torch.isnan(o[3]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_offsets_pass_32_bits(dtype):
    """Pages 2^31 + 2^20 elements apart: byte and element offsets beyond 32 bits."""
    h, hd, page, n = 2, 32, 16, 30
    stride = (1 << 31) + (1 << 20)
    g = gen(12)
    buf = torch.empty(stride + 2 * h * page * hd, dtype=dtype, device=DEV)
    kp = buf.as_strided((2, h, page, hd), (stride, page * hd, hd, 1))
    vp = buf.as_strided((2, h, page, hd), (stride, page * hd, hd, 1), storage_offset=h * page * hd)
    k, v = (torch.randn(n, h, hd, generator=g).to(dtype).to(DEV) for _ in range(2))
    slots = torch.arange(n, device=DEV)
    ops.paged_append(None, k, v, kp, vp, slots)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
    kl = torch.tensor([n], dtype=torch.int32, device=DEV)
    q = torch.randn(n, h, hd, generator=g).to(dtype).to(DEV)
    want, bound = R.attend(q, k, v, 0)
    close(ops.paged_attention(q[n - 1:], kp, vp, table, kl), want[n - 1:], bound[n - 1:])
    off = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    close(ops.paged_prefill_attention(q, off, kp, vp, table, kl), want, bound)


# ---------------------------------------------------------------------------
# prefill
# ---------------------------------------------------------------------------

def run_prefill(dtype, hq, hk, hd, new, past, page, window=0, sinks=0, max_q=None, seed=0, tail=0):
    g = gen(seed)
    lens = [a + b for a, b in zip(new, past)]
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, lens, hk, page, hd, dtype))
    n = sum(new)
    q = (1.5 * torch.randn(n + tail, hq, hd, generator=g)).to(dtype).to(DEV)
    off = torch.tensor([0] + new).cumsum(0).int().to(DEV)
    out = torch.full((n + tail, hq, hd), 7.0, dtype=dtype, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.paged_prefill_attention(q, off, kp, vp, table, kl, max_q=max_q, window=window, sinks=sinks, out=out, err=err)
    assert got is out and int(err) == 0
    assert (out[n:] == 7).all()
    at = 0
    for b, t in enumerate(new):
        if t:
            k, v = R.gather_keys(kp, table[b], lens[b]), R.gather_keys(vp, table[b], lens[b])
            want, bound = R.attend(q[at:at + t], k, v, past[b], window, sinks)
            close(out[at:at + t], want, bound)
        at += t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,hd", LAYOUTS)
@pytest.mark.parametrize("new,past,page,window,sinks", [
    ([1], [0], 16, 0, 0), ([0, 1, 2, 17, 0, 64, 65], [3, 0, 5, 0, 9, 1, 0], 16, 0, 0),
    ([130, 20], [0, 211], 7, 0, 0), ([150, 3], [0, 90], 32, 20, 3), ([129], [300], 24, 64, 0), ([40], [70], 16, 1, 1)])
def test_prefill(dtype, hq, hk, hd, new, past, page, window, sinks):
    run_prefill(dtype, hq, hk, hd, new, past, page, window, sinks, seed=page, tail=3)


@pytest.mark.parametrize("dtype,hq,hk,hd", [(torch.float16, 4, 4, 16), (torch.bfloat16, 4, 4, 32), (torch.float32, 2, 1, 64)])
def test_prefill_long(dtype, hq, hk, hd):
    run_prefill(dtype, hq, hk, hd, [1500, 700], [0, 800], 64, 0, 0)
    run_prefill(dtype, hq, hk, hd, [1500, 700], [0, 800], 64, 300, 7)


def test_prefill_max_q_only_sizes_the_grid():
    run_prefill(torch.float16, 4, 2, 32, [300, 1, 77], [5, 0, 0], 16, 0, 0, max_q=10)
    run_prefill(torch.float32, 4, 2, 32, [300, 1, 77], [5, 0, 0], 16, 50, 2, max_q=10)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prefill_tiles_without_keys_among_others(dtype):
    """More queries than keys over several tiles: the first see nothing, the later ones their keys."""
    g = gen(18)
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [70], 1, 8, 16, dtype))
    q = torch.randn(500, 1, 16, generator=g).to(dtype).to(DEV)
    off = torch.tensor([0, 500], dtype=torch.int32, device=DEV)
    for max_q in (500, 40):
        o = ops.paged_prefill_attention(q, off, kp, vp, table, kl, max_q=max_q)
        assert not o[:430].any()
        want, bound = R.attend(q[430:], R.gather_keys(kp, table[0], 70), R.gather_keys(vp, table[0], 70), 0)
        close(o[430:], want, bound)


def test_prefill_of_one_token_each_equals_decode():
    g = gen(5)
    lens, hq, hk, hd = [40, 1, 300, 129], 8, 2, 32
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, lens, hk, 16, hd, torch.float32))
    q = torch.randn(4, hq, hd, generator=g).to(DEV)
    off = torch.arange(5, dtype=torch.int32, device=DEV)
    a = ops.paged_attention(q, kp, vp, table, kl, window=100, sinks=2)
    b = ops.paged_prefill_attention(q, off, kp, vp, table, kl, window=100, sinks=2)
    torch.testing.assert_close(a, b, rtol=2e-6, atol=2e-6)


def test_prefill_more_queries_than_keys_and_bad_offsets():
    """Queries before the sequence's first key see nothing; a bad span is reported and left alone."""
    g = gen(6)
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [3, 20], 2, 8, 16, torch.float16))
    q = torch.randn(12, 2, 16, generator=g).half().to(DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 7.0)
    off = torch.tensor([0, 5, 13], dtype=torch.int32, device=DEV)
    ops.paged_prefill_attention(q, off, kp, vp, table, kl, out=out, err=err)
    assert int(err) == -9
    assert not out[:2].any() and (out[5:] == 7).all()
    k, v = R.gather_keys(kp, table[0], 3), R.gather_keys(vp, table[0], 3)
    want, bound = R.attend(q[2:5], k, v, 0)
    close(out[2:5], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hk,hd", LAYOUTS)
def test_prefill_hidden_values_that_are_not_finite(dtype, hq, hk, hd):
    """A key or value that is infinite or NaN reaches the tokens that see it and no others."""
    g = gen(14)
    n, window, sinks = 90, 20, 2
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [n], hk, 16, hd, dtype))
    q = torch.randn(n, hq, hd, generator=g).to(dtype).to(DEV)
    off = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    clean = ops.paged_prefill_attention(q, off, kp, vp, table, kl, window=window, sinks=sinks)

    def at(j):
        return int(table[0, j // 16]), j % 16

    for j, value in ((40, float("nan")), (61, float("inf")), (77, float("-inf"))):
        vp[at(j)[0], :, at(j)[1]] = value
    kp[at(30)[0], :, at(30)[1]] = float("nan")
    o = ops.paged_prefill_attention(q, off, kp, vp, table, kl, window=window, sinks=sinks)
    t = torch.arange(n, device=DEV)
    sees = lambda j: (t >= j) & (t < j + window)  # noqa: E731
    touched = sees(40) | sees(61) | sees(77) | sees(30)
    assert not torch.isfinite(o[touched].float()).any()
    # rows computed once more add in another order: one rounding of the result and
    # of the probabilities each way
    d = (o[~touched].double() - clean[~touched].double()).abs()
    k, v = R.gather_keys(kp, table[0], n), R.gather_keys(vp, table[0], n)
    k, v = torch.where(torch.isfinite(k), k, 0), torch.where(torch.isfinite(v), v, 0)
    _, bound = R.attend(q, k, v, 0, window, sinks)
    assert (d <= 2 * bound[~touched]).all()


# ---------------------------------------------------------------------------
# use: streams, graphs, repeatability
# ---------------------------------------------------------------------------

def test_calls_in_two_graphs_and_on_another_stream_repeat_bit_for_bit():
    g = gen(8)
    lens, hq, hk, hd = [3000, 900], 4, 2, 32
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, lens, hk, 16, hd, torch.bfloat16))
    qs = [torch.randn(2, hq, hd, generator=g).bfloat16().to(DEV) for _ in range(2)]
    want = [ops.paged_attention(q, kp, vp, table, kl) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [ops.paged_attention(q, kp, vp, table, kl) for q in qs]
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.paged_attention(q, kp, vp, table, kl))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for w, x, y in zip(want, again, outs):
        assert torch.equal(w, x) and torch.equal(w, y)


def test_lengths_move_between_replays_of_one_graph():
    """A captured step reads lengths and tables when it is replayed."""
    g = gen(13)
    hq = hk = 2
    hd, page = 16, 16
    kp, vp, table, kl = (t.to(DEV) for t in R.make_pool(g, [2000, 1200], hk, page, hd, torch.float16))
    kp, vp = torch.nan_to_num(kp), torch.nan_to_num(vp)
    q = torch.randn(2, hq, hd, generator=g).half().to(DEV)
    ops.paged_attention(q, kp, vp, table, kl)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(q, kp, vp, table, kl)
    for lens in ([2000, 1200], [1, 0], [513, 1199]):
        kl.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        for b, n in enumerate(lens):
            want, bound = R.attend(q[b:b + 1], R.gather_keys(kp, table[b], n), R.gather_keys(vp, table[b], n), n - 1)
            close(out[b:b + 1], want, bound)
