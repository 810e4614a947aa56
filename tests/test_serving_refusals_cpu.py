"""What the serving entry points refuse, on the host before any launch (no
GPU: the pointers are never used)."""
import pytest
import torch

from walsh_research_b200 import _lib, ops

P16 = 1 << 12  # a 16-byte aligned address that is never dereferenced


KV_FIELDS = ("k_pages", "v_pages", "dtype", "n_pages", "kv_heads", "page_size", "head_dim", "page_stride", "head_stride",
             "row_stride", "page_table", "table_stride", "table_cols", "kv_lens", "window", "sinks", "scale", "err")


def kv(**kw):
    d = dict(k_pages=P16, v_pages=P16, dtype=2, n_pages=4, kv_heads=2, page_size=16, head_dim=32, page_stride=1024,
             head_stride=512, row_stride=32, page_table=P16, table_stride=3, table_cols=3, kv_lens=P16, window=0,
             sinks=0, scale=0.25, err=None)
    d.update(kw)
    return _lib.PAGED_KV.pack(*[d[n] or 0 for n in KV_FIELDS])


def attn(k, q=P16, q_bs=128, q_hs=32, B=2, hq=4, max_len=48, scratch=P16, o=P16):
    return _lib.lib().walsh_paged_attn_fwd(k, q, q_bs, q_hs, B, hq, max_len, scratch, o, None)


def prefill(k, q=P16, q_ts=128, q_hs=32, rows=9, off=P16, B=2, hq=4, max_q=9, o=P16):
    return _lib.lib().walsh_paged_prefill_fwd(k, q, q_ts, q_hs, rows, off, B, hq, max_q, o, None)


def append(k, q=P16, q_ts=128, q_hs=32, key=P16, k_ts=64, k_hs=32, v=P16, v_ts=64, v_hs=32, n=5, hq=4, slots=P16,
           pos=P16, cos=P16, sin=P16, n_pos=8, qn=None, kn=None, eps=1e-6, q_out=P16):
    return _lib.lib().walsh_paged_append(k, q, q_ts, q_hs, key, k_ts, k_hs, v, v_ts, v_hs, n, hq, slots, pos, 1, cos, sin,
                                         n_pos, qn, kn, eps, q_out, None)


ARG, SHAPE, DTYPE, ALIGN, INJECTED = -1, -2, -3, -4, -7


@pytest.mark.parametrize("call", [attn, prefill, append])
@pytest.mark.parametrize("bad,code", [
    (dict(k_pages=None), ARG), (dict(v_pages=None), ARG), (dict(dtype=3), DTYPE), (dict(head_dim=24), SHAPE),
    (dict(head_dim=256), SHAPE), (dict(n_pages=0), SHAPE), (dict(kv_heads=0), SHAPE), (dict(page_size=0), SHAPE),
    (dict(page_stride=-8), SHAPE), (dict(row_stride=16), SHAPE), (dict(k_pages=P16 + 2), ALIGN),
    (dict(page_stride=1020), ALIGN), (dict(head_stride=516), ALIGN), (dict(row_stride=36), ALIGN)])
def test_pages_refused(call, bad, code):
    assert call(kv(**bad)) == code


@pytest.mark.parametrize("call", [attn, prefill])
@pytest.mark.parametrize("bad,code", [
    (dict(page_table=None), ARG), (dict(kv_lens=None), ARG), (dict(window=-1), ARG), (dict(sinks=-1), ARG),
    (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG), (dict(scale=float("nan")), ARG), (dict(scale=float("inf")), ARG),
    (dict(table_cols=0), SHAPE), (dict(table_cols=1 << 28), SHAPE), (dict(table_stride=-1), SHAPE)])
def test_tables_refused(call, bad, code):
    assert call(kv(**bad)) == code


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), ARG), (dict(o=None), ARG), (dict(B=-1), SHAPE), (dict(hq=3), SHAPE), (dict(hq=0), SHAPE),
    (dict(max_len=-1), SHAPE), (dict(q=P16 + 4), ALIGN), (dict(o=P16 + 2), ALIGN), (dict(q_hs=33), ALIGN),
    (dict(q_bs=-128), SHAPE), (dict(B=1 << 25), SHAPE)])
def test_decode_arguments_refused(bad, code):
    assert attn(kv(), **bad) == code


def test_decode_needs_its_scratch():
    one = kv(table_cols=1 << 16)
    need = _lib.call("walsh_paged_attn_scratch_bytes", one, 1, 2, 1 << 20)
    assert need > 0
    assert attn(one, B=1, hq=2, max_len=1 << 20, scratch=None) == ARG
    assert _lib.call("walsh_paged_attn_scratch_bytes", kv(), 4096, 4, 16) == 0
    assert _lib.call("walsh_paged_attn_scratch_bytes", kv(head_dim=7), 1, 2, 16) == -1


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), ARG), (dict(off=None), ARG), (dict(o=None), ARG), (dict(B=1 << 16), SHAPE), (dict(hq=5), SHAPE),
    (dict(rows=1 << 31), SHAPE), (dict(max_q=-1), SHAPE), (dict(q_ts=4), ALIGN), (dict(q=P16 + 8), ALIGN)])
def test_prefill_arguments_refused(bad, code):
    assert prefill(kv(), **bad) == code


@pytest.mark.parametrize("bad,code", [
    (dict(key=None), ARG), (dict(v=None), ARG), (dict(slots=None), ARG), (dict(q=None), ARG), (dict(q_out=None), ARG),
    (dict(cos=None), ARG), (dict(pos=None), ARG), (dict(kn=P16, eps=-1.0), ARG), (dict(kn=P16, eps=float("nan")), ARG),
    (dict(q=None, q_out=None, qn=P16), ARG), (dict(n=-1), SHAPE), (dict(hq=0), SHAPE), (dict(n_pos=0), SHAPE),
    (dict(k_ts=60), ALIGN), (dict(v_hs=4), ALIGN), (dict(q_ts=-8), SHAPE), (dict(v=P16 + 2), ALIGN)])
def test_append_arguments_refused(bad, code):
    assert append(kv(), **bad) == code


def sample(logits=P16, dtype=0, ld=100, rows=2, vocab=100, u=P16, t=1.0, k=0, p=1.0, m=0.0, ids=P16):
    return _lib.lib().walsh_sample_tokens(logits, dtype, ld, rows, vocab, u, t, k, p, m, None, None, None, None, ids, None,
                                          None)


@pytest.mark.parametrize("bad,code", [
    (dict(logits=None), ARG), (dict(u=None), ARG), (dict(ids=None), ARG), (dict(dtype=5), DTYPE), (dict(vocab=0), SHAPE),
    (dict(vocab=(1 << 18) + 1), SHAPE), (dict(rows=-1), SHAPE), (dict(ld=-1), SHAPE), (dict(t=-0.5), ARG),
    (dict(t=float("nan")), ARG), (dict(p=float("nan")), ARG), (dict(m=float("nan")), ARG)])
def test_sampling_arguments_refused(bad, code):
    assert sample(**bad) == code


def test_nothing_to_do_is_fine():
    assert append(kv(), n=0) == 0 and attn(kv(), B=0) == 0 and prefill(kv(), B=0) == 0 and sample(rows=0) == 0


def test_fault_injection(monkeypatch):
    for site, call in (("paged_append", append), ("paged_attn_fwd", attn), ("paged_prefill_fwd", prefill)):
        monkeypatch.setenv("WALSH_INJECT_FAULT", site)
        assert call(kv()) == INJECTED
    monkeypatch.setenv("WALSH_INJECT_FAULT", "sample_tokens")
    assert sample() == INJECTED


def test_cpu_tensors_are_rejected():
    x = torch.zeros(2, 2, 32)
    pages = torch.zeros(3, 2, 16, 32)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: ops.paged_append(x, x, x, pages, pages, lens),
                 lambda: ops.paged_attention(x, pages, pages, table, lens),
                 lambda: ops.paged_prefill_attention(x, torch.zeros(3, dtype=torch.int32), pages, pages, table, lens),
                 lambda: ops.sample_tokens(torch.zeros(2, 9), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="CUDA devices only"):
            call()


@pytest.fixture
def no_device_check(monkeypatch):
    """The wrappers' own checks, with CPU tensors standing in for device ones."""
    monkeypatch.setattr(ops, "require_cuda", lambda *a: None)


def test_wrappers_refuse_what_does_not_fit(no_device_check):
    x = torch.zeros(2, 2, 32)
    pages = torch.zeros(3, 2, 16, 32)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    off = torch.zeros(3, dtype=torch.int32)
    cases = [
        lambda: ops.paged_attention(x.half(), pages, pages, table, lens),
        lambda: ops.paged_attention(x[..., :16], pages, pages, table, lens),
        lambda: ops.paged_attention(x, pages, pages[:2], table, lens),
        lambda: ops.paged_attention(x, pages, pages.half(), table, lens),
        lambda: ops.paged_attention(x, pages, pages.transpose(0, 1).contiguous().transpose(0, 1), table, lens),
        lambda: ops.paged_attention(x, pages, pages, table.long(), lens),
        lambda: ops.paged_attention(x, pages, pages, table, lens.long()),
        lambda: ops.paged_attention(x, pages, pages, table[:1], lens),
        lambda: ops.paged_attention(x, pages, pages, table, lens[:1]),
        lambda: ops.paged_attention(x, pages, pages, table, lens, window=-1),
        lambda: ops.paged_attention(x, pages, pages, table, lens, out=torch.zeros(2, 2, 16)),
        lambda: ops.paged_attention(x, pages, pages, table, lens, out=x.half()),
        lambda: ops.paged_attention(x, pages, pages, table, lens, err=torch.zeros(2, dtype=torch.int32)),
        lambda: ops.paged_prefill_attention(x, off[:2], pages, pages, table, lens),
        lambda: ops.paged_prefill_attention(x, off.long(), pages, pages, table, lens),
        lambda: ops.paged_append(x, x, x, pages, pages, lens[:1]),
        lambda: ops.paged_append(x, x, x, pages, pages, lens.float()),
        lambda: ops.paged_append(x, x[:1], x, pages, pages, lens),
        lambda: ops.paged_append(x, x, x, pages, pages, lens, positions=lens),
        lambda: ops.paged_append(x, x, x, pages, pages, lens, positions=lens, rope=(torch.zeros(4, 8), torch.zeros(4, 8))),
        lambda: ops.paged_append(x, x, x, pages, pages, lens, q_norm=torch.ones(16)),
        lambda: ops.paged_append(None, x, x, pages, pages, lens, q_norm=torch.ones(32)),
        lambda: ops.sample_tokens(torch.zeros(9), torch.zeros(1)),
        lambda: ops.sample_tokens(torch.zeros(2, 9), torch.zeros(3)),
        lambda: ops.sample_tokens(torch.zeros(2, 9), torch.zeros(2).double()),
        lambda: ops.sample_tokens(torch.zeros(2, 9), torch.zeros(2), temperature=-1.0),
        lambda: ops.sample_tokens(torch.zeros(2, 9), torch.zeros(2), top_p=float("nan")),
        lambda: ops.sample_tokens(torch.zeros(2, 9), torch.zeros(2), top_k=torch.zeros(2)),
        lambda: ops.sample_tokens(torch.zeros(2, 9), torch.zeros(2), temperature=torch.zeros(3)),
    ]
    for i, c in enumerate(cases):
        with pytest.raises(ValueError):
            c()
            pytest.fail(f"case {i} was accepted")


def test_calls_run_on_the_tensors_device(monkeypatch):
    """Tensors on another device than the current one: the call is made under
    their device, with its stream; on the current device nothing is switched."""
    log = []

    class Guard:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            log.append(("enter", self.dev))

        def __exit__(self, *a):
            log.append(("exit", self.dev))

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(ops, "stream", lambda: 77)
    monkeypatch.setattr(ops, "call", lambda name, *a: log.append((name,) + a))
    ops._call_on(0, "x", 1)
    ops._call_on(3, "y", 2)
    assert log == [("x", 1, 77), ("enter", 3), ("y", 2, 77), ("exit", 3)]


def test_windows_sinks_and_bounds_past_31_bits_reach_the_kernel(monkeypatch):
    """2^31 and more mean no limit: clamped alike for the call and its scratch."""
    calls = []
    monkeypatch.setattr(ops, "_device_of", lambda *t: 0)
    monkeypatch.setattr(ops, "_call_on", lambda dev, name, *args: calls.append((name, args)))
    kp = torch.zeros(4, 2, 8, 16)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for kw in (dict(window=2 ** 40), dict(window=5, sinks=2 ** 31), dict(max_len=2 ** 40), dict(max_len=2 ** 32 + 1),
               dict(window=2 ** 31 - 1, sinks=2 ** 35, max_len=2 ** 31)):
        ops.paged_attention(torch.zeros(1, 2, 16), kp, kp, table, lens, **kw)
        name, args = calls.pop()
        assert name == "walsh_paged_attn_fwd" and args[6] == min(kw.get("max_len", 32), 32)  # what the table holds
        f = dict(zip(("window", "sinks"), _lib.PAGED_KV.unpack(args[0])[14:16]))
        assert all(f[k] == min(kw.get(k, 0), 2 ** 31 - 1) for k in f)


@pytest.mark.parametrize("dtype,hq,hk,hd,B", [(0, 8, 8, 128, 8192), (0, 32, 1, 128, 2 ** 20), (2, 64, 64, 128, 2 ** 20 - 1),
                                              (2, 1024, 1024, 16, 65535), (1, 40, 2, 64, 10 ** 6)])
def test_the_largest_decode_grid_counts_in_31_bits(dtype, hq, hk, hd, B):
    """The CTAs of a call (units times the ranges its scratch is for) for a bound of 2^31 - 1 keys."""
    k = kv(dtype=dtype, kv_heads=hk, head_dim=hd, page_size=2 ** 20, table_cols=2047, page_stride=2 ** 20 * hd * hk,
           head_stride=2 ** 20 * hd, row_stride=hd)
    nbytes = _lib.lib().walsh_paged_attn_scratch_bytes(k, B, hq, 2 ** 31 - 1)
    per_range = B * hq * (hd + 2) * 4
    assert nbytes > 0 and nbytes % per_range == 0
    group, tile = hq // hk, 4 if dtype == 0 else 8 if hq // hk <= 8 else 16
    assert B * hk * -(-group // tile) * (nbytes // per_range) < 2 ** 31
