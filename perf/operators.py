"""The serving operators of walsh_research_b200 as measurable cases: paged
cache append, paged decode attention, paged prefill attention with a sliding
window, and token sampling.

``listed()`` / ``draw(rng)`` give cases, ``prepare`` their inputs on the GPU,
``run`` one pass: with ``own`` false in elementary torch operations, with
``own`` true through the package's entry points.  ``exact`` gives the same
outputs from the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# (query heads, key/value heads, head dim): the 512- and 2048-wide models'
# own layouts first, then shared key/value heads
LAYOUTS = [(32, 32, 16), (64, 64, 32), (32, 8, 64), (16, 2, 128), (32, 4, 32), (8, 8, 64)]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    def case(name, op, dtype, **kw):
        return dict(name=name, op=op, dtype=dtype, **kw)

    def heads(i):
        return dict(heads=LAYOUTS[i][0], kv_heads=LAYOUTS[i][1], head_dim=LAYOUTS[i][2])

    return [
        # a single conversation's next token: latency only
        case("append_1", "append", "f16", tokens=1, **heads(0), page=16, norm=False, fused=False),
        # a batched decode step from a fused q|k|v projection, with per-head norms
        case("append_256", "append", "bf16", tokens=256, **heads(2), page=64, norm=True, fused=True),
        # prompts of a whole batch
        case("append_65536", "append", "f16", tokens=65536, **heads(0), page=64, norm=True, fused=False),
        # one conversation, some thousand tokens of context: few rows, a long axis
        case("decode_1x4099", "decode", "f16", batch=1, longest=4099, ragged=False, **heads(0), page=16, window=0,
             sinks=0),
        # the 512-wide model's batched decode, conversations of all ages
        case("decode_256x1024", "decode", "f16", batch=256, longest=1024, ragged=True, **heads(0), page=64, window=0,
             sinks=0),
        # shared key/value heads over long documents
        case("decode_12x32768", "decode", "bf16", batch=12, longest=32768, ragged=True, **heads(2), page=32, window=0,
             sinks=0),
        # endless streams of the 2048-wide model: a window and a few first tokens stay visible
        case("decode_window", "decode", "bf16", batch=48, longest=6000, ragged=True, **heads(1), page=16, window=1000,
             sinks=4),
        # short questions arriving together
        case("prefill_short", "prefill", "f16", batch=5, longest=61, ragged=True, past=0, **heads(0), page=16,
             window=0, sinks=0),
        # the 512-wide model's prompts under a window
        case("prefill_8x2048", "prefill", "f16", batch=8, longest=2048, ragged=False, past=0, **heads(0), page=64,
             window=512, sinks=4),
        # a later part of long prompts of the 2048-wide model
        case("prefill_chunk", "prefill", "bf16", batch=3, longest=3500, ragged=True, past=2500, **heads(1), page=32,
             window=1024, sinks=16),
        # one answer's next token
        case("sample_1", "sample", "f32", rows=1, vocab=50257, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0),
        # a batched decode step, nucleus sampling over the whole vocabulary
        case("sample_256", "sample", "f32", rows=256, vocab=50257, temperature=1.0, top_k=0, top_p=0.9, min_p=0.02),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill", "sample"])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    if op == "sample":
        vocab = _log_int(rng, 200, 130000)
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, max(1, min(512, 256 * 50257 // vocab))), vocab=vocab,
                    temperature=round(rng.uniform(0.3, 1.5), 2), top_k=rng.choice([0, 0, 1, 20, 64, 500]),
                    top_p=rng.choice([1.0, 0.95, 0.9, 0.5]), min_p=rng.choice([0.0, 0.0, 0.01, 0.1]))
    h, hk, hd = rng.choice(LAYOUTS)
    heads = dict(heads=h, kv_heads=hk, head_dim=hd)
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "append":
        limit = 65536 * 32 * 16 * 3 * 2 // ((h + 2 * hk) * hd * (4 if dtype == "f32" else 2))
        return dict(op=op, dtype=dtype, tokens=_log_int(rng, 1, limit), **heads, page=page,
                    norm=rng.random() < 0.5, fused=rng.random() < 0.5)
    window, sinks = rng.choice([(0, 0), (0, 0), (128, 4), (777, 1), (1024, 16), (333, 0)])
    ragged = rng.random() < 0.7
    if op == "decode":
        batch = _log_int(rng, 1, 256)
        limit = 256 * 1024 * 32 * 16 * 2 // (batch * hk * hd * (4 if dtype == "f32" else 2))
        return dict(op=op, dtype=dtype, batch=batch, longest=_log_int(rng, 1, max(2, min(40000, limit))),
                    ragged=ragged, **heads, page=page, window=window, sinks=sinks)
    batch = _log_int(rng, 1, 16)
    work = 8 * 2048 * 512 * 32 * 16 // (batch * h * hd * (8 if dtype == "f32" else 1))  # query-key pairs a sequence may have
    longest = _log_int(rng, 2, max(2, min(4000, work // window if window else int(math.sqrt(2 * work)))))
    past = rng.choice([0, 0, _log_int(rng, 1, 2000)])
    past = min(past, max(0, work // longest))
    return dict(op=op, dtype=dtype, batch=batch, longest=longest, ragged=ragged, past=past, **heads, page=page,
                window=window, sinks=sinks)


def _lengths(case):
    """The batch's lengths (new tokens for prefill), the same for every seed up to their order."""
    n, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    return [longest] + [1 + (i * 0x9E3779B1 >> 7) % longest for i in range(1, n)]


def _visible(pos, window, sinks):
    """Keys that the query at position pos sees."""
    n = pos + 1
    return n if window == 0 else min(n, window + min(sinks, max(0, n - window)))


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * 16, "flops": 8 * n}
    h, hk, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        n = case["tokens"]
        return {"bytes": 2 * n * (h + 2 * hk) * hd * e + n * (hd * 4 + 16), "flops": n * (h + hk) * hd * (7 if case["norm"] else 3)}
    lens, w, s = _lengths(case), case["window"], case["sinks"]
    if case["op"] == "decode":
        vis = sum(_visible(n - 1, w, s) for n in lens)
        return {"bytes": vis * hk * hd * 2 * e + case["batch"] * h * hd * 2 * e, "flops": 4 * vis * h * hd}
    past = case["past"]
    pairs = sum(_visible(past + t, w, s) for n in lens for t in range(n))
    keys = sum(n + (past if w == 0 else min(past, w + s)) for n in lens)
    return {"bytes": keys * hk * hd * 2 * e + sum(lens) * h * hd * 2 * e, "flops": 4 * pairs * h * hd}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    st = dict(case)
    if case["op"] == "sample":
        # a language model's logits: a wide bell, its tail the candidates
        st["logits"] = (3.0 * randn(case["rows"], case["vocab"])).to(dt)
        st["u"] = torch.rand(case["rows"], generator=g, device="cuda")
        return st
    h, hk, hd, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    if case["op"] == "append":
        n = case["tokens"]
        if case["fused"]:
            qkv = randn(n, h + 2 * hk, hd).to(dt)
            st["q"], st["k"], st["v"] = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
        else:
            st["q"], st["k"], st["v"] = randn(n, h, hd).to(dt), randn(n, hk, hd).to(dt), randn(n, hk, hd).to(dt)
        pages = -(-n // ps) + 3
        st["k_pages"] = torch.zeros(pages, hk, ps, hd, dtype=dt, device="cuda")
        st["v_pages"] = torch.zeros_like(st["k_pages"])
        # sequences of up to 1024 tokens; pages in no order
        pos = torch.arange(n, device="cuda") % 1024
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(n, device="cuda")
        st["slots"] = order[at // ps] * ps + at % ps
        st["positions"] = pos
        ang = torch.outer(torch.arange(2048, device="cuda", dtype=torch.float64),
                          10000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd))
        st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        if case["norm"]:
            st["q_norm"], st["k_norm"] = 1 + 0.1 * randn(hd), 1 + 0.1 * randn(hd)
        return st
    lens = torch.tensor(_lengths(case))
    lens = lens[torch.randperm(len(lens), generator=torch.Generator().manual_seed(seed))]
    total = lens if case["op"] == "decode" else lens + case["past"]
    st["kv_lens"] = total.to(torch.int32).cuda()
    st["max_len"] = int(total.max())
    width = -(-st["max_len"] // ps)
    need = (total + ps - 1) // ps
    pages = int(need.sum())
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    col = torch.arange(width)[None, :]
    flat = (need.cumsum(0) - need)[:, None] + col
    table = torch.where(col < need[:, None], flat, torch.zeros_like(flat)).cuda()
    st["page_table"] = order[table].contiguous()
    st["k_pages"], st["v_pages"] = randn(pages, hk, ps, hd).to(dt), randn(pages, hk, ps, hd).to(dt)
    n = case["batch"] if case["op"] == "decode" else int(lens.sum())
    # scores with a spread of 1.5: some keys stand out, as in a trained head
    st["q"] = (1.5 * randn(n, h, hd)).to(dt)
    if case["op"] == "prefill":
        off = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
        st["q_offsets"] = off.to(torch.int32).cuda()
        st["max_q"] = int(lens.max())
    return st


# ---------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits (sampling in 64: a token at a
# border of a sum is kept or dropped whole)
# ---------------------------------------------------------------------------

def _plain_rotate(x, w, st):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    c, s = st["cos"][st["positions"]][:, None], st["sin"][st["positions"]][:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _plain_append(st):
    dt = st["q"].dtype
    q = _plain_rotate(st["q"], st.get("q_norm"), st).to(dt)
    k = _plain_rotate(st["k"], st.get("k_norm"), st).to(dt)
    page, row = st["slots"] // st["page"], st["slots"] % st["page"]
    st["k_pages"][page, :, row] = k
    st["v_pages"][page, :, row] = st["v"]
    return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}


def _plain_rows(st, seq, key, ok):
    """K and V of the given keys of the given sequences, [..., Hkv, hd] in float32."""
    key = torch.where(ok, key, torch.zeros_like(key))
    page = st["page_table"].long()[seq.expand_as(key), key // st["page"]]
    return st["k_pages"][page, :, key % st["page"]].float(), st["v_pages"][page, :, key % st["page"]].float()


def _plain_attend(st, q, qpos, seq, key, seen):
    """q [S, R, Hq, hd] at positions qpos [S, R] over keys key [S, J] of sequences seq [S, 1]."""
    hk, hd = st["kv_heads"], st["head_dim"]
    k, v = _plain_rows(st, seq, key, seen.any(1))
    q = q.float().unflatten(2, (hk, -1)) * (1.0 / math.sqrt(hd))
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)                    # [S, Hkv, g R, hd]
    s = torch.matmul(q, k.permute(0, 2, 3, 1))                    # [S, Hkv, g R, J]
    mask = seen[:, None, None].expand(-1, -1, st["heads"] // hk, -1, -1).flatten(2, 3)
    s = s.masked_fill(~mask, float("-inf"))
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)).unflatten(2, (-1, qpos.shape[1]))
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3)                 # [S, R, Hq, hd]


def _plain_keys(st, first, last, span):
    """Key numbers of a query block that sees window keys first..last: the sinks, then the window. [S, J]"""
    dev = first.device
    sink = torch.arange(st["sinks"], device=dev)[None].expand(len(first), -1)
    sink = torch.where(sink < first[:, None], sink, torch.full_like(sink, -1))
    near = first[:, None] + torch.arange(span, device=dev)[None]
    near = torch.where(near <= last[:, None], near, torch.full_like(near, -1))
    return torch.cat((sink, near), 1)


def _plain_seen(st, key, qpos):
    key, qpos = key[:, None], qpos[..., None]
    seen = (key >= 0) & (key <= qpos)
    if st["window"]:
        seen &= (key > qpos - st["window"]) | (key < st["sinks"])
    return seen


def _plain_decode(st):
    lens = st["kv_lens"].long()
    first = (lens - st["window"]).clamp_min(0) if st["window"] else torch.zeros_like(lens)
    span = min(st["window"], st["max_len"]) if st["window"] else st["max_len"]
    key = _plain_keys(st, first, lens - 1, span)
    qpos = lens[:, None] - 1
    seq = torch.arange(len(lens), device=lens.device)[:, None]
    return _plain_attend(st, st["q"][:, None], qpos, seq, key, _plain_seen(st, key, qpos))[:, 0].to(st["q"].dtype)


def _plain_prefill(st, block=128):
    """Query blocks of 128, each over its own window's keys."""
    dev, off = st["q"].device, st["q_offsets"].long()
    block = min(block, st["max_q"])
    per = -(-st["max_q"] // block)
    new = off[1:] - off[:-1]
    seq = torch.arange(len(new), device=dev).repeat_interleave(per, output_size=len(new) * per)
    t = (torch.arange(per, device=dev) * block).repeat(len(new))[:, None] + torch.arange(block, device=dev)[None]
    ok = t < new[seq][:, None]
    qpos = torch.where(ok, (st["kv_lens"].long() - new)[seq][:, None] + t, torch.full_like(t, -1))
    row = torch.where(ok, off[seq][:, None] + t, torch.zeros_like(t))
    start = (st["kv_lens"].long() - new)[seq] + t[:, 0]
    first = (start - st["window"] + 1).clamp_min(0) if st["window"] else torch.zeros_like(start)
    span = min(st["window"] - 1 + block, st["max_len"]) if st["window"] else st["max_len"]
    key = _plain_keys(st, first, qpos.amax(1), span)
    o = _plain_attend(st, st["q"][row], qpos, seq[:, None], key, _plain_seen(st, key, qpos))
    out = torch.zeros(len(st["q"]) + 1, *st["q"].shape[1:], device=dev, dtype=st["q"].dtype)
    out[torch.where(ok, row, torch.full_like(row, len(st["q"])))] = o.to(out.dtype)
    return out[:-1]


def _plain_sample(st):
    z = st["logits"].double() / st["temperature"]
    vocab = z.shape[1]
    top, order = torch.sort(z, dim=1, descending=True, stable=True)
    w = torch.exp(top - top[:, :1])
    rank = torch.arange(vocab, device=z.device)[None]
    keep = rank < (st["top_k"] if 0 < st["top_k"] < vocab else vocab)
    w = w * keep
    if st["top_p"] < 1:
        before = w.cumsum(1) - w
        keep = keep & (before < st["top_p"] * w.sum(1, keepdim=True))
    if st["min_p"] > 0:
        keep = keep & (w >= st["min_p"])
    w = torch.zeros_like(w).scatter_(1, order, w * keep)
    cdf = w.cumsum(1)
    target = st["u"].double()[:, None] * cdf[:, -1:]
    ids = torch.searchsorted(cdf, target, right=True).clamp_max(vocab - 1)
    logp = torch.log(w.gather(1, ids) / cdf[:, -1:])
    return {"ids": ids[:, 0], "logprob": logp[:, 0].float()}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    if own:
        return _own(st)
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill, "sample": _plain_sample}[st["op"]](st)


def _own(st):
    from walsh_research_b200 import ops
    if st["op"] == "append":
        q = ops.paged_append(st["q"], st["k"], st["v"], st["k_pages"], st["v_pages"], st["slots"],
                             positions=st["positions"], rope=(st["cos"], st["sin"]), q_norm=st.get("q_norm"),
                             k_norm=st.get("k_norm"), eps=1e-6)
        return {"q": q, "k_pages": st["k_pages"], "v_pages": st["v_pages"]}
    if st["op"] == "decode":
        return ops.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["page_table"], st["kv_lens"],
                                   max_len=st["max_len"], window=st["window"], sinks=st["sinks"])
    if st["op"] == "prefill":
        return ops.paged_prefill_attention(st["q"], st["q_offsets"], st["k_pages"], st["v_pages"], st["page_table"],
                                           st["kv_lens"], max_q=st["max_q"], window=st["window"], sinks=st["sinks"])
    ids, logp = ops.sample_tokens(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                  top_p=st["top_p"], min_p=st["min_p"], want_logprob=True)
    return {"ids": ids, "logprob": logp}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_head_rows(x, w, cos, sin):
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w.double()
    z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * torch.complex(cos.double(), sin.double())[:, None]
    return torch.view_as_real(z).flatten(-2)


def _exact_sequence(q, k, v, pos0, window, sinks):
    """One sequence: q [T, Hq, hd] at positions pos0.., k and v [L, Hkv, hd], all float64."""
    T, h, hd = q.shape
    k = k.repeat_interleave(h // k.shape[1], 1)
    v = v.repeat_interleave(h // v.shape[1], 1)
    out = torch.empty_like(q)
    for t0 in range(0, T, 256):
        t1 = min(T, t0 + 256)
        i = pos0 + torch.arange(t0, t1, device=q.device)[:, None]
        j = torch.arange(k.shape[0], device=q.device)[None]
        hidden = j > i
        if window:
            hidden = hidden | ((i - j >= window) & (j >= sinks))
        s = torch.einsum("thd,jhd->htj", q[t0:t1], k) / math.sqrt(hd)
        p = torch.softmax(s.masked_fill(hidden, float("-inf")), -1)
        out[t0:t1] = torch.einsum("htj,jhd->thd", p, v)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]
        q = _exact_head_rows(st["q"], st.get("q_norm"), cos, sin)
        k = _exact_head_rows(st["k"], st.get("k_norm"), cos, sin)
        kp, vp = (p.double().transpose(1, 2).flatten(0, 1).contiguous() for p in (st["k_pages"], st["v_pages"]))
        kp.index_copy_(0, st["slots"], k)
        vp.index_copy_(0, st["slots"], st["v"].double())
        back = (lambda p: p.unflatten(0, (-1, case["page"])).transpose(1, 2).contiguous())
        return {"q": q, "k_pages": back(kp), "v_pages": back(vp)}
    if case["op"] == "sample":
        z = st["logits"].double().cpu().numpy() / case["temperature"]
        u = st["u"].double().cpu().numpy()
        ids, logp = [], []
        for r in range(case["rows"]):
            order = np.argsort(-z[r], kind="stable")
            if case["top_k"] > 0:
                order = order[:case["top_k"]]
            w = np.exp(z[r][order] - z[r][order[0]])
            n = len(order)
            if case["top_p"] < 1:
                n = 1 + int(np.sum(np.cumsum(w)[:-1] < case["top_p"] * w.sum()))
            n = max(1, min(n, int(np.sum(w >= case["min_p"]))))
            by_index = np.argsort(order[:n])
            cdf = np.cumsum(w[:n][by_index])
            pick = min(n - 1, int(np.searchsorted(cdf, u[r] * cdf[-1], side="right")))
            ids.append(int(order[:n][by_index][pick]))
            logp.append(float(np.log(w[:n][by_index][pick] / cdf[-1])))
        return {"ids": np.array(ids, dtype=np.int64), "logprob": np.array(logp)}
    out = []
    lens, table = st["kv_lens"].tolist(), st["page_table"].long()
    off = st["q_offsets"].tolist() if case["op"] == "prefill" else list(range(len(lens) + 1))
    for b, n in enumerate(lens):
        at = torch.arange(n, device="cuda")
        page, row = table[b][at // case["page"]], at % case["page"]
        q = st["q"][off[b]:off[b + 1]].double()
        out.append(_exact_sequence(q, st["k_pages"][page, :, row].double(), st["v_pages"][page, :, row].double(),
                                   n - len(q), case["window"], case["sinks"]))
    return torch.cat(out)
