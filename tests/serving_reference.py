"""Plain float64 forms of the serving operators (paged append, paged
attention, token sampling) that the tests compare the kernels with, and the
bounds on the difference that the kernels' arithmetic allows."""
import math
from fractions import Fraction

import numpy as np
import torch


def make_pool(g, lens, kv_heads, page, hd, dtype, spare=2, cols_extra=0, garbage=None):
    """Pages holding random keys and values for sequences of the given lengths:
    (k_pages, v_pages, page_table int32, kv_lens int32), pages in random order,
    ``spare`` unused ones and NaN in every slot that no sequence owns."""
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + spare
    cols = max(1, max(need, default=1) + cols_extra)
    order = torch.randperm(n_pages, generator=g)
    kp = torch.randn(n_pages, kv_heads, page, hd, generator=g).to(dtype)
    vp = torch.randn(n_pages, kv_heads, page, hd, generator=g).to(dtype)
    table = torch.full((len(lens), cols), -1 if garbage is None else garbage, dtype=torch.int32)
    used = torch.zeros(n_pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]]
        table[b, :need[b]] = ids.int()
        for i, p in enumerate(ids.tolist()):
            used[p, :min(page, n - i * page)] = True
        at += need[b]
    for t in (kp, vp):
        t.transpose(1, 2)[~used] = float("nan")
    return kp, vp, table, torch.tensor(lens, dtype=torch.int32)


def gather_keys(pages, table_row, n):
    """[n, Hkv, hd] of one sequence."""
    page = pages.shape[2]
    at = torch.arange(n, device=pages.device)
    return pages[table_row.long()[at // page], :, at % page]


def attend(q, k, v, pos0, window=0, sinks=0, scale=None, hide=None):
    """q [T, Hq, hd] at positions pos0.. over k, v [L, Hkv, hd], float64.
    Returns (o, bound): the bound covers one rounding of the result to q's
    type, one of each probability to it, and the float32 arithmetic."""
    T, hq, hd = q.shape
    dt, L = q.dtype, k.shape[0]
    scale = hd ** -0.5 if scale is None else scale
    if L == 0:
        return torch.zeros(T, hq, hd, dtype=torch.float64, device=q.device), torch.zeros(T, hq, hd, device=q.device)
    g = hq // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(g, 1), v.double().repeat_interleave(g, 1)
    i = pos0 + torch.arange(T, device=q.device)[:, None]
    j = torch.arange(L, device=q.device)[None]
    see = j <= i
    if window:
        see = see & ((j > i - window) | (j < sinks))
    if hide is not None:
        see = see & ~hide[None]
    s = torch.einsum("thd,jhd->htj", q, k) * scale
    s_abs = torch.einsum("thd,jhd->htj", q.abs(), k.abs()).masked_fill(~see, 0.0).amax(-1) * scale   # [h, t]
    m = s.masked_fill(~see, float("-inf")).amax(-1, keepdim=True)
    p = torch.exp(s - m.clamp_min(-1e300)).masked_fill(~see, 0.0)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    v = torch.where(see.any(0)[:, None, None], v, torch.zeros_like(v))
    o = torch.einsum("htj,jhd->thd", p, v)
    a = torch.einsum("htj,jhd->thd", p, v.abs())
    half = torch.finfo(dt).eps / 2
    # a score is a float32 sum of hd products scaled once (hd + 4 roundings of at
    # most s_abs) and its exponential good to 2^-22; numerator and denominator
    # both carry that; the sums over the keys run in at least 16 parts
    d = 2 * (2.0 ** -24 * (hd + 4) * s_abs + 2.0 ** -22) + 2 * (L / 16 + 64) * 2.0 ** -24
    bound = half * o.abs() + (half + d.t()[..., None]) * a
    # results below the type's normal range are rounded to multiples of its smallest step
    return o, bound + torch.finfo(dt).tiny * torch.finfo(dt).eps


def rotate(x, w, cos, sin, eps=1e-6):
    """Norm (w not None) and rotation (cos not None) of x [N, H, hd] in float64, with
    the bound on a result rounded once to x's type."""
    dt, hd = x.dtype, x.shape[-1]
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    mag = y.abs()
    if cos is not None:
        c, s = cos.double()[:, None], sin.double()[:, None]
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
        mag = torch.stack(((a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()), -1).flatten(-2)
    # float32: the mean of hd squares (hd roundings, halved by the root), root,
    # division, two products, and two products and a sum of the rotation
    return y, torch.finfo(dt).eps / 2 * y.abs() + (hd / 2 + 8) * 2.0 ** -24 * mag + torch.finfo(dt).tiny * torch.finfo(dt).eps


def sample_row(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One draw from logits z [V] (float64 values) by the definition; (id, log
    probability).  Weights are float64 exponentials as multiples of 2^-60, so
    that sums are exact: equal weights stay equal and a number that falls on a
    border falls on it here too."""
    z = np.where(np.isnan(z), -np.inf, z)
    m = z.max()
    if m == -np.inf:
        return -1, float("nan")
    V = len(z)
    if not temperature > 0:
        return int(z.argmax()), 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(z == m, 1.0, np.where(z == -np.inf, 0.0, np.exp((z - m) / temperature)))
    order = np.argsort(-z, kind="stable")
    if 0 < top_k < V:
        order = order[:top_k]
    whole = [int(x) for x in np.rint(w * 2.0 ** 60)]
    n = len(order)
    if top_p < 1:
        reach = top_p * float(sum(whole[i] for i in order))
        n, before = 0, 0
        while n < len(order) and (n == 0 or before < reach):
            before += whole[order[n]]
            n += 1
    kept = np.zeros(V, dtype=bool)
    kept[order[:n]] = True
    kept &= w >= min(min_p, 1.0)
    total = sum(whole[i] for i in np.flatnonzero(kept))
    t = Fraction(min(max(float(u), 0.0), 1.0) if u == u else 0.0) * total
    run, last = 0, -1
    for i in np.flatnonzero(kept):
        run += whole[i]
        if whole[i]:
            last = i
        if run > t:
            break
    return int(last), math.log(w[last] / (total / 2.0 ** 60))
