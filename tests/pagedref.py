"""Plain float64 forms of the paged-cache operators, their inputs with everything awkward in them, and the
error bounds their tests hold the kernels to (test infrastructure only).

The bounds are counted, not fitted.  With eps = 2^-24 (f32, half a step), a row's result o = sum_j p_j v_j / l
moves by at most

* half a step of the output type, relative to o (2^-8 for bf16, 2^-11 for f16);
* the rounding of P for the tensor core: f16 to nearest 2^-11 per term, two bf16 parts 2^-14, so 2^-11 of
  A = sum_j p_j |v_j| / l covers every form (f32 P: none);
* the scores' own error d_j <= (D + 4) eps scale sum_d |q_d k_jd|, which moves p_j by a factor e^(d_j), in
  numerator and denominator: 2 max_j d_j A;
* the exponentials and the f32 sums over n keys: (16 + n / 8) eps A (pairwise or MMA sums of at most n terms
  round at most n / 8 times in a row here; ex2.approx is good to 2 eps and the scaled argument, up to 2^7, to
  2^7 eps, which the 16 covers for |s| < 8 and ``arg`` below scales for larger ones).
"""
from __future__ import annotations

import math

import torch

EPS = 2.0 ** -24
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def quantise(x):
    """The stored form of rows x: (bytes, f32 scales); see ``cache_write_ir``."""
    x = x.double()
    bad = ~torch.isfinite(x).all(-1)
    amax = torch.where(torch.isfinite(x), x, 0.0).abs().amax(-1)
    s = amax.float() * torch.tensor(1.0 / 127.0, dtype=torch.float32)
    s = torch.where(bad, torch.full_like(s, math.nan), s)
    ok = s > 0
    r = (x / torch.where(ok, s, torch.ones_like(s)).double()[..., None]).float().double()
    q = torch.where(ok[..., None], torch.nan_to_num(r).round().clamp(-127, 127), 0.0)
    return (q + 128).to(torch.uint8), s


def page_of(t, b, pos, page):
    """The page of position pos of sequence b, or None."""
    m = t["table"].shape[1]
    if not 0 <= pos < m * page:
        return None
    pg = int(t["table"][b, pos // page])
    return pg if 0 <= pg < t["KC"].shape[0] else None


def write_ref(t, page, quant):
    """KC, VC (, KS, VS) after the write, from the tensors before it."""
    out = {n: t[n].clone() for n in ("KC", "VC", "KS", "VS") if n in t}
    B, C = t["K"].shape[:2]
    for b in range(B):
        n, f = int(t["lens"][b]), int(t["fresh"][b])
        for c in range(min(f, C)):
            pos = n - f + c
            pg = page_of(t, b, pos, page)
            if pg is None:
                continue
            for x in "KV":
                row = t[x][b, c]
                if quant:
                    by, s = quantise(row)
                    out[x + "C"][pg, :, pos % page] = by
                    out[x + "S"][pg, :, pos % page] = s
                else:
                    out[x + "C"][pg, :, pos % page] = row
    return out


def rows(t, n, b, upto, page):
    """(values [upto, heads, dim] float64, which positions exist) of sequence b."""
    hk, d = t[n + "C"].shape[1], t[n + "C"].shape[3]
    v = torch.zeros(upto, hk, d, dtype=torch.float64)
    ok = torch.zeros(upto, dtype=torch.bool)
    for p in range(upto):
        pg = page_of(t, b, p, page)
        if pg is None:
            continue
        ok[p] = True
        x = t[n + "C"][pg, :, p % page].double()
        if n + "S" in t:
            x = (x - 128) * t[n + "S"][pg, :, p % page].double()[:, None]
        v[p] = x
    return v, ok


def read_ref(t, page, dtype):
    out = {n: t[n].clone() for n in ("KR", "VR")}
    for b in range(t["lens"].shape[0]):
        upto = min(max(int(t["lens"][b]), 0), out["KR"].shape[1], t["table"].shape[1] * page)
        for n in "KV":
            v, ok = rows(t, n, b, upto, page)
            if n + "S" in t:
                # the product is rounded to f32 first, then to the output type
                v = v.float()
            out[n + "R"][b, :upto][ok] = v.to(DT[dtype])[ok]
    return out


def attention_ref(t, page, window=None, sinks=0, scale=None):
    """(O as float64 with untouched rows NaN-free copies of t["O"], bound, written rows) over the chunk."""
    B, C, H, D = t["Q"].shape
    hk = t["KC"].shape[1]
    g = H // hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    ref = t["O"].double().clone()
    bound = torch.zeros_like(ref)
    wrote = torch.zeros(B, C, dtype=torch.bool)
    dtype = "bf16" if t["O"].dtype == torch.bfloat16 else "f16"
    for b in range(B):
        n, f = int(t["lens"][b]), int(t["fresh"][b])
        f = min(max(f, 0), C)
        last = n - int(t["fresh"][b]) + f - 1
        upto = min(max(last + 1, 0), t["table"].shape[1] * page)
        k, ok = rows(t, "K", b, upto, page)
        v, _ = rows(t, "V", b, upto, page)
        j = torch.arange(upto)
        for c in range(f):
            wrote[b, c] = True
            pos = n - int(t["fresh"][b]) + c
            see = ok & (j <= pos)
            if window is not None:
                see = see & ((j > pos - window) | (j < sinks))
            kk, vv = k[see], v[see]
            if kk.shape[0] == 0:
                ref[b, c] = 0
                continue
            q = t["Q"][b, c].double().reshape(hk, g, D)
            s = torch.einsum("hgd,jhd->hgj", q, kk) * scale
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m))
            l = p.sum(-1, keepdim=True)
            l = torch.where(l == 0, torch.ones_like(l), l)
            w = p / l
            o = torch.zeros(hk, g, D, dtype=torch.float64)
            fin = torch.isfinite(vv).all()
            o = torch.einsum("hgj,jhd->hgd", w, vv)
            a = torch.einsum("hgj,jhd->hgd", w, torch.nan_to_num(vv).abs() if not fin else vv.abs())
            d = (torch.einsum("hgd,jhd->hgj", q.abs(), kk.abs()) * abs(scale)).amax(-1, keepdim=True)
            d = torch.nan_to_num(d, posinf=0.0)
            arg = torch.nan_to_num(s.abs().amax(-1, keepdim=True), posinf=0.0) * 4
            nk = kk.shape[0]
            bd = HALF_STEP[dtype] * o.abs() + a * (2.0 ** -11 + 2 * (D + 4) * EPS * d + (16 + nk / 8 + arg) * EPS) + 1e-30
            if dtype == "f16":
                bd = bd + 2.0 ** -25                    # half a subnormal step
            ref[b, c] = o.reshape(H, D)
            bound[b, c] = bd.reshape(H, D)
    return ref, bound, wrote


def check(got, ref, bound, what="", inf_or_nan=False):
    """``got`` within ``bound`` of ``ref``, NaN and infinities in the same places.  ``inf_or_nan`` accepts a NaN for an
    infinity: a kernel that takes P in parts, or in 16 bits, multiplies an infinity that a row sees by a part that can
    be exactly 0 (p = 2^k has no low part; p < 2^-32 of the row's largest rounds to 0 in f16), and 0 * inf is NaN."""
    g, r = got.detach().cpu().double(), ref
    inf = torch.isinf(r)
    if inf_or_nan:
        g = torch.where(inf & torch.isnan(g), r, g)
    nan = torch.isnan(r)
    assert torch.equal(torch.isnan(g), nan), f"{what}: NaN in other places ({int((torch.isnan(g) != nan).sum())})"
    assert torch.equal(g[inf], r[inf]), f"{what}: infinities differ"
    fin = ~nan & ~inf
    err = (g - r).abs()[fin]
    bd = bound[fin]
    bad = err > bd
    if bad.any():
        w = int((err / (bd + 1e-300)).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {err.numel()} outside their bounds, worst error {err[w]:.3e} "
                             f"over {bd[w]:.3e} (value {r[fin][w]:.4f})")


def make(op, batch, kv_heads, dim, page, max_pages, lens, fresh, chunk=1, heads=None, length=None, dtype="bf16",
         quant=False, seed=0, spare=2, stale="nan", sizes=1.0):
    """Inputs of an operator on the CPU.  Pages are shuffled; rows of the cache that no token owns hold
    ``stale`` ("nan" or a number), and outputs start at 7."""
    g = torch.Generator().manual_seed(seed)
    pages = batch * max_pages + spare
    order = torch.randperm(pages, generator=g)[:batch * max_pages].reshape(batch, max_pages).to(torch.int32)
    t = {"table": order, "lens": torch.tensor(lens, dtype=torch.int32), "fresh": torch.tensor(fresh, dtype=torch.int32)}
    dt = DT[dtype]
    shape = (pages, kv_heads, page, dim)
    for n in "KV":
        x = torch.randn(shape, generator=g) * sizes
        if quant:
            t[n + "C"], t[n + "S"] = quantise(x.to(dt))
        else:
            t[n + "C"] = x.to(dt)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(batch):
        for p in range(min(max(int(lens[b]), 0), max_pages * page)):
            used[int(order[b, p // page]), p % page] = True
    for n in "KV":
        fill = math.nan if stale == "nan" else float(stale)
        if quant:
            t[n + "S"].transpose(1, 2)[~used] = fill
        else:
            t[n + "C"].transpose(1, 2)[~used] = fill
    if op == "write":
        for n in "KV":
            t[n] = (torch.randn(batch, chunk, kv_heads, dim, generator=g) * sizes).to(dt)
    elif op == "read":
        for n in ("KR", "VR"):
            t[n] = torch.full((batch, length, kv_heads, dim), 7.0, dtype=dt)
    else:
        t["Q"] = torch.randn(batch, chunk, heads, dim, generator=g).to(dt)
        t["O"] = torch.full((batch, chunk, heads, dim), 7.0, dtype=dt)
    return t, pages
