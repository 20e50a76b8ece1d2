"""The paged key/value cache operators as measured work: their cases, inputs, plain forms and exact values.

Three operators belong together here, the serving side of attention:

* the cache written: the new tokens' keys and values go to the pages of their sequences, in the activations'
  own 16-bit type or as bytes with one f32 scale per token and head;
* the cache read back: the first tokens of every sequence, gathered from their pages (and scaled back);
* attention of a chunk of new tokens over the pages, causal, with grouped heads, over all keys or over a
  sliding window and a few first tokens that stay visible.

A sequence b holds ``lens[b]`` tokens, the last ``fresh[b]`` of them new; token p of it sits in row ``p % page``
of page ``table[b, p // page]``.  New token c has position ``lens[b] - fresh[b] + c``; rows c >= fresh[b] of a
chunk are padding and are not written.
"""
import math

import torch

own = False

_T = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases ------------------------------------------------------------------------------------------------


def _attn(name, batch, chunk, heads, kv_heads, dim, page, longest, shortest, dtype="bf16", quant=False, window=0,
          sinks=0):
    return {"name": name, "op": "attention", "batch": batch, "chunk": chunk, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "page": page, "longest": longest, "shortest": shortest, "dtype": dtype, "quant": quant,
            "window": window, "sinks": sinks}


def _cache(op, name, batch, chunk, kv_heads, dim, page, longest, shortest, dtype="bf16", quant=False):
    return {"name": name, "op": op, "batch": batch, "chunk": chunk, "kv_heads": kv_heads, "dim": dim, "page": page,
            "longest": longest, "shortest": shortest, "dtype": dtype, "quant": quant}


def listed():
    return [
        # one decode step's keys and values of a batch of 64 go to their pages: a call where latency counts
        _cache("write", "write_step_bf16", 64, 1, 8, 128, 16, 4000, 1, "bf16", False),
        # prompts of up to 2048 tokens are quantised as they are written, and read back (the values that a
        # check of the cache or a second model on it sees)
        _cache("write_read", "write_read_prompt_u8", 8, 2048, 8, 128, 64, 2048, 300, "bf16", True),
        # a quantised cache read back whole, at a head dim of 64 and small pages, in f16
        _cache("read", "read_u8_f16", 16, 1, 8, 64, 16, 4096, 100, "f16", True),
        # the first tokens of a single conversation: the smallest attention call
        _attn("decode_one_bf16", 1, 1, 32, 8, 128, 16, 333, 333),
        # a serving batch in decode with ragged lengths, four query heads to a key head
        _attn("decode_batch_bf16", 48, 1, 32, 8, 128, 16, 8192, 17),
        # the same serving batch on a cache of bytes
        _attn("decode_batch_u8", 48, 1, 32, 8, 128, 64, 8192, 17, quant=True),
        # one long document in decode, every query head with keys of its own, head dim 64, f16
        _attn("decode_long_f16", 1, 1, 32, 32, 64, 64, 131072, 131072, "f16"),
        # five drafted tokens a sequence to check at once, on a cache of bytes
        _attn("draft_u8", 16, 5, 32, 4, 128, 32, 5000, 800, quant=True),
        # decode behind a window of 1000 tokens and 4 first ones, on long sequences
        _attn("decode_window_bf16", 64, 1, 32, 8, 128, 16, 30000, 1, window=1000, sinks=4),
        # a chunk of a long prompt, most of it already in the cache: the largest call
        _attn("chunk_bf16", 2, 2048, 32, 8, 128, 64, 8192, 6000),
        # a ragged chunk behind a window, f16, head dim 64, six query heads to a key head
        _attn("chunk_window_f16", 4, 1111, 24, 4, 64, 16, 6000, 700, "f16", window=1024, sinks=4),
        # a chunk on a cache of bytes
        _attn("chunk_u8", 4, 512, 32, 8, 128, 64, 4096, 512, quant=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "f16"])
    quant = rng.random() < 0.5
    dim = rng.choice([64, 128])
    page = rng.choice([8, 16, 32, 64, 128])
    kind = rng.choice(["write", "write_read", "read", "decode", "decode", "chunk", "chunk", "window"])
    if kind in ("write", "write_read", "read"):
        batch = _log(rng, 1, 64)
        longest = _log(rng, 16, 32768 // batch)
        chunk = _log(rng, 1, longest) if kind != "read" else 1
        quant = quant or kind == "write_read"
        if kind == "write":
            quant = False
        return {k: v for k, v in _cache(kind, "", batch, chunk, rng.choice([1, 2, 4, 8]), dim, page, longest,
                                        rng.randint(1, longest), dtype, quant).items() if k != "name"}
    group = rng.choice([1, 2, 3, 4, 6, 8, 16])
    kv_heads = rng.choice([1, 2, 4, 8])
    if kind == "decode":
        batch = _log(rng, 1, 64)
        longest = _log(rng, 1, 262144 // batch)
        chunk = min(rng.choice([1, 1, 1, 2, 3, 7]), longest)
    else:
        batch = _log(rng, 1, 8)
        longest = _log(rng, 64, 8192 // batch)
        chunk = _log(rng, 8, min(longest, 2500 // batch))
        while group * kv_heads > 32:
            group //= 2
    window = _log(rng, 1, longest) if kind == "window" or rng.random() < 0.2 else 0
    sinks = rng.randint(0, 70) if window else 0
    return {k: v for k, v in _attn("", batch, chunk, group * kv_heads, kv_heads, dim, page, longest,
                                   rng.randint(1, longest), dtype, quant, window, sinks).items() if k != "name"}


# ---- inputs -----------------------------------------------------------------------------------------------


def _lengths(case, seed):
    """Per sequence: tokens in the cache and how many of them are new (the longest sequence first)."""
    g = torch.Generator().manual_seed(seed * 7919 + 11)
    b, lo, hi, chunk = case["batch"], case["shortest"], case["longest"], case["chunk"]
    lens = torch.randint(lo, hi + 1, (b,), generator=g, dtype=torch.int32)
    lens[0] = hi
    full = case["op"] == "write_read"            # whole prompts: every token of a sequence is new
    fresh = lens.clamp(max=chunk)
    if chunk > 1 and not full and b > 1:         # a batch in which some sequences bring less than a chunk
        some = torch.randint(1, chunk + 1, (b,), generator=g, dtype=torch.int32)
        fresh[1::2] = torch.minimum(fresh, some)[1::2]
    return lens, fresh


def _sizes(case):
    per = -(-case["longest"] // case["page"])    # pages a sequence may hold
    return per, case["batch"] * per + 3          # and pages in the pool, a few of them never used


def _quantise(x):
    """Bytes and f32 scales of rows along the last axis: scale = max|x| / 127, byte = 128 + round(x / scale)."""
    x = x.float()
    scale = x.abs().amax(-1) / 127.0
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = torch.round(x / safe[..., None]).clamp(-127, 127)
    return (q + 128).to(torch.uint8), scale


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _T[case["dtype"]]
    b, hk, d, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    per, pool = _sizes(case)
    lens, fresh = _lengths(case, seed)
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed + 5))
    st = {"table": order[:b * per].reshape(b, per).to(torch.int32).cuda(), "lens": lens.cuda(), "fresh": fresh.cuda()}

    def rows(*shape):
        # every token and head has a size of its own, as keys and values of real layers do
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
        return x * torch.exp(0.3 * torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))

    if case["quant"]:
        for n in "KV":
            st[n + "C"], st[n + "S"] = _quantise(rows(pool, hk, page, d))
    else:
        for n in "KV":
            st[n + "C"] = rows(pool, hk, page, d).to(dt)
    if case["op"] == "attention":
        st["Q"] = torch.randn((b, case["chunk"], case["heads"], d), generator=g, device="cuda").to(dt)
        st["O"] = torch.zeros_like(st["Q"])
    elif case["op"] in ("write", "write_read"):
        for n in "KV":
            st[n] = rows(b, case["chunk"], hk, d).to(dt)
    if case["op"] in ("read", "write_read"):
        for n in "KV":
            st[n + "R"] = torch.zeros((b, case["longest"], hk, d), device="cuda", dtype=dt)
    return st


def prepare(case, seed):
    state = {"case": dict(case), "t": _inputs(case, seed)}
    if own:
        from emmy_ptx_b200 import irgen
        from emmy_ptx_b200.compiler import compile_graph
        from emmy_ptx_b200.ir import Graph
        from emmy_ptx_b200.runtime import Executable
        per, pool = _sizes(case)
        common = dict(kv_heads=case["kv_heads"], dim=case["dim"], pages=pool, page=case["page"], max_pages=per,
                      dtype=case["dtype"], quant=case["quant"])
        probs = []
        if case["op"] == "attention":
            probs.append(irgen.paged_attention_ir(case["batch"], case["chunk"], case["heads"],
                                                  window=case["window"] or None, sinks=case["sinks"], **common))
        if case["op"] in ("write", "write_read"):
            probs.append(irgen.cache_write_ir(case["batch"], case["chunk"], **common))
        if case["op"] in ("read", "write_read"):
            probs.append(irgen.cache_read_ir(case["batch"], case["longest"], **common))
        state["ex"] = [Executable(compile_graph(Graph.from_dict(p.graph), p.meta())) for p in probs]
    return state


# ---- one pass ---------------------------------------------------------------------------------------------


def _positions(case, t, dev):
    """Positions [B, C] of a chunk's tokens, -1 for padding rows."""
    c = torch.arange(case["chunk"], device=dev)
    pos = (t["lens"] - t["fresh"])[:, None] + c
    return torch.where(c < t["fresh"][:, None], pos, -1)


def _plain_write(case, t):
    pos = _positions(case, t, t["K"].device).long()
    page, keep = case["page"], pos >= 0
    pid = torch.gather(t["table"].long(), 1, pos.clamp(min=0) // page)
    where = (pid[keep], pos[keep] % page)
    for n in "KV":
        x = t[n][keep]                                        # [tokens, heads, dim]
        if case["quant"]:
            q, scale = _quantise(x)
            t[n + "S"][where[0], :, where[1]] = scale
            t[n + "C"][where[0], :, where[1]] = q
        else:
            t[n + "C"][where[0], :, where[1]] = x


def _gathered(case, t, n):
    """Every sequence's tokens in order, [B, pages * page, heads, dim] in f32."""
    x = t[n + "C"][t["table"].long()].float()                 # [B, pages, heads, page, dim]
    if case["quant"]:
        x = (x - 128.0) * t[n + "S"][t["table"].long()][..., None]
    b, per, hk, page, d = x.shape
    return x.permute(0, 1, 3, 2, 4).reshape(b, per * page, hk, d)


def _plain_read(case, t):
    dt = _T[case["dtype"]]
    live = torch.arange(case["longest"], device=t["lens"].device) < t["lens"][:, None]
    for n in "KV":
        x = _gathered(case, t, n)[:, :case["longest"]].to(dt)
        t[n + "R"] = torch.where(live[:, :, None, None], x, t[n + "R"])
    return [t["KR"], t["VR"]]


def _plain_attention(case, t):
    dt = _T[case["dtype"]]
    out = torch.zeros_like(t["Q"])
    pos_all = _positions(case, t, t["Q"].device)
    group, d = case["heads"] // case["kv_heads"], case["dim"]
    step = max(1, (1 << 28) // (case["chunk"] * case["heads"] * case["longest"] + case["longest"] * case["kv_heads"] * d))
    for b0 in range(0, case["batch"], step):                  # as many sequences at once as memory holds well
        part = {k: (t[k][b0:b0 + step] if k in ("Q", "table", "lens", "fresh") else t[k]) for k in t}
        k, v = _gathered(case, part, "K"), _gathered(case, part, "V")
        n, length = k.shape[0], k.shape[1]
        q = part["Q"].float().reshape(n, case["chunk"], case["kv_heads"], group, d)
        q = q.permute(0, 2, 1, 3, 4).reshape(n, case["kv_heads"], case["chunk"] * group, d)
        s = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
        pos = pos_all[b0:b0 + step]
        key = torch.arange(length, device=q.device)
        see = key <= pos[:, :, None]
        if case["window"]:
            see = see & ((key > pos[:, :, None] - case["window"]) | (key < case["sinks"]))
        see = see[:, None, :, None, :].expand(n, 1, case["chunk"], group, length).reshape(
            n, 1, case["chunk"] * group, length)
        s = torch.where(see, s, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, torch.ones_like(total))
        o = o.reshape(n, case["kv_heads"], case["chunk"], group, d).permute(0, 2, 1, 3, 4)
        out[b0:b0 + step] = o.reshape(n, case["chunk"], case["heads"], d).to(dt)
    return [out]


def run(state):
    case, t = state["case"], state["t"]
    if own:
        for ex in state["ex"]:
            ex(t)
        if case["op"] == "attention":
            return [t["O"]]
        return [t["KC"], t["VC"]] if case["op"] == "write" else [t["KR"], t["VR"]]
    if case["op"] == "attention":
        return _plain_attention(case, t)
    if case["op"] in ("write", "write_read"):
        _plain_write(case, t)
    if case["op"] == "write":
        return [t["KC"], t["VC"]]
    return _plain_read(case, t)


# ---- what a pass cannot do without ------------------------------------------------------------------------


def work(case):
    """Bytes and operations for the lengths of seed 0 (other seeds draw others from the same range)."""
    lens, fresh = _lengths(case, 0)
    hk, d = case["kv_heads"], case["dim"]
    row = hk * ((d + 4) if case["quant"] else 2 * d)          # one token's keys (or values) in the cache
    tokens = int(fresh.sum())
    if case["op"] != "attention":
        nbytes = 0
        if case["op"] in ("write", "write_read"):
            nbytes += tokens * 2 * (hk * d * 2 + row)
        if case["op"] in ("read", "write_read"):
            nbytes += int(lens.sum()) * 2 * (hk * d * 2 + row)
        return {"bytes": nbytes, "flops": nbytes}
    w, sinks = case["window"], case["sinks"]
    keys = pairs = 0
    for n, f in zip(lens.tolist(), fresh.tolist()):
        pos = torch.arange(n - f, n, dtype=torch.int64)
        if not w:
            keys += n
            pairs += int((pos + 1).sum())
            continue
        lo = (pos - w + 1).clamp(min=0)
        first = torch.minimum(lo, torch.full_like(lo, sinks))
        pairs += int((pos + 1 - lo + first).sum())
        keys += n - int(lo[0]) + int(first[0])
    return {"bytes": keys * 2 * row + tokens * case["heads"] * d * 4, "flops": 4 * pairs * case["heads"] * d}


# ---- exact values -----------------------------------------------------------------------------------------


def _exact_rows(case, t, n, b, length):
    """The first ``length`` tokens of sequence b in float64, [heads, length, dim]."""
    page = case["page"]
    ids = t["table"][b, :-(-length // page)].long()
    x = t[n + "C"].index_select(0, ids).double()
    if case["quant"]:
        x = (x - 128) * t[n + "S"].index_select(0, ids).double().unsqueeze(-1)
    return x.transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :length]


def exact(case, seed):
    t = _inputs(case, seed)
    lens, fresh = t["lens"].tolist(), t["fresh"].tolist()
    if case["op"] == "attention":
        out = torch.zeros(t["Q"].shape, dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for b, (n, f) in enumerate(zip(lens, fresh)):
            k, v = _exact_rows(case, t, "K", b, n), _exact_rows(case, t, "V", b, n)
            j = torch.arange(n, device="cuda")
            for c0 in range(0, f, 256):
                c1 = min(f, c0 + 256)
                i = torch.arange(n - f + c0, n - f + c1, device="cuda").unsqueeze(1)
                hidden = j > i
                if case["window"]:
                    hidden |= (j <= i - case["window"]) & (j >= case["sinks"])
                for h in range(case["heads"]):
                    s = t["Q"][b, c0:c1, h].double() @ k[h // group].T / math.sqrt(case["dim"])
                    out[b, c0:c1, h] = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1) @ v[h // group]
        return [out]
    if case["op"] in ("write", "write_read"):
        page = case["page"]
        if case["op"] == "write":
            res = [t["KC"].double(), t["VC"].double()]
        else:
            res = [t["KR"].double(), t["VR"].double()]
        for b, (n, f) in enumerate(zip(lens, fresh)):
            p = torch.arange(n - f, n, device="cuda")
            for r, name in zip(res, "KV"):
                if case["op"] == "write_read":
                    r[b, :n] = _exact_rows(case, t, name, b, n).transpose(0, 1)
                x = t[name][b, :f].double()
                if case["quant"]:
                    # the scale and the ratio are defined as f32 numbers; all else is exact
                    scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()
                    ratio = (x / scale).float().double().nan_to_num(0.0)
                    x = ratio.round().clamp(-127, 127) * scale
                if case["op"] == "write":
                    r[t["table"][b, p // page].long(), :, p % page] = x
                else:
                    r[b, p] = x
        return res
    res = [t["KR"].double(), t["VR"].double()]
    for b, n in enumerate(lens):
        for r, name in zip(res, "KV"):
            r[b, :n] = _exact_rows(case, t, name, b, n).transpose(0, 1)
    return res
