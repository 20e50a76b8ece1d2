"""A paged key/value cache written and read back: one pass of wide loads and stores over the tokens.

They move rows 16 or 32 bytes a thread and compute no more than a row needs.  In 16 bits they are bound by HBM; a decode
step by the chain lengths -> table -> row; the quantising write by its instructions (72 % of the issue slots of
its active cycles), the read of bytes by the latency of lengths -> table -> row and scale -> store (52 warps an SM, 53 %):

* **write** (:func:`..irgen.cache_write_ir`): dim / 8 lanes a row, 16 bytes of K and of V each.  For a cache of
  bytes the lanes find max|x| on the 16-bit patterns (their order without the sign is the numbers' order, and the
  largest tells an infinity or a NaN in the row), a row's lanes meet in shuffles, and each packs 8 bytes.
  round(x / s) is taken from x * (1 / s), which is within 2^-15 of the quotient for |x / s| <= 127: where that
  lies within 1e-4 of a half (or s is so small that 1 / s overflows) the warp divides instead, so every
  byte is that of the rounded quotient.
* **read** (:func:`..irgen.cache_read_ir`): 16 values a thread of K and of V: 16 bytes in (or 32), 32 out.
  (byte - 128) is exact in f32 (0x4B000000 | b is 2^23 + b), times the scale, rounded once more to the output.

Measured on one B200: a decode step's write (64 tokens, 8 heads of 128, bf16) 2.0 us on the GPU in a run of calls; 16
sequences of 100 to 4096 tokens of bytes read back (8 heads of 64, f16, 107 MB) 20-24 us, 4.4-5.2 TB/s, and from a bf16
cache of 8 heads of 128 (280 MB) 43 us, 6.5 TB/s; 8 prompts of 300 to 2048 tokens written in bf16 20 us (101 MB),
quantised and read back 38-41 us for both calls.

Offsets into the pool are 64-bit.
"""
from __future__ import annotations

from .tc_paged_attention import _E, _f32

THREADS = 256
SAFE = 0.4999                    # |x * inv - round(x * inv)| below this: the quotient rounds to the same number


def _common(e):
    def gptr(pname):
        return e.o("cvta.to.global.u64", e.o("ld.param.u64", f"[{pname}]", cls="rd"), cls="rd")

    def at(base, off):
        return e.o("add.s64", base, off, cls="rd")

    def wide(x, n):
        return e.o("mul.wide.u32", x, n, cls="rd")
    return gptr, at, wide


def _page_row(e, at, wide, gptr, b, pos, kvh, kv_heads, page, pages, max_pages):
    """The pool's row (over pages, heads and rows, 64 bits) of position ``pos`` < max_pages * page; returns from the
    kernel where the table names no page."""
    o = e.o
    slot, row = o("div.u32", pos, page), o("rem.u32", pos, page)
    pg = o("ld.global.nc.u32", f"[{at(at(gptr('p_table'), wide(b, 4 * max_pages)), wide(slot, 4))}]")
    e(f"@{e.cond('ge.u32', pg, pages)} ret;")                   # negative numbers are large ones here
    return o("mad.wide.u32", pg, kv_heads * page, wide(o("mad.lo.u32", kvh, page, row), 1), cls="rd")


def _record(name, kind, e, params, cells):
    text = [f".visible .entry {name}(", ",\n".join(f"\t.param .u64 p_{p}" for p, _, _ in params), ")",
            f".reqntid {THREADS}, 1, 1", "{"] + e.decls() + e.lines + ["\tret;", "}"]
    return {"name": name, "kind": kind, "params": [n for _, n, _ in params], "raw_entry": text,
            "grid": [-(-cells // THREADS), 1, 1], "block": [THREADS, 1, 1], "dyn_smem": 0,
            "align": {n: a for _, n, a in params}, "zero_outputs": []}


def cache_write_entry(name, batch, chunk, kv_heads, dim, pages, page, max_pages, dtype, quant, names):
    """``names``: K, V, table, lens, fresh, KC, VC (, KS, VS)."""
    e = _E()
    o = e.o
    gptr, at, wide = _common(e)
    lpr = dim // 8                                              # lanes a row
    cells = batch * chunk * kv_heads * lpr
    gid = o("mad.lo.u32", o("mov.u32", "%ctaid.x"), THREADS, o("mov.u32", "%tid.x"))
    live = e.cond("lt.u32", gid, cells)
    e(f"@!{live} ret;")
    ln, r_ = o("rem.u32", gid, lpr), o("div.u32", gid, lpr)
    kvh, bc = o("rem.u32", r_, kv_heads), o("div.u32", r_, kv_heads)
    c, b = o("rem.u32", bc, chunk), o("div.u32", bc, chunk)
    b_len = o("ld.global.nc.u32", f"[{at(gptr('p_lens'), wide(b, 4))}]")
    b_new = o("ld.global.nc.u32", f"[{at(gptr('p_fresh'), wide(b, 4))}]")
    # the rows themselves do not wait for the page
    xs = []
    for n in "KV":
        src = at(gptr(f"p_{n}"), wide(gid, 16))
        ws = [e.r() for _ in range(4)]
        e(f"ld.global.nc.L1::no_allocate.v4.b32 {{{', '.join(ws)}}}, [{src}];")
        xs.append(ws)
    e(f"@{e.cond('ge.s32', c, b_new)} ret;")
    pos = o("add.s32", o("sub.s32", b_len, b_new), c)
    e(f"@{e.cond('ge.u32', pos, max_pages * page)} ret;")       # negative positions are large ones here
    row = _page_row(e, at, wide, gptr, b, pos, kvh, kv_heads, page, pages, max_pages)
    if not quant:
        for n, ws in zip("KV", xs):
            dst = at(at(gptr(f"p_{n}C"), o("mul.lo.s64", row, dim * 2, cls="rd")), wide(ln, 16))
            e(f"st.global.v4.b32 [{dst}], {{{', '.join(ws)}}};")
    else:
        inf_bits = 0x7F80 if dtype == "bf16" else 0x7C00
        # a row's lanes are all here or all gone: the shuffles' members are this row's group
        for n, ws in zip("KV", xs):
            m = None
            for x in ws:
                a_ = o("and.b32", x, "0x7FFF7FFF")
                m = a_ if m is None else o("max.u16x2", m, a_)
            m = o("max.u32", o("and.b32", m, 65535), o("shr.u32", m, 16))
            d = lpr // 2
            mask = o("shl.b32", (1 << lpr) - 1 if lpr < 32 else -1,
                     o("and.b32", o("and.b32", gid, 31), 32 - lpr) if lpr < 32 else 0)
            while d:
                m = o("max.u32", m, o("shfl.sync.bfly.b32", m, d, 31, mask))
                d //= 2
            if dtype == "bf16":
                amax = o("shl.b32", m, 16, cls="f")
            else:
                lo, hi = "%h0", "%h1"
                e(f"mov.b32 {{{lo}, {hi}}}, {m};")
                amax = o("cvt.f32.f16", lo, cls="f")
            s = o("mul.rn.f32", amax, _f32(1.0 / 127.0), cls="f")
            e(f"@{e.cond('ge.u32', m, inf_bits)} mov.b32 {s}, 0f7FFFFFFF;")
            ok = e.cond("gt.f32", s, "0f00000000")               # a zero row, or a NaN scale: all bytes 128
            inv = o("rcp.rn.f32", s, cls="f")
            vals = []
            for x in ws:
                if dtype == "bf16":
                    vals += [o("shl.b32", x, 16, cls="f"), o("and.b32", x, -65536, cls="f")]
                else:
                    e(f"mov.b32 {{%h0, %h1}}, {x};")
                    vals += [o("cvt.f32.f16", "%h0", cls="f"), o("cvt.f32.f16", "%h1", cls="f")]
            qs = []
            odd = e.cond("ne.u32", gid, gid)
            magic = "0f4B400000"                                 # 1.5 * 2^23: adding it rounds to an integer
            for v in vals:
                y = o("mul.rn.f32", v, inv, cls="f")
                q = o("sub.rn.f32", o("add.rn.f32", y, magic, cls="f"), magic, cls="f")
                dlt = o("abs.f32", o("sub.rn.f32", y, q, cls="f"), cls="f")
                p_ = e.cond("ltu.f32", _f32(SAFE), dlt)         # or a NaN
                e(f"or.pred {odd}, {odd}, {p_};")
                qs.append(q)
            l_fast = e.L("fast")
            e(f"and.pred {odd}, {odd}, {ok};")
            e(f"@!{odd} bra {l_fast};")
            for v, q in zip(vals, qs):
                y = o("div.rn.f32", v, s, cls="f")
                e(f"cvt.rni.f32.f32 {q}, {y};")
                e(f"max.f32 {q}, {q}, 0fC2FE0000;")              # a scale near f32's smallest steps past 127
                e(f"min.f32 {q}, {q}, 0f42FE0000;")
            e.label(l_fast)
            bytes_ = []
            for q in qs:
                q0 = o("selp.f32", q, "0f00000000", ok, cls="f")
                bytes_.append(o("add.rn.f32", q0, "0f4B000080", cls="f"))     # 2^23 + 128 + q: the byte is its low 8 bits
            words = []
            for i in range(0, 8, 4):
                lo_ = o("prmt.b32", bytes_[i], bytes_[i + 1], "0x0040")
                hi_ = o("prmt.b32", bytes_[i + 2], bytes_[i + 3], "0x0040")
                words.append(o("prmt.b32", lo_, hi_, "0x5410"))
            dst = at(at(gptr(f"p_{n}C"), o("mul.lo.s64", row, dim, cls="rd")), wide(ln, 8))
            e(f"st.global.v2.b32 [{dst}], {{{words[0]}, {words[1]}}};")
            sd = at(gptr(f"p_{n}S"), o("mul.lo.s64", row, 4, cls="rd"))
            e(f"@{e.cond('eq.u32', ln, 0)} st.global.f32 [{sd}], {s};")
    kn, vn, tn, lnn, fn, kcn, vcn = names[:7]
    params = [("K", kn, 16), ("V", vn, 16), ("table", tn, 4), ("lens", lnn, 4), ("fresh", fn, 4), ("KC", kcn, 16),
              ("VC", vcn, 16)]
    if quant:
        params += [("KS", names[7], 4), ("VS", names[8], 4)]
    rec = _record(name, "cache_write", e, params, cells)
    if quant and dtype == "f16":
        rec["raw_entry"].insert(rec["raw_entry"].index("{") + 1, "\t.reg .b16 %h<2>;")
    return rec


def cache_read_entry(name, batch, length, kv_heads, dim, pages, page, max_pages, dtype, quant, names):
    """``names``: KC, VC, (KS, VS,) table, lens, KR, VR."""
    e = _E()
    o = e.o
    gptr, at, wide = _common(e)
    lpr = dim // 16
    cells = batch * length * kv_heads * lpr
    gid = o("mad.lo.u32", o("mov.u32", "%ctaid.x"), THREADS, o("mov.u32", "%tid.x"))
    e(f"@{e.cond('ge.u32', gid, cells)} ret;")
    ln, r_ = o("rem.u32", gid, lpr), o("div.u32", gid, lpr)
    kvh, bt = o("rem.u32", r_, kv_heads), o("div.u32", r_, kv_heads)
    t, b = o("rem.u32", bt, length), o("div.u32", bt, length)
    b_len = o("ld.global.nc.u32", f"[{at(gptr('p_lens'), wide(b, 4))}]")
    e(f"@{e.cond('ge.s32', t, b_len)} ret;")
    if length > max_pages * page:
        e(f"@{e.cond('ge.u32', t, max_pages * page)} ret;")
    row = _page_row(e, at, wide, gptr, b, t, kvh, kv_heads, page, pages, max_pages)
    loaded = []
    for n in "KV":
        src = at(at(gptr(f"p_{n}C"), o("mul.lo.s64", row, dim * (1 if quant else 2), cls="rd")),
                 wide(ln, 16 if quant else 32))
        ws = [e.r() for _ in range(4 if quant else 8)]
        e(f"ld.global.nc.L1::no_allocate.v{len(ws)}.b32 {{{', '.join(ws)}}}, [{src}];")
        s = o("ld.global.nc.f32", f"[{at(gptr(f'p_{n}S'), o('mul.lo.s64', row, 4, cls='rd'))}]", cls="f") if quant else None
        loaded.append((ws, s))
    for n, (ws, s) in zip("KV", loaded):
        dst = at(gptr(f"p_{n}R"), wide(gid, 32))
        if quant:
            c4b = o("mov.b32", "0x4B000000")
            out = []
            for x in ws:
                f = []
                for k in range(4):
                    y = o("prmt.b32", x, c4b, f"0x744{k}", cls="f")           # 2^23 + byte k
                    f.append(o("mul.rn.f32", o("sub.rn.f32", y, "0f4B000080", cls="f"), s, cls="f"))
                pk = "cvt.rn.bf16x2.f32" if dtype == "bf16" else "cvt.rn.f16x2.f32"
                out += [o(pk, f[1], f[0]), o(pk, f[3], f[2])]
            ws = out
        e(f"st.global.v8.b32 [{dst}], {{{', '.join(ws)}}};")
    if quant:
        kcn, vcn, ksn, vsn, tn, lnn, krn, vrn = names
        params = [("KC", kcn, 16), ("VC", vcn, 16), ("KS", ksn, 4), ("VS", vsn, 4)]
    else:
        kcn, vcn, tn, lnn, krn, vrn = names
        params = [("KC", kcn, 32), ("VC", vcn, 32)]
    params += [("table", tn, 4), ("lens", lnn, 4), ("KR", krn, 32), ("VR", vrn, 32)]
    return _record(name, "cache_read", e, params, cells)
