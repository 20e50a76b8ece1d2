"""Attention of a chunk of new tokens over a paged key/value cache, on the 5th-generation tensor cores.

O = softmax(Q K^T * scale) V over the keys each token sees (:func:`..irgen.paged_attention_ir`): the keys up to
its own position, or a window of them and a few first ones, in pages that a table names.  The cache holds the
activations' 16-bit type, or bytes with one f32 scale per token and head.

**Work.**  A CTA owns up to 128 query rows of one sequence and one key head: as many tokens as fit with all
their query heads (a row is token * group + head of the group), so one pass over a key head's keys serves its
whole group.  It walks its keys in tiles of 64, the tiles of the first tokens and then those of the window
when there is one.  When that makes too few CTAs for the GPU, or leaves it to one long sequence, the tiles
of a unit are split over ``splits`` CTAs, each of at least ``min_tiles``; parts store O, the row's reference m and its sum
l in f32 and a second entry joins them (o = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s).  A unit whose
tiles fit one part writes O itself.  Two CTAs share an SM (half its TMEM columns and shared memory each), so
one's loads and softmax run beside the other's products.

**Roles.**  One thread issues the ``tcgen05.mma``: S(j+1) = Q K_(j+1)^T into one of two 64-column score buffers,
then O += P(j) V_j.  Four softmax warps hold one row a thread; warps without a row take no part, so a decode step
costs one warp's softmax.  16-bit caches are loaded by TMA, one box per page of the tile (at most 64 rows), with
the page numbers fetched 32 at a time one batch ahead.  For a cache of bytes four warps load 16 bytes a thread a
tile ahead, convert and store into the tiles' swizzled layout: a byte b is b - 128, exact in bf16
(0x4300 | (b & 127) is 128 + (b & 127), less 128 or 256) and in f16 (0x6400 | b is 1024 + b, less 1152), so no
product is rounded.  The keys' scales multiply the scores' columns, the values' scales multiply P.

**Numerics.**  The score buffers, the running reference and sum, and O are f32.  P is rounded for the tensor core:
f16 caches take f16 P, to nearest (2^-11), with 2^7 put on the exponent so that small weights keep their bits;
bf16 caches and bytes (whose P carries a scale of any size) take P as two bf16 parts, truncated, 2^-14 together.
O is rescaled only when the row's maximum grew by more than 2^8.

**What is masked.**  Scores past the row's own position, outside its window or of a page that the table does not
name become -inf; a row that sees nothing ends as 0.  Rows of a V tile that no row of the CTA sees are zeroed in
shared memory before the product (P is 0 there, but a stale row may hold NaN).

Every wait is bounded and reports a code (71-76); TMEM is always freed.
"""
from __future__ import annotations

import struct

from .ptxasm import Asm, idesc_f16, smem_desc_hi, wait_bar, wait_bar_warp

ROWS = 128                       # query rows of a CTA (the MMA's M)
BKV = 64                         # keys of a tile
STAGES = 4                       # ring items K0 V0 K1 V1: two tiles in flight
TMEM_COLS = 256                  # O (dim columns) and two score buffers; two CTAs fill an SM's 512
LOG2E = 1.4426950408889634
RESCALE = 8.0                    # log2 units the reference may lag behind the row's maximum
F16_LIFT = 7.0                   # f16 P is 2^(s - m + 7): at most 2^15, and 2^-21 of the largest is still normal

ERR_LOAD, ERR_MMA, ERR_SOFTMAX, ERR_EPILOGUE, ERR_DRAIN, ERR_Q = 71, 72, 73, 74, 75, 76

# shared memory behind the tiles: barriers, the TMEM slot, two mask words per tile (a ring of 4 tiles) and, for
# bytes, the keys' and values' scales of 4 tiles.  A ring of 4 is enough: the loads of tile j + 4 wait for
# S(j + 2), which is issued after P(j) is complete, so nobody reads slot j any more.
QFULL = 0
FULL = 8
EMPTY = FULL + 8 * STAGES
SFULL = EMPTY + 8 * STAGES
PFULL = SFULL + 16
PFREE = PFULL + 16
SLOT = PFREE + 16
KMASK = 192
KSC = 256
VSC = KSC + 4 * BKV * 4
AUX_BYTES = VSC + 4 * BKV * 4


def _f32(v: float) -> str:
    return "0f%08X" % struct.unpack("<I", struct.pack("<f", v))[0]


class _E(Asm):
    """The assembler with one helper: ``e.o("add.u32", x, y)`` emits it into a fresh register."""

    def o(self, ins, *args, cls="r"):
        d = self.r(cls)
        self(f"{ins} {d}, {', '.join(str(x) for x in args)};")
        return d

    def cond(self, cmp, x, y):
        return self.o(f"setp.{cmp}", x, y, cls="p")


def supported(dim, heads, kv_heads, page) -> bool:
    """Head dims of one or two 128-byte columns; a group that fits the tile; pages that tile 64 keys (8 rows
    are one swizzle atom) or are whole numbers of them."""
    return (dim in (64, 128) and heads // kv_heads <= ROWS
            and (page % BKV == 0 or (page >= 8 and BKV % page == 0)))


def geometry(chunk, heads, kv_heads):
    """(group, tokens per full CTA, token tiles, rows a CTA can have)."""
    group = heads // kv_heads
    tq = ROWS // group
    return group, tq, -(-chunk // tq), min(tq, chunk) * group


def plan_splits(batch, chunk, heads, kv_heads, page, max_pages, window, sinks, sms=148):
    """(splits, least tiles of a part): one part where the units fill the GPU's two CTAs an SM, otherwise as many
    parts as fill it, of at least 8 tiles.  Splitting more costs more than it evens out here: a part of 128 rows
    writes and the join reads 64 KiB of f32, as much as two tiles of keys and values (a 2048-token chunk over
    8192 keys ran at 876 TFLOP/s in one part and 647 in up to four)."""
    group, tq, ntile, rows = geometry(chunk, heads, kv_heads)
    longest = -(-max_pages * page // BKV)
    if window is not None:
        longest = min(longest, -(-sinks // BKV) + (window + min(tq, chunk) - 1) // BKV + 2)
    min_tiles = 8
    units = batch * kv_heads * ntile
    return max(1, min(longest // min_tiles, 2 * sms // units)), min_tiles


def _unit(e, k, b_len, b_new, c0, splits, min_tiles, tq, chunk, cap, window, sinks):
    """What a unit (a sequence's token tile) walks, from its length and new tokens: emitted alike by the attention
    and by the join.  Returns registers: the last token c1, first and last position, the first window key
    ``lo``, sink tiles ``st``, ``gap`` (tile = i + gap from sink tile st on), tiles ``total`` and tiles per part."""
    n = e.o("min.s32", b_new, chunk)
    c1 = e.o("min.s32", e.o("add.s32", c0, tq), n)
    c1 = e.o("sub.s32", c1, 1)
    first = e.o("sub.s32", b_len, b_new)
    pos0, pos1 = e.o("add.s32", first, c0), e.o("add.s32", first, c1)
    end = e.o("min.s32", e.o("add.s32", pos1, 1), cap)
    end = e.o("max.s32", end, 0)
    tend = e.o("shr.u32", e.o("add.u32", end, BKV - 1), 6)
    lo = st = gap = None
    total = tend
    if window is not None:
        lo = e.o("max.s32", e.o("sub.s32", pos0, window - 1), 0)
        wt0 = e.o("min.u32", e.o("shr.u32", lo, 6), tend)
        st = e.o("min.u32", wt0, -(-sinks // BKV))
        gap = e.o("sub.u32", wt0, st)
        total = e.o("sub.u32", tend, gap)
    per = total
    if splits > 1:
        per = e.o("div.u32", e.o("add.u32", total, splits - 1), splits)
        per = e.o("max.u32", per, min_tiles)
    return dict(n=n, c1=c1, pos0=pos0, pos1=pos1, end=end, lo=lo, st=st, gap=gap, total=total, per=per)


def paged_attention_entry(name, batch, chunk, heads, kv_heads, dim, pages, page, max_pages, dtype, quant, window, sinks,
                          scale, names, scratch, splits, min_tiles, prefix=""):
    """The launch record and PTX; ``names``: Q, KC, VC, (KS, VS,) table, lens, fresh, O; ``scratch``: the parts'
    buffer, all their O rows and then their m and l."""
    D = dim
    group, tq, ntile, rows = geometry(chunk, heads, kv_heads)
    units = batch * kv_heads * ntile
    grid = units * splits
    half = dtype == "f16"                    # the Q K^T operands' type
    p_f16 = half and not quant               # P and V in f16; otherwise bf16, P in two parts
    row_b = D * 2
    q_bytes, q_box = ROWS * row_b, ROWS * 128
    kv_bytes, kv_box = BKV * row_b, BKV * 128
    boxes = D // 64
    cap = max_pages * page
    pieces = max(1, BKV // page)             # pages of a tile
    box_rows = min(page, BKV)
    if quant:
        threads, soft0, mma_warp = 288, 4, 8
    else:
        threads, soft0, mma_warp = 192, 2, 1
    idesc_qk = idesc_f16(ROWS, BKV, False, False, half=half)
    idesc_pv = idesc_f16(ROWS, D, False, True, half=p_f16)
    kdesc_hi = smem_desc_hi(16, 1024)
    vdesc_hi = smem_desc_hi(kv_box, 1024)
    cscale = _f32(scale * LOG2E)
    S0 = D                                   # score buffers behind O's columns
    e = _E()
    o = e.o

    def gptr(pname):
        return o("cvta.to.global.u64", o("ld.param.u64", f"[{pname}]", cls="rd"), cls="rd")

    def wide(x, n):
        return o("mul.wide.u32", x, n, cls="rd")

    def at(base, off):
        return o("add.s64", base, off, cls="rd")

    def ldg(addr, ty="u32", cls="r"):
        return o(f"ld.global.nc.{ty}", f"[{addr}]", cls=cls)

    tid = o("mov.u32", "%tid.x")
    warp = o("shr.u32", tid, 5)
    lane = o("and.b32", tid, 31)
    cta = o("mov.u32", "%ctaid.x")
    err, o_ptr = gptr("p_err"), gptr("p_O")
    if splits > 1:
        e("griddepcontrol.launch_dependents;")                  # the join's blocks may come up and wait
        unit, sp = o("div.u32", cta, splits), o("rem.u32", cta, splits)
    else:
        unit, sp = cta, None
    kvh = o("rem.u32", unit, kv_heads)
    ub = o("div.u32", unit, kv_heads)
    b = o("rem.u32", ub, batch)
    tile = o("sub.u32", ntile - 1, o("div.u32", ub, batch))     # the longest rows of a sequence first
    b_len = ldg(at(gptr("p_lens"), wide(b, 4)))
    b_new = ldg(at(gptr("p_fresh"), wide(b, 4)))
    c0 = o("mul.lo.u32", tile, tq)
    e(f"@{e.cond('ge.s32', c0, b_new)} ret;")                   # a tile of padding
    w = _unit(e, None, b_len, b_new, c0, splits, min_tiles, tq, chunk, cap, window, sinks)
    c1, pos0, pos1, total, per = w["c1"], w["pos0"], w["pos1"], w["total"], w["per"]
    ntok = o("add.u32", o("sub.u32", c1, c0), 1)
    vrows = o("mul.lo.u32", ntok, group)
    # first row of Q and O in [batch * chunk * heads, dim], and row r's index from it
    base_row = o("mad.lo.u32", b, chunk, c0)
    base_row = o("mad.lo.u32", base_row, heads, o("mul.lo.u32", kvh, group))

    def row_index(r):
        """Row r of the CTA's tile as a row of Q and O: token r / group, head r % group."""
        if group == 1:
            return o("mad.lo.u32", r, heads, base_row)
        t_ = o("div.u32", r, group)
        return o("add.u32", o("mad.lo.u32", t_, heads, base_row), o("sub.u32", r, o("mul.lo.u32", t_, group)))

    i0, nb = None, total
    if splits > 1:
        i0 = o("mul.lo.u32", sp, per)
        p_none = e.cond("ge.u32", i0, total)
        p_later = e.cond("ne.u32", sp, 0)
        e(f"and.pred {p_none}, {p_none}, {p_later};")
        e(f"@{p_none} ret;")                                    # no tiles for this part
        nb = o("min.u32", o("sub.u32", total, i0), per)
    # a unit that sees no key at all: its rows are 0
    l_some = e.L("some")
    e(f"@{e.cond('ne.u32', total, 0)} bra {l_some};")
    zr, zero = o("mov.u32", tid), o("mov.u32", 0)
    l_z, l_zd = e.L("zero"), e.L("zerod")
    e.label(l_z)
    e(f"@{e.cond('ge.u32', zr, vrows)} bra {l_zd};")
    za = at(o_ptr, wide(row_index(zr), row_b))
    for c in range(row_b // 32):
        e(f"st.global.v8.b32 [{za}+{32 * c}], {{{', '.join([zero] * 8)}}};")
    e(f"add.u32 {zr}, {zr}, {threads};")
    e(f"bra {l_z};")
    e.label(l_zd)
    e("ret;")
    e.label(l_some)

    smem_sym = f"{prefix}paged_smem"
    raw = o("mov.u32", smem_sym)
    sQ = o("and.b32", o("add.u32", raw, 1023), -1024)
    sKV = o("add.u32", sQ, q_bytes)
    bars = o("add.u32", sKV, STAGES * kv_bytes)
    nwarps = o("shr.u32", o("add.u32", vrows, 31), 5)          # softmax warps that have a row
    l_init = e.L("noinit")
    e(f"@{e.cond('ne.u32', tid, 0)} bra {l_init};")
    e(f"mbarrier.init.shared::cta.b64 [{bars}+{QFULL}], {nwarps};")
    for s in range(STAGES):
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{FULL + 8 * s}], {2 if quant else 1};")
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{EMPTY + 8 * s}], 1;")
    for u in range(2):
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{SFULL + 8 * u}], 1;")
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{PFULL + 8 * u}], {nwarps};")
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{PFREE + 8 * u}], 1;")
    e("fence.mbarrier_init.release.cluster;")
    e("fence.proxy.async.shared::cta;")
    e.label(l_init)
    p_mma = e.cond("eq.u32", warp, mma_warp)
    l_noalloc = e.L("noalloc")
    e(f"@!{p_mma} bra {l_noalloc};")
    e(f"tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [{bars}+{SLOT}], {TMEM_COLS};")
    e("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;")
    e("tcgen05.fence::before_thread_sync;")
    e.label(l_noalloc)
    e("bar.sync 0;")
    e("tcgen05.fence::after_thread_sync;")
    taddr = o("ld.shared.b32", f"[{bars}+{SLOT}]")
    l_end, l_mma, l_soft = e.L("end"), e.L("mma"), e.L("soft")
    e(f"@{p_mma} bra {l_mma};")
    e(f"@{e.cond('ge.u32', warp, soft0)} bra {l_soft};")
    table = gptr("p_table")
    trow = at(table, wide(b, 4 * max_pages))                   # this sequence's row of the table

    def tile_of(j):
        """The key tile of the part's tile number j."""
        i = o("add.u32", j, i0) if i0 is not None else j
        if window is None:
            return i
        past = e.cond("ge.u32", i, w["st"])
        return o("selp.u32", o("add.u32", i, w["gap"]), i, past)

    def entry(dst, slot, ok):
        """dst = the page of table slot ``slot`` where ``ok``, or -1 (also for a number outside the pool)."""
        a_ = at(trow, wide(slot, 4))
        e(f"mov.u32 {dst}, -1;")
        e(f"@{ok} ld.global.nc.u32 {dst}, [{a_}];")
        return dst

    def valid(pg):
        return e.cond("lt.u32", pg, pages)

    # ------------------------------------------------------------------ loads
    if not quant:
        tk, tv = [o("cvta.param.u64", o("mov.u64", f"p_tm{x}", cls="rd"), cls="rd") for x in "KV"]
        per_batch = 32 // pieces                               # tiles whose pages one lane-load fetches
        sub = o("div.u32", lane, pieces) if pieces > 1 else lane
        piece = o("rem.u32", lane, pieces) if pieces > 1 else None

        def fetch(dst, j0):
            """Lane l: the page of piece l % pieces of tile j0 + l / pieces."""
            j = o("add.u32", j0, sub)
            ok = e.cond("lt.u32", j, nb)
            vt = tile_of(j)
            if pieces > 1:
                slot = o("mad.lo.u32", vt, pieces, piece)
            elif page == BKV:
                slot = vt
            else:
                slot = o("div.u32", vt, page // BKV)
            okm = e.cond("lt.u32", slot, max_pages)
            e(f"and.pred {ok}, {ok}, {okm};")
            return entry(dst, slot, ok)

        cur, nxt = e.r(), e.r()
        j = o("mov.u32", 0)
        fetch(cur, j)
        fetch(nxt, o("mov.u32", per_batch))
        armed = [o("mov.u32", 2) for _ in range(STAGES)]
        l_top, l_done = e.L("ld"), e.L("ldd")
        p_l0, p_pc = e.cond("eq.u32", lane, 0), e.cond("lt.u32", lane, pieces)
        e.label(l_top)
        for u in range(2):
            e(f"@{e.cond('ge.u32', j, nb)} bra {l_done};")
            ph = o("and.b32", o("shr.u32", j, 1), 1)
            at_ = o("and.b32", j, per_batch - 1)
            l_same = e.L("same")
            p_new = e.cond("eq.u32", at_, 0)
            p_j = e.cond("ne.u32", j, 0)
            e(f"and.pred {p_new}, {p_new}, {p_j};")
            e(f"@!{p_new} bra {l_same};")                      # the same for every lane
            e(f"mov.u32 {cur}, {nxt};")
            fetch(nxt, o("add.u32", j, per_batch))
            e.label(l_same)
            l0 = o("mul.lo.u32", at_, pieces) if pieces > 1 else at_
            mine = o("shfl.sync.idx.b32", cur, o("add.u32", l0, piece) if pieces > 1 else l0, 31, -1)
            # the tile's mask words: bit k of word h is set when key 32 h + k has a page
            words = []
            for h in range(2):
                if pieces == 1:
                    src = mine
                else:
                    k_ = o("div.u32", o("add.u32", lane, 32 * h), page)
                    src = o("shfl.sync.idx.b32", cur, o("add.u32", l0, k_), 31, -1)
                words.append(o("vote.sync.ballot.b32", valid(src), -1))
            vt = tile_of(j)
            pgc = o("selp.b32", mine, -1, valid(mine))         # outside the pool: the box reads zeros
            roff = o("mul.lo.u32", o("rem.u32", vt, page // BKV), BKV) if page > BKV else 0
            for kv, tm in enumerate((tk, tv)):
                st_ = 2 * u + kv
                wait_bar_warp(e, f"{bars}+{EMPTY + 8 * st_}", o("xor.b32", ph, 1), err, ERR_LOAD, l_done)
                if kv == 0:
                    ma = o("mad.lo.u32", o("and.b32", j, 3), 8, bars)
                    e(f"@{p_l0} st.shared.v2.b32 [{ma}+{KMASK}], {{{words[0]}, {words[1]}}};")
                e(f"@{p_l0} mbarrier.arrive.expect_tx.shared::cta.b64 _, [{bars}+{FULL + 8 * st_}], {kv_bytes};")
                e(f"mov.u32 {armed[st_]}, {ph};")
                e("bar.warp.sync -1;")
                for h in range(boxes):
                    dst = o("add.u32", sKV, st_ * kv_bytes + h * kv_box)
                    if pieces > 1:
                        dst = o("mad.lo.u32", piece, page * 128, dst)
                    e(f"@{p_pc} cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                      f"[{dst}], [{tm}, {{{64 * h}, {roff}, {kvh}, {pgc}}}], [{bars}+{FULL + 8 * st_}];")
            e(f"add.u32 {j}, {j}, 1;")
        e(f"bra {l_top};")
        e.label(l_done)
        for s in range(STAGES):
            skip = e.L("nodrain")
            e(f"@{e.cond('eq.u32', armed[s], 2)} bra {skip};")
            wait_bar_warp(e, f"{bars}+{FULL + 8 * s}", armed[s], err, ERR_DRAIN, skip)
            e.label(skip)
        e(f"bra {l_end};")
    else:
        # warps 0, 1 load K and both scales, warps 2, 3 load V; thread t of 64 takes 16 bytes of rows
        # t / 4 + 16 k, k = 0..3, in each 64-byte half (4 lanes a row half: whole 32-byte sectors, and the
        # 16-byte stores of 8 lanes fall into 8 different bank groups)
        t64 = o("and.b32", tid, 63)
        p_v = e.cond("ge.u32", warp, 2)
        isv = o("selp.u32", 1, 0, p_v)
        pool = o("selp.b64", gptr("p_VC"), gptr("p_KC"), p_v, cls="rd")
        ks_ptr, vs_ptr = gptr("p_KS"), gptr("p_VS")
        rsub, chunk16 = o("shr.u32", t64, 2), o("and.b32", t64, 3)
        npg = 1 if pieces == 1 else 4

        def key_rows(j):
            """(first key of the part's tile j, whether there is one)."""
            return o("shl.b32", tile_of(j), 6), e.cond("lt.u32", j, nb)

        def entries(j, regs):
            """The pages of this thread's rows of tile j: one for all, or one for each of its four; and the
            page of row t64, whose scales it loads."""
            k0, ok = key_rows(j)
            todo = [(regs[0], k0)] if npg == 1 else [(regs[k], o("add.u32", k0, o("add.u32", rsub, 16 * k)))
                                                     for k in range(4)]
            if npg > 1:
                todo.append((regs[4], o("add.u32", k0, t64)))
            for dst, key in todo:
                okk = e.cond("lt.u32", key, w["end"])
                e(f"and.pred {okk}, {okk}, {ok};")
                entry(dst, o("div.u32", key, page), okk)

        def place(pg, key):
            """Row of the pool, flattened over pages, heads and rows (64 bits), of ``key`` on page ``pg``."""
            r_ = o("mul.wide.u32", pg, kv_heads * page, cls="rd")
            in_page = o("rem.u32", key, page)
            return at(r_, wide(o("mad.lo.u32", kvh, page, in_page), 1))

        def data(j, regs, dst, sc):
            """Loads tile j: 16 bytes per row and half into ``dst``, the scales of row t64 into ``sc``; rows without
            a key read as byte 128, which is 0."""
            k0, ok = key_rows(j)
            for k in range(4):
                key = o("add.u32", k0, o("add.u32", rsub, 16 * k))
                pg = regs[0] if npg == 1 else regs[k]
                p_ = e.cond("lt.u32", key, w["end"])
                e(f"and.pred {p_}, {p_}, {ok};")
                e(f"and.pred {p_}, {p_}, {valid(pg)};")
                a_ = at(at(pool, o("mul.lo.s64", place(pg, key), D, cls="rd")), wide(chunk16, 16))
                for h in range(boxes):
                    d_ = dst[h * 4 + k]
                    for x in d_:
                        e(f"mov.b32 {x}, 0x80808080;")
                    e(f"@{p_} ld.global.nc.L1::no_allocate.v4.b32 {{{', '.join(d_)}}}, [{a_}+{64 * h}];")
            l_ = e.L("noscale")
            for x in sc:
                e(f"mov.b32 {x}, 0f00000000;")
            e(f"mov.u32 {sc_ok}, 0;")
            e(f"@{p_v} bra {l_};")
            key = o("add.u32", k0, t64)
            pg = regs[0] if npg == 1 else regs[4]
            p_ = e.cond("lt.u32", key, w["end"])
            e(f"and.pred {p_}, {p_}, {ok};")
            e(f"and.pred {p_}, {p_}, {valid(pg)};")
            off = o("mul.lo.s64", place(pg, key), 4, cls="rd")
            e(f"@{p_} ld.global.nc.f32 {sc[0]}, [{at(ks_ptr, off)}];")
            e(f"@{p_} ld.global.nc.f32 {sc[1]}, [{at(vs_ptr, off)}];")
            e(f"selp.u32 {sc_ok}, 1, 0, {p_};")
            e.label(l_)

        pgs = [e.r() for _ in range(1 if npg == 1 else 5)]
        bufs = [[[e.r() for _ in range(4)] for _ in range(4 * boxes)] for _ in range(2)]
        scs = [[e.r("f"), e.r("f")] for _ in range(2)]
        oks = [e.r() for _ in range(2)]
        j = o("mov.u32", 0)
        entries(j, pgs)
        sc_ok = oks[0]
        data(j, pgs, bufs[0], scs[0])
        entries(o("mov.u32", 1), pgs)
        l_top, l_done = e.L("ld"), e.L("ldd")
        p_l0 = e.cond("eq.u32", lane, 0)
        zero_ = o("mov.u32", 0)
        swz = o("and.b32", rsub, 7)
        e.label(l_top)
        for u in range(2):
            e(f"@{e.cond('ge.u32', j, nb)} bra {l_done};")
            ph = o("and.b32", o("shr.u32", j, 1), 1)
            j1 = o("add.u32", j, 1)
            sc_ok = oks[1 - u]
            data(j1, pgs, bufs[1 - u], scs[1 - u])             # the next tile's loads in flight,
            entries(o("add.u32", j, 2), pgs)                   # and the pages of the one after it
            fb = o("mad.lo.u32", isv, 8, bars)
            wait_bar_warp(e, f"{fb}+{EMPTY + 16 * u}", o("xor.b32", ph, 1), err, ERR_LOAD, l_done)
            stage = o("mad.lo.u32", isv, kv_bytes, sKV)
            # K in the type of Q; V in bf16
            l_v, l_cv = e.L("asbf"), e.L("cvd")

            def convert(as_half):
                for h in range(boxes):
                    for k in range(4):
                        out = []
                        for x in bufs[u][h * 4 + k]:
                            for sel in ("0x4140", "0x4342"):
                                if as_half:
                                    t_ = o("prmt.b32", x, c64, sel)
                                    out.append(o("sub.rn.f16x2", t_, c1152))
                                else:
                                    t_ = o("prmt.b32", x, zero_, sel)
                                    m_ = o("lop3.b32", t_, "0x007F007F", c4300, "0xEA")     # (t & 7F) | 4300
                                    c_ = o("lop3.b32", t_, "0x00800080", c4380, "0x6A")     # (t & 80) ^ 4380
                                    out.append(o("sub.rn.bf16x2", m_, c_))
                        # bytes 16 c.. of half h are columns 16 c..: two 16-byte chunks of the row's 128
                        ra = o("mad.lo.u32", rsub, 128, o("add.u32", stage, 2 * u * kv_bytes + h * kv_box + k * 2048))
                        for i in range(2):
                            ch = o("xor.b32", o("mad.lo.u32", chunk16, 2, i), swz)
                            sa = o("mad.lo.u32", ch, 16, ra)
                            e(f"st.shared.v4.b32 [{sa}], {{{', '.join(out[4 * i:4 * i + 4])}}};")

            if half:
                c64, c1152 = o("mov.b32", "0x64646464"), o("mov.b32", "0x64806480")
            c4300, c4380 = o("mov.b32", "0x43004300"), o("mov.b32", "0x43804380")
            if half:
                e(f"@{p_v} bra {l_v};")
                convert(True)
                e(f"bra {l_cv};")
                e.label(l_v)
            convert(False)
            e.label(l_cv)
            # K's warps: the scales of 64 keys and the mask words (a key has a page and lies below the end)
            l_ns = e.L("nosc")
            e(f"@{p_v} bra {l_ns};")
            sa = o("mad.lo.u32", o("and.b32", j, 3), BKV * 4, bars)
            sa = o("mad.lo.u32", t64, 4, sa)
            e(f"st.shared.f32 [{sa}+{KSC}], {scs[u][0]};")
            e(f"st.shared.f32 [{sa}+{VSC}], {scs[u][1]};")
            mw_ = o("vote.sync.ballot.b32", e.cond("ne.u32", oks[u], 0), -1)
            ma = o("mad.lo.u32", o("and.b32", j, 3), 8, bars)
            ma = o("mad.lo.u32", warp, 4, ma)
            e(f"@{p_l0} st.shared.b32 [{ma}+{KMASK}], {mw_};")
            e.label(l_ns)
            e("fence.proxy.async.shared::cta;")
            e("bar.warp.sync -1;")
            e(f"@{p_l0} mbarrier.arrive.shared::cta.b64 _, [{fb}+{FULL + 16 * u}];")
            e(f"mov.u32 {j}, {j1};")
        e(f"bra {l_top};")
        e.label(l_done)
        e(f"bra {l_end};")

    # ------------------------------------------------------------------ MMA issue (one thread)
    e.label(l_mma)
    e(f"@{e.cond('ne.u32', lane, 0)} bra {l_end};")
    l_mdone = e.L("mdone")
    zero2 = o("mov.u32", 0)
    wait_bar(e, f"{bars}+{QFULL}", zero2, err, ERR_MMA, l_mdone)
    e("tcgen05.fence::after_thread_sync;")
    iqk, ipv = o("mov.u32", idesc_qk), o("mov.u32", idesc_pv)
    ptrue, pfalse = e.cond("eq.u32", lane, lane), e.cond("ne.u32", lane, lane)
    khi, vhi = o("mov.b64", kdesc_hi, cls="rd"), o("mov.b64", vdesc_hi, cls="rd")

    def desc(addr, hi):
        return o("or.b64", o("cvt.u64.u32", o("shr.u32", addr, 4), cls="rd"), hi, cls="rd")

    def plus(d0, off):
        return o("add.s64", d0, off >> 4, cls="rd") if off else d0

    q0 = desc(sQ, khi)
    qd = [plus(q0, (k // 4) * q_box + (k % 4) * 32) for k in range(D // 16)]
    stg = [o("add.u32", sKV, s * kv_bytes) for s in range(STAGES)]
    kd, vd = [desc(stg[2 * u], khi) for u in range(2)], [desc(stg[2 * u + 1], vhi) for u in range(2)]
    scol = [o("add.u32", taddr, S0 + BKV * u) for u in range(2)]

    def commit(off):
        e(f"tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [{bars}+{off}];")

    def ring(st_, ph):
        wait_bar(e, f"{bars}+{FULL + 8 * st_}", ph, err, ERR_MMA, l_mdone)
        e("tcgen05.fence::after_thread_sync;")

    def qk(u):
        for k in range(D // 16):
            e(f"tcgen05.mma.cta_group::1.kind::f16 [{scol[u]}], {qd[k]}, {plus(kd[u], (k // 4) * kv_box + (k % 4) * 32)}, "
              f"{iqk}, {ptrue if k else pfalse};")
        commit(EMPTY + 8 * (2 * u))
        commit(SFULL + 8 * u)

    j = o("mov.u32", 0)
    ring(0, zero2)
    qk(0)
    l_mg = e.L("mg")
    e.label(l_mg)
    for u in range(2):                                         # tile j = 2 g + u
        ph = o("and.b32", o("shr.u32", j, 1), 1)
        jn = o("add.u32", j, 1)
        have = e.cond("lt.u32", jn, nb)
        l_nok = e.L("nok")
        e(f"@!{have} bra {l_nok};")
        ring(2 * (1 - u), ph if u == 0 else o("xor.b32", ph, 1))
        qk(1 - u)
        e.label(l_nok)
        ring(2 * u + 1, ph)
        wait_bar(e, f"{bars}+{PFULL + 8 * u}", ph, err, ERR_MMA, l_mdone)
        e("tcgen05.fence::after_thread_sync;")
        pacc = e.cond("ne.u32", j, 0)
        for part in range(1 if p_f16 else 2):
            for k in range(BKV // 16):
                e(f"tcgen05.mma.cta_group::1.kind::f16 [{taddr}], [{scol[u]}+{BKV // 2 * part + 8 * k}], "
                  f"{plus(vd[u], 2048 * k)}, {ipv}, {pacc if k == 0 and part == 0 else ptrue};")
        commit(EMPTY + 8 * (2 * u + 1))
        commit(PFREE + 8 * u)
        e(f"@!{have} bra {l_mdone};")
        e(f"mov.u32 {j}, {jn};")
    e(f"bra {l_mg};")
    e.label(l_mdone)
    e(f"bra {l_end};")

    # ------------------------------------------------------------------ softmax (one row a thread)
    e.label(l_soft)
    quad = o("and.b32", warp, 3)                               # the TMEM lanes a warp reaches
    e(f"@{e.cond('ge.u32', quad, nwarps)} bra {l_end};")
    rowl = o("mad.lo.u32", quad, 32, lane)
    # Q: each warp its own 32 rows, 16 bytes a lane, into the swizzled K-major tile
    q_ptr = gptr("p_Q")
    per_row = row_b // 16                                      # lanes a row takes
    qsub, qch = o("div.u32", lane, per_row), o("rem.u32", lane, per_row)
    passes = 32 * per_row // 32
    for p0 in range(0, passes, 8):
        ws, rr_ = [], []
        for p_ in range(p0, min(passes, p0 + 8)):
            r_ = o("mad.lo.u32", quad, 32, o("add.u32", qsub, p_ * (32 // per_row)))
            ok = e.cond("lt.u32", r_, vrows)
            qa = at(at(q_ptr, wide(row_index(r_), row_b)), wide(qch, 16))
            d_ = [o("mov.b32", 0) for _ in range(4)]
            e(f"@{ok} ld.global.nc.v4.b32 {{{', '.join(d_)}}}, [{qa}];")
            ws.append(d_)
            rr_.append(r_)
        for d_, r_ in zip(ws, rr_):
            box = o("shr.u32", qch, 3)
            ch = o("xor.b32", o("and.b32", qch, 7), o("and.b32", r_, 7))
            sa = o("mad.lo.u32", box, q_box, sQ)
            sa = o("mad.lo.u32", r_, 128, sa)
            sa = o("mad.lo.u32", ch, 16, sa)
            e(f"st.shared.v4.b32 [{sa}], {{{', '.join(d_)}}};")
    e("fence.proxy.async.shared::cta;")
    e("bar.warp.sync -1;")
    p_l0s = e.cond("eq.u32", lane, 0)
    e(f"@{p_l0s} mbarrier.arrive.shared::cta.b64 _, [{bars}+{QFULL}];")
    lanebase = o("add.u32", o("shl.b32", quad, 21), taddr)
    tok = o("div.u32", rowl, group) if group > 1 else rowl
    pos = o("min.s32", o("add.s32", pos0, tok), pos1)          # rows without a token: the last one's
    s_ = [e.r("f") for _ in range(BKV)]
    mref, lsum = o("mov.b32", "0fFF800000", cls="f"), o("mov.b32", "0f00000000", cls="f")
    j = o("mov.u32", 0)
    l_sj, l_sdone, l_noepi = e.L("sj"), e.L("sdone"), e.L("noepi")
    e.label(l_sj)
    e(f"@{e.cond('ge.u32', j, nb)} bra {l_sdone};")
    buf = o("and.b32", j, 1)
    ph = o("and.b32", o("shr.u32", j, 1), 1)
    bb = o("mad.lo.u32", buf, 8, bars)
    sc_col = o("add.u32", o("mad.lo.u32", buf, BKV, lanebase), S0)
    key0 = o("shl.b32", tile_of(j), 6)
    wait_bar_warp(e, f"{bb}+{SFULL}", ph, err, ERR_SOFTMAX, l_noepi)
    e("tcgen05.fence::after_thread_sync;")
    for c in range(BKV // 32):
        e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(s_[32 * c:32 * c + 32])}}}, [{sc_col}+{32 * c}];")
    slot_a = o("and.b32", j, 3)
    ma = o("mad.lo.u32", slot_a, 8, bars)
    km = [e.r(), e.r()]
    e(f"ld.shared.v2.b32 {{{km[0]}, {km[1]}}}, [{ma}+{KMASK}];")
    e("tcgen05.wait::ld.sync.aligned;")
    sca = None
    if quant:
        sca = o("mad.lo.u32", slot_a, BKV * 4, bars)
        for c in range(0, BKV, 4):
            kf = [e.r("f") for _ in range(4)]
            e(f"ld.shared.v4.f32 {{{', '.join(kf)}}}, [{sca}+{KSC + 4 * c}];")
            for i in range(4):
                e(f"mul.f32 {s_[c + i]}, {s_[c + i]}, {kf[i]};")
    # the keys of the tile this row sees, as 64 bits: up to its own position, inside the window or among
    # the sinks, on a page.  Tiles that every row of the warp sees whole skip all of it.
    lim = o("sub.s32", pos, key0)
    p_all = e.cond("ge.s32", lim, BKV - 1)
    kand = o("and.b32", km[0], km[1])
    pk_ = e.cond("eq.s32", kand, -1)
    e(f"and.pred {p_all}, {p_all}, {pk_};")
    wl = sk = None
    if window is not None:
        wl = o("sub.s32", o("sub.s32", pos, window), key0)      # keys up to here lie before the window
        sk = o("sub.s32", sinks, key0)                          # keys below here are sinks
        pw_ = e.cond("lt.s32", wl, 0)
        ps_ = e.cond("ge.s32", sk, BKV)
        e(f"or.pred {pw_}, {pw_}, {ps_};")
        e(f"and.pred {p_all}, {p_all}, {pw_};")
    v_all = o("vote.sync.all.pred", p_all, -1, cls="p")
    l_seen = e.L("seen")
    m0, m1 = o("mov.b32", -1), o("mov.b32", -1)
    e(f"@{v_all} bra {l_seen};")

    def below(n, cls="rd"):
        """The bits below n (clamped to 0..64)."""
        k_ = o("sub.s32", 64, o("min.s32", o("max.s32", n, 0), 64))
        return o("shr.u64", o("mov.b64", -1, cls="rd"), k_, cls="rd")        # a shift by 64 leaves 0

    bits = below(o("add.s32", o("min.s32", lim, BKV), 1))
    if window is not None:
        inside = o("not.b64", below(o("add.s32", wl, 1)), cls="rd")
        inside = o("or.b64", inside, below(sk), cls="rd")
        bits = o("and.b64", bits, inside, cls="rd")
    pages_ = e.r("rd")
    e(f"mov.b64 {pages_}, {{{km[0]}, {km[1]}}};")
    bits = o("and.b64", bits, pages_, cls="rd")
    e(f"mov.b64 {{{m0}, {m1}}}, {bits};")
    for c in range(BKV):
        t_ = o("and.b32", (m0, m1)[c // 32], 1 << (c % 32) if c % 32 < 31 else -(1 << 31))
        e(f"@{e.cond('eq.u32', t_, 0)} mov.b32 {s_[c]}, 0fFF800000;")
    e.label(l_seen)
    if not quant:
        # rows of V that no row of this CTA sees (past its last token, or between sinks and window) may
        # hold anything: zero them before the product multiplies them by P = 0
        l_vok = e.L("vok")
        vlim = o("sub.s32", pos1, key0)
        pv_ = e.cond("ge.s32", vlim, BKV - 1)
        if window is not None:
            lo_k = o("sub.s32", w["lo"], key0)
            p1_, p2_ = e.cond("le.s32", lo_k, 0), e.cond("ge.s32", sk, BKV)
            e(f"or.pred {p1_}, {p1_}, {p2_};")
            e(f"and.pred {pv_}, {pv_}, {p1_};")
        e(f"@{pv_} bra {l_vok};")                               # the same for every thread
        wait_bar_warp(e, f"{o('mad.lo.u32', buf, 16, bars)}+{FULL + 8}", ph, err, ERR_SOFTMAX, l_noepi)
        va = o("mad.lo.u32", buf, 2 * kv_bytes, o("add.u32", sKV, kv_bytes))
        z_ = o("mov.b32", 0)
        for h in range(2):
            r_ = o("add.u32", lane, 32 * h)
            pz = e.cond("gt.s32", r_, vlim)
            if window is not None:
                pa, pb = e.cond("lt.s32", r_, lo_k), e.cond("ge.s32", r_, sk)
                e(f"and.pred {pa}, {pa}, {pb};")
                e(f"or.pred {pz}, {pz}, {pa};")
            ra = o("mad.lo.u32", r_, 128, va)
            for box in range(boxes):
                for i in range(8):
                    e(f"@{pz} st.shared.v4.b32 [{ra}+{box * kv_box + 16 * i}], {{{z_}, {z_}, {z_}, {z_}}};")
        e("fence.proxy.async.shared::cta;")
        e.label(l_vok)
    # the row's maximum: 8 chains of three-input maxima
    lvl = [e.r("f") for _ in range(8)]
    for k in range(8):
        col = list(range(k, BKV, 8))
        e(f"max.f32 {lvl[k]}, {s_[col[0]]}, {s_[col[1]]}, {s_[col[2]]};")
        e(f"max.f32 {lvl[k]}, {lvl[k]}, {s_[col[3]]}, {s_[col[4]]};")
        e(f"max.f32 {lvl[k]}, {lvl[k]}, {s_[col[5]]}, {s_[col[6]]};")
        e(f"max.f32 {lvl[k]}, {lvl[k]}, {s_[col[7]]};")
    e(f"max.f32 {lvl[0]}, {lvl[0]}, {lvl[1]}, {lvl[2]};")
    e(f"max.f32 {lvl[3]}, {lvl[3]}, {lvl[4]}, {lvl[5]};")
    e(f"max.f32 {lvl[6]}, {lvl[6]}, {lvl[7]};")
    e(f"max.f32 {lvl[0]}, {lvl[0]}, {lvl[3]}, {lvl[6]};")
    mnew = o("max.f32", mref, o("mul.f32", lvl[0], cscale, cls="f"), cls="f")
    alpha = o("mov.b32", "0f3F800000", cls="f")
    l_first, l_after = e.L("first"), e.L("after")
    anyneed = e.cond("ne.u32", lane, lane)
    e(f"@{e.cond('eq.u32', j, 0)} bra {l_first};")
    need = e.cond("gt.f32", mnew, o("add.f32", mref, _f32(RESCALE), cls="f"))
    e(f"vote.sync.any.pred {anyneed}, {need}, -1;")
    e(f"@!{anyneed} bra {l_after};")
    e(f"ex2.approx.ftz.f32 {alpha}, {o('sub.f32', mref, mnew, cls='f')};")
    # a row that has seen nothing yet while another of the warp rescales: -inf - -inf must not make a NaN
    e(f"@{e.cond('eq.f32', mnew, '0fFF800000')} mov.b32 {alpha}, 0f3F800000;")
    e(f"mul.f32 {lsum}, {lsum}, {alpha};")
    e.label(l_first)
    e(f"mov.b32 {mref}, {mnew};")
    e.label(l_after)
    lift = F16_LIFT if p_f16 else 0.0
    negm = o("sub.f32", o("mov.b32", _f32(lift), cls="f"), mref, cls="f")
    e(f"@{e.cond('eq.f32', mref, '0fFF800000')} mov.b32 {negm}, 0f00000000;")
    cf = o("mov.b32", cscale, cls="f")
    cp2, np2 = e.r("rd"), e.r("rd")
    e(f"mov.b64 {cp2}, {{{cf}, {cf}}};")
    e(f"mov.b64 {np2}, {{{negm}, {negm}}};")
    acc = [o("mov.b64", 0, cls="rd") for _ in range(2)]

    def exps(cols):
        for k, idx in enumerate(cols[::2]):
            x0, x1 = s_[idx], s_[idx + 1]
            xp, ep = e.r("rd"), e.r("rd")
            e(f"mov.b64 {xp}, {{{x0}, {x1}}};")
            e(f"fma.rn.f32x2 {xp}, {xp}, {cp2}, {np2};")
            e(f"mov.b64 {{{x0}, {x1}}}, {xp};")
            e(f"ex2.approx.ftz.f32 {x0}, {x0};")
            e(f"ex2.approx.ftz.f32 {x1}, {x1};")
            e(f"mov.b64 {ep}, {{{x0}, {x1}}};")
            e(f"add.rn.f32x2 {acc[k & 1]}, {acc[k & 1]}, {ep};")

    if p_f16:
        for h in range(2):
            cols = list(range(32 * h, 32 * h + 32))
            exps(cols)
            hw = [o("cvt.rn.f16x2.f32", s_[c + 1], s_[c]) for c in cols[::2]]
            e(f"tcgen05.st.sync.aligned.32x32b.x16.b32 [{sc_col}+{16 * h}], {{{', '.join(hw)}}};")
    else:
        exps(list(range(BKV)))
        if quant:
            for c in range(0, BKV, 4):
                vf = [e.r("f") for _ in range(4)]
                e(f"ld.shared.v4.f32 {{{', '.join(vf)}}}, [{sca}+{VSC + 4 * c}];")
                for i in range(4):
                    e(f"mul.f32 {s_[c + i]}, {s_[c + i]}, {vf[i]};")
            # a masked key's scale may be NaN: its weight is 0 whatever it was multiplied by
            l_nz = e.L("nz")
            e(f"@{v_all} bra {l_nz};")
            for c in range(BKV):
                t_ = o("and.b32", (m0, m1)[c // 32], 1 << (c % 32) if c % 32 < 31 else -(1 << 31))
                e(f"@{e.cond('eq.u32', t_, 0)} mov.b32 {s_[c]}, 0f00000000;")
            e.label(l_nz)
        for h in range(2):
            hi, lo = [], []
            for c in range(32 * h, 32 * h + 32, 2):
                hi.append(o("prmt.b32", s_[c], s_[c + 1], "0x7632"))
                d0 = o("sub.f32", s_[c], o("and.b32", s_[c], -65536, cls="f"), cls="f")
                d1 = o("sub.f32", s_[c + 1], o("and.b32", s_[c + 1], -65536, cls="f"), cls="f")
                lo.append(o("prmt.b32", d0, d1, "0x7632"))
            e(f"tcgen05.st.sync.aligned.32x32b.x16.b32 [{sc_col}+{16 * h}], {{{', '.join(hi)}}};")
            e(f"tcgen05.st.sync.aligned.32x32b.x16.b32 [{sc_col}+{32 + 16 * h}], {{{', '.join(lo)}}};")
    parts = [e.r("f") for _ in range(4)]
    e(f"mov.b64 {{{parts[0]}, {parts[1]}}}, {acc[0]};")
    e(f"mov.b64 {{{parts[2]}, {parts[3]}}}, {acc[1]};")
    psum = o("add.f32", o("add.f32", parts[0], parts[1], cls="f"), o("add.f32", parts[2], parts[3], cls="f"), cls="f")
    e(f"add.f32 {lsum}, {lsum}, {psum};")
    # the lazy rescale of O, once the previous product has completed
    l_nore = e.L("norescale")
    e(f"@!{anyneed} bra {l_nore};")

    def pv_done(k, code, bail):
        br = o("mad.lo.u32", o("and.b32", k, 1), 8, bars)
        wait_bar_warp(e, f"{br}+{PFREE}", o("and.b32", o("shr.u32", k, 1), 1), err, code, bail)

    pv_done(o("sub.u32", j, 1), ERR_SOFTMAX, l_noepi)
    e("tcgen05.fence::after_thread_sync;")
    for c in range(D // 32):
        regs = s_[:32]
        e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(regs)}}}, [{lanebase}+{32 * c}];")
        e("tcgen05.wait::ld.sync.aligned;")
        for r_ in regs:
            e(f"mul.f32 {r_}, {r_}, {alpha};")
        e(f"tcgen05.st.sync.aligned.32x32b.x32.b32 [{lanebase}+{32 * c}], {{{', '.join(regs)}}};")
    e.label(l_nore)
    e("tcgen05.wait::st.sync.aligned;")
    e("tcgen05.fence::before_thread_sync;")
    e("bar.warp.sync -1;")
    e(f"@{p_l0s} mbarrier.arrive.shared::cta.b64 _, [{bb}+{PFULL}];")
    e(f"add.u32 {j}, {j}, 1;")
    e(f"bra {l_sj};")

    # epilogue: after the last product, O / l as the output type, or the part's O, m and l in f32
    e.label(l_sdone)
    pv_done(o("sub.u32", nb, 1), ERR_EPILOGUE, l_noepi)
    e("tcgen05.fence::after_thread_sync;")
    p_row = e.cond("lt.u32", rowl, vrows)
    l_part = e.L("part")
    if splits > 1:
        e(f"@{e.cond('gt.u32', total, per)} bra {l_part};")
    p_zero = e.cond("eq.f32", lsum, "0f00000000")
    inv = o("rcp.rn.f32", o("selp.f32", "0f3F800000", lsum, p_zero, cls="f"), cls="f")
    oa = at(o_ptr, wide(row_index(rowl), row_b))
    pack = "cvt.rn.f16x2.f32" if half else "cvt.rn.bf16x2.f32"
    for c in range(D // 32):
        regs = s_[:32]
        e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(regs)}}}, [{lanebase}+{32 * c}];")
        e("tcgen05.wait::ld.sync.aligned;")
        words = []
        for k in range(16):
            x0 = o("mul.f32", regs[2 * k], inv, cls="f")
            x1 = o("mul.f32", regs[2 * k + 1], inv, cls="f")
            words.append(o("selp.b32", 0, o(pack, x1, x0), p_zero))
        for i in range(2):
            e(f"@{p_row} st.global.v8.b32 [{oa}+{64 * c + 32 * i}], {{{', '.join(words[8 * i:8 * i + 8])}}};")
    if splits > 1:
        e(f"bra {l_noepi};")
        e.label(l_part)
        pi = o("mad.lo.u32", cta, rows, rowl)
        pa = at(gptr("p_part"), wide(pi, D * 4))
        for c in range(D // 32):
            regs = s_[:32]
            e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(regs)}}}, [{lanebase}+{32 * c}];")
            e("tcgen05.wait::ld.sync.aligned;")
            for i in range(4):
                e(f"@{p_row} st.global.v8.f32 [{pa}+{128 * c + 32 * i}], {{{', '.join(regs[8 * i:8 * i + 8])}}};")
        mla = at(at(gptr("p_part"), grid * rows * D * 4), wide(pi, 8))
        # the parts' O and l stand for 2^-negm; a part that saw nothing has m = -inf
        meff = o("sub.f32", mref, _f32(lift), cls="f")
        e(f"@{p_row} st.global.v2.f32 [{mla}], {{{meff}, {lsum}}};")
    e.label(l_noepi)

    e.label(l_end)
    e("barrier.sync 0;")
    e("bar.warp.sync -1;")
    l_nod = e.L("nodealloc")
    e(f"@!{p_mma} bra {l_nod};")
    e("tcgen05.fence::after_thread_sync;")
    e(f"tcgen05.dealloc.cta_group::1.sync.aligned.b32 {taddr}, {TMEM_COLS};")
    e.label(l_nod)

    if quant:
        qn, kn, vn, ksn, vsn, tn, ln, fn, on = names
        params = [("Q", qn, 16), ("KC", kn, 16), ("VC", vn, 16), ("KS", ksn, 4), ("VS", vsn, 4)]
    else:
        qn, kn, vn, tn, ln, fn, on = names
        params = [("Q", qn, 16), ("KC", kn, 16), ("VC", vn, 16)]
    params += [("table", tn, 4), ("lens", ln, 4), ("fresh", fn, 4), ("O", on, 32)]
    sc_spec = []
    if splits > 1:
        params += [("part", scratch, 32)]
        sc_spec = [{"name": scratch, "dtype": "f32", "shape": [grid * rows, D + 2], "per_call": True}]
    tmaps = []
    if not quant:
        es = 2
        tmaps = [{"name": f"tm{x}", "tensor": nm, "dtype": dtype, "dims": [D, page, kv_heads, pages],
                  "strides": [D * es, page * D * es, kv_heads * page * D * es], "box": [64, box_rows, 1, 1],
                  "swizzle": "128B"} for x, nm in (("K", kn), ("V", vn))]
    plist = [f"\t.param .u64 p_{p}" for p, _, _ in params]
    plist += [f"\t.param .align 64 .b8 p_{t['name']}[128]" for t in tmaps] + ["\t.param .u64 p_err"]
    text = [f".visible .entry {name}(", ",\n".join(plist), ")", f".reqntid {threads}, 1, 1",
            f".maxnreg {65536 // (2 * threads) // 8 * 8}", "{"]
    text += e.decls() + e.lines + ["\tret;", "}"]
    return {
        "name": name, "kind": "tcgen05_paged_attention", "params": [n for _, n, _ in params],
        "raw_entry": text, "raw_decls": [f".extern .shared .align 1024 .b8 {smem_sym}[];"],
        "grid": [grid, 1, 1], "block": [threads, 1, 1],
        "dyn_smem": q_bytes + STAGES * kv_bytes + (AUX_BYTES if quant else KSC) + 1024,
        "align": {n: a_ for _, n, a_ in params}, "zero_outputs": [], "tmaps": tmaps,
        "extra": [{"name": "__err", "kind": "errword"}], "scratch": sc_spec,
    }


def join_entry(name, batch, chunk, heads, kv_heads, dim, page, max_pages, dtype, window, sinks, names, scratch, splits,
               min_tiles, locate=None):
    """The second entry: rows whose unit was split, o = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.  One block a row;
    its four warps take every fourth part, so that a row of 100 parts is 25 loads deep.  Rows of units that
    fit one part are written already and return at once.  ``locate`` finds a row's parts (the default: ``splits`` parts
    a unit, of at least ``min_tiles`` tiles each)."""
    D = dim
    group, tq, ntile, rows = geometry(chunk, heads, kv_heads)
    per_lane = D // 32
    e = _E()
    o = e.o

    def gptr(pname):
        return o("cvta.to.global.u64", o("ld.param.u64", f"[{pname}]", cls="rd"), cls="rd")

    def at(base, x, n):
        return o("add.s64", base, o("mul.wide.u32", x, n, cls="rd"), cls="rd")

    tid = o("mov.u32", "%tid.x")
    warp, lane = o("shr.u32", tid, 5), o("and.b32", tid, 31)
    e("griddepcontrol.wait;")                                   # the parts are written
    row = o("mov.u32", "%ctaid.x")
    h, bc = o("rem.u32", row, heads), o("div.u32", row, heads)
    c, b = o("rem.u32", bc, chunk), o("div.u32", bc, chunk)
    b_len = o("ld.global.nc.u32", f"[{at(gptr('p_lens'), b, 4)}]")
    b_new = o("ld.global.nc.u32", f"[{at(gptr('p_fresh'), b, 4)}]")
    e(f"@{e.cond('ge.s32', c, b_new)} ret;")
    if locate is None:
        tile = o("div.u32", c, tq)
        c0 = o("mul.lo.u32", tile, tq)
        w = _unit(e, None, b_len, b_new, c0, splits, min_tiles, tq, chunk, max_pages * page, window, sinks)
        e(f"@{e.cond('le.u32', w['total'], w['per'])} ret;")
        nact = o("div.u32", o("sub.u32", o("add.u32", w["total"], w["per"]), 1), w["per"])
        unit = o("mad.lo.u32", o("sub.u32", ntile - 1, tile), batch, b)
        unit = o("mad.lo.u32", unit, kv_heads, o("div.u32", h, group))
        rowl = o("mad.lo.u32", o("sub.u32", c, c0), group, o("rem.u32", h, group))
        base = o("mad.lo.u32", o("mul.lo.u32", unit, splits), rows, rowl)     # part 0's row; parts are ``rows`` apart
        part_rows = batch * kv_heads * ntile * splits * rows

        def part_row(s_):
            return o("mad.lo.u32", s_, rows, base)
    else:
        def zero_row(p_none):
            """A row that sees no key, where ``p_none``: 0."""
            l_ = e.L("nz")
            e(f"@!{p_none} bra {l_};")
            e(f"@{e.cond('ge.u32', tid, D // 2)} ret;")
            e(f"st.global.b32 [{at(at(gptr('p_O'), row, D * 2), tid, 4)}], {o('mov.b32', 0)};")
            e("ret;")
            e.label(l_)
        nact, part_row, part_rows = locate(e, lambda x, y: o("add.s64", x, y, cls="rd"), gptr, lane, b, c, h, zero_row)
    part = gptr("p_part")
    ml = o("add.s64", part, part_rows * D * 4, cls="rd")
    # the largest reference of the row's parts (every warp on its own)
    m = o("mov.b32", "0fFF800000", cls="f")
    s = o("mov.u32", lane)
    l_m, l_md = e.L("m"), e.L("md")
    e.label(l_m)
    e(f"@{e.cond('ge.u32', o('and.b32', s, -32), nact)} bra {l_md};")           # the same for the warp
    v = o("mov.b32", "0fFF800000", cls="f")
    e(f"@{e.cond('lt.u32', s, nact)} ld.global.f32 {v}, [{at(ml, part_row(s), 8)}];")
    e(f"max.f32 {m}, {m}, {v};")
    e(f"add.u32 {s}, {s}, 32;")
    e(f"bra {l_m};")
    e.label(l_md)
    for d in (16, 8, 4, 2, 1):
        e(f"max.f32 {m}, {m}, {o('shfl.sync.bfly.b32', m, d, 31, -1, cls='f')};")
    e(f"@{e.cond('eq.f32', m, '0fFF800000')} mov.b32 {m}, 0f00000000;")
    acc = [o("mov.b32", "0f00000000", cls="f") for _ in range(per_lane)]
    l = o("mov.b32", "0f00000000", cls="f")
    s = o("mov.u32", warp)
    l_top, l_done = e.L("p"), e.L("pd")
    UN = 4
    vec = f"v{per_lane}"
    part_l = at(part, lane, per_lane * 4)
    e.label(l_top)
    e(f"@{e.cond('ge.u32', s, nact)} bra {l_done};")
    loaded = []
    for u in range(UN):
        su = o("add.u32", s, 4 * u)
        ok = e.cond("lt.u32", su, nact)
        idx = part_row(su)
        ms, ls = o("mov.b32", "0fFF800000", cls="f"), o("mov.b32", "0f00000000", cls="f")
        e(f"@{ok} ld.global.v2.f32 {{{ms}, {ls}}}, [{at(ml, idx, 8)}];")
        xs = [o("mov.b32", "0f00000000", cls="f") for _ in range(per_lane)]
        e(f"@{ok} ld.global.{vec}.f32 {{{', '.join(xs)}}}, [{at(part_l, idx, D * 4)}];")
        loaded.append((ms, ls, xs))
    for ms, ls, xs in loaded:
        f = o("ex2.approx.ftz.f32", o("sub.f32", ms, m, cls="f"), cls="f")
        e(f"fma.rn.f32 {l}, {f}, {ls}, {l};")
        for a_, x in zip(acc, xs):
            e(f"fma.rn.f32 {a_}, {f}, {x}, {a_};")
    e(f"add.u32 {s}, {s}, {4 * UN};")
    e(f"bra {l_top};")
    e.label(l_done)
    sm = o("mov.u32", f"{name}_sum")
    sl = o("mov.u32", f"{name}_l")
    wa = o("mad.lo.u32", warp, D * 4, sm)
    wa = o("mad.lo.u32", lane, per_lane * 4, wa)
    e(f"st.shared.{vec}.f32 [{wa}], {{{', '.join(acc)}}};")
    e(f"st.shared.f32 [{o('mad.lo.u32', warp, 4, sl)}], {l};")                 # every lane holds the same l
    e("bar.sync 0;")
    e(f"@{e.cond('ge.u32', tid, D // 2)} ret;")
    ls = [e.r("f") for _ in range(4)]
    e(f"ld.shared.v4.f32 {{{', '.join(ls)}}}, [{sl}];")
    lt = o("add.f32", o("add.f32", ls[0], ls[1], cls="f"), o("add.f32", ls[2], ls[3], cls="f"), cls="f")
    xs = [o("mov.b32", "0f00000000", cls="f") for _ in range(2)]
    ra = o("mad.lo.u32", tid, 8, sm)
    for k in range(4):
        y = [e.r("f") for _ in range(2)]
        e(f"ld.shared.v2.f32 {{{y[0]}, {y[1]}}}, [{ra}+{k * D * 4}];")
        for i in range(2):
            e(f"add.f32 {xs[i]}, {xs[i]}, {y[i]};")
    p_zero = e.cond("eq.f32", lt, "0f00000000")
    inv = o("rcp.rn.f32", o("selp.f32", "0f3F800000", lt, p_zero, cls="f"), cls="f")
    x0, x1 = (o("mul.f32", x, inv, cls="f") for x in xs)
    word = o("cvt.rn.f16x2.f32" if dtype == "f16" else "cvt.rn.bf16x2.f32", x1, x0)
    word = o("selp.b32", 0, word, p_zero)
    oa = at(at(gptr("p_O"), row, D * 2), tid, 4)
    e(f"st.global.b32 [{oa}], {word};")
    ln, fn, on = names
    params = [("lens", ln, 4), ("fresh", fn, 4), ("O", on, 4), ("part", scratch, 32)]
    text = [f".visible .entry {name}(", ",\n".join(f"\t.param .u64 p_{p}" for p, _, _ in params), ")",
            ".reqntid 128, 1, 1", "{"]
    text += e.decls() + e.lines + ["\tret;", "}"]
    return {"name": name, "kind": "paged_attention_join", "params": [n for _, n, _ in params], "raw_entry": text,
            "raw_decls": [f".shared .align 16 .b8 {name}_sum[{4 * D * 4}];", f".shared .align 16 .b8 {name}_l[16];"],
            "grid": [batch * chunk * heads, 1, 1], "block": [128, 1, 1], "dyn_smem": 0,
            "align": {n: a_ for _, n, a_ in params}, "zero_outputs": [], "pdl": True}
