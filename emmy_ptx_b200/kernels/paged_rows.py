"""Attention of a few query rows over a paged key/value cache: the decode step and short drafts.

The same operator as :mod:`.tc_paged_attention`, for units of at most 64 rows (new tokens x the group's heads).
There the products are small and the time goes into reading the cache, so nothing here is shared between warps:
a warp takes every n-th block of 16 keys of its unit, keeps the online softmax and O of its rows in registers and
meets the other warps once, at the end.

* **Work.**  One CTA a unit where sequences are short.  Otherwise the 64-key tiles of all units, in order of
  sequence and key head, are cut into equal runs, one for each CTA the GPU holds at a time: every CTA reads the
  lengths, takes prefix sums over the batch and so finds its own run, whatever the lengths are.  A run may end one
  unit, cover some and begin another; units of more than one run leave parts in f32 (O, the reference m and the sum l)
  that a second entry joins.
* **Loads.**  Each warp has a ring of ``stages`` blocks in shared memory, filled by TMA (16 rows of 128 bytes a box, or
  8 where a page is no multiple of 16) one ring ahead; page numbers are fetched a block earlier.  Only its own
  warp reads a stage, so a barrier per stage and the warp's own convergence are all the synchronisation there
  is.  Copies by ``cp.async`` (16 bytes a lane) held the same schedule at 5.0 TB/s whatever the ring and with
  the products taken out.
* **Products.**  ``mma.sync`` m16n8k16 with f32 accumulators: S = Q K^T takes a row's 16 bytes as they lie (lane
  (g, t) takes the 16-byte pieces 2 t and 2 t + 1 of each 128 bytes of key g's row, which the 128-byte swizzle puts
  into different banks for a quarter warp; Q is read in the same order, and a dot product does not mind the
  order of its terms); O += P V takes pairs of V rows, put together by byte permutes.  Eight rows
  or fewer use half of the tile's registers.  Units of more than 16 rows give each 16 rows their own warps, which
  read the same keys from L1 and L2.
* **Numerics** as in the tensor-memory form: scores, sums and O in f32; P in f16 (to nearest, lifted by 2^7) for
  f16 caches and bytes, in two bf16 parts (2^-14 together, at most 1) for bf16 caches; bytes are converted to f16
  exactly.
  The reference of a row is raised when a score exceeds it by 2^8, so most blocks need no maximum.

* **What is masked** keeps its promise: V rows that no row of the unit sees become 0 in registers, and where some rows
  see a key and others do not, an infinity or a NaN in its V row is taken out of the product and put back by two
  products of indicators (which rows see the key, which elements are +inf or NaN, -inf or NaN).

Measured on one B200 (8 key heads of 128, 4 query heads each): 48 sequences of 17 to 8192 tokens, bf16, 830 MB: the
kernel 133 us, 6.25 TB/s (0.97 of a copy), the call 136-141; the same in bytes 86 and 94-98 us, where issue slots are the
busiest resource (51 % of the active cycles); one sequence of 333 tokens 6.9 us.

The tcgen05 form holds a row a thread: four rows keep 4 of its 128 softmax threads busy, and each tile passes
through TMA, MMA, TMEM and back.
"""
from __future__ import annotations

import math

from .ptxasm import wait_bar_warp
from .tc_paged_attention import LOG2E, RESCALE, _E, _f32, _unit, lift_of, q_most

MAX_ROWS = 64
ERR_ROWS = 77                    # a block's copy never completed


def supported(dim, chunk, heads, kv_heads, page) -> bool:
    """Head dims of one or two 128-byte columns, pages of whole 8-row pieces, at most 64 rows a unit."""
    return dim in (64, 128) and page % 8 == 0 and chunk * (heads // kv_heads) <= MAX_ROWS


def few_rows(quant) -> int:
    """The most rows a unit of this form has unless it is asked for (``paged_rows``) or the tcgen05 form does not take
    the pages; larger units take that.  16 sequences of up to 5000 tokens, 4 key heads of 128, us here and there: bf16 16
    rows 33 and 35, 24 rows 43 and 37, 64 rows 72 and 39; bytes (whose conversion costs the other form more) 32 rows 39
    and 41, 40 rows 47 and 41, 64 rows 59 and 43."""
    return 32 if quant else 16


def shape(dim, chunk, heads, kv_heads, quant, wide=False):
    """(rows, 16-row tiles, warps, ring stages, bytes of a stage) of a CTA.  ``wide``: few units of up to 16 rows, one
    CTA each, that are bound by the chain of a warp's blocks, take eight warps (one sequence of 333 tokens, 8 key heads
    of 128: 6.9 us, 8.7 with four; 16 such sequences 8.8 and 11.2)."""
    rows = chunk * (heads // kv_heads)
    mt = -(-rows // 16)
    warps = 8 if wide and mt == 1 else {1: 4, 2: 4, 3: 3, 4: 4}[mt]
    stage_bytes = 2 * block_keys(quant) * dim * (1 if quant else 2)
    return rows, mt, warps, (16384 if quant else 8192) // stage_bytes, stage_bytes


def max_registers(rows, quant) -> int:
    """Registers a thread: 128 for at most 8 rows of a 16-bit cache, where 16 warps an SM with one 8 KiB block each
    keep HBM busy (a batch of 48 at 137 us; 139 with 168 registers); 168 where there is more arithmetic (the same
    batch in bytes: 90 us with two blocks a warp, 94 at 128 registers).  The cap of 128 spills 24 to 68 bytes a thread at
    dim 128 in bf16, also in the forms that it was not measured for (a CTA a unit: few short sequences, windows)."""
    return 128 if rows <= 8 and not quant else 168


def block_keys(quant) -> int:
    """Keys of a block: 16, the second product's depth; 32 for bytes, which have more work a byte to share."""
    return 32 if quant else 16


# Sequences whose lengths each CTA takes prefix sums of.  Above it a unit has one CTA, in the table's order.  Sequences of
# 17 to 3000 tokens, 8 key heads of 128, bf16, against their bytes at a copy's rate: 128 of them 143 us over 125, 129 of
# them 152 over 126, 256 of them 262 over 244; with one key head 256 units are too few to even out: 53 over 30.
MAX_SPREAD_BATCH = 128
MIN_TILES = 4                    # a run's least tiles: one for each of four warps


def _longest(chunk, page, max_pages, window, sinks):
    """The most tiles a unit can have."""
    longest = -(-max_pages * page // 64)
    return longest if window is None else min(longest, -(-sinks // 64) + (window + chunk - 1) // 64 + 2)


def most_tiles(batch, chunk, heads, kv_heads, page, max_pages, window, sinks):
    """The most tiles all units can have."""
    return batch * kv_heads * _longest(chunk, page, max_pages, window, sinks)


def plan_ctas(batch, chunk, heads, kv_heads, dim, quant, page, max_pages, window, sinks, sms=148):
    """CTAs to spread the tiles over, or 0 for one CTA a unit: for sequences of at most 8 tiles (a second launch
    would cost more than their keys), for windows when there are units for every SM (all units are alike
    then) and for batches whose prefix sums would take long (they have many units).  As many as are on the GPU at a time:
    twice as many give a batch of 48 sequences the same (137 us in bf16, 90 and 92 in bytes) and one of 16 less (35 us
    against 31 in bf16, 33 against 29 in bytes)."""
    longest = _longest(chunk, page, max_pages, window, sinks)
    units = batch * kv_heads
    if window is not None and units >= 2 * sms:
        return 0
    if longest <= 8 or batch > MAX_SPREAD_BATCH or units * longest >= 1 << 31:
        return 0
    rows, _, warps, _, _ = shape(dim, chunk, heads, kv_heads, quant)
    resident = 65536 // (max_registers(rows, quant) * 32 * warps)
    return resident * sms


def _tiles_of(e, at, lens_ptr, fresh_ptr, b, ok, chunk, cap, window, sinks):
    """Tiles a key head of sequence ``b`` walks (0 where ``ok`` is false or nothing is new)."""
    o = e.o
    n_, f_ = o("mov.u32", 0), o("mov.u32", 0)
    e(f"@{ok} ld.global.nc.u32 {n_}, [{at(lens_ptr, o('mul.wide.u32', b, 4, cls='rd'))}];")
    e(f"@{ok} ld.global.nc.u32 {f_}, [{at(fresh_ptr, o('mul.wide.u32', b, 4, cls='rd'))}];")
    total = _unit(e, n_, f_, o("mov.u32", 0), chunk, chunk, cap, window, sinks)["total"]
    return o("selp.u32", total, 0, e.cond("gt.s32", f_, 0))


def paged_rows_entry(name, batch, chunk, heads, kv_heads, dim, pages, page, max_pages, dtype, quant, window, sinks,
                     scale, names, scratch, ctas, min_tiles=MIN_TILES, prefix="", sms=148):
    """The launch record and PTX; arguments as :func:`.tc_paged_attention.paged_attention_entry`, with ``ctas`` CTAs
    to spread the tiles over (0: one a unit) in runs of at least ``min_tiles``."""
    D = dim
    group = heads // kv_heads
    eight = not ctas and batch * kv_heads <= (1 if quant else 2) * sms            # all of them on the GPU at a time
    rows, mt, warps, stages, stage_b = shape(dim, chunk, heads, kv_heads, quant, eight)
    streams = warps // mt
    threads = 32 * warps
    grid = ctas or batch * kv_heads
    few = rows <= 8                          # the tile's upper 8 rows are not there
    half = dtype == "f16"
    p_f16 = half or quant                    # P and V in f16; otherwise bf16, P in two parts
    q_f16 = half or quant                    # Q and K in f16
    es = 1 if quant else 2
    row_b = D * es                           # a cache row
    cap = max_pages * page
    ksteps, nts = D // 16, D // 8
    nk = row_b // 64                         # 16-byte pieces a lane takes of a K row
    BLK = block_keys(quant)
    NT, KB = BLK // 8, BLK // 16             # 8-key tiles of S and 16-key steps of P V in a block
    bpt = 64 // BLK                          # blocks of a 64-key tile
    prow = math.gcd(page, BLK)               # rows of a block that lie on one page at least
    pieces = range(BLK // prow)
    scan = not quant and chunk > 1           # rows of different positions share V rows that may hold anything
    sc_b = 2 * BLK * 4 if quant else 0       # bytes of a block's scales
    bw = min(row_b, 128)                     # bytes of a box row, and the swizzle's span
    boxes = row_b // bw
    v_ld = 8 if (quant and D == 64) else 16  # bytes of a lane's V pieces
    nv = (row_b // 8) // v_ld                # pieces a lane takes of a V row
    cscale = _f32(scale * LOG2E)
    e = _E()
    o = e.o
    hs = (0,) if few else (0, 1)             # the tile's row halves: rows g and g + 8

    def gptr(pname):
        return o("cvta.to.global.u64", o("ld.param.u64", f"[{pname}]", cls="rd"), cls="rd")

    def wide(x, n):
        return o("mul.wide.u32", x, n, cls="rd")

    def at(base, off):
        return o("add.s64", base, off, cls="rd")

    tid = o("mov.u32", "%tid.x")
    warp, lane = o("shr.u32", tid, 5), o("and.b32", tid, 31)
    g, t = o("shr.u32", lane, 2), o("and.b32", lane, 3)
    cta = o("mov.u32", "%ctaid.x")
    smem_sym = f"{prefix}rows_smem"
    raw = o("mov.u32", smem_sym)
    sbase = o("and.b32", o("add.u32", raw, 1023), -1024)
    wbase = o("mad.lo.u32", warp, stages * stage_b, sbase)    # this warp's ring
    scal = o("mad.lo.u32", warp, stages * sc_b, o("add.u32", sbase, warps * stages * stage_b))     # its keys' scales
    # the rings and scales, or where the warps meet (m, l and O of each, rows padded by 4 banks)
    RW = 8 if few else 16                                      # rows a warp holds
    orow = D * 4 + 16
    area = max(warps * stages * (stage_b + sc_b), warps * RW * (orow + 8))
    bars = o("add.u32", o("mad.lo.u32", warp, stages * 8, sbase), area)
    # this lane's pieces, from a stage: K rows 8 a + g at k_at[i] + 8 a rows, V rows 8 a + 2 t + j at v_at[j] + 8 a rows,
    # each box BLK rows on; the swizzle exchanges 16-byte pieces by the row's place in its 128 bytes x 8
    if bw == 128:
        k_at = [o("mad.lo.u32", o("xor.b32", o("mad.lo.u32", t, 2, i), g), 16, o("shl.b32", g, 7)) for i in range(2)]
        v_at = []
        for j in range(2):
            r_ = o("mad.lo.u32", t, 2, j)
            v_at.append(o("mad.lo.u32", o("xor.b32", g, r_), 16, o("shl.b32", r_, 7)))
    else:                                                     # 64-byte rows of bytes: pieces of 16 for K, 8 for V
        k_at = [o("mad.lo.u32", o("xor.b32", t, o("shr.u32", g, 1)), 16, o("shl.b32", g, 6))]
        v_at = []
        for j in range(2):
            r_ = o("mad.lo.u32", t, 2, j)
            x_ = o("mad.lo.u32", o("xor.b32", o("shr.u32", g, 1), t), 16, o("shl.b32", r_, 6))
            v_at.append(o("mad.lo.u32", o("and.b32", g, 1), 8, x_))
    v_off = BLK * row_b                                       # V behind K
    k_imm = [[(hb * BLK + 8 * a) * bw for hb in range(boxes)] for a in range(NT)]
    err = gptr("p_err")
    tk, tv = [o("cvta.param.u64", o("mov.u64", f"p_tm{x}", cls="rd"), cls="rd") for x in "KV"]
    p_l0 = e.cond("eq.u32", lane, 0)
    l_init = e.L("noinit")
    e(f"@!{p_l0} bra {l_init};")
    for s_ in range(stages):
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{8 * s_}], 1;")
    e("fence.mbarrier_init.release.cluster;")
    e("fence.proxy.async.shared::cta;")
    e.label(l_init)
    e("bar.warp.sync -1;")
    # a bit for each ring stage: its barrier's phase; it holds a block that needs masks; a piece of it lies on no page
    phase, edge = o("mov.u32", 0), o("mov.u32", 0)
    gone = [o("mov.u32", 0) for _ in pieces]
    failed = o("mov.u32", 0)
    lens_ptr, fresh_ptr = gptr("p_lens"), gptr("p_fresh")
    l_exit, l_seg, l_find = e.L("exit"), e.L("seg"), e.L("find")
    if ctas:
        e("griddepcontrol.launch_dependents;")                # the join's blocks may come up and wait
        # prefix sums of the sequences' tiles (over their key heads), 32 at a time
        run, sums = None, []
        for k in range(-(-batch // 32)):
            bb = o("add.u32", lane, 32 * k) if k else lane
            v = o("mul.lo.u32", _tiles_of(e, at, lens_ptr, fresh_ptr, bb, e.cond("lt.u32", bb, batch), chunk, cap, window,
                                          sinks), kv_heads)
            sums.append(v)
        for k, v in enumerate(sums):
            for d_ in (1, 2, 4, 8, 16):
                up = o("shfl.sync.up.b32", v, d_, 0, -1)
                e(f"@{e.cond('ge.u32', lane, d_)} add.u32 {v}, {v}, {up};")
            if run is not None:
                e(f"add.u32 {v}, {v}, {run};")
            run = o("shfl.sync.idx.b32", v, 31, 31, -1)
        per = o("div.u32", o("add.u32", run, ctas - 1), ctas)
        per = o("max.u32", per, min_tiles)
        start = o("mul.lo.u32", cta, per)
        e(f"@{e.cond('ge.u32', start, run)} ret;")            # no tiles for this CTA
        stop = o("min.u32", o("add.u32", start, per), run)
        # the first sequence that ends behind the start, and the tiles before it
        b, before = o("mov.u32", 0), o("mov.u32", 0)
        for v in sums:
            past = e.cond("le.u32", v, start)
            e(f"add.u32 {b}, {b}, {o('popc.b32', o('vote.sync.ballot.b32', past, -1))};")
            e(f"max.u32 {before}, {before}, {o('redux.sync.max.u32', o('selp.u32', v, 0, past), -1)};")
        now = o("mov.u32", start)
        e.label(l_find)
    else:
        kvh, b = o("rem.u32", cta, kv_heads), o("div.u32", cta, kv_heads)
    b_len = o("ld.global.nc.u32", f"[{at(lens_ptr, wide(b, 4))}]")
    b_new = o("ld.global.nc.u32", f"[{at(fresh_ptr, wide(b, 4))}]")
    if not ctas:
        e(f"@{e.cond('le.s32', b_new, 0)} ret;")              # nothing new in this sequence
    w = _unit(e, b_len, b_new, o("mov.u32", 0), chunk, chunk, cap, window, sinks)
    total, end, pos0, pos1 = w["total"], w["end"], w["pos0"], w["pos1"]
    i0, nb = None, total
    if ctas:
        tb = o("selp.u32", total, 0, e.cond("gt.s32", b_new, 0))
        behind = o("mad.lo.u32", tb, kv_heads, before)
        p_in = e.cond("lt.u32", now, behind)
        e(f"@{p_in} bra {l_seg};")
        e(f"mov.u32 {before}, {behind};")                     # the run goes on in a later sequence
        e(f"add.u32 {b}, {b}, 1;")
        e(f"bra {l_find};")
        e.label(l_seg)
        off = o("sub.u32", now, before)
        kvh = o("div.u32", off, tb)
        i0 = o("sub.u32", off, o("mul.lo.u32", kvh, tb))
        nb = o("min.u32", o("sub.u32", tb, i0), o("sub.u32", stop, now))
    vrows = o("mul.lo.u32", w["n"], group)
    base_row = o("mad.lo.u32", o("mul.lo.u32", b, chunk), heads, o("mul.lo.u32", kvh, group))

    def row_index(r):
        if group == 1:
            return o("mad.lo.u32", r, heads, base_row)
        t_ = o("div.u32", r, group)
        return o("add.u32", o("mad.lo.u32", t_, heads, base_row), o("sub.u32", r, o("mul.lo.u32", t_, group)))

    # blocks of keys, without those of the last tile that lie past the end
    nblk = o("mul.lo.u32", nb, bpt)

    def tile_of(j):
        i = o("add.u32", j, i0) if i0 is not None else j
        if window is None:
            return i
        past = e.cond("ge.u32", i, w["st"])
        return o("selp.u32", o("add.u32", i, w["gap"]), i, past)

    def key_of(n):
        """The first key of the part's block n."""
        return o("mad.lo.u32", o("and.b32", n, bpt - 1), BLK, o("shl.b32", tile_of(o("div.u32", n, bpt)), 6))

    last0 = key_of(o("sub.u32", nblk, 1))                     # total = 0: no blocks, whatever this gives
    over = o("max.s32", o("sub.s32", o("add.u32", last0, BLK), end), 0)
    p_any = e.cond("ne.u32", nb, 0)
    e(f"@{p_any} sub.u32 {nblk}, {nblk}, {o('div.u32', over, BLK)};")
    e(f"@{e.cond('ne.u32', failed, 0)} mov.u32 {nblk}, 0;")

    table = at(gptr("p_table"), wide(b, 4 * max_pages))
    if quant:
        ksp, vsp = gptr("p_KS"), gptr("p_VS")
    mtile = o("rem.u32", warp, mt) if mt > 1 else None
    stream = o("div.u32", warp, mt) if mt > 1 else warp

    def fetch(n, regs):
        """The page of each piece of block n, or -1 (past the blocks, or outside the table)."""
        ok = e.cond("lt.u32", n, nblk)
        k0 = key_of(n)
        for h in pieces:
            slot = o("div.u32", o("add.u32", k0, prow * h) if h else k0, page)
            okh = e.cond("lt.u32", slot, max_pages)
            e(f"and.pred {okh}, {okh}, {ok};")
            e(f"mov.u32 {regs[h]}, -1;")
            e(f"@{okh} ld.global.nc.u32 {regs[h]}, [{at(table, wide(slot, 4))}];")

    tt2 = o("shl.b32", t, 1)
    hoff = o("mul.lo.u32", kvh, page)

    def copy(n, regs, sbit, so, bar):
        """Block n's copies into the ring stage at byte ``so`` of the ring (bit ``sbit`` of ``edge``), by lane 0."""
        l_no = e.L("nocp")
        e(f"@{e.cond('ge.u32', n, nblk)} bra {l_no};")
        k0 = key_of(n)
        last = o("add.u32", k0, BLK)
        okp = [e.cond("lt.u32", regs[h], pages) for h in pieces]
        # plain: every row of the unit sees every key of the block
        plain = e.cond("le.s32", last, o("add.s32", pos0, 1))
        p_ = e.cond("le.u32", last, end)
        e(f"and.pred {plain}, {plain}, {p_};")
        for p_ in okp:
            e(f"and.pred {plain}, {plain}, {p_};")
        if window is not None:
            p1, p2 = e.cond("gt.s32", k0, o("sub.s32", pos1, window)), e.cond("le.u32", last, sinks)
            e(f"or.pred {p1}, {p1}, {p2};")
            e(f"and.pred {plain}, {plain}, {p1};")
        e(f"or.b32 {edge}, {edge}, {sbit};")
        e(f"@{plain} sub.u32 {edge}, {edge}, {sbit};")
        for x, p_ in zip(gone, okp):
            e(f"or.b32 {x}, {x}, {sbit};")
            e(f"@{p_} sub.u32 {x}, {x}, {sbit};")
        e(f"@!{p_l0} bra {l_no};")
        nbytes = o("mov.u32", stage_b)
        if quant:
            for p_ in okp:
                e(f"@{p_} add.u32 {nbytes}, {nbytes}, {8 * prow};")
        e(f"mbarrier.arrive.expect_tx.shared::cta.b64 _, [{bar}], {nbytes};")
        dst = o("add.u32", wbase, so)
        rows_at = [o("rem.u32", o("add.u32", k0, prow * h) if h else k0, page) for h in pieces]
        for x, tm in enumerate((tk, tv)):
            for h in pieces:
                pgc = o("selp.b32", regs[h], -1, okp[h])       # outside the pool: the box reads zeros
                ro = rows_at[h]
                for hb in range(boxes):
                    e(f"cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                      f"[{dst}+{x * v_off + (hb * BLK + prow * h) * bw}], [{tm}, {{{64 * hb}, {ro}, {kvh}, {pgc}}}], [{bar}];")
        if quant:
            sd = o("mad.lo.u32", o("div.u32", so, stage_b), sc_b, scal)
            for h in pieces:
                off = o("mad.wide.u32", regs[h], kv_heads * page * 4, wide(o("add.u32", hoff, rows_at[h]), 4), cls="rd")
                for x, ptr in enumerate((ksp, vsp)):
                    e(f"@{okp[h]} cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes "
                      f"[{sd}+{4 * (BLK * x + prow * h)}], [{at(ptr, off)}], {4 * prow}, [{bar}];")
        e.label(l_no)

    # ---- Q: the rows of this warp's tile, in the order the keys' bytes come ------------------
    q_ptr = gptr("p_Q")
    r0 = o("mad.lo.u32", mtile, 16, g) if mt > 1 else g
    qa = [[None] * 4 for _ in range(ksteps)]
    zero = o("mov.b32", 0)
    pos, crow = [], []                                         # positions; scale * log2(e) for the row's scores
    for h in hs:
        r_ = o("add.u32", r0, 8 * h) if h else r0
        okr = e.cond("lt.u32", r_, vrows)
        src = at(q_ptr, wide(row_index(r_), D * 2))
        # 16 bytes of K meet 16 (or, bytes, 32) of Q; a lane's pieces of a box row lie side by side
        per_p = 32 if quant else 16
        np_ = nk // boxes                                      # pieces a lane takes of a box row
        src = at(src, wide(t, np_ * per_p))
        got = []
        for hb in range(boxes):
            for i in range(np_):
                for x in range(per_p // 16):
                    d_ = [o("mov.b32", 0) for _ in range(4)]
                    e(f"@{okr} ld.global.nc.v4.b32 {{{', '.join(d_)}}}, [{src}+{hb * 128 + i * per_p + 16 * x}];")
                    got += d_
        if q_f16 and not half:
            # bf16 to f16: the row times a power of two that brings its largest number to 2^14 (see q_most), exact
            # but for numbers 2^-28 of the largest and less; the scores take the inverse
            big = None
            for x in got:
                a_ = o("and.b32", x, "0x7FFF7FFF")
                big = a_ if big is None else o("max.u16x2", big, a_)
            big = o("max.u32", o("and.b32", big, 65535), o("shr.u32", big, 16))
            for d_ in (1, 2):
                big = o("max.u32", big, o("shfl.sync.bfly.b32", big, d_, 31, -1))
            ex = o("sub.s32", 127 + 14, o("shr.u32", big, 7))     # 14 less the largest's exponent
            ex = o("min.s32", ex, q_most(scale))
            up = o("shl.b32", o("add.s32", ex, 127), 23, cls="f")
            down = o("shl.b32", o("sub.s32", 127, ex), 23, cls="f")
            crow.append(o("mul.f32", down, cscale, cls="f"))
            got = [o("cvt.rn.f16x2.f32", o("mul.f32", o("and.b32", x, -65536, cls="f"), up, cls="f"),
                     o("mul.f32", o("shl.b32", x, 16, cls="f"), up, cls="f")) for x in got]
        else:
            crow.append(cscale)
        for ks in range(ksteps):                               # two registers a k-step
            qa[ks][h], qa[ks][2 + h] = got[2 * ks], got[2 * ks + 1]
        tok = o("div.u32", r_, group) if group > 1 else r_
        pos.append(o("min.s32", o("add.s32", pos0, tok), pos1))
    if few:
        for ks in range(ksteps):
            qa[ks][1] = qa[ks][3] = zero

    # four registers a tile, also where its upper rows are not there: products take them in fours, and sharing the
    # upper two between tiles cost more moves than it saved registers
    acc = [[o("mov.b32", "0f00000000", cls="f") for _ in range(4)] for _ in range(nts)]
    m = [o("mov.b32", "0fFF800000", cls="f") for _ in hs]
    l = [o("mov.b32", "0f00000000", cls="f") for _ in hs]
    ty = "f16.f16" if q_f16 else "bf16.bf16"
    pty = "f16.f16" if p_f16 else "bf16.bf16"

    def mma(tys, d, a_, b_, c):
        e(f"mma.sync.aligned.m16n8k16.row.col.f32.{tys}.f32 {{{', '.join(d)}}}, {{{', '.join(a_)}}}, "
          f"{{{', '.join(b_)}}}, {{{', '.join(c)}}};")

    # ---- the ring: ``stages`` blocks ahead --------------------------------------------------
    pg = [e.r() for _ in pieces]
    nn = o("mov.u32", stream)                                  # the next block to copy
    for s_ in range(stages):
        fetch(nn, pg)
        copy(nn, pg, o("mov.u32", 1 << s_), o("mov.u32", s_ * stage_b), o("add.u32", bars, 8 * s_))
        e(f"add.u32 {nn}, {nn}, {streams};")
    fetch(nn, pg)
    n = o("mov.u32", stream)
    rd, rbit = o("mov.u32", 0), o("mov.u32", 1)                # the stage to read next, and its bit
    l_fail = e.L("fail")
    lift = lift_of(dtype, quant)
    if quant:
        c64, c1152 = o("mov.b32", "0x64646464"), o("mov.b32", "0x64806480")
        c6400 = o("mov.b32", "0x64006400")
        # P carries the values' scales over vref, a power of two at least half the largest scale (of either sign) the
        # warp's rows met: P is at most 2^15 in f16, and what is 2^-20 of the largest scale's still has 11 bits
        vref = o("mov.b32", "0f00800000", cls="f")
        vinv = o("mov.b32", "0f7E800000", cls="f")
    l_top, l_done = e.L("blk"), e.L("blkd")
    e.label(l_top)
    e(f"@{e.cond('ge.u32', n, nblk)} bra {l_done};")
    bar = o("mad.lo.u32", rd, 8, bars)
    par = o("selp.u32", 1, 0, e.cond("ne.u32", o("and.b32", phase, rbit), 0))
    wait_bar_warp(e, bar, par, err, ERR_ROWS, l_fail)
    e(f"xor.b32 {phase}, {phase}, {rbit};")
    so = o("add.u32", wbase, o("mul.lo.u32", rd, stage_b))
    if quant:
        sc = o("add.u32", o("mad.lo.u32", rd, sc_b, scal), o("shl.b32", t, 3))
    ka = [o("add.u32", so, x) for x in k_at]
    va = [o("add.u32", so, x) for x in v_at]
    # S = Q K^T, 8 keys a tile
    sv, ys = [], []
    for a in range(NT):
        bs = []
        for i in range(nk):
            d_ = [e.r() for _ in range(4)]
            e(f"ld.shared.v4.b32 {{{', '.join(d_)}}}, [{ka[i % len(ka)]}+{k_imm[a][i // len(ka)]}];")
            if not quant:
                bs += [(d_[0], d_[1]), (d_[2], d_[3])]
            else:                                              # 1024 + b less 1152
                bs += [tuple(o("sub.rn.f16x2", o("prmt.b32", x, c64, sel), c1152) for sel in ("0x4140", "0x4342"))
                       for x in d_]
        cur = [o("mov.b32", "0f00000000", cls="f") for _ in range(4)]
        for ks in range(ksteps):
            mma(ty, cur, qa[ks], bs[ks], cur)
        if quant:
            f_, y_ = [e.r("f"), e.r("f")], [e.r("f"), e.r("f")]
            e(f"ld.shared.v2.f32 {{{f_[0]}, {f_[1]}}}, [{sc}+{32 * a}];")
            e(f"ld.shared.v2.f32 {{{y_[0]}, {y_[1]}}}, [{sc}+{4 * BLK + 32 * a}];")
            for x in range(2 * len(hs)):
                e(f"mul.f32 {cur[x]}, {cur[x]}, {f_[x & 1]};")
            ys.append(y_)
        sv.append(cur)
    # which keys each row sees; blocks that every row sees whole skip this
    l_seen = e.L("seen")
    live = [e.cond("eq.u32", lane, lane) for _ in range(4)]
    sees = {(a, j, h): e.cond("eq.u32", lane, lane) for a in range(NT) for j in range(2) for h in hs}
    whole = e.cond("eq.u32", o("and.b32", edge, rbit), 0)
    e(f"@{whole} bra {l_seen};")
    key0 = key_of(n)
    pk = [e.cond("eq.u32", o("and.b32", x, rbit), 0) for x in gone]
    if not quant:
        for r_ in range(4):
            key = o("add.u32", o("add.u32", key0, 8 * (r_ // 2) + r_ % 2), tt2)
            e(f"setp.lt.u32 {live[r_]}, {key}, {end};")
            if window is not None:
                p1, p2 = e.cond("ge.u32", key, w["lo"]), e.cond("lt.u32", key, sinks)
                e(f"or.pred {p1}, {p1}, {p2};")
                e(f"and.pred {live[r_]}, {live[r_]}, {p1};")
    for a in range(NT):
        for j in range(2):
            key = o("add.u32", o("add.u32", key0, 8 * a + j), tt2)
            any_ = None
            for h in hs:
                ps = sees[a, j, h]
                e(f"setp.le.s32 {ps}, {key}, {pos[h]};")
                e(f"and.pred {ps}, {ps}, {pk[8 * a // prow]};")
                if window is not None:
                    p1 = e.cond("gt.s32", o("add.s32", key, window), pos[h])
                    p2 = e.cond("lt.s32", key, sinks)
                    e(f"or.pred {p1}, {p1}, {p2};")
                    e(f"and.pred {ps}, {ps}, {p1};")
                e(f"@!{ps} mov.b32 {sv[a][2 * h + j]}, 0fFF800000;")
                if quant and any_ is None:
                    any_ = o("selp.u32", 1, 0, ps)
                elif quant:
                    e(f"@{ps} mov.u32 {any_}, 1;")
            if quant:                                          # scales of keys that this lane's rows do not see
                e(f"@{e.cond('eq.u32', any_, 0)} mov.b32 {ys[a][j]}, 0f00000000;")
    e.label(l_seen)
    # raise the rows' references where a score passed them by 2^8, and vref where a scale reached twice it
    mx, need = [], None
    for h in hs:
        x = None
        for a in range(NT):
            y = o("max.f32", sv[a][2 * h], sv[a][2 * h + 1], cls="f")
            x = y if x is None else o("max.f32", x, y, cls="f")
        mx.append(o("mul.f32", x, crow[h], cls="f"))
        p_ = e.cond("gt.f32", mx[h], o("add.f32", m[h], _f32(RESCALE), cls="f"))
        if need is None:
            need = p_
        else:
            e(f"or.pred {need}, {need}, {p_};")
    if quant:
        ymax = o("mov.b32", "0f00000000", cls="f")
        for a in range(NT):
            for y in ys[a]:                                     # of either sign; a NaN drops out
                e(f"max.f32 {ymax}, {ymax}, {o('abs.f32', y, cls='f')};")
        p_ = e.cond("ge.f32", o("mul.f32", ymax, vinv, cls="f"), "0f40000000")
        e(f"or.pred {need}, {need}, {p_};")
    anyneed = o("vote.sync.any.pred", need, -1, cls="p")
    l_keep = e.L("keep")
    e(f"@!{anyneed} bra {l_keep};")
    if quant:
        yb = o("redux.sync.max.u32", o("mov.b32", ymax), -1)
        yb = o("min.u32", o("and.b32", yb, "0x7F800000"), "0x7E000000")
        yb = o("max.u32", yb, o("mov.b32", vref))
        e(f"mov.b32 {vinv}, {o('sub.u32', '0x7F000000', yb)};")                     # a power of two's inverse
        vscale = o("mul.f32", vref, vinv, cls="f")
        e(f"mov.b32 {vref}, {yb};")
    for h in hs:
        for d_ in (1, 2):
            e(f"max.f32 {mx[h]}, {mx[h]}, {o('shfl.sync.bfly.b32', mx[h], d_, 31, -1, cls='f')};")
        mn = o("max.f32", m[h], mx[h], cls="f")
        al = o("ex2.approx.ftz.f32", o("sub.f32", m[h], mn, cls="f"), cls="f")
        e(f"@{e.cond('eq.f32', mn, '0fFF800000')} mov.b32 {al}, 0f3F800000;")   # nothing seen yet
        e(f"mov.b32 {m[h]}, {mn};")
        e(f"mul.f32 {l[h]}, {l[h]}, {al};")
        if quant:
            al = o("mul.f32", al, vscale, cls="f")
        for nt in range(nts):
            for j in range(2):
                e(f"mul.f32 {acc[nt][2 * h + j]}, {acc[nt][2 * h + j]}, {al};")
    e.label(l_keep)
    for h in hs:
        neg = o("sub.f32", o("mov.b32", _f32(lift), cls="f"), m[h], cls="f")
        e(f"@{e.cond('eq.f32', m[h], '0fFF800000')} mov.b32 {neg}, 0f00000000;")
        part_sum = []
        for a in range(NT):
            for j in range(2):
                x = sv[a][2 * h + j]
                e(f"fma.rn.f32 {x}, {x}, {crow[h]}, {neg};")
                e(f"ex2.approx.ftz.f32 {x}, {x};")
            part_sum.append(o("add.f32", sv[a][2 * h], sv[a][2 * h + 1], cls="f"))
        while len(part_sum) > 1:
            part_sum = [o("add.f32", part_sum[i], part_sum[i + 1], cls="f") for i in range(0, len(part_sum), 2)]
        e(f"add.f32 {l[h]}, {l[h]}, {part_sum[0]};")
    if quant:
        for a in range(NT):
            for j in range(2):
                e(f"mul.f32 {ys[a][j]}, {ys[a][j]}, {vinv};")
                for h in hs:
                    e(f"mul.f32 {sv[a][2 * h + j]}, {sv[a][2 * h + j]}, {ys[a][j]};")
        # a scale that some rows do not see may be NaN: their weights are 0
        l_ok = e.L("whole")
        e(f"@{whole} bra {l_ok};")
        for (a, j, h), ps in sees.items():
            e(f"@!{ps} mov.b32 {sv[a][2 * h + j]}, 0f00000000;")
        e.label(l_ok)
    exp_mask = 0x7C00 if half else 0x7F80
    one = 0x3C00 if half else 0x3F80

    def specials(vr, nt0, n_, a0):
        """Blocks in which a key is seen by some rows only: takes infinities and NaNs out of the V rows ``vr`` and adds
        them to O for the rows that see them, by their signs (a NaN counts as both)."""
        l_out = e.L("clean")
        e(f"@{whole} bra {l_out};")
        m_ = None
        for r_ in range(4):
            for x in vr[r_]:
                x = o("and.b32", x, "0x7FFF7FFF")
                m_ = x if m_ is None else o("max.u16x2", m_, x)
        m_ = o("max.u32", o("and.b32", m_, 65535), o("shr.u32", m_, 16))
        e(f"@!{o('vote.sync.any.pred', e.cond('ge.u32', m_, exp_mask), -1, cls='p')} bra {l_out};")
        va_ = []                                               # which rows see which key: A of the indicators' products
        for a in range(2):
            for h in (0, 1):
                if h not in hs:
                    va_.append(zero)
                    continue
                lo_ = o("selp.u32", one, 0, sees[a0 + a, 0, h])
                va_.append(o("add.u32", lo_, o("selp.u32", one << 16, 0, sees[a0 + a, 1, h])))
        for x in range(n_):
            ind = [[], []]
            for k in range(2):
                sel = "0x7632" if x % 2 else "0x5410"
                w_ = o("prmt.b32", vr[2 * k][x // 2], vr[2 * k + 1][x // 2], sel)
                pos_w, neg_w = o("mov.u32", 0), o("mov.u32", 0)
                for hf in range(2):
                    mag = o("and.b32", w_, 0x7FFF << (16 * hf))
                    sg = o("and.b32", w_, 0x8000 << (16 * hf))
                    p_sp = e.cond("ge.u32", mag, exp_mask << (16 * hf))
                    p_nan = e.cond("gt.u32", mag, exp_mask << (16 * hf))
                    p_neg = e.cond("ne.u32", sg, 0)
                    p_p, p_n = e.r("p"), e.r("p")
                    e(f"not.pred {p_p}, {p_neg};")
                    e(f"or.pred {p_p}, {p_p}, {p_nan};")
                    e(f"and.pred {p_p}, {p_p}, {p_sp};")
                    e(f"or.pred {p_n}, {p_neg}, {p_nan};")
                    e(f"and.pred {p_n}, {p_n}, {p_sp};")
                    e(f"@{p_p} or.b32 {pos_w}, {pos_w}, {one << (16 * hf)};")
                    e(f"@{p_n} or.b32 {neg_w}, {neg_w}, {one << (16 * hf)};")
                ind[0].append(pos_w)
                ind[1].append(neg_w)
            for sgn, big in ((0, "0f7F800000"), (1, "0fFF800000")):
                cnt = [o("mov.b32", "0f00000000", cls="f") for _ in range(4)]
                mma(pty, cnt, va_, ind[sgn], cnt)
                for h in hs:
                    for j in range(2):
                        y = acc[nt0 + x][2 * h + j]
                        e(f"@{e.cond('gt.f32', cnt[2 * h + j], '0f00000000')} add.f32 {y}, {y}, {big};")
        for r_ in range(4):
            for x in vr[r_]:
                lo_, hi_ = o("and.b32", x, 0x7FFF), o("and.b32", x, 0x7FFF0000)
                e(f"@{e.cond('ge.u32', lo_, exp_mask)} and.b32 {x}, {x}, -65536;")
                e(f"@{e.cond('ge.u32', hi_, exp_mask << 16)} and.b32 {x}, {x}, 65535;")
        e.label(l_out)

    for kb in range(KB):
        # P as the second product's A: rows g (and g + 8), keys 2t, 2t+1 and 8 further
        pa = [[None] * 4 for _ in range(1 if p_f16 else 2)]
        for a in range(2):
            for h in (0, 1):
                if h not in hs:
                    for part in pa:
                        part[2 * a + h] = zero
                    continue
                x0, x1 = sv[2 * kb + a][2 * h], sv[2 * kb + a][2 * h + 1]
                if p_f16:
                    pa[0][2 * a + h] = o("cvt.rn.f16x2.f32", x1, x0)
                else:
                    pa[0][2 * a + h] = o("prmt.b32", x0, x1, "0x7632")
                    d0 = o("sub.f32", x0, o("and.b32", x0, -65536, cls="f"), cls="f")
                    d1 = o("sub.f32", x1, o("and.b32", x1, -65536, cls="f"), cls="f")
                    pa[1][2 * a + h] = o("prmt.b32", d0, d1, "0x7632")
        for i in range(nv):
            vr = []
            for r_ in range(4):                                # rows 2t, 2t+1, 2t+8, 2t+9
                d_ = [e.r() for _ in range(v_ld // 4)]
                off = v_off + (i * BLK + 16 * kb + 8 * (r_ // 2)) * bw
                e(f"ld.shared.v{len(d_)}.b32 {{{', '.join(d_)}}}, [{va[r_ % 2]}+{off}];")
                vr.append(d_)
            if not quant:
                # rows that no row of the unit sees may hold anything: P is 0 there, so they become 0 too
                l_live = e.L("live")
                e(f"@{whole} bra {l_live};")
                for r_ in range(4):
                    for x in vr[r_]:
                        e(f"@!{live[r_]} mov.b32 {x}, 0;")
                e.label(l_live)
            per_piece = v_ld // es
            if scan:
                specials(vr, i * per_piece, per_piece, 2 * kb)
            for x in range(per_piece):
                nt = i * per_piece + x
                bb = []
                for k in range(2):
                    lo_, hi_ = vr[2 * k], vr[2 * k + 1]
                    if quant:                                  # byte x of both rows, 1024 + b less 1152
                        t_ = o("prmt.b32", lo_[x // 4], hi_[x // 4], f"0x{4 + x % 4}{4 + x % 4}{x % 4}{x % 4}")
                        t_ = o("lop3.b32", t_, "0x00FF00FF", c6400, "0xEA")
                        bb.append(o("sub.rn.f16x2", t_, c1152))
                    else:
                        bb.append(o("prmt.b32", lo_[x // 2], hi_[x // 2], "0x7632" if x % 2 else "0x5410"))
                for part in pa:
                    mma(pty, acc[nt], part, bb, acc[nt])
    e("bar.warp.sync -1;")                                     # every lane has read the stage
    copy(nn, pg, rbit, o("mul.lo.u32", rd, stage_b), bar)
    e(f"add.u32 {nn}, {nn}, {streams};")
    fetch(nn, pg)
    e(f"add.u32 {n}, {n}, {streams};")
    e(f"add.u32 {rd}, {rd}, 1;")
    e(f"shl.b32 {rbit}, {rbit}, 1;")
    p_ = e.cond("eq.u32", rd, stages)
    e(f"@{p_} mov.u32 {rd}, 0;")
    e(f"@{p_} mov.u32 {rbit}, 1;")
    e(f"bra {l_top};")
    # a copy that never came: this warp does no more work, but meets the others
    e.label(l_fail)
    e(f"mov.u32 {failed}, 1;")
    e.label(l_done)

    # ---- the warps of a row tile meet -------------------------------------------------------
    # a warp's m, l and O go to shared memory (the ring's, once every warp is through with it: all that
    # was copied has been waited for)
    for h in hs:
        for d_ in (1, 2):
            e(f"add.f32 {l[h]}, {l[h]}, {o('shfl.sync.bfly.b32', l[h], d_, 31, -1, cls='f')};")
    e("bar.sync 0;")
    # bytes: O times the scales' power, both sums by 2^-14 first, so that weights are at most 1 (as in bf16): no sum here
    # is larger than that of p v
    out_lift = -RESCALE if quant else lift
    if quant:
        vout = o("mul.f32", vref, _f32(2.0 ** (out_lift - lift)), cls="f")
        for h in hs:
            e(f"mul.f32 {l[h]}, {l[h]}, {_f32(2.0 ** (out_lift - lift))};")
    obase = o("mad.lo.u32", warp, RW * orow, sbase)
    mlb = o("add.u32", sbase, warps * RW * orow)

    piece = v_ld // es                                         # consecutive dims of a (lane, piece)
    span = D // nv                                             # dims of all lanes' pieces i
    p_t0 = e.cond("eq.u32", t, 0)
    for h in hs:
        rr = o("add.u32", g, 8 * h) if h else g
        ra = o("mad.lo.u32", rr, orow, obase)
        ra = o("mad.lo.u32", t, 2 * piece * 4, ra)             # column n = 2t, 2t+1 of a tile: dims n * piece + x
        for i in range(nv):
            for j in range(2):
                for x0 in range(0, piece, 4):
                    vals = [acc[i * piece + x0 + x][2 * h + j] for x in range(4)]
                    if quant:
                        vals = [o("mul.f32", x, vout, cls="f") for x in vals]
                    e(f"st.shared.v4.f32 [{ra}+{(i * span + j * piece + x0) * 4}], {{{', '.join(vals)}}};")
        ma = o("mad.lo.u32", o("mad.lo.u32", warp, RW, rr), 8, mlb)
        e(f"@{p_t0} st.shared.v2.f32 [{ma}], {{{m[h]}, {l[h]}}};")
    e("bar.sync 0;")
    o_ptr = gptr("p_O")
    if ctas:
        p_split = e.cond("ne.u32", nb, tb)                     # the unit has other runs too
        slot = o("shl.b32", cta, 1)                            # a CTA's first segment leaves part 2 c, a later one 2 c + 1
        e(f"@{e.cond('ne.u32', now, start)} add.u32 {slot}, {slot}, 1;")
    cpr = D // 8                                               # 8 dims a thread
    item = o("mov.u32", tid)
    nitems = o("mul.lo.u32", vrows, cpr)
    l_it, l_itd = e.L("it"), e.L("itd")
    e.label(l_it)
    e(f"@{e.cond('ge.u32', item, nitems)} bra {l_itd};")
    r_, ch = o("div.u32", item, cpr), o("rem.u32", item, cpr)
    tile_ = o("shr.u32", r_, 4)
    rin = o("and.b32", r_, 15)
    ms, ls = [], []
    for s_ in range(streams):
        wi = o("add.u32", tile_, s_ * mt)
        ma = o("mad.lo.u32", o("mad.lo.u32", wi, RW, rin), 8, mlb)
        a_, b_ = e.r("f"), e.r("f")
        e(f"ld.shared.v2.f32 {{{a_}, {b_}}}, [{ma}];")
        ms.append(a_)
        ls.append(b_)
    mm = ms[0]
    for x in ms[1:]:
        mm = o("max.f32", mm, x, cls="f")
    mz = o("selp.f32", "0f00000000", mm, e.cond("eq.f32", mm, "0fFF800000"), cls="f")
    lt = o("mov.b32", "0f00000000", cls="f")
    ov = [o("mov.b32", "0f00000000", cls="f") for _ in range(8)]
    for s_ in range(streams):
        f_ = o("ex2.approx.ftz.f32", o("sub.f32", ms[s_], mz, cls="f"), cls="f")
        e(f"fma.rn.f32 {lt}, {f_}, {ls[s_]}, {lt};")
        wi = o("add.u32", tile_, s_ * mt)
        oa = o("mad.lo.u32", o("mad.lo.u32", wi, RW, rin), orow, sbase)
        oa = o("mad.lo.u32", ch, 32, oa)
        for x0 in (0, 4):
            y = [e.r("f") for _ in range(4)]
            e(f"ld.shared.v4.f32 {{{', '.join(y)}}}, [{oa}+{4 * x0}];")
            for x in range(4):
                e(f"fma.rn.f32 {ov[x0 + x]}, {f_}, {y[x]}, {ov[x0 + x]};")
    l_part, l_next = e.L("part"), e.L("next")
    if ctas:
        e(f"@{p_split} bra {l_part};")
    p_zero = e.cond("eq.f32", lt, "0f00000000")
    inv = o("rcp.rn.f32", o("selp.f32", "0f3F800000", lt, p_zero, cls="f"), cls="f")
    pack = "cvt.rn.f16x2.f32" if half else "cvt.rn.bf16x2.f32"
    words = []
    for x in range(0, 8, 2):
        x0, x1 = (o("mul.f32", ov[x + k], inv, cls="f") for k in range(2))
        words.append(o("selp.b32", 0, o(pack, x1, x0), p_zero))
    oa = at(at(o_ptr, wide(row_index(r_), D * 2)), wide(ch, 16))
    e(f"st.global.v4.b32 [{oa}], {{{', '.join(words)}}};")
    if ctas:
        e(f"bra {l_next};")
        e.label(l_part)
        pi = o("mad.lo.u32", slot, rows, r_)
        pa_ = at(at(gptr("p_part"), wide(pi, D * 4)), wide(ch, 32))
        e(f"st.global.v8.f32 [{pa_}], {{{', '.join(ov)}}};")
        mla = at(at(gptr("p_part"), 2 * ctas * rows * D * 4), wide(pi, 8))
        meff = o("sub.f32", mm, _f32(out_lift), cls="f")
        e(f"@{e.cond('eq.u32', ch, 0)} st.global.v2.f32 [{mla}], {{{meff}, {lt}}};")
    e.label(l_next)
    e(f"add.u32 {item}, {item}, {threads};")
    e(f"bra {l_it};")
    e.label(l_itd)
    if ctas:
        e(f"add.u32 {now}, {now}, {nb};")
        e(f"@{e.cond('ge.u32', now, stop)} bra {l_exit};")
        e("fence.proxy.async.shared::cta;")                    # these reads and writes before the next copies
        e("bar.sync 0;")                                       # the ring is free again
        e(f"bra {l_find};")
        e.label(l_exit)

    if quant:
        qn, kn, vn, ksn, vsn, tn, ln, fn, on = names
        params = [("Q", qn, 16), ("KC", kn, 16), ("VC", vn, 16), ("KS", ksn, 16), ("VS", vsn, 16)]
    else:
        qn, kn, vn, tn, ln, fn, on = names
        params = [("Q", qn, 16), ("KC", kn, 16), ("VC", vn, 16)]
    params += [("table", tn, 4), ("lens", ln, 4), ("fresh", fn, 4), ("O", on, 16)]
    sc_spec = []
    if ctas:
        params += [("part", scratch, 32)]
        sc_spec = [{"name": scratch, "dtype": "f32", "shape": [2 * ctas * rows, D + 2], "per_call": True}]
    plist = [f"\t.param .u64 p_{p}" for p, _, _ in params]
    plist += [f"\t.param .align 64 .b8 p_tm{x}[128]" for x in "KV"] + ["\t.param .u64 p_err"]
    text = [f".visible .entry {name}(", ",\n".join(plist), ")", f".reqntid {threads}, 1, 1"]
    text += [f".maxnreg {max_registers(rows, quant)}", "{"]
    text += e.decls() + e.lines + ["\tret;", "}"]
    dyn = area + warps * stages * 8 + 1024
    es_name = "u8" if quant else dtype
    tmaps = [{"name": f"tm{x}", "tensor": nm, "dtype": es_name, "dims": [D, page, kv_heads, pages],
              "strides": [row_b, page * row_b, kv_heads * page * row_b], "box": [bw // es, prow, 1, 1],
              "swizzle": f"{bw}B"} for x, nm in (("K", kn), ("V", vn))]
    return {
        "name": name, "kind": "paged_attention_rows", "params": [n for _, n, _ in params], "raw_entry": text,
        "raw_decls": [f".extern .shared .align 1024 .b8 {smem_sym}[];"],
        "grid": [grid, 1, 1], "block": [threads, 1, 1], "dyn_smem": dyn,
        "align": {n: a_ for _, n, a_ in params}, "zero_outputs": [], "scratch": sc_spec, "tmaps": tmaps, "extra": [{"name": "__err", "kind": "errword"}],
    }


def join_entry(name, batch, chunk, heads, kv_heads, dim, page, max_pages, dtype, window, sinks, names, scratch, ctas,
               min_tiles=MIN_TILES):
    """The second entry: the rows of units of more than one run, o = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.  One
    block a row, which finds its unit's runs by the same sums over the batch; its four warps take every fourth part,
    so that a row of 100 parts is 25 loads deep.  Rows of units of one run are written already; rows that see no key
    at all, which no run covers, become 0."""
    D = dim
    group = heads // kv_heads
    rows, cap = chunk * group, max_pages * page
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
    b_new = o("ld.global.nc.u32", f"[{at(gptr('p_fresh'), b, 4)}]")
    e(f"@{e.cond('ge.s32', c, b_new)} ret;")
    lens_ptr, fresh_ptr = gptr("p_lens"), gptr("p_fresh")
    run, before, tb = o("mov.u32", 0), o("mov.u32", 0), o("mov.u32", 0)
    for k in range(-(-batch // 32)):
        bb = o("add.u32", lane, 32 * k) if k else lane
        v = _tiles_of(e, lambda x, y: o("add.s64", x, y, cls="rd"), lens_ptr, fresh_ptr, bb, e.cond("lt.u32", bb, batch),
                      chunk, cap, window, sinks)
        e(f"add.u32 {run}, {run}, {v};")
        e(f"@{e.cond('lt.u32', bb, b)} add.u32 {before}, {before}, {v};")
        e(f"@{e.cond('eq.u32', bb, b)} mov.u32 {tb}, {v};")
    run, before, tb = (o("redux.sync.add.u32", x, -1) for x in (run, before, tb))
    l_some = e.L("some")
    e(f"@{e.cond('ne.u32', tb, 0)} bra {l_some};")             # a row that sees no key: 0
    e(f"@{e.cond('ge.u32', tid, D // 2)} ret;")
    e(f"st.global.b32 [{at(at(gptr('p_O'), row, D * 2), tid, 4)}], {o('mov.b32', 0)};")
    e("ret;")
    e.label(l_some)
    per = o("div.u32", o("add.u32", o("mul.lo.u32", run, kv_heads), ctas - 1), ctas)
    per = o("max.u32", per, min_tiles)
    t0 = o("mad.lo.u32", before, kv_heads, o("mul.lo.u32", o("div.u32", h, group), tb))
    first = o("div.u32", t0, per)
    last = o("div.u32", o("sub.u32", o("add.u32", t0, tb), 1), per)
    e(f"@{e.cond('eq.u32', first, last)} ret;")                # one run: written already
    nact = o("add.u32", o("sub.u32", last, first), 1)
    # the first run reaches the unit as a later segment unless it begins with it
    late = o("selp.u32", 1, 0, e.cond("ne.u32", t0, o("mul.lo.u32", first, per)))
    rowl = o("mad.lo.u32", c, group, o("rem.u32", h, group))

    def part_row(s_):
        slot = o("shl.b32", o("add.u32", first, s_), 1)
        slot = o("add.u32", slot, o("selp.u32", late, 0, e.cond("eq.u32", s_, 0)))
        return o("mad.lo.u32", slot, rows, rowl)

    part_rows = 2 * ctas * rows
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
