"""Attention of a chunk of new tokens over a paged key/value cache, on the 5th-generation tensor cores.

O = softmax(Q K^T * scale) V over the keys each token sees (:func:`..irgen.paged_attention_ir`): the keys up to
its own position, or a window of them and a few first ones, in pages that a table names.  The cache holds the
activations' 16-bit type, or bytes with one f32 scale per token and head.

**Work.**  A unit is up to 128 query rows of one sequence and one key head: as many tokens as fit with all their
query heads (a row is token * group + head of the group), so one pass over a key head's keys serves its whole
group.  It walks its keys in tiles of 64, the tiles of the first tokens and then those of the window when there is
one.  The tiles of all units, in a row, are cut into equal runs, one for each CTA the GPU holds at a time (two an
SM, half its TMEM columns and shared memory each, so that one's loads and softmax run beside the other's
products): every CTA takes prefix sums over the units and so finds its own run, whatever the lengths are.  A unit of
more than one run leaves parts in f32 (O, the row's reference m and its sum l) and a second entry joins them
(o = sum 2^(m_s - m) O_s / sum 2^(m_s - m) l_s).  Where the units fill the GPU by
themselves, and for very short sequences, a CTA takes one unit, the longest units first: every CTA counts how many come
before its own (4 x 512 tokens behind 333 to 4096 keys, bytes: 100 us, 129 in order of the table).

**Roles.**  One thread issues the ``tcgen05.mma``: S(j+1) = Q K_(j+1)^T into one of two 64-column score buffers, then
O += P(j) V_j.  Four softmax warps hold one row a thread; a warp without a row works on zeros like the others (the
barriers count four).  A warp loads by TMA, one box per page of the tile (at most 64 rows), with the page numbers
fetched 32 at a time one batch ahead.  For 16-bit caches one more warp makes a V tile fit for the product (see what is
masked): done by the softmax warps, that took 86 us in place of 61 for 4 x 1111 tokens with a window of 1024 (24 heads
of 64 on 4, f16).  For a cache of bytes the boxes land in a raw ring, and two warps convert them into the tiles the
products read: with 0x64 as its upper half a byte b is the f16 number 1024 + b, less 1152 it is b - 128, exactly.
Each quarter warp takes 64 bytes of rows r and r ^ 5, which the raw ring's swizzle and the tile's put into different
banks.  The keys' scales multiply the scores' columns, the values' scales multiply P.

**Numerics.**  The score buffers, the running reference and sum, and O are f32.  P is rounded for the tensor core:
f16 caches take f16 P, to nearest (2^-11), with 2^7 put on the exponent so that small weights keep their bits;
bf16 caches take P as two bf16 parts, truncated, 2^-14 together, lowered by the 2^8 the reference may lag behind.  Bytes
are multiplied in f16: a bf16 Q row is brought to 2^14 by a power of two (exact but for numbers 2^-28 of its largest: see
:func:`q_most`), and P carries the values' scales over a running power of two, at least half the largest scale so far (by
magnitude), so that it stays below 2^15 and what is 2^-20 of the largest still has 11 bits.  O is rescaled only when the
row's maximum grew by more than 2^8, or that power did.

**What is masked.**  Scores past the row's own position, outside its window or of a page that the table does not
name become -inf; a row that sees nothing ends as 0.  Rows of a V tile that no row of the CTA sees are zeroed in
shared memory before the product (P is 0 there, but a stale row may hold NaN).  Where some rows see a key and others
do not (the diagonal, a window's edge) the V tile is scanned: an infinity or a NaN must reach the rows that see it,
and no other.  It is added to O by those rows, and the product gets 0 in its place.

The roles (loads, conversion, products, softmax) walk the run's segments on their own, each as far ahead as the
barriers between them let it; barrier phases, ring stages and score buffers go by the tile's number in the run.
Every wait is bounded and reports a code (71-76); TMEM is always freed.
"""
from __future__ import annotations

import math
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
# bytes, the keys' and values' scales of 4 tiles with the power the latter stand over, Q's row factors and the raw
# scales.  A ring of 4 is enough: tile j + 4 comes in after tile j + 2 was converted, whose V waits for the product
# of tile j + 1, so nobody reads slot j any more.  Bytes use the ring barriers 0 and 1 for the raw stages, 2 for the
# converted K and 3 for the converted V.
QFULL = 0
FULL = 8
EMPTY = FULL + 8 * STAGES
SFULL = EMPTY + 8 * STAGES
PFULL = SFULL + 16
PFREE = PFULL + 16
SLOT = PFREE + 16
VOK = SLOT + 8                   # two barriers: a V tile is fit for the product (16-bit caches)
KMASK = 192
KSC = 256
VSC = KSC + 4 * BKV * 4
VREF = 224                       # 4 floats
VBAD = 240                       # two words per score buffer: rows of the V tile that hold an infinity or a NaN
QSC = VSC + 4 * BKV * 4
RAWSC = QSC + 4 * ROWS
AUX_BYTES = RAWSC + 2 * 2 * BKV * 4
QUANT_LIFT = 6.0                 # bytes: P's exponent is lifted by one less, since its scale may be twice vref


def lift_of(dtype, quant) -> float:
    """What P's exponent is lifted by.  In bf16, whose exponents reach as far as f32's, it is lowered by what the
    reference may lag behind, so that weights are at most 1 and a sum of p v is no larger than with the row's maximum."""
    return QUANT_LIFT if quant else F16_LIFT if dtype == "f16" else -RESCALE


def q_most(scale) -> int:
    """The largest power of two that a bf16 Q row is multiplied by for f16: the row's scores take its inverse with the
    scale, and both stay normal f32 numbers.  Rows whose largest number is 2^(14 - q_most) or more (2^-109 with the
    usual scale at dim 128) reach 2^14; a row of zeros takes any power."""
    return min(126, 126 + math.frexp(scale * LOG2E)[1] - 1)


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


MAX_SPREAD_PAIRS = 256           # (sequence, token tile) pairs each CTA takes prefix sums of
MIN_TILES = 4                    # a run's least tiles (one sequence of 5000 tokens, 40 rows: 20.5 us; 24.6 with 8)


def _longest(chunk, heads, kv_heads, page, max_pages, window, sinks):
    """The most tiles a unit can have."""
    longest = -(-max_pages * page // BKV)
    if window is None:
        return longest
    _, tq, _, _ = geometry(chunk, heads, kv_heads)
    return min(longest, -(-sinks // BKV) + (window + min(tq, chunk) - 1) // BKV + 2)


def most_tiles(batch, chunk, heads, kv_heads, page, max_pages, window, sinks):
    """The most tiles all units can have."""
    return (batch * geometry(chunk, heads, kv_heads)[2] * kv_heads
            * _longest(chunk, heads, kv_heads, page, max_pages, window, sinks))


def plan_ctas(batch, chunk, heads, kv_heads, page, max_pages, window, sinks, sms=148):
    """CTAs to spread the tiles over, or 0 for one CTA a unit: for sequences of at most 8 tiles, and where the units
    fill the GPU by themselves.  There the parts and the second launch cost more than equal runs give (a 2048-token
    chunk over 8192 keys, 1024 units: 418 us, 420 with runs; 512 units of cached bytes 100 and 129; a windowed
    chunk of 848 units 59 and 74).  Nor for more pairs than :data:`MAX_SPREAD_PAIRS`, which also go in the table's order:
    not measured, right for any number."""
    pairs = batch * geometry(chunk, heads, kv_heads)[2]
    longest = _longest(chunk, heads, kv_heads, page, max_pages, window, sinks)
    if (longest <= 8 or pairs > MAX_SPREAD_PAIRS or pairs * kv_heads >= 2 * sms
            or pairs * kv_heads * longest >= 1 << 31):
        return 0
    return 2 * sms


def _unit(e, b_len, b_new, c0, tq, chunk, cap, window, sinks):
    """What a unit (a sequence's token tile) walks, from its length and new tokens: emitted alike by the attention
    and by the join.  Returns registers: the last token c1, first and last position, the first window key
    ``lo``, sink tiles ``st``, ``gap`` (tile = i + gap from sink tile st on) and the number of tiles ``total``."""
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
    return dict(n=n, c1=c1, pos0=pos0, pos1=pos1, end=end, lo=lo, st=st, gap=gap, total=total)


class _Place:
    """A (sequence, token tile) pair's registers: sequence ``b``, its length and new tokens, the tile's first token,
    what :func:`_unit` gives, whether it has a token (``live``), its tiles (0 without one) and its rows."""

    def __init__(self, e, pair, ok, lens, fresh, batch, chunk, group, tq, ntile, cap, window, sinks):
        o = e.o
        self.b = o("rem.u32", pair, batch)
        tile = o("sub.u32", ntile - 1, o("div.u32", pair, batch))               # the longest rows of a sequence first
        off = o("mul.wide.u32", self.b, 4, cls="rd")
        n, f = o("mov.u32", 0), o("mov.u32", 0)
        g = f"@{ok} " if ok else ""
        e(f"{g}ld.global.nc.u32 {n}, [{o('add.s64', lens, off, cls='rd')}];")
        e(f"{g}ld.global.nc.u32 {f}, [{o('add.s64', fresh, off, cls='rd')}];")
        self.c0 = o("mul.lo.u32", tile, tq)
        self.w = _unit(e, n, f, self.c0, tq, chunk, cap, window, sinks)
        self.live = e.cond("lt.s32", self.c0, f)
        self.tiles = o("selp.u32", self.w["total"], 0, self.live)
        self.vrows = o("mul.lo.u32", o("add.u32", o("sub.u32", self.w["c1"], self.c0), 1), group)


def _prefix(e, lane, pairs, tiles_of, run_heads):
    """Inclusive prefix sums of ``tiles_of(pair, ok)`` times ``run_heads`` over the pairs, 32 to a register (lane l of
    register k holds pair 32 k + l), and the total."""
    o = e.o
    sums, run = [], None
    for k in range(-(-pairs // 32)):
        q = o("add.u32", lane, 32 * k) if k else lane
        sums.append(o("mul.lo.u32", tiles_of(q, e.cond("lt.u32", q, pairs)), run_heads))
    for v in sums:
        for d in (1, 2, 4, 8, 16):
            up = o("shfl.sync.up.b32", v, d, 0, -1)
            e(f"@{e.cond('ge.u32', lane, d)} add.u32 {v}, {v}, {up};")
        if run is not None:
            e(f"add.u32 {v}, {v}, {run};")
        run = o("shfl.sync.idx.b32", v, 31, 31, -1)
    return sums, run


def _first_behind(e, sums, start):
    """The first pair whose inclusive sum lies behind ``start``, and the sum before it."""
    o = e.o
    pair, before = o("mov.u32", 0), o("mov.u32", 0)
    for v in sums:
        past = e.cond("le.u32", v, start)
        e(f"add.u32 {pair}, {pair}, {o('popc.b32', o('vote.sync.ballot.b32', past, -1))};")
        e(f"max.u32 {before}, {before}, {o('redux.sync.max.u32', o('selp.u32', v, 0, past), -1)};")
    return pair, before


def paged_attention_entry(name, batch, chunk, heads, kv_heads, dim, pages, page, max_pages, dtype, quant, window, sinks,
                          scale, names, scratch, ctas, min_tiles=MIN_TILES, prefix="", sms=148):
    """The launch record and PTX; ``names``: Q, KC, VC, (KS, VS,) table, lens, fresh, O; ``scratch``: the parts'
    buffer, all their O rows and then their m and l."""
    D = dim
    group, tq, ntile, rows = geometry(chunk, heads, kv_heads)
    pairs = batch * ntile
    grid = ctas or pairs * kv_heads
    half = dtype == "f16" or quant           # the operands' type; in bf16 P comes in two parts
    p_f16 = half
    raw_b = BKV * D if quant else 0          # raw bytes of a K or V tile
    scan = not quant and min(tq, chunk) > 1  # rows of different positions share a V tile that may hold anything
    exp_mask = 0x7C00 if dtype == "f16" else 0x7F80
    row_b = D * 2
    q_bytes, q_box = ROWS * row_b, ROWS * 128
    kv_bytes, kv_box = BKV * row_b, BKV * 128
    boxes = D // 64
    cap = max_pages * page
    pieces = max(1, BKV // page)             # pages of a tile
    box_rows = min(page, BKV)
    if quant:
        threads, soft0, mma_warp = 256, 4, 1
    else:
        threads, soft0, mma_warp = 224, 2, 1
    idesc_qk = idesc_f16(ROWS, BKV, False, False, half=half)
    idesc_pv = idesc_f16(ROWS, D, False, True, half=p_f16)
    kdesc_hi = smem_desc_hi(16, 1024)
    vdesc_hi = smem_desc_hi(kv_box, 1024)
    cscale = _f32(scale * LOG2E)
    # one CTA a unit, more of them than the GPU holds at a time, of sequences that may differ
    order = not ctas and batch > 1 and pairs <= MAX_SPREAD_PAIRS and pairs * kv_heads > 2 * sms
    SCOL = D                                 # score buffers behind O's columns
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
    lens, fresh = gptr("p_lens"), gptr("p_fresh")

    def place(pair, ok=None):
        return _Place(e, pair, ok, lens, fresh, batch, chunk, group, tq, ntile, cap, window, sinks)

    def by_length(nth):
        """The pair with the nth most tiles, so that the longest units start first and no long one is left for the end:
        each thread counts how many come before its own."""
        keys, mine = o("mov.u32", f"{prefix}{name}_order"), []
        for k in range(-(-pairs // threads)):
            q = o("add.u32", tid, threads * k)
            ok = e.cond("lt.u32", q, pairs)
            key = o("min.u32", place(q, ok).tiles, (1 << 22) - 1)
            key = o("mad.lo.u32", key, 512, o("sub.u32", 2 * MAX_SPREAD_PAIRS - 1, q))      # ties: the earlier pair
            e(f"@{ok} st.shared.b32 [{o('mad.lo.u32', q, 4, keys)}], {key};")
            mine.append((q, ok, key, o("mov.u32", 0)))
        quads = -(-pairs // 4)
        pad = e.cond("lt.u32", tid, 4 * quads - pairs)
        e(f"@{pad} st.shared.b32 [{o('mad.lo.u32', tid, 4, keys)}+{4 * pairs}], {o('mov.b32', 0)};")
        e("bar.sync 0;")
        at_, last_, l_top = o("mov.u32", keys), o("add.u32", keys, 16 * quads), e.L("rank")
        e.label(l_top)
        x = [e.r() for _ in range(4)]
        e(f"ld.shared.v4.b32 {{{', '.join(x)}}}, [{at_}];")
        for _, _, key, rank in mine:
            for y in x:
                e(f"@{e.cond('gt.u32', y, key)} add.u32 {rank}, {rank}, 1;")
        e(f"add.u32 {at_}, {at_}, 16;")
        e(f"@{e.cond('lt.u32', at_, last_)} bra {l_top};")
        for q, ok, _, rank in mine:
            hit = e.cond("eq.u32", rank, nth)
            e(f"and.pred {hit}, {hit}, {ok};")
            e(f"@{hit} st.shared.b32 [{keys}+{4 * MAX_SPREAD_PAIRS}], {q};")
        e("bar.sync 0;")
        return o("ld.shared.b32", f"[{keys}+{4 * MAX_SPREAD_PAIRS}]")

    if ctas:
        e("griddepcontrol.launch_dependents;")                  # the join's blocks may come up and wait
        sums, run = _prefix(e, lane, pairs, lambda q, ok: place(q, ok).tiles, kv_heads)
        per = o("max.u32", o("div.u32", o("add.u32", run, ctas - 1), ctas), min_tiles)
        start = o("mul.lo.u32", cta, per)
        e(f"@{e.cond('ge.u32', start, run)} ret;")              # no tiles for this CTA
        stop = o("min.u32", o("add.u32", start, per), run)
        pair0, before0 = _first_behind(e, sums, start)
    else:
        kvh0, nth = o("rem.u32", cta, kv_heads), o("div.u32", cta, kv_heads)
        S0 = place(by_length(nth) if order else nth)
        e(f"@!{S0.live} ret;")                                  # a tile of padding

    class Segment:
        """One unit's share of the run, as a role sees it."""

        def __init__(self, P, kvh, i0, nb):
            self.P, self.w, self.kvh, self.i0, self.nb, self.b = P, P.w, kvh, i0, nb, P.b
            # first row of Q and O in [batch * chunk * heads, dim]
            r = o("mad.lo.u32", P.b, chunk, P.c0)
            self.base_row = o("mad.lo.u32", r, heads, o("mul.lo.u32", kvh, group))

        def row_index(self, r):
            """Row r of the unit as a row of Q and O: token r / group, head r % group."""
            if group == 1:
                return o("mad.lo.u32", r, heads, self.base_row)
            t_ = o("div.u32", r, group)
            return o("add.u32", o("mad.lo.u32", t_, heads, self.base_row), o("sub.u32", r, o("mul.lo.u32", t_, group)))

        def tile_of(self, j):
            """The key tile of the segment's tile number j."""
            i = o("add.u32", j, self.i0) if self.i0 is not None else j
            if window is None:
                return i
            past = e.cond("ge.u32", i, self.w["st"])
            return o("selp.u32", o("add.u32", i, self.w["gap"]), i, past)

    def each_segment(tag, body, out):
        """Emits ``body(segment)`` once, in a loop over the run's segments, and then a branch to ``out``."""
        if not ctas:
            body(Segment(S0, kvh0, None, S0.w["total"]))
            e(f"bra {out};")
            return
        pair, before, now = o("mov.u32", pair0), o("mov.u32", before0), o("mov.u32", start)
        l_find, l_seg = e.L(f"{tag}find"), e.L(f"{tag}seg")
        e.label(l_find)
        P = place(pair)
        behind = o("mad.lo.u32", P.tiles, kv_heads, before)
        e(f"@{e.cond('lt.u32', now, behind)} bra {l_seg};")
        e(f"mov.u32 {before}, {behind};")
        e(f"add.u32 {pair}, {pair}, 1;")
        e(f"bra {l_find};")
        e.label(l_seg)
        off = o("sub.u32", now, before)
        kvh = o("div.u32", off, P.tiles)
        i0 = o("sub.u32", off, o("mul.lo.u32", kvh, P.tiles))
        seg = Segment(P, kvh, i0, o("min.u32", o("sub.u32", P.tiles, i0), o("sub.u32", stop, now)))
        seg.now = now
        body(seg)
        e(f"add.u32 {now}, {now}, {seg.nb};")
        e(f"@{e.cond('lt.u32', now, stop)} bra {l_find};")
        e(f"bra {out};")

    if not ctas:
        # a unit that sees no key at all: its rows are 0
        l_some = e.L("some")
        e(f"@{e.cond('ne.u32', S0.w['total'], 0)} bra {l_some};")
        zs = Segment(S0, kvh0, None, None)
        zr, zero = o("mov.u32", tid), o("mov.u32", 0)
        l_z, l_zd = e.L("zero"), e.L("zerod")
        e.label(l_z)
        e(f"@{e.cond('ge.u32', zr, S0.vrows)} bra {l_zd};")
        za = at(o_ptr, wide(zs.row_index(zr), row_b))
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
    # bytes: two raw tiles, then one converted K and V
    sRaw = o("add.u32", sKV, 2 * kv_bytes) if quant else None
    bars = o("add.u32", sKV, 2 * kv_bytes + 4 * raw_b if quant else STAGES * kv_bytes)
    l_init = e.L("noinit")
    e(f"@{e.cond('ne.u32', tid, 0)} bra {l_init};")
    e(f"mbarrier.init.shared::cta.b64 [{bars}+{QFULL}], 4;")
    for s in range(STAGES):
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{FULL + 8 * s}], 1;")
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{EMPTY + 8 * s}], {2 if quant and s < 2 else 1};")
    for u in range(2):
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{SFULL + 8 * u}], 1;")
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{PFULL + 8 * u}], 4;")
        e(f"mbarrier.init.shared::cta.b64 [{bars}+{PFREE + 8 * u}], 1;")
        if not quant:
            e(f"mbarrier.init.shared::cta.b64 [{bars}+{VOK + 8 * u}], 1;")
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
    l_end, l_mma, l_soft, l_help = e.L("end"), e.L("mma"), e.L("soft"), e.L("help")
    e(f"@{p_mma} bra {l_mma};")
    if not quant:
        e(f"@{e.cond('eq.u32', warp, 6)} bra {l_help};")
    e(f"@{e.cond('ge.u32', warp, soft0)} bra {l_soft};")
    def valid(pg):
        return e.cond("lt.u32", pg, pages)

    # ------------------------------------------------------------------ loads
    l_conv = e.L("conv")
    if quant:
        e(f"@{e.cond('ge.u32', warp, 2)} bra {l_conv};")
    tk, tv = [o("cvta.param.u64", o("mov.u64", f"p_tm{x}", cls="rd"), cls="rd") for x in "KV"]
    table = gptr("p_table")
    if quant:
        ks_ptr, vs_ptr = gptr("p_KS"), gptr("p_VS")
    per_batch = 32 // pieces                                   # tiles whose pages one lane-load fetches
    sub = o("div.u32", lane, pieces) if pieces > 1 else lane
    piece = o("rem.u32", lane, pieces) if pieces > 1 else None
    cur, nxt = e.r(), e.r()
    p_l0, p_pc = e.cond("eq.u32", lane, 0), e.cond("lt.u32", lane, pieces)
    nfull = [o("mov.u32", 0) for _ in range(1 if quant else 2)]       # tiles loaded (16 bits: of K, of V)
    l_ldone = e.L("ldd")
    jj_ld = o("mov.u32", 0)                                    # the tile's number in the run

    def loads(S):
        trow = at(table, wide(S.b, 4 * max_pages))             # this sequence's row of the table

        def fetch(dst, j0):
            """Lane l: the page of piece l % pieces of tile j0 + l / pieces, or -1."""
            j = o("add.u32", j0, sub)
            ok = e.cond("lt.u32", j, S.nb)
            vt = S.tile_of(j)
            if pieces > 1:
                slot = o("mad.lo.u32", vt, pieces, piece)
            elif page == BKV:
                slot = vt
            else:
                slot = o("div.u32", vt, page // BKV)
            okm = e.cond("lt.u32", slot, max_pages)
            e(f"and.pred {ok}, {ok}, {okm};")
            a_ = at(trow, wide(slot, 4))
            e(f"mov.u32 {dst}, -1;")
            e(f"@{ok} ld.global.nc.u32 {dst}, [{a_}];")

        j, jj = o("mov.u32", 0), jj_ld
        fetch(cur, j)
        fetch(nxt, o("mov.u32", per_batch))
        l_u, l_seg = [e.L("ld0"), e.L("ld1")], e.L("ldseg")
        e(f"@{e.cond('ne.u32', o('and.b32', jj, 1), 0)} bra {l_u[1]};")
        for u in range(2):                                     # ring stages by the tile's parity
            e.label(l_u[u])
            e(f"@{e.cond('ge.u32', j, S.nb)} bra {l_seg};")
            ph = o("and.b32", o("shr.u32", jj, 1), 1)
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
            vt = S.tile_of(j)
            pgc = o("selp.b32", mine, -1, valid(mine))         # outside the pool: the box reads zeros
            roff = o("mul.lo.u32", o("rem.u32", vt, page // BKV), BKV) if page > BKV else 0
            ma = o("mad.lo.u32", o("and.b32", jj, 3), 8, bars)

            def arm(st_, nbytes, first, count):
                """Waits for ring stage st_, notes the mask words with a tile's first box, expects the bytes."""
                wait_bar_warp(e, f"{bars}+{EMPTY + 8 * st_}", o("xor.b32", ph, 1), err, ERR_LOAD, l_ldone)
                if first:
                    e(f"@{p_l0} st.shared.v2.b32 [{ma}+{KMASK}], {{{words[0]}, {words[1]}}};")
                e(f"@{p_l0} mbarrier.arrive.expect_tx.shared::cta.b64 _, [{bars}+{FULL + 8 * st_}], {nbytes};")
                e(f"add.u32 {count}, {count}, 1;")
                e("bar.warp.sync -1;")

            def box(tm, x, dst, st_):
                if pieces > 1:
                    dst = o("mad.lo.u32", piece, page * min(128, D if quant else row_b), dst)
                e(f"@{p_pc} cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                  f"[{dst}], [{tm}, {{{x}, {roff}, {S.kvh}, {pgc}}}], [{bars}+{FULL + 8 * st_}];")

            if quant:
                ok_ = valid(mine)
                here = o("and.b32", o("vote.sync.ballot.b32", ok_, -1), (1 << pieces) - 1)
                arm(u, o("mad.lo.u32", o("popc.b32", here), 2 * box_rows * 4, 2 * raw_b), True, nfull[0])
                e(f"and.pred {ok_}, {ok_}, {p_pc};")
                for kv, (tm, scp) in enumerate(((tk, ks_ptr), (tv, vs_ptr))):
                    box(tm, 0, o("add.u32", sRaw, (2 * u + kv) * raw_b), u)
                    first = o("mad.lo.u32", S.kvh, page, roff)
                    off = o("mad.wide.u32", mine, kv_heads * page * 4, wide(first, 4), cls="rd")
                    sd = o("add.u32", bars, RAWSC + (2 * u + kv) * BKV * 4)
                    if pieces > 1:
                        sd = o("mad.lo.u32", piece, page * 4, sd)
                    e(f"@{ok_} cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [{sd}], [{at(scp, off)}], "
                      f"{box_rows * 4}, [{bars}+{FULL + 8 * u}];")
            else:
                for kv, tm in enumerate((tk, tv)):
                    arm(2 * u + kv, kv_bytes, kv == 0, nfull[kv])
                    for h in range(boxes):
                        box(tm, 64 * h, o("add.u32", sKV, (2 * u + kv) * kv_bytes + h * kv_box), 2 * u + kv)
            e(f"add.u32 {j}, {j}, 1;")
            e(f"add.u32 {jj}, {jj}, 1;")
        e(f"bra {l_u[0]};")
        e.label(l_seg)

    each_segment("ld", loads, l_ldone)
    e.label(l_ldone)
    # wait for what is in flight: use k of a stage completes phase k - 1 (stage u has seen half the tiles)
    for kv in range(1 if quant else 2):
        for u in range(2):
            skip = e.L("nodrain")
            uses = o("shr.u32", o("add.u32", nfull[kv], 1 - u), 1)
            e(f"@{e.cond('eq.u32', uses, 0)} bra {skip};")
            wait_bar_warp(e, f"{bars}+{FULL + 8 * (u if quant else 2 * u + kv)}", o("and.b32", o("sub.u32", uses, 1), 1), err,
                          ERR_DRAIN, skip)
            e.label(skip)
    e(f"bra {l_end};")
    if quant:
        # ---------------------------------------------------------------- bytes to f16 (warps 2 and 3)
        e.label(l_conv)
        piece4, odd = o("and.b32", lane, 3), o("and.b32", o("shr.u32", lane, 2), 1)
        rlow = o("xor.b32", o("shl.b32", o("shr.u32", lane, 3), 1), o("mul.lo.u32", odd, 5))      # row within 8
        c64, c1152 = o("mov.b32", "0x64646464"), o("mov.b32", "0x64806480")
        if D == 128:                                            # 16-byte pieces by the row's low three bits
            raw_at = [o("mad.lo.u32", o("xor.b32", o("add.u32", piece4, 4 * h), rlow), 16, o("shl.b32", rlow, 7))
                      for h in range(2)]
        else:                                                   # 64-byte rows: by bits 1 and 2
            raw_at = [o("mad.lo.u32", o("xor.b32", piece4, o("and.b32", o("shr.u32", rlow, 1), 3)), 16,
                        o("shl.b32", rlow, 6))]
        out_at = [o("mad.lo.u32", o("xor.b32", o("mad.lo.u32", piece4, 2, i), rlow), 16, o("shl.b32", rlow, 7))
                  for i in range(2)]
        # warp 2 converts K, warp 3 V, each as far ahead as the products let it
        isv = o("sub.u32", warp, 2)
        raw_kv = o("mad.lo.u32", isv, raw_b, sRaw)
        out_kv = [o("mad.lo.u32", isv, kv_bytes, o("add.u32", sKV, x)) for x in out_at]
        kvb = o("mad.lo.u32", isv, 8, o("add.u32", bars, 16))   # K's and V's barriers behind the raw stages'
        p_l0c = e.cond("eq.u32", lane, 0)
        p_w2 = e.cond("eq.u32", warp, 2)
        jj_cv = o("mov.u32", 0)

        def convert(S):
            w = S.w
            vpow = o("mov.b32", "0x00800000")                      # the values' power of two (its f32 bits)
            j, jj = o("mov.u32", 0), jj_cv
            l_top, l_seg = e.L("cv"), e.L("cvseg")
            e.label(l_top)
            e(f"@{e.cond('ge.u32', j, S.nb)} bra {l_seg};")
            u_, ph, ph1 = o("and.b32", jj, 1), o("and.b32", o("shr.u32", jj, 1), 1), o("and.b32", jj, 1)
            rb = o("mad.lo.u32", u_, 8, bars)
            wait_bar_warp(e, f"{rb}+{FULL}", ph, err, ERR_LOAD, l_end)
            slot_c = o("and.b32", jj, 3)
            l_nosc = e.L("nosc")
            e(f"@!{p_w2} bra {l_nosc};")
            # warp 2: the tile's scales, two a lane; those of V over the power, which grows when one reaches twice it
            rs = o("mad.lo.u32", lane, 8, o("mad.lo.u32", u_, 2 * BKV * 4, bars))
            ksv, vsv = [e.r("f"), e.r("f")], [e.r("f"), e.r("f")]
            e(f"ld.shared.v2.f32 {{{ksv[0]}, {ksv[1]}}}, [{rs}+{RAWSC}];")
            e(f"ld.shared.v2.f32 {{{vsv[0]}, {vsv[1]}}}, [{rs}+{RAWSC + BKV * 4}];")
            key0c = o("mad.lo.u32", lane, 2, o("shl.b32", S.tile_of(j), 6))
            mw = o("mad.lo.u32", slot_c, 8, bars)
            mw = o("ld.shared.b32", f"[{o('mad.lo.u32', o('shr.u32', lane, 4), 4, mw)}+{KMASK}]")
            big = o("mov.b32", "0f00000000", cls="f")
            for i in range(2):
                bit = o("and.b32", o("shr.u32", mw, o("add.u32", o("shl.b32", o("and.b32", lane, 15), 1), i)), 1)
                kk = o("add.u32", key0c, i) if i else key0c
                pk2 = e.cond("lt.u32", kk, w["end"])
                pk1 = e.cond("ne.u32", bit, 0)
                e(f"and.pred {pk1}, {pk1}, {pk2};")
                if window is not None:                              # nor those that no row sees
                    p1, p2 = e.cond("ge.u32", kk, w["lo"]), e.cond("lt.u32", kk, sinks)
                    e(f"or.pred {p1}, {p1}, {p2};")
                    e(f"and.pred {pk1}, {pk1}, {p1};")
                e(f"@{pk1} max.f32 {big}, {big}, {o('abs.f32', vsv[i], cls='f')};")        # a NaN drops out
            bigb = o("redux.sync.max.u32", o("mov.b32", big), -1)
            bigb = o("min.u32", o("and.b32", bigb, "0x7F800000"), "0x7E000000")
            grow = e.cond("gt.u32", bigb, vpow)
            e(f"@{grow} mov.u32 {vpow}, {bigb};")
            vinv = o("mov.b32", o("sub.u32", "0x7F000000", vpow), cls="f")
            sd = o("mad.lo.u32", lane, 8, o("mad.lo.u32", slot_c, BKV * 4, bars))
            e(f"st.shared.v2.f32 [{sd}+{KSC}], {{{ksv[0]}, {ksv[1]}}};")
            v0, v1 = (o("mul.f32", x, vinv, cls="f") for x in vsv)
            e(f"st.shared.v2.f32 [{sd}+{VSC}], {{{v0}, {v1}}};")
            e(f"@{p_l0c} st.shared.b32 [{o('mad.lo.u32', slot_c, 4, bars)}+{VREF}], {vpow};")
            e.label(l_nosc)
            src = o("mad.lo.u32", u_, 2 * raw_b, raw_kv)
            for h in range(boxes):
                words = []
                for k in range(8):
                    d_ = [e.r() for _ in range(4)]
                    e(f"ld.shared.v4.b32 {{{', '.join(d_)}}}, [{o('add.u32', src, raw_at[h])}+{8 * k * D}];")
                    words.append(d_)
                if h == 0:
                    wait_bar_warp(e, f"{kvb}+{EMPTY}", o("xor.b32", ph1, 1), err, ERR_LOAD, l_end)
                for k in range(8):
                    out = [o("sub.rn.f16x2", o("prmt.b32", x, c64, sel), c1152)
                           for x in words[k] for sel in ("0x4140", "0x4342")]
                    for i in range(2):
                        e(f"st.shared.v4.b32 [{out_kv[i]}+{h * kv_box + 8 * k * 128}], "
                          f"{{{', '.join(out[4 * i:4 * i + 4])}}};")
            e("fence.proxy.async.shared::cta;")
            e("bar.warp.sync -1;")
            e(f"@{p_l0c} mbarrier.arrive.shared::cta.b64 _, [{rb}+{EMPTY}];")
            e(f"@{p_l0c} mbarrier.arrive.shared::cta.b64 _, [{kvb}+{FULL}];")
            e(f"add.u32 {j}, {j}, 1;")
            e(f"add.u32 {jj}, {jj}, 1;")
            e(f"bra {l_top};")
            e.label(l_seg)

        each_segment("cv", convert, l_end)

    else:
        # ---------------------------------------------------------------- V made fit for the product (warp 6)
        e.label(l_help)
        p_l0h = e.cond("eq.u32", lane, 0)
        jj_h = o("mov.u32", 0)
        # a lane takes a row's 16-byte pieces in an order of its own, so that eight lanes fill all banks
        piece = [o("xor.b32", o("shl.b32", o("and.b32", lane, 7), 4), 16 * i) for i in range(8)]

        def partial(S, key0):
            """Whether some rows of the unit see a key of the tile that others do not (the same for every thread): a
            row's own position lies in it, or a row's window begins in it and it is not all sinks."""
            p_ = e.cond("lt.s32", o("sub.s32", S.w["pos0"], key0), BKV - 1)
            if window is not None:
                p1 = e.cond("ge.s32", o("sub.s32", o("sub.s32", S.w["pos1"], window), key0), 0)
                p2 = e.cond("lt.s32", o("sub.s32", sinks, key0), BKV)
                e(f"and.pred {p1}, {p1}, {p2};")
                e(f"or.pred {p_}, {p_}, {p1};")
            return p_

        def help_(S):
            """Zeroes the rows of V that no row of the unit sees (past its last token, between sinks and window), and
            notes the rows that hold an infinity or a NaN where some rows see a key and others do not."""
            j, jj = o("mov.u32", 0), jj_h
            l_top, l_seg = e.L("hp"), e.L("hpseg")
            e.label(l_top)
            e(f"@{e.cond('ge.u32', j, S.nb)} bra {l_seg};")
            u_, ph = o("and.b32", jj, 1), o("and.b32", o("shr.u32", jj, 1), 1)
            key0 = o("shl.b32", S.tile_of(j), 6)
            bad = [o("mov.b32", 0), o("mov.b32", 0)]
            l_vok, l_clean = e.L("vok"), e.L("clean")
            sb = o("mad.lo.u32", u_, 16, bars)
            wait_bar_warp(e, f"{sb}+{FULL + 8}", ph, err, ERR_LOAD, l_end)
            va = o("mad.lo.u32", u_, 2 * kv_bytes, o("add.u32", sKV, kv_bytes))
            vlim = o("sub.s32", S.w["pos1"], key0)
            pv_ = e.cond("ge.s32", vlim, BKV - 1)
            if window is not None:
                lo_k, sk = o("sub.s32", S.w["lo"], key0), o("sub.s32", sinks, key0)
                p1_, p2_ = e.cond("le.s32", lo_k, 0), e.cond("ge.s32", sk, BKV)
                e(f"or.pred {p1_}, {p1_}, {p2_};")
                e(f"and.pred {pv_}, {pv_}, {p1_};")
            e(f"@{pv_} bra {l_vok};")
            z_ = o("mov.b32", 0)
            for h in range(2):
                r_ = o("add.u32", lane, 32 * h)
                pz = e.cond("gt.s32", r_, vlim)
                if window is not None:
                    pa, pb = e.cond("lt.s32", r_, lo_k), e.cond("ge.s32", r_, sk)
                    e(f"and.pred {pa}, {pa}, {pb};")
                    e(f"or.pred {pz}, {pz}, {pa};")
                ra = o("mad.lo.u32", r_, 128, va)
                for i in range(8):
                    pa_ = o("add.u32", ra, piece[i])
                    for box in range(boxes):
                        e(f"@{pz} st.shared.v4.b32 [{pa_}+{box * kv_box}], {{{z_}, {z_}, {z_}, {z_}}};")
            e("fence.proxy.async.shared::cta;")
            e.label(l_vok)
            if scan:
                e(f"@!{partial(S, key0)} bra {l_clean};")
                for h in range(2):
                    ra = o("mad.lo.u32", o("add.u32", lane, 32 * h), 128, va)
                    m_ = None
                    for i in range(8):
                        pa_ = o("add.u32", ra, piece[i])
                        for box in range(boxes):
                            d_ = [e.r() for _ in range(4)]
                            e(f"ld.shared.v4.b32 {{{', '.join(d_)}}}, [{pa_}+{box * kv_box}];")
                            for x in d_:
                                x = o("and.b32", x, "0x7FFF7FFF")
                                m_ = x if m_ is None else o("max.u16x2", m_, x)
                    m_ = o("max.u32", o("and.b32", m_, 65535), o("shr.u32", m_, 16))
                    e(f"vote.sync.ballot.b32 {bad[h]}, {e.cond('ge.u32', m_, exp_mask)}, -1;")
                e.label(l_clean)
                e(f"@{p_l0h} st.shared.v2.b32 [{o('mad.lo.u32', u_, 8, bars)}+{VBAD}], {{{bad[0]}, {bad[1]}}};")
            e("bar.warp.sync -1;")
            e(f"@{p_l0h} mbarrier.arrive.shared::cta.b64 _, [{o('mad.lo.u32', u_, 8, bars)}+{VOK}];")
            e(f"add.u32 {j}, {j}, 1;")
            e(f"add.u32 {jj}, {jj}, 1;")
            e(f"bra {l_top};")
            e.label(l_seg)

        each_segment("h", help_, l_end)

    # ------------------------------------------------------------------ MMA issue (one thread)
    e.label(l_mma)
    e(f"@{e.cond('ne.u32', lane, 0)} bra {l_end};")
    iqk, ipv = o("mov.u32", idesc_qk), o("mov.u32", idesc_pv)
    ptrue, pfalse = e.cond("eq.u32", lane, lane), e.cond("ne.u32", lane, lane)
    khi, vhi = o("mov.b64", kdesc_hi, cls="rd"), o("mov.b64", vdesc_hi, cls="rd")

    def desc(addr, hi):
        return o("or.b64", o("cvt.u64.u32", o("shr.u32", addr, 4), cls="rd"), hi, cls="rd")

    def plus(d0, off):
        return o("add.s64", d0, off >> 4, cls="rd") if off else d0

    q0 = desc(sQ, khi)
    qd = [plus(q0, (k // 4) * q_box + (k % 4) * 32) for k in range(D // 16)]
    ring_k, ring_v = ([2, 2], [3, 3]) if quant else ([0, 2], [1, 3])         # barriers of a tile's K and V by its parity
    stg = [o("add.u32", sKV, s * kv_bytes) for s in range(2 if quant else STAGES)]
    kd = [desc(stg[0 if quant else 2 * u], khi) for u in range(2)]
    vd = [desc(stg[1 if quant else 2 * u + 1], vhi) for u in range(2)]
    scol = [o("add.u32", taddr, SCOL + BKV * u) for u in range(2)]

    def commit(off):
        e(f"tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [{bars}+{off}];")

    def ring(st_, ph):
        wait_bar(e, f"{bars}+{FULL + 8 * st_}", ph, err, ERR_MMA, l_end)
        e("tcgen05.fence::after_thread_sync;")

    def qk(u):
        for k in range(D // 16):
            e(f"tcgen05.mma.cta_group::1.kind::f16 [{scol[u]}], {qd[k]}, {plus(kd[u], (k // 4) * kv_box + (k % 4) * 32)}, "
              f"{iqk}, {ptrue if k else pfalse};")
        commit(EMPTY + 8 * ring_k[u])
        commit(SFULL + 8 * u)

    jj_m, segs = o("mov.u32", 0), o("mov.u32", 0)

    def clear(tile_addr, bad):
        """Writes 0 over the infinities and NaNs of the V tile's rows ``bad`` (two words; one thread, a rare path)."""
        row, end_ = o("mov.u32", 0), o("mov.u32", BKV)
        l_r, l_c, l_n, l_d = e.L("clr"), e.L("clrc"), e.L("clrn"), e.L("clrd")
        e.label(l_r)
        e(f"@{e.cond('ge.u32', row, end_)} bra {l_d};")
        word = o("selp.b32", bad[0], bad[1], e.cond("lt.u32", row, 32))
        bit = o("and.b32", o("shr.u32", word, o("and.b32", row, 31)), 1)
        e(f"@{e.cond('eq.u32', bit, 0)} bra {l_n};")
        a_ = o("mad.lo.u32", row, 128, tile_addr)
        k_ = o("mov.u32", 0)
        e.label(l_c)
        for box in range(boxes):
            x = o("ld.shared.b32", f"[{a_}+{box * kv_box}]")
            lo_, hi_ = o("and.b32", x, 0x7FFF), o("and.b32", x, 0x7FFF0000)
            e(f"@{e.cond('ge.u32', lo_, exp_mask)} and.b32 {x}, {x}, -65536;")
            e(f"@{e.cond('ge.u32', hi_, exp_mask << 16)} and.b32 {x}, {x}, 65535;")
            e(f"st.shared.b32 [{a_}+{box * kv_box}], {x};")
        e(f"add.u32 {a_}, {a_}, 4;")
        e(f"add.u32 {k_}, {k_}, 1;")
        e(f"@{e.cond('lt.u32', k_, 32)} bra {l_c};")
        e.label(l_n)
        e(f"add.u32 {row}, {row}, 1;")
        e(f"bra {l_r};")
        e.label(l_d)

    def phase_of(x):
        """The phase of a ring barrier at tile x of the run: of two stages, or of one (bytes: the tile's parity)."""
        return o("and.b32", x if quant else o("shr.u32", x, 1), 1)

    def issue(S):
        j, jj = o("mov.u32", 0), jj_m
        wait_bar(e, f"{bars}+{QFULL}", o("and.b32", segs, 1), err, ERR_MMA, l_end)
        e("tcgen05.fence::after_thread_sync;")
        e(f"add.u32 {segs}, {segs}, 1;")
        l_in, l_u, l_seg = [e.L("in0"), e.L("in1")], [e.L("mg0"), e.L("mg1")], e.L("mseg")
        e(f"@{e.cond('ne.u32', o('and.b32', jj, 1), 0)} bra {l_in[1]};")
        for u in range(2):
            e.label(l_in[u])
            ring(ring_k[u], phase_of(jj))
            qk(u)
            e(f"bra {l_u[u]};")
        for u in range(2):                                     # a tile of parity u
            e.label(l_u[u])
            jn, jjn = o("add.u32", j, 1), o("add.u32", jj, 1)
            have = e.cond("lt.u32", jn, S.nb)
            l_nok = e.L("nok")
            e(f"@!{have} bra {l_nok};")
            ring(ring_k[1 - u], phase_of(jjn))
            qk(1 - u)
            e.label(l_nok)
            ring(ring_v[u], phase_of(jj))
            if not quant:
                wait_bar(e, f"{bars}+{VOK + 8 * u}", phase_of(jj), err, ERR_MMA, l_end)
            wait_bar(e, f"{bars}+{PFULL + 8 * u}", o("and.b32", o("shr.u32", jj, 1), 1), err, ERR_MMA, l_end)
            e("tcgen05.fence::after_thread_sync;")
            pacc = e.cond("ne.u32", j, 0)
            if scan:
                bad = [e.r(), e.r()]
                e(f"ld.shared.v2.b32 {{{bad[0]}, {bad[1]}}}, [{bars}+{VBAD + 8 * u}];")
                l_fine = e.L("fine")
                any_ = o("or.b32", bad[0], bad[1])
                e(f"@{e.cond('eq.u32', any_, 0)} bra {l_fine};")
                clear(stg[2 * u + 1], bad)
                e("fence.proxy.async.shared::cta;")
                e(f"setp.eq.u32 {pacc}, {lane}, {lane};")       # O holds what the rows added, also before the first product
                e.label(l_fine)
            for part in range(1 if p_f16 else 2):
                for k in range(BKV // 16):
                    e(f"tcgen05.mma.cta_group::1.kind::f16 [{taddr}], [{scol[u]}+{BKV // 2 * part + 8 * k}], "
                      f"{plus(vd[u], 2048 * k)}, {ipv}, {pacc if k == 0 and part == 0 else ptrue};")
            commit(EMPTY + 8 * ring_v[u])
            commit(PFREE + 8 * u)
            e(f"mov.u32 {j}, {jn};")
            e(f"mov.u32 {jj}, {jjn};")
            e(f"@!{have} bra {l_seg};")
        e(f"bra {l_u[0]};")
        e.label(l_seg)

    each_segment("m", issue, l_end)

    # ------------------------------------------------------------------ softmax (one row a thread)
    e.label(l_soft)
    quad = o("and.b32", warp, 3)                               # the TMEM lanes a warp reaches
    rowl = o("mad.lo.u32", quad, 32, lane)
    q_ptr = gptr("p_Q")
    per_row = row_b // 16                                      # lanes a row takes
    qsub, qch = o("div.u32", lane, per_row), o("rem.u32", lane, per_row)
    passes = 32 * per_row // 32
    recast = quant and dtype == "bf16"
    p_l0s = e.cond("eq.u32", lane, 0)
    lanebase = o("add.u32", o("shl.b32", quad, 21), taddr)
    s_ = [e.r("f") for _ in range(BKV)]
    jj_s = o("mov.u32", 0)
    out_cvt = "cvt.rn.f16x2.f32" if dtype == "f16" else "cvt.rn.bf16x2.f32"
    lift = lift_of(dtype, quant)
    out_lift = -RESCALE if quant else lift                     # of the parts: weights of at most 1 before vref comes in

    def add_specials(S, j, jj, buf, ph, key0, *rest):
        """Tiles in which a key is seen by some rows only: takes the rare path when the V rows hold an infinity or a NaN.
        Returns what emits that path, behind the loop: it adds them to O for the rows that see them; it borrows the
        scores' registers and loads them again."""
        l_out, l_rare = e.L("clean"), e.L("rare")
        e(f"@!{partial(S, key0)} bra {l_out};")
        wait_bar_warp(e, f"{o('mad.lo.u32', buf, 8, bars)}+{VOK}", ph, err, ERR_SOFTMAX, l_end)
        bad = [e.r(), e.r()]
        e(f"ld.shared.v2.b32 {{{bad[0]}, {bad[1]}}}, [{o('mad.lo.u32', buf, 8, bars)}+{VBAD}];")
        e(f"@{e.cond('ne.u32', o('or.b32', bad[0], bad[1]), 0)} bra {l_rare};")
        e.label(l_out)
        return lambda: rare(S, j, jj, buf, *rest, bad, l_rare, l_out)

    def rare(S, j, jj, buf, seen, pv_done, load_scores, bad, l_rare, l_out):
        e.label(l_rare)
        va = o("mad.lo.u32", buf, 2 * kv_bytes, o("add.u32", sKV, kv_bytes))
        # O is this warp's to change between the previous product and this tile's; before the first it is 0
        l_old, l_have = e.L("oldo"), e.L("haveo")
        zf = o("mov.b32", 0)
        e(f"@{e.cond('ne.u32', j, 0)} bra {l_old};")
        for c in range(D // 32):
            e(f"tcgen05.st.sync.aligned.32x32b.x32.b32 [{lanebase}+{32 * c}], {{{', '.join([zf] * 32)}}};")
        e("tcgen05.wait::st.sync.aligned;")
        e(f"bra {l_have};")
        e.label(l_old)
        pv_done(o("sub.u32", jj, 1), ERR_SOFTMAX, l_end)
        e("tcgen05.fence::after_thread_sync;")
        e.label(l_have)
        row = o("mov.u32", 0)
        l_r, l_n = e.L("sp"), e.L("spn")
        e.label(l_r)
        low = e.cond("lt.u32", row, 32)
        sh = o("and.b32", row, 31)
        bit = o("and.b32", o("shr.u32", o("selp.b32", bad[0], bad[1], low), sh), 1)
        e(f"@{e.cond('eq.u32', bit, 0)} bra {l_n};")            # the same for the warp
        mine = e.cond("ne.u32", o("and.b32", o("shr.u32", o("selp.b32", seen[0], seen[1], low), sh), 1), 0)
        col, sw = o("mov.u32", 0), o("and.b32", row, 7)
        l_c = e.L("spc")
        e.label(l_c)                                            # 32 columns at a time
        oc = o("add.u32", lanebase, col)
        regs = s_[:32]
        e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(regs)}}}, [{oc}];")
        e("tcgen05.wait::ld.sync.aligned;")
        ra = o("mad.lo.u32", row, 128, va)
        ra = o("mad.lo.u32", o("shr.u32", col, 6), kv_box, ra)
        first = o("and.b32", o("shr.u32", col, 3), 7)           # 16-byte pieces of the 64-column box
        for i in range(4):
            d_ = [e.r() for _ in range(4)]
            pa_ = o("mad.lo.u32", o("xor.b32", o("add.u32", first, i), sw), 16, ra)
            e(f"ld.shared.v4.b32 {{{', '.join(d_)}}}, [{pa_}];")
            for k, x in enumerate(d_):
                for h in range(2):
                    mag = o("and.b32", x, 0x7FFF << (16 * h))
                    p_ = e.cond("ge.u32", mag, exp_mask << (16 * h))
                    e(f"and.pred {p_}, {p_}, {mine};")
                    # an infinity or a NaN as f32: the same sign and kind
                    if dtype == "bf16":
                        f_ = o("shl.b32", x, 16) if h == 0 else o("and.b32", x, -65536)
                    else:
                        sign = o("shl.b32", o("and.b32", x, 0x8000), 16) if h == 0 else o("and.b32", x, -(1 << 31))
                        frac = o("shl.b32", o("and.b32", x, 0x3FF), 13) if h == 0 else o("shr.u32", o("and.b32", x,
                                                                                                    0x3FF0000), 3)
                        f_ = o("or.b32", o("or.b32", sign, 0x7F800000), frac)
                    e(f"@{p_} add.f32 {regs[8 * i + 2 * k + h]}, {regs[8 * i + 2 * k + h]}, {o('mov.b32', f_, cls='f')};")
        e(f"tcgen05.st.sync.aligned.32x32b.x32.b32 [{oc}], {{{', '.join(regs)}}};")
        e("tcgen05.wait::st.sync.aligned;")
        e(f"add.u32 {col}, {col}, 32;")
        e(f"@{e.cond('lt.u32', col, D)} bra {l_c};")
        e.label(l_n)
        e(f"add.u32 {row}, {row}, 1;")
        e(f"@{e.cond('lt.u32', row, BKV)} bra {l_r};")
        load_scores()
        e("tcgen05.wait::ld.sync.aligned;")
        e(f"bra {l_out};")

    def softmax(S):
        w, pos0, pos1, vrows = S.w, S.w["pos0"], S.w["pos1"], S.P.vrows
        # Q: each warp its own 32 rows, 16 bytes a lane, into the swizzled K-major tile
        for p0 in range(0, passes, 8):
            ws, rr_ = [], []
            for p_ in range(p0, min(passes, p0 + 8)):
                r_ = o("mad.lo.u32", quad, 32, o("add.u32", qsub, p_ * (32 // per_row)))
                ok = e.cond("lt.u32", r_, vrows)
                qa = at(at(q_ptr, wide(S.row_index(r_), row_b)), wide(qch, 16))
                d_ = [o("mov.b32", 0) for _ in range(4)]
                e(f"@{ok} ld.global.nc.v4.b32 {{{', '.join(d_)}}}, [{qa}];")
                ws.append(d_)
                rr_.append(r_)
            for d_, r_ in zip(ws, rr_):
                if recast:
                    # the row's largest number to 2^14 by a power of two, then f16: see above
                    big = None
                    for x in d_:
                        a_ = o("and.b32", x, "0x7FFF7FFF")
                        big = a_ if big is None else o("max.u16x2", big, a_)
                    big = o("max.u32", o("and.b32", big, 65535), o("shr.u32", big, 16))
                    k_ = 1
                    while k_ < per_row:
                        big = o("max.u32", big, o("shfl.sync.bfly.b32", big, k_, 31, -1))
                        k_ *= 2
                    ex = o("min.s32", o("sub.s32", 127 + 14, o("shr.u32", big, 7)), q_most(scale))
                    up = o("shl.b32", o("add.s32", ex, 127), 23, cls="f")
                    down = o("shl.b32", o("sub.s32", 127, ex), 23, cls="f")
                    qsa = o("mad.lo.u32", r_, 4, bars)
                    e(f"@{e.cond('eq.u32', qch, 0)} st.shared.f32 [{qsa}+{QSC}], {o('mul.f32', down, cscale, cls='f')};")
                    d_ = [o("cvt.rn.f16x2.f32", o("mul.f32", o("and.b32", x, -65536, cls="f"), up, cls="f"),
                            o("mul.f32", o("shl.b32", x, 16, cls="f"), up, cls="f")) for x in d_]
                box = o("shr.u32", qch, 3)
                ch = o("xor.b32", o("and.b32", qch, 7), o("and.b32", r_, 7))
                sa = o("mad.lo.u32", box, q_box, sQ)
                sa = o("mad.lo.u32", r_, 128, sa)
                sa = o("mad.lo.u32", ch, 16, sa)
                e(f"st.shared.v4.b32 [{sa}], {{{', '.join(d_)}}};")
        e("fence.proxy.async.shared::cta;")
        e("bar.warp.sync -1;")
        e(f"@{p_l0s} mbarrier.arrive.shared::cta.b64 _, [{bars}+{QFULL}];")
        tok = o("div.u32", rowl, group) if group > 1 else rowl
        pos = o("min.s32", o("add.s32", pos0, tok), pos1)          # rows without a token: the last one's
        cf = o("mov.b32", cscale, cls="f")                          # scale * log2(e) for this row's scores
        if recast:
            e(f"ld.shared.f32 {cf}, [{o('mad.lo.u32', rowl, 4, bars)}+{QSC}];")
        vref = o("mov.b32", "0f00800000", cls="f") if quant else None
        mref, lsum = o("mov.b32", "0fFF800000", cls="f"), o("mov.b32", "0f00000000", cls="f")
        j, jj = o("mov.u32", 0), jj_s
        l_sj, l_sdone, l_noepi = e.L("sj"), e.L("sdone"), e.L("noepi")

        def pv_done(k, code, bail):
            br = o("mad.lo.u32", o("and.b32", k, 1), 8, bars)
            wait_bar_warp(e, f"{br}+{PFREE}", o("and.b32", o("shr.u32", k, 1), 1), err, code, bail)

        e.label(l_sj)
        e(f"@{e.cond('ge.u32', j, S.nb)} bra {l_sdone};")
        buf = o("and.b32", jj, 1)
        ph = o("and.b32", o("shr.u32", jj, 1), 1)
        bb = o("mad.lo.u32", buf, 8, bars)
        sc_col = o("add.u32", o("mad.lo.u32", buf, BKV, lanebase), SCOL)
        key0 = o("shl.b32", S.tile_of(j), 6)
        wait_bar_warp(e, f"{bb}+{SFULL}", ph, err, ERR_SOFTMAX, l_end)
        e("tcgen05.fence::after_thread_sync;")

        def load_scores():
            for c in range(BKV // 32):
                e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(s_[32 * c:32 * c + 32])}}}, [{sc_col}+{32 * c}];")

        load_scores()
        slot_a = o("and.b32", jj, 3)
        ma = o("mad.lo.u32", slot_a, 8, bars)
        km = [e.r(), e.r()]
        e(f"ld.shared.v2.b32 {{{km[0]}, {km[1]}}}, [{ma}+{KMASK}];")
        e("tcgen05.wait::ld.sync.aligned;")
        sca = None
        if quant:
            sca = o("mad.lo.u32", slot_a, BKV * 4, bars)
            vnew = o("ld.shared.f32", f"[{o('mad.lo.u32', slot_a, 4, bars)}+{VREF}]", cls="f")

            def times(off):
                """The row times 64 numbers in shared memory, two at a time."""
                for c in range(0, BKV, 4):
                    kp = [e.r("rd"), e.r("rd")]
                    e(f"ld.shared.v2.b64 {{{kp[0]}, {kp[1]}}}, [{sca}+{off + 4 * c}];")
                    for i in range(2):
                        x0, x1 = s_[c + 2 * i], s_[c + 2 * i + 1]
                        xp = e.r("rd")
                        e(f"mov.b64 {xp}, {{{x0}, {x1}}};")
                        e(f"mul.rn.f32x2 {xp}, {xp}, {kp[i]};")
                        e(f"mov.b64 {{{x0}, {x1}}}, {xp};")
            times(KSC)
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
        e.label(l_seen)
        if scan:
            out_of_line = add_specials(S, j, jj, buf, ph, key0, (m0, m1), pv_done, load_scores)
        l_kept = e.L("kept")
        e(f"@{v_all} bra {l_kept};")
        for c in range(BKV):
            t_ = o("and.b32", (m0, m1)[c // 32], 1 << (c % 32) if c % 32 < 31 else -(1 << 31))
            e(f"@{e.cond('eq.u32', t_, 0)} mov.b32 {s_[c]}, 0fFF800000;")
        e.label(l_kept)
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
        mnew = o("max.f32", mref, o("mul.f32", lvl[0], cf, cls="f"), cls="f")
        alpha = o("mov.b32", "0f3F800000", cls="f")
        l_first, l_after = e.L("first"), e.L("after")
        anyneed = e.cond("ne.u32", lane, lane)
        e(f"@{e.cond('eq.u32', j, 0)} bra {l_first};")
        need = e.cond("gt.f32", mnew, o("add.f32", mref, _f32(RESCALE), cls="f"))
        if quant:
            e(f"or.pred {need}, {need}, {e.cond('ne.f32', vnew, vref)};")           # the same for every row
        e(f"vote.sync.any.pred {anyneed}, {need}, -1;")
        e(f"@!{anyneed} bra {l_after};")
        e(f"ex2.approx.ftz.f32 {alpha}, {o('sub.f32', mref, mnew, cls='f')};")
        # a row that has seen nothing yet while another of the warp rescales: -inf - -inf must not make a NaN
        e(f"@{e.cond('eq.f32', mnew, '0fFF800000')} mov.b32 {alpha}, 0f3F800000;")
        e(f"mul.f32 {lsum}, {lsum}, {alpha};")
        if quant:
            inv_ = o("mov.b32", o("sub.u32", "0x7F000000", o("mov.b32", vnew)), cls="f")
            e(f"mul.f32 {alpha}, {alpha}, {o('mul.f32', vref, inv_, cls='f')};")
        e.label(l_first)
        e(f"mov.b32 {mref}, {mnew};")
        if quant:
            e(f"mov.b32 {vref}, {vnew};")
        e.label(l_after)
        negm = o("sub.f32", o("mov.b32", _f32(lift), cls="f"), mref, cls="f")
        e(f"@{e.cond('eq.f32', mref, '0fFF800000')} mov.b32 {negm}, 0f00000000;")
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
            def pack(cols):
                hw = [o("cvt.rn.f16x2.f32", s_[c + 1], s_[c]) for c in cols[::2]]
                e(f"tcgen05.st.sync.aligned.32x32b.x16.b32 [{sc_col}+{cols[0] // 2}], {{{', '.join(hw)}}};")
            if quant:
                exps(list(range(BKV)))
                times(VSC)
                # a masked key's scale may be NaN: its weight is 0 whatever it was multiplied by
                l_nz = e.L("nz")
                e(f"@{v_all} bra {l_nz};")
                for c in range(BKV):
                    t_ = o("and.b32", (m0, m1)[c // 32], 1 << (c % 32) if c % 32 < 31 else -(1 << 31))
                    e(f"@{e.cond('eq.u32', t_, 0)} mov.b32 {s_[c]}, 0f00000000;")
                e.label(l_nz)
            for h in range(2):
                cols = list(range(32 * h, 32 * h + 32))
                if not quant:
                    exps(cols)
                pack(cols)
        else:
            exps(list(range(BKV)))
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

        pv_done(o("sub.u32", jj, 1), ERR_SOFTMAX, l_end)
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
        e(f"add.u32 {jj}, {jj}, 1;")
        e(f"bra {l_sj};")
        if scan:
            out_of_line()

        # epilogue: after the last product, O / l as the output type, or the part's O, m and l in f32
        e.label(l_sdone)
        pv_done(o("sub.u32", jj, 1), ERR_EPILOGUE, l_end)
        e("tcgen05.fence::after_thread_sync;")
        p_row = e.cond("lt.u32", rowl, vrows)
        l_part = e.L("part")
        if ctas:
            e(f"@{e.cond('ne.u32', S.nb, S.P.tiles)} bra {l_part};")            # the unit has other runs too
        p_zero = e.cond("eq.f32", lsum, "0f00000000")
        inv = o("rcp.rn.f32", o("selp.f32", "0f3F800000", lsum, p_zero, cls="f"), cls="f")
        oa = at(o_ptr, wide(S.row_index(rowl), row_b))
        for c in range(D // 32):
            regs = s_[:32]
            e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(regs)}}}, [{lanebase}+{32 * c}];")
            e("tcgen05.wait::ld.sync.aligned;")
            words = []
            for k in range(16):
                x0 = o("mul.f32", regs[2 * k], inv, cls="f")
                x1 = o("mul.f32", regs[2 * k + 1], inv, cls="f")
                if quant:                                       # not inv * vref: that may fall below f32's normal numbers
                    x0, x1 = o("mul.f32", x0, vref, cls="f"), o("mul.f32", x1, vref, cls="f")
                words.append(o("selp.b32", 0, o(out_cvt, x1, x0), p_zero))
            for i in range(2):
                e(f"@{p_row} st.global.v8.b32 [{oa}+{64 * c + 32 * i}], {{{', '.join(words[8 * i:8 * i + 8])}}};")
        if ctas:
            e(f"bra {l_noepi};")
            e.label(l_part)
            # a CTA's first segment leaves part 2 c, a later one 2 c + 1
            part = o("add.u32", o("shl.b32", cta, 1), o("selp.u32", 1, 0, e.cond("ne.u32", S.now, start)))
            pi = o("mad.lo.u32", part, rows, rowl)
            pa = at(gptr("p_part"), wide(pi, D * 4))
            if quant:
                vout = o("mul.f32", vref, _f32(2.0 ** (out_lift - lift)), cls="f")
                e(f"mul.f32 {lsum}, {lsum}, {_f32(2.0 ** (out_lift - lift))};")
            for c in range(D // 32):
                regs = s_[:32]
                e(f"tcgen05.ld.sync.aligned.32x32b.x32.b32 {{{', '.join(regs)}}}, [{lanebase}+{32 * c}];")
                e("tcgen05.wait::ld.sync.aligned;")
                if quant:
                    for x in regs:
                        e(f"mul.f32 {x}, {x}, {vout};")
                for i in range(4):
                    e(f"@{p_row} st.global.v8.f32 [{pa}+{128 * c + 32 * i}], {{{', '.join(regs[8 * i:8 * i + 8])}}};")
            mla = at(at(gptr("p_part"), 2 * ctas * rows * D * 4), wide(pi, 8))
            # the parts' O and l stand for 2^-negm; a part that saw nothing has m = -inf
            meff = o("sub.f32", mref, _f32(out_lift), cls="f")
            e(f"@{p_row} st.global.v2.f32 [{mla}], {{{meff}, {lsum}}};")
        e.label(l_noepi)

    each_segment("s", softmax, l_end)

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
        params = [("Q", qn, 16), ("KC", kn, 16), ("VC", vn, 16), ("KS", ksn, 16), ("VS", vsn, 16)]
    else:
        qn, kn, vn, tn, ln, fn, on = names
        params = [("Q", qn, 16), ("KC", kn, 16), ("VC", vn, 16)]
    params += [("table", tn, 4), ("lens", ln, 4), ("fresh", fn, 4), ("O", on, 32)]
    sc_spec = []
    if ctas:
        params += [("part", scratch, 32)]
        sc_spec = [{"name": scratch, "dtype": "f32", "shape": [2 * ctas * rows, D + 2], "per_call": True}]
    es = 1 if quant else 2
    span = min(128, D * es)                                     # a box row, and the swizzle
    tmaps = [{"name": f"tm{x}", "tensor": nm, "dtype": "u8" if quant else dtype, "dims": [D, page, kv_heads, pages],
              "strides": [D * es, page * D * es, kv_heads * page * D * es], "box": [span // es, box_rows, 1, 1],
              "swizzle": f"{span}B"} for x, nm in (("K", kn), ("V", vn))]
    plist = [f"\t.param .u64 p_{p}" for p, _, _ in params]
    plist += [f"\t.param .align 64 .b8 p_{t['name']}[128]" for t in tmaps] + ["\t.param .u64 p_err"]
    text = [f".visible .entry {name}(", ",\n".join(plist), ")", f".reqntid {threads}, 1, 1",
            f".maxnreg {65536 // (2 * -(-threads // 128) * 128) // 8 * 8}", "{"]
    text += e.decls() + e.lines + ["\tret;", "}"]
    return {
        "name": name, "kind": "tcgen05_paged_attention", "params": [n for _, n, _ in params],
        "raw_entry": text, "raw_decls": [f".extern .shared .align 1024 .b8 {smem_sym}[];",
                                        *([f".shared .align 16 .b8 {prefix}{name}_order[{4 * MAX_SPREAD_PAIRS + 16}];"] if order else [])],
        "grid": [grid, 1, 1], "block": [threads, 1, 1],
        "dyn_smem": q_bytes + (2 * kv_bytes + 4 * raw_b + AUX_BYTES if quant else STAGES * kv_bytes + KSC) + 1024,
        "align": {n: a_ for _, n, a_ in params}, "zero_outputs": [], "tmaps": tmaps,
        "extra": [{"name": "__err", "kind": "errword"}], "scratch": sc_spec,
    }


def join_entry(name, batch, chunk, heads, kv_heads, dim, page, max_pages, dtype, window, sinks, names, scratch, ctas,
               min_tiles=MIN_TILES):
    """The second entry: the rows of units of more than one run, o = sum_s 2^(m_s - m) O_s / sum_s 2^(m_s - m) l_s.  A
    block for every cut between two runs: it finds by the same prefix sums the unit that the cut lies in, and the unit's
    cuts share its rows.  Units of one run are written already; warps of more blocks look at a unit each and write 0
    where it sees no key at all (no run covers it).  Bound by the latency of its loads, so a warp has eight of them in
    flight, under a running maximum: two parts of four rows, or eight of one where there are many parts.  2 x
    2048 tokens over 8192 keys (295 cuts, parts of 64 KiB): 14 us, 37 by a block a unit and a row of a warp at a time; one
    sequence of 5000 tokens in 79 parts: 6 us, 16 where one block joined a unit."""
    D = dim
    group, tq, ntile, rows = geometry(chunk, heads, kv_heads)
    pairs, cuts = batch * ntile, ctas - 1
    per_lane = D // 32
    threads = 512
    e = _E()
    o = e.o

    def gptr(pname):
        return o("cvta.to.global.u64", o("ld.param.u64", f"[{pname}]", cls="rd"), cls="rd")

    def at(base, x, n):
        return o("add.s64", base, o("mul.wide.u32", x, n, cls="rd"), cls="rd")

    tid = o("mov.u32", "%tid.x")
    warp, lane = o("shr.u32", tid, 5), o("and.b32", tid, 31)
    e("griddepcontrol.wait;")                                   # the parts are written
    cta = o("mov.u32", "%ctaid.x")
    lens, fresh = gptr("p_lens"), gptr("p_fresh")

    def place(pair, ok=None):
        return _Place(e, pair, ok, lens, fresh, batch, chunk, group, tq, ntile, max_pages * page, window, sinks)

    vec = f"v{per_lane}"
    o_l = at(gptr("p_O"), lane, per_lane * 2)

    def first_row(P, kvh):
        return o("mad.lo.u32", o("mad.lo.u32", P.b, chunk, P.c0), heads, o("mul.lo.u32", kvh, group))

    def out_row(base, r):
        t_ = o("div.u32", r, group)
        return o("add.u32", o("mad.lo.u32", t_, heads, base), o("sub.u32", r, o("mul.lo.u32", t_, group)))

    def store(p_, base, r, words):
        e(f"{p_}st.global.{'b32' if per_lane == 2 else 'v2.b32'} [{at(o_l, out_row(base, r), D * 2)}], "
          f"{words[0] if per_lane == 2 else '{' + ', '.join(words) + '}'};")

    l_cut, l_zero = e.L("cut"), e.L("zero")
    e(f"@{e.cond('lt.u32', cta, cuts)} bra {l_cut};")
    unit = o("mad.lo.u32", o("sub.u32", cta, cuts), threads // 32, warp)
    e(f"@{e.cond('ge.u32', unit, pairs * kv_heads)} ret;")
    P = place(o("div.u32", unit, kv_heads))
    p_ = e.cond("eq.u32", P.tiles, 0)
    e(f"and.pred {p_}, {p_}, {P.live};")
    e(f"@!{p_} ret;")
    base, r, z_ = first_row(P, o("rem.u32", unit, kv_heads)), o("mov.u32", 0), o("mov.b32", 0)
    e.label(l_zero)
    store("", base, r, [z_] * (per_lane // 2))
    e(f"add.u32 {r}, {r}, 1;")
    e(f"@{e.cond('lt.u32', r, P.vrows)} bra {l_zero};")
    e("ret;")
    e.label(l_cut)
    sums, run = _prefix(e, lane, pairs, lambda q, ok: place(q, ok).tiles, kv_heads)
    per = o("max.u32", o("div.u32", o("add.u32", run, ctas - 1), ctas), min_tiles)
    pos = o("mul.lo.u32", o("add.u32", cta, 1), per)
    e(f"@{e.cond('ge.u32', pos, run)} ret;")                    # nothing behind the cut
    pair, before = _first_behind(e, sums, pos)
    P = place(pair)
    kvh = o("div.u32", o("sub.u32", pos, before), P.tiles)
    t0 = o("mad.lo.u32", kvh, P.tiles, before)
    first = o("div.u32", t0, per)
    last = o("div.u32", o("sub.u32", o("add.u32", t0, P.tiles), 1), per)
    e(f"@{e.cond('eq.u32', pos, t0)} ret;")                     # between two units
    ncut = o("sub.u32", last, first)
    nth = o("sub.u32", cta, first)
    row0 = o("div.u32", o("mul.lo.u32", nth, P.vrows), ncut)
    row1 = o("div.u32", o("mad.lo.u32", nth, P.vrows, P.vrows), ncut)
    nact = o("add.u32", o("sub.u32", last, first), 1)
    # the first run reaches the unit as a later segment (part 2 c + 1) unless it begins with it
    late = o("selp.u32", 1, 0, e.cond("ne.u32", t0, o("mul.lo.u32", first, per)))
    r0 = o("mad.lo.u32", o("mul.lo.u32", first, 2), rows, 0)
    r_late = o("mad.lo.u32", late, rows, r0)
    base_row = first_row(P, kvh)
    part = gptr("p_part")
    ml = o("add.s64", part, 2 * ctas * rows * D * 4, cls="rd")
    part_l = at(part, lane, per_lane * 4)
    nwarp = threads // 32
    none_m, zero = o("mov.b32", "0fFF800000", cls="f"), o("mov.b32", "0f00000000", cls="f")

    def join_rows(at_once, parts):
        """The block's rows, ``at_once`` of a warp at a time and ``parts`` parts of each."""
        row = o("add.u32", row0, warp)
        l_row, l_out, l_top, l_done = e.L("row"), e.L("out"), e.L("p"), e.L("pd")
        e.label(l_row)
        e(f"@{e.cond('ge.u32', row, row1)} bra {l_out};")
        rws = [o("add.u32", row, nwarp * i) if i else row for i in range(at_once)]
        live = [e.cond("lt.u32", r, row1) for r in rws]
        ms, ls = [o("mov.b32", none_m, cls="f") for _ in rws], [o("mov.b32", zero, cls="f") for _ in rws]
        accs = [[o("mov.b32", zero, cls="f") for _ in range(per_lane)] for _ in rws]
        s = o("mov.u32", 0)
        e.label(l_top)
        e(f"@{e.cond('ge.u32', s, nact)} bra {l_done};")
        loaded = []
        for u in range(parts):
            su = o("add.u32", s, u) if u else s
            base = o("selp.u32", r_late, o("mad.lo.u32", su, 2 * rows, r0), e.cond("eq.u32", su, 0))
            for i, r in enumerate(rws):
                ok = e.cond("lt.u32", su, nact)
                e(f"and.pred {ok}, {ok}, {live[i]};")
                idx = o("add.u32", base, r)
                pm, pl = o("mov.b32", none_m, cls="f"), o("mov.b32", zero, cls="f")
                e(f"@{ok} ld.global.v2.f32 {{{pm}, {pl}}}, [{at(ml, idx, 8)}];")
                xs = [o("mov.b32", zero, cls="f") for _ in range(per_lane)]
                e(f"@{ok} ld.global.{vec}.f32 {{{', '.join(xs)}}}, [{at(part_l, idx, D * 4)}];")
                loaded.append((i, pm, pl, xs))
        for i in range(at_once):
            mine = [x for x in loaded if x[0] == i]
            top = ms[i]
            for _, pm, _, _ in mine:
                top = o("max.f32", top, pm, cls="f")
            ref = o("selp.f32", zero, top, e.cond("eq.f32", top, none_m), cls="f")
            f = o("ex2.approx.ftz.f32", o("sub.f32", ms[i], ref, cls="f"), cls="f")
            for x in (ls[i], *accs[i]):
                e(f"mul.f32 {x}, {x}, {f};")
            for _, pm, pl, xs in mine:
                f = o("ex2.approx.ftz.f32", o("sub.f32", pm, ref, cls="f"), cls="f")
                e(f"fma.rn.f32 {ls[i]}, {f}, {pl}, {ls[i]};")
                for a_, x in zip(accs[i], xs):
                    e(f"fma.rn.f32 {a_}, {f}, {x}, {a_};")
            e(f"mov.b32 {ms[i]}, {top};")
        e(f"add.u32 {s}, {s}, {parts};")
        e(f"bra {l_top};")
        e.label(l_done)
        for i, r in enumerate(rws):
            p_zero = e.cond("eq.f32", ls[i], zero)
            inv = o("rcp.rn.f32", o("selp.f32", "0f3F800000", ls[i], p_zero, cls="f"), cls="f")
            words = []
            for x in range(0, per_lane, 2):
                x0, x1 = (o("mul.f32", accs[i][x + k], inv, cls="f") for k in range(2))
                word = o("cvt.rn.f16x2.f32" if dtype == "f16" else "cvt.rn.bf16x2.f32", x1, x0)
                words.append(o("selp.b32", 0, word, p_zero))
            store(f"@{live[i]} ", base_row, r, words)
        e(f"add.u32 {row}, {row}, {nwarp * at_once};")
        e(f"bra {l_row};")
        e.label(l_out)

    l_many = e.L("many")
    e(f"@{e.cond('gt.u32', nact, 4)} bra {l_many};")
    join_rows(4, 2)
    e("ret;")
    e.label(l_many)
    join_rows(1, 8)
    ln, fn, on = names
    params = [("lens", ln, 4), ("fresh", fn, 4), ("O", on, 8), ("part", scratch, 32)]
    text = [f".visible .entry {name}(", ",\n".join(f"\t.param .u64 p_{p}" for p, _, _ in params), ")",
            f".reqntid {threads}, 1, 1", "{"]
    text += e.decls() + e.lines + ["\tret;", "}"]
    return {"name": name, "kind": "paged_attention_join", "params": [n for _, n, _ in params], "raw_entry": text,
            "grid": [cuts + -(-pairs * kv_heads // (threads // 32)), 1, 1], "block": [threads, 1, 1], "dyn_smem": 0,
            "align": {n: a_ for _, n, a_ in params}, "zero_outputs": [], "pdl": True}
