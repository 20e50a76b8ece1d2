"""The paged key/value cache operators on the CPU: the IR's meaning (oracle), the emitted CUDA-core kernels and the
tensor-core form (emulators) against plain float64, with ragged batches, padding, stale rows of NaN, missing
pages, empty sequences and windows; and what the builders refuse."""
import ctypes
import json
import math

import pytest
import torch

from emmy_ptx_b200 import irgen, launcher
from emmy_ptx_b200.codegen.generic import Unsupported
from emmy_ptx_b200.compiler import compile_graph
from emmy_ptx_b200.data import from_numpy_storage, to_numpy_storage
from emmy_ptx_b200.ir import Graph
from emmy_ptx_b200.launcher import EmmyError
from emmy_ptx_b200.runtime import Executable
from oracle.interp import Interpreter
from tests import pagedemu as PE
from tests import pagedref as R


def by_oracle(p, t):
    """The IR's outputs from the interpreter, on outputs that start as ``t`` holds them."""
    bufs = {a.name: to_numpy_storage(t[a.name]) for a in p.args}
    Interpreter(Graph.from_dict(p.graph)).run(bufs, p.grid, p.block)
    return {a.name: from_numpy_storage(bufs[a.name], a.dtype).reshape(a.shape) for a in p.outputs}


def by_emitter(p, t):
    """The outputs of the statement-at-a-time CUDA-core PTX, run instruction by instruction."""
    got, code, mod = PE.run(p, t, {"patterns": False})
    assert code == 0 and [r["kind"] for r in mod.kernels] == ["generic"]
    return got


def by_kernel(p, t):
    """The outputs of the hand-written kernel the nest is lowered to."""
    got, code, mod = PE.run(p, t)
    assert code == 0 and [r["kind"] for r in mod.kernels] == [p.entry]
    return got


def same(got, want, what):
    """Equal bit for bit, any NaN equal to any other."""
    if got.dtype.is_floating_point:
        assert torch.equal(torch.isnan(got), torch.isnan(want)), what
        got, want = torch.nan_to_num(got.float()), torch.nan_to_num(want.float())
    assert torch.equal(got, want), f"{what}: {int((got != want).sum())} elements differ"


def broken_table(t, pages):
    """Entries that name no page: below zero, one past the pool, far past it."""
    t["table"][0, -1] = -1
    t["table"][-1, 0] = pages
    if t["table"].shape[1] > 2:
        t["table"][0, 1] = 2 ** 31 - 1


def awkward_rows(t, d):
    """Rows for the byte rounding: a scale of exactly 1 with quotients at halves (to even) and their neighbours, a row
    of the type's smallest numbers (the scale's own steps are coarse or it is 0), one of its largest."""
    x = (torch.arange(d) % 64 + 0.5) * (1 - 2 * (torch.arange(d) % 2))
    x[0] = 127.0
    t["K"][-1, 0, 0] = x.to(t["K"].dtype)
    tiny, big = torch.finfo(t["K"].dtype).smallest_normal, torch.finfo(t["K"].dtype).max
    t["V"][-1, 0, 0] = (x * (tiny / 100)).to(t["V"].dtype)
    t["V"][0, -1, -1] = (x / 127 * big).to(t["V"].dtype)


WRITES = [
    # batch, chunk, kv_heads, dim, page, max_pages, lens, fresh
    (3, 4, 2, 64, 8, 3, [4, 9, 24], [4, 2, 0]),
    (2, 1, 1, 128, 16, 2, [1, 32], [1, 1]),
    (2, 5, 3, 32, 3, 4, [3, 14], [5, 5]),              # positions below 0 and past the last page: not written
    (1, 3, 1, 256, 1, 5, [5], [2]),
]


@pytest.mark.parametrize("run", [by_oracle, by_emitter, by_kernel])
@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("case", WRITES, ids=lambda c: "x".join(map(str, c[:6])))
def test_cache_write(case, dtype, quant, run):
    B, C, hk, d, page, mp, lens, fresh = case
    t, pages = R.make("write", B, hk, d, page, mp, lens, fresh, chunk=C, dtype=dtype, quant=quant, seed=B + d)
    broken_table(t, pages)
    t["K"][0, 0, 0] = 0.0                                # a row of zeros
    t["V"][0, 0, 0, 3] = math.inf                        # a row with an infinity, one with a NaN
    t["V"][-1, -1, -1, 5] = math.nan
    awkward_rows(t, d)
    p = irgen.cache_write_ir(B, C, hk, d, pages, page, mp, dtype, quant)
    got = run(p, t)
    want = R.write_ref(t, page, quant)
    for n in want:
        same(got[n], want[n], f"{n} {run.__name__}")


READS = [(3, 20, 2, 64, 8, 3, [0, 9, 24]), (2, 33, 1, 128, 16, 2, [1, 40]), (1, 7, 3, 32, 3, 2, [-4])]


@pytest.mark.parametrize("run", [by_oracle, by_emitter, by_kernel])
@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("case", READS, ids=lambda c: "x".join(map(str, c[:6])))
def test_cache_read(case, dtype, quant, run):
    B, L, hk, d, page, mp, lens = case
    t, pages = R.make("read", B, hk, d, page, mp, lens, [0] * B, length=L, dtype=dtype, quant=quant, seed=L)
    broken_table(t, pages)
    p = irgen.cache_read_ir(B, L, hk, d, pages, page, mp, dtype, quant)
    got = run(p, t)
    want = R.read_ref(t, page, dtype)
    for n in want:
        same(got[n], want[n], f"{n} {run.__name__}")


ATTENDS = [
    # batch, chunk, heads, kv_heads, dim, page, max_pages, lens, fresh, window, sinks
    (3, 3, 4, 2, 32, 8, 3, [3, 9, 20], [3, 2, 0], None, 0),
    (2, 1, 3, 1, 64, 4, 4, [1, 16], [1, 1], None, 0),
    (2, 4, 2, 2, 32, 3, 5, [2, 15], [4, 4], 4, 2),          # two rows at positions below 0: zero
    (1, 2, 2, 1, 64, 8, 2, [19], [2], 1, 0),                 # past the last page; a window of one
]


@pytest.mark.parametrize("run", [by_oracle, by_emitter])
@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("f16", True)])
@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "x".join(map(str, c[:7])))
def test_paged_attention_nest(case, dtype, quant, run):
    B, C, H, hk, d, page, mp, lens, fresh, window, sinks = case
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, dtype=dtype, quant=quant, seed=H)
    if mp == 3:
        broken_table(t, pages)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, dtype, quant, window, sinks)
    got = run(p, t)
    ref, bound, _ = R.attention_ref(t, page, window, sinks)
    R.check(got["O"], ref, bound, run.__name__)


def test_offsets_past_32_bits_are_refused_by_the_cuda_core_form():
    # 2^31 elements and more: the statement-at-a-time emitter computes element offsets in 32 bits
    p = irgen.cache_write_ir(1, 1, 8, 128, 1 << 17, 16, 4)
    with pytest.raises(Unsupported, match="32-bit"):
        compile_graph(Graph.from_dict(p.graph), p.meta(), {"patterns": False})
    p = irgen.cache_write_ir(1, 1, 8, 128, (1 << 17) - 1, 16, 4)
    compile_graph(Graph.from_dict(p.graph), p.meta(), {"patterns": False})


GOOD = dict(batch=1, chunk=1, kv_heads=1, dim=64, pages=4, page=8, max_pages=2)


@pytest.mark.parametrize("change,word", [
    (dict(dim=48), "dim"), (dict(dim=96), "dim"), (dict(page=0), "page"), (dict(kv_heads=True), "kv_heads"),
    (dict(pages=1 << 30), "pages"), (dict(page=1 << 15, max_pages=1 << 15), "positions"), (dict(batch=-1), "batch"),
    (dict(chunk=1 << 27), "threads"), (dict(dtype="f32"), "dtype"), (dict(quant=1), "quant"), (dict(chunk=2.0), "chunk"),
])
def test_builders_refuse(change, word):
    kw = {**GOOD, **change}
    with pytest.raises(ValueError, match=word):
        irgen.cache_write_ir(**kw)
    with pytest.raises(ValueError, match=word):
        irgen.paged_attention_ir(heads=1, **kw)
    kw["length"] = kw.pop("chunk")
    with pytest.raises(ValueError, match="length" if word == "chunk" else word):
        irgen.cache_read_ir(**kw)


@pytest.mark.parametrize("change,word", [
    (dict(heads=3, kv_heads=2), "heads"), (dict(window=0), "window"), (dict(window=2.5), "window"), (dict(sinks=2), "sinks"),
    (dict(window=4, sinks=-1), "sinks"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(scale=0.0), "scale"), (dict(scale=-0.5), "scale"),
    (dict(window=1 << 30), "window"),
])
def test_paged_attention_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        irgen.paged_attention_ir(**{**GOOD, "heads": 2, **change})


# ---- the tensor-core form --------------------------------------------------------------------

TENSOR = [
    # batch, chunk, heads, kv_heads, dim, page, max_pages, lens, fresh, window, sinks, options
    (2, 1, 2, 1, 64, 16, 8, [1, 128], [1, 1], None, 0, {}),
    (3, 1, 4, 2, 128, 32, 6, [190, 0, 64], [1, 0, 1], None, 0, {}),
    (1, 1, 6, 2, 64, 64, 5, [300], [1], None, 0, {"paged_ctas": 5, "paged_min_tiles": 1}),
    (2, 5, 3, 1, 64, 8, 20, [77, 160], [5, 3], None, 0, {"paged_ctas": 3, "paged_min_tiles": 1}),
    (1, 70, 5, 1, 64, 128, 2, [150], [70], None, 0, {}),                     # 25 tokens a tile, 125 rows
    (1, 130, 1, 1, 128, 64, 3, [140], [130], None, 0, {}),                   # a tile of 128 tokens and one of 2
    (2, 1, 2, 2, 64, 16, 20, [320, 40], [1, 1], 70, 3, {}),                  # sink tile, then the window's
    (1, 40, 2, 1, 64, 32, 12, [380], [40], 100, 5, {"paged_ctas": 3, "paged_min_tiles": 1}),
    (1, 9, 2, 1, 64, 64, 4, [256], [9], 1, 0, {}),
    (1, 9, 2, 1, 64, 64, 4, [200], [9], 3, 150, {}),                         # more sinks than a tile
    (2, 6, 2, 1, 64, 16, 2, [4, 40], [6, 6], None, 0, {}),                   # positions below 0, past the table
    (2, 5, 7, 1, 128, 8, 20, [77, 160], [5, 3], 40, 3, {"paged_ctas": 3, "paged_min_tiles": 1}),   # 35 rows
    (1, 8, 8, 1, 64, 16, 9, [131], [8], None, 0, {}),                         # 64 rows
]
FORMS = {"rows": "paged_attention_rows", "tiles": "tcgen05_paged_attention"}


def form_opts(form, case):
    """The options that make a case take one form, or None when it cannot."""
    if form == "rows" and case[1] * (case[2] // case[3]) > 64:
        return None
    return {**case[-1], "paged_rows": 64 if form == "rows" else 0}


@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("form,case", [(f, c) for f in FORMS for c in TENSOR if form_opts(f, c)],
                         ids=lambda c: c if isinstance(c, str) else "x".join(map(str, c[:7])))
def test_paged_attention_tensor_cores_emulated(form, case, dtype, quant):
    B, C, H, hk, d, page, mp, lens, fresh, window, sinks, _ = case
    opts = form_opts(form, case)
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, dtype=dtype, quant=quant, seed=H + C)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, dtype, quant, window, sinks)
    got, code, mod = PE.run(p, t, opts)
    assert code == 0
    kinds = [k["kind"] for k in mod.kernels]
    assert kinds == [FORMS[form]] + ["paged_attention_join"] * (opts.get("paged_ctas", 0) > 0)
    ref, bound, _ = R.attention_ref(t, page, window, sinks)
    R.check(got["O"], ref, bound, form)


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("page", [8, 64])
def test_paged_attention_late_completions_and_missing_pages(page, quant, rows):
    # asynchronous work completes as late as the barriers allow; table entries name no page
    mp = 320 // page
    t, pages = R.make("attend", 2, 1, 64, page, mp, [320, 250], [3, 3], chunk=3, heads=2, quant=quant, seed=page)
    t["table"][0, 1] = -1
    t["table"][0, mp - 2] = pages
    t["table"][1, 0] = 2 ** 31 - 1
    p = irgen.paged_attention_ir(2, 3, 2, 1, 64, pages, page, mp, "bf16", quant)
    got, code, _ = PE.run(p, t, {"paged_ctas": 3, "paged_min_tiles": 2, "paged_rows": rows}, defer=True)
    assert code == 0
    ref, bound, _ = R.attention_ref(t, page)
    R.check(got["O"], ref, bound, "late completions")


SPREAD = [
    # batch, chunk, heads, kv_heads, dim, page, max_pages, lens, fresh, window, sinks
    (5, 2, 4, 2, 64, 16, 13, [70, 0, 200, 1, 65], [2, 0, 1, 2, 2], None, 0),       # 4's first row sees no key
    (3, 70, 2, 1, 64, 64, 4, [250, 69, 130], [70, 70, 3], None, 0),                 # two token tiles, one of padding
    (3, 3, 2, 1, 64, 8, 25, [200, 5, 150], [3, 3, 3], 66, 4),
]


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("ctas", [1, 2, 3, 7])
@pytest.mark.parametrize("form,case", [(f, c) for f in FORMS for c in SPREAD if f == "tiles" or c[1] <= 32],
                         ids=lambda c: c if isinstance(c, str) else "x".join(map(str, c[:7])))
def test_paged_attention_runs_over_many_units(form, case, ctas, quant):
    # runs that end in one unit, cover others and begin a third, at odd and even tiles; sequences without work
    B, C, H, hk, d, page, mp, lens, fresh, window, sinks = case
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, quant=quant, seed=ctas)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, "bf16", quant, window, sinks)
    ref, bound, _ = R.attention_ref(t, page, window, sinks)
    got, code, _ = PE.run(p, t, {"paged_rows": 64 if form == "rows" else 0, "paged_ctas": ctas, "paged_min_tiles": 1},
                          defer=ctas == 2)
    assert code == 0
    R.check(got["O"], ref, bound, f"{form} {ctas}")


SPECIAL = [
    # chunk, heads, kv_heads, dim, lens, window, sinks, positions of V rows with an infinity or a NaN
    (5, 2, 1, 64, 70, None, 0, [65, 67, 69]),
    (3, 3, 1, 128, 3, None, 0, [0, 1, 2]),                           # the first tile, before any product
    (6, 2, 2, 64, 200, 70, 3, [1, 127, 128, 131, 199]),                # the window begins for some rows only
    (1, 2, 1, 64, 130, 70, 3, [2, 59, 60, 129]),                       # one token: keys behind the window are not read
    (9, 1, 1, 64, 150, 5, 64, [3, 64, 138, 140, 143, 145]),
]


def with_specials(case, dtype, page):
    """Inputs with infinities and NaNs in the values (and a NaN key) of keys that some rows see and others do not."""
    C, H, hk, d, n, window, sinks, where = case
    t, pages = R.make("attend", 1, hk, d, page, -(-n // page), [n], [C], chunk=C, heads=H, dtype=dtype, seed=n)
    for i, pos in enumerate(where):
        pg = int(t["table"][0, pos // page])
        t["VC"][pg, :, pos % page, 3 * i] = (math.inf, -math.inf, math.nan)[i % 3]
        t["VC"][pg, 0, pos % page, 3] = math.inf                      # the same column with both signs
    if C > 1:                                                            # seen by the last token alone
        t["KC"][int(t["table"][0, (n - 1) // page]), 0, (n - 1) % page, 5] = math.nan
    return t, pages


@pytest.mark.parametrize("form", ["rows", "tiles", "oracle"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", SPECIAL, ids=lambda c: "x".join(map(str, c[:5])))
def test_infinities_and_nans_reach_only_rows_that_see_them(case, dtype, form):
    C, H, hk, d, n, window, sinks, _ = case
    t, pages = with_specials(case, dtype, 16)
    p = irgen.paged_attention_ir(1, C, H, hk, d, pages, 16, t["table"].shape[1], dtype, False, window, sinks)
    ref, bound, _ = R.attention_ref(t, 16, window, sinks)
    for ctas in (0,) if form == "oracle" else (0, 2):
        if form == "oracle":
            got = by_oracle(p, t)
        else:
            got, code, _ = PE.run(p, t, {"paged_rows": 64 if form == "rows" else 0, "paged_ctas": ctas, "paged_min_tiles": 1})
            assert code == 0
        assert torch.isfinite(got["O"]).any()
        R.check(got["O"], ref, bound, form, inf_or_nan=form != "oracle")


@pytest.mark.parametrize("missing", range(0, 17, 2))
def test_paged_attention_a_missing_page_masks_no_other(missing):
    # the masks of a ring stage that held a missing page must be gone when the next block comes to it
    t, pages = R.make("attend", 1, 1, 64, 16, 17, [271], [9], chunk=9, heads=2, quant=bool(missing % 4), seed=missing)
    t["table"][0, missing] = -1
    p = irgen.paged_attention_ir(1, 9, 2, 1, 64, pages, 16, 17, "bf16", bool(missing % 4))
    ref, bound, _ = R.attention_ref(t, 16)
    for rows in (0, 64):
        got, code, _ = PE.run(p, t, {"paged_rows": rows})
        assert code == 0
        R.check(got["O"], ref, bound, f"rows {rows}")


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("quant", [False, True])
def test_paged_attention_all_pages_missing_is_zero(quant, rows):
    t, pages = R.make("attend", 1, 1, 64, 16, 8, [100], [2], chunk=2, heads=2, quant=quant)
    t["table"].fill_(-1)
    p = irgen.paged_attention_ir(1, 2, 2, 1, 64, pages, 16, 8, "bf16", quant)
    for opts in ({}, {"paged_ctas": 3, "paged_min_tiles": 1}):
        got, code, _ = PE.run(p, t, {**opts, "paged_rows": rows})
        assert code == 0 and not got["O"].any()


def test_paged_attention_lowering_rule():
    """What the tensor cores take: head dim 64 or 128; pages of whole 8-row pieces for few rows a unit (at most 64
    where the tcgen05 form does not take the pages), else a group of at most 128 heads and pages that tile 64 keys; a changed nest stays on the CUDA
    cores."""
    def kind(change=None, **kw):
        base = dict(batch=1, chunk=1, heads=2, kv_heads=1, dim=64, pages=4, page=16, max_pages=2)
        p = irgen.paged_attention_ir(**{**base, **kw})
        if change:
            change(p.graph["nodes"]["paged_attention"])
        return compile_graph(Graph.from_dict(p.graph), p.meta()).kernels[0]["kind"]
    assert kind() == kind(page=24) == kind(heads=16) == kind(chunk=8) == "paged_attention_rows"
    assert kind(heads=64, page=24) == kind(chunk=32, page=96) == kind(heads=32, quant=True) == "paged_attention_rows"
    assert kind(heads=17) == kind(chunk=9) == kind(heads=33, quant=True) == "tcgen05_paged_attention"
    assert kind(chunk=40, dim=128, page=192, window=3, sinks=1, scale=0.25) == "tcgen05_paged_attention"
    for kw in (dict(dim=32), dict(dim=256), dict(page=4), dict(page=12), dict(heads=129), dict(chunk=40, page=24),
               dict(chunk=40, page=96)):
        assert kind(**kw) == "generic", kw

    def swap(node):                                        # K and V exchanged in the nest
        s = json.dumps(node["op_fields"]).replace('"KC"', '"XX"').replace('"VC"', '"KC"').replace('"XX"', '"VC"')
        node["op_fields"] = json.loads(s)
    assert kind(swap) == "generic"

    def late(node):                                        # the causal limit one key further
        s = json.dumps(node["op_fields"])
        i = s.index('"minimum"')
        node["op_fields"] = json.loads(s[:i] + s[i:].replace('"right": 1', '"right": 2', 1))
    assert kind(late) == "generic"


# ---- the runtime's side, through a device that only records ----------------------------------------------


class PlanDevice:
    """Stands in for :class:`launcher.Device`: keeps the plans it is given and the parameters they are launched
    with."""

    def __init__(self):
        self.plans, self.log = [], []

    def load_ptx(self, ptx):
        return "module"

    def function(self, mod, entry):
        return entry

    def set_max_dyn_smem(self, fn, nbytes):
        pass

    def plan(self, fn, grid, block, dyn_smem, align, cluster=(1, 1, 1), pdl=False, tmaps=(), tail=None):
        self.plans.append(dict(fn=fn, grid=grid, align=align, pdl=pdl, tmaps=tmaps, tail=tail))
        return len(self.plans) - 1

    def launch_plan(self, plan, params, stream):
        for a, x in zip(self.plans[plan]["align"], params):
            if x % a:
                raise EmmyError(10003, "emmy_plan_launch", "aligned")
        self.log.append((self.plans[plan]["fn"], list(params), stream))

    def destroy_plan(self, plan):
        self.log.append(("destroyed", plan))

    def unload(self, mod):
        pass


class HostExecutable(Executable):
    def _device_tensor(self, shape, dtype):
        return torch.empty(shape, dtype=dtype)


@pytest.fixture
def exe(monkeypatch):
    dev = PlanDevice()
    monkeypatch.setattr(launcher.Device, "get", classmethod(lambda cls, index=0: dev))
    t, pages = R.make("attend", 2, 1, 64, 16, 8, [100, 20], [40, 3], chunk=40, heads=4)
    p = irgen.paged_attention_ir(2, 40, 4, 1, 64, pages, 16, 8)
    ex = HostExecutable(compile_graph(Graph.from_dict(p.graph), p.meta()), device=0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)          # CPU tensors pass for cuda:0's
    return ex, t, dev


def test_a_plan_gets_pointers_maps_and_the_status_word(exe):
    ex, t, dev = exe
    ex.run(t, 55)
    (fn, params, stream), = dev.log
    rec = ex.records[0]
    assert (fn, stream) == ("paged_attention", 55) and rec["kind"] == "tcgen05_paged_attention"
    assert params == [t[n].data_ptr() for n in rec["params"]]
    plan, = dev.plans
    assert [m[0] for m in plan["tmaps"]] == [rec["params"].index(n) for n in ("KC", "VC")]
    assert plan["tail"] == ex.err.data_ptr()
    ex.close()
    assert dev.log[-1] == ("destroyed", 0)


@pytest.mark.parametrize("name,make", [
    ("Q", lambda t: t["Q"].float()), ("Q", lambda t: t["Q"][:, :39]), ("KC", lambda t: t["KC"].transpose(1, 2)),
    ("lens", lambda t: t["lens"].long()), ("table", lambda t: t["table"].repeat(1, 2)[:, ::2]),
    ("O", lambda t: t["O"].transpose(0, 1)), ("fresh", lambda t: None),
    ("O", lambda t: torch.empty(t["O"].numel() + 1, dtype=t["O"].dtype)[1:].view(t["O"].shape)),
], ids=["type", "shape", "order", "index-type", "strides", "transposed", "missing", "alignment"])
def test_tensors_of_another_kind_are_refused_before_a_launch(exe, name, make):
    ex, t, dev = exe
    with pytest.raises(ValueError, match=repr(name)):
        ex.run({**t, name: make(t)}, 55)
    assert dev.log == []


def test_tensors_of_another_device_are_refused(exe, monkeypatch):
    ex, t, dev = exe
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: -1)
    with pytest.raises(ValueError, match="cuda:0"):
        ex.run(t, 55)
    assert dev.log == []


def test_plan_arguments_are_checked_before_the_driver():
    lib = launcher.load_library()
    u3 = (ctypes.c_uint32 * 3)(1, 1, 1)
    al = (ctypes.c_uint32 * 17)(*[16] * 17)
    fn, h = ctypes.c_void_p(0x1000), ctypes.c_void_p()
    assert lib.emmy_plan_create(None, u3, u3, None, 0, 0, al, 1, ctypes.byref(h)) != 0
    assert lib.emmy_plan_create(fn, u3, u3, None, 0, 0x80, al, 1, ctypes.byref(h)) != 0
    assert lib.emmy_plan_create(fn, u3, u3, None, 0, 0, al, 17, ctypes.byref(h)) != 0 and "16" in launcher.last_error()
    assert lib.emmy_plan_create(fn, u3, u3, None, 0, 0, al, 2, ctypes.byref(h)) == 0
    d = (ctypes.c_uint64 * 2)(64, 64)
    b = (ctypes.c_uint32 * 2)(64, 8)
    assert lib.emmy_plan_add_tmap(h, 2, 9, 2, d, d, b, 3, 2) != 0            # a parameter the plan does not have
    assert lib.emmy_plan_add_tmap(h, 0, 9, 6, d, d, b, 3, 2) != 0
    assert lib.emmy_plan_launch(h, d, 1, None) != 0 and "2 parameters" in launcher.last_error()
    bad = (ctypes.c_uint64 * 2)(64, 72)
    assert lib.emmy_plan_launch(h, bad, 2, None) != 0 and "parameter 1" in launcher.last_error()
    assert lib.emmy_plan_launch(None, d, 2, None) != 0
    assert lib.emmy_plan_destroy(h) == 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a library that has no device")
def test_a_plan_without_a_context_is_not_launched():
    lib = launcher.load_library()
    u3, al, h = (ctypes.c_uint32 * 3)(1, 1, 1), (ctypes.c_uint32 * 1)(16), ctypes.c_void_p()
    assert lib.emmy_plan_create(ctypes.c_void_p(0x1000), u3, u3, None, 0, 0, al, 1, ctypes.byref(h)) == 0
    assert lib.emmy_plan_launch(h, (ctypes.c_uint64 * 1)(64), 1, None) != 0 and "emmy_init" in launcher.last_error()
    assert lib.emmy_plan_destroy(h) == 0


@pytest.mark.parametrize("scale", [2.0 ** -65, 2.0 ** 65, 1e-38, 1e38])
def test_scales_whose_products_leave_f32_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        irgen.paged_attention_ir(**{**GOOD, "heads": 2, "scale": scale})


def test_a_closed_executable_refuses(exe):
    ex, t, dev = exe
    ex.close()
    with pytest.raises(ValueError, match="closed"):
        ex.run(t, 55)
    assert dev.log == [("destroyed", 0)]


@pytest.mark.parametrize("quant", [False, True])
def test_units_start_with_the_longest(quant):
    """More units than an SM count of 1 holds: which unit a CTA takes goes by the lengths (equal ones and none among
    them), and every unit is taken once."""
    B, C, H, hk, d, page, mp = 5, 130, 1, 1, 64, 64, 5
    t, pages = R.make("attend", B, hk, d, page, mp, [140, 300, 0, 140, 219], [130, 70, 0, 130, 3], chunk=C, heads=H,
                      quant=quant, seed=6)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, "bf16", quant)
    got, code, mod = PE.run(p, t, {"sms": 1, "paged_ctas": 0})
    assert code == 0 and mod.kernels[0]["grid"] == [10, 1, 1] and "_order" in mod.ptx
    ref, bound, _ = R.attention_ref(t, page)
    R.check(got["O"], ref, bound, "longest first")


@pytest.mark.parametrize("opts", [{"paged_ctas": -1}, {"paged_ctas": 1 << 15}, {"paged_min_tiles": 0},
                                  {"paged_min_tiles": 1 << 17}])
@pytest.mark.parametrize("rows", [0, 64])
def test_options_out_of_range_are_refused(opts, rows):
    p = irgen.paged_attention_ir(2, 1, 2, 1, 64, 8, 64, 4)
    with pytest.raises(ValueError, match="paged_ctas"):
        compile_graph(Graph.from_dict(p.graph), p.meta(), {**opts, "paged_rows": rows})


@pytest.mark.parametrize("rows", [0, 64])
def test_more_tiles_than_32_bits_are_not_cut_into_runs(rows):
    p = irgen.paged_attention_ir(128, 1, 2, 2, 64, 1 << 20, 64, (1 << 24) - 1)
    for opts in ({}, {"paged_ctas": 0}):
        assert len(compile_graph(Graph.from_dict(p.graph), p.meta(), {**opts, "paged_rows": rows}).kernels) == 1
    with pytest.raises(ValueError, match="tiles"):
        compile_graph(Graph.from_dict(p.graph), p.meta(), {"paged_ctas": 8, "paged_rows": rows})
