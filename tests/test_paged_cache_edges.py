"""The paged key/value cache at the edges of what its definition allows, on the CPU (emulated kernels, recording
devices) against plain float64."""
import contextlib
import ctypes
import json
from types import SimpleNamespace

import pytest
import torch

from emmy_ptx_b200 import data, irgen, launcher
from emmy_ptx_b200.codegen.generic import Unsupported
from emmy_ptx_b200.compiler import compile_graph
from emmy_ptx_b200.ir import Graph
from emmy_ptx_b200.runtime import Executable
from tests import pagedemu as PE
from tests import pagedref as R
from tests.test_paged_cache import PlanDevice, same

#: scales as other programs may leave them: a factor for every token of every head
SIGNS = {"negative": lambda n: -torch.ones(n), "alternating": lambda n: 1.0 - 2.0 * (torch.arange(n) % 2),
         "large-negative": lambda n: torch.where(torch.arange(n) % 7 == 3, -1024.0, 1.0)}
SIGNED = [
    # batch, chunk, heads, kv_heads, dim, page, max_pages, lens, fresh, options
    (1, 1, 4, 1, 128, 16, 5, [70], [1], {}),
    (2, 3, 2, 1, 64, 16, 9, [130, 20], [3, 2], {"paged_ctas": 3, "paged_min_tiles": 1}),
]


def signed_case(case, dtype, signs):
    """Inputs whose key and value scales carry signs (the keys' only the signs: their sizes would make every score
    but one vanish)."""
    B, C, H, hk, d, page, mp, lens, fresh, _ = case
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, dtype=dtype, quant=True, seed=d)
    f = SIGNS[signs](t["VS"].numel()).reshape(t["VS"].shape)
    t["VS"] = t["VS"] * f
    t["KS"] = t["KS"] * torch.sign(f).flip(0)
    return t, irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, dtype, True)


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("signs", SIGNS)
@pytest.mark.parametrize("case,dtype", [(SIGNED[0], "f16"), (SIGNED[1], "bf16")], ids=["decode-f16", "draft-runs-bf16"])
def test_scales_of_any_sign(case, dtype, signs, rows):
    t, p = signed_case(case, dtype, signs)
    got, code, _ = PE.run(p, t, {**case[-1], "paged_rows": rows})
    assert code == 0
    ref, bound, _ = R.attention_ref(t, case[5])
    R.check(got["O"], ref, bound, signs)


# ---- values near both ends of f32 ------------------------------------------------------------


def ramp_case(quant, k, n=230):
    """Scores that grow by almost 2^8 along the keys (a kernel that takes its reference from the first ones has weights
    up to 2^8 here), values times 2^k.  Values of one sign, so that no sum cancels."""
    d, page = 64, 16
    t, pages = R.make("attend", 1, 1, d, page, -(-n // page), [n], [2], chunk=2, heads=2, quant=quant, seed=4)
    u = torch.ones(d)
    x = torch.zeros(pages, 1, page, d)
    for j in range(n):
        x[int(t["table"][0, j // page]), 0, j % page] = u * (j / n) * 5.4 / 8
    t["Q"][:] = 1.0                                           # the last key's score: 64 * 5.4 / 8 / 8
    v = (x + 1) * torch.rand(x.shape, generator=torch.Generator().manual_seed(1)).add(0.25)
    for name, y in (("K", x), ("V", v)):
        if quant:
            t[name + "C"], t[name + "S"] = R.quantise(y.to(torch.bfloat16))
        else:
            t[name + "C"] = y.to(torch.bfloat16)
    big = dict(t)
    if quant:
        big["VS"] = t["VS"] * 2.0 ** k
    else:
        big["VC"] = t["VC"] * 2.0 ** k
    return t, big, irgen.paged_attention_ir(1, 2, 2, 1, d, pages, page, -(-n // page), "bf16", quant)


#: bytes down to scales of 2^-126, both kinds up to sums of 2^127 with weights of at most 1
RANGES = [(False, 119), (True, 119), (True, -119)]


def check_scaled(got, base, k):
    """Values times 2^k give the output times 2^k: everything between is a product with a power of two, exact but where
    it leaves the normal numbers (by 2^-141 here, which may turn the last rounding: one step of bf16)."""
    want = base.double() * 2.0 ** k
    err = (got.double() - want).abs()
    assert bool((err <= (2.0 ** -7 * want.abs() + 2.0 ** -133 if k < 0 else 0 * want)).all()), (err / want).max()


@pytest.mark.parametrize("opts", [{}, {"paged_ctas": 3, "paged_min_tiles": 1}], ids=["whole", "runs"])
@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("quant,k", RANGES)
def test_values_near_the_ends_of_f32(quant, k, rows, opts):
    t, big, p = ramp_case(quant, k)
    base, c0, _ = PE.run(p, t, {**opts, "paged_rows": rows})
    got, c1, _ = PE.run(p, big, {**opts, "paged_rows": rows})
    assert c0 == c1 == 0
    ref, bound, _ = R.attention_ref(t, 16)
    R.check(base["O"], ref, bound, "before")
    check_scaled(got["O"], base["O"], k)


# ---- queries of any size over a cache of bytes -----------------------------------------------


QSIZES = [(-60, 60, None), (-97, 97, None), (-109, 100, 64.0), (-40, 97, 2.0 ** -60), (100, -100, None), (-26, 26, None)]


def sized_case(q2, k2, scale):
    """Queries times 2^q2 against key scales times 2^k2: ordinary scores, times 2^(q2 + k2)."""
    t, pages = R.make("attend", 1, 2, 64, 16, 8, [120], [2], chunk=2, heads=4, quant=True, seed=11)
    t["Q"] = t["Q"] * 2.0 ** q2
    t["Q"][0, 1, 1] = 0.0                                     # a row of zeros: the mean of the values
    t["KS"] = t["KS"] * 2.0 ** k2
    return t, irgen.paged_attention_ir(1, 2, 4, 2, 64, pages, 16, 8, "bf16", True, scale=scale)


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("q2,k2,scale", QSIZES)
def test_queries_of_any_size_over_bytes(q2, k2, scale, rows):
    t, p = sized_case(q2, k2, scale)
    got, code, _ = PE.run(p, t, {"paged_rows": rows})
    assert code == 0
    ref, bound, _ = R.attention_ref(t, 16, scale=scale)
    R.check(got["O"], ref, bound, "sizes")


# ---- several kernels in one graph ------------------------------------------------------------


def joined(*problems):
    """(graph, meta) of the problems' kernels one after the other, tensors of one name shared."""
    nodes = {}
    for p in problems:
        nodes.update({n: x for n, x in p.graph["nodes"].items() if x["op"] == "KernelOp"})
    made = {o["name"] for x in nodes.values() for o in x["outputs"]}
    ins = {n: x for p in problems for n, x in p.graph["nodes"].items() if x["op"] == "InputOp" and n not in made}
    graph = {"nodes": {**ins, **nodes}, "inputs": list(ins), "outputs": sorted(made)}
    return graph, {"kernels": [k for p in problems for k in p.meta()["kernels"]]}


def step_problems(quant=False):
    """A decode step's write, attention and read back, and all their tensors."""
    B, H, hk, d, page, mp = 2, 4, 2, 64, 16, 6
    lens = [30, 61]
    w, pages = R.make("write", B, hk, d, page, mp, lens, [1, 1], quant=quant, seed=3)
    a, _ = R.make("attend", B, hk, d, page, mp, lens, [1, 1], heads=H, quant=quant, seed=4)
    r, _ = R.make("read", B, hk, d, page, mp, lens, [1, 1], length=mp * page, quant=quant, seed=5)
    c = (hk, d, pages, page, mp, "bf16", quant)
    return {**r, **a, **w}, (irgen.cache_write_ir(B, 1, *c), irgen.paged_attention_ir(B, 1, H, *c),
                             irgen.cache_read_ir(B, mp * page, *c))


def step_refs(t, quant, page=16):
    """The tensors after the step, and the attention's bound."""
    t = {**t, **R.write_ref(t, page, quant)}
    ref, bound, _ = R.attention_ref(t, page)
    return {**t, **R.read_ref(t, page, "bf16")}, ref, bound


class Recorder:
    """A device that notes what it is asked to launch, from plans and without; see :class:`tests.test_paged_cache.PlanDevice`."""

    def __init__(self):
        self.plans, self.log, self.maps = [], [], []

    def load_ptx(self, ptx):
        return "module"

    def function(self, mod, entry):
        return entry

    def set_max_dyn_smem(self, fn, nbytes):
        pass

    def plan(self, fn, *args, **kw):
        self.plans.append(fn)
        return fn

    def launch_plan(self, plan, params, stream):
        self.log.append(("plan", plan, list(params), stream))

    def launch(self, fn, grid, block, dyn_smem, stream, arg_ptrs, cluster=(1, 1, 1), pdl=False):
        self.log.append(("launch", fn, [ctypes.cast(a, ctypes.POINTER(ctypes.c_uint64))[0] for a in arg_ptrs], stream))

    def launch_u64(self, fn, grid, block, dyn_smem, stream, params, align=None, pdl=False):
        self.log.append(("launch", fn, list(params), stream))

    def tmap_encode_tiled(self, out_buf, dtype, gaddr, dims, strides, box, **kw):
        self.maps.append((gaddr, tuple(box)))

    def memset_d32(self, ptr, value, count, stream):
        self.log.append(("zero", ptr, count, stream))

    def destroy_plan(self, plan):
        pass

    def unload(self, mod):
        pass


class HostExecutable(Executable):
    def _device_tensor(self, shape, dtype):
        return torch.empty(shape, dtype=dtype)

    def _call_scratch(self, stream):
        return {n: torch.empty(k, dtype=dt) for n, (k, dt) in self._temp.items()}


@pytest.fixture
def recorder(monkeypatch):
    dev = Recorder()
    monkeypatch.setattr(launcher.Device, "get", classmethod(lambda cls, index=0: dev))
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)          # CPU tensors pass for cuda:0's
    return dev


def shifted(x, by=2):
    """The same tensor ``by`` bytes past a 64-byte boundary."""
    raw = torch.empty(x.numel() * x.element_size() + 128, dtype=torch.uint8)
    at = -raw.data_ptr() % 64 + by
    y = raw[at:at + x.numel() * x.element_size()].view(x.dtype).view(x.shape)
    return y.copy_(x)


RUNS = {"paged_ctas": 3, "paged_min_tiles": 1}


def host_executable(problems, opts=None):
    g, meta = joined(*problems)
    return HostExecutable(compile_graph(Graph.from_dict(g), meta, opts or {}), device=0)


def test_a_graph_of_cache_operators_runs_from_plans(recorder):
    t, problems = step_problems()
    ex = host_executable(problems, RUNS)
    names = ["cache_write", "paged_attention", "paged_attention_join", "cache_read"]
    assert [r["entry"] for r in ex.records] == names == recorder.plans
    ex.run(t, 55)
    assert [(x[0], x[1], x[3]) for x in recorder.log] == [("plan", n, 55) for n in names]
    for (_, _, ptrs, _), rec in zip(recorder.log, ex.records):
        want = [t[n].data_ptr() if n in t else None for n in rec["params"]]
        assert [x for x, y in zip(ptrs, want) if y is not None] == [y for y in want if y is not None]
    part = [x[2][ex.records[i]["params"].index("paged_attention__paged_attention__part")] for i, x in enumerate(recorder.log)
            if i in (1, 2)]
    assert part[0] == part[1] and part[0]
    for name in ("K", "Q", "KR"):                                  # every kernel's tensors are checked before any launch
        for other in (t[name].float(), shifted(t[name]))[:1 if name == "K" else 2]:      # K's plan checks K itself
            recorder.log.clear()
            with pytest.raises(ValueError, match=repr(name)):
                ex.run({**t, name: other}, 55)
            assert recorder.log == []


def other_first():
    """A kernel that zeroes its output before it runs, beside the cache's."""
    return irgen.SMALL["c2"]()


@pytest.mark.parametrize("first", [True, False])
def test_a_cache_operator_beside_another_kernel(recorder, first):
    t, problems = step_problems()
    q = other_first()
    t = {**t, **data.make_inputs(q)}
    ex = host_executable([q, problems[1]] if first else [problems[1], q], RUNS)
    assert ex.plans is None and recorder.plans == []
    ex.run(t, 55)
    mine = [("launch", "paged_attention"), ("launch", "paged_attention_join")]
    other = [("zero", t["out"].data_ptr()), ("launch", q.entry)]
    assert [x[:2] for x in recorder.log] == (other + mine if first else mine + other)
    calls = {x[1]: x[2] for x in recorder.log if x[0] == "launch"}
    for rec in ex.records:
        for n, x in zip(rec["params"], calls[rec["entry"]]):
            if n in t:
                assert x == t[n].data_ptr(), (rec["entry"], n)
    i, j = (r["params"].index("paged_attention__paged_attention__part") for r in ex.records if "join" in r["entry"]
            or r["entry"] == "paged_attention")
    assert calls["paged_attention"][i] == calls["paged_attention_join"][j]
    for other in (t["Q"][:, :, :3], shifted(t["Q"])):
        recorder.log.clear()
        with pytest.raises(ValueError, match="'Q'"):
            ex.run({**t, "Q": other}, 55)
        assert recorder.log == []


def test_a_closed_executable_of_several_kernels_refuses(recorder):
    t, problems = step_problems()
    q = other_first()
    ex = host_executable([q, problems[1]], RUNS)
    ex.close()
    with pytest.raises(ValueError, match="closed"):
        ex.run({**t, **data.make_inputs(q)}, 55)
    assert recorder.log == []


def test_two_attentions_of_one_graph_have_their_own_tensor_maps(recorder):
    # both name their map of the pool alike; their boxes differ
    B, H, hk, d, page, mp = 1, 2, 1, 64, 64, 3
    t, pages = R.make("attend", B, hk, d, page, mp, [150], [1], heads=H)
    b, _ = R.make("attend", B, hk, d, page, mp, [150], [70], chunk=70, heads=H)
    one = irgen.paged_attention_ir(B, 1, H, hk, d, pages, page, mp)
    many = irgen.paged_attention_ir(B, 70, H, hk, d, pages, page, mp)
    many.graph = json.loads(json.dumps(many.graph).replace('"Q"', '"Q2"').replace('"O"', '"O2"').replace(
        '"paged_attention"', '"chunk_attention"'))
    many.entry = "chunk_attention"
    for a in many.args:
        a.name = {"Q": "Q2", "O": "O2"}.get(a.name, a.name)
    q = other_first()
    t = {**t, "Q2": b["Q"], "O2": b["O"], **data.make_inputs(q)}
    ex = host_executable([one, many, q])
    assert [r["kind"] for r in ex.records[:2]] == ["paged_attention_rows", "tcgen05_paged_attention"] and ex.plans is None
    ex.run(t, 55)
    boxes = [tuple(s["box"]) for r in ex.records[:2] for s in r["tmaps"]]
    assert [x for _, x in recorder.maps] == boxes and boxes[0] != boxes[2]
    ex.run(t, 55)
    assert len(recorder.maps) == len(boxes)                       # kept for the same pointers


@pytest.mark.parametrize("quant", [False, True])
def test_a_serving_step_as_one_graph_emulated(quant):
    t, problems = step_problems(quant)
    g, meta = joined(*problems)
    mod = compile_graph(Graph.from_dict(g), meta, RUNS)
    specs = {a.name: a for p in problems for a in p.args}
    outs = [specs[n] for n in g["outputs"]]
    whole = SimpleNamespace(args=list(specs.values()), outputs=outs)
    got, code, _ = PE.run(whole, t, mod=mod)
    assert code == 0
    want, ref, bound = step_refs(t, quant)
    R.check(got["O"], ref, bound, "step")
    for n in got:
        if n != "O":
            same(got[n], want[n], n)


# ---- what the documents promise of addresses -------------------------------------------------


@pytest.mark.parametrize("quant", [False, True])
def test_tensors_on_32_byte_boundaries_are_taken(recorder, monkeypatch, quant):
    # what a plan's first entry checks itself is checked by the stand-in of tests.test_paged_cache
    dev = PlanDevice()
    monkeypatch.setattr(launcher.Device, "get", classmethod(lambda cls, index=0: dev))
    t, problems = step_problems(quant)
    for p, opts in [(problems[0], {}), (problems[1], {}), (problems[1], {"paged_rows": 0}), (problems[2], {})]:
        ex = HostExecutable(compile_graph(Graph.from_dict(p.graph), p.meta(), opts), device=0)
        mine = {a.name: shifted(t[a.name], 32) for a in p.args}
        ex.run(mine, 55)
        assert dev.log
        for rec in ex.records:
            for n, a in rec["align"].items():
                assert a <= 32, (rec["entry"], n)
        # 16 bytes are enough for what is loaded in pieces of 16, and refused before a launch where they are not
        for name, a in ex.records[0]["align"].items():
            if name in t:
                dev.log.clear()
                call = {**mine, name: shifted(t[name], 16)}
                if a <= 16:
                    ex.run(call, 55)
                    assert dev.log
                else:
                    assert name in ("KC", "VC", "KR", "VR", "O")
                    with pytest.raises(ValueError, match=f"'{name}' must be 32-byte"):
                        ex.run(call, 55)
                    assert dev.log == []


# ---- buffers past 32 bits on the CUDA-core path ----------------------------------------------


def big_buffer(shape, index, extra=()):
    """y[i] = x[index] of 1024 elements, x of ``shape``."""
    i = irgen
    body = [i.Tile([i.Axis("i", 1024)], [*extra, i.Load(["a"], "x", index, "f32"), i.Write("y", ["a"], [i.V("i")], "f32")])]
    args = [i.TensorSpec("x", shape, "f32"), i.TensorSpec("at", (1024,), "i32", ("randint", 0, 8)),
            i.TensorSpec("y", (1024,), "f32", output=True)]
    p = i.Problem("big", "test", "big", i._graph("big", args, body), args, grid=8, block=128)
    return lambda: compile_graph(Graph.from_dict(p.graph), p.meta())


def test_a_low_part_of_a_large_buffer_is_addressed():
    i = irgen
    at = [i.Load(["k"], "at", [i.V("i")], "i32")]
    huge = 1 << 33
    big_buffer((huge,), [i.V("i")])()                              # a range that is known, and short
    big_buffer((1 << 10, huge >> 10), [0, i.Bin("*", i.V("i"), 4)])()
    big_buffer((1 << 10, huge >> 10), [i.Bin("/", i.V("i"), 256), i.V("i")])()          # up to 3 rows of 2^23
    big_buffer((huge,), [i.V("k")], at)()                          # a 32-bit number as it is
    with pytest.raises(Unsupported, match="32-bit"):               # rows up to 1023 of 2^23: past 2^32
        big_buffer((1 << 10, huge >> 10), [i.V("i"), 0])()
    with pytest.raises(Unsupported, match="32-bit"):               # a row that only the data know
        big_buffer((1 << 10, huge >> 10), [i.V("k"), i.V("i")], at)()
    big_buffer((1 << 10, (1 << 31 >> 10) - 1), [i.V("k"), i.V("i")], at)()


# ---- the byte rows' scale --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_the_scale_is_the_product_with_the_rounded_inverse(dtype):
    """s = max|x| * f32(1/127), which for some rows is not max|x| / 127 rounded to f32: there by one f32 step (both
    round once, the constant is half a step off at most), which moves a stored value by half a step s / 2 at most
    more than the rounding, as the byte may be the next one where x / s lies next to a half."""
    dt = R.DT[dtype]
    top = 1 + torch.arange(1 << (7 if dtype == "bf16" else 10)) / (1 << (7 if dtype == "bf16" else 10))
    x = torch.randn(len(top), 64, generator=torch.Generator().manual_seed(2)).clamp(-0.99, 0.99)
    x[:, 5] = top
    x = x.to(dt)
    by, s = R.quantise(x)
    quotient = (x.double().abs().amax(-1) / 127).float()
    other = s != quotient
    assert 4 <= int(other.sum()) < len(s)
    step = (s.view(torch.int32) - quotient.view(torch.int32)).abs()
    assert int(step.max()) == 1
    # bytes * s is within half a step of x: |q - x / s| <= 1/2, and the ratio's own rounding (half a step of f32 at 127)
    err = ((by.double() - 128) * s.double()[:, None] - x.double()).abs() / s.double()[:, None]
    assert float(err.max()) <= 0.5 + 127 * R.EPS
    x = x[other][:8]
    n = len(x)
    t, pages = R.make("write", 1, 1, 64, 8, 2, [n], [n], chunk=n, dtype=dtype, quant=True)
    t["K"][0, :, 0], t["V"][0, :, 0] = x, -x
    p = irgen.cache_write_ir(1, n, 1, 64, pages, 8, 2, dtype, True)
    want = R.write_ref(t, 8, True)
    for opts in ({}, {"patterns": False}):
        got, code, _ = PE.run(p, t, opts)
        assert code == 0
        for name in want:
            same(got[name], want[name], name)


# ---- streams by their handles ----------------------------------------------------------------


class PlanExecutable(Executable):
    """Allocates a call's scratch as the real one does."""

    def _device_tensor(self, shape, dtype):
        return torch.empty(shape, dtype=dtype)


def test_a_call_allocates_on_the_stream_it_launches_on(recorder, monkeypatch):
    # 0 and 1 are the handles of the default stream, which torch makes no external stream of (it gives another one, or
    # refuses); 2 is another stream in every thread
    t, problems = step_problems()
    p = problems[1]
    ex = PlanExecutable(compile_graph(Graph.from_dict(p.graph), p.meta(), RUNS), device=0)
    on, empty = [], torch.empty

    @contextlib.contextmanager
    def stream(s):
        on.append(s)
        yield
        on.append(None)
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda h, device=None: ("external", h, str(device)))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: ("default", str(device)))
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **kw: empty(*a, **kw))
    for handle, want in ((55, ("external", 55, "cuda:0")), (0, ("default", "cuda:0")), (1, ("default", "cuda:0"))):
        on.clear()
        ex.run(t, handle)
        assert on == [want, None] and recorder.log[-1][-1] == handle
    recorder.log.clear()
    with pytest.raises(ValueError, match="per-thread"):
        ex.run(t, 2)
    assert recorder.log == []
