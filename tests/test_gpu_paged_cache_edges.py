"""The paged key/value cache at the edges of what its definition allows, on a B200 against plain float64 (the CPU's
cases and references: :mod:`tests.test_paged_cache_edges`, :mod:`tests.pagedref`)."""
import ctypes
import threading

import pytest
import torch

from emmy_ptx_b200 import data
from emmy_ptx_b200.compiler import compile_graph
from emmy_ptx_b200.ir import Graph
from emmy_ptx_b200.runtime import Executable
from tests import pagedref as R
from tests.test_paged_cache_edges import (QSIZES, RANGES, RUNS, SIGNED, SIGNS, check_scaled, joined, other_first, ramp_case, signed_case,
                                          sized_case, step_problems, step_refs)
from tests.test_paged_cache import same

pytestmark = pytest.mark.gpu


def go(p, t, opts=None):
    ex = Executable(compile_graph(Graph.from_dict(p.graph), p.meta(), opts or {}), device=0)
    g = {k: v.cuda() for k, v in t.items()}
    ex(g)
    torch.cuda.synchronize()
    ex.check()
    ex.close()
    return {a.name: g[a.name].cpu() for a in p.outputs}


@pytest.mark.parametrize("opts", [{"paged_rows": 0}, {"paged_rows": 64}, {"patterns": False}],
                         ids=["tiles", "rows", "CUDA-cores"])
@pytest.mark.parametrize("signs", SIGNS)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", SIGNED, ids=["decode", "draft-runs"])
def test_scales_of_any_sign(case, dtype, signs, opts):
    t, p = signed_case(case, dtype, signs)
    got = go(p, t, {**case[-1], **opts})
    ref, bound, _ = R.attention_ref(t, case[5])
    R.check(got["O"], ref, bound, signs)


@pytest.mark.parametrize("opts", [{"paged_ctas": 0}, {"paged_ctas": 3, "paged_min_tiles": 1}], ids=["whole", "runs"])
@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("n", [230, 8000])
@pytest.mark.parametrize("quant,k", [*RANGES, (True, 112), (False, 112)])
def test_values_near_the_ends_of_f32(quant, k, n, rows, opts):
    if k == 119 and n == 8000:
        k = 114                                               # the weights sum to more: 2^119 would leave f32 with any kernel
    t, big, p = ramp_case(quant, k, n)
    base = go(p, t, {**opts, "paged_rows": rows})["O"]
    got = go(p, big, {**opts, "paged_rows": rows})["O"]
    ref, bound, _ = R.attention_ref(t, 16)
    R.check(base, ref, bound, "before")
    check_scaled(got, base, k)


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("q2,k2,scale", QSIZES)
def test_queries_of_any_size_over_bytes(q2, k2, scale, rows):
    t, p = sized_case(q2, k2, scale)
    ref, bound, _ = R.attention_ref(t, 16, scale=scale)
    R.check(go(p, t, {"paged_rows": rows})["O"], ref, bound, "sizes")


def step_graph(more=(), opts=None):
    t, problems = step_problems()
    g, meta = joined(*more, *problems)
    return t, Executable(compile_graph(Graph.from_dict(g), meta, opts or RUNS), device=0)


def check_step(g, t):
    want, ref, bound = step_refs(t, False)
    R.check(g["O"], ref, bound, "step")
    for n in ("KC", "VC", "KR", "VR"):
        same(g[n].cpu(), want[n], n)


def test_a_serving_step_as_one_graph():
    """Write, attend and read back as one module's plans: called, and captured and replayed with other inputs."""
    t, ex = step_graph()
    assert len(ex.plans) == 4
    g = {k: v.cuda() for k, v in t.items()}
    ex(g)
    torch.cuda.synchronize()
    check_step(g, t)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=s):
        ex(g)
    gen = torch.Generator().manual_seed(9)
    host = {k: v.cpu().clone() for k, v in g.items()}
    for n in ("K", "V", "Q"):
        host[n] = torch.randn(host[n].shape, generator=gen).to(host[n].dtype)
        g[n].copy_(host[n])
    host["lens"] += 1
    g["lens"].copy_(host["lens"])
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    check_step(g, host)
    ex.check()


def test_a_cache_operator_beside_another_kernel():
    """A kernel that is no cache operator in the same module: the general path, on the current stream, on a stream
    given by its handle, and captured."""
    q = other_first()
    t, ex = step_graph([q])
    assert ex.plans is None
    t = {**t, **data.make_inputs(q)}
    g = {k: v.cuda() for k, v in t.items()}
    x = next(a.name for a in q.inputs)
    total = t[x].double().sum().item()
    tol = t[x].numel() * 2.0 ** -24 * t[x].double().abs().sum().item()            # an f32 sum in any order

    def fresh():
        for n in t:
            g[n].copy_(t[n])
        torch.cuda.synchronize()

    def check():
        torch.cuda.synchronize()
        check_step(g, t)
        assert abs(g["out"].double().sum().item() - total) <= tol
    ex(g)
    check()
    fresh()
    s = torch.cuda.Stream()
    ex.run(g, s.cuda_stream)
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ex(g)
    for _ in range(2):
        fresh()
        graph.replay()
        check()
    ex.check()


def test_a_thread_without_a_context_has_none_after_a_call():
    cuda = ctypes.CDLL("libcuda.so.1")
    t, problems = step_problems()
    p = problems[0]
    ex = Executable(compile_graph(Graph.from_dict(p.graph), p.meta()), device=0)
    g = {k: v.cuda() for k, v in t.items()}
    stream, seen = torch.cuda.Stream(), []
    torch.cuda.synchronize()

    def current():
        ctx = ctypes.c_void_p()
        assert cuda.cuCtxGetCurrent(ctypes.byref(ctx)) == 0
        return ctx.value

    def work():
        seen.append(current())
        ex.run(g, stream.cuda_stream)
        seen.append(current())
    th = threading.Thread(target=work)
    th.start()
    th.join()
    stream.synchronize()
    assert seen == [None, None]
    want = R.write_ref(t, 16, False)
    for n in want:
        same(g[n].cpu(), want[n], n)
    assert current() is not None
    mine = current()
    ex(g)
    assert current() == mine


def test_the_default_stream_by_its_handle(monkeypatch):
    t, problems = step_problems()
    p = problems[1]
    ex = Executable(compile_graph(Graph.from_dict(p.graph), p.meta(), RUNS), device=0)
    g = {k: v.cuda() for k, v in t.items()}
    ref, bound, _ = R.attention_ref(t, 16)
    seen, empty, side = [], torch.empty, torch.cuda.Stream()
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: (seen.append(torch.cuda.current_stream().cuda_stream), empty(*a, **kw))[1])
    for current in (torch.cuda.default_stream(), side):
        for handle, want in ((0, 0), (1, 0), (side.cuda_stream, side.cuda_stream)):
            g["O"].fill_(7)
            torch.cuda.synchronize()
            seen.clear()
            with torch.cuda.stream(current):
                ex.run(g, handle)
            torch.cuda.synchronize()
            assert seen == [want]
            R.check(g["O"], ref, bound, handle)
    ex.check()


def test_a_call_captured_by_its_handle_owns_its_scratch():
    """What the graph's call allocated stays the graph's: memory taken and filled later is not what a replay writes."""
    t, problems = step_problems()
    p = problems[1]
    ex = Executable(compile_graph(Graph.from_dict(p.graph), p.meta(), RUNS), device=0)
    g = {k: v.cuda() for k, v in t.items()}
    ref, bound, _ = R.attention_ref(t, 16)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        ex.run(g, s.cuda_stream)
    with torch.cuda.stream(s):
        n = sum(k for k, _ in ex._temp.values())
        junk = [torch.full((n,), float("nan"), device="cuda") for _ in range(32)]
    for _ in range(3):
        g["O"].fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        R.check(g["O"], ref, bound, "replay")
    assert all(bool(x.isnan().all()) for x in junk)
    ex.check()
