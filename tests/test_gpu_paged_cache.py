"""The paged key/value cache operators on a B200 against plain float64 (:mod:`tests.pagedref`): every type, ragged
batches, padding, stale rows of NaN, missing pages, windows, split units, and the calls a serving program
makes: write then attend then read, captured and replayed, on another stream."""
import pytest
import torch

from emmy_ptx_b200 import irgen
from emmy_ptx_b200.compiler import compile_graph
from emmy_ptx_b200.ir import Graph
from emmy_ptx_b200.runtime import Executable
from tests import pagedref as R
from tests.test_paged_cache import ATTENDS, FORMS, READS, SPECIAL, SPREAD, TENSOR, WRITES, awkward_rows, broken_table, form_opts, same, with_specials

pytestmark = pytest.mark.gpu


def build(p, opts=None):
    return Executable(compile_graph(Graph.from_dict(p.graph), p.meta(), opts or {}), device=0)


def on_gpu(t):
    return {k: v.cuda() for k, v in t.items()}


def go(p, t, opts=None):
    ex = build(p, opts)
    g = on_gpu(t)
    ex(g)
    torch.cuda.synchronize()
    ex.check()
    kinds = [r["kind"] for r in ex.records]
    ex.close()
    return {a.name: g[a.name].cpu() for a in p.outputs}, kinds


@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("form,case", [(f, c) for f in FORMS for c in TENSOR if form_opts(f, c)],
                         ids=lambda c: c if isinstance(c, str) else "x".join(map(str, c[:7])))
def test_paged_attention(form, case, dtype, quant):
    B, C, H, hk, d, page, mp, lens, fresh, window, sinks, _ = case
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, dtype=dtype, quant=quant, seed=H + C)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, dtype, quant, window, sinks)
    got, kinds = go(p, t, form_opts(form, case))
    assert kinds[0] == FORMS[form]
    ref, bound, _ = R.attention_ref(t, page, window, sinks)
    R.check(got["O"], ref, bound, form)


@pytest.mark.parametrize("form", ["rows", "tiles"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", SPECIAL, ids=lambda c: "x".join(map(str, c[:5])))
def test_infinities_and_nans_reach_only_rows_that_see_them(case, dtype, form):
    C, H, hk, d, n, window, sinks, _ = case
    t, pages = with_specials(case, dtype, 16)
    p = irgen.paged_attention_ir(1, C, H, hk, d, pages, 16, t["table"].shape[1], dtype, False, window, sinks)
    ref, bound, _ = R.attention_ref(t, 16, window, sinks)
    for ctas in (0, 2):
        got, _ = go(p, t, {"paged_rows": 64 if form == "rows" else 0, "paged_ctas": ctas, "paged_min_tiles": 1})
        R.check(got["O"], ref, bound, form, inf_or_nan=True)


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("form,case", [(f, c) for f in FORMS for c in SPREAD if f == "tiles" or c[1] <= 32],
                         ids=lambda c: c if isinstance(c, str) else "x".join(map(str, c[:7])))
def test_paged_attention_runs_over_many_units(form, case, quant):
    B, C, H, hk, d, page, mp, lens, fresh, window, sinks = case
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, quant=quant, seed=B)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, "bf16", quant, window, sinks)
    ref, bound, _ = R.attention_ref(t, page, window, sinks)
    for ctas in (1, 2, 3, 4, 5, 7, 11, 40):
        got, _ = go(p, t, {"paged_rows": 64 if form == "rows" else 0, "paged_ctas": ctas, "paged_min_tiles": 1})
        R.check(got["O"], ref, bound, f"{form} {ctas}")


@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("f16", True)])
@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "x".join(map(str, c[:7])))
def test_paged_attention_cuda_cores(case, dtype, quant):
    B, C, H, hk, d, page, mp, lens, fresh, window, sinks = case
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, dtype=dtype, quant=quant, seed=H)
    if mp == 3:
        broken_table(t, pages)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, dtype, quant, window, sinks)
    got, _ = go(p, t, {"patterns": False})
    ref, bound, _ = R.attention_ref(t, page, window, sinks)
    R.check(got["O"], ref, bound, "CUDA cores")


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("B,C,H,hk,d,page,lens,window,sinks", [
    (3, 1, 8, 2, 128, 16, [2111, 63, 1024], None, 0),
    (2, 4, 12, 2, 64, 64, [1500, 700], None, 0),
    (1, 200, 4, 1, 128, 32, [900], None, 0),
    (1, 150, 6, 2, 64, 8, [1300], 333, 70),
    (4, 1, 16, 1, 128, 128, [2000, 1, 129, 800], 500, 4),
], ids=["decode", "draft", "chunk", "chunk-window", "decode-window"])
def test_paged_attention_longer(B, C, H, hk, d, page, lens, window, sinks, quant, rows):
    mp = -(-max(lens) // page) + 1
    fresh = [min(C, n) for n in lens]
    t, pages = R.make("attend", B, hk, d, page, mp, lens, fresh, chunk=C, heads=H, quant=quant, seed=d + C, sizes=2.0)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, "bf16", quant, window, sinks)
    got, kinds = go(p, t, {"paged_rows": rows})
    assert kinds[0] == FORMS["rows" if C * (H // hk) <= rows else "tiles"]
    ref, bound, _ = R.attention_ref(t, page, window, sinks)
    R.check(got["O"], ref, bound, "longer")


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("page", [8, 64])
def test_paged_attention_missing_pages(page, quant):
    mp = 320 // page
    t, pages = R.make("attend", 2, 1, 64, page, mp, [320, 250], [3, 3], chunk=3, heads=2, quant=quant, seed=page)
    t["table"][0, 1] = -1
    t["table"][0, mp - 2] = pages
    t["table"][1, 0] = 2 ** 31 - 1
    p = irgen.paged_attention_ir(2, 3, 2, 1, 64, pages, page, mp, "bf16", quant)
    ref, bound, _ = R.attention_ref(t, page)
    for rows in (0, 64):
        for opts in ({}, {"paged_ctas": 3, "paged_min_tiles": 2}):
            got, _ = go(p, t, {**opts, "paged_rows": rows})
            R.check(got["O"], ref, bound, "missing pages")
    t["table"].fill_(-1)
    for rows in (0, 64):
        got, _ = go(p, t, {"paged_rows": rows})
        assert not got["O"][:, :3].any()


@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("f16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("case", WRITES, ids=lambda c: "x".join(map(str, c[:6])))
def test_cache_write(case, dtype, quant):
    B, C, hk, d, page, mp, lens, fresh = case
    t, pages = R.make("write", B, hk, d, page, mp, lens, fresh, chunk=C, dtype=dtype, quant=quant, seed=B + d)
    broken_table(t, pages)
    t["K"][0, 0, 0] = 0.0
    t["V"][0, 0, 0, 3] = float("inf")
    t["V"][-1, -1, -1, 5] = float("nan")
    awkward_rows(t, d)
    p = irgen.cache_write_ir(B, C, hk, d, pages, page, mp, dtype, quant)
    want = R.write_ref(t, page, quant)
    for opts, kind in (({}, "cache_write"), ({"patterns": False}, "generic")):
        got, kinds = go(p, t, opts)
        assert kinds == [kind]
        for n in want:
            same(got[n], want[n], f"{n} {kind}")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_cache_write_many_quotients(dtype):
    # a million rows' worth of quotients, many of them next to a half
    t, pages = R.make("write", 4, 8, 128, 64, 8, [512] * 4, [512] * 4, chunk=512, dtype=dtype, quant=True, seed=21)
    p = irgen.cache_write_ir(4, 512, 8, 128, pages, 64, 8, dtype, True)
    got, _ = go(p, t)
    for x in "KV":
        by, s = R.quantise(t[x])
        pg = t["table"].long().repeat_interleave(64, 1)
        row = (torch.arange(512) % 64).expand(4, 512)
        same(got[x + "C"][pg, :, row], by, x)
        same(got[x + "S"][pg, :, row], s, x)


@pytest.mark.parametrize("dtype,quant", [("bf16", False), ("bf16", True), ("f16", True)])
@pytest.mark.parametrize("case", READS, ids=lambda c: "x".join(map(str, c[:6])))
def test_cache_read(case, dtype, quant):
    B, L, hk, d, page, mp, lens = case
    t, pages = R.make("read", B, hk, d, page, mp, lens, [0] * B, length=L, dtype=dtype, quant=quant, seed=L)
    broken_table(t, pages)
    p = irgen.cache_read_ir(B, L, hk, d, pages, page, mp, dtype, quant)
    want = R.read_ref(t, page, dtype)
    for opts, kind in (({}, "cache_read"), ({"patterns": False}, "generic")):
        got, kinds = go(p, t, opts)
        assert kinds == [kind]
        for n in want:
            same(got[n], want[n], f"{n} {kind}")


@pytest.mark.parametrize("quant", [False, True])
def test_a_serving_step_captured_and_replayed(quant):
    """Write, attend and read back, as one decode step after another from one captured graph, on a stream of
    its own; lengths and inputs change between replays, as they do in serving."""
    B, H, hk, d, page, mp = 2, 4, 2, 64, 16, 6
    t, pages = R.make("write", B, hk, d, page, mp, [30, 61], [1, 1], quant=quant, seed=3)
    a, _ = R.make("attend", B, hk, d, page, mp, [30, 61], [1, 1], heads=H, quant=quant, seed=4)
    r, _ = R.make("read", B, hk, d, page, mp, [30, 61], [1, 1], length=mp * page, quant=quant, seed=5)
    t = {**r, **a, **t}
    common = (hk, d, pages, page, mp, "bf16", quant)
    steps = [build(irgen.cache_write_ir(B, 1, *common)), build(irgen.paged_attention_ir(B, 1, H, *common),
             {"paged_ctas": 3, "paged_min_tiles": 1}), build(irgen.cache_read_ir(B, mp * page, *common))]
    g = on_gpu(t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        for ex in steps:
            ex(g)                                            # warm-up: modules loaded, descriptors made
        with torch.cuda.graph(graph, stream=s):
            for ex in steps:
                ex(g)
    s.synchronize()
    host = {k: v.clone() for k, v in t.items()}
    host.update({k: v.cpu() for k, v in g.items()})          # the state after the warm-up
    gen = torch.Generator().manual_seed(9)
    for step in range(3):
        host["lens"] = host["lens"] + 1
        for n in ("K", "V", "Q"):
            host[n] = torch.randn(host[n].shape, generator=gen).to(host[n].dtype)
        for n in ("lens", "K", "V", "Q"):
            g[n].copy_(host[n])
        torch.cuda.current_stream().synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        s.synchronize()
        host.update(R.write_ref(host, page, quant))
        ref, bound, _ = R.attention_ref(host, page)
        R.check(g["O"], ref, bound, f"step {step}")
        back = R.read_ref(host, page, "bf16")
        host.update(back)
        for n in ("KC", "VC", "KR", "VR"):
            same(g[n].cpu(), host[n], f"{n} step {step}")
    for ex in steps:
        ex.check()


# ---- calls that overlap, other threads, sizes past 32 bits -------------------------------------


def decode_case(quant=False, seed=0, rows=64, B=3, C=1, lens=(700, 90, 1500), H=4, hk=2, d=64, page=16):
    mp = -(-max(lens) // page)
    t, pages = R.make("attend", B, hk, d, page, mp, list(lens), [min(C, n) for n in lens], chunk=C, heads=H, quant=quant,
                      seed=seed)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp, "bf16", quant)
    return t, build(p, {"paged_rows": rows, "paged_ctas": 9, "paged_min_tiles": 1})


@pytest.mark.parametrize("rows", [0, 64])
def test_calls_of_one_executable_overlap(rows):
    """Two streams run one Executable at a time, each with its own inputs, output and (the call's own) scratch."""
    t, ex = decode_case(rows=rows)
    assert ex.records[0]["scratch"]
    sets = [on_gpu(t), on_gpu({**t, "Q": torch.randn(t["Q"].shape).to(t["Q"].dtype)})]
    ex(sets[0]), ex(sets[1])
    torch.cuda.synchronize()
    want = [g["O"].clone() for g in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for g in sets:
            g["O"].fill_(7)
        torch.cuda.synchronize()
        for _ in range(8):
            for g, s in zip(sets, streams):
                with torch.cuda.stream(s):
                    ex(g)
        torch.cuda.synchronize()
        for g, w in zip(sets, want):
            assert torch.equal(g["O"], w)
    ex.check()


def test_two_graphs_of_one_executable_replay_at_once():
    t, ex = decode_case()
    sets = [on_gpu(t), on_gpu({**t, "Q": torch.randn(t["Q"].shape).to(t["Q"].dtype)})]
    want, graphs, streams = [], [], []
    for g in sets:
        ex(g)
        torch.cuda.synchronize()
        want.append(g["O"].clone())
        graphs.append(torch.cuda.CUDAGraph())
        streams.append(torch.cuda.Stream())
        with torch.cuda.graph(graphs[-1], stream=streams[-1]):
            for _ in range(4):
                ex(g)
    for _ in range(20):
        for g in sets:
            g["O"].fill_(7)
        torch.cuda.synchronize()
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for g, w in zip(sets, want):
            assert torch.equal(g["O"], w)
    ex.check()


def test_a_stream_given_by_its_handle():
    t, ex = decode_case()
    g = on_gpu(t)
    ex(g)
    torch.cuda.synchronize()
    want = g["O"].clone()
    s = torch.cuda.Stream()
    g["O"].fill_(7)
    torch.cuda.synchronize()
    for _ in range(5):
        ex.run(g, s.cuda_stream)
    s.synchronize()
    assert torch.equal(g["O"], want)


def test_a_call_from_another_thread():
    """A thread that has made no CUDA call before: the plan brings its context."""
    import threading
    t, ex = decode_case()
    g = on_gpu(t)
    ex(g)
    torch.cuda.synchronize()
    want = g["O"].clone()
    g["O"].fill_(7)
    torch.cuda.synchronize()
    stream, failed = torch.cuda.Stream(), []

    def work():
        try:
            ex.run(g, stream.cuda_stream)
        except Exception as err:                                 # reported by the test's own thread
            failed.append(err)
    th = threading.Thread(target=work)
    th.start()
    th.join()
    torch.cuda.synchronize()
    assert not failed and torch.equal(g["O"], want)


def test_an_empty_batch_of_lengths_keeps_what_is_there():
    """Lengths of zero, nothing new: the write and the read leave everything, attention answers its rows as unseen."""
    B, H, hk, d, page, mp = 3, 4, 2, 64, 16, 40
    for quant in (False, True):
        common = (hk, d, B * mp + 2, page, mp, "bf16", quant)
        w, _ = R.make("write", B, hk, d, page, mp, [0] * B, [0] * B, quant=quant, seed=1)
        got, _ = go(irgen.cache_write_ir(B, 1, *common), w)
        for n in got:
            same(got[n], w[n], n)
        r, _ = R.make("read", B, hk, d, page, mp, [0] * B, [0] * B, length=mp * page, quant=quant, seed=1)
        got, _ = go(irgen.cache_read_ir(B, mp * page, *common), r)
        for n in got:
            same(got[n], r[n], n)
        a, _ = R.make("attend", B, hk, d, page, mp, [0] * B, [0] * B, heads=H, quant=quant, seed=1)
        for rows in (0, 64):
            got, _ = go(irgen.paged_attention_ir(B, 1, H, *common), a, {"paged_rows": rows})
            ref, bound, _ = R.attention_ref(a, page)
            R.check(got["O"], ref, bound, "empty")


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("B,C,lens", [(140, 1, 700), (300, 1, 30)])
def test_more_sequences_than_a_prefix_sum_takes(B, C, lens, rows):
    H, hk, d, page = 2, 1, 64, 64
    gen = torch.Generator().manual_seed(B)
    ls = torch.randint(0, lens + 1, (B,), generator=gen).tolist()
    mp = -(-lens // page)
    t, pages = R.make("attend", B, hk, d, page, mp, ls, [min(C, n) for n in ls], chunk=C, heads=H, seed=B)
    p = irgen.paged_attention_ir(B, C, H, hk, d, pages, page, mp)
    got, _ = go(p, t, {"paged_rows": rows})
    ref, bound, _ = R.attention_ref(t, page)
    R.check(got["O"], ref, bound, "many sequences")


@pytest.mark.parametrize("rows", [0, 64])
@pytest.mark.parametrize("quant", [False, True])
def test_pages_named_twice(quant, rows):
    """Sequences that share the pages of a common beginning, and a page named twice by one sequence."""
    t, pages = R.make("attend", 2, 2, 64, 16, 20, [300, 310], [4, 2], chunk=4, heads=4, quant=quant, seed=8)
    t["table"][1, :9] = t["table"][0, :9]
    t["table"][0, 3] = t["table"][0, 5]
    p = irgen.paged_attention_ir(2, 4, 4, 2, 64, pages, 16, 20, "bf16", quant)
    ref, bound, _ = R.attention_ref(t, 16)
    for ctas in (0, 5):
        got, _ = go(p, t, {"paged_rows": rows, "paged_ctas": ctas, "paged_min_tiles": 1})
        R.check(got["O"], ref, bound, "shared pages")


@pytest.mark.parametrize("quant", [False, True])
def test_caches_past_32_bits(quant):
    """The same pages in a pool whose elements (and bytes) pass 2^32, first, last and around both powers, give the
    same bits as in a small one."""
    B, C, H, hk, d, page, mp = 2, 5, 4, 2, 128, 64, 4
    small, pages = R.make("write", B, hk, d, page, mp, [250, 199], [C, 3], chunk=C, quant=quant, seed=2)
    a, _ = R.make("attend", B, hk, d, page, mp, [250, 199], [C, 3], chunk=C, heads=H, quant=quant, seed=2)
    small["Q"], small["O"] = a["Q"], a["O"]
    r, _ = R.make("read", B, hk, d, page, mp, [250, 199], [C, 3], length=mp * page, quant=quant, seed=2)
    small["KR"], small["VR"] = r["KR"], r["VR"]
    for n in ("KC", "VC", "KS", "VS"):
        if n in a:
            small[n] = a[n]
    per = hk * page * d
    big = (1 << 32) // per + 9
    half, full = (1 << 31) // per, (1 << 32) // per
    where = torch.tensor([0, 1, half - 1, half, half + 1, full - 1, full, full + 1, big - 2, big - 1])[:pages]
    assert len(where) == pages
    g = on_gpu(small)
    h = dict(g)
    h["table"] = where[small["table"].long()].to(torch.int32).cuda()
    for n in ("KC", "VC", "KS", "VS"):
        if n in g:
            h[n] = torch.empty((big, *g[n].shape[1:]), dtype=g[n].dtype, device="cuda")
            h[n][where.cuda()] = g[n]
    for n in ("O", "KR", "VR"):
        h[n] = g[n].clone()
    for t, n in ((g, pages), (h, big)):
        common = (hk, d, n, page, mp, "bf16", quant)
        for p, opts in ((irgen.cache_write_ir(B, C, *common), {}), (irgen.paged_attention_ir(B, C, H, *common), {}),
                        (irgen.cache_read_ir(B, mp * page, *common), {})):
            ex = build(p, opts)
            ex(t)
            torch.cuda.synchronize()
            ex.check()
            ex.close()
    for n in ("O", "KR", "VR"):
        same(h[n].cpu(), g[n].cpu(), n)
    for n in ("KC", "VC", "KS", "VS"):
        if n in g:
            same(h[n][where.cuda()].cpu(), g[n].cpu(), n)
    tiles = [build(irgen.paged_attention_ir(B, C, H, hk, d, n, page, mp, "bf16", quant), {"paged_rows": 0})
             for n in (pages, big)]
    tiles[0](g), tiles[1](h)
    torch.cuda.synchronize()
    same(h["O"].cpu(), g["O"].cpu(), "tiles")
