"""The paged key/value cache at the edges of what its definition allows, on a B200 against plain float64 (the CPU's
cases and references: :mod:`tests.test_paged_cache_edges`, :mod:`tests.pagedref`)."""
import pytest
import torch

from emmy_ptx_b200.compiler import compile_graph
from emmy_ptx_b200.ir import Graph
from emmy_ptx_b200.runtime import Executable
from tests import pagedref as R
from tests.test_paged_cache_edges import QSIZES, RANGES, SIGNED, SIGNS, check_scaled, ramp_case, signed_case, sized_case

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
