"""The paged key/value cache at the edges of what its definition allows, on the CPU (emulated kernels, recording
devices) against plain float64."""
import pytest
import torch

from emmy_ptx_b200 import irgen
from tests import pagedemu as PE
from tests import pagedref as R

#: scales as other programs may leave them: a factor for every token of every head
SIGNS = {"negative": lambda n: -torch.ones(n), "alternating": lambda n: 1.0 - 2.0 * (torch.arange(n) % 2),
         "large-negative": lambda n: torch.where(torch.arange(n) % 7 == 3, -1024.0, 1.0)}
SIGNED = [
    # batch, chunk, heads, kv_heads, dim, page, max_pages, lens, fresh, options
    (1, 1, 4, 1, 64, 16, 8, [100], [1], {}),
    (2, 3, 4, 2, 128, 16, 13, [200, 40], [3, 2], {"paged_ctas": 5, "paged_min_tiles": 1}),
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
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", SIGNED, ids=["decode", "draft-runs"])
def test_scales_of_any_sign(case, dtype, signs, rows):
    t, p = signed_case(case, dtype, signs)
    got, code, _ = PE.run(p, t, {**case[-1], "paged_rows": rows})
    assert code == 0
    ref, bound, _ = R.attention_ref(t, case[5])
    R.check(got["O"], ref, bound, signs)
