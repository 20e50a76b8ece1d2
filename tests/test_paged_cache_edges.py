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
