"""shared_prefix_attention where magnitudes differ: between the queries of a batch, and between the values of a row's keys.

Tolerances, per element of a row of queries, with p the softmax weights and u = eps / 2 of the output's type:
* u * (sum p|v| + |out|) for the weights' and the output's rounding, and (2 d + 64 * 2^-24) sum p|v| for scores that are off
  by at most d, exp2 and the join.  d = (D + 8) * 2^-24 * scale * max_j sum |q||k_j|, and for bf16 queries that became fp16
  numbers D * 2^-29 * scale * max|q| * max|k|: a row's power of two leaves its largest at 2^4 or more, where 2^-25, half the
  least fp16 step, is 2^-29 of it.
* Weights of an 8-bit cache, times the value's scale, are fp16 numbers relative to the largest of their row so far, which is
  at 2^6 or more: one below 2^-14 is off by 2^-25, 2^-31 of the largest.  Over n keys n * 2^-31 * max_j p_j max|v_j|.
* Weights of an fp16 cache are fp16 numbers relative to the largest weight, which is at 2^7 or more, whatever the values are:
  each is off by 2^-25, so 2^-32 max p, which its value multiplies: 2^-32 max p * sum |v_j|.
"""
import math

import pytest
import torch

from oracle import cache_ops_oracle as o
from tests.test_gpu_cache_ops import BF16, FP16, attention_case, gen, run_attention, status

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def op(cuda_device):
    import pcie_through  # noqa: F401

    torch.ops.pcie_through.device_status()
    return torch.ops.pcie_through


def check_rows(c, out, lse, rows):
    """The rows of queries that `rows` ([seqs, q_heads] truth values) names, against the definition in 64 bits."""
    k, v = (o.values(c[x], c["block"], c["heads"], c["dim"], c["fmt"]).double() for x in ("k", "v"))
    kp, ok = o.rows_of(k, c["prefix_table"], c["prefix"], c["block"])
    vp, _ = o.rows_of(v, c["prefix_table"], c["prefix"], c["block"])
    assert ok.all()
    out, lse = out.cpu().double(), lse.cpu().double()
    u, group = torch.finfo(c["q"].dtype).eps / 2, c["q"].shape[1] // c["heads"]
    assert rows.any()
    for s, head in rows.nonzero().tolist():
        n, h = int(c["lens"][s]), head // group
        kk = torch.cat([kp, o.rows_of(k, c["tables"][s], n, c["block"])[0]])[:, h]
        vv = torch.cat([vp, o.rows_of(v, c["tables"][s], n, c["block"])[0]])[:, h]
        q = c["q"][s, head].double()
        z = kk @ q * c["scale"]
        p = torch.softmax(z, 0)
        want, spread = p @ vv, p @ vv.abs()
        d = (c["dim"] + 8) * 2 ** -24 * abs(c["scale"]) * (kk.abs() @ q.abs()).max()
        if c["fmt"] != "raw" and c["q"].dtype == BF16:
            d = d + c["dim"] * 2 ** -29 * abs(c["scale"]) * q.abs().max() * kk.abs().max()
        tol = u * (spread + want.abs()) + (2 * d + 64 * 2 ** -24) * spread
        if c["fmt"] != "raw":
            tol = tol + len(kk) * 2 ** -31 * (p * vv.abs().amax(1)).max()
        elif c["q"].dtype == FP16:
            tol = tol + 2 ** -32 * p.max() * vv.abs().sum(0)
        if c["q"].dtype == FP16:
            tol = tol + 2 ** -25                                   # the output's least step
        worst = float(((out[s, head] - want).abs() / tol).max())
        assert worst <= 1, f"row {s}, {head}: {worst:.2f} of the bound"
        true_lse = torch.logsumexp(z, 0)
        assert abs(lse[s, head] - true_lse) <= d + 64 * 2 ** -24 * (1 + true_lse.abs())


# ------------------------------------------------------------------ queries ---
@pytest.mark.parametrize("fmt", ["e4m3", "int8", "raw"])
@pytest.mark.parametrize("seqs,group,dim,aiv", [(40, 4, 128, None), (9, 4, 64, 1), (70, 5, 128, 1), (2, 4, 128, None)])
def test_a_row_does_not_see_its_neighbours_queries(op, cuda_device, fmt, seqs, group, dim, aiv):
    """Ordinary rows of a batch in which single heads have queries of 1e6 to the largest finite number, as rows that nobody
    wrote (padding of a captured batch) may have."""
    c = attention_case(fmt, BF16, 1, group, dim, 16, 300, [5, 0, 33] * (seqs // 3) + [1] * (seqs % 3), seed=1)
    ordinary = torch.ones(seqs, group, dtype=torch.bool)
    for i, power in enumerate((1e6, 1e10, 1e12, 1e20, 1e30, 3e38)):
        s, head = (i * 7 + 1) % seqs, i % group
        c["q"][s, head] = (torch.randn(dim, generator=gen(i)).clamp(-1, 1) * power).to(BF16)
        ordinary[s, head] = False
    ordinary[0] = True
    c["q"][0] = (torch.randn(group, dim, generator=gen(9)) * 2).to(BF16)
    out, lse = run_attention(op, c, cuda_device, aiv=aiv)
    assert status() == 0
    check_rows(c, out, lse, ordinary)
    # the same rows in a batch of ordinary queries: what a row gets does not hang on the others beyond rounding
    assert out.isfinite().all(-1)[ordinary.to(cuda_device)].all()


@pytest.mark.parametrize("fmt,dtype,dim", [("e4m3", BF16, 128), ("int8", FP16, 128), ("int8", BF16, 64), ("raw", BF16, 128)])
def test_alternating_batches_give_the_same_bits(op, cuda_device, fmt, dtype, dim):
    """Two batches with caches, pages and prefixes of their own, in turn: what a CTA's shared memory holds of the call before is
    never used (the places of a tile's rows are all written when the first of them is read)."""
    cases = [attention_case(fmt, dtype, 1, 4, dim, 16, prefix, [3, 0, 20] * 4, seed=prefix) for prefix in (1900, 700)]
    dev = [{n: c[n].to(cuda_device) for n in ("q", "k", "v", "prefix_table", "tables", "lens")} for c in cases]
    for aiv in (1, None):
        first = [run_attention(op, c, cuda_device, aiv=aiv) for c in cases]
        for c, (out, lse) in zip(cases, first):
            check_rows(c, out, lse, torch.ones(c["q"].shape[:2], dtype=torch.bool))
        out, lse = [torch.empty_like(x) for x in first[0]]
        for _ in range(100):
            for c, d, (want, want_lse) in zip(cases, dev, first):
                op.shared_prefix_attention(d["q"], out, d["k"], d["v"], d["prefix_table"], c["prefix"], d["tables"], d["lens"], 16, 1,
                                           {"raw": 0, "e4m3": 1, "int8": 2}[fmt], c["scale"], lse, None, aiv)
                assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("scale", [0.11, -0.11])
def test_queries_that_grow_from_row_to_row(op, cuda_device, fmt, scale):
    """Rows of all magnitudes from 2^-30 to 2^30, with scores of order one in the rows that `scale` suits, masked pages and an
    odd end of the prefix in the same tiles."""
    c = attention_case(fmt, BF16, 1, 8, 128, 16, 517, [3] * 8, seed=5)
    power = torch.linspace(-30, 30, 64).round().view(8, 8, 1)
    c["q"] = (torch.randn(8, 8, 128, generator=gen(1)) * 2.0 ** power).to(BF16)
    c["q"][3, 3] = 0
    c["scale"] = scale
    for aiv in (None, 1):
        out, lse = run_attention(op, c, cuda_device, aiv=aiv)
        assert status() == 0
        check_rows(c, out, lse, torch.ones(8, 8, dtype=torch.bool))


def test_queries_far_below_their_neighbours(op, cuda_device):
    """Rows of 2^-112 next to rows of 2^56, keys of 2^66: the small rows' scores are 2^-40, so every key has the same weight."""
    c = attention_case("e4m3", BF16, 1, 2, 128, 16, 300, [2] * 40, seed=12)
    o.split_pages(c["k"], 16, 1, 128, "e4m3")[1].mul_(2.0 ** 66)
    c["q"] = torch.randn(40, 2, 128, generator=gen(3)).to(BF16)
    c["q"][:, 0] *= 2.0 ** -112
    c["q"][:, 1] *= 2.0 ** 56
    rows = torch.zeros(40, 2, dtype=torch.bool)
    rows[:, 0] = True
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0
    check_rows(c, out, lse, rows)


@pytest.mark.parametrize("seqs", [2, 40])
@pytest.mark.parametrize("dtype,powers", [(BF16, (8, 20, 25, 31, 40, 70)), (FP16, (8, 13))])
def test_scores_of_any_magnitude(op, cuda_device, seqs, dtype, powers):
    """16-bit caches, queries of up to 2^70: the scores' last place is far above one, and the largest has the weight 1."""
    c = attention_case("raw", dtype, 1, 4, 128, 16, 300, [5] * seqs, seed=8)
    c["scale"] = 1.0
    for power in powers:
        c["q"] = (torch.randn(seqs, 4, 128, generator=gen(power)).clamp(-3, 3) * 2.0 ** power).to(dtype)
        out, lse = run_attention(op, c, cuda_device)
        assert status() == 0
        check_rows(c, out, lse, torch.ones(seqs, 4, dtype=torch.bool))


# ------------------------------------------------------- scales of the values ---
def placed_case(fmt, dtype, dim, seqs, group, prefix, score, size, seed=0):
    """One K/V head; key j of the prefix has the score score[j] log2 e^-1 for every row (in units of log2, up to the cache's
    rounding) and values of about 2^size[j]."""
    c = attention_case(fmt, dtype, 1, group, dim, 16, prefix, [2] * seqs, seed=seed)
    g = gen(seed + 40)
    c["q"] = (0.01 * torch.randn(seqs, group, dim, generator=g)).to(dtype)
    c["q"][..., 0] = 2
    k = 0.01 * torch.randn(prefix, 1, dim, generator=g)
    k[:, 0, 0] = torch.as_tensor(score) * math.log(2) / 2
    c["scale"] = 1.0
    v = torch.randn(prefix, 1, dim, generator=g) * 2.0 ** torch.as_tensor(size, dtype=torch.float32)[:, None, None]
    at = torch.arange(prefix)
    slots = c["prefix_table"][at // 16] * 16 + at % 16
    o.write(k.to(dtype), c["k"], slots, 16, fmt)
    o.write(v.to(dtype), c["v"], slots, 16, fmt)
    for s in range(seqs):                                          # the own tokens: far below
        rows = torch.zeros(2, 1, dim)
        rows[:, 0, 0] = -200
        mine = c["tables"][s, 0] * 16 + torch.arange(2)
        o.write(rows.to(dtype), c["k"], mine, 16, fmt)
    return c


def check_all(op, device, c):
    for aiv in (None, 1):
        out, lse = run_attention(op, c, device, aiv=aiv)
        assert status() == 0
        check_rows(c, out, lse, torch.ones(c["q"].shape[:2], dtype=torch.bool))


@pytest.mark.parametrize("fmt,dtype", [("e4m3", BF16), ("int8", BF16), ("e4m3", FP16), ("int8", FP16)])
@pytest.mark.parametrize("seqs", [2, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_large_value_that_a_row_does_not_weigh(op, cuda_device, fmt, dtype, seqs, dim):
    """One key of the prefix has values 2^14 (fp16: 2^10) or, in bf16, 2^20 to 2^90 times the others' and a weight of 2^-60 and
    less: the others keep their bits, wherever the key lies."""
    n = 500
    for power, far in ((14, 60), (20, 60), (90, 190)) if dtype == BF16 else ((10, 60),):
        for place in (0, 130, n - 1):
            score, size = -torch.rand(n, generator=gen(power)) * 9, torch.zeros(n)
            score[place], size[place] = -far, power
            check_all(op, cuda_device, placed_case(fmt, dtype, dim, seqs, 2, n, score, size, seed=place))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("seqs", [2, 40])
@pytest.mark.parametrize("rise", [0.03, 0.3, -0.3])
def test_value_scales_that_rise_along_the_prefix(op, cuda_device, fmt, seqs, rise):
    """Values of 2^(rise j), so that o is rescaled from tile to tile while the rows' maxima stay; with the scores falling by as
    much every key counts, and with steep scores only one side does."""
    n = 400
    j = torch.arange(n)
    for slope in (0.0, -rise, -1.1 * rise):
        check_all(op, cuda_device, placed_case(fmt, BF16, 128, seqs, 2, n, slope * j - max(0.0, slope * n), rise * j - max(0.0, rise * n / 2), seed=3))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("seqs", [2, 40])
def test_a_first_key_with_a_large_weight_and_small_values(op, cuda_device, fmt, seqs):
    """The first key takes nearly all weight and has values of 2^-12 of the others' or none at all."""
    n = 300
    score, size = torch.full((n,), -16.0) - torch.rand(n, generator=gen(2)) * 4, torch.zeros(n)
    score[0] = 0
    for small in (-12, -200):
        size[0] = small
        check_all(op, cuda_device, placed_case(fmt, BF16, 128, seqs, 2, n, score, size, seed=4))
    c = placed_case(fmt, BF16, 128, seqs, 2, n, score, torch.full((n,), -200.0), seed=5)     # values of nothing but zeros
    out, _ = run_attention(op, dict(c, lens=torch.zeros(seqs, dtype=torch.int64)), cuda_device)
    assert (out == 0).all() and status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("seqs", [2, 40])
def test_values_of_nearly_the_largest_number(op, cuda_device, fmt, seqs):
    """Values of 2^120, and next to them values of 1 with a weight 2^100 times as large: sum and result stay finite and right."""
    n = 200
    score = -torch.rand(n, generator=gen(2)) * 30
    check_all(op, cuda_device, placed_case(fmt, BF16, 128, seqs, 2, n, score, torch.full((n,), 120.0), seed=6))
    size = torch.where(torch.arange(n) % 3 == 0, 100.0, 0.0)
    check_all(op, cuda_device, placed_case(fmt, BF16, 128, seqs, 2, n, score - size, size, seed=7))


@pytest.mark.parametrize("seqs", [2, 40])
def test_very_many_keys_of_very_small_weight(op, cuda_device, seqs):
    """An fp16 cache: one key with values of 0 takes nearly all weight, 16383 with a weight of 2^-25.5 each make up the result."""
    n = 16384
    score, size = torch.full((n,), -25.5), torch.zeros(n)
    score[5], size[5] = 0, -200
    c = placed_case("raw", FP16, 64, seqs, 2, n, score, size, seed=9)
    slots = c["prefix_table"][torch.arange(n) // 16], torch.arange(n) % 16
    c["v"][slots] = c["v"][slots].abs() + 1                          # of one sign, so that they do not cancel
    c["v"][slots[0][5], slots[1][5]] = 0
    check_all(op, cuda_device, c)
