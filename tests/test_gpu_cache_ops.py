"""The operators that fill and read the cache of an attention layer, against their definition.

Tolerances.  A rounding to type t is off by at most u = eps(t) / 2 relative to the value.
* 16-bit writes, codes, scales and read-back values are compared bit for bit: the definition names every rounding.
* norm and rotation run in fp32: mean, rsqrt, weight, two products and a sum are fewer than 32 roundings of 2^-24 of
  terms that are at most |a| + |b| of the pair; then one rounding to the output's type, or to a code (half a code step:
  2^-4 relative or 2^-10 of the scale for e4m3, half a scale for int8).
* attention: weights are rounded to q's type before the second product (u of each, so u * sum p|v| / l), the result
  once more (u * |out|).  The scores are fp32 sums of D products, off by at most (D + 8) * 2^-24 * scale * sum |q||k|; an
  error d of a score changes a weight by d relative, in numerator and denominator, so 2 d * sum p|v| / l.  exp2 and the
  joining of partial results: 64 * 2^-24 relative.  fp16 weights below 2^-14 are off by 2^-25 each, not relative.
"""
import ctypes as C
import math

import pytest
import torch

from oracle import cache_ops_oracle as o
from tests.helpers import u8

pytestmark = pytest.mark.gpu

FMT = {"raw": 0, "e4m3": 1, "int8": 2}
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def op(cuda_device):
    import pcie_through  # noqa: F401

    torch.ops.pcie_through.device_status()
    return torch.ops.pcie_through


def status():
    return int(torch.ops.pcie_through.device_status())


def gen(seed):
    return torch.Generator().manual_seed(seed)


def empty_pages(blocks, block, heads, dim, fmt, dtype, poison=0xFF):
    """CPU pages filled with bytes that are NaN in every 16-bit type, in e4m3 and in the scales."""
    if fmt == "raw":
        return torch.full((blocks, block, heads, dim), float("nan"), dtype=dtype)
    return torch.full((blocks, o.block_bytes(block, heads, dim, fmt)), poison, dtype=torch.uint8)


def filled_pages(blocks, block, heads, dim, fmt, dtype, seed, spread=1.0):
    rows = torch.randn(blocks * block, heads, dim, generator=gen(seed))
    rows *= (torch.randn(blocks * block, heads, 1, generator=gen(seed + 1)) * spread).exp() if spread != 1.0 else 1.0
    rows = rows.to(dtype)
    return o.write(rows, empty_pages(blocks, block, heads, dim, fmt, dtype), torch.arange(blocks * block), block, fmt)


def same(a, b):
    return torch.equal(u8(a.cpu()), u8(b.cpu()))


# ---------------------------------------------------------------- kv_write ---
@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,heads,dim,block", [(1, 8, 128, 16), (1, 1, 16, 1), (37, 2, 64, 8), (129, 3, 96, 16), (70, 5, 256, 7),
                                                    (513, 1, 128, 128), (33, 4, 48, 3)])
def test_kv_write_is_bit_exact(op, cuda_device, fmt, dtype, tokens, heads, dim, block):
    blocks = -(-tokens // block) + 2
    x = torch.randn(tokens, 2, heads, dim, generator=gen(tokens + dim)).to(dtype)
    x[0, 0, 0] = 0                                                  # a row of zeros
    if tokens > 4:
        x[1] *= 1e-3
        x[2, :, :, 3] = 6e4                                          # one value far above the others
        x[3] = torch.finfo(dtype).tiny / 2 if dtype == BF16 else 6e-8
    slots = torch.randperm(blocks * block, generator=gen(7))[:tokens]
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]               # padding
    want = [o.write(x[:, i], empty_pages(blocks, block, heads, dim, fmt, dtype), slots, block, fmt) for i in range(2)]
    dev = x.to(cuda_device)
    for ids in (slots.to(cuda_device), slots.to(torch.int32).to(cuda_device)):
        got = [empty_pages(blocks, block, heads, dim, fmt, dtype).to(cuda_device) for _ in range(2)]
        op.kv_write(dev[:, 0], dev[:, 1], got[0], got[1], ids, block, FMT[fmt])   # strided slices of one tensor
        assert same(got[0], want[0]) and same(got[1], want[1])        # unwritten rows and padding bytes included
    assert status() == 0


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype,tokens,heads,dim,block", [(BF16, 8200, 1, 128, 16), (FP16, 1030, 8, 64, 16), (BF16, 2800, 3, 48, 8),
                                                          (FP16, 1700, 5, 256, 7), (BF16, 9000, 1, 16, 16), (FP16, 1400, 6, 112, 32)])
def test_kv_write_of_many_rows_is_bit_exact(op, cuda_device, fmt, dtype, tokens, heads, dim, block):
    test_kv_write_is_bit_exact(op, cuda_device, fmt, dtype, tokens, heads, dim, block)


def test_kv_write_rows_with_inf_or_nan_read_back_as_nan(op, cuda_device):
    for fmt in ("e4m3", "int8"):
        x = torch.ones(3, 2, 64, dtype=BF16)
        x[0, 0, 5], x[1, 1, 0] = float("inf"), float("nan")
        pages = empty_pages(1, 16, 2, 64, fmt, BF16, poison=0).to(cuda_device)
        d = x.to(cuda_device)
        op.kv_write(d, d, pages, pages.clone(), torch.arange(3, device=cuda_device), 16, FMT[fmt])
        v = o.values(pages.cpu(), 16, 2, 64, fmt)[0]
        assert v[0, 0].isnan().all() and v[1, 1].isnan().all()
        assert (v[0, 1] == 1).all() and (v[1, 0] == 1).all() and (v[2] == 1).all()
    assert status() == 0


def test_kv_write_slot_beyond_the_cache_is_skipped_and_reported(op, cuda_device):
    x = torch.randn(4, 1, 64, generator=gen(3)).to(BF16)
    pages = empty_pages(2, 4, 1, 64, "e4m3", BF16)
    slots = torch.tensor([7, 8, 0, 1 << 40])
    want = o.write(x, pages.clone(), slots, 4, "e4m3")
    got = pages.to(cuda_device)
    op.kv_write(x.to(cuda_device), x.to(cuda_device), got, got.clone(), slots.to(cuda_device), 4, 1)
    assert same(got, want) and status() == 0x1


def test_kv_write_and_read_back_beyond_4_gib(op, cuda_device):
    """Pages whose byte offset does not fit 32 bits."""
    block, heads, dim = 16, 8, 128
    page = o.block_bytes(block, heads, dim, "e4m3")
    blocks = (5 << 30) // page
    cache = torch.zeros(2, blocks, page, dtype=torch.uint8, device=cuda_device)
    ids = torch.tensor([blocks - 1, 3, blocks - 7], device=cuda_device)
    x = torch.randn(40, heads, dim, generator=gen(1)).to(BF16)
    slots = (ids.cpu()[torch.arange(40) // block] * block + torch.arange(40) % block)
    d = x.to(cuda_device)
    op.kv_write(d, d, cache[0], cache[1], slots.to(cuda_device), block, 1)
    ptr = [torch.tensor([c.data_ptr()], device=cuda_device) for c in cache]
    out = torch.zeros(2, 1, 40, heads, dim, dtype=FP32, device=cuda_device)
    op.paged_gather_dequant(ptr[0], ptr[1], out[0], out[1], ids[None], torch.tensor([40], device=cuda_device), block, blocks, 1)
    codes, scales = o.encode(x, "e4m3")
    want = codes.float() * scales.unsqueeze(-1)
    assert torch.equal(out[0, 0].cpu(), want) and torch.equal(out[1, 0].cpu(), want)
    q = torch.randn(1, heads, dim, generator=gen(2)).to(BF16).to(cuda_device)
    res, lse = torch.empty_like(q), torch.empty(1, heads, device=cuda_device)
    op.shared_prefix_attention(q, res, cache[0], cache[1], ids, 16, ids[None, 1:], torch.tensor([24], device=cuda_device), block, heads, 1,
                               None, lse)
    z = torch.einsum("hd,thd->ht", q[0].cpu().double(), want.double()) * dim ** -0.5
    assert torch.allclose(lse[0].cpu().double(), torch.logsumexp(z, 1), atol=1e-4)
    assert status() == 0


# ------------------------------------------------------ qk_norm_rope_write ---
@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype,tokens,heads,group,dim,rot,interleaved,norm", [
    (BF16, 1, 8, 4, 128, 128, False, "qk"), (FP16, 5, 2, 7, 128, 64, True, "qk"), (BF16, 40, 1, 1, 64, 64, False, ""),
    (FP16, 33, 3, 2, 96, 96, False, "k"), (BF16, 17, 2, 3, 256, 32, True, "q"), (FP16, 9, 1, 8, 48, 16, False, "qk"),
    (BF16, 6, 2, 2, 80, 48, False, "qk"), (BF16, 6, 2, 2, 128, 0, False, "qk")])
def test_qk_norm_rope_write(op, cuda_device, fmt, dtype, tokens, heads, group, dim, rot, interleaved, norm):
    from heterofusedkernels_b200.connector import rope_table

    block, hq, eps, longest = 16, heads * group, 1e-5, 4000
    blocks = -(-tokens // block) + 1
    qkv = (torch.randn(tokens, hq + 2 * heads, dim, generator=gen(dim + tokens)) * 3).to(dtype)
    q, k, v = qkv.split([hq, heads, heads], 1)
    wq, wk = (1 + 0.2 * torch.randn(2, dim, generator=gen(5))).to(dtype)
    wq, wk = (wq if "q" in norm else None), (wk if "k" in norm else None)
    table = rope_table(longest, rot, 1e4, device="cpu") if rot else torch.zeros(longest, 0)
    positions = torch.randint(0, longest, (tokens,), generator=gen(6))
    positions[0] = longest - 1
    slots = torch.randperm(blocks * block, generator=gen(7))[:tokens]
    if tokens > 4:
        slots[2], positions[2] = -1, -5                                # a padding row needs no position
    want_q = o.norm_rope(q, positions.clamp(min=0), table, wq, eps, interleaved)
    want_k = o.norm_rope(k, positions.clamp(min=0), table, wk, eps, interleaved)
    dev = qkv.to(cuda_device)
    dq, dk, dv = dev.split([hq, heads, heads], 1)
    up = lambda t: None if t is None else t.to(cuda_device)  # noqa: E731
    kc, vc = (empty_pages(blocks, block, heads, dim, fmt, dtype).to(cuda_device) for _ in range(2))
    out = torch.full((tokens, hq, dim), 7.0, dtype=dtype, device=cuda_device)
    op.qk_norm_rope_write(dq, dk, dv, out, kc, vc, up(slots), up(positions).to(torch.int32), up(table), block, FMT[fmt], up(wq), up(wk),
                          eps, interleaved)
    assert status() == 0
    # V is written as kv_write does, bit for bit
    assert same(vc, o.write(v, empty_pages(blocks, block, heads, dim, fmt, dtype), slots, block, fmt))
    u = torch.finfo(dtype).eps / 2
    row = lambda x: x.abs().amax(-1, keepdim=True) * 2  # noqa: E731  (|a| + |b| of a pair)
    live = slots >= 0
    err = (out.cpu().double() - want_q).abs()
    assert (err <= u * want_q.abs() + 32 * 2 ** -24 * row(want_q) + 2 ** -25)[live].all()
    assert (out.cpu()[~live] == 7).all()
    held = o.values(kc.cpu(), block, heads, dim, fmt).double().flatten(0, 1)
    got, want = held[slots[live]], want_k[live]
    slop = 32 * 2 ** -24 * row(want)
    if fmt == "raw":
        bound = u * want.abs() + slop + 2 ** -25
    else:
        scale = want.abs().amax(-1, keepdim=True) / o.TOP[fmt]
        bound = (torch.maximum(2 ** -4 * want.abs(), 2 ** -10 * scale) if fmt == "e4m3" else 0.5 * scale) * 1.0001 + slop
    assert ((got - want).abs() <= bound).all()
    used = torch.zeros(blocks * block, dtype=torch.bool)
    used[slots[live]] = True
    assert held[~used].isnan().all()
    # in place
    op.qk_norm_rope_write(dq, dk, dv, dq, kc, vc, up(slots), up(positions), up(table), block, FMT[fmt], up(wq), up(wk), eps, interleaved)
    assert torch.equal(dq[live.to(cuda_device)], out[live.to(cuda_device)])


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype,tokens,heads,group,dim,rot,interleaved,norm", [
    (BF16, 1400, 2, 4, 128, 128, False, "qk"), (FP16, 1000, 2, 7, 128, 64, True, "qk"), (BF16, 5500, 1, 1, 64, 64, False, ""),
    (FP16, 1400, 3, 2, 96, 96, False, "k"), (BF16, 1700, 2, 3, 256, 32, True, "q"), (FP16, 1700, 1, 8, 48, 16, False, "qk"),
    (BF16, 2100, 2, 2, 80, 48, False, "qk"), (BF16, 2100, 2, 2, 128, 0, False, "qk"), (FP16, 2100, 2, 2, 16, 16, False, "qk")])
def test_qk_norm_rope_write_of_many_rows(op, cuda_device, fmt, dtype, tokens, heads, group, dim, rot, interleaved, norm):
    test_qk_norm_rope_write(op, cuda_device, fmt, dtype, tokens, heads, group, dim, rot, interleaved, norm)


def test_norm_rope_position_outside_the_table_is_skipped_and_reported(op, cuda_device):
    from heterofusedkernels_b200.connector import rope_table

    x = torch.randn(3, 4, 64, generator=gen(1)).to(BF16).to(cuda_device)
    table = rope_table(10, 64)
    pages = empty_pages(1, 4, 1, 64, "raw", BF16).to(cuda_device)
    v, out = pages.clone(), torch.zeros(3, 2, 64, dtype=BF16, device=cuda_device)
    op.qk_norm_rope_write(x[:, :2], x[:, 2:3], x[:, 3:], out, pages, v, torch.arange(3, device=cuda_device),
                          torch.tensor([0, 10, -1], device=cuda_device), table, 4, 0)
    assert status() == 0x40
    assert (out[1:] == 0).all() and pages[0, 1:].isnan().all() and v[0, 1:].isnan().all()
    assert torch.equal(out[0], x[0, :2]) and torch.equal(pages[0, 0], x[0, 2:3])      # position 0 turns nothing


# ---------------------------------------------------- paged_gather_dequant ---
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("out_type", [BF16, FP16, FP32])
@pytest.mark.parametrize("layers,lens,heads,dim,block", [(2, [40, 100], 8, 128, 16), (1, [1], 1, 16, 1), (3, [0, 5, 0, 17, 64], 2, 64, 8),
                                                         (2, [300, 1, 33], 3, 96, 7), (1, [257, 128], 1, 128, 128), (5, [9] * 70, 1, 256, 4)])
def test_paged_gather_dequant_is_exact(op, cuda_device, fmt, out_type, layers, lens, heads, dim, block):
    from heterofusedkernels_b200.workloads import block_tables_for

    blocks = sum(-(-n // block) for n in lens) + 4
    pages = [filled_pages(blocks, block, heads, dim, fmt, BF16, 10 * i) for i in range(2 * layers)]
    tables = block_tables_for(lens, block, blocks, 3)
    want = [torch.cat([o.rows_of(o.values(p, block, heads, dim, fmt), tables[s], n, block)[0] for s, n in enumerate(lens)])
            for p in pages]
    dev = [p.to(cuda_device) for p in pages]
    kp = torch.tensor([p.data_ptr() for p in dev[:layers]], device=cuda_device)
    vp = torch.tensor([p.data_ptr() for p in dev[layers:]], device=cuda_device)
    total = sum(lens)
    for ids in (torch.int64, torch.int32):
        k, v = torch.full((2, layers, total + 3, heads, dim), 5.0, dtype=out_type, device=cuda_device)
        op.paged_gather_dequant(kp, vp, k, v, tables.to(ids).to(cuda_device), torch.tensor(lens, dtype=ids, device=cuda_device), block,
                                blocks, FMT[fmt])
        for l in range(layers):
            assert torch.equal(k[l, :total].cpu(), want[l].to(out_type)) and torch.equal(v[l, :total].cpu(), want[layers + l].to(out_type))
        assert (k[:, total:] == 5).all() and (v[:, total:] == 5).all()       # rows behind the last sequence
    assert status() == 0


def test_paged_gather_dequant_bad_pages_and_lengths(op, cuda_device):
    pages = filled_pages(4, 8, 2, 64, "int8", BF16, 1).to(cuda_device)
    ptr = torch.tensor([pages.data_ptr()], device=cuda_device)
    tables = torch.tensor([[1, 9], [2, -1]], device=cuda_device)
    k, v = torch.full((2, 1, 32, 2, 64), 5.0, device=cuda_device)
    op.paged_gather_dequant(ptr, ptr, k, v, tables, torch.tensor([16, 8], device=cuda_device), 8, 4, 2)
    assert status() == 0x1
    held = o.values(pages.cpu(), 8, 2, 64, "int8")
    assert torch.equal(k[0, :8].cpu(), held[1]) and (k[0, 8:16] == 5).all() and torch.equal(v[0, 16:24].cpu(), held[2])
    op.paged_gather_dequant(ptr, ptr, k, v, tables[1:], torch.tensor([17], device=cuda_device), 8, 4, 2)
    assert status() & 0x8
    null = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    op.paged_gather_dequant(null, null, k, v, tables[1:], torch.tensor([8], device=cuda_device), 8, 4, 2)
    assert status() == 0x20


def test_paged_gather_dequant_of_more_than_1024_sequences(op, cuda_device):
    n = 1500
    pages = filled_pages(n, 4, 1, 64, "e4m3", BF16, 2)
    lens = torch.arange(n) % 5
    tables = torch.randperm(n, generator=gen(1))[:, None]
    want = torch.cat([o.values(pages, 4, 1, 64, "e4m3")[tables[s, 0], :lens[s]] for s in range(n)])
    d = pages.to(cuda_device)
    ptr = torch.tensor([d.data_ptr()], device=cuda_device)
    k, v = torch.zeros(2, 1, len(want), 1, 64, device=cuda_device)
    op.paged_gather_dequant(ptr, ptr, k, v, tables.to(cuda_device), lens.to(cuda_device), 4, n, 1)
    assert torch.equal(k[0].cpu(), want) and torch.equal(v[0].cpu(), want) and status() == 0


# ------------------------------------------------- shared_prefix_attention ---
def attention_case(fmt, dtype, heads, group, dim, block, prefix, lens, seed=0, spread=1.0, q_gain=2.0, bad=False):
    own = [-(-n // block) for n in lens]
    front = -(-prefix // block)
    blocks = sum(own) + front + 2
    k, v = (filled_pages(blocks, block, heads, dim, fmt, dtype, seed + 100 * i, spread) for i in range(2))
    perm = torch.randperm(blocks, generator=gen(seed))
    tables = torch.full((len(lens), max(own + [1]) + 1), -1)
    at = front
    for s, n in enumerate(own):
        tables[s, :n] = perm[at:at + n]
        at += n
    # what no sequence has written: NaN behind the last token of a page and in the pages of nobody
    for pages in (k, v):
        held = torch.zeros(blocks * block, dtype=torch.bool)
        for table, n in [(perm[:front], prefix)] + [(tables[s], n) for s, n in enumerate(lens)]:
            i = torch.arange(n)
            held[table[i // block] * block + i % block] = True
        dead = (~held).nonzero()[:, 0]
        if fmt == "raw":
            pages[dead // block, dead % block] = float("nan")
        else:
            codes, scales = o.split_pages(pages, block, heads, dim, fmt)
            codes.view(torch.uint8)[dead // block, dead % block] = 0xFF
            scales[dead // block, dead % block] = float("nan")
    q = (torch.randn(len(lens), heads * group, dim, generator=gen(seed + 9)) * q_gain).to(dtype)
    return dict(fmt=fmt, q=q, k=k, v=v, prefix_table=perm[:front].clone(), prefix=prefix, tables=tables, lens=torch.tensor(lens), block=block,
                heads=heads, dim=dim, scale=dim ** -0.5)


def run_attention(op, c, device, ids=torch.int64, q=None, out=None, **more):
    up = lambda t: t.to(ids).to(device)  # noqa: E731
    q = c["q"].to(device) if q is None else q
    out = torch.full_like(q, 3.0) if out is None else out
    lse = torch.full(q.shape[:2], 3.0, device=device)
    op.shared_prefix_attention(q, out, c["k"].to(device), c["v"].to(device), up(c["prefix_table"]), c["prefix"], up(c["tables"]),
                               up(c["lens"]), c["block"], c["heads"], FMT[c["fmt"]], c["scale"], lse, **more)
    return out, lse


def check_attention(c, out, lse, keys=None):
    held = [o.values(c[x], c["block"], c["heads"], c["dim"], c["fmt"]) for x in ("k", "v")]
    want, want_lse, spread, reach = o.attention(c["q"], held[0], held[1], c["prefix_table"], c["prefix"], c["tables"], c["lens"], c["block"],
                                                c["scale"])
    u = torch.finfo(c["q"].dtype).eps / 2
    score = (c["dim"] + 8) * 2 ** -24 * reach
    tol = u * (spread + want.abs()) + (2 * score + 64 * 2 ** -24)[..., None] * spread
    if c["q"].dtype == FP16:
        n = c["prefix"] + int(c["lens"].max()) if len(c["lens"]) else 0
        biggest = held[1].nan_to_num(0.0).abs().max()
        tol = tol + n * 2 ** -25 * biggest + 2 ** -25
    err = (out.cpu().double() - want).abs()
    assert not out.isnan().any()
    assert (err <= tol).all(), f"worst {float((err / tol.clamp(min=1e-30)).max()):.2f} of the bound"
    dead = want_lse == -math.inf
    assert (lse.cpu()[dead] == -math.inf).all() and (out.cpu()[dead] == 0).all()
    lse_err = (lse.cpu().double() - want_lse).abs()[~dead]
    assert (lse_err <= (score + 64 * 2 ** -24 * (1 + want_lse.abs()))[~dead]).all()


SHAPES = [
    # heads, group, dim, block, prefix, lens
    (1, 1, 64, 16, 0, [1]),
    (2, 4, 128, 16, 0, [0, 1, 15, 16, 17, 63, 64, 65, 200]),
    (1, 8, 128, 16, 33, [0, 5]),
    (4, 7, 64, 16, 130, [3, 0, 0, 129]),
    (2, 1, 128, 8, 64, [9, 70, 8]),
    (1, 5, 128, 7, 100, [50, 13, 0]),
    (1, 3, 64, 1, 3, [2, 40]),
    (1, 20, 128, 128, 300, [257, 1]),
    (2, 33, 64, 32, 40, [64]),
    (1, 16, 128, 16, 1000, list(range(0, 40))),
    (2, 4, 128, 16, 513, [0] * 17),
    (1, 8, 64, 128, 129, [7] * 40),
    (2, 2, 128, 48, 0, [0, 0, 0]),
    (1, 4, 128, 16, 2000, [1500]),
]


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_shared_prefix_attention(op, cuda_device, fmt, dtype, shape):
    c = attention_case(fmt, dtype, *shape, seed=len(shape[5]))
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0
    check_attention(c, out, lse)
    # int32 ids, few CTAs, a workspace of the caller's: the same numbers but for the order of sums
    need = op.shared_prefix_attention_workspace(c["q"].to(cuda_device), c["prefix"], c["tables"], c["block"], c["heads"], 3)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=cuda_device)
    out, lse = run_attention(op, c, cuda_device, ids=torch.int32, workspace=ws, aiv=3)
    assert status() == 0
    check_attention(c, out, lse)


LONG = [
    # rows on both sides of a tile of 128 and of a block of 256; key tiles on both sides of 128; many tiles for a CTA
    (1, 8, 128, 16, 2900, [20] * 5), (2, 1, 128, 16, 1157, [3] * 128), (1, 3, 64, 32, 900, [0, 5] * 22), (1, 7, 128, 128, 641, [1] * 37),
    (1, 2, 128, 16, 128, [0] * 129), (3, 40, 64, 8, 257, [17]), (1, 11, 128, 7, 390, [9, 0, 30, 2]),
]


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", LONG, ids=[str(i) for i in range(len(LONG))])
def test_attention_behind_a_longer_prefix(op, cuda_device, fmt, dtype, shape):
    """More than 32 rows of queries to a K/V head: the tensor-core kernel, with one CTA (every tile of the prefix in one run)
    and with as many as it likes."""
    c = attention_case(fmt, dtype, *shape, seed=11)
    for aiv in (None, 1):
        out, lse = run_attention(op, c, cuda_device, aiv=aiv)
        assert status() == 0
        check_attention(c, out, lse)
    again, lse_again = run_attention(op, c, cuda_device, aiv=1)
    assert torch.equal(out, again) and torch.equal(lse, lse_again)


@pytest.mark.parametrize("fmt", ["raw", "e4m3"])
@pytest.mark.parametrize("seqs", [3, 60])
@pytest.mark.parametrize("scale", [-0.11, 0.0, 3.0])
def test_attention_with_any_finite_scale(op, cuda_device, fmt, seqs, scale):
    """Negative scales turn the order of the keys round, 0 makes them equal; keys that do not count stay out."""
    c = attention_case(fmt, BF16, 1, 4, 128, 16, 133, [7, 0, 20] * (seqs // 3), seed=2, q_gain=0.5)
    c["scale"] = scale
    out, lse = run_attention(op, c, cuda_device)
    check_attention(c, out, lse)


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("seqs", [2, 50])
def test_attention_bad_prefix_pages_and_rising_maxima(op, cuda_device, fmt, seqs):
    """Pages that are not there, among them the first tile's whole, and keys whose scores rise from tile to tile, so that the
    maximum in use has to follow; both ways the prefix is read."""
    c = attention_case(fmt, BF16, 1, 2, 64, 16, 700, [5] * seqs, seed=6)
    steep = torch.linspace(0.05, 6, 700)
    x = torch.randn(700, 1, 64, generator=gen(3)).sign() * steep[:, None, None]
    at = torch.arange(700)
    slots = c["prefix_table"][at // 16] * 16 + at % 16
    o.write(x.to(BF16), c["k"], slots, 16, fmt)
    c["q"] = (torch.randn(seqs, 2, 64, generator=gen(4)).sign() * 0.7).to(BF16)
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0
    check_attention(c, out, lse)
    c["prefix_table"][:8] = -1                                     # keys 0..127
    c["prefix_table"][20] = 10 ** 6
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0x1
    check_attention(c, out, lse)
    c["prefix_table"][:] = -7
    c["lens"] = torch.zeros(seqs, dtype=torch.int64)
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0x1
    check_attention(c, out, lse)


@pytest.mark.parametrize("seqs", [2, 40])
def test_attention_queries_of_very_different_magnitude(op, cuda_device, seqs):
    """bf16 queries over an 8-bit cache become fp16 numbers times a power of two: rows from 1e-30 to 1e30, and zeros."""
    c = attention_case("e4m3", BF16, 1, 4, 128, 16, 150, [12] * seqs, seed=7)
    power = torch.linspace(-30, -1, seqs * 4).view(seqs, 4, 1)
    c["q"] = (torch.randn(seqs, 4, 128, generator=gen(1)) * 10.0 ** power).to(BF16)
    c["q"][0, 0] = 0
    out, lse = run_attention(op, c, cuda_device)
    check_attention(c, out, lse)
    c["q"] = (torch.randn(seqs, 4, 128, generator=gen(1)).double() * 10.0 ** (power.double() + 31)).to(BF16)
    c["scale"] = 1e-30
    out, lse = run_attention(op, c, cuda_device)
    check_attention(c, out, lse)


def test_attention_passes_nan_and_inf_of_queries_on(op, cuda_device):
    for fmt, seqs in (("raw", 2), ("raw", 40), ("int8", 2), ("int8", 40)):
        c = attention_case(fmt, BF16, 1, 2, 64, 16, 40, [3] * seqs, seed=1)
        c["q"][0, 1, 5], c["q"][1, 0, 0] = float("nan"), float("inf")
        out, _ = run_attention(op, c, cuda_device)
        assert out[0, 1].isnan().all() and out[1, 0].isnan().all()
        assert not out[0, 0].isnan().any() and not out[1, 1].isnan().any()


@pytest.mark.parametrize("fmt,dtype", [("e4m3", FP16), ("int8", FP16), ("int8", BF16), ("raw", BF16)])
def test_attention_scales_over_many_orders_of_magnitude(op, cuda_device, fmt, dtype):
    """Rows of the cache whose magnitudes differ by up to 2^20: weight times scale leaves the range of fp16 that is held with full precision."""
    c = attention_case(fmt, dtype, 2, 4, 128, 16, 200, [90, 300, 2], seed=3, spread=2.0, q_gain=0.05)
    out, lse = run_attention(op, c, cuda_device)
    check_attention(c, out, lse)


def test_attention_takes_strided_queries_and_in_place_output(op, cuda_device):
    c = attention_case("raw", BF16, 2, 4, 128, 16, 70, [20, 0, 33], seed=4)
    wide = torch.zeros(3, 12, 128, dtype=BF16, device=cuda_device)
    wide[:, 2:10] = c["q"].to(cuda_device)
    out, lse = run_attention(op, c, cuda_device, q=wide[:, 2:10], out=torch.zeros(8, 3, 128, dtype=BF16, device=cuda_device).transpose(0, 1))
    check_attention(c, out, lse)
    first = out.clone()
    out, lse = run_attention(op, c, cuda_device, q=wide[:, 2:10], out=wide[:, 2:10])
    assert torch.equal(out, first) and (wide[:, :2] == 0).all() and (wide[:, 10:] == 0).all()


def test_attention_bad_pages_and_lengths(op, cuda_device):
    c = attention_case("e4m3", BF16, 1, 4, 64, 16, 40, [30, 20], seed=5)
    c["tables"][0, 1], c["prefix_table"][1] = 999, -3
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0x1
    check_attention(c, out, lse)
    c = attention_case("raw", FP16, 1, 4, 64, 16, 40, [32, 20], seed=5)
    c["tables"] = c["tables"][:, :2].contiguous()
    c["lens"] = torch.tensor([33, -1])                              # clamped to 32 and 0
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0x8
    check_attention(c, out, lse)
    c["lens"] = torch.tensor([1 << 40, 1 << 33])
    c["tables"][1] = c["tables"][0]
    out, lse = run_attention(op, c, cuda_device)
    assert status() == 0x8
    check_attention(c, out, lse)


def test_attention_of_more_than_1024_sequences(op, cuda_device):
    c = attention_case("int8", BF16, 1, 2, 64, 4, 6, [i % 4 for i in range(1100)], seed=6)
    out, lse = run_attention(op, c, cuda_device)
    check_attention(c, out, lse)


def test_attention_of_no_sequences_and_of_an_empty_table(op, cuda_device):
    c = attention_case("raw", BF16, 1, 2, 64, 16, 20, [3], seed=6)
    c["tables"] = c["tables"][:, :0]
    c["lens"] = torch.tensor([0])
    out, lse = run_attention(op, c, cuda_device)
    check_attention(c, out, lse)
    q = torch.zeros(0, 2, 64, dtype=BF16, device=cuda_device)
    run_attention(op, dict(c, tables=torch.zeros(0, 4), lens=torch.zeros(0)), cuda_device, q=q)
    assert status() == 0


def test_the_same_call_gives_the_same_bits(op, cuda_device):
    c = attention_case("e4m3", BF16, 2, 4, 128, 16, 700, [400, 30, 0, 250], seed=8)
    a, la = run_attention(op, c, cuda_device)
    b, lb = run_attention(op, c, cuda_device)
    assert torch.equal(a, b) and torch.equal(la, lb)


# ------------------------------------------------------- streams and graphs ---
def test_calls_on_several_streams_and_replayed_graphs(op, cuda_device):
    """Two streams at once without workspaces of their own, then a captured call replayed with other lengths and queries."""
    cases = [attention_case("int8", BF16, 2, 4, 128, 16, 300, [100, 40, 7], seed=20 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append((c, run_attention(op, c, cuda_device)))
    torch.cuda.synchronize()
    for c, (out, lse) in got:
        check_attention(c, out, lse)

    c = cases[0]
    d = {n: c[n].to(cuda_device) for n in ("q", "k", "v", "prefix_table", "tables", "lens")}
    out, lse = torch.empty_like(d["q"]), torch.empty(d["q"].shape[:2], device=cuda_device)
    new = torch.randn(3, 2, 2, 128, generator=gen(4)).to(BF16)
    rows, slots = new.to(cuda_device), torch.full((3,), -1, device=cuda_device)

    def step():
        op.kv_write(rows[:, 0], rows[:, 1], d["k"], d["v"], slots, 16, 2)
        op.shared_prefix_attention(d["q"], out, d["k"], d["v"], d["prefix_table"], 300, d["tables"], d["lens"], 16, 2, 2, c["scale"], lse)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        c["q"] = torch.randn(3, 8, 128, generator=gen(30 + turn)).to(BF16)
        c["lens"] = torch.tensor([100 + turn, 40, 7 - turn])
        place = torch.tensor([int(c["tables"][0, (99 + turn) // 16]) * 16 + (99 + turn) % 16, -1, -1])
        o.write(new[:, 0], c["k"], place, 16, "int8")
        o.write(new[:, 1], c["v"], place, 16, "int8")
        for n in ("q", "lens"):
            d[n].copy_(c[n])
        slots.copy_(place)
        graph.replay()
        torch.cuda.synchronize()
        check_attention(c, out, lse)
    assert status() == 0


def test_a_captured_call_with_a_shared_prefix_replays(op, cuda_device):
    """The three dependent launches (prefix, own tokens, join) in a graph, two graphs replayed in turn and on two streams."""
    graphs = []
    for seed in (1, 2):
        c = attention_case("e4m3", BF16, 2, 4, 128, 16, 600, [30, 0, 77] * 5, seed=seed)
        d = {n: c[n].to(cuda_device) for n in ("q", "k", "v", "prefix_table", "tables", "lens")}
        out, lse = torch.empty_like(d["q"]), torch.empty(d["q"].shape[:2], device=cuda_device)

        def call(c=c, d=d, out=out, lse=lse):
            op.shared_prefix_attention(d["q"], out, d["k"], d["v"], d["prefix_table"], 600, d["tables"], d["lens"], 16, 2, 1, c["scale"], lse)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((c, d, out, lse, graph))
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(3):
        for i, (c, d, out, lse, graph) in enumerate(graphs):
            c["q"] = torch.randn(15, 8, 128, generator=gen(50 + turn + 10 * i)).to(BF16)
            d["q"].copy_(c["q"])
            out.zero_()
        torch.cuda.synchronize()
        for (c, d, out, lse, graph), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for c, d, out, lse, graph in graphs:
            check_attention(c, out, lse)
    assert status() == 0


# ------------------------------------------------------------- used together ---
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("mover", [None, 1, 2, "staged"])
def test_an_8_bit_cache_through_prompt_swap_and_decoding(op, cuda_device, fmt, mover):
    """A prompt is normed, rotated and written; its pages go to the host and come back in other places; two sequences behind
    it decode a token; what they read equals the read-back of the cache, and attention of these values."""
    from heterofusedkernels_b200.connector import QuantizedPagedKVCache, rope_table

    heads, group, dim, block, prompt = 2, 4, 128, 16, 100
    cache = QuantizedPagedKVCache(2, 24, block, heads, dim, fmt, cuda_device, host_slots=16)
    for t in cache.k_caches + cache.v_caches:
        t.fill_(0xFF)
    table = rope_table(256, dim)
    pages = torch.randperm(24, generator=gen(1))
    where = pages[torch.arange(prompt) // block] * block + torch.arange(prompt) % block
    x = torch.randn(2, prompt, (group + 2) * heads, dim, generator=gen(2)).to(BF16).to(cuda_device)
    w = torch.ones(dim, dtype=BF16, device=cuda_device)
    for layer in range(2):
        q, k, v = x[layer].split([group * heads, heads, heads], 1)
        cache.norm_rope_write(layer, q, k, v, where.to(cuda_device), torch.arange(prompt, device=cuda_device), table, w, w)
    n = -(-prompt // block)
    lens = torch.tensor([prompt])
    before = cache.paged_gather(pages[None, :n], lens)
    slots = cache.swap_out(pages[:n], mover=mover)
    for t in cache.k_caches + cache.v_caches:
        t.fill_(0xFF)
    front = pages[n:2 * n]                       # other places
    cache.swap_in(front, slots, mover=mover, release=True)
    after = cache.paged_gather(front[None], lens)
    assert not before[0].isnan().any()
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])
    # two sequences behind the prompt, 17 tokens each
    own = torch.stack([pages[2 * n:2 * n + 2], pages[2 * n + 2:2 * n + 4]])
    at = torch.arange(17)
    where = (own[:, at // block] * block + at % block).flatten()
    y = torch.randn(2, 34, (group + 2) * heads, dim, generator=gen(3)).to(BF16).to(cuda_device)
    for layer in range(2):
        q, k, v = y[layer].split([group * heads, heads, heads], 1)
        turned = cache.norm_rope_write(layer, q, k, v, where.to(cuda_device), (prompt + at).repeat(2).to(cuda_device), table)
        q = turned[[16, 33]]
        lse = torch.empty(2, heads * group, device=cuda_device)
        out = cache.attend(layer, q, front.to(cuda_device), prompt, own.to(cuda_device), torch.tensor([17, 17], device=cuda_device), lse=lse)
        c = dict(fmt=fmt, q=q.cpu(), k=cache.k_caches[layer].cpu(), v=cache.v_caches[layer].cpu(), prefix_table=front, prefix=prompt,
                 tables=own, lens=torch.tensor([17, 17]), block=block, heads=heads, dim=dim, scale=dim ** -0.5)
        check_attention(c, out, lse)
    assert cache.status() == 0


def test_an_8_bit_cache_in_the_layer_wise_pipeline_and_migration(op, cuda_device):
    from heterofusedkernels_b200.connector import LayerwisePrefetcher, QuantizedPagedKVCache

    cache = QuantizedPagedKVCache(3, 16, 16, 4, 64, "int8", cuda_device, host_slots=24, pool_layout="layer_major", dtype=FP32)
    other = QuantizedPagedKVCache(3, 20, 16, 4, 64, "int8", cuda_device, dtype=FP32)
    for t in other.k_caches + other.v_caches:
        t.zero_()
    x = torch.randn(3, 100, 2, 4, 64, generator=gen(1)).to(BF16).to(cuda_device)
    for layer in range(3):
        cache.write(layer, x[layer, :, 0], x[layer, :, 1], torch.arange(100, device=cuda_device))
    want = cache.paged_gather(torch.arange(7)[None], torch.tensor([100]))
    assert want[0].dtype == FP32
    ids, slots = torch.arange(7, device=cuda_device), torch.arange(3, 10, device=cuda_device)
    pipe = LayerwisePrefetcher(cache)
    pipe.evict((0, 3), ids, slots)
    pipe.quiesce()
    pipe.prefetch((0, 3), ids + 8, slots)
    pipe.quiesce()
    cache.migrate_to(other, ids + 8, ids + 11)
    for where, first in ((cache, 8), (other, 11)):
        got = where.paged_gather(torch.arange(first, first + 7)[None], torch.tensor([100]))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(AssertionError):
        cache.migrate_to(QuantizedPagedKVCache(3, 4, 16, 4, 64, "e4m3", cuda_device), ids[:1], ids[:1])
    with pytest.raises(ValueError, match="mover"):
        cache.paged_gather(torch.arange(7)[None], torch.tensor([100]), mover=1)
    assert cache.status() == 0


def test_a_16_bit_cache_of_the_connector_writes_and_attends(op, cuda_device):
    from heterofusedkernels_b200.connector import PagedKVCache

    cache = PagedKVCache(1, 8, 16, 2, 64, FP16, cuda_device)
    x = torch.randn(40, 2, 2, 64, generator=gen(1)).to(FP16).to(cuda_device)
    cache.write(0, x[:, 0], x[:, 1], torch.arange(40, device=cuda_device))
    k, v = cache.paged_gather(torch.arange(3)[None], torch.tensor([40]))
    assert torch.equal(k[0], x[:, 0]) and torch.equal(v[0], x[:, 1])
    q = torch.randn(1, 6, 64, generator=gen(2)).to(FP16).to(cuda_device)
    lse = torch.empty(1, 6, device=cuda_device)
    out = cache.attend(0, q, torch.arange(2, device=cuda_device), 32, torch.tensor([[2]], device=cuda_device),
                       torch.tensor([8], device=cuda_device), lse=lse)
    c = dict(fmt="raw", q=q.cpu(), k=cache.k_caches[0].cpu(), v=cache.v_caches[0].cpu(), prefix_table=torch.arange(2), prefix=32,
             tables=torch.tensor([[2]]), lens=torch.tensor([8]), block=16, heads=2, dim=64, scale=0.125)
    c["v"][~c["v"].isfinite()] = 0
    check_attention(c, out, lse)
    assert cache.status() == 0


def test_refusals_on_the_device(op, cuda_device):
    """What the operators refuse before anything is enqueued; the sizes themselves are tested without a GPU."""
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=cuda_device)  # noqa: E731
    k, cache, ids = z(4, 2, 64), z(3, 16, 2, 64), torch.arange(4, device=cuda_device)
    page = z(3, o.block_bytes(16, 2, 64, "e4m3"), dtype=torch.uint8)
    op.kv_write(k, k, cache, cache.clone(), ids, 16, 0)
    for args, text in [((k, k, cache.half(), cache.half(), ids, 16, 0), "dtype of the call"), ((k, k, cache, cache, ids, 8, 0), "blockSize"),
                       ((k, k, page, page, ids, 16, 0), "dtype of the call"), ((k, k, cache, cache, ids, 16, 1), "uint8"),
                       ((k, k, page[:, :100], page[:, :100], ids, 16, 1), "a page of this cache"), ((k, k, page, page, ids, 16, 3), "kvFormat"),
                       ((k, k[:2], cache, cache, ids, 16, 0), "same shape"), ((k, k, cache, cache, ids[:3], 16, 0), "slot ids"),
                       ((k, k, cache, cache, ids.float(), 16, 0), "int64 or int32"), ((k, k, cache, cache, ids.cpu(), 16, 0), "one device"),
                       ((z(4, 2, 72)[:, :, 4:68], k, cache, cache, ids, 16, 0), "multiples of 16"),
                       ((k.float(), k.float(), cache, cache, ids, 16, 0), "bfloat16 or float16")]:
        with pytest.raises(RuntimeError, match=text):
            op.kv_write(*args)
    q, tab, lens, pre = z(2, 4, 64), z(2, 1, dtype=torch.int64), z(2, dtype=torch.int64), z(2, dtype=torch.int64)
    good = [q, torch.empty_like(q), cache, cache, pre, 32, tab, lens, 16, 2, 0]
    op.shared_prefix_attention(*good)
    for i, bad, text in [(5, 33, "needs 3"), (9, 3, "multiple of kvHeads"), (0, z(2, 4, 96), "out must have"), (4, pre.int(), "same dtype"),
                         (7, lens[:1], "num_seqs"), (8, 8, "blockSize"), (3, cache[:2], "same shape"), (6, tab.t(), "num_seqs"),
                         (1, z(2, 1, 64).expand(2, 4, 64), "overlap"), (5, -1, "negative"),
                         (6, tab[:1].expand(2, 1), "block_table_stride")]:
        args = list(good)
        args[i] = bad
        with pytest.raises(RuntimeError, match=text):
            op.shared_prefix_attention(*args)
    with pytest.raises(RuntimeError, match="needed"):
        op.shared_prefix_attention(*good, workspace=z(1024, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="256-byte"):
        op.shared_prefix_attention(*good, workspace=z(1 << 24, dtype=torch.uint8)[16:])
    with pytest.raises(RuntimeError, match="not finite"):
        op.shared_prefix_attention(*good, float("nan"))
    with pytest.raises(RuntimeError, match="64 or 128"):
        op.shared_prefix_attention(z(2, 4, 96), z(2, 4, 96), z(3, 16, 2, 96), z(3, 16, 2, 96), pre, 32, tab, lens, 16, 2, 0)
    table = torch.zeros(8, 64, device=cuda_device)
    pos = torch.arange(4, device=cuda_device)
    rope = [z(4, 4, 64), k, k, z(4, 4, 64), cache, cache, ids, pos, table, 16, 0]
    op.qk_norm_rope_write(*rope)
    for i, bad, text in [(8, table[:, :24].contiguous(), "rot_dim"), (8, table.double(), "float32"), (7, pos[:3], "positions"),
                         (3, z(4, 1, 64).expand(4, 4, 64), "overlap"), (0, z(3, 4, 64), "qHeads"), (8, torch.zeros(8, 128, device=cuda_device), "larger")]:
        args = list(rope)
        args[i] = bad
        with pytest.raises(RuntimeError, match=text):
            op.qk_norm_rope_write(*args)
    with pytest.raises(RuntimeError, match="kWeight"):
        op.qk_norm_rope_write(*rope, None, z(32))
    with pytest.raises(RuntimeError, match="eps"):
        op.qk_norm_rope_write(*rope, None, None, -1.0)
    out = torch.zeros(1, 16, 2, 64, device=cuda_device)
    ptr = torch.tensor([page.data_ptr()], device=cuda_device)
    for args, text in [((ptr, ptr, out, out, tab, lens, 16, 3, 0), "paged_gather reads"), ((ptr, ptr, out.double(), out.double(), tab, lens, 16, 3, 1), "float32"),
                       ((ptr, ptr, out, out, tab, lens, 16, 3, 1, 1024), "smaller than one"), ((ptr, ptr, out, out, tab, lens.int(), 16, 3, 1), "same dtype"),
                       ((ptr, ptr, out, out, tab[:1].expand(3, tab.shape[1]), lens[:1].repeat(3), 16, 3, 1), "block_table_stride")]:
        with pytest.raises(RuntimeError, match=text):
            op.paged_gather_dequant(*args)
    torch.cuda.synchronize()
    assert status() == 0
