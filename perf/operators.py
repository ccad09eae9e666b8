"""Cases of the operators that fill, keep and read the paged K/V cache: `kv_write`, `qk_norm_rope_write`,
`paged_gather_dequant` and `shared_prefix_attention`.

`run` computes a case in elementary torch operations, or (where `own` is true) through the framework's operators.

A page of a 16-bit cache is [block_size][kv_heads][head_dim].  A page of an 8-bit cache is one run of bytes: the codes
[block_size][kv_heads][head_dim], then the fp32 scales [block_size][kv_heads], padded to a multiple of 16 bytes.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FORMATS = {"raw": 0, "e4m3": 1, "int8": 2}          # kvFormat of the operators
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}
TINY = 2.0 ** -126                                  # least scale: the smallest normal fp32 number
EPS = 1e-6                                          # of the root mean square


def listed():
    return [
        # one decoding step of 64 sequences: the new tokens' K and V of one layer go to their pages
        dict(name="write_decode_64", op="write", tokens=64, kv_heads=8, dim=128, block=16, fmt="e4m3", type="bf16"),
        # several prompts at once, packed: K and V of one layer
        dict(name="write_prompt_65536", op="write", tokens=65536, kv_heads=8, dim=128, block=16, fmt="int8", type="fp16"),
        # the whole prologue of attention for one token: the smallest call there is
        dict(name="rope_decode_1", op="rope", tokens=1, kv_heads=8, group=4, dim=128, rot=128, interleaved=False, norm=True,
             block=16, fmt="e4m3", type="bf16"),
        # ... for a prompt, odd length, 7 query heads to a K/V head, 16-bit cache, half of the head rotated in pairs
        dict(name="rope_prompt_8191", op="rope", tokens=8191, kv_heads=4, group=7, dim=128, rot=64, interleaved=True, norm=True,
             block=16, fmt="raw", type="bf16"),
        # ... for packed prompts into the 8-bit cache
        dict(name="rope_prompt_16384", op="rope", tokens=16384, kv_heads=8, group=4, dim=128, rot=128, interleaved=False,
             norm=False, block=16, fmt="e4m3", type="fp16"),
        # reading two short sequences back, all layers
        dict(name="gather_small", op="gather", layers=2, seqs=2, low=40, high=100, kv_heads=8, dim=128, block=16, fmt="int8",
             type="fp16"),
        # reading a batch of 64 long sequences back: four layers of the 32
        dict(name="gather_64_seqs", op="gather", layers=4, seqs=64, low=512, high=8192, kv_heads=8, dim=128, block=16, fmt="e4m3",
             type="bf16"),
        # decoding, few sequences behind a system prompt
        dict(name="attend_4", op="attend", seqs=4, group=4, kv_heads=8, dim=128, block=16, prefix=512, low=1, high=64, fmt="raw",
             type="bf16"),
        # decoding, a batch behind a long prompt
        dict(name="attend_64_prefix_8192", op="attend", seqs=64, group=4, kv_heads=8, dim=128, block=16, prefix=8192, low=256,
             high=2048, fmt="raw", type="bf16"),
        # ragged everything: 7 query heads to a K/V head, prefix that ends inside a page, sequences without own tokens, int8
        dict(name="attend_33_ragged", op="attend", seqs=33, group=7, kv_heads=4, dim=128, block=16, prefix=4099, low=0, high=2900,
             fmt="int8", type="fp16"),
        # no common prefix: long sequences of their own
        dict(name="attend_8_long", op="attend", seqs=8, group=4, kv_heads=8, dim=128, block=16, prefix=0, low=16384, high=131072,
             fmt="raw", type="bf16"),
        # one K/V head a GPU, large batch behind a very long prefix, large pages, 8-bit cache
        dict(name="attend_256_prefix_32768", op="attend", seqs=256, group=8, kv_heads=1, dim=128, block=128, prefix=32768, low=1,
             high=1024, fmt="e4m3", type="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))


def draw(rng):
    op = rng.choice(["write", "rope", "gather", "attend", "attend"])
    c = dict(op=op, kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), block=rng.choice([8, 16, 32, 128]),
             fmt=rng.choice(["raw", "e4m3", "int8"]), type=rng.choice(["bf16", "fp16"]))
    if op == "write":
        c.update(tokens=_log(rng, 1, 65536), dim=rng.choice([64, 96, 128, 256]))
        c["tokens"] = min(c["tokens"], 65536 * 8 * 128 // (c["kv_heads"] * c["dim"]))
    elif op == "rope":
        c.update(tokens=_log(rng, 1, 16384), group=rng.randint(1, 8), dim=rng.choice([64, 96, 128, 256]),
                 interleaved=rng.random() < 0.5, norm=rng.random() < 0.7)
        c["rot"] = rng.choice([c["dim"], 32])
        c["tokens"] = min(c["tokens"], 16384 * 40 * 128 // (c["kv_heads"] * (c["group"] + 2) * c["dim"]))
    elif op == "gather":
        c.update(layers=rng.randint(1, 8), seqs=_log(rng, 1, 64), high=_log(rng, 1, 8192), fmt=rng.choice(["e4m3", "int8"]),
                 type=rng.choice(["bf16", "fp16", "fp32"]))
        c["low"] = rng.randint(1, c["high"])
        c["layers"] = max(1, min(c["layers"], 4 * 64 * 4096 * 1024 // (c["seqs"] * c["high"] * c["kv_heads"] * c["dim"])))
    else:
        c.update(seqs=_log(rng, 1, 256), group=rng.randint(1, 8), prefix=rng.choice([0, _log(rng, 1, 32768), _log(rng, 1, 32768)]),
                 high=_log(rng, 1, 8192))
        c["high"] = min(c["high"], 4 * 1024 * 1024 // (c["seqs"] * c["kv_heads"]))
        c["prefix"] = min(c["prefix"], 256 * 8 * 32768 // (c["seqs"] * c["group"] * c["kv_heads"]))
        c["low"] = rng.randint(0, c["high"])
    return c


# ---- pages ---------------------------------------------------------------------------------------------------------
def _block_bytes(c):
    return -(-c["block"] * c["kv_heads"] * (c["dim"] + 4) // 16) * 16


def _codes(pages, c):
    n = c["block"] * c["kv_heads"] * c["dim"]
    return pages[..., :n].unflatten(-1, (c["block"], c["kv_heads"], c["dim"]))


def _scales(pages, c):
    n = c["block"] * c["kv_heads"]
    return pages[..., n * c["dim"]:n * (c["dim"] + 4)].view(torch.float32).unflatten(-1, (c["block"], c["kv_heads"]))


def _seen(pages, c):
    """What a cache holds, as outputs: the pages, or codes and scales."""
    return pages if c["fmt"] == "raw" else [_codes(pages, c).view(CODES[c["fmt"]]), _scales(pages, c)]


def _encode(x, fmt):
    """fp32 rows [..., dim] -> codes (as bytes) and scales [...]."""
    scale = (x.abs().amax(-1) / TOP[fmt]).clamp(min=TINY)
    y = x * (1 / scale)[..., None]
    y = y.to(CODES["e4m3"]) if fmt == "e4m3" else y.round().to(torch.int8)
    return y.view(torch.uint8), scale


def _pages(c, layers, blocks, g):
    """A cache as it is in use: every page written, values of unit variance."""
    shape = (layers, blocks, c["block"], c["kv_heads"], c["dim"])
    if c["fmt"] == "raw":
        out = torch.empty(shape, dtype=TYPES[c["type"]], device="cuda")
        for layer in out:
            layer.normal_(generator=g)
        return out
    out = torch.zeros(layers, blocks, _block_bytes(c), dtype=torch.uint8, device="cuda")
    for layer in out:
        for part in layer.split(max(1, (1 << 28) // _block_bytes(c))):
            codes, scales = _encode(torch.randn((len(part),) + shape[2:], generator=g, device="cuda"), c["fmt"])
            _codes(part, c).copy_(codes)
            _scales(part, c).copy_(scales)
    return out


def _lengths(c, g):
    n = torch.linspace(c["low"], c["high"], c["seqs"], dtype=torch.float64).round().to(torch.int64).cuda()
    return n[torch.randperm(c["seqs"], generator=g, device="cuda")]


def _total(c):
    return int(torch.linspace(c["low"], c["high"], c["seqs"], dtype=torch.float64).round().sum())


def _tables(lens, block, ids):
    """Rows of page ids for these lengths, -1 behind the last page; `ids` are used in order."""
    n = (lens + block - 1) // block
    width = max(1, int(n.max()))
    at = (n.cumsum(0) - n)[:, None] + torch.arange(width, device="cuda")
    used = torch.arange(width, device="cuda") < n[:, None]
    return torch.where(used, ids[at.clamp(max=len(ids) - 1)], -1)


# ---- inputs --------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"c": c, "fmt": FORMATS[c["fmt"]], "type": TYPES[c["type"]]}
    new = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(s["type"])  # noqa: E731
    if c["op"] in ("write", "rope"):
        # K, V (and queries) are slices of one projection's output, as a model has them
        t, hk, d = c["tokens"], c["kv_heads"], c["dim"]
        hq = hk * c.get("group", 0)
        qkv = new(t, hq + 2 * hk, d)
        s["q"], s["k"], s["v"] = qkv.split([hq, hk, hk], 1)
        blocks = -(-t // c["block"]) + 2
        s["k_cache"], s["v_cache"] = _pages(c, 2, blocks, g)
        if t <= 256:    # decoding: one token of each sequence
            s["slots"] = torch.randperm(blocks * c["block"], generator=g, device="cuda")[:t]
        else:           # prompts: page after page
            at = torch.arange(t, device="cuda")
            s["slots"] = torch.randperm(blocks, generator=g, device="cuda")[at // c["block"]] * c["block"] + at % c["block"]
        if c["op"] == "rope":
            s["k"].mul_(3)
            s["q_out"] = torch.empty(t, hq, d, dtype=s["type"], device="cuda")
            longest = 32768
            angle = torch.arange(longest, dtype=torch.float64, device="cuda")[:, None] * \
                5e5 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
            s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
            s["positions"] = torch.randint(0, longest, (t,), generator=g, device="cuda")
            s["q_weight"], s["k_weight"] = (1 + 0.1 * new(2, d)).to(s["type"]) if c["norm"] else (None, None)
        return s
    lens = _lengths(c, g)
    pages = int(((lens + c["block"] - 1) // c["block"]).sum())
    front = -(-c.get("prefix", 0) // c["block"])
    blocks = pages + front + 3
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    s["tables"], s["lens"] = _tables(lens, c["block"], ids[front:]).to(torch.int32), lens.to(torch.int32)
    if c["op"] == "gather":
        s["pages"] = _pages(c, 2 * c["layers"], blocks, g)
        at = torch.tensor([p.data_ptr() for p in s["pages"]], device="cuda")
        s["k_ptrs"], s["v_ptrs"] = at[:c["layers"]].clone(), at[c["layers"]:].clone()
        s["k_out"], s["v_out"] = torch.empty(2, c["layers"], _total(c), c["kv_heads"], c["dim"], dtype=s["type"], device="cuda")
        return s
    s["k_cache"], s["v_cache"] = _pages(c, 2, blocks, g)
    s["prefix_table"] = ids[:front].clone()
    s["q"] = 2 * new(c["seqs"], c["kv_heads"] * c["group"], c["dim"])
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
    s["scale"] = c["dim"] ** -0.5
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def _store(x, pages, s):
    """fp32 rows [tokens, kv_heads, dim] to their slots."""
    c = s["c"]
    block, at = s["slots"] // c["block"], s["slots"] % c["block"]
    if c["fmt"] == "raw":
        pages[block, at] = x.to(pages.dtype)
    else:
        codes, scales = _encode(x, c["fmt"])
        _codes(pages, c)[block, at] = codes
        _scales(pages, c)[block, at] = scales


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(x, cos_sin, c):
    cos, sin = cos_sin[:, None].chunk(2, -1)
    turned, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if c["interleaved"] else turned.chunk(2, -1)
    pair = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack(pair, -1).flatten(-2) if c["interleaved"] else torch.cat(pair, -1)
    return torch.cat([turned, rest], -1)


def _rows(pages, ids, c):
    """Pages by id, [..., width * block, kv_heads, dim] in fp32; ids below 0 stand for any page."""
    got = pages[ids.clamp(min=0).long()]
    if c["fmt"] != "raw":
        got = _codes(got, c).view(CODES[c["fmt"]]).float() * _scales(got, c)[..., None]
    return got.float().flatten(ids.dim() - 1, ids.dim())


def run(s):
    c = s["c"]
    if own:
        return _run_own(s, c)
    if c["op"] == "write":
        _store(s["k"].float(), s["k_cache"], s)
        _store(s["v"].float(), s["v_cache"], s)
        return [_seen(s["k_cache"], c), _seen(s["v_cache"], c)]
    if c["op"] == "rope":
        turn = s["cos_sin"][s["positions"]]
        s["q_out"].copy_(_rotated(_normed(s["q"].float(), s["q_weight"]), turn, c))
        _store(_rotated(_normed(s["k"].float(), s["k_weight"]), turn, c), s["k_cache"], s)
        _store(s["v"].float(), s["v_cache"], s)
        return [s["q_out"], _seen(s["k_cache"], c), _seen(s["v_cache"], c)]
    used = torch.arange(s["tables"].shape[1] * c["block"], device="cuda") < s["lens"][:, None]
    if c["op"] == "gather":
        rows = _rows(s["pages"].flatten(0, 1), _per_layer(s["tables"], s["pages"]), c)
        out = rows[:, used].to(s["type"])
        s["k_out"].copy_(out[:c["layers"]])
        s["v_out"].copy_(out[c["layers"]:])
        return [s["k_out"], s["v_out"]]
    q = s["q"].float().unflatten(1, (c["kv_heads"], c["group"])) * s["scale"]
    k, v = (_rows(p, s["prefix_table"], c)[:c["prefix"]] for p in (s["k_cache"], s["v_cache"]))
    scores = torch.einsum("shgd,lhd->shgl", q, k)
    ks, vs = (_rows(p, s["tables"], c) for p in (s["k_cache"], s["v_cache"]))
    mine = torch.einsum("shgd,slhd->shgl", q, ks).masked_fill(~used[:, None, None], -math.inf)
    top = torch.maximum(mine.amax(-1), scores.amax(-1) if c["prefix"] else mine.amax(-1)).clamp(min=-1e30)[..., None]
    scores, mine = (scores - top).exp(), (mine - top).exp()
    total = scores.sum(-1) + mine.sum(-1)
    vs = vs.masked_fill(~used[:, :, None, None], 0)
    out = torch.einsum("shgl,lhd->shgd", scores, v) + torch.einsum("shgl,slhd->shgd", mine, vs)
    out = torch.where(total[..., None] > 0, out / total[..., None], 0)
    s["out"].copy_(out.flatten(1, 2))
    s["lse"].copy_((top[..., 0] + total.log()).flatten(1, 2))
    return [s["out"], s["lse"]]


def _per_layer(tables, pages):
    """Page ids in the layers one behind the other, -1 kept: [layers, seqs, width]."""
    at = tables.long() + torch.arange(pages.shape[0], device="cuda")[:, None, None] * pages.shape[1]
    return torch.where(tables >= 0, at, -1)


def _run_own(s, c):
    import heterofusedkernels_b200
    heterofusedkernels_b200.load_ops()
    ops = torch.ops.pcie_through
    if c["op"] == "write":
        ops.kv_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], c["block"], s["fmt"])
        return [_seen(s["k_cache"], c), _seen(s["v_cache"], c)]
    if c["op"] == "rope":
        ops.qk_norm_rope_write(s["q"], s["k"], s["v"], s["q_out"], s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                               s["cos_sin"], c["block"], s["fmt"], s["q_weight"], s["k_weight"], EPS, c["interleaved"])
        return [s["q_out"], _seen(s["k_cache"], c), _seen(s["v_cache"], c)]
    if c["op"] == "gather":
        ops.paged_gather_dequant(s["k_ptrs"], s["v_ptrs"], s["k_out"], s["v_out"], s["tables"], s["lens"], c["block"],
                                 s["pages"].shape[1], s["fmt"])
        return [s["k_out"], s["v_out"]]
    ops.shared_prefix_attention(s["q"], s["out"], s["k_cache"], s["v_cache"], s["prefix_table"], c["prefix"], s["tables"],
                                s["lens"], c["block"], c["kv_heads"], s["fmt"], s["scale"], s["lse"])
    return [s["out"], s["lse"]]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c = case
    elt = {"bf16": 2, "fp16": 2, "fp32": 4}[c["type"]]
    row = c["dim"] * elt if c["fmt"] == "raw" else c["dim"] + 4   # bytes of one head's row in a page
    hk, d = c["kv_heads"], c["dim"]
    if c["op"] == "write":
        return {"bytes": c["tokens"] * (2 * hk * (d * elt + row) + 8), "flops": 4 * c["tokens"] * hk * d}
    if c["op"] == "rope":
        hq = hk * c["group"]
        turn = min(c["tokens"], 32768) * c["rot"] * 4
        return {"bytes": c["tokens"] * ((2 * hq + 2 * hk) * d * elt + 2 * hk * row + 16) + turn,
                "flops": c["tokens"] * (10 * (hq + hk) + 3 * hk) * d}
    total = _total(c)
    if c["op"] == "gather":
        return {"bytes": total * 2 * c["layers"] * hk * (row + d * elt), "flops": total * 2 * c["layers"] * hk * d}
    hq = hk * c["group"]
    return {"bytes": (c["prefix"] + total) * 2 * hk * row + c["seqs"] * hq * (2 * d * elt + 4),
            "flops": 4 * d * hq * (c["seqs"] * c["prefix"] + total)}


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------------
def _grid(y):
    """The e4m3 numbers nearest to y (ties to even): steps of 2^-9 below 2^-6, 8 steps to a factor of two above."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 4).clamp(min=-9))
    return torch.round(y / step) * step


def _exact_store(x, pages, s):
    c = s["c"]
    at = s["slots"]
    if c["fmt"] == "raw":
        held = pages.double()
        held.flatten(0, 1)[at] = x
        return held
    values, scales = _codes(pages, c).view(CODES[c["fmt"]]).double(), _scales(pages, c).double()
    biggest = x.abs().max(-1).values / TOP[c["fmt"]]
    biggest = torch.where(biggest < TINY, TINY, biggest)
    scales = scales.flatten(0, 1).index_copy(0, at, biggest).unflatten(0, (-1, c["block"]))
    if c["fmt"] == "int8":
        return [None, scales]
    values = values.flatten(0, 1).index_copy(0, at, _grid(x / biggest[..., None])).unflatten(0, (-1, c["block"]))
    return [values, scales]


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "write":
        return [_exact_store(s["k"].double(), s["k_cache"], s), _exact_store(s["v"].double(), s["v_cache"], s)]
    if c["op"] == "rope":
        return _exact_rope(s, c)
    lens, tables = s["lens"].tolist(), s["tables"].long()

    def page_rows(pages, ids, n, head=slice(None)):
        got = pages[ids[:-(-n // c["block"])]]
        if c["fmt"] == "raw":
            return got.double().reshape(-1, c["kv_heads"], c["dim"])[:n, head]
        x = _codes(got, c).view(CODES[c["fmt"]]).double() * _scales(got, c).double()[..., None]
        return x.reshape(-1, c["kv_heads"], c["dim"])[:n, head]

    if c["op"] == "gather":
        if _total(c) * c["layers"] * c["kv_heads"] * c["dim"] > 600_000_000:
            return None
        out = [torch.cat([page_rows(p, t, n) for t, n in zip(tables, lens)]) for p in s["pages"]]
        return [torch.stack(out[:c["layers"]]), torch.stack(out[c["layers"]:])]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for h in range(c["kv_heads"]):
        heads = slice(h * c["group"], (h + 1) * c["group"])
        q = s["q"][:, heads].double()
        kp, vp = (page_rows(p, s["prefix_table"].long(), c["prefix"], h) for p in (s["k_cache"], s["v_cache"]))
        for i, n in enumerate(lens):
            k, v = (torch.cat([a, page_rows(p, tables[i], n, h)]) for a, p in ((kp, s["k_cache"]), (vp, s["v_cache"])))
            if len(k):
                z = q[i] @ k.T * s["scale"]
                lse[i, heads] = torch.logsumexp(z, -1)
                out[i, heads] = torch.softmax(z, -1) @ v
    return [out, lse]


def _exact_rope(s, c):
    turn = s["cos_sin"].double()[s["positions"]]
    half = c["rot"] // 2
    z = torch.complex(turn[:, None, :half], turn[:, None, half:])

    def norm_and_turn(x, weight):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + EPS) * weight.double()
        a, b = ((x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]) if c["interleaved"] else (x[..., :half], x[..., half:c["rot"]]))
        w = torch.complex(a.contiguous(), b.contiguous()) * z
        out = x.clone()
        if c["interleaved"]:
            out[..., 0:c["rot"]:2], out[..., 1:c["rot"]:2] = w.real, w.imag
        else:
            out[..., :half], out[..., half:c["rot"]] = w.real, w.imag
        return out

    return [norm_and_turn(s["q"], s["q_weight"]), _exact_store(norm_and_turn(s["k"], s["k_weight"]), s["k_cache"], s),
            _exact_store(s["v"].double(), s["v_cache"], s)]
