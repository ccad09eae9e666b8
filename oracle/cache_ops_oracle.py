"""CPU oracle of the operators that fill and read the cache of an attention layer.  TEST INFRASTRUCTURE ONLY.

Codes and scales follow the definition in fp32 (they are compared bit for bit); norms, rotations and attention are
in 64 bits.  Loops over tokens and sequences, no batching: the restatement is meant to be read.
"""
from __future__ import annotations

import math

import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
TINY = 2.0 ** -126


def block_bytes(block_size, heads, dim, fmt, elt=2):
    if fmt == "raw":
        return block_size * heads * dim * elt
    return -(-block_size * heads * (dim + 4) // 16) * 16


def encode(x, fmt):
    """Rows [..., dim] -> (codes [..., dim], scales [...]); codes as float8_e4m3fn or int8."""
    x = x.float()
    scale = (x.abs().amax(-1) * (1 / torch.tensor(TOP[fmt]))).clamp(min=TINY)
    scale = torch.where(scale.isfinite(), scale, torch.nan)
    y = x * (1 / scale).unsqueeze(-1)
    return (y.to(torch.float8_e4m3fn) if fmt == "e4m3" else y.round().to(torch.int8)), scale


def split_pages(pages, block_size, heads, dim, fmt):
    """uint8 [blocks, bytes] -> views (codes [blocks, B, H, D], scales [blocks, B, H])."""
    n = block_size * heads
    codes = pages[:, :n * dim].unflatten(1, (block_size, heads, dim))
    scales = pages[:, n * dim:n * (dim + 4)].view(torch.float32).unflatten(1, (block_size, heads))
    return codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8), scales


def values(pages, block_size, heads, dim, fmt):
    """What the pages hold, fp32 (exact products of code and scale are rounded to fp32, as the read-back does)."""
    if fmt == "raw":
        return pages.float()
    codes, scales = split_pages(pages, block_size, heads, dim, fmt)
    return codes.float() * scales.unsqueeze(-1)


def write(rows, pages, slots, block_size, fmt):
    """In place; rows [tokens, heads, dim]."""
    heads, dim = rows.shape[1:]
    if fmt != "raw":
        codes, scales = split_pages(pages, block_size, heads, dim, fmt)
        row_codes, row_scales = encode(rows, fmt)
    for t, slot in enumerate(slots.tolist()):
        if slot < 0 or slot >= pages.shape[0] * block_size:
            continue
        b, at = divmod(slot, block_size)
        if fmt == "raw":
            pages[b, at] = rows[t]
        else:
            codes.view(torch.uint8)[b, at] = row_codes.view(torch.uint8)[t]
            scales[b, at] = row_scales[t]
    return pages


def norm_rope(x, positions, cos_sin, weight, eps, interleaved):
    """[tokens, heads, dim] in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = cos_sin.shape[1] // 2
    out = x.clone()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    for t, p in enumerate(positions.tolist()):
        c, s = cos_sin[p, :half].double(), cos_sin[p, half:].double()
        out[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
        out[t, :, b] = x[t, :, b] * c + x[t, :, a] * s
    return out


def rows_of(held, table, n, block_size):
    """Tokens 0..n of a page list: (rows [n, heads, dim], which of them lie in valid pages)."""
    rows, ok = [], []
    for i in range(n):
        b = int(table[i // block_size])
        good = 0 <= b < held.shape[0]
        ok.append(good)
        rows.append(held[b if good else 0, i % block_size])
    if not rows:
        return held.new_zeros((0,) + held.shape[2:]), torch.zeros(0, dtype=torch.bool)
    return torch.stack(rows), torch.tensor(ok)


def attention(q, k_held, v_held, prefix_table, prefix_len, tables, lens, block_size, scale):
    """Returns out, lse, and what an error bound needs: sum p|v| / l and the largest sum |q||k| * scale; all 64 bits."""
    seqs, q_heads, dim = q.shape
    heads = k_held.shape[2]
    group = q_heads // heads
    out, spread = torch.zeros(2, seqs, q_heads, dim, dtype=torch.float64)
    lse, reach = torch.full((seqs, q_heads), -math.inf, dtype=torch.float64), torch.zeros(seqs, q_heads, dtype=torch.float64)
    kp, okp = rows_of(k_held, prefix_table, prefix_len, block_size)
    vp, _ = rows_of(v_held, prefix_table, prefix_len, block_size)
    cap = tables.shape[1] * block_size
    for s in range(seqs):
        n = min(max(int(lens[s]), 0), cap)
        ks, oks = rows_of(k_held, tables[s], n, block_size)
        vs, _ = rows_of(v_held, tables[s], n, block_size)
        ok = torch.cat([okp, oks])
        k, v = torch.cat([kp, ks])[ok].double(), torch.cat([vp, vs])[ok].double()
        if len(k) == 0:
            continue
        for head in range(q_heads):
            z = k[:, head // group] @ q[s, head].double() * scale
            lse[s, head] = torch.logsumexp(z, 0)
            p = torch.softmax(z, 0)
            out[s, head] = p @ v[:, head // group]
            spread[s, head] = p @ v[:, head // group].abs()
            reach[s, head] = (k[:, head // group].abs() @ q[s, head].double().abs()).max() * abs(scale)
    return out, lse, spread, reach
