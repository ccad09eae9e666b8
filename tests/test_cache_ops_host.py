"""The operators that fill and read the cache of an attention layer, without a GPU: sizes of pages, the checks of the
C ABI (each returns before any CUDA call), struct layouts, and the oracle against its own definitions."""
import ctypes as C
import re
from pathlib import Path

import pytest
import torch

from oracle import cache_ops_oracle as o

HEADER = (Path(__file__).resolve().parent.parent / "include" / "hfk_b200.h").read_text()


def test_struct_layouts_follow_the_header_order(hfk):
    for struct, cname in ((hfk.Rows, "hfk_rows"), (hfk.KvWriteDesc, "hfk_kv_write_desc"), (hfk.NormRopeDesc, "hfk_norm_rope_desc"),
                          (hfk.PrefixAttentionDesc, "hfk_prefix_attention_desc")):
        m = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), HEADER, flags=re.S)
        body = re.sub(r"/\*.*?\*/", "", m.group(1), flags=re.S)
        assert [re.split(r"[\s\*]+", f.strip())[-1] for f in body.split(";") if f.strip()] == [f[0] for f in struct._fields_]


@pytest.mark.parametrize("block,heads,dim", [(16, 8, 128), (1, 1, 16), (7, 3, 48), (128, 1, 128), (3, 1, 32)])
def test_page_bytes(hfk, block, heads, dim):
    f = hfk.lib().hfk_kv_block_bytes
    assert f(block, heads, dim, hfk.HFK_KV_RAW) == block * heads * dim * 2
    for code, fmt in ((hfk.HFK_KV_E4M3, "e4m3"), (hfk.HFK_KV_INT8, "int8")):
        n = f(block, heads, dim, code)
        assert n == o.block_bytes(block, heads, dim, fmt) and n % 16 == 0


def test_page_bytes_of_bad_arguments_are_zero(hfk):
    f = hfk.lib().hfk_kv_block_bytes
    for args in ((0, 1, 16, 1), (16, -1, 16, 1), (16, 1, 0, 1), (16, 1, 16, 3), (16, 1, 16, -1), (1 << 40, 1 << 40, 16, 1), (1 << 20, 1 << 20, 16, 0)):
        assert f(*args) == 0


def write_desc(hfk, **over):
    d = hfk.KvWriteDesc()
    for r in (d.k, d.v):
        r.base, r.token_stride, r.head_stride = 0x10000, 2048, 256
    d.k_cache, d.v_cache, d.slot_ids = 0x20000, 0x30000, 0x40000
    d.ids_are_int64, d.type, d.kv_format, d.kv_heads, d.head_dim = 1, hfk.HFK_TYPE_BF16, hfk.HFK_KV_E4M3, 8, 128
    d.tokens, d.block_size, d.num_device_blocks = 4, 16, 10
    d.device_block_stride = hfk.lib().hfk_kv_block_bytes(16, 8, 128, hfk.HFK_KV_E4M3)
    for k, v in over.items():
        if k in ("k", "v"):
            for n, x in v.items():
                setattr(getattr(d, k), n, x)
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,code", [
    (dict(k_cache=0), "INVALID_ARG"), (dict(v_cache=0x30008), "ALIGNMENT"), (dict(slot_ids=0), "INVALID_ARG"), (dict(type=2), "INVALID_ARG"),
    (dict(kv_format=3), "INVALID_ARG"), (dict(kv_heads=0), "INVALID_ARG"), (dict(head_dim=120), "UNSUPPORTED"), (dict(head_dim=272, device_block_stride=1 << 20), "UNSUPPORTED"),
    (dict(tokens=-1), "INVALID_ARG"), (dict(block_size=0), "INVALID_ARG"), (dict(num_device_blocks=1 << 28), "TOO_LARGE"),
    (dict(tokens=1 << 28), "TOO_LARGE"), (dict(device_block_stride=16 * 8 * 128), "INVALID_ARG"), (dict(device_block_stride=17000), "ALIGNMENT"),
    (dict(k=dict(base=0)), "INVALID_ARG"), (dict(v=dict(token_stride=2050)), "ALIGNMENT"), (dict(k=dict(base=0x10002)), "ALIGNMENT"),
    (dict(kv_heads=1 << 20, block_size=1 << 20), "TOO_LARGE")])
def test_kv_write_refusals(hfk, over, code):
    d = write_desc(hfk, **over)
    assert hfk.lib().hfk_kv_write(C.byref(d), None) == getattr(hfk, "HFK_ERR_" + code), hfk.last_error()


def test_no_tokens_is_no_work(hfk):
    d = write_desc(hfk, tokens=0, slot_ids=0, k=dict(base=0), v=dict(base=0))
    assert hfk.lib().hfk_kv_write(C.byref(d), None) == hfk.HFK_OK
    assert hfk.lib().hfk_kv_write(None, None) == hfk.HFK_ERR_INVALID_ARG
    assert hfk.lib().hfk_qk_norm_rope_write(C.byref(d), None, None) == hfk.HFK_ERR_INVALID_ARG


@pytest.mark.parametrize("over,code", [
    (dict(q_heads=0), "INVALID_ARG"), (dict(rot_dim=24), "UNSUPPORTED"), (dict(rot_dim=144), "UNSUPPORTED"), (dict(rot_dim=-16), "UNSUPPORTED"),
    (dict(max_positions=0), "INVALID_ARG"), (dict(eps=-1.0), "INVALID_ARG"), (dict(eps=float("nan")), "INVALID_ARG"), (dict(positions=0), "INVALID_ARG"),
    (dict(cos_sin=0), "INVALID_ARG"), (dict(cos_sin=0x60004), "ALIGNMENT"), (dict(q_weight=0x70008), "ALIGNMENT"), (dict(q_heads=1 << 30), "TOO_LARGE"),
    (dict(q_out=(0x80000, 8192, 128)), "INVALID_ARG"), (dict(q_out=(0x80000, 0, 256)), "INVALID_ARG"), (dict(q=(0, 8192, 256)), "INVALID_ARG")])
def test_norm_rope_refusals(hfk, over, code):
    d, n = write_desc(hfk), hfk.NormRopeDesc()
    for r in (n.q, n.q_out):
        r.base, r.token_stride, r.head_stride = 0x50000, 8192, 256
    n.q_heads, n.rot_dim, n.positions, n.cos_sin, n.max_positions, n.eps = 32, 128, 0x90000, 0x60000, 100, 1e-6
    for k, v in over.items():
        if k in ("q", "q_out"):
            getattr(n, k).base, getattr(n, k).token_stride, getattr(n, k).head_stride = v
        else:
            setattr(n, k, v)
    assert hfk.lib().hfk_qk_norm_rope_write(C.byref(d), C.byref(n), None) == getattr(hfk, "HFK_ERR_" + code), hfk.last_error()


@pytest.mark.parametrize("over,more,code", [
    (dict(), dict(kv_format=0), "INVALID_ARG"), (dict(), dict(kv_format=3), "INVALID_ARG"), (dict(), dict(out_type=3), "INVALID_ARG"),
    (dict(), dict(kv_heads=0), "UNSUPPORTED"), (dict(), dict(kv_heads=3), "UNSUPPORTED"), (dict(device_block_stride=16 * 1024), dict(), "INVALID_ARG"),
    (dict(k_out=0), dict(), "INVALID_ARG"), (dict(block_size=0), dict(), "INVALID_ARG"), (dict(out_layer_stride=1024 * 100 * 2 - 32), dict(), "INVALID_ARG"),
    (dict(out_layer_stride=1024 * 100 * 2 + 8), dict(), "ALIGNMENT"), (dict(block_table_stride=2), dict(), "INVALID_ARG")])
def test_gather_dequant_refusals(hfk, over, more, code):
    d = hfk.PagedGatherDesc()
    d.k_layer_ptrs = d.v_layer_ptrs = d.block_tables = d.seq_lens = 0x1000
    d.k_out, d.v_out = 0x20000, 0x30000
    d.ids_are_int64, d.layers, d.num_seqs, d.max_blocks_per_seq, d.block_table_stride = 1, 2, 2, 4, 4
    d.block_size, d.token_bytes, d.device_block_stride = 16, 1024, 16 * 1024 + 16 * 8 * 4
    d.num_device_blocks, d.total_tokens, d.out_layer_stride = 8, 100, 1024 * 100 * 2
    for k, v in over.items():
        setattr(d, k, v)
    a = dict(kv_format=1, kv_heads=8, out_type=0, **{})
    a.update(more)
    assert hfk.lib().hfk_paged_gather_dequant(C.byref(d), a["kv_format"], a["kv_heads"], a["out_type"], 0, None) == getattr(hfk, "HFK_ERR_" + code), hfk.last_error()


def attention_desc(hfk, **over):
    d = hfk.PrefixAttentionDesc()
    for r in (d.q, d.out):
        r.base, r.token_stride, r.head_stride = 0x10000, 8192, 256
    d.k_cache = d.v_cache = 0x20000
    d.prefix_table = d.block_tables = d.seq_lens = 0x30000
    d.ids_are_int64, d.type, d.kv_format, d.kv_heads, d.group, d.head_dim = 0, 0, 0, 8, 4, 128
    d.num_seqs, d.prefix_len, d.max_blocks_per_seq, d.block_table_stride, d.block_size = 4, 100, 8, 8, 16
    d.device_block_stride, d.num_device_blocks, d.scale = 16 * 8 * 128 * 2, 64, 0.1
    d.workspace, d.workspace_bytes = 0x100000, 1 << 30
    for k, v in over.items():
        if k in ("q", "out"):
            getattr(d, k).base, getattr(d, k).token_stride, getattr(d, k).head_stride = v
        else:
            setattr(d, k, v)
    return d


@pytest.mark.parametrize("over,code", [
    (dict(head_dim=96), "UNSUPPORTED"), (dict(group=0), "INVALID_ARG"), (dict(group=300), "TOO_LARGE"), (dict(kv_heads=0), "INVALID_ARG"),
    (dict(prefix_len=-1), "INVALID_ARG"), (dict(prefix_len=1 << 31), "TOO_LARGE"), (dict(max_blocks_per_seq=1 << 28, block_table_stride=1 << 28), "TOO_LARGE"),
    (dict(num_seqs=1 << 31), "TOO_LARGE"), (dict(block_size=0), "INVALID_ARG"), (dict(device_block_stride=4096), "INVALID_ARG"),
    (dict(block_table_stride=7), "INVALID_ARG"), (dict(scale=float("inf")), "INVALID_ARG"), (dict(seq_lens=0), "INVALID_ARG"), (dict(prefix_table=0), "INVALID_ARG"),
    (dict(block_tables=0), "INVALID_ARG"), (dict(workspace=0), "ALIGNMENT"), (dict(workspace=0x100010), "ALIGNMENT"), (dict(workspace_bytes=4096), "INVALID_ARG"),
    (dict(type=2), "INVALID_ARG"), (dict(kv_format=5), "INVALID_ARG"), (dict(q=(0x10008, 8192, 256)), "ALIGNMENT"), (dict(out=(0x10000, 4096, 256)), "INVALID_ARG"),
    (dict(out=(0x10000, -8192, 256)), "INVALID_ARG"), (dict(k_cache=0), "INVALID_ARG")])
def test_attention_refusals(hfk, over, code):
    d = attention_desc(hfk, **over)
    assert hfk.lib().hfk_shared_prefix_attention(C.byref(d), 0, None) == getattr(hfk, "HFK_ERR_" + code), hfk.last_error()


def test_attention_workspace(hfk):
    f = hfk.lib().hfk_prefix_attention_workspace
    sizes = [f(C.byref(attention_desc(hfk, num_seqs=n)), 0) for n in (1, 4, 64, 1024, 5000)]
    assert sizes[0] > 0 and sizes == sorted(sizes) and sizes[3] == sizes[4]     # beyond 1024 sequences: in turns
    assert f(C.byref(attention_desc(hfk, head_dim=80)), 0) == 0
    assert f(None, 0) == 0
    d = attention_desc(hfk, num_seqs=0, seq_lens=0, block_tables=0)
    assert hfk.lib().hfk_shared_prefix_attention(C.byref(d), 0, None) == hfk.HFK_OK


def test_operators_refuse_host_tensors():
    import pcie_through  # noqa: F401

    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError):
        torch.ops.pcie_through.kv_write(x, x, torch.zeros(2, 16, 2, 64), torch.zeros(2, 16, 2, 64), torch.zeros(2, dtype=torch.long), 16, 0)


# ---- the oracle ----------------------------------------------------------------------------------------------------
def test_codes_are_the_nearest_and_ties_go_to_even():
    x = torch.tensor([[448.0, 1.0, 1.0625, 1.1875, -17.0, 2.0 ** -9, 2.0 ** -10, 0.0]])
    codes, scale = o.encode(x, "e4m3")
    assert float(scale) == 1.0
    assert codes.float().tolist() == [[448.0, 1.0, 1.0, 1.25, -16.0, 2.0 ** -9, 0.0, 0.0]]
    codes, scale = o.encode(torch.tensor([[127.0, 0.5, 1.5, -2.5, -126.6]]), "int8")
    assert float(scale) == 1.0 and codes.tolist() == [[127, 0, 2, -2, -127]]
    codes, scale = o.encode(torch.zeros(1, 8), "e4m3")
    assert float(scale) == 2.0 ** -126 and (codes.float() == 0).all()


def test_attention_of_the_oracle_is_softmax_over_the_concatenated_keys():
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(2, 6, 4, 2, 8, generator=g)
    q = torch.randn(2, 4, 8, generator=g)
    tables = torch.tensor([[2, 5], [4, -1]])
    out, lse, _, _ = o.attention(q, k, v, torch.tensor([1, 0]), 6, tables, torch.tensor([5, 0]), 4, 0.3)
    kk = torch.cat([k[1], k[0, :2], k[2], k[5, :1]])
    vv = torch.cat([v[1], v[0, :2], v[2], v[5, :1]])
    want = torch.nn.functional.scaled_dot_product_attention(q[0, 1:2].double(), kk[:, 0].double(), vv[:, 0].double(), scale=0.3)
    assert torch.allclose(out[0, 1:2], want)
    want = torch.nn.functional.scaled_dot_product_attention(q[1, 3:].double(), kk[:6, 1].double(), vv[:6, 1].double(), scale=0.3)
    assert torch.allclose(out[1, 3:], want)


def test_rope_table_and_rotation_keep_lengths():
    from heterofusedkernels_b200.connector import rope_table

    t = rope_table(50, 16, 100.0, scale=2.0, device="cpu")
    assert t.shape == (50, 16) and t.dtype == torch.float32
    assert torch.allclose(t[:, :8] ** 2 + t[:, 8:] ** 2, torch.ones(50, 8))
    assert torch.allclose(t[7, 3], torch.tensor(3.5 * 100.0 ** (-6 / 16)).cos())
    x = torch.randn(3, 2, 32, generator=torch.Generator().manual_seed(1))
    for inter in (False, True):
        y = o.norm_rope(x, torch.tensor([0, 9, 49]), t, None, 0.0, inter)
        assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1)) and torch.equal(y[0], x[0].double())
        assert torch.equal(y[..., 16:], x[..., 16:].double())
