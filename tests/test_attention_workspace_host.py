"""Sizes of shared_prefix_attention's workspace, without a GPU: one that is sized for the largest call holds every smaller one.  What a
call needs shows in what it refuses: the size is checked last of all, before any CUDA call that a host without a GPU fails in."""
import ctypes as C
import random

import pytest

from tests.test_cache_ops_host import attention_desc


def need(hfk, **over):
    """Bytes below which the call is refused, from its message."""
    d = attention_desc(hfk, workspace_bytes=0, **over)
    ctas = over.get("ctas", 0)
    assert hfk.lib().hfk_shared_prefix_attention(C.byref(d), ctas, None) == hfk.HFK_ERR_INVALID_ARG
    words = hfk.last_error().split()
    assert words[-1] == "needed", hfk.last_error()
    return int(words[-2])


def given(hfk, ctas=0, **over):
    return hfk.lib().hfk_prefix_attention_workspace(C.byref(attention_desc(hfk, **over)), ctas)


GEOMETRIES = [dict(kv_heads=8, group=4), dict(kv_heads=1, group=8), dict(kv_heads=4, group=7, head_dim=64, device_block_stride=16 * 4 * 64 * 2),
              dict(kv_heads=2, group=1), dict(kv_heads=1, group=64)]


def shaped(geometry, **more):
    g = dict(geometry, **more)
    d, h = g.get("head_dim", 128), g["kv_heads"]
    row = h * g["group"] * d * 2
    return dict(g, device_block_stride=16 * h * d * 2, q=(0x10000, row, d * 2), out=(0x10000, row, d * 2))


@pytest.mark.parametrize("geometry", GEOMETRIES, ids=[str(i) for i in range(len(GEOMETRIES))])
@pytest.mark.parametrize("prefix", [0, 100, 897, 8192, 32768])
def test_the_size_for_a_batch_holds_every_smaller_batch(hfk, geometry, prefix):
    most = 0
    for n in range(1, 1100):
        over = shaped(geometry, num_seqs=n, prefix_len=prefix)
        most = max(most, need(hfk, **over))
        assert most <= given(hfk, **over)


def test_the_size_holds_every_shorter_prefix_and_narrower_table(hfk):
    rng = random.Random(1)
    for _ in range(300):
        geometry = rng.choice(GEOMETRIES)
        big = dict(num_seqs=rng.randint(1, 1500), prefix_len=rng.randint(0, 40000), max_blocks_per_seq=rng.randint(0, 3000))
        big["block_table_stride"] = big["max_blocks_per_seq"]
        ctas = rng.choice([0, 0, 1, 7, 148, 1000])
        bound = given(hfk, ctas, **shaped(geometry, **big))
        for _ in range(20):
            small = dict(num_seqs=rng.randint(1, big["num_seqs"]), prefix_len=rng.choice([0, rng.randint(0, big["prefix_len"]), big["prefix_len"]]),
                         max_blocks_per_seq=rng.randint(0, big["max_blocks_per_seq"]), block_table_stride=big["block_table_stride"])
            d = attention_desc(hfk, workspace_bytes=0, **shaped(geometry, **small))
            assert hfk.lib().hfk_shared_prefix_attention(C.byref(d), ctas, None) == hfk.HFK_ERR_INVALID_ARG
            assert int(hfk.last_error().split()[-2]) <= bound, (geometry, big, small, ctas)
