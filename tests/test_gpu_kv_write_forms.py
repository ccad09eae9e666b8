"""kv_write and qk_norm_rope_write at the numbers of rows where heads up to 64 change to the form with 32 elements a lane."""
import pytest

from tests.test_gpu_cache_ops import BF16, FP16, op, test_kv_write_is_bit_exact, test_qk_norm_rope_write  # noqa: F401

one_write, one_rope = test_kv_write_is_bit_exact, test_qk_norm_rope_write
del test_kv_write_is_bit_exact, test_qk_norm_rope_write        # not collected here a second time

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype,tokens,heads,dim,block", [(BF16, 16400, 2, 64, 16), (FP16, 11000, 3, 48, 7), (BF16, 4100, 8, 16, 16), (FP16, 5462, 6, 32, 128)])
def test_many_rows_of_small_heads_are_bit_exact(op, cuda_device, fmt, dtype, tokens, heads, dim, block):  # noqa: F811
    assert tokens * 2 * heads >= 1 << 16
    one_write(op, cuda_device, fmt, dtype, tokens, heads, dim, block)


@pytest.mark.parametrize("fmt", ["raw", "e4m3", "int8"])
@pytest.mark.parametrize("dtype,tokens,heads,group,dim,rot,interleaved,norm", [
    (BF16, 5500, 2, 4, 64, 64, False, "qk"), (FP16, 7400, 1, 7, 64, 32, True, "k"), (BF16, 6600, 2, 3, 48, 16, False, "q"),
    (FP16, 17000, 1, 2, 16, 16, False, "qk")])
def test_many_rotated_rows_of_small_heads(op, cuda_device, fmt, dtype, tokens, heads, group, dim, rot, interleaved, norm):  # noqa: F811
    assert tokens * heads * (group + 2) >= 1 << 16
    one_rope(op, cuda_device, fmt, dtype, tokens, heads, group, dim, rot, interleaved, norm)
