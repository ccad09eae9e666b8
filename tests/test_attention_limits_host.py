"""Limits of shared_prefix_attention's arguments, without a GPU."""
import ctypes as C

import pytest

from tests.test_cache_ops_host import attention_desc


@pytest.mark.parametrize("scale,fine", [(2.3e38, True), (-2.3e38, True), (0.0, True), (1e-45, True), (2.4e38, False), (-2.4e38, False), (3.4e38, False),
                                        (float("nan"), False), (float("-inf"), False)])
def test_a_scale_whose_product_with_log2_e_is_not_finite_is_refused(hfk, scale, fine):
    """What is not refused goes on to the next check, that of the workspace."""
    d = attention_desc(hfk, scale=scale, workspace_bytes=0)
    assert hfk.lib().hfk_shared_prefix_attention(C.byref(d), 0, None) == hfk.HFK_ERR_INVALID_ARG
    assert ("workspace" if fine else "scale is not finite") in hfk.last_error()
