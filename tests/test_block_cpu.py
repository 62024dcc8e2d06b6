"""Rotary and block-cache entries without a device: what they refuse before touching one."""
import ctypes as C

import numpy as np


def test_null_checks_without_device(skv):
    L = skv.lib()
    pos = np.zeros(1, np.int32).ctypes.data_as(C.c_void_p)
    h = C.c_void_p()
    assert L.swiftkv_rotary_create(None, 64, 10, 10000.0, None, C.byref(h)) == skv.EINVAL
    assert L.swiftkv_rope_lut_generate_scaled(None, 10, 10000.0, None, C.byref(h)) == skv.EINVAL
    assert L.swiftkv_rotary(None, None, None, 0, None, 0, 0, 0, 0, pos, 1, 1, 1, 64) == skv.EINVAL
    assert L.swiftkv_block_cache_create(None, 1, 1, 1, 1, 64, 64, C.byref(h)) == skv.EINVAL
    assert L.swiftkv_block_append(None, None, 0, None, 0, 0, None, 0, 0, pos, 1, 1) == skv.EINVAL
    assert L.swiftkv_block_values(None, None, 0, 0, pos, 1, 1, 0, None, None) == skv.EINVAL
    assert L.swiftkv_block_attention(None, None, 0, None, 0, None, 0, 0, None, 0, 0, pos, 1, 1, 0.0, None, None,
                                     0) == skv.EINVAL
    assert b"null" in L.swiftkv_last_error()
    assert L.swiftkv_block_evict(None, None, 0, 1, 0, pos, 1, 2, 0, 1, None, None, None) == skv.EINVAL
    assert L.swiftkv_block_cache_bytes(None) == 0 and L.swiftkv_block_cache_blocks(None) == 0
    assert L.swiftkv_rotary_destroy(None) == skv.OK and L.swiftkv_block_cache_destroy(None) == skv.OK


def test_scaling_structure(skv):
    """The mirror of swiftkv_rope_scaling: two 32-bit numbers, then four doubles."""
    assert C.sizeof(skv.RopeScaling) == 40
    s = skv.RopeScaling(skv.ROPE_BANDS, 8.0, 4096, 1.0, 4.0)
    assert (s.kind, s.original_positions, s.factor, s.low, s.high, s.magnitude) == (3, 4096, 8.0, 1.0, 4.0, 1.0)
