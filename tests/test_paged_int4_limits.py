"""Scales of the 4-bit paged decode that its powers of two cannot hold, refused before a device is touched."""
from butterfly_b200 import _lib

from .test_paged_int4_validation import _decode


def test_scales_beyond_fp32():
    assert _decode(scale=2.4e38) == _lib.BAD_SHAPE  # times log2(e) it is infinite
    assert _decode(scale=float("inf")) == _lib.BAD_SHAPE and _decode(scale=-1.0) == _lib.BAD_SHAPE
    assert _decode(q=(0, 8, 1, 128), scale=1e38) == _lib.OK
