"""The dense feed-forward operators at the ends of what their calls allow: alignment, the range of the norm's statistics, kernels that only some
sizes reach, results of a row in calls of different row counts.  References as in test_dense_ffn.py."""
import ctypes

import pytest

from helpers import native
from test_dense_ffn import fake_context


def test_scales_of_prepared_weights_lie_at_16_bytes():
    """The many-row products copy them into LDS sixteen bytes a lane, so every call that writes or reads them asks for that alignment.  Addresses
    are never followed."""
    lib, memory = native.load(), fake_context()
    ctx, P, Q, i64 = ctypes.addressof(memory), 1 << 20, 1 << 21, ctypes.c_int64
    for off in (4, 8, 12):
        assert lib.ca_mxfp4_prepare(ctx, 16, 64, P, P, Q, Q + off, None) == -1
        assert lib.ca_mxfp4_linear(ctx, 64, 16, 256, P, P, 0, P, P + off, P, i64(16), None) == -1
        assert lib.ca_mxfp4_swiglu(ctx, 64, 256, 256, P, P, 0, P, P + off, P, P, P, P, P, 0, None) == -1
        assert lib.ca_mxfp4_swiglu(ctx, 64, 256, 256, P, P, 0, P, P, P, P + off, P, P, P, 0, None) == -1
