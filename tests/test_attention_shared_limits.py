"""CPU: the sizes up to which the shared decode counts in 32 bits."""
import ctypes

import pytest
import torch

from myvllm_amd import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="host pointers in the calls")
RANGE = -11


def call(B, cols, page=16):
    """B sequences with tables of `cols` pages: the shapes of such a call over
    small tensors, which are not read (refused, or without a device to run on)."""
    n = _lib.load().paged_attention_decode_shared_workspace_size(B, 1, 1, 1, 64)
    i32 = torch.zeros(2, 2, dtype=torch.int32)
    q, c = torch.zeros(1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, page, 1, 64, dtype=torch.bfloat16)
    d = dict(q=_lib.describe(q), kc=_lib.describe(c), vc=_lib.describe(c), tab=_lib.describe(i32),
             ctx=_lib.describe(i32[0]), lens=_lib.describe(i32[0, :1]), groups=None, out=_lib.describe(q),
             ws=_lib.describe(torch.zeros(4)))
    for t in ("q", "tab", "ctx", "out"):
        d[t].shape[0] = B
    d["tab"].shape[1] = cols
    d["tab"].stride[0] = cols
    d["ws"].shape[0] = n
    return _lib.load().paged_attention_decode_shared(*(None if t is None else ctypes.byref(t) for t in d.values()),
                                                     1.0, None)


@pytest.mark.parametrize("B, cols, page, refused", [
    (32768, 65533, 16, True),  # 2^15 (65,533 tiles + 4 for a start) is 2^31 + 2^15
    (65535, 32766, 16, True),  # as many as one less than the plain decode's limit
    (32768, 65532, 16, True),  # 2^31
    (32768, 65531, 16, False),
    (65535, 32764, 16, False),
    (65535, 65529, 8, True),  # 32,765 tiles of 16 keys, the last one of 8 keys
    (65535, 65528, 8, False),
    (1, 2**26, 16, False),  # 2^30 positions
    (1, 2**26 + 1, 16, True),
    (1, 2**30 // 48 + 1, 48, True),
])
def test_prices_and_positions(B, cols, page, refused):
    assert (call(B, cols, page) == RANGE) == refused
