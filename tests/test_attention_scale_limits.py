"""CPU: the scales that the biased attention refuses.  Its kernels hold the bias in
units of the scale, slope x distance / (scale log2 e) in fp32: with a slope of 1
and 2^31 keys that is past 3.4e38 from a scale of 4e-30 down."""
import ctypes

import pytest
import torch

from myvllm_amd import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="host pointers in the calls")
ARG = -13


def D(t):
    return None if t is None else ctypes.byref(_lib.describe(t))


def calls(scale, cap, slopes):
    q, k, c = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((2, 4, 64), (2, 2, 64), (6, 16, 2, 64)))
    i = torch.zeros(2, 3, dtype=torch.int32)
    s = D(slopes)
    lib, o = _lib.load(), D(q.clone())
    return (lib.flash_attention_varlen_scored(D(q), D(k), D(k), D(i[0]), o, s, None, 2, scale, cap, 1, None),
            lib.paged_attention_prefill_scored(D(q), D(c), D(c), D(i), D(i[0, :2]), D(i[0]), o, None, s, None, 2, scale,
                                               cap, None),
            lib.paged_attention_decode_scored(D(q), D(c), D(c), D(i), D(i[0, :2]), o, None, s, 1, scale, cap, None))


@pytest.mark.parametrize("scale, cap, biased, refused", [
    (1e-38, 0.0, True, True), (-1e-30, 0.0, True, True), (9e-21, 0.0, True, True),
    (1.1e-20, 0.0, True, False), (0.0, 0.0, True, False), (1e-38, 5.0, True, False), (1e-38, 5.0, False, False),
])
def test_scales_with_slopes(scale, cap, biased, refused):
    slopes = torch.ones(4) if biased else None
    assert [c == ARG for c in calls(scale, cap, slopes)] == [refused] * 3
