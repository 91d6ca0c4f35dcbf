"""CPU: what the scored and the shared attention refuse, and the reference of their scores."""
import ctypes
import math

import pytest
import torch

from myvllm_amd import _lib, flash_attention_prefill, paged_flash_attention_decode, paged_flash_attention_decode_shared
from oracle.attention import attention_weights_ref

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="host pointers in the calls")
Z, BF, I32 = torch.zeros, torch.bfloat16, torch.int32
NULL, NDIM, SHAPE, DTYPE, STRIDE, HEADS, HEAD_DIM, ALIGN, RANGE, ARG = -1, -2, -3, -4, -5, -6, -7, -9, -11, -13


def D(t):
    return t if t is None or not isinstance(t, torch.Tensor) else ctypes.byref(_lib.describe(t))


SCORES = [
    (dict(slopes=Z(3)), SHAPE), (dict(slopes=Z(4, dtype=BF)), DTYPE), (dict(slopes=Z(8)[::2]), STRIDE),
    (dict(slopes=Z(4, 1)), NDIM), (dict(cap=-1.0), ARG), (dict(cap=4097.0), ARG), (dict(cap=9e-4), ARG),
    (dict(cap=math.nan), ARG), (dict(cap=math.inf), ARG),
]
MASKS = [(dict(pfx=Z(3, dtype=I32)), SHAPE), (dict(pfx=Z(2)), DTYPE), (dict(pfx=Z(4, dtype=I32)[::2]), STRIDE)]


@cpu_only
@pytest.mark.parametrize("change, code", SCORES + MASKS + [(dict(pfx=Z(2, dtype=I32), causal=0), ARG),
                                                           (dict(D=72), HEAD_DIM), (dict(cu=Z(3)), DTYPE)])
def test_varlen_refusals(change, code):
    a = dict(slopes=None, pfx=None, cap=5.0, causal=1, D=64, cu=Z(3, dtype=I32)) | change
    q, k = Z(5, 4, a["D"], dtype=BF), Z(5, 2, a["D"], dtype=BF)
    assert _lib.load().flash_attention_varlen_scored(D(q), D(k), D(k), D(a["cu"]), D(q.clone()), D(a["slopes"]),
                                                     D(a["pfx"]), 5, 1.0, a["cap"], a["causal"], None) == code


@cpu_only
@pytest.mark.parametrize("change, code", SCORES + MASKS + [(dict(ctx=Z(3, dtype=I32)), SHAPE),
                                                           (dict(ws=Z(4, dtype=BF)), DTYPE)])
def test_paged_prefill_refusals(change, code):
    a = dict(slopes=None, pfx=None, cap=0.0, ctx=Z(2, dtype=I32), ws=None) | change
    q, c = Z(5, 4, 64, dtype=BF), Z(6, 16, 2, 64, dtype=BF)
    assert _lib.load().paged_attention_prefill_scored(
        D(q), D(c), D(c), D(Z(2, 3, dtype=I32)), D(a["ctx"]), D(Z(3, dtype=I32)), D(q.clone()), D(a["ws"]),
        D(a["slopes"]), D(a["pfx"]), 5, 1.0, a["cap"], None) == code


@cpu_only
@pytest.mark.parametrize("change, code", SCORES + [(dict(splits=2), NULL), (dict(splits=0), RANGE)])
def test_decode_refusals(change, code):
    a = dict(slopes=None, cap=0.0, splits=1) | change
    q, c = Z(2, 4, 64, dtype=BF), Z(6, 16, 2, 64, dtype=BF)
    assert _lib.load().paged_attention_decode_scored(
        D(q), D(c), D(c), D(Z(2, 3, dtype=I32)), D(Z(2, dtype=I32)), D(q.clone()), None, D(a["slopes"]), a["splits"],
        1.0, a["cap"], None) == code


def shared_args():
    n = _lib.load().paged_attention_decode_shared_workspace_size(4, 2, 4, 2, 64)
    return dict(q=Z(4, 4, 64, dtype=BF), kc=Z(6, 16, 2, 64, dtype=BF), vc=Z(6, 16, 2, 64, dtype=BF),
                tab=Z(4, 3, dtype=I32), ctx=Z(4, dtype=I32), lens=Z(2, dtype=I32), groups=Z(3, dtype=I32),
                out=Z(4, 4, 64, dtype=BF), ws=Z(n))


@cpu_only
@pytest.mark.parametrize(
    "change, code",
    [
        (dict(lens=None), NULL), (dict(lens=Z(2)), DTYPE), (dict(lens=Z(4, dtype=I32)[::2]), STRIDE),
        (dict(lens=Z(1, 2, dtype=I32)), NDIM), (dict(lens=Z(3, dtype=I32)), SHAPE), (dict(groups=None), SHAPE),
        (dict(groups=Z(3)), DTYPE), (dict(groups=Z(6, dtype=I32)[::2]), STRIDE), (dict(groups=Z(2, dtype=I32)), SHAPE),
        (dict(ws=None), NULL), (dict(ws=Z(8)), SHAPE),
        (dict(ws=Z(2 * 10**7, dtype=BF)), DTYPE), (dict(ws=Z(2 * 10**7)[1:]), ALIGN), (dict(ws=Z(2, 2 * 10**7)), NDIM),
        (dict(q=Z(4, 3, 64, dtype=BF), out=Z(4, 3, 64, dtype=BF)), HEADS), (dict(ctx=Z(3, dtype=I32)), SHAPE),
        (dict(out=Z(4, 4, 64)), DTYPE), (dict(kc=Z(6, 16, 2, 72, dtype=BF), vc=Z(6, 16, 2, 72, dtype=BF)), SHAPE),
    ],
)
def test_shared_refusals(change, code):
    a = shared_args() | change
    assert _lib.load().paged_attention_decode_shared(*(D(t) for t in a.values()), 1.0, None) == code


@cpu_only
def test_shared_range():
    """2^27 columns of 16 keys are 2^31 positions (refused before any HIP call)."""
    a = shared_args()
    tab = _lib.describe(a.pop("tab"))
    tab.shape[1] = 2**27
    d = [D(t) for t in a.values()]
    d.insert(3, ctypes.byref(tab))
    assert _lib.load().paged_attention_decode_shared(*d, 1.0, None) == RANGE


def test_shared_workspace():
    """Partials of the own keys' pieces (a slot per sequence and unit) and their
    prices, the plan, 128 rows of D + 4 floats per workgroup of shared keys
    (none for single sequences)."""
    size = _lib.load().paged_attention_decode_shared_workspace_size

    def want(B, G, Hq, D, units, wgs):
        return ((B + units) * Hq * (D + 4) + (B + 4) // 4 * 4 + 4 + 4 * B + 8 * G + 8 * (-(-wgs // 8) * 8)
                + wgs * 128 * (D + 4))

    assert size(1, 1, 16, 2, 256) == want(1, 1, 16, 256, 256, 0)
    assert size(64, 0, 16, 2, 256) == want(64, 0, 16, 256, 256, 0)
    assert size(4, 1, 16, 2, 256) == want(4, 1, 16, 256, 256, 256)
    assert size(4, 1, 128, 2, 64) == want(4, 1, 128, 64, 64, 768)
    assert size(4, 1, 16, 2, 96) == 0 and size(4, 1, 16, 3, 64) == 0
    rows = 2 * (65535 * 8 // 128 + 1)
    assert size(65535, 1, 16, 2, 256) == want(65535, 1, 16, 256, 16384, rows)


def test_python_refusals():
    q, c, i = Z(2, 4, 64, dtype=BF), Z(6, 16, 2, 64, dtype=BF), Z(2, 3, dtype=I32)
    with pytest.raises(ValueError, match="block_size"):
        paged_flash_attention_decode_shared(q, c, c, i, i[0, :2], i[0, :1], 1.0, 8)
    for fn in (lambda: paged_flash_attention_decode_shared(q, c, c, i, i[0, :2], i[0, :1], 1.0, 16),
               lambda: paged_flash_attention_decode(q, c, c, i, i[0, :2], 1.0, 16, softcap=2.0),
               lambda: flash_attention_prefill(q, q, q, i[0, :2], 1.0, 4, 4, 64, 64, True, alibi_slopes=Z(4))):
        with pytest.raises(ValueError, match="GPU tensors"):
            fn()


def test_reference_scores():
    q = torch.randn(3, 2, 4, dtype=torch.float64)
    k = torch.randn(5, 1, 4, dtype=torch.float64)
    x, p = attention_weights_ref(q, k, [0, 2, 4], 0.5, softcap=1.5, slopes=torch.tensor([0.25, 2.0]), prefix=2)
    for n, i in enumerate((0, 2, 4)):
        for h, s in enumerate((0.25, 2.0)):
            w = [1.5 * math.tanh(0.5 * float(q[n, h] @ k[j, 0]) / 1.5) - s * abs(i - j)
                 if j <= i or j < 2 else -math.inf for j in range(5)]
            assert x[n, h].tolist() == pytest.approx(w)
            z = sum(math.exp(v) for v in w)
            assert p[n, h].tolist() == pytest.approx([math.exp(v) / z for v in w])
    assert attention_weights_ref(q, k, [-1, -1, -1], 1.0)[1].abs().sum() == 0
