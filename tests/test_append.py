"""CPU: what the paged append refuses, and its oracle."""
import ctypes

import pytest
import torch

from myvllm_amd import _lib, paged_kv_append
from oracle.attention import paged_kv_append_ref, rotate_ref

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="host pointers in the calls")
ERR = {"NULL": -1, "NDIM": -2, "SHAPE": -3, "DTYPE": -4, "STRIDE": -5, "HEADS": -6, "HEAD_DIM": -7, "ALIGN": -9,
       "RANGE": -11}
Z = torch.zeros
BF = torch.bfloat16


def args(D=128, T=5, N=2):
    return dict(k=Z(T, 2, D, dtype=BF), v=Z(T, 2, D, dtype=BF), kc=Z(6, 16, 2, D, dtype=BF),
                vc=Z(6, 16, 2, D, dtype=BF), tab=Z(N, 3, dtype=torch.int32), ctx=Z(N, dtype=torch.int32), q=Z(T, 4, D, dtype=BF),
                out=Z(T, 4, D, dtype=BF), cu=Z(N + 1, dtype=torch.int32), cos=Z(48, 32), sin=Z(48, 32))


def call(a):
    d = [None if t is None else (t if isinstance(t, _lib.GdnTensor) else _lib.describe(t)) for t in a.values()]
    return _lib.load().paged_kv_append(*(None if t is None else ctypes.byref(t) for t in d), 0, None)


@cpu_only
@pytest.mark.parametrize(
    "change, code",
    [
        (dict(k=None), "NULL"),
        (dict(k=Z(5, 256, dtype=BF)), "NDIM"),
        (dict(v=Z(4, 2, 128, dtype=BF)), "SHAPE"),
        (dict(kc=Z(6, 16, 4, 128, dtype=BF), vc=Z(6, 16, 4, 128, dtype=BF)), "SHAPE"),
        (dict(vc=Z(7, 16, 2, 128, dtype=BF)), "SHAPE"),
        (dict(ctx=Z(3, dtype=torch.int32)), "SHAPE"),
        (dict(tab=Z(2, 3)), "DTYPE"),
        (dict(k=Z(5, 2, 128), v=Z(5, 2, 128)), "DTYPE"),
        (dict(vc=Z(6, 16, 2, 128, dtype=torch.float16)), "DTYPE"),
        (dict(q=Z(5, 4, 128, dtype=torch.float16)), "DTYPE"),
        (dict(q=None), "NULL"),
        (dict(out=None), "NULL"),
        (dict(out=Z(5, 2, 128, dtype=BF)), "SHAPE"),
        (dict(q=Z(4, 4, 128, dtype=BF)), "SHAPE"),
        (dict(cu=None), "SHAPE"),  # five tokens, two sequences
        (dict(cu=Z(4, dtype=torch.int32)), "SHAPE"),
        (dict(cu=Z(3)), "DTYPE"),
        (dict(cu=Z(6, dtype=torch.int32)[::2]), "STRIDE"),
        (dict(sin=None), "NULL"),
        (dict(sin=Z(47, 32)), "SHAPE"),
        (dict(cos=Z(48, 12), sin=Z(48, 12)), "SHAPE"),
        (dict(cos=Z(48, 72), sin=Z(48, 72)), "SHAPE"),
        (dict(cos=Z(48, 0), sin=Z(48, 0)), "SHAPE"),
        (dict(cos=Z(48, 32, dtype=BF), sin=Z(48, 32, dtype=BF)), "DTYPE"),
        (dict(cos=Z(32, 48).t()), "STRIDE"),
        (dict(cos=Z(48 * 32 + 1)[1:].view(48, 32)), "ALIGN"),
        (dict(k=Z(5 * 256 + 1, dtype=BF)[1:].view(5, 2, 128)), "ALIGN"),
        (dict(kc=Z(6 * 4096 + 1, dtype=BF)[1:].view(6, 16, 2, 128)), "ALIGN"),
        (dict(k=Z(5, 128, 2, dtype=BF).transpose(1, 2)), "STRIDE"),
        (dict(k=Z(5, 0, 128, dtype=BF), v=Z(5, 0, 128, dtype=BF), kc=Z(6, 16, 0, 128, dtype=BF),
              vc=Z(6, 16, 0, 128, dtype=BF)), "HEADS"),
    ],
)
def test_refusals(change, code):
    a = args()
    a.update(change)
    assert call(a) == ERR[code]


@cpu_only
def test_refused_sizes():
    assert call(args(D=96) | dict(cos=None, sin=None)) == ERR["HEAD_DIM"]
    a = args()
    a["tab"] = _lib.describe(a["tab"])
    a["tab"].shape[1] = 2**27  # x 16 keys = 2^31 positions
    assert call(a) == ERR["RANGE"]


def test_python_refusals():
    a = args()
    pos = [a[n] for n in ("q", "k", "v", "kc", "vc", "tab", "ctx")]
    with pytest.raises(ValueError, match="block_size"):
        paged_kv_append(*pos, 32)
    with pytest.raises(ValueError, match="GPU tensors"):
        paged_kv_append(*pos, 16, cu_seqlens=a["cu"])
    with pytest.raises(ValueError, match="none without q"):
        paged_kv_append(None, *pos[1:], 16, cu_seqlens=a["cu"], out=a["out"])


def test_oracle_rotation():
    """Norms of pairs stay, angles add, and the two layouts are each other's permutation."""
    x = torch.randn(3, 2, 8, dtype=torch.float64)
    ang = torch.rand(3, 3, dtype=torch.float64)
    y = rotate_ref(x, ang.cos(), ang.sin())
    assert torch.allclose(y[..., :3]**2 + y[..., 3:6]**2, x[..., :3]**2 + x[..., 3:6]**2)
    assert torch.equal(y[..., 6:], x[..., 6:])
    assert torch.allclose(rotate_ref(y, ang.cos(), ang.sin()), rotate_ref(x, (2 * ang).cos(), (2 * ang).sin()))
    to = [0, 3, 1, 4, 2, 5, 6, 7]
    assert torch.allclose(rotate_ref(x[..., to], ang.cos(), ang.sin(), True), y[..., to])


def test_oracle_append():
    k = torch.arange(5.0).view(5, 1, 1).expand(5, 1, 2) + 1
    kc, vc = Z(3, 2, 1, 2, dtype=torch.float64), Z(3, 2, 1, 2, dtype=torch.float64)
    q = paged_kv_append_ref(k, k, -k, kc, vc, torch.tensor([[2, 0], [1, -1]]), torch.tensor([3, 4]), [0, 2, 5])
    assert kc[..., 0, 0].tolist() == [[2, 0], [0, 3], [0, 1]]  # the second's tokens at 2 and 3 have no page
    assert torch.equal(vc, -kc) and torch.equal(q, k.double())
