"""CPU: the 4-bit oracle, and what the entries of 4-bit caches, of positions of
their own and of the read refuse."""
import ctypes

import pytest
import torch

import myvllm_amd as ops
from myvllm_amd import _lib
from oracle.fp4 import GRID, TOP, axis_of, pack_ref, unpack_ref

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="host pointers in the calls")
ERR = {"NULL": -1, "NDIM": -2, "SHAPE": -3, "DTYPE": -4, "STRIDE": -5, "HEADS": -6, "HEAD_DIM": -7, "ALIGN": -9,
       "RANGE": -11, "ARG": -13}
Z = torch.zeros
BF, U8, I32 = torch.bfloat16, torch.uint8, torch.int32


def test_oracle_values_stay():
    """Rows of representable values are their own packing."""
    g = torch.Generator().manual_seed(0)
    for dt, top in TOP.items():
        for e in (-top, -3, 0, top):
            x = torch.tensor(GRID)[torch.randint(0, 8, (6, 32), generator=g)] * (1 - 2 * torch.randint(0, 2, (6, 32), generator=g))
            x[:, 0] = 6  # (the scale is then 2^e)
            x = (x.double() * 2.0**e).to(dt)
            codes, scales = pack_ref(x)
            assert (scales == e + 127).all()
            assert torch.equal(unpack_ref(codes, scales), x.double())


def test_oracle_rounding():
    x = torch.zeros(32)
    x[:12] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5, 0.26, 5.01, -0.24])
    got = unpack_ref(*pack_ref(x.to(torch.float16)))
    assert got[:12].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -4, 0.5, 6, 0]
    # past 1.5 * 2^k the scale goes up: 6.01 / 2 rounds to 3
    x[0] = 6.01
    assert unpack_ref(*pack_ref(x.to(torch.float16)))[0] == 6
    x[0] = 7.9
    assert unpack_ref(*pack_ref(x.to(torch.float16)))[0] == 8
    for bad in (float("inf"), float("nan")):
        x[0] = bad
        assert unpack_ref(*pack_ref(x.to(BF))).isnan().all()
    # limits of the exponent: fp16's largest saturates, its small numbers are coarse
    y = torch.full((32,), 65504.0, dtype=torch.float16)
    assert (unpack_ref(*pack_ref(y)) == 6 * 2.0**13).all()
    y = torch.full((32,), 2.0**-14, dtype=torch.float16)
    assert (unpack_ref(*pack_ref(y)) == 2.0**-14).all()
    assert (unpack_ref(*pack_ref(y / 4)) == 0).all()


def test_oracle_error_bound():
    """Half the widest step: 6 - 4 of the scale is 2, and the largest of a block is above 3 scales."""
    x = torch.randn(50, 256, generator=torch.Generator().manual_seed(1)).to(BF)
    err = (unpack_ref(*pack_ref(x)) - x.double()).abs().unflatten(-1, (-1, 32))
    most = x.double().abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
    assert (err <= most / 3).all()


def test_axis_order():
    assert axis_of([1, 3, 2], False) == [0, 1, 1, 1, 2, 2]
    assert axis_of([3, 2, 2], True) == [0, 1, 2, 0, 1, 2, 0]
    assert axis_of([1, 3, 0, 2], True) == [0, 1, 3, 1, 3, 1]


def append_args(D=128, T=5, N=2, page=16):
    return dict(k=Z(T, 2, D, dtype=BF), v=Z(T, 2, D, dtype=BF), kc=Z(6, page, 2, D // 2, dtype=U8),
                vc=Z(6, page, 2, D // 2, dtype=U8), tab=Z(N, 3, dtype=I32), ctx=Z(N, dtype=I32),
                q=Z(T, 4, D, dtype=BF), out=Z(T, 4, D, dtype=BF), cu=Z(N + 1, dtype=I32), cos=Z(48, 32), sin=Z(48, 32),
                pos=Z(3, T, dtype=I32), ks=Z(6, 2, D // 32, page, dtype=U8), vs=Z(6, 2, D // 32, page, dtype=U8))


def code_of(fn, a, *scalars):
    d = [None if t is None else ctypes.byref(t if isinstance(t, _lib.GdnTensor) else _lib.describe(t)) for t in a]
    return getattr(_lib.load(), fn)(*d, *scalars, None)


SCALE_REFUSALS = [
    (dict(ks=None), "NULL"),
    (dict(kc=Z(6, 16, 2, 128, dtype=BF), vc=Z(6, 16, 2, 128, dtype=BF)), "SHAPE"),
    (dict(kc=Z(6, 16, 2, 64, dtype=BF), vc=Z(6, 16, 2, 64, dtype=BF)), "DTYPE"),
    (dict(ks=Z(6, 2, 4, 16)), "DTYPE"),
    (dict(vs=Z(6, 2, 4, 17, dtype=U8)), "SHAPE"),
    (dict(ks=Z(6, 2, 8, 16, dtype=U8)), "SHAPE"),
    (dict(ks=Z(5, 2, 4, 16, dtype=U8)), "SHAPE"),
    (dict(ks=Z(6, 2, 4, dtype=U8)), "NDIM"),
    (dict(ks=Z(6, 2, 16, 4, dtype=U8).transpose(2, 3)), "STRIDE"),
    (dict(vs=Z(6 * 2 * 4 * 16 + 1, dtype=U8)[1:].view(6, 2, 4, 16)), "ALIGN"),
    (dict(ks=Z(6, 2, 4, 18, dtype=U8)[..., :16]), "ALIGN"),
    (dict(kc=Z(6, 16, 2, 72, dtype=U8)[..., :64], vc=Z(6, 16, 2, 72, dtype=U8)[..., :64]), "ALIGN"),
]


@cpu_only
@pytest.mark.parametrize(
    "change, code",
    SCALE_REFUSALS + [
        (dict(pos=Z(5, 5, dtype=I32)), "SHAPE"),
        (dict(pos=Z(3, 4, dtype=I32)), "SHAPE"),
        (dict(pos=Z(3, 5)), "DTYPE"),
        (dict(pos=Z(5, dtype=I32)), "NDIM"),
        (dict(pos=Z(5, 3, dtype=I32).t()), "STRIDE"),
        (dict(pos=Z(2, 5, dtype=I32)), "ARG"),  # two axes of the three sections
        (dict(cos=Z(48, 40), sin=Z(48, 40)), "ARG"),
        (dict(cos=None, sin=None), "NULL"),
    ],
)
def test_append_refusals(change, code):
    a = append_args()
    a.update(change)
    assert code_of("paged_kv_append_ex", a.values(), 0, 12, 10, 10, 0, 0) == ERR[code]


@cpu_only
def test_append_refused_sizes():
    a = append_args(page=8)  # no whole 16-key groups
    assert code_of("paged_kv_append_ex", a.values(), 0, 12, 10, 10, 0, 0) == ERR["SHAPE"]
    assert code_of("paged_kv_append_ex", append_args().values(), 0, 40, -8, 0, 0, 0) == ERR["ARG"]
    for name, dim, value in (("kc", 0, 2**32), ("ks", 0, 2**32), ("vc", 1, 2**28), ("vs", 2, 2**30), ("ks", 1, 2**31)):
        a = append_args()
        a[name] = _lib.describe(a[name])
        a[name].stride[dim] = value
        assert code_of("paged_kv_append_ex", a.values(), 0, 12, 10, 10, 0, 0) == ERR["RANGE"], (name, dim)
    for name in ("kc", "vs"):
        a = append_args()
        a[name] = _lib.describe(a[name])
        a[name].stride[0] = -1024
        assert code_of("paged_kv_append_ex", a.values(), 0, 12, 10, 10, 0, 0) == ERR["STRIDE"]


def attention_args(D=128, N=2):
    a = append_args(D, T=N, N=N)
    return dict(q=a["q"], kc=a["kc"], vc=a["vc"], ks=a["ks"], vs=a["vs"], tab=a["tab"], ctx=a["ctx"], cu=a["cu"],
                out=a["out"], ws=None)


def attention_code(a, decode, splits=1):
    if decode:
        return code_of("paged_attention_decode_fp4", [t for n, t in a.items() if n != "cu"], splits, ctypes.c_float(1.0))
    return code_of("paged_attention_prefill_fp4", a.values(), 4, ctypes.c_float(1.0))


@cpu_only
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("change, code", SCALE_REFUSALS + [(dict(q=Z(2, 3, 128, dtype=BF), out=Z(2, 3, 128, dtype=BF)), "HEADS"),
                                                           (dict(q=Z(2, 4, 128), out=Z(2, 4, 128)), "DTYPE")])
def test_attention_refusals(decode, change, code):
    a = attention_args()
    a.update(change)
    assert attention_code(a, decode) == ERR[code]


@cpu_only
def test_attention_refused_sizes():
    a = attention_args()
    a["tab"] = _lib.describe(a["tab"])
    a["tab"].shape[1] = 2**27
    assert attention_code(a, True) == attention_code(a, False) == ERR["RANGE"]
    a = attention_args()
    a["tab"] = Z(2, 0, dtype=I32)
    assert attention_code(a, False) == ERR["SHAPE"]
    assert attention_code(attention_args(), True, splits=3) == ERR["NULL"]  # no workspace
    assert attention_code(attention_args(), True, splits=257) == ERR["RANGE"]


@cpu_only
def test_few_refusals():
    def code(splits=2, most=3, ws=True, **change):
        a = attention_args()
        a.update(change)
        n = _lib.workspace_size("paged_attention_decode_workspace_size", 2, max(most, 0) * 4, 128, splits)
        a["ws"] = Z(n) if ws else None
        return code_of("paged_attention_few_fp4", a.values(), splits, ctypes.c_int64(most), ctypes.c_float(1.0))

    for change, want in SCALE_REFUSALS:
        assert code(**change) == ERR[want], change
    assert code(ws=False) == ERR["NULL"]
    assert code(splits=1) == code(splits=257) == ERR["RANGE"]
    assert code(most=0) == code(most=-1) == ERR["SHAPE"]
    assert code(cu=Z(1, dtype=I32), tab=Z(0, 3, dtype=I32), ctx=Z(0, dtype=I32)) == ERR["SHAPE"]
    a = attention_args()
    a["ws"] = Z(8)
    assert code_of("paged_attention_few_fp4", a.values(), 2, ctypes.c_int64(3), ctypes.c_float(1.0)) == ERR["SHAPE"]
    assert code_of("paged_attention_few_fp4", a.values(), 2, ctypes.c_int64(2**30), ctypes.c_float(1.0)) == ERR["RANGE"]


@cpu_only
def test_read_refusals():
    def code(scales=True, **change):
        a = append_args()
        a.update(change)
        return code_of("paged_kv_read", [a[n] for n in ("k", "v", "kc", "vc", "tab", "ctx", "cu")]
                       + ([a["ks"], a["vs"]] if scales else [None, None]))

    for change, want in SCALE_REFUSALS[:1] + SCALE_REFUSALS[2:]:
        assert code(**change) == ERR[want], change
    assert code(scales=False) == ERR["SHAPE"]
    sixteen = dict(kc=Z(6, 16, 2, 128, dtype=BF), vc=Z(6, 16, 2, 128, dtype=BF))
    assert code(scales=False, cu=None, **sixteen) == ERR["SHAPE"]  # five tokens of two sequences
    assert code(scales=False, cu=Z(3), **sixteen) == ERR["DTYPE"]
    assert code(scales=False, k=Z(5, 2, 128, dtype=torch.float16), v=Z(5, 2, 128, dtype=torch.float16), **sixteen) == ERR["DTYPE"]


def test_python_refusals():
    a = append_args()
    pos = [a[n] for n in ("q", "k", "v", "kc", "vc", "tab", "ctx")]
    scales = dict(k_scales=a["ks"], v_scales=a["vs"])
    rope = dict(cos=a["cos"], sin=a["sin"])
    for kw, match in (
        (dict(k_scales=a["ks"]), "come together"),
        (dict(sections=(16, 16)), "those of positions"),
        (dict(sections=(16, 16), **scales), "those of positions"),
        (dict(positions=a["pos"], sections=(12, 10, 10)), "cos and sin"),
        (dict(positions=a["pos"], **rope), "as many sections"),
        (dict(positions=a["pos"], sections=(12, 10), **rope), "as many sections"),
        (dict(positions=a["pos"], sections=(12, 10, 11), **rope), "32 frequencies"),
        (dict(positions=a["pos"], sections=(40, -4, -4), **rope), "32 frequencies"),
        (dict(positions=Z(5, 5, dtype=I32), sections=(8, 8, 8, 8, 0), **rope), "one to four"),
        (scales, "GPU tensors"),
    ):
        with pytest.raises(ValueError, match=match):
            ops.paged_kv_append(*pos, 16, cu_seqlens=a["cu"], **kw)
    caches = [a["kc"], a["vc"], a["tab"], a["ctx"]]
    q = a["q"][:2]
    for kw in (dict(softcap=20.0), dict(alibi_slopes=Z(4))):
        with pytest.raises(ValueError, match="plain scores"):
            ops.paged_flash_attention_decode(q, *caches, 1.0, 16, **scales, **kw)
    with pytest.raises(ValueError, match="plain scores"):
        ops.paged_flash_attention_prefill(q, *caches, a["cu"], None, 1.0, 16, prefix_lens=a["ctx"], **scales)
    with pytest.raises(ValueError, match="GPU tensors"):
        ops.paged_kv_read(*caches, 16, cu_seqlens=a["cu"], **scales)
    with pytest.raises(ValueError, match="block_size"):
        ops.paged_kv_read(*caches, 32, **scales)


def test_few_tokens_workspace():
    """At most 512 MiB, as the prefill's docstring says: one long sequence among many sizes all slots."""
    from myvllm_amd.full_attention import _few_workspace

    size = lambda *s: _lib.workspace_size("paged_attention_decode_workspace_size", *s)  # noqa: E731
    for N, rows, D, splits in ((1024, 64 * 16, 64, 2), (4096, 8 * 16, 256, 2)):
        assert size(N, rows, D, splits) > 2**27
        assert _few_workspace(N, rows, D, splits, "meta") is None
    for N in range(950, 1000):
        n, ws = size(N, 1024, 64, 2), _few_workspace(N, 1024, 64, 2, "meta")
        assert (ws is None) == (n > 2**27) and (ws is None or ws.numel() == n)
    assert size(950, 1024, 64, 2) <= 2**27 < size(999, 1024, 64, 2)


@pytest.mark.parametrize("T", [1, 2, 5])
@pytest.mark.parametrize("axes", [1, 3])
def test_positions_of_any_stride(T, axes):
    """Positions kept token by token, (T, axes) turned over, and every other one of a longer list: copied, one token
    as several."""
    from myvllm_amd.full_attention import _axes

    cos = Z(48, 32)
    wide = torch.arange(8 * 4 * axes, dtype=I32).view(8, 4 * axes)
    for p in (wide[:T, :axes].t(), wide[:T, ::4].t(), wide.t()[::4, :2 * T:2]) + ((wide[:T, 0],) if axes == 1 else ()):
        rows = p if p.dim() == 2 else p[None]
        got, of = _axes(p, (32,) if axes == 1 else (12, 10, 10), cos)
        assert torch.equal(got, rows) and got.stride(1) == 1 and sum(of) == 32
