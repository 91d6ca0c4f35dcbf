"""GPU: the append into caches held in 4 bits and with positions of several axes,
and the read, against the float64 oracle.

Codes and scale bytes have to be equal: keys are rotated in fp64 (products of a
16-bit and an fp32 number are exact there, and one fused step and one rounding of
the sum give the same), rounded to the 16-bit type through fp32 on both sides, and
the rest is comparisons.  Rotated q, and keys in 16-bit caches, as in the tests of the
plain append: two products and a sum in fp32 (below 4 x 2^-24 (|a| + |b|)), one
rounding, eps / 2 (fp16's subnormals: 2^-25)."""
import pytest
import torch

import myvllm_amd as ops
from oracle.fp4 import append_ref, cache_values, pack_ref, unpack_ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def rope(rows, rot, base=10000.0):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return a.cos().float(), a.sin().float()


def make(new, prefix, Hq=4, Hkv=2, D=128, page=16, dtype=BF, index=torch.int32, seed=0, spare=3, cols=0, bits=4):
    g = torch.Generator().manual_seed(seed)
    ctx = [n + p for n, p in zip(new, prefix)]
    pages = [-(-c // page) for c in ctx]
    blocks = sum(pages) + spare
    perm = torch.randperm(blocks, generator=g)
    tab = torch.full((len(new), max(pages + [1, cols])), -1, dtype=index)
    at = 0
    for n, p in enumerate(pages):
        tab[n, :p] = perm[at:at + p].to(index)
        at += p
    T = sum(new)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    cu = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=index)
    c = dict(q=r(T, Hq, D), k=r(T, Hkv, D), v=r(T, Hkv, D), tab=tab, ctx=torch.tensor(ctx, dtype=index), cu=cu)
    byte = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)  # noqa: E731
    if bits == 4:
        c.update(kc=byte(blocks, page, Hkv, D // 2), vc=byte(blocks, page, Hkv, D // 2),
                 ks=byte(blocks, Hkv, D // 32, page), vs=byte(blocks, Hkv, D // 32, page))
    else:
        c.update(kc=r(blocks, page, Hkv, D), vc=r(blocks, page, Hkv, D))
    return c


def close(got, ref, big):
    eps = torch.finfo(got.dtype).eps / 2
    bound = eps * (1 + 2**-10) * ref.abs() + 2**-22 * 2 * big + (2**-25 if got.dtype == HF else 0)
    err = (got.double().cpu() - ref).abs()
    assert got.shape == ref.shape and (err <= bound).all(), f"{int((err > bound).sum())} off, max {err.max():.3e}"


def append(d, page, use_cu=True, with_q=True, out=None, **kw):
    scales = dict(k_scales=d["ks"], v_scales=d["vs"]) if "ks" in d else {}
    return ops.paged_kv_append(d["q"] if with_q else None, d["k"], d["v"], d["kc"], d["vc"], d["tab"], d["ctx"], page,
                               cu_seqlens=d["cu"] if use_cu else None, out=out, **scales, **kw)


def check(c, dev, use_cu=True, with_q=True, cos=None, sin=None, interleaved=False, positions=None, sections=None,
          dealt=False, put=None, out=None):
    d = {n: (put or (lambda n, t: t.to(dev)))(n, t) for n, t in c.items()}
    page = c["kc"].shape[1]
    gpu = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = append(d, page, use_cu, with_q, out(d) if out else None, cos=gpu(cos), sin=gpu(sin), interleaved=interleaved,
                 positions=gpu(positions), sections=sections, sections_interleaved=dealt)
    torch.cuda.synchronize()
    rq, rk, rv, places = append_ref(c["q"] if with_q else None, c["k"], c["v"], c["tab"], c["ctx"],
                                    c["cu"] if use_cu else None, page, c["kc"].shape[0], cos, sin, interleaved,
                                    positions, sections, dealt)
    dt = c["k"].dtype
    t, b, s = ([p[i] for p in places] for i in range(3))
    big = float(max(x.float().nan_to_num(0, 0, 0).abs().max() if x.numel() else 0 for x in (c["q"], c["k"])))
    want = {n: c[n].clone() for n in ("kc", "vc", "ks", "vs") if n in c}
    for x, rows in (("k", rk), ("v", rv.double())):
        if "ks" in c:
            codes, scales = pack_ref(rows.float().to(dt))
            want[x + "c"][b, s] = codes[t]
            want[x + "s"][b, :, :, s] = scales[t]
            assert torch.equal(d[x + "c"].cpu(), want[x + "c"]), f"{x} codes"
            assert torch.equal(d[x + "s"].cpu(), want[x + "s"]), f"{x} scales"
        else:
            mine = d[x + "c"].cpu()
            close(mine[b, s], rows[t], big)
            mine[b, s] = c[x + "c"][b, s]
            assert torch.equal(mine, c[x + "c"]), "rows that nobody wrote"
    if with_q:
        close(got, rq, big)
        rot = 0 if cos is None else 2 * cos.shape[1]
        assert torch.equal(got.cpu()[..., rot:].double(), rq[..., rot:])
    else:
        assert got is None
    return d, got


CASES = [
    ([1], [0], 16, 2, 256, 16, 64, False, BF, torch.int32),
    ([1, 31, 0, 17], [0, 300, 5, 16], 16, 2, 256, 16, 256, False, BF, torch.int32),
    ([33, 64], [100, 0], 16, 4, 128, 32, 128, True, HF, torch.int64),
    ([5, 0, 0, 90], [11, 0, 3, 1], 4, 4, 64, 48, 16, False, HF, torch.int32),
    ([20, 3], [1000, 2], 6, 2, 64, 16, 48, True, BF, torch.int64),
    ([65], [1], 5, 1, 128, 16, 112, False, BF, torch.int32),
    ([40], [70], 1, 1, 256, 16, 0, False, HF, torch.int32),
    ([9, 9], [7, 8], 70, 10, 256, 64, 32, False, BF, torch.int32),
    ([13, 50], [3, 0], 3, 3, 64, 16, 64, False, BF, torch.int32),
    ([21], [6], 8, 2, 128, 16, 80, False, HF, torch.int64),
]


def split_sections(half, axes):
    cuts = [half // 4, half // 3, half // 6][: axes - 1]
    return [half - sum(cuts)] + cuts


@pytest.mark.parametrize("new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index", CASES)
def test_fp4_append(dev, new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index):
    print(f"fp4 append new={new} prefix={prefix} {Hq}/{Hkv}x{D} page={page} rot={rot} {inter} {dtype}", flush=True)
    c = make(new, prefix, Hq, Hkv, D, page, dtype, index, seed=sum(new))
    cos, sin = rope(max(c["ctx"]) + 1, rot) if rot else (None, None)
    check(c, dev, cos=cos, sin=sin, interleaved=inter)
    check(c, dev, cos=cos, sin=sin, interleaved=inter, with_q=False)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index", [c for c in CASES if c[6]][:6])
def test_axes(dev, bits, axes, new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index):
    print(f"axes {axes} bits {bits} new={new} {Hq}/{Hkv}x{D} rot={rot} {inter} {dtype}", flush=True)
    c = make(new, prefix, Hq, Hkv, D, page, dtype, index, seed=axes, bits=bits)
    cos, sin = rope(500, rot)  # (the tables do not have to reach the cache's positions)
    pos = torch.randint(0, 500, (axes, sum(new)), generator=torch.Generator().manual_seed(rot), dtype=index)
    sections = split_sections(rot // 2, axes)
    for dealt in (False, True):
        check(c, dev, cos=cos, sin=sin, interleaved=inter, positions=pos, sections=sections, dealt=dealt)
    if axes == 1:
        check(c, dev, cos=cos, sin=sin, interleaved=inter, positions=pos[0])


def test_axes_uneven_sections(dev):
    """An empty section, one of everything, and positions of a strided and of another integer type."""
    c = make([30, 7], [0, 90], bits=16)
    cos, sin = rope(64, 128)
    g = torch.Generator().manual_seed(3)
    wide = torch.randint(0, 64, (37, 3), generator=g)
    for sections, dealt in (([0, 64, 0], True), ([0, 64, 0], False), ([1, 0, 63], True), ([61, 2, 1], False)):
        check(c, dev, cos=cos, sin=sin, positions=wide.t().contiguous(), sections=sections, dealt=dealt)
    check(c, dev, cos=cos, sin=sin, positions=wide.t(), sections=[20, 22, 22])  # (copied: its tokens lie apart)
    deep = torch.zeros(5, 37, dtype=torch.int32)
    deep[::2] = wide.t().int()
    check(c, dev, cos=cos, sin=sin, positions=deep[::2], sections=[20, 22, 22])


def test_axes_agree_with_the_plain_append(dev):
    """All axes at the cache's position: the plain rotation (either may fuse another one
    of the two products into the sum, so each is held to the oracle by check())."""
    c = make([12, 1, 60], [0, 33, 7], bits=16)
    cos, sin = rope(80, 64)
    a, qa = check(c, dev, cos=cos, sin=sin)
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip([12, 1, 60], c["ctx"].tolist())])
    b, qb = check(c, dev, cos=cos, sin=sin, positions=pos.expand(3, -1).contiguous(), sections=[11, 11, 10], dealt=True)
    assert torch.equal(a["vc"], b["vc"])
    big = float(c["q"].float().abs().max())
    assert ((qa.double() - qb.double()).abs() <= 2 * (2**-8 * qa.double().abs() + 2**-21 * big)).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_tokens_without_a_place(dev, bits):
    """Positions past the rotation on one axis, past the table, below 0, foreign blocks, rows outside the offsets."""
    c = make([10, 20, 6], [0, 40, 0], bits=bits)
    c["ctx"] = torch.tensor([7, 200, 6], dtype=torch.int32)  # three below 0; all past the table
    c["tab"][2, 0] = 10**6
    cos, sin = rope(32, 64)
    pos = torch.randint(0, 32, (3, 36), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    pos[1, 5], pos[2, 6], pos[0, 34] = 32, -1, 2**31 - 1
    check(c, dev, cos=cos, sin=sin, positions=pos, sections=[10, 11, 11])
    c["cu"] = torch.tensor([2, 10, 10, 30], dtype=torch.int32)
    check(c, dev, cos=cos, sin=sin, positions=pos, sections=[10, 11, 11])
    check(c, dev)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_every_kind_of_number(dev, dtype):
    """Blocks of zeros, of the type's limits, next to the codes' borders, with infinities and NaN."""
    g = torch.Generator().manual_seed(5)
    rows = []
    grid = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7], dtype=torch.float64)
    info = torch.finfo(dtype)
    for e in (-133, -126, -30, -24, -15, -14, -13, -12, -3, 0, 5, 12, 13, 14, 125, 126):
        x = grid[torch.randint(0, 16, (256,), generator=g)] * (1 - 2 * torch.randint(0, 2, (256,), generator=g))
        rows.append((x * 2.0**e).clamp(info.min, info.max).to(dtype))
        near = torch.nextafter(rows[-1].float(), torch.randn(256, generator=g)).to(dtype)
        rows.append((near.double() * (1 + info.eps * torch.randint(-1, 2, (256,), generator=g))).clamp(info.min, info.max).to(dtype))
    for bad in (float("inf"), -float("inf"), float("nan")):
        x = torch.randn(256, generator=g).to(dtype)
        x[[3, 100, 255]] = bad
        rows.append(x)
    rows += [torch.zeros(256, dtype=dtype), torch.full((256,), info.max, dtype=dtype),
             torch.full((256,), info.smallest_normal / 2, dtype=dtype)]
    T = len(rows)
    c = make([T], [0], Hq=2, Hkv=1, D=256, dtype=dtype)
    c["v"] = torch.stack(rows)[:, None]
    c["k"] = c["v"].clone()
    d, _ = check(c, dev)
    k, v = ops.paged_kv_read(d["kc"], d["vc"], d["tab"], d["ctx"], 16, cu_seqlens=d["cu"], dtype=dtype,
                             k_scales=d["ks"], v_scales=d["vs"])
    ref = unpack_ref(*pack_ref(c["v"]))
    for x in (k, v):
        assert torch.equal(x.cpu().double().nan_to_num(-1), ref.nan_to_num(-1))
    assert ref.abs().nan_to_num(0).max() <= info.max


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_keys_are_rounded_through_fp32(dev, dtype, inter):
    """A sum 2^-30 below the middle of two 16-bit numbers is that middle in fp32, so the even one of
    them: 1.75, the border between 1.5 and 2, which becomes 2.  Rounded once it would be the lower
    one, and 1.5.  (Magnitudes up to 4 give the scale 1.)"""
    D, rot = 64, 64
    c = make([40], [0], Hq=1, Hkv=1, D=D, dtype=dtype)
    middle = 1.75 - torch.finfo(dtype).eps / 2
    cos, sin = torch.full((40, rot // 2), middle), torch.full((40, rot // 2), 2.0**-30)
    a, b = (slice(0, D, 2), slice(1, D, 2)) if inter else (slice(0, D // 2), slice(D // 2, D))
    c["k"][:, :, a], c["k"][:, :, b] = 1.0, 1.0
    c["k"][::2, 0, 6] = 2.0
    c["k"][::2, 0, 7 + (25 if not inter else 0)] = 2.0
    c["k"][1::2] *= -1
    check(c, dev, cos=cos, sin=sin, interleaved=inter)


def test_strides_streams_and_in_place(dev):
    """Caches as slices of a cache of layers with wider rows; q turned where it lies; another stream."""
    c = make([40, 3], [5, 70], D=256, Hq=8, Hkv=2)
    cos, sin = rope(200, 96)

    def put(n, t):
        if n in ("kc", "vc"):
            w = torch.full((3, *t.shape[:2], t.shape[2] + 1, t.shape[3] + 16), 7, dtype=t.dtype, device=dev)
            w[1, :, :, :t.shape[2], :t.shape[3]] = t.to(dev)
            return w[1, :, :, :t.shape[2], :t.shape[3]]
        if n in ("ks", "vs"):
            w = torch.full((3, *t.shape[:2], t.shape[2] + 2, t.shape[3] + 4), 7, dtype=t.dtype, device=dev)
            w[1, :, :, :t.shape[2], :t.shape[3]] = t.to(dev)
            return w[1, :, :, :t.shape[2], :t.shape[3]]
        if n == "q":
            w = torch.zeros(t.shape[0], 12, 256, dtype=t.dtype, device=dev)
            w[:, 2:10] = t.to(dev)
            return w[:, 2:10]
        return t.to(dev)

    d, got = check(c, dev, cos=cos, sin=sin, put=put, out=lambda d: d["q"])
    assert got is d["q"]
    for n in ("kc", "vc", "ks", "vs"):
        w = d[n]._base
        inner = w[1, :, :, :c[n].shape[2], :c[n].shape[3]]
        assert (w == 7).sum() >= w.numel() - inner.numel() and (w[0] == 7).all() and (w[2] == 7).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(c, dev, cos=cos, sin=sin)
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index", CASES[:8])
def test_read(dev, bits, new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index):
    c = make(new, prefix, Hq, Hkv, D, page, dtype, index, seed=D, bits=bits)
    if bits == 4:  # finite values of the type
        top = 125 if dtype == BF else 13
        for n in ("ks", "vs"):
            c[n] = (c[n].int() % (2 * top + 1) + 127 - top).to(torch.uint8)
    d = {n: t.to(dev) for n, t in c.items()}
    scales = dict(k_scales=d["ks"], v_scales=d["vs"]) if bits == 4 else {}
    whole = {x: (cache_values(c[x + "c"], c[x + "s"]) if bits == 4 else c[x + "c"].double()) for x in "kv"}
    full = torch.tensor([0] + c["ctx"].cumsum(0).tolist(), dtype=index)
    for cu, lens in ((c["cu"], new), (full, c["ctx"].tolist())):
        got = ops.paged_kv_read(d["kc"], d["vc"], d["tab"], d["ctx"], page, cu_seqlens=cu.to(dev),
                                dtype=dtype if bits == 4 else None, **scales)
        for x, y in zip("kv", got):
            rows = [whole[x][int(c["tab"][n, p // page]), p % page]
                    for n, m in enumerate(lens) for p in range(int(c["ctx"][n]) - m, int(c["ctx"][n]))]
            assert y.dtype == dtype and torch.equal(y.cpu().double(), torch.stack(rows))
    some = c["ctx"] > 0
    last = ops.paged_kv_read(d["kc"], d["vc"], d["tab"], d["ctx"], page, dtype=dtype if bits == 4 else None, **scales)
    for x, y in zip("kv", last):
        for n in range(len(new)):
            m = int(c["ctx"][n])
            ref = whole[x][int(c["tab"][n, (m - 1) // page]), (m - 1) % page] if some[n] else torch.zeros(Hkv, D)
            assert torch.equal(y[n].cpu().double(), ref.double())


def test_read_edges(dev):
    """Rows without a place and of foreign blocks are zero; many empty sequences; no tokens."""
    c = make([10, 20], [0, 0], bits=16)
    c["ctx"] = torch.tensor([7, 200], dtype=torch.int32)
    c["tab"][0, 0] = -5
    d = {n: t.to(dev) for n, t in c.items()}
    for x in ops.paged_kv_read(d["kc"], d["vc"], d["tab"], d["ctx"], 16, cu_seqlens=d["cu"]):
        assert x.shape == (30, 2, 128) and not x.any()
    cu = torch.tensor([3, 3, 4], dtype=torch.int32, device=dev)  # rows before, after and of one token
    d["ctx"] = torch.tensor([9, 2], dtype=torch.int32, device=dev)
    k, _ = ops.paged_kv_read(d["kc"], d["vc"], d["tab"], d["ctx"], 16, num_tokens=6, cu_seqlens=cu)
    assert torch.equal(k[3].cpu(), c["kc"][int(c["tab"][1, 0]), 1]) and not k[[0, 1, 2, 4, 5]].any()
    for N in (64, 100, 4097):
        new = [0] * N
        for i in (0, 1, N // 2, N - 2, N - 1):
            new[i] = 2 + i % 3
        c = make(new, [0] * N, bits=16)
        d = {n: t.to(dev) for n, t in c.items()}
        append(d, 16)
        k, v = ops.paged_kv_read(d["kc"], d["vc"], d["tab"], d["ctx"], 16, cu_seqlens=d["cu"])
        assert torch.equal(k, d["k"]) and torch.equal(v, d["v"])
    k, v = ops.paged_kv_read(d["kc"], d["vc"], d["tab"][:0], d["ctx"][:0], 16)
    assert k.shape == (0, 2, 128)


def test_read_of_no_sequences(dev):
    """Offsets of an empty batch: every row is one that nobody wrote."""
    c = {n: t.to(dev) for n, t in make([3], [20]).items()}
    k, v = ops.paged_kv_read(c["kc"], c["vc"], c["tab"][:0], c["ctx"][:0], 16, num_tokens=5, cu_seqlens=c["cu"][:1],
                             k_scales=c["ks"], v_scales=c["vs"])
    assert k.shape == (5, 2, 128) and not k.any() and not v.any()


def test_append_and_read_in_a_graph(dev):
    c = make([1] * 20, list(range(20)), seed=9)
    cos, sin = (t.to(dev) for t in rope(64, 64))
    pos = torch.randint(0, 64, (3, 20), dtype=torch.int32, device=dev)
    d = {n: t.to(dev) for n, t in c.items()}

    def step():
        q = append(d, 16, use_cu=False, cos=cos, sin=sin, positions=pos, sections=[12, 10, 10])
        return [q, *ops.paged_kv_read(d["kc"], d["vc"], d["tab"], d["ctx"], 16, k_scales=d["ks"], v_scales=d["vs"])]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        for n in ("q", "k", "v"):
            d[n].copy_(torch.randn(d[n].shape, generator=torch.Generator().manual_seed(i)).to(BF))
        pos.copy_(torch.randint(0, 64, (3, 20), generator=torch.Generator().manual_seed(i), dtype=torch.int32))
        d["kc"].zero_()
        d["ks"].zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, cache = [t.clone() for t in held], (d["kc"].clone(), d["ks"].clone())
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(cache[0], d["kc"]) and torch.equal(cache[1], d["ks"])


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rot, inter", [(0, False), (16, False), (48, True), (64, False)])
def test_block_maxima(dev, D, rot, inter):
    """A block's scale is its own largest magnitude's, whichever lane has it and whatever the
    wave's other rows and earlier steps left: each of the block's places in turn, blocks
    2^20 apart next to each other and after each other.  (A block of 16 of turned and 16 of other numbers
    is shared by lanes of both halves.)"""
    T, Hkv = 96, 8
    c = make([T], [0], Hq=1, Hkv=Hkv, D=D, seed=rot)
    t, h, b = torch.meshgrid(torch.arange(T), torch.arange(Hkv), torch.arange(D // 32), indexing="ij")
    size = 2.0 ** (20.0 * ((t + h + b) % 2) - 10.0 * (h % 3))
    for x, shift in (("k", 0), ("v", 7)):
        rows = c[x].float().clamp(-0.4, 0.4).unflatten(-1, (-1, 32))
        at = ((t + 5 * h + 11 * b + shift) % 32)[..., None]
        rows = rows.scatter(-1, at, (1.0 + t / 128)[..., None].float() * (1 - 2 * (t % 2))[..., None])
        c[x] = (rows * size[..., None]).flatten(-2).to(BF)
    cos, sin = rope(T, rot) if rot else (None, None)
    check(c, dev, cos=cos, sin=sin, interleaved=inter)


@pytest.mark.parametrize("bits", [16, 4])
def test_one_token_with_positions_kept_token_by_token(dev, bits):
    """One token's positions as a column of (T, axes), whose tokens lie `axes` apart, as of several tokens."""
    cos, sin = rope(64, 128)
    wide = torch.randint(0, 64, (6, 3), generator=torch.Generator().manual_seed(1)).int().to(dev)
    for n in (1, 2, 6):
        c = make([n], [40], bits=bits, seed=n)
        d = {x: t.to(dev) for x, t in c.items()}
        q = append(d, 16, cos=cos.to(dev), sin=sin.to(dev), positions=wide[:n].t(), sections=(22, 21, 21))
        e = {x: t.to(dev) for x, t in c.items()}
        want, _ = check(c, dev, cos=cos, sin=sin, positions=wide[:n].t().cpu().contiguous(), sections=(22, 21, 21))
        turned = append(e, 16, cos=cos.to(dev), sin=sin.to(dev), positions=wide[:n].cpu().t().contiguous().to(dev),
                        sections=(22, 21, 21))
        torch.cuda.synchronize()
        assert torch.equal(q, turned) and all(torch.equal(d[x], want[x]) for x in ("kc", "vc"))


def test_append_past_4_gib(dev):
    """Rows other than those that are there, into blocks whose bytes lie past 2^32 of the cache's start; the blocks at
    those addresses less 2^32 stay as they were."""
    page, Hkv, D = 16, 2, 256
    per = page * Hkv * D // 2
    blocks = (2**32 + 2**28) // per
    low = 2**32 // per
    g = torch.Generator().manual_seed(9)
    kc, vc = (torch.zeros(blocks, page, Hkv, D // 2, dtype=torch.uint8, device=dev) for _ in range(2))
    ks, vs = (torch.full((blocks, Hkv, D // 32, page), 127, dtype=torch.uint8, device=dev) for _ in range(2))
    at = [blocks - 1, low, low + 77]
    tab, ctx = torch.tensor([at], dtype=torch.int32, device=dev), torch.tensor([41], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, 41], dtype=torch.int32, device=dev)
    for turn in range(2):
        k, v = (torch.randn(41, Hkv, D, generator=g).to(BF) for _ in range(2))
        ops.paged_kv_append(None, k.to(dev), v.to(dev), kc, vc, tab, ctx, page, cu_seqlens=cu, k_scales=ks, v_scales=vs)
        got = ops.paged_kv_read(kc, vc, tab, ctx, page, 41, cu, k_scales=ks, v_scales=vs)
        torch.cuda.synchronize()
        for mine, rows, codes, scales in ((got[0], k, kc, ks), (got[1], v, vc, vs)):
            c, s = pack_ref(rows)
            assert torch.equal(mine.cpu().double(), unpack_ref(c, s))
            for i, b in enumerate(at):
                m = min(41 - 16 * i, 16)
                assert torch.equal(codes[b, :m].cpu(), c[16 * i:16 * i + m])
                assert torch.equal(scales[b, :, :, :m].cpu(), s[16 * i:16 * i + m].permute(1, 2, 0))
                assert not codes[b - low].any() and (scales[b - low] == 127).all()
