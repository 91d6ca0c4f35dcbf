"""GPU: decode and paged prefill over caches held in 4 bits, against the float64
attention over the values that the codes stand for, with the bound of the 16-bit
kernels (attention_bounds): the codes become 16-bit numbers exactly.  To it comes
what a weight below 2^-126, the smallest normal number of fp32 and bf16, loses where it
becomes 0: with the row's weights summing to at least 1 in the kernel's units (its
base is no higher than the largest score), 2^-126 |v| of each of m keys, and as much of
|o| by the sum: at most 2^-125 m max|v|."""
import pytest
import torch

import myvllm_amd as ops
from attention_bounds import assert_within, ref_and_bound
from myvllm_amd import _lib
from oracle.fp4 import cache_values, pack_ref

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(ctx, new, Hq=16, Hkv=2, D=256, page=16, dtype=BF, index=torch.int32, seed=0, cols=0, stale=True):
    """Random rows packed; what no sequence covers is full of NaN scales."""
    g = torch.Generator().manual_seed(seed)
    pages = [-(-c // page) for c in ctx]
    blocks = sum(pages) + 2
    perm = torch.randperm(blocks, generator=g)
    tab = torch.full((len(ctx), max(pages + [1, cols])), -1, dtype=index)
    at = 0
    used = torch.zeros(blocks, page, dtype=torch.bool)
    for n, p in enumerate(pages):
        tab[n, :p] = perm[at:at + p].to(index)
        at += p
        j = torch.arange(ctx[n])
        used[tab[n, j // page].long(), j % page] = True
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = dict(q=(2 * r(sum(new), Hq, D)).to(dtype), tab=tab, ctx=torch.tensor(ctx, dtype=index),
             cu=torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=index))
    for x in ("k", "v"):
        rows = (r(blocks, page, Hkv, D) * 2.0 ** torch.randint(-2, 3, (blocks, page, Hkv, 1), generator=g)).to(dtype)
        codes, scales = pack_ref(rows)
        if stale:
            codes[~used], scales[~used] = 255, 255
        c[x + "c"], c[x + "s"] = codes, scales.permute(0, 2, 3, 1).contiguous()
    return c


def rows_of(c, x, n, page, whole=None):
    m = int(c["ctx"][n])
    j = torch.arange(m)
    b = c["tab"][n, j // page].long()
    ok = (b >= 0) & (b < c["kc"].shape[0])
    whole = cache_values(c[x + "c"], c[x + "s"]) if whole is None else whole
    v = whole[b.clamp(0, c["kc"].shape[0] - 1), j % page]
    return torch.where(ok[:, None, None], v, 0.0)


def reference(c, new, scale):
    page = c["kc"].shape[1]
    refs, bounds, at = [], [], 0
    whole = {x: cache_values(c[x + "c"], c[x + "s"]) for x in "kv"}
    for n, m in enumerate(new):
        k, v = (rows_of(c, x, n, page, whole[x]) for x in "kv")
        L = k.shape[0]
        o, b = ref_and_bound(c["q"][at:at + m], k, v, torch.arange(L - m, L), scale, c["q"].dtype)
        refs.append(o)
        bounds.append(b + 2.0**-125 * L * (v.abs().nan_to_num(0).max() if L else 0))
        at += m
    return torch.cat(refs), torch.cat(bounds)


def decode(c, dev, scale, splits=None, out=None, put=None):
    d = {n: (put or (lambda n, t: t.to(dev)))(n, t) for n, t in c.items()}
    o = ops.paged_flash_attention_decode(d["q"], d["kc"], d["vc"], d["tab"], d["ctx"], scale, c["kc"].shape[1],
                                         num_splits=splits, out=out, k_scales=d["ks"], v_scales=d["vs"])
    torch.cuda.synchronize()
    return o


def prefill(c, dev, scale, put=None, out=None, **kw):
    d = {n: (put or (lambda n, t: t.to(dev)))(n, t) for n, t in c.items()}
    o = ops.paged_flash_attention_prefill(d["q"], d["kc"], d["vc"], d["tab"], d["ctx"], d["cu"], None, scale,
                                          c["kc"].shape[1], out=out, k_scales=d["ks"], v_scales=d["vs"], **kw)
    torch.cuda.synchronize()
    return o


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 700]
HEADS = [(16, 2, 256, BF), (16, 2, 256, HF), (16, 4, 128, HF), (16, 16, 64, BF), (6, 2, 64, HF), (5, 1, 128, BF),
         (3, 3, 64, BF), (6, 6, 64, BF), (40, 1, 256, BF), (34, 2, 128, BF), (21, 3, 256, HF), (8, 1, 64, HF)]


@pytest.mark.parametrize("Hq, Hkv, D, dtype", HEADS)
@pytest.mark.parametrize("page, index", [(16, torch.int32), (48, torch.int64)])
def test_decode_heads(dev, Hq, Hkv, D, dtype, page, index):
    print(f"fp4 decode {Hq}/{Hkv}x{D} {dtype} page={page}", flush=True)
    c = make(EDGES, [1] * len(EDGES), Hq, Hkv, D, page, dtype, index, seed=D + Hq)
    ref, bound = reference(c, [1] * len(EDGES), D**-0.5)
    for splits in (None, 1, 2, 9):
        assert_within(decode(c, dev, D**-0.5, splits), ref, bound, f"splits {splits}")


@pytest.mark.parametrize("splits", [1, 2, 3, 17, 64, 256])
def test_decode_splits(dev, splits):
    """Pieces that end inside tiles and pages, several sequences in a unit and units without work."""
    ctx = [1, 0, 2000, 16, 33, 700]
    for Hq, Hkv, D in ((16, 2, 256), (4, 4, 64), (8, 2, 128)):
        print(f"fp4 decode splits={splits} {Hq}/{Hkv}x{D}", flush=True)
        c = make(ctx, [1] * 6, Hq, Hkv, D, seed=splits, cols=150)
        ref, bound = reference(c, [1] * 6, 0.1)
        a = decode(c, dev, 0.1, splits)
        assert_within(a, ref, bound)
        assert torch.equal(a, decode(c, dev, 0.1, splits))


def test_decode_batches(dev):
    """One sequence to more than the waves price by themselves (1,024)."""
    for B in (1, 63, 65, 1025):
        g = torch.Generator().manual_seed(B)
        ctx = torch.randint(0, 70, (B,), generator=g).tolist()
        c = make(ctx, [1] * B, 4, 2, 128, seed=B)
        ref, bound = reference(c, [1] * B, 0.1)
        print(f"fp4 decode B={B}", flush=True)
        for splits in (None, 3):
            assert_within(decode(c, dev, 0.1, splits), ref, bound, f"B={B}")
    c = make([5], [1], 4, 2, 128)
    c = dict(c, q=c["q"][:0], tab=c["tab"][:0], ctx=c["ctx"][:0])
    assert decode(c, dev, 0.1, 1).shape == (0, 4, 128)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0, 1e-8])
def test_scales(dev, scale):
    c = make([40, 100], [1, 1], seed=1)
    ref, bound = reference(c, [1, 1], scale)
    for splits in (1, 4):
        assert_within(decode(c, dev, scale, splits), ref, bound)
    c = make([40, 100], [30, 40], seed=1)
    assert_within(prefill(c, dev, scale), *reference(c, [30, 40], scale))


def test_extreme_scales(dev):
    """Values near the ends of the type, and single NaN blocks, which reach their own head alone.

    bf16 up to the scale 2^110: a key's weight in the fp32 sums is up to 2^8, so they
    hold 90 keys of 6 * 2^e for 2^8 * 90 * 6 * 2^e < 2^128, e < 110.93 (at 2^125 the
    sums are infinite, as the 16-bit kernels' are over such values)."""
    for dtype, top in ((BF, 110), (HF, 13)):
        c = make([50, 90], [1, 1], 4, 2, 128, dtype=dtype, stale=False)
        c["vs"][:] = 127 + top
        c["vc"] &= 0x77
        o = decode(c, dev, 0.1)
        ref, bound = reference(c, [1, 1], 0.1)
        assert_within(o, ref, bound)
        c["vs"][:] = 127 - top
        if dtype == BF:  # (fp16's own steps are coarser than the sums there)
            assert_within(decode(c, dev, 0.1), *reference(c, [1, 1], 0.1))
    c = make([50, 90], [1, 1], 4, 2, 128)
    c["ks"][int(c["tab"][0, 2]), 1, 3, 4] = 255
    o = decode(c, dev, 0.1).cpu()
    assert o[0, 2:].isnan().all() and not o[0, :2].isnan().any() and not o[1].isnan().any()
    c["cu"] = torch.tensor([0, 1, 2], dtype=torch.int32)
    o = prefill(c, dev, 0.1).cpu()
    assert o[0, 2:].isnan().all() and not o[0, :2].isnan().any() and not o[1].isnan().any()


def test_foreign_blocks_and_long_lengths(dev):
    """Table entries outside the cache read as zero keys; lengths past the table end at it."""
    c = make([60, 100], [1, 1], cols=8)
    c["tab"][0, 1], c["tab"][1, 0], c["tab"][1, 5] = 10**6, -1, c["kc"].shape[0]
    ref, bound = reference(c, [1, 1], 0.1)
    for splits in (1, 3):
        assert_within(decode(c, dev, 0.1, splits), ref, bound)
    assert_within(prefill(c, dev, 0.1), ref, bound)
    c["tab"][1] = c["tab"][0].clone()
    far = dict(c, ctx=torch.tensor([60, 10**6], dtype=torch.int32))
    near = dict(c, ctx=torch.tensor([60, 128], dtype=torch.int32))
    far["ks"], far["vs"] = (t.clone().fill_(120) for t in (c["ks"], c["vs"]))
    near["ks"], near["vs"] = far["ks"], far["vs"]
    assert torch.equal(decode(far, dev, 0.1, 2), decode(near, dev, 0.1, 2))


@pytest.mark.parametrize("Hq, Hkv, D, dtype", HEADS)
@pytest.mark.parametrize("page, index", [(16, torch.int32), (32, torch.int64)])
def test_prefill_heads(dev, Hq, Hkv, D, dtype, page, index):
    print(f"fp4 prefill {Hq}/{Hkv}x{D} {dtype} page={page}", flush=True)
    new, prefix = [1, 3, 0, 40, 65, 130], [0, 100, 7, 33, 0, 16]
    c = make([n + p for n, p in zip(new, prefix)], new, Hq, Hkv, D, page, dtype, index, seed=Hq + D)
    assert_within(prefill(c, dev, D**-0.5), *reference(c, new, D**-0.5))


@pytest.mark.parametrize("Hq, Hkv, D, dtype", HEADS[:6])
def test_prefill_split(dev, Hq, Hkv, D, dtype):
    """Few rows over long contexts, split over the keys; the same within the bound as unsplit."""
    new, prefix = [2, 9, 70], [4000, 2001, 1500]
    c = make([n + p for n, p in zip(new, prefix)], new, Hq, Hkv, D, 16, dtype, seed=D, cols=1000)
    T, cap = sum(new), 16 * c["tab"].shape[1]
    assert _lib.workspace_size("paged_attention_prefill_workspace_size", T, 3, Hq, Hkv, D, cap) > 0
    print(f"fp4 split prefill {Hq}/{Hkv}x{D}", flush=True)
    ref, bound = reference(c, new, D**-0.5)
    a = prefill(c, dev, D**-0.5)
    assert_within(a, ref, bound)
    assert torch.equal(a, prefill(c, dev, D**-0.5))
    d = {n: t.to(dev) for n, t in c.items()}
    o = torch.empty_like(d["q"])
    _lib.call("paged_attention_prefill_fp4", d["q"], d["kc"], d["vc"], d["ks"], d["vs"], d["tab"], d["ctx"], d["cu"], o,
              None, max(new), D**-0.5)
    assert_within(o, ref, bound, "unsplit")


LAYOUTS = [(16, ""), (32, ""), (16, "vc"), (16, "ks"), (16, "vs"), (16, "kc")]


def laid_out(dev, apart):
    """Tensors on the GPU, the one called `apart` with larger strides than the others."""
    def put(n, t):
        if n != apart:
            return t.to(dev)
        w = torch.full((t.shape[0] + 1, t.shape[1] + 1, t.shape[2] + 1, t.shape[3] + 32), 255, dtype=t.dtype,
                       device=dev)
        w = w[1:, :t.shape[1], :t.shape[2], :t.shape[3]]
        w.copy_(t)
        return w

    return put


@pytest.mark.parametrize("Hq, Hkv, D, dtype", [(16, 2, 256, BF), (8, 4, 128, HF), (4, 4, 64, BF)])
@pytest.mark.parametrize("page, apart", LAYOUTS)
def test_layouts(dev, Hq, Hkv, D, dtype, page, apart):
    """Pages of 16 keys with k and v laid out alike, and every other layout: prefill whole and split,
    a few tokens, decode."""
    print(f"fp4 layouts {Hq}/{Hkv}x{D} {dtype} page={page} apart={apart}", flush=True)
    put = laid_out(dev, apart)
    for new, ctx in (([70, 0, 129, 1, 33, 64], [70, 40, 300, 1000, 800, 64]), ([1, 33], [3000, 2000])):
        c = make(ctx, new, Hq, Hkv, D, page, dtype, seed=D + page)
        ref, bound = reference(c, new, D**-0.5)
        assert_within(prefill(c, dev, D**-0.5, put=put), ref, bound)
        d = {n: put(n, t) for n, t in c.items()}
        o = torch.empty_like(d["q"])
        _lib.call("paged_attention_prefill_fp4", d["q"], d["kc"], d["vc"], d["ks"], d["vs"], d["tab"], d["ctx"],
                  d["cu"], o, None, max(new), D**-0.5)
        assert_within(o, ref, bound, "unsplit")
    for new, ctx in (([1, 3, 0, 4], [900, 70, 5, 4]), ([2] * 20, [50 + 7 * i for i in range(20)])):
        c = make(ctx, new, Hq, Hkv, D, page, dtype, seed=D + page)
        assert is_few(c, max(new))
        assert_within(prefill(c, dev, D**-0.5, put=put), *reference(c, new, D**-0.5))
    for ctx in ([900, 70, 0, 4], [50 + 7 * i for i in range(20)]):
        c = make(ctx, [1] * len(ctx), Hq, Hkv, D, page, dtype, seed=D + page)
        ref, bound = reference(c, [1] * len(ctx), D**-0.5)
        for splits in (None, 1, 4):
            assert_within(decode(c, dev, D**-0.5, splits, put=put), ref, bound)


def is_few(c, most):
    from myvllm_amd.full_attention import _few_tokens

    return _few_tokens(c["q"], c["kc"], c["tab"], most)


@pytest.mark.parametrize("Hq, Hkv, D, dtype", HEADS)
@pytest.mark.parametrize("page, index", [(16, torch.int32), (48, torch.int64)])
def test_few_tokens_heads(dev, Hq, Hkv, D, dtype, page, index):
    """A few tokens of each sequence, as the decode's columns: groups that end inside a
    token, empty sequences, tokens that see one key and whole contexts of new tokens."""
    print(f"fp4 few {Hq}/{Hkv}x{D} {dtype} page={page}", flush=True)
    most = 64 // (Hq // Hkv)
    new = [1, 0, most, min(3, most), min(2, most), most, 1, min(5, most)]
    ctx = [1, 20, most, 3 + 40, 33, most + 700, 300, 64 + 5]
    ctx = [max(c, n) for c, n in zip(ctx, new)]
    c = make(ctx, new, Hq, Hkv, D, page, dtype, index, seed=Hq + D, cols=60)
    assert is_few(c, most) and not is_few(c, most + 64)
    ref, bound = reference(c, new, D**-0.5)
    a = prefill(c, dev, D**-0.5)
    assert_within(a, ref, bound)
    assert torch.equal(a, prefill(c, dev, D**-0.5))
    d = {n: t.to(dev) for n, t in c.items()}
    for splits in (2, 3, 40, 256):
        ws = torch.full((_lib.workspace_size("paged_attention_decode_workspace_size", len(new), most * Hq, D, splits),),
                        float("nan"), device=dev)
        o = torch.full_like(d["q"], 7.0)
        _lib.call("paged_attention_few_fp4", d["q"], d["kc"], d["vc"], d["ks"], d["vs"], d["tab"], d["ctx"], d["cu"],
                  o, ws, splits, most, D**-0.5)
        assert_within(o, ref, bound, f"splits {splits}")


@pytest.mark.parametrize("Hq, Hkv, D", [(8, 2, 128), (16, 2, 256), (4, 4, 64)])
def test_few_tokens_edges(dev, Hq, Hkv, D):
    """Rows outside the offsets and before position 0 are zero; lengths past the table; foreign blocks; NaN."""
    c = make([30, 20], [8, 7], Hq, Hkv, D, cols=4)
    c["cu"] = torch.tensor([2, 5, 10], dtype=torch.int32)
    o = prefill(c, dev, 0.1)
    assert is_few(c, 5) and not o[:2].any() and not o[10:].any()
    assert_within(o[2:10], *reference(dict(c, q=c["q"][2:10]), [3, 5], 0.1))
    c = make([3, 0], [5, 4], Hq, Hkv, D)
    o = prefill(c, dev, 0.1)
    assert not o[:2].any() and not o[5:].any()
    assert_within(o[2:5], *reference(dict(c, q=c["q"][2:5], ctx=c["ctx"][:1]), [3], 0.1))
    c = make([60, 100], [3, 4], Hq, Hkv, D, cols=8)
    c["tab"][0, 1], c["tab"][1, 0], c["tab"][1, 5] = 10**6, -1, c["kc"].shape[0]
    assert_within(prefill(c, dev, 0.1), *reference(c, [3, 4], 0.1))
    c["ks"][int(c["tab"][0, 2]), 0, 0, 4] = 255  # key 36 of the first sequence, kv head 0
    o = prefill(c, dev, 0.1).cpu()
    R = Hq // Hkv
    assert o[:3, :R].isnan().all() and not o[:3, R:].isnan().any() and not o[3:].isnan().any()
    full = make([200, 30], [2, 3], Hq, Hkv, D)
    short = dict(full, tab=full["tab"][:, :2].contiguous())  # 32 keys of the 200: queries past them see them all
    k, v = (cache_values(full[x + "c"], full[x + "s"])[full["tab"][0, :2].long()].flatten(0, 1) for x in "kv")
    ref, bound = ref_and_bound(full["q"][:2], k, v, torch.tensor([198, 199]), 0.1, BF)
    assert_within(prefill(short, dev, 0.1)[:2], ref, bound)


def test_few_tokens_batches(dev):
    """More sequences than the waves price by themselves; scales of either sign and zero; one graph's replays."""
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 4, (1100,), generator=g).tolist()
    ctx = [n + int(x) for n, x in zip(new, torch.randint(0, 60, (1100,), generator=g))]
    c = make(ctx, new, 4, 2, 128)
    assert_within(prefill(c, dev, 0.1), *reference(c, new, 0.1))
    c = make([40, 100, 1000], [2, 3, 1], 4, 2, 128)
    for scale in (-0.1, 0.0, 2.0):
        assert_within(prefill(c, dev, scale), *reference(c, [2, 3, 1], scale))
    d = {n: t.to(dev) for n, t in c.items()}
    step = lambda: ops.paged_flash_attention_prefill(  # noqa: E731
        d["q"], d["kc"], d["vc"], d["tab"], d["ctx"], d["cu"], None, 0.1, 16, max_seqlen=3, k_scales=d["ks"], v_scales=d["vs"])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        d["q"].copy_(torch.randn(d["q"].shape, generator=torch.Generator().manual_seed(i)).to(BF))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        assert torch.equal(got, step())


def test_empty_cache(dev):
    """No blocks at all: every row is zero."""
    c = make([30, 20], [3, 1], 4, 2, 128)
    for n in ("kc", "vc", "ks", "vs"):
        c[n] = c[n][:0]
    assert not prefill(c, dev, 0.1).any()
    wide = make([300, 20], [290, 1], 4, 2, 128)
    assert not prefill(dict(wide, **{n: c[n] for n in ("kc", "vc", "ks", "vs")}), dev, 0.1).any()
    one = make([30, 20], [1, 1], 4, 2, 128)
    for splits in (1, 3):
        assert not decode(dict(one, **{n: c[n] for n in ("kc", "vc", "ks", "vs")}), dev, 0.1, splits).any()


def test_prefill_uncovered_rows(dev):
    """Rows outside the offsets, and queries before position 0, are zero."""
    c = make([30, 20], [10, 20])
    c["cu"] = torch.tensor([2, 10, 25], dtype=torch.int32)
    o = prefill(c, dev, 0.1).cpu()
    assert not o[:2].any() and not o[25:].any()
    sub = dict(c, q=c["q"][2:25])
    assert_within(o[2:25], *reference(sub, [8, 15], 0.1))
    c = make([3, 0], [10, 20])
    assert not is_few(c, 20)
    o = prefill(c, dev, 0.1).cpu()
    assert not o[:7].any() and not o[10:].any()
    sub = dict(c, q=c["q"][7:10], ctx=c["ctx"][:1])
    assert_within(o[7:10], *reference(sub, [3], 0.1))
    c = make([3, 0], [10, 20])
    c["cu"] = torch.zeros(1, dtype=torch.int32)
    c["tab"], c["ctx"] = c["tab"][:0], c["ctx"][:0]
    assert not prefill(c, dev, 0.1).any()


def test_strides(dev):
    """Slices of caches of layers with wider rows, strided q and out, misaligned tensors (copied)."""
    c = make([70, 33, 5], [1, 1, 1], 8, 2, 128)
    ref, bound = reference(c, [1] * 3, 0.1)

    def put(n, t):
        if n in ("kc", "vc", "ks", "vs"):
            pad = 16 if n in ("kc", "vc") else 4
            w = torch.full((3, *t.shape[:2], t.shape[2] + 1, t.shape[3] + pad), 255, dtype=t.dtype, device=dev)
            w[1, :, :, :t.shape[2], :t.shape[3]] = t.to(dev)
            return w[1, :, :, :t.shape[2], :t.shape[3]]
        if n == "q":
            w = torch.zeros(t.shape[0], 3 * t.shape[1], 128, dtype=t.dtype, device=dev)
            w[:, ::3] = t.to(dev)
            return w[:, ::3]
        return t.to(dev)

    def odd(n, t):
        w = torch.empty(t.numel() + 1, dtype=t.dtype, device=dev)
        return w[1:].view(t.shape).copy_(t) if n in ("kc", "vc", "ks", "vs", "q") else t.to(dev)

    for how in (put, odd):
        out = torch.full((3, 10, 128), 9.0, dtype=BF, device=dev)
        o = decode(c, dev, 0.1, 3, out=out[:, 1:9], put=how)
        assert_within(o, ref, bound)
        assert o.data_ptr() == out[:, 1:9].data_ptr() and (out[:, [0, 9]] == 9).all()
        out.fill_(9)
        assert_within(prefill(c, dev, 0.1, put=how, out=out[:, 1:9]), ref, bound)
        assert (out[:, [0, 9]] == 9).all()


def test_far_offsets(dev):
    """Blocks whose bytes lie past 2^32 of the cache's start."""
    page, Hkv, D = 16, 2, 256
    per = page * Hkv * D // 2
    blocks = (2**32 + 2**28) // per
    c = make([100], [1], 8, Hkv, D)
    big = {x: torch.zeros(blocks, page, Hkv, D // 2, dtype=torch.uint8, device=dev) for x in ("kc", "vc")}
    small = {x: torch.zeros(blocks, Hkv, D // 32, page, dtype=torch.uint8, device=dev) for x in ("ks", "vs")}
    at = [blocks - 1 - i * (blocks // 7) for i in range(7)]
    for i, b in enumerate(at):
        for x in big:
            big[x][b] = c[x][int(c["tab"][0, i])].to(dev)
        for x in small:
            small[x][b] = c[x][int(c["tab"][0, i])].to(dev)
    ref, bound = reference(c, [1], 0.1)
    tab = torch.tensor([at], dtype=torch.int32, device=dev)
    q, ctx, cu = c["q"].to(dev), c["ctx"].to(dev), c["cu"].to(dev)
    scales = dict(k_scales=small["ks"], v_scales=small["vs"])
    assert_within(ops.paged_flash_attention_decode(q, big["kc"], big["vc"], tab, ctx, 0.1, page, **scales), ref, bound)
    assert_within(ops.paged_flash_attention_prefill(q, big["kc"], big["vc"], tab, ctx, cu, None, 0.1, page, **scales), ref, bound)
    k, v = ops.paged_kv_read(big["kc"], big["vc"], tab, ctx, page, **scales)
    assert torch.equal(k[0].cpu().double(), rows_of(c, "k", 0, 16)[99])
    ops.paged_kv_append(None, k, v, big["kc"], big["vc"], tab, ctx, page, **scales)
    k2, v2 = ops.paged_kv_read(big["kc"], big["vc"], tab, ctx, page, **scales)
    assert torch.equal(k2, k) and torch.equal(v2, v)


def test_serving_run(dev):
    """Prompts appended and attended to, a fork, decode steps of all, a compaction: the
    4-bit run against the 16-bit kernels over the values that it holds."""
    Hq, Hkv, D, page, L = 8, 2, 128, 16, 2
    cache = ops.PagedKVCache(L, 64, page, Hkv, D, BF, dev, bits=4)
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(BF).to(dev)  # noqa: E731
    a = torch.arange(512, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    cos, sin = a.cos().float().to(dev), a.sin().float().to(dev)

    def step(ids, new):
        cache.extend(ids, new)
        tab, ctx = cache.tables(ids)
        one = all(n == 1 for n in new)
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=dev)
        T = sum(new)
        pos = torch.randint(0, 512, (3, T), generator=g, dtype=torch.int32).to(dev)
        for layer in range(L):
            kc, vc, ks, vs = cache.layer(layer)
            scales = dict(k_scales=ks, v_scales=vs)
            q = ops.paged_kv_append(r(T, Hq, D), r(T, Hkv, D), r(T, Hkv, D), kc, vc, tab, ctx, page, cos=cos, sin=sin,
                                    cu_seqlens=cu, positions=pos, sections=(11, 11, 10), sections_interleaved=True, **scales)
            if one:
                o = ops.paged_flash_attention_decode(q, kc, vc, tab, ctx, D**-0.5, page, **scales)
            else:
                o = ops.paged_flash_attention_prefill(q, kc, vc, tab, ctx, cu, None, D**-0.5, page, **scales)
            # whole sequences read back, attended to by the 16-bit kernels
            lens = ctx.tolist()
            k, v = ops.paged_kv_read(kc, vc, tab, ctx, page, sum(lens), dtype=BF, **scales,
                                     cu_seqlens=torch.tensor([0] + ctx.cumsum(0).tolist(), dtype=torch.int32, device=dev))
            at, q0 = 0, 0
            for n, m in enumerate(lens):
                ks_, vs_ = k[at:at + m].cpu().double(), v[at:at + m].cpu().double()
                o_ref, bound = ref_and_bound(q[q0:q0 + new[n]].cpu(), ks_, vs_, torch.arange(m - new[n], m), D**-0.5, BF)
                assert_within(o[q0:q0 + new[n]], o_ref, bound, f"layer {layer} of {ids}")
                at, q0 = at + m, q0 + new[n]

    x, y = cache.allocate(), cache.allocate()
    step([x, y], [37, 100])
    z = cache.fork(x)
    before = ops.paged_kv_read(*cache.layer(1)[:2], *cache.tables([z]), page, k_scales=cache.layer(1)[2],
                               v_scales=cache.layer(1)[3])[0]
    step([x, y, z], [1, 1, 1])
    w = cache.fork(y)
    step([z, w, x], [1, 1, 1])
    cache.free([y])
    assert cache.compact() > 0
    step([x, w, z], [1, 1, 1])
    step([w, z], [20, 3])
    # the fork's first tokens are still its sequence's
    tab, ctx = cache.tables([z])
    old = torch.tensor([37], dtype=torch.int32, device=dev)
    kc, vc, ks, vs = cache.layer(1)
    assert torch.equal(ops.paged_kv_read(kc, vc, tab, old, page, k_scales=ks, v_scales=vs)[0], before)


def test_graphs_share_no_workspace(dev):
    """Two captured decodes of one shape, replayed in turn with eager work between."""
    cs = [make([900, 1200, 40], [1] * 3, seed=s) for s in (1, 2)]
    ds = [{n: t.to(dev) for n, t in c.items()} for c in cs]

    def step(d):
        return ops.paged_flash_attention_decode(d["q"], d["kc"], d["vc"], d["tab"], d["ctx"], 0.1, 16,
                                                k_scales=d["ks"], v_scales=d["vs"])

    want = [step(d).clone() for d in ds]
    torch.cuda.synchronize()
    graphs, held = [], []
    for d in ds:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(step(d))
        graphs.append(g)
    for _ in range(3):
        for h in held:
            h.zero_()
        for g in graphs:
            g.replay()
        eager = step(ds[0])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(h, w) for h, w in zip(held, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step(ds[1])
    b = step(ds[0])
    torch.cuda.synchronize()
    assert torch.equal(a, want[1]) and torch.equal(b, want[0])


@pytest.mark.parametrize("Hq, Hkv, D, dtype", HEADS)
@pytest.mark.parametrize("most", [1, 2, 3])
def test_more_tokens_than_said(dev, Hq, Hkv, D, dtype, most):
    """Sequences of more tokens than max_seqlen: every row is written, and right (as over 16-bit caches)."""
    print(f"fp4 few, more than {most}, {Hq}/{Hkv}x{D} {dtype}", flush=True)
    new = [most, 0, most + 1, 40, 1, most + 16]
    ctx = [300, 20, 70, 40, 9, 900]
    c = make(ctx, new, Hq, Hkv, D, dtype=dtype, seed=D + Hq)
    ref, bound = reference(c, new, D**-0.5)
    d = {n: t.to(dev) for n, t in c.items()}
    for splits in (2, 3, 40):
        ws = torch.full((_lib.workspace_size("paged_attention_decode_workspace_size", 6, most * Hq, D, splits),),
                        float("nan"), device=dev)
        o = torch.full_like(d["q"], float("nan"))
        _lib.call("paged_attention_few_fp4", d["q"], d["kc"], d["vc"], d["ks"], d["vs"], d["tab"], d["ctx"], d["cu"],
                  o, ws, splits, most, D**-0.5)
        assert_within(o, ref, bound, f"splits {splits}")
    if is_few(c, most):
        out = torch.full_like(d["q"], float("nan"))
        assert_within(prefill(c, dev, D**-0.5, max_seqlen=most, out=out), ref, bound)


def test_more_tokens_in_a_later_replay(dev):
    """A captured graph whose offsets, lengths and table then hold other batches: longer sequences, empty ones, a
    lone one, rows of no sequence."""
    Hq, Hkv, D = 8, 2, 128
    c = make([300, 200, 90, 500], [6] * 4, Hq, Hkv, D, cols=40)
    d = {n: t.to(dev) for n, t in c.items()}
    out = torch.empty_like(d["q"])
    step = lambda: ops.paged_flash_attention_prefill(  # noqa: E731
        d["q"], d["kc"], d["vc"], d["tab"], d["ctx"], d["cu"], None, 0.1, 16, max_seqlen=6, out=out, k_scales=d["ks"],
        v_scales=d["vs"])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for ctx, new in (([300, 200, 90, 500], [6] * 4), ([24, 7, 60, 600], [20, 0, 1, 3]), ([0, 0, 640, 0], [0, 0, 24, 0]),
                     ([5, 31, 16, 2], [5, 7, 8, 2])):
        x = make(ctx, new, Hq, Hkv, D, seed=sum(ctx))
        rows = sum(new)
        d["q"][:rows] = x["q"].to(dev)
        d["cu"].copy_(x["cu"])
        d["ctx"].copy_(x["ctx"])
        d["tab"].fill_(-1)
        d["tab"][:, :x["tab"].shape[1]] = x["tab"].to(dev)
        for n in ("kc", "vc", "ks", "vs"):
            m = min(x[n].shape[0], c[n].shape[0])
            d[n][:m] = x[n][:m].to(dev)
            x[n] = d[n].cpu()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert_within(out[:rows], *reference(x, new, 0.1))
        assert not out[rows:].any()


def test_few_tokens_of_many(dev):
    """One sequence of 64 tokens among 1,023 of one: the few-tokens form's slots would take 544 MiB, so it goes in
    tiles, within the 512 MiB."""
    Hq = Hkv = 16
    D, new = 64, [1] * 700 + [64] + [1] * 323
    g = torch.Generator().manual_seed(4)
    ctx = [n + int(x) for n, x in zip(new, torch.randint(0, 12, (1024,), generator=g))]
    c = make(ctx, new, Hq, Hkv, D)
    assert is_few(c, 64)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    torch.cuda.reset_peak_memory_stats(dev)
    o = prefill(c, dev, 0.1, max_seqlen=64)
    inputs = sum(t.numel() * t.element_size() for t in c.values())
    assert torch.cuda.max_memory_allocated(dev) - before < 2**29 + 2 * inputs
    assert_within(o, *reference(c, new, 0.1))


@pytest.mark.parametrize("most", [0, 1])
def test_tiles_of_more_tokens_than_said(dev, most):
    """The prefill in tiles takes its sequences from the offsets alone; with empty ones only, every row is zero."""
    new = [70, 0, 1, 33]
    for Hq, Hkv, D, dtype in HEADS[:4]:
        c = make([90, 4, 300, 33], new, Hq, Hkv, D, dtype=dtype)
        d = {n: t.to(dev) for n, t in c.items()}
        o = torch.full_like(d["q"], float("nan"))
        _lib.call("paged_attention_prefill_fp4", d["q"], d["kc"], d["vc"], d["ks"], d["vs"], d["tab"], d["ctx"], d["cu"],
                  o, None, most, 0.1)
        assert_within(o, *reference(c, new, 0.1))
        if most == 0:
            assert_within(prefill(c, dev, 0.1, max_seqlen=0), *reference(c, new, 0.1))
        out = torch.full_like(d["q"], float("nan"))
        assert not prefill(dict(c, cu=torch.zeros_like(c["cu"])), dev, 0.1, out=out).any()


@pytest.mark.parametrize("new", [[3, 1], [290, 1]])
def test_tables_without_columns(dev, new):
    """No keys at all: zero rows, in a few tokens and in tiles, as over 16-bit caches."""
    c = make([300, 20], new, 4, 2, 128)
    c["tab"] = c["tab"][:, :0]
    out = torch.full_like(c["q"], float("nan")).to(dev)
    assert not prefill(c, dev, 0.1, out=out).any()
    k, v = (cache_values(c[x + "c"], c[x + "s"]).nan_to_num(0).to(BF).to(dev) for x in "kv")
    o = ops.paged_flash_attention_prefill(c["q"].to(dev), k, v, c["tab"].to(dev), c["ctx"].to(dev), c["cu"].to(dev), None,
                                          0.1, 16)
    torch.cuda.synchronize()
    assert not o.any()
