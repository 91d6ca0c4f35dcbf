"""GPU: attention with capped or biased scores and prefix masks, against float64
(tests/attention_bounds.py derives the bound)."""
import pytest
import torch

from attention_bounds import assert_within, ref_and_bound
from myvllm_amd import (_lib, flash_attention_prefill, paged_flash_attention_decode, paged_flash_attention_prefill,
                        paged_kv_append)
from myvllm_amd.workloads import attn_varlen_case, paged_case
from oracle.attention import gather_paged

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def alibi(H):
    return 2.0 ** (-8 * (torch.arange(H) + 1.0) / H)


def form_of(kind, Hq, lens, dev, index=torch.int32):
    """Keywords of the ops and of the reference: cap, slopes, and prefix lengths from none to past the end."""
    kw, ref = {}, {}
    if "cap" in kind:
        kw["softcap"] = ref["softcap"] = 3.0
    if "slope" in kind:
        ref["slopes"] = alibi(Hq)
        kw["alibi_slopes"] = ref["slopes"].to(dev)
    pre = [0] * len(lens)
    if "mask" in kind:
        pre = [(0, n // 2 + 1, n + 9, 5)[i % 4] for i, n in enumerate(lens)]
        kw["prefix_lens"] = torch.tensor(pre, dtype=index, device=dev)
    return kw, ref, pre


def check_varlen(dev, case, causal, kw, ref_kw, pre):
    Hq, Hkv, D = case.q.shape[1], case.k.shape[1], case.q.shape[2]
    out = flash_attention_prefill(case.q.to(dev), case.k.to(dev), case.v.to(dev), case.cu.to(dev), case.scale, Hq, Hkv, D,
                                  D, causal, **kw).cpu()
    cu = case.cu.tolist()
    for n, (s, e) in enumerate(zip(cu, cu[1:])):
        ref, bound = ref_and_bound(case.q[s:e], case.k[s:e], case.v[s:e], torch.arange(e - s), case.scale, case.q.dtype,
                                   causal, prefix=pre[n], **ref_kw)
        assert_within(out[s:e], ref, bound, f"sequence {n}")
    return out


@pytest.mark.parametrize("kind", ["cap", "slope", "mask", "cap slope mask"])
@pytest.mark.parametrize(
    "lengths, Hq, Hkv, D, dtype",
    [
        ([1, 31, 33, 100, 257], 16, 2, 256, BF),
        ([70, 0, 129], 4, 4, 128, HF),
        ([300, 17], 8, 4, 64, BF),  # key tiles of 64
        ([96, 1, 45], 3, 1, 64, HF),
        ([130], 6, 2, 128, BF),
    ],
)
def test_varlen(dev, lengths, Hq, Hkv, D, dtype, kind):
    print(f"scored varlen {lengths} {Hq}/{Hkv}x{D} {dtype} {kind}", flush=True)
    case = attn_varlen_case(lengths, seed=sum(lengths), Hq=Hq, Hkv=Hkv, D=D, dtype=dtype)
    check_varlen(dev, case, True, *form_of(kind, Hq, lengths, dev, torch.int64 if D == 128 else torch.int32))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_varlen_both_directions(dev, D):
    case = attn_varlen_case([150, 33], seed=D, Hq=4, Hkv=2, D=D)
    print(f"scored bidirectional D={D}", flush=True)
    check_varlen(dev, case, False, *form_of("cap slope", 4, [150, 33], dev))


@pytest.mark.parametrize("scale, cap, slope", [(4.0, 2.0, 0.0), (4.0, 4096.0, 0.5), (-0.3, 5.0, 0.1), (0.0, 1.0, 0.25),
                                               (0.1, None, -0.02), (0.05, 0.25, 30.0), (1.0, 1e-3, 0.0), (1e30, 50.0, 0.0)])
def test_varlen_scales(dev, scale, cap, slope):
    """Saturated, hardly capped, folded signs, growing with distance, one key wide."""
    case = attn_varlen_case([65, 200], seed=7, Hq=4, Hkv=2, D=128)
    case.scale = scale
    print(f"scored scale={scale} cap={cap} slope={slope}", flush=True)
    slopes = torch.full((4,), slope)
    kw = dict(softcap=cap, alibi_slopes=slopes.to(dev))
    if scale == 1e30:  # every score is at the cap's end, of the sign of q.k
        out = flash_attention_prefill(case.q.to(dev), case.k.to(dev), case.v.to(dev), case.cu.to(dev), scale, 4, 2, 128,
                                      128, True, **kw).cpu()
        s = torch.einsum("nhd,mhd->nhm", case.q[:65].double(), case.k[:65].double().repeat_interleave(2, 1))
        p = torch.softmax((50 * s.sign()).masked_fill((torch.arange(65) > torch.arange(65)[:, None])[:, None],
                                                      -torch.inf), -1)
        ref = torch.einsum("nhm,mhd->nhd", p, case.v[:65].double().repeat_interleave(2, 1))
        big = torch.einsum("nhm,mhd->nhd", p, case.v[:65].double().abs().repeat_interleave(2, 1))
        assert_within(out[:65], ref, big * 2**-6.9)
        return
    check_varlen(dev, case, True, kw, dict(softcap=cap, slopes=slopes), [0, 0])


@pytest.mark.parametrize("cap, dtype", [(40.0, BF), (40.0, HF), (6.0, HF), (1.0, BF)])
def test_varlen_small_head_dim_caps(dev, cap, dtype):
    """At D = 64 tiles whose scores stay below 3/4 of the cap go another way: all, some and none of them."""
    case = attn_varlen_case([400, 33], seed=11, Hq=4, Hkv=2, D=64, dtype=dtype)
    print(f"scored D=64 cap={cap} {dtype}", flush=True)
    for slopes in (None, alibi(4)):
        kw = dict(softcap=cap, alibi_slopes=None if slopes is None else slopes.to(dev))
        check_varlen(dev, case, True, kw, dict(softcap=cap, slopes=slopes), [0, 0])


def test_varlen_other_head_dim_strides_and_out(dev):
    """A head dim that runs padded; views of a packed projection into a given tensor."""
    case = attn_varlen_case([50, 20], seed=3, Hq=4, Hkv=4, D=72)
    kw, ref, pre = form_of("cap slope mask", 4, [50, 20], dev)
    check_varlen(dev, case, True, kw, ref, pre)
    case = attn_varlen_case([50, 20], seed=3, Hq=4, Hkv=2, D=64)
    want = check_varlen(dev, case, True, kw, ref, pre)
    packed = torch.cat([case.q.flatten(1), case.k.flatten(1), case.v.flatten(1)], 1).to(dev)
    q, k, v = (t.unflatten(1, (-1, 64)) for t in packed.split([256, 128, 128], 1))
    for out in (torch.empty(70, 4, 96, dtype=BF, device=dev)[..., :64],
                torch.empty(70 * 256 + 1, dtype=BF, device=dev)[1:].view(70, 4, 64)):
        got = flash_attention_prefill(q, k, v, case.cu.to(dev), case.scale, 4, 2, 64, 64, True, out=out, **kw)
        assert got is out and torch.equal(out.cpu(), want)


def test_no_form_is_the_plain_op(dev):
    """softcap 0 and nothing else leaves the scores as they are, to the last product's rounding."""
    case = attn_varlen_case([100, 3], seed=1, Hq=4, Hkv=2, D=128)
    check_varlen(dev, case, True, dict(softcap=0.0), {}, [0, 0])


def poison(case, dev):
    """The cache with NaN wherever no sequence has a key."""
    kc, vc = case.k_cache.clone(), case.v_cache.clone()
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for n, L in enumerate(case.context_lens.tolist()):
        j = torch.arange(min(L, case.block_tables.shape[1] * case.page))
        used[case.block_tables[n, j // case.page].long(), j % case.page] = True
    kc[~used] = float("nan")
    vc[~used] = float("nan")
    return kc.to(dev), vc.to(dev)


def check_paged(dev, case, kw, ref_kw, pre, lib=False):
    kc, vc = poison(case, dev)
    d = [t.to(dev) for t in (case.q, case.block_tables, case.context_lens, case.cu)]
    out = paged_flash_attention_prefill(d[0], kc, vc, d[1], d[2], d[3], None, case.scale, case.page, **kw)
    if lib:  # the same without a workspace
        whole = torch.empty_like(out)
        _lib.call("paged_attention_prefill_scored", d[0], kc, vc, *d[1:], whole, None, kw.get("alibi_slopes"),
                  kw.get("prefix_lens"), case.max_len, case.scale, kw.get("softcap") or 0.0)
        outs = (out, whole)
    else:
        outs = (out,)
    cu = case.cu.tolist()
    for n, L in enumerate(case.context_lens.tolist()):
        s, e = cu[n], cu[n + 1]
        k, v = (gather_paged(c, case.block_tables[n], L) for c in (case.k_cache, case.v_cache))
        ref, bound = ref_and_bound(case.q[s:e], k, v, torch.arange(L - (e - s), L), case.scale, case.q.dtype,
                                   prefix=pre[n], **ref_kw)
        for o in outs:
            assert_within(o[s:e], ref, bound, f"sequence {n}")
    return out


@pytest.mark.parametrize("kind", ["cap", "slope mask", "cap slope mask"])
@pytest.mark.parametrize(
    "ctx, new, page, Hq, Hkv, D, dtype, index",
    [
        ([40, 300, 17], [40, 100, 1], 16, 16, 2, 256, BF, torch.int32),
        ([77, 130], [33, 130], 7, 4, 4, 128, HF, torch.int64),
        ([64, 0, 5], [10, 0, 5], 16, 8, 2, 64, BF, torch.int64),
        ([4, 20, 0], [9, 50, 3], 16, 4, 2, 128, BF, torch.int32),  # queries before the first key, and without any
        ([4096, 37, 1500], [3, 37, 40], 16, 16, 2, 256, BF, torch.int32),  # split over the keys
        ([3000, 3001], [33, 70], 48, 4, 4, 128, HF, torch.int64),  # split
        ([2500, 700], [31, 90], 32, 8, 4, 64, HF, torch.int32),  # split
    ],
)
def test_paged_prefill(dev, ctx, new, page, Hq, Hkv, D, dtype, index, kind):
    print(f"scored paged prefill {ctx} {new} page={page} {Hq}/{Hkv}x{D} {kind}", flush=True)
    case = paged_case(ctx, new, page=page, seed=sum(ctx), Hq=Hq, Hkv=Hkv, D=D, dtype=dtype)
    case.block_tables, case.context_lens = case.block_tables.to(index), case.context_lens.to(index)
    check_paged(dev, case, *form_of(kind, Hq, ctx, dev, index), lib=True)


def test_paged_prefill_uncovered_rows(dev):
    case = paged_case([40, 30], [10, 30], page=16, seed=2, Hq=4, Hkv=2, D=64)
    kw, _, _ = form_of("cap slope mask", 4, [40, 30], dev)
    d = [t.to(dev) for t in (case.k_cache, case.v_cache, case.block_tables, case.context_lens)]
    q = torch.cat([case.q[:3], case.q, case.q[:5]]).to(dev)
    out = torch.full_like(q, float("nan"))
    paged_flash_attention_prefill(q, *d, case.cu.to(dev) + 3, None, case.scale, 16, out=out, **kw)
    ref = paged_flash_attention_prefill(case.q.to(dev), *d, case.cu.to(dev), None, case.scale, 16, **kw)
    assert torch.equal(out[3:-5], ref) and not out[:3].any() and not out[-5:].any()


@pytest.mark.parametrize("splits", [1, 3, None])
@pytest.mark.parametrize(
    "ctx, Hq, Hkv, D, page, dtype, index",
    [
        ([1, 17, 300, 0, 64], 16, 2, 256, 16, BF, torch.int32),
        ([33, 500], 4, 4, 128, 7, HF, torch.int64),
        ([129, 16, 3], 64, 2, 64, 32, BF, torch.int32),  # two head groups per kv head
        ([5000, 1, 40], 8, 1, 128, 48, HF, torch.int32),
    ],
)
def test_decode(dev, ctx, Hq, Hkv, D, page, dtype, index, splits):
    print(f"scored decode {ctx} {Hq}/{Hkv}x{D} page={page} splits={splits}", flush=True)
    case = paged_case(ctx, [1] * len(ctx), page=page, seed=sum(ctx), Hq=Hq, Hkv=Hkv, D=D, dtype=dtype)
    kc, vc = poison(case, dev)
    d = [t.to(dev) for t in (case.q, case.block_tables.to(index), case.context_lens.to(index))]
    for kind in ("cap", "slope", "cap slope"):
        kw, ref_kw, _ = form_of(kind, Hq, ctx, dev)
        out = paged_flash_attention_decode(d[0], kc, vc, d[1], d[2], case.scale, page, num_splits=splits, **kw)
        for n, L in enumerate(ctx):
            k, v = (gather_paged(c, case.block_tables[n], L) for c in (case.k_cache, case.v_cache))
            ref, bound = ref_and_bound(case.q[n:n + 1], k, v, [L - 1], case.scale, dtype, **ref_kw)
            assert_within(out[n:n + 1], ref, bound, f"{kind} {n}")


def test_decode_many_sequences(dev):
    """Past 1,024 sequences the prices come from a launch of their own."""
    g = torch.Generator().manual_seed(6)
    ctx = torch.randint(0, 70, (1100,), generator=g).tolist()
    case = paged_case(ctx, [1] * 1100, seed=1, Hq=4, Hkv=2, D=64)
    kw, ref_kw, _ = form_of("cap slope", 4, ctx, dev)
    print("scored decode B=1100", flush=True)
    d = [t.to(dev) for t in (case.q, case.k_cache, case.v_cache, case.block_tables, case.context_lens)]
    out = paged_flash_attention_decode(*d, case.scale, 16, num_splits=2, **kw)
    for n in list(range(0, 1100, 37)) + [1099]:
        k, v = (gather_paged(c, case.block_tables[n], ctx[n]) for c in (case.k_cache, case.v_cache))
        ref, bound = ref_and_bound(case.q[n:n + 1], k, v, [ctx[n] - 1], case.scale, BF, **ref_kw)
        assert_within(out[n:n + 1], ref, bound, str(n))


def test_append_prefill_decode(dev):
    """A prompt in two chunks and two decode steps through the cache that the
    append fills, against the packed op over the whole of it."""
    g = torch.Generator().manual_seed(8)
    Hq, Hkv, D, T = 8, 2, 128, 90
    q, k, v = (torch.randn(T, h, D, generator=g).to(BF).to(dev) for h in (Hq, Hkv, Hkv))
    ang = torch.arange(T)[:, None] * 100.0 ** (-torch.arange(32) / 32)
    cos, sin = ang.cos().to(dev), ang.sin().to(dev)
    kc, vc = (torch.full((8, 16, Hkv, D), float("nan"), dtype=BF, device=dev) for _ in range(2))
    tab = torch.tensor([[5, 0, 3, 7, 1, 2]], dtype=torch.int32, device=dev)
    kw = dict(softcap=20.0, alibi_slopes=alibi(Hq).to(dev))
    out, rot = [], []
    for a, b in ((0, 50), (50, 88), (88, 89), (89, 90)):
        ctx = torch.tensor([b], dtype=torch.int32, device=dev)
        cu = torch.tensor([0, b - a], dtype=torch.int32, device=dev)
        qr = paged_kv_append(q[a:b], k[a:b], v[a:b], kc, vc, tab, ctx, 16, cos, sin, cu_seqlens=cu)
        rot.append(qr)
        out.append(paged_flash_attention_decode(qr, kc, vc, tab, ctx, 0.1, 16, **kw) if b - a == 1 else
                   paged_flash_attention_prefill(qr, kc, vc, tab, ctx, cu, None, 0.1, 16, **kw))
    keys = gather_paged(kc.cpu(), tab[0].cpu(), T)
    ref, bound = ref_and_bound(torch.cat(rot).cpu(), keys, v.cpu(), torch.arange(T), 0.1, BF, softcap=20.0,
                               slopes=alibi(Hq))
    assert_within(torch.cat(out), ref, bound)
    whole = flash_attention_prefill(torch.cat(rot), keys.to(dev), v, torch.tensor([0, T], device=dev), 0.1, Hq, Hkv, D,
                                    D, True, **kw)
    assert_within(whole, ref, bound)


def test_scored_calls_captured(dev):
    """Prefill and decode in one graph, replayed with other inputs and lengths."""
    case = paged_case([200, 90], [20, 20], seed=4, Hq=8, Hkv=2, D=64)
    one = paged_case([200, 90], [1, 1], seed=5, Hq=8, Hkv=2, D=64)
    kw, _, _ = form_of("cap slope mask", 8, [200, 90], dev)
    dkw = {n: kw[n] for n in ("softcap", "alibi_slopes")}
    d = {n: getattr(case, n).to(dev) for n in ("q", "k_cache", "v_cache", "block_tables", "context_lens", "cu")}
    q1 = one.q.to(dev)

    def step():
        a = paged_flash_attention_prefill(d["q"], d["k_cache"], d["v_cache"], d["block_tables"], d["context_lens"],
                                          d["cu"], None, 0.2, 16, max_seqlen=20, **kw)
        b = paged_flash_attention_decode(q1, d["k_cache"], d["v_cache"], d["block_tables"], d["context_lens"], 0.2, 16,
                                         **dkw)
        return a, b

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = step()
        for i in range(4):
            d["context_lens"] -= 13
            kw["prefix_lens"] += 7
            kw["alibi_slopes"] *= 0.5
            q1.mul_(-0.5)
            graph.replay()
            want = step()
            s.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
