"""GPU: the paged append against the float64 oracle, token by token.

Bound per element, derived: the rotation is two products and a sum in fp32
(below 4 x 2^-24 (|a| + |b|)), then one rounding to the output type (at most
half a step, eps / 2 relative, or half fp16's subnormal step 2^-25).  What is
not rotated is moved and has to be equal, as has every cache row not written.
"""
import pytest
import torch

from myvllm_amd import paged_flash_attention_decode, paged_kv_append
from oracle.attention import paged_kv_append_ref

pytestmark = pytest.mark.gpu


def rope(rows, rot, base=10000.0):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return a.cos().float(), a.sin().float()


def make(new, prefix, Hq=4, Hkv=2, D=128, page=16, dtype=torch.bfloat16, index=torch.int32, seed=0, spare=3, cols=0):
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
    return dict(q=r(T, Hq, D), k=r(T, Hkv, D), v=r(T, Hkv, D), k_cache=r(blocks, page, Hkv, D),
                v_cache=r(blocks, page, Hkv, D), block_tables=tab, context_lens=torch.tensor(ctx, dtype=index), cu=cu)


def close(got, ref, big):
    eps = torch.finfo(got.dtype).eps / 2
    bound = eps * (1 + 2**-10) * ref.abs() + 2**-22 * 2 * big + (2**-25 if got.dtype == torch.float16 else 0)
    err = (got.double().cpu() - ref).abs()
    assert got.shape == ref.shape and (err <= bound).all(), f"{int((err > bound).sum())} off, max {err.max():.3e}"


def check(c, dev, cu=True, cos=None, sin=None, interleaved=False, out=None, with_q=True):
    d = {n: t.to(dev) for n, t in c.items()}
    page = c["k_cache"].shape[1]
    got = paged_kv_append(d["q"] if with_q else None, d["k"], d["v"], d["k_cache"], d["v_cache"], d["block_tables"],
                          d["context_lens"], page, cos=None if cos is None else cos.to(dev),
                          sin=None if sin is None else sin.to(dev), cu_seqlens=d["cu"] if cu else None,
                          interleaved=interleaved, out=out)
    torch.cuda.synchronize()
    kc, vc = c["k_cache"].double(), c["v_cache"].double()
    ref = paged_kv_append_ref(c["q"] if with_q else None, c["k"], c["v"], kc, vc, c["block_tables"], c["context_lens"],
                              c["cu"] if cu else None, cos, sin, interleaved)
    big = float(max(c["q"].abs().max() if c["q"].numel() else 0, c["k"].abs().max() if c["k"].numel() else 0))
    assert torch.equal(d["v_cache"].cpu().double(), vc)
    written = (kc != c["k_cache"].double()).flatten(2).any(-1)
    assert torch.equal(d["k_cache"].cpu()[~written], c["k_cache"][~written])
    rot = 0 if cos is None else 2 * cos.shape[1]
    assert torch.equal(d["k_cache"].cpu()[..., rot:].double(), kc[..., rot:])
    close(d["k_cache"], kc, big)
    if with_q:
        close(got, ref, big)
        assert torch.equal(got.cpu()[..., rot:].double(), ref[..., rot:])
    else:
        assert got is None
    return got


@pytest.mark.parametrize(
    "new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index",
    [
        ([1], [0], 16, 2, 256, 16, 64, False, torch.bfloat16, torch.int32),
        ([1, 31, 0, 17], [0, 300, 5, 16], 16, 2, 256, 16, 256, False, torch.bfloat16, torch.int32),
        ([33, 64], [100, 0], 16, 4, 128, 7, 128, True, torch.float16, torch.int64),
        ([5, 0, 0, 90], [11, 0, 3, 1], 4, 4, 64, 48, 16, False, torch.float16, torch.int32),
        ([20, 3], [1000, 2], 6, 2, 64, 16, 48, True, torch.bfloat16, torch.int64),
        ([65], [1], 5, 1, 128, 1, 112, False, torch.bfloat16, torch.int32),
        ([40], [70], 1, 1, 256, 16, 0, False, torch.float16, torch.int32),
        ([9, 9], [7, 8], 70, 10, 256, 32, 32, False, torch.bfloat16, torch.int32),
    ],
)
def test_append(dev, new, prefix, Hq, Hkv, D, page, rot, inter, dtype, index):
    print(f"append new={new} prefix={prefix} {Hq}/{Hkv}x{D} page={page} rot={rot} {inter} {dtype}", flush=True)
    c = make(new, prefix, Hq, Hkv, D, page, dtype, index, seed=sum(new))
    cos, sin = rope(max(c["context_lens"]) + 1, rot) if rot else (None, None)
    check(c, dev, cos=cos, sin=sin, interleaved=inter)
    check(c, dev, cos=cos, sin=sin, interleaved=inter, with_q=False)


@pytest.mark.parametrize("B", [1, 64, 65, 257])
def test_append_one_token_each(dev, B):
    g = torch.Generator().manual_seed(B)
    c = make([1] * B, torch.randint(0, 100, (B,), generator=g).tolist(), seed=B)
    cos, sin = rope(101, 64)
    print(f"append decode B={B}", flush=True)
    a = check(c, dev, cu=False, cos=cos, sin=sin)
    b = check(c, dev, cu=True, cos=cos, sin=sin)
    assert torch.equal(a, b)


def test_append_many_sequences(dev):
    """Past 64 and 64^2 sequences the search takes further rounds; most are empty."""
    for N in (64, 100, 4097, 5000):
        new = [0] * N
        for i in (0, 1, N // 2, N - 2, N - 1):
            new[i] = 2 + i % 3
        print(f"append N={N}", flush=True)
        c = make(new, [0] * N, Hq=1, Hkv=1, D=64, seed=N)
        check(c, dev, cos=rope(16, 64)[0], sin=rope(16, 64)[1])


def test_append_tokens_without_a_place(dev):
    """Negative positions, positions past the table and past the rotation, table
    entries outside the cache, rows that no sequence covers."""
    c = make([10, 40, 20, 30], [0, 0, 5, 60], seed=3, cols=5)
    c["context_lens"] = torch.tensor([4, 95, 25, 90], dtype=torch.int32)  # 6 before 0; 55..94 of 80; 60..89 of 80
    c["block_tables"][1, 3] = c["k_cache"].shape[0]
    c["block_tables"][2, 1] = -7
    extra = 3
    for n in ("q", "k", "v"):
        c[n] = torch.cat([c[n][:extra], c[n], c[n][:extra]])
    c["cu"] = c["cu"] + extra
    cos, sin = rope(75, 128)
    print("append tokens without a place", flush=True)
    got = check(c, dev, cos=cos, sin=sin).cpu()
    assert (got[:extra] == 0).all() and (got[-extra:] == 0).all() and (got[extra:extra + 6] == 0).all()
    check(c, dev)


def test_append_strides_in_place_and_out(dev):
    """q, k, v as views of a packed projection, caches as views of a stack of
    layers; q rotated where it lies, into another tensor, and into a misaligned one."""
    c = make([30, 7], [3, 20], Hq=4, Hkv=2, D=128, seed=5)
    cos, sin = rope(64, 64)
    T = c["q"].shape[0]
    packed = torch.cat([c["q"].flatten(1), c["k"].flatten(1), c["v"].flatten(1)], 1).to(dev)
    ref = check(c, dev, cos=cos, sin=sin)
    stack = torch.zeros(2, 3, *c["k_cache"].shape, dtype=torch.bfloat16, device=dev)
    kc, vc = stack[0, 1], stack[1, 2]
    kc.copy_(c["k_cache"])
    vc.copy_(c["v_cache"])
    q, k, v = (x.unflatten(1, (-1, 128)) for x in packed.split([512, 256, 256], dim=1))
    args = [c[n].to(dev) for n in ("block_tables", "context_lens")]
    kw = dict(cos=cos.to(dev), sin=sin.to(dev), cu_seqlens=c["cu"].to(dev))
    o = paged_kv_append(q, k, v, kc, vc, *args, 16, **kw)
    assert torch.equal(o, ref)
    keep = stack.clone()
    wide = torch.empty(T, 4, 256, dtype=torch.bfloat16, device=dev)[..., 64:192]
    odd = torch.empty(T * 512 + 1, dtype=torch.bfloat16, device=dev)[1:].view(T, 4, 128)
    for out in (wide, odd):
        assert paged_kv_append(q, k, v, kc, vc, *args, 16, out=out, **kw) is out
        assert torch.equal(out, ref)
    moved = torch.empty(T * 512 + 1, dtype=torch.bfloat16, device=dev)[1:].view(T, 4, 128).copy_(q)
    assert torch.equal(paged_kv_append(moved, k, v, kc, vc, *args, 16, out=moved, **kw), ref)
    before = packed[:, 512:].clone()
    assert paged_kv_append(q, k, v, kc, vc, *args, 16, out=q, **kw) is q
    assert torch.equal(q, ref) and torch.equal(packed[:, 512:], before)
    assert torch.equal(stack, keep) and not stack[0, 0].any() and not stack[1, 1].any()


def test_append_far_blocks(dev):
    """Cache offsets past 2^31 elements and 2^32 bytes."""
    blocks = (1 << 31) // (16 * 2 * 256) + 10
    kc = torch.zeros(blocks, 16, 2, 256, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros(blocks, 16, 2, 256, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(20, 2, 256, generator=g).bfloat16().to(dev) for _ in range(2))
    tab = torch.tensor([[blocks - 1, blocks // 2]], device=dev)
    paged_kv_append(None, k, v, kc, vc, tab, torch.tensor([20], device=dev), 16,
                    cu_seqlens=torch.tensor([0, 20], device=dev))
    assert torch.equal(kc[blocks - 1], k[:16]) and torch.equal(vc[blocks // 2, :4], v[16:])
    assert int(torch.count_nonzero(kc.view(torch.int16).amax(dim=(1, 2, 3)))) <= 2


def test_append_then_decode_captured(dev):
    """A decode step's append and attention in one graph, replayed while the
    lengths grow, against the eager calls; on a stream of its own."""
    c = make([1, 1, 1], [20, 31, 0], Hq=4, Hkv=2, D=64, seed=9, cols=4)
    for n, row in enumerate(([0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11])):
        c["block_tables"][n, :4] = torch.tensor(row)
    g = torch.Generator().manual_seed(2)
    c["k_cache"] = torch.randn(12, 16, 2, 64, generator=g).bfloat16()
    c["v_cache"] = torch.randn(12, 16, 2, 64, generator=g).bfloat16()
    d = {n: t.to(dev) for n, t in c.items()}
    cos, sin = (t.to(dev) for t in rope(64, 64))
    eager = {n: d[n].clone() for n in ("k_cache", "v_cache")}

    def step(kc, vc):
        q = paged_kv_append(d["q"], d["k"], d["v"], kc, vc, d["block_tables"], d["context_lens"], 16, cos=cos, sin=sin)
        return paged_flash_attention_decode(q, kc, vc, d["block_tables"], d["context_lens"], 0.125, 16)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(d["k_cache"], d["v_cache"])
        step(eager["k_cache"], eager["v_cache"])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            o = step(d["k_cache"], d["v_cache"])
        for i in range(4):
            d["context_lens"] += 1
            for n in ("q", "k", "v"):
                d[n].copy_(torch.randn(d[n].shape, generator=g).bfloat16())
            graph.replay()
            ref = step(eager["k_cache"], eager["v_cache"])
            s.synchronize()
            assert torch.equal(o, ref)
            assert torch.equal(d["k_cache"], eager["k_cache"]) and torch.equal(d["v_cache"], eager["v_cache"])
