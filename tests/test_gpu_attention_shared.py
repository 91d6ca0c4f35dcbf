"""GPU: decode of sequences that share their first keys, against float64 over
each sequence's own table (tests/attention_bounds.py derives the bound) and
against the plain decode."""
import pytest
import torch

from attention_bounds import assert_within, ref_and_bound
from myvllm_amd import paged_flash_attention_decode, paged_flash_attention_decode_shared, paged_kv_append
from oracle.attention import gather_paged

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(groups, Hq, Hkv, D, page=16, dtype=BF, index=torch.int32, seed=0, cols=0):
    """groups: (shared keys, [own keys of each sequence]); an own count below 0
    is a sequence that much shorter than the shared keys (it still holds them as
    far as it goes).  Whole shared pages are the same ones, the rest of the
    shared keys is copied into each sequence's own page; NaN wherever no
    sequence has a key."""
    g = torch.Generator().manual_seed(seed)
    ctx = [max(0, p + n) for p, own in groups for n in own]
    need = sum(-(-c // page) for c in ctx) + 3
    order = torch.randperm(need, generator=g).tolist()
    tab = torch.full((len(ctx), max([cols, 1] + [-(-c // page) for c in ctx])), -1, dtype=index)
    kc, vc = (torch.full((need, page, Hkv, D), float("nan"), dtype=dtype) for _ in range(2))
    b = 0
    for p, own in groups:
        # keys of the longest possible prefix, then each sequence's own
        pk, pv = (torch.randn(p, Hkv, D, generator=g).to(dtype) for _ in range(2))
        whole = [order.pop() for _ in range(min(p, max([p + n for n in own] + [0])) // page)]
        for n in own:
            L = max(0, p + n)
            mine = whole[:L // page] if L < p else whole
            mine = mine + [order.pop() for _ in range(-(-L // page) - len(mine))]
            tab[b, :len(mine)] = torch.tensor(mine, dtype=index)
            k, v = (torch.cat([x, torch.randn(max(n, 0), Hkv, D, generator=g).to(dtype)])[:L] for x in (pk, pv))
            j = torch.arange(L)
            kc[tab[b, j // page].long(), j % page] = k
            vc[tab[b, j // page].long(), j % page] = v
            b += 1
    q = torch.randn(len(ctx), Hq, D, generator=g).to(dtype)
    cu = [0]
    for _, own in groups:
        cu.append(cu[-1] + len(own))
    return dict(q=q, k_cache=kc, v_cache=vc, block_tables=tab, context_lens=torch.tensor(ctx, dtype=index),
                prefix_lens=torch.tensor([p for p, _ in groups], dtype=index)), torch.tensor(cu, dtype=index)


def check(dev, c, cu, scale=None, rows=None, plain=True):
    d = {n: t.to(dev) for n, t in c.items()}
    page, D = c["k_cache"].shape[1], c["q"].shape[2]
    scale = D**-0.5 if scale is None else scale
    out = paged_flash_attention_decode_shared(*d.values(), scale, page, cu_groups=None if cu is None else cu.to(dev))
    for b in range(len(c["q"])) if rows is None else rows:
        L = int(c["context_lens"][b])
        k, v = (gather_paged(c[n], c["block_tables"][b], L) for n in ("k_cache", "v_cache"))
        ref, bound = ref_and_bound(c["q"][b:b + 1], k, v, [L - 1], scale, c["q"].dtype)
        assert_within(out[b:b + 1], ref, bound, f"sequence {b}")
    if plain:
        d.pop("prefix_lens")
        want = paged_flash_attention_decode(*d.values(), scale, page)
        assert torch.isfinite(out).all()
        assert (out.double() - want.double()).norm() <= 6e-3 * want.double().norm().clamp_min(1e-12)
    return out


@pytest.mark.parametrize(
    "groups, Hq, Hkv, D, page, dtype, index",
    [
        ([(1000, [1, 5, 64, 33])], 16, 2, 256, 16, BF, torch.int32),
        ([(1000, [17, 1, 300])], 16, 4, 128, 16, HF, torch.int64),
        ([(500, [3, 40] * 20)], 4, 4, 64, 16, BF, torch.int32),  # one head per kv head
        ([(331, [1, 2, 3])], 6, 2, 128, 7, BF, torch.int32),  # a lookup per row
        ([(2000, [0, 1, 48])], 64, 2, 64, 48, HF, torch.int64),  # 32 heads per kv head; nothing of its own
        ([(15, [9, 30]), (16, [9, 0]), (17, [1, 2]), (0, [4, 5])], 8, 2, 128, 16, BF, torch.int32),
        ([(64, [10]), (700, [1, 2, 3]), (90, []), (31, [5] * 9), (2500, [7, 800])], 16, 2, 256, 16, BF, torch.int64),
        ([(400, [-400, 5, -1, -100, 60])], 8, 1, 256, 16, BF, torch.int32),  # padding first, shorter ones between
        ([(400, [-10, -20, -400])], 8, 2, 64, 32, HF, torch.int32),  # all shorter
        ([(40, [3] * 130)], 16, 2, 256, 16, BF, torch.int32),  # several blocks of 128 rows
        ([(33 + i, [2, 1 + i]) for i in range(70)], 4, 2, 64, 16, BF, torch.int32),  # past 64 groups
        ([(9000, [30, 2])], 2, 1, 128, 16, BF, torch.int32),  # two rows, many pieces
    ],
)
def test_shared(dev, groups, Hq, Hkv, D, page, dtype, index):
    print(f"shared decode {str(groups)[:70]} {Hq}/{Hkv}x{D} page={page} {dtype}", flush=True)
    c, cu = make(groups, Hq, Hkv, D, page, dtype, index, seed=len(groups))
    out = check(dev, c, cu)
    assert (out[c["context_lens"] == 0] == 0).all()
    if len(groups) == 1:
        assert torch.equal(check(dev, c, None), out)


def test_one_sequence_and_none(dev):
    c, cu = make([(100, [7])], 16, 2, 256)
    print("shared decode of one and of none", flush=True)
    check(dev, c, cu)
    d = {n: t.to(dev) for n, t in c.items()}
    empty = paged_flash_attention_decode_shared(d["q"][:0], d["k_cache"], d["v_cache"], d["block_tables"][:0],
                                                d["context_lens"][:0], d["prefix_lens"], 1.0, 16)
    assert empty.shape == (0, 16, 256)
    check(dev, c | dict(prefix_lens=c["prefix_lens"][:0]), cu[:1])  # no groups


def test_sequences_outside_the_groups(dev):
    c, cu = make([(50, [3, 4]), (200, [1, 9, 2]), (60, [5, 5])], 8, 2, 128, seed=4)
    print("shared decode, sequences in no group", flush=True)
    check(dev, c | dict(prefix_lens=c["prefix_lens"][1:2]), cu[1:3])


def test_prefix_past_the_table(dev):
    """More shared keys than the table holds: all sequences are shorter."""
    c, cu = make([(64, [0, 0, 0])], 8, 2, 128)
    print("shared decode, prefix past the table", flush=True)
    for p in (64, 65, 10**6, -5):
        check(dev, c | dict(prefix_lens=torch.tensor([p], dtype=torch.int32)), cu)


@pytest.mark.parametrize("scale", [4.0, -0.2, 0.0])
def test_scales(dev, scale):
    c, cu = make([(300, [20, 70, 1])], 4, 2, 64, seed=2)
    print(f"shared decode scale={scale}", flush=True)
    check(dev, c, cu, scale=scale, plain=False)


@pytest.mark.parametrize("D, page, index", [(64, 16, torch.int32), (64, 48, torch.int64), (128, 32, torch.int32),
                                            (256, 16, torch.int64)])
def test_long_own_keys(dev, D, page, index):
    """Many kv heads leave few units: pieces of over 1,024 own keys, whose pages are looked up in batches."""
    c, cu = make([(100, [3000, 17, 2500, 1])], 64, 64, D, page, index=index, seed=6)
    print(f"shared decode, long own keys D={D} page={page}", flush=True)
    check(dev, c, cu)


def test_many_sequences(dev):
    """Past 1,024 sequences the prices come from a launch of their own; more row blocks than the chip has room for."""
    g = torch.Generator().manual_seed(3)
    own = torch.randint(0, 50, (1500,), generator=g).tolist()
    c, cu = make([(100, own[:700]), (333, own[700:])], 4, 2, 64, seed=3)
    print("shared decode B=1500", flush=True)
    check(dev, c, cu, rows=list(range(0, 1500, 41)) + [699, 700, 1499])


def test_views_and_out(dev):
    """Caches and queries as views, a misaligned output."""
    c, cu = make([(90, [7, 20, 1])], 4, 2, 64, seed=8)
    want = check(dev, c, cu)
    d = {n: t.to(dev) for n, t in c.items()}
    stack = torch.stack([d["k_cache"], d["v_cache"]], 1)
    d["k_cache"], d["v_cache"] = stack[:, 0], stack[:, 1]
    wide = torch.zeros(3, 4, 200, dtype=BF, device=dev)
    wide[..., 8:72] = d["q"]
    d["q"] = wide[..., 8:72]
    tab = torch.full((3, 50), -1, dtype=torch.int32, device=dev)
    tab[:, 5:5 + d["block_tables"].shape[1]] = d["block_tables"]
    d["block_tables"] = tab[:, 5:5 + d["block_tables"].shape[1]]
    for out in (torch.empty(3, 4, 128, dtype=BF, device=dev)[..., 64:],
                torch.empty(3 * 256 + 1, dtype=BF, device=dev)[1:].view(3, 4, 64)):
        got = paged_flash_attention_decode_shared(*d.values(), 0.125, 16, out=out)
        assert got is out and torch.equal(out, want)


def test_far_pages(dev):
    """Shared and own pages past 2^31 elements of the cache."""
    c, cu = make([(100, [40, 3])], 4, 2, 256, seed=9)
    blocks = (1 << 31) // (16 * 2 * 256) + len(c["k_cache"])
    d = {n: t.to(dev) for n, t in c.items()}
    for n in ("k_cache", "v_cache"):
        far = torch.empty(blocks, 16, 2, 256, dtype=BF, device=dev)
        far[-len(c[n]):] = d[n]
        d[n] = far
    off = blocks - len(c["k_cache"])
    d["block_tables"] = torch.where(d["block_tables"] >= 0, d["block_tables"] + off, d["block_tables"])
    got = paged_flash_attention_decode_shared(*d.values(), 256**-0.5, 16)
    assert torch.equal(got, check(dev, c, cu))


def test_without_room_for_a_workspace(dev, monkeypatch):
    """The plain decode's result, bit for bit."""
    c, cu = make([(90, [7, 20, 1])], 4, 2, 64, seed=8)
    d = {n: t.to(dev) for n, t in c.items()}
    want = paged_flash_attention_decode(*list(d.values())[:5], 0.125, 16)
    real, refused = torch.empty, []

    def empty(*a, **kw):
        if kw.get("dtype") == torch.float32 and not refused:
            refused.append(a)
            raise torch.OutOfMemoryError("none left")
        return real(*a, **kw)

    monkeypatch.setattr(torch, "empty", empty)
    got = paged_flash_attention_decode_shared(*d.values(), 0.125, 16, cu_groups=cu.to(dev))
    assert refused and torch.equal(got, want)


def test_append_and_shared_decode_captured(dev):
    """Decode steps of a batch behind one prompt, append and attention, in two
    graphs that share a memory pool, replayed in turn against eager calls."""
    g = torch.Generator().manual_seed(5)
    c, cu = make([(200, [1, 9, 30, 5])], 8, 2, 128, seed=5, cols=20)
    used = 0
    for b, L in enumerate(c["context_lens"].tolist()):  # pages of their own for the steps to come
        n = -(-L // 16)
        c["block_tables"][b, n:n + 2] = torch.tensor([len(c["k_cache"]) + used, len(c["k_cache"]) + used + 1])
        used += 2
    for n in ("k_cache", "v_cache"):
        c[n] = torch.cat([c[n], torch.full((used, 16, 2, 128), float("nan"), dtype=BF)])
    d = {n: t.to(dev) for n, t in c.items()}
    eager = {n: d[n].clone() for n in ("k_cache", "v_cache")}
    k, v = (torch.randn(4, 2, 128, generator=g).to(BF).to(dev) for _ in range(2))
    cos, sin = torch.rand(512, 64, device=dev), torch.rand(512, 64, device=dev)

    def step(kc, vc, prefix):
        q = paged_kv_append(d["q"], k, v, kc, vc, d["block_tables"], d["context_lens"], 16, cos, sin)
        return paged_flash_attention_decode_shared(q, kc, vc, d["block_tables"], d["context_lens"], prefix, 0.1, 16)

    prefixes = [d["prefix_lens"], d["prefix_lens"] - 90]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(eager["k_cache"], eager["v_cache"], prefixes[0])
        step(d["k_cache"], d["v_cache"], prefixes[0])
        graphs, outs = [], []
        for p in prefixes:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s, pool=graphs[0].pool() if len(graphs) > 1 else None):
                outs.append(step(d["k_cache"], d["v_cache"], p))
        for i in range(6):
            d["context_lens"] += 1
            k.mul_(-0.75)
            d["q"].mul_(-1.1)
            graphs[i % 2].replay()
            got = outs[i % 2].clone()
            want = step(eager["k_cache"], eager["v_cache"], prefixes[i % 2])
            s.synchronize()
            assert torch.isfinite(got).all() and torch.equal(got, want)
