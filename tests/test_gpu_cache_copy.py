"""GPU: copies of blocks inside caches, and the forks and compaction made of them."""
import random

import pytest
import torch

from myvllm_amd import LinearAttentionCache, PagedKVCache, cache_copy
from myvllm_amd._lib import GdnError

pytestmark = pytest.mark.gpu


def check(caches, src, dst, to=list):
    want = [t.clone() for t in caches]
    for t in want:
        t[:, dst] = t[:, src]
    cache_copy(caches, to(src), to(dst))
    torch.cuda.synchronize()
    for a, b in zip(caches, want):
        assert torch.equal(a, b)


def pairs(blocks, n, seed=0):
    ids = random.Random(seed).sample(range(blocks), 2 * n)
    return ids[:n], ids[n:]


@pytest.mark.parametrize(
    "shape, dtype",
    [((3, 20, 16, 2, 128), torch.bfloat16), ((1, 20, 4096), torch.float16), ((2, 20, 4, 3, 5), torch.float32),
     ((4, 20, 7), torch.uint8), ((2, 20, 1), torch.int64), ((1, 20, 16385), torch.uint8), ((2, 20, 4, 8), torch.bool),
     ((2, 20, 8, 4), torch.float64), ((2, 20, 0), torch.float32), ((0, 20, 4), torch.float32)])
def test_shapes_and_types(dev, shape, dtype):
    print(f"cache copy {shape} {dtype}", flush=True)
    t = (torch.randn(shape, device=dev) * 50).to(dtype)
    for n in (1, 3, 10):
        check([t], *pairs(20, n, n))
    check([t], [], [])


@pytest.mark.parametrize("n", [31, 32, 33, 447, 448, 449, 1000])
def test_many_pairs(dev, n):
    print(f"cache copy {n} pairs", flush=True)
    blocks = 2 * n + 3
    a = torch.randn(2, blocks, 24, device=dev)
    b = torch.randint(0, 256, (3, blocks, 40), dtype=torch.uint8, device=dev)
    src, dst = pairs(blocks, n, n)
    check([a, b], src, dst)
    check([b], [src[0]] * n, dst, to=torch.tensor)  # one source for all


def test_views_and_several_caches(dev):
    """Layers of a larger cache, blocks with room between them, five caches in one call."""
    w = torch.randn(4, 12, 2, 40, device=dev)
    keep = w.clone()
    v = w[1:3, :, 1]
    want = v.clone()
    want[:, [4, 5]] = want[:, [0, 1]]
    cache_copy(v, [0, 1], [4, 5])
    torch.cuda.synchronize()
    assert torch.equal(v, want)
    keep[1:3, :, 1] = want
    assert torch.equal(w, keep)
    check([torch.randn(i + 1, 12, 5 * i + 4, device=dev) for i in range(5)], [3, 3, 9], [1, 11, 0])
    odd = torch.randn(2 * 12 * 8 + 1, device=dev)[1:].view(2, 12, 8)
    check([odd], [0, 2], [1, 3])


def test_refusals(dev):
    t = torch.zeros(2, 6, 32, device=dev)
    for src, dst in (([0], [6]), ([-1], [2]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(GdnError):
            cache_copy(t, src, dst)
    for args, match in (((t[0], [0], [1]), "layers, blocks"), (([t, t[:, :5]], [0], [1]), "one number"),
                        ((t.transpose(1, 2)[:, :6], [0], [1]), "side by side"),
                        ((t, torch.zeros(1, dtype=torch.int32, device=dev), [1]), "on the host")):
        with pytest.raises(ValueError, match=match):
            cache_copy(*args)
    assert not t.any()


def test_in_a_graph_and_on_a_stream(dev):
    t = torch.randn(2, 600, 64, device=dev)
    src, dst = pairs(600, 300)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache_copy(t, src, dst)
    for _ in range(3):
        t.copy_(torch.randn_like(t))
        want = t.clone()
        want[:, dst] = want[:, src]
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(t, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check([t], dst[:5], src[:5])


def test_state_cache_forks(dev):
    c = LinearAttentionCache(3, 8, 4, 128, 128, 2, 4, torch.bfloat16, dev)
    a = c.allocate()
    c.conv_cache[:, a].normal_()
    c.recurrent_cache[:, a].normal_()
    b = c.fork(a)
    more = c.fork_many([a, b, a])
    torch.cuda.synchronize()
    for s in [b, *more]:
        assert torch.equal(c.conv_cache[:, s], c.conv_cache[:, a])
        assert torch.equal(c.recurrent_cache[:, s], c.recurrent_cache[:, a])
    assert not c.recurrent_cache[:, list(c.free_slot_ids)].any()


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_cache_compaction(dev, bits):
    c = PagedKVCache(2, 1200, 16, 2, 64, torch.float16, dev, bits=bits)
    ids = [c.allocate() for _ in range(60)]
    r = random.Random(0)
    c.extend(ids, [r.randint(1, 300) for _ in ids])
    for t in c._tensors():
        t.copy_(torch.randint(0, 120, t.shape, device=dev))
    c.free(ids[::2])
    rows = {s: [t[:, c.blocks[s]].clone() for t in c._tensors()] for s in ids[1::2]}
    assert c.compact() > 100
    torch.cuda.synchronize()
    for s, was in rows.items():
        assert all(torch.equal(t[:, c.blocks[s]], x) for t, x in zip(c._tensors(), was))
    assert c.compact() == 0


@pytest.mark.parametrize("n, streams", [(779, False), (780, True), (1300, True)])
def test_large_copies(dev, n, streams):
    """32 MiB and more go by stores past the caches: two caches, several launches of 448 pairs, blocks that end inside a
    workgroup's 4 KB, and a kernel that reads the blocks straight after the copy."""
    print(f"cache copy of {n} large blocks", flush=True)
    blocks = 2 * n + 5
    a = torch.randint(-128, 127, (4, blocks, 4352), dtype=torch.int16, device=dev)  # blocks of 8,704 bytes
    b = torch.randint(0, 256, (2, blocks, 257, 16), dtype=torch.uint8, device=dev)  # of 4,112
    assert (n * (4 * 8704 + 2 * 4112) >= 2**25) == streams
    src, dst = pairs(blocks, n, n)
    s, d = (torch.tensor(x, device=dev) for x in (src, dst))
    want = [t.clone().index_copy_(1, d, t[:, s]) for t in (a, b)]
    torch.cuda.synchronize()
    cache_copy([a, b], src, dst)
    read = [t[:, d] + 1 for t in (a, b)]
    torch.cuda.synchronize()
    for t, w, r in zip((a, b), want, read):
        assert torch.equal(t, w) and torch.equal(r, w[:, d] + 1)
