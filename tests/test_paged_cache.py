"""CPU: the allocator of the paged cache (forks, copies on write, compaction), the
forks of the state cache, and what the block copy refuses."""
import ctypes
import random

import pytest
import torch

import myvllm_amd.cache as cache_module
from myvllm_amd import LinearAttentionCache, PagedKVCache, _lib, cache_copy

cpu_only = pytest.mark.skipif(torch.cuda.is_available(), reason="host pointers in the calls")
ERR = {"NULL": -1, "NDIM": -2, "SHAPE": -3, "DTYPE": -4, "STRIDE": -5, "RANGE": -11, "ARG": -13}
CPU = torch.device("cpu")


def copy_ref(caches, src, dst):
    """The copy in plain torch, with the checks of the entry."""
    assert len(set(dst)) == len(dst) and not set(dst) & set(src)
    for t in caches:
        t[:, dst] = t[:, src]


@pytest.fixture
def plain_copy(monkeypatch):
    calls = []

    def copy(caches, src, dst):
        calls.append((list(src), list(dst)))
        copy_ref(caches, list(src), list(dst))

    monkeypatch.setattr(cache_module, "cache_copy", copy)
    return calls


def paged(bits=16, blocks=8, size=16):
    return PagedKVCache(2, blocks, size, 2, 64, torch.bfloat16, CPU, bits=bits)


def test_layouts():
    c = paged()
    assert c.k_cache.shape == c.v_cache.shape == (2, 8, 16, 2, 64) and c.k_cache.dtype == torch.bfloat16
    k, v, ks, vs = c.layer(1)
    assert k.shape == (8, 16, 2, 64) and ks is None and vs is None
    assert PagedKVCache.bytes_per_block(2, 16, 2, 64, torch.bfloat16) * 8 == 2 * c.k_cache.numel() * 2
    c = paged(4)
    assert c.k_cache.shape == (2, 8, 16, 2, 32) and c.k_scales.shape == (2, 8, 2, 2, 16)
    assert c.layer(0)[2].shape == (8, 2, 2, 16)
    per = PagedKVCache.bytes_per_block(2, 16, 2, 64, torch.bfloat16, bits=4)
    assert per * 8 == 2 * (c.k_cache.numel() + c.k_scales.numel())
    for kw in (dict(bits=8), dict(bits=4, size=24)):
        with pytest.raises(ValueError):
            paged(**kw)


def test_extend_fork_free(plain_copy):
    c = paged()
    a, b = c.allocate(), c.allocate()
    c.extend([a, b], [20, 16])
    assert c.blocks[a] == [0, 1] and c.blocks[b] == [2] and c.lengths == {a: 20, b: 16}
    tab, ctx = c.tables([b, a])
    assert tab.tolist() == [[2, -1], [0, 1]] and ctx.tolist() == [16, 20]
    f = c.fork(a)
    assert c.blocks[f] == [0, 1] and c.holders[:3] == [2, 2, 1]
    c.k_cache[:, 1] = 3
    c.extend([f], [1])  # into the shared, partly filled block: a copy
    assert plain_copy == [([1], [3])] and c.blocks[f] == [0, 3] and (c.k_cache[:, 3] == 3).all()
    c.extend([a], [13])  # now its own; a third block
    assert c.blocks[a] == [0, 1, 4] and len(plain_copy) == 1
    g = c.fork(b)
    c.extend([g, b], [1, 1])  # a full block is shared as it is
    assert c.blocks[g] == [2, 5] and c.blocks[b] == [2, 6] and len(plain_copy) == 1
    c.free([a, b])
    assert c.holders == [1, 0, 1, 1, 0, 1, 0, 0] and set(c.free_block_ids) == {1, 4, 6, 7}
    c.free([f, g])
    assert sorted(c.free_block_ids) == list(range(8)) and not any(c.holders) and not c.blocks


def test_one_of_the_holders_keeps_the_block(plain_copy):
    c = paged()
    a = c.allocate()
    c.extend([a], [5])
    b, d = c.fork(a), c.fork(a)
    c.extend([a, b, d], [1, 0, 1])  # b does not write: both others copy
    assert plain_copy == [([0, 0], [1, 2])] and c.blocks == {a: [1], b: [0], d: [2]}
    e = c.fork(b)
    c.extend([b, e], [1, 1])  # both write: the last one stays
    assert plain_copy[1:] == [([0], [3])] and c.blocks[b] == [3] and c.blocks[e] == [0]


def test_refusals_change_nothing(plain_copy):
    c = paged(blocks=3)
    a = c.allocate()
    c.extend([a], [40])
    b = c.fork(a)
    before = (c.blocks[a][:], c.lengths.copy(), list(c.free_block_ids), c.holders[:])
    for ids, counts in (([a], [9]), ([b], [1])):
        with pytest.raises(RuntimeError):
            c.extend(ids, counts)
    for ids, counts in (([a, a], [1, 1]), ([7], [1]), ([a], [-1]), ([a], [])):
        with pytest.raises(ValueError):
            c.extend(ids, counts)
    for ids in ([9], [a, a]):
        with pytest.raises(ValueError):
            c.free(ids)
    with pytest.raises(ValueError):
        c.fork(9)
    with pytest.raises(ValueError):
        c.tables([9])
    assert before == (c.blocks[a], c.lengths, list(c.free_block_ids), c.holders) and not plain_copy


@pytest.mark.parametrize("bits", [16, 4])
def test_random_life(plain_copy, bits):
    """Every sequence reads back its own tokens after any order of calls."""
    r = random.Random(bits)
    c = paged(bits, blocks=40)
    said: dict[int, list[int]] = {}
    for step in range(400):
        do = r.random()
        ids = list(said)
        if do < 0.25 or not ids:
            said[c.allocate()] = []
        elif do < 0.65:
            some = r.sample(ids, r.randint(1, len(ids)))
            counts = [r.randint(0, 20) for _ in some]
            old = {s: c.lengths[s] for s in some}
            try:
                c.extend(some, counts)
            except RuntimeError:
                continue
            for s, n in zip(some, counts):
                for p in range(old[s], old[s] + n):
                    x = r.randrange(100)
                    said[s].append(x)
                    for t in c._tensors():
                        at = t[:, c.blocks[s][p // 16]]
                        (at[..., p % 16] if t is c.k_scales or t is c.v_scales else at[:, p % 16]).fill_(x)
        elif do < 0.8:
            s = r.choice(ids)
            said[c.fork(s)] = said[s][:]
        elif do < 0.95:
            gone = r.sample(ids, r.randint(1, max(1, len(ids) // 2)))
            c.free(gone)
            for s in gone:
                del said[s]
        else:
            c.compact()
            used = {b for x in c.blocks.values() for b in x}
            assert used == set(range(len(used)))
        held = [0] * 40
        for x in c.blocks.values():
            for b in x:
                held[b] += 1
        assert held == c.holders and sorted(c.free_block_ids) == [b for b in range(40) if not held[b]]
    for s, x in said.items():
        assert c.lengths[s] == len(x)
        for p, v in enumerate(x):
            assert (c.k_cache[:, c.blocks[s][p // 16], p % 16] == v).all()
            if bits == 4:
                assert (c.v_scales[:, c.blocks[s][p // 16], ..., p % 16] == v).all()


def test_state_forks(plain_copy):
    c = LinearAttentionCache(3, 4, 4, 8, 16, 2, 4, torch.bfloat16, CPU)
    a = c.allocate()
    c.conv_cache[:, a], c.recurrent_cache[:, a] = 2, 5
    assert c.fork(a) == 1 and (c.recurrent_cache[:, 1] == 5).all() and (c.conv_cache[:, 1] == 2).all()
    assert c.fork_many([a, 1]) == [2, 3] and (c.recurrent_cache == 5).all()
    with pytest.raises(RuntimeError):
        c.fork(a)
    c.deallocate(2)
    with pytest.raises(ValueError):
        c.fork(2)
    assert c.fork_many([]) == [] and len(c.free_slot_ids) == 1


def call(caches, pairs):
    d = [None if t is None else ctypes.byref(t if isinstance(t, _lib.GdnTensor) else _lib.describe(t)) for t in caches]
    return _lib.load().cache_copy(*(d + [None] * 4)[:4], None if pairs is None else ctypes.byref(_lib.describe(pairs)), None)


@cpu_only
def test_copy_entry_refusals():
    t = torch.zeros(2, 6, 32)
    p = lambda src, dst: torch.tensor([src, dst], dtype=torch.int32)  # noqa: E731
    ok = p([0, 1], [2, 3])
    many = list(range(40))
    big = torch.zeros(1, 200, 8)
    for caches, pairs, code in (
        ([], ok, "NULL"),
        ([t], None, "NULL"),
        ([t[0]], ok, "NDIM"),
        ([t, torch.zeros(2, 5, 32)], ok, "SHAPE"),
        ([t], ok.long(), "DTYPE"),
        ([t], torch.zeros(3, 2, dtype=torch.int32), "SHAPE"),
        ([t], torch.zeros(2, 4, dtype=torch.int32)[:, ::2], "STRIDE"),
        ([torch.zeros(2, 32, 6).transpose(1, 2)], ok, "STRIDE"),
        ([t], p([0, 6], [2, 3]), "RANGE"),
        ([t], p([0, 1], [2, -1]), "RANGE"),
        ([t], p([0, 1], [2, 2]), "ARG"),
        ([t], p([0, 1], [1, 2]), "ARG"),
        ([t], p([3], [3]), "ARG"),
        ([big], p(many, [50 + i for i in many[:-1]] + [50]), "ARG"),
        ([big], p(many, [39 + i for i in many]), "ARG"),
        ([big], p(many, [161 + i for i in many]), "RANGE"),
    ):
        assert call(caches, pairs) == ERR[code], (code, pairs)
    huge = _lib.describe(t)
    huge.shape[0] = 2**31
    huge.stride[0] = 0
    assert call([huge], ok) == ERR["RANGE"]
    assert call([t], torch.zeros(2, 0, dtype=torch.int32)) == 0
    assert call([torch.zeros(0, 6, 32)], ok) == 0


def test_copy_python_refusals():
    t = torch.zeros(2, 6, 32)
    for args, match in ((([], [0], [1]), "no caches"), ((t, [0], [1]), "GPU tensors")):
        with pytest.raises(ValueError, match=match):
            cache_copy(*args)
    from myvllm_amd.cache import _pairs
    with pytest.raises(ValueError, match="2 sources for 1"):
        _pairs([0, 1], [2])
    with pytest.raises(ValueError, match="outside"):
        _pairs([2**31], [1])
    assert _pairs(torch.tensor([4, 5]), [6, 7]).tolist() == [[4, 5], [6, 7]]
    assert _pairs([], []).shape == (2, 0)


@cpu_only
def test_copy_of_overlapping_blocks():
    """Blocks that share memory are refused (their copies would race); any order of layers and blocks is not."""
    w = torch.zeros(4000)
    none = torch.zeros(2, 0, dtype=torch.int32)
    pairs = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    for size, stride in (((2, 6, 32), (192, 0, 1)), ((2, 6, 32), (0, 32, 1)), ((1, 6, 32), (0, 31, 1)),
                         ((2, 6, 32), (191, 32, 1)), ((3, 6, 32), (32, 95, 1)), ((2, 6, 32), (31, 64, 1)), ((2, 2, 32), (32, 32, 1))):
        t = w.as_strided(size, stride)
        assert call([t], none) == call([t], pairs) == ERR["STRIDE"], stride
        assert call([torch.zeros(2, size[1], 32), t], none) == ERR["STRIDE"]
    for size, stride in (((2, 6, 32), (192, 32, 1)), ((2, 6, 32), (32, 64, 1)), ((1, 6, 32), (0, 32, 1)),
                         ((3, 1, 32), (40, 0, 1)), ((2, 6, 32), (32, 70, 1)), ((2, 6, 0), (0, 0, 1)), ((1, 1, 32), (0, 0, 1))):
        assert call([w.as_strided(size, stride)], none) == 0, stride
