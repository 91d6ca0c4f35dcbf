"""GPU: NaN among queries, keys and values.  A row is NaN where one of the scores that it
sees is, and in the dims of a value that it sees: whatever the splits, the other sequences
of the batch and the kernel that a call goes by.  All other rows are as without it."""
import pytest
import torch

import myvllm_amd as ops
from attention_bounds import assert_within
from myvllm_amd import _lib
from oracle.fp4 import cache_values
from test_gpu_fp4_attention import decode, is_few, make, prefill, reference

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
NAN = float("nan")
SHAPES = [(16, 2, 256, BF), (8, 4, 128, HF), (4, 4, 64, BF)]
SPLITS = (None, 1, 2, 9, 64)


def set_nan(c, x, n, j, h, blocks=slice(None)):
    """The scales of key or value j (slices too) of sequence n, kv head h."""
    page = c["kc"].shape[1]
    for i in range(*j.indices(int(c["ctx"][n]))) if isinstance(j, slice) else [j]:
        c[x + "s"][int(c["tab"][n, i // page]), h, blocks, i % page] = 255


def check(o, clean, bound, nan):
    """NaN where `nan` says so, else as the clean result."""
    o = o.cpu()
    assert o[nan].isnan().all()
    assert_within(torch.where(nan, 0.0, o.double()), torch.where(nan, 0.0, clean), bound)


@pytest.mark.parametrize("Hq, Hkv, D, dtype", SHAPES)
def test_decode_fp4(dev, Hq, Hkv, D, dtype):
    """A NaN query; one whole sequence of NaN keys; a NaN key alone in the last group of 16
    keys, and in a unit of its own; a NaN value far below the others' weights."""
    R, ctx = Hq // Hkv, [700, 16 * 30 + 1, 2000, 33, 1]
    new = [1] * len(ctx)
    for kind in ("q", "all keys", "last key", "value"):
        print(f"fp4 decode NaN {kind} {Hq}/{Hkv}x{D}", flush=True)
        c = make(ctx, new, Hq, Hkv, D, dtype=dtype, seed=D)
        if kind == "value":  # (head 1 of sequence 2: its first 64 keys weigh less than 2^-149 of the others)
            c["q"][2].fill_(-20.0)
            codes = c["tab"][2, :4].long()
            c["kc"][codes, :, 1] = 0x77  # 6
            c["ks"][codes, 1] = 127
            for b in c["tab"][2, 4:].tolist():
                if b >= 0:
                    c["kc"][b, :, 1], c["ks"][b, 1] = 0, 127
        ref, bound = reference(c, new, D**-0.5)
        nan = torch.zeros(ref.shape, dtype=torch.bool)
        if kind == "q":
            for n, h in ((0, 0), (1, Hq - 1), (2, 1), (4, 0)):
                c["q"][n, h, 3 * n] = NAN
                nan[n, h] = True
        elif kind == "all keys":
            for n, h in ((0, 1), (2, 0), (3, 1)):
                set_nan(c, "k", n, slice(None), h, 1)
                nan[n, h * R:(h + 1) * R] = True
        elif kind == "last key":
            for n, h in ((1, 0), (2, 1), (3, 0)):
                set_nan(c, "k", n, ctx[n] - 1, h, 0)
                nan[n, h * R:(h + 1) * R] = True
        else:
            set_nan(c, "v", 2, 5, 1, 1)
            nan[2, R:2 * R, 32:64] = True
        for splits in SPLITS:
            check(decode(c, dev, D**-0.5, splits), ref, bound, nan)


@pytest.mark.parametrize("Hq, Hkv, D, dtype", SHAPES)
def test_decode(dev, Hq, Hkv, D, dtype):
    """The same over 16-bit caches."""
    R, ctx, page = Hq // Hkv, [700, 16 * 30 + 1, 2000, 33, 1], 16
    c = make(ctx, [1] * 5, Hq, Hkv, D, dtype=dtype, seed=D, stale=False)
    kc, vc = (cache_values(c[x + "c"], c[x + "s"]).to(dtype) for x in "kv")
    ref, bound = reference(c, [1] * 5, D**-0.5)
    nan = torch.zeros(ref.shape, dtype=torch.bool)
    q = c["q"].clone()
    q[0, 0, 5], nan[0, 0] = NAN, True
    for n, h, keys in ((2, 1, range(2000)), (1, 0, [480]), (3, 1, [32])):
        for j in keys:
            kc[int(c["tab"][n, j // page]), j % page, h, 7] = NAN
        nan[n, h * R:(h + 1) * R] = True
    vc[int(c["tab"][0, 3]), 4, 1, 9] = NAN
    nan[0, R:2 * R, 9] = True
    d = [t.to(dev) for t in (q, kc, vc, c["tab"], c["ctx"])]
    for splits in SPLITS:
        print(f"decode NaN {Hq}/{Hkv}x{D} splits {splits}", flush=True)
        o = ops.paged_flash_attention_decode(*d, D**-0.5, page, num_splits=splits)
        torch.cuda.synchronize()
        check(o, ref, bound, nan)


@pytest.mark.parametrize("Hq, Hkv, D, dtype", SHAPES)
@pytest.mark.parametrize("few", [True, False])
def test_prefill_fp4(dev, Hq, Hkv, D, dtype, few):
    """NaN queries and keys in a prefill over 4-bit caches, of a few tokens and in tiles, split and not: a key
    makes the rows NaN that see it."""
    R = Hq // Hkv
    new = [3, 1, 0, 4] if few else [70, 1, 0, 130]
    ctx = [700, 481, 20, 3000] if few else [700, 481, 20, 130]
    c = make(ctx, new, Hq, Hkv, D, dtype=dtype, seed=D)
    assert is_few(c, max(new)) == few
    ref, bound = reference(c, new, D**-0.5)
    nan = torch.zeros(ref.shape, dtype=torch.bool)
    at = [0, new[0], new[0] + new[1], new[0] + new[1], sum(new)]
    c["q"][1, 0, 3], nan[1, 0] = NAN, True
    set_nan(c, "k", 1, 480, 0, 0)  # alone in its group of 16
    nan[at[1], :R] = True
    if few:
        set_nan(c, "k", 3, slice(0, 2000), 1, 1)  # whole units without another key
        nan[at[3]:at[4], R:2 * R] = True
    set_nan(c, "k", 3, ctx[3] - 2, 0, 0)  # the two last queries see it
    nan[at[4] - 2:at[4], :R] = True
    print(f"fp4 prefill NaN {Hq}/{Hkv}x{D} few {few}", flush=True)
    check(prefill(c, dev, D**-0.5), ref, bound, nan)


@pytest.mark.parametrize("Hq, Hkv, D, dtype", SHAPES)
@pytest.mark.parametrize("new, ctx", [([4, 3, 1, 0, 4], [700, 35, 481, 20, 4]), ([70, 3, 130, 0, 33], [700, 35, 130, 20, 4000]),
                                      ([2, 9, 70], [4000, 2001, 1500])])
def test_values_that_only_later_queries_see(dev, Hq, Hkv, D, dtype, new, ctx):
    """NaN among the values of the new tokens: rows before them are as without it (a weight of 0 would not keep it
    out), in the few-tokens form and in tiles, split and not."""
    R, far = Hq // Hkv, len(new) == 3
    c = make(ctx, new, Hq, Hkv, D, dtype=dtype, seed=D, cols=1000 if far else 0)
    few = is_few(c, max(new))
    assert few == (max(new) * R <= 64)
    ref, bound = reference(c, new, D**-0.5)
    nan = torch.zeros(ref.shape, dtype=torch.bool)
    at = [sum(new[:i]) for i in range(len(new) + 1)]

    def bad(n, j, h, blocks):  # key j: the rows from position j on see it
        set_nan(c, "v", n, j, h, blocks)
        row = at[n] + max(0, j - (ctx[n] - new[n]))
        for b in blocks:
            nan[row:at[n + 1], h * R:(h + 1) * R, 32 * b:32 * b + 32] = True

    bad(0, ctx[0] - 1, 0, [0])
    bad(0, ctx[0] - 2, 1, [1])
    bad(1, ctx[1] - 2, 0, range(D // 32))
    bad(1, 7, 1, [0])  # all rows see it
    bad(1, ctx[1] - 1, 1, [0, 1])
    bad(2, ctx[2] - 1, 1, [D // 32 - 1])
    if new[2] > 20:
        bad(2, ctx[2] - 17, 1, [0])
        bad(2, ctx[2] - 33, 0, [0])
        bad(2, ctx[2] - 20, 0, [0, 1])
    if len(new) > 4:
        bad(4, ctx[4] - 1, 0, [1])
        bad(4, ctx[4] - 3, 0, [1])
    print(f"fp4 NaN values {Hq}/{Hkv}x{D} new={new} few={few}", flush=True)
    check(prefill(c, dev, D**-0.5), ref, bound, nan)
    d = {n: t.to(dev) for n, t in c.items()}
    o = torch.empty_like(d["q"])
    _lib.call("paged_attention_prefill_fp4", d["q"], d["kc"], d["vc"], d["ks"], d["vs"], d["tab"], d["ctx"], d["cu"], o,
              None, max(new), D**-0.5)
    check(o, ref, bound, nan)
    for splits in (2, 40):
        ws = torch.empty(_lib.workspace_size("paged_attention_decode_workspace_size", len(new), 4 * Hq, D, splits),
                         device=dev)
        o.fill_(float("inf"))
        _lib.call("paged_attention_few_fp4", d["q"], d["kc"], d["vc"], d["ks"], d["vs"], d["tab"], d["ctx"], d["cu"], o,
                  ws, splits, 4, D**-0.5)
        check(o, ref, bound, nan)


@pytest.mark.parametrize("few", [True, False])
def test_rows_that_see_no_key(dev, few):
    """Queries before position 0 are zero whatever the values, and the stale ones past the length, hold."""
    Hq, Hkv, D = 8, 2, 128
    new, ctx = ([6, 4], [3, 2]) if few else ([60, 40], [33, 2])
    c = make(ctx, new, Hq, Hkv, D)
    assert is_few(c, max(new)) == few
    set_nan(c, "v", 0, slice(None), 0)
    set_nan(c, "v", 1, 1, 1)
    o = prefill(c, dev, 0.1).cpu()
    a, b = new[0] - ctx[0], new[0] + new[1] - ctx[1]
    assert not o[:a].any() and o[a:new[0], :4].isnan().all() and not o[a:new[0], 4:].isnan().any()
    assert not o[new[0]:b].any() and not o[b:, :4].isnan().any() and not o[b, 4:].isnan().any()
    assert o[b + 1, 4:].isnan().all()


@pytest.mark.parametrize("Hq, Hkv, D, dtype", SHAPES)
def test_other_forms(dev, Hq, Hkv, D, dtype):
    """Capped and biased scores, sequences that share their first keys, a split prefill: over 16-bit caches."""
    R, page = Hq // Hkv, 16
    ctx = [700, 16 * 30 + 1, 2000, 33, 1]
    c = make(ctx, [1] * 5, Hq, Hkv, D, dtype=dtype, seed=D, stale=False)
    kc, vc = (cache_values(c[x + "c"], c[x + "s"]).to(dtype) for x in "kv")
    q = c["q"].clone()
    nan = torch.zeros(q.shape, dtype=torch.bool)
    q[0, 0, 5], nan[0, 0] = NAN, True
    for n, h, keys in ((2, 1, range(2000)), (1, 0, [480]), (3, 1, [32])):
        for j in keys:
            kc[int(c["tab"][n, j // page]), j % page, h, 7] = NAN
        nan[n, h * R:(h + 1) * R] = True
    d = [t.to(dev) for t in (q, kc, vc, c["tab"], c["ctx"])]
    for kw in (dict(softcap=20.0), dict(alibi_slopes=torch.full((Hq,), 0.01, device=dev))):
        for splits in SPLITS:
            o = ops.paged_flash_attention_decode(*d, D**-0.5, page, num_splits=splits, **kw).cpu()
            assert o[nan].isnan().all() and not o[~nan].isnan().any(), (kw, splits)
    cu = torch.arange(6, dtype=torch.int32, device=dev)
    o = ops.paged_flash_attention_prefill(*d, cu, None, D**-0.5, page).cpu()
    assert o[nan].isnan().all() and not o[~nan].isnan().any()
    # four sequences that share 32 keys; the last one's own keys of head 1 are all NaN
    tab = torch.full((4, 20), -1, dtype=torch.int32)
    tab[:, :2] = c["tab"][0, :2]
    tab[0, 2:20], tab[1, 2:20], tab[2, 2:4], tab[3, 2:20] = (c["tab"][2, a:b] for a, b in ((4, 22), (24, 42), (44, 46), (48, 66)))
    k = cache_values(c["kc"], c["ks"]).to(dtype)
    k[tab[3, 2:].long(), :, 1, 3] = NAN
    q = c["q"][:4].clone()
    q[1, 2, 9] = NAN
    nan = torch.zeros(q.shape, dtype=torch.bool)
    nan[1, 2], nan[3, R:2 * R] = True, True
    lens = torch.tensor([320, 300, 50, 311], dtype=torch.int32)
    o = ops.paged_flash_attention_decode_shared(q.to(dev), k.to(dev), d[2], tab.to(dev), lens.to(dev),
                                                torch.tensor([32], dtype=torch.int32, device=dev), D**-0.5, page).cpu()
    assert o[nan].isnan().all() and not o[~nan].isnan().any()
