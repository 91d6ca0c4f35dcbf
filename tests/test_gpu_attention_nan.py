"""GPU: NaN among queries, keys and values.  A row is NaN where one of the scores that it
sees is, and in the dims of a value that it sees: whatever the splits, the other sequences
of the batch and the kernel that a call goes by.  All other rows are as without it."""
import pytest
import torch

import myvllm_amd as ops
from attention_bounds import assert_within
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
