"""GPU: the plan of the shared decode at its limits -- more groups than threads,
more row blocks than pieces fit, prefixes of up to 2^30 keys."""
import pytest
import torch

from myvllm_amd import paged_flash_attention_decode_shared
from test_gpu_attention_shared import check, make

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("G, every, own", [
    (300, 7, [2, 0, 5]),  # 43 groups of three sequences, the others empty: past the 256 threads of small batches
    (1100, 1, [3]),  # groups of one, which share nothing, past the 1,024 of large ones
    (1100, 2, [1, 4]),
    (2100, 6, [0, 9]),
    (600, 200, [1] * 20),  # three groups, far apart
])
def test_many_groups(dev, G, every, own):
    groups = [(20 + g % 50, own if g % every == every - 1 else []) for g in range(G)]
    c, cu = make(groups, 4, 2, 64, seed=G)
    B = len(c["q"])
    print(f"shared decode of {B} sequences in {G} groups", flush=True)
    check(dev, c, cu, rows=sorted({*range(0, B, 23), B - 1}))


@pytest.mark.parametrize("keys", [40, 2000])
def test_more_row_blocks_than_room_for_pieces(dev, keys):
    """2,048 blocks of 128 rows, where the workspace holds one piece of each."""
    c, cu = make([(keys, [1 + b % 3 for b in range(8192)])], 32, 1, 256, seed=1)
    print(f"shared decode of 2,048 row blocks, {keys} keys", flush=True)
    check(dev, c, cu, rows=[0, 1, 4000, 4095, 4096, 8190, 8191], plain=False)


@pytest.mark.parametrize("keys", [2**20 + 3, 2**24 + 33, 3 * 2**25, 2**30 - 16])
def test_long_prefixes(dev, keys):
    """Tables that repeat one page of zero keys, with 16 pages of other keys put
    into the shared part, the first, the last and some between; query row i scores
    60 at the i-th and 0 at every other key, so it returns that page's mean (the
    others together weigh 2^30 e^-60, below 1e-16)."""
    g = torch.Generator().manual_seed(keys & 0xffff)
    cols = -(-keys // 16) + 1
    kc, vc = torch.zeros(19, 16, 1, 64, dtype=BF), torch.randn(19, 16, 1, 64, generator=g).to(BF)
    for i in range(16):
        kc[i, :, 0, i] = 1.0
    row = torch.full((cols,), 16, dtype=torch.int32, device=dev)
    row[-1] = 17  # the sequences' own keys
    at = torch.randint(1, keys // 16 - 1, (16,), generator=g)
    at[0], at[1] = 0, keys // 16 - 1
    row[at.to(dev)] = torch.arange(16, dtype=torch.int32, device=dev)
    assert torch.unique(at).numel() == 16
    q = torch.zeros(4, 4, 64, dtype=BF)
    for i in range(16):
        q[i // 4, i % 4, i] = 60.0
    ctx = torch.full((4,), 16 * cols, dtype=torch.int32, device=dev)
    print(f"shared decode behind {keys} keys", flush=True)
    got = paged_flash_attention_decode_shared(q.to(dev), kc.to(dev), vc.to(dev), row.expand(4, cols), ctx,
                                              torch.tensor([keys], dtype=torch.int32, device=dev), 1.0, 16)
    v = vc[:16, :, 0].double()
    # half a step of P and of the result, and fp32 sums
    bound = 2**-8 * (v.abs().mean(1) + v.mean(1).abs()) * 1.02
    err = (got.double().cpu().view(16, 64) - v.mean(1)).abs()
    assert (err <= bound).all(), f"rows {(err > bound).any(1).nonzero().flatten().tolist()}"
