"""GPU: scored attention over values far from 1, against float64
(tests/attention_bounds.py derives the bound)."""
import pytest
import torch

from attention_bounds import assert_within, ref_and_bound
from myvllm_amd import flash_attention_prefill, paged_flash_attention_prefill

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def run(dev, q, k, v, scale, causal=True, paged=False, **kw):
    """One sequence; paged: its keys in pages of 16 (a whole number of them)."""
    (T, Hq, D), (L, Hkv, _) = q.shape, k.shape
    q, k, v = q.to(dev), k.to(dev), v.to(dev)
    if paged:
        kc, vc = (t.reshape(-1, 16, Hkv, D) for t in (k, v))
        tab = torch.arange(len(kc), dtype=torch.int32, device=dev)[None]
        return paged_flash_attention_prefill(q, kc, vc, tab, torch.tensor([L], dtype=torch.int32, device=dev),
                                             torch.tensor([0, T], dtype=torch.int32, device=dev), None, scale, 16, **kw)
    return flash_attention_prefill(q, k, v, torch.tensor([0, T], dtype=torch.int32, device=dev), scale, Hq, Hkv, D, D,
                                   causal, **kw)


def normal(seed, *shape, std=1.0, dtype=BF):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


@pytest.mark.parametrize("size", [1e-26, 1e33])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_values_far_from_one(dev, D, paged, size):
    """bf16 values of 1e-26 and of 1e33 behind slopes of 0.7 to 0.004: the base
    of the softmax must not run so far from the maximum that the products leave
    fp32's range."""
    slopes = 2.0 ** (-torch.arange(1.0, 9.0)) * 1.4
    q, k, v = normal(7, 320, 8, D), normal(8, 320, 2, D), normal(9, 320, 2, D, std=size)
    print(f"values of {size} D={D} paged={paged}", flush=True)
    got = run(dev, q, k, v, D**-0.5, paged=paged, alibi_slopes=slopes.to(dev))
    ref, bound = ref_and_bound(q, k, v, torch.arange(320), D**-0.5, BF, slopes=slopes)
    assert_within(got, ref, bound)


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_values_and_rising_capped_scores(dev, D, paged):
    """Scores that rise by 14 from key tile to key tile, capped, over values of
    1e33: a base that trails by 2^20 would overflow where the plain op does not."""
    q, k = torch.zeros(4 if paged else 256, 2, D), torch.zeros(256, 1, D)
    q[..., 0] = 1.0
    k[:, 0, 0] = 7.0 * (torch.arange(256) // 64)
    q, k, v = q.to(BF), k.to(BF), normal(11, 256, 1, D, std=1e33)
    print(f"rising scores D={D} paged={paged}", flush=True)
    every = dict(prefix_lens=torch.tensor([256], dtype=torch.int32, device=dev)) if paged else dict(causal=False)
    got = run(dev, q, k, v, 2.0, paged=paged, softcap=1000.0, **every)
    ref, bound = ref_and_bound(q, k, v, torch.arange(len(q)), 2.0, BF, causal=False, softcap=1000.0)
    assert_within(got, ref, bound)
