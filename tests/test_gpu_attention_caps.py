"""GPU: capped attention at D = 64 over all scales and caps, against float64
(tests/attention_bounds.py derives the bound)."""
import pytest
import torch

from attention_bounds import assert_within, ref_and_bound
from myvllm_amd import flash_attention_prefill, paged_flash_attention_decode, paged_flash_attention_prefill

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


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


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("ratio", [1e-1, 1e-4, 2e-5, 1e-6, 1e-9, 1e-14])
def test_small_scales_at_64_dims(dev, ratio, paged):
    """scale / cap down to 1e-14, q and k so large that the scores are spread to
    3/4 of the cap and past it; a polynomial in powers of the ratio would lose
    its high terms (0.06 of the cap at 3/4 without those past the third)."""
    cap = 8.0
    std = (0.3 / (ratio * 8)) ** 0.5  # scale q.k / cap has a standard deviation of 0.3 (8: the root of 64 dims)
    q, k, v = normal(1, 96, 4, 64, std=std), normal(2, 96, 2, 64, std=std), normal(3, 96, 2, 64)
    print(f"scale / cap = {ratio} paged={paged}", flush=True)
    got = run(dev, q, k, v, ratio * cap, paged=paged, softcap=cap)
    ref, bound = ref_and_bound(q, k, v, torch.arange(96), ratio * cap, BF, softcap=cap)
    assert_within(got, ref, bound)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale, cap, at", [(1 / 16, 4096.0, 0.68), (0.125, 4096.0, 0.6), (0.01, 1000.0, 0.68),
                                            (1 / 64, 1000.0, 0.65), (1.0, 50.0, 0.68),
                                            (1e-7, 0.125, 0.68), (1e-12, 8.0, 0.65)])
def test_tiles_near_the_cap_and_past_it(dev, scale, cap, at, dtype):
    """Query 0 scores the same at every key, `at` times the cap before it is
    capped, so its result is the mean of the values; in the second tile of keys
    query 1 scores past the range that the polynomial covers, so that the tile
    goes through the exponential: the two have to agree."""
    q, k = torch.zeros(128, 1, 64), torch.zeros(128, 1, 64)
    x = at * cap / scale / 64  # (query 0's share of each dim's product)
    # dims 0..31 of both queries; dim 63 only query 1's, and only of a key of the second half
    q[:2, 0, :32], k[:, 0, :32] = round((2 * x) ** 0.5), round((2 * x) ** 0.5)
    q[1, 0, 63], k[100, 0, 63] = round((20 * x) ** 0.5), round((20 * x) ** 0.5)
    if scale < 1e-3 and dtype == HF:
        pytest.skip("products past fp16's range")
    q, k = q.to(dtype), k.to(dtype)
    v = torch.cat([torch.ones(64, 1, 64), -torch.ones(64, 1, 64)]).to(dtype)
    print(f"scale={scale} cap={cap} at={at} {dtype}", flush=True)
    got = run(dev, q, k, v, scale, causal=False, softcap=cap)
    ref, bound = ref_and_bound(q, k, v, torch.arange(128), scale, dtype, causal=False, softcap=cap)
    assert 0.5 < float(scale * (q[0, 0].double() @ k[0, 0].double())) / cap < 0.75
    assert_within(got[:1], ref[:1], bound[:1])


@pytest.mark.parametrize("scale", [1e-3, 0.05, 1.0, 4.0])
@pytest.mark.parametrize("cap", [1e-3, 0.3, 30.0, 1000.0, 4096.0])
def test_caps_and_scales_at_64_dims(dev, cap, scale):
    """Over the accepted caps, with scores spread over +- 3/4 of the cap."""
    std = min((0.3 * cap / scale / 8) ** 0.5, 1e3)
    q, k, v = normal(4, 70, 2, 64, std=std), normal(5, 70, 1, 64, std=std), normal(6, 70, 1, 64)
    print(f"cap={cap} scale={scale}", flush=True)
    got = run(dev, q, k, v, scale, softcap=cap)
    ref, bound = ref_and_bound(q, k, v, torch.arange(70), scale, BF, softcap=cap)
    assert_within(got, ref, bound)


@pytest.mark.parametrize("scale", [1e36, -1e38])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scales_past_the_cap(dev, D, scale):
    """scale / cap past fp32's range: a score of exactly 0 stays 0, every other one
    is at the cap's end."""
    q, k, v = normal(12, 64, 4, D), normal(13, 64, 2, D), normal(14, 64, 2, D)
    q[::2] = 0
    print(f"scale={scale} D={D}", flush=True)
    tab = torch.arange(4, dtype=torch.int32, device=dev)[None]
    kc, vc = (t.to(dev).reshape(4, 16, 2, D) for t in (k, v))
    none = (q == 0).all(-1, keepdim=True)
    for cap in (1e-3, 2.0):
        got = run(dev, q, k, v, scale, softcap=cap)
        flat, big = ref_and_bound(q, k, v, torch.arange(64), 0.0, BF)
        assert_within(torch.where(none.to(dev), got, 0), torch.where(none, flat, 0.0), torch.where(none, big, 0.0))
        assert torch.isfinite(got).all()
        ctx = torch.tensor([64], dtype=torch.int32, device=dev)
        one = paged_flash_attention_decode(q[:1].to(dev), kc, vc, tab, ctx, scale, 16, softcap=cap)
        mean = v.double().mean(0).repeat_interleave(2, 0)[None]
        assert_within(one, mean, 2**-7 * v.double().abs().mean(0).repeat_interleave(2, 0)[None])
