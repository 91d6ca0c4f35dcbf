"""Reference and elementwise error bound of the attention kernels, derived.

With weights p, their errors: the score in fp32 is off by at most dx = D 2^-24
scale |q|.|k| (the dot product), 3e-7 softcap (the tanh by exp2 and reciprocal,
each within an ulp, and its sums), and 2^-22 of the magnitudes that are added
and multiplied in fp32 (x, the bias); p then by 2 dx relative (and its share in
the sum, once more), plus half a step of p's 16-bit rounding, eps / 2, and for
fp16 half the subnormal step, 2^-25 (the sum is at least 1 in p's units).  The
result is rounded once more, eps / 2; fp32 sums and merges are within 2^-18.
"""
import torch

from oracle.attention import attention_weights_ref


def ref_and_bound(q, k, v, pos, scale, dtype, causal=True, softcap=None, slopes=None, prefix=0):
    """q (n, Hq, D) at pos over keys k, v (m, Hkv, D): result and bound, fp64."""
    r = q.shape[1] // k.shape[1]
    n, m = q.shape[0], k.shape[0]
    if m == 0:
        return torch.zeros(n, *q.shape[1:], dtype=torch.float64), torch.zeros(n, *q.shape[1:], dtype=torch.float64)
    x, p = attention_weights_ref(q, k, pos, scale, causal, softcap, slopes, prefix)
    vr = v.double().repeat_interleave(r, 1)
    mix = lambda w, u: torch.einsum("nhm,mhd->nhd", w, u)  # noqa: E731
    o, big = mix(p, vr), mix(p, vr.abs())
    dots = torch.einsum("nhd,mhd->nhm", q.double().abs(), k.double().abs().repeat_interleave(r, 1)) * abs(scale)
    dx = q.shape[2] * 2.0**-24 * dots + 3e-7 * (softcap or 0) + 2.0**-22 * (1 + x.abs().clamp(max=1e30))
    if slopes is not None:
        far = (torch.as_tensor(pos)[:, None] - torch.arange(m)).abs()
        dx = dx + 2.0**-22 * slopes.double().abs()[None, :, None] * far[:, None]
    half = torch.finfo(dtype).eps / 2
    pd = torch.where(p > 0, p * dx, 0.0)
    bound = half * (big + o.abs()) * (1 + 2.0**-6) + 2 * (mix(pd, vr.abs()) + big * pd.sum(-1, keepdim=True)) \
        + 2.0**-18 * big
    if dtype == torch.float16:
        seen = torch.isfinite(x).double()
        bound = bound + 2.0**-25 * (mix(seen, vr.abs()) + seen.sum(-1, keepdim=True) * o.abs() + 1)
    return o, bound


def assert_within(got, ref, bound, what=""):
    got = got.double().cpu()
    assert got.shape == ref.shape
    err = (got - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())}/{bad.numel()} off, worst {(err / bound.clamp_min(1e-300)).max():.2f} x"
