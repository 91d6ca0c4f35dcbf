"""CPU: the capped score's stated accuracy, from the constants in the source: the
steps of attention_common.h in float32 against float64."""
import pathlib
import re

import numpy as np

ROOT = pathlib.Path(__file__).parent.parent
F = np.float32


def stated():
    """In units of the cap."""
    return float(re.search(r"the tanh is within (\S+) softcap", (ROOT / "include/gdn_hip.h").read_text())[1])


def fma(a, b, c):
    return F(np.float64(a) * np.float64(b) + np.float64(c))  # (the product of two float32 is exact in float64)


def test_near_scores():
    """tanh(x) / 2 - 1 / 2 by the polynomial, for every x that it is used at."""
    src = (ROOT / "myvllm_amd/csrc/attention_common.h").read_text()
    src = src[src.index("struct CapNear"):]
    src = src[:src.index("};")]
    lim = F(re.search(r"\? ([\d.]+)f / h", src)[1])
    coef = [F(0.5) * F(c) for c in re.findall(r"0\.5f \* (-?[\d.]+)f", src)]
    assert len(coef) == 5
    x = np.concatenate([np.linspace(-lim, lim, 1_000_001), np.logspace(-30, 0, 10_001) * lim]).astype(F)
    u = x * x
    p = np.full_like(x, coef[0])
    for c in coef[1:]:
        p = fma(p, u, c)
    y = fma(x, p, F(-0.5))
    err = np.abs(2 * (y.astype(np.float64) + 0.5) - np.tanh(x.astype(np.float64)))
    assert err.max() <= stated(), err.max()


def test_exponential():
    """1 - 2 / (1 + e): e and the quotient within an ulp each, the sum rounded."""
    x = np.linspace(-12, 12, 200_001)
    e = np.exp(2 * x)
    y = 1 / (1 + e)
    ulp = lambda v: 2.0 ** (np.floor(np.log2(v)) - 23)  # noqa: E731
    err = ulp(e) / (1 + e) ** 2 + ulp(1 + e) / 2 / (1 + e) ** 2 + ulp(y)
    assert 2 * err.max() <= stated(), 2 * err.max()
