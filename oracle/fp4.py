"""CPU restatement of caches held in 4 bits and of the append with rotary
positions of several axes (no counterpart in the reference), in float64."""
from __future__ import annotations

import torch

from .attention import rotate_ref

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TOP = {torch.bfloat16: 125, torch.float16: 13}  # largest exponent of a scale


def pack_ref(x):
    """Rows x (..., D), bf16 or fp16, as codes (..., D / 2) and scale bytes
    (..., D / 32): by trying exponents and all eight magnitudes of each number."""
    y = x.double().unflatten(-1, (-1, 32))
    top = TOP[x.dtype]
    finite = torch.isfinite(y).all(-1)
    y = torch.where(finite[..., None], y, 0.0)
    most = y.abs().amax(-1)
    e = torch.full(most.shape, top, dtype=torch.int64)
    for k in range(top - 1, -top - 1, -1):
        e = torch.where(most <= 6 * 2.0**k, k, e)
    z = y / 2.0 ** e.double()[..., None]
    far = (z.abs().clamp(max=6.0)[..., None] - torch.tensor(GRID, dtype=torch.float64)).abs()
    near = far.amin(-1, keepdim=True)
    # of two as near, the even code: odd ones count as a little further
    code = (far + torch.arange(8) % 2 * 2.0**-60 * (far == near)).argmin(-1)
    tie = (far == near).sum(-1) == 2
    first = (far == near).int().argmax(-1)
    code = torch.where(tie, first + first % 2, code)
    code = code + 8 * torch.signbit(z)
    code = torch.where(finite[..., None], code, 0).flatten(-2)
    byte = torch.where(finite, e + 127, 255)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), byte.to(torch.uint8)


def unpack_ref(codes, scales):
    """The numbers, float64, of codes (..., D / 2) and scale bytes (..., D / 32)."""
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2).long()
    v = torch.tensor(GRID, dtype=torch.float64)[c % 8] * (1 - 2 * (c // 8))
    s = torch.where(scales == 255, float("nan"), 2.0 ** (scales.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def cache_values(codes, scales):
    """Codes (blocks, page, H, D / 2) and scales (blocks, H, D / 32, page) as (blocks, page, H, D)."""
    return unpack_ref(codes, scales.permute(0, 3, 1, 2))


def axis_of(sections, dealt):
    """The axis of each frequency."""
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    order = sorted((turn, a) for a, n in enumerate(sections) for turn in range(n))
    return [a for _, a in order]


def append_ref(q, k, v, block_tables, context_lens, cu_seqlens, page, num_blocks, cos=None, sin=None, interleaved=False,
               positions=None, sections=None, dealt=False):
    """Rows of the append: q rotated (fp64, zero where a token has no place; None
    for None), k rotated (fp64) and v, and for every token that is written
    (token, block, slot)."""
    T = k.shape[0]
    cu = list(range(T + 1)) if cu_seqlens is None else [int(c) for c in cu_seqlens]
    turn_q = torch.zeros(q.shape, dtype=torch.float64) if q is not None else None
    turn_k = k.double().clone()
    half = 0 if cos is None else cos.shape[1]
    if positions is not None:
        positions = positions.view(-1, T)
        of = axis_of(sections or [half], dealt)
    places = []
    for n in range(block_tables.shape[0]):
        for t in range(cu[n], cu[n + 1]):
            p = int(context_lens[n]) - cu[n + 1] + t
            ok = 0 <= p < block_tables.shape[1] * page
            if positions is not None:
                turns = [int(x) for x in positions[:, t]]
                ok = ok and all(0 <= x < cos.shape[0] for x in turns)
            elif cos is not None:
                turns, of = [p], [0] * half
                ok = ok and p < cos.shape[0]
            if not ok:
                continue
            if cos is not None:
                at = [turns[a] for a in of]
                c, s = cos[at, range(half)][None], sin[at, range(half)][None]
                turn = lambda x: rotate_ref(x[t:t + 1], c, s, interleaved)[0]  # noqa: E731
            else:
                turn = lambda x: x[t].double()  # noqa: E731
            if q is not None:
                turn_q[t] = turn(q)
            turn_k[t] = turn(k)
            b = int(block_tables[n, p // page])
            if 0 <= b < num_blocks:
                places.append((t, b, p % page))
    return turn_q, turn_k, v, places
