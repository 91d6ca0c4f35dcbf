"""Performance cases of paged caches held in 4 bits, of rotary positions with several axes, and
of copies inside the caches.

Each case is one call, or two that follow each other, as a serving program makes it.  Heads,
head dims and pages are those of this repository's attention workloads (16 / 2 heads of 256,
16 / 4 of 128, 16 / 16 of 64, 16-token pages), the state cache that of its Gated DeltaNet
layers, lengths those of its prefill and decode workloads.  ``listed()`` holds the fixed cases,
``draw`` more of the same ranges.  Where ``own`` is false ``run`` computes the operators in plain
float32 torch (keys that are rounded to 4 bits are rotated in float64, next to whose borders
float32 would choose another value now and then); ``exact`` restates them in float64 on its own.

The 4-bit form of a row of D numbers: blocks of 32 share a scale 2^e, e the smallest with
max|x| <= 6 * 2^e, held to the exponents that keep every value a normal number of the 16-bit type
(-125..125 for bf16, -13..13 for fp16); a number is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 times the
scale with a sign, the nearest, of two as near the one with an even code.  Caches hold two codes
a byte (blocks, page, heads, D / 2), the first in the low half, and e + 127 as bytes
(blocks, heads, D / 32, page).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROPE_ROWS = 32768  # positions of the rotation table that a serving program keeps
ROPE_BASE = 10000.0
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EXPONENTS = {torch.bfloat16: 125, torch.float16: 13}


def listed() -> list[dict]:
    return [
        # a decode batch of chats about images: each new token has its time, height and width position
        dict(name="axes_decode_64", kind="axes", seqs=64, lo=1, hi=1, prefix=4096, len_seed=1, hq=16, hkv=2, dim=256,
             rot=64, deal=True, page=16, dtype="bf16"),
        # a prefill batch of prompts with images in them
        dict(name="axes_prefill_8", kind="axes", seqs=8, lo=512, hi=4096, prefix=0, len_seed=2, hq=16, hkv=4, dim=128,
             rot=128, deal=False, page=16, dtype="fp16"),
        # one short prompt put into a 4-bit cache, and its keys and values read back; a latency
        dict(name="append4_17", kind="append4", seqs=1, lo=17, hi=17, prefix=0, len_seed=3, hq=16, hkv=2, dim=256,
             rot=64, page=16, dtype="bf16"),
        # a full prefill batch of ragged prompts into a 4-bit cache, read back as a program that moves it does
        dict(name="append4_16", kind="append4", seqs=16, lo=512, hi=4096, prefix=0, len_seed=4, hq=16, hkv=2, dim=256,
             rot=256, page=16, dtype="bf16"),
        # one user's chat: a decode step over a 4-bit cache; a latency
        dict(name="decode4_1", kind="decode4", seqs=1, lo=2943, hi=2943, len_seed=5, hq=16, hkv=2, dim=256, page=16,
             dtype="bf16"),
        # an ordinary serving batch's decode step
        dict(name="decode4_64", kind="decode4", seqs=64, lo=1024, hi=8192, len_seed=6, hq=16, hkv=2, dim=256, page=16,
             dtype="bf16"),
        # a large batch of long contexts, which the smaller cache makes room for
        dict(name="decode4_256_fp16", kind="decode4", seqs=256, lo=512, hi=16384, len_seed=7, hq=16, hkv=4, dim=128,
             page=16, dtype="fp16"),
        # chunks of long prompts over what is already in the 4-bit cache
        dict(name="prefill4_chunks", kind="prefill4", seqs=4, lo=256, hi=2048, prefix=16384, len_seed=8, hq=16, hkv=2,
             dim=256, page=16, dtype="bf16"),
        # a few tokens each of several sequences that are to be checked at once, heads without groups, odd lengths
        dict(name="prefill4_few", kind="prefill4", seqs=12, lo=3, hi=9, prefix=6000, len_seed=9, hq=16, hkv=16, dim=64,
             page=32, dtype="fp16"),
        # sixteen answers branch off: the last page of each is copied in every layer
        dict(name="copy_fork_16", kind="copy", of="pages", pairs=16, blocks=301, layers=8, hkv=2, dim=256, page=16,
             len_seed=10, dtype="bf16"),
        # the recurrent and conv states of eight sequences that branch off
        dict(name="copy_states_8", kind="copy", of="states", pairs=8, blocks=24, layers=6, len_seed=11, hk=16, hv=32,
             dtype="bf16"),
        # a cache after many requests have ended: the pages in use move to its front
        dict(name="copy_compact", kind="copy", of="pages", pairs=1501, blocks=4001, layers=8, hkv=2, dim=256, page=16,
             len_seed=12, dtype="bf16"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng: random.Random) -> dict:
    """One more case; sizes stay at or below the listed cases'."""
    kind = rng.choice(["axes", "axes_decode", "append4", "append4", "decode4", "decode4", "decode4", "prefill4",
                       "prefill4", "copy"])
    hq, hkv, dim = rng.choice([(16, 2, 256), (16, 2, 256), (8, 1, 256), (16, 4, 128), (16, 16, 64)])
    c = dict(len_seed=rng.randrange(1 << 20), hq=hq, hkv=hkv, dim=dim, page=rng.choice([16, 16, 16, 32, 64]),
             dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "axes_decode":
        return dict(c, kind="axes", seqs=_log(rng, 1, 256), lo=1, hi=1, prefix=_log(rng, 16, 8192),
                    rot=rng.choice([dim, dim // 4]), deal=rng.choice([True, False]))
    if kind in ("axes", "append4"):
        hi = _log(rng, 2, 4096)
        c.update(kind=kind, seqs=max(1, min(_log(rng, 1, 16), 32768 // hi)), lo=max(1, hi // 8), hi=hi, prefix=0,
                 rot=rng.choice([dim, dim // 4]))
        return dict(c, deal=rng.choice([True, False])) if kind == "axes" else c
    if kind == "decode4":
        hi = _log(rng, 64, 16384)
        return dict(c, kind=kind, seqs=max(1, min(_log(rng, 1, 256), 1_000_000 // hi)), lo=max(1, hi // 8), hi=hi)
    if kind == "prefill4":
        hi, prefix = _log(rng, 2, 2048), _log(rng, 64, 16384)
        return dict(c, kind=kind, seqs=max(1, min(_log(rng, 1, 12), 50_000_000 // (hi * (prefix + hi)))),
                    lo=max(1, hi // 8), hi=hi, prefix=prefix)
    layers, c["dtype"] = _log(rng, 1, 8), rng.choice(["bf16", "fp16"])
    if rng.random() < 0.4:
        pairs = _log(rng, 1, 16)
        return dict(kind="copy", of="states", pairs=pairs, blocks=2 * pairs + rng.randint(1, 8), layers=min(layers, 4),
                    len_seed=c["len_seed"], hk=16, hv=rng.choice([16, 32]), dtype=c["dtype"])
    pairs = _log(rng, 1, 1500)
    return dict(kind="copy", of="pages", pairs=pairs, blocks=2 * pairs + rng.randint(1, 900), layers=layers, hkv=hkv,
                dim=dim, page=16, len_seed=c["len_seed"], dtype=c["dtype"])


# ---- sizes ---------------------------------------------------------------------------


def _lengths(c: dict) -> list[int]:
    """New tokens per sequence, or the keys of each (decode)."""
    r = random.Random(c["len_seed"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]


def _contexts(c: dict) -> list[int]:
    """Keys of each sequence once the new ones are in the cache."""
    r = random.Random(c["len_seed"] + 1)
    return [n + (r.randint(c["prefix"] // 2, c["prefix"]) if c.get("prefix") else 0) for n in _lengths(c)]


def _cu(lens: list[int]) -> list[int]:
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _sections(c: dict) -> list[int]:
    """Frequencies of the time, height and width axis."""
    n = c["rot"] // 2
    if c["deal"]:
        return [n - 2 * (n // 3), n // 3, n // 3]
    return [n // 4, 3 * n // 8, n - n // 4 - 3 * n // 8]


def _axis_of(c: dict) -> list[int]:
    """The axis of each frequency: section after section, or dealt to the axes in turn."""
    left = _sections(c)
    if not c["deal"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    of: list[int] = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                of.append(a)
    return of


def _pairs(c: dict) -> tuple[list[int], list[int]]:
    """Blocks copied and where to: the sources lie behind the places, as when a cache is compacted."""
    r = random.Random(c["len_seed"])
    ids = sorted(r.sample(range(c["blocks"]), 2 * c["pairs"]))
    return ids[c["pairs"]:], ids[: c["pairs"]]


# ---- inputs --------------------------------------------------------------------------


def prepare(case: dict, seed: int) -> dict:
    c = case
    dev, dt = torch.device("cuda:0"), DTYPES[c["dtype"]]
    gen, cpu = torch.Generator(device=dev).manual_seed(seed), random.Random(seed)
    normal = lambda *shape, std=1.0: (torch.randn(*shape, generator=gen, device=dev) * std).to(dt)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    kind = c["kind"]
    if kind == "copy":
        s = dict(case=c)
        s["src"], s["dst"] = _pairs(c)  # (what the program's allocator holds)
        s["src_ids"], s["dst_ids"] = (torch.tensor(x, device=dev) for x in (s["src"], s["dst"]))
        if c["of"] == "pages":
            shape = (c["layers"], c["blocks"], c["page"], c["hkv"], c["dim"])
            s["caches"] = [normal(*shape), normal(*shape)]
        else:
            s["caches"] = [normal(c["layers"], c["blocks"], 3, 256 * c["hk"] + 128 * c["hv"]),
                           torch.randn(c["layers"], c["blocks"], c["hv"], 128, 128, generator=gen, device=dev)]
        return s
    hq, hkv, D, page = c["hq"], c["hkv"], c["dim"], c["page"]
    lens = _lengths(c)
    T = c["seqs"] if kind == "decode4" else sum(lens)
    # scores of a few units, as after the q and k norms of a trained layer
    s = dict(q=normal(T, hq, D, std=1.0 if kind in ("axes", "append4") else 2.0), scale=D ** -0.5, case=c,
             longest=max(lens))
    ctx = lens if kind == "decode4" else _contexts(c)
    if kind == "prefill4" or c["hi"] > 1 and kind != "decode4":
        s["cu"] = ints(_cu(lens))
    pages = [-(-n // page) for n in ctx]
    total = sum(pages) + 3
    order = list(range(total))
    cpu.shuffle(order)
    rows, at = [], 0
    for p in pages:
        rows.append(order[at: at + p])
        at += p
    s["tables"] = ints([r + [-1] * (max(pages) - len(r)) for r in rows])
    s["ctx"] = ints(ctx)
    if kind in ("axes", "append4"):
        s["k"], s["v"] = normal(T, hkv, D), normal(T, hkv, D)
        f = ROPE_BASE ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=dev) / c["rot"])
        a = torch.arange(ROPE_ROWS, dtype=torch.float64, device=dev)[:, None] * f
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
    if kind == "axes":
        s["k_cache"], s["v_cache"] = normal(total, page, hkv, D), normal(total, page, hkv, D)
        s["positions"] = _positions(lens, ctx, cpu, dev)
        return s
    for x in ("k", "v"):
        codes = torch.zeros(total, page, hkv, D // 2, dtype=torch.uint8, device=dev)
        scales = torch.zeros(total, hkv, D // 32, page, dtype=torch.uint8, device=dev)
        if kind != "append4":
            step = max(1, (1 << 26) // (page * hkv * D))
            for b in range(0, total, step):
                n = min(step, total - b)
                codes[b: b + n], e = _pack(normal(n, page, hkv, D))
                scales[b: b + n] = e.permute(0, 2, 3, 1)
        s[x + "_cache"], s[x + "_scales"] = codes, scales
    return s


def _positions(lens, ctx, cpu, dev):
    """(3, T): words share one position on all axes; an image's patches share a time and lie on a grid."""
    parts = []
    for n, m in zip(lens, ctx):
        t = torch.arange(n)
        text = n // 4 if n > 8 else n
        wide = max(1, int(math.sqrt(max(1, n // 2)))) + cpu.randint(0, 3)
        image = torch.stack([torch.full_like(t, text), text + (t - text) // wide, text + (t - text) % wide])
        p = torch.where((t >= text) & (t < text + n // 2), image, t.expand(3, n))
        parts.append(p + (m - n))
    return torch.cat(parts, 1).to(torch.int32).to(dev)


# ---- one pass ------------------------------------------------------------------------


def run(s: dict):
    c = s["case"]
    if own:
        return _run_own(s, c)
    kind = c["kind"]
    if kind == "copy":
        src, dst = s["src_ids"], s["dst_ids"]
        return {"a": s["caches"][0].index_copy_(1, dst, s["caches"][0].index_select(1, src)),
                "b": s["caches"][1].index_copy_(1, dst, s["caches"][1].index_select(1, src))}
    if kind in ("axes", "append4"):
        return _plain_append(s, c)
    D = c["dim"]
    tab = s["tables"].clamp(min=0).long()
    k = _unpack(s["k_cache"][tab], s["k_scales"][tab].permute(0, 1, 4, 2, 3)).flatten(1, 2)
    v = _unpack(s["v_cache"][tab], s["v_scales"][tab].permute(0, 1, 4, 2, 3)).flatten(1, 2)
    keys = s["ctx"].long()
    if kind == "decode4":
        o = _plain_attend(s["q"][:, None].float(), k, v, keys[:, None] - 1, keys, s["scale"])
        return {"o": o[:, 0].to(s["q"].dtype)}
    # packed rows -> (sequences, longest) rows, those past an end masked, and back
    start, n = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    i = torch.arange(s["longest"], device=n.device)
    at = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1)
    o = _plain_attend(s["q"][at].float(), k, v, (keys - n)[:, None] + i, keys, s["scale"])
    t = torch.arange(s["q"].shape[0], device=n.device)
    of = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    return {"o": o[of, t - start[of]].to(s["q"].dtype)}


def _plain_attend(q, k, v, pos, keys, scale):
    """q (N, Lq, Hq, D) at positions pos (N, Lq); k, v (N, Lk, Hkv, D) of which keys (N,) count."""
    N, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    r = Hq // Hkv
    qh = q.view(N, Lq, Hkv, r, D).permute(0, 2, 3, 1, 4).reshape(N, Hkv, r * Lq, D)
    sc = (qh @ k.permute(0, 2, 3, 1).contiguous()).view(N, Hkv, r, Lq, Lk) * scale
    j = torch.arange(Lk, device=q.device)
    seen = (j <= pos[..., None]) & (j < keys[:, None, None])
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    l = p.sum(-1, keepdim=True)
    o = (p.view(N, Hkv, r * Lq, Lk) @ v.permute(0, 2, 1, 3).contiguous()).view(N, Hkv, r, Lq, D)
    o = torch.where(l > 0, o / l, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(N, Lq, Hq, D)


def _pack(x):
    """Rows of 16-bit numbers (..., D) as two codes a byte (..., D / 2) and scale bytes (..., D / 32)."""
    y = x.float().unflatten(-1, (-1, 32))
    m, e = torch.frexp(y.abs().amax(-1))
    top = EXPONENTS[x.dtype]
    e = (e - 2 - (m <= 0.75).int()).clamp(-top, top)
    z = torch.ldexp(y, -e[..., None])
    a = z.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    r = (a / step).round() * step
    code = torch.where(r < 2, 2 * r, torch.where(r < 4, r + 2, 4 + r / 2)).to(torch.uint8)
    code = (code | (torch.signbit(z).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _unpack(codes, scales):
    """The numbers, in float32, of codes (..., D / 2) with scales (..., D / 32)."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    z = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).flatten(-2)
    return torch.ldexp(z.unflatten(-1, (-1, 32)), scales[..., None].int() - 127).flatten(-2)


def _plain_append(s, c):
    page = c["page"]
    T = s["q"].shape[0]
    t = torch.arange(T, device=s["q"].device)
    if "cu" in s:
        n = torch.searchsorted(s["cu"][1:].long(), t, right=True)
        pos = s["ctx"].long()[n] - s["cu"].long()[n + 1] + t
    else:
        n, pos = t, s["ctx"].long() - 1
    block, slot = s["tables"][n, pos // page].long(), pos % page
    if c["kind"] == "axes":
        j = torch.arange(c["rot"] // 2, device=t.device)
        p = s["positions"].long()[torch.tensor(_axis_of(c), device=t.device)].t()
        cos, sin = s["cos"][p, j][:, None], s["sin"][p, j][:, None]
        s["k_cache"][block, slot] = _plain_rotate(s["k"], cos, sin, c["rot"])
        s["v_cache"][block, slot] = s["v"]
        return {"q": _plain_rotate(s["q"], cos, sin, c["rot"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    out = {"q": _plain_rotate(s["q"], cos, sin, c["rot"])}
    for x, y in (("k", _plain_rotate(s["k"], cos.double(), sin.double(), c["rot"])), ("v", s["v"])):
        codes, scales = _pack(y)
        s[x + "_cache"][block, slot] = codes
        s[x + "_scales"][block, :, :, slot] = scales
        out[x] = _unpack(s[x + "_cache"][block, slot], s[x + "_scales"][block, :, :, slot]).to(y.dtype)
    return out


def _plain_rotate(x, cos, sin, rot):
    """The first `rot` dims of x turned by halves, in the tables' type, rounded once to x's."""
    y = x[..., :rot].to(cos.dtype)
    a, b = y[..., : rot // 2], y[..., rot // 2:]
    y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y.float().to(x.dtype), x[..., rot:]], -1)


def _run_own(s, c):
    import myvllm_amd as ops

    kind = c["kind"]
    if kind == "copy":
        ops.cache_copy(s["caches"], s["src"], s["dst"])
        return {"a": s["caches"][0], "b": s["caches"][1]}
    caches = (s["k_cache"], s["v_cache"], s["tables"], s["ctx"])
    if kind == "axes":
        q = ops.paged_kv_append(s["q"], s["k"], s["v"], *caches, c["page"], cos=s["cos"], sin=s["sin"],
                                cu_seqlens=s.get("cu"), positions=s["positions"], sections=_sections(c),
                                sections_interleaved=c["deal"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    scales = dict(k_scales=s["k_scales"], v_scales=s["v_scales"])
    if kind == "append4":
        q = ops.paged_kv_append(s["q"], s["k"], s["v"], *caches, c["page"], cos=s["cos"], sin=s["sin"],
                                cu_seqlens=s["cu"], **scales)
        k, v = ops.paged_kv_read(*caches, c["page"], num_tokens=s["q"].shape[0], cu_seqlens=s["cu"],
                                 dtype=s["q"].dtype, **scales)
        return {"q": q, "k": k, "v": v}
    if kind == "decode4":
        return {"o": ops.paged_flash_attention_decode(s["q"], *caches, s["scale"], c["page"], **scales)}
    return {"o": ops.paged_flash_attention_prefill(s["q"], *caches, s["cu"], None, s["scale"], c["page"],
                                                   max_seqlen=s["longest"], **scales)}


# ---- what a pass cannot do without ---------------------------------------------------


def work(case: dict) -> dict:
    c, kind = case, case["kind"]
    es = 2
    if kind == "copy":
        if c["of"] == "pages":
            row = 2 * c["page"] * c["hkv"] * c["dim"] * es
        else:
            row = 3 * (256 * c["hk"] + 128 * c["hv"]) * es + c["hv"] * 128 * 128 * 4
        return {"bytes": 2 * c["pairs"] * c["layers"] * row, "flops": 0}
    hq, hkv, D = c["hq"], c["hkv"], c["dim"]
    lens = _lengths(c)
    T = sum(lens)
    row4 = D // 2 + D // 32
    if kind == "axes":
        return {"bytes": 2 * T * (hq + 2 * hkv) * D * es + T * (c["rot"] * 4 + 16),
                "flops": 3 * T * (hq + hkv) * c["rot"]}
    if kind == "append4":
        # q read and written; k and v read, written in 4 bits, read in 4 bits and written
        return {"bytes": 2 * T * hq * D * es + 2 * T * hkv * (2 * D * es + 2 * row4) + T * (c["rot"] * 4 + 4),
                "flops": 3 * T * (hq + hkv) * c["rot"]}
    if kind == "decode4":
        return {"bytes": c["seqs"] * 2 * hq * D * es + T * 2 * hkv * row4 + T // c["page"] * 4,
                "flops": 4 * D * hq * T}
    ctx = _contexts(c)
    pairs = sum(n * m - n * (n - 1) // 2 for n, m in zip(lens, ctx))
    return {"bytes": T * 2 * hq * D * es + sum(ctx) * 2 * hkv * row4, "flops": 4 * D * hq * pairs}


# ---- the same in 64 bits -------------------------------------------------------------


def exact(case: dict, seed: int):
    c, kind = case, case["kind"]
    if kind == "copy":
        return None  # (nothing is computed)
    s = prepare(case, seed)
    hq, hkv, D, page = c["hq"], c["hkv"], c["dim"], c["page"]
    r = hq // hkv
    lens = _lengths(c)
    ctx = lens if kind == "decode4" else _contexts(c)
    if kind in ("axes", "append4"):
        dt = s["k"].dtype
        out = {x: s[x].double() for x in ("q", "k", "v")}
        if kind == "axes":
            caches = {x: s[x].double() for x in ("k_cache", "v_cache")}
        half, at = c["rot"] // 2, 0
        of = _axis_of(c) if kind == "axes" else [0] * half
        for n, (m, new) in enumerate(zip(ctx, lens)):
            own_pos = torch.arange(m - new, m, device=s["q"].device)
            pos = s["positions"][:, at: at + new].long() if kind == "axes" else own_pos[None]
            turn = torch.stack([torch.complex(s["cos"][pos[a], f].double(), s["sin"][pos[a], f].double())
                                for f, a in enumerate(of)], -1)[:, None]
            for x in ("q", "k"):
                y = out[x][at: at + new]
                z = torch.complex(y[..., :half].contiguous(), y[..., half:c["rot"]].contiguous()) * turn
                y[..., :half], y[..., half:c["rot"]] = z.real, z.imag
            if kind == "axes":
                rows = (s["tables"][n].long()[own_pos // page], own_pos % page)
                caches["k_cache"][rows], caches["v_cache"][rows] = out["k"][at: at + new], out["v"][at: at + new]
            at += new
        if kind == "axes":
            return dict(q=out["q"], **caches)
        return dict(q=out["q"], k=_nearest(out["k"].float().to(dt).double(), EXPONENTS[dt]),
                    v=_nearest(out["v"], EXPONENTS[dt]))
    decoded = {}
    for x in ("k", "v"):
        table = torch.tensor([g * t for t in (1.0, -1.0) for g in GRID], dtype=torch.float64, device=s["q"].device)
        decoded[x] = lambda blocks, h, x=x: (
            table[torch.stack([s[x + "_cache"][blocks, :, h] % 16, s[x + "_cache"][blocks, :, h] // 16], -1).long()]
            .reshape(len(blocks), page, D // 32, 32)
            * 2.0 ** (s[x + "_scales"][blocks, h].double().transpose(1, 2)[..., None] - 127)).reshape(-1, D)
    q, out = s["q"].double(), []
    cu = list(range(c["seqs"] + 1)) if kind == "decode4" else _cu(lens)
    for n, m in enumerate(ctx):
        a, e = cu[n], cu[n + 1]
        blocks = s["tables"][n, : -(-m // page)].long()
        o = torch.empty(e - a, hq, D, dtype=torch.float64, device=q.device)
        j = torch.arange(m, device=q.device)
        for h in range(hkv):
            kt, vh = decoded["k"](blocks, h)[:m].t().contiguous(), decoded["v"](blocks, h)[:m]
            for x in range(a, e, 1024):
                y = min(e, x + 1024)
                i = torch.arange(x - e + m, y - e + m, device=q.device)
                w = (q[x:y, h * r: (h + 1) * r].transpose(0, 1).reshape(-1, D) @ kt).view(r, y - x, m) * s["scale"]
                w = torch.softmax(w.masked_fill(j > i[:, None], -math.inf), -1)
                o[x - a: y - a, h * r: (h + 1) * r] = (w.flatten(0, 1) @ vh).view(r, y - x, D).transpose(0, 1)
        out.append(o)
    return {"o": torch.cat(out)}


def _nearest(x, top):
    """The 4-bit values next to x, by the borders between neighbouring ones: of a tie the even code's."""
    y = x.unflatten(-1, (-1, 32))
    most = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(most.clamp(min=1e-300) / 6))
    e = torch.where(6 * 2.0 ** (e - 1) >= most, e - 1, e)
    e = torch.where(6 * 2.0 ** e < most, e + 1, e)
    scale = 2.0 ** e.clamp(-top, top)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    a = (y / scale).abs()
    code = torch.zeros_like(a, dtype=torch.long)
    for k in range(7):  # past the border, or on it where the next code is even
        code += (a >= mid[k]) if k % 2 else (a > mid[k])
    return (grid[code] * scale).copysign(y).flatten(-2)
