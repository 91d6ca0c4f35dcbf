"""Performance cases of the paged-cache append, of the decode of batches that share a prefix,
and of attention with capped or biased scores or a prefix mask.

Each case is one call as a serving program makes it.  Heads, head dims and
pages are those of this repository's attention workloads (16 / 2 heads of 256,
16 / 4 of 128, 16 / 16 of 64, 16-token pages), lengths those of its prefill
and decode workloads.  ``listed()`` holds the fixed cases, ``draw`` more of
the same ranges.  Where ``own`` is false ``run`` computes the operators in
plain float32 torch; ``exact`` restates them in float64 on its own.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PAGE = 16
ROPE_ROWS = 32768  # positions of the rotation table that a serving program keeps
ROPE_BASE = 10000.0


def listed() -> list[dict]:
    return [
        # one user's chat: the new token of a decode step, rotated and put into the cache; a latency
        dict(name="append_decode_1", kind="append", seqs=1, lo=1, hi=1, prefix=2943, len_seed=1, hq=16, hkv=2, dim=256,
             rot=64, interleaved=False, dtype="bf16"),
        # an ordinary batch's decode step
        dict(name="append_decode_256", kind="append", seqs=256, lo=1, hi=1, prefix=4096, len_seed=2, hq=16, hkv=2,
             dim=256, rot=64, interleaved=False, dtype="bf16"),
        # a full prefill batch of ragged prompts
        dict(name="append_prefill_16", kind="append", seqs=16, lo=512, hi=4096, prefix=0, len_seed=3, hq=16, hkv=2,
             dim=256, rot=256, interleaved=False, dtype="bf16"),
        # chunks of odd lengths over what is already cached, rotation of neighbouring pairs
        dict(name="append_chunks_fp16", kind="append", seqs=7, lo=33, hi=1025, prefix=16384, len_seed=4, hq=16, hkv=4,
             dim=128, rot=128, interleaved=True, dtype="fp16"),
        # a few answers sampled from one prompt
        dict(name="shared_decode_4", kind="shared", seqs=4, groups=1, plo=1000, phi=1000, lo=1, hi=64, len_seed=5,
             hq=16, hkv=2, dim=256, dtype="bf16"),
        # a serving batch behind one long system prompt
        dict(name="shared_decode_64", kind="shared", seqs=64, groups=1, plo=8192, phi=8192, lo=16, hi=1024, len_seed=6,
             hq=16, hkv=2, dim=256, dtype="bf16"),
        # a large batch that asks about one long document
        dict(name="shared_decode_256", kind="shared", seqs=256, groups=1, plo=16384, phi=16384, lo=128, hi=2048,
             len_seed=7, hq=16, hkv=2, dim=256, dtype="bf16"),
        # several prompts, each with its own answers
        dict(name="shared_groups_fp16", kind="shared", seqs=45, groups=5, plo=500, phi=6000, lo=1, hi=700, len_seed=8,
             hq=16, hkv=4, dim=128, dtype="fp16"),
        # prompts through an attention layer whose scores are capped
        dict(name="capped_prefill_8", kind="prefill", seqs=8, lo=256, hi=4096, len_seed=9, hq=16, hkv=2, dim=256,
             cap=50.0, slopes=False, pmask=0, dtype="bf16"),
        # chunks over cached prefixes, scores biased by distance
        dict(name="biased_paged_prefill", kind="paged_prefill", seqs=4, lo=256, hi=1024, prefix=16384, len_seed=10,
             hq=16, hkv=4, dim=128, cap=0.0, slopes=True, pmask=0, dtype="bf16"),
        # a batch's decode step with capped scores
        dict(name="capped_decode_64", kind="decode", seqs=64, lo=1024, hi=8192, len_seed=11, hq=16, hkv=2, dim=256,
             cap=30.0, slopes=False, dtype="bf16"),
        # documents read in both directions before the answer is: a prefix mask, capped and biased
        dict(name="prefix_mask_fp16", kind="prefill", seqs=6, lo=200, hi=2048, len_seed=12, hq=16, hkv=16, dim=64,
             cap=20.0, slopes=True, pmask=1500, dtype="fp16"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    """A whole number in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng: random.Random) -> dict:
    """One more case; sizes stay at or below the listed cases'."""
    kind = rng.choice(["append", "append_decode", "shared", "shared", "shared", "prefill", "paged_prefill", "decode",
                       "decode"])
    hq, hkv, dim = rng.choice([(16, 2, 256), (16, 2, 256), (8, 1, 256), (16, 4, 128), (16, 16, 64)])
    c = dict(len_seed=rng.randrange(1 << 20), hq=hq, hkv=hkv, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if kind == "append_decode":
        return dict(c, kind="append", seqs=_log(rng, 1, 512), lo=1, hi=1, prefix=_log(rng, 16, 16384),
                    rot=rng.choice([dim, dim // 4]), interleaved=rng.choice([False, False, True]))
    if kind == "append":
        hi = _log(rng, 2, 4096)
        return dict(c, kind="append", seqs=max(1, min(_log(rng, 1, 16), 32768 // hi)), lo=max(1, hi // 8), hi=hi,
                    prefix=rng.choice([0, _log(rng, 16, 16384)]), rot=rng.choice([dim, dim // 4]),
                    interleaved=rng.choice([False, False, True]))
    if kind == "shared":
        phi, hi = _log(rng, 64, 16384), _log(rng, 8, 2048)
        seqs = max(2, min(_log(rng, 2, 256), 4_000_000 // (phi + hi)))
        groups = rng.choice([1, 1, rng.randint(1, max(1, seqs // 2))])
        return dict(c, kind="shared", seqs=seqs, groups=groups, plo=phi if groups == 1 else max(1, phi // 8), phi=phi,
                    lo=max(1, hi // 16), hi=hi)
    form = rng.choice(["cap", "slopes", "both"])
    c.update(cap=0.0 if form == "slopes" else float(rng.choice([15, 30, 50])), slopes=form != "cap")
    if kind == "prefill":
        hi = _log(rng, 64, 4096)
        return dict(c, kind="prefill", seqs=max(1, min(_log(rng, 1, 16), 100_000_000 // (hi * hi))),
                    lo=max(1, hi // 8), hi=hi, pmask=rng.choice([0, 0, max(1, hi // 2)]))
    if kind == "paged_prefill":
        hi, prefix = _log(rng, 16, 1024), _log(rng, 64, 16384)
        return dict(c, kind="paged_prefill", seqs=max(1, min(_log(rng, 1, 8), 50_000_000 // (hi * (prefix + hi)))),
                    lo=max(1, hi // 8), hi=hi, prefix=prefix, pmask=rng.choice([0, 0, max(1, (prefix + hi) // 2)]))
    hi = _log(rng, 64, 8192)
    return dict(c, kind="decode", seqs=max(1, min(_log(rng, 1, 128), 524288 // hi)), lo=max(1, hi // 8), hi=hi)


# ---- sizes ---------------------------------------------------------------------------


def _lengths(c: dict) -> list[int]:
    """New tokens per sequence, or the keys of each (decode), or the own keys of each (shared prefix)."""
    r = random.Random(c["len_seed"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["seqs"])]


def _contexts(c: dict) -> list[int]:
    """Keys of each sequence once the new ones are in the cache."""
    lens, r = _lengths(c), random.Random(c["len_seed"] + 1)
    if c["kind"] == "shared":
        of, pre = _groups(c)
        return [pre[of[b]] + n for b, n in enumerate(lens)]
    return [n + (r.randint(c["prefix"] // 2, c["prefix"]) if c.get("prefix") else 0) for n in lens]


def _groups(c: dict) -> tuple[list[int], list[int]]:
    """The group of each sequence (in order, none empty) and the keys that each group shares."""
    r = random.Random(c["len_seed"] + 2)
    cuts = sorted(r.sample(range(1, c["seqs"]), c["groups"] - 1)) if c["groups"] > 1 else []
    return ([sum(b >= x for x in cuts) for b in range(c["seqs"])],
            [r.randint(c["plo"], c["phi"]) for _ in range(c["groups"])])


def _prefix_masks(c: dict) -> list[int]:
    r = random.Random(c["len_seed"] + 3)
    return [r.randint(0, c["pmask"]) for _ in range(c["seqs"])]


def _cu(lens: list[int]) -> list[int]:
    cu = [0]
    cu.extend(sum(lens[: n + 1]) for n in range(len(lens)))
    return cu


# ---- inputs --------------------------------------------------------------------------


def prepare(case: dict, seed: int) -> dict:
    c = case
    dev, dt = torch.device("cuda:0"), DTYPES[c["dtype"]]
    gen, cpu = torch.Generator(device=dev).manual_seed(seed), random.Random(seed)
    normal = lambda *shape, std=1.0: (torch.randn(*shape, generator=gen, device=dev) * std).to(dt)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    kind, hq, hkv, D = c["kind"], c["hq"], c["hkv"], c["dim"]
    lens = _lengths(c)
    T = c["seqs"] if kind in ("decode", "shared") else sum(lens)
    # scores of a few units, as after the q and k norms of a trained layer
    s = dict(q=normal(T, hq, D, std=1.0 if kind == "append" else 2.0), scale=D ** -0.5, case=c, longest=max(lens))
    if c.get("slopes"):
        s["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / hq) for h in range(hq)], device=dev)
    if c.get("pmask"):
        s["pmask"] = ints(_prefix_masks(c))
    if kind in ("append", "prefill"):
        s["k"], s["v"] = normal(T, hkv, D), normal(T, hkv, D)
    if kind in ("prefill", "paged_prefill") or (kind == "append" and c["hi"] > 1):
        s["cu"] = ints(_cu(lens))
    if kind == "prefill":
        return s
    ctx = _contexts(c)
    of, pre = _groups(c) if kind == "shared" else ([], [])
    pages = [-(-n // PAGE) for n in ctx]
    total = sum(pages) + 3
    order = list(range(total))
    cpu.shuffle(order)
    rows, at = [], 0
    for p in pages:
        rows.append(order[at: at + p])
        at += p
    s["k_cache"], s["v_cache"] = normal(total, PAGE, hkv, D), normal(total, PAGE, hkv, D)
    first = {}
    for b, g in enumerate(of):
        # the whole pages of the shared keys are the group's; the keys past them lie in each one's own page
        lead = first.setdefault(g, b)
        n, rest = pre[g] // PAGE, pre[g] % PAGE
        rows[b][:n] = rows[lead][:n]
        if rest and lead != b:
            for x in ("k_cache", "v_cache"):
                s[x][rows[b][n], :rest] = s[x][rows[lead][n], :rest]
    s["tables"] = ints([r + [-1] * (max(pages) - len(r)) for r in rows])
    s["ctx"] = ints(ctx)
    if kind == "shared":
        s["prefix_lens"] = ints(pre)
        s["cu_groups"] = ints([0] + [sum(x <= g for x in of) for g in range(c["groups"])])
    if kind == "append":
        f = ROPE_BASE ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device=dev) / c["rot"])
        a = torch.arange(ROPE_ROWS, dtype=torch.float64, device=dev)[:, None] * f
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
    return s


# ---- one pass ------------------------------------------------------------------------


def run(s: dict):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "append":
        return _plain_append(s, c)
    hkv, D = c["hkv"], c["dim"]
    if c["kind"] == "prefill":
        # packed rows -> (sequences, longest) rows, those past an end masked below
        start, n = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
        i = torch.arange(s["longest"], device=n.device)
        at = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1)
        q, k, v = s["q"][at], s["k"][at], s["v"][at]
        pos, keys = i.expand(at.shape), n
    else:
        tab = s["tables"].clamp(min=0).long()
        k = s["k_cache"][tab].view(tab.shape[0], -1, hkv, D)
        v = s["v_cache"][tab].view(tab.shape[0], -1, hkv, D)
        keys = s["ctx"].long()
        if c["kind"] == "paged_prefill":
            start, n = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
            i = torch.arange(s["longest"], device=n.device)
            at = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1)
            q, pos = s["q"][at], (keys - n)[:, None] + i
        else:
            q, pos = s["q"][:, None], keys[:, None] - 1
    o = _plain_attend(q.float(), k.float(), v.float(), pos, keys, s["scale"], c.get("cap", 0.0), s.get("slopes"),
                      s.get("pmask")).to(s["q"].dtype)
    if c["kind"] in ("decode", "shared"):
        return {"o": o[:, 0]}
    return {"o": _packed(o, s)}


def _packed(o, s):
    """(sequences, longest) rows back to packed ones."""
    t = torch.arange(s["q"].shape[0], device=o.device)
    n = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    return o[n, t - s["cu"].long()[n]]


def _plain_attend(q, k, v, pos, keys, scale, cap, slopes, pmask):
    """q (N, Lq, Hq, D) at positions pos (N, Lq); k, v (N, Lk, Hkv, D) of which keys (N,) count."""
    N, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    r = Hq // Hkv
    qh = q.view(N, Lq, Hkv, r, D).permute(0, 2, 3, 1, 4).reshape(N, Hkv, r * Lq, D)
    sc = (qh @ k.permute(0, 2, 3, 1).contiguous()).view(N, Hkv, r, Lq, Lk) * scale
    if cap:
        sc = cap * torch.tanh(sc / cap)
    j = torch.arange(Lk, device=q.device)
    if slopes is not None:
        sc = sc - slopes.view(Hkv, r, 1, 1) * (pos[..., None] - j).abs().float()[:, None, None]
    seen = j <= pos[..., None]
    if pmask is not None:
        seen = seen | (j < pmask.long()[:, None, None])
    seen = seen & (j < keys[:, None, None])
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    l = p.sum(-1, keepdim=True)
    o = (p.view(N, Hkv, r * Lq, Lk) @ v.permute(0, 2, 1, 3).contiguous()).view(N, Hkv, r, Lq, D)
    o = torch.where(l > 0, o / l, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(N, Lq, Hq, D)


def _plain_append(s, c):
    T = s["q"].shape[0]
    t = torch.arange(T, device=s["q"].device)
    if "cu" in s:
        n = torch.searchsorted(s["cu"][1:].long(), t, right=True)
        pos = s["ctx"].long()[n] - s["cu"].long()[n + 1] + t
    else:
        n, pos = t, s["ctx"].long() - 1
    block, slot = s["tables"][n, pos // PAGE].long(), pos % PAGE
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    s["k_cache"][block, slot] = _plain_rotate(s["k"], cos, sin, c)
    s["v_cache"][block, slot] = s["v"]
    return {"q": _plain_rotate(s["q"], cos, sin, c), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_rotate(x, cos, sin, c):
    rot = c["rot"]
    y = x[..., :rot].float()
    if c["interleaved"]:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = y[..., : rot // 2], y[..., rot // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y.to(x.dtype), x[..., rot:]], -1)


def _run_own(s, c):
    import myvllm_amd as ops

    kind = c["kind"]
    if kind == "append":
        q = ops.paged_kv_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["tables"], s["ctx"], PAGE,
                                cos=s["cos"], sin=s["sin"], cu_seqlens=s.get("cu"), interleaved=c["interleaved"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if kind == "shared":
        return {"o": ops.paged_flash_attention_decode_shared(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["ctx"],
                                                             s["prefix_lens"], s["scale"], PAGE,
                                                             cu_groups=s["cu_groups"])}
    form = dict(softcap=c["cap"] or None, alibi_slopes=s.get("slopes"))
    if kind == "decode":
        return {"o": ops.paged_flash_attention_decode(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["ctx"],
                                                      s["scale"], PAGE, **form)}
    form["prefix_lens"] = s.get("pmask")
    if kind == "paged_prefill":
        return {"o": ops.paged_flash_attention_prefill(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["ctx"],
                                                       s["cu"], None, s["scale"], PAGE, max_seqlen=s["longest"],
                                                       **form)}
    return {"o": ops.flash_attention_prefill(s["q"], s["k"], s["v"], s["cu"], s["scale"], c["hq"], c["hkv"], c["dim"],
                                             c["dim"], True, max_seqlen=s["longest"], **form)}


# ---- what a pass cannot do without ---------------------------------------------------


def work(case: dict) -> dict:
    c, kind, lens = case, case["kind"], _lengths(case)
    hq, hkv, D, es = c["hq"], c["hkv"], c["dim"], 2
    if kind == "append":
        T = sum(lens)
        return {"bytes": 2 * T * (hq + 2 * hkv) * D * es + T * (c["rot"] * 4 + 4),
                "flops": 3 * T * (hq + hkv) * c["rot"]}
    if kind == "shared":
        of, pre = _groups(c)
        keys = sum(lens) + sum(pre)
        return {"bytes": (c["seqs"] * 2 * hq + keys * 2 * hkv) * D * es + keys // PAGE * 4,
                "flops": 4 * D * hq * sum(_contexts(c))}
    if kind == "decode":
        return {"bytes": (c["seqs"] * 2 * hq + sum(lens) * 2 * hkv) * D * es + sum(lens) // PAGE * 4,
                "flops": 4 * D * hq * sum(lens)}
    ctx, masks = (lens if kind == "prefill" else _contexts(c)), _prefix_masks(c) if c["pmask"] else [0] * len(lens)
    pairs = 0
    for n, m, p in zip(lens, ctx, masks):
        # query i sees max(m - n + i + 1, min(p, m)) keys
        p = min(p, m)
        low = max(0, min(n, p - (m - n)))  # queries that see p keys
        pairs += low * p + sum(range(m - n + low + 1, m + 1))
    return {"bytes": (sum(lens) * 2 * hq + sum(ctx) * 2 * hkv) * D * es, "flops": 4 * D * hq * pairs}


# ---- the same in 64 bits -------------------------------------------------------------


def exact(case: dict, seed: int):
    c, kind = case, case["kind"]
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v
         for k, v in prepare(case, seed).items()}
    hq, hkv, D = c["hq"], c["hkv"], c["dim"]
    r = hq // hkv
    lens, N = _lengths(c), c["seqs"]
    if kind == "append":
        # the rotation as a complex product
        at = 0
        half = c["rot"] // 2
        q = s["q"].clone()
        for n, (m, new) in enumerate(zip(_contexts(c), lens)):
            p = torch.arange(m - new, m, device=q.device)
            turn = torch.complex(s["cos"][p], s["sin"][p])[:, None]
            kk = s["k"][at: at + new].clone()
            for x in (q[at: at + new], kk):
                if c["interleaved"]:
                    re, im = x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]
                else:
                    re, im = x[..., :half], x[..., half:c["rot"]]
                z = torch.complex(re.contiguous(), im.contiguous()) * turn
                re.copy_(z.real)
                im.copy_(z.imag)
            rows = (s["tables"][n].long()[p // PAGE], p % PAGE)
            s["k_cache"][rows] = kk
            s["v_cache"][rows] = s["v"][at: at + new]
            at += new
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    out = []
    one = kind in ("decode", "shared")
    cu = list(range(N + 1)) if one else _cu(lens)
    ctx = _contexts(c) if kind in ("shared", "paged_prefill") else lens
    masks = _prefix_masks(c) if c.get("pmask") else [0] * N
    for n, m in enumerate(ctx):
        a, e = cu[n], cu[n + 1]
        if kind == "prefill":
            k, v = s["k"][a:e], s["v"][a:e]
        else:
            pages = s["tables"][n, : -(-m // PAGE)].long()
            k, v = s["k_cache"][pages].flatten(0, 1)[:m], s["v_cache"][pages].flatten(0, 1)[:m]
        j = torch.arange(m, device=k.device)
        o = torch.empty(e - a, hq, D, dtype=torch.float64, device=k.device)
        for h in range(hkv):
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            for x in range(a, e, 1024):
                y = min(e, x + 1024)
                i = torch.arange(x - e + m, y - e + m, device=k.device)
                w = (s["q"][x:y, h * r: (h + 1) * r].transpose(0, 1).reshape(-1, D) @ kt).view(r, y - x, m) * s["scale"]
                if c.get("cap"):
                    w = torch.tanh(w / c["cap"]) * c["cap"]
                if c.get("slopes"):
                    w = w - s["slopes"][h * r: (h + 1) * r, None, None] * (i[:, None] - j).abs()
                hidden = (j > i[:, None]) & (j >= masks[n])
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                o[x - a: y - a, h * r: (h + 1) * r] = (w.flatten(0, 1) @ vh).view(r, y - x, D).transpose(0, 1)
        out.append(o)
    return {"o": torch.cat(out)}
