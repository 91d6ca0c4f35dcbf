"""Full attention of the hybrid stack's attention layers, on HIP kernels.

Same names, arguments and results as ``ops/full_attention.py`` of
yuyifanbupt/myvllm (``flash_attention_prefill`` ``:114-173``,
``paged_flash_attention_decode`` ``:282-335``, ``paged_flash_attention_prefill``
``:454-512``), with the output on q's device in q's dtype.  GQA: query head h
reads kv head ``h // (Hq // Hkv)``.  Supported: bf16 / fp16, head dim 64, 128
or 256 for q, k and v alike.

Differences from the reference kernels, all in the reference's disfavour
(each is a defect of its Triton code, not an intended behaviour): K and V of
sequence n are read from that sequence's rows (``:57-72`` read from token 0),
the output's dim stride is the dim stride (``:76``), the non-causal path masks
keys past the sequence end, and the paged prefill reads its work list and
``cu_seqlens`` correctly (``:378-380``); a query with no visible key gives a
zero row instead of 0/0.

The three ops take other forms of scores as keywords (``softcap``,
``alibi_slopes``, ``prefix_lens``), and beside them stand the append that fills
the caches (:func:`paged_kv_append`) and the decode of sequences that share
their first keys (:func:`paged_flash_attention_decode_shared`).
"""
from __future__ import annotations

import torch

from . import _lib


def _out_for(out, shape, dtype, dev):
    """The tensor the kernel writes: `out` itself when it has 16-byte aligned
    rows, else a temporary copied into `out` afterwards (_finish)."""
    if out is not None and _lib.vec16_ok(out):
        return out
    return torch.empty(shape, dtype=dtype, device=dev)


def _finish(out, o):
    if out is not None and o is not out:
        out.copy_(o)
        return out
    return o


_DECODE_MIN_SPLIT_KEYS = 256
_DECODE_TARGET_WAVES = 512   # unit x kv-head waves aimed at with splits
_DECODE_SPLIT_ROWS = 2048    # (sequence, kv head) rows from which one split is enough
_DECODE_MAX_SPLITS = 256


def _max_seqlen(cu_seqlens: torch.Tensor) -> int:
    if cu_seqlens.numel() < 2:
        return 0
    return int((cu_seqlens[1:] - cu_seqlens[:-1]).max().item())


def flash_attention_prefill(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: torch.Tensor,
    scale: float,
    num_heads: int,
    num_kv_heads: int,
    head_dim: int,
    head_v_dim: int,
    is_causal: bool,
    max_seqlen: int | None = None,
    out: torch.Tensor | None = None,
    softcap: float | None = None,
    alibi_slopes: torch.Tensor | None = None,
    prefix_lens: torch.Tensor | None = None,
) -> torch.Tensor:
    """Varlen attention over packed sequences: q (T, Hq, D), k, v (T, Hkv, D) ->
    (T, Hq, D).  ``max_seqlen`` (the longest sequence) is read from
    ``cu_seqlens`` when not given, one host sync as in the reference (``:139``).

    Other forms of scores x = scale q.k, applied in this order: ``softcap``
    (1e-3 to 4096): x <- softcap tanh(x / softcap); ``alibi_slopes``
    (Hq,) fp32: x <- x - slope_h |i - j| (without a cap for scales from 1e-20
    on, or 0); ``prefix_lens`` (N,), causal only: the first ``prefix_lens[n]``
    keys are visible to every query of sequence n.  A packed batch is its own
    document mask: each document a sequence."""
    if q.shape[1] != num_heads or k.shape[1] != num_kv_heads or q.shape[2] != head_dim or v.shape[2] != head_v_dim:
        raise ValueError("q/k/v shapes disagree with num_heads/num_kv_heads/head_dim/head_v_dim")
    dev = _lib.require_device(q, k, v, cu_seqlens, alibi_slopes, prefix_lens)
    if max_seqlen is None:
        max_seqlen = _max_seqlen(cu_seqlens)
    own = head_dim in _KERNEL_HEAD_DIMS and head_v_dim == head_dim
    scored = _scored(softcap, alibi_slopes, prefix_lens)
    if not own and (scored or not _direct_head_dim(q, k, v, head_dim, head_v_dim, max_seqlen)):
        return _padded_prefill(q, k, v, cu_seqlens, scale, head_dim, head_v_dim, is_causal, max_seqlen, out,
                               softcap=softcap, alibi_slopes=alibi_slopes, prefix_lens=prefix_lens)
    q, k, v = _lib.vec16(q), _lib.vec16(k), _lib.vec16(v)
    if scored:
        o = _out_for(out, (q.shape[0], q.shape[1], head_v_dim), q.dtype, dev)
        _lib.call("flash_attention_varlen_scored", q, k, v, cu_seqlens, o, alibi_slopes, prefix_lens, int(max_seqlen),
                  float(scale), float(softcap or 0.0), int(bool(is_causal)))
        return _finish(out, o)
    o = _out_for(out if own or _apart(out, q, k, v) else None, (q.shape[0], q.shape[1], head_v_dim), q.dtype, dev)
    _lib.call("flash_attention_varlen" if own else "flash_attention_varlen_any_dim", q, k, v, cu_seqlens, o,
              int(max_seqlen), float(scale), int(bool(is_causal)))
    return _finish(out, o)


_KERNEL_HEAD_DIMS = (64, 128, 256)


def _scored(softcap, alibi_slopes, prefix_lens=None) -> bool:
    return softcap is not None or alibi_slopes is not None or prefix_lens is not None


def _direct_head_dim(q, k, v, head_dim, head_v_dim, max_seqlen) -> bool:
    """Whether the kernels of any head dim read q, k and v as they lie: 16-bit
    rows of a multiple of 8 elements (the vision tower's 1152 / 16 = 72,
    ``models/qwen/vision.py:18``, ``configs/qwen3_5.py:11``, ``:16``), each
    inside its token stride, within the kernels' 32-bit offsets.  The rest is
    padded: other dims, v narrower or wider than k, overlapping rows."""
    if head_dim != head_v_dim or head_dim % 8 or not 0 < head_dim <= _KERNEL_HEAD_DIMS[-1]:
        return False
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or k.shape[0] != q.shape[0] or v.shape != k.shape:
        return False
    st = max(k.stride(0), v.stride(0), k.shape[1] * head_dim)
    return min(k.stride(0), v.stride(0)) >= head_dim and max(max_seqlen, 64) * st * q.element_size() < 2**31


def _apart(out, q, k, v) -> bool:
    """Whether a result of q's shape can go to `out` directly: of the same shape,
    dtype and device and in memory of its own.  The padded path copies its result
    into whatever `out` is, one of the inputs among them."""
    return (out is not None and out.shape == q.shape and out.dtype == q.dtype and out.device == q.device
            and out.untyped_storage().data_ptr() not in {t.untyped_storage().data_ptr() for t in (q, k, v)})


def _crosses(out, q, k, v) -> bool:
    """Whether a result of q's form written to `out` row by row, each after its own
    row of q is read, could land on other rows of q, k or v first: `out` in their
    memory, and not q itself."""
    if out is q or out.shape != q.shape or out.dtype != q.dtype:
        return False  # (another shape or type is refused further on)
    if out.data_ptr() == q.data_ptr() and out.stride() == q.stride():
        return False
    return any(_meet(out, t) for t in (q, k, v))


def _meet(a, b) -> bool:
    """Whether two tensors (tokens, heads, dim) of one type may share memory: not
    where one ends before the other begins, nor as column blocks of one matrix."""
    es, pa, pb = a.element_size(), a.data_ptr(), b.data_ptr()
    if a.numel() == 0 or b.numel() == 0 or pa + es * _span(a) <= pb or pb + es * _span(b) <= pa:
        return False
    row = a.stride(0) * es
    at = (pa - pb) % row if row > 0 else 0
    return not (a.stride(0) == b.stride(0) and es * _span(b[0]) <= at and at + es * _span(a[0]) <= row)


def _span(t) -> int:
    """Elements from a tensor's first to its last."""
    return 1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))


def _padded_prefill(q, k, v, cu_seqlens, scale, head_dim, head_v_dim, is_causal, max_seqlen, out, **form):
    """Head dims no kernel reads as they lie (:func:`_direct_head_dim`) run
    zero-padded to the next of 64, 128 and 256: zero dims add nothing to q.k
    and give zero output columns, which are dropped.  The padded copies cost
    one pass over q, k and v."""
    Dp = next((d for d in _KERNEL_HEAD_DIMS if d >= max(head_dim, head_v_dim)), None)
    if Dp is None:
        raise ValueError(f"head dims {head_dim}/{head_v_dim} above {_KERNEL_HEAD_DIMS[-1]} are not supported")
    pad = lambda t: torch.nn.functional.pad(t, (0, Dp - t.shape[-1]))
    o = flash_attention_prefill(pad(q), pad(k), pad(v), cu_seqlens, scale, q.shape[1], k.shape[1], Dp, Dp, is_causal,
                                max_seqlen=max_seqlen, **form)
    return _finish(out, o[..., :head_v_dim]) if out is not None else o[..., :head_v_dim]


def decode_num_splits(num_seqs: int, num_q_heads: int, num_kv_heads: int, capacity: int) -> int:
    """Splits of the decode launch.  With num_splits > 1 the kernel deals the
    batch's 16-key tiles evenly over num_seqs x (num_splits - 1) units
    (whatever the context lengths), and each unit's waves write partials that
    a second launch merges; with one split a wave streams a whole sequence.
    Balanced units saturate HBM from about 512 waves (unit x kv head x
    query-head group) on; more waves only add partials and concurrent page
    streams (256 sequences of U[512, 4096] keys, 2 kv heads: 256 units 232
    us, 512 units 245, 1,024 units 245; 64 of U[2k, 32k]: 192 units 397 us,
    1,024 units 429).  So: about 512 waves, at least one unit per sequence
    (one split leaves ragged batches unbalanced), one split once the batch
    alone has 2048 rows, and at least 256 keys of the table's capacity per
    unit."""
    rows = max(1, num_seqs * num_kv_heads * ((num_q_heads // max(num_kv_heads, 1) + 15) // 16))
    if rows >= _DECODE_SPLIT_ROWS:
        return 1
    units = max(1, round(_DECODE_TARGET_WAVES / rows))
    by_keys = -(-max(capacity, 1) // _DECODE_MIN_SPLIT_KEYS)
    return max(1, min(_DECODE_MAX_SPLITS, 1 + min(units, by_keys)))


def paged_flash_attention_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float,
    block_size: int,
    num_splits: int | None = None,
    out: torch.Tensor | None = None,
    softcap: float | None = None,
    alibi_slopes: torch.Tensor | None = None,
) -> torch.Tensor:
    """One query per sequence over its paged cache: q (B, Hq, D), caches
    (num_blocks, block_size, Hkv, D), block_tables (B, max_blocks),
    context_lens (B,) -> (B, Hq, D).  No host sync.  ``softcap`` and
    ``alibi_slopes`` as in :func:`flash_attention_prefill`."""
    if k_cache.shape[1] != block_size:
        raise ValueError(f"block_size {block_size} != k_cache.shape[1] {k_cache.shape[1]}")
    dev = _lib.require_device(q, k_cache, v_cache, block_tables, context_lens, alibi_slopes)
    B, Hq, Dh = q.shape
    if num_splits is None:
        num_splits = decode_num_splits(B, Hq, k_cache.shape[2], block_tables.shape[1] * block_size)
    ws = None
    n_ws = _lib.workspace_size("paged_attention_decode_workspace_size", B, Hq, Dh, int(num_splits))
    if n_ws > 0:
        ws = torch.empty(n_ws, dtype=torch.float32, device=dev)
    q, k_cache, v_cache = _lib.vec16(q), _lib.vec16(k_cache), _lib.vec16(v_cache)
    o = _out_for(out, (B, Hq, v_cache.shape[-1]), q.dtype, dev)
    if _scored(softcap, alibi_slopes):
        _lib.call("paged_attention_decode_scored", q, k_cache, v_cache, block_tables, context_lens, o, ws,
                  alibi_slopes, int(num_splits), float(scale), float(softcap or 0.0))
    else:
        _lib.call("paged_attention_decode", q, k_cache, v_cache, block_tables, context_lens, o, ws, int(num_splits),
                  float(scale))
    return _finish(out, o)


def paged_flash_attention_decode_shared(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    prefix_lens: torch.Tensor,
    scale: float,
    block_size: int,
    cu_groups: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """:func:`paged_flash_attention_decode` for sequences that begin with the
    same keys (a common prompt): the same result, with those keys read once per
    group and not once per sequence.

    The sequences ``[cu_groups[g], cu_groups[g + 1])`` (all of them without
    ``cu_groups``, then ``prefix_lens`` has one element) hold the same first
    ``prefix_lens[g]`` keys and values, counted in ``context_lens`` as any
    others.  Their tables name pages that hold them, as a rule the same ones;
    they are read through the table of the group's first sequence that is long
    enough.  A shorter sequence, and one in no group, is read through its own
    table alone.  No host sync; where the workspace is not to be had it runs as
    the plain decode."""
    if k_cache.shape[1] != block_size:
        raise ValueError(f"block_size {block_size} != k_cache.shape[1] {k_cache.shape[1]}")
    dev = _lib.require_device(q, k_cache, v_cache, block_tables, context_lens, prefix_lens, cu_groups)
    B, Hq, Dh = q.shape
    n_ws = _lib.workspace_size("paged_attention_decode_shared_workspace_size", B, prefix_lens.numel(), Hq,
                               k_cache.shape[2], Dh)
    q, k_cache, v_cache = _lib.vec16(q), _lib.vec16(k_cache), _lib.vec16(v_cache)
    o = _out_for(out, (B, Hq, v_cache.shape[-1]), q.dtype, dev)
    try:
        ws = torch.empty(n_ws, dtype=torch.float32, device=dev)
    except torch.OutOfMemoryError:
        return paged_flash_attention_decode(q, k_cache, v_cache, block_tables, context_lens, scale, block_size, out=out)
    _lib.call("paged_attention_decode_shared", q, k_cache, v_cache, block_tables, context_lens, prefix_lens, cu_groups,
              o, ws, float(scale))
    return _finish(out, o)


def paged_flash_attention_decode_noalloc(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float,
    block_size: int,
    num_splits: int,
    out: torch.Tensor,
) -> torch.Tensor:
    """:func:`paged_flash_attention_decode` for callers that cannot allocate
    device memory: ``out`` is required, ``num_splits`` is explicit, and the
    split partials live in the library's static device array (C entry
    ``paged_attention_decode_noalloc``; at most ``GDN_DECODE_SCRATCH_FLOATS``
    fp32 values, else ``GdnError``).  Calls that overlap in time on one GPU
    share that array and race; order them on one stream."""
    if k_cache.shape[1] != block_size:
        raise ValueError(f"block_size {block_size} != k_cache.shape[1] {k_cache.shape[1]}")
    _lib.require_device(q, k_cache, v_cache, block_tables, context_lens, out)
    _lib.call("paged_attention_decode_noalloc", q, k_cache, v_cache, block_tables, context_lens, out, int(num_splits),
              float(scale))
    return out


def _prefill_workspace(q, k_cache, v_cache, block_tables, cu_seqlens, page):
    """Workspace of the split paged prefill when these sizes run split, else
    None: one workgroup per row, also where the memory is not to be had.
    Pages of a multiple of 16 keys only, with block strides below 4 GiB: the
    launcher serves the others by a kernel that looks every row up and is not
    split."""
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.dim() != 4 or block_tables.dim() != 2 or cu_seqlens.dim() != 1:
        return None  # (the entry refuses the call)
    if page % 16 or max(k_cache.stride(0), v_cache.stride(0)) * k_cache.element_size() >= 2**32:
        return None
    n = _lib.workspace_size("paged_attention_prefill_workspace_size", q.shape[0], cu_seqlens.numel() - 1, q.shape[1],
                            k_cache.shape[2], q.shape[2], block_tables.shape[1] * page)
    if n <= 0:
        return None
    try:
        return torch.empty(n, dtype=torch.float32, device=q.device)
    except torch.OutOfMemoryError:
        return None


def paged_flash_attention_prefill(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    block_m_indices: torch.Tensor | None,
    scale: float,
    page_block_size: int,
    max_seqlen: int | None = None,
    out: torch.Tensor | None = None,
    softcap: float | None = None,
    alibi_slopes: torch.Tensor | None = None,
    prefix_lens: torch.Tensor | None = None,
) -> torch.Tensor:
    """Prefill over a paged cache that already holds the new keys: query i of
    sequence n sits at position ``context_lens[n] - len_n + i`` and attends
    causally to the cached keys.  ``block_m_indices`` (the reference's
    per-16-row work list) is accepted for interface parity and not needed:
    the kernel tiles the queries itself from ``cu_seqlens``.  Few new tokens
    over a long cache are split over the keys as well; the partials then take a
    temporary workspace of up to 512 MiB, without which nothing is split.
    ``softcap``, ``alibi_slopes`` and ``prefix_lens`` as in
    :func:`flash_attention_prefill`, positions and keys counted over the cache."""
    if k_cache.shape[1] != page_block_size:
        raise ValueError(f"page_block_size {page_block_size} != k_cache.shape[1] {k_cache.shape[1]}")
    dev = _lib.require_device(q, k_cache, v_cache, page_block_tables, context_lens, cu_seqlens, alibi_slopes,
                              prefix_lens)
    if max_seqlen is None:
        max_seqlen = _max_seqlen(cu_seqlens)
    q, k_cache, v_cache = _lib.vec16(q), _lib.vec16(k_cache), _lib.vec16(v_cache)
    o = _out_for(out, (q.shape[0], q.shape[1], v_cache.shape[-1]), q.dtype, dev)
    ws = _prefill_workspace(q, k_cache, v_cache, page_block_tables, cu_seqlens, page_block_size)
    if _scored(softcap, alibi_slopes, prefix_lens):
        _lib.call("paged_attention_prefill_scored", q, k_cache, v_cache, page_block_tables, context_lens, cu_seqlens,
                  o, ws, alibi_slopes, prefix_lens, int(max_seqlen), float(scale), float(softcap or 0.0))
    elif ws is not None:
        _lib.call("paged_attention_prefill_split", q, k_cache, v_cache, page_block_tables, context_lens, cu_seqlens, o,
                  ws, int(max_seqlen), float(scale))
    else:
        _lib.call("paged_attention_prefill", q, k_cache, v_cache, page_block_tables, context_lens, cu_seqlens, o,
                  int(max_seqlen), float(scale))
    return _finish(out, o)


def paged_kv_append(
    q: torch.Tensor | None,
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    block_size: int,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    interleaved: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Puts the new tokens' k, v (T, Hkv, D) into the paged caches and rotates
    q and k on the way: the step before the paged attention ops, with their
    tables and lengths.  ``context_lens`` (N,) counts the new tokens, so token i
    of sequence n sits at position ``context_lens[n] - len_n + i``; without
    ``cu_seqlens`` every sequence has one token (a decode step).

    ``cos`` and ``sin`` (positions, rot / 2), fp32, turn the first ``rot`` dims
    of q and k (halves ``(j, j + rot / 2)`` as the reference's
    ``layers/rotary_embedding.py:20-31``, or neighbours ``(2 j, 2 j + 1)`` when
    ``interleaved``); without them nothing is rotated.  Returns the rotated q
    (None for ``q=None``), into ``out`` where given, which may be q itself (on other
    rows of q, k or v it goes through a copy).

    A token in no sequence or at a position without a table column or a row of
    the rotation is not appended and its row of q is zero; table entries
    outside ``[0, num_blocks)`` are not written.  No host sync.  The caches are
    written where they lie, so their rows must be 16-byte aligned."""
    if k_cache.shape[1] != block_size:
        raise ValueError(f"block_size {block_size} != k_cache.shape[1] {k_cache.shape[1]}")
    if q is None and out is not None:
        raise ValueError("out is the rotated q's: none without q")
    tensors = (k, v, k_cache, v_cache, block_tables, context_lens, q, out, cu_seqlens, cos, sin)
    if not _lib.same_device(*tensors):
        _lib.require_device(*tensors)
    if not _lib.vec16_all(q, k, v, cos, sin):
        q, k, v, cos, sin = (t if t is None else _lib.vec16(t) for t in (q, k, v, cos, sin))
    # (rows aligned already are rotated where they lie when out is q)
    o = None if q is None else torch.empty_like(q) if out is None or _crosses(out, q, k, v) else \
        _out_for(out, q.shape, q.dtype, q.device)
    _lib.call("paged_kv_append", k, v, k_cache, v_cache, block_tables, context_lens, q, o, cu_seqlens, cos, sin,
              int(bool(interleaved)))
    return o if out is None else _finish(out, o)
