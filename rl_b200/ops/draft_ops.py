"""Operators of speculative decoding over the paged key/value cache: the rows of trees of drafted tokens, their attention, the verification of the
drafted tokens against the target's logits, and the move of the accepted rows' keys and values to the places that they keep.

A step of a program that decodes this way: :func:`tree_rows` gives what each row sees, its position and its cache slot; every layer writes its rows'
keys and values (``rope_kv_cache_write`` of :mod:`rl_b200.ops.engine_ops`) and attends with :func:`tree_paged_decode`; :func:`verify_drafts` walks down the
trees on the logits of the rows; :func:`kv_cache_keep` moves what was accepted to the end of the context.

The rows of all sequences' trees lie one after the other: sequence ``b``'s are ``cu_rows[b]`` to ``cu_rows[b + 1]`` (int32 [B + 1], as ``cu_seqlens`` elsewhere), at most
``max_rows`` <= 256 of them; none for a padding row of the batch. Row 0 is the last token that is decided and not yet in the cache, the others are drafted. ``parents``
[T] int32 has the row, counted within the sequence, that a row continues: smaller than its own, -1 for row 0. ``ctx_lens`` [B] int32 tokens stand in the cache
before the tree; row ``j``'s key and value stand at place ``ctx_lens[b] + j`` of the pages that ``block_table`` [B, pages] int32 names.

On the GPU offsets that do not ascend, rows over ``max_rows``, parents that are not above their row, pages that are not there and places outside the table are left
out. The status word then has ``RLB_ERR_BOUNDS``: from :func:`tree_rows` for offsets, rows, parents and places, from :func:`verify_drafts` for offsets and rows, from
:func:`tree_paged_decode` for pages, from :func:`kv_cache_keep` for rows, pages and places. Where offsets that do not ascend have several sequences name a row, :func:`tree_paged_decode` gives it
the attention of one of them. CPU tensors run the PyTorch restatement. Everything here is for inference: nothing has a gradient.
"""

from __future__ import annotations

import ctypes as C
import math
from functools import lru_cache
from typing import Optional, Sequence

import torch

from . import lib as _L
from .lib import call, use_native

_P, _I, _LL, _F = _L.P, _L.I, _L.L, _L.F
_L.register("rlb_tree_rows", [_P, _P, _P, _P, _LL, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P])
_L.register("rlb_kv_keep", [_P, _I, _P, _LL, _I, _I, _I, _I, _I, _P, _P, _I, _P, _I, _P, _P])
_L.register("rlb_verify_drafts", [_P, _LL, _P, _LL, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P, _P, C.c_double, _I, _P, _P, _P, _P, _P, _P])
_L.register("rlb_tree_decode", [_P, _LL, _P, _P, _I, _I, _P, _LL, _I, _P, _P, _I, _I, _I, _I, _I, _I, _P, _LL, _P, _I, _F, _I, _I, _I, _P, _P, _P, _P, _LL, _P, _P])

BF16 = torch.bfloat16
HEAD_DIMS = (64, 128)
MAX_ROWS = 256
COLDEST = torch.finfo(torch.float32).tiny
MAX_SCALE = torch.finfo(torch.float32).max / 2      # (times log2(e) it has to be a number still)
MAX_VOCAB = 1 << 30
MAX_TOKENS = 0x7FFF0000      # of a sequence: places are 32-bit numbers
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda index: torch.cuda.current_stream(index).cuda_stream


def _same_device(device: torch.device, *ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on several devices: {device} and {t.device}")


def _launch(device: torch.device, name: str, *args) -> None:
    """Enqueues on the device's current stream, whichever device is the current one; the status word and the stream are the entry's last arguments."""
    index = device.index
    if torch.cuda.current_device() == index:
        call(name, *args, _L.status_word(device).data_ptr(), _raw_stream(index))
        return
    with torch.cuda.device(index):
        call(name, *args, _L.status_word(device).data_ptr(), _raw_stream(index))


def _ints(t: torch.Tensor, shape: tuple, what: str) -> torch.Tensor:
    if t.dtype is not torch.int32 or t.shape != shape:
        raise ValueError(f"{what} is int32 {list(shape)}, not {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def _rows_of(cu_rows: torch.Tensor, max_rows: int) -> int:
    """Sequences of the batch."""
    if cu_rows.dim() != 1 or cu_rows.dtype is not torch.int32 or cu_rows.numel() < 1:
        raise ValueError(f"cu_rows is int32 [B + 1], not {cu_rows.dtype} {tuple(cu_rows.shape)}")
    if not 1 <= max_rows <= MAX_ROWS:
        raise ValueError(f"max_rows is 1 to {MAX_ROWS}, not {max_rows}")
    return cu_rows.numel() - 1


def _table(block_table: torch.Tensor, B: int, block_size: int) -> torch.Tensor:
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype is not torch.int32:
        raise ValueError(f"block_table is int32 [{B}, pages], not {block_table.dtype} {tuple(block_table.shape)}")
    if block_size < 1 or block_table.shape[1] * block_size > MAX_TOKENS:
        raise ValueError(f"pages of {block_size} tokens, {block_table.shape[1]} to a sequence: the kernels count to {MAX_TOKENS}")
    return block_table if block_table.stride(1) == 1 else block_table.contiguous()


def _no_gradient(*ts: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise ValueError("speculative decoding has no gradient: call under torch.no_grad()")


def _spans(cu_rows: torch.Tensor, T: int, max_rows: int) -> list[tuple[int, int]]:
    """(first row, rows) of each sequence."""
    cu, got = cu_rows.tolist(), []
    for a, e in zip(cu[:-1], cu[1:]):
        lo = min(max(a, 0), T)
        got.append((lo, min(min(max(e, lo), T) - lo, max_rows)))
    return got


# --------------------------------------------------------------------------------------- rows
def tree_rows(parents: torch.Tensor, cu_rows: torch.Tensor, ctx_lens: torch.Tensor, block_table: torch.Tensor, block_size: int, *, max_rows: int,
              ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """What the layers need of the trees' rows: ``masks`` int32 [T, ceil(max_rows / 32)], in which bit ``i % 32`` of word ``i // 32`` says that a row sees row ``i`` of its
    sequence (itself and the rows that it continues); ``positions`` int32 [T], the context's length and the rows before it on its path; ``slots`` int64 [T], the
    cache places as ``rope_kv_cache_write`` takes them. Rows of no sequence (behind the last, before the first, over ``max_rows``) see nothing, with position 0 and slot -1 (which is skipped).
    Where offsets do not ascend, a row that several sequences name is the first one's."""
    B = _rows_of(cu_rows, max_rows)
    T, device, words = parents.shape[0] if parents.dim() == 1 else -1, parents.device, -(-max_rows // 32)
    parents = _ints(parents, (T,), "parents")
    _same_device(device, cu_rows, ctx_lens, block_table)
    table, ctx, cu = _table(block_table, B, block_size), _ints(ctx_lens, (B,), "ctx_lens"), cu_rows.contiguous()
    if not use_native(parents):
        masks, positions = torch.zeros((T, words), dtype=torch.int32), torch.zeros(T, dtype=torch.int32)
        slots = torch.full((T,), -1, dtype=torch.int64)
        room, taken = table.shape[1] * block_size, 0      # taken: rows before are earlier sequences'
        for b, (lo, n) in enumerate(_spans(cu, T, max_rows)):
            seen: list[int] = []
            taken = max(taken, min(int(cu[b]), T))
            for j in range(n):
                p, place = int(parents[lo + j]), int(ctx[b]) + j
                seen.append(1 << j | (seen[p] if 0 <= p < j else 0))
                if lo + j < taken:
                    continue
                for w in range(words):
                    x = seen[j] >> (32 * w) & 0xFFFFFFFF
                    masks[lo + j, w] = x - (1 << 32) if x >> 31 else x
                positions[lo + j] = int(ctx[b]) + bin(seen[j]).count("1") - 1
                if 0 <= place < room:
                    slots[lo + j] = int(table[b, place // block_size]) * block_size + place % block_size
        return masks, positions, slots
    masks, positions, slots = parents.new_empty((T, words)), parents.new_empty(T), parents.new_empty(T, dtype=torch.int64)
    _launch(device, "rlb_tree_rows", parents.data_ptr(), cu.data_ptr(), ctx.data_ptr(), table.data_ptr(), table.stride(0), table.shape[1], block_size, B, T, max_rows, words,
            masks.data_ptr(), positions.data_ptr(), slots.data_ptr())
    return masks, positions, slots


# --------------------------------------------------------------------------------------- attention
def _tree_decode_ref(q, k_cache, v_cache, table, ctx, spans, Hq, Hkv, D, masks, positions, window, scale, out):
    block, g = k_cache.shape[2], Hq // Hkv
    for b, (lo, n) in enumerate(spans):
        if n == 0:
            continue
        room = table.shape[1] * block
        c = min(max(int(ctx[b]), 0), room)
        keys = min(c + n, room)
        pages = table[b, : -(-keys // block)].long()
        there = (pages >= 0) & (pages < k_cache.shape[0])
        k, v = (torch.where(there[:, None, None, None], x[torch.where(there, pages, 0)], 0).transpose(0, 1).reshape(Hkv, -1, D)[:, :keys].float() for x in (k_cache, v_cache))
        i = torch.arange(keys) - c
        sees = (i < 0).expand(n, -1).clone()
        for j in range(n):
            for t in range(keys - c):
                sees[j, c + t] = bool(int(masks[lo + j, t // 32]) >> (t % 32) & 1) if masks is not None else t <= j
        if window:
            pos = positions[lo : lo + n].long().clamp(min=c)
            own = positions[lo : lo + n].long()
            sees &= pos[:, None] - torch.cat([torch.arange(c), own[: keys - c]]) < window
        sees &= there.repeat_interleave(block)[:keys]
        s = torch.einsum("nhgd,htd->hgnt", q[lo : lo + n, : Hq * D].reshape(n, Hkv, g, D).float() * scale, k)
        p = torch.softmax(s.masked_fill(~sees, float("-inf")), -1)
        p = torch.where(sees.any(-1)[:, None], p, 0.0)      # (rows that see nothing)
        finite = v.isfinite()
        o = torch.einsum("hgnt,htd->nhgd", p, torch.where(finite, v, 0))
        for t in (~finite).any(-1).any(0).nonzero().flatten().tolist():      # (a weight of zero times these is not zero)
            o[sees[:, t]] += torch.where(finite, 0, v)[:, t, None]
        out[lo : lo + n] = o.reshape(n, Hq * D).to(out.dtype)
    return out


@lru_cache(maxsize=4096)
def tree_plan(B: int, Hq: int, Hkv: int, D: int, max_rows: int, max_len: int, sm_count: int = 148) -> tuple[int, int]:
    """How :func:`tree_paged_decode` is cut up. A unit is a sequence, a key/value head and a block of 128 / (Hq / Hkv) rows of its tree; keys go by in tiles of 64. (0, 1): a CTA
    for each unit, the longest sequences' first. (n, 1): n CTAs share all tiles evenly, units one after another, and a second kernel joins what they cut through. (n, blocks): the CTAs of a
    sequence's blocks have the same tiles, so that its keys and values come from memory once.

    Two CTAs are on an SM at a time. With fewer units than that, sharing pays where the longest unit has six tiles more than a share (us in a graph, a CTA each / shared: one
    sequence of 1000 tokens, 8 KV heads of 128, trees of 8: 18.7 / 13.8; two of 500 13.1 / 13.7; 16 of 8000 with trees of 64 146 / 103). With more, sharing keeps the loads of the next unit on
    their way (128 of 1000, trees of 8: 83 / 73; 180 of 500 79 / 64; 64 of 1200 49 / 49), but for less than twice as many of 64 rows and more, whose parts are large
    (64 of 1280 with trees of 17, 4 query heads each: 52 / 56; 16 of 500 with trees of 128: 36 / 46). Blocks one after another read a sequence of 131072 tokens, trees of 33 with 5 query
    heads, twice from memory: 189, beside one another 154; where all keys stay in the second level cache there is no difference, and trees of fewer blocks leave CTAs without work."""
    blocks = -(-max_rows // (128 // (Hq // Hkv)))
    units, tiles, slots = B * Hkv * blocks, -(-max_len // 64), 2 * sm_count
    group = blocks if blocks <= 4 and B * Hkv * max_len * 4 * D > 2**27 else 1
    if units > slots:
        share = units > 2 * slots or min(max_rows, 128 // (Hq // Hkv)) * (Hq // Hkv) < 64
    else:
        share = tiles * (slots - units) > 6 * slots
    return (slots - slots % group, group) if share else (0, 1)


def tree_scratch_size(ctas: int, Hq: int, Hkv: int, D: int, max_rows: int) -> int:
    """Floats of the scratch tensor of :func:`tree_paged_decode` with this many CTAs."""
    return 2 * ctas * min(max_rows, 128 // (Hq // Hkv)) * (Hq // Hkv) * (D + 2) + 16 * ctas


def tree_paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, ctx_lens: torch.Tensor, cu_rows: torch.Tensor,
                      Hq: int, Hkv: int, D: int, *, max_rows: int, masks: Optional[torch.Tensor] = None, scale: Optional[float] = None, window: int = 0,
                      positions: Optional[torch.Tensor] = None, plan: Optional[tuple[int, int]] = None, scratch: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the trees' rows, ``q`` [T, >= Hq D] (rows may be strided: the fused rows do), against the paged cache [blocks, Hkv, block size, D], which holds their own
    keys and values behind the context. A row sees the whole context of its sequence and the tree rows whose bits ``masks`` (as :func:`tree_rows` gives them; any bits
    do) has set; without ``masks`` the rows up to itself, which is a chain. ``window`` > 0: of these only keys whose position is less than ``window`` before the row's own
    (sliding-window layers): ``positions`` [T] int32 has the rows' (from the context's end on), a context place's is its number. A row that sees nothing gives zeros. Rows of no sequence are left as
    they are in ``out`` (a new ``out`` has no values there). Heads of 64 and 128, at most 128 query heads to a key/value head, pages of a multiple of 16 tokens. ``plan``: as
    :func:`tree_plan` gives it (None: for the table's width); ``scratch``: float32 tensor of :func:`tree_scratch_size` elements, for callers that keep their own (one call at a
    time). Returns [T, Hq D].

    Scores, maxima and sums are in 32 bits, weights are rounded to bf16 before they meet the values."""
    B = _rows_of(cu_rows, max_rows)
    width, device = Hq * D, q.device
    if D not in HEAD_DIMS:
        raise ValueError(f"heads of {HEAD_DIMS} dimensions, not {D}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv or Hq // Hkv > 128 or q.dim() != 2 or q.shape[1] < width:
        raise ValueError(f"q is [T, {width}] with {Hq} heads, 1 to 128 times {Hkv}, not {tuple(q.shape)}")
    T, shape = q.shape[0], k_cache.shape
    if len(shape) != 4 or shape != v_cache.shape or shape[1] != Hkv or shape[3] != D or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError(f"the caches are contiguous [blocks, {Hkv}, block size, {D}], not {tuple(shape)} and {tuple(v_cache.shape)}")
    blocks, block = shape[0], shape[2]
    if block < 16 or block % 16:
        raise ValueError(f"pages hold a multiple of 16 tokens, not {block}")
    dtype = q.dtype
    if dtype != k_cache.dtype or dtype != v_cache.dtype:
        raise ValueError(f"queries and caches are of one type, not {q.dtype}, {k_cache.dtype} and {v_cache.dtype}")
    _same_device(device, k_cache, v_cache, block_table, ctx_lens, cu_rows, masks, positions, out)
    table, ctx, cu = _table(block_table, B, block), _ints(ctx_lens, (B,), "ctx_lens"), cu_rows.contiguous()
    if masks is not None:
        if masks.dtype is not torch.int32 or masks.dim() != 2 or masks.shape[0] != T or masks.shape[1] * 32 < max_rows:
            raise ValueError(f"masks is int32 [{T}, {-(-max_rows // 32)}], not {masks.dtype} {tuple(masks.shape)}")
        masks = masks if masks.stride(1) == 1 else masks.contiguous()
    if window < 0 or (window and positions is None):
        raise ValueError(f"window {window} is negative, or has no positions")
    window = min(window, MAX_TOKENS)
    if window:
        positions = _ints(positions, (T,), "positions")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not abs(scale) <= MAX_SCALE:
        raise ValueError(f"scale {scale} is no number of at most {MAX_SCALE}")
    _no_gradient(q, k_cache, v_cache)
    if out is None:
        out = q.new_empty((T, width))
    elif out.shape != (T, width) or out.dtype != q.dtype:
        raise ValueError(f"out is {q.dtype} [{T}, {width}], not {out.dtype} {tuple(out.shape)}")
    elif out.stride(1) != 1 or (T > 1 and out.stride(0) < width):
        raise ValueError(f"out has whole rows one after the other, not strides {out.stride()}")
    if T == 0 or B == 0:
        return out
    if not use_native(q):
        return _tree_decode_ref(q, k_cache, v_cache, table, ctx, _spans(cu, T, max_rows), Hq, Hkv, D, masks, positions, window, scale, out)
    if dtype is not BF16:
        raise ValueError(f"the kernels take bf16 queries and caches, not {q.dtype}")
    if (k_cache.data_ptr() | v_cache.data_ptr()) % 16 or blocks < 1 or blocks * Hkv * block > 0x7FFFFFFE or B > 65535 or Hkv * -(-max_rows // (128 // (Hq // Hkv))) > 65535:
        raise ValueError(f"caches {tuple(k_cache.shape)} start on 16 bytes and have some pages, and less than 2^31 - 1 places of all heads, for at most 65535 sequences, and units of a sequence")
    pages = table.shape[1]
    room = pages * block
    longest = min(room, window + max_rows) if window else room
    blocks_of = -(-max_rows // (128 // (Hq // Hkv)))
    ctas, group = tree_plan(B, Hq, Hkv, D, max_rows, longest) if plan is None else plan
    if not 0 <= ctas <= 65535 or group not in (1, blocks_of) or ctas % group or (group > 1 and not ctas):
        raise ValueError(f"plan {(ctas, group)} is neither (0, 1) nor up to 65535 CTAs in groups of 1 or {blocks_of}")
    if ctas and B * Hkv * blocks_of * (longest // 64 + 2) + 64 * ctas > 0x7FFFFFFF:
        ctas, group = 0, 1      # (more tiles than the kernel counts to)
    parts = sums = cuts = None
    if ctas:
        size = tree_scratch_size(ctas, Hq, Hkv, D, max_rows)
        if scratch is None:
            scratch = torch.empty(size, dtype=torch.float32, device=device)
        elif scratch.dtype is not torch.float32 or not scratch.is_contiguous() or scratch.numel() < size or scratch.data_ptr() % 32 or scratch.device != device:
            raise ValueError(f"scratch is a contiguous float32 tensor of {size} elements on {device} that starts on 32 bytes")
        cuts = scratch.data_ptr()
        parts = cuts + 64 * ctas
        sums = parts + (size - 16 * ctas) // (D + 2) * D * 4
    stride = q.stride()
    if stride[1] != 1 or stride[0] % 8 or stride[0] < width or q.data_ptr() % 16:      # rows that do not start on 16 bytes, or share places
        q = q[:, :width].clone(memory_format=torch.contiguous_format)
    _launch(device, "rlb_tree_decode", q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), blocks, block, table.data_ptr(), table.stride(0), pages,
            ctx.data_ptr(), cu.data_ptr(), B, T, max_rows, Hq, Hkv, D, _L.ptr(masks), masks.stride(0) if masks is not None else 0, _L.ptr(positions) if window else None,
            window, scale, ctas, group, 4, parts, sums, cuts, out.data_ptr(), out.stride(0))
    return out


# --------------------------------------------------------------------------------------- verification
def _rounded_down(x: float) -> float:
    f = torch.tensor(x, dtype=torch.float32)
    return float(f) if float(f) <= x else float(torch.nextafter(f, torch.tensor(-math.inf)))


def _usable(z: torch.Tensor) -> torch.Tensor:
    """Logits in 64 bits, -inf for what is not a number, the largest number for +inf."""
    z = z.double()
    return torch.where(z.isnan(), -math.inf, z).clamp(max=torch.finfo(torch.float32).max)


def _weights(z: torch.Tensor, temp: float) -> tuple[torch.Tensor, torch.Tensor]:
    """Probabilities and their logarithms in 64 bits; zeros and -inf where no number is above -inf."""
    z = _usable(z)
    top = z.max()
    if top == -math.inf:
        return torch.zeros_like(z), z
    e = torch.where((z == -math.inf) | (z < top - _rounded_down(1000 * math.log(2) * temp)), -math.inf, (z - top) / temp)
    logp = e - torch.log(torch.exp(e).sum())
    return torch.exp(logp), logp


def _verify_ref(logits, tokens, parents, spans, uniforms, draft, temps, greedy, steps, out):
    got_tokens, got_counts, got_rows, got_logprobs = out
    V = logits.shape[1]
    for b, (lo, n) in enumerate(spans):
        warm = torch.tensor(temps[b], dtype=torch.float32) >= COLDEST
        cold, temp = greedy or not warm, temps[b] if warm else 1.0
        node, step = 0, 0
        while n:
            p, logp = _weights(logits[lo + node], temp)
            some = bool(p.sum() > 0)
            best = int(torch.argmax(_usable(logits[lo + node]))) if some else 0
            q = _weights(draft[lo + node], temp)[0] if draft is not None and not cold else None
            w, left, went = p.clone(), 1.0, -1
            for j in range(node + 1, n) if step + 1 < steps else ():
                if int(parents[lo + j]) != node:
                    continue
                t, u = int(tokens[lo + j]), float(uniforms[lo + j])
                if cold:
                    if some and t == best:
                        went = j
                        break
                    continue
                if not 0 <= t < V:
                    continue
                if u * (float(q[t]) if q is not None else 1.0) * left < float(w[t]):
                    went = j
                    break
                if q is not None:
                    w = (w / left - q.clamp(min=2.0**-1000 * float(q.max()))).clamp_(min=0.0)
                    left = float(w.sum())
                    if not left > 0:
                        break
                else:
                    left -= float(w[t])
                    w[t] = 0.0
            if went >= 0:
                t = int(tokens[lo + went])
            elif cold or not some:
                t = best
            else:
                w = w if bool(w.sum() > 0) else p
                run = w.cumsum(0)
                over = ((run > float(uniforms[lo]) * run[-1]) & (w > 0)).nonzero()
                t = int(over[0]) if len(over) else int((w > 0).nonzero()[-1])
            got_rows[b, step], got_tokens[b, step] = node, t
            got_logprobs[b, step] = float(logp[t]) if some else -math.inf
            step += 1
            if went < 0:
                break
            node = went
        got_counts[b] = step
    return out


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, cu_rows: torch.Tensor, uniforms: torch.Tensor, *, max_rows: int,
                  draft_logits: Optional[torch.Tensor] = None, temperature: float = 1.0, temps: Optional[torch.Tensor] = None, greedy: bool = False,
                  max_steps: Optional[int] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accepts drafted tokens so that what is kept is distributed as the target's own samples. ``logits`` [T, V] (bf16 or fp32) of every row's next token, ``tokens`` [T] int32
    the rows' own tokens, ``uniforms`` [T] fp32 in [0, 1): a drafted row's number decides on it, row 0's draws the last token. ``temperature``, ``temps`` [B] fp32 and
    ``greedy`` as in :func:`rl_b200.ops.engine_ops.sample` (temperatures below 2^-126 are greedy too).

    From row 0 on, with p the target's probabilities at the node and w = p, Z = 1: the node's children are tried in order of their rows. Child c with token x and number u is
    accepted if u Z q(x) < w(x), and is the next node. Otherwise, with ``draft_logits`` [T, V] (the logits, at the same temperature, that a row's children were drawn from,
    independently), w becomes max(w / Z - q, 0) and Z its sum; without (children were taken without chance, each token once; q = 1) Z loses w(x) and x is out. Where no child
    is accepted, the last token is the first whose running sum of w passes row 0's number times the whole sum. Greedy: a child is accepted if its token has the largest logit (of equal ones the lowest), which is the last token too.
    Logits that are not numbers weigh nothing, nor does what is less than 2^-1000 of the largest (what the draft takes off a token is at least that); +inf as much as the largest number. At most ``max_steps`` tokens (None: ``max_rows``).

    Returns ``tokens`` int32 [B, max_steps] (accepted ones and the last; -1 behind them), ``counts`` int32 [B], ``rows`` int32 [B, max_steps] (row 0 and the accepted rows, as :func:`kv_cache_keep`
    takes them; -1 behind them) and ``logprobs`` fp32 [B, max_steps], the tokens' logarithms of p (0 behind them; -inf where no logit is above -inf, whose token is 0). Sums are in 64 bits, weights to 1.5e-13; on the GPU a draft's probabilities count as 2^-41 more, so
    that of tokens as probable in both nothing is left."""
    B = _rows_of(cu_rows, max_rows)
    if logits.dim() != 2 or logits.dtype not in (torch.float32, BF16) or not 1 <= logits.shape[1] <= MAX_VOCAB:
        raise ValueError(f"logits are fp32 or bf16 [T, V] with V up to 2^30, not {logits.dtype} {tuple(logits.shape)}")
    T, V = logits.shape
    device = logits.device
    if draft_logits is not None and (draft_logits.shape != logits.shape or draft_logits.dtype != logits.dtype):
        raise ValueError(f"draft_logits are {logits.dtype} [{T}, {V}], not {draft_logits.dtype} {tuple(draft_logits.shape)}")
    _same_device(device, tokens, parents, cu_rows, uniforms, draft_logits, temps)
    tokens, parents, cu = _ints(tokens, (T,), "tokens"), _ints(parents, (T,), "parents"), cu_rows.contiguous()
    for x, shape, what in ((uniforms, (T,), "uniforms"), (temps, (B,), "temps")):
        if x is not None and (x.dtype is not torch.float32 or x.shape != shape):
            raise ValueError(f"{what} is float32 {list(shape)}, not {x.dtype} {tuple(x.shape)}")
    if math.isnan(temperature):
        raise ValueError("temperature is not a number")
    steps = max_rows if max_steps is None else max_steps
    if not 1 <= steps <= max_rows:
        raise ValueError(f"max_steps is 1 to max_rows = {max_rows}, not {steps}")
    _no_gradient(logits, draft_logits)
    out = tokens.new_empty((B, steps)), tokens.new_empty(B), tokens.new_empty((B, steps)), uniforms.new_empty((B, steps))
    if B == 0:
        return out
    if not use_native(logits):
        for x, fill in zip(out, (-1, 0, -1, 0.0)):
            x.fill_(fill)
        each = temps.tolist() if temps is not None else [float(temperature)] * B
        return _verify_ref(logits, tokens, parents, _spans(cu, T, max_rows), uniforms, draft_logits, each, greedy, steps, out)
    logits = logits if logits.stride(1) == 1 else logits.contiguous()
    if draft_logits is not None and draft_logits.stride(1) != 1:
        draft_logits = draft_logits.contiguous()
    uniforms, temps = uniforms.contiguous(), None if temps is None else temps.contiguous()
    _launch(device, "rlb_verify_drafts", logits.data_ptr(), logits.stride(0), _L.ptr(draft_logits), draft_logits.stride(0) if draft_logits is not None else 0,
            int(logits.dtype is torch.float32), V, T, B, max_rows, steps, tokens.data_ptr(), parents.data_ptr(), cu.data_ptr(), uniforms.data_ptr(), _L.ptr(temps),
            float(temperature), int(greedy), *(x.data_ptr() for x in out))
    return out


# --------------------------------------------------------------------------------------- keep
def kv_cache_keep(caches: Sequence[tuple[torch.Tensor, torch.Tensor]], block_table: torch.Tensor, ctx_lens: torch.Tensor, rows: torch.Tensor, counts: torch.Tensor) -> None:
    """Moves the keys and values of accepted rows to the places that they keep, in the (keys, values) ``caches`` [blocks, heads, block size, D] of all layers: place
    ``ctx_lens[b] + i`` takes what stands at ``ctx_lens[b] + rows[b, i]``, for ``i < counts[b]``. ``rows`` and ``counts`` as :func:`verify_drafts` gives them: ``rows[b]`` ascends and
    ``rows[b, i] >= i`` (an entry that does not is left out). Layers without a cache are None, a cache that several layers share is moved once. Places of 16-byte multiples, any type."""
    if rows.dim() != 2:
        raise ValueError(f"rows is int32 [B, steps], not {rows.dtype} {tuple(rows.shape)}")
    B, S = rows.shape
    rows, counts, ctx = _ints(rows, (B, S), "rows"), _ints(counts, (B,), "counts"), _ints(ctx_lens, (B,), "ctx_lens")
    _same_device(rows.device, block_table, counts, ctx)
    kinds: dict[tuple, dict[int, torch.Tensor]] = {}
    last, places, grad = None, {}, torch.is_grad_enabled()
    for pair in caches:
        for x in pair if pair is not None else ():
            if x is None:
                continue
            at, kind = x.data_ptr(), (x.shape, x.dtype)
            if kind != last:
                if x.dim() != 4 or x.shape[3] * x.element_size() % 16:
                    raise ValueError(f"caches are [blocks, heads, block size, D] in places of 16 bytes, not {x.dtype} {tuple(x.shape)}")
                last = kind
                places = kinds.setdefault((x.shape[0], x.shape[1], x.shape[2], x.shape[3] * x.element_size() // 16), {})
            if at % 16 or not x.is_contiguous() or x.device != rows.device or (grad and x.requires_grad):
                raise ValueError(f"caches are contiguous, start on 16 bytes, lie on {rows.device} and have no gradient, not {x.dtype} {tuple(x.shape)} on {x.device}")
            places[at] = x
    for (blocks, heads, block, vecs), tensors in kinds.items():
        table = _table(block_table, B, block)
        if B == 0 or blocks == 0:
            continue
        one = next(iter(tensors.values()))
        if not use_native(one):
            room = table.shape[1] * block
            for b in range(B):
                c, last = int(ctx[b]), -1
                for i in range(min(int(counts[b]), S)):
                    r = int(rows[b, i])
                    if r <= last or r < i:
                        continue
                    last = r
                    if r == i or not (0 <= c + i and c + r < room):
                        continue
                    to, source = int(table[b, (c + i) // block]), int(table[b, (c + r) // block])
                    if not (0 <= to < blocks and 0 <= source < blocks):
                        continue
                    for x in tensors.values():
                        x[to, :, (c + i) % block] = x[source, :, (c + r) % block]
            continue
        _launch(one.device, "rlb_kv_keep", (C.c_void_p * len(tensors))(*tensors), len(tensors), table.data_ptr(), table.stride(0), table.shape[1], block, blocks, heads, vecs,
                ctx.data_ptr(), rows.data_ptr(), S, counts.data_ptr(), B)
