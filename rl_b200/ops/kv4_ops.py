"""Operators of the generation engine's 4-bit key/value cache (``kv_cache_dtype: int4``): the write behind the q/k/v projection with the rotary
embedding applied on the way, the read-back that prefix reuse and chunked prefill need, and decode attention over the pages.

The cache is a uint8 tensor [num_blocks, Hkv, page bytes]. A page holds ``block_size`` tokens of one key/value head: 4-bit codes of the keys, of the
values, and a bf16 scale per group of 32 consecutive dimensions of a token. With ``a`` a group's largest magnitude, its scale is ``s = bf16(a / 7.5)``
(0 where ``a < 2^-100``; NaN where a value of the group is not finite) and the code of ``x`` is ``clamp(floor(x / s) + 8, 0, 15)``, which stands for
``(code - 7.5) * s``. 4.5 bits a value: 3.6 times the tokens of a bf16 cache in the same memory. ``csrc/kv4.cuh`` has the order of the codes in a page.

Head dimensions 64, 128 and 256, pages of a multiple of 16 tokens, any number of query heads to a key/value head. bf16 rows on the GPU; CPU tensors run
the PyTorch restatement. The cache is for inference: nothing here has a gradient.
"""

from __future__ import annotations

import math
from contextlib import nullcontext
from typing import Optional

import torch

from . import lib as _L
from .lib import call, ptr, stream_ptr, use_native

_P, _I, _LL, _F = _L.P, _L.I, _L.L, _L.F
_L.register("rlb_rope_kv4_cache_write", [_P, _P, _P, _P, _P, _LL, _I, _I, _I, _I, _LL, _LL, _P, _P])
_L.register("rlb_kv4_cache_read", [_P, _P, _P, _P, _LL, _LL, _LL, _I, _I, _I, _LL, _P, _P])
_L.register("rlb_kv4_paged_decode", [_P, _LL, _P, _LL, _P, _LL, _I, _P, _I, _I, _I, _I, _I, _I, _F, _I, _P, _P, _P, _LL, _P, _P])

BF16 = torch.bfloat16
HEAD_DIMS = (64, 128, 256)
GROUP = 32
TINY = 2.0 ** -100
MAX_BLOCK = 65536


def kv4_page_bytes(block_size: int, D: int) -> int:
    """Bytes of a page of ``block_size`` tokens of one key/value head."""
    if D not in HEAD_DIMS:
        raise ValueError(f"the 4-bit cache holds heads of {HEAD_DIMS} dimensions, not {D}")
    if block_size < 16 or block_size % 16 or block_size > MAX_BLOCK:
        raise ValueError(f"pages of the 4-bit cache hold a multiple of 16 tokens up to {MAX_BLOCK}, not {block_size}")
    return block_size * D * 9 // 8


def kv4_cache(num_blocks: int, Hkv: int, block_size: int, D: int, device) -> torch.Tensor:
    """An empty cache (every place holds zeros)."""
    return torch.zeros((num_blocks, Hkv, kv4_page_bytes(block_size, D)), dtype=torch.uint8, device=device)


def _block_size(cache: torch.Tensor, Hkv: int, D: int) -> int:
    """Tokens of a page, from its bytes; refuses what is not a cache of this shape."""
    if D not in HEAD_DIMS:
        raise ValueError(f"the 4-bit cache holds heads of {HEAD_DIMS} dimensions, not {D}")
    if cache.dtype != torch.uint8 or cache.dim() != 3 or not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError("the 4-bit cache is a contiguous uint8 tensor [blocks, heads, page bytes] that starts on 16 bytes")
    size = cache.shape[2] * 8 // (9 * D)
    if cache.shape[1] != Hkv or size < 16 or kv4_page_bytes(size - size % 16, D) != cache.shape[2]:
        raise ValueError(f"cache {tuple(cache.shape)} does not hold pages of {Hkv} heads of {D} dimensions")
    return size


def _same_device(*ts: Optional[torch.Tensor]) -> None:
    devices = {t.device for t in ts if t is not None}
    if len(devices) > 1:
        raise ValueError(f"tensors on several devices: {sorted(map(str, devices))}")


def _on(device: torch.device):
    """Kernels go to the current stream of the tensors' device, whichever device is current."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _index(t: torch.Tensor, dtype: torch.dtype, n: int, what: str) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != n or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what} is a vector of {n} integers, not {t.dtype} {tuple(t.shape)}")
    return t.to(dtype).contiguous()


# --------------------------------------------------------------------------------------- PyTorch restatement
def quantize_ref(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., D] -> codes uint8 [..., D / 32, 32] and bf16 scales [..., D / 32]."""
    g = x.double().unflatten(-1, (-1, GROUP))
    a = g.abs().amax(-1)
    s = (a / 7.5).to(BF16)
    s = torch.where(a < TINY, torch.zeros_like(s), s)
    s = torch.where(torch.isfinite(g).all(-1), s, torch.full_like(s, math.nan))
    d = s.double().unsqueeze(-1)
    c = torch.where((d > 0) & torch.isfinite(d), torch.floor(g / d) + 8, torch.full_like(g, 8.0))
    return c.clamp(0, 15).to(torch.uint8), s


def _pack_pages(kc, vc, ks, vs) -> torch.Tensor:
    """Codes [..., block, G, 32] and scales [..., block, G] of whole pages -> their bytes."""
    *lead, block, G, _ = kc.shape
    k = kc.unflatten(-1, (4, 2, 4)).transpose(-4, -3)
    n = len(lead)
    v = vc.unflatten(-1, (8, 4)).unflatten(n, (block // 2, 2))                # [.., pairs, 2, G, 8, 4]
    v = v.permute(*range(n), n, n + 3, n + 2, n + 1, n + 4)
    codes = [(u[..., 0::2] | u[..., 1::2] << 4).reshape(*lead, -1) for u in (k, v)]
    s = torch.stack([ks, vs], -2).contiguous().view(torch.uint8).reshape(*lead, -1)
    return torch.cat([*codes, s], -1)


def _unpack_pages(pages: torch.Tensor, D: int) -> tuple[torch.Tensor, ...]:
    """Bytes of pages [..., bytes] -> codes of keys and values [..., block, G, 32], scales [..., block, G]."""
    *lead, size = pages.shape
    block, G = size * 8 // (9 * D), D // GROUP
    n, at = block * D // 2, len(lead)
    nib = torch.stack([pages[..., : 2 * n] & 15, pages[..., : 2 * n] >> 4], -1).reshape(*lead, 2, -1)
    k = nib.select(-2, 0).reshape(*lead, block, 4, G, 2, 4).transpose(-4, -3).reshape(*lead, block, G, GROUP)
    v = nib.select(-2, 1).reshape(*lead, block // 2, 8, G, 2, 4)
    v = v.permute(*range(at), at, at + 3, at + 2, at + 1, at + 4).reshape(*lead, block, G, GROUP)
    s = pages[..., 2 * n :].contiguous().view(BF16).reshape(*lead, block, 2, G)
    return k, v, s[..., 0, :], s[..., 1, :]


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    return ((codes.float() - 7.5) * scales.float().unsqueeze(-1)).flatten(-2)


def _rotate_ref(x: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor) -> torch.Tensor:
    """[T, heads, D]: angles in 64 bits, sines and cosines rounded to 32, products and sums in 32."""
    a = positions.double()[:, None] * inv_freq.double()
    c, s = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    lo, hi = x.float().chunk(2, -1)
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1).to(x.dtype)


# --------------------------------------------------------------------------------------- operators
def rope_kv4_cache_write(qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, slots: torch.Tensor, cache: torch.Tensor,
                         Hq: int, Hkv: int, D: int) -> torch.Tensor:
    """Rotary embedding of the q and k heads of fused rows [T, (Hq + 2 Hkv) D] (in place on CUDA) and the write of the rotated k and of v into the
    4-bit ``cache``, in one launch; returns the rotated fused rows. ``slots`` [T]: block * block_size + offset of each token (negative: rotate only);
    the slots of one call differ from each other. The angles are taken in 64 bits, whatever the position."""
    block = _block_size(cache, Hkv, D)
    T = qkv.shape[0]
    if qkv.dim() != 2 or qkv.shape[1] != (Hq + 2 * Hkv) * D:
        raise ValueError(f"qkv is [T, {(Hq + 2 * Hkv) * D}], not {tuple(qkv.shape)}")
    if inv_freq.dtype != torch.float32 or inv_freq.shape != (D // 2,):
        raise ValueError(f"inv_freq is a float32 vector of {D // 2}, not {inv_freq.dtype} {tuple(inv_freq.shape)}")
    _same_device(qkv, positions, inv_freq, slots, cache)
    positions, slots = _index(positions, torch.int32, T, "positions"), _index(slots, torch.int64, T, "slots")
    if not use_native(qkv):
        out = qkv.clone()
        out[:, : (Hq + Hkv) * D] = _rotate_ref(qkv[:, : (Hq + Hkv) * D].reshape(T, Hq + Hkv, D), positions, inv_freq).reshape(T, -1)
        ok = slots >= 0
        blk, off = slots[ok] // block, slots[ok] % block
        kv = out[ok][:, Hq * D :].reshape(-1, 2, Hkv, D)
        codes, scales = quantize_ref(kv)
        for b in blk.unique().tolist():
            kc, vc, ks, vs = _unpack_pages(cache[b], D)
            mine = blk == b
            at = off[mine]
            kc[:, at], vc[:, at] = codes[mine][:, 0].transpose(0, 1), codes[mine][:, 1].transpose(0, 1)
            ks[:, at], vs[:, at] = scales[mine][:, 0].transpose(0, 1), scales[mine][:, 1].transpose(0, 1)
            cache[b] = _pack_pages(kc, vc, ks, vs)
        return out
    if qkv.dtype != BF16:
        raise ValueError(f"the 4-bit cache takes bf16 rows, not {qkv.dtype}")
    rows = qkv
    if qkv.stride(1) != 1 or qkv.stride(0) % 8 or qkv.data_ptr() % 16:      # rows that do not start on 16 bytes: turned in a copy
        rows = qkv.clone(memory_format=torch.contiguous_format)
    with _on(qkv.device):
        call("rlb_rope_kv4_cache_write", ptr(rows), ptr(positions), ptr(inv_freq.contiguous()), ptr(slots), ptr(cache), T, Hq, Hkv, D, block,
             rows.stride(0), cache.shape[0], ptr(_L.status_word(qkv.device)), stream_ptr())
        if rows is not qkv:
            qkv.copy_(rows)
    return qkv


def kv4_cache_read(cache: torch.Tensor, slots: torch.Tensor, Hkv: int, D: int, *, out: Optional[torch.Tensor] = None,
                   rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keys and values of the tokens at ``slots`` [n] as bf16 rows [k heads | v heads]. ``out`` [m, >= 2 Hkv D]: where they go (its other columns
    stay); ``rows`` [n]: token i goes to row ``rows[i]`` of ``out`` (None: row i), each row named once. A negative slot gives a row of zeros."""
    block = _block_size(cache, Hkv, D)
    n, width = slots.shape[0], 2 * Hkv * D
    _same_device(cache, slots, out, rows)
    slots = _index(slots, torch.int64, n, "slots")
    if rows is not None:
        if out is None:
            raise ValueError("rows name rows of out: give both")
        rows = _index(rows, torch.int64, n, "rows")
    if out is None:
        out = torch.empty((n, width), dtype=BF16, device=cache.device)
    elif out.dim() != 2 or out.shape[1] < width or (rows is None and out.shape[0] < n):
        raise ValueError(f"out {tuple(out.shape)} has no room for {n} rows of {width}")
    if not use_native(cache):
        kc, vc, ks, vs = _unpack_pages(cache[(slots // block).clamp(min=0)], D)      # [n, Hkv, block, ...]
        ar, off = torch.arange(n), slots.clamp(min=0) % block
        kv = torch.stack([_values(kc, ks)[ar, :, off], _values(vc, vs)[ar, :, off]], 1).reshape(n, width)
        kv = torch.where(slots[:, None] < 0, torch.zeros_like(kv), kv)
        out[torch.arange(n) if rows is None else rows, :width] = kv.to(out.dtype)
        return out
    if out.dtype != BF16:
        raise ValueError(f"the 4-bit cache is read into bf16 rows, not {out.dtype}")
    to = out
    if out.stride(1) != 1 or out.stride(0) % 8 or out.data_ptr() % 16:      # rows that do not start on 16 bytes: read into a copy
        to = out.clone(memory_format=torch.contiguous_format)
        if to.stride(0) % 8:
            to = torch.empty((out.shape[0], -(-out.shape[1] // 8) * 8), dtype=BF16, device=out.device)[:, : out.shape[1]].copy_(out)
    with _on(cache.device):
        call("rlb_kv4_cache_read", ptr(cache), ptr(slots), ptr(rows), ptr(to), n, to.stride(0), to.shape[0], Hkv, D, block, cache.shape[0],
             ptr(_L.status_word(cache.device)), stream_ptr())
        if to is not out:
            out.copy_(to)
    return out


def kv4_splits(B: int, Hq: int, Hkv: int, max_len: int, sm_count: int = 148) -> int:
    """KV splits of decode attention over the 4-bit cache: as many CTAs as the device holds at a time, no split of less than 256 tokens."""
    ctas = max(1, B) * Hkv * -(-(Hq // Hkv) // 8)
    return int(max(1, min(4 * sm_count // ctas, max_len // 256, 128)))


def kv4_scratch_sizes(B: int, Hq: int, num_splits: int, D: int) -> tuple[int, int]:
    """Floats of the two scratch tensors of :func:`kv4_paged_decode` with this many splits."""
    return B * Hq * num_splits * D, B * Hq * num_splits * 2


def kv4_paged_decode(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, Hq: int, Hkv: int, D: int, *,
                     scale: Optional[float] = None, window: int = 0, num_splits: int = 0,
                     scratch: Optional[tuple[torch.Tensor, torch.Tensor]] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per sequence, ``q`` [B, >= Hq D] (rows may be strided: the fused rows do), against the 4-bit ``cache``:
    ``seq_lens`` [B] int32 tokens in the pages that ``block_table`` [B, pages] int32 names, of which ``window`` > 0 leaves the last ``window``. A
    sequence without tokens gives zeros. ``num_splits``: parts that a sequence's tokens are cut into (0: by :func:`kv4_splits` from the table's width);
    ``scratch``: fp32 tensors of :func:`kv4_scratch_sizes` elements, for callers that keep their own. Returns [B, Hq D]."""
    block = _block_size(cache, Hkv, D)
    B = q.shape[0]
    if Hq < 1 or Hq % Hkv or q.dim() != 2 or q.shape[1] < Hq * D:
        raise ValueError(f"q is [B, {Hq * D}] with {Hq} heads, a multiple of {Hkv}, not {tuple(q.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] != B or seq_lens.shape != (B,):
        raise ValueError(f"block_table is [{B}, pages] and seq_lens [{B}], not {tuple(block_table.shape)} and {tuple(seq_lens.shape)}")
    if any(t.dtype not in (torch.int32, torch.int64) for t in (block_table, seq_lens)):
        raise ValueError("block_table and seq_lens are integers")
    if window < 0:
        raise ValueError(f"window {window} is negative")
    _same_device(q, cache, block_table, seq_lens, out, *(scratch or ()))
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, Hq * D), dtype=q.dtype, device=q.device)
    elif out.shape != (B, Hq * D) or out.dtype != q.dtype:
        raise ValueError(f"out is {q.dtype} [{B}, {Hq * D}], not {out.dtype} {tuple(out.shape)}")
    if not use_native(q):
        for b in range(B):
            n = int(seq_lens[b])
            if n <= 0:
                out[b] = 0
                continue
            lo = max(0, n - window) if window else 0
            kc, vc, ks, vs = _unpack_pages(cache[block_table[b, : -(-n // block)].long()].transpose(0, 1), D)
            k, v = (_values(c, s).flatten(1, 2)[:, lo:n] for c, s in ((kc, ks), (vc, vs)))
            p = torch.softmax(q[b, : Hq * D].reshape(Hkv, Hq // Hkv, D).float() * scale @ k.transpose(1, 2), dim=-1)
            out[b] = (p @ v).reshape(Hq * D).to(out.dtype)
        return out
    if q.dtype != BF16:
        raise ValueError(f"the 4-bit cache takes bf16 queries, not {q.dtype}")
    if q.stride(1) != 1 or q.stride(0) % 8 or q.data_ptr() % 16:      # rows that do not start on 16 bytes
        q = q[:, : Hq * D].clone(memory_format=torch.contiguous_format)
    table = block_table.to(torch.int32)
    if table.stride(1) != 1:
        table = table.contiguous()
    lens = seq_lens.to(torch.int32).contiguous()
    num_splits = num_splits or kv4_splits(B, Hq, Hkv, table.shape[1] * block)
    if num_splits < 1:
        raise ValueError(f"num_splits {num_splits} is negative")
    to = out if out.stride(1) == 1 and out.stride(0) % 4 == 0 and out.data_ptr() % 8 == 0 else torch.empty((B, Hq * D), dtype=BF16, device=q.device)
    with _on(q.device):
        po = pml = None
        if num_splits > 1:
            no, nml = kv4_scratch_sizes(B, Hq, num_splits, D)
            po, pml = scratch if scratch is not None else (torch.empty(no, dtype=torch.float32, device=q.device),
                                                           torch.empty(nml, dtype=torch.float32, device=q.device))
            if any(t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < size for t, size in ((po, no), (pml, nml))):
                raise ValueError(f"scratch is two contiguous float32 tensors of {no} and {nml} elements")
        call("rlb_kv4_paged_decode", ptr(q), q.stride(0), ptr(cache), cache.shape[0], ptr(table), table.stride(0), table.shape[1], ptr(lens), B, Hq, Hkv,
             D, block, window, scale, num_splits, ptr(po), ptr(pml), ptr(to), to.stride(0), ptr(_L.status_word(q.device)), stream_ptr())
        if to is not out:
            out.copy_(to)
    return out
