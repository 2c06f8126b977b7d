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
from functools import lru_cache
from typing import Optional

import torch

from . import lib as _L
from .lib import call, ptr, use_native

_P, _I, _LL, _F = _L.P, _L.I, _L.L, _L.F
_L.register("rlb_rope_kv4_cache_write", [_P, _P, _P, _P, _P, _LL, _I, _I, _I, _I, _LL, _LL, _P, _P])
_L.register("rlb_kv4_cache_read", [_P, _P, _P, _P, _LL, _LL, _LL, _I, _I, _I, _LL, _P, _P])
_L.register("rlb_kv4_paged_decode", [_P, _LL, _P, _LL, _P, _LL, _I, _P, _I, _I, _I, _I, _I, _I, _F, _I, _I, _P, _P, _P, _LL, _P, _P])

BF16 = torch.bfloat16
HEAD_DIMS = (64, 128, 256)
GROUP = 32
TINY = 2.0 ** -100
MAX_BLOCK = 65536
MAX_CLUSTER = 8
MAX_SCALE = torch.finfo(torch.float32).max
MAX_TOKENS = 0x7FFF0000      # of a sequence: places are 32-bit numbers, with room for the steps that are requested ahead
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else lambda index: torch.cuda.current_stream(index).cuda_stream


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


@lru_cache(maxsize=256)
def _page_tokens(page_bytes: int, D: int) -> int:
    """Tokens of a page of so many bytes; 0 where no page has as many."""
    if D not in HEAD_DIMS:
        raise ValueError(f"the 4-bit cache holds heads of {HEAD_DIMS} dimensions, not {D}")
    size = page_bytes * 8 // (9 * D)
    return size if 16 <= size <= MAX_BLOCK and size % 16 == 0 and size * D * 9 // 8 == page_bytes else 0


def block_size_of(cache: torch.Tensor, Hkv: int, D: int) -> int:
    """Tokens of a page, from its bytes; refuses what is not a cache of this shape."""
    shape = cache.shape
    if cache.dtype is not torch.uint8 or len(shape) != 3 or not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError("the 4-bit cache is a contiguous uint8 tensor [blocks, heads, page bytes] that starts on 16 bytes")
    size = _page_tokens(shape[2], D)
    if shape[1] != Hkv or Hkv < 1 or not size:
        raise ValueError(f"cache {tuple(shape)} does not hold pages of {Hkv} heads of {D} dimensions")
    return size


def _same_device(device: torch.device, *ts: torch.Tensor) -> None:
    for t in ts:
        if t.device != device:
            raise ValueError(f"tensors on several devices: {device} and {t.device}")


def _index(t: torch.Tensor, dtype: torch.dtype, shape: tuple, what: str) -> torch.Tensor:
    if t.shape != shape or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{what} is an integer tensor {shape}, not {t.dtype} {tuple(t.shape)}")
    return t if t.dtype is dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _aligned(t: torch.Tensor) -> bool:
    """Whether the kernels can move these rows 16 bytes at a time."""
    stride = t.stride()
    return stride[1] == 1 and stride[0] % 8 == 0 and t.data_ptr() % 16 == 0


def _apart(t: torch.Tensor, width: int) -> bool:
    """Whether rows that lie one after the other are written, none of which reaches into the next."""
    stride = t.stride()
    return stride[1] == 1 and (t.shape[0] < 2 or stride[0] >= width)


def _refuse_overlap(t: torch.Tensor, width: int) -> None:
    """Refuses rows that are written where two numbers have one place: numbers (i, j) and (k, l) with (i - k) a = (l - j) b for the strides a and b, first at b / g rows and a / g
    columns with g the greatest common divisor."""
    a, b = t.stride()
    n = t.shape[0]
    g = math.gcd(a, b)
    if (n > b // g and width > a // g) if a and b else (n > 1 and not a) or (width > 1 and not b):
        raise RuntimeError(f"rows {n} x {width} with strides ({a}, {b}) share places: nothing is written to rows that overlap")


def _no_gradient(t: torch.Tensor) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("the 4-bit cache has no gradient: call under torch.no_grad()")


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
    the slots of one call differ from each other. The angles are taken in 64 bits, whatever the (32-bit) position; the policy's own passes and the write of a bf16 cache take them in
    32 bits (``elementwise.cu``, ``paged_attention.cu``), which is half a unit in the last place of the angle away: 0.001 near position 32768, 0.004 near 131072, on the pairs that turn
    fastest."""
    block = block_size_of(cache, Hkv, D)
    if qkv.dim() != 2 or Hq < 0 or qkv.shape[1] != (Hq + 2 * Hkv) * D:
        raise ValueError(f"qkv is [T, {(Hq + 2 * Hkv) * D}], not {tuple(qkv.shape)}")
    if inv_freq.dtype is not torch.float32 or inv_freq.shape != (D // 2,):
        raise ValueError(f"inv_freq is a float32 vector of {D // 2}, not {inv_freq.dtype} {tuple(inv_freq.shape)}")
    T = qkv.shape[0]
    _no_gradient(qkv)
    _same_device(qkv.device, positions, inv_freq, slots, cache)
    positions, slots = _index(positions, torch.int32, (T,), "positions"), _index(slots, torch.int64, (T,), "slots")
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
    if qkv.dtype is not BF16:
        raise ValueError(f"the 4-bit cache takes bf16 rows, not {qkv.dtype}")
    index = qkv.device.index
    if torch.cuda.current_device() != index:      # kernels go to the current stream of the tensors' device, whichever device is current
        with torch.cuda.device(qkv.device):
            return rope_kv4_cache_write(qkv, positions, inv_freq, slots, cache, Hq, Hkv, D)
    rows = qkv
    if not (_aligned(qkv) and _apart(qkv, qkv.shape[1])):      # rows that do not start on 16 bytes: turned in a copy
        _refuse_overlap(qkv, qkv.shape[1])
        rows = qkv.clone(memory_format=torch.contiguous_format)
    inv_freq = inv_freq.contiguous()
    call("rlb_rope_kv4_cache_write", rows.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), slots.data_ptr(), cache.data_ptr(), T, Hq, Hkv, D, block,
         rows.stride(0), cache.shape[0], _L.status_word(qkv.device).data_ptr(), _raw_stream(index))
    if rows is not qkv:
        qkv.copy_(rows)
    return qkv


def kv4_cache_read(cache: torch.Tensor, slots: torch.Tensor, Hkv: int, D: int, *, out: Optional[torch.Tensor] = None,
                   rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keys and values of the tokens at ``slots`` [n] as bf16 rows [k heads | v heads]. ``out`` [m, >= 2 Hkv D]: where they go (its other columns
    stay); ``rows`` [n]: token i goes to row ``rows[i]`` of ``out`` (None: row i), each row named once. A negative slot gives a row of zeros."""
    block = block_size_of(cache, Hkv, D)
    n, width, device = slots.numel(), 2 * Hkv * D, cache.device
    _same_device(device, slots)
    slots = _index(slots, torch.int64, (n,), "slots")
    if rows is not None:
        if out is None:
            raise ValueError("rows name rows of out: give both")
        _same_device(device, rows)
        rows = _index(rows, torch.int64, (n,), "rows")
    if out is None:
        out = torch.empty((n, width), dtype=BF16, device=device)
    elif out.dim() != 2 or out.shape[1] < width or (rows is None and out.shape[0] < n):
        raise ValueError(f"out {tuple(out.shape)} has no room for {n} rows of {width}")
    else:
        _same_device(device, out)
        if not _apart(out, width):
            _refuse_overlap(out, width)
    if not use_native(cache):
        kc, vc, ks, vs = _unpack_pages(cache[(slots // block).clamp(min=0)], D)      # [n, Hkv, block, ...]
        ar, off = torch.arange(n, device=device), slots.clamp(min=0) % block
        kv = torch.stack([_values(kc, ks)[ar, :, off], _values(vc, vs)[ar, :, off]], 1).reshape(n, width)
        kv = torch.where(slots[:, None] < 0, torch.zeros_like(kv), kv)
        out[ar if rows is None else rows, :width] = kv.to(out.dtype)
        return out
    if out.dtype is not BF16:
        raise ValueError(f"the 4-bit cache is read into bf16 rows, not {out.dtype}")
    index = device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(device):
            return kv4_cache_read(cache, slots, Hkv, D, out=out, rows=rows)
    to = out
    if not (_aligned(out) and _apart(out, width)):      # rows that do not start on 16 bytes: read into a copy
        to = torch.empty((out.shape[0], width), dtype=BF16, device=device).copy_(out[:, :width])
    call("rlb_kv4_cache_read", cache.data_ptr(), slots.data_ptr(), ptr(rows), to.data_ptr(), n, to.stride(0), to.shape[0], Hkv, D, block, cache.shape[0],
         _L.status_word(device).data_ptr(), _raw_stream(index))
    if to is not out:
        out[:, :width] = to
    return out


@lru_cache(maxsize=4096)
def kv4_plan(B: int, Hq: int, Hkv: int, D: int, max_len: int, sm_count: int = 148) -> tuple[int, int]:
    """How decode attention over the 4-bit cache is cut up: (cluster, 0): a cluster of CTAs per sequence and key/value head (with up to eight query
    heads), or (1, n): n CTAs, as many as the device holds, share all tokens evenly, and a second kernel joins what they cut through.

    A cluster of twice the CTAs is taken while they run at once and keep six steps of 32 tokens each, eight more in all where some SMs get two (us in a graph with one,
    two, four, eight CTAs: one sequence of 1200 tokens with 8 KV heads of 128 10.6, 8.6, 7.3, 7.1; 12 of 600 7.3, 8.3, 8.0, 14.5; 26 of 2400 with 4 heads
    21.0, 17.8, 15.6; 48 of 2400 26.6, 22.5, 28.5). Sharing has its search and its join, some 5 us, and pays off from 50 steps per CTA on (8 heads of 128, best cluster /
    shared: one sequence of 4800 tokens 9.7 / 10.7, of 40000 36 / 23; 64 of 4000 71 / 67, of 16000 255 / 214), where there are at most two CTAs for each that
    the device holds (128 of 4000: 112 / 120); with two CTAs an SM where they would get less than 20 steps otherwise (one of 19200: 15.9, all places 18.8). Of 732
    calls with 8 to 384 sequences times heads the mean is 1.0 % above the best of five choices, the worst 20 %."""
    segments, steps = max(1, B) * Hkv * -(-(Hq // Hkv) // 8), -(-max_len // 32)
    slots = (4 if D == 64 else 3 if D == 128 else 2) * sm_count
    cluster = 1
    while cluster < MAX_CLUSTER and 2 * cluster * segments <= slots and steps >= 12 * cluster + (8 if 2 * cluster * segments > sm_count else 0):
        cluster *= 2
    if steps >= max(100, 50 * cluster) and segments < 2 * slots and segments * (steps + 2) < 2**30:
        return 1, 2 * sm_count if segments * steps < 20 * slots else slots
    return cluster, 0


def kv4_scratch_size(num_ctas: int, D: int) -> int:
    """Floats of the scratch tensor of :func:`kv4_paged_decode` with this many CTAs."""
    return num_ctas * (16 * D + 36)


def kv4_paged_decode(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, Hq: int, Hkv: int, D: int, *,
                     scale: Optional[float] = None, window: int = 0, plan: Optional[tuple[int, int]] = None,
                     scratch: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per sequence, ``q`` [B, >= Hq D] (rows may be strided: the fused rows do), against the 4-bit ``cache``:
    ``seq_lens`` [B] int32 tokens in the pages that ``block_table`` [B, pages] int32 names, of which ``window`` > 0 leaves the last ``window``. A
    sequence without tokens gives zeros. ``plan``: (cluster, num_ctas): a cluster of up to eight CTAs per sequence and key/value head, or with (1, n) n CTAs
    that share all tokens evenly (None: :func:`kv4_plan` for the table's width); ``scratch``: float32 tensor of :func:`kv4_scratch_size` elements, for callers that
    keep their own (one call at a time). Returns [B, Hq D].

    Scores and sums are in 32 bits, a weight times a value's scale is rounded to bf16. A token's share of a group of 32 dimensions keeps these eight bits where weight times
    scale (weights: 1 for the largest) is at least 2^-100 and 2^-80 of the head's largest scale in that sequence."""
    block = block_size_of(cache, Hkv, D)
    device, width = q.device, Hq * D
    if Hq < 1 or Hq % Hkv or q.dim() != 2 or q.shape[1] < width:
        raise ValueError(f"q is [B, {width}] with {Hq} heads, a multiple of {Hkv}, not {tuple(q.shape)}")
    if window < 0 or (scale is not None and not abs(scale) <= MAX_SCALE):
        raise ValueError(f"window {window} is negative, or scale {scale} not a number of 32 bits")
    B = q.shape[0]
    _same_device(device, cache, block_table, seq_lens)
    if block_table.dim() != 2:
        raise ValueError(f"block_table is [{B}, pages], not {tuple(block_table.shape)}")
    pages = block_table.shape[1]
    if block_table.shape[0] != B or seq_lens.shape != (B,) or block_table.dtype is not torch.int32 or seq_lens.dtype is not torch.int32:
        raise ValueError(f"block_table is int32 [{B}, pages] and seq_lens int32 [{B}], not {block_table.dtype} {tuple(block_table.shape)} and {seq_lens.dtype} {tuple(seq_lens.shape)}")
    room = pages * block
    if room > MAX_TOKENS:
        raise ValueError(f"block_table has room for {room} tokens a sequence, the kernels count to {MAX_TOKENS}")
    _no_gradient(q)
    window = min(window, MAX_TOKENS)      # (no sequence is longer, and the kernels count in 32 bits)
    table = block_table if block_table.stride(1) == 1 else block_table.contiguous()      # (rows of a wider table are read where they are)
    lens = seq_lens.contiguous()
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, width), dtype=q.dtype, device=device)
    elif out.shape != (B, width) or out.dtype != q.dtype:
        raise ValueError(f"out is {q.dtype} [{B}, {width}], not {out.dtype} {tuple(out.shape)}")
    else:
        _same_device(device, out)
        if not _apart(out, width):
            _refuse_overlap(out, width)
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
    if q.dtype is not BF16:
        raise ValueError(f"the 4-bit cache takes bf16 queries, not {q.dtype}")
    if plan is None:
        plan = kv4_plan(B, Hq, Hkv, D, min(room, window) if window else room)
    cluster, num_ctas = plan
    if not 1 <= cluster <= MAX_CLUSTER or num_ctas < 0 or (num_ctas and cluster != 1):
        raise ValueError(f"plan {plan} is neither (1 to {MAX_CLUSTER}, 0) nor (1, CTAs)")
    if num_ctas:
        if B * Hkv * -(-(Hq // Hkv) // 8) * ((min(room, window) if window else room) // 32 + 2) + num_ctas > 0x7FFFFFFF:
            raise ValueError(f"plan {plan} shares more steps than it can count: take a cluster, or a window or a narrower block_table")
        size = kv4_scratch_size(num_ctas, D)
        if scratch is None:
            scratch = torch.empty(size, dtype=torch.float32, device=device)
        elif scratch.dtype is not torch.float32 or not scratch.is_contiguous() or scratch.numel() < size or scratch.data_ptr() % 16 or scratch.device != device:
            raise ValueError(f"scratch is a contiguous float32 tensor of {size} elements on {device} that starts on 16 bytes")
        sums = scratch.data_ptr()
        parts = sums + num_ctas * 64 * D
    else:
        sums = parts = None
    index = device.index
    if torch.cuda.current_device() != index:
        with torch.cuda.device(device):
            return kv4_paged_decode(q, cache, table, lens, Hq, Hkv, D, scale=scale, window=window, plan=plan, scratch=scratch, out=out)
    if not _aligned(q):      # rows that do not start on 16 bytes
        q = q[:, :width].clone(memory_format=torch.contiguous_format)
    stride = out.stride()
    to = out if stride[1] == 1 and stride[0] % 4 == 0 and out.data_ptr() % 8 == 0 and _apart(out, width) else torch.empty((B, width), dtype=BF16, device=device)
    call("rlb_kv4_paged_decode", q.data_ptr(), q.stride(0), cache.data_ptr(), cache.shape[0], table.data_ptr(), table.stride(0), pages, lens.data_ptr(), B, Hq, Hkv,
         D, block, window, scale, cluster, num_ctas, sums, parts, to.data_ptr(), to.stride(0), _L.status_word(device).data_ptr(), _raw_stream(index))
    if to is not out:
        out.copy_(to)
    return out
