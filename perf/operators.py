"""The operators of the generation engine's 4-bit key/value cache as they are timed: the cache write behind the q/k/v projection, the read-back
that prefix reuse and chunked prefill need, and decode attention over the cache's pages.

A page holds ``block`` tokens of one key/value head: keys' codes, values' codes, scales. A group is 32 consecutive dimensions of a token: its scale
is bf16(largest magnitude / 7.5) and a value x is the code floor(x / scale) + 8, which stands for (code - 7.5) * scale.
"""

import math
import zlib

import torch

own = False

GROUP = 32
TINY = 2.0 ** -100       # a group whose largest magnitude is below this is held as zeros


def listed():
    return [
        # one row of a small model's decode step: launch and latency
        dict(name="write-one", kind="write", tokens=1, Hq=32, Hkv=4, D=64, block=64),
        # the decode step of 64 sequences with 32 query and 8 key/value heads of 128
        dict(name="write-decode", kind="write", tokens=64, Hq=32, Hkv=8, D=128, block=64),
        # ragged prompts of a prefill round, packed
        dict(name="write-prompts", kind="write", tokens=15003, Hq=32, Hkv=8, D=128, block=64),
        # one more turn of a short conversation
        dict(name="read-turn", kind="read", tokens=517, Hkv=4, D=64, block=16),
        # the cached prefixes of a chunked prefill round
        dict(name="read-prefix", kind="read", tokens=32771, Hkv=8, D=128, block=64),
        # one user's short question
        dict(name="decode-one", kind="decode", batch=1, context=300, Hq=32, Hkv=8, D=128, block=64, ragged=True, window=0),
        # the rollout of 64 sequences of the benchmark's length
        dict(name="decode-rollout", kind="decode", batch=64, context=1280, Hq=32, Hkv=8, D=128, block=64, ragged=True, window=0),
        # many sequences, seven query heads to a key/value head, small pages
        dict(name="decode-wide", kind="decode", batch=256, context=2001, Hq=28, Hkv=4, D=128, block=16, ragged=True, window=0),
        # a small model's heads of 64
        dict(name="decode-64", kind="decode", batch=96, context=3001, Hq=14, Hkv=2, D=64, block=32, ragged=True, window=0),
        # sliding-window layers with heads of 256
        dict(name="decode-window", kind="decode", batch=48, context=9001, Hq=16, Hkv=8, D=256, block=64, ragged=True, window=1024),
        # one long document
        dict(name="decode-document", kind="decode", batch=1, context=131072, Hq=40, Hkv=8, D=128, block=128, ragged=True, window=0),
        # long responses of many sequences: the cache is most of the card's traffic
        dict(name="decode-long", kind="decode", batch=32, context=32768, Hq=32, Hkv=8, D=128, block=64, ragged=False, window=0),
    ]


HEADS = {64: [(32, 4), (14, 2), (8, 8), (16, 1)], 128: [(32, 8), (28, 4), (40, 8), (16, 16), (32, 2), (12, 2)], 256: [(16, 8), (8, 4), (8, 1)]}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode"])
    D = rng.choice([64, 128, 128, 256])
    Hq, Hkv = rng.choice(HEADS[D])
    block = rng.choice([16, 32, 64, 128])
    if kind == "write":
        return dict(kind=kind, tokens=_log(rng, 1, 16000), Hq=Hq, Hkv=Hkv, D=D, block=block)
    if kind == "read":
        return dict(kind=kind, tokens=_log(rng, 1, 40000), Hkv=Hkv, D=D, block=block)
    context = _log(rng, 1, 60000)
    most = max(1, min(256, 30_000_000 // (context * Hkv * D // 32)))
    return dict(kind=kind, batch=_log(rng, 1, most), context=context, Hq=Hq, Hkv=Hkv, D=D, block=block,
                ragged=rng.random() < 0.7, window=rng.choice([0, 0, 0, 128, 1024, 4096]))


# ------------------------------------------------------------------------------------------- what the inputs are
def _lengths(case):
    """Cached tokens of each sequence: the longest has ``context``; of eight and more the last is a padding row of the batch."""
    B, n = case["batch"], case["context"]
    if not case["ragged"]:
        return [n] * B
    lens = [max(1, int(n * (0.25 + 0.75 * ((0.618034 * i) % 1.0)))) for i in range(B)]
    lens[0] = n
    if B >= 8:
        lens[-1] = 0
    return lens


def _generator(case, seed):
    key = zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()) ^ (seed * 0x9E3779B1 & 0xFFFFFFFF)
    return torch.Generator(device="cuda").manual_seed(key)


def _normal(shape, g, D):
    """Keys and values as projections give them: normal, some channels of each head far larger than the rest."""
    x = torch.randn(shape, generator=g, device="cuda")
    scale = torch.ones(D, device="cuda")
    scale[3::29] = 4.0
    return x * scale


def _random_pages(pages, Hkv, D, block, g):
    """A cache in use: [pages, Hkv, page bytes] of quantised normal keys and values."""
    n = block * D // 2
    pool = torch.empty((pages, Hkv, 2 * n + block * D // 8), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (Hkv * block * D))
    for p in range(0, pages, step):
        e = min(pages, p + step)
        parts, scales = [], []
        for keys in (True, False):
            x = _normal((e - p, Hkv, block, D), g, D).unflatten(-1, (-1, GROUP))
            s = (x.abs().amax(-1) / 7.5).to(torch.bfloat16)
            c = (torch.floor(x / s.float().unsqueeze(-1)) + 8).clamp_(0, 15).to(torch.uint8)      # [.., block, groups, 32]
            if keys:      # 16-bit units [4][groups][2] of a token, four dimensions each
                u = c.unflatten(-1, (4, 2, 4)).permute(0, 1, 2, 4, 3, 5, 6)
            else:         # 16-bit units [8][groups][2 tokens] of two tokens, four dimensions each
                u = c.unflatten(-1, (8, 4)).unflatten(2, (-1, 2)).permute(0, 1, 2, 5, 4, 3, 6)
            u = u.reshape(e - p, Hkv, n, 2)
            parts.append(u[..., 0] | (u[..., 1] << 4))
            scales.append(s)
        sc = torch.stack(scales, 3).contiguous().view(torch.uint8).reshape(e - p, Hkv, -1)
        pool[p:e] = torch.cat([*parts, sc], -1)
    return pool


def prepare(case, seed):
    g = _generator(case, seed)
    Hkv, D, block = case["Hkv"], case["D"], case["block"]
    dev = "cuda"
    if case["kind"] == "write":
        T, Hq = case["tokens"], case["Hq"]
        qkv = _normal((T, Hq + 2 * Hkv, D), g, D).reshape(T, -1).to(torch.bfloat16)
        pages = T // block + 17
        if T <= 256:      # one token of each sequence, wherever the sequences are
            positions = torch.randint(0, 32768, (T,), generator=g, device=dev).to(torch.int32)
            slots = torch.randperm(pages * block, generator=g, device=dev)[:T]
            if T >= 8:
                slots[-3:] = -1      # padding rows of the batch
        else:             # prompts one after the other, pages in any order
            positions = (torch.arange(T, device=dev) % 1201).to(torch.int32)
            page = torch.randperm(pages, generator=g, device=dev)
            at = torch.arange(T, device=dev)
            slots = page[at // block] * block + at % block
        inv_freq = 500000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float32) / D)
        cache = torch.zeros((pages, Hkv, block * D * 9 // 8), dtype=torch.uint8, device=dev)
        return dict(case=case, qkv=qkv, positions=positions, inv_freq=inv_freq, slots=slots, cache=cache)
    if case["kind"] == "read":
        pages = case["tokens"] // block + 3
        cache = _random_pages(pages, Hkv, D, block, g)
        page = torch.randperm(pages, generator=g, device=dev)
        at = torch.arange(case["tokens"], device=dev)
        return dict(case=case, cache=cache, slots=page[at // block] * block + at % block)
    lens = _lengths(case)
    need = [-(-n // block) for n in lens]
    cache = _random_pages(sum(need) + 2, Hkv, D, block, g)
    order = torch.randperm(sum(need) + 2, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((len(lens), max(need) + 1), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    rows = _normal((len(lens), case["Hq"] + 2 * Hkv, D), g, D).reshape(len(lens), -1).to(torch.bfloat16)     # the fused rows of the projection
    return dict(case=case, q=rows[:, : case["Hq"] * D], cache=cache, table=table, lens=torch.tensor(lens, dtype=torch.int32, device=dev))


# ------------------------------------------------------------------------------------------- plain forms
def _rotated(qkv, positions, inv_freq, heads, D):
    """The first ``heads`` heads turned: angles in 64 bits, cosines and sines rounded to 32, the rest in 32."""
    x = qkv[:, : heads * D].float().reshape(len(qkv), heads, 2, D // 2)
    a = positions.double()[:, None] * inv_freq.double()
    c, s = torch.cos(a).float()[:, None], torch.sin(a).float()[:, None]
    lo, hi = x[:, :, 0], x[:, :, 1]
    return torch.stack([lo * c - hi * s, hi * c + lo * s], 2).reshape(len(qkv), heads * D).to(torch.bfloat16)


def _held(x):
    """bf16 [..., D] -> what the cache keeps of it, in bf16. In 64 bits: values lie next to the borders of their codes."""
    g = x.double().unflatten(-1, (-1, GROUP))
    a = g.abs().amax(-1, keepdim=True)
    s = (a / 7.5).to(torch.bfloat16).double()
    s = torch.where(a < TINY, 0.0, s)
    c = (torch.floor(g / s) + 8).clamp(0, 15)
    return torch.where(s == 0, 0.0, (c - 7.5) * s).flatten(-2).float().to(torch.bfloat16)


def _codes(pages, D, block):
    """[..., page bytes] -> codes of keys and values [..., block, D] and their scales [..., block, groups, 1] in 32 bits."""
    n, lead, G = block * D // 2, pages.shape[:-1], D // GROUP
    raw = torch.stack([pages[..., : 2 * n] & 15, pages[..., : 2 * n] >> 4], -1)
    k = raw[..., :n, :].reshape(*lead, block, 4, G, 2, 4).transpose(-4, -3).reshape(*lead, block, G, GROUP)
    v = raw[..., n:, :].reshape(*lead, block // 2, 8, G, 2, 4)
    v = v.permute(*range(len(lead)), -5, -2, -3, -4, -1).reshape(*lead, block, G, GROUP)
    s = pages[..., 2 * n :].contiguous().view(torch.bfloat16).float().reshape(*lead, block, 2, G, 1)
    return k, v, s[..., 0, :, :], s[..., 1, :, :]


def _plain_write(st):
    c = st["case"]
    T, Hq, Hkv, D = len(st["qkv"]), c["Hq"], c["Hkv"], c["D"]
    qkv = st["qkv"]
    qkv[:, : (Hq + Hkv) * D] = _rotated(qkv, st["positions"], st["inv_freq"], Hq + Hkv, D)
    kept = _held(qkv[:, Hq * D :].reshape(T, 2 * Hkv, D)).reshape(T, -1)
    return dict(rows=qkv, kept=torch.where(st["slots"][:, None] < 0, torch.zeros_like(kept), kept))


def _plain_read(st):
    c = st["case"]
    block, slots = c["block"], st["slots"]
    k, v, ks, vs = _codes(st["cache"], c["D"], block)
    both = []
    for codes, scale in ((k, ks), (v, vs)):
        x = ((codes.float() - 7.5) * scale).flatten(-2)              # [pages, Hkv, block, D]
        both.append(x[slots // block, :, slots % block].flatten(1))
    return torch.cat(both, 1).to(torch.bfloat16)


def _plain_decode(st):
    c = st["case"]
    Hq, Hkv, D, block, lens = c["Hq"], c["Hkv"], c["D"], c["block"], st["lens"]
    B = len(lens)
    k, v, ks, vs = _codes(st["cache"][st["table"].long()], D, block)                       # [B, pages, Hkv, block, ...]
    k = ((k.float() - 7.5) * ks).flatten(-2).transpose(1, 2).flatten(2, 3)                 # [B, Hkv, tokens, D]
    s = torch.matmul(st["q"].float().reshape(B, Hkv, Hq // Hkv, D), k.transpose(2, 3)) / math.sqrt(D)
    del k
    at = torch.arange(s.shape[-1], device=s.device)
    live = at < lens[:, None]
    if c["window"]:
        live = live & (at >= lens[:, None] - c["window"])
    live = live[:, None, None]
    s = s.masked_fill(~live, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    v = ((v.float() - 7.5) * vs).flatten(-2).transpose(1, 2).flatten(2, 3)
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.reshape(B, Hq * D).to(torch.bfloat16)


def run(state):
    c = state["case"]
    if own:
        from rl_b200.ops import kv4_ops as K

        if c["kind"] == "write":
            rows = K.rope_kv4_cache_write(state["qkv"], state["positions"], state["inv_freq"], state["slots"], state["cache"], c["Hq"], c["Hkv"], c["D"])
            return dict(rows=rows, kept=K.kv4_cache_read(state["cache"], state["slots"], c["Hkv"], c["D"]))
        if c["kind"] == "read":
            return K.kv4_cache_read(state["cache"], state["slots"], c["Hkv"], c["D"])
        return K.kv4_paged_decode(state["q"], state["cache"], state["table"], state["lens"], c["Hq"], c["Hkv"], c["D"], window=c["window"])
    return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode}[c["kind"]](state)


def work(case):
    Hkv, D = case["Hkv"], case["D"]
    held = 2 * Hkv * D * 9 / 16          # bytes of a cached token: 4 bits a value and a bf16 scale for 32
    if case["kind"] == "write":          # rows read, rotated heads written back, codes written; and read back into bf16
        T, Hq = case["tokens"], case["Hq"]
        return dict(bytes=T * (2 * (Hq + 2 * Hkv) * D + 2 * (Hq + Hkv) * D + 2 * held + 4 * Hkv * D + 20), flops=T * (Hq + 2 * Hkv) * D * 6)
    if case["kind"] == "read":
        return dict(bytes=case["tokens"] * (held + 4 * Hkv * D + 8), flops=case["tokens"] * 4 * Hkv * D)
    lens = _lengths(case)
    seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
    return dict(bytes=seen * held + len(lens) * (4 * case["Hq"] * D + 4) + 4 * seen / case["block"], flops=4 * case["Hq"] * D * seen)


# ------------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _levels(x):
    """float64 [..., 32]: a value's code is the number of borders k * scale, k from -7 to 7, that it has reached."""
    a = x.abs().amax(-1, keepdim=True)
    s = (a / 7.5).to(torch.bfloat16).double() * (a >= TINY)
    c = torch.zeros_like(x)
    for k in range(-7, 8):
        c += x >= k * s
    return (c - 7.5) * s


def _token(pool, case, page, off):
    """float64 keys and values [tokens, Hkv, D] of places (page, off), unit by unit."""
    D, block, G = case["D"], case["block"], case["D"] // GROUP
    n = block * D // 2
    units = pool.view(torch.int16)[page].int() & 0xFFFF                                # [tokens, Hkv, 16-bit units]
    d = torch.arange(D, device=pool.device)
    g, quad, j = d // GROUP, d % GROUP // 4, d % 4
    ku = off[:, None] * (D // 4) + ((quad // 2) * G + g) * 2 + quad % 2
    vu = n // 2 + (off[:, None] // 2) * (D // 2) + (quad * G + g) * 2 + off[:, None] % 2
    su = n + off[:, None] * 2 * G + g
    got = []
    for u, s in ((ku, su), (vu, su + G)):
        code = torch.gather(units, 2, u[:, None].expand(-1, units.shape[1], -1)) >> (4 * j) & 15
        scale = (torch.gather(units, 2, s[:, None].expand(-1, units.shape[1], -1)) << 16).view(torch.float32)
        got.append((code.double() - 7.5) * scale.double())
    return got


def exact(case, seed):
    st = prepare(case, seed)
    Hkv, D, block = case["Hkv"], case["D"], case["block"]
    if case["kind"] == "write":
        T, Hq = case["tokens"], case["Hq"]
        x = st["qkv"].double().reshape(T, Hq + 2 * Hkv, D)
        z = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), st["positions"].double()[:, None] * st["inv_freq"].double())[:, None]
        turned = torch.complex(x[:, : Hq + Hkv, : D // 2], x[:, : Hq + Hkv, D // 2 :]) * z
        rows = torch.cat([torch.cat([turned.real, turned.imag], -1), x[:, Hq + Hkv :]], 1)
        kept = _levels(rows[:, Hq:].to(torch.bfloat16).double().unflatten(-1, (-1, GROUP))).reshape(T, -1)
        kept[st["slots"] < 0] = 0.0
        return dict(rows=rows.reshape(T, -1), kept=kept)
    if case["kind"] == "read":
        parts = [_token(st["cache"], case, s // block, s % block) for s in st["slots"].split(4096)]
        return torch.cat([torch.cat([p[i] for p in parts]).flatten(1) for i in (0, 1)], 1)
    lens = _lengths(case)
    out = torch.zeros((len(lens), case["Hq"], D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n <= first:
            continue
        q = st["q"][b].double().reshape(Hkv, -1, D)
        top, total, acc = None, 0.0, 0.0
        for at in torch.arange(first, n, device="cuda").split(4096):
            k, v = _token(st["cache"], case, st["table"][b].long()[at // block], at % block)
            s = torch.einsum("hgd,thd->hgt", q, k) / math.sqrt(D)
            m = s.amax(-1, keepdim=True) if top is None else torch.maximum(top, s.amax(-1, keepdim=True))
            keep = 0.0 if top is None else torch.exp(top - m)
            p = torch.exp(s - m)
            total, acc, top = total * keep + p.sum(-1, keepdim=True), acc * keep + torch.einsum("hgt,thd->hgd", p, v), m
        out[b] = (acc / total).reshape(-1, D)
    return out.reshape(len(lens), -1)
