"""The operators of speculative decoding as they are timed: the rows of trees of drafted tokens, attention of those rows over the paged key/value cache,
verification of the drafted tokens against the target's logits, and the move of the accepted rows' keys and values to the places they keep.

The rows of all sequences' trees lie one after the other, sequence b's at cu_rows[b] to cu_rows[b + 1]. Its row 0 is the last token that is decided,
the others are drafted; parents[t] is the row, within the sequence, that row t continues (smaller than its own; -1 for row 0). Row j's key and value
stand in the cache at place ctx_lens[b] + j.
"""

import math
import zlib

import torch

own = False


def listed():
    return [
        # a small model's answer to one short question: launch and latency
        dict(name="attend-one", kind="attend", batch=1, rows=6, context=300, Hq=14, Hkv=2, D=64, block=16, chain=False, ragged=True, window=0),
        # the rollout of 64 sequences of the benchmark's length
        dict(name="attend-rollout", kind="attend", batch=64, rows=17, context=1280, Hq=32, Hkv=8, D=128, block=64, chain=False, ragged=True, window=0),
        # few users and wide trees, small pages
        dict(name="attend-wide", kind="attend", batch=16, rows=64, context=8001, Hq=28, Hkv=4, D=128, block=16, chain=False, ragged=True, window=0),
        # one long document
        dict(name="attend-document", kind="attend", batch=1, rows=33, context=131072, Hq=40, Hkv=8, D=128, block=128, chain=False, ragged=True, window=0),
        # long responses of many sequences with a draft head's chain of four tokens: the cache is most of the card's traffic
        dict(name="attend-long", kind="attend", batch=32, rows=5, context=32768, Hq=32, Hkv=8, D=128, block=64, chain=True, ragged=False, window=0),
        # one user, a chain of drafted tokens
        dict(name="verify-one", kind="verify", batch=1, rows=6, vocab=32000, dtype="float32", draft=False, children=1, temperature=1.0),
        # the rollout of 64 sequences, trees of the most probable continuations
        dict(name="verify-rollout", kind="verify", batch=64, rows=17, vocab=128256, dtype="float32", draft=False, children=4, temperature=1.0),
        # tokens that were drawn from a draft model's distribution, two to a node
        dict(name="verify-drawn", kind="verify", batch=48, rows=8, vocab=151936, dtype="bfloat16", draft=True, children=2, temperature=0.8),
        # rows of one sequence's tree
        dict(name="rows-one", kind="rows", batch=1, rows=6, context=300, block=16, chain=False),
        # rows of many trees
        dict(name="rows-batch", kind="rows", batch=256, rows=64, context=4000, block=64, chain=False),
        # accepted rows of one sequence, in the caches of four layers
        dict(name="keep-one", kind="keep", batch=1, layers=4, accepted=3, Hkv=2, D=64, block=16),
        # accepted rows of 64 sequences, in the caches of a small model's 16 layers
        dict(name="keep-rollout", kind="keep", batch=64, layers=16, accepted=4, Hkv=8, D=64, block=32),
    ]


HEADS = {64: [(32, 8), (14, 2), (8, 8), (16, 1)], 128: [(32, 8), (28, 4), (40, 8), (16, 16), (32, 2), (12, 2)]}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "verify", "verify", "rows", "keep"])
    D = rng.choice([64, 128, 128])
    Hq, Hkv = rng.choice(HEADS[D])
    block = rng.choice([16, 32, 64, 128])
    chain = rng.random() < 0.3
    if kind == "rows":
        rows = _log(rng, 1, 200)
        return dict(kind=kind, batch=_log(rng, 1, 256), rows=rows, context=_log(rng, 1, 30000), block=block, chain=chain)
    if kind == "keep":
        return dict(kind=kind, batch=_log(rng, 1, 64), layers=_log(rng, 1, 16), accepted=rng.randint(1, 7), Hkv=Hkv, D=D, block=rng.choice([16, 32]))
    if kind == "verify":
        draft = rng.random() < 0.4
        rows = _log(rng, 1, 24 if draft else 64)
        vocab = rng.choice([2048, 32000, 50257, 128256, 151936])
        batch = _log(rng, 1, max(1, min(64, (50_000_000 if draft else 140_000_000) // (rows * vocab))))
        return dict(kind=kind, batch=batch, rows=rows, vocab=vocab, dtype=rng.choice(["float32", "bfloat16"]), draft=draft,
                    children=rng.choice([1, 1, 2, 3] if draft else [1, 2, 4, 8]), temperature=rng.choice([0.7, 1.0, 1.0, 1.3]))
    rows, context = _log(rng, 1, 200), _log(rng, 1, 60000)
    most = min(256, 30_000_000 // (context * Hkv * D // 32 + 1), 300_000_000 // (context * Hq * rows) + 1)
    return dict(kind=kind, batch=_log(rng, 1, max(1, most)), rows=rows, context=context, Hq=Hq, Hkv=Hkv, D=D, block=block, chain=chain,
                ragged=rng.random() < 0.7, window=rng.choice([0, 0, 0, 128, 1024, 4096]))


# ------------------------------------------------------------------------------------------- what the inputs are
def _contexts(case):
    """Cached tokens of each sequence before its tree: the longest has ``context``."""
    B, n = case["batch"], case["context"]
    if not case.get("ragged", True):
        return [n] * B
    lens = [max(1, int(n * (0.25 + 0.75 * ((0.618034 * i) % 1.0)))) for i in range(B)]
    lens[0] = n
    return lens


def _sizes(case):
    """Rows of each sequence: the largest tree has ``rows``; of eight sequences and more the last is a padding row of the batch, without rows."""
    B, n = case["batch"], case["rows"]
    if case.get("chain"):
        sizes = [n] * B
    else:
        sizes = [max(1, n - int(0.5 * n * ((0.754878 * i) % 1.0))) for i in range(B)]
    if B >= 8:
        sizes[-1] = 0
    return sizes


def _generator(case, seed, device="cuda"):
    key = zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()) ^ (seed * 0x9E3779B1 & 0xFFFFFFFF)
    return torch.Generator(device=device).manual_seed(key)


def _trees(sizes, g, chain, children=3):
    """Parents of all rows [T] on the CPU: every node has at most ``children``, the newest ones first to be continued."""
    parents = []
    for n in sizes:
        pick = torch.rand(max(n, 1), generator=g).tolist()
        free, got, has = [], [], [0] * n
        for j in range(n):
            if j == 0:
                got.append(-1)
            elif chain:
                got.append(j - 1)
            else:
                at = max(0, len(free) - 1 - int(pick[j] ** 2 * 2 * len(free)))
                got.append(free[at])
                has[free[at]] += 1
                if has[free[at]] == children:
                    del free[at]
            free.append(j)
        parents += got
    return torch.tensor(parents, dtype=torch.int32)


def _offsets(sizes):
    return torch.tensor([0] + sizes, dtype=torch.int64).cumsum(0).to(torch.int32)


def _pages(lens, block, g):
    """int32 [sequences, pages] block table of so many tokens each, in any order, and the number of pages."""
    need = [-(-n // block) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(need) + 1), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    return table, sum(need) + 2


def _normal(shape, g, D):
    """Keys, values and queries as projections give them: normal, some channels of each head larger than the rest."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    x[..., 3::29] *= 3.0
    return x


def _seen(parents, cu, n):
    """bool [B, n, n]: row i of a sequence sees row j: itself, and the rows it continues. Ancestors by doubling."""
    B, dev = len(cu) - 1, parents.device
    at = cu[:-1, None].long() + torch.arange(n, device=dev)
    there = at < cu[1:, None]
    up = torch.where(there, parents[at.clamp(max=max(len(parents) - 1, 0))].long(), -1)
    seen = torch.eye(n, dtype=torch.float32, device=dev).repeat(B, 1, 1)
    seen[up >= 0] += torch.nn.functional.one_hot(up[up >= 0], n).float()
    reach = 1
    while reach < n:
        seen = (torch.matmul(seen, seen) > 0).float()
        reach *= 2
    return (seen > 0) & there[:, :, None], at, there


def _words(bits):
    """bool [..., n] -> int32 [..., ceil(n / 32)], bit j of word w is place 32 w + j."""
    n = bits.shape[-1]
    x = torch.nn.functional.pad(bits, (0, -n % 32)).unflatten(-1, (-1, 32)).long()
    x = (x << torch.arange(32, device=bits.device)).sum(-1)
    return torch.where(x >= 2**31, x - 2**32, x).to(torch.int32)


def _tree(case, seed, children=3):
    sizes = _sizes(case)
    parents = _trees(sizes, _generator(case, seed, "cpu"), case.get("chain", False), children)
    return parents.cuda(), _offsets(sizes).cuda()


def prepare(case, seed):
    g = _generator(case, seed)
    dev = "cuda"
    if case["kind"] == "keep":
        B, n, block, layers = case["batch"], case["accepted"], case["block"], case["layers"]
        lens = [20 + 7 * i % 23 for i in range(B)]
        table, pages = _pages([m + 4 * (n + 1) for m in lens], block, g)
        shape = (pages, case["Hkv"], block, case["D"])
        caches = [(_normal(shape, g, case["D"]), _normal(shape, g, case["D"])) for _ in range(layers)]
        step = torch.randint(1, 4, (B, n), generator=g, device=dev)
        rows = torch.cat([torch.zeros((B, 1), dtype=torch.int64, device=dev), n + step.cumsum(1)], 1).to(torch.int32)      # (behind every place that is written)
        counts = torch.randint(1, n + 2, (B,), generator=g, device=dev).to(torch.int32)
        counts[0] = n + 1
        if B >= 8:
            counts[-1] = 0
        return dict(case=case, caches=caches, table=table, ctx=torch.tensor(lens, dtype=torch.int32, device=dev), rows=rows, counts=counts)
    parents, cu = _tree(case, seed, case.get("children", 3))
    T = len(parents)
    if case["kind"] == "verify":
        V, dt = case["vocab"], getattr(torch, case["dtype"])
        # logits of a language model: a few tokens have most of the probability, on some rows nearly all of it
        logits = torch.empty((T, V), dtype=dt, device=dev)
        guess = torch.empty((T, V), dtype=dt, device=dev) if case["draft"] else None
        tokens = torch.zeros(T, dtype=torch.int32, device=dev)
        up = torch.where(parents >= 0, parents.long() + torch.repeat_interleave(cu[:-1].long(), (cu[1:] - cu[:-1]).long(), output_size=T), -1)
        rank = torch.zeros(T, dtype=torch.int64)
        seen = {}
        for t, p in enumerate(up.tolist()):
            rank[t] = seen[p] = seen.get(p, -1) + 1
        best = torch.zeros((T, case["children"]), dtype=torch.int64, device=dev)
        for t in range(0, T, 64):
            z = torch.randn((min(64, T - t), V), generator=g, device=dev) * (3.0 + 5.0 * torch.rand((min(64, T - t), 1), generator=g, device=dev))
            logits[t : t + 64] = z.to(dt)
            z += 0.6 * torch.randn(z.shape, generator=g, device=dev)      # what the draft makes of it
            if case["draft"]:
                guess[t : t + 64] = z.to(dt)
                p = torch.softmax(guess[t : t + 64].float() / case["temperature"], -1)
                best[t : t + 64] = torch.multinomial(p, case["children"], replacement=True, generator=g)
            else:
                best[t : t + 64] = z.topk(case["children"], -1).indices
        child = up >= 0
        tokens[child] = best[up[child], rank.to(dev)[child].clamp(max=case["children"] - 1)].to(torch.int32)
        return dict(case=case, logits=logits, guess=guess, tokens=tokens, parents=parents, cu=cu, uniforms=torch.rand(T, generator=g, device=dev))
    lens = _contexts(case)
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    table, pages = _pages([a + b for a, b in zip(lens, _sizes(case))], case["block"], g)
    if case["kind"] == "rows":
        return dict(case=case, parents=parents, cu=cu, ctx=ctx, table=table)
    Hq, Hkv, D, n = case["Hq"], case["Hkv"], case["D"], case["rows"]
    seen, at, there = _seen(parents, cu, n)
    masks = torch.zeros((T, -(-n // 32)), dtype=torch.int32, device=dev)
    masks[at[there]] = _words(seen)[there]
    positions = torch.zeros(T, dtype=torch.int32, device=dev)
    positions[at[there]] = (ctx[:, None] + seen.sum(-1) - 1).to(torch.int32)[there]
    shape = (pages, Hkv, case["block"], D)
    rows = _normal((T, Hq + 2 * Hkv, D), g, D).reshape(T, -1)      # the fused rows of the projection
    return dict(case=case, q=rows[:, : Hq * D], k=_normal(shape, g, D), v=_normal(shape, g, D), table=table, ctx=ctx, cu=cu,
                masks=None if case["chain"] else masks, positions=positions)


# ------------------------------------------------------------------------------------------- plain forms
def _plain_rows(st):
    c = st["case"]
    n, block, dev = c["rows"], c["block"], st["cu"].device
    seen, at, there = _seen(st["parents"], st["cu"], n)
    masks = torch.zeros((len(st["parents"]), -(-n // 32)), dtype=torch.int32, device=dev)
    positions = torch.zeros(len(st["parents"]), dtype=torch.int32, device=dev)
    slots = torch.full((len(st["parents"]),), -1, dtype=torch.int64, device=dev)
    masks[at[there]] = _words(seen)[there]
    positions[at[there]] = (st["ctx"][:, None] + seen.sum(-1) - 1).to(torch.int32)[there]
    place = st["ctx"][:, None].long() + torch.arange(n, device=dev)
    page = torch.gather(st["table"].long(), 1, (place // block).clamp(max=st["table"].shape[1] - 1))
    slots[at[there]] = (page * block + place % block)[there]
    return dict(masks=masks, positions=positions, slots=slots)


def _plain_attend(st):
    c = st["case"]
    Hq, Hkv, D, n, cu = c["Hq"], c["Hkv"], c["D"], c["rows"], st["cu"].long()
    B, T, dev = len(cu) - 1, len(st["q"]), st["q"].device
    at = cu[:-1, None] + torch.arange(n, device=dev)
    there = at < cu[1:, None]
    at = torch.where(there, at, 0)
    k = st["k"][st["table"].long()].transpose(1, 2).flatten(2, 3).float()                 # [B, Hkv, tokens, D]
    q = st["q"].float()[at].reshape(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = (torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D)).unflatten(2, (Hq // Hkv, n))    # [B, Hkv, group, rows, tokens]
    del k
    places = torch.arange(s.shape[-1], device=dev)
    j = places - st["ctx"][:, None]                                                       # row of the tree, below 0: context
    j_in = ((j >= 0) & (j < n))[:, None].expand(-1, n, -1)
    if st["masks"] is None:
        bit = j[:, None] <= torch.arange(n, device=dev)[:, None]
    else:
        jc = j.clamp(0, n - 1)[:, None].expand(-1, n, -1)
        bit = (torch.gather(st["masks"][at].long(), 2, jc // 32) >> (jc % 32)) & 1 == 1
    live = ((j < 0)[:, None] | (j_in & bit)) & there[:, :, None]
    if c["window"]:
        key = torch.where(j_in, torch.gather(st["positions"][at], 1, j.clamp(0, n - 1))[:, None], places.to(torch.int32))
        live = live & (st["positions"][at][:, :, None] - key < c["window"])
    s = s.masked_fill_(~live[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    v = st["v"][st["table"].long()].transpose(1, 2).flatten(2, 3).float()
    o = torch.matmul(p.flatten(2, 3), v) / p.flatten(2, 3).sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.unflatten(2, (Hq // Hkv, n)).permute(0, 3, 1, 2, 4).reshape(B, n, Hq * D).to(torch.bfloat16)
    out = torch.zeros((T, Hq * D), dtype=torch.bfloat16, device=dev)
    out[at[there]] = o[there]
    return out


def _plain_verify(st):
    """In 64 bits: whole numbers depend on values next to a border."""
    c = st["case"]
    n, cu, dev = c["rows"], st["cu"].long(), st["cu"].device
    B, T, V = len(cu) - 1, len(st["tokens"]), c["vocab"]
    owner = torch.searchsorted(cu[1:].contiguous(), torch.arange(T, device=dev), right=True)
    up = torch.where(st["parents"] >= 0, st["parents"].long() + cu[owner], -1)
    z = st["logits"].double() / c["temperature"]
    e = torch.exp(z - z.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    del z, e
    q = None
    if c["draft"]:
        z = st["guess"].double() / c["temperature"]
        e = torch.exp(z - z.amax(-1, keepdim=True))
        q = e / e.sum(-1, keepdim=True)
        del z, e
    rank = ((up[:, None] == up[None, :]) & (torch.arange(T, device=dev)[None, :] < torch.arange(T, device=dev)[:, None])).sum(1)     # older siblings
    child = up >= 0
    tok, u = st["tokens"].long(), st["uniforms"].double()
    left, total = p.clone(), torch.ones(T, dtype=torch.float64, device=dev)      # of each node: what is still to be given, and its sum
    follow = torch.full((T,), -1, dtype=torch.int64, device=dev)
    for r in range(c["children"]):      # the children of a node one after the other
        at = torch.where(child & (rank == r), up, T)
        mine = torch.full((T + 1,), -1, dtype=torch.int64, device=dev).scatter_(0, at, torch.arange(T, device=dev))[:T]
        has = (mine >= 0) & (follow < 0)
        row = mine.clamp(min=0)
        w = torch.gather(left, 1, tok[row][:, None])[:, 0]
        chance = torch.gather(q, 1, tok[row][:, None])[:, 0] if c["draft"] else 1.0
        yes = has & (u[row] * chance * total < w)
        follow = torch.where(yes, row, follow)
        no = has & ~yes
        if c["draft"]:
            left = torch.where(no[:, None], (left / total[:, None] - q).clamp_min_(0.0), left)
            total = torch.where(no, left.sum(-1), total)
        else:
            left.scatter_(1, tok[row][:, None], torch.where(no, 0.0, w)[:, None])
            total = torch.where(no, total - w, total)
    node = torch.where(cu[1:] > cu[:-1], cu[:-1], -1)
    out = dict(tokens=torch.full((B, n), -1, dtype=torch.int32, device=dev), counts=torch.zeros(B, dtype=torch.int32, device=dev),
               rows=torch.full((B, n), -1, dtype=torch.int32, device=dev), logprobs=torch.zeros((B, n), dtype=torch.float32, device=dev))
    final = node
    for s in range(n):      # down the accepted rows
        live, here = node >= 0, node.clamp(min=0)
        to = torch.where(live, follow[here], -1)
        final = torch.where(live, node, final)
        out["rows"][:, s] = torch.where(live, here - cu[:-1], -1).to(torch.int32)
        out["counts"] += live.to(torch.int32)
        out["tokens"][:, s] = torch.where(to >= 0, tok[to.clamp(min=0)], -1).to(torch.int32)
        out["logprobs"][:, s] = torch.where(to >= 0, torch.log(p[here, tok[to.clamp(min=0)]]), 0.0).float()
        node = to
    # the token behind the last accepted one: the first whose share of the running sum passes the sequence's own number
    live, here = final >= 0, final.clamp(min=0)
    w = left[here]
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p[here])
    run = w.cumsum(-1)
    passed = run > u[cu[:-1].clamp(max=T - 1)][:, None] * run[:, -1:]
    last = torch.where(passed.any(-1), passed.int().argmax(-1), V - 1 - (w > 0).flip(-1).int().argmax(-1))
    b = torch.arange(B, device=dev)
    end = (out["counts"].long() - 1).clamp(min=0)
    out["tokens"][b, end] = torch.where(live, last, -1).to(torch.int32)
    out["logprobs"][b, end] = torch.where(live, torch.log(p[here, last]), 0.0).float()
    return out


def _plain_keep(st):
    block, table, ctx, rows = st["case"]["block"], st["table"].long(), st["ctx"].long()[:, None], st["rows"].long()
    i = torch.arange(rows.shape[1], device=rows.device)
    b, i = torch.where((i < st["counts"][:, None]) & (rows != i))
    source, target = (ctx[b, 0] + rows[b, i], ctx[b, 0] + i)
    sp, tp = table[b, source // block], table[b, target // block]
    for pair in st["caches"]:
        for x in pair:
            x[tp, :, target % block] = x[sp, :, source % block]
    return [x for pair in st["caches"] for x in pair]


def run(state):
    c = state["case"]
    if own:
        from rl_b200.ops import draft_ops as S

        if c["kind"] == "rows":
            masks, positions, slots = S.tree_rows(state["parents"], state["cu"], state["ctx"], state["table"], c["block"], max_rows=c["rows"])
            return dict(masks=masks, positions=positions, slots=slots)
        if c["kind"] == "attend":
            return S.tree_paged_decode(state["q"], state["k"], state["v"], state["table"], state["ctx"], state["cu"], c["Hq"], c["Hkv"], c["D"],
                                       max_rows=c["rows"], masks=state["masks"], window=c["window"], positions=state["positions"] if c["window"] else None)
        if c["kind"] == "verify":
            tokens, counts, rows, logprobs = S.verify_drafts(state["logits"], state["tokens"], state["parents"], state["cu"], state["uniforms"],
                                                             max_rows=c["rows"], draft_logits=state["guess"], temperature=c["temperature"])
            return dict(tokens=tokens, counts=counts, rows=rows, logprobs=logprobs)
        S.kv_cache_keep(state["caches"], state["table"], state["ctx"], state["rows"], state["counts"])
        return [x for pair in state["caches"] for x in pair]
    return {"rows": _plain_rows, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[c["kind"]](state)


def _visited(case):
    """Nodes of a sequence whose logits decide something, in the mean of these inputs: the accepted rows and the one behind which the last token is drawn."""
    n = case["rows"]
    take = 0.47 if not case["draft"] and case["children"] > 1 else 0.40 if not case["draft"] else 0.78 if case["children"] > 1 else 0.80
    depth = n if case["children"] == 1 else max(1.0, 1.6 * math.sqrt(n))
    return min(float(n), (1 - take ** depth) / (1 - take))


def work(case):
    if case["kind"] == "keep":      # half of the sequences' rows, and they move
        moved = case["batch"] * (case["accepted"] / 2) * case["layers"] * 2 * case["Hkv"] * case["D"]
        return dict(bytes=2 * 2 * moved, flops=0)
    sizes = _sizes(case)
    T = sum(sizes)
    if case["kind"] == "rows":
        return dict(bytes=T * (4 + 4 * -(-case["rows"] // 32) + 4 + 8) + 8 * len(sizes), flops=T * case["rows"])
    if case["kind"] == "verify":
        live = sum(n > 0 for n in sizes)
        nodes = live * _visited(case)
        return dict(bytes=nodes * case["vocab"] * (4 if case["dtype"] == "float32" else 2) * (2 if case["draft"] else 1) + 12 * T + 12 * live * case["rows"],
                    flops=nodes * case["vocab"] * (8 if case["draft"] else 4))
    Hq, Hkv, D, w = case["Hq"], case["Hkv"], case["D"], case["window"]
    seen = [(min(c, w) if w else c, n) for c, n in zip(_contexts(case), sizes) if n]
    tokens = sum(c + n for c, n in seen)
    return dict(bytes=tokens * 4 * Hkv * D + T * 4 * Hq * D + 4 * tokens / case["block"], flops=4 * Hq * D * sum(n * (c + (n + 1) / 2) for c, n in seen))


# ------------------------------------------------------------------------------------------- in 64 bits, from the definitions
def _exact_attend(case, st):
    Hq, Hkv, D, block, w = case["Hq"], case["Hkv"], case["D"], case["block"], case["window"]
    cu, ctx = st["cu"].tolist(), st["ctx"].tolist()
    out = torch.zeros((len(st["q"]), Hkv, Hq // Hkv, D), dtype=torch.float64, device="cuda")
    for b, c in enumerate(ctx):
        lo, hi = cu[b], cu[b + 1]
        n = hi - lo
        if not n:
            continue
        q = st["q"][lo:hi].double().reshape(n, Hkv, -1, D)
        pos = st["positions"][lo:hi].long()
        tree = torch.zeros((n, n), dtype=torch.bool, device="cuda")
        for j in range(n):
            tree[:, j] = torch.arange(n, device="cuda") >= j if st["masks"] is None else (st["masks"][lo:hi, j // 32].long() >> (j % 32)) & 1 == 1
        top, total, acc = torch.full((n, Hkv, Hq // Hkv, 1), -math.inf, dtype=torch.float64, device="cuda"), 0.0, 0.0
        for at in torch.arange(max(0, c - w) if w else 0, c + n, device="cuda").split(4096):
            page, off = st["table"][b].long()[at // block], at % block
            k, v = st["k"][page, :, off].double(), st["v"][page, :, off].double()
            sees = torch.ones((n, len(at)), dtype=torch.bool, device="cuda")
            j = at - c
            sees[:, j >= 0] = tree[:, j[j >= 0]]
            if w:
                sees &= pos[:, None] - torch.where(j >= 0, pos[j.clamp(min=0)], at) < w
            s = torch.einsum("nhgd,thd->nhgt", q, k) / math.sqrt(D)
            s = s.masked_fill(~sees[:, None, None], -math.inf)
            m = torch.maximum(top, s.amax(-1, keepdim=True))
            base = torch.where(m == -math.inf, 0.0, m)
            keep, p = torch.exp(top - base), torch.exp(s - base)
            total, acc, top = total * keep + p.sum(-1, keepdim=True), acc * keep + torch.einsum("nhgt,thd->nhgd", p, v), m
        out[lo:hi] = torch.where(total > 0, acc / total, 0.0)
    return out.reshape(len(st["q"]), -1)


def _exact_verify(case, st):
    n, V = case["rows"], case["vocab"]
    cu, parents, tokens, u = st["cu"].tolist(), st["parents"].tolist(), st["tokens"].tolist(), st["uniforms"].double().tolist()
    B = len(cu) - 1
    got = dict(tokens=torch.full((B, n), -1, dtype=torch.int32), counts=torch.zeros(B, dtype=torch.int32), rows=torch.full((B, n), -1, dtype=torch.int32),
               logprobs=torch.zeros((B, n), dtype=torch.float64))
    for b in range(B):
        lo, hi = cu[b], cu[b + 1]
        node, step = 0, 0
        while lo < hi:
            logp = torch.log_softmax(st["logits"][lo + node].double() / case["temperature"], -1)
            p = logp.exp()
            q = torch.softmax(st["guess"][lo + node].double() / case["temperature"], -1) if case["draft"] else None
            now, went = p.clone(), None
            got["rows"][b, step] = node
            for j in range(1, hi - lo):
                if parents[lo + j] != node:
                    continue
                x = tokens[lo + j]
                share = now / now.sum()
                if u[lo + j] < float(share[x]) / (float(q[x]) if case["draft"] else 1.0):
                    went = j
                    break
                if case["draft"]:
                    now = torch.relu(share - q)
                else:
                    now[x] = 0.0
            if went is None:
                run = torch.cumsum(now, 0)
                x = int(torch.searchsorted(run, u[lo] * run[-1], right=True).clamp(max=V - 1))
            got["tokens"][b, step], got["logprobs"][b, step] = x, logp[x]
            step += 1
            if went is None:
                break
            node = went
        got["counts"][b] = step
    return {k: v.cuda() for k, v in got.items()}


def exact(case, seed):
    if case["kind"] in ("rows", "keep"):      # nothing but whole numbers and moved values
        return None
    st = prepare(case, seed)
    return _exact_attend(case, st) if case["kind"] == "attend" else _exact_verify(case, st)
