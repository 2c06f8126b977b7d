"""Operators of speculative decoding on the CPU: the restatements against plain 64-bit forms, and what is refused."""

import math

import draft_oracle as O
import pytest
import torch

from rl_b200.ops import draft_ops as S
from rl_b200.ops import engine_ops as E


def _attend_case(sizes, ctx, Hq, Hkv, D, block, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    parents, cu = O.forest(sizes, seed)
    table, count = O.pages([c + n for c, n in zip(ctx, sizes)], block, seed)
    k, v = (torch.randn((count, Hkv, block, D), generator=g).to(dtype) for _ in range(2))
    q = torch.randn((int(cu[-1]), (Hq + 2 * Hkv) * D), generator=g).to(dtype)
    return q, k, v, table, torch.tensor(ctx, dtype=torch.int32), cu, parents


@pytest.mark.parametrize("sizes,ctx", [([1], [0]), ([5], [17]), ([3, 0, 40, 1], [9, 3, 64, 0])])
def test_rows(sizes, ctx):
    parents, cu = O.forest(sizes, 3)
    block, most = 16, max(sizes)
    table, _ = O.pages([c + n for c, n in zip(ctx, sizes)], block)
    masks, positions, slots = S.tree_rows(parents, cu, torch.tensor(ctx, dtype=torch.int32), table, block, max_rows=most)
    assert masks.shape == (sum(sizes), -(-most // 32)) and slots.dtype == torch.int64
    for b, (n, c) in enumerate(zip(sizes, ctx)):
        lo = int(cu[b])
        bits = O.sees(parents[lo : lo + n])
        assert torch.equal(masks[lo : lo + n], O.words(bits, masks.shape[1]))
        assert torch.equal(positions[lo : lo + n], (c + bits.sum(1) - 1).to(torch.int32))
        for j in range(n):
            assert int(slots[lo + j]) == int(table[b, (c + j) // block]) * block + (c + j) % block


def test_rows_behind_the_last_sequence_and_bad_parents():
    parents = torch.tensor([-1, 0, 5, 1, -1, 9, 9], dtype=torch.int32)
    masks, positions, slots = S.tree_rows(parents, torch.tensor([0, 4, 5], dtype=torch.int32), torch.tensor([2, 14], dtype=torch.int32), torch.tensor([[3], [1]], dtype=torch.int32),
                                          16, max_rows=4)
    assert masks[:, 0].tolist() == [1, 3, 4, 11, 1, 0, 0] and positions.tolist() == [2, 3, 2, 4, 14, 0, 0]
    assert slots.tolist() == [50, 51, 52, 53, 30, -1, -1]


@pytest.mark.parametrize("window", [0, 6])
@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,block", [(4, 2, 64, 16), (3, 3, 128, 48)])
def test_attention_restatement(Hq, Hkv, D, block, chain, window):
    sizes, ctx = [4, 1, 0, 9], [20, 0, 5, 47]
    q, k, v, table, ctx_t, cu, parents = _attend_case(sizes, ctx, Hq, Hkv, D, block)
    masks, positions, _ = S.tree_rows(parents, cu, ctx_t, table.clamp(min=0), block, max_rows=9)
    if chain:
        masks, positions = None, torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, sizes)]).to(torch.int32)
    bits = None if chain else [O.sees(parents[cu[b] : cu[b + 1]]) for b in range(4)]
    want, _ = O.attend(q, k, v, table, ctx_t, cu, Hq, Hkv, D, bits, window=window, positions=positions)
    got = S.tree_paged_decode(q, k, v, table, ctx_t, cu, Hq, Hkv, D, max_rows=9, masks=masks, window=window, positions=positions)
    assert torch.allclose(got.double(), want, rtol=1e-4, atol=1e-5)      # (32 bits; sums of at most 128 products and 56 keys)


def test_one_row_is_paged_decode():
    """A tree of one row whose key stands in the cache sees what paged decode's query does."""
    q, k, v, table, ctx, cu, _ = _attend_case([1, 1], [33, 5], 4, 2, 64, 16)
    got = S.tree_paged_decode(q, k, v, table, ctx, cu, 4, 2, 64, max_rows=1)
    assert torch.allclose(got, E.paged_decode(q, k, v, table, ctx + 1, 4, 2, 64), rtol=1e-5, atol=1e-6)


def _verify_case(sizes, V, seed, children=2, draft=False, dtype=torch.float32, chain=False):
    g = torch.Generator().manual_seed(seed)
    parents, cu = O.forest(sizes, seed, children, chain)
    T = int(cu[-1])
    logits = (torch.randn((T, V), generator=g) * 2).to(dtype)
    guess = (logits.float() + torch.randn((T, V), generator=g)).to(dtype)
    tokens = torch.zeros(T, dtype=torch.int32)
    for b, n in enumerate(sizes):
        used = {}
        for j in range(1, n):
            p = int(cu[b]) + int(parents[int(cu[b]) + j])
            used[p] = used.get(p, -1) + 1
            x = torch.multinomial(torch.softmax(guess[p].float(), -1), 1, generator=g) if draft else guess[p].float().topk(children).indices[used[p]]
            tokens[int(cu[b]) + j] = int(x)
    return logits, guess if draft else None, tokens, parents, cu, torch.rand(T, generator=g)


def _same(got, want, steps):
    tokens, counts, rows, logprobs = (x.cpu() for x in got)
    for b, (t, r, lp, _) in enumerate(want):
        n = len(t)
        pad = [-1] * (steps - n)
        assert int(counts[b]) == n and tokens[b].tolist() == t + pad and rows[b].tolist() == r + pad
        for i in range(steps):
            x, y = float(logprobs[b, i]), lp[i] if i < n else 0.0
            assert x == y or abs(x - y) <= 2.0**-23 * abs(y) + 1e-12      # (one rounding to 32 bits of what is computed in 64)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("sizes,V,children", [([1], 3, 1), ([2, 5], 40, 1), ([7, 0, 16, 3], 300, 3), ([33], 1000, 2)])
def test_verify_restatement(sizes, V, children, draft):
    most = max(sizes)
    for seed in range(4):
        logits, guess, tokens, parents, cu, u = _verify_case(sizes, V, seed, children, draft)
        for kw in (dict(), dict(temperature=0.7), dict(greedy=True), dict(temps=torch.tensor([0.5 + i for i in range(len(sizes))])), dict(max_steps=max(1, most // 2))):
            temps = kw.get("temps", torch.full((len(sizes),), kw.get("temperature", 1.0), dtype=torch.float64))
            steps = kw.get("max_steps", most)
            want = O.verify(logits, tokens, parents, cu, u, guess, temps, kw.get("greedy", False), steps)
            if min(w[3] for w in want) > 1e-9:
                _same(S.verify_drafts(logits, tokens, parents, cu, u, max_rows=most, draft_logits=guess, **kw), want, steps)


@pytest.mark.parametrize("draft,children", [(False, 2), (True, 1), (True, 2)])
def test_verify_keeps_the_targets_distribution(draft, children):
    """The first kept token of many trees is distributed as the target's samples: chi-square of 7 tokens below 36 (six degrees of freedom, chance 3e-6)."""
    V, B = 7, 4000
    g = torch.Generator().manual_seed(5)
    row = torch.randn(V, generator=g)
    guess = row + torch.randn(V, generator=g)
    n = 1 + children
    parents = torch.tensor([-1] + [0] * children, dtype=torch.int32).repeat(B)
    cu = torch.arange(0, (B + 1) * n, n, dtype=torch.int32)
    tokens = torch.zeros((B, n), dtype=torch.int32)
    if draft:
        tokens[:, 1:] = torch.multinomial(torch.softmax(guess, -1), B * children, replacement=True, generator=g).reshape(B, children)
    else:
        tokens[:, 1:] = guess.topk(children).indices
    T = B * n
    got = S.verify_drafts(row.expand(T, V).contiguous(), tokens.reshape(-1), parents, cu, torch.rand(T, generator=g), max_rows=n,
                          draft_logits=guess.expand(T, V).contiguous() if draft else None, max_steps=2)[0][:, 0]
    want = torch.softmax(row, -1) * B
    assert float(((torch.bincount(got.long(), minlength=V) - want) ** 2 / want).sum()) < 36


def test_a_draft_that_is_the_target_is_always_kept():
    logits, _, tokens, parents, cu, _ = _verify_case([6, 4], 50, 2, 1, True, chain=True)
    u = torch.full((10,), 1 - 2.0**-24)
    tokens, counts, rows, _ = S.verify_drafts(logits, tokens, parents, cu, u, max_rows=6, draft_logits=logits)
    assert counts.tolist() == [6, 4] and rows[1].tolist() == [0, 1, 2, 3, -1, -1]


def test_verify_of_rows_without_probabilities():
    """Logits that are not numbers weigh nothing; +inf shares with the largest number; a row without a number above -inf gives token 0."""
    logits = torch.tensor([[math.nan, 1.0, 2.0], [-math.inf] * 3, [math.inf, 0.0, O.FMAX], [math.nan] * 3])
    parents, cu = torch.tensor([-1, -1, -1, -1], dtype=torch.int32), torch.arange(5, dtype=torch.int32)
    tokens, counts, rows, lp = S.verify_drafts(logits, torch.zeros(4, dtype=torch.int32), parents, cu, torch.tensor([0.0, 0.5, 0.75, 0.1]), max_rows=1)
    assert tokens[:, 0].tolist() == [1, 0, 2, 0] and counts.tolist() == [1] * 4
    assert lp[1, 0] == -math.inf and lp[3, 0] == -math.inf and abs(float(lp[2, 0]) + math.log(2)) < 1e-6


def test_keep():
    g = torch.Generator().manual_seed(0)
    block, ctx, S_ = 16, [5, 14, 30], 4
    table, count = O.pages([c + 12 for c in ctx], block)
    caches = [(torch.randn((count, 2, block, 8), generator=g), torch.randn((count, 2, block, 8), generator=g)) for _ in range(3)]
    before = [(k.clone(), v.clone()) for k, v in caches]
    rows = torch.tensor([[0, 2, 3, 7], [0, 1, 2, 3], [0, 4, 11, -1]], dtype=torch.int32)
    counts = torch.tensor([4, 3, 0], dtype=torch.int32)
    shared = caches[1][0]
    S.kv_cache_keep([caches[0], None, (caches[1][0], caches[1][1]), (shared, caches[2][1])], table, torch.tensor(ctx, dtype=torch.int32), rows, counts)
    for x, y in [(caches[0], before[0]), (caches[1], before[1])]:
        for a, b in zip(x, y):
            want = b.clone()
            for i, r in enumerate([0, 2, 3, 7]):
                p, s = 5 + i, 5 + r
                want[table[0, p // block], :, p % block] = b[table[0, s // block], :, s % block]
            assert torch.equal(a, want)
    assert torch.equal(caches[2][0], before[2][0])


def test_refusals():
    q, k, v, table, ctx, cu, parents = _attend_case([2, 3], [5, 9], 4, 2, 64, 16)
    ok = dict(max_rows=3)
    run = lambda **kw: S.tree_paged_decode(**{**dict(q=q, k_cache=k, v_cache=v, block_table=table, ctx_lens=ctx, cu_rows=cu, Hq=4, Hkv=2, D=64), **ok, **kw})  # noqa: E731
    run()
    for bad in (dict(D=32), dict(Hq=5), dict(Hkv=3), dict(max_rows=0), dict(max_rows=257), dict(cu_rows=cu.long()), dict(ctx_lens=ctx.long()), dict(block_table=table.long()),
                dict(block_table=table[:1]), dict(k_cache=k.bfloat16()), dict(k_cache=k[:, :, :8]), dict(k_cache=k[:1]), dict(v_cache=v.transpose(0, 1)), dict(window=-1), dict(window=4),
                dict(scale=math.nan), dict(scale=math.inf), dict(masks=torch.zeros((5, 0), dtype=torch.int32)), dict(masks=torch.zeros((4, 1), dtype=torch.int32)),
                dict(masks=torch.zeros((5, 1))), dict(window=4, positions=torch.zeros(4, dtype=torch.int32)), dict(out=torch.zeros(5, 255)), dict(out=torch.zeros(5, 256).bfloat16()),
                dict(out=torch.zeros(256).expand(5, 256)), dict(out=torch.zeros(5, 512)[:, ::2]), dict(q=q[:, :128]), dict(q=q.clone().requires_grad_())):
        with pytest.raises(ValueError):
            run(**bad)
    for bad in (dict(parents=parents.long()), dict(block_size=0), dict(max_rows=300), dict(ctx_lens=ctx[:1])):
        with pytest.raises(ValueError):
            S.tree_rows(**{**dict(parents=parents, cu_rows=cu, ctx_lens=ctx, block_table=table, block_size=16, max_rows=3), **bad})
    logits, guess, tokens, parents, cu, u = _verify_case([2, 3], 20, 0, 2, True)
    for bad in (dict(logits=logits.double()), dict(logits=logits[0]), dict(tokens=tokens.long()), dict(parents=parents[:3]), dict(uniforms=u.double()), dict(uniforms=u[:2]),
                dict(draft_logits=guess.bfloat16()), dict(draft_logits=guess[:, :4]), dict(temps=torch.ones(3)), dict(temperature=math.nan), dict(max_steps=0), dict(max_steps=4),
                dict(logits=logits.clone().requires_grad_())):
        with pytest.raises(ValueError):
            S.verify_drafts(**{**dict(logits=logits, tokens=tokens, parents=parents, cu_rows=cu, uniforms=u, max_rows=3, draft_logits=guess), **bad})
    rows, counts = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for bad in (dict(caches=[(k[..., :3], v)]), dict(caches=[(k.transpose(0, 1), v)]), dict(rows=rows.long()), dict(rows=rows[0]), dict(counts=counts[:1]), dict(ctx_lens=ctx.long()),
                dict(block_table=table[:1])):
        with pytest.raises(ValueError):
            S.kv_cache_keep(**{**dict(caches=[(k, v)], block_table=table, ctx_lens=ctx, rows=rows, counts=counts), **bad})


def test_refusals_of_what_32_bits_do_not_count():
    """Scales that are infinite times log2(e), more tokens than places of a row are counted to (rows of none, so that nothing of that size is held)."""
    q, k, v, table, ctx, cu, _ = _attend_case([2], [5], 4, 2, 64, 16)
    for scale in (3e38, -2.4e38):
        with pytest.raises(ValueError):
            S.tree_paged_decode(q, k, v, table, ctx, cu, 4, 2, 64, max_rows=3, scale=scale)
    none, zero = torch.zeros(0, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        S.verify_drafts(torch.zeros((0, 2**30 + 1)), none, none, zero, torch.zeros(0), max_rows=4)
    assert S.verify_drafts(torch.zeros((0, 2**30)), none, none, zero, torch.zeros(0), max_rows=4)[1].tolist() == [0]


def test_empty_batches():
    none = torch.zeros(0, dtype=torch.int32)
    cu, table = torch.zeros(1, dtype=torch.int32), torch.zeros((0, 1), dtype=torch.int32)
    assert S.tree_rows(none, cu, none, table, 16, max_rows=4)[0].shape == (0, 1)
    k = torch.zeros((1, 1, 16, 64))
    assert S.tree_paged_decode(torch.zeros(0, 64), k, k, table, none, cu, 1, 1, 64, max_rows=4).shape == (0, 64)
    assert S.verify_drafts(torch.zeros(0, 5), none, none, cu, torch.zeros(0), max_rows=4)[0].shape == (0, 4)
    S.kv_cache_keep([(k, k)], table, none, torch.zeros((0, 4), dtype=torch.int32), none)


def masked_case(V, sizes, seed, draft, dtype=torch.float32, most=6):
    """Rows of which a filter or a grammar has left a few tokens (the draft's has left others beside some of them), children that are often turned down, and row 0's number zero for
    every other sequence."""
    g = torch.Generator().manual_seed(seed)
    parents, cu = O.forest(sizes, seed, 3)
    T = int(cu[-1])
    logits, guess = torch.full((T, V), -math.inf), torch.full((T, V), -math.inf)
    for t in range(T):
        few = torch.randperm(V, generator=g)[: 2 + int(torch.randint(most - 1, (1,), generator=g))]
        logits[t, few] = torch.randn(len(few), generator=g)
        both = few[torch.rand(len(few), generator=g) < 0.8]
        guess[t, both] = logits[t, both] + torch.randn(len(both), generator=g)
        guess[t, torch.randint(V, (2,), generator=g)] = 0.3
    logits, guess = logits.to(dtype), guess.to(dtype)
    tokens, used = torch.zeros(T, dtype=torch.int32), {}
    for b, n in enumerate(sizes):
        for j in range(1, n):
            p = int(cu[b]) + int(parents[int(cu[b]) + j])
            used[p] = used.get(p, -1) + 1
            best = logits[p].float().topk(min(2, V)).indices
            tokens[int(cu[b]) + j] = int(torch.multinomial(torch.softmax(guess[p].float(), -1), 1, generator=g)) if draft else int(best[-1 - used[p] % len(best)])
    u = torch.rand(T, generator=g) ** 0.1
    u = u.clamp(max=1 - 2.0**-20)
    u[cu[:-1].long()[::2]] = 0.0
    u[cu[:-1].long()[1::2]] = torch.rand(len(u[cu[:-1].long()[1::2]]), generator=g)
    return logits, guess if draft else None, tokens, parents, cu, u


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("V", [9, 1000])
def test_verify_restatement_on_masked_logits(V, draft):
    for seed in range(4):
        sizes = [4, 1, 7, 2, 5, 3]
        logits, guess, tokens, parents, cu, u = masked_case(V, sizes, seed, draft)
        want = O.verify(logits, tokens, parents, cu, u, guess)
        assert min(w[3] for w in want) > 1e-9
        _same(S.verify_drafts(logits, tokens, parents, cu, u, max_rows=7, draft_logits=guess), want, 7)


def test_greedy_takes_the_largest_logit_at_any_temperature():
    """Logits that are alike once a large temperature has divided them."""
    z = torch.tensor([[0.0, 1.0, 5.0, 2.0], [3.0, 3.0 + 2.0**-21, math.nan, -1.0], [O.FMAX, math.inf, 0.0, O.FMAX], [-math.inf, -2.0, -2.0, -math.inf]])
    parents, cu = torch.tensor([-1, -1, -1, -1], dtype=torch.int32), torch.arange(5, dtype=torch.int32)
    for kw in (dict(temperature=x) for x in (1e-30, 1.0, 1e20, math.inf)):
        got = S.verify_drafts(z, torch.zeros(4, dtype=torch.int32), parents, cu, torch.full((4,), 0.9), max_rows=1, greedy=True, **kw)
        assert got[0][:, 0].tolist() == [2, 1, 0, 1]
    tokens, _, rows, _ = S.verify_drafts(z[[0, 0, 0]], torch.tensor([0, 0, 2], dtype=torch.int32), torch.tensor([-1, 0, 0], dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32),
                                         torch.zeros(3), max_rows=3, greedy=True, temperature=1e20)
    assert tokens[0].tolist() == [2, 2, -1] and rows[0].tolist() == [0, 2, -1]


@pytest.mark.parametrize("cu,T,owners", [([0, 5, 2], 5, [0] * 5), ([0, 5, 3, 8], 9, [0] * 5 + [2] * 3 + [None]), ([4, 2, 6], 7, [None] * 4 + [1] * 2 + [None]), ([0, 4, 1, 3, 6], 6, [0] * 4 + [3] * 2),
                                         ([0, 9, 2], 5, [0] * 5)])
def test_rows_that_several_sequences_name(cu, T, owners):
    """Offsets that do not ascend: a row is the first one's that names it, and one that a sequence has is not one behind the last."""
    ctx = torch.arange(len(cu) - 1, dtype=torch.int32) * 100
    table = torch.arange(30 * len(ctx), dtype=torch.int32).reshape(-1, 30)
    parents = torch.full((T,), -1, dtype=torch.int32)
    masks, positions, slots = S.tree_rows(parents, torch.tensor(cu, dtype=torch.int32), ctx, table, 16, max_rows=8)
    for t, b in enumerate(owners):
        j = t - cu[b] if b is not None else 0
        assert int(masks[t, 0]) == (1 << j if b is not None else 0) and int(positions[t]) == (int(ctx[b]) if b is not None else 0)
        assert int(slots[t]) == (30 * 16 * b + int(ctx[b]) + j if b is not None else -1)


def test_pages_that_are_not_there_are_left_out():
    """Of a table's entries below zero and behind the cache's last page nothing is read, moved or written."""
    q, k, v, table, ctx, cu, _ = _attend_case([5, 18], [70, 3], 4, 2, 64, 16, seed=6)
    bad = table.clone()
    bad[0, 1], bad[0, 3] = k.shape[0], -1
    got = S.tree_paged_decode(q, k, v, bad, ctx, cu, 4, 2, 64, max_rows=18)
    left = torch.tensor([t for t in range(75) if not (16 <= t < 32 or 48 <= t < 64)])
    kk, vv = (torch.zeros((3, 2, 16, 64)) for _ in range(2))
    for x, y in ((kk, k), (vv, v)):
        for i, t in enumerate(left.tolist()):
            x[i // 16, :, i % 16] = y[table[0, t // 16], :, t % 16]
    want = S.tree_paged_decode(q[:5], kk, vv, torch.arange(3, dtype=torch.int32)[None], torch.tensor([38], dtype=torch.int32), torch.tensor([0, 5], dtype=torch.int32), 4, 2, 64, max_rows=18)
    assert torch.allclose(got[:5], want, rtol=1e-4, atol=1e-5)
    assert torch.equal(got[5:], S.tree_paged_decode(q, k, v, table, ctx, cu, 4, 2, 64, max_rows=18)[5:])
    none = S.tree_paged_decode(q, k, v, torch.full_like(table, -1), ctx, cu, 4, 2, 64, max_rows=18)
    assert not none.any()
    for page, rows in ((-1, [0, 1, 2, 20]), (9, [0, 1, 2, 20]), (-3, [0, 17, 20, 21])):      # the source's page, the targets'
        caches = [(torch.randn((4, 2, 16, 8)), torch.randn((4, 2, 16, 8)))]
        t = torch.tensor([[1, page]] if rows[1] == 1 else [[page, 2]], dtype=torch.int32)
        before = caches[0][0].clone(), caches[0][1].clone()
        S.kv_cache_keep(caches, t, torch.tensor([0], dtype=torch.int32), torch.tensor([rows], dtype=torch.int32), torch.tensor([4], dtype=torch.int32))
        assert torch.equal(caches[0][0], before[0]) and torch.equal(caches[0][1], before[1])


def test_values_that_are_not_finite_reach_the_rows_that_see_them():
    """And no others: rows of other branches, rows whose window or context ends before."""
    q, k, v, table, ctx, _, _ = _attend_case([6, 4], [20, 33], 4, 2, 64, 16, seed=3)
    parents, cu = torch.tensor([-1, 0, 0, 1, 2, 4, -1, 0, 1, 1], dtype=torch.int32), torch.tensor([0, 6, 10], dtype=torch.int32)
    masks, positions, _ = S.tree_rows(parents, cu, ctx, table.clamp(min=0), 16, max_rows=6)
    run = lambda values, **kw: S.tree_paged_decode(q, k, values, table, ctx, cu, 4, 2, 64, max_rows=6, masks=masks, **kw)  # noqa: E731
    for place, blind, window in ((22, [0, 1, 3, 6, 7, 8, 9], 0), (0, [0, 1, 2, 3, 4, 5, 6, 7, 8, 9], 8), (14, [1, 2, 3, 4, 5, 6, 7, 8, 9], 7)):
        kw = dict(window=window, positions=positions) if window else {}
        bad = v.clone()
        bad[table[0, place // 16], :, place % 16] = torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(64) % 3]
        got, want = run(bad, **kw), run(v, **kw)
        assert torch.equal(got[blind], want[blind])
        for r in set(range(10)) - set(blind):
            x = got[r].reshape(4, 64)
            assert x[:, 0::3].isnan().all() and (x[:, 1::3] == math.inf).all() and (x[:, 2::3] == -math.inf).all()


def faint_case(V=4096):
    """Two tokens have the target's weight and two the draft's; all others are so faint (2^-999 and 2^-1001 of the largest) that a draft which took nothing off them would leave them."""
    z, d = torch.full((4, V), -692.2), torch.full((4, V), -690.4)
    z[:, 300], z[:, 2000], d[:, 300], d[:, 17] = 0.0, 0.02, 3.0, 0.3
    tokens, parents = torch.tensor([0, 17, 300, 300], dtype=torch.int32), torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
    return (z, tokens, parents, torch.tensor([0, 4], dtype=torch.int32), torch.tensor([0.0, 0.999, 0.999, 0.999])), d


def test_verify_of_what_is_nearly_nothing():
    args, d = faint_case()
    want = O.verify(args[0], *args[1:4], args[4], d)
    assert want[0][:2] == ([2000], [0])
    _same(S.verify_drafts(*args, max_rows=4, draft_logits=d), want, 4)
