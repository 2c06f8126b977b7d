"""Kernels of speculative decoding: trees' rows and the accepted rows' move exactly, attention within the roundings that the oracle counts, verification by its decisions."""

import math

import draft_oracle as O
import pytest
import torch
from test_draft_ops import _same, _verify_case, faint_case, masked_case

from rl_b200.ops import draft_ops as S
from rl_b200.ops import engine_ops as E
from rl_b200.ops import lib as L

pytestmark = pytest.mark.gpu

I32 = torch.int32


def _dev(*ts):
    return [t.cuda() if t is not None else None for t in ts]


@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("sizes,ctx,block", [([1], [0], 16), ([6], [300], 16), ([33, 0, 1, 64, 17], [0, 5, 15, 63, 1000], 64), ([256, 255, 1], [31, 1, 0], 48)])
def test_rows(native_lib, sizes, ctx, block, chain):
    parents, cu = O.forest(sizes, 1, chain=chain)
    table, _ = O.pages([c + n for c, n in zip(ctx, sizes)], block)
    parents = torch.cat([parents, torch.full((5,), -1, dtype=I32)])      # rows behind the last sequence
    ctx = torch.tensor(ctx, dtype=I32)
    want = S.tree_rows(parents, cu, ctx, table, block, max_rows=max(sizes))
    wide = torch.full((table.shape[0], table.shape[1] + 3), -1, dtype=I32).cuda()
    wide[:, : table.shape[1]] = table.cuda()
    got = S.tree_rows(*_dev(parents, cu, ctx), wide[:, : table.shape[1]], block, max_rows=max(sizes))
    for x, y in zip(got, want):
        assert torch.equal(x.cpu(), y)
    assert L.check_status() == 0


def test_rows_reports_what_is_left_out(native_lib):
    """Parents that are not above their row, rows over max_rows, places outside the table."""
    for parents, cu, ctx, most in (([-1, 0, 5, 1], [0, 4], [2], 4), ([-1, 0, 1, 2], [0, 4], [2], 3), ([-1, 0, 1, 2], [0, 4], [14], 4), ([-1, 0, 1, 2], [2, 0], [0], 4)):
        args = [torch.tensor(x, dtype=I32) for x in (parents, cu, ctx, [[3]])]
        want = S.tree_rows(*args, 16, max_rows=most)
        got = S.tree_rows(*_dev(*args), 16, max_rows=most)
        cut = most if most < 4 else 0 if cu[1] == 0 else 4
        for x, y in zip(got, want):
            assert torch.equal(x.cpu()[:cut], y[:cut])
        assert L.check_status() == 8


@pytest.mark.parametrize("cu,most", [([3, 5, 9], 4), ([0, 6, 9], 4), ([2, 300, 301], 256)])
def test_rows_that_are_left_out_have_no_place(native_lib, cu, most):
    """Rows before the first sequence, and those over max_rows: whatever the results' memory held."""
    T = cu[-1] + 3
    args = [torch.tensor(x, dtype=I32) for x in ([-1] * T, cu, [7, 20], [list(range(30)), list(range(30, 60))])]
    want = S.tree_rows(*args, 16, max_rows=most)
    held = [torch.full((T, n), 77, dtype=t, device="cuda") for n, t in ((-(-most // 32), I32), (1, I32), (1, torch.int64))]
    del held      # (their places are the next ones to be given out)
    got = S.tree_rows(*_dev(*args), 16, max_rows=most)
    for x, y in zip(got, want):
        assert torch.equal(x.cpu(), y)
    assert L.check_status() == (8 if cu[1] - cu[0] > most else 0)


def _attend_case(sizes, ctx, Hq, Hkv, D, block, seed=0, chain=False):
    g = torch.Generator().manual_seed(seed)
    parents, cu = O.forest(sizes, seed, chain=chain)
    table, count = O.pages([c + n for c, n in zip(ctx, sizes)], block, seed)
    k, v = (torch.randn((count, Hkv, block, D), generator=g).bfloat16() for _ in range(2))
    k[..., 3] *= 4
    q = (torch.randn((int(cu[-1]), (Hq + 2 * Hkv) * D), generator=g) * 1.5).bfloat16()
    return q, k, v, table, torch.tensor(ctx, dtype=I32), cu, parents


def _bits(parents, cu):
    return [O.sees(parents[int(cu[b]) : int(cu[b + 1])]) for b in range(len(cu) - 1)]


def _masks(bits, most):
    return torch.cat([O.words(x, -(-most // 32)) for x in bits])


def _check(case, Hq, Hkv, D, most, bits=None, plan=None, **kw):
    q, k, v, table, ctx, cu, _ = case
    masks = _masks(bits, most) if bits is not None else None
    want, tol = O.attend(q, k, v, table, ctx, cu, Hq, Hkv, D, bits, **kw)
    if "positions" in kw:
        kw["positions"] = kw["positions"].cuda()
    got = S.tree_paged_decode(q.cuda()[:, : Hq * D], *_dev(k, v, table, ctx, cu), Hq, Hkv, D, max_rows=most, masks=masks.cuda() if masks is not None else None, plan=plan, **kw)
    assert L.check_status() == 0
    n = int(cu[-1])
    off = (got.cpu().double() - want).abs()[:n] - tol[:n] - 1e-30
    assert got.isfinite().all() and float(off.max()) <= 0, f"{int((off > 0).sum())} of {off.numel()} outside, worst {float((off / (tol[:n] + 1e-30)).max())} of the tolerance over it"
    return got


HEADS = {64: [(14, 2), (16, 1), (4, 4)], 128: [(8, 2), (7, 1), (3, 3), (32, 2)]}


@pytest.mark.parametrize("D,Hq,Hkv", [(D, *h) for D in HEADS for h in HEADS[D]])
@pytest.mark.parametrize("chain", [False, True])
@pytest.mark.parametrize("sizes,ctx,block", [([1], [0], 16), ([5], [1], 16), ([6, 0, 17, 1], [300, 7, 0, 63], 16), ([9, 8, 40], [55, 64, 129], 48), ([33, 3], [127, 1001], 128)])
def test_attention(native_lib, D, Hq, Hkv, sizes, ctx, block, chain):
    case = _attend_case(sizes, ctx, Hq, Hkv, D, block, seed=len(sizes), chain=chain)
    _check(case, Hq, Hkv, D, max(sizes), None if chain else _bits(case[6], case[5]))


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 8), (128, 16, 2)])
@pytest.mark.parametrize("sizes,ctx", [([256], [1]), ([129, 200], [70, 300]), ([16] * 70, list(range(70)))])
def test_attention_of_many_rows(native_lib, sizes, ctx, D, Hq, Hkv):
    case = _attend_case(sizes, ctx, Hq, Hkv, D, 64, seed=7)
    _check(case, Hq, Hkv, D, max(sizes), _bits(case[6], case[5]))


@pytest.mark.parametrize("D,Hq,Hkv,batch,context", [(128, 8, 2, 1, 20000), (64, 4, 1, 3, 9000), (128, 4, 4, 2, 5001)])
def test_attention_of_long_contexts(native_lib, D, Hq, Hkv, batch, context):
    """Contexts that are cut into parts."""
    sizes, ctx = [7] * batch, [context // (i + 1) + i for i in range(batch)]
    case = _attend_case(sizes, ctx, Hq, Hkv, D, 64, seed=9)
    _check(case, Hq, Hkv, D, 7, _bits(case[6], case[5]))


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 4, 4)])
@pytest.mark.parametrize("window", [1, 3, 64, 100, 5000])
def test_attention_in_a_window(native_lib, window, D, Hq, Hkv):
    sizes, ctx = [20, 0, 5, 1], [300, 0, 63, 4]
    case = _attend_case(sizes, ctx, Hq, Hkv, D, 32, seed=window)
    bits = _bits(case[6], case[5])
    positions = torch.cat([c + x.sum(1) - 1 for c, x in zip(ctx, bits)]).to(I32)
    _check(case, Hq, Hkv, D, 20, bits, window=window, positions=positions)
    positions = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, sizes)]).to(I32)
    _check(case, Hq, Hkv, D, 20, None, window=window, positions=positions)


def test_masks_of_any_kind(native_lib):
    """Bits that are no tree's, a row without a key (zeros), rows that do not see themselves."""
    sizes, ctx = [40, 64, 3], [0, 130, 0]
    case = _attend_case(sizes, ctx, 8, 2, 128, 16, seed=4)
    g = torch.Generator().manual_seed(4)
    bits = [torch.rand((n, n), generator=g) < 0.4 for n in sizes]
    bits[0][7], bits[2][:] = False, False
    got = _check(case, 8, 2, 128, 64, bits)
    assert not got[7].any() and not got[104:].any()


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-38, 3.0])
def test_scales(native_lib, scale):
    case = _attend_case([5, 18], [70, 3], 8, 2, 128, 16, seed=2)
    _check(case, 8, 2, 128, 18, _bits(case[6], case[5]), scale=scale)


def test_nothing_comes_from_what_is_hidden(native_lib):
    """Infinities and values that are not numbers in other branches, behind the rows, in other sequences' pages and in places outside the window."""
    D, Hq, Hkv, block = 128, 8, 2, 32
    sizes, ctx = [6, 4], [70, 200]
    q, k, v, table, ctx_t, cu, _ = _attend_case(sizes, ctx, Hq, Hkv, D, block, seed=3)
    parents = torch.tensor([-1, 0, 0, 1, 2, 4, -1, 0, 1, 1], dtype=I32)
    bits = _bits(parents, cu)
    used = torch.zeros(k.shape[0], block, dtype=torch.bool)
    for b, (c, n) in enumerate(zip(ctx, sizes)):
        at = torch.arange(c + n)
        used[table[b].long()[at // block], at % block] = True
    poison = torch.tensor([math.nan, math.inf, -math.inf]).bfloat16()
    for x in (k, v):
        x.permute(0, 2, 1, 3)[~used] = poison[torch.arange(D) % 3]
    clean = (k.clone(), v.clone())
    want = S.tree_paged_decode(*_dev(q, *clean, table, ctx_t, cu), Hq, Hkv, D, max_rows=6, masks=_masks(bits, 6).cuda()).cpu()
    ref, tol = O.attend(q, k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0), table, ctx_t, cu, Hq, Hkv, D, bits)
    assert ((want.double() - ref).abs() <= tol).all()
    place = 70 + 2      # row 2 of the first tree: seen by rows 2, 4 and 5 alone
    for x in (k, v):
        x[table[0, place // block], :, place % block] = poison[torch.arange(D) % 3]
    got = S.tree_paged_decode(*_dev(q, k, v, table, ctx_t, cu), Hq, Hkv, D, max_rows=6, masks=_masks(bits, 6).cuda()).cpu()
    blind = [0, 1, 3, 6, 7, 8, 9]
    assert torch.equal(got[blind], want[blind]) and not got[[2, 4, 5]].isfinite().all(-1).any()
    # values alone: a row that sees an infinite value has it
    k2, v2 = clean
    v2[table[0, place // block], :, place % block] = poison[torch.arange(D) % 3]
    got = S.tree_paged_decode(*_dev(q, k2, v2, table, ctx_t, cu), Hq, Hkv, D, max_rows=6, masks=_masks(bits, 6).cuda()).cpu()
    assert torch.equal(got[blind], want[blind])
    for r in (2, 4, 5):
        x = got[r].reshape(Hq, D)
        assert x[:, 0::3].isnan().all() and (x[:, 1::3] == math.inf).all() and (x[:, 2::3] == -math.inf).all()
    # in a window, places before it
    positions = torch.cat([c + x.sum(1) - 1 for c, x in zip(ctx, bits)]).to(I32)
    k3, v3 = (x.clone() for x in (k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)))
    before = S.tree_paged_decode(*_dev(q, k3, v3, table, ctx_t, cu), Hq, Hkv, D, max_rows=6, masks=_masks(bits, 6).cuda(), window=10, positions=positions.cuda()).cpu()
    for x in (k3, v3):
        for b, c in enumerate(ctx):
            for place in range(c - 9):
                x[table[b, place // block], :, place % block] = poison[torch.arange(D) % 3]
    after = S.tree_paged_decode(*_dev(q, k3, v3, table, ctx_t, cu), Hq, Hkv, D, max_rows=6, masks=_masks(bits, 6).cuda(), window=10, positions=positions.cuda()).cpu()
    assert torch.equal(before, after) and L.check_status() == 0


def test_rows_of_any_place(native_lib):
    """Fused rows, rows that start on an odd element, wider outputs, rows behind the last sequence, tables cut from wider ones: the same numbers, and nothing else is written."""
    D, Hq, Hkv = 64, 6, 2
    q, k, v, table, ctx, cu, parents = _attend_case([5, 18], [70, 3], Hq, Hkv, D, 16, seed=6)
    masks = _masks(_bits(parents, cu), 18)
    args = _dev(k, v, table, ctx, cu)
    q = torch.cat([q, q[:4]]).cuda()      # 23 rows of sequences and 4 others
    masks = torch.cat([masks, masks[:4]]).cuda()
    want = S.tree_paged_decode(q[:, : Hq * D].contiguous(), *args, Hq, Hkv, D, max_rows=18, masks=masks)[:23]
    odd = torch.empty(27, Hq * D + 3, dtype=torch.bfloat16, device="cuda")[:, 1 : 1 + Hq * D].copy_(q[:, : Hq * D])
    wide = torch.full((23 + 4, masks.shape[1] + 2), -1, dtype=I32, device="cuda")
    wide[:, : masks.shape[1]] = masks
    same = q[:1, : Hq * D].expand(27, -1)      # rows that share their place
    one = S.tree_paged_decode(same.contiguous(), *args, Hq, Hkv, D, max_rows=18, masks=masks)[:23]
    assert torch.equal(S.tree_paged_decode(same, *args, Hq, Hkv, D, max_rows=18, masks=masks)[:23], one)
    for x, m in ((q, masks), (odd, masks), (q, wide[:, : masks.shape[1]])):
        out = torch.full((27, Hq * D + 5), 9.0, dtype=torch.bfloat16, device="cuda")
        for place in (out[:, : Hq * D], out[:, 3 : 3 + Hq * D]):
            out.fill_(9.0)
            got = S.tree_paged_decode(x, *args, Hq, Hkv, D, max_rows=18, masks=m, out=place)
            assert got is place and torch.equal(place[:23], want) and (place[23:] == 9).all()
            place[:23] = 9.0
            assert (out == 9).all()
    assert L.check_status() == 0


def test_bad_pages_are_left_out(native_lib):
    """Pages that are not there and a context longer than the table are reported, and the rest is attended."""
    q, k, v, table, ctx, cu, parents = _attend_case([5, 18], [70, 3], 8, 2, 128, 16, seed=6)
    bad = table.clone()
    bad[0, 1], bad[0, 3] = k.shape[0], -1
    got = S.tree_paged_decode(*_dev(q, k, v, bad, ctx, cu), 8, 2, 128, max_rows=18).cpu()
    assert L.check_status() == 8
    keep = torch.ones(75, dtype=torch.bool)
    keep[16:32], keep[48:64] = False, False
    left = torch.arange(75)[keep]
    kk, vv = (torch.zeros(table.shape[1] + 1, 2, 16, 128).bfloat16() for _ in range(2))
    for i, p in enumerate(left.tolist()):
        for x, y in ((kk, k), (vv, v)):
            x[i // 16, :, i % 16] = y[table[0, p // 16], :, p % 16]
    want, tol = O.attend(q[:5], kk, vv, torch.arange(table.shape[1])[None], torch.tensor([38]), torch.tensor([0, 5]), 8, 2, 128)
    assert ((got[:5].double() - want).abs() <= tol).all()
    ok = S.tree_paged_decode(*_dev(q, k, v, table, ctx, cu), 8, 2, 128, max_rows=18).cpu()
    assert torch.equal(got[5:], ok[5:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("sizes,V,children", [([1], 1, 1), ([6], 3, 1), ([6], 32000, 1), ([7, 0, 16, 3] * 3, 300, 3), ([33, 2], 50257, 2), ([256, 1], 1025, 3), ([8] * 9, 4096, 2)])
def test_verify(native_lib, sizes, V, children, draft, dtype):
    most = max(sizes)
    if children > V:
        children = 1
    logits, guess, tokens, parents, cu, u = _verify_case(sizes, V, 11, min(children, V), draft, dtype)
    args, more = _dev(logits, tokens, parents, cu, u), dict(max_rows=most, draft_logits=guess.cuda() if draft else None)
    for kw in (dict(), dict(temperature=0.7), dict(greedy=True), dict(temps=torch.tensor([0.5 + 0.3 * i for i in range(len(sizes))])), dict(max_steps=max(1, most // 2))):
        temps = kw.get("temps", torch.full((len(sizes),), kw.get("temperature", 1.0), dtype=torch.float64))
        if "temps" in kw:
            temps[-1] = 0.0      # greedy
        steps = kw.get("max_steps", most)
        want = O.verify(logits, tokens, parents, cu, u, guess, temps, kw.get("greedy", False), steps)
        assert min(w[3] for w in want) > 1e-11      # (what both sides' 64 bits leave undecided; the generator's numbers are not that near to a border)
        _same(S.verify_drafts(*args, **more, **{k: x.cuda() if torch.is_tensor(x) else x for k, x in kw.items()}), want, steps)
    assert L.check_status() == 0


def test_verify_of_special_logits(native_lib):
    """As on the CPU: what is not a number, infinities, rows without probabilities, tokens outside the vocabulary, numbers at the ends of their range, equal largest logits."""
    V = 77
    g = torch.Generator().manual_seed(1)
    z = torch.randn((12, V), generator=g)
    z[0, :70], z[1], z[2, 5], z[2, 9], z[3] = math.nan, -math.inf, math.inf, O.FMAX, math.nan
    z[4, 3] = z[4, 50] = 9.0
    z[5, 1:] = -math.inf
    z[6] = z[6] * 1e30
    parents, cu = torch.tensor([-1] * 6 + [-1, 0, 0, 1, 0, 3], dtype=I32), torch.tensor([0, 1, 2, 3, 4, 5, 6, 12], dtype=I32)
    tokens = torch.tensor([0] * 6 + [0, -5, V, 1, int(z[6].argmax()), 2], dtype=I32)
    for u0 in (0.0, 0.3, 1 - 2.0**-24, 1.0, math.nan):
        u = torch.full((12,), u0)
        for kw in (dict(), dict(greedy=True), dict(temperature=0.01), dict(temperature=math.inf), dict(temperature=-1.0)):
            want = S.verify_drafts(z, tokens, parents, cu, u, max_rows=6, **kw)
            got = S.verify_drafts(*_dev(z, tokens, parents, cu, u), max_rows=6, **kw)
            for x, y in zip(got[:3], want[:3]):
                assert torch.equal(x.cpu(), y)
            assert torch.allclose(got[3].cpu(), want[3], rtol=2.0**-23, atol=1e-12)
    assert L.check_status() == 0


def test_verify_reads_rows_where_they_are(native_lib):
    """Wider logits, rows that start on odd elements, rows behind the last sequence."""
    logits, guess, tokens, parents, cu, u = _verify_case([7, 3, 5], 1000, 3, 2, True)
    want = S.verify_drafts(logits, tokens, parents, cu, u, max_rows=7, draft_logits=guess)
    wide = torch.full((18, 1013), 50.0, device="cuda")
    pad = torch.zeros(3, dtype=I32)
    for dtype in (torch.float32, torch.bfloat16):
        want = S.verify_drafts(logits.to(dtype), tokens, parents, cu, u, max_rows=7, draft_logits=guess.to(dtype))
        for off in (0, 1, 8):
            w = wide.to(dtype)
            w[:15, off : off + 1000] = logits.to(dtype).cuda()
            d = torch.cat([guess, guess[:3]]).to(dtype).cuda()
            got = S.verify_drafts(w[:, off : off + 1000], *_dev(torch.cat([tokens, pad]), torch.cat([parents, pad]), cu, torch.cat([u, u[:3]])), max_rows=7, draft_logits=d)
            for x, y in zip(got[:3], want[:3]):
                assert torch.equal(x.cpu(), y)
    assert L.check_status() == 0


@pytest.mark.parametrize("draft,children", [(False, 2), (True, 2)])
def test_verify_keeps_the_targets_distribution(native_lib, draft, children):
    """Chi-square of 50 tokens below 120 (49 degrees of freedom: chance 6e-8)."""
    V, B, n = 50, 20000, 1 + children
    g = torch.Generator().manual_seed(5)
    row = torch.randn(V, generator=g)
    guess = row + torch.randn(V, generator=g)
    parents = torch.tensor([-1] + [0] * children, dtype=I32).repeat(B)
    cu = torch.arange(0, (B + 1) * n, n, dtype=I32)
    tokens = torch.zeros((B, n), dtype=I32)
    tokens[:, 1:] = torch.multinomial(torch.softmax(guess, -1), B * children, replacement=True, generator=g).reshape(B, children) if draft else guess.topk(children).indices
    T = B * n
    got = S.verify_drafts(row.cuda().expand(T, V).contiguous(), *_dev(tokens.reshape(-1), parents, cu, torch.rand(T, generator=g)), max_rows=n,
                          draft_logits=guess.cuda().expand(T, V).contiguous() if draft else None, max_steps=2)[0][:, 0].cpu()
    want = torch.softmax(row, -1) * B
    assert float(((torch.bincount(got.long(), minlength=V) - want) ** 2 / want).sum()) < 120


def test_a_draft_that_is_the_target_is_always_kept(native_lib):
    logits, _, tokens, parents, cu, _ = _verify_case([6, 4], 5000, 2, 1, True, chain=True)
    u = torch.full((10,), 1 - 2.0**-24)
    dev = _dev(logits, tokens, parents, cu, u)
    _, counts, rows, _ = S.verify_drafts(*dev, max_rows=6, draft_logits=dev[0])
    assert counts.tolist() == [6, 4] and rows[1].tolist() == [0, 1, 2, 3, -1, -1]


@pytest.mark.parametrize("dtype,D,Hkv,block", [(torch.bfloat16, 64, 2, 16), (torch.bfloat16, 128, 8, 64), (torch.float32, 20, 3, 7), (torch.uint8, 16, 1, 16)])
def test_keep(native_lib, dtype, D, Hkv, block):
    """As on the CPU, with sources that are targets of later rows, entries that do not ascend, and rows outside the table."""
    g = torch.Generator().manual_seed(0)
    ctx, steps = [5, 14, 30, 0, 61], 9
    table, count = O.pages([c + 20 for c in ctx], block)
    caches = [tuple((torch.randn((count, Hkv, block, D), generator=g) * 50).to(dtype) for _ in range(2)) for _ in range(3)]
    rows = torch.stack([torch.arange(steps), torch.arange(steps) + torch.arange(steps).clamp(max=1), torch.arange(steps) * 2, torch.tensor([0, 5, 3, 6, 6, 9, 1, 8, 19]),
                        torch.randperm(18, generator=g)[:steps].sort().values]).to(I32)
    counts = torch.tensor([9, 9, 5, 9, 8], dtype=I32)
    dev = [tuple(x.cuda() for x in pair) for pair in caches]
    ctx = torch.tensor(ctx, dtype=I32)
    S.kv_cache_keep(caches, table, ctx, rows, counts)
    S.kv_cache_keep([*dev, None, (dev[0][0], dev[1][1])], *_dev(table, ctx, rows, counts))
    for pair, want in zip(dev, caches):
        for x, y in zip(pair, want):
            assert torch.equal(x.cpu(), y)
    assert L.check_status() == 8      # (the fourth sequence's rows do not ascend)


def test_keep_of_many_layers(native_lib):
    """More tensors than one launch has room for."""
    caches = [(torch.arange(32.0).reshape(1, 1, 32, 1).repeat(1, 1, 1, 4).cuda() + i, torch.zeros(1, 1, 32, 4, device="cuda")) for i in range(70)]
    S.kv_cache_keep(caches, *_dev(torch.zeros((1, 1), dtype=I32), torch.tensor([3], dtype=I32), torch.tensor([[0, 4, 9]], dtype=I32), torch.tensor([3], dtype=I32)))
    for i, (k, _) in enumerate(caches):
        assert k[0, 0, 3:6, 0].tolist() == [3 + i, 7 + i, 12 + i]
    assert L.check_status() == 0


def _step(st):
    """One step of a program that decodes speculatively: rows, cache write, attention, verification, keep."""
    masks, positions, slots = S.tree_rows(st["parents"], st["cu"], st["ctx"], st["table"], 16, max_rows=9)
    qkv = st["qkv"].clone()
    E.rope_kv_cache_write(qkv, positions, st["freq"], slots, st["k"], st["v"], 4, 2, 64)
    y = S.tree_paged_decode(qkv, st["k"], st["v"], st["table"], st["ctx"], st["cu"], 4, 2, 64, max_rows=9, masks=masks)
    logits = (y.float() @ st["head"]).contiguous()
    tokens, counts, rows, logprobs = S.verify_drafts(logits, st["tokens"], st["parents"], st["cu"], st["u"], max_rows=9)
    S.kv_cache_keep([(st["k"], st["v"])], st["table"], st["ctx"], rows, counts)
    return y, logits, tokens, counts, rows, logprobs


def _program(seed=0):
    g = torch.Generator().manual_seed(seed)
    sizes, ctx, V = [9, 4, 0, 7], [20, 0, 3, 33], 40
    parents, cu = O.forest(sizes, seed)
    table, count = O.pages([c + 9 for c in ctx], 16, seed)
    T = sum(sizes)
    st = dict(parents=parents, cu=cu, ctx=torch.tensor(ctx, dtype=I32), table=table.clamp(min=0), qkv=torch.randn((T, 8 * 64), generator=g).bfloat16(), freq=0.5 ** torch.arange(32.0),
              k=torch.randn((count, 2, 16, 64), generator=g).bfloat16(), v=torch.randn((count, 2, 16, 64), generator=g).bfloat16(), head=torch.randn((256, V), generator=g) * 0.3,
              tokens=torch.randint(0, V, (T,), generator=g).to(I32), u=torch.rand(T, generator=g) * 0.1)
    return {k: x.cuda() for k, x in st.items()}


def test_a_step_of_all_operators(native_lib):
    """A row's logits are those of a program that decodes its path one token at a time, the accepted rows' keys and values end up behind the context, and the step captured in a graph and
    replayed on new inputs, two such graphs in turn, gives the same."""
    st = _program()
    k0, v0 = st["k"].clone(), st["v"].clone()
    y, logits, tokens, counts, rows, _ = _step(st)
    parents, cu = st["parents"].cpu(), st["cu"].cpu()
    for b in range(4):
        lo, c = int(cu[b]), int(st["ctx"][b])
        for j in range(int(cu[b + 1]) - lo):
            path = [i for i in range(j + 1) if O.sees(parents[lo : int(cu[b + 1])])[j, i]]
            kc, vc = k0.clone(), v0.clone()
            for i, r in enumerate(path):      # one token at a time
                place = c + i
                slot = st["table"][b, place // 16].long() * 16 + place % 16
                row = E.rope_kv_cache_write(st["qkv"][lo + r : lo + r + 1].clone(), torch.tensor([place], dtype=I32, device="cuda"), st["freq"], slot[None], kc, vc, 4, 2, 64)
            one = E.paged_decode(row, kc, vc, st["table"][b : b + 1], torch.tensor([c + len(path)], dtype=I32, device="cuda"), 4, 2, 64)
            # (both are within two bf16 roundings of the same numbers: weights and result, of values up to 4)
            assert (one[0].float() - y[lo + j].float()).abs().max() <= 4 * 2 * 2 * 2.0**-8
        n = int(counts[b])
        kept = rows[b, :n].tolist()
        kc, vc = k0.clone(), v0.clone()
        for i, r in enumerate(kept):
            place = c + i
            slot = st["table"][b, place // 16].long() * 16 + place % 16
            E.rope_kv_cache_write(st["qkv"][lo + r : lo + r + 1].clone(), torch.tensor([place], dtype=I32, device="cuda"), st["freq"], slot[None], kc, vc, 4, 2, 64)
            for x, want in ((st["k"], kc), (st["v"], vc)):
                assert torch.equal(x[st["table"][b, place // 16], :, place % 16], want[st["table"][b, place // 16], :, place % 16])
    # graphs
    progs = [_program(1), _program(2)]
    graphs, outs = [], []
    for p in progs:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(p)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(p))
        graphs.append(graph)
    for seed in (3, 4):
        fresh = [_program(seed), _program(seed + 10)]
        wants = [_step({k: x.clone() for k, x in f.items()}) for f in fresh]
        for p, f in zip(progs, fresh):
            for key in ("qkv", "k", "v", "tokens", "u", "head"):
                p[key].copy_(f[key])
            for key in ("parents", "table"):
                p[key].copy_(f[key]) if p[key].shape == f[key].shape else None
        wants = [_step({k: x.clone() for k, x in p.items()}) for p in progs]
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, wants):
            for x, y in zip(got, want):
                assert torch.equal(x, y)
    assert L.check_status() == 0


def test_streams(native_lib):
    """Calls on a side stream, two at once."""
    case = _attend_case([5, 18], [700, 3], 8, 2, 128, 16, seed=6)
    q, k, v, table, ctx, cu, parents = _dev(*case)
    masks = _masks(_bits(case[6], case[5]), 18).cuda()
    want = S.tree_paged_decode(q, k, v, table, ctx, cu, 8, 2, 128, max_rows=18, masks=masks)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(S.tree_paged_decode(q, k, v, table, ctx, cu, 8, 2, 128, max_rows=18, masks=masks))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got) and L.check_status() == 0


def test_verify_on_two_streams(native_lib):
    """Calls on side streams, two at once: the same results every time, whoever of a cluster is first."""
    cases = []
    for draft, dtype in ((False, torch.float32), (True, torch.bfloat16)):
        logits, guess, tokens, parents, cu, u = _verify_case([9, 1, 6, 0, 9] * 4, 30011, 5, 2, draft, dtype)
        cases.append((_dev(logits, tokens, parents, cu, u), dict(max_rows=9, draft_logits=guess.cuda() if draft else None)))
    want = [S.verify_drafts(*args, **more) for args, more in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, S.verify_drafts(*cases[i][0], **cases[i][1])))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for i, g in got for x, y in zip(g, want[i])) and L.check_status() == 0


def test_verify_of_logits_that_grow(native_lib):
    """Ranges whose later logits weigh far more than their first ones, up to what has no place beside them."""
    V = 40000
    for step in (0.01, 0.1, 30.0):
        z = torch.arange(V).float().flip(0).reshape(2, -1).flip(0).reshape(-1) * step      # (each half falls)
        z = torch.stack([z, z.flip(0), torch.arange(V).float() * step, torch.where(torch.arange(V) % 700 == 650, 600.0 + torch.arange(V) % 3, 0.0)])
        tokens, parents, cu = torch.zeros(4, dtype=I32), torch.full((4,), -1, dtype=I32), torch.arange(5, dtype=I32)
        for u in (0.0, 0.37, 0.99):
            want = S.verify_drafts(z, tokens, parents, cu, torch.full((4,), u), max_rows=1)
            got = S.verify_drafts(*_dev(z, tokens, parents, cu, torch.full((4,), u)), max_rows=1)
            assert torch.equal(got[0].cpu(), want[0])
            assert torch.allclose(got[3].cpu(), want[3], rtol=2.0**-23, atol=1e-12)


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 7, 1), (128, 40, 1)])
@pytest.mark.parametrize("ctas", [0, 1, 3, 40, 296])
def test_every_plan_is_the_same_attention(native_lib, D, Hq, Hkv, ctas):
    """A CTA for each unit, few and many CTAs that share the tiles, blocks one after another or beside one another, trees of fewer blocks than others, callers' own scratch."""
    sizes, ctx = [70, 3, 0, 40, 33, 1], [700, 1000, 9, 64, 0, 127]
    case = _attend_case(sizes, ctx, Hq, Hkv, D, 32, seed=8)
    q, k, v, table, ctx_t, cu, parents = case
    bits = _bits(parents, cu)
    want, tol = O.attend(q, k, v, table, ctx_t, cu, Hq, Hkv, D, bits)
    blocks = -(-70 // (128 // (Hq // Hkv)))
    for group in {1, blocks} if ctas else {1}:
        n = max(group, ctas - ctas % group)
        scratch = torch.full((S.tree_scratch_size(n, Hq, Hkv, D, 70) + 3,), math.nan, device="cuda") if ctas else None
        got = S.tree_paged_decode(*_dev(q, k, v, table, ctx_t, cu), Hq, Hkv, D, max_rows=70, masks=_masks(bits, 70).cuda(), plan=(n if ctas else 0, group), scratch=scratch)
        assert ((got.cpu().double() - want).abs() <= tol).all() and L.check_status() == 0


def test_attention_of_more_sequences_than_a_block_counts_at_once(native_lib):
    sizes, ctx = [1 + i % 3 if i % 7 else 0 for i in range(500)], [i % 90 for i in range(500)]
    case = _attend_case(sizes, ctx, 4, 2, 64, 16, seed=1)
    for plan in (None, (0, 1), (296, 1)):
        _check(case, 4, 2, 64, 3, _bits(case[6], case[5]), plan=plan)


def test_plans_that_are_refused(native_lib):
    q, k, v, table, ctx, cu, _ = _dev(*_attend_case([5, 18], [70, 3], 8, 2, 128, 16, seed=6))
    for plan in ((-1, 1), (70000, 1), (10, 2), (0, 2)):
        with pytest.raises(ValueError):
            S.tree_paged_decode(q, k, v, table, ctx, cu, 8, 2, 128, max_rows=18, plan=plan)
    for scratch in (torch.zeros(10, device="cuda"), torch.zeros(10**6, device="cuda", dtype=torch.bfloat16), torch.zeros(10**6), torch.zeros(10**6, device="cuda")[1:]):
        with pytest.raises(ValueError):
            S.tree_paged_decode(q, k, v, table, ctx, cu, 8, 2, 128, max_rows=18, plan=(8, 1), scratch=scratch)


def _poisoned(args, **kw):
    """A call whose results' memory held other numbers."""
    held = [torch.full((n,), 77, dtype=I32, device="cuda") for n in (len(args[3]) - 1, (len(args[3]) - 1) * kw["max_rows"]) for _ in range(4)]
    torch.cuda.synchronize()
    del held      # (their places are the next ones to be given out)
    return S.verify_drafts(*_dev(*args), **{k: x.cuda() if torch.is_tensor(x) else x for k, x in kw.items()})


def _as_on_the_cpu(args, **kw):
    want = S.verify_drafts(*args, **kw)
    for x, y in zip(_poisoned(args, **kw)[:3], want[:3]):
        assert torch.equal(x.cpu(), y)
    got = _poisoned(args, **kw)[3].cpu()
    assert torch.allclose(got, want[3], rtol=2.0**-23, atol=1e-12)
    assert L.check_status() == 0
    return want


def test_verify_behind_the_only_token_of_a_range(native_lib):
    """A turned-down token that is all, or nearly all, of what its range of the vocabulary weighs: the range has nothing left, or what is far below the sum's roundings."""
    V = 128256
    for low, high in ((0.0, 1.0), (0.3, -0.2), (-1.7, 2.9), (0.11, 0.13)):
        for third in (-math.inf, -35.0, -60.0, -300.0):
            z = torch.full((2, V), -math.inf)
            z[:, 5], z[:, 6], z[:, 2000] = low, third, high
            for u0 in (0.0, 0.3, 1 - 2.0**-24):
                want = _as_on_the_cpu((z, *(torch.tensor(x, dtype=I32) for x in ([0, 5], [-1, 0], [0, 2])), torch.tensor([u0, 0.999])), max_rows=2)
                assert int(want[0][0, 0]) == (6 if u0 == 0 and third > -math.inf else 2000)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,batch", [(9, 3), (1003, 40), (30011, 6), (4096, 400)])
def test_verify_of_masked_logits(native_lib, V, batch, dtype):
    for seed in range(3):
        logits, _, tokens, parents, cu, u = masked_case(V, [1 + (3 * b + seed) % 7 for b in range(batch)], seed, False, dtype)
        _as_on_the_cpu((logits, tokens, parents, cu, u), max_rows=7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,batch", [(9, 3), (1003, 40), (30011, 6), (4096, 400)])
def test_verify_of_masked_logits_of_both_models(native_lib, V, batch, dtype):
    for seed in range(3):
        logits, guess, tokens, parents, cu, u = masked_case(V, [1 + (3 * b + seed) % 7 for b in range(batch)], seed, True, dtype)
        _as_on_the_cpu((logits, tokens, parents, cu, u), max_rows=7, draft_logits=guess)


@pytest.mark.parametrize("hidden", [-math.inf, math.nan, O.FMAX * -1, -3e4])
def test_verify_of_one_allowed_token(native_lib, hidden):
    """One token is left in both models and a child is a hidden one: nothing is left behind it, and the last token comes from the target's own probabilities."""
    V = 4000
    z, d = torch.full((2, V), hidden), torch.full((2, V), hidden)
    z[:, 7], d[:, 7] = 0.3, 0.1
    for u0 in (0.0, 1e-30, 0.3, 0.999, 1 - 2.0**-24):
        want = _as_on_the_cpu((z, *(torch.tensor(x, dtype=I32) for x in ([0, 3], [-1, 0], [0, 2])), torch.tensor([u0, 0.5])), max_rows=2, draft_logits=d)
        assert want[0][0].tolist() == [7, -1] and want[1].tolist() == [1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-30, 1.0, 1e20, math.inf])
def test_greedy_takes_the_largest_logit_at_any_temperature(native_lib, temperature, dtype):
    """As on the CPU, where a large temperature makes logits alike and where some are not numbers or infinite."""
    logits, _, tokens, parents, cu, u = _verify_case([9, 1, 5, 7], 3001, 6, 2, False, dtype)
    logits[0, 70], logits[3, 5:9], logits[9, 2999] = math.nan, math.inf, math.inf
    _as_on_the_cpu((logits, tokens, parents, cu, u), max_rows=9, greedy=True, temperature=temperature)


@pytest.mark.parametrize("cu,T", [([0, 5, 2], 5), ([0, 5, 3, 8], 9), ([4, 2, 6], 7), ([0, 4, 1, 3, 6], 6), ([0, 9, 2], 5), ([0, 256, 1, 256] * 60 + [300], 310)])
def test_rows_that_several_sequences_name(native_lib, cu, T):
    """As on the CPU, every time."""
    g = torch.Generator().manual_seed(T)
    args = [(torch.rand(T, generator=g) * 3).to(I32) - 1, torch.tensor(cu, dtype=I32), torch.arange(len(cu) - 1, dtype=I32), torch.arange(30 * (len(cu) - 1), dtype=I32).reshape(-1, 30)]
    want = S.tree_rows(*args, 16, max_rows=256)
    dev = _dev(*args)
    for _ in range(20):
        for x, y in zip(S.tree_rows(*dev, 16, max_rows=256), want):
            assert torch.equal(x.cpu(), y)
    assert L.check_status() == 8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 0.7, 20.0])
def test_verify_where_both_models_agree(native_lib, temperature, dtype):
    """Tokens that are as probable in the draft as in the target have nothing left behind a rejection: of all tokens (the child is a hidden one: the last token is the target's own), and of all but
    one, which is the last token whatever the number is. Logits are whole numbers and differ by a constant, so that the probabilities are equal in exact arithmetic."""
    V, g = 4096, torch.Generator().manual_seed(3)
    for seed in range(12):
        few = torch.randperm(V, generator=g)[:6].sort().values
        z, d = torch.full((2, V), -math.inf), torch.full((2, V), -math.inf)
        z[:, few] = torch.randint(-3, 4, (6,), generator=g).float() if seed % 2 else 0.0
        d[:, few] = z[:, few] + 10.0 * seed + 1
        child = int((few[-1] + 1) % V)
        one = seed % 4 > 1 and seed % 2 == 0      # the draft has the hidden child in place of the last token
        if one:
            d[:, child], d[:, few[-1]] = d[0, few[-1]].item(), -math.inf
        for u0 in (0.0, 1e-9, 0.4, 1 - 2.0**-24):
            args = (z.to(dtype), torch.tensor([0, child], dtype=I32), torch.tensor([-1, 0], dtype=I32), torch.tensor([0, 2], dtype=I32), torch.tensor([u0, 0.5]))
            want = _as_on_the_cpu(args, max_rows=2, draft_logits=d.to(dtype), temperature=temperature)
            assert not one or want[0][0].tolist() == [int(few[-1]), -1]


def test_verify_of_what_is_nearly_nothing(native_lib):
    args, d = faint_case()
    assert int(_as_on_the_cpu(args, max_rows=4, draft_logits=d)[0][0, 0]) == 2000
