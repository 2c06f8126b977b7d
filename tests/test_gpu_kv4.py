"""Kernels of the 4-bit key/value cache. The write and the read-back give the bytes and values of the definition exactly; decode attention is held to
soft-max attention in 64 bits over the values that stand in the cache."""

import math

import pytest
import torch
from kv4_oracle import replayed

from rl_b200.ops import kv4_ops as K
from rl_b200.ops import lib as L

pytestmark = pytest.mark.gpu

HEADS = {64: [(14, 2), (16, 1), (8, 8)], 128: [(8, 2), (12, 2), (7, 1), (5, 5), (32, 2)], 256: [(8, 4), (10, 1)]}


def _freq(D, base=500000.0):
    return base ** (-torch.arange(0, D, 2).float() / D)


def _rows(T, Hq, Hkv, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, (Hq + 2 * Hkv) * D, generator=g) * (1 + 3 * (torch.arange((Hq + 2 * Hkv) * D) % 29 == 3))).bfloat16()


def _write_both(rows, pos, freq, slots, cache, Hq, Hkv, D):
    """On the CPU and on the GPU: (rows, cache) of each."""
    ref = cache.clone()
    want = K.rope_kv4_cache_write(rows, pos, freq, slots, ref, Hq, Hkv, D)
    dev, mine = rows.cuda(), cache.cuda()
    got = K.rope_kv4_cache_write(dev, pos.cuda(), freq.cuda(), slots.cuda(), mine, Hq, Hkv, D)
    assert got is dev
    torch.cuda.synchronize()
    return want, ref, got.cpu(), mine.cpu()


@pytest.mark.parametrize("T", [1, 2, 3, 67, 500, 2400])
@pytest.mark.parametrize("D,Hq,Hkv,block", [(64, 14, 2, 16), (64, 16, 1, 48), (128, 8, 2, 64), (128, 5, 5, 128), (256, 8, 1, 16)])
def test_write_is_exact(native_lib, T, D, Hq, Hkv, block):
    """Every rounding is the definition's: equal bytes."""
    pages = T // block + 3
    g = torch.Generator().manual_seed(T)
    pos = torch.randint(0, 200_000, (T,), generator=g)
    pos[0] = 2**31 - 1 if T == 2 else 0
    slots = torch.randperm(pages * block, generator=g)[:T]
    slots[T // 2 :: 9] = -1
    cache = torch.randint(0, 255, (pages, Hkv, K.kv4_page_bytes(block, D)), generator=g, dtype=torch.uint8)      # what is not written stays
    want, ref, got, mine = _write_both(_rows(T, Hq, Hkv, D, T), pos, _freq(D), slots, cache, Hq, Hkv, D)
    assert torch.equal(got, want) and torch.equal(mine, ref) and L.check_status() == 0
    back = K.kv4_cache_read(mine.cuda(), slots.cuda(), Hkv, D)
    assert torch.equal(back.cpu(), K.kv4_cache_read(ref, slots, Hkv, D))


@pytest.mark.parametrize("T,D,Hq,Hkv,block", [(2003, 64, 32, 4, 32), (1001, 128, 32, 8, 64), (1333, 128, 28, 4, 16), (701, 256, 20, 10, 16)])
def test_write_of_more_rows_than_the_device_holds_threads(native_lib, T, D, Hq, Hkv, block):
    """Blocks of several whole rows, the last one short."""
    test_write_is_exact(native_lib, T, D, Hq, Hkv, block)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_write_of_special_values(native_lib, D):
    T, Hq, Hkv, block = 12, 1, 1, 16
    x = torch.zeros(T, 3 * D)
    x[1] = -0.0
    x[2, D + 5], x[3, 2 * D + 40], x[4, 2 * D] = math.inf, math.nan, -math.inf
    x[5] = 2.0 ** -101
    x[6] = 2.0 ** -100
    x[7] = torch.finfo(torch.bfloat16).max * torch.linspace(-1, 1, 3 * D)
    x[8] = ((torch.arange(3 * D) % 32) - 16) * 0.125        # multiples of the scale: borders of codes
    x[9] = (15 - (torch.arange(3 * D) % 32)) * 0.125
    x[10] = 1e-39
    x[11] = ((torch.arange(3 * D) * 37 % 256) - 128) * 2.0 ** -80
    pos = torch.zeros(T, dtype=torch.int64)                  # no rotation: the values are what is held
    want, ref, got, mine = _write_both(x.bfloat16(), pos, _freq(D), torch.arange(T), K.kv4_cache(1, Hkv, block, D, "cpu"), Hq, Hkv, D)
    assert torch.equal(mine, ref)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())
    kv, kr = K.kv4_cache_read(mine.cuda(), torch.arange(T).cuda(), Hkv, D).cpu(), K.kv4_cache_read(ref, torch.arange(T), Hkv, D)
    assert torch.equal(kv.isnan(), kr.isnan()) and torch.equal(kv.nan_to_num(), kr.nan_to_num())


def test_write_and_read_of_odd_views(native_lib):
    """Rows that do not start on 16 bytes, wider buffers, 32-bit indices, an inner stride, rows of the output by number."""
    T, Hq, Hkv, D, block = 37, 4, 2, 64, 16
    rows, pos, freq, slots = _rows(T, Hq, Hkv, D), torch.arange(T), _freq(D), torch.randperm(64)[:T]
    ref = K.kv4_cache(4, Hkv, block, D, "cpu")
    want = K.rope_kv4_cache_write(rows, pos, freq, slots, ref, Hq, Hkv, D)
    W = rows.shape[1]
    wide = torch.zeros(T, W + 24, dtype=torch.bfloat16, device="cuda")
    for view in (wide[:, 8 : 8 + W], wide[:, 3 : 3 + W], torch.zeros(W, T, dtype=torch.bfloat16, device="cuda").t()):
        wide.fill_(5.0)
        view.copy_(rows)
        cache = K.kv4_cache(4, Hkv, block, D, "cuda")
        assert K.rope_kv4_cache_write(view, pos.int().cuda(), freq.cuda(), slots.int().cuda(), cache, Hq, Hkv, D) is view
        assert torch.equal(view.cpu(), want) and torch.equal(cache.cpu(), ref)
    assert (wide[:, -4:] == 5).all()
    kv = K.kv4_cache_read(ref, slots, Hkv, D)
    to = torch.randperm(T)
    for off, extra in ((0, 0), (8, 16), (1, 7)):
        out = torch.full((T + 2, off + kv.shape[1] + extra), 3.0, dtype=torch.bfloat16, device="cuda")
        got = K.kv4_cache_read(cache, slots.cuda(), Hkv, D, out=out[:, off:], rows=to.cuda())
        assert got.data_ptr() == out[:, off:].data_ptr() and torch.equal(got[to.cuda(), : kv.shape[1]].cpu(), kv)
        assert (out[T:] == 3).all() and (out[:, :off] == 3).all() and (out[:, off + kv.shape[1] :] == 3).all()
    assert L.check_status() == 0


def test_rows_that_overlap_are_refused_before_anything_is_written(native_lib):
    """Rows that share places by any strides; the cache and the rows stay as they were. Views whose rows interleave without sharing a place are served."""
    T, Hq, Hkv, D, block = 4, 2, 1, 64, 16
    W, Wkv = 4 * D, 2 * D
    pos, freq, slots = torch.arange(T).cuda(), _freq(D).cuda(), torch.arange(T).cuda()
    held = torch.randint(0, 255, (2, Hkv, K.kv4_page_bytes(block, D)), dtype=torch.uint8).cuda()
    held[..., block * D :].view(torch.bfloat16).fill_(0.5)
    mem = _rows(1, Hq, Hkv, 16 * D).cuda().flatten()
    q, table, n = _rows(T, Hq, Hkv, D).cuda(), torch.zeros((T, 1), dtype=torch.int32, device="cuda"), torch.full((T,), 9, dtype=torch.int32, device="cuda")
    for strides in ((0, 1), (8, 1), (1, 1), (W - 8, 1), (W, 2), (3, 2), (W, 0)):
        cache, was = held.clone(), mem.clone()
        with pytest.raises(RuntimeError):
            K.rope_kv4_cache_write(mem.as_strided((T, W), strides), pos, freq, slots, cache, Hq, Hkv, D)
        assert torch.equal(cache, held) and torch.equal(mem, was)
    for strides in ((0, 1), (8, 1), (Wkv - 4, 1), (Wkv, 2), (Wkv, 0)):
        for call in (lambda out: K.kv4_cache_read(held, slots, Hkv, D, out=out), lambda out: K.kv4_paged_decode(q, held, table, n, Hq, Hkv, D, out=out)):
            was = mem.clone()
            with pytest.raises(RuntimeError):
                call(mem.as_strided((T, Wkv), strides))
            assert torch.equal(mem, was)
    ref = K.kv4_cache(2, Hkv, block, D, "cuda")
    want = K.rope_kv4_cache_write(q.clone(), pos, freq, slots, ref, Hq, Hkv, D)
    for strides in ((1, T), (3 * W - 1, 3), (1, 2 * T + 1)):
        view, cache = torch.zeros(4 * T * W, dtype=torch.bfloat16, device="cuda").as_strided((T, W), strides), torch.zeros_like(ref)
        view.copy_(q)
        assert K.rope_kv4_cache_write(view, pos, freq, slots, cache, Hq, Hkv, D) is view and torch.equal(view, want) and torch.equal(cache, ref)
    one = mem.as_strided((1, W), (0, 1))      # one row overlaps with none
    assert K.rope_kv4_cache_write(one, pos[:1], freq, slots[:1], cache, Hq, Hkv, D) is one
    assert L.check_status() == 0


def test_bad_slots_are_reported_and_skipped(native_lib):
    T, Hq, Hkv, D, block = 3, 2, 1, 128, 16
    rows, slots = _rows(T, Hq, Hkv, D), torch.tensor([32, 5, 10**12])
    cache, ref = K.kv4_cache(2, Hkv, block, D, "cuda"), K.kv4_cache(2, Hkv, block, D, "cpu")
    K.rope_kv4_cache_write(rows.cuda(), torch.arange(T).cuda(), _freq(D).cuda(), slots.cuda(), cache, Hq, Hkv, D)
    assert L.check_status() == 6
    K.rope_kv4_cache_write(rows, torch.arange(T), _freq(D), torch.tensor([-1, 5, -1]), ref, Hq, Hkv, D)
    assert torch.equal(cache.cpu(), ref)
    out = torch.full((2, 256), 9.0, dtype=torch.bfloat16, device="cuda")
    K.kv4_cache_read(cache, torch.tensor([32, 5], device="cuda"), Hkv, D, out=out)
    assert L.check_status() == 6 and (out[0] == 9).all() and torch.equal(out[1:].cpu(), K.kv4_cache_read(ref, torch.tensor([5]), Hkv, D))
    K.kv4_cache_read(cache, torch.tensor([5], device="cuda"), Hkv, D, out=out, rows=torch.tensor([2], device="cuda"))
    assert L.check_status() == 6
    assert not K.kv4_cache_read(cache, torch.tensor([-1], device="cuda"), Hkv, D).any() and L.check_status() == 0


# ------------------------------------------------------------------------------------------- decode
def _pool(pages, Hkv, D, block, seed, big=1.0):
    """A cache of normal values, and a garbage value in every byte that no token owns is made by the tests themselves."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(2, pages, Hkv, block, D, generator=g, device="cuda") * big
    x[..., 3::29] *= 4
    (kc, ks), (vc, vs) = (K.quantize_ref(t.bfloat16()) for t in x)
    return K._pack_pages(kc, vc, ks, vs)


def _check(got, q, cache, table, lens, Hq, Hkv, D, window=0, scale=None):
    """Every output within what the roundings give: the result's to bf16 (2^-8 of it), each token's weight times its scale to bf16 (2^-8 of
    the token's share), and the scores' to 32 bits. A score's sum over a group has 32 terms of at most 15 |q| and the offset of 7.5 times the sum of the query's values: 33
    roundings at that size, times the key's scale; a score's error e changes a weight by e and the sum by as much."""
    block, B = cache.shape[2] * 8 // (9 * D), got.shape[0]
    scale = scale or 1 / math.sqrt(D)
    for b in range(B):
        n = int(lens[b])
        lo = max(0, n - window) if window else 0
        if n == 0:
            assert not got[b].any()
            continue
        kc, vc, ks, vs = K._unpack_pages(cache[table[b, : -(-n // block)].long()].transpose(0, 1), D)
        k, v = (((c.double() - 7.5) * s.double().unsqueeze(-1)).flatten(-2).flatten(1, 2)[:, lo:n] for c, s in ((kc, ks), (vc, vs)))
        qb = q[b, : Hq * D].double().reshape(Hkv, Hq // Hkv, D)
        p = torch.softmax(qb @ k.transpose(1, 2) * scale, -1)
        want, share = p @ v, p @ v.abs()
        e = abs(scale) * 33 * 2.0 ** -24 * 15 * torch.einsum("hgd,hd->hg", qb.abs(), ks.double().repeat_interleave(32, -1).flatten(1, 2)[:, lo:n].amax(1)).unsqueeze(-1)
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * e + 2.0 ** -18) * share
        off = (got[b].double().reshape(want.shape) - want).abs()
        assert (off <= tol).all(), f"row {b}: {(off / tol).max().item():.2f} times the tolerance"


def _decode_case(lens, Hq, Hkv, D, block, seed=0, spare=2, big=1.0):
    need = [-(-n // block) for n in lens]
    g = torch.Generator().manual_seed(seed)
    pages = sum(need) + spare
    cache = _pool(pages, Hkv, D, block, seed, big)
    order, at = torch.randperm(pages, generator=g).int(), 0
    table = torch.full((len(lens), max(1, max(need)) + 1), 10**9, dtype=torch.int32)      # entries behind a sequence's pages are never read
    for i, k in enumerate(need):
        table[i, :k] = order[at : at + k]
        at += k
    q = _rows(len(lens), Hq, Hkv, D, seed).cuda()
    return q, cache, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


LENGTHS = [[1], [0], [2, 15, 16, 17, 0, 31, 33], [63, 64, 65, 1, 127, 128, 129], [300, 0, 1025], [4100]]


@pytest.mark.parametrize("lens", LENGTHS, ids=lambda l: "-".join(map(str, l)))
@pytest.mark.parametrize("D,Hq,Hkv", [(D, *h) for D in HEADS for h in HEADS[D]])
def test_decode(native_lib, lens, D, Hq, Hkv):
    for block in (16, 64) if D != 128 else (48, 128):
        q, cache, table, n = _decode_case(lens, Hq, Hkv, D, block, seed=len(lens))
        for plan in (None, (1, 0), (3, 0), (8, 0), (1, 1), (1, 5), (1, 37)):
            got = K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=plan)
            assert L.check_status() == 0
            _check(got, q, cache, table, n, Hq, Hkv, D)
            assert torch.equal(got, K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=plan))      # the same bits again


@pytest.mark.parametrize("window", [1, 5, 16, 100, 5000])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 14, 2), (128, 8, 2), (256, 8, 4)])
def test_decode_window(native_lib, window, D, Hq, Hkv):
    q, cache, table, n = _decode_case([1, 17, 100, 0, 1000, 333, 16], Hq, Hkv, D, 32, seed=window)
    for plan in (None, (1, 0), (2, 0), (7, 0), (1, 3), (1, 40)):
        _check(K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, window=window, plan=plan), q, cache, table, n, Hq, Hkv, D, window)
    assert L.check_status() == 0


@pytest.mark.parametrize("big,scale", [(1e-20, 0.1), (1e-3, 30.0), (40.0, None), (1e15, 1e-17)])
def test_decode_of_small_large_and_peaked(native_lib, big, scale):
    """Values far from one, and scores of hundreds: one token takes nearly all."""
    q, cache, table, n = _decode_case([700, 33, 260], 8, 2, 128, 64, seed=5, big=big)
    for plan in ((1, 0), (4, 0), (1, 7)):
        _check(K.kv4_paged_decode(q, cache, table, n, 8, 2, 128, scale=scale, plan=plan), q, cache, table, n, 8, 2, 128, scale=scale)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-38])
def test_decode_scales(native_lib, scale):
    """A negative scale, and scales that leave every token the same weight."""
    for Hq in (4, 10):
        q, cache, table, n = _decode_case([700, 33, 1], Hq, 2, 64, 16, seed=6)
        for plan in ((1, 0), (4, 0), (1, 7)):
            got = K.kv4_paged_decode(q, cache, table, n, Hq, 2, 64, scale=scale, plan=plan)
            _check(got, q, cache, table, n, Hq, 2, 64, scale=scale or 1e-300)
    with pytest.raises(ValueError):
        K.kv4_paged_decode(q, cache, table, n, 10, 2, 64, scale=math.nan)


@pytest.mark.parametrize("q_by,big,scale", [(2.0 ** -120, 2.0 ** 118, 0.1), (2.0 ** 104, 2.0 ** -88, 2.0 ** -16), (1.0, 2.0 ** 118, 0.0), (2.0 ** -125, 1.0, None)])
def test_decode_of_scores_from_far_apart_factors(native_lib, q_by, big, scale):
    """Queries, keys and scales at the ends of their type whose products are ordinary scores, or none at all."""
    for Hq in (4, 10):
        q, cache, table, n = _decode_case([700, 33, 1], Hq, 2, 64, 16, seed=7, big=big)
        q = (q.double() * q_by).bfloat16()
        for plan in ((1, 0), (4, 0), (1, 7)):
            got = K.kv4_paged_decode(q, cache, table, n, Hq, 2, 64, scale=scale, plan=plan)
            _check(got, q, cache, table, n, Hq, 2, 64, scale=1e-300 if scale == 0 else scale)


def _with_value_scales(cache, table, lens, D, power):
    """The cache with the values' scales of each sequence's token t times 2^power(t) ([tokens] or [tokens, groups])."""
    kc, vc, ks, vs = K._unpack_pages(cache, D)
    block, s = kc.shape[2], vs.double()
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        s[table[b, t // block].long(), :, t % block] *= 2.0 ** power(t).double().reshape(n, 1, -1)
    assert (s.abs() < 2.0 ** 124).all() and (s[s > 0] > 2.0 ** -100).all()
    return K._pack_pages(kc, vc, ks, s.to(torch.bfloat16))


@pytest.mark.parametrize("low,high", [(-60, 75), (-94, 118), (0, 100)])
@pytest.mark.parametrize("D,Hq", [(64, 4), (64, 10), (128, 4), (128, 10), (256, 2), (256, 16)])
def test_decode_of_values_from_far_apart_scales(native_lib, D, Hq, low, high):
    """Tokens of tiny values keep their weight beside tokens of huge ones: within a warp, between warps, clusters' CTAs and shared parts. Queries of zeros
    give every token the same weight, so that each that is left out of the denominator shows."""
    lens = [700, 33, 300]
    q, cache, table, n = _decode_case(lens, Hq, 2, D, 16, seed=11)
    orders = [lambda t, cut=cut: t >= cut for cut in (16, 32, 128, 350)]
    orders += [lambda t: t < 350, lambda t: t // 32 % 2 == 1, lambda t: t == 290]
    for order in orders:
        c = _with_value_scales(cache, table, lens, D, lambda t: torch.where(order(t), high, low))
        for x in (q, torch.zeros_like(q)):
            for plan in ((1, 0), (4, 0), (1, 7), (1, 1)):
                _check(K.kv4_paged_decode(x, c, table, n, Hq, 2, D, plan=plan), x, c, table, n, Hq, 2, D)
    assert L.check_status() == 0


@pytest.mark.parametrize("D,Hq", [(64, 4), (64, 10), (128, 4), (128, 10), (256, 2), (256, 16)])
def test_decode_of_groups_far_below_the_largest(native_lib, D, Hq):
    """A group of dimensions whose scales lie 2^-80 times the head's largest and above keeps its bits; sequences of one token to some steps a warp, also of tiny values."""
    lens, G = [700, 33, 1, 300], D // 32
    q, cache, table, n = _decode_case(lens, Hq, 2, D, 16, seed=12)
    for powers in ([0, -79], [-40, 0], [118, 40], [-15, -94], [-94, -90], [0, -60, -79, -20]):
        power = torch.tensor((powers * G)[:G], device="cuda")
        c = _with_value_scales(cache, table, lens, D, lambda t: power.expand(len(t), G))
        for x in (q, torch.zeros_like(q)):
            for plan in ((1, 0), (4, 0), (1, 7)):
                _check(K.kv4_paged_decode(x, c, table, n, Hq, 2, D, plan=plan), x, c, table, n, Hq, 2, D)
    assert L.check_status() == 0


@pytest.mark.parametrize("Hq", [4, 16])
def test_a_query_that_is_not_finite_spoils_its_head_alone(native_lib, Hq):
    q, cache, table, n = _decode_case([50, 300], Hq, 2, 128, 16, seed=2)
    for plan in ((1, 0), (3, 0), (1, 5)):
        clean = K.kv4_paged_decode(q, cache, table, n, Hq, 2, 128, plan=plan).view(2, Hq, 128)
        for bad in (math.nan, math.inf):
            x = q.clone()
            x[1, 128 + 77] = bad
            got = K.kv4_paged_decode(x, cache, table, n, Hq, 2, 128, plan=plan).view(2, Hq, 128)
            assert got[1, 1].isnan().all()
            got[1, 1] = clean[1, 1]
            assert torch.equal(got, clean)


@pytest.mark.parametrize("plan", [(1, 0), (5, 0), (1, 2), (1, 33)])
def test_decode_ignores_what_stands_behind_the_end(native_lib, plan):
    """NaN and infinite scales, and any codes, in places that the sequence does not see: before the window and behind its last token."""
    Hq, Hkv, D, block, lens, window = 8, 2, 128, 64, [70, 129, 1, 64, 300], 50
    q, cache, table, n = _decode_case(lens, Hq, Hkv, D, block, seed=3)
    dirty = cache.clone()
    for b, m in enumerate(lens):
        for t in list(range(m, -(-m // block) * block)) + list(range(0, max(0, m - window))):
            page, off = dirty[int(table[b, t // block])], t % block
            s = page[:, block * D :].view(torch.bfloat16).view(Hkv, block, 8)
            s[:, off] = torch.tensor([math.nan, math.inf, -math.inf, 3e38] * 2, device="cuda").bfloat16()
            page[:, : block * D // 2].view(Hkv, block, -1)[:, off] = 0xA5
    want = K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, window=window, plan=plan)
    got = K.kv4_paged_decode(q, dirty, table, n, Hq, Hkv, D, window=window, plan=plan)
    assert got.isfinite().all() and torch.equal(got, want)


def test_decode_hands_on_what_is_not_finite(native_lib):
    """A visible key with a NaN scale makes its heads NaN, a value's its group; other heads and sequences keep their numbers."""
    Hq, Hkv, D, block = 4, 2, 128, 16
    q, cache, table, n = _decode_case([40, 40], Hq, Hkv, D, block, seed=9)
    for plan in ((1, 0), (2, 0), (1, 3)):
        clean = K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=plan)
        for value, group in ((0, 2), (1, 1)):
            c = cache.clone()
            c[int(table[1, 1]), 1, block * D :].view(torch.bfloat16).view(block, 2, 4)[3, value, group] = math.nan
            got = K.kv4_paged_decode(q, c, table, n, Hq, Hkv, D, plan=plan).view(2, Hq, D)
            nan = torch.zeros(2, Hq, D, dtype=torch.bool, device="cuda")
            nan[1, 2:, slice(None) if value == 0 else slice(32, 64)] = True
            assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], clean.view(2, Hq, D)[~nan])


def test_decode_of_odd_views(native_lib):
    Hq, Hkv, D, block = 4, 2, 64, 16
    q, cache, table, n = _decode_case([50, 3, 0, 77], Hq, Hkv, D, block)
    want = K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D)
    _check(want, q, cache, table, n, Hq, Hkv, D)
    odd = torch.zeros(4, Hq * D + 5, dtype=torch.bfloat16, device="cuda")[:, 3 : 3 + Hq * D]
    odd.copy_(q[:, : Hq * D])
    wide = torch.full((4, 2 * Hq * D), 7.0, dtype=torch.bfloat16, device="cuda")
    for out in (wide[:, 4 : 4 + Hq * D], wide[:, 1 : 1 + Hq * D], wide[:, ::2]):
        wide.fill_(7.0)
        got = K.kv4_paged_decode(odd, cache, table.t().contiguous().t(), torch.stack([n, n], 1)[:, 0], Hq, Hkv, D, out=out)
        assert got is out and torch.equal(out, want) and int((wide == 7).sum()) >= 4 * Hq * D
    assert K.kv4_paged_decode(q[:0], cache, table[:0], n[:0], Hq, Hkv, D).shape == (0, Hq * D)
    scratch = torch.empty(K.kv4_scratch_size(3, D) + 4, device="cuda")
    _check(K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=(1, 3), scratch=scratch), q, cache, table, n, Hq, Hkv, D)
    for bad in (scratch[:-5], scratch.double(), scratch.cpu(), scratch[1:], scratch[::2]):
        with pytest.raises(ValueError):
            K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=(1, 3), scratch=bad)
    for bad in ((0, 0), (9, 0), (2, 5), (1, -1)):
        with pytest.raises(ValueError):
            K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=bad)
    for bad in (q.float(), q.half(), q.cpu(), q.clone().requires_grad_()):
        with pytest.raises(ValueError):
            K.kv4_paged_decode(bad, cache, table, n, Hq, Hkv, D)
    with pytest.raises(RuntimeError):      # rows that overlap
        K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, out=torch.zeros(1, Hq * D, dtype=torch.bfloat16, device="cuda").expand(4, -1))
    with pytest.raises(RuntimeError):
        K.rope_kv4_cache_write(q[:1].expand(4, -1), n, _freq(D).cuda(), torch.arange(4, device="cuda"), cache.clone(), Hq, Hkv, D)
    with pytest.raises(RuntimeError):
        K.kv4_cache_read(cache, n, Hkv, D, out=torch.zeros(1, 2 * Hkv * D, dtype=torch.bfloat16, device="cuda").expand(4, -1))
    with pytest.raises(ValueError):
        K.rope_kv4_cache_write(q.float(), n, _freq(D).cuda(), n, cache, Hq, Hkv, D)
    with pytest.raises(ValueError):
        K.kv4_cache_read(cache, n, Hkv, D, out=torch.zeros(4, 2 * Hkv * D, device="cuda"))


def test_bad_pages_and_lengths_are_reported(native_lib):
    """Page numbers outside the cache are left out, lengths beyond the table end there: an error is on record and nothing else is read."""
    Hq, Hkv, D, block = 8, 2, 128, 16
    q, cache, table, n = _decode_case([64, 64], Hq, Hkv, D, block)
    for plan in ((1, 0), (2, 0), (1, 3)):
        want = K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=plan)
        for page in (-1, cache.shape[0], 2**31 - 1):
            bad = table.clone()
            bad[1, 2] = page
            got = K.kv4_paged_decode(q, cache, bad, n, Hq, Hkv, D, plan=plan)
            assert L.check_status() == 6 and torch.equal(got[0], want[0]) and got.isfinite().all()
        got = K.kv4_paged_decode(q, cache, table[:, :4], torch.tensor([64, 2**31 - 1], dtype=torch.int32, device="cuda"), Hq, Hkv, D, plan=plan)
        assert L.check_status() == 6 and torch.equal(got, want)
        got = K.kv4_paged_decode(q, cache, table, torch.tensor([64, -5], dtype=torch.int32, device="cuda"), Hq, Hkv, D, plan=plan)
        assert L.check_status() == 0 and not got[1].any()
        _check(got[:1], q, cache, table, n, Hq, Hkv, D)


@pytest.mark.parametrize("plan", [None, (1, 0), (2, 0), (1, 444)])
def test_decode_of_more_rows_than_a_grid_has_in_one_direction(native_lib, plan):
    """70001 sequences: the rows of the same call in two halves."""
    B, Hq, Hkv, D, block = 70001, 2, 1, 64, 16
    cache = _pool(40, Hkv, D, block, 4)
    g = torch.Generator().manual_seed(1)
    n = torch.randint(0, 100, (B,), generator=g).int().cuda()
    table = torch.randint(0, 40, (B, 7), generator=g).int().cuda()
    q = torch.randn(B, Hq * D, generator=g).bfloat16().cuda()
    got = K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=plan)
    half = B // 2
    want = torch.cat([K.kv4_paged_decode(q[r], cache, table[r], n[r], Hq, Hkv, D, plan=plan or (1, 0)) for r in (slice(0, half), slice(half, B))])
    if plan and plan[1]:      # other shares, so other parts: on both sides half a step of the result and half a step of each token's share, neither above the largest value
        for r in (slice(0, 50), slice(B - 50, B)):
            _check(got[r], q[r], cache, table[r], n[r], Hq, Hkv, D)
        largest = K._unpack_pages(cache, D)[3].float().max() * 7.5
        assert ((got.float() - want.float()).abs() <= 4.1 * 2.0 ** -8 * largest).all()
    else:
        assert torch.equal(got, want)
    assert L.check_status() == 0


def test_decode_window_over_a_very_wide_table(native_lib):
    """A table with room for 2^31 tokens a sequence, of which a window is visible: planned and shared by the window. What no plan can share is refused by name."""
    B, Hq, Hkv, D, block, window = 8, 8, 8, 64, 65536, 16384
    cache = _pool(9, Hkv, D, block, 5)
    table = torch.zeros((B, 32767), dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(8)
    n = torch.tensor([20000, 16384, 16385, 1, 0, 65000, 30000, 16500], dtype=torch.int32, device="cuda")
    q = _rows(B, Hq, Hkv, D).cuda()
    assert K.kv4_plan(B, Hq, Hkv, D, window)[1] > 0
    for plan in (None, (1, 100), (4, 0)):
        _check(K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, window=window, plan=plan), q, cache, table, n, Hq, Hkv, D, window)
    _check(K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D), q, cache, table, n, Hq, Hkv, D)
    assert L.check_status() == 0
    with pytest.raises(ValueError):
        K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, plan=(1, 444))
    with pytest.raises(ValueError):
        K.kv4_paged_decode(q, cache, torch.zeros((B, 32768), dtype=torch.int32, device="cuda"), n, Hq, Hkv, D)


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 + 7, 2**32, 2**32 + 5, 2**40 + 1])
def test_decode_of_windows_beyond_32_bits(native_lib, window):
    """A window wider than any sequence leaves everything."""
    q, cache, table, n = _decode_case([1, 17, 100, 0, 1000, 333, 16], 4, 2, 64, 32, seed=3)
    for plan in ((1, 0), (2, 0), (1, 3)):
        assert torch.equal(K.kv4_paged_decode(q, cache, table, n, 4, 2, 64, window=window, plan=plan), K.kv4_paged_decode(q, cache, table, n, 4, 2, 64, plan=plan))
    assert L.check_status() == 0


def test_places_beyond_32_bits(native_lib):
    """A cache of more than 4 GiB: pages at its far end."""
    Hq, Hkv, D, block = 8, 8, 128, 128
    size = K.kv4_page_bytes(block, D) * Hkv
    pages = 2**32 // size + 40
    if torch.cuda.mem_get_info()[0] < 2 * pages * size:
        pytest.skip("no room")
    cache = K.kv4_cache(pages, Hkv, block, D, "cuda")
    small = K.kv4_cache(4, Hkv, block, D, "cuda")
    T = 300
    rows, pos, freq = _rows(T, Hq, Hkv, D), torch.arange(T).cuda(), _freq(D).cuda()
    at = torch.arange(T).cuda()
    far = torch.tensor([pages - 1, pages - 7, pages - 3], device="cuda")
    for c, page in ((cache, far), (small, torch.tensor([3, 0, 1], device="cuda"))):
        K.rope_kv4_cache_write(rows.cuda(), pos, freq, page[at // block] * block + at % block, c, Hq, Hkv, D)
    n = torch.tensor([T], dtype=torch.int32, device="cuda")
    for i, j in zip(far.tolist(), (3, 0, 1)):
        assert torch.equal(cache[i], small[j])
    got = K.kv4_paged_decode(rows[:1].cuda(), cache, far[None].int(), n, Hq, Hkv, D)
    assert torch.equal(got, K.kv4_paged_decode(rows[:1].cuda(), small, torch.tensor([[3, 0, 1]], device="cuda").int(), n, Hq, Hkv, D))
    s = far[at // block] * block + at % block
    assert torch.equal(K.kv4_cache_read(cache, s, Hkv, D), K.kv4_cache_read(small, torch.tensor([3, 0, 1], device="cuda")[at // block] * block + at % block, Hkv, D))
    assert L.check_status() == 0


def test_graphs_and_streams(native_lib):
    """A decode step (write, then attention) captured twice, replayed in turn on changing inputs, next to eager calls on another stream."""
    Hq, Hkv, D, block, B = 8, 2, 128, 16, 5
    q, cache, table, n = _decode_case([30, 200, 1, 64, 17], Hq, Hkv, D, block, spare=8)
    table = table.clamp(max=cache.shape[0] - 1)
    freq = _freq(D).cuda()
    state = dict(rows=q.clone(), pos=n.long() - 1, lens=n.clone())

    def step(c, plan):
        slots = table[torch.arange(B, device="cuda"), state["pos"] // block].long() * block + state["pos"] % block
        rows = K.rope_kv4_cache_write(state["rows"].clone(), state["pos"], freq, slots, c, Hq, Hkv, D)
        return K.kv4_paged_decode(rows, c, table, state["lens"], Hq, Hkv, D, plan=plan)

    caches = [cache.clone() for _ in range(3)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in ((1, 0), (1, 40), (4, 0)):
            step(cache.clone(), s)
    torch.cuda.current_stream().wait_stream(side)
    for c, s in zip(caches, ((1, 0), (1, 40), (4, 0))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c, s))
        graphs.append(g)
    for c in caches:
        c.copy_(cache)
    eager = cache.clone()
    for i in range(3):
        state["rows"].copy_(_rows(B, Hq, Hkv, D, 50 + i))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        with torch.cuda.stream(side):
            want = step(eager, (1, 0))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and all(torch.equal(c, eager) for c in caches)
        for got in outs[1:]:
            _check(got, K.rope_kv4_cache_write(state["rows"].clone(), state["pos"], freq, torch.full((B,), -1, device="cuda"), eager, Hq, Hkv, D), eager, table, n, Hq, Hkv, D)
    assert L.check_status() == 0


# ------------------------------------------------------------------------------------------- the engine
def _model(**kw):
    from rl_b200.models.config import ModelConfig
    from rl_b200.models.transformer import CausalLM

    mc = ModelConfig(**{**dict(model_type="llama", vocab_size=4096, hidden_size=512, intermediate_size=1408, num_hidden_layers=2, num_attention_heads=8,
                               num_key_value_heads=2, head_dim=128, rope_theta=500000.0), **kw})
    return CausalLM(mc, dtype=torch.bfloat16, device="cuda", seed=3)


def _engine(model, **kw):
    from rl_b200.engine.engine import GenerationEngine

    return GenerationEngine(model, **{**dict(block_size=16, num_blocks=600, max_running=16, max_model_len=1024, kv_cache_dtype="int4"), **kw})


@pytest.mark.parametrize("kw", [dict(), dict(head_dim=64, num_key_value_heads=4), dict(num_attention_heads=7, num_key_value_heads=1, qk_norm=True), dict(head_dim=256, num_attention_heads=4)],
                         ids=["128", "64", "7-heads", "256"])
def test_engine_on_the_4_bit_cache(native_lib, kw):
    """Decoding by graphs and without, prompts in portions and after cached prefixes, against the layers in plain PyTorch over what the cache holds. The bound is that
    of the bf16 engine against the trainer's pass."""
    from rl_b200.engine.engine import SamplingParams

    model = _model(**kw)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(1, 4096, (n,), generator=g).tolist() for n in (40, 3, 100, 17, 64)]
    prompts += [prompts[0], prompts[2]]
    sp = SamplingParams(max_new_tokens=24, stop_token_ids=[], seed=3, temperature=1.0)
    results = []
    for opts in (dict(use_cuda_graphs=True), dict(use_cuda_graphs=False), dict(max_prefill_tokens=48)):
        eng = _engine(model, **opts)
        seen = {}
        rounds = eng._prefill_round
        eng._prefill_round = lambda items, *a, **k: ([seen.setdefault(tuple(q), []).append(p + n) for _, q, p, n in items], rounds(items, *a, **k))[1]
        recs = eng.generate(prompts, sp)
        assert L.check_status() == 0
        results.append([r.out_tokens for r in recs])
        gaps = []
        for r in recs:
            want = replayed(model, r, sorted(set(seen.get(tuple(r.prompt), [len(r.prompt)]))), 1.0).cpu()
            gaps.append((want - torch.tensor(r.out_logprobs)).abs())
        gaps = torch.cat(gaps)
        assert gaps.mean() < 0.03 and gaps.max() < 0.5, (opts, gaps.mean(), gaps.max())
    assert results[0] == results[1]
    # a later prompt that begins with cached pages
    eng = _engine(model)
    eng.generate([prompts[2]], SamplingParams(max_new_tokens=2, stop_token_ids=[], seed=3))
    eng.generate([prompts[2] + prompts[3]], SamplingParams(max_new_tokens=4, stop_token_ids=[], seed=3))
    assert eng.stats["cached_prefix_tokens"] >= 96 and L.check_status() == 0


def test_engine_sliding_windows(native_lib):
    from rl_b200.engine.engine import SamplingParams
    from rl_b200.models.config import preset
    from rl_b200.models.transformer import CausalLM

    mc = preset("gemma3-1b", vocab_size=2048, hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=256,
                sliding_window=32, embed_scale=1.0, layer_types=["sliding_attention", "full_attention", "sliding_attention"])
    model = CausalLM(mc, dtype=torch.bfloat16, device="cuda", seed=1)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(1, 2048, (n,), generator=g).tolist() for n in (70, 5, 33)]
    eng = _engine(model)
    recs = eng.generate(prompts, SamplingParams(max_new_tokens=40, stop_token_ids=[], seed=3, temperature=1.0))
    assert L.check_status() == 0
    gaps = torch.cat([(replayed(model, r, [len(r.prompt)], 1.0).cpu() - torch.tensor(r.out_logprobs)).abs() for r in recs])
    assert gaps.mean() < 0.03 and gaps.max() < 0.5, (gaps.mean(), gaps.max())


def test_generation_by_configuration(native_lib):
    """``generation.kv_cache_dtype: int4`` through the policy worker: half and more of the cache's memory is saved, the rollout stays near the policy."""
    from rl_b200.distributed.batched_data_dict import BatchedDataDict
    from rl_b200.models.config import ModelConfig
    from rl_b200.policy.worker import PolicyWorker

    mc = ModelConfig(model_type="llama", vocab_size=4096, hidden_size=512, intermediate_size=1408, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                     head_dim=128, rope_theta=500000.0)
    g = dict(max_new_tokens=24, stop_token_ids=[], kv_cache_tokens=8192, block_size=64, max_running=32, vllm_cfg=dict(kv_cache_dtype="int4"))
    p = PolicyWorker(dict(precision="bfloat16", train_global_batch_size=8, train_micro_batch_size=4, max_total_sequence_length=256,
                          optimizer=dict(name="torch.optim.AdamW", kwargs=dict(lr=1e-4)), generation=g), model_cfg=mc, device="cuda:0", init_reference_model=False, seed=3)
    gen = p.build_generation()
    assert gen.engine.kv4
    gen.prepare_for_generation()
    ids = torch.randint(1, 4095, (8, 40), generator=torch.Generator().manual_seed(0))
    out = gen.generate(BatchedDataDict(input_ids=ids, input_lengths=torch.full((8,), 40)))
    lp = p.get_logprobs(BatchedDataDict(input_ids=out["output_ids"], input_lengths=out["unpadded_sequence_lengths"]))["logprobs"]
    err = (lp - out["logprobs"]).abs()[out["logprobs"] != 0]
    assert L.check_status() == 0 and (out["generation_lengths"] == 24).all()
    assert 0 < err.mean().item() < 0.3 and err.max().item() < 2.0      # the bounds of the other quantised rollouts
    assert gen.engine.kv_cache_bytes() * 32 == 2 * 2 * gen.engine.num_blocks * 2 * 64 * 128 * 2 * 9


@pytest.mark.parametrize("kind", ["hybrid", "experts"])
def test_engine_of_hybrid_and_expert_models(native_lib, kind):
    """Attention blocks between others, and expert layers: by graphs and without the same tokens, near the log-probabilities of the model's own pass (the bounds of the other
    quantised rollouts)."""
    from rl_b200.engine.engine import SamplingParams
    from rl_b200.models.config import preset
    from rl_b200.models.transformer import PackedBatch, build_model

    if kind == "hybrid":
        mc = preset("tiny-nemotron-h", vocab_size=4096, hidden_size=512, intermediate_size=1024, head_dim=128, num_attention_heads=4, num_key_value_heads=2)
    else:
        mc = preset("tiny-llama-oracle", num_experts=8, num_experts_per_tok=2, moe_intermediate_size=128, norm_topk_prob=True, hidden_size=256, num_attention_heads=2,
                    num_key_value_heads=1, head_dim=128, vocab_size=2048)
    model = build_model(mc, device="cuda", dtype=torch.bfloat16, seed=7)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(1, mc.vocab_size, (n,), generator=g).tolist() for n in (9, 170, 5, 30)]
    runs = [_engine(model, use_cuda_graphs=graphs).generate(prompts, SamplingParams(max_new_tokens=24, stop_token_ids=[], seed=3, temperature=1.0)) for graphs in (True, False)]
    assert L.check_status() == 0
    assert sum(a.out_tokens == b.out_tokens for a, b in zip(*runs)) >= 3      # (the few-token expert layer's sums may split a tie)
    gaps = []
    for r in runs[0]:
        seq = torch.tensor([r.prompt + r.out_tokens], device="cuda")
        with torch.no_grad():
            lp, _ = model.next_token_logprobs(PackedBatch.from_padded(seq, torch.tensor([seq.shape[1]], device="cuda")), temperature=1.0)
        gaps.append((lp[len(r.prompt) :].float().cpu() - torch.tensor(r.out_logprobs)).abs())
    gaps = torch.cat(gaps)
    assert 0 < gaps.mean() < 0.3 and gaps.max() < 2.0, (gaps.mean(), gaps.max())
