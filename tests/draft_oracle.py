"""Speculative decoding in 64 bits, row by row, and the batches that the tests of its operators run on."""

import math

import torch

FMAX = torch.finfo(torch.float32).max


def tree(n, g, children=3, chain=False):
    """Parents of ``n`` rows."""
    got, has = [], [0] * n
    for j in range(n):
        if j == 0:
            got.append(-1)
            continue
        free = [i for i in range(j) if has[i] < children]
        p = j - 1 if chain else free[int(torch.randint(len(free), (1,), generator=g))]
        has[p] += 1
        got.append(p)
    return got


def forest(sizes, seed=0, children=3, chain=False):
    """(parents [T], cu_rows [B + 1]) of trees of these sizes."""
    g = torch.Generator().manual_seed(seed)
    parents = [p for n in sizes for p in tree(n, g, children, chain)]
    return torch.tensor(parents, dtype=torch.int32), torch.tensor([0] + sizes).cumsum(0).to(torch.int32)


def sees(parents):
    """bool [n, n] of one tree."""
    n = len(parents)
    got = torch.eye(n, dtype=torch.bool)
    for j in range(n):
        p = int(parents[j])
        if 0 <= p < j:
            got[j] |= got[p]
    return got


def words(bits, count):
    """bool [n, k] -> int32 [n, count]."""
    got = torch.zeros((bits.shape[0], count), dtype=torch.int32)
    for j in range(bits.shape[0]):
        for w in range(count):
            x = sum(1 << i for i, on in enumerate(bits[j, 32 * w : 32 * w + 32].tolist()) if on)
            got[j, w] = x - (1 << 32) if x >> 31 else x
    return got


def pages(lens, block, seed=0, spare=2):
    """int32 [B, pages] table of so many tokens each in any order, and the number of pages."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // block) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)      # behind a sequence's own pages the table holds no page
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    return table, sum(need) + spare


def attend(q, k, v, table, ctx, cu, Hq, Hkv, D, bits=None, scale=None, window=0, positions=None):
    """float64 [T, Hq D] and how far a kernel may be from it, for bf16 inputs. ``bits``: bool [n, n] of each sequence (None: chains).

    A weight is rounded to bf16 before the second product (at most 2^-8 of its share), the result to bf16 (2^-8 of it). Scores are sums of D products in 32 bits, scaled: off by
    D 2^-24 of the sum of their magnitudes, and once more in the largest score that they are compared with; exponentials, the sum of n weights and the scale are some 2^-20 more."""
    T, block = q.shape[0], k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, tol = torch.zeros((T, Hq, D), dtype=torch.float64), torch.zeros((T, Hq, D), dtype=torch.float64)
    for b, c in enumerate(ctx.tolist()):
        lo, hi = int(cu[b]), int(cu[b + 1])
        n = hi - lo
        if n <= 0:
            continue
        at = torch.arange(c + n)
        kk, vv = (x[table[b].long()[at // block], :, at % block].double().repeat_interleave(Hq // Hkv, 1) for x in (k, v))
        vis = torch.ones((n, c + n), dtype=torch.bool)
        vis[:, c:] = torch.ones(n, n).tril().bool() if bits is None else bits[b]
        if window:
            pos = positions[lo:hi].long()
            vis &= pos[:, None] - torch.cat([torch.arange(c), pos]) < window
        qq = q[lo:hi, : Hq * D].reshape(n, Hq, D).double()
        for i in range(n):
            ok = vis[i]
            if not ok.any():
                continue
            s = torch.einsum("hd,thd->ht", qq[i], kk[ok]) * scale
            size = torch.einsum("hd,thd->ht", qq[i].abs(), kk[ok].abs()).amax(-1) * abs(scale)
            p = torch.softmax(s, -1)
            out[lo + i] = torch.einsum("ht,thd->hd", p, vv[ok])
            soft = 2.0**-8 + 2 * D * 2.0**-24 * size[:, None] + 2.0**-20
            tol[lo + i] = 2.0**-8 * out[lo + i].abs() + soft * torch.einsum("ht,thd->hd", p, vv[ok].abs())
    return out.reshape(T, -1), tol.reshape(T, -1)


def probabilities(z, temp):
    z = torch.where(z.isnan(), -math.inf, z.double()).clamp(max=FMAX)
    if z.max() == -math.inf:
        return torch.zeros_like(z)
    return torch.softmax(torch.where(z == -math.inf, z, (z - z.max()) / temp), -1)


def verify(logits, tokens, parents, cu, uniforms, draft=None, temps=None, greedy=False, steps=256):
    """(tokens, rows, logprobs) of each sequence as lists, and how near each decision was to the other one."""
    got = []
    for b in range(len(cu) - 1):
        lo, n = int(cu[b]), int(cu[b + 1]) - int(cu[b])
        T = float(temps[b]) if temps is not None else 1.0
        cold, T = greedy or not T > 0, T if T > 0 else 1.0
        toks, rows, lps, near = [], [], [], 1.0
        node = 0
        while n > 0:
            p = probabilities(logits[lo + node], T)
            some = bool(p.sum() > 0)
            z = torch.where(logits[lo + node].isnan(), -math.inf, logits[lo + node].double()).clamp(max=FMAX)
            best = int((z == z.max()).nonzero()[0]) if some else 0
            q = probabilities(draft[lo + node], T) if draft is not None else None
            w, went = p.clone(), -1
            if len(toks) + 1 < steps:
                for j in range(1, n):
                    if int(parents[lo + j]) != node:
                        continue
                    x, u = int(tokens[lo + j]), float(uniforms[lo + j])
                    if cold:
                        if some and x == best:
                            went = j
                            break
                        continue
                    if not 0 <= x < len(p) or not w.sum() > 0:
                        continue
                    share = w / w.sum()
                    limit = float(share[x] / q[x]) if draft is not None and q[x] > 0 else math.inf if draft is not None and share[x] > 0 else float(share[x])
                    near = min(near, abs(limit - u))
                    if u < limit:
                        went = j
                        break
                    if draft is not None:
                        w = (share - q).clamp(min=0)
                    else:
                        w[x] = 0
            if went >= 0:
                x = int(tokens[lo + went])
            elif cold or not some:
                x = best
            else:
                w = w if w.sum() > 0 else p
                run = w.cumsum(0)
                aim = float(uniforms[lo]) * float(run[-1])
                near = min(near, float((run - aim).abs()[w > 0].min() / run[-1]))
                over = ((run > aim) & (w > 0)).nonzero()
                x = int(over[0]) if len(over) else int((w > 0).nonzero()[-1])
            toks.append(x)
            rows.append(node)
            lps.append(math.log(float(p[x])) if some and p[x] > 0 else -math.inf if some is False else float(((z[x] - z.max()) / T - torch.log(torch.exp((z - z.max()) / T).sum()))))
            if went < 0:
                break
            node = went
        got.append((toks, rows, lps, near))
    return got
