"""What the generation engine computes on a 4-bit key/value cache, layer by layer in plain PyTorch."""

import math

import torch

from rl_b200.ops import kv4_ops as K


@torch.no_grad()
def replayed(model, r, portions, temperature):
    """Log-probabilities of a request's generated tokens, token by token: a token of a prompt sees the tokens of its own portion as they are and the
    ones before as the cache holds them; a generated token sees all, itself too, as the cache holds them."""
    from rl_b200.ops import functional as F

    c, dev = model.cfg, model.embed_tokens.device
    seq, P = r.prompt + r.out_tokens, len(r.prompt)
    edges = portions + list(range(P + 1, len(seq) + 1))
    held = [[] for _ in model.layers]
    out = []
    for a, b in zip([0] + edges, edges):
        pos = torch.arange(a, b, device=dev)
        h = F.embedding(torch.tensor(seq[a:b], dtype=torch.int32 if dev.type == "cuda" else torch.int64, device=dev), model.embed_tokens)
        h = h if c.embed_scale == 1.0 else h * c.embed_scale
        for li, layer in enumerate(model.layers):
            at = layer.self_attn
            qkv = at.project_qkv(F.rmsnorm(h, layer.input_layernorm, c.rms_norm_eps), pos, model.inv_freq, apply_rope=False).reshape(b - a, -1, c.head_dim)
            freq = model.inv_freq_local if layer.window and model.inv_freq_local is not None else model.inv_freq
            qk = K._rotate_ref(qkv[:, : at.hq + at.hkv], pos, freq)
            kv = torch.stack([qk[:, at.hq :], qkv[:, at.hq + at.hkv :]], 1)
            codes, s = K.quantize_ref(kv)
            stored = K._values(codes, s)
            seen = kv if a < P else stored
            k, v = torch.cat(held[li] + [seen.to(stored.dtype)]).transpose(0, 1).repeat_interleave(at.hq // at.hkv, 2)
            held[li].append(stored)
            z = torch.einsum("thd,shd->hts", qk[:, : at.hq].to(k.dtype), k) * (c.attn_scale if c.attn_scale is not None else c.head_dim ** -0.5)
            i, j = pos[:, None], torch.arange(b, device=dev)[None]
            z = z.masked_fill((j > i) | ((j <= i - layer.window) if layer.window else j > i), -math.inf)
            h = layer.tail(h, torch.einsum("hts,shd->thd", torch.softmax(z, -1), v).reshape(b - a, -1).to(h.dtype))
        if b >= P and b < len(seq):
            logits = F.rmsnorm(h[-1:], model.norm, c.rms_norm_eps).float() @ model.output_weight.float().t()
            out.append(torch.log_softmax(logits / temperature, -1)[0, seq[b]])
    return torch.stack(out)
