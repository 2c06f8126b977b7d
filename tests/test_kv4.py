"""The 4-bit key/value cache on the CPU: what a page holds, against loops over the definition in 64 bits, and what the operators refuse."""

import math

import pytest
import torch
from kv4_oracle import replayed

from rl_b200.ops import kv4_ops as K

SHAPES = [(64, 2, 16), (128, 3, 48), (256, 1, 64)]      # D, Hkv, tokens of a page


def _group(x):
    """(scale, codes) of 32 Python floats."""
    a = max(abs(v) for v in x)
    if not all(map(math.isfinite, x)):
        return math.nan, [8] * 32
    if a < 2.0 ** -100:
        return 0.0, [8] * 32
    s = float(torch.tensor(a / 7.5, dtype=torch.float64).to(torch.bfloat16))
    return s, [min(15, max(0, math.floor(v / s) + 8)) for v in x]


def _place(page, D, block, off, value, d):
    """(code, scale) of one number in a page's bytes, by the order that csrc/kv4.cuh states."""
    G, n, (g, i) = D // 32, block * D // 2, divmod(d, 32)
    if value:
        unit = n + (off // 2) * D + ((i // 4) * G + g) * 4 + (off % 2) * 2
    else:
        unit = off * (D // 2) + ((i // 8) * G + g) * 4 + (i // 4 % 2) * 2
    word = int(page[unit]) | int(page[unit + 1]) << 8
    at = 2 * n + (off * 2 + value) * 2 * G + 2 * g
    return word >> (4 * (i % 4)) & 15, float(page[at : at + 2].clone().view(torch.bfloat16))


def _rows(T, Hq, Hkv, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, (Hq + 2 * Hkv) * D, generator=g) * (1 + 3 * (torch.arange((Hq + 2 * Hkv) * D) % 29 == 3))).bfloat16()


def _freq(D):
    return 10000.0 ** (-torch.arange(0, D, 2).float() / D)


@pytest.mark.parametrize("D,Hkv,block", SHAPES)
def test_page_order_and_codes(D, Hkv, block):
    T, Hq = 5, Hkv
    cache = K.kv4_cache(3, Hkv, block, D, "cpu")
    assert cache.shape == (3, Hkv, block * D * 9 // 8)
    slots = torch.tensor([2 * block + 7, 3, -1, block + block - 1, 0])
    out = K.rope_kv4_cache_write(_rows(T, Hq, Hkv, D), torch.arange(T), _freq(D), slots, cache, Hq, Hkv, D)
    back = K.kv4_cache_read(cache, slots, Hkv, D)
    for t, slot in enumerate(slots.tolist()):
        for value in (0, 1):
            for h in range(Hkv):
                at = (Hq + value * Hkv + h) * D
                for g in range(D // 32):
                    x = [float(v) for v in out[t, at + 32 * g : at + 32 * g + 32]]
                    s, codes = _group(x)
                    for i in range(32):
                        if slot < 0:
                            assert float(back[t, (value * Hkv + h) * D + 32 * g + i]) == 0.0
                            continue
                        assert _place(cache[slot // block, h], D, block, slot % block, value, 32 * g + i) == (codes[i], s)
                        want = torch.tensor((codes[i] - 7.5) * s, dtype=torch.float64).to(torch.bfloat16)
                        assert back[t, (value * Hkv + h) * D + 32 * g + i] == want
                        assert abs(float(want) - x[i]) <= s * (0.5 + 2.0 ** -4)      # half a level, and 7.5 levels' worth of the scale's rounding 2^-8 and the result's
    assert not cache[0, :, : block * D // 2].view(Hkv, block, -1)[:, [1, 2, 4, 5]].any()


def test_rotation_is_that_of_the_formula():
    T, Hq, Hkv, D = 7, 2, 1, 64
    pos = torch.tensor([0, 1, 1000, 131071, 20_000_003, 2**31 - 1, 77])
    x = _rows(T, Hq, Hkv, D)
    out = K.rope_kv4_cache_write(x, pos, _freq(D), torch.full((T,), -1), K.kv4_cache(1, Hkv, 16, D, "cpu"), Hq, Hkv, D)
    z = torch.polar(torch.ones((), dtype=torch.float64), pos.double()[:, None] * _freq(D).double())[:, None]
    v = x.double().reshape(T, Hq + 2 * Hkv, D)[:, : Hq + Hkv]
    want = torch.complex(v[..., : D // 2], v[..., D // 2 :]) * z
    want = torch.cat([want.real, want.imag], -1).reshape(T, -1)
    got = out[:, : (Hq + Hkv) * D].double()
    # one rounding to bf16, and the cosine, sine, products and sum in 32 bits (4 roundings of at most 2 max|x|)
    assert ((got - want).abs() <= want.abs() * 2.0 ** -8 + 4 * 2.0 ** -24 * 2 * v.abs().max()).all()
    assert torch.equal(out[:, (Hq + Hkv) * D :], x[:, (Hq + Hkv) * D :])


def test_special_values():
    D = 64
    x = torch.zeros(8, 64)
    x[1] = -0.0
    x[2, 5], x[3, 40], x[4, 0] = math.inf, math.nan, -math.inf
    x[5] = 2.0 ** -101
    x[6] = torch.finfo(torch.bfloat16).max * torch.linspace(-1, 1, 64)
    x[7] = torch.cat([torch.arange(-16, 16), torch.arange(-15, 17)]) * 0.125      # multiples of the scale: the upper code
    x = x.bfloat16()
    codes, s = K.quantize_ref(x)
    for i in range(8):
        for g in range(2):
            ws, wc = _group([float(v) for v in x[i, 32 * g : 32 * g + 32]])
            assert (math.isnan(ws) and bool(s[i, g].isnan())) or float(s[i, g]) == ws
            assert codes[i, g].tolist() == wc
    kv = K._values(codes, s)
    assert not kv[0].any() and not kv[1].any() and not kv[5].any() and kv[6].isfinite().all()
    assert kv[2, :32].isnan().all() and not kv[2, 32:].any() and kv[3, 32:].isnan().all() and kv[4, :32].isnan().all()


@pytest.mark.parametrize("D,Hkv,block", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 9, 40])
def test_decode_and_write_together(D, Hkv, block, window):
    """Tokens written one step at a time and attended to, as a decode loop does, against soft-max attention over the values that stand in the cache."""
    Hq, n = 3 * Hkv, 2 * block + 3
    cache = K.kv4_cache(5, Hkv, block, D, "cpu")
    table = torch.tensor([[4, 0, 3, 1]], dtype=torch.int32)
    kv = []
    for t in range(n):
        slot = int(table[0, t // block]) * block + t % block
        row = K.rope_kv4_cache_write(_rows(1, Hq, Hkv, D, seed=t).float(), torch.tensor([t]), _freq(D), torch.tensor([slot]), cache, Hq, Hkv, D)
        codes, s = K.quantize_ref(row[:, Hq * D :].reshape(2, Hkv, D))
        kv.append(K._values(codes, s).double())
        if t % 7 and t != n - 1:
            continue
        k, v = torch.stack(kv, 2)[:, :, max(0, t + 1 - window) if window else 0 :]
        q = row[0, : Hq * D].double().reshape(Hkv, 3, D)
        want = (torch.softmax(q @ k.transpose(1, 2) / math.sqrt(D), -1) @ v).reshape(-1)
        got = K.kv4_paged_decode(row, cache, table, torch.tensor([t + 1], dtype=torch.int32), Hq, Hkv, D, window=window)[0].double()
        # all in 32 bits: sums over D and over n, both below 2^9 terms
        assert (got - want).abs().max() <= 2.0 ** -24 * 2 ** 9 * 8 * v.abs().max()
    assert not K.kv4_paged_decode(row, cache, table, torch.tensor([0], dtype=torch.int32), Hq, Hkv, D).any()


def test_refusals():
    cache = K.kv4_cache(2, 2, 16, 64, "cpu")
    x, f, one = _rows(1, 4, 2, 64), _freq(64), torch.zeros(1, dtype=torch.int64)
    bt, ln = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    bad = [
        lambda: K.kv4_page_bytes(16, 96),
        lambda: K.kv4_page_bytes(24, 64),
        lambda: K.kv4_page_bytes(0, 64),
        lambda: K.kv4_page_bytes(2 * K.MAX_BLOCK, 64),
        lambda: K.rope_kv4_cache_write(x, one, f, one, cache, 4, 2, 80),
        lambda: K.rope_kv4_cache_write(x, one, f, one, cache, 3, 2, 64),
        lambda: K.rope_kv4_cache_write(x, one, f.double(), one, cache, 4, 2, 64),
        lambda: K.rope_kv4_cache_write(x, one, f[:-1], one, cache, 4, 2, 64),
        lambda: K.rope_kv4_cache_write(x, one.float(), f, one, cache, 4, 2, 64),
        lambda: K.rope_kv4_cache_write(x, one, f, torch.zeros(2, dtype=torch.int64), cache, 4, 2, 64),
        lambda: K.rope_kv4_cache_write(x, one, f, one, cache.float(), 4, 2, 64),
        lambda: K.rope_kv4_cache_write(x, one, f, one, cache[:, :, :-8], 4, 2, 64),
        lambda: K.rope_kv4_cache_write(x, one, f, one, K.kv4_cache(2, 3, 16, 64, "cpu"), 4, 2, 64),
        lambda: K.kv4_cache_read(cache, one, 2, 128),
        lambda: K.kv4_cache_read(cache, one, 2, 64, rows=one),
        lambda: K.kv4_cache_read(cache, one, 2, 64, out=torch.zeros(1, 255)),
        lambda: K.kv4_cache_read(cache, one, 2, 64, out=torch.zeros(0, 256)),
        lambda: K.kv4_cache_read(cache, one, 2, 64, out=torch.zeros(3, 256), rows=torch.zeros(2, dtype=torch.int64)),
        lambda: K.kv4_paged_decode(x, cache, bt, ln, 3, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt, ln, 16, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt[0], ln, 4, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt, ln[:0], 4, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt.float(), ln, 4, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt.long(), ln, 4, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt, ln.long(), 4, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt, ln, 4, 2, 64, scale=math.inf),
        lambda: K.kv4_paged_decode(x.float().requires_grad_(), cache, bt, ln, 4, 2, 64),
        lambda: K.rope_kv4_cache_write(x.float().requires_grad_(), one, f, one, cache, 4, 2, 64),
        lambda: K.kv4_paged_decode(x, cache, bt, ln, 4, 2, 64, window=-1),
        lambda: K.kv4_paged_decode(x, cache, bt, ln, 4, 2, 64, out=torch.zeros(1, 256)),
        lambda: K.kv4_paged_decode(x, cache, bt, ln, 4, 2, 64, out=torch.zeros(2, 256).bfloat16()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} went through")
    assert not cache.any()


def test_plan():
    """A cluster or CTAs that share, never both; no cluster without eight steps for each of its CTAs."""
    for D in (64, 128, 256):
        for B in (0, 1, 3, 16, 64, 500, 5000):
            for Hq, Hkv in ((32, 8), (16, 1), (8, 8)):
                for n in (0, 1, 256, 300, 1000, 4000, 20000, 10**6):
                    cluster, ctas = K.kv4_plan(B, Hq, Hkv, D, n)
                    assert 1 <= cluster <= K.MAX_CLUSTER and (ctas == 0 or cluster == 1) and (cluster == 1 or n > 32 * 8 * (cluster - 1))
                    assert ctas in (0, 148 * 2, 148 * {64: 4, 128: 3, 256: 2}[D])


# ------------------------------------------------------------------------------------------- the engine
def _model(**kw):
    from rl_b200.models.config import ModelConfig
    from rl_b200.models.transformer import CausalLM

    torch.manual_seed(0)
    mc = ModelConfig(**{**dict(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                               head_dim=64, torch_dtype="float32"), **kw})
    return CausalLM(mc, dtype=torch.float32, device="cpu", seed=1)


def _engine(model, **kw):
    from rl_b200.engine.engine import GenerationEngine

    return GenerationEngine(model, **{**dict(block_size=16, num_blocks=64, max_running=8, max_model_len=128, use_cuda_graphs=False, kv_cache_dtype="int4"), **kw})


@pytest.mark.parametrize("kind", ["llama", "qk_norm", "window"])
def test_engine_on_the_4_bit_cache(kind):
    """Whole prompts, shared prompts, prompts in portions and cached prefixes give the log-probabilities of the model whose cached keys and values are what 4 bits hold."""
    from rl_b200.engine.engine import SamplingParams
    from rl_b200.models.config import preset
    from rl_b200.models.transformer import CausalLM

    model = _model(qk_norm=True) if kind == "qk_norm" else _model()
    if kind == "window":
        mc = preset("gemma3-1b", torch_dtype="float32", vocab_size=97, hidden_size=32, intermediate_size=64, num_hidden_layers=3, num_attention_heads=4,
                    num_key_value_heads=2, head_dim=64, sliding_window=6, attn_scale=0.1, embed_scale=32 ** 0.5,
                    layer_types=["sliding_attention", "full_attention", "sliding_attention"])
        model = CausalLM(mc, dtype=torch.float32, device="cpu", seed=1)
    long = [(7 * i) % 90 + 1 for i in range(37)]
    prompts = [long, long, [9, 8, 7], [11] * 16, [5] * 17]
    sp = SamplingParams(max_new_tokens=9, stop_token_ids=[], seed=3, temperature=0.8)
    for kw, portions in ((dict(), lambda n: [n]), (dict(max_prefill_tokens=16), None)):
        eng = _engine(model, **kw)
        seen = {}
        if portions is None:      # (a round's budget is shared by its prompts: what each portion is, is looked at)
            rounds = eng._prefill_round
            eng._prefill_round = lambda items, *a, **k: ([seen.setdefault(tuple(q), []).append(p + n) for _, q, p, n in items], rounds(items, *a, **k))[1]
        for r in eng.generate(prompts, sp):
            n = len(r.prompt)
            cut = portions(n) if portions else seen.get(tuple(r.prompt), [n])
            want = replayed(model, r, cut, 0.8)
            # float32 on both sides, sums in other orders; a value may fall on the other side of its code's border: one level of one value of 64
            assert (want - torch.tensor(r.out_logprobs)).abs().max() < 5e-3, (kw, n)
        assert portions is not None or any(len(v) > 1 for v in seen.values())


def test_engine_shares_and_evicts_like_the_other_cache():
    """Siblings of a prompt whose last page is copied, and sequences that lose their pages and are prefilled again, are greedy alike."""
    from rl_b200.engine.engine import SamplingParams

    model = _model()
    prompt = [(5 * i) % 90 + 1 for i in range(21)]
    sp = SamplingParams(max_new_tokens=20, stop_token_ids=[], seed=3, temperature=0.0)
    one = _engine(model).generate([prompt], sp)[0].out_tokens
    assert all(r.out_tokens == one for r in _engine(model).generate([prompt] * 6, sp))
    tight = _engine(model, num_blocks=9)
    assert all(len(r.out_tokens) == 20 for r in tight.generate([prompt, [3] * 20, [4] * 30], sp))


def test_engine_memory_and_refusals():
    from rl_b200.engine.engine import GenerationEngine
    from rl_b200.engine.generation import NativeGeneration
    from rl_b200.models.config import preset
    from rl_b200.models.transformer import CausalLM

    model = _model()
    small, big = _engine(model), _engine(model, kv_cache_dtype="auto")
    small.wake()
    big.wake()
    assert small.kv_cache_bytes() == sum(t.numel() for t in small.k_cache) and small.v_cache == [None, None]
    assert small.kv_cache_bytes() * 32 == big.kv_cache_bytes() * 9 // 2      # 4.5 bits a value; the model here has 32
    for bad in (dict(kv_cache_dtype="int3"), dict(block_size=24), dict(block_size=4)):
        with pytest.raises(ValueError):
            _engine(model, **bad)
    with pytest.raises(ValueError):
        _engine(_model(head_dim=32))
    layered = CausalLM(preset("tiny-gadarax", torch_dtype="float32"), dtype=torch.float32, device="cpu", seed=1)
    with pytest.raises(NotImplementedError):
        GenerationEngine(layered, block_size=16, num_blocks=8, max_running=2, max_model_len=64, use_cuda_graphs=False, kv_cache_dtype="int4")
    cfg = dict(block_size=16, kv_cache_tokens=256, max_running=4, max_model_len=64, use_cuda_graphs=False)
    assert NativeGeneration(model, dict(cfg, kv_cache_dtype="int4")).engine.kv4 and NativeGeneration(model, dict(cfg, vllm_cfg=dict(kv_cache_dtype="int4"))).engine.kv4
    assert not NativeGeneration(model, dict(cfg, vllm_cfg=dict(kv_cache_dtype="fp8"))).engine.kv4 and not NativeGeneration(model, cfg).engine.kv4
    for bad in (dict(kv_cache_dtype="int8"), dict(vllm_cfg=dict(kv_cache_dtype="int"))):
        with pytest.raises(ValueError):
            NativeGeneration(model, {**cfg, **bad})


def _generation_rank(generation):
    from rl_b200.algorithms.noncolocated import build_generation_rank
    from rl_b200.models.config import ModelConfig

    mc = ModelConfig(vocab_size=97, hidden_size=64, intermediate_size=96, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1, head_dim=64, torch_dtype="float32")
    g = dict(block_size=16, kv_cache_tokens=64, max_running=2, use_cuda_graphs=False, **generation)
    return build_generation_rank(dict(policy=dict(precision="float32", max_total_sequence_length=64, generation=g)), None, mc, torch.device("cpu")).engine


@pytest.mark.parametrize("section", [None, "vllm_cfg", "native_cfg"])
def test_generation_ranks_read_every_section(section):
    """A rank of its own for generation holds its cache as the section, ``vllm_cfg`` or ``native_cfg`` says."""
    for name in ("int4", "auto"):
        asked = dict(kv_cache_dtype=name)
        assert _generation_rank({section: asked} if section else asked).kv4 == (name == "int4")


@pytest.mark.parametrize("section", ["vllm_cfg", "native_cfg"])
@pytest.mark.parametrize("unset", ["auto", None])
def test_auto_in_a_subsection_asks_for_nothing(section, unset):
    """``auto`` there, the reference's default, leaves the choice to the section itself."""
    from rl_b200.engine.generation import NativeGeneration
    from rl_b200.policy.worker import PolicyWorker

    asked = {"kv_cache_dtype": "int4", section: dict(kv_cache_dtype=unset)}
    assert _generation_rank(asked).kv4
    cfg = dict(block_size=16, kv_cache_tokens=256, max_running=4, max_model_len=64, use_cuda_graphs=False, **asked)
    assert NativeGeneration(_model(), cfg).engine.kv4
    both = dict(native_cfg=dict(kv_cache_dtype="auto"), vllm_cfg=dict(kv_cache_dtype="int4"))
    assert _generation_rank(both).kv4
    p = PolicyWorker(dict(precision="float32", train_global_batch_size=2, train_micro_batch_size=2, max_total_sequence_length=64,
                          optimizer=dict(name="torch.optim.AdamW", kwargs=dict(lr=1e-4)), generation=cfg), model_cfg=_model().cfg, device="cpu", init_reference_model=False, seed=3)
    assert p.build_generation().engine.kv4


@pytest.mark.parametrize("name", ["auto", "bfloat16", "bf16", "float16", "fp16", "half", "float32", "fp32", "float", "fp8", "fp8_e4m3", "fp8_e5m2"])
def test_names_of_the_models_type(name):
    """Every name of a type without a 4-bit cache serves the model's type, as before there was one; a name that nobody knows is refused."""
    from rl_b200.engine.generation import kv_cache_dtype_of

    for section in (None, "vllm_cfg", "native_cfg"):
        asked = dict(kv_cache_dtype=name)
        assert not _generation_rank({section: asked} if section else asked).kv4
    for unknown in ("int8", "bfloat", "bf16x", "INT4 "):
        assert kv_cache_dtype_of(dict(kv_cache_dtype=unknown)) == unknown
        with pytest.raises(ValueError):
            _generation_rank(dict(kv_cache_dtype=unknown))


def test_outputs_whose_rows_overlap_are_refused():
    T, Hq, Hkv, D, block = 4, 2, 1, 64, 16
    cache, slots, mem = K.kv4_cache(2, Hkv, block, D, "cpu"), torch.arange(T), torch.zeros(4 * T * 2 * D)
    q, table, n = _rows(T, Hq, Hkv, D).float(), torch.zeros((T, 1), dtype=torch.int32), torch.full((T,), 9, dtype=torch.int32)
    for strides in ((0, 1), (8, 1), (2 * D - 4, 1), (2 * D, 2), (2 * D, 0)):
        for call in (lambda out: K.kv4_cache_read(cache, slots, Hkv, D, out=out), lambda out: K.kv4_paged_decode(q, cache, table, n, Hq, Hkv, D, out=out)):
            with pytest.raises(RuntimeError):
                call(mem.as_strided((T, 2 * D), strides))
    for strides in ((1, T), (2 * D, 1), (6 * D - 1, 3)):
        assert K.kv4_cache_read(cache, slots, Hkv, D, out=mem.as_strided((T, 2 * D), strides)).shape == (T, 2 * D)


# ------------------------------------------------------------------------------------------- the engine's other paths, against a cache of the model's type that holds what 4 bits hold
def held_write(qkv, positions, inv_freq, slots, k_cache, v_cache, Hq, Hkv, D):
    """The write of the model's type's cache, with what the 4-bit cache would keep in the place of keys and values."""
    T = qkv.shape[0]
    out = qkv.clone()
    out[:, : (Hq + Hkv) * D] = K._rotate_ref(qkv[:, : (Hq + Hkv) * D].reshape(T, Hq + Hkv, D), positions, inv_freq).reshape(T, -1)
    kv = K._values(*K.quantize_ref(out[:, Hq * D :].reshape(T, 2, Hkv, D))).to(k_cache.dtype)
    ok = slots >= 0
    page, off = slots[ok] // k_cache.shape[2], slots[ok] % k_cache.shape[2]
    k_cache[page, :, off], v_cache[page, :, off] = kv[ok, 0], kv[ok, 1]
    return out


def _against_held(monkeypatch, model, prompts, sp, **kw):
    """Runs both engines. Log-probabilities agree for as long as both sample the same tokens (float32, sums in other orders: a value may fall on the other side of its code's border,
    one level of one value), which is most of the way. Returns the 4-bit engine."""
    from rl_b200.ops import engine_ops as E

    eng = _engine(model, **kw)
    got = eng.generate(prompts, sp)
    with monkeypatch.context() as m:
        m.setattr(E, "rope_kv_cache_write", held_write)
        want = _engine(model, kv_cache_dtype="auto", **kw).generate(prompts, sp)
    compared = 0
    for a, b in zip(got, want):
        assert len(a.out_tokens) == len(b.out_tokens) == sp.max_new_tokens
        same = next((i for i, (x, y) in enumerate(zip(a.out_tokens, b.out_tokens)) if x != y), len(a.out_tokens))
        compared += same
        gap = (torch.tensor(a.out_logprobs[:same]) - torch.tensor(b.out_logprobs[:same])).abs()
        assert same == 0 or gap.max() < 5e-3, gap
    assert compared * 2 > sp.max_new_tokens * len(prompts), compared
    return eng


def _louder(model):
    with torch.no_grad():
        for n, p in model.named_parameters():
            if p.dim() >= 2 and "conv" not in n:
                p.mul_(3.0)
    return model


def test_engine_prefills_again_what_lost_its_pages(monkeypatch):
    """A cache so small that sequences are preempted and come back: prompt and generated tokens are prefilled again into other pages."""
    from rl_b200.engine.engine import SamplingParams

    prompts = [[(5 * i) % 90 + 1 for i in range(21)], [3] * 20, [4] * 30]
    for temperature in (0.0, 0.8):
        eng = _against_held(monkeypatch, _model(), prompts, SamplingParams(max_new_tokens=40, stop_token_ids=[], seed=3, temperature=temperature), num_blocks=9)
        assert eng.sched.num_preemptions > 0


def test_engine_serves_hybrid_models_on_the_4_bit_cache(monkeypatch):
    """Nemotron-H blocks: the attention blocks' keys and values in 4 bits, no rotation, prompts whole and in portions."""
    from rl_b200.engine.engine import SamplingParams

    model = _louder(_model(model_type="nemotron_h", layers_block_type=["mamba", "mlp", "attention", "mamba", "moe", "attention"], num_hidden_layers=6, mamba_num_heads=4, mamba_head_dim=8,
                           ssm_state_size=8, mamba_n_groups=2, mamba_chunk_size=4, use_rope=False, mlp_gated=False, hidden_act="relu2", num_experts=4, num_experts_per_tok=2,
                           moe_intermediate_size=16, n_shared_experts=1, moe_shared_expert_intermediate_size=24, scoring_func="sigmoid"))
    prompts = [[1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11] * 3, [9, 8, 7], [11] * 9, [5, 4, 3, 2, 1, 2, 3, 4, 5, 6, 7, 8, 9]]
    for kw in (dict(), dict(max_prefill_tokens=16)):
        eng = _against_held(monkeypatch, model, prompts, SamplingParams(max_new_tokens=10, stop_token_ids=[], seed=3, temperature=0.8), **kw)
        assert eng.hybrid and sum(c is not None for c in eng.k_cache) == 2


def test_engine_serves_expert_models_on_the_4_bit_cache(monkeypatch):
    from rl_b200.engine.engine import SamplingParams

    model = _model(model_type="qwen3_moe", qk_norm=True, num_hidden_layers=3, num_experts=8, num_experts_per_tok=2, moe_intermediate_size=16)
    prompts = [[1, 2, 3, 4, 5, 6, 7, 8, 9] * 3, [9, 8, 7], [1, 2, 3, 4, 5, 6, 7, 8, 9] * 3]
    for kw in (dict(), dict(max_prefill_tokens=16)):
        _against_held(monkeypatch, model, prompts, SamplingParams(max_new_tokens=12, stop_token_ids=[], seed=3, temperature=0.8), **kw)


_TENSOR_PARALLEL = dict(precision="float32", train_global_batch_size=4, train_micro_batch_size=2, max_total_sequence_length=96,
                        optimizer=dict(name="torch.optim.AdamW", kwargs=dict(lr=1e-3)),
                        generation=dict(max_new_tokens=12, temperature=1.0, stop_token_ids=[], kv_cache_tokens=2048, block_size=16, max_running=8, kv_cache_dtype="int4"))


def _served(ranks):
    from rl_b200.distributed.batched_data_dict import BatchedDataDict
    from rl_b200.models.config import preset
    from rl_b200.policy.worker import PolicyWorker

    w = PolicyWorker(dict(_TENSOR_PARALLEL, parallel=dict(tensor_parallel_size=ranks)), model_cfg=preset("tiny-llama-oracle", torch_dtype="float32"), init_reference_model=False, seed=4)
    gen = w.build_generation()
    assert gen.engine.kv4 and gen.engine.hkv * ranks == w.model_cfg.num_key_value_heads
    gen.prepare_for_generation()
    ids = torch.randint(1, 2048, (3, 40), generator=torch.Generator().manual_seed(20))
    out = gen.generate(BatchedDataDict(input_ids=ids, input_lengths=torch.full((3,), 40)), greedy=True)
    return out["output_ids"].tolist(), out["logprobs"].tolist()


def _served_by_two(rank, world):
    return _served(world)


def test_tensor_parallel_engine_on_the_4_bit_cache():
    """Two ranks, each with half of the key/value heads in 4 bits: the tokens and log-probabilities of one rank."""
    from test_parallel_cpu import _spawn

    from rl_b200.parallel.state import reset_parallel

    got = _spawn(_served_by_two, 2)
    reset_parallel()
    ids, lp = _served(1)
    assert got[0][0] == got[1][0] == ids
    assert (torch.tensor(got[0][1]) - torch.tensor(lp)).abs().max() < 5e-3


def test_plan_at_its_thresholds():
    """Twice the CTAs from six steps of 32 tokens for each on, eight steps more where some multiprocessors get two of them, and only while all run at once."""
    for cluster, steps in ((2, 12), (4, 24), (8, 48)):
        assert K.kv4_plan(1, 32, 8, 128, 32 * steps) == (cluster, 0) and K.kv4_plan(1, 32, 8, 128, 32 * steps - 31) == (cluster, 0)
        assert K.kv4_plan(1, 32, 8, 128, 32 * (steps - 1)) == (cluster // 2, 0)
    for B, Hkv, D in ((1, 1, 64), (3, 2, 128), (20, 4, 64), (40, 8, 128), (12, 8, 256), (9, 3, 256)):
        slots = {64: 4, 128: 3, 256: 2}[D] * 148
        for n in range(1, 3000, 31):
            cluster, ctas = K.kv4_plan(B, Hkv, Hkv, D, n)
            assert cluster == 1 or (ctas == 0 and -(-n // 32) >= 6 * cluster + (8 if B * Hkv * cluster > 148 else 0) and B * Hkv * cluster <= slots)


def test_scales_beyond_32_bits_are_refused():
    """The kernels take the scale in 32 bits, where these would be infinite."""
    cache, q = K.kv4_cache(1, 1, 16, 64, "cpu"), _rows(1, 1, 1, 64)
    for scale in (1e39, -1e300, math.inf, math.nan):
        with pytest.raises(ValueError):
            K.kv4_paged_decode(q, cache, torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), 1, 1, 64, scale=scale)
    assert K.kv4_paged_decode(q, cache, torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32), 1, 1, 64, scale=3e38).shape == (1, 64)
