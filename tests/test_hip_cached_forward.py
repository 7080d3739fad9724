"""Cached forwards of the denoiser (DreamModel_length.forward_cached, diffusion_generate(cache_interval=R)) and models with
per-head norms, on the GPU against a float64 forward with the same cache semantics.

Bars: the ones this package states for whole forwards -- fp32 logits within 1e-3 absolute, bf16 logits within 3 % of their
range."""
import math

import pytest
import torch

from dark_amd import DreamConfig, DreamGenerationConfig, DreamModel_length, kv_cache, synth

pytestmark = pytest.mark.gpu
DEV = "cuda"


def config(**kw):
    base = dict(vocab_size=512, hidden_size=192, intermediate_size=384, num_hidden_layers=2, num_attention_heads=2,
                num_key_value_heads=2, max_position_embeddings=512, mask_token_id=synth.MASK, pad_token_id=synth.END)
    base.update(kw)
    return DreamConfig(**base)


def build(cfg, dtype):
    w = synth.make_weights(cfg, seed=0, rich=True)
    if cfg.qk_norm:
        g = torch.Generator().manual_seed(5)
        for i in range(cfg.num_hidden_layers):
            for n in ("q_norm", "k_norm"):
                w[f"model.layers.{i}.self_attn.{n}.weight"] = 1 + 0.2 * torch.randn(cfg.head_dim, generator=g)
    m = DreamModel_length(cfg)
    m.load_state_dict(w, strict=True)
    m = m.to(DEV).to(dtype)
    return m, {k: v.detach().cpu().double() for k, v in m.state_dict().items()}


def reference(w, cfg, ids, index, store, kv_len, key_mask=None, causal=False):
    """Logits of tokens `ids` at places `index` of ONE sequence in float64; store: per layer (k, v) [kv_len, H, D], updated."""
    H, D, eps = cfg.num_attention_heads, cfg.head_dim, cfg.rms_norm_eps
    rms = lambda x, g: x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * g
    ang = index.double()[:, None] * float(cfg.rope_theta) ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    cos, sin = ang.cos()[:, None], ang.sin()[:, None]

    def rope(x):
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    x = w["model.embed_tokens.weight"][ids]
    for i in range(cfg.num_hidden_layers):
        p = f"model.layers.{i}."
        n = rms(x, w[p + "input_layernorm.weight"])
        q, k, v = ((n @ w[p + f"self_attn.{s}_proj.weight"].t() + w[p + f"self_attn.{s}_proj.bias"]).view(-1, H, D) for s in "qkv")
        if cfg.qk_norm:
            q, k = rms(q, w[p + "self_attn.q_norm.weight"]), rms(k, w[p + "self_attn.k_norm.weight"])
        q, k = rope(q), rope(k)
        K, V = store[i]
        K[index], V[index] = k, v
        s = torch.einsum("qhd,khd->hqk", q, K[:kv_len]) / math.sqrt(D)
        hide = torch.zeros(len(index), kv_len, dtype=torch.bool)
        if key_mask is not None:
            hide |= ~key_mask[:kv_len].bool()
        if causal:
            hide |= torch.arange(kv_len) > index[:, None]
        s = s.masked_fill(hide, -math.inf)
        o = torch.einsum("hqk,khd->qhd", s.softmax(-1), V[:kv_len]).reshape(len(index), -1)
        x = x + o @ w[p + "self_attn.o_proj.weight"].t()
        n = rms(x, w[p + "post_attention_layernorm.weight"])
        gate, up = n @ w[p + "mlp.gate_proj.weight"].t(), n @ w[p + "mlp.up_proj.weight"].t()
        x = x + (torch.nn.functional.silu(gate) * up) @ w[p + "mlp.down_proj.weight"].t()
    return rms(x, w["model.norm.weight"]) @ w["lm_head.weight"].t()


def new_store(cfg, n):
    return [tuple(torch.zeros(n, cfg.num_attention_heads, cfg.head_dim, dtype=torch.float64) for _ in range(2))
            for _ in range(cfg.num_hidden_layers)]


def close(got, want, dtype):
    tol = 1e-3 if dtype == torch.float32 else 0.03 * float(want.max() - want.min())
    err = (got.double().cpu() - want).abs().max()
    assert float(err) <= tol, (float(err), tol)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_all_positions_are_the_plain_forward(dtype, qk_norm):
    """Every position a new token: the plain forward, here with its padding mask and position ids."""
    cfg = config(qk_norm=qk_norm)
    m, w = build(cfg, dtype)
    B, N = 5, 46
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(7, 500, (B, N), generator=g)
    am = torch.ones(B, N, dtype=torch.bool)
    am[1, :9], am[3, :1] = False, False
    pos = (am.long().cumsum(-1) - 1).masked_fill(~am, 1)
    full = m(ids.to(DEV), attention_mask=am.to(DEV), position_ids=pos.to(DEV)).logits
    cache = m.make_cache(B * 48)
    table = torch.tensor([cache.allocate(N) for _ in range(B)], dtype=torch.int32, device=DEV)
    seq, index = torch.arange(B, device=DEV).repeat_interleave(N), torch.arange(N, dtype=torch.int32, device=DEV).repeat(B)
    out = m.forward_cached(cache, ids.view(-1).to(DEV), seq, index, table, torch.arange(0, B * N + 1, N, dtype=torch.int32, device=DEV),
                           torch.full((B,), N, dtype=torch.int32, device=DEV), N, N, position_ids=pos.view(-1).int().to(DEV),
                           key_mask=am.to(torch.uint8).to(DEV)).logits.view(B, N, -1)
    assert out.dtype == full.dtype
    keep = am.to(DEV)
    close(out[keep], full[keep].double().cpu(), dtype)
    for b in (0, 2):     # unpadded rows against float64
        close(out[b], reference(w, cfg, ids[b], torch.arange(N), new_store(cfg, N), N), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
def test_long_windows_in_chunks(dtype, causal):
    """Windows longer than the plain forward takes, two sequences of different lengths, filled in chunks and by single
    tokens; each chunk's logits against float64 with the same cache."""
    cfg = config(qk_norm=True)
    m, w = build(cfg, dtype)
    g = torch.Generator().manual_seed(2)
    lens = (300, 171)
    ids = [torch.randint(7, 500, (n,), generator=g) for n in lens]
    cache = m.make_cache(512, page_size=32)
    table = torch.full((2, 10), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        pages = cache.allocate(n)
        table[b, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
    store = [new_store(cfg, n) for n in lens]
    at = [0, 0]
    for step in ((150, 1), (100, 90), (1, 1), (49, 79)):
        n = list(step)
        kv = [at[b] + n[b] for b in range(2)]
        index = torch.cat([torch.arange(at[b], kv[b]) for b in range(2)])
        seq = torch.cat([torch.full((n[b],), b) for b in range(2)])
        new = torch.cat([ids[b][at[b]:kv[b]] for b in range(2)])
        out = m.forward_cached(cache, new.to(DEV), seq.to(DEV), index.int().to(DEV), table.to(DEV), i32(0, n[0], n[0] + n[1]), i32(*kv),
                               max(n), max(kv), causal=causal).logits
        want = torch.cat([reference(w, cfg, ids[b][at[b]:kv[b]], torch.arange(at[b], kv[b]), store[b], kv[b], causal=causal) for b in range(2)])
        close(out, want, dtype)
        at = kv


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_single_tokens(dtype):
    """One step of single tokens captured once and replayed along two sequences (ids, places and lengths written into the
    captured tensors), with eager steps on a cache of their own in between: the same bits."""
    cfg = config()
    m, _ = build(cfg, dtype)
    g = torch.Generator().manual_seed(3)
    lens, room = [40, 7], 64
    caches = [m.make_cache(2 * room, page_size=16) for _ in range(2)]
    tables = [torch.tensor([c.allocate(room) for _ in range(2)], dtype=torch.int32, device=DEV) for c in caches]
    ids = torch.randint(7, 500, (2, room), generator=g).to(DEV)
    seq, cu = torch.arange(2, device=DEV), i32(0, 1, 2)
    for c, t in zip(caches, tables):
        n = sum(lens)
        index = torch.cat([torch.arange(x) for x in lens]).int().to(DEV)
        m.forward_cached(c, torch.cat([ids[b, :x] for b, x in enumerate(lens)]), torch.repeat_interleave(seq, i32(*lens)), index, t,
                         i32(0, lens[0], n), i32(*lens), max(lens), room, causal=True)
    new, index, kv = ids[:, 0].clone(), i32(*lens), i32(*[x + 1 for x in lens])

    def step(c, t):
        return m.forward_cached(c, new, seq, index, t, cu, kv, 1, room, causal=True).logits

    side = torch.cuda.Stream()      # a first step outside the capture, on places that the loop writes again
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0], tables[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0], tables[0])
    for i in range(6):
        at = torch.tensor([x + i for x in lens])
        new.copy_(ids.cpu()[torch.arange(2), at])
        index.copy_(at.int())
        kv.copy_(at.int() + 1)
        graph.replay()
        want = step(caches[1], tables[1])
        torch.cuda.synchronize()
        assert torch.equal(got, want), i


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_some_positions_against_a_stale_cache(dtype):
    """kv_cache.WindowCache: a whole forward, then one for the masked positions and their left neighbours after tokens were
    committed; the other positions keep the first forward's keys and values."""
    cfg = config()
    m, w = build(cfg, dtype)
    B, N, mask = 4, 46, synth.MASK
    g = torch.Generator().manual_seed(3)
    x = torch.randint(7, 500, (B, N), generator=g)
    for b, (lo, hi) in enumerate(((1, 11), (12, 44), (45, 46), (0, 3))):
        x[b, lo:hi] = mask
    key_mask = torch.ones(B, N, dtype=torch.uint8)
    key_mask[2, :4] = 0
    st = m._hip_state(B, N)
    wc = kv_cache.WindowCache(m, B, N, None, key_mask.to(DEV), 3)
    wc.forward(st, x.to(DEV), mask)
    store = [new_store(cfg, N) for _ in range(B)]
    for b in range(B):
        want = reference(w, cfg, x[b], torch.arange(N), store[b], N, key_mask[b])
        got = st.head_rows(torch.arange(b * N, (b + 1) * N, dtype=torch.int32, device=DEV), N).clone()
        close(got[4 * (b == 2):], want[4 * (b == 2):], dtype)
    assert wc.min_masked == 1
    rows = [list(range(0, 11)), list(range(11, 44)), [44, 45], [0, 1, 2]]
    assert wc.rows.tolist() == [b * N + j for b in range(B) for j in rows[b]]
    x[0, 4], x[1, 20], x[2, 45], x[3, 0] = 100, 200, 300, 400
    wc.committed(1)
    wc.forward(st, x.to(DEV), mask)
    assert wc.done == 1
    for b in range(B):
        idx = torch.tensor(rows[b])
        want = reference(w, cfg, x[b][idx], idx, store[b], N, key_mask[b])
        got = st.head_rows((b * N + idx).int().to(DEV), len(idx)).clone()
        close(got, want, dtype)
    wc.committed(1)                      # row 2 has no mask left: something else gets re-masked
    assert wc.rows is None


def _generate(m, ids, steps, **kw):
    g = torch.Generator().manual_seed(7)
    noises = {}

    def noise(step, M, V):
        if (step, M) not in noises:
            noises[step, M] = torch.empty(M, V).exponential_(1, generator=g)
        return noises[step, M]

    trace = {}
    gc = DreamGenerationConfig(mask_token_id=synth.MASK, pad_token_id=synth.END, max_length=46)
    out = m.diffusion_generate(inputs=ids.to(DEV), generation_config=gc, return_dict_in_generate=True, output_history=True,
                               steps=steps, alg="entropy", alg_temp=0, top_p=0.9, temperature=0.1, _noise_fn=noise, _trace=trace, **kw)
    return torch.stack(out.history).cpu(), trace


@pytest.mark.parametrize("mode", ["abd", "ded"])
def test_generate_with_a_cache(mode):
    """R = 1 computes every position every time: the plain loop's confidences to fp32 accuracy and its tokens.  R = 4: the
    prompt stays, every mask is filled, as many tokens a step as without a cache."""
    cfg = config(max_position_embeddings=64)
    m, _ = build(cfg, torch.float32)
    ids = synth.make_inputs(6, mode, nentity=300, nrelation=111, seed=4)
    plain, t0 = _generate(m, ids, 12)
    every, t1 = _generate(m, ids, 12, cache_interval=1)
    torch.testing.assert_close(t1["confidence"][0], t0["confidence"][0], rtol=1e-4, atol=1e-4)
    assert t0["k"] == t1["k"] and t0["M"] == t1["M"]
    assert torch.equal(t0["x0"][0], t1["x0"][0])
    cached, t4 = _generate(m, ids, 12, cache_interval=4)
    assert t4["k"] == t0["k"] and t4["M"] == t0["M"]
    prompt = ids != synth.MASK
    assert torch.equal(cached[-1][:, :45][prompt], ids[prompt])
    assert not bool((cached[-1] == synth.MASK).any())
    assert torch.equal(cached[0], every[0]), "the first step runs a whole forward either way"


def test_generate_in_bf16_and_with_padding():
    cfg = config(max_position_embeddings=64, qk_norm=True)
    m, _ = build(cfg, torch.bfloat16)
    ids = synth.make_inputs(9, "abd", nentity=300, nrelation=111, seed=4)
    am = torch.ones_like(ids)
    am[2, :3] = 0
    out, _ = _generate(m, ids, 8, cache_interval=3, attention_mask=am.to(DEV))
    assert not bool((out[-1] == synth.MASK).any())


def test_refusals():
    cfg = config(max_position_embeddings=64)
    m, _ = build(cfg, torch.float32)
    ids = synth.make_inputs(2, "abd", nentity=300, nrelation=111)
    gc = DreamGenerationConfig(mask_token_id=synth.MASK, pad_token_id=synth.END, max_length=46)
    for kw in (dict(alg="origin"), dict(alg="entropy", generation_tokens_hook_func=lambda s, x, l: x)):
        with pytest.raises(NotImplementedError, match="cache_interval"):
            m.diffusion_generate(ids.to(DEV), generation_config=gc, steps=2, cache_interval=2, **kw)
    with pytest.raises(ValueError, match="cache_interval"):
        m.diffusion_generate(ids.to(DEV), generation_config=gc, steps=2, alg="entropy", cache_interval=-1)
    cache = m.make_cache(160)
    z = torch.zeros(1, dtype=torch.int64, device=DEV)
    args = (z, z, z.int(), torch.zeros(1, 10, dtype=torch.int32, device=DEV), i32(0, 1), i32(1), 1)
    assert m.forward_cached(cache, *args, 1).logits.shape == (1, 512)
    with pytest.raises(ValueError, match="rotation tables"):
        m.forward_cached(cache, *args, 129)
    with pytest.raises(ValueError, match="int32"):
        m.forward_cached(cache, z, z, z, *args[3:], 1)
    with pytest.raises(ValueError, match="not the model's"):
        m.forward_cached(kv_cache.PagedKVCache(2, 4, 16, 2, 64, torch.float32, DEV), *args, 1)
    with pytest.raises(ValueError, match="dtype"):
        m.forward_cached(kv_cache.PagedKVCache(2, 4, 16, 2, 96, torch.bfloat16, DEV), *args, 1)


def test_autograd_knows_of_a_cached_forward():
    cfg = config(max_position_embeddings=64)
    m, _ = build(cfg, torch.float32)
    cache = m.make_cache(16)
    z = torch.zeros(1, dtype=torch.int64, device=DEV)
    w = torch.ones_like(cache.k(0), requires_grad=True)
    cache._k.zero_()
    y = (w * cache.k(0)).sum()
    m.forward_cached(cache, z, z, z.int(), torch.zeros(1, 1, dtype=torch.int32, device=DEV), i32(0, 1), i32(1), 1, 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_the_expanding_model_in_windows_of_a_fixed_length():
    """DreamModel.diffusion_generate_length with a cache is DreamModel_length.diffusion_generate with one."""
    from dark_amd import DreamModel
    cfg = config(max_position_embeddings=64)
    m, _ = build(cfg, torch.float32)
    d = DreamModel(cfg)
    d.load_state_dict(m.state_dict(), strict=True)
    d = d.to(DEV)
    ids = synth.make_inputs(4, "abd", nentity=300, nrelation=111, seed=4)
    want, _ = _generate(m, ids, 9, cache_interval=3)
    d.diffusion_generate = d.diffusion_generate_length
    got, _ = _generate(d, ids, 9, cache_interval=3)
    assert torch.equal(got, want)
