"""The paged cache's operators without a GPU: what their entry points refuse (C and Python), the packed argument
structs, and the float64 oracle of the GPU tests against a dense attention."""
import ctypes as C
import math

import pytest
import torch

from dark_amd import _hip, kv_cache
from oracle import kv_cache_oracle as O


def test_structs_match_the_header(tmp_path):
    """Sizes and last fields of the ctypes structs against what a C compiler makes of include/dark_hip.h."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"dark_paged_kv": _hip.PagedKV, "dark_qk_norm_rope_args": _hip.QkNormRopeArgs, "dark_kv_append_args": _hip.KVAppendArgs,
             "dark_paged_attention_args": _hip.PagedAttentionArgs, "dark_cached_tokens": _hip.CachedTokens,
             "dark_layer_weights": _hip.LayerWeights, "dark_model_desc": _hip.ModelDesc}
    src = '#include "dark_hip.h"\n#include <stdio.h>\nint main(void) {\n' + "".join(
        f'  printf("{n} %zu %zu\\n", sizeof({n}), offsetof({n}, {s._fields_[-1][0]}));\n' for n, s in names.items()) + "  return 0;\n}\n"
    (tmp_path / "s.c").write_text(src)
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    for line in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.splitlines():
        n, size, last = line.split()
        s = names[n]
        assert C.sizeof(s) == int(size) and getattr(s, s._fields_[-1][0]).offset == int(last), n


def _kv(**kw):
    f = dict(k=4096, v=8192, page_stride=16 * 8 * 96, slot_stride=8 * 96, head_stride=96, dtype=1, n_pages=4, page_size=16,
             n_kv_heads=8, head_dim=96)
    f.update(kw)
    return _hip.PagedKV(**f)


def _refused(fn, args, msg):
    lib = _hip.load()
    assert getattr(lib, fn)(C.byref(args) if args is not None else None, None) == _hip.DARK_ERR_ARG
    text = lib.dark_hip_last_error().decode()
    assert msg in text, text


@pytest.mark.parametrize("kw,msg", [(dict(dtype=2), "dtype"), (dict(head_dim=80), "head_dim"), (dict(n_tokens=-1), "n_tokens"),
                                    (dict(q=None), "null pointer"), (dict(q=4104), "16 bytes"), (dict(k_ts=100), "16 bytes"),
                                    (dict(rope_cos=None), "go together"), (dict(pos=None), "positions"), (dict(eps=-1.0), "eps"),
                                    (dict(eps=math.nan), "eps")])
def test_qk_norm_rope_refuses(kw, msg):
    f = dict(q=4096, k=4096, q_out=8192, k_out=8192, rope_cos=4096, rope_sin=4096, pos=4096, q_ts=768, q_hs=96, k_ts=768, k_hs=96,
             qo_ts=768, qo_hs=96, ko_ts=768, ko_hs=96, dtype=1, n_tokens=3, n_heads=8, n_kv_heads=8, head_dim=96, max_pos=64, eps=1e-6)
    f.update(kw)
    _refused("dark_qk_norm_rope", _hip.QkNormRopeArgs(**f), msg)


@pytest.mark.parametrize("kw,msg", [(dict(kv=_kv(page_size=24)), "power of two"), (dict(kv=_kv(k=None)), "null cache"),
                                    (dict(kv=_kv(slot_stride=100)), "16 bytes"), (dict(kv=_kv(n_kv_heads=0)), "n_kv_heads"),
                                    (dict(kv=_kv(page_stride=-768)), "negative"), (dict(slots=None), "null pointer"),
                                    (dict(q=None), "go together"), (dict(rope_sin=None), "go together"), (dict(max_pos=0), "positions"),
                                    (dict(v_hs=4), "16 bytes"), (dict(n_heads=5000), "heads")])
def test_kv_append_refuses(kw, msg):
    f = dict(kv=_kv(), q=4096, k=4096, v=4096, q_out=8192, rope_cos=4096, rope_sin=4096, pos=4096, slots=4096, q_ts=768, q_hs=96,
             k_ts=768, k_hs=96, v_ts=768, v_hs=96, qo_ts=768, qo_hs=96, n_tokens=3, n_heads=8, max_pos=64, eps=1e-6)
    f.update(kw)
    _refused("dark_kv_append", _hip.KVAppendArgs(**f), msg)


@pytest.mark.parametrize("kw,msg", [(dict(n_heads=9), "multiple"), (dict(kv=_kv(head_dim=32)), "head_dim"), (dict(q=None), "null pointer"),
                                    (dict(block_table=None), "null pointer"), (dict(max_kv=-1), "negative"), (dict(scale=math.inf), "scale"),
                                    (dict(o_ts=4), "16 bytes"), (dict(table_stride=1), "table_stride"), (dict(table_width=1 << 28), "2^30"),
                                    (dict(max_kv=100000), "workspace"),
                                    (dict(max_q=64, kv=_kv(page_stride=8 * ((1 << 27) + 1), n_pages=64)), "spans more")])
def test_paged_attention_refuses(kw, msg):
    f = dict(kv=_kv(), q=4096, out=8192, block_table=4096, cu_q=4096, kv_len=4096, q_ts=768, q_hs=96, o_ts=768, o_hs=96,
             table_stride=4, n_tokens=3, n_heads=8, n_seqs=2, table_width=4, max_q=2, max_kv=64, scale=0.1)
    f.update(kw)
    _refused("dark_paged_attention", _hip.PagedAttentionArgs(**f), msg)


def test_keys_and_values_into_one_cache_are_refused():
    """Two rows for every slot: whichever came last would stay."""
    f = dict(kv=_kv(v=4096), k=4096, v=4096, slots=4096, k_ts=768, k_hs=96, v_ts=768, v_hs=96, n_tokens=3, max_pos=64, eps=1e-6)
    _refused("dark_kv_append", _hip.KVAppendArgs(**f), "same memory")


def test_null_arguments():
    for fn in ("dark_qk_norm_rope", "dark_kv_append", "dark_paged_attention"):
        _refused(fn, None, "null arguments")
    assert _hip.load().dark_paged_attention_workspace_bytes(None) == 0


def test_head_norms_go_together():
    """A layer with one of the two norms is refused by both forwards before anything is launched."""
    lib = _hip.load()
    w = (_hip.LayerWeights * 1)()
    for name, _ in _hip.LayerWeights._fields_:
        setattr(w[0], name, 4096)
    desc = _hip.ModelDesc(dtype=1, vocab=512, vocab_pad=512, d=192, ff=384, n_layers=1, n_heads=2, head_dim=96, max_pos=64, rms_eps=1e-6,
                          resid_dtype=1, embed=4096, final_norm=4096, lm_head=4096, rope_cos=4096, rope_sin=4096,
                          layers=C.cast(w, C.POINTER(_hip.LayerWeights)))
    cached = _hip.CachedTokens(ids=4096, pos=4096, slots=4096)
    cached.attn.n_tokens = 1
    for q, k, ident in ((4096, None, 4096), (None, 4096, 4096), (4096, 4096, None)):
        w[0].q_norm, w[0].k_norm, desc.ident_cos, desc.ident_sin = q, k, ident, ident
        for rc in (lib.dark_forward_hidden(C.byref(desc), 4096, None, None, 1, 46, 4096, 1 << 40, 4096, None),
                   lib.dark_forward_cached(C.byref(desc), C.byref(cached), 4096, 1 << 40, 4096, None)):
            assert rc == _hip.DARK_ERR_ARG and b"go together" in lib.dark_hip_last_error()


def test_workspace_bytes():
    """A function of the sizes alone: none for a short axis, parts of (O, m, l) for few rows over a long one."""
    lib = _hip.load()
    a = _hip.PagedAttentionArgs(kv=_kv(), n_tokens=3, n_heads=8, n_seqs=2, table_width=1 << 14, max_q=2, max_kv=64, scale=0.1)
    assert lib.dark_paged_attention_workspace_bytes(C.byref(a)) == 0
    a.max_kv = 100000
    n = lib.dark_paged_attention_workspace_bytes(C.byref(a))
    assert n > 0 and n >= 2 * 3 * 8 * (96 + 2) * 4


@pytest.mark.parametrize("dtype", [_hip.DARK_F32, _hip.DARK_BF16])
def test_workspace_does_not_grow_with_tokens_times_keys(dtype):
    """Long chunks fill the card by themselves: their keys are not cut (or into a bounded number of parts), and many single
    tokens beside one long sequence stay within 1 GiB."""
    lib = _hip.load()

    def need(seqs, new, keys, tokens=None, heads=32, kv_heads=8, dim=128):
        kv = _kv(dtype=dtype, n_kv_heads=kv_heads, head_dim=dim, slot_stride=dim, head_stride=16 * dim, page_stride=16 * kv_heads * dim)
        a = _hip.PagedAttentionArgs(kv=kv, n_tokens=tokens or seqs * new, n_heads=heads, n_seqs=seqs, table_width=-(-keys // 16),
                                    max_q=new, max_kv=keys, scale=0.1)
        return lib.dark_paged_attention_workspace_bytes(C.byref(a))

    for seqs, new, keys in ((1, 16384, 16384), (1, 32768, 32768), (8, 4096, 65536), (1, 131072, 131072), (4, 1024, 9216)):
        assert need(seqs, new, keys) == 0, (seqs, new, keys)
    for seqs, new, keys, tokens in ((128, 4096, 16384, 4096 + 127), (64, 40, 131072, 2560), (2, 300, 60300, 600), (1, 100, 1 << 20, 100),
                                    (1024, 1, 131072, 1024), (4096, 1, 1 << 20, 4096), (1 << 16, 4, 1 << 18, 1 << 18)):
        for heads, kv_heads, dim in ((32, 8, 128), (12, 12, 64), (8, 8, 96)):
            assert need(seqs, new, keys, tokens, heads, kv_heads, dim) <= (1 << 30) + 512, (seqs, new, keys, heads)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 8, 96)
    cache = torch.zeros(2, 16, 8, 96)
    with pytest.raises(RuntimeError, match="HIP device"):
        kv_cache.qk_norm_rope(q, q, None, None, None, None, None)
    with pytest.raises(RuntimeError, match="HIP device"):
        kv_cache.append_kv(q, q, cache, cache, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="HIP device"):
        kv_cache.paged_attention(q, cache, cache, torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32),
                                 torch.tensor([5], dtype=torch.int32), 1, 5)


def test_oracle_against_dense_attention():
    g = torch.Generator().manual_seed(1)
    B, n, H, Hk, D, page = 2, 21, 4, 2, 64, 8
    q, k, v = (torch.randn(B, n, h, D, generator=g, dtype=torch.float64) for h in (H, Hk, Hk))
    per = 3
    table = torch.randperm(B * per, generator=g).view(B, per)
    kc, vc = (torch.full((B * per, page, Hk, D), math.nan, dtype=torch.float64) for _ in range(2))
    slots = table[torch.arange(B).repeat_interleave(n), torch.arange(n).repeat(B) // page] * page + torch.arange(n).repeat(B) % page
    kc, vc = O.append(kc, k.view(B * n, Hk, D), slots), O.append(vc, v.view(B * n, Hk, D), slots)
    mask = torch.rand(B, n, generator=g) > 0.3
    mask[:, 0] = True
    for causal in (False, True):
        out, lse, _, _ = O.attention(q.view(B * n, H, D), kc, vc, table, [0, n, 2 * n], [n, n], key_mask=mask, causal=causal)
        s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(2, 2)) * D ** -0.5
        s = s.masked_fill(~mask[:, None, None], -math.inf)
        if causal:
            s = s.masked_fill(torch.ones(n, n).triu(1).bool(), -math.inf)
        want = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v.repeat_interleave(2, 2))
        torch.testing.assert_close(out.view(B, n, H, D), want, rtol=0, atol=1e-12)
        torch.testing.assert_close(lse.view(B, n, H), s.logsumexp(-1).transpose(1, 2), rtol=0, atol=1e-12)


# --------------------------------------------------------------------------- pages and windows
def test_pages_and_slots():
    c = kv_cache.PagedKVCache(2, 7, 16, 4, 64, torch.float32, "cpu")
    assert c.k(1).shape == (7, 16, 4, 64) and c.k(1).stride() == c.v(0).stride() and c.pages_for(0) == 0
    a, b = c.allocate(33), c.allocate(16)
    assert len(a) == 3 and len(b) == 1 and len(set(a + b)) == 4
    with pytest.raises(MemoryError):
        c.allocate(49)
    assert len(c.allocate(48)) == 3
    c.free(a)
    for bad in ([a[0]], [99], [b[0], b[0]]):
        with pytest.raises(ValueError, match="not held"):
            c.free(bad)
    table = torch.tensor([[5, -1], [2, 9]], dtype=torch.int32)
    seq, index = torch.tensor([0, 0, 0, 1, 1, 1, 1]), torch.tensor([0, 15, 16, 3, 17, 32, -1], dtype=torch.int32)
    assert c.slots(table, seq, index).tolist() == [80, 95, -1, 35, -1, -1, -1]
    assert c.slots(table, torch.tensor([2, -1, 1]), torch.tensor([0, 0, 0])).tolist() == [-1, -1, 32]    # no such sequence
    assert c.slots(table[:, :0], seq, index).tolist() == [-1] * 7 and c.slots(table[:0], seq, index).tolist() == [-1] * 7
    with pytest.raises(ValueError, match="power of two"):
        kv_cache.PagedKVCache(1, 1, 24, 1, 64, torch.float32, "cpu")


def test_window_cache_schedule(monkeypatch):
    """Whole forwards every third time; a row that runs out of masks, or a change from outside, brings one forward."""
    from types import SimpleNamespace
    seen = []
    monkeypatch.setattr(kv_cache, "forward_cached", lambda m, c, ids, seq, index, *a, out=None, **k: (
        seen.append(ids.shape[0]), out if out is not None else torch.zeros(ids.shape[0], 64))[1])
    cfg = SimpleNamespace(num_hidden_layers=1, num_attention_heads=1, head_dim=64)
    model = SimpleNamespace(config=cfg, device=torch.device("cpu"), packed=lambda: SimpleNamespace(dtype=torch.float32))
    x = torch.full((2, 20), 9)
    x[0, 5:9], x[1, 0:7] = 6, 6
    wc = kv_cache.WindowCache(model, 2, 20, None, None, 3)
    st = SimpleNamespace(hidden=torch.zeros(40, 64), rows_valid=True)
    for k in (1, 1, 1):
        wc.forward(st, x, 6)
        wc.committed(k)
    assert seen == [40, 12, 12] and not st.rows_valid and wc.min_masked == 1
    assert wc.cu.tolist() == [0, 5, 12] and wc.max_q == 7
    assert wc.rows.tolist() == [4, 5, 6, 7, 8] + [20 + j for j in range(7)]
    wc.forward(st, x, 6)                       # the third since the whole one: whole again
    wc.committed(4)
    wc.forward(st, x, 6)
    assert seen[3:] == [40, 12]
    wc.committed(1)                            # row 0 had none left
    wc.forward(st, x, 6)
    wc.expire()
    wc.forward(st, x, 6)
    assert seen[5:] == [40, 40]
    assert kv_cache.WindowCache(model, 2, 20, None, None, 1).forward(st, x, 6) is None and seen[-1] == 40


def test_a_binding_of_another_version_is_refused(monkeypatch):
    import sys
    from types import SimpleNamespace

    import dark_amd
    assert kv_cache._ops().ABI_VERSION == _hip.ABI_VERSION
    for stale in (SimpleNamespace(ABI_VERSION=_hip.ABI_VERSION - 1), SimpleNamespace()):
        monkeypatch.setattr(kv_cache, "_bind", None)
        monkeypatch.setattr(dark_amd, "_bind", stale, raising=False)
        monkeypatch.setitem(sys.modules, "dark_amd._bind", stale)
        with pytest.raises(ImportError, match="ABI version"):
            kv_cache._ops()


@pytest.mark.parametrize("goal", ["all", "probes"])
def test_changed_flags_reach_every_object(goal):
    """A changed Makefile compiles everything anew: a library of objects with other flags would pass for a built one."""
    import glob
    import os
    import subprocess
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dark_amd", "csrc")
    plan = subprocess.run(["make", "-C", src, "-n", "-W", "Makefile", goal], check=True, capture_output=True, text=True).stdout
    for f in glob.glob(os.path.join(src, "*.hip")):
        assert f"-c {os.path.basename(f)} " in plan, f
    assert goal != "all" or "bind.cpp -o ../_bind.so" in plan


def test_pages_are_freed_all_or_none():
    c = kv_cache.PagedKVCache(1, 6, 16, 1, 64, torch.float32, "cpu")
    a = c.allocate(64)
    for bad in ([a[0], a[1], 99], [a[0], a[0]], [a[2], -1], [a[0], 5 - a[0] if 5 - a[0] not in a else 6]):
        with pytest.raises(ValueError, match="not held"):
            c.free(bad)
        with pytest.raises(MemoryError):
            c.allocate(48)                     # two pages are free, as before
    c.free(torch.tensor(a))
    assert sorted(c.allocate(96)) == list(range(6))


def test_a_cache_interval_that_is_not_served_is_refused():
    """The variable-length loop and the GPT-2 backbone say so instead of running without a cache."""
    from dark_amd import DreamConfig, DreamModel, synth
    from dark_amd.custom_gpt import DiffusionModel, GPT2DiffusionConfig
    dream = DreamModel(DreamConfig(vocab_size=512, hidden_size=192, intermediate_size=384, num_hidden_layers=1, num_attention_heads=2,
                                   num_key_value_heads=2, max_position_embeddings=64, mask_token_id=synth.MASK, pad_token_id=synth.END))
    gpt2 = DiffusionModel(GPT2DiffusionConfig(vocab_size=512, n_positions=64, n_embd=128, n_layer=1, n_head=2, mask_token_id=synth.MASK))
    ids = torch.full((1, 8), synth.MASK)
    for call in (dream.diffusion_generate, gpt2.diffusion_generate, gpt2.diffusion_generate_length):
        with pytest.raises(NotImplementedError, match="cache_interval"):
            call(ids, max_length=16, steps=2, alg="entropy", cache_interval=2)
        with pytest.raises(RuntimeError, match="HIP device"):          # none asked for: as without the argument
            call(ids, max_length=16, steps=2, alg="entropy", cache_interval=0, expand_token_id=5, eos_token_id=2)
    with pytest.raises(NotImplementedError, match="cache_interval"):
        dream.diffusion_generate_batch([ids[0]], max_length=16, cache_interval=4)


def test_no_source_is_compiled_with_packed_fp32():
    """hipcc makes v_pk_{add,mul,fma}_f32 of ordinary float code unless it is told not to, some forms of which have given wrong
    results on this card: every compile line of the library says so."""
    import os
    import subprocess
    src = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dark_amd", "csrc")
    plan = subprocess.run(["make", "-C", src, "-n", "-W", "Makefile", "all", "probes"], check=True, capture_output=True, text=True).stdout
    lines = [x for x in plan.splitlines() if ".hip -o" in x]
    assert len(lines) >= 13
    for x in lines:
        assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in x, x


@pytest.mark.parametrize("dtype", [_hip.DARK_F32, _hip.DARK_BF16])
def test_sizes_beyond_any_call_are_refused(dtype):
    """Products of the largest sizes that the fields hold: an error, no division by a product that wrapped round to 0."""
    lib = _hip.load()
    kv = _kv(dtype=dtype, n_kv_heads=4096, head_dim=64, slot_stride=64, head_stride=1024, page_stride=1024 * 4096)
    a = _hip.PagedAttentionArgs(kv=kv, q=4096, out=8192, block_table=4096, cu_q=4096, kv_len=4096, o_ts=64 * 4096, q_ts=64 * 4096, q_hs=64,
                                o_hs=64, n_tokens=1, n_heads=4096, n_seqs=1 << 30, table_width=64, table_stride=64, max_q=1 << 30, max_kv=1000,
                                scale=0.1)
    assert lib.dark_paged_attention_workspace_bytes(C.byref(a)) == 0
    _refused("dark_paged_attention", a, "too many rows")
    for big in (dict(max_q=1 << 30, n_seqs=1), dict(max_q=1, n_seqs=1 << 30), dict(max_q=1 << 20, n_seqs=1 << 20), dict(max_q=(1 << 31) - 200, n_seqs=(1 << 31) - 1)):
        for k, v in big.items():
            setattr(a, k, v)
        lib.dark_paged_attention_workspace_bytes(C.byref(a))
        assert lib.dark_paged_attention(C.byref(a), None) == _hip.DARK_ERR_ARG


def test_what_knows_nothing_of_the_cache_still_works():
    """The package imports beside a torch without a HIP runtime's bindings; a config object of the caller's own, without the
    field of the per-head norms, makes a model."""
    import os
    import subprocess
    import sys
    from types import SimpleNamespace

    from dark_amd import DreamConfig, DreamModel_length
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = "import torch; del torch._C._cuda_getCurrentRawStream; import dark_amd; dark_amd.DreamConfig()"
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root)
    cfg = DreamConfig(vocab_size=512, hidden_size=192, intermediate_size=384, num_hidden_layers=1, num_attention_heads=2,
                      num_key_value_heads=2, max_position_embeddings=64)
    other = SimpleNamespace(**cfg.__dict__, head_dim=cfg.head_dim, to_dict=cfg.to_dict)
    assert set(DreamModel_length(other).state_dict()) == set(DreamModel_length(cfg).state_dict())
