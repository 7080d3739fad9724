"""What the paged key / value cache's operators are measured on.

Three operators that stand around one cache: `qk_norm_rope` (RMS norm of every query and key head and the position
rotation), `append_kv` (rotation of new tokens and their placement in the pages) and `paged_attention` (attention of a
chunk of new tokens over what the pages hold).  Head counts and widths come from this repository's models (8 heads of 96
at d = 768, 12 of 64 for the GPT-2 backbone) and from the usual grouped layout (32 query heads on 8 key heads of 128).
"""
import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp32": 4}
_EPS = 1e-6
_THETA = 1000.0


def listed():
    own_heads = {"heads": 8, "kv_heads": 8, "dim": 96}        # this repository's denoiser
    gpt2 = {"heads": 12, "kv_heads": 12, "dim": 64}           # its GPT-2 backbone
    grouped = {"heads": 32, "kv_heads": 8, "dim": 128}        # the usual grouped layout
    return [
        # one token of one sequence: nothing but latency
        {"name": "norm_rope 1 token", "op": "norm_rope", "tokens": 1, "max_pos": 128, "dtype": "bf16", **own_heads},
        # every position of 512 windows of 46, as a denoise step's full forward has them
        {"name": "norm_rope 512 x 46", "op": "norm_rope", "tokens": 23552, "max_pos": 64, "dtype": "bf16", **own_heads},
        # a long prompt's chunk, far positions, in fp32
        {"name": "norm_rope 16383 fp32", "op": "norm_rope", "tokens": 16383, "max_pos": 65536, "dtype": "fp32", **grouped},
        # one new token for each of 200 sequences being served
        {"name": "append 200 x 1", "op": "append", "seqs": 200, "new": 1, "context": 8191, "page": 16, "norm": False,
         "max_pos": 16384, "dtype": "bf16", **grouped},
        # the 11 masked positions of 1024 windows of 46: what a denoise step between two refreshes writes
        {"name": "append 1024 x 11 of 46", "op": "append", "seqs": 1024, "new": 11, "context": 35, "page": 16,
         "norm": False, "max_pos": 64, "dtype": "bf16", **own_heads},
        # prompts of up to 4096 tokens being filled in, with the norms of queries and keys
        {"name": "append 8 x 4096 norm", "op": "append", "seqs": 8, "new": 4096, "context": 0, "page": 64, "norm": True,
         "max_pos": 8192, "dtype": "bf16", **grouped},
        # one token of one sequence over a short context: latency
        {"name": "attend 1 x 1 over 777", "op": "attend", "seqs": 1, "new": 1, "context": 776, "page": 16,
         "causal": True, "masked": False, "dtype": "bf16", **own_heads},
        # the denoise step between two refreshes: 11 masked positions see the whole window of 46, padding masked out
        {"name": "attend 1024 x 11 over 46", "op": "attend", "seqs": 1024, "new": 11, "context": 35, "page": 16,
         "causal": False, "masked": True, "dtype": "bf16", **own_heads},
        # serving: one token for each of 64 sequences of very different lengths
        {"name": "attend 64 x 1 over 16384", "op": "attend", "seqs": 64, "new": 1, "context": 16383, "page": 16,
         "causal": True, "masked": False, "dtype": "bf16", **grouped},
        # a block of 4 tokens over a very long context: few rows, a long axis
        {"name": "attend 2 x 4 over 131072", "op": "attend", "seqs": 2, "new": 4, "context": 131068, "page": 64,
         "causal": False, "masked": False, "dtype": "bf16", **grouped},
        # a long prompt in chunks: 1024 new tokens of each of 4 sequences over up to 16384 cached ones
        {"name": "attend 4 x 1024 over 17408", "op": "attend", "seqs": 4, "new": 1024, "context": 16384, "page": 64,
         "causal": True, "masked": False, "dtype": "bf16", **grouped},
        # fp32 models: the causal backbone's windows
        {"name": "attend 16 x 128 fp32", "op": "attend", "seqs": 16, "new": 128, "context": 384, "page": 32,
         "causal": True, "masked": True, "dtype": "fp32", **gpt2},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges, no dearer than the dearest listed one of its operator."""
    op = rng.choice(["norm_rope", "append", "attend", "attend"])
    heads, kv_heads, dim = rng.choice([(8, 8, 96), (12, 12, 64), (32, 8, 128), (16, 4, 128), (32, 32, 64), (28, 4, 128), (8, 1, 96)])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    most = max((work(c) for c in listed() if c["op"] == op), key=lambda w: w["bytes"])["bytes"]
    most_flops = max(work(c)["flops"] for c in listed() if c["op"] == op)
    while True:
        c = {"op": op}
        if op == "norm_rope":
            c.update(tokens=_log_int(rng, 1, 24000), max_pos=rng.choice([64, 1000, 65536]))
        else:
            c.update(seqs=_log_int(rng, 1, 1024), new=_log_int(rng, 1, 4096 if op == "append" else 1024),
                     context=_log_int(rng, 1, 131072) - 1, page=rng.choice([16, 32, 64, 128]))
            if op == "append":
                c.update(norm=rng.random() < 0.5, max_pos=131072 + 4096)
            else:
                c.update(causal=rng.random() < 0.6, masked=rng.random() < 0.3)
        c.update(dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim)
        w = work(c)
        # the padded length counts for the plain form; fp32 products cost about eight times as much
        padded = 1 if op == "norm_rope" else c["seqs"] * (c["new"] + c["context"]) * kv_heads * dim
        pairs = 1 if op != "attend" else c["seqs"] * c["new"] * (c["new"] + c["context"]) * heads
        if (w["bytes"] <= most and w["flops"] * (8 if dtype == "fp32" else 1) <= most_flops
                and padded <= (1 << 31 if op == "attend" else 1 << 28) and pairs <= 1 << 31):
            return c


def _lengths(c):
    """(new tokens, tokens in the cache with them) of every sequence: ragged as in a served batch, the longest as named.
    Plain values of the case, the same for every seed."""
    rng = random.Random("%d %d %d" % (c["seqs"], c["new"], c["context"]))
    new = [c["new"] if b == 0 or c["new"] < 16 else rng.randint(1, c["new"]) for b in range(c["seqs"])]
    ctx = [c["context"] if b == 0 or c["context"] < 64 else rng.randint(0, c["context"]) for b in range(c["seqs"])]
    return new, [n + x for n, x in zip(new, ctx)]


def _table(positions, dim, dev):
    freq = _THETA ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=dev) / dim)
    ang = torch.arange(positions, dtype=torch.float64, device=dev)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, H, Hk, D = _DT[c["dtype"]], c["heads"], c["kv_heads"], c["dim"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    st = {"case": c}
    if c["op"] == "norm_rope":
        T = c["tokens"]
        qkv = randn(T, H + 2 * Hk, D)                         # the projection's output, as the model has it
        st.update(q=qkv[:, :H], k=qkv[:, H:H + Hk], pos=torch.randint(0, c["max_pos"], (T,), generator=g, device=dev, dtype=torch.int32))
        st.update(qw=1 + 0.1 * torch.randn(D, generator=g, device=dev), kw=1 + 0.1 * torch.randn(D, generator=g, device=dev))
        st["cos"], st["sin"] = _table(c["max_pos"], D, dev)
        st.update(q_out=torch.empty(T, H, D, dtype=dt, device=dev), k_out=torch.empty(T, Hk, D, dtype=dt, device=dev))
        return st
    new, kv = _lengths(c)
    B, T, page = c["seqs"], sum(new), c["page"]
    per = [-(-n // page) for n in kv]
    # pages are handed out in any order, a few of them to nobody
    n_pages = sum(per) + 3
    ids = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    width = max(per)
    per_t = torch.tensor(per, device=dev)
    first = per_t.cumsum(0) - per_t
    j = torch.arange(width, device=dev)
    table = torch.where(j < per_t[:, None], ids[(first[:, None] + j).clamp(max=n_pages - 1)], -1).to(torch.int32).contiguous()
    new_t, kv_t = torch.tensor(new, device=dev), torch.tensor(kv, device=dev)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    cu[1:] = new_t.cumsum(0)
    seq = torch.repeat_interleave(torch.arange(B, device=dev), new_t)
    index = kv_t[seq] - new_t[seq] + torch.arange(T, device=dev) - cu[seq]      # a token's place in its sequence
    st.update(k_cache=randn(n_pages, page, Hk, D), v_cache=randn(n_pages, page, Hk, D))
    if c["op"] == "append":
        qkv = randn(T, H + 2 * Hk, D)
        st.update(q=qkv[:, :H], k=qkv[:, H:H + Hk], v=qkv[:, H + Hk:], pos=index.to(torch.int32))
        st["slots"] = table[seq, index // page].long() * page + index % page
        st["cos"], st["sin"] = _table(c["max_pos"], D, dev)
        st["q_out"] = torch.empty(T, H, D, dtype=dt, device=dev)
        st["qw"] = 1 + 0.1 * torch.randn(D, generator=g, device=dev) if c["norm"] else None
        st["kw"] = 1 + 0.1 * torch.randn(D, generator=g, device=dev) if c["norm"] else None
        return st
    st.update(q=randn(T, H, D), table=table, cu=cu, kv=kv_t.to(torch.int32), seq=seq, index=index, max_q=max(new), max_kv=max(kv))
    st["mask"] = None
    if c["masked"]:
        mask = torch.rand(B, max(kv), generator=g, device=dev) > 0.2
        mask[:, 0] = True
        st["mask"] = mask.to(torch.uint8)
    return st


def _rotated(x, w, cos, sin, pos):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def run(state):
    st, c = state, state["case"]
    if own:
        from dark_amd import kv_cache
        if c["op"] == "norm_rope":
            return kv_cache.qk_norm_rope(st["q"], st["k"], st["qw"], st["kw"], st["cos"], st["sin"], st["pos"], eps=_EPS,
                                         q_out=st["q_out"], k_out=st["k_out"])
        if c["op"] == "append":
            q = kv_cache.append_kv(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"], st["cos"], st["sin"], st["pos"],
                                   q=st["q"], q_out=st["q_out"], q_weight=st["qw"], k_weight=st["kw"], eps=_EPS)
            return q, st["k_cache"], st["v_cache"]
        return kv_cache.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu"], st["kv"], st["max_q"],
                                        st["max_kv"], key_mask=st["mask"], causal=c["causal"])
    dt = _DT[c["dtype"]]
    if c["op"] == "norm_rope":
        st["q_out"].copy_(_rotated(st["q"], st["qw"], st["cos"], st["sin"], st["pos"]))
        st["k_out"].copy_(_rotated(st["k"], st["kw"], st["cos"], st["sin"], st["pos"]))
        return st["q_out"], st["k_out"]
    Hk, D = c["kv_heads"], c["dim"]
    if c["op"] == "append":
        st["q_out"].copy_(_rotated(st["q"], st["qw"], st["cos"], st["sin"], st["pos"]))
        st["k_cache"].view(-1, Hk, D)[st["slots"]] = _rotated(st["k"], st["kw"], st["cos"], st["sin"], st["pos"]).to(dt)
        st["v_cache"].view(-1, Hk, D)[st["slots"]] = st["v"]
        return st["q_out"], st["k_cache"], st["v_cache"]
    # every sequence padded to the longest: [B, key heads, queries of the group, keys]
    B, G, M, N = c["seqs"], c["heads"] // Hk, st["max_q"], st["max_kv"]
    pages = st["table"].clamp(min=0).long()
    K = st["k_cache"][pages].flatten(1, 2)[:, :N].permute(0, 2, 3, 1).float().contiguous()
    V = st["v_cache"][pages].flatten(1, 2)[:, :N].permute(0, 2, 1, 3).float().contiguous()
    place = torch.arange(st["q"].shape[0], device="cuda") - st["cu"].long()[st["seq"]]
    Q = torch.zeros(B, M, Hk, G, D, device="cuda")
    Q[st["seq"], place] = st["q"].float().view(-1, Hk, G, D)
    S = torch.matmul(Q.permute(0, 2, 3, 1, 4).reshape(B, Hk, G * M, D) * (D ** -0.5), K).view(B, Hk, G, M, N)
    key = torch.arange(N, device="cuda")
    off = (key >= st["kv"][:, None])[:, None]                                   # [B, 1, N]
    if st["mask"] is not None:
        off = off | (st["mask"] == 0)[:, None]
    if c["causal"]:
        at = torch.zeros(B, M, dtype=torch.long, device="cuda")
        at[st["seq"], place] = st["index"]
        off = off | (key > at[:, :, None])
    S = S.masked_fill_(off[:, None, None], -math.inf)
    S = S.sub_(S.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    O = torch.matmul(S.view(B, Hk, G * M, N), V) / S.view(B, Hk, G * M, N).sum(-1, keepdim=True).clamp(min=1e-30)
    O = O.view(B, Hk, G, M, D).permute(0, 3, 1, 2, 4)[st["seq"], place]
    return O.reshape(-1, c["heads"], D).to(dt)


def work(case):
    c = case
    es, D, H, Hk = _ES[c["dtype"]], c["dim"], c["heads"], c["kv_heads"]
    if c["op"] == "norm_rope":
        T = c["tokens"]
        return {"bytes": 2 * T * (H + Hk) * D * es + 4 * T + min(T, c["max_pos"]) * D * 4 + 8 * D, "flops": 8 * T * (H + Hk) * D}
    new, kv = _lengths(c)
    T = sum(new)
    if c["op"] == "append":
        rows = min(max(kv), T)
        return {"bytes": 2 * T * (H + 2 * Hk) * D * es + 12 * T + rows * D * 4, "flops": (8 if c["norm"] else 4) * T * (H + Hk) * D}
    pairs = sum(n * m - (n * (n - 1) // 2 if c["causal"] else 0) for n, m in zip(new, kv))
    return {"bytes": 2 * T * H * D * es + 2 * sum(kv) * Hk * D * es + (sum(kv) if c["masked"] else 0) + 4 * sum(-(-m // c["page"]) for m in kv),
            "flops": 4 * D * H * pairs}


def exact(case, seed):
    """From the definitions, in 64 bits, sequence by sequence."""
    c, st = case, prepare(case, seed)

    def turn(x, w):
        x = x.double()
        if w is not None:
            x = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt()
        h = x.shape[-1] // 2
        c_, s_ = (t.double().index_select(0, st["pos"].long()).unsqueeze(1) for t in (st["cos"], st["sin"]))
        y = torch.empty_like(x)
        y[..., :h] = x[..., :h] * c_ - x[..., h:] * s_
        y[..., h:] = x[..., h:] * c_ + x[..., :h] * s_
        return y

    if c["op"] == "norm_rope":
        return turn(st["q"], st["qw"]), turn(st["k"], st["kw"])
    if c["op"] == "append":
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        page, slot = st["slots"] // c["page"], st["slots"] % c["page"]
        kc[page, slot] = turn(st["k"], st["kw"])
        vc[page, slot] = st["v"].double()
        return turn(st["q"], st["qw"]), kc, vc
    new, kv = _lengths(c)
    G, D = c["heads"] // c["kv_heads"], c["dim"]
    out = torch.zeros(sum(new), c["heads"], D, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        pages = st["table"][b, :-(-m // c["page"])].long()
        K = st["k_cache"].index_select(0, pages).flatten(0, 1)[:m].double().repeat_interleave(G, 1)     # [m, H, D]
        V = st["v_cache"].index_select(0, pages).flatten(0, 1)[:m].double().repeat_interleave(G, 1)
        s = torch.matmul(st["q"][at:at + n].double().transpose(0, 1), K.permute(1, 2, 0).contiguous()) / math.sqrt(D)
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen = seen.tril(m - n)
        if st["mask"] is not None:
            seen = seen & st["mask"][b, :m].bool()
        s = s.where(seen, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
        out[at:at + n] = torch.matmul((s - s.logsumexp(-1, keepdim=True)).exp(), V.transpose(0, 1).contiguous()).transpose(0, 1)
        at += n
    return out
