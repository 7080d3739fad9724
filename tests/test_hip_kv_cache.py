"""The paged key / value cache's operators (dark_amd/kv_cache.py) on the GPU against float64 (oracle/kv_cache_oracle.py).

Tolerances are bounds by arithmetic, with u = 2^-24 and, for bf16, h = 2^-8 (half a step, relative):
  norm + rotation: a lane adds 16 squares and 4 partial sums (20 u, halved by the root), mean, eps, root, division, weight,
    product and the rotation's sum: below 24 u of |first term| + |second term|; bf16 adds its one rounding, h |y|.
  attention: a score is a sum of D products, off by at most (D + 3) u z (z = scale * sum |q_i k_i|), the exponent and the
    hardware's exp2 by a few u (1 + |s|): a weight is off by a relative d = (D + 8) u (z + 1), a normalised one by 2 d;
    n keys added up in any order, and rescaled once a tile, add (2 n + 64) u: together (2 d + (2 n + 64) u) a with
    a = sum_j p_j |v_j|.  bf16 rounds every weight once (h a) and the output once (h |out|).
  lse: d + (2 n + 64) u + 4 u |lse|.
"""
import math

import pytest
import torch

from dark_amd import _hip, kv_cache
from oracle import kv_cache_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U, HALF = 2.0 ** -24, 2.0 ** -8


def tables(n, D, theta=1000.0):
    f = theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * f
    return ang.cos().float().contiguous(), ang.sin().float().contiguous()


def check_rows(got, y, a, dtype):
    tol = 24 * U * a + (HALF * y.abs() if dtype == torch.bfloat16 else 0) + 1e-37
    err = (got.cpu().double() - y).abs()
    assert bool((err <= tol).all()), (err / tol).max()


def check_attention(got, ref, n, D, dtype, lse=None):
    out, l, a, z = ref
    own = ~out.isnan().any(-1).any(-1) | False
    d = (D + 8) * U * (z + 1)
    tol = (2 * d[..., None] + (2 * n + 64) * U) * a + 1e-30
    if dtype == torch.bfloat16:
        tol = tol + HALF * a + HALF * out.abs()
    err = (got.cpu().double() - out).abs()
    assert bool((err <= tol)[own].all()), (err / tol)[own].max()
    if lse is not None:
        fin = own[:, None] & (l > -math.inf)
        e = (lse.cpu().double() - l).abs()
        assert bool((e <= d + (2 * n + 64) * U + 4 * U * l.abs())[fin].all())
        assert bool((lse.cpu()[own[:, None] & (l == -math.inf)] == -math.inf).all())


# --------------------------------------------------------------------------- norm + rotation
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,Hk,D", [(1, 8, 8, 96), (5, 12, 12, 64), (77, 32, 8, 128), (3, 7, 1, 96), (130, 1, 1, 128),
                                      (9, 40, 10, 64)])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False), (False, False)])
def test_qk_norm_rope(dtype, T, H, Hk, D, norm, rope):
    g = torch.Generator().manual_seed(T * 31 + H + D)
    qkv = (torch.randn(T, H + 2 * Hk, D, generator=g) * 2).to(dtype)
    qkv[0, 0] = 0                                             # a row of zeros: eps alone under the root
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)) if norm else None for _ in range(2))
    cos, sin = tables(300, D) if rope else (None, None)
    pos = torch.randint(-3, 310, (T,), generator=g, dtype=torch.int32) if rope else None   # clamped to the table
    d = lambda t: None if t is None else t.to(DEV)
    x = qkv.to(DEV)
    q, k = kv_cache.qk_norm_rope(x[:, :H], x[:, H:H + Hk], d(qw), d(kw), d(cos), d(sin), d(pos), eps=1e-6)
    for got, src, w in ((q, qkv[:, :H], qw), (k, qkv[:, H:H + Hk], kw)):
        check_rows(got, *O.norm_rope(src, w, cos, sin, pos, 1e-6), dtype)
    assert torch.equal(x.cpu(), qkv)
    # in place on the fused projection's output: the same bits, v untouched
    kv_cache.qk_norm_rope(x[:, :H], x[:, H:H + Hk], d(qw), d(kw), d(cos), d(sin), d(pos), eps=1e-6, q_out=x[:, :H],
                          k_out=x[:, H:H + Hk])
    assert torch.equal(x[:, :H], q) and torch.equal(x[:, H:H + Hk], k) and torch.equal(x[:, H + Hk:].cpu(), qkv[:, H + Hk:])


def test_qk_norm_rope_strides():
    """[H, T, D] memory order, one norm only, far positions, huge and tiny rows, and inputs the kernel cannot take as
    they are (a misaligned view, a last dimension with a stride)."""
    g = torch.Generator().manual_seed(3)
    T, H, D = 33, 4, 128
    cos, sin = tables(70000, D)
    pos = torch.randint(60000, 70000, (T,), generator=g, dtype=torch.int32)
    q = torch.randn(H, T, D, generator=g) * torch.logspace(-15, 15, T)[None, :, None]
    w = torch.randn(D, generator=g)
    ref = O.norm_rope(q.transpose(0, 1), w, cos, sin, pos, 1e-6)
    args = [t.to(DEV) for t in (cos, sin, pos)]
    qd = q.to(DEV).transpose(0, 1)
    a, b = kv_cache.qk_norm_rope(qd, qd, w.to(DEV), None, *args, eps=1e-6)
    check_rows(a, *ref, torch.float32)
    check_rows(b, *O.norm_rope(q.transpose(0, 1), None, cos, sin, pos, 1e-6), torch.float32)
    buf = torch.zeros(H * T * D + 1, device=DEV)
    off = buf[1:].view(T, H, D)
    off.copy_(qd)
    odd = torch.empty(T, H, 2 * D, device=DEV)[..., ::2]
    odd.copy_(qd)
    for x in (off, odd):
        y, _ = kv_cache.qk_norm_rope(x, x, w.to(DEV), None, *args, eps=1e-6)
        assert torch.equal(y, a)


@pytest.mark.parametrize("dtype,T,H,Hk,D", [(torch.bfloat16, 150001, 4, 3, 128), (torch.float32, 180000, 5, 1, 64), (torch.bfloat16, 470000, 2, 1, 96)])
@pytest.mark.parametrize("norm", [False, True])
def test_more_rows_than_the_caches_hold(dtype, T, H, Hk, D, norm):
    """Over 256 MB of rows, normed, rotated and stored; a sample of them checked."""
    assert T * (H + 2 * Hk) * D * dtype.itemsize > 256 << 20
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H + 2 * Hk, D, generator=g).to(dtype)
    w = 1 + 0.2 * torch.randn(D, generator=g)
    cos, sin = tables(1000, D)
    pos = torch.randint(0, 1000, (T,), generator=g, dtype=torch.int32)
    at = torch.cat([torch.tensor([0, T - 1]), torch.randint(0, T, (500,), generator=g)])
    d = lambda t: t.to(DEV)
    args = (d(w), d(w)) if norm else (None, None)
    xd = d(x)
    ref = {r: O.norm_rope(x[at, h], w if norm else None, cos, sin, pos[at], 1e-6) for r, h in (("q", slice(0, H)), ("k", slice(H, H + Hk)))}
    if T * (H + Hk) * D * dtype.itemsize > 256 << 20:
        q, k = kv_cache.qk_norm_rope(xd[:, :H], xd[:, H:H + Hk], *args, d(cos), d(sin), d(pos), eps=1e-6)
        check_rows(q[d(at)], *ref["q"], dtype)
        check_rows(k[d(at)], *ref["k"], dtype)
    n_pages = -(-T // 64)
    kc = torch.zeros(n_pages, 64, Hk, D, dtype=dtype, device=DEV)
    vc = torch.zeros_like(kc)
    slots = torch.randperm(n_pages * 64, generator=g)[:T]
    q = kv_cache.append_kv(xd[:, H:H + Hk], xd[:, H + Hk:], kc, vc, d(slots), d(cos), d(sin), d(pos), q=xd[:, :H], q_weight=args[0],
                           k_weight=args[1], eps=1e-6)
    check_rows(q[d(at)], *ref["q"], dtype)
    check_rows(kc.view(-1, Hk, D)[d(slots[at])], *ref["k"], dtype)
    assert torch.equal(vc.view(-1, Hk, D)[d(slots)], xd[:, H + Hk:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False), (False, False)])
def test_more_rows_than_the_caches_hold_of_each_kind(dtype, D, norm, rope):
    """Over 256 MB of rows of each type and width, with and without norm and rotation; a sample of them checked."""
    T, H, Hk = (257 << 20) // (3 * D * dtype.itemsize) + 5, 2, 1
    g = torch.Generator(device=DEV).manual_seed(D)
    x = torch.randn(T, H + Hk, D, generator=g, device=DEV).to(dtype)
    w = 1 + 0.2 * torch.randn(D, generator=g, device=DEV) if norm else None
    cos, sin = tables(1000, D) if rope else (None, None)
    pos = torch.randint(0, 1000, (T,), generator=g, device=DEV, dtype=torch.int32) if rope else None
    d = lambda t: None if t is None else t.to(DEV)
    q, k = kv_cache.qk_norm_rope(x[:, :H], x[:, H:], w, w, d(cos), d(sin), pos, eps=1e-6)
    if not norm and not rope:
        assert torch.equal(q, x[:, :H]) and torch.equal(k, x[:, H:])
    at = torch.cat([torch.tensor([0, T - 1]), torch.randint(0, T, (300,), generator=torch.Generator().manual_seed(1))])
    c = lambda t: None if t is None else t.cpu()
    for got, src in ((q, x[:, :H]), (k, x[:, H:])):
        check_rows(got[d(at)], *O.norm_rope(src[d(at)].cpu(), c(w), cos, sin, pos[d(at)].cpu() if rope else None, 1e-6), dtype)


# --------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,Hk,D,page", [(1, 8, 8, 96, 16), (53, 12, 12, 64, 1), (200, 32, 8, 128, 64), (7, 3, 1, 96, 4096)])
@pytest.mark.parametrize("norm,heads_first", [(False, False), (True, True)])
def test_append_kv(dtype, T, H, Hk, D, page, norm, heads_first):
    g = torch.Generator().manual_seed(T + D + page)
    n_pages = T // page + 2
    shape = (n_pages, Hk, page, D) if heads_first else (n_pages, page, Hk, D)
    view = (lambda t: t.transpose(1, 2)) if heads_first else (lambda t: t)
    kc, vc = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
    qkv = torch.randn(T, H + 2 * Hk, D, generator=g).to(dtype)
    qkv[0, H + Hk, 0] = math.nan                              # values are carried, not computed
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)) if norm else None for _ in range(2))
    cos, sin = tables(500, D)
    pos = torch.randint(0, 500, (T,), generator=g, dtype=torch.int32)
    slots = torch.randperm(n_pages * page, generator=g)[:T]
    slots[T // 2] = -1                                        # not stored
    if T > 9:
        slots[3], slots[9] = n_pages * page, 1 << 40
    d = lambda t: None if t is None else t.to(DEV)
    kd, vd, x = kc.to(DEV), vc.to(DEV), qkv.to(DEV)
    q = kv_cache.append_kv(x[:, H:H + Hk], x[:, H + Hk:], view(kd), view(vd), d(slots), d(cos), d(sin), d(pos), q=x[:, :H],
                           q_weight=d(qw), k_weight=d(kw))
    check_rows(q, *O.norm_rope(qkv[:, :H], qw, cos, sin, pos, 1e-6), dtype)
    y, a = O.norm_rope(qkv[:, H:H + Hk], kw, cos, sin, pos, 1e-6)
    check_rows(view(kd), O.append(view(kc).double(), y, slots), O.append(torch.zeros_like(view(kc)).double(), a, slots), dtype)
    want = O.append(view(vc), qkv[:, H + Hk:], slots)
    assert torch.equal(view(vd).cpu().nan_to_num(7.0), want.nan_to_num(7.0)) and int(view(vd).isnan().sum()) == int(want.isnan().sum())
    # what is not stored stays bit for bit
    rest = torch.ones(n_pages * page, dtype=torch.bool)
    rest[slots[(slots >= 0) & (slots < n_pages * page)]] = False
    assert torch.equal(view(kd).cpu().reshape(-1, Hk, D)[rest], view(kc).reshape(-1, Hk, D)[rest])
    # without q: the same cache; without a rotation: the keys as they are
    k2, v2 = kc.to(DEV), vc.to(DEV)
    assert kv_cache.append_kv(x[:, H:H + Hk], x[:, H + Hk:], view(k2), view(v2), d(slots), d(cos), d(sin), d(pos), k_weight=d(kw)) is None
    assert torch.equal(k2, kd)
    kv_cache.append_kv(x[:, H:H + Hk], x[:, H + Hk:], view(k2), view(v2), d(slots))
    assert torch.equal(view(k2).cpu(), O.append(view(kc), qkv[:, H:H + Hk], slots))


def bits(t):
    return t.contiguous().view(torch.int16 if t.dtype == torch.bfloat16 else torch.int32).cpu()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,H,Hk,D", [(5, 8, 2, 96), (40, 3, 3, 64), (3, 32, 8, 128)])
def test_rows_without_a_rotation(dtype, T, H, Hk, D):
    """No tables: infinities, NaN and zeros of either sign stay in their own elements.  Without a norm too the rows are
    carried bit for bit; a norm on one side leaves the other side's so."""
    g = torch.Generator().manual_seed(D)
    x = torch.randn(T, H + 2 * Hk, D, generator=g).to(dtype)
    h = D // 2
    for r in (0, H):                                          # a query's and a key's head
        x[0, r, 3], x[0, r, h + 7] = math.inf, -math.inf      # one half each
        x[1, r, h + 1], x[1, r, 5] = math.nan, -0.0
        x[2, r] = -0.0
        x[2, r, :4] = 2.0 ** -130                             # denormal
    xd, w = x.to(DEV), 1 + 0.2 * torch.randn(D, generator=g)
    q, k = kv_cache.qk_norm_rope(xd[:, :H], xd[:, H:H + Hk], None, None, None, None, None)
    assert torch.equal(bits(q), bits(x[:, :H])) and torch.equal(bits(k), bits(x[:, H:H + Hk]))
    q, k = kv_cache.qk_norm_rope(xd[:, :H], xd[:, H:H + Hk], w.to(DEV), None, None, None, None)
    assert torch.equal(bits(k), bits(x[:, H:H + Hk]))
    check_rows(q[2:], *O.norm_rope(x[2:, :H], w, None, None, None, 1e-6), dtype)
    n = q[1, 0].cpu()                                         # (a NaN under the root reaches its own row only)
    assert bool(n.isnan().all()) and not bool(q[1, 1:].isnan().any())
    kc, vc = (torch.zeros(2, 64, Hk, D, dtype=dtype, device=DEV) for _ in range(2))
    slots = torch.randperm(128, generator=g)[:T].to(DEV)
    q = kv_cache.append_kv(xd[:, H:H + Hk], xd[:, H + Hk:], kc, vc, slots, q=xd[:, :H])
    assert torch.equal(bits(q), bits(x[:, :H]))
    assert torch.equal(bits(kc.view(128, Hk, D)[slots]), bits(x[:, H:H + Hk]))
    assert torch.equal(bits(vc.view(128, Hk, D)[slots]), bits(x[:, H + Hk:]))


# --------------------------------------------------------------------------- attention
def paged(q_lens, kv_lens, H, Hk, D, page, dtype, seed=0, spare=3, lead=0, tail=0, heads_first=False, fill=math.nan):
    """A batch over shuffled pages; every slot no sequence uses holds `fill`."""
    g = torch.Generator().manual_seed(seed + sum(kv_lens) + D)
    B, per = len(q_lens), [-(-n // page) for n in kv_lens]
    n_pages = sum(per) + spare
    ids = torch.randperm(n_pages, generator=g).int()
    table = torch.full((B, max(per + [1])), -7, dtype=torch.int32)
    kc = torch.full((n_pages, page, Hk, D), fill).to(dtype)
    vc = kc.clone()
    at = 0
    for b in range(B):
        table[b, :per[b]] = ids[at:at + per[b]]
        at += per[b]
        for j in range(kv_lens[b]):
            kc[table[b, j // page], j % page] = torch.randn(Hk, D, generator=g).to(dtype)
            vc[table[b, j // page], j % page] = torch.randn(Hk, D, generator=g).to(dtype)
    T = lead + sum(q_lens) + tail
    cu = torch.tensor([lead + sum(q_lens[:b]) for b in range(B + 1)], dtype=torch.int32)
    q = (torch.randn(T, H, D, generator=g) * 1.5).to(dtype)
    return dict(q=q, k=kc, v=vc, table=table, cu=cu, kv=torch.tensor(kv_lens, dtype=torch.int32), max_q=max(q_lens + [0]),
                max_kv=max(kv_lens + [0]), heads_first=heads_first)


def run_paged(p, **kw):
    if p["heads_first"]:
        k, v = (t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (p["k"], p["v"]))
    else:
        k, v = p["k"].to(DEV), p["v"].to(DEV)
    kw = {n: (t.to(DEV) if isinstance(t, torch.Tensor) else t) for n, t in kw.items()}
    return kv_cache.paged_attention(kw.pop("q", p["q"].to(DEV)), k, v, p["table"].to(DEV), p["cu"].to(DEV), p["kv"].to(DEV),
                                    p["max_q"], p["max_kv"], **kw)


SHAPES = [  # q_lens, kv_lens, H, Hk, D, page
    ([1], [1], 8, 8, 96, 16),
    ([1, 1, 1], [0, 33, 64], 8, 8, 96, 16),                       # nothing cached, one key past a tile, whole tiles
    ([11, 0, 11, 3], [46, 46, 11, 3], 8, 8, 96, 16),              # a denoise step; a sequence without new tokens
    ([1, 5, 2], [130, 257, 5], 32, 8, 128, 64),
    ([17, 64, 1], [17, 200, 95], 12, 12, 64, 32),
    ([70, 33], [333, 33], 4, 1, 128, 128),                        # one key head; pages longer than a tile
    ([150], [400], 6, 3, 64, 1),                                  # pages of one slot
    ([3, 2], [40, 9], 28, 4, 128, 8),
    ([129, 257], [129, 700], 2, 2, 96, 16),
    ([46, 30], [46, 100], 8, 8, 96, 16),                          # whole windows of a denoise step
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_paged_attention(dtype, causal, shape):
    q_lens, kv_lens, H, Hk, D, page = SHAPES[shape]
    p = paged(q_lens, kv_lens, H, Hk, D, page, dtype, seed=shape, heads_first=shape % 2 == 1)
    out, lse = run_paged(p, causal=causal, return_lse=True)
    check_attention(out, O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], causal=causal), max(kv_lens), D, dtype, lse)
    again, _ = run_paged(p, causal=causal, return_lse=True)
    assert torch.equal(again, out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("q_lens,H,Hk,D", [([11, 40, 1, 2], 4, 2, 96), ([1, 1, 1, 2], 8, 8, 64), ([200, 130, 7, 2], 2, 1, 128)])
def test_masks_and_what_lies_in_masked_places(dtype, causal, q_lens, H, Hk, D):
    """Key masks with NaN and infinities in what they hide, a sequence masked whole, block-table entries that name no
    page, given places, a scale of its own, tokens before and behind the batch left as they were."""
    kv_lens = [200, 77, 33, 2]
    p = paged(q_lens, kv_lens, H, Hk, D, 16, dtype, seed=5, lead=2, tail=3)
    g = torch.Generator().manual_seed(9)
    mask = torch.rand(4, 210, generator=g) > 0.4
    mask[2] = False                                               # nothing left for this sequence
    mask[0, 64:96] = False                                        # a whole tile
    for b in range(4):
        for j in range(kv_lens[b]):
            if not mask[b, j]:
                pg, s = p["table"][b, j // 16], j % 16
                p["k"][pg, s], p["v"][pg, s] = math.nan, math.inf
    p["table"][0, 1], p["table"][1, 2] = -1, p["k"].shape[0]      # no such pages: their keys are out
    index = torch.cat([torch.randint(-2, n + 3, (m,), generator=g) for n, m in zip([0] + kv_lens + [0], [2] + q_lens + [3])]).int()
    kw = dict(causal=causal, q_index=index, key_mask=mask, scale=0.3)
    out = torch.full(p["q"].shape, 5.0, dtype=dtype, device=DEV)
    got, lse = run_paged(p, out=out, return_lse=True, **kw)
    ref = O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], **kw)
    check_attention(got, ref, 200, D, dtype, lse)
    assert bool((got[:2] == 5).all()) and bool((got[-3:] == 5).all())
    at = int(p["cu"][2])
    assert bool((got[at:at + q_lens[2]] == 0).all())
    assert torch.equal(run_paged(p, **{**kw, "key_mask": mask.to(torch.uint8)})[2:-3], got[2:-3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("n,q_len,H,Hk", [(150, 150, 2, 2), (45, 6, 8, 2), (300, 300, 4, 1)])
def test_infinities_and_nan_behind_a_causal_token(dtype, D, n, q_len, H, Hk):
    """Infinities and NaN in a later token's keys and values reach only the tokens that see it, element by element."""
    p = paged([q_len], [n], H, Hk, D, 16, dtype, seed=2)
    clean = O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], causal=True)
    put = lambda j, h, i, x, t="v": p[t].__setitem__((int(p["table"][0, j // 16]), j % 16, h, i), x)
    j0 = n - q_len + q_len // 2
    put(j0, 0, 3, math.nan)
    put(j0 + 1, 0, 5, math.inf)
    put(j0 + 1, 0, 7, -math.inf)
    put(j0 + 2, 0, 5, -math.inf)                                  # +inf and -inf together: NaN
    put(n - 1, 0, 9, math.nan, "k")                               # the last key: only the last token sees it
    got = run_paged(p, causal=True).cpu()
    G, i0 = H // Hk, q_len // 2
    last = q_len - 1
    check_attention(got[:i0], tuple(x[:i0] for x in clean), n, D, dtype)
    assert bool(got[last, :G].isnan().all()), "the last token of the head group that holds the NaN key"
    check_attention(got[:last, G:], tuple(x[:last, G:] for x in clean), n, D, dtype)    # the other key heads
    sel = [i for i in range(D) if i not in (3, 5, 7)]
    mid = slice(i0, last)
    check_attention(got[mid][:, :G, sel], (clean[0][mid][:, :G, sel], clean[1][mid][:, :G], clean[2][mid][:, :G, sel], clean[3][mid][:, :G]), n, D, dtype)
    if last > i0:
        assert bool(got[mid][:, :G, 3].isnan().all())
    if last > i0 + 1:
        assert bool((got[i0 + 1:last][:, :G, 7] == -math.inf).all()) and bool((got[i0 + 1, :G, 5] == math.inf).all())
    if last > i0 + 2:
        assert bool(got[i0 + 2:last][:, :G, 5].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_lens,kv_lens,H,Hk,D,page", [([1], [5000], 8, 8, 96, 16), ([1, 1, 4], [3001, 1, 700], 8, 2, 128, 64),
                                                       ([4], [2500], 32, 8, 128, 32), ([40], [2111], 4, 4, 64, 16)])
@pytest.mark.parametrize("causal", [False, True])
def test_long_key_axis(dtype, q_lens, kv_lens, H, Hk, D, page, causal):
    """Few rows over many keys: the axis is split over workgroups and joined; the same bits every time."""
    p = paged(q_lens, kv_lens, H, Hk, D, page, dtype, seed=1)
    out, lse = run_paged(p, causal=causal, return_lse=True)
    check_attention(out, O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], causal=causal), max(kv_lens), D, dtype, lse)
    for _ in range(3):
        assert torch.equal(run_paged(p, causal=causal), out)


@pytest.mark.parametrize("q_lens,kv_lens,H,Hk,D,page", [([1, 1, 4], [3001, 1, 700], 8, 2, 128, 64), ([1, 0, 2], [5000, 3, 0], 8, 4, 96, 16),
                                                       ([1, 3], [2111, 65], 4, 4, 64, 16), ([9, 31], [3000, 40], 8, 2, 128, 16),
                                                       ([20, 1], [300, 2000], 4, 4, 64, 32)])
@pytest.mark.parametrize("causal", [False, True])
def test_tables_wider_than_the_caches_hold(q_lens, kv_lens, H, Hk, D, page, causal):
    """Tables with room for over 256 MB of keys (their rows are then read past the caches), of which the sequences have a few."""
    p = paged(q_lens, kv_lens, H, Hk, D, page, torch.bfloat16, seed=6)
    p["max_kv"] = 140000
    assert len(q_lens) * 140000 * Hk * D * 4 > 256 << 20
    p["table"] = torch.cat([p["table"], torch.full((len(q_lens), -(-140000 // page) - p["table"].shape[1]), -3, dtype=torch.int32)], 1)
    out, lse = run_paged(p, causal=causal, return_lse=True)
    check_attention(out, O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], causal=causal), max(kv_lens), D, torch.bfloat16, lse)
    assert torch.equal(run_paged(p, causal=causal), out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [-0.3, 0.0])
@pytest.mark.parametrize("q_lens,kv_lens,H,Hk,D", [([150, 9], [200, 41], 4, 2, 96), ([3, 1], [70, 400], 8, 2, 128)])
def test_scales_that_are_not_positive(dtype, scale, q_lens, kv_lens, H, Hk, D):
    """The smallest product becomes the largest score; all keys that are seen count alike.  Left-out keys stay out."""
    p = paged(q_lens, kv_lens, H, Hk, D, 16, dtype, seed=3)
    mask = torch.rand(2, 400, generator=torch.Generator().manual_seed(1)) > 0.3
    for causal in (False, True):
        kw = dict(scale=scale, key_mask=mask, causal=causal)
        out, lse = run_paged(p, return_lse=True, **kw)
        check_attention(out, O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], **kw), max(kv_lens), D, dtype, lse)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("n,max_q", [(24, 1000), (64, 400), (65, 400), (2, 9000)])
def test_chunks_of_sequences_of_very_different_lengths(n, max_q, causal):
    """The longest sequence's rows begin first wherever it stands; equal lengths, empty sequences, more room than any has."""
    kv_lens = [(37 * i) % 90 for i in range(n)]
    kv_lens[n // 2], kv_lens[-1], kv_lens[0] = 1100, 1100, 0
    q_lens = [min(k, (5 * i) % 7) for i, k in enumerate(kv_lens)]
    q_lens[n // 2] = 70
    p = paged(q_lens, kv_lens, 16, 8, 64, 32, torch.bfloat16, seed=12, lead=1)
    p["max_q"], p["max_kv"] = max_q, 1200
    out, lse = run_paged(p, causal=causal, return_lse=True)
    check_attention(out, O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], causal=causal), 1100, 64, torch.bfloat16, lse)
    assert torch.equal(run_paged(p, causal=causal)[1:], out[1:])


@pytest.mark.parametrize("dtype,n,max_q,max_kv,H,Hk,D,page", [
    (torch.bfloat16, (1 << 21) + 77, 1, 100, 8, 8, 64, 128),       # a wave a problem
    (torch.bfloat16, (1 << 17) + 5, 4, 9000, 32, 8, 64, 4096),     # parts of the keys, and 2^24 rows to join one by one
    (torch.bfloat16, (1 << 17) + 5, 4, 1500, 32, 8, 96, 512),      # ... four by four
    (torch.bfloat16, (1 << 17) + 5, 600, 700, 8, 8, 96, 256),      # row tiles
    (torch.float32, (1 << 17) + 5, 600, 1000, 8, 8, 64, 256),      # 2^32 threads and more
    (torch.float32, (1 << 17) + 5, 600, 1000, 8, 8, 128, 256),
])
def test_more_workgroups_than_a_launch_holds(dtype, n, max_q, max_kv, H, Hk, D, page):
    """Room for so many sequences that one call takes several launches; a few of them have tokens, the first and last too."""
    assert n * Hk * max(1, max_q * (H // Hk) // 128) >= 1 << 20
    q_lens = [min(max_q, x) for x in (1, 3, 130, 2, 1)]
    kv_lens = [min(max_kv, x) for x in (max_kv, 40, 1030, 77, max_kv - 3)]
    p = paged(q_lens, kv_lens, H, Hk, D, page, dtype, seed=3, tail=2)
    ref = O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], causal=True)
    at = torch.tensor([0, 1, n // 2 + 3, n - 2, n - 1])
    new = torch.zeros(n, dtype=torch.int32)
    new[at] = torch.tensor(q_lens, dtype=torch.int32)
    kv = torch.zeros(n, dtype=torch.int32)
    kv[at] = p["kv"]
    table = torch.full((n, p["table"].shape[1]), -1, dtype=torch.int32)
    table[at] = p["table"]
    p.update(table=table, kv=kv, cu=torch.cat([torch.zeros(1, dtype=torch.int32), new.cumsum(0).int()]), max_q=max_q, max_kv=max_kv)
    out, lse = run_paged(p, causal=True, out=torch.full(p["q"].shape, 5.0, dtype=dtype, device=DEV), return_lse=True)
    check_attention(out, ref, max_kv, D, dtype, lse)
    assert bool((out[-2:] == 5).all())


F32, BF16 = torch.float32, torch.bfloat16
PLANS = [  # dtype, sequences, new tokens, keys, room for (new tokens, keys), H, Hk, D
    (F32, 9, 40, 1100, (2000, 1200), 8, 8, 128),         # 8192 problems and more: a wave each, 32 rows
    (F32, 9, 23, 700, (1000, 900), 16, 4, 96),
    (F32, 10, 20, 200, (160, 256), 12, 12, 64),          # ... of few keys: 16 rows
    (F32, 10, 20, 200, (160, 250), 4, 4, 128),
    (F32, 3, 40, 500, (40, 500), 8, 8, 64),              # four waves a problem, a key head's tiles on one XCD
    (F32, 70, 20, 290, (20, 300), 4, 2, 96),             # all of a sequence's
    (F32, 70, 3, 100, (9, 128), 12, 12, 64),             # four problems a workgroup, a sequence's on one XCD
    (F32, 8, 100, 2900, (100, 3000), 8, 8, 64),          # many row tiles whose keys are cut
    (F32, 16, 40, 2500, (80, 2600), 16, 8, 128),
    (F32, 40, 1, 2900, (1, 3000), 32, 8, 128),           # single tokens in parts of 512 keys
    (BF16, 40, 1, 2900, (1, 3000), 32, 8, 128),
    (F32, 70, 1, 2900, (1, 3000), 8, 8, 96),             # ... of 1024
    (BF16, 70, 1, 2900, (1, 3000), 8, 8, 96),
    (BF16, 70, 2, 2900, (2, 3000), 24, 8, 64),
    (F32, 70, 1, 9900, (1, 10000), 12, 12, 64),          # more than eight parts
    (BF16, 70, 1, 9900, (1, 10000), 32, 8, 128),
    (BF16, 130, 11, 46, (11, 46), 8, 8, 96),             # a denoise step between two whole ones
    (BF16, 130, 46, 46, (46, 46), 2, 2, 96),             # a whole one
    (BF16, 66, 3, 120, (3, 128), 32, 8, 128),
    (BF16, 70, 3, 200, (3, 250), 12, 12, 64),            # four waves a problem, keys that stay in the caches
    (BF16, 40, 200, 1500, (200, 1500), 4, 4, 64),        # row tiles in parts
]


@pytest.mark.parametrize("plan", range(len(PLANS)))
@pytest.mark.parametrize("causal", [False, True])
def test_large_batches(plan, causal):
    """The divisions of work that many sequences, or room for long ones, bring: most sequences short, one whole, some without
    tokens or keys.  Causal calls are masked as well."""
    dtype, n, new, keys, room, H, Hk, D = PLANS[plan]
    kv_lens = [(23 * i) % min(60, keys) for i in range(n)]
    kv_lens[n // 3], kv_lens[-1], kv_lens[1] = keys, keys // 2, min(keys, 1 + keys * 2 // 3)
    q_lens = [1 if new == 1 else min(kv_lens[i], (5 * i) % min(new + 1, 8)) for i in range(n)]
    q_lens[n // 3], q_lens[-1] = new, min(new, 5)
    p = paged(q_lens, kv_lens, H, Hk, D, 32, dtype, seed=plan, lead=1, tail=1)
    p["max_q"], p["max_kv"] = room
    mask = torch.rand(n, room[1], generator=torch.Generator().manual_seed(plan)) > 0.2 if causal else None
    kw = dict(causal=causal, key_mask=mask)
    out, lse = run_paged(p, out=torch.full(p["q"].shape, 5.0, dtype=dtype, device=DEV), return_lse=True, **kw)
    check_attention(out[1:-1], tuple(x[1:-1] for x in O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], **kw)), keys, D, dtype, lse[1:-1])
    assert bool((out[:1] == 5).all()) and bool((out[-1:] == 5).all())
    assert torch.equal(run_paged(p, **kw)[1:-1], out[1:-1])


def test_views_strides_and_scores_far_apart():
    """q and out as views of larger tensors; scores so far apart that one key takes the whole row."""
    p = paged([9, 2], [100, 50], 8, 8, 96, 16, torch.float32, seed=8)
    p["q"] *= 40
    wide = torch.zeros(11, 24, 96, device=DEV)
    wide[:, 8:16] = p["q"].to(DEV)
    o = torch.full((8, 11, 96), 3.0, device=DEV).transpose(0, 1)
    got = run_paged(p, q=wide[:, 8:16], out=o)
    assert got is o
    check_attention(got, O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"]), 100, 96, torch.float32)
    buf = torch.zeros(p["q"].numel() + 1, device=DEV)
    odd = buf[1:].view(11, 8, 96)
    odd.copy_(p["q"])
    assert torch.equal(run_paged(p, q=odd), got)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements, the sequence in its last pages."""
    page, Hk, D = 64, 8, 128
    n_pages = (1 << 31) // (page * Hk * D) + 40
    kc = torch.zeros(n_pages, page, Hk, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    assert kc.numel() > 1 << 31
    T = 100
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(T, 3 * Hk, D, generator=g).bfloat16()
    pages = torch.tensor([[n_pages - 1, n_pages - 7]], dtype=torch.int32)
    idx = torch.arange(T)
    slots = (pages[0, idx // page].long() * page + idx % page).to(DEV)
    x = qkv.to(DEV)
    kv_cache.append_kv(x[:, Hk:2 * Hk], x[:, 2 * Hk:], kc, vc, slots)
    out = kv_cache.paged_attention(x[:, :Hk], kc, vc, pages.to(DEV), torch.tensor([0, T], dtype=torch.int32, device=DEV),
                                   torch.tensor([T], dtype=torch.int32, device=DEV), T, T, causal=True)
    small = torch.stack([qkv[:64, Hk:2 * Hk], torch.cat([qkv[64:, Hk:2 * Hk], torch.zeros(28, Hk, D).bfloat16()])])
    smallv = torch.stack([qkv[:64, 2 * Hk:], torch.cat([qkv[64:, 2 * Hk:], torch.zeros(28, Hk, D).bfloat16()])])
    ref = O.attention(qkv[:, :Hk], small, smallv, torch.tensor([[0, 1]]), [0, T], [T], causal=True)
    check_attention(out, ref, T, D, torch.bfloat16)
    last = tuple(r[-1:] for r in ref)      # a single token's stream of the same keys, with room for more as well
    for room in (T, 2000, 200000):
        wide = torch.cat([pages, torch.full((1, -(-room // page) - 2 if room > T else 0), -1, dtype=torch.int32)], 1).to(DEV)
        one = kv_cache.paged_attention(x[T - 1:, :Hk], kc, vc, wide, torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                                       torch.tensor([T], dtype=torch.int32, device=DEV), 1, room, causal=True)
        check_attention(one, last, T, D, torch.bfloat16)


# --------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prefill_then_tokens(dtype):
    """A prompt in two chunks, then single tokens, all with norms and rotation, against the whole computed at once."""
    g = torch.Generator().manual_seed(4)
    B, H, Hk, D, page, n = 3, 8, 2, 96, 16, 61
    x = torch.randn(B, n, H + 2 * Hk, D, generator=g).to(dtype)
    qw, kw = 1 + 0.1 * torch.randn(D, generator=g), 1 + 0.1 * torch.randn(D, generator=g)
    cos, sin = tables(64, D)
    per = -(-n // page)
    table = torch.randperm(B * per, generator=g).view(B, per).int()
    kc = torch.full((B * per, page, Hk, D), math.nan, dtype=dtype, device=DEV)
    vc = kc.clone()
    td, cd, sd, qd, kd = (t.to(DEV) for t in (table, cos, sin, qw, kw))
    got = torch.empty(B, n, H, D, dtype=dtype)
    at = 0
    for step in (40, 17, 1, 1, 2):
        idx = torch.arange(at, at + step).repeat(B)
        seq = torch.arange(B).repeat_interleave(step)
        slots = table[seq, idx // page].long() * page + idx % page
        c = x[:, at:at + step].reshape(B * step, H + 2 * Hk, D).to(DEV)
        q = kv_cache.append_kv(c[:, H:H + Hk], c[:, H + Hk:], kc, vc, slots.to(DEV), cd, sd, idx.int().to(DEV), q=c[:, :H],
                               q_weight=qd, k_weight=kd)
        o = kv_cache.paged_attention(q, kc, vc, td, torch.arange(0, B * step + 1, step, dtype=torch.int32, device=DEV),
                                     torch.full((B,), at + step, dtype=torch.int32, device=DEV), step, at + step, causal=True)
        got[:, at:at + step] = o.cpu().view(B, step, H, D)
        at += step
    # the oracle takes the operands as they were stored: rounded to the cache's type
    pos = torch.arange(n).repeat(B)
    rows = x.view(B * n, H + 2 * Hk, D)
    q = O.norm_rope(rows[:, :H], qw, cos, sin, pos, 1e-6)[0].to(dtype)
    k = kc[table.view(-1).long().to(DEV)].cpu().view(B, per * page, Hk, D)[:, :n].reshape(B * n, Hk, D)
    check_rows(k, *O.norm_rope(rows[:, H:H + Hk], kw, cos, sin, pos, 1e-6), dtype)
    pad = lambda t: torch.cat([t.view(B, n, Hk, D), torch.zeros(B, per * page - n, Hk, D, dtype=dtype)], 1).view(B * per, page, Hk, D)
    ref = O.attention(q, pad(k), pad(rows[:, H + Hk:].contiguous()), torch.arange(B * per).view(B, per), [0, n, 2 * n, 3 * n], [n] * 3, causal=True)
    out, _, a, z = ref
    # q's own rounding (its float64 value may sit next to a border): half a step of z in the score
    step = (HALF if dtype == torch.bfloat16 else 24 * U)
    tol = (2 * ((D + 8) * U * (z + 1) + 2 * step * z)[..., None] + (2 * n + 64) * U) * a
    if dtype == torch.bfloat16:
        tol = tol + HALF * a + HALF * out.abs()
    assert bool(((got.view(B * n, H, D).double() - out).abs() <= tol).all())


def test_other_stream_and_graph():
    """The calls on a side stream, and captured: every replay on new inputs equals the eager result, with eager calls and
    two graphs in between (each capture holds its own workspace)."""
    ps = [paged([1, 4], [3000, 900], 8, 2, 128, 16, torch.bfloat16, seed=s) for s in (1, 2)]
    dev = [{n: t.to(DEV) for n, t in p.items() if isinstance(t, torch.Tensor)} for p in ps]
    cos, sin = (t.to(DEV) for t in tables(4096, 128))
    pos = torch.tensor([2999, 896, 897, 898, 899], dtype=torch.int32, device=DEV)
    seq = torch.tensor([0, 1, 1, 1, 1], device=DEV)

    def call(d):
        slots = d["table"][seq, (pos // 16).long()].long() * 16 + pos % 16
        new = d["q"][:, :4]
        q = kv_cache.append_kv(new[:, :2], new[:, 2:], d["k"], d["v"], slots, cos, sin, pos, q=d["q"])
        return kv_cache.paged_attention(q, d["k"], d["v"], d["table"], d["cu"], d["kv"], 4, 3000, causal=True)

    want = [call(d).clone() for d in dev]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [call(d) for d in dev]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for d in dev:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = call(d)
        graphs.append((gr, o))
    for rep in range(4):
        for d in dev:
            d["q"].copy_(torch.randn(d["q"].shape, device=DEV))
        for gr, _ in graphs:
            gr.replay()
        got = [o.clone() for _, o in graphs]
        want = [call(d) for d in dev]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


def test_nothing_to_do():
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    q, k = kv_cache.qk_norm_rope(z(0, 8, 96), z(0, 8, 96), None, None, None, None, None)
    assert q.shape == (0, 8, 96)
    cache = z(2, 16, 8, 96)
    assert kv_cache.append_kv(z(0, 8, 96), z(0, 8, 96), cache, cache.clone(), z(0, dtype=torch.int64)) is None
    assert kv_cache.paged_attention(z(0, 8, 96), cache, cache, z(1, 2, dtype=torch.int32), i32(0, 0), i32(5), 0, 5).shape == (0, 8, 96)
    # an empty cache, no table, nothing cached: zeros
    none = z(0, 16, 8, 96)
    out, lse = kv_cache.paged_attention(z(2, 8, 96) + 1, none, none, z(1, 0, dtype=torch.int32), i32(0, 2), i32(7), 2, 7, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 40, 200])
@pytest.mark.parametrize("causal", [False, True])
def test_sequences_without_keys(dtype, n, causal):
    """No table, no room, no keys, keys of another sequence only: zeros, and the other sequence as if it were alone."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    p = paged([n, 3], [0, 700], 4, 2, 96, 16, dtype, seed=4)
    q, k, v = (p[x].to(DEV) for x in "qkv")
    cu = p["cu"].to(DEV)
    for table, kv, room in ((torch.zeros(2, 0, dtype=torch.int32), i32(9, 9), 9), (p["table"], i32(0, 700), 0), (p["table"], i32(0, 0), 5000),
                            (p["table"], i32(-5, -1), 700)):
        out, lse = kv_cache.paged_attention(q, k, v, table.to(DEV), cu, kv, n, room, causal=causal, return_lse=True)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    got = run_paged(p, causal=causal)
    assert bool((got[:n] == 0).all())
    check_attention(got, O.attention(p["q"], p["k"], p["v"], p["table"], p["cu"], p["kv"], causal=causal), 700, 96, dtype)


def test_refused_operands():
    """What a call cannot be given: said by name before anything is enqueued."""
    z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device=DEV)
    q, k, cache = z(2, 8, 96), z(2, 4, 96), z(3, 16, 4, 96)
    slots = torch.arange(2, device=DEV)
    cos, sin, pos = z(64, 48), z(64, 48), z(2, dtype=torch.int32)
    norm = lambda **kw: kv_cache.qk_norm_rope(*[{**dict(q=q, k=k, w=None, x=None, cos=cos, sin=sin, pos=pos), **kw}[n] for n in ("q", "k", "w", "x", "cos", "sin", "pos")])
    for kw, msg in ((dict(q=q.double()), "float32 and bfloat16"), (dict(k=k.bfloat16()), "k is torch.bfloat16"), (dict(k=z(3, 4, 96)), r"k is \(3, 4, 96\)"),
                    (dict(q=z(2, 8 * 96)), "q has 2 dimensions"), (dict(w=z(95)), "q_weight must be contiguous with 96"),
                    (dict(sin=None), "go together"), (dict(pos=pos.long()), "pos is torch.int64"), (dict(pos=z(3, dtype=torch.int32)), "pos must be"),
                    (dict(cos=z(64, 47)), "max_pos, 48"), (dict(k=k.cpu()), "k is on cpu")):
        with pytest.raises(ValueError, match=msg):
            norm(**kw)
    with pytest.raises(TypeError, match="k must be a tensor"):
        norm(k=None)
    with pytest.raises(RuntimeError, match="HIP device"):
        norm(q=q.cpu())
    with pytest.raises(RuntimeError, match="q requires gradients"):
        norm(q=z(2, 8, 96).requires_grad_())
    with torch.no_grad():
        norm(q=z(2, 8, 96).requires_grad_())
    with pytest.raises(ValueError, match="expanded"):
        kv_cache.qk_norm_rope(q, k, None, None, None, None, None, q_out=z(1, 8, 96).expand(2, 8, 96))
    with pytest.raises(ValueError, match="q_out is"):
        kv_cache.qk_norm_rope(q, k, None, None, None, None, None, q_out=z(2, 7, 96))
    with pytest.raises(_hip.DarkHipError, match="head_dim"):
        kv_cache.qk_norm_rope(z(1, 2, 80), z(1, 2, 80), None, None, None, None, None)
    app = lambda **kw: kv_cache.append_kv(*[{**dict(k=k, v=k, kc=cache, vc=cache.clone(), slots=slots), **kw}[n] for n in ("k", "v", "kc", "vc", "slots")])
    for kw, msg in ((dict(slots=slots.int()), "slots is torch.int32"), (dict(kc=z(3, 12, 4, 96), vc=z(3, 12, 4, 96)), "power of two"),
                    (dict(vc=z(3, 4, 16, 96).transpose(1, 2)), "same shape and strides"), (dict(kc=z(3, 16, 5, 96), vc=z(3, 16, 5, 96)), "heads of 96"),
                    (dict(kc=z(1, 16, 4, 96).expand(3, 16, 4, 96), vc=z(1, 16, 4, 96).expand(3, 16, 4, 96)), "expanded"),
                    (dict(v=z(2, 3, 96)), "the cache holds")):
        with pytest.raises(ValueError, match=msg):
            app(**kw)
    with pytest.raises(TypeError, match="slots"):
        app(slots=None)
    with pytest.raises(ValueError, match="q_out without q"):
        kv_cache.append_kv(k, k, cache, cache.clone(), slots, q_out=q)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    base = dict(q=q, kc=cache, vc=cache, table=z(1, 3, dtype=torch.int32), cu=i32(0, 2), kv=i32(5))
    att = lambda mq=2, mk=5, **kw: kv_cache.paged_attention(*[{**base, **kw}[n] for n in ("q", "kc", "vc", "table", "cu", "kv")], mq, mk,
                                                            **{n: v for n, v in kw.items() if n not in base})
    assert att().shape == (2, 8, 96)
    for kw, msg in ((dict(q=z(2, 6, 96)), "q is"), (dict(cu=i32(0, 1, 2)), "cu_q must be"), (dict(kv=i32(5).long()), "kv_len is torch.int64"),
                    (dict(table=z(1, 3)), "block_table is torch.float32"), (dict(key_mask=z(1, 4, dtype=torch.uint8)), "key_mask is"),
                    (dict(key_mask=z(1, 5)), "uint8 or bool"), (dict(mk=-1), "max_kv=-1"), (dict(q_index=i32(0)), "q_index must be"),
                    (dict(out=z(2, 8, 96).bfloat16()), "out is torch.bfloat16"), (dict(out=q), "overlap")):
        with pytest.raises(ValueError, match=msg):
            att(**kw)
    with pytest.raises(_hip.DarkHipError, match="scale"):
        att(scale=math.nan)


def test_autograd_knows_of_the_calls():
    """Operands with a forward-mode tangent are refused as those that ask for gradients are; what a call writes counts as
    written, so that a backward pass which saved it before fails instead of using the new values."""
    import torch.autograd.forward_ad as fw
    z = lambda *s: torch.randn(s, device=DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    q, k, slots = z(2, 8, 96), z(2, 4, 96), torch.arange(2, device=DEV)
    kc, vc, table, cu, kv = z(1, 16, 4, 96), z(1, 16, 4, 96), i32(0).view(1, 1), i32(0, 2), i32(2)
    calls = {"q": [lambda x: kv_cache.qk_norm_rope(x, k, None, None, None, None, None),
                   lambda x: kv_cache.append_kv(k, k, kc, vc, slots, q=x),
                   lambda x: kv_cache.paged_attention(x, kc, vc, table, cu, kv, 2, 2)],
             "k_cache": [lambda x: kv_cache.append_kv(k, k, x, vc, slots), lambda x: kv_cache.paged_attention(q, x, vc, table, cu, kv, 2, 2)]}
    with fw.dual_level():
        for name, fs in calls.items():
            x = {"q": q, "k_cache": kc}[name]
            for f in fs:
                with pytest.raises(RuntimeError, match=f"{name} carries a forward-mode tangent"):
                    f(fw.make_dual(x, torch.ones_like(x)))
                f(x)
    for out, f in ((q.clone(), lambda o: kv_cache.qk_norm_rope(q, k, None, None, None, None, None, q_out=o)),
                   (k.clone(), lambda o: kv_cache.qk_norm_rope(q, k, None, None, None, None, None, k_out=o)),
                   (kc.clone(), lambda o: kv_cache.append_kv(k, k, o, vc, slots)), (vc.clone(), lambda o: kv_cache.append_kv(k, k, kc, o, slots)),
                   (q.clone(), lambda o: kv_cache.append_kv(k, k, kc, vc, slots, q=q, q_out=o)),
                   (q.clone(), lambda o: kv_cache.paged_attention(q, kc, vc, table, cu, kv, 2, 2, out=o))):
        w = torch.ones_like(out, requires_grad=True)
        y = (w * out).sum()                                   # saves `out` for w's gradient
        f(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    before = q._version, k._version                           # inputs are not written
    kv_cache.paged_attention(q, kc, vc, table, cu, kv, 2, 2)
    kv_cache.append_kv(k, k, kc, vc, slots, q=q)
    assert (q._version, k._version) == before
    with torch.inference_mode():
        o = torch.empty_like(q)
        assert kv_cache.paged_attention(q, kc, vc, table, cu, kv, 2, 2, out=o) is o
