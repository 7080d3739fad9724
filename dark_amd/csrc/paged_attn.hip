// Attention of a chunk of new tokens over a paged key / value cache.
//
// A query head group shares its keys, so the rows of one product are (token, head of the group) pairs: row r of a
// sequence's key head is token r / G, head r % G of the group, G = n_heads / n_kv_heads.
//
// Online softmax: with m = running maximum of a row's scores (in units of log2), l = running sum, O = running product,
//   m' = max(m, max_j s_j);  O' = O 2^(m - m') + sum_j 2^(s_j - m') v_j;  l' = l 2^(m - m') + sum_j 2^(s_j - m').
// Scores are computed TRANSPOSED (S^T = K Q^T) and so is the output (O^T = V^T P^T): a lane then holds ONE row's scores and
// output, so the statistics are per-lane scalars, and P^T leaves the first product in the layout the second one reads --
// with the keys of a 32-key slot permuted, and V's rows fetched in the same permuted order -- without touching LDS.
//
// A long key axis is split over workgroups where there are few rows; parts (O, m, l) are joined by a second kernel.
#include <math.h>

#include <type_traits>

#include "common.h"

namespace dark {

int check_paged_kv(const dark_paged_kv* kv, const char* who);
int check_stream_device(hipStream_t st);

// n / d for 0 <= n < 2^31 as one multiplication (a division by a run-time number is some 30 instructions, and a kernel of a
// few microseconds is fetched from memory as it runs): m = ceil(2^(31 + s) / d), s = ceil(log2 d), n m / 2^(31 + s) is exact.
struct Div {
  uint32_t d, m, s;
  __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)(__umulhi((uint32_t)n, m) >> s); }
  __device__ __forceinline__ int divmod(int& n) const {   // quotient; n becomes the remainder
    const int q = div(n);
    n -= q * (int)d;
    return q;
  }
};
static Div make_div(int d) {
  Div x = {(uint32_t)d, 0, 0};
  while ((1ll << x.s) < d) ++x.s;
  if (d > 1) {
    x.m = (uint32_t)(((1ull << (31 + x.s)) + d - 1) / d);
    x.s -= 1;
  }
  return x;
}

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int32_t *table, *cu_q, *kv_len, *q_index;
  const uint8_t* kmask;
  float *part_o, *part_ml;     // [n_split][T][H][HD], [n_split][T][H][2]; null when n_split == 1
  int64_t q_ts, q_hs, o_ts, o_hs, table_stride, mask_stride, page_stride, slot_stride, head_stride;
  int32_t T, H, Hk, G, B, width, n_pages, page_log2, unit, causal, n_split, split_keys, n_tiles, cap, max_q, n_units, n_inner, by_length, block0;   // block0: workgroups (join: rows) of the call before this launch's; n_units: problems of the launch: sequences x key heads x row tiles x parts
  Div by_hk, by_tiles, by_split, by_group, by_inner, by_heads, by_rows;   // by_rows: max_q * n_heads
  float scale_log2, q_factor;  // scale * log2(e); row tiles: its absolute value (1 for a scale of 0), what q is multiplied by
};

// Workgroups are handed to the eight XCDs, each with an L2 of its own, in turn.  `n_inner` units that follow each other and
// read the same memory (row tiles of a key head; key heads of one token row) go to one XCD: unit number of this workgroup.
__device__ __forceinline__ int unit_of_block(const PagedArgs& a) {
  const int block = a.block0 + blockIdx.x;
  if (a.n_inner <= 1) return block;
  int k = block >> 3;
  const int group = a.by_inner.divmod(k);
  return (group * 8 + (block & 7)) * a.n_inner + k;
}

// keys of a sequence: what it says, within the table and the caller's bound (hence within the mask's rows)
__device__ __forceinline__ int seq_len(const PagedArgs& a, int b) {
  const int len = a.kv_len[b];
  return len < 0 ? 0 : (len > a.cap ? a.cap : len);
}

// Infinities and NaN of a V row that some row of the tile must not see (P = 0 there): 0 * inf would be NaN.  They are taken
// out of the product and counted by a second one over P's indicator, +inf as 1, -inf as 128, NaN as both (at most 64 keys a
// tile; 129 is a bf16), and added to the rows that do see them.
__device__ __forceinline__ float odd_code(float x) { return (x == INFINITY ? 1.f : 0.f) + (x == -INFINITY ? 128.f : 0.f) + (x != x ? 129.f : 0.f); }
__device__ __forceinline__ float odd_apply(float acc, float code) {
  const float neg = floorf(code * 0.0078125f), pos = __builtin_fmaf(neg, -128.f, code);
  acc += pos > 0.f ? INFINITY : 0.f;
  return acc + (neg > 0.f ? -INFINITY : 0.f);   // (inf - inf: NaN)
}

// 1 / l; a row without keys has l = 0 and gets zeros, a NaN sum stays one
__device__ __forceinline__ float norm_of(float l) { return l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l); }
__device__ __forceinline__ float lse_of(float m, float l) {
  return l > 0.f ? (m + log2f(l)) * 0.69314718055994530942f : (l == 0.f ? -INFINITY : l);
}

// over the four lanes l, l ^ 16, l ^ 32, l ^ 48 that hold one row (swaps of 16- and 32-lane rows, no LDS)
__device__ __forceinline__ float quad_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// over the two lanes l, l ^ 32 that hold one row
__device__ __forceinline__ float pair_max(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The running maximum is a reference, not a result: it is only raised -- and the output rescaled -- once a score exceeds it
// by this much (log2 units; weights then reach 2^8, which floating types hold as exactly as they hold 1).
constexpr float kSlack = 8.f;

// 16 dims x 32 keys of V^T as the first operand of the second product: two transposed LDS reads (each 16-lane group fetches
// a 4-key x 16-dim block row-wise and receives it column-wise), keys in the order P^T has them
template <int LD>
__device__ __forceinline__ bf16x8 read_vt(const bf16_t* Vs, int li, int g, int dt) {
  typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
  const bf16_t* vrow = Vs + (4 * g + (li >> 2)) * LD + dt * 16 + 4 * (li & 3);
  const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)vrow);
  const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(vrow + 16 * LD));
  return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
}

// a finished row (its lanes hold 4 of every 16 columns): the output, or the part of a split axis
template <typename T, int HD>
__device__ __forceinline__ void write_row(const PagedArgs& a, bool parts, int64_t at, int tok, int hq, int g,
                                          const f32x4 (&O)[HD / 16], float m, float l) {
  if (parts) {
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) *(f32x4*)(a.part_o + at * HD + dt * 16 + 4 * g) = O[dt];
    if (g == 0) { a.part_ml[at * 2] = m; a.part_ml[at * 2 + 1] = l; }
    return;
  }
  const float inv = norm_of(l);
  T* orow = (T*)a.out + (int64_t)tok * a.o_ts + hq * a.o_hs;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt)
    store4(orow + dt * 16 + 4 * g, make_float4(O[dt][0] * inv, O[dt][1] * inv, O[dt][2] * inv, O[dt][3] * inv));
  if (a.lse && g == 0) a.lse[(int64_t)tok * a.H + hq] = lse_of(m, l);
}

// orders a wave's LDS writes before its lanes' reads of each other's (no instruction: LDS serves a wave in order)
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __attribute__((aligned(16))) const unsigned kZeroRow[128] = {};   // 512 bytes, the longest row: a key that is left out

constexpr int PT_KEYS = 32;   // keys of a streamed tile

// A load from global memory.  Said so, because the choice between a row and kZeroRow leaves the compiler a pointer of no known
// memory: it then loads with instructions that LDS may serve as well, and waits for those before it touches LDS
// (1024 x 11 over 46: 29.4 us so, 27.2).
template <bool NT = false, typename V>
__device__ __forceinline__ V load_global(const V* p) {
  typedef const __attribute__((address_space(1))) V global_v;
  return NT ? __builtin_nontemporal_load((global_v*)p) : *(global_v*)p;
}

// ---- what a wave of the streaming kernels works on: RT times 16 rows of one key head against a part of its sequence's keys
template <int RT> struct Unit {
  int b, hk, split, t0, row0, rows, lo, n_parts, k_begin, k_end;   // row0: its first; lo: the fewest keys any row may look at
  int tok[RT], hq[RT], seen[RT];                                   // this lane's rows (16 t + (lane & 15)); keys they may look at
  bool live[RT];
};
// which it is (arithmetic alone), ...
template <int RT>
__device__ __forceinline__ void place_unit(const PagedArgs& a, int id, Unit<RT>& u) {
  int q = a.by_tiles.divmod(id);
  u.row0 = id * 16 * RT;             // (the tiles of a key head read the same keys, ...
  id = a.by_hk.divmod(q);
  u.hk = q;                          // ... the key heads of a token lie next to each other)
  u.b = a.by_split.divmod(id);
  // each sequence begins its round of the XCDs with another part: the first parts, which short sequences have as well, would
  // all fall to the same XCDs (64 x 1 over up to 16384: 462 us without, 404 with)
  int shift = (int)(((uint32_t)u.b * 0x9E3779B1u) >> 16);
  a.by_split.divmod(shift);
  u.split = id + shift - (id + shift >= a.n_split ? a.n_split : 0);
  u.k_begin = u.split * a.split_keys;
}
// ... and what it holds
template <int RT>
__device__ __forceinline__ bool open_unit(const PagedArgs& a, int li, Unit<RT>& u) {
  int t0 = a.cu_q[u.b], t1 = a.cu_q[u.b + 1];
  const int len = seq_len(a, u.b);
  t0 = t0 < 0 ? 0 : (t0 > a.T ? a.T : t0);
  t1 = t1 < t0 ? t0 : (t1 > a.T ? a.T : t1);
  u.t0 = t0;
  u.rows = (t1 - t0) * a.G;
  if (u.row0 >= u.rows) return false;
  const int n = t1 - t0;
  auto clip = [&](int64_t last) { return last + 1 < len ? (last + 1 < 0 ? 0 : (int)(last + 1)) : len; };
  int hi = len;
  u.lo = len;
  if (a.causal && !a.q_index) {   // the sequence's last places: rows see more and more
    u.lo = clip((int64_t)len - n + a.by_group.div(u.row0));
    hi = clip((int64_t)len - n + a.by_group.div(min(u.row0 + 16 * RT, u.rows) - 1));
  } else if (a.causal) {
    hi = 0;
    u.lo = 0x7fffffff;
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = u.row0 + 16 * t + li;
    u.live[t] = row < u.rows;
    const int rr = u.live[t] ? row : u.row0, ri = a.by_group.div(rr);
    u.tok[t] = t0 + ri;
    u.hq[t] = u.hk * a.G + rr - ri * a.G;
    u.seen[t] = u.live[t] ? len : 0;
    if (a.causal && a.q_index) {
      u.seen[t] = u.live[t] ? clip(a.q_index[u.tok[t]]) : 0;
      hi = max(hi, u.seen[t]);
      u.lo = min(u.lo, u.live[t] ? u.seen[t] : 0x7fffffff);
    } else if (a.causal && u.live[t]) {
      u.seen[t] = clip((int64_t)len - n + ri);
    }
  }
  if (a.causal && a.q_index) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      hi = max(hi, __shfl_xor(hi, o, 64));
      u.lo = min(u.lo, __shfl_xor(u.lo, o, 64));
    }
    hi = __builtin_amdgcn_readfirstlane(hi);
    u.lo = __builtin_amdgcn_readfirstlane(u.lo);
  }
  u.n_parts = len <= a.split_keys ? 1 : 2;   // (one, or more)
  if (u.split > 0 && u.k_begin >= len) return false;
  u.k_end = min(hi, u.split == a.n_split - 1 ? hi : u.k_begin + a.split_keys);
  return true;
}

// ---- joins the WPP waves of a workgroup, whose (O [16][HD], m [16], l [16]) lie where `of(wave)` says: wave w of the first
// four the rows 4 w .. 4 w + 3, a lane four columns of each 64
template <typename T, int HD, int WPP, int RT, typename Of>
__device__ __forceinline__ void join_waves(const PagedArgs& a, const Unit<RT>& u, int row0, bool parts, int wave, int lane, Of of) {
  const int li = lane & 15, r = wave * 4 + (lane >> 4);
  if (wave >= 4 || row0 + r >= u.rows) return;
  float mm = -INFINITY;
#pragma unroll
  for (int w = 0; w < WPP; ++w) mm = fmaxf(mm, of(w)[16 * HD + r]);
  const float mz = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  f32x4 acc[(HD + 63) / 64] = {};
#pragma unroll
  for (int w = 0; w < WPP; ++w) {
    const float* o = of(w);
    const float f = __builtin_amdgcn_exp2f(o[16 * HD + r] - mz);
    ll += o[16 * HD + 16 + r] * f;
#pragma unroll
    for (int c = 0; c < (HD + 63) / 64; ++c) {
      const int col = c * 64 + li * 4;
      acc[c] += *(const f32x4*)(o + r * HD + (col < HD ? col : 0)) * f;   // (read anyway: a branch a wave would wait for each in turn)
    }
  }
  const int ti = a.by_group.div(row0 + r), tk = u.t0 + ti, h = u.hk * a.G + (row0 + r) - ti * a.G;
  const int64_t pa = ((int64_t)u.split * a.T + tk) * a.H + h;
  const float inv = parts ? 1.f : norm_of(ll);
#pragma unroll
  for (int c = 0; c < (HD + 63) / 64; ++c)
    if (c * 64 + li * 4 < HD) {
      if (parts) *(f32x4*)(a.part_o + pa * HD + c * 64 + li * 4) = acc[c];
      else store4((T*)a.out + (int64_t)tk * a.o_ts + h * a.o_hs + c * 64 + li * 4,
                  make_float4(acc[c][0] * inv, acc[c][1] * inv, acc[c][2] * inv, acc[c][3] * inv));
    }
  if (li == 0) {
    if (parts) { a.part_ml[pa * 2] = mm; a.part_ml[pa * 2 + 1] = ll; }
    else if (a.lse) a.lse[(int64_t)tk * a.H + h] = lse_of(mm, ll);
  }
}

// ---- few rows (one token and its head group, a handful of masked positions): 16 rows of one key head against a stream of
// keys that is read once.  Bound by HBM; what counts is bytes in flight, so every wave streams tiles of its own -- tile t's
// successor is on its way into the registers t is done with, the pages of the one behind it are looked up -- and waits for
// nobody.  K and V rows are read whole (16 lanes a row of 256 bytes) and turned into operands by way of LDS of the wave's
// own: read from memory as the first product wants them, 64 bytes of each of 16 rows an instruction, they come slower (64 x 1
// over up to 16384, 32 heads on 8 of 128: 518 us so, 439 whole, 401 = 6.1 TB/s whole and past the caches, see NT; a plain stream
// of such rows reads 6.0 and 6.8 TB/s).  Two waves a SIMD: 502 us with three, 522 with one.
// WPP waves share one problem (tiles dealt out in turn, joined in LDS at the end); WPP = 1: four problems a workgroup.
template <int HD, int WPP, bool ODD, bool NT>
__global__ __launch_bounds__(WPP == 8 ? 512 : 256, HD == 64 ? 3 : 2) void paged_few_kernel(const PagedArgs a) {
  constexpr int LD = HD + 8, NC = HD / 32, NW = WPP == 8 ? 8 : 4;   // NC: 32-dim steps of the first product
  constexpr int CH = HD / 8, NL = CH / 2;   // 16-byte chunks of a row; of a tile's K or V that a lane loads
  __shared__ __attribute__((aligned(16))) bf16_t Vall[NW][PT_KEYS * LD];
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  bf16_t* Vs = Vall[wave];
  int id = unit_of_block(a);
  if (WPP == 1) id = id * NW + wave;
  if (id < 0 || id >= a.n_units) return;
  Unit<1> u;
  place_unit(a, id, u);
  const int32_t* tab = a.table + u.b * a.table_stride;
  const uint8_t* km = a.kmask ? a.kmask + u.b * a.mask_stride : nullptr;
  // pages and masks of this lane's two keys of a tile as they stand in memory: looked at two tiles ahead and made sense of
  // one tile ahead, so that nothing waits for them -- the first even before the sequence's length is known, within the table
  int rp[2] = {-1, -1}, rm[2] = {1, 1};
  auto look = [&](int k0) {
#pragma unroll
    for (int jt = 0; jt < 2; ++jt) {
      const int key = min(k0 + jt * 16 + li, a.cap - 1);
      rp[jt] = tab[key >> a.page_log2];
      if (km) rm[jt] = km[key];
    }
  };
  const int first = u.k_begin + (WPP == 1 ? 0 : wave * PT_KEYS);
  if (a.cap > 0) look(first);
  if (!open_unit(a, li, u)) return;
  const int k_end = u.k_end, seen = u.seen[0], lo = u.lo;

  const bf16_t* qrow = (const bf16_t*)a.q + (int64_t)u.tok[0] * a.q_ts + u.hq[0] * a.q_hs;
  bf16x8 qb[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) qb[i] = *(const bf16x8*)(qrow + i * 32 + g * 8);

  const bf16_t* kbase = (const bf16_t*)a.k + (int64_t)u.hk * a.head_stride;
  const bf16_t* vbase = (const bf16_t*)a.v + (int64_t)u.hk * a.head_stride;
  const int pmask = (1 << a.page_log2) - 1;
  // page of a key, -1 where it is left out
  auto place = [&](int k0, int (&pg)[2]) {
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
      pg[jt] = (k0 + jt * 16 + li < k_end && rp[jt] < a.n_pages && rm[jt] != 0) ? rp[jt] : -1;
  };
  // where a lane's chunks of 32 rows lie: chunk n is number n * 64 + lane of the tile, its row's place comes from the lane that
  // looked it up.  Rows are read whole, 1 KB an instruction.
  auto spread = [&](int k0, const int (&pg)[2], int64_t (&off)[NL]) {
    int64_t at[2];
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
      at[jt] = pg[jt] < 0 ? -1 : (int64_t)pg[jt] * a.page_stride + (int64_t)((k0 + jt * 16 + li) & pmask) * a.slot_stride;
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int c = n % (NL / 2) * 64 + lane, row = c / CH, jt = n / (NL / 2);
      const unsigned lo32 = (unsigned)__builtin_amdgcn_ds_bpermute(row * 4, (int)(uint32_t)at[jt]);
      const int hi32 = __builtin_amdgcn_ds_bpermute(row * 4, (int)(at[jt] >> 32));
      off[n] = (int64_t)hi32 << 32 | lo32;
    }
  };
  auto fetch = [&](const bf16_t* base, const int64_t (&off)[NL], bf16x8 (&x)[NL]) {
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int col = (n % (NL / 2) * 64 + lane) % CH * 8;
      const bf16_t* p = off[n] < 0 ? (const bf16_t*)kZeroRow : base + off[n];   // a key that is left out is read as zeros
      x[n] = load_global<NT>((const bf16x8*)(p + col));
    }
  };
  auto to_lds = [&](const bf16x8 (&x)[NL]) {   // (row = key, padded by 16 bytes: no bank conflict in either direction)
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int c = n * 64 + lane;
      *(bf16x8*)(Vs + c / CH * LD + c % CH * 8) = x[n];
    }
  };

  f32x4 O[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) O[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // One turn of the loop brings tile t + 1 in and works on tile t; the first only brings (the code of both is there once:
  // short kernels are fetched as they run).
  const int step = WPP * PT_KEYS;
  int k0 = first - step;
  int pg[2] = {-1, -1}, pn[2];
  bf16x8 kr[NL], vr[NL];
  int64_t off[NL];
  for (bool work = false; k0 < k_end; k0 += step, work = true) {
    if (k0 + step >= k_end && !work) break;
    place(k0 + step, pn);
    if (k0 + 2 * step < k_end) look(k0 + 2 * step);   // (before the rows: who waits for it does not wait for them)
    spread(k0 + step, pn, off);
    // ---- S^T = K Q^T by way of LDS; K's registers then take the next tile's
    f32x4 S[2];
    if (work) to_lds(kr);
    fetch(kbase, off, kr);
    if (work) {
      wave_fence();   // lanes read what other lanes of the wave have written
#pragma unroll
      for (int jt = 0; jt < 2; ++jt) {
        S[jt] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NC; ++i)
          S[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)(Vs + (jt * 16 + li) * LD + i * 32 + g * 8), qb[i], S[jt], 0, 0, 0);
      }
      wave_fence();
    }
    // ---- V -> LDS in K's place; V's registers likewise
    bool odd = false;
    if (work) {
      if (ODD && k0 + PT_KEYS > lo && lo < k_end) {   // some row does not see a key that others do
#pragma unroll
        for (int n = 0; n < NL; ++n)
#pragma unroll
          for (int e = 0; e < 8; ++e) odd |= !(fabsf((float)vr[n][e]) < INFINITY);
        odd = __any(odd);
      }
      to_lds(vr);
    }
    fetch(vbase, off, vr);
    if (work) {
      // ---- softmax
      float mx = -INFINITY;
#pragma unroll
      for (int jt = 0; jt < 2; ++jt) {
        const unsigned on = (unsigned)__ballot(pg[jt] >= 0) >> (4 * g);   // (lanes 0..15 hold the tile's 16 keys)
        const int room = seen - (k0 + jt * 16 + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          S[jt][r] = ((on >> r) & 1) && r < room ? S[jt][r] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, S[jt][r]);
        }
      }
      mx = quad_max(mx);
      if (__any(mx > m + kSlack)) {
        const float mn = fmaxf(m, mx);
        const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        m = mn;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) O[i] *= alpha;
      }
      const float mz = m == -INFINITY ? 0.f : m;   // nothing seen yet: 2^(-inf - 0) = 0 everywhere
      bf16x8 pb;
#pragma unroll
      for (int jt = 0; jt < 2; ++jt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          S[jt][r] = __builtin_amdgcn_exp2f(S[jt][r] - mz);
          l += S[jt][r];
          pb[jt * 4 + r] = (bf16_t)S[jt][r];   // (rounded for the matrix instruction: relative 2^-8 a weight)
        }
      // ---- O^T += V^T P^T
      wave_fence();
      if (ODD && odd) {
        bf16x8 ind;
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) ind[jj] = S[jj >> 2][jj & 3] > 0.f ? (bf16_t)1.f : (bf16_t)0.f;
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt) {
          const bf16x8 v = read_vt<LD>(Vs, li, g, dt);
          bf16x8 vs = v, vc;
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) {
            const float c = odd_code((float)v[jj]);
            vc[jj] = (bf16_t)c;
            vs[jj] = c == 0.f ? v[jj] : (bf16_t)0.f;
          }
          const f32x4 code = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vc, ind, (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
          O[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vs, pb, O[dt], 0, 0, 0);
#pragma unroll
          for (int r = 0; r < 4; ++r) O[dt][r] = odd_apply(O[dt][r], code[r]);
        }
      } else {
#pragma unroll
        for (int dt = 0; dt < HD / 16; ++dt)
          O[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(read_vt<LD>(Vs, li, g, dt), pb, O[dt], 0, 0, 0);
      }
      wave_fence();
    }
    pg[0] = pn[0]; pg[1] = pn[1];
  }
  l = quad_sum(l);
  const bool parts = u.n_parts > 1 && a.n_split > 1;
  if constexpr (WPP == 1) {
    if (!u.live[0]) return;
    write_row<bf16_t, HD>(a, parts, ((int64_t)u.split * a.T + u.tok[0]) * a.H + u.hq[0], u.tok[0], u.hq[0], g, O, m, l);
  } else {
    // O [16][HD] fp32, then m and l of the 16 rows, in the wave's own LDS
    float* mine = (float*)Vs;
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) *(f32x4*)(mine + li * HD + dt * 16 + 4 * g) = O[dt];
    if (g == 0) { mine[16 * HD + li] = m; mine[16 * HD + 16 + li] = l; }
    __syncthreads();
    join_waves<bf16_t, HD, WPP>(a, u, u.row0, parts, wave, lane, [&](int w) { return (const float*)Vall[w]; });
  }
}

// ---- fp32: the same stream for any number of rows, 16 a workgroup, on 16 x 16 x 4 fp32 matrix instructions; nothing passes
// through LDS.  The output's columns are dealt to the second product's rows so that a lane reads a V row's 16 bytes at
// 64 c + 4 (lane & 15) -- 16 lanes a whole row piece -- and its four (HD 96: the last two) floats go to four instructions.
// 16 sequences of 9 to 128 new tokens over 31 to 512 keys, 12 heads of 64: 24 us, 29 TFLOP/s; the SIMDs that get the
// long sequences' rows work twice as long as the average.  (Eight waves a problem: 28.5 us; one: 47.)  Long chunks (4 x 1024
// over 9216, head_dim 128) 118 TFLOP/s of the 152 that a large fp32 product reaches: a read of K and V serves the wave's 32 rows
// alone (16 for heads of 64), 16 flops a byte, so that 7.4 TB/s of them go into registers, beside the softmax's vector
// instructions, which overlap with the matrix instructions of two or three waves only in part.  Single tokens over long
// contexts are bound by HBM (64 x 1 over up to 16384, 32 heads on 8 of 128: 812 us, 6.1 TB/s, every byte fetched once).
template <int HD, int WPP, int RT, bool ODD>
__global__ __launch_bounds__(256, HD == 64 ? 3 : 2) void paged_f32_kernel(const PagedArgs a) {
  constexpr int NC = HD / 16, KEYS = 16, NV = (HD + 63) / 64;   // NV: pieces of a V row a lane reads
  constexpr int E1 = HD == 96 ? 2 : 4;                                                      // floats of the second one
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  __shared__ __attribute__((aligned(16))) float Oall[WPP == 1 ? 1 : 4][RT][WPP == 1 ? 4 : 16 * HD + 32];
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int id = unit_of_block(a);
  if (WPP == 1) id = id * 4 + wave;
  if (id < 0 || id >= a.n_units) return;
  Unit<RT> u;
  place_unit(a, id, u);
  const int32_t* tab = a.table + u.b * a.table_stride;
  const uint8_t* km = a.kmask ? a.kmask + u.b * a.mask_stride : nullptr;
  int rp = -1, rm = 1;   // page and mask of key k0 + li as they stand in memory
  auto look = [&](int k0) {
    const int key = min(k0 + li, a.cap - 1);
    rp = tab[key >> a.page_log2];
    if (km) rm = km[key];
  };
  const int first = u.k_begin + (WPP == 1 ? 0 : wave * KEYS);
  if (a.cap > 0) look(first);
  if (!open_unit(a, li, u)) return;
  const int k_end = u.k_end, lo = u.lo;

  f32x4 qf[RT][NC];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const float* qrow = (const float*)a.q + (int64_t)u.tok[t] * a.q_ts + u.hq[t] * a.q_hs + g * 4;
#pragma unroll
    for (int i = 0; i < NC; ++i) qf[t][i] = *(const f32x4*)(qrow + 16 * i);
  }
  const float* kbase = (const float*)a.k + (int64_t)u.hk * a.head_stride;
  const float* vbase = (const float*)a.v + (int64_t)u.hk * a.head_stride;
  const int pmask = (1 << a.page_log2) - 1;
  // where key k0 + li lies, in elements from its head's first; -1: left out, read as zeros
  auto place = [&](int k0) -> int64_t {
    const bool on = k0 + li < k_end && rp >= 0 && rp < a.n_pages && rm != 0;
    return on ? (int64_t)rp * a.page_stride + (int64_t)((k0 + li) & pmask) * a.slot_stride : -1;
  };
  f32x4 kr[NC], v0[4], v1[4];
  auto fetch_k = [&](int64_t at) {
    const float* p = (at < 0 ? (const float*)kZeroRow : kbase + at) + g * 4;
#pragma unroll
    for (int i = 0; i < NC; ++i) kr[i] = load_global((const f32x4*)(p + i * 16));
  };
  auto fetch_v = [&](int64_t at) {   // rows 4 g + r: the keys whose weights this lane group holds
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const unsigned lo32 = (unsigned)__builtin_amdgcn_ds_bpermute((4 * g + r) * 4, (int)(uint32_t)at);
      const int hi32 = __builtin_amdgcn_ds_bpermute((4 * g + r) * 4, (int)(at >> 32));
      const float* p = hi32 < 0 ? (const float*)kZeroRow : vbase + ((int64_t)hi32 << 32 | lo32);
      v0[r] = load_global((const f32x4*)(p + li * 4));
      if constexpr (E1 == 2) {
        const f32x2 x = load_global((const f32x2*)(p + 64 + li * 2));
        v1[r] = (f32x4){x[0], x[1], 0.f, 0.f};
      } else if constexpr (NV == 2) {
        v1[r] = load_global((const f32x4*)(p + 64 + li * 4));
      }
    }
  };

  f32x4 O[RT][NC];   // [4 c + e]: column 64 c + 4 (4 g + r) + e (HD 96, c = 1: 64 + 2 (4 g + r) + e) in element r
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int i = 0; i < NC; ++i) O[t][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m[RT], l[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) { m[t] = -INFINITY; l[t] = 0.f; }
  // (one turn brings tile t + 1 in and works on tile t, as above)
  const int step = WPP * KEYS;
  int k0 = first - step;
  int64_t pg = -1, pn;
  for (bool work = false; k0 < k_end; k0 += step, work = true) {
    if (k0 + step >= k_end && !work) break;
    pn = place(k0 + step);
    if (k0 + 2 * step < k_end) look(k0 + 2 * step);
    f32x4 S[RT];
    if (work) {   // two sums a row tile: an instruction does not wait for the one before it
      f32x4 S2[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) S[t] = S2[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int e = 0; e < 4; e += 2)
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            S[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[i][e], qf[t][i][e], S[t], 0, 0, 0);
            S2[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[i][e + 1], qf[t][i][e + 1], S2[t], 0, 0, 0);
          }
#pragma unroll
      for (int t = 0; t < RT; ++t) S[t] += S2[t];
    }
    fetch_k(pn);
    if (work) {
      const unsigned on = (unsigned)__ballot(pg >= 0) >> (4 * g);   // (lanes 0..15 hold the 16 keys)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float mx = -INFINITY;
        const int room = u.seen[t] - (k0 + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          S[t][r] = ((on >> r) & 1) && r < room ? S[t][r] * a.scale_log2 : -INFINITY;
          mx = fmaxf(mx, S[t][r]);
        }
        mx = quad_max(mx);
        if (__any(mx > m[t] + kSlack)) {
          const float mn = fmaxf(m[t], mx);
          const float alpha = __builtin_amdgcn_exp2f(m[t] - (mn == -INFINITY ? 0.f : mn));
          m[t] = mn;
          l[t] *= alpha;
#pragma unroll
          for (int i = 0; i < NC; ++i) O[t][i] *= alpha;
        }
        const float mz = m[t] == -INFINITY ? 0.f : m[t];   // nothing seen yet: 2^(-inf - 0) = 0 everywhere
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          S[t][r] = __builtin_amdgcn_exp2f(S[t][r] - mz);
          l[t] += S[t][r];   // (this lane's keys only: the four lanes of a row are added up at the end)
        }
      }
      // ---- O^T += V^T P^T
      if (ODD && k0 + KEYS > lo && lo < k_end) {
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < NC; ++i) odd |= !(fabsf(i < 4 ? v0[r][i & 3] : v1[r][i & 3]) < INFINITY);
        if (__any(odd)) {
#pragma unroll
          for (int i = 0; i < NC; ++i) {
            f32x4 code[RT] = {};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float c = odd_code(i < 4 ? v0[r][i & 3] : v1[r][i & 3]);
#pragma unroll
              for (int t = 0; t < RT; ++t) code[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(c, S[t][r] > 0.f ? 1.f : 0.f, code[t], 0, 0, 0);
              if (i < 4) v0[r][i & 3] = c == 0.f ? v0[r][i & 3] : 0.f;
              else v1[r][i & 3] = c == 0.f ? v1[r][i & 3] : 0.f;
            }
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
              for (int x = 0; x < 4; ++x) O[t][i][x] = odd_apply(O[t][i][x], code[t][x]);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int t = 0; t < RT; ++t)
            O[t][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(i < 4 ? v0[r][i & 3] : v1[r][i & 3], S[t][r], O[t][i], 0, 0, 0);
    }
    fetch_v(pn);
    pg = pn;
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) l[t] = quad_sum(l[t]);
  const bool parts = u.n_parts > 1 && a.n_split > 1;
  // four (two) neighbouring columns of this lane's row for each r
  auto emit = [&](float* row, const f32x4 (&o)[NC], float inv) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      *(f32x4*)(row + 4 * (4 * g + r)) = (f32x4){o[0][r], o[1][r], o[2][r], o[3][r]} * inv;
      if constexpr (E1 == 2) *(f32x2*)(row + 64 + 2 * (4 * g + r)) = (f32x2){o[4][r], o[5][r]} * inv;
      else if constexpr (NV == 2) *(f32x4*)(row + 64 + 4 * (4 * g + r)) = (f32x4){o[NC - 4][r], o[NC - 3][r], o[NC - 2][r], o[NC - 1][r]} * inv;
    }
  };
  if constexpr (WPP == 1) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (!u.live[t]) continue;
      const int64_t at = ((int64_t)u.split * a.T + u.tok[t]) * a.H + u.hq[t];
      if (parts) {
        emit(a.part_o + at * HD, O[t], 1.f);
        if (g == 0) { a.part_ml[at * 2] = m[t]; a.part_ml[at * 2 + 1] = l[t]; }
      } else {
        emit((float*)a.out + (int64_t)u.tok[t] * a.o_ts + u.hq[t] * a.o_hs, O[t], norm_of(l[t]));
        if (a.lse && g == 0) a.lse[(int64_t)u.tok[t] * a.H + u.hq[t]] = lse_of(m[t], l[t]);
      }
    }
  } else {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float* mine = Oall[wave][t];
      emit(mine + li * HD, O[t], 1.f);
      if (g == 0) { mine[16 * HD + li] = m[t]; mine[16 * HD + 16 + li] = l[t]; }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t)
      join_waves<float, HD, WPP>(a, u, u.row0 + 16 * t, parts, wave, lane, [&](int w) { return (const float*)Oall[w][t]; });
  }
}

// ---- many rows (chunks of a prompt): 128 rows of one key head (32 a wave) against tiles of 64 keys that the workgroup's
// four waves share through LDS, on 32 x 32 x 16 matrix instructions.  Two tile buffers: the next tile is written into LDS by
// the memory pipe itself while this one is computed; one barrier a tile.
// LDS rows are not padded (the direct writes are linear), their 16-byte chunks are permuted instead: by the row's number,
// so that the 16 rows a K read touches at once, and the 4 rows of a transposed V read, lie in different banks.
// Bound by matrix and vector instructions in turn: 32 and some 220 of them for 32 x 64 scores of head_dim 128, two waves a SIMD.
// 4 x 1024 tokens over 9216, 8 key heads of 128, groups of 4: 668 us, 926 TFLOP/s (causal 626 us, 933); head_dim 96 527 us, 880;
// 64 388 us, 797; over up to 17408, ragged, 525 us, 896.  The next tile's first product between this tile's exponentials (by
// scheduling groups, by source order): 841 and 920 TFLOP/s, the other wave of the SIMD fills those gaps already.
template <int HD> struct TileSwz {
  static constexpr int CH = HD / 8;   // chunks of a row
  // 128: 16 chunks = all banks; 64: two rows are; 96: rows start 4 chunks apart, K's chunks are rotated, V's are apart as is
  __device__ static __forceinline__ int k_pos(int r, int c) {
    if constexpr (HD == 96) { const int x = c + ((r >> 2) & 3); return x >= CH ? x - CH : x; }
    else return c ^ (HD == 128 ? r & 15 : (r >> 1) & 7);
  }
  __device__ static __forceinline__ int k_chunk(int r, int pos) {
    if constexpr (HD == 96) { const int x = pos - ((r >> 2) & 3); return x < 0 ? x + CH : x; }
    else return k_pos(r, pos);
  }
  __device__ static __forceinline__ int v_pos(int r, int c) {
    return HD == 96 ? c : c ^ (HD == 128 ? (r & 7) * 2 : ((r >> 1) & 3) * 2);
  }
};

constexpr int TT_ROWS = 128, TT_KEYS = 64;

// The sequence with the n-th most keys (of 64 at most, a lane each): the longest begin first and the shortest
// fill up what is left (32 heads on 8 of 128: 24 x up to 200 over up to 6200 180 us, 238 in the batch's order; 12 x up to
// 400 over up to 10400 302 and 365.  Not by rows times keys: a workgroup has 128 rows whatever the sequence has).
__device__ __forceinline__ int nth_longest(const PagedArgs& a, int n, int lane) {
  const int len = lane < a.B ? seq_len(a, lane) : -1;
  int ahead = 0;   // longer sequences, or as long ones before it
  for (int i = 0; i < a.B; ++i) {
    const int other = __builtin_amdgcn_readlane(len, i);
    ahead += other > len || (other == len && i < lane) ? 1 : 0;
  }
  return __builtin_ctzll(__ballot(lane < a.B && ahead == n));   // (exactly one is the n-th)
}

template <int HD, bool ODD, bool NT>
__global__ __launch_bounds__(256, 2) void paged_tile_kernel(const PagedArgs a) {
  typedef TileSwz<HD> Z;
  typedef __attribute__((address_space(3))) void lds_void;
  typedef const __attribute__((address_space(1))) void gl_void;
  typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
  constexpr int CH = Z::CH, TILE = TT_KEYS * HD * 2, NI = CH / 4;   // NI: 1-KB pieces of a tile that a wave brings in
  extern __shared__ __attribute__((aligned(16))) char smem[];       // [2][K tile | V tile]
  __shared__ int red[8];

  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, c32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int id = unit_of_block(a);
  if (id < 0 || id >= a.n_units) return;
  int rest = a.by_tiles.divmod(id);
  const int tile = a.n_tiles - 1 - id;                // (the tiles of a key head read the same keys; the last see most and come
                                                      // first: 2 chunks of 4096 tokens, causal, 343 us otherwise, 312)
  id = a.by_split.divmod(rest);
  const int split = rest;
  int b = a.by_hk.divmod(id);
  const int hk = id;
  if (a.by_length) b = nth_longest(a, b, lane);
  // the page and the mask of key k0 + lane as they stand in memory (made sense of one tile later, so that nothing waits here;
  // the first even before the sequence's length is known, within the table) ...
  const int32_t* tab = a.table + b * a.table_stride;
  const uint8_t* km = a.kmask ? a.kmask + b * a.mask_stride : nullptr;
  int raw_page = -1, raw_mask = 1;
  auto look = [&](int k0) {
    const int key = min(k0 + lane, a.cap - 1);
    raw_page = tab[key >> a.page_log2];
    if (km) raw_mask = km[key];
  };
  const int k_begin = split * a.split_keys;
  if (a.cap > 0) look(k_begin);
  int t0 = a.cu_q[b], t1 = a.cu_q[b + 1];
  t0 = t0 < 0 ? 0 : (t0 > a.T ? a.T : t0);
  t1 = t1 < t0 ? t0 : (t1 > a.T ? a.T : t1);
  const int rows = (t1 - t0) * a.G;
  const int row0 = tile * TT_ROWS;
  if (row0 >= rows) return;
  const int len = seq_len(a, b);
  const int row = row0 + wave * 32 + c32;
  const bool live = row < rows;
  const int ri = a.by_group.div(live ? row : row0), tok = t0 + ri, hq = hk * a.G + (live ? row : row0) - ri * a.G;
  int seen = live ? len : 0;   // keys this lane's row may look at
  if (a.causal && live) {
    const int64_t last = a.q_index ? (int64_t)a.q_index[tok] : (int64_t)len - (t1 - tok);
    seen = last + 1 < len ? (last + 1 < 0 ? 0 : (int)(last + 1)) : len;
  }
  int whi = seen, wlo = live ? seen : 0x7fffffff;   // largest and smallest bound of the wave's rows, then the workgroup's
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    whi = max(whi, __shfl_xor(whi, o, 64));
    wlo = min(wlo, __shfl_xor(wlo, o, 64));
  }
  whi = __builtin_amdgcn_readfirstlane(whi);
  wlo = __builtin_amdgcn_readfirstlane(wlo);
  if (lane == 0) { red[wave] = whi; red[4 + wave] = wlo; }
  __syncthreads();
  const int hi = __builtin_amdgcn_readfirstlane(max(max(red[0], red[1]), max(red[2], red[3])));
  const int lo = __builtin_amdgcn_readfirstlane(min(min(red[4], red[5]), min(red[6], red[7])));
  const int n_parts = len <= a.split_keys ? 1 : 2;   // (one, or more)
  if (split > 0 && k_begin >= len) return;
  const int k_end = min(hi, split == a.n_split - 1 ? hi : k_begin + a.split_keys);

  const bf16_t* qrow = (const bf16_t*)a.q + (int64_t)tok * a.q_ts + hq * a.q_hs;
  bf16x8 qb[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) qb[i] = *(const bf16x8*)(qrow + i * 16 + h * 8);
  // below, a larger product is a larger score: a scale that is not positive goes over to the queries (-1 and 0 times a bf16 are exact)
  if (a.q_factor != 1.f) {
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) qb[i][e] = (bf16_t)((float)qb[i][e] * a.q_factor);
  }

  const char* kbase = (const char*)((const bf16_t*)a.k + (int64_t)hk * a.head_stride);
  const char* vbase = (const char*)((const bf16_t*)a.v + (int64_t)hk * a.head_stride);
  const int pmask = (1 << a.page_log2) - 1;
  // ... and where its row lies, in units of 2^unit elements from its head's first; ~0: left out
  auto place = [&](int k0) -> unsigned {
    const int key = k0 + lane;
    const bool on = key < k_end && raw_page >= 0 && raw_page < a.n_pages && raw_mask != 0;
    return on ? (unsigned)(((int64_t)raw_page * a.page_stride + (int64_t)(key & pmask) * a.slot_stride) >> a.unit) : ~0u;
  };
  // this wave's pieces of a tile: lane l of piece n fills chunk (n * 4 + wave) * 64 + l of the tile
  auto stage = [&](int buf, unsigned off) {
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int at = (n * 4 + wave) * 64 + lane, r = at / CH, pos = at - r * CH;
      const unsigned o = __shfl(off, r, 64);
      const bool on = o != ~0u;
      const char* zr = (const char*)kZeroRow;
      const char* kp = (on ? kbase + ((uint64_t)o << (a.unit + 1)) : zr) + Z::k_chunk(r, pos) * 16;
      const char* vp = (on ? vbase + ((uint64_t)o << (a.unit + 1)) : zr) + Z::v_pos(r, pos) * 16;
      char* to = smem + buf * (2 * TILE) + (n * 4 + wave) * 1024;
      __builtin_amdgcn_global_load_lds((gl_void*)kp, (lds_void*)to, 16, 0, NT ? 2 : 0);   // (2: nt, past the caches)
      __builtin_amdgcn_global_load_lds((gl_void*)vp, (lds_void*)(to + TILE), 16, 0, NT ? 2 : 0);
    }
  };

  f32x16 O[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) O[i] = (f32x16){};
  float m = -INFINITY, l = 0.f;

  // this lane's places in a tile: K chunk 2i + h of row c32, V rows 4h + li / 4, columns 16 x + 4 (li & 3) of 32
  const int vr = 4 * h + (li >> 2), x = (lane >> 4) & 1;
  int k_at[HD / 16], v_at[HD / 32];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) k_at[i] = c32 * (HD * 2) + Z::k_pos(c32, 2 * i + h) * 16;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) v_at[i] = TILE + vr * (HD * 2) + Z::v_pos(vr, 4 * i + 2 * x + ((li & 3) >> 1)) * 16 + (li & 1) * 8;

  uint64_t on = 0, on_next = 0;   // which keys of the tile are used at all
  if (k_begin < k_end) {          // (no direct write may be under way when the workgroup ends)
    const unsigned off = place(k_begin);
    on = __ballot(off != ~0u);
    stage(0, off);
    look(k_begin + TT_KEYS);
  }
  // PART: some row may not see a key of the tile that others do
  auto turn = [&](auto part_tag, int k0, int buf) {
    constexpr bool PART = decltype(part_tag)::value;
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0): this wave's pieces of the tile are in LDS, its reads are done;
    __builtin_amdgcn_s_barrier();         // everybody's are: the tile may be read, the other buffer refilled
    if (k0 + TT_KEYS < k_end) {
      const unsigned off = place(k0 + TT_KEYS);
      on_next = __ballot(off != ~0u);
      stage(buf ^ 1, off);
      look(k0 + 2 * TT_KEYS);
    }
    const char* tl = smem + buf * (2 * TILE);
    int odd = 0;
    if (PART) {   // look for infinities and NaN in V
#pragma unroll
      for (int n = 0; n < CH / 4; ++n) {
        const bf16x8 v = *(const bf16x8*)(tl + TILE + (n * 256 + tid) * 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) odd |= !(fabsf((float)v[e]) < INFINITY);
      }
      odd = __syncthreads_or(odd);
    }
    // ---- S^T = K Q^T (a wave whose rows see nothing of the tile passes it by, but for the barriers)
    f32x16 S[2];
    if (k0 < whi) {
      bf16x8 kf[2][HD / 16];
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) kf[t][i] = *(const bf16x8*)(tl + t * 32 * HD * 2 + k_at[i]);
#pragma unroll
      for (int t = 0; t < 2; ++t) S[t] = (f32x16){};
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t) S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[t][i], qb[i], S[t], 0, 0, 0);
      // four LDS reads ahead of the matrix instructions, then one for one
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < HD / 8 - 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
    }
    if (PART && odd) {   // (rare) V's infinities and NaN out of the tile, their codes in K's place
      __syncthreads();
#pragma unroll 1
      for (int n = 0; n < CH / 4; ++n) {
        bf16x8* pv = (bf16x8*)(smem + buf * (2 * TILE) + TILE + (n * 256 + tid) * 16);
        bf16x8 v = *pv, c;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float code = odd_code((float)v[e]);
          c[e] = (bf16_t)code;
          v[e] = code == 0.f ? v[e] : (bf16_t)0.f;
        }
        *pv = v;
        *(bf16x8*)(smem + buf * (2 * TILE) + (n * 256 + tid) * 16) = c;
      }
      __syncthreads();
    }
    if (k0 < whi) {
      // ---- softmax: this lane's keys are 32 t + (i & 3) + 8 (i >> 2) + 4 h
      if (on != ~0ull || (PART && k0 + TT_KEYS > wlo)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          unsigned out = ~((unsigned)(on >> (32 * t)) >> (4 * h));   // keys left out, by the numbers of this lane's
          if (PART) {
            const int room = seen - (k0 + 32 * t + 4 * h);
            out |= room <= 0 ? ~0u : room >= 32 ? 0u : ~0u << room;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {   // (the bit over the whole word, then one word or the other: 1 x 725 over 939, masked, 34.9 -> 31.5 us)
            const unsigned bits = (unsigned)((int)(out << (31 - ((i & 3) + 8 * (i >> 2)))) >> 31);
            S[t][i] = __uint_as_float((bits & 0xff800000u) | (~bits & __float_as_uint(S[t][i])));   // (-inf, or as it is)
          }
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, S[t][i]);
      mx = pair_max(mx) * a.scale_log2;
      if (__any(mx > m + kSlack)) {
        const float mn = fmaxf(m, mx);
        const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
        m = mn;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) O[i] *= alpha;
      }
      const float mz = m == -INFINITY ? 0.f : m;
      bf16x8 pb[4];   // P^T, 16 keys each: rounded for the matrix instruction (relative 2^-8 a weight)
      float ls[2] = {0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(S[t][i], a.scale_log2, -mz));
          ls[i & 1] += e;
          pb[2 * t + (i >> 3)][i & 7] = (bf16_t)e;
        }
      l += ls[0] + ls[1];
      // ---- O^T += V^T P^T
      auto read_v = [&](const char* at, int s, int dt) {
        const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(at + s * 16 * HD * 2 + v_at[dt]));
        const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(at + (s * 16 + 8) * HD * 2 + v_at[dt]));
        return __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
      };
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) O[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_v(tl, s, dt), pb[s], O[dt], 0, 0, 0);
      if (PART && odd) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) pb[s][jj] = (float)pb[s][jj] > 0.f ? (bf16_t)1.f : (bf16_t)0.f;
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) {
          f32x16 code = {};
#pragma unroll
          for (int s = 0; s < 4; ++s) code = __builtin_amdgcn_mfma_f32_32x32x16_bf16(read_v(tl - TILE, s, dt), pb[s], code, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 16; ++i) O[dt][i] = odd_apply(O[dt][i], code[i]);
        }
      }
    }
    on = on_next;
  };
  int k0 = k_begin, buf = 0;
  for (const int whole = ODD && lo < k_end ? lo - TT_KEYS : k_end - 1; k0 <= whole; k0 += TT_KEYS, buf ^= 1) turn(std::false_type(), k0, buf);
  if constexpr (ODD)
    for (; k0 < k_end; k0 += TT_KEYS, buf ^= 1) turn(std::true_type(), k0, buf);
  l = pair_sum(l);
  if (!live) return;
  const bool parts = n_parts > 1 && a.n_split > 1;
  const int64_t at = ((int64_t)split * a.T + tok) * a.H + hq;
  const float inv = norm_of(l);
  bf16_t* orow = (bf16_t*)a.out + (int64_t)tok * a.o_ts + hq * a.o_hs;
#pragma unroll
  for (int dt = 0; dt < HD / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = dt * 32 + 8 * i + 4 * h;
      const f32x4 o = {O[dt][4 * i], O[dt][4 * i + 1], O[dt][4 * i + 2], O[dt][4 * i + 3]};
      if (parts) *(f32x4*)(a.part_o + at * HD + d) = o;
      else store4(orow + d, make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv));
    }
  if (h == 0) {
    if (parts) { a.part_ml[at * 2] = m; a.part_ml[at * 2 + 1] = l; }
    else if (a.lse) a.lse[(int64_t)tok * a.H + hq] = lse_of(m, l);
  }
}

// ---- joins the parts of a split key axis: WPR waves a (token, head), each an equal share of the parts (4 where there are
// many: the parts are then read side by side and not one after the other).  Latency: 5 us for 32 parts of 256 rows.
template <typename T, int HD, int WPR>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a) {
  __shared__ float so[4][HD], sl[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int h = a.block0 + (WPR == 4 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave);
  const int b = a.by_rows.divmod(h);
  if (b >= a.B) return;
  const int i = a.by_heads.divmod(h);
  const int t0 = a.cu_q[b], t1 = a.cu_q[b + 1], len = seq_len(a, b);
  const int tok = t0 + i;
  if (tok < 0 || tok >= t1 || tok >= a.T) return;
  const int n_all = len <= 0 ? 1 : (len + a.split_keys - 1) / a.split_keys;
  if (n_all <= 1) return;                       // written whole by the first kernel
  const int n = min(n_all, a.n_split);
  const int64_t step = (int64_t)a.T * a.H, row = (int64_t)tok * a.H + h;
  float m = -INFINITY;
  for (int s = lane; s < n; s += 64) m = fmaxf(m, a.part_ml[(s * step + row) * 2]);
  m = wave_max(m);
  const float mz = m == -INFINITY ? 0.f : m;
  const bool on = lane * 2 < HD;
  float l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 4
  for (int s = WPR == 4 ? wave : 0; s < n; s += WPR) {   // (every part in its fixed place: the same bits every time)
    const int64_t at = s * step + row;
    const float2 ml = *(const float2*)(a.part_ml + at * 2);
    const float2 v = on ? *(const float2*)(a.part_o + at * HD + lane * 2) : make_float2(0.f, 0.f);
    const float f = __builtin_amdgcn_exp2f(ml.x - mz);
    l += ml.y * f;
    o0 += v.x * f;
    o1 += v.y * f;
  }
  T* orow = (T*)a.out + (int64_t)tok * a.o_ts + h * a.o_hs;
  if constexpr (WPR == 4) {
    if (on) { so[wave][lane * 2] = o0; so[wave][lane * 2 + 1] = o1; }
    if (lane == 0) sl[wave] = l;
    __syncthreads();
    if (wave > 0) return;
    l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    if (on) {
      o0 = (so[0][lane * 2] + so[1][lane * 2]) + (so[2][lane * 2] + so[3][lane * 2]);
      o1 = (so[0][lane * 2 + 1] + so[1][lane * 2 + 1]) + (so[2][lane * 2 + 1] + so[3][lane * 2 + 1]);
    }
  }
  const float inv = norm_of(l);
  if (on) {
    orow[lane * 2] = ElemTraits<T>::from_f32(o0 * inv);
    orow[lane * 2 + 1] = ElemTraits<T>::from_f32(o1 * inv);
  }
  if (a.lse && lane == 0) a.lse[row] = lse_of(m, l);
}

// Workgroups of one launch at most, a multiple of the XCDs; a call of more takes several.  (A launch of 2^32 threads or more is
// not refused: it runs the rest of a division by 2^32.)
constexpr int MAX_BLOCKS = 1 << 22;

struct PagedPlan {
  int few, rt;           // waves a problem in the streaming kernels (0: tiles of rows) and their 16-row tiles
  int n_tiles, n_split, split_keys;
  int64_t ws_o, ws_ml;   // bytes
};

// The row tiles' kernel hands a key's place from lane to lane as 32 bits: in units of the largest power of two that divides
// the cache's strides (256 bytes for one head of 128 bf16, a cache of 1 TiB then).
static int place_step(const dark_paged_kv& kv) {
  const uint64_t strides = (uint64_t)kv.page_stride | (uint64_t)kv.slot_stride | 1ull << 20;
  return __builtin_ctzll(strides);
}

static PagedPlan plan_paged(const dark_paged_attention_args* p) {
  PagedPlan s;
  const int64_t rows = (int64_t)p->max_q * (p->n_heads / p->kv.n_kv_heads);
  const int64_t heads = (int64_t)p->kv.n_kv_heads * p->n_seqs;
  s.few = 0;
  s.rt = 1;
  if (p->kv.dtype == DARK_F32) {
    // A wave a problem where keys are few, or problems many: four waves of a workgroup then read the same keys, and nothing is
    // joined (16 heads on 4 of 128: 634 x up to 42 over up to 247 303 us, 322 with four waves a problem; 116 x up to 349 over up to
    // 353 322 and 436; 12 heads of 64, 21 x up to 346 over up to 531: 69 and 54 the other way).
    // 32 rows a wave where they are there and dims enough to be worth it (4 x 512 over 2048, 32 heads on 8 of 128: 653 us, 811 with
    // 16; 8 of 96, 8 x 512 over 2048: 289 and 358; 12 heads of 64, 64 x 40 over 440: 76 and 62 the other way).
    const int64_t problems = heads * ((rows + 15) / 16);
    const bool many = problems >= 8192 && p->max_kv <= 2048 && p->kv.head_dim > 64 && rows > 16;
    s.few = p->max_kv <= 128 || (p->max_kv <= 256 && problems >= 1024) || many ? 1 : 4;
    if (rows > 16 && p->kv.head_dim > 64 && (s.few == 4 || (many && p->max_kv > 256))) s.rt = 2;
  }
  else if (rows <= 16 || (rows <= 48 && p->max_kv <= 128)) {   // (512 x 46 over 46, 8 heads of 96: 42.3 us, 44.6 by row tiles;
                                                               // 64 x 8 over 2000, 32 rows: 160 and 88 the other way)
    // Waves a problem: one where keys are few, eight where CUs are left over and the axis is short (16 x 1 over 900, 8 heads of
    // 128: 20.1 us, 21.2 with four; over 1900: 32.4, 29.8 with four and a join; 12 heads of 64 over 1900: 22.2 and 25.8;
    // 256 problems, 32 x 1 over 900: 27.4 and 23.5)
    const bool wide = heads <= 192 && p->max_kv <= (p->kv.head_dim == 64 ? 2048 : 1024);
    s.few = p->max_kv <= 128 ? 1 : wide ? 8 : 4;
  }
  const int tile_rows = s.few ? 16 * s.rt : TT_ROWS;
  s.n_tiles = (int)((rows + tile_rows - 1) / tile_rows);
  if (s.n_tiles < 1) s.n_tiles = 1;
  const int64_t wgs = (int64_t)s.n_tiles * heads;
  // Parts of a key axis (8 key heads of 128 where nothing else is said; "up to": ragged).  Few problems: 512 of them fill the
  // card once (2 x 4 over 131072, 16 problems: 180 us in 32 parts; 191 in 24, 185 in 48, 189 in 64), 1024 where key heads have
  // several row tiles, of which shorter sequences lack some (8 x up to 512 over up to 4512: 105 us in 4 parts, 120 whole, 120 in 8;
  // 8 x 64 over 8064, one tile: 71 and 59 the other way), and of 2048 keys at most where those are longer, as far as 4096 parts
  // go (11 x up to 142 over up to 25082: 155 us, 185 without, 612 whole; 6 x up to 366 over up to 38700 307, 960 whole; 4 x up to 334
  // over up to 12305, 32 heads of 64, 119, 139 without, 213 whole; but 18 x up to 200 over up to 36946 381 and 363, 2 x up to
  // 300 over up to 60300 250 and 231).  Many with one row tile a key head, as with one token for each of many sequences: parts
  // of 1024 keys, because lengths differ and the longest must not finish alone (64 x 1 over up to 16384: 403 us; 425 with parts
  // of 512, 405 with 2048, 417 with 4096, 477 whole), of 512 where the card would be filled twice at most (32 x 1 over up to 4000:
  // 56.6 us, 62.4 with parts of 1024, 59.6 whole; but equal lengths would rather stay whole: 32 x 1 over 1900 48.7 and 42.7); many
  // row tiles in fp32 as far as 4096 parts go, or else what is joined grows with tokens times keys (4 x 1024 over 9216: 4.95 ms
  // whole, 5.78 in 9 parts; 1 x 1500 over 20000, 8 heads of 96: 1.21 and 0.97 in 10).  Never below 256 keys (a part's (O, m, l) is
  // then 1/16 of the keys' bytes at most for 16 rows, 1/2 for the 128 of a row tile), nor below 1024 for the many rows of one
  // sequence, all there (1 x 643 over 645, 32 heads of 64: 16.9 us, 29.6 in three parts; 1 x 1024 over 8024: 61.8 and 73.1; but 4 x
  // up to 199 over up to 1559: 27.0, 32.9 in two parts of 832); none where there are no more than 512 (5 x 279 over 284: 14.7
  // us, 22.8 in two parts).
  int64_t keys = p->max_kv;
  if ((s.few == 0 || s.few == 4) && p->max_kv > 512) {
    const bool tiles = s.n_tiles > 1, ragged = p->n_seqs > 1;
    if (wgs < (s.few == 0 && tiles && ragged ? 1024 : 256)) {
      int64_t n = ((tiles && ragged ? 1024 : 512) + wgs / 2) / wgs;
      if (s.few == 0 && tiles && ragged) {
        const int64_t even = (p->max_kv + 2047) / 2048, room = 4096 / wgs;
        if (n < even) n = even < room ? even : (n < room ? room : n);
      }
      const int64_t least = s.few == 0 && tiles && (!ragged || wgs >= 256) ? 1024 : 256, most = (p->max_kv + least - 1) / least;
      if (n > most) n = most;
      keys = (p->max_kv + n - 1) / n;
    }
    if (s.few && wgs >= 256 && keys > 1024) {
      if (s.n_tiles == 1) {
        keys = wgs * ((keys + 1023) / 1024) <= (p->kv.head_dim == 64 ? 2048 : 1024) ? 512 : 1024;
      } else {
        int64_t n = (keys + 1023) / 1024;
        if (n > 4096 / wgs) n = 4096 / wgs;
        if (n > 1) keys = (keys + n - 1) / n;
      }
    }
    // no more than 1 GiB of parts (a token has room in every part, however short its own axis; 1024 single tokens, one of them
    // over 131072 keys, 8 key heads of 128: 977 us in 62 parts, 1772 in 128, 2 GiB)
    const int64_t part = (int64_t)p->n_tokens * p->n_heads * (p->kv.head_dim * 4 + 8), room = ((int64_t)1 << 30) / (part > 0 ? part : 1);
    if ((p->max_kv + keys - 1) / keys > room) keys = room > 1 ? (p->max_kv + room - 1) / room : p->max_kv;
  }
  s.split_keys = (int)((keys + 63) / 64 * 64);
  if (s.split_keys < 64) s.split_keys = 64;
  s.n_split = (int)((p->max_kv + s.split_keys - 1) / s.split_keys);
  if (s.n_split < 1) s.n_split = 1;
  s.ws_o = s.ws_ml = 0;
  if (s.n_split > 1) {
    const int64_t n = (int64_t)s.n_split * p->n_tokens * p->n_heads;
    s.ws_o = (int64_t)align_up((size_t)n * p->kv.head_dim * 4, 256);
    s.ws_ml = (int64_t)align_up((size_t)n * 8, 256);
  }
  return s;
}

static int check_paged_attention(const dark_paged_attention_args* p) {
  const char* who = "paged_attention";
  DARK_CHECK_ARG(p != nullptr, "%s: null arguments", who);
  DARK_TRY(check_paged_kv(&p->kv, who));
  DARK_CHECK_ARG(p->n_heads >= 1 && p->n_heads <= 4096 && p->n_heads % p->kv.n_kv_heads == 0,
                 "%s: n_heads=%d must be a multiple of n_kv_heads=%d", who, p->n_heads, p->kv.n_kv_heads);
  DARK_CHECK_ARG(p->n_tokens >= 0 && p->n_seqs >= 0 && p->table_width >= 0 && p->max_q >= 0 && p->max_kv >= 0 &&
                     p->n_tokens < (1 << 30), "%s: negative or too large size", who);
  DARK_CHECK_ARG((int64_t)p->table_width * p->kv.page_size < (1ll << 30) && p->max_kv < (1 << 30), "%s: 2^30 keys a sequence or more", who);
  const int64_t G = p->n_heads / p->kv.n_kv_heads;
  DARK_CHECK_ARG(p->n_tokens * G < (1ll << 31) - 128 && p->max_q * G < (1ll << 31) - 128, "%s: 2^31 rows of a key head or more", who);
  // (far beyond what a call is refused for; below, the plan's products of them stay within 64 bits)
  DARK_CHECK_ARG((double)p->n_seqs * p->kv.n_kv_heads * ((double)p->max_q * G / 16 + 1) < 1e12, "%s: too many rows", who);
  DARK_CHECK_ARG(p->scale == p->scale && fabsf(p->scale) < INFINITY, "%s: scale is not finite", who);
  return DARK_OK;
}

}  // namespace dark

using namespace dark;

extern "C" {

size_t dark_paged_attention_workspace_bytes(const dark_paged_attention_args* p) {
  if (check_paged_attention(p) != DARK_OK || p->n_tokens == 0 || p->n_seqs == 0) return 0;
  const PagedPlan s = plan_paged(p);
  return (size_t)(s.ws_o + s.ws_ml);
}

int dark_paged_attention(const dark_paged_attention_args* p, void* stream) {
  const char* who = "paged_attention";
  DARK_TRY(check_paged_attention(p));
  if (p->n_tokens == 0 || p->n_seqs == 0 || p->max_q == 0) return DARK_OK;
  const int es = p->kv.dtype == DARK_BF16 ? 2 : 4;
  DARK_CHECK_ARG(p->q && p->out && p->cu_q && p->kv_len && (p->block_table || p->table_width == 0), "%s: null pointer", who);
  DARK_CHECK_ARG(((uintptr_t)p->q & 15) == 0 && ((uintptr_t)p->out & 15) == 0 && p->q_ts * es % 16 == 0 && p->q_hs * es % 16 == 0 &&
                     p->o_ts * es % 16 == 0 && p->o_hs * es % 16 == 0,
                 "%s: pointers and strides must be multiples of 16 bytes", who);
  DARK_CHECK_ARG(p->table_stride >= p->table_width || p->n_seqs == 1, "%s: table_stride %lld < table_width %d", who, (long long)p->table_stride, p->table_width);
  hipStream_t st = (hipStream_t)stream;
  const PagedPlan s = plan_paged(p);
  const int unit = place_step(p->kv);
  DARK_CHECK_ARG(s.few || (double)p->kv.page_stride * (p->kv.n_pages > 0 ? p->kv.n_pages - 1 : 0) +
                              (double)p->kv.slot_stride * (p->kv.page_size - 1) < 4294967295.0 * (double)(1ll << unit),
                 "%s: the cache spans more than 2^32 times the power of two in its strides (%lld elements)", who, 1ll << unit);
  DARK_CHECK_ARG(s.ws_o + s.ws_ml == 0 || (p->workspace && ((uintptr_t)p->workspace & 15) == 0 && p->workspace_bytes >= s.ws_o + s.ws_ml),
                 "%s: workspace %lld < required %lld bytes (or not 16-byte aligned)", who, (long long)p->workspace_bytes, (long long)(s.ws_o + s.ws_ml));
  DARK_TRY(check_stream_device(st));
  PagedArgs a = {};
  a.q = p->q; a.k = p->kv.k; a.v = p->kv.v; a.out = p->out; a.lse = p->lse;
  a.table = p->block_table; a.cu_q = p->cu_q; a.kv_len = p->kv_len; a.q_index = p->q_index; a.kmask = p->key_mask;
  if (s.n_split > 1) {
    a.part_o = (float*)p->workspace;
    a.part_ml = (float*)((char*)p->workspace + s.ws_o);
  }
  a.q_ts = p->q_ts; a.q_hs = p->q_hs; a.o_ts = p->o_ts; a.o_hs = p->o_hs; a.table_stride = p->table_stride; a.mask_stride = p->mask_stride;
  a.page_stride = p->kv.page_stride; a.slot_stride = p->kv.slot_stride; a.head_stride = p->kv.head_stride;
  a.T = p->n_tokens; a.H = p->n_heads; a.Hk = p->kv.n_kv_heads; a.G = p->n_heads / p->kv.n_kv_heads; a.B = p->n_seqs;
  a.width = p->table_width; a.n_pages = p->kv.n_pages; a.page_log2 = __builtin_ctz((unsigned)p->kv.page_size);
  a.unit = unit; a.causal = p->causal != 0; a.n_split = s.n_split; a.split_keys = s.split_keys; a.n_tiles = s.n_tiles;
  const int64_t cap = (int64_t)p->table_width * p->kv.page_size;
  a.cap = (int)(cap < p->max_kv ? cap : p->max_kv);
  a.scale_log2 = p->scale * 1.44269504088896340736f;
  a.q_factor = 1.f;
  if (!s.few && !(a.scale_log2 > 0.f)) {
    a.q_factor = a.scale_log2 < 0.f ? -1.f : 0.f;
    a.scale_log2 = a.scale_log2 < 0.f ? -a.scale_log2 : 1.f;
  }
  const int64_t wgs = (int64_t)s.n_tiles * p->kv.n_kv_heads * p->n_seqs * s.n_split;
  DARK_CHECK_ARG(wgs < (1ll << 30), "%s: %lld workgroups", who, (long long)wgs);
  a.n_units = (int)wgs;
  a.max_q = p->max_q;
  // (not for short ones, which wait for the ranking: 60 x up to 200 over up to 700 91 us, 106 with it; nor for few, split evenly;
  // more than 64 sequences, a lane each, begin in the batch's order)
  a.by_length = s.few == 0 && p->n_seqs > 1 && p->n_seqs <= 64 && p->max_kv >= 1024 && (s.n_split == 1 || wgs >= 512 * (int64_t)s.n_split);

  a.by_hk = make_div(a.Hk); a.by_tiles = make_div(s.n_tiles); a.by_split = make_div(s.n_split); a.by_group = make_div(a.G);
  a.by_heads = make_div(a.H); a.by_rows = make_div((int)(s.n_split > 1 ? (int64_t)p->max_q * a.H : 1));
  const int64_t jrows = s.n_split > 1 ? (int64_t)p->n_seqs * p->max_q * p->n_heads : 0;   // (padded: a sequence's last may not be there)
  DARK_CHECK_ARG(jrows < (1ll << 31) - MAX_BLOCKS * 4, "%s: too many rows", who);
  // Units that share memory on one XCD: all heads and row tiles of a part, or else the row tiles of a key head -- where there
  // are enough such groups to even out what they hold, or eight heads that hold the same (16 sequences of up to 512 keys,
  // 12 heads, fp32: 26.3 us, 34.9 with the units dealt out one by one).
  int blocks = s.few == 1 ? (int)((wgs + 3) / 4) : (int)wgs;
  a.n_inner = 1;
  for (const bool all : {true, false}) {
    int inner = (all ? p->kv.n_kv_heads : 1) * s.n_tiles;
    if (all && !s.few) continue;    // (its units are ordered by heads first)
    if (s.few == 1) inner /= 4;     // (four units a workgroup)
    const int groups = inner > 1 ? cdiv(blocks, inner) : 0;
    if (groups >= 64 || (groups > 0 && !all && p->kv.n_kv_heads % 8 == 0)) {
      a.n_inner = inner;
      blocks = cdiv(groups, 8) * 8 * inner;
      break;
    }
  }
  a.by_inner = make_div(a.n_inner);
  auto launch = [&](auto kernel, int lds) {
    for (a.block0 = 0; a.block0 < blocks; a.block0 += MAX_BLOCKS)
      hipLaunchKernelGGL(kernel, dim3(blocks - a.block0 < MAX_BLOCKS ? blocks - a.block0 : MAX_BLOCKS), dim3(s.few == 8 ? 512 : 256), lds, st, a);
  };
  auto join = [&](auto kernel, int per) {   // `per` rows a workgroup
    for (int64_t row = 0; row < jrows; row += (int64_t)MAX_BLOCKS * per) {
      const int64_t n = (jrows - row + per - 1) / per;
      a.block0 = (int)row;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(n < MAX_BLOCKS ? n : MAX_BLOCKS)), dim3(256), 0, st, a);
    }
  };
#define DARK_JOIN(T, HDv)                                                 \
  if (s.n_split > 8) join(paged_join_kernel<T, HDv, 4>, 1);               \
  else if (s.n_split > 1) join(paged_join_kernel<T, HDv, 1>, 4)
#define DARK_PAGED_BF16(HDv)                                                                                        \
  do {                                                                                                              \
    if (s.few == 1) launch(paged_few_kernel<HDv, 1, ODD, false>, 0);                                                \
    else if (s.few == 4 && past) launch(paged_few_kernel<HDv, 4, ODD, HDv % 64 == 0>, 0);                           \
    else if (s.few == 4) launch(paged_few_kernel<HDv, 4, ODD, false>, 0);                                           \
    else if (s.few == 8) launch(paged_few_kernel<HDv, 8, ODD, false>, 0);                                           \
    else {                                                                                                          \
      constexpr int lds = 4 * TT_KEYS * HDv * 2;                                                                    \
      static SmemOptIn optin, optin_nt;                                                                             \
      if (past && s.n_tiles == 1) {                                                                                 \
        DARK_TRY(optin_nt.ensure((const void*)paged_tile_kernel<HDv, ODD, HDv % 64 == 0>, lds, st));                \
        launch(paged_tile_kernel<HDv, ODD, HDv % 64 == 0>, lds);                                                    \
      } else {                                                                                                      \
        DARK_TRY(optin.ensure((const void*)paged_tile_kernel<HDv, ODD, false>, lds, st));                           \
        launch(paged_tile_kernel<HDv, ODD, false>, lds);                                                            \
      }                                                                                                             \
    }                                                                                                               \
    DARK_JOIN(bf16_t, HDv);                                                                                         \
  } while (0)
#define DARK_PAGED_F32(HDv)                                                             \
  do {                                                                                  \
    if (s.rt == 1 && s.few == 1) launch(paged_f32_kernel<HDv, 1, 1, ODD>, 0);           \
    else if (s.rt == 1) launch(paged_f32_kernel<HDv, 4, 1, ODD>, 0);                    \
    else if constexpr (HDv > 64) {   /* (32 rows a wave, see plan_paged) */             \
      if (s.few == 1) launch(paged_f32_kernel<HDv, 1, 2, ODD>, 0);                      \
      else launch(paged_f32_kernel<HDv, 4, 2, ODD>, 0);                                 \
    }                                                                                   \
    DARK_JOIN(float, HDv);                                                              \
  } while (0)
  const int HD = p->kv.head_dim;
  // NT: keys that, with four layers of them, cannot stay in the 256 MB behind the L2s until they are read again go past the
  // caches (64 x 1 over up to 16384, 2.5 GB: 403 us, 439 without; 12 heads of 64: 289 and 326; 64 x 1 over 900, 118 MB, among other
  // layers': 42.6 and 47.7, again and again 42.0 and 40.1; 64 x 8 over 2000, one tile of rows: 88 us, 99 without) -- if their rows
  // are whole 128-byte lines (head_dim 96: 604 past them, 543 through them)
  const bool past = HD % 64 == 0 && (int64_t)p->n_seqs * a.cap * p->kv.n_kv_heads * HD * es * 2 > (int64_t)64 << 20;
  // rows of one tile see different keys only where a token's own place bounds them and a tile holds several tokens
  if (p->causal && p->max_q > 1) {
    constexpr bool ODD = true;
    if (p->kv.dtype == DARK_BF16) {
      if (HD == 64) DARK_PAGED_BF16(64); else if (HD == 96) DARK_PAGED_BF16(96); else DARK_PAGED_BF16(128);
    } else {
      if (HD == 64) DARK_PAGED_F32(64); else if (HD == 96) DARK_PAGED_F32(96); else DARK_PAGED_F32(128);
    }
  } else {
    constexpr bool ODD = false;
    if (p->kv.dtype == DARK_BF16) {
      if (HD == 64) DARK_PAGED_BF16(64); else if (HD == 96) DARK_PAGED_BF16(96); else DARK_PAGED_BF16(128);
    } else {
      if (HD == 64) DARK_PAGED_F32(64); else if (HD == 96) DARK_PAGED_F32(96); else DARK_PAGED_F32(128);
    }
  }
#undef DARK_JOIN
#undef DARK_PAGED_BF16
#undef DARK_PAGED_F32
  DARK_CHECK_LAUNCH();
  return DARK_OK;
}

}  // extern "C"
