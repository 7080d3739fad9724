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

#include "common.h"

namespace dark {

int check_paged_kv(const dark_paged_kv* kv, const char* who);
int check_stream_device(hipStream_t st);

struct PagedArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int32_t *table, *cu_q, *kv_len, *q_index;
  const uint8_t* kmask;
  float *part_o, *part_ml;     // [n_split][T][H][HD], [n_split][T][H][2]; null when n_split == 1
  int64_t q_ts, q_hs, o_ts, o_hs, table_stride, mask_stride, page_stride, slot_stride, head_stride;
  int32_t T, H, Hk, G, B, width, n_pages, page_log2, causal, n_split, split_keys, n_tiles, cap;
  float scale_log2;            // scale * log2(e)
};

// keys of a sequence: what it says, within the table and the caller's bound (hence within the mask's rows)
__device__ __forceinline__ int seq_len(const PagedArgs& a, int b) {
  const int len = a.kv_len[b];
  return len < 0 ? 0 : (len > a.cap ? a.cap : len);
}

template <typename T> struct PVec;
template <> struct PVec<bf16_t> { static constexpr int N = 8; typedef bf16x8 raw; };
template <> struct PVec<float> { static constexpr int N = 4; typedef f32x4 raw; };

// infinities and NaN of a V row that some row of the tile must not see (P = 0 there): 0 * inf would be NaN.  They are taken
// out of the product and counted by a second one over P's indicator: +inf 1, -inf 2^8, NaN 2^16 (at most 32 keys a tile).
__device__ __forceinline__ float odd_code(float x) {
  return x != x ? 65536.f : x == INFINITY ? 1.f : x == -INFINITY ? 256.f : 0.f;
}
__device__ __forceinline__ float odd_apply(float acc, float code) {
  if (code == 0.f) return acc;
  const int c = (int)code;
  const bool nan = c >= 65536, neg = (c & 0xff00) != 0, pos = (c & 0xff) != 0;
  return (nan || (neg && pos)) ? NAN : acc + (pos ? INFINITY : -INFINITY);
}

constexpr int PT_ROWS = 64, PT_KEYS = 32;   // rows of a workgroup (16 a wave), keys of a tile

template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_attn_kernel(const PagedArgs a) {
  constexpr int VEC = PVec<T>::N, LD = HD + VEC, CH = HD / VEC, NT = PT_KEYS / 16;
  constexpr bool kF32 = sizeof(T) == 4;
  typedef typename PVec<T>::raw raw;
  __shared__ __attribute__((aligned(16))) T Ks[PT_KEYS * LD];
  __shared__ __attribute__((aligned(16))) T Vs[PT_KEYS * LD];
  __shared__ float kbias[PT_KEYS];
  __shared__ int red[8];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, g = lane >> 4;
  int bid = blockIdx.x;
  const int split = bid % a.n_split; bid /= a.n_split;
  const int tile = bid % a.n_tiles; bid /= a.n_tiles;
  const int hk = bid % a.Hk, b = bid / a.Hk;
  int t0 = a.cu_q[b], t1 = a.cu_q[b + 1];
  t0 = t0 < 0 ? 0 : (t0 > a.T ? a.T : t0);
  t1 = t1 < t0 ? t0 : (t1 > a.T ? a.T : t1);
  const int64_t rows = (int64_t)(t1 - t0) * a.G;
  const int64_t row0 = (int64_t)tile * PT_ROWS;
  if (row0 >= rows) return;
  const int len = seq_len(a, b);

  const int64_t row = row0 + wave * 16 + li;
  const bool live = row < rows;
  const int tok = t0 + (int)((live ? row : row0) / a.G), hq = hk * a.G + (int)((live ? row : row0) % a.G);
  int seen = live ? len : 0;   // keys this lane's row may look at
  if (a.causal && live) {
    const int64_t last = a.q_index ? (int64_t)a.q_index[tok] : (int64_t)len - (t1 - tok);
    seen = last + 1 < len ? (last + 1 < 0 ? 0 : (int)(last + 1)) : len;
  }
  int hi = seen, lo = live ? seen : 0x7fffffff;   // largest and smallest bound of the workgroup's rows
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    hi = max(hi, __shfl_xor(hi, o, 64));
    lo = min(lo, __shfl_xor(lo, o, 64));
  }
  if (lane == 0) { red[wave] = hi; red[4 + wave] = lo; }
  __syncthreads();
  hi = max(max(red[0], red[1]), max(red[2], red[3]));
  lo = min(min(red[4], red[5]), min(red[6], red[7]));
  const int n_parts = len <= 0 ? 1 : (len + a.split_keys - 1) / a.split_keys;   // parts of this sequence that hold keys
  if (split >= n_parts) return;
  const int k_begin = split * a.split_keys;
  const int k_end = min(hi, split == a.n_split - 1 ? hi : k_begin + a.split_keys);

  // ---- this lane's share of the queries
  const T* qrow = (const T*)a.q + tok * a.q_ts + hq * a.q_hs;
  bf16x8 qb[HD / 32];
  float qf[HD / 4];
  if constexpr (kF32) {
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) qf[i] = qrow[i * 4 + g];
  } else {
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) qb[i] = *(const bf16x8*)(qrow + i * 32 + g * 8);
  }

  f32x4 O[HD / 16];
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) O[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const int32_t* tab = a.table + b * a.table_stride;
  const uint8_t* km = a.kmask ? a.kmask + b * a.mask_stride : nullptr;

  for (int k0 = k_begin; k0 < k_end; k0 += PT_KEYS) {
    // ---- K and V of the tile; a key that no row may use is stored as zeros
    int odd = 0;
    for (int it = tid; it < PT_KEYS * CH; it += 256) {
      const int j = it / CH, c = it - j * CH;
      const int key = k0 + j;
      raw rk = {}, rv = {};
      bool on = key < hi && (!km || km[key] != 0);
      int page = on ? tab[key >> a.page_log2] : -1;
      on = on && page >= 0 && page < a.n_pages;
      if (on) {
        const int64_t off = (int64_t)page * a.page_stride + (int64_t)(key & ((1 << a.page_log2) - 1)) * a.slot_stride +
                            (int64_t)hk * a.head_stride + c * VEC;
        rk = *(const raw*)((const T*)a.k + off);
        rv = *(const raw*)((const T*)a.v + off);
#pragma unroll
        for (int e = 0; e < VEC; ++e) odd |= !(fabsf((float)rv[e]) < INFINITY);
      }
      *(raw*)(Ks + j * LD + c * VEC) = rk;
      *(raw*)(Vs + j * LD + c * VEC) = rv;
      if (c == 0) kbias[j] = on ? 0.f : -INFINITY;
    }
    const bool partial = k0 + PT_KEYS > lo;   // some row does not see all of this tile
    odd = __syncthreads_or(odd && partial);

    f32x4 S[NT];
    float mx = m;
#pragma unroll
    for (int jt = 0; jt < NT; ++jt) {
      S[jt] = (f32x4){0.f, 0.f, 0.f, 0.f};
      const T* kr = Ks + (jt * 16 + li) * LD;
      if constexpr (kF32) {
#pragma unroll
        for (int i = 0; i < HD / 4; ++i) S[jt] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[i * 4 + g], qf[i], S[jt], 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < HD / 32; ++i)
          S[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)(kr + i * 32 + g * 8), qb[i], S[jt], 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = jt * 16 + 4 * g + r;
        const float s = (kbias[j] == 0.f && k0 + j < seen) ? S[jt][r] * a.scale_log2 : -INFINITY;
        S[jt][r] = s;
        mx = fmaxf(mx, s);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mz = mx == -INFINITY ? 0.f : mx;   // nothing seen yet: 2^(-inf - 0) = 0 everywhere
    const float alpha = __builtin_amdgcn_exp2f(m - mz);
    m = mx;
    float sum = 0.f;
#pragma unroll
    for (int jt = 0; jt < NT; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        S[jt][r] = __builtin_amdgcn_exp2f(S[jt][r] - mz);
        sum += S[jt][r];
      }
    l = l * alpha + sum;   // (this lane's keys only: the four lanes of a row are added up at the end)
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) O[i] *= alpha;

    // ---- O^T += V^T P^T
    if constexpr (kF32) {
#pragma unroll
      for (int dt = 0; dt < HD / 16; ++dt) {
        f32x4 code = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int jt = 0; jt < NT; ++jt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float v = Vs[(jt * 16 + 4 * g + r) * LD + dt * 16 + li];
            if (odd) {
              const float c = odd_code(v);
              code = __builtin_amdgcn_mfma_f32_16x16x4f32(c, S[jt][r] > 0.f ? 1.f : 0.f, code, 0, 0, 0);
              v = c == 0.f ? v : 0.f;
            }
            O[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, S[jt][r], O[dt], 0, 0, 0);
          }
        if (odd) {
#pragma unroll
          for (int r = 0; r < 4; ++r) O[dt][r] = odd_apply(O[dt][r], code[r]);
        }
      }
    } else {
      // P is rounded to bf16 for the matrix instruction (relative 2^-8 a weight, as the operands of every product here)
      bf16x8 pb, ind;
#pragma unroll
      for (int jj = 0; jj < 8; ++jj) {
        pb[jj] = (bf16_t)S[jj >> 2][jj & 3];
        ind[jj] = S[jj >> 2][jj & 3] > 0.f ? (bf16_t)1.f : (bf16_t)0.f;
      }
#pragma unroll
      for (int dt = 0; dt < HD / 16; ++dt) {
        // transposed LDS reads: each 16-lane group fetches a 4-key x 16-dim block row-wise and receives it column-wise
        typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
        const T* vrow = Vs + (4 * g + (li >> 2)) * LD + dt * 16 + 4 * (li & 3);
        const bf16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)vrow);
        const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(vrow + 16 * LD));
        bf16x8 v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
        f32x4 code = {0.f, 0.f, 0.f, 0.f};
        if (odd) {
          bf16x8 vc;
#pragma unroll
          for (int jj = 0; jj < 8; ++jj) {
            const float c = odd_code((float)v[jj]);
            vc[jj] = (bf16_t)c;
            v[jj] = c == 0.f ? v[jj] : (bf16_t)0.f;
          }
          code = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vc, ind, code, 0, 0, 0);
        }
        O[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb, O[dt], 0, 0, 0);
        if (odd) {
#pragma unroll
          for (int r = 0; r < 4; ++r) O[dt][r] = odd_apply(O[dt][r], code[r]);
        }
      }
    }
    __syncthreads();
  }

  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (!live) return;
  if (n_parts > 1 && a.n_split > 1) {
    const int64_t at = ((int64_t)split * a.T + tok) * a.H + hq;
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) *(f32x4*)(a.part_o + at * HD + dt * 16 + 4 * g) = O[dt];
    if (g == 0) { a.part_ml[at * 2] = m; a.part_ml[at * 2 + 1] = l; }
    return;
  }
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);   // (a NaN sum stays one)
  T* orow = (T*)a.out + tok * a.o_ts + hq * a.o_hs;
#pragma unroll
  for (int dt = 0; dt < HD / 16; ++dt)
    store4(orow + dt * 16 + 4 * g, make_float4(O[dt][0] * inv, O[dt][1] * inv, O[dt][2] * inv, O[dt][3] * inv));
  if (a.lse && g == 0) a.lse[(int64_t)tok * a.H + hq] = l > 0.f ? (m + log2f(l)) * 0.69314718055994530942f : (l == 0.f ? -INFINITY : l);
}

// ---- joins the parts of a split key axis: one wave per (token, head)
template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.T * a.H) return;
  const int tok = (int)(row / a.H), h = (int)(row - (int64_t)tok * a.H);
  // the token's sequence: the last b with cu_q[b] <= tok
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= tok) lo = mid; else hi = mid;
  }
  if (tok < a.cu_q[lo] || tok >= a.cu_q[lo + 1]) return;
  const int len = seq_len(a, lo);
  const int n_all = len <= 0 ? 1 : (len + a.split_keys - 1) / a.split_keys;
  if (n_all <= 1) return;                       // written whole by the first kernel
  const int n = min(n_all, a.n_split);
  const int64_t step = (int64_t)a.T * a.H;
  float m = -INFINITY;
  for (int s = 0; s < n; ++s) m = fmaxf(m, a.part_ml[(s * step + row) * 2]);
  const float mz = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[2] = {0.f, 0.f};
  for (int s = 0; s < n; ++s) {                 // (in order: the same bits every time)
    const int64_t at = s * step + row;
    const float f = __builtin_amdgcn_exp2f(a.part_ml[at * 2] - mz);
    l += a.part_ml[at * 2 + 1] * f;
    if (lane * 2 < HD) {
      const float2 v = *(const float2*)(a.part_o + at * HD + lane * 2);
      o[0] += v.x * f;
      o[1] += v.y * f;
    }
  }
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  if (lane * 2 < HD) {
    T* d = (T*)a.out + tok * a.o_ts + h * a.o_hs + lane * 2;
    d[0] = ElemTraits<T>::from_f32(o[0] * inv);
    d[1] = ElemTraits<T>::from_f32(o[1] * inv);
  }
  if (a.lse && lane == 0) a.lse[row] = l > 0.f ? (m + log2f(l)) * 0.69314718055994530942f : (l == 0.f ? -INFINITY : l);
}

struct PagedPlan {
  int n_tiles, n_split, split_keys;
  int64_t ws_o, ws_ml;   // bytes
};

static PagedPlan plan_paged(const dark_paged_attention_args* p) {
  PagedPlan s;
  const int G = p->n_heads / p->kv.n_kv_heads;
  s.n_tiles = (int)(((int64_t)p->max_q * G + PT_ROWS - 1) / PT_ROWS);
  if (s.n_tiles < 1) s.n_tiles = 1;
  const int64_t wgs = (int64_t)s.n_tiles * p->kv.n_kv_heads * p->n_seqs;
  // enough workgroups for 256 CUs x 4, parts of 256 keys at least
  int64_t want = (1024 + wgs - 1) / (wgs > 0 ? wgs : 1);
  const int64_t most = (p->max_kv + 255) / 256;
  if (want > most) want = most;
  if (want < 1) want = 1;
  s.split_keys = (int)(((p->max_kv + want - 1) / want + 63) / 64 * 64);
  if (s.split_keys < 64) s.split_keys = 64;
  s.n_split = (int)((p->max_kv + s.split_keys - 1) / s.split_keys);
  if (s.n_split < 1) s.n_split = 1;
  s.ws_o = s.ws_ml = 0;
  if (s.n_split > 1) {
    const int64_t rows = (int64_t)s.n_split * p->n_tokens * p->n_heads;
    s.ws_o = (int64_t)align_up((size_t)rows * p->kv.head_dim * 4, 256);
    s.ws_ml = (int64_t)align_up((size_t)rows * 8, 256);
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
  DARK_CHECK_ARG((int64_t)p->table_width * p->kv.page_size < (1ll << 31) - 64 && p->max_kv < 0x7fffffc0, "%s: more than 2^31 keys a sequence", who);
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
  a.causal = p->causal != 0; a.n_split = s.n_split; a.split_keys = s.split_keys; a.n_tiles = s.n_tiles;
  const int64_t cap = (int64_t)p->table_width * p->kv.page_size;
  a.cap = (int)(cap < p->max_kv ? cap : p->max_kv);
  a.scale_log2 = p->scale * 1.44269504088896340736f;
  const int64_t wgs = (int64_t)s.n_tiles * p->kv.n_kv_heads * p->n_seqs * s.n_split;
  DARK_CHECK_ARG(wgs < (1ll << 31), "%s: %lld workgroups", who, (long long)wgs);
  const dim3 grid((unsigned)wgs), block(256), jgrid((unsigned)(((int64_t)p->n_tokens * p->n_heads + 3) / 4));
#define DARK_PAGED(T, HDv)                                                                          \
  do {                                                                                              \
    hipLaunchKernelGGL((paged_attn_kernel<T, HDv>), grid, block, 0, st, a);                         \
    if (s.n_split > 1) hipLaunchKernelGGL((paged_join_kernel<T, HDv>), jgrid, block, 0, st, a);     \
  } while (0)
  const int HD = p->kv.head_dim;
  if (p->kv.dtype == DARK_BF16) {
    if (HD == 64) DARK_PAGED(bf16_t, 64); else if (HD == 96) DARK_PAGED(bf16_t, 96); else DARK_PAGED(bf16_t, 128);
  } else {
    if (HD == 64) DARK_PAGED(float, 64); else if (HD == 96) DARK_PAGED(float, 96); else DARK_PAGED(float, 128);
  }
#undef DARK_PAGED
  DARK_CHECK_LAUNCH();
  return DARK_OK;
}

}  // extern "C"
