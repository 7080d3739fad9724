// Per-head RMS norm + position rotation of queries and keys, and the placement of new tokens in the pages of a
// key / value cache.  The three jobs are one kernel: a token's rows (heads of q, k and v) are read once, normed and
// rotated in fp32 registers and stored once, wherever they belong.
//
// Bound by HBM: 2 * (heads read) * head_dim elements a token against ~8 flops an element.  A row is held by LPR lanes, lane
// c of them with the 16 bytes at chunk c of the row's first half and of its second half -- the two elements of every rotated
// pair in one lane -- so the 64 / LPR rows of a pass need no exchange but the norm's sum (log2(LPR) xor-shuffles).  A wave
// keeps its pass (which heads, hence its pointers, strides and weights) and walks over the tokens, the next one's rows,
// rotation and, one further, position on their way while it computes.  Read and written, each time other inputs: 16383 tokens
// x 40 fp32 heads of 128 in 121 us (5.6 TB/s), 512 x 46 x 16 bf16 heads of 96 in 34.7 us (4.2; a copy of as much takes 28.7),
// 1024 x 11 x 24 such heads into their pages in 21.7 us (4.8), 8 x up to 4096 x 48 bf16 heads of 128 with norms in 115 us (5.7);
// one token in 2.4 us.  Rows two tokens ahead instead of one: 39.7 us for 38.5, registers cost a wave.
#include "common.h"

namespace dark {

struct RowsArgs {
  // role 0 = q -> q_out, 1 = k -> k_out / pages, 2 = v -> pages
  const void* src[3];
  void* dst[3];
  const float* w[2];
  const float *cosT, *sinT;
  const int32_t* pos;
  const int64_t* slots;       // null: dst[1] is a plain [T, heads, HD] output
  int64_t src_ts[3], src_hs[3], dst_ts[3], dst_hs[3];
  int64_t page_stride, n_slots;
  int32_t T, h_end[3];        // rows [0, h_end[0]) are q heads, then k heads, then v heads
  int32_t max_pos, page_log2, n_pass, t_step, pos_period;   // passes of a token, tokens under way at a time
  float eps;
};

template <typename T> struct RowVec;
template <> struct RowVec<bf16_t> {
  static constexpr int N = 8;
  typedef bf16x8 raw;
  __device__ static __forceinline__ void up(const raw& r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)r[i];
  }
  __device__ static __forceinline__ raw down(const float (&f)[8]) {
    raw r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (bf16_t)f[i];
    return r;
  }
};
template <> struct RowVec<float> {
  static constexpr int N = 4;
  typedef f32x4 raw;
  __device__ static __forceinline__ void up(const raw& r, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = r[i];
  }
  __device__ static __forceinline__ raw down(const float (&f)[4]) { return (raw){f[0], f[1], f[2], f[3]}; }
};

// 1 / sqrt(x), off by one unit in the last place (the instruction takes small denormals for zeros)
__device__ __forceinline__ float rsqrt_of(float x) {
  const bool tiny = x < 0x1p-100f;
  return __builtin_amdgcn_rsqf(tiny ? x * 0x1p100f : x) * (tiny ? 0x1p50f : 1.f);
}

// Every condition around a load is the same for the whole wave: lanes without a row of their own load the last one, a side
// without weights the other's (a branch of its own around each had every load waited for: 512 x 46 40.8 us so, 36.5).
// ROPE = there are tables; asked at run time, the two ways of a row had its loads waited for (1024 x 11: 27.3 us so, 21.7).
template <typename T, int HD, bool NORM, bool ROPE, bool PAST>
__global__ __launch_bounds__(256) void head_rows_kernel(const RowsArgs a) {
  constexpr int N = RowVec<T>::N, HALF = HD / 2, CH = HALF / N;         // CH lanes hold a row
  constexpr int LPR = CH <= 4 ? 4 : CH <= 8 ? 8 : 16, RPP = 64 / LPR;   // lanes a row is given, rows of one pass
  typedef typename RowVec<T>::raw raw;
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));   // (weights may begin at any float)
  const int lane = threadIdx.x & 63;
  const int unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pass = unit % a.n_pass, step = a.t_step;
  int t = unit / a.n_pass;
  if (t >= step || t >= a.T) return;
  const int c = lane & (LPR - 1), r = pass * RPP + lane / LPR;
  const bool on = c < CH && r < a.h_end[2];
  const int rr = r < a.h_end[2] ? r : a.h_end[2] - 1, at = (c < CH ? c : 0) * N;
  const int role = rr < a.h_end[0] ? 0 : rr < a.h_end[1] ? 1 : 2;
  const int h = rr - (role == 0 ? 0 : role == 1 ? a.h_end[0] : a.h_end[1]);
  const int64_t src_ts = role == 0 ? a.src_ts[0] : role == 1 ? a.src_ts[1] : a.src_ts[2];
  const T* src = (const T*)(role == 0 ? a.src[0] : role == 1 ? a.src[1] : a.src[2]) +
                 h * (role == 0 ? a.src_hs[0] : role == 1 ? a.src_hs[1] : a.src_hs[2]) + t * src_ts + at;
  const bool paged = role > 0 && a.slots;
  const int64_t dst_ts = role == 0 ? a.dst_ts[0] : role == 1 ? a.dst_ts[1] : a.dst_ts[2];
  T* dst = (T*)(role == 0 ? a.dst[0] : role == 1 ? a.dst[1] : a.dst[2]) +
           h * (role == 0 ? a.dst_hs[0] : role == 1 ? a.dst_hs[1] : a.dst_hs[2]) + (paged ? 0 : t * dst_ts) + at;
  float w[2 * N];
  bool normed = false;
  if constexpr (NORM) {
    normed = role == 0 ? a.w[0] != nullptr : role == 1 && a.w[1] != nullptr;
    const float* wp = normed ? (role == 0 ? a.w[0] : a.w[1]) : (a.w[0] ? a.w[0] : a.w[1]);
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      *(f32x4*)(w + i) = *(const f32x4_any*)(wp + at + i);
      *(f32x4*)(w + N + i) = *(const f32x4_any*)(wp + HALF + at + i);
    }
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) w[i] = normed ? w[i] : 1.f;
  }
  raw x1, x2;
  float cs[N] = {}, sn[N] = {};
  int64_t slot = 0;
  auto position = [&](int tt) {
    if (!ROPE || tt >= a.T) return 0;
    const int q = a.pos ? a.pos[tt] : tt % a.pos_period;
    return q < 0 ? 0 : (q >= a.max_pos ? a.max_pos - 1 : q);
  };
  auto fetch = [&](int tt, int pp) {   // (src is at token tt)
    x1 = *(const raw*)src;
    x2 = *(const raw*)(src + HALF);
    if (a.slots) slot = a.slots[tt];
    if constexpr (ROPE) {
      const float* cp = a.cosT + (int64_t)pp * HALF + at;
      const float* sp = a.sinT + (int64_t)pp * HALF + at;
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        *(f32x4*)(cs + i) = *(const f32x4*)(cp + i);
        *(f32x4*)(sn + i) = *(const f32x4*)(sp + i);
      }
    }
  };
  fetch(t, position(t));
  int p_next = position(t + step);
  while (true) {
    // this token's rows and rotation, then its successor's take their place
    raw y1 = x1, y2 = x2;
    float cc[N], ss[N];
#pragma unroll
    for (int i = 0; i < N; ++i) { cc[i] = cs[i]; ss[i] = sn[i]; }
    const int64_t to = slot;
    const int tn = t + step;
    if (tn < a.T) {
      src += step * src_ts;
      fetch(tn, p_next);
      p_next = position(tn + step);
    }
    float f1[N], f2[N], o1[N], o2[N];
    RowVec<T>::up(y1, f1);
    RowVec<T>::up(y2, f2);
    if constexpr (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) sum += f1[i] * f1[i] + f2[i] * f2[i];
      if (CH < LPR && c >= CH) sum = 0.f;   // (lanes without a chunk of the row)
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
      const float inv = normed ? rsqrt_of(sum * (1.f / HD) + a.eps) : 1.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        f1[i] *= inv * w[i];
        f2[i] *= inv * w[N + i];
      }
    }
    // (without tables no turn by an angle of 0: an infinity times its sine would make the other half's element a NaN)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o1[i] = ROPE ? f1[i] * cc[i] - f2[i] * ss[i] : f1[i];
      o2[i] = ROPE ? f2[i] * cc[i] + f1[i] * ss[i] : f2[i];
    }
    if (role < 2 && (ROPE || normed)) {   // (values, and rows with neither norm nor rotation, are carried as they are)
      y1 = RowVec<T>::down(o1);
      y2 = RowVec<T>::down(o2);
    }
    const bool kept = !paged || (to >= 0 && to < a.n_slots);
    if (on && kept) {
      T* d = dst + (paged ? (to >> a.page_log2) * a.page_stride + (to & (((int64_t)1 << a.page_log2) - 1)) * dst_ts : 0);
      if constexpr (PAST) {
        __builtin_nontemporal_store(y1, (raw*)d);
        __builtin_nontemporal_store(y2, (raw*)(d + HALF));
      } else {
        *(raw*)d = y1;
        *(raw*)(d + HALF) = y2;
      }
    }
    if (tn >= a.T) return;
    if (!paged) dst += step * dst_ts;
    t = tn;
  }
}

static bool aligned16(const void* p, int64_t s0, int64_t s1, int es) {
  return ((uintptr_t)p & 15) == 0 && (s0 * es) % 16 == 0 && (s1 * es) % 16 == 0;
}

// a stream of another device than the current one would run there on this device's pointers
int check_stream_device(hipStream_t st) {
  if (st == nullptr) return DARK_OK;
  int cur = 0;
  hipDevice_t sdev = 0;
  DARK_CHECK_HIP(hipGetDevice(&cur));
  DARK_CHECK_HIP(hipStreamGetDevice(st, &sdev));
  DARK_CHECK_ARG((int)sdev == cur, "stream belongs to device %d but device %d is current (make the tensors' device current "
                 "before calling)", (int)sdev, cur);
  return DARK_OK;
}

int check_paged_kv(const dark_paged_kv* kv, const char* who) {
  DARK_CHECK_ARG(kv->dtype == DARK_F32 || kv->dtype == DARK_BF16, "%s: bad dtype %d", who, kv->dtype);
  const int es = kv->dtype == DARK_BF16 ? 2 : 4;
  DARK_CHECK_ARG(kv->head_dim == 64 || kv->head_dim == 96 || kv->head_dim == 128, "%s: head_dim=%d must be 64, 96 or 128", who, kv->head_dim);
  DARK_CHECK_ARG(kv->n_kv_heads >= 1 && kv->n_kv_heads <= 4096, "%s: n_kv_heads=%d", who, kv->n_kv_heads);
  DARK_CHECK_ARG(kv->page_size >= 1 && kv->page_size <= 4096 && (kv->page_size & (kv->page_size - 1)) == 0,
                 "%s: page_size=%d must be a power of two up to 4096", who, kv->page_size);
  DARK_CHECK_ARG(kv->n_pages >= 0, "%s: n_pages=%d", who, kv->n_pages);
  DARK_CHECK_ARG(kv->n_pages == 0 || (kv->k && kv->v), "%s: null cache pointer", who);
  DARK_CHECK_ARG(kv->page_stride >= 0 && kv->slot_stride >= 0 && kv->head_stride >= 0, "%s: negative cache stride", who);
  DARK_CHECK_ARG(aligned16(kv->k, kv->page_stride, kv->slot_stride, es) && aligned16(kv->v, kv->head_stride, 0, es),
                 "%s: the cache's pointers and strides must be multiples of 16 bytes", who);
  return DARK_OK;
}

static int launch_head_rows(RowsArgs& a, int dtype, int HD, hipStream_t st) {
  DARK_TRY(check_stream_device(st));
  const int ch = HD / 2 / (dtype == DARK_BF16 ? 8 : 4), rpp = 64 / (ch <= 4 ? 4 : ch <= 8 ? 8 : 16);
  a.n_pass = cdiv(a.h_end[2], rpp);
  // Tokens a wave walks over: some 32768 waves in all, so that the card sweeps over the tokens in order (8 x up to 4096, 48 heads:
  // 116 us; 119 with 16384 waves, 135 with 8192), but two at least where there are enough and weights to fetch first (512 x 46:
  // 34.8 us, 39.8 with one, 36.1 with three)
  const bool norm = a.w[0] || a.w[1];
  const int64_t units = (int64_t)a.T * a.n_pass;
  int64_t walk = norm && units >= 16384 ? 2 : 1;
  if (walk < (units + 16384) / 32768) walk = (units + 16384) / 32768;
  a.t_step = (int)((a.T + walk - 1) / walk);
  // rows that the 256 MB behind the L2s cannot hold for their reader are written past them (16383 tokens x 40 fp32 heads of
  // 128, 0.7 GB moved: 120 us, 129 without; 512 x 46 x 16 bf16 heads of 96, 72 MB: 31.0 and 34.8, but then they are there to
  // be read)
  const bool past = (int64_t)a.T * a.h_end[2] * HD * (dtype == DARK_BF16 ? 2 : 4) > (int64_t)256 << 20;
  const dim3 grid((unsigned)cdiv(a.t_step * a.n_pass, 4)), block(256);
#define DARK_ROWS_AT(T, HDv, ROPE)                                                                               \
  do {                                                                                                           \
    if (norm && past) hipLaunchKernelGGL((head_rows_kernel<T, HDv, true, ROPE, true>), grid, block, 0, st, a);   \
    else if (norm) hipLaunchKernelGGL((head_rows_kernel<T, HDv, true, ROPE, false>), grid, block, 0, st, a);     \
    else if (past) hipLaunchKernelGGL((head_rows_kernel<T, HDv, false, ROPE, true>), grid, block, 0, st, a);     \
    else hipLaunchKernelGGL((head_rows_kernel<T, HDv, false, ROPE, false>), grid, block, 0, st, a);              \
  } while (0)
#define DARK_ROWS(T, HDv)                                                                    \
  do {                                                                                       \
    if (a.cosT) DARK_ROWS_AT(T, HDv, true); else DARK_ROWS_AT(T, HDv, false);                \
  } while (0)
  if (dtype == DARK_BF16) {
    if (HD == 64) DARK_ROWS(bf16_t, 64); else if (HD == 96) DARK_ROWS(bf16_t, 96); else DARK_ROWS(bf16_t, 128);
  } else {
    if (HD == 64) DARK_ROWS(float, 64); else if (HD == 96) DARK_ROWS(float, 96); else DARK_ROWS(float, 128);
  }
#undef DARK_ROWS
#undef DARK_ROWS_AT
  DARK_CHECK_LAUNCH();
  return DARK_OK;
}

static int check_rows(const char* who, int dtype, int T, int Hq, int Hk, int HD, float eps) {
  DARK_CHECK_ARG(dtype == DARK_F32 || dtype == DARK_BF16, "%s: bad dtype %d", who, dtype);
  DARK_CHECK_ARG(HD == 64 || HD == 96 || HD == 128, "%s: head_dim=%d must be 64, 96 or 128", who, HD);
  DARK_CHECK_ARG(T >= 0 && T < (1 << 30), "%s: n_tokens=%d", who, T);
  DARK_CHECK_ARG(Hq >= 0 && Hq <= 4096 && Hk >= 0 && Hk <= 4096, "%s: heads %d / %d", who, Hq, Hk);
  DARK_CHECK_ARG(eps >= 0.f, "%s: eps=%g", who, (double)eps);
  return DARK_OK;
}

}  // namespace dark

using namespace dark;

extern "C" {

int dark_qk_norm_rope(const dark_qk_norm_rope_args* p, void* stream) {
  const char* who = "qk_norm_rope";
  DARK_CHECK_ARG(p != nullptr, "%s: null arguments", who);
  DARK_TRY(check_rows(who, p->dtype, p->n_tokens, p->n_heads, p->n_kv_heads, p->head_dim, p->eps));
  if (p->n_tokens == 0 || p->n_heads + p->n_kv_heads == 0) return DARK_OK;
  const int es = p->dtype == DARK_BF16 ? 2 : 4;
  DARK_CHECK_ARG((p->n_heads == 0 || (p->q && p->q_out)) && (p->n_kv_heads == 0 || (p->k && p->k_out)), "%s: null pointer", who);
  DARK_CHECK_ARG((p->rope_cos == nullptr) == (p->rope_sin == nullptr), "%s: rope_cos and rope_sin go together", who);
  DARK_CHECK_ARG(!p->rope_cos || ((p->pos || p->pos_period > 0) && p->max_pos >= 1), "%s: a rotation needs positions and a table", who);
  DARK_CHECK_ARG(aligned16(p->q, p->q_ts, p->q_hs, es) && aligned16(p->k, p->k_ts, p->k_hs, es) &&
                     aligned16(p->q_out, p->qo_ts, p->qo_hs, es) && aligned16(p->k_out, p->ko_ts, p->ko_hs, es),
                 "%s: pointers and strides must be multiples of 16 bytes", who);
  RowsArgs a = {};
  a.src[0] = p->q; a.src[1] = p->k; a.dst[0] = p->q_out; a.dst[1] = p->k_out;
  a.w[0] = p->q_w; a.w[1] = p->k_w; a.cosT = p->rope_cos; a.sinT = p->rope_sin; a.pos = p->pos;
  a.src_ts[0] = p->q_ts; a.src_hs[0] = p->q_hs; a.src_ts[1] = p->k_ts; a.src_hs[1] = p->k_hs;
  a.dst_ts[0] = p->qo_ts; a.dst_hs[0] = p->qo_hs; a.dst_ts[1] = p->ko_ts; a.dst_hs[1] = p->ko_hs;
  a.T = p->n_tokens; a.max_pos = p->max_pos; a.eps = p->eps; a.pos_period = p->pos_period > 0 ? p->pos_period : 1;
  a.h_end[0] = p->n_heads; a.h_end[1] = a.h_end[2] = p->n_heads + p->n_kv_heads;
  return launch_head_rows(a, p->dtype, p->head_dim, (hipStream_t)stream);
}

int dark_kv_append(const dark_kv_append_args* p, void* stream) {
  const char* who = "kv_append";
  DARK_CHECK_ARG(p != nullptr, "%s: null arguments", who);
  DARK_TRY(check_paged_kv(&p->kv, who));
  DARK_TRY(check_rows(who, p->kv.dtype, p->n_tokens, p->n_heads, p->kv.n_kv_heads, p->kv.head_dim, p->eps));
  if (p->n_tokens == 0) return DARK_OK;
  const int es = p->kv.dtype == DARK_BF16 ? 2 : 4;
  DARK_CHECK_ARG(p->k && p->v && p->slots, "%s: null pointer", who);
  DARK_CHECK_ARG(p->kv.n_pages == 0 || p->kv.k != p->kv.v, "%s: k and v would go to the same memory", who);
  DARK_CHECK_ARG((p->q == nullptr) == (p->q_out == nullptr) && (p->n_heads == 0 || p->q), "%s: q and q_out go together", who);
  DARK_CHECK_ARG((p->rope_cos == nullptr) == (p->rope_sin == nullptr), "%s: rope_cos and rope_sin go together", who);
  DARK_CHECK_ARG(!p->rope_cos || (p->pos && p->max_pos >= 1), "%s: a rotation needs positions and a table", who);
  DARK_CHECK_ARG(aligned16(p->q, p->q_ts, p->q_hs, es) && aligned16(p->k, p->k_ts, p->k_hs, es) &&
                     aligned16(p->v, p->v_ts, p->v_hs, es) && aligned16(p->q_out, p->qo_ts, p->qo_hs, es),
                 "%s: pointers and strides must be multiples of 16 bytes", who);
  RowsArgs a = {};
  const int Hq = p->q ? p->n_heads : 0, Hk = p->kv.n_kv_heads;
  a.src[0] = p->q; a.src[1] = p->k; a.src[2] = p->v;
  a.dst[0] = p->q_out; a.dst[1] = p->kv.k; a.dst[2] = p->kv.v;
  a.w[0] = p->q_w; a.w[1] = p->k_w; a.cosT = p->rope_cos; a.sinT = p->rope_sin; a.pos = p->pos; a.slots = p->slots;
  a.src_ts[0] = p->q_ts; a.src_hs[0] = p->q_hs; a.src_ts[1] = p->k_ts; a.src_hs[1] = p->k_hs; a.src_ts[2] = p->v_ts; a.src_hs[2] = p->v_hs;
  a.dst_ts[0] = p->qo_ts; a.dst_hs[0] = p->qo_hs;
  a.dst_ts[1] = a.dst_ts[2] = p->kv.slot_stride; a.dst_hs[1] = a.dst_hs[2] = p->kv.head_stride;
  a.page_stride = p->kv.page_stride; a.n_slots = (int64_t)p->kv.n_pages * p->kv.page_size;
  a.T = p->n_tokens; a.max_pos = p->max_pos; a.eps = p->eps; a.page_log2 = __builtin_ctz((unsigned)p->kv.page_size);
  a.h_end[0] = Hq; a.h_end[1] = Hq + Hk; a.h_end[2] = Hq + 2 * Hk;
  return launch_head_rows(a, p->kv.dtype, p->kv.head_dim, (hipStream_t)stream);
}

}  // extern "C"
