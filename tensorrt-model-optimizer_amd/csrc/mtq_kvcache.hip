// mtq_kvcache.hip — a KV cache held in 4 bits (NVFP4), in pages, and the attention that reads it.
//
// A row (one token of one KV head, head_dim values) is D / 2 bytes of E2M1 codes (even column low)
// and D / 16 E4M3 scales; with the tensor's gs = RN(amax / 2688) a value is
//   code * RN(scale * gs),   scale = e4m3(min(RN(max|x| / RN(6 gs)), 448)) of its 16 columns,
// code = e2m1(RN(x / RN(scale * gs))): element for element the NVFP4 fake quant that the K/V
// quantizers simulate (mtq_nvfp4_fake_quant), whose blocks with scale * gs < 1e-5 come out as zeros
// (stored here as scale 0, codes 0).
//
// Position p of sequence b lives on page table[b][p / page_size], place p % page_size.  The new
// tokens of a call are the last len_q[b] of its len_k[b] positions; token i of sequence b is row
// start[b] + i of q / k / v / o.  A table entry outside the cache's pages stands for no page: rows
// for it are dropped, reads give zeros, the attention does not see its keys.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "mtq_amd.h"
#include "mtq_device.hpp"

using namespace mtq;

namespace mtq {
int host_check_launch();
int host_num_cus();
}

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

inline bool al16p(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr float kNegInf = -__builtin_inff();
// probabilities are held as 2^kShift exp2(x - m), m at most kSlack below the largest x so far
constexpr float kShift = 6.0f, kSlack = 8.0f;

struct Cache {
  uint8_t *data[2], *scale[2];                        // K, V
  int64_t d_page[2], d_head[2], d_tok[2];             // byte strides of the codes
  int64_t s_page[2], s_head[2], s_tok[2];             // ... and of the scales
  const float *amax[2];
  const int32_t *table, *start, *len_q, *len_k;
  int64_t table_stride;
  int table_cols, num_pages, shift, hkv, head_dim;
};

__device__ __forceinline__ float global_scale_of(const float *amax) {
  const float gs = div_rn(*amax, 2688.0f, 1.0f / 2688.0f);
  return gs > 0.f ? gs : 1e-12f;
}

// the page of position pos, -1 where there is none: the table's entry, which is loaded without a branch
// (page_entry) so that a loop can have it in flight, and what it says (page_at)
__device__ __forceinline__ int page_entry(const Cache &c, int b, int pos) {
  const int slot = pos >> c.shift;
  return c.table[(int64_t)b * c.table_stride + ((uint32_t)slot < (uint32_t)c.table_cols ? slot : 0)];
}
__device__ __forceinline__ int page_at(const Cache &c, int pos, int entry) {
  return (uint32_t)(pos >> c.shift) < (uint32_t)c.table_cols && (uint32_t)entry < (uint32_t)c.num_pages ? entry : -1;
}
__device__ __forceinline__ int page_of(const Cache &c, int b, int pos) { return page_at(c, pos, page_entry(c, b, pos)); }

// ---- rows into pages and back -------------------------------------------------------------------
// A lane takes 8 columns of a row, two lanes a block, so that 16-bit rows move in whole 16-byte pieces of
// neighbouring lanes.  A workgroup takes tokens of one head where the call has them (2^lt of them, then heads):
// in the cache's layout these lie behind each other, 16 of them at head_dim 128 being 1 KiB of codes and a
// line of scales, while k and v are met in pieces of a row (256 bytes there).  Bound by HBM (16 + 4.5 bytes a
// lane): 3.7 TB/s each way at the size below.
struct RowArgs {
  Cache c;
  void *x[2];             // k, v
  int64_t xt[2], xh[2];   // element strides (token, head)
  int64_t rows;
  int lt, passes;
  int max_len;  // tokens of a sequence from max_len on are left out, also where its last pass reaches them
};
// Tokens of a lane in flight at once, and whether it loops over more.  us for the prompts of 7 sequences, 27954 tokens
// of 8 heads of 128 (147 MB each way), each call for itself: append, 1 / 2 / 4 tokens, looping with at most 48
// workgroups a CU 39 / 40 / 46, without a loop 2 / 4 tokens 44 / 47; read 1 / 2 / 4 / 8 tokens 50 / 45 / 39 / 39.  (Right
// behind the append, whose codes are still in the caches, the read takes 26 to 30.)
constexpr int kAppendAhead = 2, kReadAhead = 4, kAppendWgs = 48;

// what a lane works on: false where there is none of it
struct RowLane {
  int kv, h, col, first, step, end;  // tokens first, first + step, .. below end
};
template <int AHEAD> __device__ __forceinline__ bool row_lane(const RowArgs &a, int lq, RowLane &r) {
  const int ll = 28 - __builtin_clz(a.c.head_dim), lr = 8 - ll;  // 2^ll lanes a row, 2^lr rows a pass
  const int row = threadIdx.x >> ll;
  const int kvh = (blockIdx.z << (lr - a.lt)) + (row >> a.lt);
  r.col = 8 * (threadIdx.x & ((1 << ll) - 1));
  r.kv = kvh >= a.c.hkv ? 1 : 0;
  r.h = kvh - r.kv * a.c.hkv;
  r.step = 1 << a.lt;
  r.first = (blockIdx.x * a.passes * AHEAD << a.lt) + (row & (r.step - 1));
  const int64_t end = (int64_t)(blockIdx.x + 1) * a.passes * AHEAD << a.lt;
  lq = lq < a.max_len ? lq : a.max_len;
  r.end = end < lq ? (int)end : lq;
  return kvh < 2 * a.c.hkv;
}

template <typename T, bool VEC> struct Row8 {
  static constexpr int NV = 8 / Vec<T>::N;
  Vec<T> v[NV];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = ldg_vec(p + i * Vec<T>::N);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i / Vec<T>::N].e[i % Vec<T>::N] = p[i];
    }
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NV; ++i) stg_vec(p + i * Vec<T>::N, v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = v[i / Vec<T>::N].e[i % Vec<T>::N];
    }
  }
  __device__ __forceinline__ T &operator[](int i) { return v[i / Vec<T>::N].e[i % Vec<T>::N]; }
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void cache_append_kernel(RowArgs a) {
  const Cache &c = a.c;
  const int b = blockIdx.y, lq = c.len_q[b], lk = c.len_k[b];
  RowLane r;
  if (!row_lane<kAppendAhead>(a, lq, r)) return;
  const int64_t start = c.start[b];
  const int kv = r.kv;
  const float g = global_scale_of(kv ? c.amax[1] : c.amax[0]), six = 6.0f * g, rsix = 1.0f / six;
  const T *x = reinterpret_cast<const T *>(kv ? a.x[1] : a.x[0]) + r.h * (kv ? a.xh[1] : a.xh[0]) + r.col;
  uint8_t *d = (kv ? c.data[1] : c.data[0]) + r.h * (kv ? c.d_head[1] : c.d_head[0]) + (r.col >> 1);
  uint8_t *s = (kv ? c.scale[1] : c.scale[0]) + r.h * (kv ? c.s_head[1] : c.s_head[0]) + (r.col >> 4);
  const int64_t xt = kv ? a.xt[1] : a.xt[0], dp = kv ? c.d_page[1] : c.d_page[0], dt = kv ? c.d_tok[1] : c.d_tok[0];
  const int64_t sp = kv ? c.s_page[1] : c.s_page[0], st = kv ? c.s_tok[1] : c.s_tok[0];
  for (int i0 = r.first; i0 < r.end; i0 += kAppendAhead * r.step) {
    Row8<T, VEC> in[kAppendAhead];
    int page[kAppendAhead];
#pragma unroll
    for (int u = 0; u < kAppendAhead; ++u) {
      const int i = i0 + u * r.step;
      const int64_t row = start + i;
      const bool ok = i < r.end && row >= 0 && row < a.rows;
      if (ok) in[u].load(x + row * xt);
      page[u] = ok ? page_of(c, b, lk - lq + i) : -1;
    }
#pragma unroll
    for (int u = 0; u < kAppendAhead; ++u) {
      if (page[u] < 0) continue;  // both lanes of a block alike
      float v[8], m = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = Elem<T>::ld(in[u][j]);
        m = max_skip_nan(m, v[j]);
      }
      m = fmaxf(m, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(m), 0xB1, 0xf, 0xf, true)));  // lane ^ 1
      float s8 = div_rn(m, six, rsix);
      s8 = s8 < kE4M3Max ? s8 : kE4M3Max;
      int sb = __builtin_amdgcn_cvt_pk_fp8_f32(s8, s8, 0, false) & 0xff;
      const float q = __builtin_amdgcn_cvt_f32_fp8(sb, 0) * g;
      uint32_t w = 0;
      if (q >= 1e-5f) {
        const float rq = 1.0f / q;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float t = fminf(div_rn(fabsf(v[j]), q, rq), 6.0f);  // inf and NaN: 6
          v[j] = v[j] >= 0.f ? t : -t;
        }
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.0f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.0f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.0f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.0f, 3);
      } else {
        sb = 0;
      }
      const int64_t at = (lk - lq + i0 + u * r.step) & ((1 << c.shift) - 1);
      *reinterpret_cast<uint32_t *>(d + page[u] * dp + at * dt) = w;
      if (!(r.col & 8)) s[page[u] * sp + at * st] = (uint8_t)sb;
    }
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void cache_read_kernel(RowArgs a) {
  const Cache &c = a.c;
  const int b = blockIdx.y, lq = c.len_q[b], lk = c.len_k[b];
  RowLane r;
  if (!row_lane<kReadAhead>(a, lq, r)) return;
  const int64_t start = c.start[b];
  const int kv = r.kv;
  const float g = global_scale_of(kv ? c.amax[1] : c.amax[0]);
  T *x = reinterpret_cast<T *>(kv ? a.x[1] : a.x[0]) + r.h * (kv ? a.xh[1] : a.xh[0]) + r.col;
  const uint8_t *d = (kv ? c.data[1] : c.data[0]) + r.h * (kv ? c.d_head[1] : c.d_head[0]) + (r.col >> 1);
  const uint8_t *s = (kv ? c.scale[1] : c.scale[0]) + r.h * (kv ? c.s_head[1] : c.s_head[0]) + (r.col >> 4);
  const int64_t xt = kv ? a.xt[1] : a.xt[0], dp = kv ? c.d_page[1] : c.d_page[0], dt = kv ? c.d_tok[1] : c.d_tok[0];
  const int64_t sp = kv ? c.s_page[1] : c.s_page[0], st = kv ? c.s_tok[1] : c.s_tok[0];
  uint32_t w[kReadAhead];
  int sb[kReadAhead];
#pragma unroll
  for (int u = 0; u < kReadAhead; ++u) {
    const int i = r.first + u * r.step, pos = lk - lq + i, page = i < r.end ? page_of(c, b, pos) : -1;
    const int64_t at = pos & ((1 << c.shift) - 1);
    w[u] = 0, sb[u] = 0;
    if (page >= 0) {
      w[u] = *reinterpret_cast<const uint32_t *>(d + page * dp + at * dt);
      sb[u] = s[page * sp + at * st];
    }
  }
#pragma unroll
  for (int u = 0; u < kReadAhead; ++u) {
    const int i = r.first + u * r.step;
    const int64_t row = start + i;
    if (i >= r.end || row < 0 || row >= a.rows) continue;
    const float q = __builtin_amdgcn_cvt_f32_fp8(sb[u], 0) * g;
    Row8<T, VEC> o;
    auto pair = [&](auto e, int j) { o[j] = Elem<T>::st(e[0] * q), o[j + 1] = Elem<T>::st(e[1] * q); };
    pair(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 0), 0);
    pair(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 1), 2);
    pair(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 2), 4);
    pair(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], 1.0f, 3), 6);
    o.store(x + row * xt);
  }
}

// ---- attention -----------------------------------------------------------------------------------
// o = softmax(sm_scale q k^T) v over the pages of a sequence, G query heads to a KV head.
//
// A row is (query token, head of the group); 16 rows are one column block of the matrix
// instructions.  Scores are computed transposed, S^T = K q^T (v_mfma_f32_16x16x32_f16: lane
// (c = lane & 15, g = lane >> 4) holds row c's scores of keys 4 g .. 4 g + 3), so a row's maximum and
// sum are in-lane work and two exchanges, and the probabilities are already the second operand of
// O^T += V^T P^T, whose contraction takes the keys in the order the lanes hold them.
//   K: lane (t = lane & 15, g) loads the codes of key t's columns [D / 4 g, D / 4 (g + 1)) and turns
//      them into fp16 products code * scale: exact (at most 6 significant bits, 2^-10 .. 2688); gs goes
//      into the softmax factor.  The contraction over head_dim takes the columns in that order, q too.
//   q: to fp16 with a power of two of its row that puts its largest value into [2^14, 2^15): 8
//      (bf16) or 11 (fp16) bits stay exact down to 2^-28 of it.
//   V: the same products, through LDS rows that ds_read_b64_tr_b16 reads transposed.
//   P: fp16, 2^6 exp2(x - m), off by 2^-12 of each weight and a normal number down to 2^-20 of the
//      largest; the row sum carries the same 2^6.  m follows the running maximum only where a key exceeds it
//      by 2^8 (weights then reach 2^14, inside fp16): most steps neither exchange maxima nor rescale O.
// Sums and the accumulators are fp32.
//
// A wave takes 32 keys at a time, the waves of a workgroup every fourth 32 keys, and keep statistics
// of their own, joined through LDS at the end (in wave order).  Where there are few sequences the
// keys are cut into splits; their partial results are joined by a second small kernel, in order.
// Bound by the cache's bytes: 64 single tokens over up to 16384 keys, 32 / 8 heads of 128: 163 us (717 MB, 4.4
// TB/s; matrix cores busy 14 % of the time); head_dim 64: 110 (3.2 TB/s), 256 with 16 / 4 heads: 179 (4.0).
struct AttnArgs {
  Cache c;
  const void *q;
  void *o;
  float *part;  // the splits' rows: o, m, l
  int64_t qt, qh, ot, oh, rows;
  int group, causal, splits, chunk, tiles, part_tiles, batch;  // tiles: of the kernel's rows, part_tiles: of 16
  int max_q;  // new tokens of a sequence that the grid and `part` have room for
  float sm_log2;  // softmax_scale * log2(e)
};

// where a row of a split's results lies: [splits][batch][hkv][16-row tiles][16][D + 4]
template <int D> __device__ __forceinline__ int64_t part_row(const AttnArgs &a, int split, int b, int kvh, int row) {
  return (((((int64_t)split * a.batch + b) * a.c.hkv + kvh) * a.part_tiles + (row >> 4)) * 16 + (row & 15)) * (D + 4);
}

// rows of a sequence of lq new tokens: those past max_q, should the device hold a longer length, are left out
__device__ __forceinline__ int attn_rows(const AttnArgs &a, int lq) {
  lq = lq < a.max_q ? lq : a.max_q;
  return lq > 0 ? lq * a.group : 0;
}

// Weights are 2^(s qs - m) in one fused step, so that m, which is rounded, leaves the rounding of the largest
// score in the exponent: the same for all keys, and below 1 while |s qs| < 2^24.  Rows that could get past
// that (|s| <= D 2^15 2688, so real scores beyond 10^7) have their scores multiplied by pre before, where they
// would be masked, and qs = 1: every product with m is then exact.
template <int D> __device__ __forceinline__ bool split_scale(float &qs, float &pre) {
  const bool far = qs * (float)(D * 2688) > 512.f;
  pre = far ? qs : 1.f;
  qs = far ? 1.f : qs;
  return far;
}

// fp16 values of a lane's D / 4 codes times their block scales; ok false: zeros
template <int D>
__device__ __forceinline__ void dequant(const uint32_t (&w)[D / 32], uint32_t sc, bool ok, h8 (&f)[D / 32]) {
  // the lane's columns are D / 64 blocks of 16 = 2 dwords each
#pragma unroll
  for (int k = 0; k < D / 64; ++k) {
    const float s = ok ? (k == 0 ? __builtin_amdgcn_cvt_f32_fp8(sc, 0) : k == 1 ? __builtin_amdgcn_cvt_f32_fp8(sc, 1) : k == 2 ? __builtin_amdgcn_cvt_f32_fp8(sc, 2) : __builtin_amdgcn_cvt_f32_fp8(sc, 3)) : 0.f;
    const _Float16 h = (_Float16)s;
    const h2 hs = {h, h};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t u = w[2 * k + i];
      const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, 1.0f, 0)) * hs;
      const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, 1.0f, 1)) * hs;
      const h2 c = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, 1.0f, 2)) * hs;
      const h2 d = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(u, 1.0f, 3)) * hs;
      f[2 * k + i] = h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    }
  }
}

template <int D>
__device__ __forceinline__ void load_codes(const uint8_t *d, const uint8_t *s, uint32_t (&w)[D / 32], uint32_t &sc) {
  if constexpr (D == 64) {
    const uint2 a = *reinterpret_cast<const uint2 *>(d);
    w[0] = a.x, w[1] = a.y;
    sc = *s;
  } else {
#pragma unroll
    for (int i = 0; i < D / 128; ++i) {
      const uint4 a = *reinterpret_cast<const uint4 *>(d + 16 * i);
      w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
    }
    if constexpr (D == 128)
      sc = *reinterpret_cast<const uint16_t *>(s);
    else
      sc = *reinterpret_cast<const uint32_t *>(s);
  }
}

__device__ __forceinline__ float max_g(float v) {  // over the 4 lanes of a row (lane ^ 16, lane ^ 32)
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum_g(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

template <typename T, int D>
__global__ __launch_bounds__(256, D == 256 ? 2 : 4) void attn_decode_kernel(AttnArgs a) {
  constexpr int NF = D / 32;                // fragments of a row in the contraction over head_dim
  constexpr int NB = D / 16;                // 16-column blocks of the output
  constexpr int VP = 2 * D + 32;            // V row pitch in LDS
  constexpr int kVBytes = 32 * VP;
  constexpr int kOBytes = 4 * 16 * (D + 4) * 4;
  constexpr int kBytes = 4 * kVBytes > kOBytes ? 4 * kVBytes : kOBytes;
  __shared__ __attribute__((aligned(16))) unsigned char lds[kBytes];
  __shared__ float ml[2][4][16];
  const Cache &c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), t = lane & 15, g = lane >> 4;
  const int tile = blockIdx.x / a.splits, split = blockIdx.x - tile * a.splits, kvh = blockIdx.y, b = blockIdx.z;
  const int lq = c.len_q[b];
  int lk = c.len_k[b];
  const int cap = c.table_cols << c.shift;
  const int off = lk - lq;  // a query token's place in its sequence
  lk = lk < cap ? lk : cap;
  const int nrows = attn_rows(a, lq);
  if (16 * tile >= nrows) return;
  const int last_tok = (16 * tile + 15 < nrows ? 16 * tile + 15 : nrows - 1) / a.group;
  int kv_end = a.causal ? off + last_tok + 1 : lk;
  kv_end = kv_end < lk ? kv_end : lk;
  const int t0 = split * a.chunk;
  if (split > 0 && t0 >= kv_end) return;  // the join knows the splits that there are
  // the last split takes what is left, should a sequence be longer than the call's max_len_k
  const int t1 = split + 1 < a.splits && t0 + a.chunk < kv_end ? t0 + a.chunk : kv_end;

  // ---- this lane's row of q
  const int row = 16 * tile + t, rtok = row / a.group, head = kvh * a.group + row % a.group;
  const int64_t qrow = (int64_t)c.start[b] + rtok;
  const bool row_ok = row < nrows && qrow >= 0 && qrow < a.rows;
  const int see = row_ok ? (a.causal ? (off + rtok + 1 < lk ? off + rtok + 1 : lk) : lk) : 0;  // keys it sees
  h8 qf[NF];
  float qscale, pre;
  bool far;
  {
    float v[NF][8];
    float m = 0.f;
    const T *qp = reinterpret_cast<const T *>(a.q) + (row_ok ? qrow : 0) * a.qt + head * a.qh + g * (D / 4);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const Vec<T> x = row_ok ? ldg_vec(qp + 8 * f) : Vec<T>{};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[f][j] = row_ok ? Elem<T>::ld(x.e[j]) : 0.f;
        m = max_skip_nan(m, v[f][j]);
      }
    }
    m = max_g(m);
    int e = (int)(__float_as_uint(m) >> 23) - 127;   // m >= 0
    e = m == 0.f || e == 128 ? 0 : e < -100 ? -100 : e;  // inf: left as it is
    const float up = pow2f(14 - e < 127 ? 14 - e : 127);
    qscale = fmaxf(a.sm_log2 * global_scale_of(c.amax[0]) * (1.0f / up), 1e-37f);  // > 0: scores of -inf stay -inf
    far = split_scale<D>(qscale, pre);
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[f][j] = (_Float16)(v[f][j] * up);
  }

  f32x4 acc[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kNegInf, l = 0.f;
  // keys below wmin need neither a mask nor pre in any of the wave's rows
  int wmin = row_ok ? (far ? 0 : see) : 0x7fffffff;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const int v = __shfl_xor(wmin, o, 64);
    wmin = v < wmin ? v : wmin;
  }
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  unsigned char *const vb = lds + wave * kVBytes;
  // a key's codes: the page's place (uniform) + a lane's offset in 16 keys (32 bits: token strides are below 2^26)
  const uint32_t kdo = t * (uint32_t)c.d_tok[0] + g * (D / 8), kso = t * (uint32_t)c.s_tok[0] + g * (D / 64);
  const uint32_t vdo = t * (uint32_t)c.d_tok[1] + g * (D / 8), vso = t * (uint32_t)c.s_tok[1] + g * (D / 64);

  // 32 keys' codes: K's registers are loaded anew (the wave's next 32 keys) as soon as its fp16 products are
  // made, V's as soon as its are; the pages of the 32 keys after those are in flight too
  uint32_t kw[2][NF], vw[2][NF], ksc[2], vsc[2];
  auto entries = [&](int kv, int (&e)[2]) {  // 16 keys: one page
#pragma unroll
    for (int u = 0; u < 2; ++u) e[u] = page_entry(c, b, __builtin_amdgcn_readfirstlane(kv + 16 * u));
  };
  auto fetch = [&](int i, int kv, const int (&page)[2], uint32_t (&w)[2][NF], uint32_t (&sc)[2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t pg = page[u] >= 0 ? page[u] : 0, at = (kv + 16 * u) & ((1 << c.shift) - 1);
      load_codes<D>(c.data[i] + (kvh * c.d_head[i] + pg * c.d_page[i] + at * c.d_tok[i]) + (i ? vdo : kdo),
                    c.scale[i] + (kvh * c.s_head[i] + pg * c.s_page[i] + at * c.s_tok[i]) + (i ? vso : kso), w[u], sc[u]);
    }
  };
  int ent[2], page[2] = {-1, -1};
  const int kv_first = t0 + 32 * wave;
  if (kv_first < t1) {
    entries(kv_first, ent);
#pragma unroll
    for (int u = 0; u < 2; ++u) page[u] = page_at(c, kv_first + 16 * u, ent[u]);
    entries(kv_first + 128, ent);
    fetch(0, kv_first, page, kw, ksc);
    fetch(1, kv_first, page, vw, vsc);
  }
  for (int kv = kv_first; kv < t1; kv += 128) {
    const bool has[2] = {page[0] >= 0, page[1] >= 0};
#pragma unroll
    for (int u = 0; u < 2; ++u) page[u] = page_at(c, kv + 128 + 16 * u, ent[u]);
    entries(kv + 256, ent);
    // ---- scores
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      h8 kf[NF];
      dequant<D>(kw[u], ksc[u], true, kf);
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < NF; ++f) s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[f], qf[f], s[u], 0, 0, 0);
    }
    fetch(0, kv + 128, page, kw, ksc);  // past the end: keys of any page, not used
    // ---- V to LDS (rows that hold no token of this sequence as zeros: 0 * NaN is NaN)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      h8 vf[NF];
      dequant<D>(vw[u], vsc[u], has[u] && kv + 16 * u + t < lk, vf);
#pragma unroll
      for (int f = 0; f < NF; ++f)
        *reinterpret_cast<h8 *>(vb + (16 * u + t) * VP + g * (D / 2) + 16 * f) = vf[f];
    }
    fetch(1, kv + 128, page, vw, vsc);
    // ---- softmax: keys kv + 16 u + 4 g + j
    if (kv + 32 > wmin || !has[0] || !has[1]) {  // wave-uniform
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[u][j] = has[u] && kv + 16 * u + 4 * g + j < see ? s[u][j] * pre : kNegInf;
    }
    float mx = s[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, s[j >> 2][j & 3]);
    mx *= qscale;
    // the running maximum moves only where a key of the wave exceeds its row's by 2^kSlack
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack)) {
      const float mn = fmaxf(m, max_g(mx));
      const float corr = __builtin_amdgcn_exp2f(m - (mn == kNegInf ? 0.f : mn));
      m = mn;
      l *= corr;
#pragma unroll
      for (int d = 0; d < NB; ++d) acc[d] *= corr;
    }
    const float mu = (m == kNegInf ? 0.f : m) - kShift;
    h8 p;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], qscale, -mu));
      const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][(j & 3) + 1], qscale, -mu));
      l += e0;  // this lane's keys only; joined at the end
      l += e1;
      const h2 h = __builtin_convertvector((f2v{e0, e1}), h2);
      p[j] = h.x, p[j + 1] = h.y;
    }
    // ---- O^T += V^T P^T
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < NB; ++d) {
      const unsigned char *base = vb + (4 * g + (t >> 2)) * VP + 32 * d + 8 * (t & 3);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)base);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(base + 16 * VP));
      const h4 a0 = __builtin_bit_cast(h4, lo), a1 = __builtin_bit_cast(h4, hi);
      const h8 vt = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, p, acc[d], 0, 0, 0);
    }
    __builtin_amdgcn_wave_barrier();
  }

  // ---- join the waves: rows t, columns 16 d + 4 g + j
  l = sum_g(l);
  __syncthreads();  // every wave is done with its V rows
  float *ob = reinterpret_cast<float *>(lds) + wave * 16 * (D + 4);
#pragma unroll
  for (int d = 0; d < NB; ++d) *reinterpret_cast<f32x4 *>(ob + t * (D + 4) + 16 * d + 4 * g) = acc[d];
  if (g == 0) {
    ml[0][wave][t] = m;
    ml[1][wave][t] = l;
  }
  __syncthreads();
  const float gv = global_scale_of(c.amax[1]);
  for (int i = tid; i < 16 * (D / 4); i += 256) {
    const int r = i / (D / 4), d4 = 4 * (i % (D / 4)), rr = 16 * tile + r;
    if (rr >= nrows) continue;
    float mm = kNegInf;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[0][w][r]);
    const float mu = mm == kNegInf ? 0.f : mm;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float ls = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(ml[0][w][r] - mu);
      ls += ml[1][w][r] * f;
      o += *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(lds) + (w * 16 + r) * (D + 4) + d4) * f;
    }
    if (a.splits > 1) {
      float *pp = a.part + part_row<D>(a, split, b, kvh, rr);
      *reinterpret_cast<f32x4 *>(pp + d4) = o;
      if (d4 == 0) pp[D] = mm, pp[D + 1] = ls;
    } else {
      const int64_t orow = (int64_t)c.start[b] + rr / a.group;
      if (orow < 0 || orow >= a.rows) continue;
      const float inv = ls > 0.f ? gv / ls : 0.f;
      T *op = reinterpret_cast<T *>(a.o) + orow * a.ot + (kvh * a.group + rr % a.group) * a.oh + d4;
#pragma unroll
      for (int j = 0; j < 4; ++j) op[j] = Elem<T>::st(ls == ls && ls == 0.f ? 0.f : o[j] * inv);
    }
  }
}

// the splits of a row, in order: a workgroup a row, D / 4 lanes for its columns, 1024 / D splits at a time
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  constexpr int LN = D / 4, NG = 256 / LN;
  __shared__ f32x4 ob[NG][LN];
  __shared__ float lb[NG];
  const Cache &c = a.c;
  const int kvh = blockIdx.y, row = blockIdx.x, b = blockIdx.z, grp = threadIdx.x / LN, d4 = 4 * (threadIdx.x % LN);
  const int lq = c.len_q[b], off = c.len_k[b] - lq, cap = c.table_cols << c.shift;
  const int lk = c.len_k[b] < cap ? c.len_k[b] : cap;
  if (row >= attn_rows(a, lq)) return;
  const int64_t orow = (int64_t)c.start[b] + row / a.group;
  if (orow < 0 || orow >= a.rows) return;
  int kv_end = a.causal ? off + row / a.group + 1 : lk;
  kv_end = kv_end < lk ? kv_end : lk;
  int n = kv_end > 0 ? (kv_end + a.chunk - 1) / a.chunk : 1;
  n = n < a.splits ? n : a.splits;
  const int64_t step = (int64_t)a.batch * c.hkv * a.part_tiles * 16 * (D + 4);
  const float *pp = a.part + part_row<D>(a, 0, b, kvh, row);
  float m = kNegInf;
  for (int s = threadIdx.x % 64; s < n; s += 64) m = fmaxf(m, pp[s * step + D]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float mu = m == kNegInf ? 0.f : m;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
  for (int s = grp; s < n; s += NG) {
    const float f = __builtin_amdgcn_exp2f(pp[s * step + D] - mu);
    l += pp[s * step + D + 1] * f;
    o += *reinterpret_cast<const f32x4 *>(pp + s * step + d4) * f;
  }
  ob[grp][threadIdx.x % LN] = o;
  if (d4 == 0) lb[grp] = l;
  __syncthreads();
  if (grp) return;
  for (int g = 1; g < NG; ++g) o += ob[g][threadIdx.x], l += lb[g];
  const float inv = global_scale_of(c.amax[1]) / l;
  T *op = reinterpret_cast<T *>(a.o) + orow * a.ot + (kvh * a.group + row % a.group) * a.oh + d4;
#pragma unroll
  for (int j = 0; j < 4; ++j) op[j] = Elem<T>::st(l == 0.f ? 0.f : o[j] * inv);
}

// ---- attention of prompts ------------------------------------------------------------------------
// The same sums where every KV head has rows by the hundred: bound by the matrix cores and, nearly as
// much, by the exponentials (a quarter of the VALU's rate) and by LDS (K and V of a 32 x 32 tile of scores
// are 16 KiB of fragments: 128 cycles of LDS beside 512 of one SIMD's matrix core, four SIMDs at once).  A
// workgroup is 8 waves of 32 rows (v_mfma_f32_32x32x16_f16) on one KV head, two waves a SIMD; 64 keys at
// a time are turned into fp16 by the whole workgroup, once per 256 rows, into one of three LDS stages.
// Chunks of 500 to 1024 tokens behind contexts of up to 8192, 4 sequences, 32 / 8 heads of 128: 370 us (800 TFLOP/s)
// back to back, 380 to 455 where each call is waited for; matrix cores busy 41 % of the time, LDS 36 %, 29 % of that
// in conflicts.  head_dim 64: 277 us (536 TFLOP/s).  64 rows a wave, one wave a SIMD, half the LDS reads took 546
// where this layout took 409 (before its page entries were loaded ahead): nothing of its one wave overlaps.
// The loop over 32-key tiles is pipelined in registers: the step of tile j multiplies K of tile j + 1
// and V of tile j - 1 while the softmax of tile j runs, three chains without a dependency between them.
__device__ __forceinline__ float xmax32(float v) {  // v and its lane ^ 32 partner
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xadd32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
typedef float f32x16 __attribute__((ext_vector_type(16)));

// key (of a 32-key tile) of score register j in half hi
__device__ __forceinline__ int crow(int j, int hi) { return (j & 3) + 8 * (j >> 2) + 4 * hi; }

template <typename T, int D>
__global__ __launch_bounds__(512, 2) void attn_prompt_kernel(AttnArgs a) {
  constexpr int KP = 2 * D + 16, VP = 2 * D + 64;  // row pitches: conflict-free b128 reads / transposed reads
  constexpr int KIMG = 64 * KP, VIMG = 64 * VP, STAGE = KIMG + VIMG;
  constexpr int QS = D / 16, DB = D / 32, NW = D / 32;  // steps over head_dim, output blocks, code dwords a lane
  __shared__ __attribute__((aligned(16))) unsigned char lds[3 * STAGE];
  const Cache &c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), fr = lane & 31, hi = lane >> 5;
  // the tiles of one (sequence, KV head) on one XCD, longest first
  const int xcd = blockIdx.x % 8, li = blockIdx.x / 8;
  const int pair = (li / a.tiles) * 8 + xcd, tile = a.tiles - 1 - li % a.tiles;
  if (pair >= a.batch * c.hkv) return;
  const int b = pair / c.hkv, kvh = pair - b * c.hkv;
  const int lq = c.len_q[b], off = c.len_k[b] - lq, cap = c.table_cols << c.shift;
  const int lk = c.len_k[b] < cap ? c.len_k[b] : cap;
  const int nrows = attn_rows(a, lq);
  if (256 * tile >= nrows) return;  // the whole workgroup
  const int last_tok = (256 * tile + 255 < nrows ? 256 * tile + 255 : nrows - 1) / a.group;
  int kv_end = a.causal ? off + last_tok + 1 : lk;
  kv_end = kv_end < lk ? kv_end : lk;
  // this split's stages of 64 keys (the last split takes what is left); the join knows the splits there are
  const int split = blockIdx.y, t0 = split * (a.chunk / 64);
  if (split > 0 && 64 * t0 >= kv_end) return;
  int stages = kv_end > 0 ? (kv_end + 63) / 64 : 0;
  if (split + 1 < a.splits && t0 + a.chunk / 64 < stages) stages = t0 + a.chunk / 64;

  // ---- this lane's row of q
  h8 qf[QS];
  float qs, pre;
  int see, wmin = 0x7fffffff;  // keys a row sees; keys below wmin need neither a mask nor pre in any of the wave's rows
  {
    const int row = 256 * tile + 32 * wave + fr, rtok = row / a.group, head = kvh * a.group + row % a.group;
    const int64_t qrow = (int64_t)c.start[b] + rtok;
    const bool ok = row < nrows && qrow >= 0 && qrow < a.rows;
    see = ok ? (a.causal ? (off + rtok + 1 < lk ? off + rtok + 1 : lk) : lk) : 0;
    const T *qp = reinterpret_cast<const T *>(a.q) + (ok ? qrow : 0) * a.qt + head * a.qh + 8 * hi;
    Vec<T> x[QS];
    float m = 0.f;
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      x[s].raw = make_uint4(0, 0, 0, 0);
      if (ok) x[s] = ldg_vec(qp + 16 * s);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max_skip_nan(m, Elem<T>::ld(x[s].e[j]));
    }
    m = xmax32(m);
    int e = (int)(__float_as_uint(m) >> 23) - 127;
    e = m == 0.f || e == 128 ? 0 : e < -100 ? -100 : e;
    const float up = pow2f(14 - e < 127 ? 14 - e : 127);
    qs = fmaxf(a.sm_log2 * global_scale_of(c.amax[0]) * (1.0f / up), 1e-37f);
    const bool far = split_scale<D>(qs, pre);
    wmin = ok ? (far ? 0 : see) : wmin;
#pragma unroll
    for (int s = 0; s < QS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) qf[s][j] = (_Float16)(Elem<T>::ld(x[s].e[j]) * up);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int v = __shfl_xor(wmin, o, 64);
    wmin = v < wmin ? v : wmin;
  }
  wmin = __builtin_amdgcn_readfirstlane(wmin);

  f32x16 acc[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[d][e] = 0.f;
  float m = kNegInf, l = 0.f;

  // ---- staging: the first 256 lanes unpack K, the others V; lane -> key of the stage, quarter of its columns
  const int skey = (tid & 255) >> 2, sg = tid & 3, skv = wave >> 2;
  uint32_t cw[NW], csc = 0;
  bool cok = false;
  int pages = 0;  // of the stage in the registers: bit u: keys 16 u .. 16 u + 15 have a page
  const int64_t d_page = skv ? c.d_page[1] : c.d_page[0], d_tok = skv ? c.d_tok[1] : c.d_tok[0];
  const int64_t s_page = skv ? c.s_page[1] : c.s_page[0], s_tok = skv ? c.s_tok[1] : c.s_tok[0];
  const uint8_t *const dbase = (skv ? c.data[1] + kvh * c.d_head[1] : c.data[0] + kvh * c.d_head[0]) + sg * (D / 8);
  const uint8_t *const sbase = (skv ? c.scale[1] + kvh * c.s_head[1] : c.scale[0] + kvh * c.s_head[0]) + sg * (D / 64);
  struct Entries {
    int group[4], mine;
  };
  auto entries = [&](int t, Entries &e) {
#pragma unroll
    for (int u = 0; u < 4; ++u) e.group[u] = page_entry(c, b, 64 * t + 16 * u);
    e.mine = page_entry(c, b, 64 * t + skey);
  };
  auto gload = [&](int t, const Entries &e) {
    pages = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u) pages |= (page_at(c, 64 * t + 16 * u, e.group[u]) >= 0 ? 1 : 0) << u;
    const int key = 64 * t + skey, page = page_at(c, key, e.mine), at = key & ((1 << c.shift) - 1);
    const int64_t pg = page >= 0 ? page : 0;
    load_codes<D>(dbase + pg * d_page + at * d_tok, sbase + pg * s_page + at * s_tok, cw, csc);
    cok = skv == 0 || (page >= 0 && key < lk);  // V of no token of this sequence: zeros (0 * NaN is NaN)
  };
  auto swrite = [&](int slot) {
    h8 f[NW];
    dequant<D>(cw, csc, cok, f);
    unsigned char *o = lds + slot * STAGE + (skv ? KIMG + skey * VP : skey * KP) + sg * (D / 2);
#pragma unroll
    for (int i = 0; i < NW; ++i) *reinterpret_cast<h8 *>(o + 16 * i) = f[i];
  };
  // S^T of a tile
  auto score = [&](const unsigned char *K, f32x16 &s) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int st = 0; st < QS; ++st) {
      const h8 kf = *reinterpret_cast<const h8 *>(K + fr * KP + (16 * st + 8 * hi) * 2);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[st], s, 0, 0, 0);
    }
  };
  const int trq = (lane & 15) >> 2, trp = lane & 3, trg = lane >> 4;
  const int tr_off = (4 * (trg >> 1) + trq) * VP + (16 * (trg & 1) + 4 * trp) * 2;
  auto pv = [&](const unsigned char *V, const h8 (&p)[2]) {
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const unsigned char *base = V + tr_off + 16 * g * VP + 64 * d;
        const h4 lo = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)base));
        const h4 up = __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(base + 8 * VP)));
        const h8 vf = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, p[g], acc[d], 0, 0, 0);
      }
  };
  // the softmax of one tile; returns whether some row's maximum moved (corr: what O and l of before are worth)
  auto soft = [&](const f32x16 &s, h8 (&p)[2], float &corr) -> bool {
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = xmax32(mx) * qs;
    const bool up = mx > m + kSlack;
    corr = up ? __builtin_amdgcn_exp2f(m - mx) : 1.f;  // m = -inf: 0
    m = up ? mx : m;
    const float mu = (m == kNegInf ? 0.f : m) - kShift;
    float ls = 0.f;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * g + i], qs, -mu));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * g + i + 1], qs, -mu));
        ls += e0;
        ls += e1;
        const h2 h = __builtin_convertvector((f2v{e0, e1}), h2);
        p[g][i] = h.x;
        p[g][i + 1] = h.y;
      }
    l = l * corr + ls;  // this lane's keys only; joined at the end
    return up;
  };
  auto mask = [&](f32x16 &s, int kv0, int pg) {
    if (kv0 + 32 <= wmin && pg == 3) return;  // wave-uniform
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int k = crow(e, hi);
      s[e] = kv0 + k < see && (pg >> (k >> 4) & 1) ? s[e] * pre : kNegInf;
    }
  };

  if (t0 < stages) {
    // V of "tile -1" is multiplied by weights of zero: it has to be finite
    for (int i = tid; i < VIMG / 16; i += 512) *reinterpret_cast<uint4 *>(lds + 2 * STAGE + KIMG + 16 * i) = make_uint4(0, 0, 0, 0);
    Entries ent;
    entries(t0, ent);
    gload(t0, ent);
    entries(t0 + 1, ent);
    int pg0 = pages;
    swrite(0);
    gload(t0 + 1, ent);  // past the end: keys of any page, not used
    entries(t0 + 2, ent);
    int pg1 = pages;
    __syncthreads();
    f32x16 sc, sn;
    score(lds, sc);
    h8 pp[2], pc[2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) pp[g][i] = (_Float16)0.f;
    int slot = 0;
    float corr;
    auto rescale = [&](bool moved) {
      if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[d][e] *= corr;
      }
    };
    for (int t = t0; t < stages; ++t) {
      const int nx = slot == 2 ? 0 : slot + 1, pv_slot = slot == 0 ? 2 : slot - 1;
      const unsigned char *Kc = lds + slot * STAGE, *Vc = Kc + KIMG, *Vp = lds + pv_slot * STAGE + KIMG + 32 * VP;
      // tile 2 t: scores of 2 t + 1, V of 2 t - 1
      mask(sc, 64 * t, pg0 & 3);
      swrite(nx);                                   // stage t + 1 (read by none before the barrier below)
      gload(t + 2, ent);                            // in flight under the rest of this stage
      entries(t + 3, ent);
      const int pg2 = pages;
      score(Kc + 32 * KP, sn);
      bool moved = soft(sc, pc, corr);
      pv(Vp, pp);
      rescale(moved);
      __syncthreads();
      // tile 2 t + 1: scores of 2 t + 2, V of 2 t
      mask(sn, 64 * t + 32, pg0 >> 2);
      score(lds + nx * STAGE, sc);
      moved = soft(sn, pp, corr);
      pv(Vc, pc);
      rescale(moved);
      slot = nx;
      pg0 = pg1, pg1 = pg2;
    }
    pv(lds + (slot == 0 ? 2 : slot - 1) * STAGE + KIMG + 32 * VP, pp);
  }

  // ---- o = acc gv / l: lane holds columns 32 d + crow(e, hi) of its row
  const float ls = xadd32(l);
  const int row = 256 * tile + 32 * wave + fr;
  if (row >= nrows) return;
  if (a.splits > 1) {
    float *pp = a.part + part_row<D>(a, split, b, kvh, row);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4)
        *reinterpret_cast<f32x4 *>(pp + 32 * d + 8 * e4 + 4 * hi) = f32x4{acc[d][4 * e4], acc[d][4 * e4 + 1], acc[d][4 * e4 + 2], acc[d][4 * e4 + 3]};
    if (hi == 0) pp[D] = m, pp[D + 1] = ls;
    return;
  }
  const int64_t orow = (int64_t)c.start[b] + row / a.group;
  if (orow < 0 || orow >= a.rows) return;
  const float inv = global_scale_of(c.amax[1]) / ls;
  T *op = reinterpret_cast<T *>(a.o) + orow * a.ot + (kvh * a.group + row % a.group) * a.oh;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
      struct alignas(4 * sizeof(T)) Pack {
        T h[4];
      } pk;
#pragma unroll
      for (int i = 0; i < 4; ++i) pk.h[i] = Elem<T>::st(ls == 0.f ? 0.f : acc[d][4 * e4 + i] * inv);
      *reinterpret_cast<Pack *>(op + 32 * d + 8 * e4 + 4 * hi) = pk;
    }
}

bool make_cache(const mtq_kv_cache *k, const int32_t *table, int64_t table_stride, int table_cols, const int32_t *start,
                const int32_t *len_q, const int32_t *len_k, int batch, Cache &c) {
  if (!k || !table || !start || !len_q || !len_k || batch < 1 || table_cols < 1 || (batch > 1 && table_stride < table_cols)) return false;
  if (k->page_size < 16 || k->page_size > 32768 || (k->page_size & (k->page_size - 1))) return false;
  if (k->num_pages < 1 || k->num_kv_heads < 1) return false;
  if (k->head_dim != 64 && k->head_dim != 128 && k->head_dim != 256) return false;
  if ((int64_t)table_cols * k->page_size > (int64_t)INT32_MAX / 2) return false;  // positions are ints
  for (int i = 0; i < 2; ++i) {
    c.data[i] = (uint8_t *)k->data[i], c.scale[i] = (uint8_t *)k->scale[i], c.amax[i] = k->amax[i];
    c.d_page[i] = k->data_strides[i][0], c.d_head[i] = k->data_strides[i][1], c.d_tok[i] = k->data_strides[i][2];
    c.s_page[i] = k->scale_strides[i][0], c.s_head[i] = k->scale_strides[i][1], c.s_tok[i] = k->scale_strides[i][2];
    if (!c.data[i] || !c.scale[i] || !c.amax[i]) return false;
    const int sb = k->head_dim / 16;
    // rows: 16-byte aligned codes, scales aligned to a row of theirs
    if ((uintptr_t)c.data[i] % 16 || (uintptr_t)c.scale[i] % sb) return false;
    for (int j = 0; j < 3; ++j)
      if (k->data_strides[i][j] < 0 || k->data_strides[i][j] % 16 || k->scale_strides[i][j] < 0 || k->scale_strides[i][j] % sb) return false;
    if (k->data_strides[i][2] >= (1 << 26) || k->scale_strides[i][2] >= (1 << 26)) return false;
  }
  c.table = table, c.start = start, c.len_q = len_q, c.len_k = len_k, c.table_stride = table_stride;
  c.table_cols = table_cols, c.num_pages = k->num_pages, c.hkv = k->num_kv_heads, c.head_dim = k->head_dim;
  c.shift = 0;
  while ((1 << c.shift) < k->page_size) c.shift++;
  return true;
}

int rows_call(bool append, const mtq_kv_cache *cache, void *k, void *v, const int64_t *strides, int64_t rows,
              const int32_t *table, int64_t table_stride, int table_cols, const int32_t *start, const int32_t *len_q,
              const int32_t *len_k, int batch, int max_len, int dtype, hipStream_t stream) {
  if (dtype != MTQ_BF16 && dtype != MTQ_F16 && dtype != MTQ_F32) return MTQ_ERR_DTYPE;
  RowArgs a;
  if (!strides || rows < 0 || max_len < 0 || batch < 0 || batch > 65535) return MTQ_ERR_INVALID_ARG;
  if (batch == 0 || max_len == 0 || rows == 0) return MTQ_OK;
  if (!k || !v || !make_cache(cache, table, table_stride, table_cols, start, len_q, len_k, batch, a.c)) return MTQ_ERR_INVALID_ARG;
  a.x[0] = k, a.x[1] = v;
  a.xt[0] = strides[0], a.xh[0] = strides[1], a.xt[1] = strides[2], a.xh[1] = strides[3];
  a.rows = rows;
  if (max_len > rows) max_len = (int)rows;  // a sequence has no more new tokens than there are rows
  if (max_len > 1 << 30) return MTQ_ERR_INVALID_ARG;
  a.max_len = max_len;
  // tokens of a head a pass of the workgroup takes: as many as there are, at most the pass's rows
  const int rows_wg = 2048 / a.c.head_dim;
  a.lt = 0;
  while ((2 << a.lt) <= rows_wg && (1 << a.lt) < max_len) a.lt++;
  const int es = dtype == MTQ_F32 ? 4 : 2;
  bool vec = al16p(k) && al16p(v);
  for (int i = 0; i < 4; ++i) {
    if (strides[i] < 0) return MTQ_ERR_INVALID_ARG;
    vec = vec && (strides[i] * es) % 16 == 0;
  }
  const int toks = (append ? kAppendAhead : kReadAhead) << a.lt, heads = rows_wg >> a.lt;
  const int64_t gz = (2 * (int64_t)a.c.hkv + heads - 1) / heads, all = ((int64_t)max_len + toks - 1) / toks * batch * gz;
  const int64_t most = (int64_t)kAppendWgs * host_num_cus();
  const int64_t passes = (all + most - 1) / most, enough = ((int64_t)max_len + toks - 1) / toks;
  a.passes = append ? (int)(passes < enough ? passes : enough) : 1;
  const int64_t gx = ((int64_t)max_len + (int64_t)toks * a.passes - 1) / ((int64_t)toks * a.passes);
  if (gz > 65535 || gx > UINT32_MAX / 256) return MTQ_ERR_INVALID_ARG;  // (a grid's dimension has fewer than 2^32 lanes)
  const dim3 g((unsigned)gx, (unsigned)batch, (unsigned)gz);
  auto go = [&](auto t) {
    using T = decltype(t);
    if (append)
      vec ? cache_append_kernel<T, true><<<g, 256, 0, stream>>>(a) : cache_append_kernel<T, false><<<g, 256, 0, stream>>>(a);
    else
      vec ? cache_read_kernel<T, true><<<g, 256, 0, stream>>>(a) : cache_read_kernel<T, false><<<g, 256, 0, stream>>>(a);
    return host_check_launch();
  };
  return dtype == MTQ_BF16 ? go(__bf16{}) : dtype == MTQ_F16 ? go(_Float16{}) : go(float{});
}

struct Plan {
  int tiles, part_tiles, chunk, splits;
  bool prompt;
};
// Rows of a KV head from which the prompt kernel is taken.  us, prompt / decode kernel, 32 / 8 heads of 128 (4 rows a
// token): 1 sequence of 8192 keys, 64 rows 29 / 22, 96 30 / 27, 128 32 / 30, 256 41 / 40, 512 46 / 58; 8 of them, 64 rows
// 78 / 53, 96 83 / 76, 128 86 / 97, 256 99 / 159; 64 of 2048 keys, 64 rows 142 / 73, 128 144 / 139.  Few workgroups
// on short contexts would gain from more rows: 1 prompt of 128 tokens alone 15 / 7, of 512 27 / 20, of 1024 71 / 45; 4 of 128
// 16 / 12, but of 256 21 / 26, and 16 of 64 15 / 20.
constexpr int kPromptRows = 128;

// the rows of a KV head that a call has room for (ints in the kernels)
bool attn_rows_fit(int max_len_q, int group) { return (int64_t)max_len_q * group <= INT32_MAX - 256; }

// Splits of the keys: enough workgroups to fill the card (decode: 6 a CU, a split at least 256 keys, two
// 32-key steps a wave; prompts: one a CU, at least 512 keys).  Up to 512 keys stay in one piece, which needs no
// join: 9.7 us against 10.9 for one sequence of 500 keys, 10.1 / 13.8 for 32 of them; at 1000, split is faster
// (10.8 / 12.8).
// The workspace's size and the call's plan are this function's of the same arguments, max_len_k as the caller gave it
// (the size is no monotone function of it: fewer keys can mean more splits).
Plan attn_plan(int batch, int hkv, int group, int head_dim, int max_len_q, int max_len_k) {
  Plan p;
  if (max_len_k > INT32_MAX / 2) max_len_k = INT32_MAX / 2;  // the most positions that a cache can have
  const int64_t rows = (int64_t)max_len_q * group;
  // head_dim 256: the prompt kernel's three stages do not fit LDS, and the decode kernel unpacks every key again for 16
  // rows (the chunks above with 16 / 4 heads of 256: 713 us, 416 TFLOP/s)
  p.prompt = rows >= kPromptRows && head_dim <= 128;
  p.part_tiles = (int)((rows + 15) / 16);
  p.tiles = p.prompt ? (int)((rows + 255) / 256) : p.part_tiles;
  const int64_t wgs = (int64_t)batch * hkv * p.tiles, cus = host_num_cus();
  const int least = p.prompt || max_len_k <= 512 ? 512 : 256;
  int64_t splits = p.prompt ? cus / wgs : (6 * cus + wgs - 1) / wgs;
  const int64_t most = (max_len_k + least - 1) / least;
  splits = splits < most ? splits : most;
  splits = splits < 1 ? 1 : splits > 256 ? 256 : splits;
  int64_t chunk = (max_len_k + splits - 1) / splits;
  chunk = (chunk + 127) / 128 * 128;
  p.chunk = (int)(chunk < least ? least : chunk);
  p.splits = (max_len_k + p.chunk - 1) / p.chunk;
  if (p.splits < 1) p.splits = 1;
  return p;
}

}  // namespace

extern "C" {

int mtq_kv_append(const mtq_kv_cache *cache, const void *k, const void *v, const int64_t *strides, int64_t rows,
                  const int32_t *block_table, int64_t table_stride, int table_cols, const int32_t *b_start_loc,
                  const int32_t *b_seq_len, const int32_t *b_seq_len_k, int batch, int max_len, int dtype, hipStream_t stream) {
  return rows_call(true, cache, const_cast<void *>(k), const_cast<void *>(v), strides, rows, block_table, table_stride,
                   table_cols, b_start_loc, b_seq_len, b_seq_len_k, batch, max_len, dtype, stream);
}

int mtq_kv_read(const mtq_kv_cache *cache, void *k, void *v, const int64_t *strides, int64_t rows, const int32_t *block_table,
                int64_t table_stride, int table_cols, const int32_t *b_start_loc, const int32_t *b_seq_len,
                const int32_t *b_seq_len_k, int batch, int max_len, int dtype, hipStream_t stream) {
  return rows_call(false, cache, k, v, strides, rows, block_table, table_stride, table_cols, b_start_loc, b_seq_len,
                   b_seq_len_k, batch, max_len, dtype, stream);
}

size_t mtq_kv_attention_workspace_bytes(int batch, int num_q_heads, int num_kv_heads, int head_dim, int max_len_q, int max_len_k) {
  if (batch < 1 || num_kv_heads < 1 || num_q_heads < num_kv_heads || max_len_q < 1 || max_len_k < 0 || head_dim < 1) return 0;
  if (!attn_rows_fit(max_len_q, num_q_heads / num_kv_heads)) return 0;  // which mtq_kv_attention refuses
  const Plan p = attn_plan(batch, num_kv_heads, num_q_heads / num_kv_heads, head_dim, max_len_q, max_len_k);
  return p.splits > 1 ? (size_t)p.splits * batch * num_kv_heads * p.part_tiles * 16 * (head_dim + 4) * sizeof(float) : 0;
}

int mtq_kv_attention(const mtq_kv_cache *cache, const void *q, void *o, const int64_t *strides, int64_t rows, int num_q_heads,
                     const int32_t *block_table, int64_t table_stride, int table_cols, const int32_t *b_start_loc,
                     const int32_t *b_seq_len, const int32_t *b_seq_len_k, int batch, int max_len_q, int max_len_k,
                     int is_causal, double softmax_scale, int dtype, void *ws, size_t ws_bytes, hipStream_t stream) {
  if (dtype != MTQ_BF16 && dtype != MTQ_F16) return MTQ_ERR_DTYPE;
  if (!strides || rows < 0 || max_len_q < 0 || max_len_k < 0 || batch < 0 || batch > 65535) return MTQ_ERR_INVALID_ARG;
  if (batch == 0 || max_len_q == 0 || rows == 0) return MTQ_OK;
  AttnArgs a;
  if (!q || !o || !make_cache(cache, block_table, table_stride, table_cols, b_start_loc, b_seq_len, b_seq_len_k, batch, a.c))
    return MTQ_ERR_INVALID_ARG;
  if (num_q_heads < 1 || num_q_heads % a.c.hkv) return MTQ_ERR_INVALID_ARG;
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0 || strides[i] % 8) return MTQ_ERR_INVALID_ARG;
  if (!al16p(q) || !al16p(o) || !(softmax_scale > 0.0 && softmax_scale < 3.4e38)) return MTQ_ERR_INVALID_ARG;
  a.group = num_q_heads / a.c.hkv;
  if (!attn_rows_fit(max_len_q, a.group)) return MTQ_ERR_INVALID_ARG;
  const Plan p = attn_plan(batch, a.c.hkv, a.group, a.c.head_dim, max_len_q, max_len_k);
  const int64_t pg = ((int64_t)batch * a.c.hkv + 7) / 8 * 8 * p.tiles;  // the prompt kernel's grid
  // (a grid's dimension has fewer than 2^32 lanes)
  if (p.prompt ? pg > UINT32_MAX / 512 : (int64_t)p.tiles * p.splits > UINT32_MAX / 256) return MTQ_ERR_INVALID_ARG;
  if (a.c.hkv > 65535) return MTQ_ERR_INVALID_ARG;
  const size_t need = mtq_kv_attention_workspace_bytes(batch, num_q_heads, a.c.hkv, a.c.head_dim, max_len_q, max_len_k);
  if (need && (!ws || ws_bytes < need || !al16p(ws))) return MTQ_ERR_INVALID_ARG;
  a.q = q, a.o = o, a.part = (float *)ws;
  a.qt = strides[0], a.qh = strides[1], a.ot = strides[2], a.oh = strides[3], a.rows = rows;
  a.causal = is_causal ? 1 : 0;
  a.splits = p.splits, a.chunk = p.chunk, a.tiles = p.tiles, a.part_tiles = p.part_tiles, a.batch = batch;
  a.max_q = max_len_q;
  a.sm_log2 = (float)(softmax_scale * 1.44269504088896);
  const dim3 g((unsigned)(p.tiles * p.splits), (unsigned)a.c.hkv, (unsigned)batch), gj((unsigned)(max_len_q * a.group), (unsigned)a.c.hkv, (unsigned)batch);
  auto go = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    if constexpr (D <= 128) {
      if (p.prompt)
        attn_prompt_kernel<T, D><<<dim3((unsigned)pg, (unsigned)p.splits), 512, 0, stream>>>(a);
      else
        attn_decode_kernel<T, D><<<g, 256, 0, stream>>>(a);
    } else {
      attn_decode_kernel<T, D><<<g, 256, 0, stream>>>(a);
    }
    const int st = host_check_launch();
    if (st != MTQ_OK || p.splits == 1) return st;
    attn_join_kernel<T, D><<<gj, 256, 0, stream>>>(a);
    return host_check_launch();
  };
  auto dims = [&](auto t) {
    switch (a.c.head_dim) {
    case 64: return go(t, std::integral_constant<int, 64>{});
    case 128: return go(t, std::integral_constant<int, 128>{});
    default: return go(t, std::integral_constant<int, 256>{});
    }
  };
  return dtype == MTQ_BF16 ? dims(__bf16{}) : dims(_Float16{});
}

}  // extern "C"
