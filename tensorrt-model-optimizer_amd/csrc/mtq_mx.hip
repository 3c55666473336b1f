// mtq_mx.hip — microscaled operands and their products on gfx950: quantising activations, the RMS
// norm that quantises its output, and y = xq . W^T with W packed as MXFP4.
//
// Formats.  A row of K values is held as K / 32 blocks; block b has an exponent e_b (E8M0 byte
// e_b + 127) and 32 elements q, value = q * 2^e_b:
//   e_b = ceil(log2(max|x| / most)), q = round(x / 2^e_b), most = 6 (E2M1, two codes a byte, the
//   even column low) or 448 (E4M3, a byte each)
// -- the values of the dynamic block fake quant (mtq_fused_amax_convert with E8M0 scales): a block
// of zeros has e = 0, NaN is left out of the maximum, an infinity counts as FLT_MAX and saturates,
// a NaN element becomes +6 in E2M1 and stays NaN in E4M3.  Two plain FP8 formats stand beside them:
// per tensor (values of mtq_fake_e4m3fy: q = e4m3(x * s), s = RN(RN(1 / amax) * 448), factor 1 / s)
// and per token (factor max|x| / 448 of the row, 1 for a row of zeros, q = e4m3(x / factor)).
#include <hip/hip_runtime.h>
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
typedef int i32x8 __attribute__((ext_vector_type(8)));

inline bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool is_mx(int kind) { return kind == MTQ_MXFP4 || kind == MTQ_MXFP8; }

// A grid's dimension holds fewer than 2^32 lanes and wraps silently beyond: `rows` rows of `lanes` lanes each
// (rounded up by less than 1024 in all) go in as few launches as they need, launch(first row, rows of it).
template <typename F> int in_launches(int64_t rows, int64_t lanes, F launch) {
  const int64_t most = (UINT32_MAX - 1024) / lanes;
  for (int64_t r = 0; r < rows; r += most) {
    launch(r, rows - r < most ? rows - r : most);
    const int st = host_check_launch();
    if (st != MTQ_OK) return st;
  }
  return MTQ_OK;
}

// ---- 8 consecutive values --------------------------------------------------------------------
// VEC: 16-byte aligned groups of 8 columns, none of them past the row; else element by element.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, int64_t col, int64_t cols, float (&v)[8]) {
  if constexpr (VEC) {
    constexpr int N = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      const Vec<T> a = ldg_vec(p + col + i);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i + j] = Elem<T>::ld(a.e[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? Elem<T>::ld(p[col + i]) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *p, int64_t col, int64_t cols, const float (&v)[8]) {
  if constexpr (VEC) {
    constexpr int N = Vec<T>::N;
#pragma unroll
    for (int i = 0; i < 8; i += N) {
      Vec<T> a;
#pragma unroll
      for (int j = 0; j < N; ++j) a.e[j] = Elem<T>::st(v[i + j]);
      stg_vec(p + col + i, a);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < cols) p[col + i] = Elem<T>::st(v[i]);
  }
}

// |x| for a block's maximum: NaN left out, infinities as FLT_MAX
__device__ __forceinline__ float mx_abs(float v) { return clamp_flt_max(abs_or_zero(v)); }

// 8 values -> 8 E2M1 codes of v / 2^e (unscale = 2^e): v_cvt_scalef32_pk_fp4_f32 rounds to nearest,
// halves to the even code, and saturates; it turns NaN into +-6, so NaN enters as +inf
// (the convert is checked for scales 2^-125 .. 2^125: blocks further out are moved by 2^64, exactly)
__device__ __forceinline__ uint32_t e2m1_codes8(const float (&v)[8], float unscale) {
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = v[j] != v[j] ? __builtin_inff() : v[j];
  if (!(unscale >= 0x1p-100f && unscale <= 0x1p100f)) {
    const float k = unscale < 1.f ? 0x1p64f : 0x1p-64f;
    unscale *= k;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] *= k;
  }
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[0], a[1], unscale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[2], a[3], unscale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[4], a[5], unscale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, a[6], a[7], unscale, 3);
  return w;
}
// 8 values of at most 448 (or NaN) -> their E4M3 bytes
__device__ __forceinline__ uint2 e4m3_bytes8(const float (&a)[8]) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[0], a[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[2], a[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(a[4], a[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(a[6], a[7], hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}
// ... of v * s, saturating, NaN kept
__device__ __forceinline__ uint2 e4m3_codes8(const float (&v)[8], float s) {
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = clamp_nan(v[j] * s, -kE4M3Max, kE4M3Max);
  return e4m3_bytes8(a);
}
// A row's own factor d = max|x| / 448 (1 where that is 0): codes of the quotient x / d, rounded once.  A product with
// 1 / d would be rounded twice (codes flip at their borders), and 1 / d is past fp32 for d < 2^-128: rows of a
// small d have both sides multiplied by 2^64 first, exactly.
struct RowFactor {
  float d, by, lo, up, r, most;  // x / d = x up / by, r = 1 / by; |x up| is cut at `most`: infinities, a d rounded down
};
__device__ __forceinline__ RowFactor row_factor(float most) {
  RowFactor f;
  f.d = most / kE4M3Max;
  f.d = f.d > 0.f ? f.d : 1.f;
  f.up = f.d < 0x1p-64f ? 0x1p64f : 1.f;
  f.by = f.d * f.up;
  f.r = 1.0f / f.by;
  f.most = clamp_flt_max(f.by * kE4M3Max);
  return f;
}
// The quotients x / (most / 448) before the divisor is rounded, for rows whose factor d is that times something
// that they all share: by + lo is most / 448, |x| <= most.
__device__ __forceinline__ RowFactor row_quotient(float most, float d) {
  RowFactor f;
  f.d = d;
  f.up = most < 0x1p-56f ? 0x1p64f : 1.f;
  f.by = most * f.up / kE4M3Max;
  f.lo = __builtin_fmaf(-f.by, kE4M3Max, most * f.up) / kE4M3Max;
  f.r = 1.0f / f.by;
  return f;
}
__device__ __forceinline__ uint2 e4m3_quotients8(const float (&v)[8], const RowFactor &f) {
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = v[j] * f.up, y = x * f.r;
    const float e = __builtin_fmaf(-y, f.lo, __builtin_fmaf(-y, f.by, x));
    a[j] = __builtin_copysignf(__builtin_fmaf(e, f.r, y), x);
  }
  return e4m3_bytes8(a);
}
__device__ __forceinline__ uint2 e4m3_codes8(const float (&v)[8], const RowFactor &f) {
  float a[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = div_rn(clamp_nan(v[j] * f.up, -f.most, f.most), f.by, f.r);
  return e4m3_bytes8(a);
}

// One block of 32 in 4 consecutive lanes of 8 values: codes to the row q, the exponent byte to sc[]
template <int KIND>
__device__ __forceinline__ void mx_store8(const float (&v)[8], int64_t col, uint8_t *q, uint8_t *sc, bool live) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, mx_abs(v[j]));
  m = group_max_f<4>(m);
  float scale, unscale;
  e8m0_scale(m, KIND == MTQ_MXFP4 ? 6.0f : kE4M3Max, scale, unscale);
  if (!live) return;
  if constexpr (KIND == MTQ_MXFP4)
    *reinterpret_cast<uint32_t *>(q + col / 2) = e2m1_codes8(v, unscale);
  else
    *reinterpret_cast<uint2 *>(q + col) = e4m3_codes8(v, scale);
  if ((col & 31) == 0) {
    // unscale = 2^e, e in [-127, 127]: its exponent field, 0 for the subnormal 2^-127
    sc[col / 32] = (uint8_t)((__float_as_uint(unscale) >> 23) & 0xff);
  }
}
template <bool VEC>
__device__ __forceinline__ void fp8_store8(uint2 w, int64_t col, int64_t cols, uint8_t *q) {
  if constexpr (VEC) {
    *reinterpret_cast<uint2 *>(q + col) = w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (col + j < cols) q[col + j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
  }
}

// ---- sums and maxima over a workgroup (its waves' results through LDS, in wave order) ----------
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// ---- residual addition + RMS norm + quantised output ------------------------------------------
// h = RN_T(x + r); y = h * rsqrt(mean(h^2) + eps) * w in fp32, quantised from the fp32 value (no
// rounding of y to T in between: an unfused norm rounds there because it has to store y).
// Bound by HBM: x, r, h and a byte of codes per element, each touched once.  A workgroup takes one
// row and keeps it in registers (NV groups of 8 columns a lane) between the sum of squares and the
// output, so nothing is read twice.
// A code flips where y lies within its own error of a rounding border, a block's exponent where its maximum
// does, so that error is kept small: squares are summed in fp32 by eights and those sums in double, rsqrt is a
// pair of floats, and x * w of 16-bit operands is exact before the one product.  The MX formats, whose
// factors are powers of two, take y rounded to odd where it matters (round_odd): rounding that again to a code,
// or comparing it with a border, is then as good as y itself (16384 x 4096: 2 to 5 codes off by a step, 20 to
// 40 without; 94 us with, 88 without).  FP8 per token takes y / (max|y| / 448) = p / (max|p| / 448), p = x w: the
// root cancels, and of 2501 x 5000 codes 1 to 3 are off by a step (quotients that fp32 rounds onto a border).
// us: 16 x 4096 with residual 5 (a launch); 16384 x 4096 with residual 94 to MXFP8 and MXFP4, 85 to FP8 per tensor, 90
// per token (472 MB: 5.0 TB/s, 5.5, 5.2; a copy of 1 GiB 5.2, a sum of two such tensors 6.0); 2501 x 5000 fp16 per
// token 15.6 (37 MB, 2.4 TB/s; a row is less than a workgroup can hide).
struct NormArgs {
  const void *x, *r, *w;
  void *h;
  uint8_t *q;
  void *scale;
  const float *amax;
  int64_t xs, rs, cols;
  double eps;
  int w_dtype;
};

// v = p * (rh + rl) rounded to nearest -> toward zero, the last bit set where something was cut
__device__ __forceinline__ float round_odd(float v, float p, float rh, float rl) {
  const float rest = __builtin_fmaf(p, rh, -v) + p * rl;
  const uint32_t cut = rest < 0.f || rest > 0.f ? 1u : 0u;  // (an infinite v: rest is NaN)
  const uint32_t up = (__float_as_uint(rest) ^ __float_as_uint(v)) >> 31;
  return __uint_as_float((__float_as_uint(v) - (up & cut)) | cut);
}

template <typename T, int KIND, int NV, bool VEC>
__global__ __launch_bounds__(1024) void rms_norm_kernel(NormArgs a) {
  __shared__ double red[16];
  __shared__ float redm[16];
  constexpr bool MX = KIND == MTQ_MXFP4 || KIND == MTQ_MXFP8, TOKEN = KIND == MTQ_FP8_TOKEN;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nw = blockDim.x >> 6;
  const T *x = reinterpret_cast<const T *>(a.x) + row * a.xs;
  float f[NV][8];
  double ss = 0.0;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int64_t col = 8 * ((int64_t)u * blockDim.x + tid);
    if (col >= a.cols) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[u][j] = 0.f;
      continue;
    }
    load8<T, VEC>(x, col, a.cols, f[u]);
    if (a.r) {
      float r[8];
      load8<T, VEC>(reinterpret_cast<const T *>(a.r) + row * a.rs, col, a.cols, r);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[u][j] = Elem<T>::ld(Elem<T>::st(f[u][j] + r[j]));
      store8<T, VEC>(reinterpret_cast<T *>(a.h) + row * a.cols, col, a.cols, f[u]);
    }
    float s8 = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s8 = __builtin_fmaf(f[u][j], f[u][j], s8);
    ss += (double)s8;
  }
  ss = wave_sum(ss);
  if (lane == 0) red[wave] = ss;
  __syncthreads();
  ss = 0.0;
  for (int i = 0; i < nw; ++i) ss += red[i];
  const double rd = 1.0 / __builtin_sqrt(ss / (double)a.cols + a.eps);
  const float rh = (float)rd, rl = (float)(rd - (double)rh);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int64_t col = 8 * ((int64_t)u * blockDim.x + tid);
    if (col >= a.cols) continue;
    float w[8];
    if (a.w_dtype == MTQ_F32)
      load8<float, VEC>(reinterpret_cast<const float *>(a.w), col, a.cols, w);
    else
      load8<T, VEC>(reinterpret_cast<const T *>(a.w), col, a.cols, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = f[u][j] * w[j];
      f[u][j] = MX || TOKEN ? p : __builtin_fmaf(p, rh, p * rl);
    }
  }
  float s = 1.f;
  RowFactor rf{};
  bool regular = true;
  if constexpr (TOKEN) {
    float m = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, mx_abs(f[u][j]));  // columns past the row are 0
    m = wave_max(m);
    if (lane == 0) redm[wave] = m;
    __syncthreads();
    m = 0.f;
    for (int i = 0; i < nw; ++i) m = fmaxf(m, redm[i]);
    // y / (max|y| / 448) = p / (max|p| / 448): the root cancels, and with it y's own roundings
    const double top = (double)m * rd;  // max|y|
    const float d = (float)(top / (double)kE4M3Max);
    regular = rd < __builtin_inf() && m < 3.402823466e38f && d > 0.f && (float)top < __builtin_inff();
    if (regular) {
      rf = row_quotient(m, d);
    } else {  // rows of y = 0, NaN, infinities, or below what a factor can be: through y itself
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) f[u][j] *= (float)rd;
      const bool inf = rd > 0.0 && (m == 3.402823466e38f || (m > 0.f && (float)top == __builtin_inff()));
      rf = row_factor(inf ? 3.402823466e38f : 0.f);
    }
    if (tid == 0) reinterpret_cast<float *>(a.scale)[row] = rf.d;
  } else if constexpr (KIND == MTQ_FP8_TENSOR) {
    const Fp8Q p = make_fp8q(*a.amax);
    s = p.s;
    if (row == 0 && tid == 0) *reinterpret_cast<float *>(a.scale) = p.inv;
  }
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int64_t col = 8 * ((int64_t)u * blockDim.x + tid);
    if constexpr (MX) {
      // a block's 4 lanes are all live or all past the row (cols % 32 == 0)
      uint8_t *q = a.q + row * (KIND == MTQ_MXFP4 ? a.cols / 2 : a.cols);
      float v[8];
      uint32_t low = ~0u;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = __builtin_fmaf(f[u][j], rh, f[u][j] * rl);
        const uint32_t b = __float_as_uint(v[j]) & 0x7ffff;
        low = low < b ? low : b;
      }
      // halfway between codes, or a border, only where the bits below the 4th are zeros
      if (__builtin_amdgcn_ballot_w64(low == 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = round_odd(v[j], f[u][j], rh, rl);
      }
      mx_store8<KIND>(v, col, q, reinterpret_cast<uint8_t *>(a.scale) + row * (a.cols / 32), col < a.cols);
    } else if (col < a.cols) {
      const uint2 w = !TOKEN ? e4m3_codes8(f[u], s) : regular ? e4m3_quotients8(f[u], rf) : e4m3_codes8(f[u], rf);
      fp8_store8<VEC>(w, col, a.cols, a.q + row * a.cols);
    }
  }
}

template <typename T, int KIND, bool VEC>
int launch_norm(const NormArgs &all, int64_t rows, hipStream_t stream) {
  // 256 lanes of 8 columns a group, up to 4 groups in registers; wider rows take more lanes
  const int64_t groups = (all.cols + 7) / 8;
  int threads = 256;
  while (threads < 1024 && groups > 4 * threads) threads *= 2;
  if (groups < 256) threads = (int)((groups + 63) / 64 * 64);
  const int nv = (int)((groups + threads - 1) / threads);
  return in_launches(rows, threads, [&](int64_t r, int64_t n) {
    NormArgs a = all;
    a.x = reinterpret_cast<const T *>(all.x) + r * all.xs;
    if (all.r) a.r = reinterpret_cast<const T *>(all.r) + r * all.rs, a.h = reinterpret_cast<T *>(all.h) + r * all.cols;
    a.q = all.q + r * (KIND == MTQ_MXFP4 ? all.cols / 2 : all.cols);
    if (KIND == MTQ_FP8_TOKEN) a.scale = reinterpret_cast<float *>(all.scale) + r;
    if (KIND == MTQ_MXFP4 || KIND == MTQ_MXFP8) a.scale = reinterpret_cast<uint8_t *>(all.scale) + r * (all.cols / 32);
    const unsigned g = (unsigned)n;
    if (nv <= 1)
      rms_norm_kernel<T, KIND, 1, VEC><<<g, threads, 0, stream>>>(a);
    else if (nv <= 2)
      rms_norm_kernel<T, KIND, 2, VEC><<<g, threads, 0, stream>>>(a);
    else if (nv <= 4)
      rms_norm_kernel<T, KIND, 4, VEC><<<g, threads, 0, stream>>>(a);
    else
      rms_norm_kernel<T, KIND, 8, VEC><<<g, threads, 0, stream>>>(a);
  });
}
template <typename T, int KIND> int launch_norm_v(const NormArgs &a, bool vec, int64_t rows, hipStream_t stream) {
  return vec ? launch_norm<T, KIND, true>(a, rows, stream) : launch_norm<T, KIND, false>(a, rows, stream);
}
template <typename T> int launch_norm_k(const NormArgs &a, int kind, bool vec, int64_t rows, hipStream_t stream) {
  switch (kind) {
  case MTQ_MXFP4: return launch_norm_v<T, MTQ_MXFP4>(a, vec, rows, stream);
  case MTQ_MXFP8: return launch_norm_v<T, MTQ_MXFP8>(a, vec, rows, stream);
  case MTQ_FP8_TENSOR: return launch_norm_v<T, MTQ_FP8_TENSOR>(a, vec, rows, stream);
  default: return launch_norm_v<T, MTQ_FP8_TOKEN>(a, vec, rows, stream);
  }
}

// v_cvt_scalef32_pk_fp4_{bf16,f16} into byte SEL of a dword of codes
template <typename T> struct Fp4Pair;
template <> struct Fp4Pair<__bf16> {
  typedef bf16x2_t v2;
  template <int SEL> static __device__ __forceinline__ uint32_t cvt(uint32_t w, v2 p, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, p, s, SEL);
  }
};
template <> struct Fp4Pair<_Float16> {
  typedef f16x2_t v2;
  template <int SEL> static __device__ __forceinline__ uint32_t cvt(uint32_t w, v2 p, float s) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, p, s, SEL);
  }
};

// 8 packed 16-bit values of one lane, 4 lanes a block: MXFP4 codes as block_codes() below makes them
template <typename T>
__device__ __forceinline__ void mxfp4_store8_packed(const u32x4 &x, int64_t col, uint8_t *q, uint8_t *sc, bool live) {
  u16x2_t mx = {0, 0};
#pragma unroll
  for (int j = 0; j < 4; ++j) mx = __builtin_elementwise_max(mx, __builtin_bit_cast(u16x2_t, x[j] & 0x7fff7fffu));
  const uint32_t mb = group_max_u32<4>(mx.x > mx.y ? mx.x : mx.y);
  float un, scale;
  e8m0_scale(mb >= Fp4Native<T>::kInfBits ? 3.402823466e38f : half_bits_to_float<T>(mb), 6.0f, scale, un);
  if (mb <= Fp4Native<T>::kInfBits && un >= 0x1p-100f && un <= 0x1p100f) {  // uniform over the block's lanes
    if (!live) return;
    uint32_t w = 0;
    w = Fp4Pair<T>::template cvt<0>(w, __builtin_bit_cast(typename Fp4Pair<T>::v2, (uint32_t)x[0]), un);
    w = Fp4Pair<T>::template cvt<1>(w, __builtin_bit_cast(typename Fp4Pair<T>::v2, (uint32_t)x[1]), un);
    w = Fp4Pair<T>::template cvt<2>(w, __builtin_bit_cast(typename Fp4Pair<T>::v2, (uint32_t)x[2]), un);
    w = Fp4Pair<T>::template cvt<3>(w, __builtin_bit_cast(typename Fp4Pair<T>::v2, (uint32_t)x[3]), un);
    *reinterpret_cast<uint32_t *>(q + col / 2) = w;
    if ((col & 31) == 0) sc[col / 32] = (uint8_t)((__float_as_uint(un) >> 23) & 0xff);
  } else {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = half_bits_to_float<T>(x[j] & 0xffffu), v[2 * j + 1] = half_bits_to_float<T>(x[j] >> 16);
    mx_store8<MTQ_MXFP4>(v, col, q, sc, live);
  }
}

// ---- quantising rows ---------------------------------------------------------------------------
// MX and per-tensor FP8: 8 values a lane over all rows (a block's 4 lanes are neighbours).  Bound by HBM: 16384 x 4096
// bf16 to MXFP4 32 us (5.3 TB/s), to MXFP8 43 (4.8), to FP8 per tensor 38 (5.4), per token 45 (4.5).
template <typename T, int KIND, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *__restrict__ x, int64_t xs, int64_t rows, int64_t cols,
                                                          const float *__restrict__ amax, uint8_t *__restrict__ q,
                                                          void *__restrict__ scale) {
  const int64_t gpr = (cols + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / gpr, col = (i - row * gpr) * 8;
  const bool live = row < rows;
  if constexpr (KIND == MTQ_MXFP4 && VEC && sizeof(T) == 2) {
    u32x4 w = {0, 0, 0, 0};
    if (live) w = *reinterpret_cast<const u32x4 *>(x + row * xs + col);
    mxfp4_store8_packed<T>(w, col, q + row * (cols / 2), reinterpret_cast<uint8_t *>(scale) + row * (cols / 32), live);
    return;
  }
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live) load8<T, VEC>(x + row * xs, col, cols, v);
  if constexpr (KIND == MTQ_FP8_TENSOR) {
    const Fp8Q p = make_fp8q(*amax);
    if (i == 0) *reinterpret_cast<float *>(scale) = p.inv;
    if (live) fp8_store8<VEC>(e4m3_codes8(v, p.s), col, cols, q + row * cols);
  } else {
    mx_store8<KIND>(v, col, q + row * (KIND == MTQ_MXFP4 ? cols / 2 : cols),
                    reinterpret_cast<uint8_t *>(scale) + row * (cols / 32), live);
  }
}

// per token: one workgroup a row, two passes over it (the second from the caches)
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void token_quantize_kernel(const T *__restrict__ x, int64_t xs, int64_t cols,
                                                             uint8_t *__restrict__ q, float *__restrict__ scale) {
  __shared__ float red[4];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  x += row * xs;
  float m = 0.f;
  for (int64_t col = 8 * tid; col < cols; col += 2048) {
    float v[8];
    load8<T, VEC>(x, col, cols, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, mx_abs(v[j]));
  }
  m = wave_max(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const RowFactor f = row_factor(m);
  if (tid == 0) scale[row] = f.d;
  for (int64_t col = 8 * tid; col < cols; col += 2048) {
    float v[8];
    load8<T, VEC>(x, col, cols, v);
    fp8_store8<VEC>(e4m3_codes8(v, f), col, cols, q + row * cols);
  }
}

template <typename T, bool VEC>
int launch_quantize(const T *x, int64_t xs, int64_t rows, int64_t cols, int kind, const float *amax, uint8_t *q,
                    void *scale, hipStream_t stream) {
  const int64_t gpr = (cols + 7) / 8;
  return in_launches(rows, kind == MTQ_FP8_TOKEN ? 256 : gpr, [&](int64_t r, int64_t n) {
    const T *const xr = x + r * xs;
    uint8_t *const qr = q + r * (kind == MTQ_MXFP4 ? cols / 2 : cols);
    void *const sr = is_mx(kind) ? (uint8_t *)scale + r * (cols / 32) : scale;
    const unsigned g = (unsigned)((n * gpr + 255) / 256);
    switch (kind) {
    case MTQ_MXFP4: mx_quantize_kernel<T, MTQ_MXFP4, VEC><<<g, 256, 0, stream>>>(xr, xs, n, cols, amax, qr, sr); break;
    case MTQ_MXFP8: mx_quantize_kernel<T, MTQ_MXFP8, VEC><<<g, 256, 0, stream>>>(xr, xs, n, cols, amax, qr, sr); break;
    case MTQ_FP8_TENSOR:
      mx_quantize_kernel<T, MTQ_FP8_TENSOR, VEC><<<g, 256, 0, stream>>>(xr, xs, n, cols, amax, qr, sr);
      break;
    default: token_quantize_kernel<T, VEC><<<(unsigned)n, 256, 0, stream>>>(xr, xs, cols, qr, (float *)scale + r); break;
    }
  });
}

// 4 consecutive columns of a row of y: v * f + bias, rounded once
template <typename T>
__device__ __forceinline__ void out4(T *y, const f32x4 &v, float f, const void *bias, int bias_f32, int64_t n, int N) {
  float o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    o[k] = v[k] * f;
    if (bias && n + k < N) o[k] += bias_f32 ? reinterpret_cast<const float *>(bias)[n + k] : Elem<T>::ld(reinterpret_cast<const T *>(bias)[n + k]);
  }
  if (n + 4 <= N) {  // one store, of any alignment (rows of an odd N)
    T e[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) e[k] = Elem<T>::st(o[k]);
    __builtin_memcpy(y + n, e, sizeof(e));
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < N) y[n + k] = Elem<T>::st(o[k]);
  }
}

// 32 values of one lane in 16 packed 16-bit pairs -> its block's E2M1 codes and exponent byte: the
// largest magnitude from packed integer maxima of the bit patterns (NaN patterns sort above infinity),
// the codes from v_cvt_scalef32_pk_fp4_{bf16,f16}; a block with a NaN or an exponent outside -100 .. 100
// takes the fp32 forms
template <typename T> __device__ __forceinline__ void block_codes(const u32x4 (&x)[4], u32x4 &codes, int &exponent) {
  u16x2_t mx = {0, 0};
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = __builtin_elementwise_max(mx, __builtin_bit_cast(u16x2_t, x[t][j] & 0x7fff7fffu));
  const uint32_t mb = mx.x > mx.y ? mx.x : mx.y;
  float m = mb == Fp4Native<T>::kInfBits ? 3.402823466e38f : half_bits_to_float<T>(mb);
  const bool nan = mb > Fp4Native<T>::kInfBits;
  if (nan) {
    m = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m = fmaxf(m, mx_abs(half_bits_to_float<T>(x[t][j] & 0xffffu)));
        m = fmaxf(m, mx_abs(half_bits_to_float<T>(x[t][j] >> 16)));
      }
  }
  float scale, un;
  e8m0_scale(m, 6.0f, scale, un);
  exponent = (int)((__float_as_uint(un) >> 23) & 0xff);
  if (!nan && un >= 0x1p-100f && un <= 0x1p100f) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      uint32_t w = 0;
      typename Fp4Pair<T>::v2 p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = __builtin_bit_cast(typename Fp4Pair<T>::v2, (uint32_t)x[t][j]);
      w = Fp4Pair<T>::template cvt<0>(w, p[0], un);
      w = Fp4Pair<T>::template cvt<1>(w, p[1], un);
      w = Fp4Pair<T>::template cvt<2>(w, p[2], un);
      w = Fp4Pair<T>::template cvt<3>(w, p[3], un);
      codes[t] = w;
    }
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = half_bits_to_float<T>(x[t][j] & 0xffffu), v[2 * j + 1] = half_bits_to_float<T>(x[t][j] >> 16);
      codes[t] = e2m1_codes8(v, un);
    }
  }
}

// ---- y = xq . W^T for few rows -------------------------------------------------------------------
// v_mfma_scale_f32_16x16x128_f8f6f4, first operand 16 rows of W, second 16 rows of xq: lane
// (r = lane & 15, g = lane >> 4) gives row r's block g of a 128-column step (E2M1: 16 bytes) and that
// block's exponent byte; an E4M3 operand gives columns 16 g .. + 15 and 64 + 16 g .. + 15 of the step
// (the layout was read off the instruction on the card), its lane's byte still being block g's.  The
// result holds y^T: lane (r, g) has row r of xq and 4 consecutive rows 4 g .. of W.
//
// Rounding, read off the instruction with chosen codes: products of E2M1 by E2M1 are added exactly and then in
// fp32 (cut below 2^-23 of the largest term).  With an E4M3 operand the products of eight neighbouring columns
// are first added in fixed point whose last bit is 2^-13 of 2^(their largest sum of exponents), cut toward
// zero.  That is kept: it is far below the 2^-4 with which E4M3 rounded x, on average 2^-19 of sum |x w| (at
// most 7 * 2^-13 of the largest product of every eight), and exact sums would need fp16 operands at half the
// rate and twice the LDS.
//
// The call is bound by reading W once (17/32 byte per weight), so a workgroup is WAVES waves that split
// K over the same 16 * NT rows of W, every wave streaming its part straight into the operand registers
// (nothing of W is shared, so LDS would only add a trip), and the partial tiles meet in LDS at the end,
// summed in wave order.  A wave takes 512 columns at a time: 4 NT loads of codes, one 16-byte load of
// exponents a row, all in flight together; the other waves of the SIMD cover the rest.
// 1 x 4096 x 4096, quantised on the way: 6.0 us (8.9 MB).
struct SkinnyArgs {
  const void *x;             // xq, or the 16-bit activations (FUSED)
  const uint8_t *xsc;        // exponent bytes [M, K / 32] (MX formats)
  const float *xf;           // factor per row (per token) or one (per tensor)
  const uint8_t *w, *wsc;    // [N, K / 2], [N, K / 32]
  const void *bias;
  void *y;
  int64_t xs;                // row stride of the 16-bit activations
  int M, N, K, tiles_n;
  int xf_stride;             // 1: a factor per row, 0: one
  int bias_f32;
};

enum { kOpFp4 = 0, kOpFp8 = 1, kOpFused = 2 };

__device__ __forceinline__ u32x4 load16_any(const uint8_t *p) {  // any alignment
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

template <typename T, int OP, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, NT == 4 ? 2 : 4) void mx_skinny_kernel(SkinnyArgs a) {
  __shared__ f32x4 red[WAVES][NT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
  const int n0 = (blockIdx.x % a.tiles_n) * 16 * NT, m0 = (blockIdx.x / a.tiles_n) * 16;
  const int nb = a.K / 32, batches = (nb + 15) / 16;
  const int b0 = (int)((int64_t)batches * wave / WAVES), b1 = (int)((int64_t)batches * (wave + 1) / WAVES);
  const uint8_t *wp[NT], *wsp[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + 16 * j + r < a.N ? n0 + 16 * j + r : a.N - 1;  // rows past N: never stored
    wp[j] = a.w + (int64_t)n * (a.K / 2);
    wsp[j] = a.wsc + (int64_t)n * nb;
  }
  const int64_t xm = m0 + r < a.M ? m0 + r : a.M - 1;
  const uint8_t *const xp = reinterpret_cast<const uint8_t *>(a.x) + xm * (OP == kOpFused ? a.xs * 2 : OP == kOpFp4 ? a.K / 2 : a.K);
  const uint8_t *const xsp = a.xsc + xm * nb;
  f32x4 acc[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

  constexpr int XV = OP == kOpFused ? 4 : OP == kOpFp8 ? 2 : 1;
  constexpr bool XS = OP != kOpFused;
  struct Batch {
    u32x4 w[NT][4], ws[NT], x[4][XV], xs;
  } st;
  auto load = [&](int b, Batch &d) {
    const int blk0 = 16 * b + g;
    if (16 * b + 16 <= nb) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int u = 0; u < 4; ++u) d.w[j][u] = *reinterpret_cast<const u32x4 *>(wp[j] + (int64_t)(blk0 + 4 * u) * 16);
        d.ws[j] = load16_any(wsp[j] + 16 * b);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int t = 0; t < XV; ++t)
          d.x[u][t] = *reinterpret_cast<const u32x4 *>(
              OP == kOpFp8 ? xp + 512 * (int64_t)b + 128 * u + 64 * t + 16 * g
                           : xp + (int64_t)(blk0 + 4 * u) * (OP == kOpFused ? 64 : 16) + 16 * t);
      if constexpr (XS) {
        d.xs = u32x4{0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu};
        if (a.xsc) d.xs = load16_any(xsp + 16 * b);
      }
    } else {  // the end of a K that 512 does not divide: what lies past it becomes zero codes of W
      const uint32_t sh = 8 * g;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int blk = blk0 + 4 * u, bc = blk < nb ? blk : 0;
        const bool in = blk < nb;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const u32x4 v = *reinterpret_cast<const u32x4 *>(wp[j] + (int64_t)bc * 16);
          d.w[j][u] = in ? v : u32x4{0, 0, 0, 0};
          d.ws[j][u] = (uint32_t)(in ? wsp[j][bc] : 127) << sh;
        }
#pragma unroll
        for (int t = 0; t < XV; ++t) {
          const int k = 512 * b + 128 * u + 64 * t + 16 * g;
          d.x[u][t] = *reinterpret_cast<const u32x4 *>(OP == kOpFp8 ? xp + (k < a.K ? k : 0)
                                                                    : xp + (int64_t)bc * (OP == kOpFused ? 64 : 16) + 16 * t);
        }
        if constexpr (XS) d.xs[u] = (uint32_t)(a.xsc ? xsp[bc] : 127) << sh;
      }
    }
  };
  auto use = [&](const Batch &d) {
    const uint32_t sh = 8 * g;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      i32x8 xf;
      int xs;
      if constexpr (OP == kOpFused) {
        u32x4 c;
        block_codes<T>(d.x[u], c, xs);
        xf = i32x8{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
      } else {
        xs = (int)(d.xs[u] >> sh);
        if constexpr (OP == kOpFp4)
          xf = i32x8{(int)d.x[u][0].x, (int)d.x[u][0].y, (int)d.x[u][0].z, (int)d.x[u][0].w, 0, 0, 0, 0};
        else
          xf = i32x8{(int)d.x[u][0].x, (int)d.x[u][0].y, (int)d.x[u][0].z, (int)d.x[u][0].w,
                     (int)d.x[u][XV - 1].x, (int)d.x[u][XV - 1].y, (int)d.x[u][XV - 1].z, (int)d.x[u][XV - 1].w};
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const i32x8 wf = {(int)d.w[j][u].x, (int)d.w[j][u].y, (int)d.w[j][u].z, (int)d.w[j][u].w, 0, 0, 0, 0};
        acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[j], 4, OP == kOpFp8 ? 0 : 4, 0, (int)(d.ws[j][u] >> sh), 0, xs);
      }
    }
  };
  for (int b = b0; b < b1; ++b) {
    load(b, st);
    use(st);
  }

#pragma unroll
  for (int j = 0; j < NT; ++j) red[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave < NT) {
    const int m = m0 + r, n = n0 + 16 * wave + 4 * g;
    f32x4 v = red[0][wave][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += red[w][wave][lane];
    if (m < a.M) {
      const float f = a.xf ? a.xf[(int64_t)m * a.xf_stride] : 1.f;
      out4<T>(reinterpret_cast<T *>(a.y) + (int64_t)m * a.N, v, f, a.bias, a.bias_f32, n, a.N);
    }
  }
}

template <typename T, int OP> int launch_skinny(const SkinnyArgs &all, hipStream_t stream) {
  // tiles of W that share a read of xq: four where that leaves a workgroup for nearly every CU (16 rows of
  // E4M3 against 28672 x 8192: 33 us, two 40, one 49), one where there are too few of them
  const int64_t gm = (all.M + 15) / 16, cus = host_num_cus();
  auto go = [&](auto nt, auto waves) {
    constexpr int NT = decltype(nt)::value, WAVES = decltype(waves)::value;
    const int tiles_n = (all.N + 16 * NT - 1) / (16 * NT);
    return in_launches(gm, (int64_t)tiles_n * 64 * WAVES, [&](int64_t t, int64_t n) {
      SkinnyArgs a = all;
      const int64_t m = 16 * t;
      a.x = reinterpret_cast<const uint8_t *>(all.x) + m * (OP == kOpFused ? all.xs * 2 : OP == kOpFp4 ? all.K / 2 : all.K);
      if (all.xsc) a.xsc = all.xsc + m * (all.K / 32);
      if (all.xf) a.xf = all.xf + m * all.xf_stride;
      a.y = reinterpret_cast<T *>(all.y) + m * all.N;
      a.M = (int)(all.M - m < 16 * n ? all.M - m : 16 * n);
      a.tiles_n = tiles_n;
      mx_skinny_kernel<T, OP, NT, WAVES><<<(unsigned)(n * tiles_n), 64 * WAVES, 0, stream>>>(a);
    });
  };
  if constexpr (OP != kOpFused) {
    if (all.N >= 48 * cus) return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
  }
  return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
}

// ---- y = xq . W^T for many rows ------------------------------------------------------------------
// Bound by the matrix cores (16x16x128: 16 cycles of E2M1 x E2M1, 32 with an E4M3 operand).  A
// workgroup is 8 waves on a 256 x 256 tile of y, a wave on 128 rows of xq x 64 of W; K advances by
// BK = 256 columns (E2M1) or 128 (E4M3 rows of xq), so a K tile is 128 bytes of each xq row in LDS and
// as many MFMA cycles in both forms.  The schedule is that of the 16-bit search kernel
// (mtq_awq_gemm.hip, awq_search_pp_kernel): operands come by LDS-DMA into two buffers of four
// half-tiles, a K tile is four phases of a 64 x 32 quadrant each, every phase issues the DMA of one
// half-tile two to five phases ahead and waits with a counted vmcnt, and waves 4-7 run one barrier
// behind waves 0-3, so that one wave of a SIMD reads LDS while the other multiplies.  The K tiles of all
// the workgroup's tiles of y are one stream: what is loaded ahead at a tile's end is the next tile's.
// us for xq 8192 x 4096, W 14336 x 4096: 247 to 254 E2M1 (3.8 PFLOP/s; each further 4096 columns:
// 193, 5.0), 371 to 384 E4M3 (2.5); without the stores 222 (of 254) and 349 (of 371): they come from all CUs at
// once, 128 KiB a tile, and loads are waited for in order behind them.
// The exponent bytes are laid out by K tile first ([K tile][row][BK / 32], zero past the matrix; one
// small pass per operand), so a tile's are two DMAs a wave into a ring of three; a lane's exponents of
// both 128-column steps are one 16-bit read (bytes 2 g + s for its block 4 s + g).
// LDS rows are 16-byte chunks stored at chunk ^ f(row) (the XOR is applied to the global address),
// f = row / 2 for 128-byte rows and -(row / 4) for 64-byte ones: a 128-bit read serves lanes 0-3, 12-15
// and 20-27 together (then the others of 0-31), whose 16 chunks then fall on different banks
// (SQ_LDS_BANK_CONFLICT is 6 % of SQ_LDS_IDX_ACTIVE; blocks 2 g + s, which conflict, 266 us against 260).
// Columns past K (K % BK != 0): chunks there are read from the row's first chunk of the tile, and
// their exponents are 2^-127 on both sides, so what they add vanishes (below 2^-230).
struct PpArgs {
  const uint8_t *x, *w, *xsc, *wsc;  // xsc / wsc: tiled exponents; xsc null: all 2^0
  const float *xf;
  const void *bias;
  void *y;
  int M, N, K, tiles_m, tiles_n, xf_stride, bias_f32;
};
constexpr int kPpTile = 256, kPpThreads = 512;
constexpr int pp_bk(bool f8) { return f8 ? 128 : 256; }

template <int N> __device__ __forceinline__ void wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t wave_rsrc(const void *base, uint32_t bytes) {
  const uint64_t a = (uint64_t)base;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void *)(((uint64_t)hi << 32) | lo), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}
// buffer_load ... lds: BYTES (4 or 16) a lane to lds + lane * BYTES (the builtin exists in the device pass only)
#if defined(__HIP_DEVICE_COMPILE__)
#define MX_DMA(rsrc, lds, bytes, voff, soff) \
  __builtin_amdgcn_raw_ptr_buffer_load_lds((rsrc), (__attribute__((address_space(3))) void *)(lds), bytes, (voff), (soff), 0, 0)
#else
#define MX_DMA(rsrc, lds, bytes, voff, soff) ((void)(rsrc), (void)(lds), (void)(voff), (void)(soff))
#endif

template <bool F8> __device__ __forceinline__ f32x4 pp_mma(const i32x8 &w, const i32x8 &x, f32x4 c, int s, int ws, int xs) {
  if (F8) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 0, 0, ws, 0, xs);
  return s ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, 1, ws, 1, xs)
           : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, 0, ws, 0, xs);
}

// 16 bytes of a row of y
template <typename T> __device__ __forceinline__ void pp_store(T *y, const T (&e)[16 / sizeof(T)], int64_t n, int N) {
  constexpr int EC = 16 / sizeof(T);
  if (n + EC <= N) {  // of any alignment (rows of an odd N)
    __builtin_memcpy(y + n, e, 16);
  } else {
#pragma unroll
    for (int k = 0; k < EC; ++k)
      if (n + k < N) y[n + k] = e[k];
  }
}

// W's row at LDS row r of 32 (two operands of 16): operand 1's rows come between operand 0's by fours, so that a
// lane's results of both (rows 4 fq .. of each) are 8 columns of y in a piece
__device__ __forceinline__ int pp_wrow(int r) { return (r & 12) << 1 | (r & 16) >> 2 | (r & 3); }

template <typename T, bool F8>
__global__ __launch_bounds__(kPpThreads) void mx_pp_kernel(PpArgs p) {
  constexpr int BK = pp_bk(F8), NB = BK / 32;         // K tile, its blocks
  constexpr int AH = 128 * 128, BH = 128 * (BK / 2);  // bytes of a half-tile of xq, of W
  constexpr int BUF = 2 * AH + 2 * BH, SOP = kPpTile * NB, SBUF = 2 * SOP;
  constexpr int AU = 2, BU = F8 ? 1 : 2, SU = F8 ? 1 : 2;  // DMAs a wave: half-tiles, a tile's exponents
  constexpr int CNT = 2 * AU + 2 * BU + SU;
  constexpr int NS = F8 ? 1 : 2;                       // 128-column steps of a K tile
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * BUF + 3 * SBUF + 8 * 2048];
  unsigned char *const sring = lds + 2 * BUF;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2, wn = wave & 3, fr = lane & 15, fq = lane >> 4;

  const int xrow = F8 ? p.K : p.K / 2, wrow = p.K / 2;  // bytes of a row
  const int nt = (p.K + BK - 1) / BK;
  const int xpad = p.tiles_m * kPpTile, wpad = p.tiles_n * kPpTile;  // rows of the tiled exponents
  const int xs_step = (p.xsc ? xpad : wpad) * NB, ws_step = wpad * NB;
  const int a_chunk = (lane & 7) ^ (((wave * 8 + (lane >> 3)) >> 1) & 7);
  const int b_chunk = F8 ? (lane & 3) ^ (-(lane >> 4) & 3) : a_chunk;
  // what to step back by where the chunk lies past K in the last tile (a chunk: 16 columns of E4M3, 32 of E2M1)
  const unsigned a_tail = (nt - 1) * BK + a_chunk * (F8 ? 16 : 32) < p.K ? 0 : a_chunk * 16;
  const unsigned b_tail = (nt - 1) * BK + b_chunk * 32 < p.K ? 0 : b_chunk * 16;

  // ---- a tile of y and its DMA sources.  Tile order: units of 8 row tiles x 4 column tiles on one
  // XCD at a time (its L2 then holds 12 operand panels for 32 workgroups), consecutive units on the
  // 8 XCDs; the workgroups (a multiple of 8) step through the order.
  const int mgn = (p.tiles_m + 7) / 8, total = (mgn * ((p.tiles_n + 3) / 4) + 7) / 8 * 8 * 32;
  int tm = 0, tn = 0;
  auto next_tile = [&](int &id) -> bool {
    for (; id < total; id += gridDim.x) {
      const int xcd = id % 8, li = id / 8, slot = li % 32, u = (li / 32) * 8 + xcd;
      tm = (u % mgn) * 8 + slot % 8;
      tn = (u / mgn) * 4 + slot / 8;
      if (tm < p.tiles_m && tn < p.tiles_n) return true;
    }
    return false;
  };
  __amdgpu_buffer_rsrc_t xr, wr, xsr, wsr;
  auto set_tile = [&]() {
    const int64_t m0 = (int64_t)tm * kPpTile, n0 = (int64_t)tn * kPpTile;
    const int rows_x = (int)(p.M - m0 < kPpTile ? p.M - m0 : kPpTile), rows_w = (int)(p.N - n0 < kPpTile ? p.N - n0 : kPpTile);
    xr = wave_rsrc(p.x + m0 * xrow, (uint32_t)rows_x * (uint32_t)xrow);
    wr = wave_rsrc(p.w + n0 * wrow, (uint32_t)rows_w * (uint32_t)wrow);
    // rows without exponents: any bytes (not read from LDS)
    xsr = wave_rsrc(p.xsc ? p.xsc + m0 * NB : p.wsc + n0 * NB, (uint32_t)(nt - 1) * xs_step + SOP);
    wsr = wave_rsrc(p.wsc + n0 * NB, (uint32_t)(nt - 1) * ws_step + SOP);
  };

  // xq half h, round u: LDS row rr = u * 64 + wave * 8 + lane / 8, chunk slot lane % 8, is row u * 128 + h * 64 +
  // rr % 64 of the tile; W half h: the same, or (64-byte rows) rr = wave * 16 + lane / 4, slot lane % 4, is row
  // rr / 32 * 64 + h * 32 + pp_wrow(rr % 32).  Rows past the matrix are out of their buffer's range (the row is
  // in the vector offset): they read as zeros and their results are not stored.
  const int b_rr = F8 ? wave * 16 + (lane >> 2) : wave * 8 + (lane >> 3);
  const unsigned a_off = (unsigned)(wave * 8 + (lane >> 3)) * (unsigned)xrow + a_chunk * 16;
  const unsigned b_off = (unsigned)((b_rr >> 5) * 64 + pp_wrow(b_rr & 31)) * (unsigned)wrow + b_chunk * 16;
  // K tile tt of set_tile's tile, into buffer `buf`
  auto load_a = [&](int h, int tt, int buf) {
    unsigned char *dst = lds + buf * BUF + h * AH + wave * 1024;
    const uint32_t soff = __builtin_amdgcn_readfirstlane((uint32_t)tt * 128);
    const unsigned off = a_off - (tt == nt - 1 ? a_tail : 0);
#pragma unroll
    for (int u = 0; u < AU; ++u) MX_DMA(xr, dst + u * 8192, 16, off + (unsigned)((u * 128 + h * 64) * xrow), soff);
  };
  auto load_b = [&](int h, int tt, int buf) {
    unsigned char *dst = lds + buf * BUF + 2 * AH + h * BH + wave * 1024;
    const uint32_t soff = __builtin_amdgcn_readfirstlane((uint32_t)tt * (BK / 2));
    const unsigned off = b_off - (tt == nt - 1 ? b_tail : 0);
#pragma unroll
    for (int u = 0; u < BU; ++u) MX_DMA(wr, dst + u * 8192, 16, off + (unsigned)((u * 128 + h * 32) * wrow), soff);
  };
  auto load_s = [&](int tt, int slot) {
    unsigned char *dst = sring + slot * SBUF;
    const uint32_t sx = __builtin_amdgcn_readfirstlane((uint32_t)tt * xs_step), sw = __builtin_amdgcn_readfirstlane((uint32_t)tt * ws_step);
    if constexpr (F8) {  // 1 KiB each: waves 0-3 and 4-7
      if (wave < 4)
        MX_DMA(xsr, dst + wave * 256, 4, (unsigned)(wave * 256 + lane * 4), sx);
      else
        MX_DMA(wsr, dst + SOP + (wave - 4) * 256, 4, (unsigned)((wave - 4) * 256 + lane * 4), sw);
    } else {
      MX_DMA(xsr, dst + wave * 256, 4, (unsigned)(wave * 256 + lane * 4), sx);
      MX_DMA(wsr, dst + SOP + wave * 256, 4, (unsigned)(wave * 256 + lane * 4), sw);
    }
  };
  // stream order of the DMAs: per K tile t  B1(t+1) | A1(t+1) | B0(t+2) | S(t+2) A0(t+2); CNT are those
  // issued after the half-tile that the next phase reads.  Past a tile's end comes the next tile of y: what is
  // two K tiles ahead belongs to it from the second half of K tile nt - 2 on, where the offsets change.

  // ---- fragments.  E2M1 operand, step s: block 4 s + fq (E4M3 form: block fq of 4); E4M3 operand:
  // columns 16 fq .. and 64 + 16 fq ..
  const int sw8 = (lane >> 1) & 7, sw4 = -(fr >> 2) & 3;
  auto ld4 = [&](const unsigned char *q) -> i32x8 {
    const u32x4 d = *reinterpret_cast<const u32x4 *>(q);
    return i32x8{(int)d.x, (int)d.y, (int)d.z, (int)d.w, 0, 0, 0, 0};
  };
  auto read_a = [&](const unsigned char *buf, int i, int s) -> i32x8 {
    const unsigned char *row = buf + (i >> 2) * AH + (grp * 64 + (i & 3) * 16 + fr) * 128;
    if constexpr (F8) {
      const u32x4 d = *reinterpret_cast<const u32x4 *>(row + ((fq ^ sw8) << 4));
      const u32x4 e = *reinterpret_cast<const u32x4 *>(row + (((4 + fq) ^ sw8) << 4));
      return i32x8{(int)d.x, (int)d.y, (int)d.z, (int)d.w, (int)e.x, (int)e.y, (int)e.z, (int)e.w};
    } else {
      return ld4(row + (((4 * s + fq) ^ sw8) << 4));
    }
  };
  auto read_b = [&](const unsigned char *buf, int j, int s) -> i32x8 {
    const unsigned char *row = buf + 2 * AH + (j >> 1) * BH + (wn * 32 + (j & 1) * 16 + fr) * (BK / 2);
    return ld4(row + (F8 ? (fq ^ sw4) << 4 : ((4 * s + fq) ^ sw8) << 4));
  };
  auto read_s = [&](const unsigned char *base, int row) -> int {
    if constexpr (F8) return base[row * NB + fq];
    return *reinterpret_cast<const uint16_t *>(base + row * NB + 2 * fq);
  };

  int id = blockIdx.x;
  if (!next_tile(id)) return;  // the whole workgroup, before any barrier
  set_tile();
  // what the phases before the first K tile would have issued
  load_b(0, 0, 0);
  load_s(0, 0);
  load_a(0, 0, 0);
  load_b(1, 0, 0);
  load_a(1, 0, 0);
  load_b(0, 1, 1);
  load_s(1, 1);
  load_a(0, 1, 1);
  wait_vm<CNT>();
  __builtin_amdgcn_s_barrier();
  int buf = 0, slot = 0;  // of the stream
  for (bool more = true; more;) {
    const int64_t m0 = (int64_t)tm * kPpTile + grp * 128, n0 = (int64_t)tn * kPpTile + wn * 64;
    f32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (grp == 1) __builtin_amdgcn_s_barrier();  // one barrier behind
    i32x8 af[4][NS], b0f[2][NS], b1f[2][NS];
    int sa[4], sb0[2], sb1[2];
    for (int t = 0; t < nt; ++t) {
      const unsigned char *cur = lds + buf * BUF;
      const unsigned char *sx = sring + slot * SBUF, *sw = sx + SOP;
      const int slot2 = slot == 0 ? 2 : slot - 1;  // two ahead
      const int t1 = t + 1 < nt ? t + 1 : 0, t2 = t + 2 < nt ? t + 2 : t + 2 - nt;
      // rows without exponents: 2^0, past K 2^-127
      const int unit = F8 && !p.xsc ? ((t == nt - 1 && (nt - 1) * BK + 32 * fq >= p.K) ? 0 : 127) : 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int mq = (q == 0 || q == 1) ? 0 : 1;
        const int nq = (q == 1 || q == 2) ? 1 : 0;
        if (q == 0 || q == 2) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int s = 0; s < NS; ++s) af[i][s] = read_a(cur, 4 * mq + i, s);
            sa[i] = F8 && !p.xsc ? unit : read_s(sx, grp * 128 + 16 * (4 * mq + i) + fr);
          }
        }
        if (q == 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int s = 0; s < NS; ++s) b0f[j][s] = read_b(cur, j, s);
            sb0[j] = read_s(sw, wn * 64 + pp_wrow(16 * j + fr));
          }
        }
        if (q == 1) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int s = 0; s < NS; ++s) b1f[j][s] = read_b(cur, 2 + j, s);
            sb1[j] = read_s(sw, wn * 64 + 32 + pp_wrow(16 * j + fr));
          }
        }
        if (q == 0) load_b(1, t1, buf ^ 1);
        if (q == 1) load_a(1, t1, buf ^ 1);
        if (q == 2) {
          if (t == nt - 2) {  // (nt >= 2)
            id += gridDim.x;
            more = next_tile(id);
            if (more) set_tile();  // else the last tile's own K tiles again, which nothing reads
          }
          load_b(0, t2, buf);
        }
        if (q == 3) {
          load_s(t2, slot2);
          load_a(0, t2, buf);
        }
        wait_vm<CNT>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[4 * mq + i][2 * nq + j] =
                  pp_mma<F8>(nq ? b1f[j][s] : b0f[j][s], af[i][s], acc[4 * mq + i][2 * nq + j], s, nq ? sb1[j] : sb0[j], sa[i]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_s_barrier();
      }
      slot = slot == 2 ? 0 : slot + 1;
      buf ^= 1;
    }
    // both halves of the workgroup store at a time: one behind the other, each would wait for the other's stores
    // (282 against 269 us)
    if (grp == 0) __builtin_amdgcn_s_barrier();
    // ---- y of the wave's 128 x 64: a lane holds y[m][n .. n + 7], m = 16 i + er, n = 32 h + 8 eq.  Through LDS (2 KiB
    // of the wave's own: 16 rows of 128 bytes, chunk c of row r at c ^ r % 8), so that 8 lanes store 128 bytes of
    // a row (64 bytes of 16 rows at once, what the lanes hold: 1 to 5 us slower of 390)
    int el = lane;
    asm volatile("" : "+v"(el));  // (addresses made here, not kept over the K tiles)
    const int er = el & 15, eq = el >> 4, sr = el >> 3, sc = el & 7;
    unsigned char *const stage = lds + 2 * BUF + 3 * SBUF + wave * 2048;
    float bias[2][8];
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int64_t n = n0 + 32 * (k >> 3) + 8 * eq + (k & 7), nk = n < p.N ? n : p.N - 1;
      bias[k >> 3][k & 7] = !p.bias ? 0.f : p.bias_f32 ? reinterpret_cast<const float *>(p.bias)[nk] : Elem<T>::ld(reinterpret_cast<const T *>(p.bias)[nk]);
    }
    constexpr int EC = 16 / sizeof(T), PASSES = 64 / (8 * EC);  // columns of a chunk; 128-byte pieces of a row
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t mf = m0 + 16 * i + er;
      const float f = p.xf ? p.xf[(mf < p.M ? mf : p.M - 1) * p.xf_stride] : 1.f;
#pragma unroll
      for (int ps = 0; ps < PASSES; ++ps) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // the lane's two chunks of this piece
          const int h = PASSES == 1 ? c : ps, k0 = PASSES == 1 ? 0 : 4 * c;
          const int chunk = PASSES == 1 ? 4 * c + eq : 2 * eq + c;
          T e[EC];
#pragma unroll
          for (int k = 0; k < EC; ++k) e[k] = Elem<T>::st(acc[i][2 * h + ((k0 + k) >> 2)][(k0 + k) & 3] * f + bias[h][k0 + k]);
          __builtin_memcpy(stage + er * 128 + 16 * (chunk ^ (er & 7)), e, 16);
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          T e[EC];
          __builtin_memcpy(e, stage + (8 * u + sr) * 128 + 16 * (sc ^ sr), 16);
          const int64_t m = m0 + 16 * i + 8 * u + sr;
          if (m < p.M) pp_store<T>(reinterpret_cast<T *>(p.y) + m * p.N, e, n0 + ps * 8 * EC + EC * sc, p.N);
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
  wait_vm<0>();                                // the re-loads past the last tile
}

// ---- y = xq . W^T in between ---------------------------------------------------------------------
// Too many rows to stream W past registers, too few tiles of 256 x 256 to fill the card: BM x BN tiles
// (64 or 128), 4 waves of (BM / 2) x (BN / 2), K tiles as above in a ring of STAGES in LDS, filled by
// DMA STAGES - 1 ahead, one barrier a K tile (a stage is refilled after the barrier behind its last
// read).  Where there are still fewer tiles than CUs, K is cut into splits whose fp32 tiles a second
// small kernel adds in order.  Exponents: [rows][stride], stride a multiple of 4, zero past K.
// us: 48 x 28672 x 8192 E4M3 rows 43 (2.9 TB/s of W); 1531 x 6151 x 1696 E4M3 rows 37 to 46, E2M1 34.
struct MidArgs {
  const uint8_t *x, *w, *xsc, *wsc;
  const float *xf;
  const void *bias;
  void *y;
  float *part;  // [splits][M][N]
  int M, N, K, tiles_m, tiles_n, xs_stride, ws_stride, xf_stride, bias_f32, splits;
};

template <typename T, bool F8, int BM, int BN, int STAGES>
__global__ __launch_bounds__(256, 2) void mx_mid_kernel(MidArgs p) {
  constexpr int BK = pp_bk(F8), NB = BK / 32, WR = BK / 2;  // K tile, its blocks, bytes of a W row in it
  constexpr int AB = BM * 128, BB = BN * WR, SA = BM * NB, SB = BN * NB;
  constexpr int AU = AB / 4096, BU = BB / 4096;          // 16-byte DMAs a wave
  constexpr int SI = (SA + SB + 1023) / 1024;            // 4-byte DMAs a wave (the last ones may be idle copies)
  constexpr int SBYTES = SI * 1024;
  constexpr int STAGE = AB + BB + SBYTES, CNT = (STAGES - 2) * (AU + BU + SI);
  constexpr int NS = F8 ? 1 : 2, MI = BM / 32, NJ = BN / 32;
  __shared__ __attribute__((aligned(16))) unsigned char lds[STAGES * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, fr = lane & 15, fq = lane >> 4;

  // tiles of one column of W on one XCD, row tiles fastest: W's panel is read from HBM once
  const int per = p.tiles_m * p.tiles_n, split = blockIdx.x / per, rest = blockIdx.x - split * per;
  const int q8 = per / 8, r8 = per % 8, xcd = rest % 8;
  const int li = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + rest / 8;
  const int tn = li / p.tiles_m, tm = li - tn * p.tiles_m;
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
  const int xrow = F8 ? p.K : p.K / 2, wrow = p.K / 2;
  const int nt_all = (p.K + BK - 1) / BK;
  const int t0 = (int)((int64_t)nt_all * split / p.splits), t1 = (int)((int64_t)nt_all * (split + 1) / p.splits);
  const int rows_x = (int)(p.M - m0 < BM ? p.M - m0 : BM), rows_w = (int)(p.N - n0 < BN ? p.N - n0 : BN);

  // ---- DMA sources.  Operand rows of 128 bytes: LDS row u * 32 + wave * 8 + lane / 8, chunk slot lane % 8; of 64
  // bytes: u * 64 + wave * 16 + lane / 4, slot lane % 4.  Rows past the matrix re-read its last one.
  const int a_chunk = (lane & 7) ^ (((wave * 8 + (lane >> 3)) >> 1) & 7);
  const int b_chunk = F8 ? (lane & 3) ^ (-(lane >> 4) & 3) : a_chunk;
  unsigned a_off[AU], b_off[BU], s_off[SI];
#pragma unroll
  for (int u = 0; u < AU; ++u) {
    const int row = u * 32 + wave * 8 + (lane >> 3);
    a_off[u] = (unsigned)(row < rows_x ? row : rows_x - 1) * (unsigned)xrow + a_chunk * 16;
  }
#pragma unroll
  for (int u = 0; u < BU; ++u) {
    const int row = F8 ? u * 64 + wave * 16 + (lane >> 2) : u * 32 + wave * 8 + (lane >> 3);
    b_off[u] = (unsigned)(row < rows_w ? row : rows_w - 1) * (unsigned)wrow + b_chunk * 16;
  }
  // exponents: dword d of [xq rows][NB] then [W rows][NB]; a wave-sized piece is one operand's
  bool s_x[SI];
#pragma unroll
  for (int u = 0; u < SI; ++u) {
    int d = (u * 4 + wave) * 64 + lane;
    s_x[u] = p.xsc && (u * 4 + wave) * 256 < SA;
    if ((u * 4 + wave) * 256 >= SA) d -= SA / 4;
    const int rows = s_x[u] ? rows_x : rows_w;
    int row = d / (NB / 4);
    row = row < rows ? row : rows - 1;
    s_off[u] = (unsigned)row * (unsigned)(s_x[u] ? p.xs_stride : p.ws_stride) + 4 * (d % (NB / 4));
  }
  const int k_last = (nt_all - 1) * BK;
  const unsigned a_tail = k_last + a_chunk * (F8 ? 16 : 32) < p.K ? 0 : a_chunk * 16;
  const unsigned b_tail = k_last + b_chunk * 32 < p.K ? 0 : b_chunk * 16;
  const __amdgpu_buffer_rsrc_t xr = wave_rsrc(p.x + m0 * xrow, (uint32_t)rows_x * (uint32_t)xrow);
  const __amdgpu_buffer_rsrc_t wr = wave_rsrc(p.w + n0 * wrow, (uint32_t)rows_w * (uint32_t)wrow);
  const __amdgpu_buffer_rsrc_t xsr = wave_rsrc(p.xsc ? p.xsc + m0 * p.xs_stride : p.wsc + n0 * p.ws_stride,
                                               p.xsc ? (uint32_t)rows_x * p.xs_stride : (uint32_t)rows_w * p.ws_stride);
  const __amdgpu_buffer_rsrc_t wsr = wave_rsrc(p.wsc + n0 * p.ws_stride, (uint32_t)rows_w * p.ws_stride);
  auto load = [&](int t, int slot) {
    unsigned char *dst = lds + slot * STAGE;
    const int tt = t < t1 ? t : t1 - 1;  // past the end: harmless re-loads
    const uint32_t sa = __builtin_amdgcn_readfirstlane((uint32_t)tt * 128), sb = __builtin_amdgcn_readfirstlane((uint32_t)tt * WR);
    const uint32_t ss = __builtin_amdgcn_readfirstlane((uint32_t)tt * NB);
    const bool last = tt == nt_all - 1;
#pragma unroll
    for (int u = 0; u < AU; ++u) MX_DMA(xr, dst + u * 4096 + wave * 1024, 16, a_off[u] - (last ? a_tail : 0), sa);
#pragma unroll
    for (int u = 0; u < BU; ++u) MX_DMA(wr, dst + AB + u * 4096 + wave * 1024, 16, b_off[u] - (last ? b_tail : 0), sb);
#pragma unroll
    for (int u = 0; u < SI; ++u) {
      if (s_x[u])
        MX_DMA(xsr, dst + AB + BB + (u * 4 + wave) * 256, 4, s_off[u], ss);
      else
        MX_DMA(wsr, dst + AB + BB + (u * 4 + wave) * 256, 4, s_off[u], ss);
    }
  };

  const int sw8 = (fr >> 1) & 7, sw4 = -(fr >> 2) & 3;
  auto ld4 = [&](const unsigned char *q) -> i32x8 {
    const u32x4 d = *reinterpret_cast<const u32x4 *>(q);
    return i32x8{(int)d.x, (int)d.y, (int)d.z, (int)d.w, 0, 0, 0, 0};
  };
  f32x4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (t0 < t1) {
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load(t0 + s, s);
    int slot = 0;
    for (int t = t0; t < t1; ++t) {
      wait_vm<CNT>();                 // this wave's part of stage t has landed ...
      __builtin_amdgcn_s_barrier();   // ... every wave's; and stage t - 1 has been read by all
      load(t + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
      const unsigned char *st = lds + slot * STAGE, *sx = st + AB + BB, *sw = sx + SA;
      const int unit = F8 && !p.xsc ? ((t == nt_all - 1 && k_last + 32 * fq >= p.K) ? 0 : 127) : 0;
      i32x8 bf[NJ][NS];
      int sb[NJ][NS];
      // exponent byte of block 4 s + fq in a lane's lowest byte
      auto read_s = [&](const unsigned char *row, int (&e)[NS]) {
        if constexpr (F8) {
          e[0] = row[fq];
        } else {
          e[0] = row[fq], e[1] = row[4 + fq];
        }
      };
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = wn * (BN / 2) + 16 * j + fr;
#pragma unroll
        for (int s = 0; s < NS; ++s) bf[j][s] = ld4(st + AB + row * WR + (F8 ? (fq ^ sw4) << 4 : ((4 * s + fq) ^ sw8) << 4));
        read_s(sw + row * NB, sb[j]);
      }
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int row = wm * (BM / 2) + 16 * i + fr;
        i32x8 af[NS];
        int sa[NS];
        if constexpr (F8) {
          const u32x4 d = *reinterpret_cast<const u32x4 *>(st + row * 128 + ((fq ^ sw8) << 4));
          const u32x4 e = *reinterpret_cast<const u32x4 *>(st + row * 128 + (((4 + fq) ^ sw8) << 4));
          af[0] = i32x8{(int)d.x, (int)d.y, (int)d.z, (int)d.w, (int)e.x, (int)e.y, (int)e.z, (int)e.w};
          if (p.xsc)
            read_s(sx + row * NB, sa);
          else
            sa[0] = unit;
        } else {
#pragma unroll
          for (int s = 0; s < NS; ++s) af[s] = ld4(st + row * 128 + (((4 * s + fq) ^ sw8) << 4));
          read_s(sx + row * NB, sa);
        }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = pp_mma<F8>(bf[j][s], af[s], acc[i][j], 0, sb[j][s], sa[s]);
      }
      slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
    wait_vm<0>();  // the re-loads past the end land before the workgroup's LDS is given away
  }

#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = m0 + wm * (BM / 2) + 16 * i + fr;
    if (m >= p.M) continue;
    const float f = p.xf ? p.xf[m * p.xf_stride] : 1.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int64_t n = n0 + wn * (BN / 2) + 16 * j + 4 * fq;
      if (p.splits > 1)
        out4<float>(p.part + ((int64_t)split * p.M + m) * p.N, acc[i][j], 1.f, nullptr, 0, n, p.N);
      else
        out4<T>(reinterpret_cast<T *>(p.y) + m * p.N, acc[i][j], f, p.bias, p.bias_f32, n, p.N);
    }
  }
}

template <typename T> __global__ __launch_bounds__(256) void mx_join_kernel(MidArgs p) {
  const int64_t groups = (p.N + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / groups, n = 4 * (i - m * groups);
  if (m >= p.M) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  const int64_t step = (int64_t)p.M * p.N;
  const float *q = p.part + m * p.N + n;
  if (p.N % 4 == 0) {
    for (int s = 0; s < p.splits; ++s) v += *reinterpret_cast<const f32x4 *>(q + s * step);
  } else {
    for (int s = 0; s < p.splits; ++s)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < p.N) v[k] += q[s * step + k];
  }
  out4<T>(reinterpret_cast<T *>(p.y) + m * p.N, v, p.xf ? p.xf[m * p.xf_stride] : 1.f, p.bias, p.bias_f32, n, p.N);
}

// exponents [rows][nb] -> [rows][stride], zero past nb
__global__ __launch_bounds__(256) void mx_pad_scales_kernel(const uint8_t *__restrict__ s, int64_t rows, int nb, int stride,
                                                            uint8_t *__restrict__ o) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = stride / 4, row = i / per;
  const int b = 4 * (int)(i - row * per);
  if (row >= rows) return;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (b + j < nb) w |= (uint32_t)s[row * nb + b + j] << (8 * j);
  *reinterpret_cast<uint32_t *>(o + row * stride + b) = w;
}

// exponents [rows][nb] -> [K tile][rows padded to 256][NB], 0 past the matrix; both operands' in one launch
struct TileScales {
  const uint8_t *s[2];
  uint8_t *o[2];
  int rows[2], pad[2], blocks0, nb, nt;  // blocks0: workgroups of the first
};
template <int NB> __global__ __launch_bounds__(256) void mx_tile_scales_kernel(TileScales a) {
  const int op = (int)blockIdx.x >= a.blocks0 ? 1 : 0;
  const int64_t i = (int64_t)(blockIdx.x - (op ? a.blocks0 : 0)) * 256 + threadIdx.x;
  const int64_t row = i / a.nt;
  const int t = (int)(i - row * a.nt), nb = a.nb, pad = op ? a.pad[1] : a.pad[0];
  if (row >= pad) return;
  const uint8_t *s = (op ? a.s[1] : a.s[0]) + row * nb + t * NB;
  const bool in = row < (op ? a.rows[1] : a.rows[0]);
  uint32_t w[NB / 4];
#pragma unroll
  for (int k = 0; k < NB / 4; ++k) {
    w[k] = 0;
    const int left = nb - t * NB - 4 * k;
    if (in && nb % 4 == 0 && left > 0) {  // 4-byte aligned rows: a dword is inside or outside
      w[k] = *reinterpret_cast<const uint32_t *>(s + 4 * k);
    } else if (in) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) w[k] |= (uint32_t)s[4 * k + j] << (8 * j);
    }
  }
  uint32_t *d = reinterpret_cast<uint32_t *>((op ? a.o[1] : a.o[0]) + ((int64_t)t * pad + row) * NB);
  if constexpr (NB == 8) {  // E2M1: a lane's two blocks g and 4 + g of a K tile next to each other
    d[0] = __builtin_amdgcn_perm(w[1], w[0], 0x05010400);
    d[1] = __builtin_amdgcn_perm(w[1], w[0], 0x07030602);
  } else {
    d[0] = w[0];
  }
}

// Rows up to which the weight-streaming kernel is taken: one 16-row operand, since each further one reads W again.
// us for rows handed over quantised, streaming / tiles:
//   16 rows  4096 x 4096 E4M3 5.7 / 10.3, E2M1 4.9 / 8.1; 28672 x 8192 E4M3 34 / 39; 14336 x 4096 E2M1 9.3 / 9.4
//   17 rows  7.3 / 10.4, 6.1 / 8.2; 53 / 40; 13.6 / 9.8        48 rows  11.7 / 12.5, 9.1 / 9.1; 82 / 43; 19.8 / 10.1
// (a small W, which the caches hold, would gain from more rows)
constexpr int kSkinnyRows = 16;
// MXFP4 rows of at most 8 tokens against at most 8 MiB of W: quantised by every workgroup for itself, in
// registers (kOpFused); else once, by a launch of its own.  us, fused / in two launches:
// 1024 x 4096: 1 row 5.4 / 7.4; 4096 x 4096: 1 row 6.1 / 7.4, 8 rows 6.9 / 7.2, 16 rows 8.0 / 7.7; 8192 x 4096: 1 row
// 8.5 / 7.9, 8 rows 10.4 / 8.7
constexpr int kFusedRows = 8;
constexpr int64_t kFusedWeights = 1 << 24;

// which kernel, and its tile
struct LinearPlan {
  enum { kSkinny, kMid, kPp } form;
  int bm, bn, splits;
};
LinearPlan linear_plan(int64_t M, int64_t N, int64_t K, int kind) {
  LinearPlan p{LinearPlan::kSkinny, 0, 0, 1};
  // 32-bit offsets inside a panel of 256 rows and inside the tiled exponents
  const int64_t pad = (M > N ? M : N) + kPpTile;
  if (M <= kSkinnyRows || pad * (K / 32 + 8) >= (1ll << 31)) return p;
  const int64_t cus = host_num_cus();
  auto tiles = [&](int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  // 256 x 256 tiles for three quarters of the CUs, and two K tiles at least.  Their order goes by units of 8 x 4 tiles,
  // and a unit that the matrix fills by half costs as much as a whole one: more than 9/16 of the slots have to hold a
  // tile.  us, E2M1 rows / E4M3 rows, the tiles below in brackets: x 14336 x 4096, 1024 rows (1/2 of the slots) 68 (60) /
  // 104 (89), 1280 (5/8) 69 (83) / 105 (101), 1536 69 (85) / 105 (121), 2304 (9/16) 130 (120) / 208 (184), 2560 (5/8)
  // 129 (140) / 209 (205); 300 x 28672 x 8192 (1/4) 227 (94) / 384 (129); 30000 x 512 x 4096 68 (63) / 107 (98).
  // x 4096 x 4096: 2048 rows (128 tiles) 42 (31) / 60 (46), 2560 (160) 41 (51) / 56 (62), 3328 (208) 40 (55) / 56 (82).
  const int64_t slots = (M + 2047) / 2048 * 8 * ((N + 1023) / 1024 * 4);
  if (tiles(256, 256) * 4 >= cus * 3 && tiles(256, 256) * 16 > slots * 9 && K > pp_bk(kind != MTQ_MXFP4)) {
    p.form = LinearPlan::kPp;
    return p;
  }
  p.form = LinearPlan::kMid;
  // The smaller tiles where the larger ones leave CUs idle.  us, 128 / 64 rows: 1024 x 8192 x 4096 (512 tiles of 128 x 128)
  // E2M1 rows 30 / 42, E4M3 46 / 63; 512 x 8192 x 4096 (256) 20.1 / 20.9, 32.5 / 31.4; 512 x 4096 x 4096 (128) 25 / 13, 26 / 18;
  // but 128 x 28672 x 8192 (224) 46 / 55, 61 / 68.  128 / 64 columns of 64 rows: 64 x 28672 x 8192 (224 tiles of 128) 36 / 44,
  // 44 / 52; 512 x 4096 x 4096 (256) 13.0 / 13.7, 18.0 / 19.4; 64 x 14336 x 4096 (112) 17.9 / 11.0, 24 / 14.
  p.bm = M > 64 && tiles(128, 128) >= cus ? 128 : 64;
  p.bn = p.bm == 128 || tiles(64, 128) * 4 >= cus * 3 ? 128 : 64;
  // K is split where fewer than three quarters of the CUs have a tile.  us, split / whole: 64 x 4096 x 14336 E4M3
  // 19.5 / 39, 128 x 4096 x 14336 E2M1 21.8 / 27.7, 32 x 4096 x 4096 E4M3 11.1 / 11.6 (but 64 rows 13.8 / 11.6, 128 rows
  // 14.7 / 11.7); with more tiles than that: 256 x 4096 x 4096 E4M3 18.2 / 12.0, 64 x 14336 x 4096 20.8 / 14.2, 48 x
  // 28672 x 8192 48.8 / 42.9.
  const int bk = pp_bk(kind != MTQ_MXFP4);
  const int64_t nt = (K + bk - 1) / bk, have = tiles(p.bm, p.bn);
  int64_t splits = have * 4 >= 3 * cus ? 1 : (2 * cus + have - 1) / have;
  if (splits > nt / 4) splits = nt / 4;  // a split of fewer than 4 K tiles is mostly its start
  p.splits = (int)(splits < 1 ? 1 : splits > 16 ? 16 : splits);
  return p;
}
struct LinearWs {
  size_t q, scale, xt, wt, part, bytes;  // offsets: codes and scales of x, both operands' exponents laid out anew, splits
};
LinearWs linear_ws(int64_t M, int64_t N, int64_t K, int kind, bool quantise) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  LinearWs w;
  w.q = 0;
  w.scale = quantise ? up((size_t)M * (kind == MTQ_MXFP4 ? K / 2 : K)) : 0;
  w.xt = w.scale + (quantise ? up(is_mx(kind) ? (size_t)M * (K / 32) : kind == MTQ_FP8_TOKEN ? 4 * (size_t)M : 4) : 0);
  w.wt = w.part = w.bytes = w.xt;
  const LinearPlan p = linear_plan(M, N, K, kind);
  const int bk = pp_bk(kind != MTQ_MXFP4);
  const size_t nt = (size_t)((K + bk - 1) / bk), per = nt * (bk / 32);
  if (p.form == LinearPlan::kPp) {
    w.wt = w.xt + (is_mx(kind) ? up(M) * per : 0);
    w.part = w.bytes = w.wt + up(N) * per;
  } else if (p.form == LinearPlan::kMid) {
    if (K % bk) {  // rows of exponents padded to whole K tiles
      w.wt = w.xt + (is_mx(kind) ? up((size_t)M * per) : 0);
      w.part = w.wt + up((size_t)N * per);
    }
    w.bytes = w.part + (p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0);
  }
  return w;
}
template <typename T, bool F8> int launch_mid(MidArgs a, const LinearPlan &p, hipStream_t stream) {
  a.tiles_m = (a.M + p.bm - 1) / p.bm, a.tiles_n = (a.N + p.bn - 1) / p.bn, a.splits = p.splits;
  const unsigned g = (unsigned)((int64_t)a.tiles_m * a.tiles_n * a.splits);
  if (p.bm == 128)
    mx_mid_kernel<T, F8, 128, 128, 2><<<g, 256, 0, stream>>>(a);
  else if (p.bn == 128)
    mx_mid_kernel<T, F8, 64, 128, F8 ? 4 : 3><<<g, 256, 0, stream>>>(a);
  else
    mx_mid_kernel<T, F8, 64, 64, 3><<<g, 256, 0, stream>>>(a);
  int st = host_check_launch();
  if (st != MTQ_OK || a.splits == 1) return st;
  mx_join_kernel<T><<<(unsigned)(((int64_t)a.M * ((a.N + 3) / 4) + 255) / 256), 256, 0, stream>>>(a);
  return host_check_launch();
}
// xs may be null: W's only
template <bool F8>
int launch_tile_scales(const uint8_t *xs, int M, uint8_t *xo, const uint8_t *ws, int N, uint8_t *wo, int K, hipStream_t stream) {
  constexpr int BK = pp_bk(F8);
  TileScales a{{xs, ws}, {xo, wo}, {M, N}, {(M + 255) / 256 * 256, (N + 255) / 256 * 256}, 0, K / 32, (K + BK - 1) / BK};
  auto blocks = [&](int pad) { return ((int64_t)pad * a.nt + 255) / 256; };
  a.blocks0 = xs ? (int)blocks(a.pad[0]) : 0;
  mx_tile_scales_kernel<BK / 32><<<(unsigned)(a.blocks0 + blocks(a.pad[1])), 256, 0, stream>>>(a);
  return host_check_launch();
}
template <typename T, bool F8> int launch_pp(PpArgs a, hipStream_t stream) {
  a.tiles_m = (a.M + kPpTile - 1) / kPpTile, a.tiles_n = (a.N + kPpTile - 1) / kPpTile;
  // one workgroup a CU (its LDS), each going through several tiles of y
  const int64_t order = ((int64_t)((a.tiles_m + 7) / 8) * ((a.tiles_n + 3) / 4) + 7) / 8 * 8 * 32;
  const int64_t cus = (host_num_cus() + 7) / 8 * 8;
  mx_pp_kernel<T, F8><<<(unsigned)(order < cus ? order : cus), kPpThreads, 0, stream>>>(a);
  return host_check_launch();
}

bool known_kind(int kind) { return kind >= MTQ_MXFP4 && kind <= MTQ_FP8_TOKEN; }

}  // namespace

extern "C" {

int mtq_mx_quantize(const void *x, int64_t row_stride, int64_t rows, int64_t cols, int dtype, int kind, const float *amax,
                    uint8_t *q, void *scale, hipStream_t stream) {
  if (!known_kind(kind)) return MTQ_ERR_FORMAT;
  if (dtype != MTQ_BF16 && dtype != MTQ_F16 && dtype != MTQ_F32) return MTQ_ERR_DTYPE;
  if (rows < 0 || cols < 1 || (is_mx(kind) && cols % 32) || (rows > 1 && row_stride < cols)) return MTQ_ERR_INVALID_ARG;
  if (rows == 0) return MTQ_OK;
  if (!x || !q || !scale || (kind == MTQ_FP8_TENSOR && !amax)) return MTQ_ERR_INVALID_ARG;
  if (rows > (int64_t)INT32_MAX || (cols + 7) / 8 > (int64_t)INT32_MAX) return MTQ_ERR_INVALID_ARG;
  if ((uintptr_t)q % 8) return MTQ_ERR_INVALID_ARG;
  const int es = dtype == MTQ_F32 ? 4 : 2;
  const bool vec = al16(x) && cols % 8 == 0 && (rows == 1 || (row_stride * es) % 16 == 0);
  auto go = [&](auto t) {
    using T = decltype(t);
    const T *p = reinterpret_cast<const T *>(x);
    return vec ? launch_quantize<T, true>(p, row_stride, rows, cols, kind, amax, q, scale, stream)
               : launch_quantize<T, false>(p, row_stride, rows, cols, kind, amax, q, scale, stream);
  };
  return dtype == MTQ_BF16 ? go(__bf16{}) : dtype == MTQ_F16 ? go(_Float16{}) : go(float{});
}

int mtq_rms_norm_quantize(const void *x, int64_t x_stride, const void *residual, int64_t r_stride, const void *weight,
                          int weight_dtype, double eps, void *h, uint8_t *q, void *scale, const float *amax, int64_t rows,
                          int64_t cols, int dtype, int kind, hipStream_t stream) {
  if (!known_kind(kind)) return MTQ_ERR_FORMAT;
  if (dtype != MTQ_BF16 && dtype != MTQ_F16 && dtype != MTQ_F32) return MTQ_ERR_DTYPE;
  if (weight_dtype != dtype && weight_dtype != MTQ_F32) return MTQ_ERR_DTYPE;
  if (rows < 0 || cols < 1 || cols > 65536 || (is_mx(kind) && cols % 32)) return MTQ_ERR_INVALID_ARG;
  if (rows > (int64_t)INT32_MAX || (rows > 1 && (x_stride < cols || (residual && r_stride < cols)))) return MTQ_ERR_INVALID_ARG;
  if (!(eps >= 0.0 && eps < 3.4e38)) return MTQ_ERR_INVALID_ARG;
  if (rows == 0) return MTQ_OK;
  if (!x || !weight || !q || !scale || (residual && !h) || (kind == MTQ_FP8_TENSOR && !amax)) return MTQ_ERR_INVALID_ARG;
  if ((uintptr_t)q % 8) return MTQ_ERR_INVALID_ARG;
  const int es = dtype == MTQ_F32 ? 4 : 2;
  const bool vec = cols % 8 == 0 && al16(x) && al16(weight) && (rows == 1 || (x_stride * es) % 16 == 0) &&
                   (!residual || (al16(residual) && al16(h) && (rows == 1 || (r_stride * es) % 16 == 0)));
  const NormArgs a{x, residual, weight, h, q, scale, amax, x_stride, r_stride, cols, eps, weight_dtype};
  if (dtype == MTQ_BF16) return launch_norm_k<__bf16>(a, kind, vec, rows, stream);
  if (dtype == MTQ_F16) return launch_norm_k<_Float16>(a, kind, vec, rows, stream);
  return launch_norm_k<float>(a, kind, vec, rows, stream);
}

size_t mtq_mx_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int kind, int x_dtype) {
  if (M < 1 || N < 1 || K < 32 || !known_kind(kind)) return 0;
  return linear_ws(M, N, K, kind, x_dtype >= 0).bytes;
}

int mtq_mx_linear(const void *x, int64_t x_stride, int x_dtype, const void *x_scale, int kind, const float *amax,
                  const uint8_t *w, const uint8_t *w_scale, const void *bias, int bias_dtype, void *y, int y_dtype, int64_t M,
                  int64_t N, int64_t K, void *ws, size_t ws_bytes, hipStream_t stream) {
  if (!known_kind(kind)) return MTQ_ERR_FORMAT;
  if (y_dtype != MTQ_BF16 && y_dtype != MTQ_F16 && y_dtype != MTQ_F32) return MTQ_ERR_DTYPE;
  if (x_dtype >= 0 && x_dtype != MTQ_BF16 && x_dtype != MTQ_F16 && x_dtype != MTQ_F32) return MTQ_ERR_DTYPE;
  if (bias && bias_dtype != y_dtype && bias_dtype != MTQ_F32) return MTQ_ERR_DTYPE;
  if (M < 0 || N < 1 || K < 32 || K % 32 || M > (1 << 24) || N > (1 << 24) || K > (1 << 22)) return MTQ_ERR_INVALID_ARG;
  if (M == 0) return MTQ_OK;
  if (!x || !w || !w_scale || !y || !al16(w) || (uintptr_t)w_scale % 4) return MTQ_ERR_INVALID_ARG;
  if (x_dtype < 0 ? !x_scale || !al16(x) || (uintptr_t)x_scale % 4 : (M > 1 && x_stride < K) || (kind == MTQ_FP8_TENSOR && !amax)) return MTQ_ERR_INVALID_ARG;
  SkinnyArgs a{};
  a.w = w, a.wsc = w_scale, a.bias = bias, a.y = y, a.M = (int)M, a.N = (int)N, a.K = (int)K;
  a.bias_f32 = bias && bias_dtype == MTQ_F32;
  const bool vec = x_dtype >= 0 && x_dtype != MTQ_F32 && al16(x) && (M == 1 || x_stride % 8 == 0);
  const bool fused = vec && kind == MTQ_MXFP4 && M <= kFusedRows && N * K <= kFusedWeights && x_dtype == y_dtype;
  if (fused) {
    a.x = x, a.xs = x_stride;
    return y_dtype == MTQ_BF16 ? launch_skinny<__bf16, kOpFused>(a, stream) : launch_skinny<_Float16, kOpFused>(a, stream);
  }
  const LinearWs o = linear_ws(M, N, K, kind, x_dtype >= 0);
  if (o.bytes && (!ws || ws_bytes < o.bytes || !al16(ws))) return MTQ_ERR_INVALID_ARG;
  if (x_dtype >= 0) {
    uint8_t *q = (uint8_t *)ws + o.q;
    void *sc = (uint8_t *)ws + o.scale;
    const int st = mtq_mx_quantize(x, x_stride, M, K, x_dtype, kind, amax, q, sc, stream);
    if (st != MTQ_OK) return st;
    x = q, x_scale = sc;
  }
  a.x = x;
  if (is_mx(kind)) {
    a.xsc = (const uint8_t *)x_scale;
  } else {
    a.xf = (const float *)x_scale;
    a.xf_stride = kind == MTQ_FP8_TOKEN;
  }
  const LinearPlan plan = linear_plan(M, N, K, kind);
  if (plan.form != LinearPlan::kSkinny) {
    const bool f8 = kind != MTQ_MXFP4;
    const int bk = pp_bk(f8), nb = (int)(K / 32), per = (int)((K + bk - 1) / bk * (bk / 32));
    const uint8_t *xt = a.xsc, *wt = w_scale;
    int st = MTQ_OK;
    uint8_t *const xo = (uint8_t *)ws + o.xt, *const wo = (uint8_t *)ws + o.wt;
    if (plan.form == LinearPlan::kPp) {
      st = f8 ? launch_tile_scales<true>(xt, a.M, xo, wt, a.N, wo, a.K, stream) : launch_tile_scales<false>(xt, a.M, xo, wt, a.N, wo, a.K, stream);
      xt = xt ? xo : nullptr, wt = wo;
    } else if (K % bk) {  // else as they are (4-byte aligned: checked)
      auto pad = [&](const uint8_t *&s, int64_t rows, uint8_t *d) {
        if (!s || st != MTQ_OK) return;
        mx_pad_scales_kernel<<<(unsigned)((rows * (per / 4) + 255) / 256), 256, 0, stream>>>(s, rows, nb, per, d);
        st = host_check_launch();
        s = d;
      };
      pad(xt, M, xo);
      pad(wt, N, wo);
    }
    if (st != MTQ_OK) return st;
    auto go = [&](auto t) {
      using T = decltype(t);
      if (plan.form == LinearPlan::kPp) {
        const PpArgs p{(const uint8_t *)x, w, xt, wt, a.xf, bias, y, a.M, a.N, a.K, 0, 0, a.xf_stride, a.bias_f32};
        return f8 ? launch_pp<T, true>(p, stream) : launch_pp<T, false>(p, stream);
      }
      const MidArgs p{(const uint8_t *)x, w, xt, wt, a.xf, bias, y, (float *)((uint8_t *)ws + o.part), a.M, a.N, a.K, 0, 0, per, per,
                      a.xf_stride, a.bias_f32, 1};
      return f8 ? launch_mid<T, true>(p, plan, stream) : launch_mid<T, false>(p, plan, stream);
    };
    return y_dtype == MTQ_BF16 ? go(__bf16{}) : y_dtype == MTQ_F16 ? go(_Float16{}) : go(float{});
  }
  auto go = [&](auto t) {
    using T = decltype(t);
    return kind == MTQ_MXFP4 ? launch_skinny<T, kOpFp4>(a, stream) : launch_skinny<T, kOpFp8>(a, stream);
  };
  return y_dtype == MTQ_BF16 ? go(__bf16{}) : y_dtype == MTQ_F16 ? go(_Float16{}) : go(float{});
}

}  // extern "C"
