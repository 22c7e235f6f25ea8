// row_quant.cu -- rows to 8 bits: RMS norm with the residual's addition, and the plain
// row-wise quantiser, with int8 or e4m3 codes and one fp32 scale per row.
//
//   s = x + r                              (fp32; sum_out = s rounded to x's type)
//   y_k = s_k * rstd * w_k,  rstd = 1 / sqrt(mean(s^2) + eps)
//   scale = max(max_k |y_k| / Q, 1e-12),   Q = 127 (int8) or 448 (e4m3)
//   q_k = round(y_k / scale)               (to nearest, ties to even)
//
// rstd is one number per row, so max|y| = rstd * max|s w|: the sum of squares and
// the maximum are reduced together, in one pass over the row, and the codes are
// s_k w_k * (rstd / scale) from the registers that hold the row. The norm works on
// the fp32 sum, not on the rounded one: sum_out is rounded once and nothing
// computed here is rounded twice.
//
// A row with a NaN, or an infinity, has the scale NaN (max.NaN keeps it), so what
// its codes stand for is NaN; int8 codes of it are 0.
#include "sm100.cuh"
#include "srdit_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace srdit {
namespace rq {

struct Args {
  const void* x;
  const void* res;
  const void* w;
  void* sum;
  uint8_t* q;
  float* scale;
  long long ldx, ldr, lds, ldq;
  int M, K;
  int warps;  // warps per row
  float eps, inv_k;
};

template <typename T>
SRDIT_DEV float to_f(T v);
template <>
SRDIT_DEV float to_f(float v) { return v; }
template <>
SRDIT_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
SRDIT_DEV float to_f(__half v) { return __half2float(v); }
template <typename T>
SRDIT_DEV T from_f(float v);
template <>
SRDIT_DEV float from_f(float v) { return v; }
template <>
SRDIT_DEV __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
SRDIT_DEV __half from_f(float v) { return __float2half_rn(v); }

// V values of type T as one aligned access of at most 16 bytes each
template <typename T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Vec {
  T v[V];
};

// plain loads: sum may be x or the residual itself, so these are not read-only
template <typename T, int V>
SRDIT_DEV void load(const T* p, float (&o)[V]) {
  const Vec<T, V> t = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = to_f<T>(t.v[i]);
}
template <typename T, int V>
SRDIT_DEV void store(T* p, const float (&o)[V]) {
  Vec<T, V> t;
#pragma unroll
  for (int i = 0; i < V; ++i) t.v[i] = from_f<T>(o[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = t;
}

SRDIT_DEV float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
SRDIT_DEV uint32_t code_i8(float v) {
  int d;
  asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(d) : "f"(v));
  return static_cast<uint32_t>(d) & 0xffu;
}
SRDIT_DEV uint32_t code_e4m3x2(float lo, float hi) {
  uint16_t h;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(hi), "f"(lo));
  return h;
}

// V codes as one aligned store
template <bool kInt8, int V>
SRDIT_DEV void store_codes(uint8_t* p, const float (&y)[V]) {
  if constexpr (V == 1) {
    *p = static_cast<uint8_t>(kInt8 ? code_i8(y[0]) : code_e4m3x2(y[0], 0.f) & 0xffu);
  } else {
    uint32_t h[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      h[i] = kInt8 ? (code_i8(y[2 * i]) | code_i8(y[2 * i + 1]) << 8)
                   : code_e4m3x2(y[2 * i], y[2 * i + 1]);
    if constexpr (V == 2) {
      *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(h[0]);
    } else {
      static_assert(V == 8, "1, 2 or 8 codes");
      *reinterpret_cast<uint2*>(p) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
  }
}

// One row per `warps` warps of the block; a thread holds 8 * NV values of its row as
// vectors of V (V = 8: 16-byte loads of 16-bit values; 2 and 1 for rows whose width,
// pitch or base is not so aligned), vector i of thread t at (i * threads + t) * V.
template <typename T, bool kInt8, bool kNorm, bool kRes, int V, int NV>
__global__ void __launch_bounds__(1024) rows_kernel(const Args a) {
  pdl_begin();
  constexpr int N = 8 * NV / V;
  __shared__ float2 part[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tpr = a.warps * 32;
  const int sub = warp / a.warps;  // row of the block
  const int t = threadIdx.x - sub * tpr;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + sub;
  const bool on = row < a.M;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = kRes ? static_cast<const T*>(a.res) + row * a.ldr : nullptr;
  const T* w = static_cast<const T*>(a.w);
  float s[N][V];
  float ss = 0.f, mx = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * tpr + t) * V;
    if (on && c < a.K) {
      load<T, V>(x + c, s[i]);
      if constexpr (kRes) {
        float rr[V];
        load<T, V>(r + c, rr);
#pragma unroll
        for (int e = 0; e < V; ++e) s[i][e] += rr[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) s[i][e] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * tpr + t) * V;
    if (on && c < a.K) {
      if constexpr (kRes) store<T, V>(static_cast<T*>(a.sum) + row * a.lds + c, s[i]);
      float ww[V];
      if constexpr (kNorm) load<T, V>(w + c, ww);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (kNorm) {
          ss = fmaf(s[i][e], s[i][e], ss);
          s[i][e] *= ww[e];
        }
        mx = max_nan(mx, fabsf(s[i][e]));
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if constexpr (kNorm) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (a.warps > 1) {
    if (lane == 0) part[warp] = make_float2(ss, mx);
    __syncthreads();
    // every warp reduces its row's partials itself, in the same order
    const float2 p = lane < a.warps ? part[sub * a.warps + lane] : make_float2(0.f, 0.f);
    ss = p.x;
    mx = p.y;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      if constexpr (kNorm) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
  }
  if (!on) return;
  const float rstd = kNorm ? 1.0f / sqrtf(fmaf(ss, a.inv_k, a.eps)) : 1.0f;
  const float scale = max_nan(mx * rstd / (kInt8 ? 127.f : 448.f), 1e-12f);
  const float inv = rstd / scale;
  if (t == 0) a.scale[row] = scale;
  uint8_t* q = a.q + row * a.ldq;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * tpr + t) * V;
    if (c < a.K) {
      float y[V];
#pragma unroll
      for (int e = 0; e < V; ++e) y[e] = s[i][e] * inv;
      store_codes<kInt8, V>(q + c, y);
    }
  }
}

template <typename T, bool kInt8, bool kNorm, bool kRes, int V>
static int launch_v(Args& a, cudaStream_t stream) {
  // 8 values per thread up to 8192 columns, 32 above (a row is one block's). With 16, 24
  // and 32 a row of 4096 takes 2.9, 3.2 and 3.6 us in place of 2.6; 6912 rows of 3072 take
  // 31.6, 30.5 and 32.2 in place of 30.9.
  const int nv = a.K <= 8192 ? 1 : 4;
  a.warps = (a.K + nv * 256 - 1) / (nv * 256);
  const int rows = a.warps >= 4 ? 1 : 4 / a.warps;
  const int threads = rows * a.warps * 32;
  const unsigned grid = static_cast<unsigned>((a.M + rows - 1) / rows);
  if (nv == 1)
    SRDIT_LAUNCH((rows_kernel<T, kInt8, kNorm, kRes, V, 1>), grid, threads, 0, stream, a);
  else
    SRDIT_LAUNCH((rows_kernel<T, kInt8, kNorm, kRes, V, 4>), grid, threads, 0, stream, a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, bool kInt8, bool kNorm, bool kRes>
static int launch_r(Args& a, cudaStream_t stream) {
  // the widest vector that every row of every operand is aligned for
  const uintptr_t e = sizeof(T);
  uintptr_t in = reinterpret_cast<uintptr_t>(a.x) | a.ldx * e | a.K * e;
  if (kNorm) in |= reinterpret_cast<uintptr_t>(a.w);
  if (kRes)
    in |= reinterpret_cast<uintptr_t>(a.res) | a.ldr * e | reinterpret_cast<uintptr_t>(a.sum) |
          a.lds * e;
  const uintptr_t out = reinterpret_cast<uintptr_t>(a.q) | a.ldq | a.K;
  if (in % (e == 4 ? 32 : 16) == 0 && out % 8 == 0)
    return launch_v<T, kInt8, kNorm, kRes, 8>(a, stream);
  if (in % (2 * e) == 0 && out % 2 == 0) return launch_v<T, kInt8, kNorm, kRes, 2>(a, stream);
  return launch_v<T, kInt8, kNorm, kRes, 1>(a, stream);
}

template <typename T, bool kInt8, bool kNorm>
static int launch_n(Args& a, cudaStream_t stream) {
  if constexpr (kNorm) {
    if (a.res) return launch_r<T, kInt8, true, true>(a, stream);
  }
  return launch_r<T, kInt8, kNorm, false>(a, stream);
}

template <bool kNorm>
static int run(Args& a, int dtype, int q_type, cudaStream_t stream) {
  const bool i8 = q_type == SRDIT_Q_INT8;
  if (!i8 && q_type != SRDIT_Q_E4M3) return SRDIT_EINVAL;
  switch (dtype) {
    case SRDIT_BF16:
      return i8 ? launch_n<__nv_bfloat16, true, kNorm>(a, stream)
                : launch_n<__nv_bfloat16, false, kNorm>(a, stream);
    case SRDIT_FP16:
      return i8 ? launch_n<__half, true, kNorm>(a, stream)
                : launch_n<__half, false, kNorm>(a, stream);
    case SRDIT_FP32:
      return i8 ? launch_n<float, true, kNorm>(a, stream)
                : launch_n<float, false, kNorm>(a, stream);
    default: return SRDIT_EINVAL;
  }
}

}  // namespace rq
}  // namespace srdit

using namespace srdit;

static bool elem_aligned(const void* p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == SRDIT_FP32 ? 4 : 2) == 0;
}

static int check_rows(const void* x, long long ldx, int M, int K, int dtype, const void* q,
                      long long ldq, const float* scale) {
  if (M < 0 || K <= 0 || !x || !q || !scale || dtype < SRDIT_BF16 || dtype > SRDIT_FP32)
    return SRDIT_EINVAL;
  if (ldx < K || ldq < K) return SRDIT_EINVAL;
  if (!elem_aligned(x, dtype) || (reinterpret_cast<uintptr_t>(scale) & 3u)) return SRDIT_EALIGN;
  if (K > 32768) return SRDIT_EUNSUPPORTED;
  return 0;
}

extern "C" int srdit_add_rms_quant(const void* x, long long ldx, int M, int K, int dtype,
                                   const void* residual, long long ldr, const void* weight,
                                   float eps, void* sum, long long ld_sum, void* q, long long ldq,
                                   int q_type, float* scale, cudaStream_t stream) {
  if (M == 0) return 0;
  const int rc = check_rows(x, ldx, M, K, dtype, q, ldq, scale);
  if (rc) return rc;
  if (!weight || !(eps >= 0.f) || (residual == nullptr) != (sum == nullptr)) return SRDIT_EINVAL;
  if (residual && (ldr < K || ld_sum < K)) return SRDIT_EINVAL;
  if (!elem_aligned(weight, dtype) || !elem_aligned(residual, dtype) || !elem_aligned(sum, dtype))
    return SRDIT_EALIGN;
  rq::Args a = {};
  a.x = x;
  a.res = residual;
  a.w = weight;
  a.sum = sum;
  a.q = static_cast<uint8_t*>(q);
  a.scale = scale;
  a.ldx = ldx;
  a.ldr = ldr;
  a.lds = ld_sum;
  a.ldq = ldq;
  a.M = M;
  a.K = K;
  a.eps = eps;
  a.inv_k = 1.0f / static_cast<float>(K);
  return rq::run<true>(a, dtype, q_type, stream);
}

extern "C" int srdit_quant_rows(const void* x, long long ldx, int M, int K, int dtype, void* q,
                                long long ldq, int q_type, float* scale, cudaStream_t stream) {
  if (M == 0) return 0;
  const int rc = check_rows(x, ldx, M, K, dtype, q, ldq, scale);
  if (rc) return rc;
  rq::Args a = {};
  a.x = x;
  a.q = static_cast<uint8_t*>(q);
  a.scale = scale;
  a.ldx = ldx;
  a.ldq = ldq;
  a.M = M;
  a.K = K;
  return rq::run<false>(a, dtype, q_type, stream);
}
