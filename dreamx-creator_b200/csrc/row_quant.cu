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
// What cannot be held: a row with a NaN has the scale NaN (max.NaN keeps it). One with an
// infinity has the scale NaN after a norm (inf * 0) and infinity without one, and int8 codes
// 0. Either way what its codes stand for is NaN. A finite row whose sum of squares is not
// finite (values from 2^56 on) is no such row: far_rstd.
#include "elem.cuh"
#include "srdit_internal.h"

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
  int rows;   // rows per block
  float eps, inv_k;
};

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
  for (int i = 0; i < V; ++i) o[i] = to_f(t.v[i]);
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
// the largest magnitude of three
SRDIT_DEV float amax3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
SRDIT_DEV float warp_amax(float v) {
  float d;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(v));
  return d;
}
SRDIT_DEV uint32_t code_e4m3x2(uint64_t v) {
  const float2 f = f2_split(v);
  uint16_t h;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(f.y), "f"(f.x));
  return h;
}
// The integers nearest to s * inv, for |s * inv| < 2^22: one fma to 1.5 2^23, whose sum has
// the integer in its low bits (to nearest, ties to even, from the exact product).
SRDIT_DEV uint64_t near_ints(uint64_t s, uint64_t inv) {
  return f2_fma(s, inv, f2_pack(12582912.f, 12582912.f));
}
SRDIT_DEV uint32_t low_bytes(uint64_t ab) {
  const float2 f = f2_split(ab);
  return __byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x0040);
}

// V codes of s * inv as one aligned store. `zero`: the row has no finite scale; its int8
// codes are 0 (e4m3 codes become NaN by themselves)
template <bool kInt8, int V>
SRDIT_DEV void store_codes(uint8_t* p, const float (&s)[V], uint64_t inv, bool zero) {
  uint32_t h[(V + 1) / 2];
#pragma unroll
  for (int i = 0; i < (V + 1) / 2; ++i) {
    const uint64_t v = f2_pack(s[2 * i], V > 1 ? s[2 * i + 1] : 0.f);
    h[i] = kInt8 ? low_bytes(near_ints(v, inv)) : code_e4m3x2(f2_mul(v, inv));
    if (kInt8 && zero) h[i] = 0u;
  }
  if constexpr (V == 1) {
    *p = static_cast<uint8_t>(h[0]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(h[0]);
  } else {
    static_assert(V == 8, "1, 2 or 8 codes");
    *reinterpret_cast<uint2*>(p) =
        make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
  }
}

// What a row's values need: the sum of squares and the largest magnitude.
template <bool kNorm, int V>
SRDIT_DEV void accumulate(float (&s)[V], const float (&w)[V], uint64_t& ss2, float& mx) {
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    const bool two = e + 1 < V;
    if constexpr (kNorm) {
      const uint64_t v = f2_pack(s[e], two ? s[e + 1] : 0.f);
      ss2 = f2_fma(v, v, ss2);
      const float2 y = f2_split(f2_mul(v, f2_pack(w[e], two ? w[e + 1] : 0.f)));
      s[e] = y.x;
      if (two) s[e + 1] = y.y;
    }
    mx = amax3(mx, s[e], two ? s[e + 1] : 0.f);
  }
}

// 1 / sqrt(mean(s^2) + eps) of a finite row x [+ r] whose sum of squares is beyond fp32 (values
// from 2^56 on): of the values times 2^-72, whose squares' sum is not, read once more by each
// of the row's warps.
template <typename T>
SRDIT_DEV float far_rstd(const T* x, const T* r, int K, float inv_k, float eps) {
  constexpr float down = 0x1p-72f;
  float ss = 0.f;
  __syncwarp();
#pragma unroll 1
  for (int c = threadIdx.x & 31; c < K; c += 32) {
    const float v = (to_f(x[c]) + (r ? to_f(r[c]) : 0.f)) * down;
    ss = fmaf(v, v, ss);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  return rsqrtf(fmaf(ss, inv_k, eps * down * down)) * down;
}

// (a call where the code inlined would cost a row of narrow vectors 6 registers)
template <typename T>
__device__ __noinline__ float far_rstd_call(const T* x, const T* r, int K, float inv_k, float eps) {
  return far_rstd<T>(x, r, K, inv_k, eps);
}

// The row's sums over its `warps` warps, the first of them `warp0` of the block, in the same
// order in every thread; then its scale and the factor from values to codes. far(): the norm's
// factor where the sum is beyond fp32.
template <typename T, bool kInt8, bool kNorm, typename F>
SRDIT_DEV void row_scale(const Args& a, uint64_t ss2, float mx, int warps, int warp0, float2* part,
                         float& scale, float& inv, F far) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float2 sp = f2_split(ss2);
  float ss = sp.x + sp.y;
  mx = warp_amax(mx);
  if constexpr (kNorm) {
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  if (warps > 1) {
    if (lane == 0) part[warp] = make_float2(ss, mx);
    __syncthreads();
    const float2 p = lane < warps ? part[warp0 + lane] : make_float2(0.f, 0.f);
    mx = warp_amax(p.y);
    if constexpr (kNorm) {
      ss = p.x;
#pragma unroll
      for (int o = 16; o; o >>= 1)
        if (o < warps) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      ss = __shfl_sync(0xffffffffu, ss, 0);
    }
  }
  // Approximate root and quotient, 2 units in the last place: every thread computes these.
  float rstd = kNorm ? rsqrtf(fmaf(ss, a.inv_k, a.eps)) : 1.0f;
  if constexpr (kNorm && !__is_same(T, __half)) {  // (fp16 has no such rows)
    constexpr float inf = __builtin_huge_valf();
    if (ss == inf && mx < inf) rstd = far();
  }
  scale = max_nan(mx * rstd * (kInt8 ? 1.f / 127.f : 1.f / 448.f), 1e-12f);
  inv = __fdividef(rstd, scale);
}

// Rows of up to 8192: one row per `warps` warps of the block, 8 values of it in a thread's
// registers as vectors of V (V = 8: 16-byte loads of 16-bit values; 2 and 1 for rows whose
// width, pitch or base is not so aligned), vector i of thread t at (i * threads + t) * V.
// Bounded by memory: 6912 x 3072 bf16 with the residual takes 27.5 us, 5.41 TB/s, what a
// copy of as many bytes reaches. (With scalar arithmetic, an exact root and quotients in every
// thread it took 34 instructions a value, 70% of the issue slots, and 30.9 us. With 16, 24
// and 32 values in a thread this one takes 29.3, 29.5 and 31.2 us, and a single row of 4096
// 2.9, 3.3 and 3.8 us in place of 2.5. Without far_rstd: 27.3.)
template <typename T, bool kInt8, bool kNorm, bool kRes, int V>
__global__ void __launch_bounds__(1024) rows_kernel(const Args a) {
  pdl_begin();
  constexpr int N = 8 / V;
  __shared__ float2 part[32];
  const int warp = threadIdx.x >> 5;
  const int tpr = a.warps * 32;
  const int sub = a.warps < 4 ? warp / a.warps : 0;  // row of the block
  const int t = threadIdx.x - sub * tpr;
  const long long row = static_cast<long long>(blockIdx.x) * a.rows + sub;
  const bool on = row < a.M;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = kRes ? static_cast<const T*>(a.res) + row * a.ldr : nullptr;
  const T* w = static_cast<const T*>(a.w);
  float s[N][V];
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
    }
  }
  uint64_t ss2 = f2_pack(0.f, 0.f);
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * tpr + t) * V;
    if (on && c < a.K) {
      if constexpr (kRes) store<T, V>(static_cast<T*>(a.sum) + row * a.lds + c, s[i]);
      float ww[V];
      if constexpr (kNorm) load<T, V>(w + c, ww);
      accumulate<kNorm, V>(s[i], ww, ss2, mx);
    }
  }
  float scale, inv;
  row_scale<T, kInt8, kNorm>(a, ss2, mx, a.warps, sub * a.warps, part, scale, inv, [&] {
    // (of the sum as it was stored, rounded: it may have taken the place of x or of r)
    const T* far = kRes ? static_cast<const T*>(a.sum) + row * a.lds
                        : static_cast<const T*>(a.x) + row * a.ldx;
    return V == 8 ? far_rstd<T>(far, nullptr, a.K, a.inv_k, a.eps)
                  : far_rstd_call<T>(far, nullptr, a.K, a.inv_k, a.eps);
  });
  if (!on) return;
  const bool zero = !(scale < __int_as_float(0x7f800000));
  if (t == 0) a.scale[row] = scale;
  uint8_t* q = a.q + row * a.ldq;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = (i * tpr + t) * V;
    if (c < a.K) store_codes<kInt8, V>(q + c, s[i], f2_pack(inv, inv), zero);
  }
}

// Wider rows: one block of 512 threads a row, which it reads twice, the second time out of
// the caches. The sum is stored in the second pass, since it may be x or the residual.
// Four blocks an SM: 6912 x 14336 bf16 67 to 70 us, with the residual 115 to 128 (with what the
// compiler takes by itself, 32 to 44 registers: 66 to 73, and 122 to 140).
template <typename T, bool kInt8, bool kNorm, bool kRes, int V>
__global__ void __launch_bounds__(512, 4) wide_rows_kernel(const Args a) {
  pdl_begin();
  __shared__ float2 part[16];
  const long long row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = kRes ? static_cast<const T*>(a.res) + row * a.ldr : nullptr;
  const T* w = static_cast<const T*>(a.w);
  auto value = [&](int c, float(&s)[V]) {
    load<T, V>(x + c, s);
    if constexpr (kRes) {
      float rr[V];
      load<T, V>(r + c, rr);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += rr[e];
    }
  };
  uint64_t ss2 = f2_pack(0.f, 0.f);
  float mx = 0.f;
#pragma unroll 4
  for (int c = threadIdx.x * V; c < a.K; c += 512 * V) {
    float s[V], ww[V];
    value(c, s);
    if constexpr (kNorm) load<T, V>(w + c, ww);
    accumulate<kNorm, V>(s, ww, ss2, mx);
  }
  float scale, inv;
  row_scale<T, kInt8, kNorm>(a, ss2, mx, 16, 0, part, scale, inv, [&] {
    const float rstd = far_rstd<T>(x, r, a.K, a.inv_k, a.eps);
    __syncthreads();  // every warp has read the row: the sum may take the place of x or of r
    return rstd;
  });
  const bool zero = !(scale < __int_as_float(0x7f800000));
  if (threadIdx.x == 0) a.scale[row] = scale;
  uint8_t* q = a.q + row * a.ldq;
#pragma unroll 4
  for (int c = threadIdx.x * V; c < a.K; c += 512 * V) {
    float s[V];
    value(c, s);
    if constexpr (kRes) store<T, V>(static_cast<T*>(a.sum) + row * a.lds + c, s);
    if constexpr (kNorm) {
      float ww[V];
      load<T, V>(w + c, ww);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] *= ww[e];
    }
    store_codes<kInt8, V>(q + c, s, f2_pack(inv, inv), zero);
  }
}

template <typename T, bool kInt8, bool kNorm, bool kRes, int V>
static int launch_v(Args& a, cudaStream_t stream) {
  if (a.K > 8192) {
    SRDIT_LAUNCH((wide_rows_kernel<T, kInt8, kNorm, kRes, V>), static_cast<unsigned>(a.M), 512, 0,
                 stream, a);
    return static_cast<int>(cudaGetLastError());
  }
  a.warps = (a.K + 255) / 256;
  a.rows = a.warps >= 4 ? 1 : 4 / a.warps;
  const unsigned grid = static_cast<unsigned>((a.M + a.rows - 1) / a.rows);
  SRDIT_LAUNCH((rows_kernel<T, kInt8, kNorm, kRes, V>), grid, a.rows * a.warps * 32, 0, stream, a);
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
  if (a.M == 1) a.ldx = a.ldr = a.lds = a.ldq = a.K;  // of one row they may be anything
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
  if (M > 1 && (ldx < K || ldq < K)) return SRDIT_EINVAL;
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
  if (residual && M > 1 && (ldr < K || ld_sum < K)) return SRDIT_EINVAL;
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
