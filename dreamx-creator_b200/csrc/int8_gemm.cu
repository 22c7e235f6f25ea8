// int8_gemm.cu -- row-wise scaled int8 GEMM.
//
//   out[m, n] = a_scale[m] * w_scale[n] * sum_k A[m, k] W[n, k] + bias[n]
//
// The sum is exact in int32 (|A|, |W| <= 128 and K <= 131072 keep it below 2^31).
#include "sm100.cuh"
#include "srdit_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace srdit {
namespace i8 {

struct Params {
  const int8_t* a;
  const int8_t* w;
  const float* a_scale;
  const float* w_scale;
  const void* bias;
  void* out;
  long long lda, ldw, ldo;
  int M, N, K;
};

template <typename T>
SRDIT_DEV float to_f(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else return static_cast<float>(v);
}

// One output per thread, four products per dp4a.
template <typename T>
__global__ void __launch_bounds__(256) simple_kernel(const Params p) {
  pdl_begin();
  const int n = blockIdx.x * 16 + (threadIdx.x & 15);
  const int m = blockIdx.y * 16 + (threadIdx.x >> 4);
  if (m >= p.M || n >= p.N) return;
  const int8_t* a = p.a + m * p.lda;
  const int8_t* w = p.w + n * p.ldw;
  int acc = 0;
  int k = 0;
  for (; k + 4 <= p.K; k += 4)
    acc = __dp4a(*reinterpret_cast<const int*>(a + k), *reinterpret_cast<const int*>(w + k), acc);
  for (; k < p.K; ++k) acc += static_cast<int>(a[k]) * static_cast<int>(w[k]);
  float y = static_cast<float>(acc) * p.a_scale[m] * p.w_scale[n];
  if (p.bias) y += to_f<T>(static_cast<const T*>(p.bias)[n]);
  static_cast<T*>(p.out)[m * p.ldo + n] = static_cast<T>(y);
}

template <typename T>
static int launch(const Params& p, cudaStream_t stream) {
  const dim3 grid((p.N + 15) / 16, (p.M + 15) / 16);
  SRDIT_LAUNCH((simple_kernel<T>), grid, 256, 0, stream, p);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace i8
}  // namespace srdit

using namespace srdit;

extern "C" int srdit_int8_gemm(const void* a, const float* a_scale, const void* w,
                               const float* w_scale, const void* bias, void* out, int dtype, int M,
                               int N, int K, long long lda, long long ldw, long long ldo,
                               uint32_t* status, cudaStream_t stream) {
  (void)status;
  if (M < 0 || N < 0 || K <= 0) return SRDIT_EINVAL;
  if (M == 0 || N == 0) return 0;
  if (!a || !a_scale || !w || !w_scale || !out) return SRDIT_EINVAL;
  if (lda < K || ldw < K || ldo < N) return SRDIT_EINVAL;
  if (K > 131072) return SRDIT_EUNSUPPORTED;
  if ((lda % 16) || (ldw % 16) || (reinterpret_cast<uintptr_t>(a) & 15u) ||
      (reinterpret_cast<uintptr_t>(w) & 15u))
    return SRDIT_EALIGN;
  i8::Params p = {static_cast<const int8_t*>(a), static_cast<const int8_t*>(w), a_scale, w_scale,
                  bias, out, lda, ldw, ldo, M, N, K};
  switch (dtype) {
    case SRDIT_BF16: return i8::launch<__nv_bfloat16>(p, stream);
    case SRDIT_FP16: return i8::launch<__half>(p, stream);
    case SRDIT_FP32: return i8::launch<float>(p, stream);
    default: return SRDIT_EINVAL;
  }
}
