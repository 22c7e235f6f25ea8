// cross_attn.cu -- attention of queries over an encoder's keys and values of another
// length, with per-sample key lengths, a key mask and grouped heads.
//
//   o[b, i, h] = sum_j p_j v[b, j, g] / sum_j p_j,   p_j = exp(scale q.k_j - max)
//
// over the keys j < kv_lens[b] with key_mask[b, j]; g = h / (H / Hkv). A row that
// sees no key is 0. A key that is not seen is never used: whatever its row holds
// (NaN, infinities) does not reach the output.
#include "sm100.cuh"
#include "srdit_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace srdit {
namespace xattn {

// One warp per (sample, query, head); a lane holds 4 of the head's values.
template <typename T>
__global__ void __launch_bounds__(256) simple_kernel(const srdit_cross_attn_args a) {
  pdl_begin();
  const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= static_cast<long long>(a.B) * a.Lq * a.H) return;
  const int h = static_cast<int>(item % a.H);
  const long long bi = item / a.H;
  const int i = static_cast<int>(bi % a.Lq), b = static_cast<int>(bi / a.Lq);
  const int g = h / (a.H / a.Hkv);
  const int len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Lk) : a.Lk;
  const T* q = static_cast<const T*>(a.q) + b * a.q_stride[0] + i * a.q_stride[1] + h * a.q_stride[2];
  const T* k = static_cast<const T*>(a.k) + b * a.k_stride[0] + g * a.k_stride[2];
  const T* v = static_cast<const T*>(a.v) + b * a.v_stride[0] + g * a.v_stride[2];
  const uint8_t* mask = a.key_mask ? a.key_mask + b * a.mask_stride : nullptr;
  float qv[4], o[4];
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < a.D ? static_cast<float>(q[d]) * a.scale : 0.f;
    o[e] = 0.f;
  }
  float m = -__int_as_float(0x7f800000), l = 0.f;
  for (long long j = 0; j < len; ++j) {
    if (mask && !mask[j]) continue;
    float s = 0.f;
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 32 * e;
      if (d < a.D) s += qv[e] * static_cast<float>(k[j * a.k_stride[1] + d]);
    }
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s);
    const float c = expf(m - mn), p = expf(s - mn);
    m = mn;
    l = l * c + p;
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 32 * e;
      if (d < a.D) o[e] = o[e] * c + p * static_cast<float>(v[j * a.v_stride[1] + d]);
    }
  }
  T* out = static_cast<T*>(a.out) + b * a.o_stride[0] + i * a.o_stride[1] + h * a.o_stride[2];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 32 * e;
    if (d < a.D) out[d] = static_cast<T>(o[e] * inv);
  }
}

}  // namespace xattn
}  // namespace srdit

using namespace srdit;

// 16-byte rows: base and every stride that is used
static bool check_view(const void* p, const long long st[3], int b, int l, int h) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  const int n[3] = {b, l, h};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] < 0 || st[i] % 8)) return false;
  return true;
}

extern "C" int srdit_cross_attn(const srdit_cross_attn_args* args, cudaStream_t stream) {
  if (!args) return SRDIT_EINVAL;
  const srdit_cross_attn_args& a = *args;
  if (a.B < 0 || a.Lq < 0 || a.Lk < 0 || a.H < 0 || a.Hkv <= 0 || a.H % a.Hkv) return SRDIT_EINVAL;
  if (a.B == 0 || a.Lq == 0 || a.H == 0) return 0;
  if (!a.q || !a.out || (a.Lk > 0 && (!a.k || !a.v)) || !(a.scale > 0.f)) return SRDIT_EINVAL;
  if (a.D <= 0 || a.D > 128 || a.D % 8) return SRDIT_EUNSUPPORTED;
  if (!check_view(a.q, a.q_stride, a.B, a.Lq, a.H) || !check_view(a.k, a.k_stride, a.B, a.Lk, a.Hkv) ||
      !check_view(a.v, a.v_stride, a.B, a.Lk, a.Hkv) || !check_view(a.out, a.o_stride, a.B, a.Lq, a.H))
    return SRDIT_EALIGN;
  // an output entry is one place
  if ((a.B > 1 && a.o_stride[0] == 0) || (a.Lq > 1 && a.o_stride[1] == 0) ||
      (a.H > 1 && a.o_stride[2] == 0))
    return SRDIT_EINVAL;
  const unsigned grid = static_cast<unsigned>((static_cast<long long>(a.B) * a.Lq * a.H + 7) / 8);
  if (a.dtype == SRDIT_BF16)
    SRDIT_LAUNCH((xattn::simple_kernel<__nv_bfloat16>), grid, 256, 0, stream, a);
  else if (a.dtype == SRDIT_FP16)
    SRDIT_LAUNCH((xattn::simple_kernel<__half>), grid, 256, 0, stream, a);
  else
    return SRDIT_EINVAL;
  return static_cast<int>(cudaGetLastError());
}

extern "C" int srdit_cross_attn_splits(const srdit_cross_attn_args* args) {
  (void)args;
  return 1;
}
