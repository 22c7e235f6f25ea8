// seq_attn.cu -- attention of packed sequences of queries over keys in the pages of a cache (16
// bits, or 8-bit codes with a scale per token and head) or in packed rows of their own.
//
//   o[i, h] = sum_j p_j v[j, g] / sum_j p_j,   p_j = exp(scale q.k_j - max)
//
// over the L keys of the query's sequence, or with a causal mask over those up to its own
// token, j <= L - n + i for query i of n; g = h / (H / Hkv). A row that sees no key is 0.
// The softmax is one pass over the keys with a running maximum m and sum l, in fp32 and base
// 2: p = 2^(s c - m) with c = scale log2(e).
#include <atomic>

#include "seq.cuh"

namespace srdit {
namespace sattn {

struct Args {
  const void* q;
  void* out;
  long long qs[2], os[2];
  const void* kv[2];
  long long ps[2][3], ss[2][3];  // strides {page, token, head}; packed keys are one page
  const float* scale[2];
  Table table;
  Offsets rows, keys;
  Divisor by_each;
  const int32_t* lens;
  int B, H, Hkv, D, group, paged, causal;
  float c;
};

// The simplest form: a warp per query row, a lane four of its values, key after key.
template <typename T, int CODE>
__global__ void __launch_bounds__(256) row_kernel(const __grid_constant__ Args a) {
  pdl_begin();
  const int lane = threadIdx.x & 31, col = lane * 4;
  const long long task = blockIdx.x * 8ll + (threadIdx.x >> 5);
  const int t = static_cast<int>(task / a.H), h = static_cast<int>(task % a.H);
  if (t >= a.rows.rows) return;
  const int b = find_sequence(a.rows, a.B, t, a.by_each);
  if (b >= a.B) return;
  const bool on = col < a.D;
  const int len = a.paged ? a.table.clamp_len(__ldg(a.lens + b)) : a.keys.end(b) - a.keys.begin(b);
  const int last = a.causal ? min(len, len - (a.rows.end(b) - t) + 1) : len;
  auto four = [&](const void* p, long long at, float (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = 0.f;
      if (!on) continue;
      if constexpr (CODE == SRDIT_KV_PLAIN) {
        f[e] = to_f(static_cast<const T*>(p)[at + e]);
      } else if constexpr (CODE == SRDIT_Q_INT8) {
        f[e] = static_cast<const int8_t*>(p)[at + e];
      } else {
        uint32_t h2;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;"
            : "=r"(h2)
            : "h"(static_cast<uint16_t>(static_cast<const uint8_t*>(p)[at + e])));
        f[e] = __low2float(*reinterpret_cast<const __half2*>(&h2));
      }
    }
  };
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = neg_inf(), l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    q[e] = on ? to_f(static_cast<const T*>(a.q)[t * a.qs[0] + h * a.qs[1] + col + e]) : 0.f;
  for (int j = 0; j < last; ++j) {
    long long page = 0, row = a.keys.begin(b) + j;
    if (a.paged) {
      const int n = a.table.by_page.div(j);
      page = a.table.page(b, n);
      if (page < 0) continue;
      row = j - n * a.table.page_size;
    }
    const int g = h / a.group;
    float k[4], v[4], s = 0.f;
    four(a.kv[0], page * a.ps[0][0] + row * a.ps[0][1] + g * a.ps[0][2] + col, k);
    four(a.kv[1], page * a.ps[1][0] + row * a.ps[1][1] + g * a.ps[1][2] + col, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(q[e], k[e], s);
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    float f = 1.f;
    if constexpr (CODE != SRDIT_KV_PLAIN) {
      s *= a.scale[0][page * a.ss[0][0] + row * a.ss[0][1] + g * a.ss[0][2]];
      f = a.scale[1][page * a.ss[1][0] + row * a.ss[1][1] + g * a.ss[1][2]];
    }
    s *= a.c;
    const float mn = max2(m, s), neg = mn == neg_inf() ? 0.f : -mn;
    const float alpha = ex2(m + neg), p = ex2(s + neg);
    m = mn;
    l = fmaf(l, alpha, p);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(p * f, v[e], o[e] * alpha);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (on)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + t * a.os[0] + h * a.os[1] + col) =
        make_uint2(pack2(o[0] * inv, o[1] * inv, T{}), pack2(o[2] * inv, o[3] * inv, T{}));
}

template <typename T, int CODE>
static int run(const Args& a, cudaStream_t stream) {
  const long long tasks = static_cast<long long>(a.rows.rows) * a.H;
  SRDIT_LAUNCH((row_kernel<T, CODE>), static_cast<unsigned>((tasks + 7) / 8), 256, 0, stream, a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T>
static int run_code(const Args& a, int code, cudaStream_t stream) {
  switch (code) {
    case SRDIT_Q_INT8: return run<T, SRDIT_Q_INT8>(a, stream);
    case SRDIT_Q_E4M3: return run<T, SRDIT_Q_E4M3>(a, stream);
    default: return run<T, SRDIT_KV_PLAIN>(a, stream);
  }
}

// 16-byte rows: base and the strides that are used; entries of an output are one place each
static int check_view(const void* p, const long long st[2], int n, int h, bool one_place) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return SRDIT_EALIGN;
  const int dims[2] = {n, h};
  for (int i = 0; i < 2; ++i) {
    if (dims[i] <= 1) continue;
    if (st[i] < 0 || st[i] % 8) return SRDIT_EALIGN;
    if (st[i] == 0 && (one_place || i == 0)) return SRDIT_EINVAL;
  }
  return 0;
}

// argument checks; 1: nothing to do
static int check(const srdit_seq_attn_args& a) {
  if (a.B < 0 || a.T < 0 || a.H < 0 || a.Hkv <= 0 || a.H % a.Hkv || a.max_q < 0 || a.max_kv < 0)
    return SRDIT_EINVAL;
  if (a.dtype != SRDIT_BF16 && a.dtype != SRDIT_FP16) return SRDIT_EINVAL;
  const bool paged = a.pages != nullptr;
  if (paged) {
    const int rc = check_pages(*a.pages);
    if (rc) return rc;
    if (a.pages->B != a.B || a.pages->Hkv != a.Hkv || a.pages->D != a.D ||
        a.pages->dtype != a.dtype)
      return SRDIT_EINVAL;
  } else if (a.Tk < 0) {
    return SRDIT_EINVAL;
  }
  if (a.B == 0 || a.T == 0 || a.H == 0) return 1;
  if (!a.q || !a.out || !(a.scale > 0.f) || a.scale > 3.4028234e38f) return SRDIT_EINVAL;
  if (!a.cu_q && a.T % a.B) return SRDIT_EINVAL;
  if (paged ? !a.kv_lens : (a.Tk > 0 && (!a.k || !a.v)) || (!a.cu_k && !a.cu_q && a.Tk % a.B))
    return SRDIT_EINVAL;
  if (a.D <= 0 || a.D > 128 || a.D % 8) return SRDIT_EUNSUPPORTED;
  if (static_cast<long long>(a.B) * a.Hkv > 65535 ||
      static_cast<long long>(a.T) * a.H > (1ll << 26))
    return SRDIT_EUNSUPPORTED;
  int rc = check_view(a.q, a.q_stride, a.T, a.H, false);
  if (!rc) rc = check_view(a.out, a.o_stride, a.T, a.H, true);
  if (!rc && !paged) rc = check_view(a.k, a.k_stride, a.Tk, a.Hkv, false);
  if (!rc && !paged) rc = check_view(a.v, a.v_stride, a.Tk, a.Hkv, false);
  if (rc) return rc;
  if ((reinterpret_cast<uintptr_t>(a.cu_q) | reinterpret_cast<uintptr_t>(a.cu_k) |
       reinterpret_cast<uintptr_t>(a.kv_lens)) & 3u)
    return SRDIT_EALIGN;
  return 0;
}

}  // namespace sattn
}  // namespace srdit

using namespace srdit;

extern "C" int srdit_seq_attn_workspace(const srdit_seq_attn_args* args) {
  if (!args || sattn::check(*args) != 0) return 0;
  return 0;
}

extern "C" int srdit_seq_attn(const srdit_seq_attn_args* args, cudaStream_t stream) {
  if (!args) return SRDIT_EINVAL;
  const srdit_seq_attn_args& u = *args;
  const int rc = sattn::check(u);
  if (rc) return rc < 0 ? rc : 0;
  sattn::Args a = {};
  a.q = u.q;
  a.out = u.out;
  a.paged = u.pages != nullptr;
  const long long* const st[2] = {u.k_stride, u.v_stride};
  if (u.pages) {
    const srdit_kv_pages& p = *u.pages;
    a.table = table_of(p);
    const void* const kv[2] = {p.k, p.v};
    const long long* const ps[2] = {p.k_stride, p.v_stride};
    const long long* const ss[2] = {p.ks_stride, p.vs_stride};
    const float* const scale[2] = {p.k_scale, p.v_scale};
    for (int i = 0; i < 2; ++i) {
      a.kv[i] = kv[i];
      a.scale[i] = scale[i];
      for (int d = 0; d < 3; ++d) {
        a.ps[i][d] = ps[i][d];
        a.ss[i][d] = ss[i][d];
      }
    }
  } else {
    a.kv[0] = u.k;
    a.kv[1] = u.v;
    for (int i = 0; i < 2; ++i) {
      a.ps[i][1] = st[i][0];
      a.ps[i][2] = st[i][1];
    }
    a.keys = {u.cu_k ? u.cu_k : u.cu_q, u.Tk, u.Tk / u.B};
  }
  for (int i = 0; i < 2; ++i) {
    a.qs[i] = u.q_stride[i];
    a.os[i] = u.o_stride[i];
  }
  a.rows = {u.cu_q, u.T, u.T / u.B};
  a.by_each = Divisor::of(u.cu_q ? 1 : u.T / u.B);
  a.lens = u.kv_lens;
  a.B = u.B;
  a.H = u.H;
  a.Hkv = u.Hkv;
  a.D = u.D;
  a.group = u.H / u.Hkv;
  a.causal = u.causal;
  a.c = u.scale * kLog2e;
  const int code = u.pages ? u.pages->code : SRDIT_KV_PLAIN;
  return u.dtype == SRDIT_BF16 ? sattn::run_code<__nv_bfloat16>(a, code, stream)
                               : sattn::run_code<__half>(a, code, stream);
}
