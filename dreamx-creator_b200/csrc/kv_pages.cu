// kv_pages.cu -- a key/value cache in pages: new tokens' keys and values written into them, in
// 16 bits or as 8-bit codes with one fp32 scale per token and head, and read back.
//
//   token i of the n new ones of sequence b is its token p = kv_lens[b] - n + i, which lies in
//   row p % page_size of page table[b, p / page_size]
//   scale = max(max_d |x_d| * (1 / Q), 1e-12),  Q = 127 (int8) or 448 (e4m3)
//   code_d = round(x_d * (1 / scale)), ties to even; read back: code_d * scale, rounded once
//
// Every operation is rounded as it stands here, so codes are the same wherever they are
// computed in this way. A row holding a NaN gets the scale NaN, one with an infinity the scale
// infinity, and what their codes stand for is NaN, as with the row quantisers.
#include "seq.cuh"

namespace srdit {

// base and the strides {page, token, head} that are used in units of 16 bytes
static bool pool_aligned(const void* p, const long long st[3], const int n[3], int unit) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && st[i] % unit) return false;
  return true;
}

int check_pages(const srdit_kv_pages& p) {
  const bool codes = p.code != SRDIT_KV_PLAIN;
  if (p.B < 0 || p.pages < 0 || p.Hkv <= 0 || p.D <= 0 || p.page_size <= 0 || p.table_width < 0)
    return SRDIT_EINVAL;
  if (p.dtype != SRDIT_BF16 && p.dtype != SRDIT_FP16) return SRDIT_EINVAL;
  if (codes && p.code != SRDIT_Q_INT8 && p.code != SRDIT_Q_E4M3) return SRDIT_EINVAL;
  if (p.pages > 0 && (!p.k || !p.v || (codes && (!p.k_scale || !p.v_scale)))) return SRDIT_EINVAL;
  if (p.B > 0 && p.table_width > 0 && !p.table) return SRDIT_EINVAL;
  const int unit = codes ? 16 : 8;
  if (p.D > 128 || p.D % unit || p.Hkv > 1024 ||
      !(p.page_size % 128 == 0 || p.page_size == 16 || p.page_size == 32 || p.page_size == 64) ||
      static_cast<long long>(p.table_width) * p.page_size > 0x7fffff00ll)
    return SRDIT_EUNSUPPORTED;
  const int n[3] = {p.pages, p.page_size, p.Hkv};
  if (!pool_aligned(p.k, p.k_stride, n, unit) || !pool_aligned(p.v, p.v_stride, n, unit) ||
      (reinterpret_cast<uintptr_t>(p.table) & 3u) ||
      (reinterpret_cast<uintptr_t>(p.k_scale) & 3u) || (reinterpret_cast<uintptr_t>(p.v_scale) & 3u))
    return SRDIT_EALIGN;
  // an entry of the cache is one place, ahead of the base
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (p.k_stride[i] <= 0 || p.v_stride[i] <= 0 ||
                     (codes && (p.ks_stride[i] <= 0 || p.vs_stride[i] <= 0))))
      return SRDIT_EINVAL;
  return 0;
}

namespace kvp {

struct Args {
  Table table;
  Offsets rows;           // of the packed tensors
  Divisor by_each, by_groups;
  const int32_t* lens;    // write: tokens of each sequence with the new ones
  int B, Hkv, D;
  int groups;             // of ROWS rows: 2 Hkv rows a token (keys, then values)
  uint8_t* page[2];       // k, v
  float* scale[2];
  long long ps[2][3];     // strides {page, token, head} of pages
  long long ss[2][3];     // ... and of scales
  uint8_t* x[2];          // packed rows
  long long xs[2][2];     // strides {token, head}
};

constexpr int ROWS = 8;  // rows of a warp: two at a time, a lane 8 values

template <typename T>
SRDIT_DEV void widen(uint4 w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T* t = reinterpret_cast<const T*>(&u[i]);
    f[2 * i] = to_f(t[0]);
    f[2 * i + 1] = to_f(t[1]);
  }
}
SRDIT_DEV uint2 codes_int8(const float (&f)[8], float inv, bool zero) {
  uint32_t h[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)  // 1.5 2^23 + n has n in its low byte
      b[e] = __float_as_uint(__fadd_rn(__fmul_rn(f[4 * i + e], inv), 12582912.f));
    h[i] = zero ? 0u
                : __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040),
                              0x5410);
  }
  return make_uint2(h[0], h[1]);
}
SRDIT_DEV uint2 codes_e4m3(const float (&f)[8], float inv) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;"
        : "=h"(c)
        : "f"(__fmul_rn(f[2 * i + 1], inv)), "f"(__fmul_rn(f[2 * i], inv)));
    h[i] = c;
  }
  return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// A warp takes 8 rows (heads of k, then of v) of one token, two at a time, half a warp a row.
// The rows' loads do not wait for the search of their sequence.
template <typename T, int CODE>
__global__ void __launch_bounds__(256) write_kernel(const __grid_constant__ Args a) {
  pdl_begin();
  const int lane = threadIdx.x & 31, half = lane >> 4, col = (lane & 15) * 8;
  const int task = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = a.by_groups.div(task);
  const int r0 = (task - t * a.groups) * ROWS;
  if (t >= a.rows.rows) return;
  const bool on = col < a.D;
  uint4 w[ROWS / 2];
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) {
    const int r = r0 + 2 * i + half, side = r >= a.Hkv, h = r - side * a.Hkv;
    w[i] = make_uint4(0, 0, 0, 0);
    if (on && r < 2 * a.Hkv)
      w[i] = __ldg(reinterpret_cast<const uint4*>(
          a.x[side] + (t * a.xs[side][0] + h * a.xs[side][1] + col) * 2));
  }
  const int b = find_sequence(a.rows, a.B, t, a.by_each);
  if (b >= a.B) return;
  const int p = __ldg(a.lens + b) - (a.rows.end(b) - t);  // this token's place in it
  if (p < 0) return;
  const int n = a.table.by_page.div(p);
  const long long page = a.table.page(b, n);
  if (page < 0) return;
  const long long row = p - n * a.table.page_size;
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) {
    const int r = r0 + 2 * i + half, side = r >= a.Hkv, h = r - side * a.Hkv;
    const bool here = on && r < 2 * a.Hkv;
    const long long at =
        page * a.ps[side][0] + row * a.ps[side][1] + h * a.ps[side][2] + col;
    if constexpr (CODE == SRDIT_KV_PLAIN) {
      if (here) *reinterpret_cast<uint4*>(a.page[side] + at * 2) = w[i];
    } else {
      constexpr float q = CODE == SRDIT_Q_INT8 ? 127.f : 448.f;
      float f[8];
      widen<T>(w[i], f);
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = max2(mx, fabsf(f[e]));
#pragma unroll
      for (int o = 8; o; o >>= 1) mx = max2(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float scale = max2(__fmul_rn(mx, 1.f / q), 1e-12f);
      const float inv = __fdiv_rn(1.f, scale);
      if (here) {
        const bool zero = !(scale < __int_as_float(0x7f800000));
        *reinterpret_cast<uint2*>(a.page[side] + at) =
            CODE == SRDIT_Q_INT8 ? codes_int8(f, inv, zero) : codes_e4m3(f, inv);
        if (col == 0)
          a.scale[side][page * a.ss[side][0] + row * a.ss[side][1] + h * a.ss[side][2]] = scale;
      }
    }
  }
}

// The same the other way: token t - begin(b) of sequence b, whose rows of the packed tensors
// are [begin(b), end(b)). Rows of a page that the table does not have are zeros.
template <typename T, int CODE>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ Args a) {
  pdl_begin();
  const int lane = threadIdx.x & 31, half = lane >> 4, col = (lane & 15) * 8;
  const int task = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = a.by_groups.div(task);
  const int r0 = (task - t * a.groups) * ROWS;
  if (t >= a.rows.rows) return;
  const int b = find_sequence(a.rows, a.B, t, a.by_each);
  if (b >= a.B) return;
  const int p = t - a.rows.begin(b);
  const int n = a.table.by_page.div(p);
  const long long page = a.table.page(b, n);
  const long long row = p - n * a.table.page_size;
  const bool on = col < a.D;
  uint4 w[ROWS / 2];
  float s[ROWS / 2];
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) {
    const int r = r0 + 2 * i + half, side = r >= a.Hkv, h = r - side * a.Hkv;
    w[i] = make_uint4(0, 0, 0, 0);
    s[i] = 0.f;
    if (!on || r >= 2 * a.Hkv || page < 0) continue;
    const long long at =
        page * a.ps[side][0] + row * a.ps[side][1] + h * a.ps[side][2] + col;
    if constexpr (CODE == SRDIT_KV_PLAIN) {
      w[i] = *reinterpret_cast<const uint4*>(a.page[side] + at * 2);
    } else {
      const uint2 c = *reinterpret_cast<const uint2*>(a.page[side] + at);
      w[i].x = c.x;
      w[i].y = c.y;
      s[i] = a.scale[side][page * a.ss[side][0] + row * a.ss[side][1] + h * a.ss[side][2]];
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS / 2; ++i) {
    const int r = r0 + 2 * i + half, side = r >= a.Hkv, h = r - side * a.Hkv;
    if (!on || r >= 2 * a.Hkv) continue;
    uint4 o = w[i];
    if constexpr (CODE != SRDIT_KV_PLAIN) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t c = (e & 2 ? w[i].y : w[i].x) >> (16 * (e & 1));
        float2 v;
        if constexpr (CODE == SRDIT_Q_INT8) {
          v = make_float2(static_cast<int8_t>(c), static_cast<int8_t>(c >> 8));
        } else {
          uint32_t h2;
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(c)));
          v = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        }
        u[e] = pack2(__fmul_rn(v.x, s[i]), __fmul_rn(v.y, s[i]), T{});
      }
      o = make_uint4(u[0], u[1], u[2], u[3]);
    }
    *reinterpret_cast<uint4*>(a.x[side] + (t * a.xs[side][0] + h * a.xs[side][1] + col) * 2) = o;
  }
}

template <bool kWrite, typename T, int CODE>
static int launch(const Args& a, unsigned blocks, cudaStream_t stream) {
  if constexpr (kWrite)
    SRDIT_LAUNCH((write_kernel<T, CODE>), blocks, 256, 0, stream, a);
  else
    SRDIT_LAUNCH((read_kernel<T, CODE>), blocks, 256, 0, stream, a);
  return static_cast<int>(cudaGetLastError());
}

template <bool kWrite, typename T>
static int launch_code(const Args& a, int code, unsigned blocks, cudaStream_t stream) {
  switch (code) {
    case SRDIT_Q_INT8: return launch<kWrite, T, SRDIT_Q_INT8>(a, blocks, stream);
    case SRDIT_Q_E4M3: return launch<kWrite, T, SRDIT_Q_E4M3>(a, blocks, stream);
    default: return launch<kWrite, T, SRDIT_KV_PLAIN>(a, blocks, stream);
  }
}

// packed rows of T tokens in sequences of cu (or T / B each)
template <bool kWrite>
static int run(const srdit_kv_pages* pages, const void* k, const long long* k_stride,
               const void* v, const long long* v_stride, int T, const int32_t* cu,
               const int32_t* lens, cudaStream_t stream) {
  if (!pages || !k_stride || !v_stride || T < 0) return SRDIT_EINVAL;
  const srdit_kv_pages& p = *pages;
  const int rc = check_pages(p);
  if (rc) return rc;
  if (T == 0 || p.B == 0) return 0;
  if (!k || !v || (kWrite && !lens) || (!cu && T % p.B)) return SRDIT_EINVAL;
  const void* x[2] = {k, v};
  const long long* st[2] = {k_stride, v_stride};
  for (int i = 0; i < 2; ++i) {
    if (reinterpret_cast<uintptr_t>(x[i]) & 15u) return SRDIT_EALIGN;
    const int n[2] = {T, p.Hkv};
    for (int d = 0; d < 2; ++d)
      if (n[d] > 1) {
        if (st[i][d] % 8) return SRDIT_EALIGN;
        if (!kWrite && st[i][d] <= 0) return SRDIT_EINVAL;  // each row is one place
      }
  }
  if ((reinterpret_cast<uintptr_t>(cu) & 3u) || (reinterpret_cast<uintptr_t>(lens) & 3u))
    return SRDIT_EALIGN;
  Args a = {};
  a.table = table_of(p);
  a.rows = {cu, T, T / p.B};
  a.by_each = Divisor::of(cu ? 1 : T / p.B);
  a.lens = lens;
  a.B = p.B;
  a.Hkv = p.Hkv;
  a.D = p.D;
  a.groups = (2 * p.Hkv + ROWS - 1) / ROWS;
  a.by_groups = Divisor::of(a.groups);
  const long long tasks = static_cast<long long>(T) * a.groups;
  if (tasks > 0x7ffffff0ll) return SRDIT_EUNSUPPORTED;
  void* const page[2] = {p.k, p.v};
  float* const scale[2] = {p.k_scale, p.v_scale};
  const long long* const ps[2] = {p.k_stride, p.v_stride};
  const long long* const ss[2] = {p.ks_stride, p.vs_stride};
  for (int i = 0; i < 2; ++i) {
    a.page[i] = static_cast<uint8_t*>(page[i]);
    a.scale[i] = scale[i];
    for (int d = 0; d < 3; ++d) {
      a.ps[i][d] = ps[i][d];
      a.ss[i][d] = ss[i][d];
    }
    a.x[i] = const_cast<uint8_t*>(static_cast<const uint8_t*>(x[i]));
    a.xs[i][0] = st[i][0];
    a.xs[i][1] = st[i][1];
  }
  const unsigned blocks = static_cast<unsigned>((tasks + 7) / 8);
  return p.dtype == SRDIT_BF16 ? launch_code<kWrite, __nv_bfloat16>(a, p.code, blocks, stream)
                               : launch_code<kWrite, __half>(a, p.code, blocks, stream);
}

}  // namespace kvp
}  // namespace srdit

using namespace srdit;

extern "C" int srdit_kv_write(const srdit_kv_pages* pages, const void* k,
                              const long long* k_stride, const void* v, const long long* v_stride,
                              int T, const int32_t* cu_q, const int32_t* kv_lens,
                              cudaStream_t stream) {
  return kvp::run<true>(pages, k, k_stride, v, v_stride, T, cu_q, kv_lens, stream);
}

extern "C" int srdit_kv_read(const srdit_kv_pages* pages, void* k, const long long* k_stride,
                             void* v, const long long* v_stride, int T, const int32_t* cu_k,
                             cudaStream_t stream) {
  return kvp::run<false>(pages, k, k_stride, v, v_stride, T, cu_k, nullptr, stream);
}
