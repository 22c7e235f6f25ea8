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

constexpr int ROWS = 16;  // rows of a warp

// A row is LPR lanes' 16 values each: 4 lanes up to 64 wide, else 8. This lane's row of a warp's
// i-th 32 / LPR.
template <int LPR>
struct Place {
  int side, h;  // k or v, head
  bool on;
  SRDIT_DEV Place(const Args& a, int r0, int i) {
    const int lane = threadIdx.x & 31;
    const int r = r0 + i * (32 / LPR) + lane / LPR;
    side = r >= a.Hkv;
    h = r - side * a.Hkv;
    on = r < 2 * a.Hkv && lane % LPR * 16 < a.D;
  }
};

// the larger magnitude of each half, NaN if one is
template <typename T>
SRDIT_DEV uint32_t max_abs2(uint32_t m, uint32_t w) {
  uint32_t d;
  if constexpr (__is_same(T, __half))
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(m), "r"(w));
  else
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(m), "r"(w));
  return d;
}
template <typename T>
SRDIT_DEV uint64_t widen2(uint32_t w) {
  if constexpr (__is_same(T, __half)) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2_pack(f.x, f.y);
  } else {
    return bf2_unpack(w);
  }
}
// two pairs as four codes: values times inv, each product rounded, then the code
template <int CODE>
SRDIT_DEV uint32_t codes4(uint64_t x, uint64_t y, uint64_t inv) {
  x = f2_mul(x, inv);
  y = f2_mul(y, inv);
  if constexpr (CODE == SRDIT_Q_INT8) {
    // 1.5 2^23 + n has n in its low byte. (Single additions: the compiler makes one rounding of a
    // product and a sum of pairs.)
    auto whole = [](float v) { return __float_as_uint(__fadd_rn(v, 12582912.f)); };
    const float2 a = f2_split(x), b = f2_split(y);
    return __byte_perm(__byte_perm(whole(a.x), whole(a.y), 0x0040),
                       __byte_perm(whole(b.x), whole(b.y), 0x0040), 0x5410);
  } else {
    const float2 a = f2_split(x), b = f2_split(y);
    uint32_t d;
    asm("{.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1; cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};}"
        : "=r"(d)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
  }
}

// A warp takes 16 rows (heads of k, then of v) of one token. The rows' loads do not wait for the
// search of their sequence, which is one trip to memory; the page is another.
// Bounded by memory: 6912 tokens of 24 heads of 128, bf16 to e4m3, 24.4 us, 5.3 TB/s (with 8 rows a warp,
// 8 values a lane and the search in three trips 39); in 16 bits 30 us, 5.6 TB/s.
template <typename T, int CODE, int LPR>
__global__ void __launch_bounds__(256) write_kernel(const __grid_constant__ Args a) {
  pdl_begin();
  constexpr int N = ROWS * LPR / 32;
  const int lane = threadIdx.x & 31, col = lane % LPR * 16;
  const int task = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = a.by_groups.div(task);
  const int r0 = (task - t * a.groups) * ROWS;
  if (t >= a.rows.rows) return;
  uint4 w[N][2];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Place<LPR> p(a, r0, i);
    w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
    if (p.on) {
      const uint4* x = reinterpret_cast<const uint4*>(
          a.x[p.side] + (t * a.xs[p.side][0] + p.h * a.xs[p.side][1] + col) * 2);
      w[i][0] = __ldg(x);
      if (col + 8 < a.D) w[i][1] = __ldg(x + 1);
    }
  }
  int len, begin, end;
  const int b = find_sequence(a.rows, a.B, t, a.by_each, a.lens, len, begin, end);
  if (b >= a.B) return;
  const int place = len - (end - t);  // this token's in its sequence
  if (place < 0) return;
  const int n = a.table.by_page.div(place);
  const long long page = a.table.page(b, n);
  if (page < 0) return;
  const long long row = place - n * a.table.page_size;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Place<LPR> p(a, r0, i);
    const long long at = page * a.ps[p.side][0] + row * a.ps[p.side][1] + p.h * a.ps[p.side][2] + col;
    const uint32_t u[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w,
                           w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
    if constexpr (CODE == SRDIT_KV_PLAIN) {
      if (!p.on) continue;
      uint4* dst = reinterpret_cast<uint4*>(a.page[p.side] + at * 2);
      dst[0] = w[i][0];
      if (col + 8 < a.D) dst[1] = w[i][1];
    } else {
      constexpr float q = CODE == SRDIT_Q_INT8 ? 127.f : 448.f;
      uint32_t m = u[0];
#pragma unroll
      for (int x = 1; x < 8; ++x) m = max_abs2<T>(m, u[x]);
      const float2 mf = f2_split(widen2<T>(m));
      float mx = max2(fabsf(mf.x), fabsf(mf.y));
#pragma unroll
      for (int o = LPR / 2; o; o >>= 1) mx = max2(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float scale = max2(__fmul_rn(mx, 1.f / q), 1e-12f);
      const float inv = __fdiv_rn(1.f, scale);
      const uint64_t inv2 = f2_pack(inv, inv);
      uint32_t c[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        c[x] = codes4<CODE>(widen2<T>(u[2 * x]), widen2<T>(u[2 * x + 1]), inv2);
      if (CODE == SRDIT_Q_INT8 && !(scale < __int_as_float(0x7f800000)))
        c[0] = c[1] = c[2] = c[3] = 0u;  // no finite scale
      if (p.on) {
        *reinterpret_cast<uint4*>(a.page[p.side] + at) = make_uint4(c[0], c[1], c[2], c[3]);
        if (col == 0)
          a.scale[p.side][page * a.ss[p.side][0] + row * a.ss[p.side][1] + p.h * a.ss[p.side][2]] =
              scale;
      }
    }
  }
}

// The same the other way: token t - begin(b) of sequence b, whose rows of the packed tensors
// are [begin(b), end(b)). Rows of a page that the table does not have are zeros.
// Bounded by memory: 4 x 16384 tokens of 8 heads of 128, e4m3 to bf16, 68 to 71 us, 5.8 to 6.0 TB/s (as
// above 85); in 16 bits 84 us, 6.4 TB/s.
template <typename T, int CODE, int LPR>
__global__ void __launch_bounds__(256) read_kernel(const __grid_constant__ Args a) {
  pdl_begin();
  constexpr int N = ROWS * LPR / 32;
  const int lane = threadIdx.x & 31, col = lane % LPR * 16;
  const int task = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int t = a.by_groups.div(task);
  const int r0 = (task - t * a.groups) * ROWS;
  if (t >= a.rows.rows) return;
  int len, begin, end;
  const int b = find_sequence(a.rows, a.B, t, a.by_each, nullptr, len, begin, end);
  if (b >= a.B) return;
  const int place = t - begin;
  const int n = a.table.by_page.div(place);
  const long long page = a.table.page(b, n);
  const long long row = place - n * a.table.page_size;
  uint4 w[N][2];
  float s[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Place<LPR> p(a, r0, i);
    w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
    s[i] = 0.f;
    if (!p.on || page < 0) continue;
    const long long at = page * a.ps[p.side][0] + row * a.ps[p.side][1] + p.h * a.ps[p.side][2] + col;
    if constexpr (CODE == SRDIT_KV_PLAIN) {
      const uint4* src = reinterpret_cast<const uint4*>(a.page[p.side] + at * 2);
      w[i][0] = src[0];
      if (col + 8 < a.D) w[i][1] = src[1];
    } else {
      w[i][0] = *reinterpret_cast<const uint4*>(a.page[p.side] + at);
      s[i] = a.scale[p.side][page * a.ss[p.side][0] + row * a.ss[p.side][1] + p.h * a.ss[p.side][2]];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Place<LPR> p(a, r0, i);
    if (!p.on) continue;
    if constexpr (CODE != SRDIT_KV_PLAIN) {
      const uint32_t u[4] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w};
      uint32_t o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t c = u[e >> 1] >> (16 * (e & 1));
        float2 v;
        if constexpr (CODE == SRDIT_Q_INT8) {
          v = make_float2(static_cast<int8_t>(c), static_cast<int8_t>(c >> 8));
        } else {
          uint32_t h2;
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(c)));
          v = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        }
        o[e] = pack2(__fmul_rn(v.x, s[i]), __fmul_rn(v.y, s[i]), T{});
      }
      w[i][0] = make_uint4(o[0], o[1], o[2], o[3]);
      w[i][1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
    uint4* dst = reinterpret_cast<uint4*>(
        a.x[p.side] + (t * a.xs[p.side][0] + p.h * a.xs[p.side][1] + col) * 2);
    dst[0] = w[i][0];
    if (col + 8 < a.D) dst[1] = w[i][1];
  }
}

template <bool kWrite, typename T, int CODE>
static int launch(const Args& a, unsigned blocks, cudaStream_t stream) {
  if (kWrite && a.D <= 64)
    SRDIT_LAUNCH((write_kernel<T, CODE, 4>), blocks, 256, 0, stream, a);
  else if (kWrite)
    SRDIT_LAUNCH((write_kernel<T, CODE, 8>), blocks, 256, 0, stream, a);
  else if (a.D <= 64)
    SRDIT_LAUNCH((read_kernel<T, CODE, 4>), blocks, 256, 0, stream, a);
  else
    SRDIT_LAUNCH((read_kernel<T, CODE, 8>), blocks, 256, 0, stream, a);
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
