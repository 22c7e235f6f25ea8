// seq_attn.cuh -- what the kernels of attention over packed sequences are given, and how a call
// is run.
#pragma once
#include "seq.cuh"

namespace srdit {
namespace sattn {

constexpr int TILE = 128;

struct Args {
  const void* q;
  void* out;
  long long qs[2], os[2];   // {token, head}, elements (keys and values go by tensor maps)
  const float* scale[2];    // of the codes of k, v
  long long ss[2][3];       // ... strides {page, token, head}
  Table table;              // pages (page_size 0: packed keys)
  Offsets rows, keys;       // queries; packed keys
  Divisor by_each;
  const int32_t* lens;      // pages: keys of each sequence
  int T, B, H, Hkv, D, group;
  int causal, max_q;
  float c;                  // scale * log2(e)
  float* ws;                // parts of rows: O
  float* ml;                // ... their {m, l}
  uint32_t* status;
  // chunk_kernel
  int pack, pack_log, rt;   // heads of a group side by side in a query tile (2^n), its tokens
  int slots, nhp;           // pieces of 2 rt tokens (some empty), head packs
  Divisor by_nhp, by_slots, by_piece;  // ... and 2 rt
  Divisor by_packs, by_ctas;           // ... the packs of a group, the CTAs
  int ranged, box_log;      // items shared out by key tiles; log2 of the keys of a page's box
  void* cuts;
  // step_kernel
  int splits, shared;       // parts of the keys; shares of all keys
  Divisor by_group;

  SRDIT_DEV bool paged() const { return table.page_size > 0; }
  SRDIT_DEV int key_count(int b) const {
    return paged() ? table.clamp_len(__ldg(lens + b)) : keys.end(b) - keys.begin(b);
  }
};

// How a call is run: the launch and the workspace's size go by it.
struct Plan {
  bool step;                    // step_kernel (few rows per key head), else chunk_kernel
  int splits, cluster, parts;   // step_kernel; parts in the workspace per row (1: none)
  bool shared;                  // ... all keys in equal shares
  int pack, rt, slots, nhp;     // chunk_kernel
  int ranged;                   // 0: whole items, 1: shared out by key tiles, 2: the last round
  int ctas;
  long long ws_floats;
};

Plan plan_step(const srdit_seq_attn_args& u, int sms);
Plan plan_chunk(const srdit_seq_attn_args& u, int sms);
int run_step(const srdit_seq_attn_args& u, Args& a, const Plan& p, cudaStream_t stream);
int run_chunk(const srdit_seq_attn_args& u, Args& a, const Plan& p, cudaStream_t stream);

// the element type that products are computed in: fp16 for codes, which it holds exactly
template <typename T, int CODE>
struct Compute {
  using type = __half;
};
template <typename T>
struct Compute<T, SRDIT_KV_PLAIN> {
  using type = T;
};

// Over codes parts of rows have sums of weights l in the unit of 2^(m - 24), where m is the maximum of
// score + exponent of the value's scale: with exponents from -80 to 125 they are in range.
constexpr int L_UNIT = 24;
// What takes O and l from one maximum to another that is x larger (x <= 0): a factor for O; l, in which
// a much smaller factor may count, by two halves of it.
template <bool CODES>
struct Fall {
  float f, half;
  SRDIT_DEV explicit Fall(float x) : f(0.f), half(ex2(CODES ? x * 0.5f : x)) {
    f = CODES ? half * half : half;
  }
  SRDIT_DEV float add(float l, float sum) const {  // sum + 2^x l
    return CODES ? fmaf(l * half, half, sum) : fmaf(l, f, sum);
  }
};

// 4 codes as fp16 values, exactly: the first two in x, the others in y
template <int CODE>
SRDIT_DEV void widen4(uint32_t u, uint32_t& x, uint32_t& y) {
  if constexpr (CODE == SRDIT_Q_INT8) {
    // n + 128 behind the exponent of 1024, less 1152
    const uint32_t b = u ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    const uint32_t lo = __byte_perm(b, 0x64646464u, 0x4140), hi = __byte_perm(b, 0x64646464u, 0x4342);
    const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&lo), off);
    const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&hi), off);
    x = *reinterpret_cast<const uint32_t*>(&p);
    y = *reinterpret_cast<const uint32_t*>(&q);
  } else {
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}"
        : "=r"(x), "=r"(y)
        : "r"(u));
  }
}
// 16 codes, in order (word i: values 2i and 2i + 1)
template <int CODE>
SRDIT_DEV void widen_codes(uint4 w, uint32_t (&h)[8]) {
  widen4<CODE>(w.x, h[0], h[1]);
  widen4<CODE>(w.y, h[2], h[3]);
  widen4<CODE>(w.z, h[4], h[5]);
  widen4<CODE>(w.w, h[6], h[7]);
}
// whether one of 4 e4m3 codes is NaN
SRDIT_DEV bool nan_codes(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u;
}
// the larger magnitudes' bits of two pairs of 16-bit floats
SRDIT_DEV uint32_t max_bits(uint32_t m, uint32_t w) { return __vmaxu2(m, w & 0x7fff7fffu); }
// whether one of a pair of magnitudes is an infinity or NaN
template <typename T>
SRDIT_DEV bool not_finite(uint32_t m) {
  constexpr uint32_t top = __is_same(T, __half) ? 0x7c00u : 0x7f80u;
  return (m & 0xffffu) >= top || (m >> 16) >= top;
}

// bf16 rows as fp16: times 2^k, by which the row's largest magnitude (its bits) lies in [2^14,
// 2^15). What falls below fp16 then is 2^-29 of the largest or less. A row with an infinity or a
// NaN keeps its size.
SRDIT_DEV int fp16_exponent(uint32_t max_bf16) {
  const int e = static_cast<int>(max_bf16 >> 7);
  return e == 255 ? 0 : min(141 - e, 120);
}
SRDIT_DEV float exp2_int(int k) { return __int_as_float((k + 127) << 23); }
SRDIT_DEV uint32_t bf16x2_as_fp16(uint32_t w, float f) {
  const float2 v = f2_split(bf2_unpack(w));
  return pack2(v.x * f, v.y * f, __half{});
}

// A tensor map over pages of keys or values, or packed ones as one page: boxes of `rows` keys
// of one head. Extents of one entry may have any stride.
inline int key_map(CUtensorMap* m, const srdit_seq_attn_args& u, bool v, int cols, int rows) {
  const bool paged = u.pages != nullptr;
  const srdit_kv_pages* p = u.pages;
  const bool codes = paged && p->code != SRDIT_KV_PLAIN;
  const void* base = paged ? (v ? p->v : p->k) : (v ? u.v : u.k);
  long long n[3] = {paged ? p->pages : 1, paged ? p->page_size : u.Tk, u.Hkv};
  const long long* s3 = paged ? (v ? p->v_stride : p->k_stride) : nullptr;
  const long long* s2 = v ? u.v_stride : u.k_stride;
  long long st[3] = {s3 ? s3[0] : 0, s3 ? s3[1] : s2[0], s3 ? s3[2] : s2[1]};
  if (n[0] == 0 || n[1] == 0) {  // nothing is loaded; the map only has to be valid
    base = u.q;
    n[0] = n[1] = n[2] = 1;
  }
  const int e = codes ? 1 : 2;
  const long long row = (static_cast<long long>(u.D) * e + 15) / 16 * 16;
  for (int i = 0; i < 3; ++i) {
    if (st[i] == 0) n[i] = 1;  // one entry for all
    st[i] = n[i] > 1 ? st[i] * e : row;
  }
  const long long dims[4] = {u.D, n[2], n[1], n[0]};
  const long long strides[3] = {st[2], st[1], st[0]};
  const int box[4] = {cols, 1, rows, 1};
  return make_tmap_4d(m, base, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                      e, dims, strides, box);
}

}  // namespace sattn
}  // namespace srdit
