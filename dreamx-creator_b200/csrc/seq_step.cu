// seq_step.cu -- attention of a few query rows per key head (single tokens of a serving step)
// over the pages of a cache: bounded by the bytes of keys and values.
//
// mma.sync m16n8k16 with the keys as its rows, S^T = K Q^T and O^T = V^T P^T: the query rows of
// one key head (tokens x grouped heads) are the columns, NT times 8 of them. A warp takes blocks
// of 16 keys, which lie in one page, through a ring of its own that TMA boxes fill. The
// contraction over the head's dims may run in any order, so thread c of a quad holds dims 16c to
// 16c + 15 of each 64 for both operands (16-byte loads), and O's rows may be numbered in any
// order, so a lane group holds value columns that lie together.
//
// Codes are widened to fp16 in registers, which is exact; a key's scale multiplies its scores, a
// value's scale its weights, both in fp32, so the only rounding is the weights' to fp16. The
// weights' running maximum is that of score + log2(largest scale of the block's values): weight
// times scale stays at 1 or below, whatever size the scales have, and the sum l is of weights in the
// same unit.
#include <atomic>

#include "seq_attn.cuh"

namespace srdit {
namespace sattn {

constexpr int WARPS = 4;

template <int DP, int NT, int CODE>
struct StepCfg {
  static constexpr bool CODES = CODE != SRDIT_KV_PLAIN;
  static constexpr int PER_SM = NT == 1 ? 3 : 2;
  static constexpr int NC = DP / 32;                  // 8-value pieces of a row of q and k
  static constexpr int NV = DP / 64;                  // 64-column pieces of v
  static constexpr int SLAB = 16 * 128;               // 16 rows of 128 bytes, swizzled
  static constexpr int SLABS = CODES ? 1 : DP / 64;   // of 16 keys
  static constexpr int BLK = 2 * SLABS * SLAB;        // a block: k, then v
  static constexpr int STAGES = 6 / PER_SM * 8192 / BLK;
  static constexpr int RING = WARPS * STAGES * BLK;
  // after the keys: each warp's O [8 NT][DP + 4], then the CTA's, over the ring
  static constexpr int SMEM = RING + 1024;
  static_assert(RING >= (WARPS + 1) * 8 * NT * (DP + 4) * 4, "O fits the ring");
};

SRDIT_DEV void cp_async4(uint32_t dst, const float* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src),
               "r"(on ? 4 : 0)
               : "memory");
}
// an arrival of this thread (of those that the barrier counts) when its copies have landed
SRDIT_DEV void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// blockIdx.x: part of the keys, blockIdx.y: (sequence, key head). The parts of a row that run
// as one cluster are joined in its shared memory.
template <typename T, int DP, int NT, int CODE>
__global__ void __launch_bounds__(WARPS * 32, StepCfg<DP, NT, CODE>::PER_SM)
    step_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ Args a, int cluster) {
  pdl_begin();
  using C = StepCfg<DP, NT, CODE>;
  using E = typename Compute<T, CODE>::type;
  constexpr int NC = C::NC, NV = C::NV, STAGES = C::STAGES, R = 8 * NT;
  constexpr bool CODES = C::CODES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float(*so)[R][DP + 4] = reinterpret_cast<float(*)[R][DP + 4]>(ring);
  float(*co)[DP + 4] = so[WARPS];   // the CTA's own part
  __shared__ float2 sml[WARPS][R];  // {m, l} of each warp
  __shared__ float2 cml[R];
  __shared__ uint64_t bars[WARPS][STAGES];
  __shared__ float sc[CODES ? WARPS : 1][CODES ? STAGES : 1][32];  // scales: 16 keys', 16 values'
  if (cluster > 1) cluster_arrive();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int part = blockIdx.x;
  // sequences of different lengths side by side, so that an SM gets some of each
  const int b = blockIdx.y % a.B, kvh = blockIdx.y / a.B;
  const int row0 = a.rows.begin(b), n_all = a.rows.end(b) - row0;
  const int rows = min(n_all, a.max_q) * a.group;
  const int len = rows > 0 ? a.key_count(b) : 0;
  const int first = len - n_all;  // the first query's token
  const int nblk = (len + 15) / 16;
  const int blk0 = static_cast<int>(static_cast<long long>(nblk) * part / a.splits);
  const int blk1 = static_cast<int>(static_cast<long long>(nblk) * (part + 1) / a.splits);

  uint64_t* full = bars[warp];
  if (lane == 0) {
    if (warp == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    for (int x = 0; x < STAGES; ++x) mbar_init(&full[x], CODES ? 33 : 1);
    fence_barrier_init();
  }
  __syncwarp();
  uint8_t* mine = ring + warp * STAGES * C::BLK;
  // pages of this warp's next blocks, a lane one, read 32 blocks ahead
  auto pages_at = [&](int n) {
    const int blk = blk0 + warp + (n + lane) * WARPS;
    return blk < blk1 ? a.table.page(b, a.table.by_page.div(blk * 16)) : -1;
  };
  int page_now = -1, page_next = pages_at(0);
  int fetched = 0;
  uint32_t there = 0;  // slots whose page is one
  auto fetch = [&](int slot) {
    if ((fetched & 31) == 0) {
      page_now = page_next;
      page_next = pages_at(fetched + 32);
    }
    const int page = __shfl_sync(0xffffffffu, page_now, fetched & 31);
    const int blk = blk0 + warp + fetched * WARPS;
    ++fetched;
    if (blk >= blk1) return;
    there = page >= 0 ? there | 1u << slot : there & ~(1u << slot);
    const int row = blk * 16 - a.table.by_page.div(blk * 16) * a.table.page_size;
    if (lane == 0) {
      uint8_t* dst = mine + slot * C::BLK;
      const int at = page >= 0 ? page : max(a.table.pages, 1);  // (past the pages: zeros)
      mbar_arrive_expect_tx(&full[slot], C::BLK);
#pragma unroll
      for (int x = 0; x < C::SLABS; ++x) {
        tma_load_4d(dst + x * C::SLAB, &tmK, &full[slot], x * 64, kvh, row, at);
        tma_load_4d(dst + (C::SLABS + x) * C::SLAB, &tmV, &full[slot], x * 64, kvh, row, at);
      }
    }
    if constexpr (CODES) {
      const int side = lane >> 4, key = lane & 15;
      const bool on = page >= 0 && blk * 16 + key < len;
      const float* src = a.scale[side];
      if (on) src += page * a.ss[side][0] + (row + key) * a.ss[side][1] + kvh * a.ss[side][2];
      cp_async4(smem_u32(&sc[warp][slot][lane]), src, on);
      cp_async_arrive(&full[slot]);
    }
  };
#pragma unroll
  for (int x = 0; x < STAGES; ++x) fetch(x);
  __syncwarp();
  // column r: token r / group, head kvh * group + r % group
  uint4 qf[NT][NC];
  float cq[NT][2];  // scale * log2(e) over the query's own factor, of columns 2c and 2c + 1
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = g + 8 * n, tok = a.by_group.div(r);
    const T* qp = static_cast<const T*>(a.q) + (row0 + tok) * a.qs[0] +
                  (static_cast<long long>(kvh) * a.group + r - tok * a.group) * a.qs[1];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      const int d = (x >> 1) * 64 + c * 16 + (x & 1) * 8;
      qf[n][x] = r < rows && d < a.D ? *reinterpret_cast<const uint4*>(qp + d)
                                     : make_uint4(0, 0, 0, 0);
    }
    cq[n][0] = cq[n][1] = a.c;
    if constexpr (CODES && !__is_same(T, __half)) {
      uint32_t m = 0;
#pragma unroll
      for (int x = 0; x < NC; ++x)
        m = max_bits(max_bits(max_bits(max_bits(m, qf[n][x].x), qf[n][x].y), qf[n][x].z),
                     qf[n][x].w);
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
      const int k = fp16_exponent(max(m & 0xffffu, m >> 16));
      const float f = exp2_int(k), back = a.c * exp2_int(-k);
#pragma unroll
      for (int x = 0; x < NC; ++x)
        qf[n][x] = make_uint4(bf16x2_as_fp16(qf[n][x].x, f), bf16x2_as_fp16(qf[n][x].y, f),
                              bf16x2_as_fp16(qf[n][x].z, f), bf16x2_as_fp16(qf[n][x].w, f));
      cq[n][0] = __shfl_sync(0xffffffffu, back, 8 * c);
      cq[n][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
    }
  }
  // the last key that columns 2c and 2c + 1 see
  int lim[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      lim[n][e] = a.causal ? first + a.by_group.div(8 * n + 2 * c + e) : len;
  float o[NT][NV * 4][4];
  // of columns 2c and 2c + 1, in every lane group; l: this lane's keys only
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int x = 0; x < NV * 4; ++x)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][x][e] = 0.f;
    m[n][0] = m[n][1] = neg_inf();
    l[n][0] = l[n][1] = 0.f;
  }

  // a lane's pieces of a swizzled slab: k row g, v rows 2c and 2c + 1
  const uint32_t k_at = static_cast<uint32_t>(g * 128 + (((CODES ? c : 2 * c) ^ g) << 4));
  const uint32_t vg = CODES && DP == 64 ? g >> 1 : g;
  const uint32_t v_low = CODES && DP == 64 ? (g & 1) * 8u : 0u;
  const uint32_t v_at = static_cast<uint32_t>(2 * c * 128 + ((vg ^ (2 * c)) << 4)) + v_low;
  const uint32_t v_at1 =
      static_cast<uint32_t>((2 * c + 1) * 128 + ((vg ^ (2 * c + 1)) << 4)) + v_low;
  int slot = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (int blk = blk0 + warp; blk < blk1; blk += WARPS) {
    const int key0 = blk * 16;
    const bool ok_page = (there >> slot) & 1u;
    if (!mbar_wait_warp(&full[slot], phase, a.status)) {
      // having given up, let the loads in flight land before the ring is used again
      for (int i = 0; i < 200; ++i) __nanosleep(1000);
      break;
    }
    // k rows g and g + 8; v rows 2c, 2c + 1, 2c + 8, 2c + 9
    const uint32_t src = smem_u32(mine) + static_cast<uint32_t>(slot * C::BLK);
    uint4 kf[2][NC], vf[4][NV];
    float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
    bool nan_code[4] = {false, false, false, false};
    if constexpr (!CODES) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < NC; ++x)
          kf[h][x] = lds16(src + (x >> 1) * C::SLAB + h * 1024 + ((x & 1) ? k_at ^ 16u : k_at));
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int x = 0; x < NV; ++x)
          vf[r][x] = lds16(src + (NV + x) * C::SLAB + (r >> 1) * 1024 + ((r & 1) ? v_at1 : v_at));
    } else {
      uint4 kc[2][NV], vc[4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < NV; ++x)
          kc[h][x] = lds16(src + h * 1024 + (x ? k_at ^ 64u : k_at));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t at = src + C::SLAB + (r >> 1) * 1024 + ((r & 1) ? v_at1 : v_at);
        if constexpr (DP == 128) {
          vc[r] = lds16(at);
        } else {
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(vc[r].x), "=r"(vc[r].y) : "r"(at));
          vc[r].z = vc[r].w = 0u;
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[h] = sc[warp][slot][g + 8 * h];
        vs[h] = sc[warp][slot][16 + g + 8 * h];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < NV; ++x) {
          uint32_t w[8];
          widen_codes<CODE>(kc[h][x], w);
          kf[h][2 * x] = make_uint4(w[0], w[1], w[2], w[3]);
          kf[h][2 * x + 1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (CODE == SRDIT_Q_E4M3) {
          nan_code[r] = nan_codes(vc[r].x) || nan_codes(vc[r].y) || nan_codes(vc[r].z) ||
                        nan_codes(vc[r].w);
          if (nan_code[r]) vc[r] = make_uint4(0, 0, 0, 0);
        }
        uint32_t w[8];
        widen_codes<CODE>(vc[r], w);
        vf[r][0] = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (NV == 2) vf[r][1] = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
    __syncwarp();  // every lane has read the slot
    fetch(slot);
    __syncwarp();
    if (++slot == STAGES) {
      slot = 0;
      phase ^= 1u;
    }
    // keys of the block that the sequence has
    const int have = ok_page ? min(16, len - key0) : 0;
    if (!CODES && have < 16) {  // values of others: zeros
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (2 * c + (r & 1) + (r >> 1) * 8 >= have)
#pragma unroll
          for (int x = 0; x < NV; ++x) vf[r][x] = make_uint4(0, 0, 0, 0);
    }
    const bool hidden = a.causal && key0 + 15 > first;  // from some of the queries
    // Values that are not finite: where some queries do not see them they are taken out, and the
    // queries that do get a NaN; a NaN code is one always.
    uint32_t bad[2] = {0u, 0u};  // keys g and g + 8
    if ((!CODES && hidden && n_all > 1) || CODE == SRDIT_Q_E4M3) {
      uint32_t all[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        bool here = nan_code[r];
        if constexpr (!CODES) {
          uint32_t mx = 0;
#pragma unroll
          for (int x = 0; x < NV; ++x)
            mx = max_bits(max_bits(max_bits(max_bits(mx, vf[r][x].x), vf[r][x].y), vf[r][x].z),
                          vf[r][x].w);
          here = not_finite<E>(mx);
        }
        all[r] = __ballot_sync(0xffffffffu, here);
        if (!CODES && (all[r] & (0x11111111u << c)))
#pragma unroll
          for (int x = 0; x < NV; ++x) vf[r][x] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        bad[h] = ((g & 1) ? all[2 * h + 1] : all[2 * h]) & (0x11111111u << (g >> 1));
    }
    float lv = 0.f;
    if constexpr (CODES) {  // log2 of the block's largest scale of a value
      float top = fmaxf(vs[0] < 3e38f ? vs[0] : 0.f, vs[1] < 3e38f ? vs[1] : 0.f);
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      lv = __log2f(fmaxf(top, 1e-30f));
    }
    uint32_t pf[NT][2];
    bool moved = false;
    float alpha[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // two chains of products, joined at the end
      float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        mma16816<E>(s, kf[0][x].x, kf[1][x].x, kf[0][x].y, kf[1][x].y, qf[n][x].x, qf[n][x].y);
        mma16816<E>(s2, kf[0][x].z, kf[1][x].z, kf[0][x].w, kf[1][x].w, qf[n][x].z, qf[n][x].w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] += s2[e];
        if constexpr (CODES) s[e] *= ks[e >> 1];
      }
      // s[0], s[2]: column 2c, keys g and g + 8; s[1], s[3]: column 2c + 1
      if (have < 16 || hidden) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = g + (e >> 1) * 8;
          if (key >= have || key0 + key > lim[n][e & 1]) s[e] = neg_inf();
        }
      }
      float w[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = max2(s[e], s[2 + e]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = max2(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float mn = max2(m[n][e], fmaf(top, cq[n][e], lv));
        const float neg = mn == neg_inf() ? 0.f : -mn;
        alpha[n][e] = ex2(m[n][e] + neg);
        moved |= mn != m[n][e];
        m[n][e] = mn;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool seen = s[2 * h + e] != neg_inf();
          const float p = ex2(fmaf(s[2 * h + e], cq[n][e], neg));
          s[2 * h + e] = p;
          w[2 * h + e] = !CODES ? p : seen ? p * vs[h] : 0.f;
          if (bad[h] && seen) l[n][e] = __int_as_float(0x7fc00000);
        }
        l[n][e] = fmaf(l[n][e], alpha[n][e], s[e] + s[2 + e]);
      }
      pf[n][0] = transpose8x8(pack2(w[0], w[1], E{}));
      pf[n][1] = transpose8x8(pack2(w[2], w[3], E{}));
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < NV * 4; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][x][e] *= alpha[n][e & 1];
    }
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      const uint32_t r0[4] = {vf[0][x].x, vf[0][x].y, vf[0][x].z, vf[0][x].w};
      const uint32_t r1[4] = {vf[1][x].x, vf[1][x].y, vf[1][x].z, vf[1][x].w};
      const uint32_t r2[4] = {vf[2][x].x, vf[2][x].y, vf[2][x].z, vf[2][x].w};
      const uint32_t r3[4] = {vf[3][x].x, vf[3][x].y, vf[3][x].z, vf[3][x].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // the lane group's columns 2w (operand row g) and 2w + 1 (row g + 8)
        const uint32_t a0 = __byte_perm(r0[w], r1[w], 0x5410);
        const uint32_t a1 = __byte_perm(r0[w], r1[w], 0x7632);
        const uint32_t a2 = __byte_perm(r2[w], r3[w], 0x5410);
        const uint32_t a3 = __byte_perm(r2[w], r3[w], 0x7632);
#pragma unroll
        for (int n = 0; n < NT; ++n)
          mma16816<E>(o[n][x * 4 + w], a0, a1, a2, a3, pf[n][0], pf[n][1]);
      }
    }
  }
  // every warp is done with its ring; O takes its place
  __syncthreads();
  // this warp's part: o[n][x * 4 + w][e] is query column 8n + 2c + (e & 1) and the lane group's
  // value column 2w + (e >> 1) of its x-th eight
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
      const int row = 8 * n + 2 * c + e;
      if (g == 0) sml[warp][row] = make_float2(m[n][e], l[n][e]);
      if (row < rows) {
#pragma unroll
        for (int x = 0; x < NV * 4; ++x) {
          const int col = CODES && DP == 128 ? g * 16 + (x >> 2) * 8 : (x >> 2) * 64 + g * 8;
          *reinterpret_cast<float2*>(&so[warp][row][col + (x & 3) * 2]) =
              make_float2(o[n][x][e], o[n][x][2 + e]);
        }
      }
    }
  }
  __syncthreads();
  // the CTA's part, four columns a thread
  constexpr int DQ = DP / 4;
  for (int x = threadIdx.x; x < rows * DQ; x += WARPS * 32) {
    const int row = x / DQ, d = x % DQ * 4;
    float top = neg_inf();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = max2(top, sml[w][row].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (top != neg_inf()) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float2 ml = sml[w][row];
        const float f = ex2(ml.x - top);
        const float4 v = *reinterpret_cast<const float4*>(&so[w][row][d]);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
        sum = fmaf(ml.y, f, sum);
      }
    }
    *reinterpret_cast<float4*>(&co[row][d]) = acc;
    if (d == 0) cml[row] = make_float2(top, sum);
  }
  int share = 0, shares = 1;
  if (cluster > 1) {
    cluster_wait();  // the arrival at the start: every CTA of the cluster runs
    cluster_arrive();
    cluster_wait();  // every part is in its CTA's shared memory
    share = static_cast<int>(cluster_ctarank());
    shares = cluster;
  } else {
    __syncthreads();
  }
  // CTA `share` of the cluster joins every shares-th four columns of the parts
  const long long all_rows = static_cast<long long>(a.T) * a.H;
  const int wparts = a.splits / cluster;
  const int dq = a.D / 4;
  for (int x = threadIdx.x * shares + share; x < rows * dq; x += WARPS * 32 * shares) {
    const int row = x / dq, d = (x - row * dq) * 4;
    float top = neg_inf(), sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (cluster > 1) {
      const uint32_t ml0 = smem_u32(&cml[row]), o0 = smem_u32(&co[row][d]);
      float pm[8], pl[8];
      float4 po[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        pm[s] = neg_inf();
        pl[s] = 0.f;
        po[s] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < cluster) {
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                       : "=f"(pm[s]), "=f"(pl[s])
                       : "r"(mapa_shared(ml0, s)));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(po[s].x), "=f"(po[s].y), "=f"(po[s].z), "=f"(po[s].w)
                       : "r"(mapa_shared(o0, s)));
        }
        top = max2(top, pm[s]);
      }
      if (top != neg_inf()) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const float f = ex2(pm[s] - top);
          acc.x = fmaf(po[s].x, f, acc.x);
          acc.y = fmaf(po[s].y, f, acc.y);
          acc.z = fmaf(po[s].z, f, acc.z);
          acc.w = fmaf(po[s].w, f, acc.w);
          sum = fmaf(pl[s], f, sum);
        }
      }
    } else {
      top = cml[row].x;
      sum = cml[row].y;
      acc = *reinterpret_cast<const float4*>(&co[row][d]);
    }
    const int i = a.by_group.div(row);
    const long long tok = row0 + i;
    const int head = kvh * a.group + row - i * a.group;
    if (wparts == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + tok * a.os[0] + head * a.os[1] + d) =
          make_uint2(pack2(acc.x * inv, acc.y * inv, T{}), pack2(acc.z * inv, acc.w * inv, T{}));
    } else {
      const long long at = (part / cluster) * all_rows + tok * a.H + head;
      *reinterpret_cast<float4*>(a.ws + at * a.D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(a.ml + at * 2) = make_float2(top, sum);
    }
  }
  if (cluster > 1) {  // no CTA leaves while another reads its shared memory
    cluster_arrive();
    cluster_wait();
  }
}

// One warp per (token, head): joins the parts that went through the workspace, four parts'
// loads in flight.
template <typename T>
__global__ void __launch_bounds__(128) join_step_kernel(const __grid_constant__ Args a, int parts) {
  pdl_begin();
  const long long rows = static_cast<long long>(a.T) * a.H;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int lane = threadIdx.x & 31;
  const int t = static_cast<int>(row / a.H), h = static_cast<int>(row - static_cast<long long>(t) * a.H);
  const int b = find_sequence(a.rows, a.B, t, a.by_each);
  if (b >= a.B || t - a.rows.begin(b) >= a.max_q) return;
  const float2* ml = reinterpret_cast<const float2*>(a.ml);
  float m = neg_inf(), l = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const bool on = lane * 4 < a.D;
  for (int p0 = 0; p0 < parts; p0 += 4) {
    float2 pm[4];
    float4 v[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      pm[x] = make_float2(neg_inf(), 0.f);
      v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p0 + x < parts) {
        const long long at = (p0 + x) * rows + row;
        pm[x] = ml[at];
        if (on) v[x] = *reinterpret_cast<const float4*>(a.ws + at * a.D + lane * 4);
      }
    }
    float mn = m;
#pragma unroll
    for (int x = 0; x < 4; ++x) mn = max2(mn, pm[x].x);
    if (mn == neg_inf()) continue;  // no key seen yet
    const float f = ex2(m - mn);
    m = mn;
    l *= f;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (pm[x].x == neg_inf()) continue;  // a part that saw no key
      const float k = ex2(pm[x].x - m);
      l = fmaf(pm[x].y, k, l);
      acc[0] = fmaf(v[x].x, k, acc[0]);
      acc[1] = fmaf(v[x].y, k, acc[1]);
      acc[2] = fmaf(v[x].z, k, acc[2]);
      acc[3] = fmaf(v[x].w, k, acc[3]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (on)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + t * a.os[0] + h * a.os[1] + lane * 4) =
        make_uint2(pack2(acc[0] * inv, acc[1] * inv, T{}), pack2(acc[2] * inv, acc[3] * inv, T{}));
}

// ---------------------------------------------------------------- launch
Plan plan_step(const srdit_seq_attn_args& u, int sms) {
  Plan p = {};
  p.step = true;
  const int group = u.H / u.Hkv;
  const long long pairs = static_cast<long long>(u.B) * u.Hkv;
  const int per_sm = u.max_q * group <= 8 ? 3 : 2;
  const long long held = static_cast<long long>(u.pages->table_width) * u.pages->page_size;
  const long long keys = u.max_kv > 0 && u.max_kv < held ? u.max_kv : held;
  const long long blocks = (keys + 15) / 16;
  // The keys are split until every SM has its CTAs, each with a block per warp at least, within a
  // cluster; more than a cluster's 8 parts go through the workspace, from 8 blocks a warp.
  const long long most = (blocks + WARPS - 1) / WARPS;
  p.cluster = p.parts = 1;
  while (p.cluster < 8 && 2 * p.cluster <= most &&
         (pairs * p.cluster < sms || 2 * pairs * p.cluster <= per_sm * sms))
    p.cluster *= 2;
  p.splits = p.cluster;
  const int warps = 8 * WARPS;
  if (p.cluster == 8 && blocks >= 8 * warps) {
    long long parts = (sms + 5 * pairs / 2) / (5 * pairs);
    if (parts > blocks / (4 * warps)) parts = blocks / (4 * warps);
    p.parts = parts < 1 ? 1 : static_cast<int>(parts);
    p.splits = 8 * p.parts;
  }
  p.ws_floats = p.parts > 1 ? static_cast<long long>(p.parts) * u.T * u.H * (u.D + 2) : 0;
  return p;
}

template <typename T, int DP, int NT, int CODE>
static int launch(const srdit_seq_attn_args& u, const Args& a, const Plan& p, cudaStream_t stream) {
  using C = StepCfg<DP, NT, CODE>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  int rc = set_smem(step_kernel<T, DP, NT, CODE>, C::SMEM, attr_done);
  if (rc) return rc;
  CUtensorMap tk, tv;
  const int cols = C::CODES ? 128 : 64;
  rc = key_map(&tk, u, false, cols, 16);
  if (!rc) rc = key_map(&tv, u, true, cols, 16);
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.B * a.Hkv));
  return launch_clusters(p.cluster, step_kernel<T, DP, NT, CODE>, grid, WARPS * 32, C::SMEM, stream,
                         tk, tv, a, p.cluster);
}

template <typename T, int CODE>
static int launch_size(const srdit_seq_attn_args& u, const Args& a, const Plan& p,
                       cudaStream_t stream) {
  const bool one = u.max_q * a.group <= 8;
  if (u.D <= 64)
    return one ? launch<T, 64, 1, CODE>(u, a, p, stream) : launch<T, 64, 2, CODE>(u, a, p, stream);
  return one ? launch<T, 128, 1, CODE>(u, a, p, stream) : launch<T, 128, 2, CODE>(u, a, p, stream);
}

template <typename T>
static int run_typed(const srdit_seq_attn_args& u, const Args& a, const Plan& p,
                     cudaStream_t stream) {
  int rc;
  switch (u.pages->code) {
    case SRDIT_Q_INT8: rc = launch_size<T, SRDIT_Q_INT8>(u, a, p, stream); break;
    case SRDIT_Q_E4M3: rc = launch_size<T, SRDIT_Q_E4M3>(u, a, p, stream); break;
    default: rc = launch_size<T, SRDIT_KV_PLAIN>(u, a, p, stream);
  }
  if (rc || p.parts == 1) return rc;
  const long long rows = static_cast<long long>(u.T) * u.H;
  SRDIT_LAUNCH((join_step_kernel<T>), static_cast<unsigned>((rows + 3) / 4), 128, 0, stream, a,
               p.parts);
  return static_cast<int>(cudaGetLastError());
}

int run_step(const srdit_seq_attn_args& u, Args& a, const Plan& p, cudaStream_t stream) {
  a.splits = p.splits;
  a.by_group = Divisor::of(a.group);
  a.ml = a.ws + static_cast<long long>(p.parts) * u.T * u.H * u.D;
  return u.dtype == SRDIT_BF16 ? run_typed<__nv_bfloat16>(u, a, p, stream)
                               : run_typed<__half>(u, a, p, stream);
}

}  // namespace sattn
}  // namespace srdit
