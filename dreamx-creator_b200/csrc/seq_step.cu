// seq_step.cu -- attention of a few query rows per key head (single tokens of a serving step)
// over the pages of a cache: bounded by the bytes of keys and values.
//
// mma.sync m16n8k16 with the keys as its rows, S^T = K Q^T and O^T = V^T P^T: the query rows of
// one key head (tokens x grouped heads) are the columns, NT times 8 of them. A warp takes blocks
// of 16 keys, or 32 of codes, through a ring of its own that TMA boxes fill, a box or more a page.
// A block goes to registers whole, and its slot is refilled before the block is computed. The
// contraction over the head's dims may run in any order, so thread c of a quad holds dims 16c to
// 16c + 15 of each 64 for both operands (16-byte loads), and O's rows may be numbered in any
// order, so a lane group holds value columns that lie together.
//
// Codes are widened to fp16 in registers, which is exact; a key's scale multiplies its scores, a
// value's scale its weights, both in fp32, so the only rounding is the weights' to fp16. The
// weights' running maximum m is that of score + e, where e is the exponent of the value's scale:
// weight times scale stays below 2, and some are near 1, whatever size the scales have, those of keys
// that are hidden among them. The sum l is of 2^(score - m + 24): with e from -80 (and scales below it
// lose digits) to 125 it is in range, and a weight is lost from it when it is 2^-25 of the largest, of
// scales up to kv_write's 2^121 2^-29. (From weights times 2^-e it would be lost where another's
// scale is 2^126 times its own.) What takes l from one maximum to the next, 2^(m - m'), may be out of
// range, and is taken in two halves.
//
// The keys are split in one of two ways. Little work: every (sequence, key head) over a cluster of
// up to 8 CTAs, which join their parts in shared memory. Much: two CTAs on every SM (three over
// codes) take equal shares of all blocks, whatever the sequences' lengths, and join_share_kernel
// joins what the shares cut. 32 sequences of up to 4096 keys, 32 heads over 8 of 128, bf16: 52 us,
// 5.2 TB/s; 8 of 32768 169 us, 6.4 TB/s, in e4m3 107, 5.2 TB/s, in int8 107 to 116, where widening the
// codes takes 46% of the issue slots.
#include <atomic>

#include "seq_attn.cuh"

namespace srdit {
namespace sattn {

constexpr int WARPS = 4;
constexpr int MAX_SHARED = 1024;  // sequences of a launch by shares
constexpr int MIN_BLOCKS = 8;     // blocks of a share, at least
constexpr int SHARE_BLOCKS = 64;  // ... of a CTA, from which shares are taken
constexpr int LEAST = -80, MOST = 125;  // exponents of values' scales

template <int DP, int NT, int CODE>
struct StepCfg {
  static constexpr bool CODES = CODE != SRDIT_KV_PLAIN;
  static constexpr int PER_SM = NT == 1 ? 3 : 2;
  static constexpr int KB = CODES ? 32 : 16;          // keys of a block
  static constexpr int NB = KB / 16;
  static constexpr int NC = DP / 32;                  // 8-value pieces of a row of q and k
  static constexpr int NV = DP / 64;                  // 64-column pieces of v
  static constexpr int SLAB = KB * 128;               // KB rows of 128 bytes, swizzled
  static constexpr int SLABS = CODES ? 1 : DP / 64;
  static constexpr int BLK = 2 * SLABS * SLAB;        // a block: k, then v
  static constexpr int STAGES = 6 / PER_SM * 8192 / BLK;
  static constexpr int RING = WARPS * STAGES * BLK;
  // after the keys: each warp's O [8 NT][DP + 4], then the CTA's, over the ring
  static constexpr int SMEM = RING + 1024;
  static_assert(RING >= (WARPS + 1) * 8 * NT * (DP + 4) * 4, "O fits the ring");
};

// What a CTA leaves for join_share_kernel: the (sequence, key head) that it begins and does not
// end.
struct StepCut {
  int parts, b, kvh, pad;
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

template <typename T, int DP, int NT, int CODE>
__global__ void __launch_bounds__(WARPS * 32, StepCfg<DP, NT, CODE>::PER_SM)
    step_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ Args a, int cluster) {
  pdl_begin();
  using C = StepCfg<DP, NT, CODE>;
  using E = typename Compute<T, CODE>::type;
  constexpr int NC = C::NC, NV = C::NV, NB = C::NB, KB = C::KB, STAGES = C::STAGES, R = 8 * NT;
  constexpr bool CODES = C::CODES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float(*so)[R][DP + 4] = reinterpret_cast<float(*)[R][DP + 4]>(ring);
  float(*co)[DP + 4] = so[WARPS];   // the CTA's own part
  __shared__ float2 sml[WARPS][R];  // {m, l} of each warp
  __shared__ float2 cml[R];
  __shared__ uint64_t bars[WARPS][STAGES];
  __shared__ float sc[CODES ? WARPS : 1][CODES ? STAGES : 1][2 * KB];  // scales: keys', values'
  __shared__ int before[MAX_SHARED + 1];  // shares: blocks of the sequences before one
  __shared__ int sums[WARPS];
  if (cluster > 1) cluster_arrive();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
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
  uint32_t phases = 0;  // of the ring's slots

  // What this CTA does: (sequence, key head) pairs and blocks of their keys.
  auto blocks_of = [&](int b) {
    const int from = a.rows.begin(b), to = a.rows.end(b), n = max(1, (a.key_count(b) + KB - 1) / KB);
    return to > from ? n : 0;
  };
  int s = 0, s1 = 1, share = 1, b = 0, kvh = 0;
  if (a.shared) {
    const int each = (a.B + WARPS * 32 - 1) / (WARPS * 32);
    const int b0 = min(static_cast<int>(threadIdx.x) * each, a.B), b1 = min(b0 + each, a.B);
    int sum = 0;
    for (int x = b0; x < b1; ++x) {
      const int w = blocks_of(x);
      before[x] = sum;
      sum += w;
    }
    int up = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += y;
    }
    if (lane == 31) sums[warp] = up;
    __syncthreads();
    int base = up - sum;
    for (int w = 0; w < warp; ++w) base += sums[w];
    for (int x = b0; x < b1; ++x) before[x] += base;
    if (threadIdx.x == WARPS * 32 - 1) before[a.B] = base + sum;
    __syncthreads();
    // the same blocks for every key head at the same time: their rows lie side by side
    const int total = before[a.B], groups = static_cast<int>(gridDim.x) / a.Hkv;
    const int group = static_cast<int>(blockIdx.x) / a.Hkv;
    kvh = static_cast<int>(blockIdx.x) - group * a.Hkv;
    share = max((total + groups - 1) / groups, MIN_BLOCKS);
    s = min(group * share, total);
    s1 = min(s + share, total);
    if (threadIdx.x == 0) static_cast<StepCut*>(a.cuts)[blockIdx.x].parts = 0;
  } else {
    // sequences of different lengths side by side, so that an SM gets some of each
    b = blockIdx.y % a.B;
    kvh = blockIdx.y / a.B;
  }
  // (The body of this loop, to the end of the kernel but for its last lines, is not indented.)
#pragma unroll 1
  while (s < s1) {
  int blk0, blk1, part = 0, slot_of_part = -1;
  if (a.shared) {
    int lo = 0, hi = a.B;  // the sequence that block s is of
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= s) lo = mid; else hi = mid;
    }
    b = lo;
    const int w = before[b + 1] - before[b];
    blk0 = s - before[b];
    blk1 = min(w, blk0 + (s1 - s));
    const int cta = static_cast<int>(blockIdx.x);
    if (blk0 > 0 || blk1 < w) slot_of_part = blk0 > 0 ? 2 * cta : 2 * cta + 1;
    if (blk0 == 0 && blk1 < w && threadIdx.x == 0) {
      const StepCut cut = {(s + w - 1) / share - s / share + 1, b, kvh, 0};
      static_cast<StepCut*>(a.cuts)[cta] = cut;
    }
    s += blk1 - blk0;
  } else {
    s = s1;
    part = blockIdx.x;
    blk0 = blk1 = 0;
  }
  const int row0 = a.rows.begin(b), n_all = a.rows.end(b) - row0;
  const int rows = min(n_all, a.max_q) * a.group;
  const int len = rows > 0 ? a.key_count(b) : 0;
  const int first = len - n_all;  // the first query's token
  const int nblk = (len + KB - 1) / KB;
  if (!a.shared) {
    blk0 = static_cast<int>(static_cast<long long>(nblk) * part / a.splits);
    blk1 = static_cast<int>(static_cast<long long>(nblk) * (part + 1) / a.splits);
  }
  blk1 = min(blk1, nblk);

  // Pages of this warp's next blocks, a lane one, read 32 blocks ahead (pages of 16 keys and
  // blocks of 32: 16 blocks, two lanes one).
  const int pages_log = NB == 2 && a.table.page_size == 16 ? 1 : 0;
  auto pages_at = [&](int n) {
    const int blk = blk0 + warp + (n + (lane >> pages_log)) * WARPS;
    const int key = blk * KB + (pages_log ? (lane & 1) * 16 : 0);
    return blk < blk1 && key < len ? a.table.page(b, a.table.by_page.div(key)) : -1;
  };
  int page_now = -1, page_next = pages_at(0);
  int fetched = 0;
  uint32_t there = 0;  // two bits a slot: whether the halves' pages are ones
  const float* k_scale = CODES ? a.scale[0] + kvh * a.ss[0][2] : nullptr;
  const float* v_scale = CODES ? a.scale[1] + kvh * a.ss[1][2] : nullptr;
  auto fetch = [&](int slot) {
    const int in = fetched & ((32 >> pages_log) - 1);
    if (in == 0) {
      page_now = page_next;
      page_next = pages_at(fetched + (32 >> pages_log));
    }
    int page[NB];
    page[0] = __shfl_sync(0xffffffffu, page_now, in << pages_log);
    if constexpr (NB == 2)
      page[1] = __shfl_sync(0xffffffffu, page_now, (in << pages_log) + pages_log);
    const int blk = blk0 + warp + fetched * WARPS;
    ++fetched;
    if (blk >= blk1) return;
    uint32_t here = 0;
#pragma unroll
    for (int x = 0; x < NB; ++x) here |= page[x] >= 0 ? 1u << x : 0u;
    there = (there & ~(3u << (2 * slot))) | here << (2 * slot);
    const int row = blk * KB - a.table.by_page.div(blk * KB) * a.table.page_size;
    if (lane == 0) {
      uint8_t* dst = mine + slot * C::BLK;
      mbar_arrive_expect_tx(&full[slot], C::BLK);
#pragma unroll
      for (int y = 0; y < NB; ++y) {
        if (y > pages_log) break;
        const int at = page[y] >= 0 ? page[y] : max(a.table.pages, 1);  // (past the pages: zeros)
#pragma unroll
        for (int x = 0; x < C::SLABS; ++x) {
          tma_load_4d(dst + x * C::SLAB + y * 2048, &tmK, &full[slot], x * 64, kvh, row, at);
          tma_load_4d(dst + (C::SLABS + x) * C::SLAB + y * 2048, &tmV, &full[slot], x * 64, kvh,
                      row, at);
        }
      }
    }
    if constexpr (CODES) {
      const int half = (lane >> 4) & pages_log, p = half ? page[NB - 1] : page[0];
      const bool on = p >= 0 && blk * KB + lane < len;
      const long long in_page = row + lane - half * 16;
      const float* k = a.scale[0];
      const float* v = a.scale[1];
      if (on) {
        k = k_scale + (p * a.ss[0][0] + in_page * a.ss[0][1]);
        v = v_scale + (p * a.ss[1][0] + in_page * a.ss[1][1]);
      }
      cp_async4(smem_u32(&sc[warp][slot][lane]), k, on);
      cp_async4(smem_u32(&sc[warp][slot][KB + lane]), v, on);
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
      const float f = exp2_int(k), back = fmaxf(a.c * exp2_int(-k), 1.2e-38f);  // (0 times -inf is NaN)
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

  // a lane's pieces of a swizzled slab: k row g, v rows 2c and 2c + 1 (of 8)
  const uint32_t k_at = static_cast<uint32_t>(g * 128 + (((CODES ? c : 2 * c) ^ g) << 4));
  const uint32_t vg = CODES && DP == 64 ? g >> 1 : g;
  const uint32_t v_low = CODES && DP == 64 ? (g & 1) * 8u : 0u;
  const uint32_t v_at = static_cast<uint32_t>(2 * c * 128 + ((vg ^ (2 * c)) << 4)) + v_low;
  const uint32_t v_at1 =
      static_cast<uint32_t>((2 * c + 1) * 128 + ((vg ^ (2 * c + 1)) << 4)) + v_low;
  int slot = 0;
#pragma unroll 1
  for (int blk = blk0 + warp; blk < blk1; blk += WARPS) {
    const int key0 = blk * KB;
    const uint32_t ok_pages = (there >> (2 * slot)) & 3u;
    if (!mbar_wait_warp(&full[slot], (phases >> slot) & 1u, a.status)) {
      // having given up, let the loads in flight land before the ring is used again
      for (int i = 0; i < 200; ++i) __nanosleep(1000);
      break;
    }
    phases ^= 1u << slot;
    // per 16 keys: k rows g and g + 8; v rows 2c, 2c + 1, 2c + 8, 2c + 9
    const uint32_t src = smem_u32(mine) + static_cast<uint32_t>(slot * C::BLK);
    // 16 bits: rows' pieces as the products take them; codes: 16 bytes of codes each
    constexpr int KP = CODES ? NV : NC, VP = CODES ? 1 : NV;
    uint4 kr[NB][2][KP], vr[NB][4][VP];
    float ks[NB][2], vs[NB][2];
#pragma unroll
    for (int y = 0; y < NB; ++y) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < KP; ++x)
          kr[y][h][x] =
              CODES ? lds16(src + y * 2048 + h * 1024 + (x ? k_at ^ 64u : k_at))
                    : lds16(src + (x >> 1) * C::SLAB + h * 1024 + ((x & 1) ? k_at ^ 16u : k_at));
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int x = 0; x < VP; ++x) {
          const uint32_t at = src + (C::SLABS + x) * C::SLAB + y * 2048 + (r >> 1) * 1024 +
                              ((r & 1) ? v_at1 : v_at);
          if constexpr (CODES && DP == 64) {
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];"
                         : "=r"(vr[y][r][x].x), "=r"(vr[y][r][x].y)
                         : "r"(at));
            vr[y][r][x].z = vr[y][r][x].w = 0u;
          } else {
            vr[y][r][x] = lds16(at);
          }
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ks[y][h] = CODES ? sc[CODES ? warp : 0][CODES ? slot : 0][y * 16 + g + 8 * h] : 1.f;
        vs[y][h] = CODES ? sc[CODES ? warp : 0][CODES ? slot : 0][KB + y * 16 + g + 8 * h] : 1.f;
      }
    }
    __syncwarp();  // every lane has read the slot
    fetch(slot);
    __syncwarp();
    if (++slot == STAGES) slot = 0;
    // keys that the sequence has, of the block and of its halves with a page
    const int have = len - key0;
    const bool part_of = have < KB || ok_pages != (pages_log ? 3u : NB == 2 ? 3u : 1u);
    auto is_key = [&](int y, int key) {  // key of half y
      return y * 16 + key < have && ((ok_pages >> y) & 1u);
    };
    if (CODE != SRDIT_Q_INT8 && part_of) {  // values of others, which may be NaN: zeros
#pragma unroll
      for (int y = 0; y < NB; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!is_key(y, 2 * c + (r & 1) + (r >> 1) * 8))
#pragma unroll
            for (int x = 0; x < VP; ++x) vr[y][r][x] = make_uint4(0, 0, 0, 0);
    }
    const bool hidden = a.causal && key0 + KB - 1 > first;  // from some of the queries
    // Values that are not finite, where some queries do not see them, are taken out, and the
    // queries that do get a NaN.
    uint32_t bad[NB][2];  // keys g and g + 8
#pragma unroll
    for (int y = 0; y < NB; ++y) bad[y][0] = bad[y][1] = 0u;
    if (hidden && CODE != SRDIT_Q_INT8) {
#pragma unroll
      for (int y = 0; y < NB; ++y) {
        uint32_t all[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bool here;
          if constexpr (CODES) {
            here = nan_codes(vr[y][r][0].x) || nan_codes(vr[y][r][0].y) ||
                   nan_codes(vr[y][r][0].z) || nan_codes(vr[y][r][0].w);
          } else {
            uint32_t mx = 0;
#pragma unroll
            for (int x = 0; x < VP; ++x)
              mx = max_bits(max_bits(max_bits(max_bits(mx, vr[y][r][x].x), vr[y][r][x].y),
                                     vr[y][r][x].z),
                            vr[y][r][x].w);
            here = not_finite<E>(mx);
          }
          all[r] = __ballot_sync(0xffffffffu, here);
          if (all[r] & (0x11111111u << c))
#pragma unroll
            for (int x = 0; x < VP; ++x) vr[y][r][x] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
          bad[y][h] = ((g & 1) ? all[2 * h + 1] : all[2 * h]) & (0x11111111u << (g >> 1));
      }
    }
    // the exponent of a value's scale, less 24, and the scale over it (0, an infinity and a NaN stay)
    float lv[NB][2];
    if constexpr (CODES) {
#pragma unroll
      for (int y = 0; y < NB; ++y)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int bits = static_cast<int>(__float_as_uint(vs[y][h]) >> 23 & 255u);
          const int e = min(max(bits, 127 + LEAST), 127 + MOST);
          vs[y][h] *= exp2_int(127 - e);
          lv[y][h] = __int_as_float(0x4b000000 | e) - (8388608.f + 127.f + L_UNIT);
        }
    }
    float p[NT][NB][4];
#pragma unroll
    for (int y = 0; y < NB; ++y) {
      uint4 kf[2][NC];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 0; x < KP; ++x) {
          if constexpr (CODES) {
            uint32_t w[8];
            widen_codes<CODE>(kr[y][h][x], w);
            kf[h][2 * x] = make_uint4(w[0], w[1], w[2], w[3]);
            kf[h][2 * x + 1] = make_uint4(w[4], w[5], w[6], w[7]);
          } else {
            kf[h][x] = kr[y][h][x];
          }
        }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        // two chains of products, joined at the end
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < NC; ++x) {
          mma16816<E>(s0, kf[0][x].x, kf[1][x].x, kf[0][x].y, kf[1][x].y, qf[n][x].x, qf[n][x].y);
          mma16816<E>(s2, kf[0][x].z, kf[1][x].z, kf[0][x].w, kf[1][x].w, qf[n][x].z, qf[n][x].w);
        }
        // [0], [2]: column 2c, keys g and g + 8; [1], [3]: column 2c + 1
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[n][y][e] = s0[e] + s2[e];
          if constexpr (CODES) p[n][y][e] *= ks[y][e >> 1];
        }
        if (part_of || hidden) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = g + (e >> 1) * 8;
            if (!is_key(y, key) || key0 + y * 16 + key > lim[n][e & 1]) p[n][y][e] = neg_inf();
          }
        }
      }
    }
    uint32_t pf[NT][NB][2];
    bool moved = false;
    float alpha[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // (rounded before the maximum is taken from them: however large they are, that of the
        // largest is 0)
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& x = p[n][y][2 * h + e];
            x = CODES ? __fmaf_rn(x, cq[n][e], lv[y][h]) : __fmul_rn(x, cq[n][e]);  // (both 24 less)
          }
        float top = max2(p[n][0][e], p[n][0][2 + e]);
        if constexpr (NB == 2) top = max2(top, max2(p[n][1][e], p[n][1][2 + e]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = max2(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float mn = max2(m[n][e], top);
        const float neg = mn == neg_inf() ? 0.f : -mn;
        const Fall<CODES> fall(m[n][e] + neg);
        alpha[n][e] = fall.f;
        moved |= mn != m[n][e];
        m[n][e] = mn;
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float& x = p[n][y][2 * h + e];
            const bool seen = x != neg_inf();
            const float z = __fadd_rn(x, neg);
            x = ex2(z);
            if constexpr (CODES) {
              sum += ex2(z - lv[y][h]);
              x = seen ? x * vs[y][h] : 0.f;
            } else {
              sum += x;
            }
            if (bad[y][h] && seen) sum = __int_as_float(0x7fc00000);
          }
        l[n][e] = fall.add(l[n][e], sum);
      }
#pragma unroll
      for (int y = 0; y < NB; ++y) {
        pf[n][y][0] = transpose8x8(pack2(p[n][y][0], p[n][y][1], E{}));
        pf[n][y][1] = transpose8x8(pack2(p[n][y][2], p[n][y][3], E{}));
      }
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
    for (int y = 0; y < NB; ++y) {
      // the operand rows are the lane group's value columns 2w and 2w + 1 of its x-th eight: of each
      // the keys of rows 2c and 2c + 1 (a0, a1) and those 8 further on side by side
      if constexpr (CODES) {
        const uint32_t r0[4] = {vr[y][0][0].x, vr[y][0][0].y, vr[y][0][0].z, vr[y][0][0].w};
        const uint32_t r1[4] = {vr[y][1][0].x, vr[y][1][0].y, vr[y][1][0].z, vr[y][1][0].w};
        const uint32_t r2[4] = {vr[y][2][0].x, vr[y][2][0].y, vr[y][2][0].z, vr[y][2][0].w};
        const uint32_t r3[4] = {vr[y][3][0].x, vr[y][3][0].y, vr[y][3][0].z, vr[y][3][0].w};
#pragma unroll
        for (int j = 0; j < 2 * NV; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // (codes of two columns of two rows, by column)
            uint32_t a0, a1, a2, a3;
            widen4<CODE>(__byte_perm(r0[j], r1[j], e ? 0x7362 : 0x5140), a0, a1);
            widen4<CODE>(__byte_perm(r2[j], r3[j], e ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816<E>(o[n][2 * j + e], a0, a1, a2, a3, pf[n][y][0], pf[n][y][1]);
          }
      } else {
#pragma unroll
        for (int x = 0; x < NV; ++x) {
          const uint32_t r0[4] = {vr[y][0][x].x, vr[y][0][x].y, vr[y][0][x].z, vr[y][0][x].w};
          const uint32_t r1[4] = {vr[y][1][x].x, vr[y][1][x].y, vr[y][1][x].z, vr[y][1][x].w};
          const uint32_t r2[4] = {vr[y][2][x].x, vr[y][2][x].y, vr[y][2][x].z, vr[y][2][x].w};
          const uint32_t r3[4] = {vr[y][3][x].x, vr[y][3][x].y, vr[y][3][x].z, vr[y][3][x].w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = __byte_perm(r0[w], r1[w], 0x5410);
            const uint32_t a1 = __byte_perm(r0[w], r1[w], 0x7632);
            const uint32_t a2 = __byte_perm(r2[w], r3[w], 0x5410);
            const uint32_t a3 = __byte_perm(r2[w], r3[w], 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma16816<E>(o[n][x * 4 + w], a0, a1, a2, a3, pf[n][y][0], pf[n][y][1]);
          }
        }
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
        const Fall<CODES> fall(ml.x - top);
        const float f = fall.f;
        const float4 v = *reinterpret_cast<const float4*>(&so[w][row][d]);
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
        sum = fall.add(ml.y, sum);
      }
    }
    *reinterpret_cast<float4*>(&co[row][d]) = acc;
    if (d == 0) cml[row] = make_float2(top, sum);
  }
  int share_of = 0, shares = 1;
  if (cluster > 1) {
    cluster_wait();  // the arrival at the start: every CTA of the cluster runs
    cluster_arrive();
    cluster_wait();  // every part is in its CTA's shared memory
    share_of = static_cast<int>(cluster_ctarank());
    shares = cluster;
  } else {
    __syncthreads();
  }
  // CTA `share_of` of the cluster joins every shares-th four columns of the parts
  const long long all_rows = static_cast<long long>(a.T) * a.H;
  const int wparts = a.splits / cluster;
  const int dq = a.D / 4;
  for (int x = threadIdx.x * shares + share_of; x < rows * dq; x += WARPS * 32 * shares) {
    const int row = x / dq, d = (x - row * dq) * 4;
    float top = neg_inf(), sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (cluster > 1) {
      const uint32_t ml0 = smem_u32(&cml[row]), o0 = smem_u32(&co[row][d]);
      float pm[8], pl[8];
      float4 po[8];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        pm[y] = neg_inf();
        pl[y] = 0.f;
        po[y] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (y < cluster) {
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                       : "=f"(pm[y]), "=f"(pl[y])
                       : "r"(mapa_shared(ml0, y)));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(po[y].x), "=f"(po[y].y), "=f"(po[y].z), "=f"(po[y].w)
                       : "r"(mapa_shared(o0, y)));
        }
        top = max2(top, pm[y]);
      }
      if (top != neg_inf()) {
#pragma unroll
        for (int y = 0; y < 8; ++y) {
          const Fall<CODES> fall(pm[y] - top);
          const float f = fall.f;
          acc.x = fmaf(po[y].x, f, acc.x);
          acc.y = fmaf(po[y].y, f, acc.y);
          acc.z = fmaf(po[y].z, f, acc.z);
          acc.w = fmaf(po[y].w, f, acc.w);
          sum = fall.add(pl[y], sum);
        }
      }
    } else {
      top = cml[row].x;
      sum = cml[row].y;
      acc = *reinterpret_cast<const float4*>(&co[row][d]);
    }
    if (slot_of_part >= 0) {  // a share's part
      *reinterpret_cast<float4*>(a.ws + (static_cast<long long>(slot_of_part) * R + row) * DP + d) =
          acc;
      if (d == 0)
        reinterpret_cast<float2*>(a.ml)[slot_of_part * R + row] = make_float2(top, sum);
      continue;
    }
    const int i = a.by_group.div(row);
    const long long tok = row0 + i;
    const int head = kvh * a.group + row - i * a.group;
    if (wparts == 1) {
      const float inv = sum == 0.f ? 0.f : (CODES ? exp2_int(L_UNIT) : 1.f) / sum;
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + tok * a.os[0] + head * a.os[1] + d) =
          make_uint2(pack2(acc.x * inv, acc.y * inv, T{}), pack2(acc.z * inv, acc.w * inv, T{}));
    } else {
      const long long at = (part / cluster) * all_rows + tok * a.H + head;
      *reinterpret_cast<float4*>(a.ws + at * a.D + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(a.ml + at * 2) = make_float2(top, sum);
    }
  }
  if (a.shared) {
    // the ring takes O's place again: TMA writes follow these reads
    fence_proxy_async_smem();
    __syncthreads();
  }
  }
  if (cluster > 1) {  // no CTA leaves while another reads its shared memory
    cluster_arrive();
    cluster_wait();
  }
}

// One block per CTA: joins the parts of the rows that its share begins and does not end, which
// are in its second slot and the first slots of the CTAs that go on with the same key head. A
// thread takes four columns of a row and every fourth part, four parts' loads in flight: bounded
// by their latency.
template <typename T, int DP, int NT, bool CODES>
__global__ void __launch_bounds__(512) join_share_kernel(const __grid_constant__ Args a) {
  pdl_begin();
  constexpr int R = 8 * NT;
  const StepCut cut = static_cast<const StepCut*>(a.cuts)[blockIdx.x];
  if (cut.parts == 0) return;
  __shared__ float4 acc_of[4][128];
  __shared__ float2 ml_of[4][128];
  const int row0 = a.rows.begin(cut.b);
  const int rows = min(a.rows.end(cut.b) - row0, a.max_q) * a.group;
  const int dq = a.D / 4, way = threadIdx.x >> 7, task = threadIdx.x & 127;
  for (int x0 = 0; x0 < rows * dq; x0 += 128) {
    const int x = min(x0 + task, rows * dq - 1);
    const int row = x / dq, d = (x - row * dq) * 4;
    float m = neg_inf(), l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 q, float4 v) {
      if (q.x == neg_inf()) return;  // it saw no key
      const float mn = max2(m, q.x);
      const Fall<CODES> fall0(m - mn), fall1(q.x - mn);
      const float f0 = fall0.f, f1 = fall1.f;
      m = mn;
      l = fall1.add(q.y, fall0.add(l, 0.f));
      acc.x = acc.x * f0 + v.x * f1;
      acc.y = acc.y * f0 + v.y * f1;
      acc.z = acc.z * f0 + v.z * f1;
      acc.w = acc.w * f0 + v.w * f1;
    };
    for (int p0 = way; p0 < cut.parts; p0 += 16) {
      float2 q[4];
      float4 v[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int p = p0 + 4 * y, cta = static_cast<int>(blockIdx.x) + p * a.Hkv;
        const int at = (p == 0 ? 2 * cta + 1 : 2 * cta) * R + row;
        q[y] = make_float2(neg_inf(), 0.f);
        v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p < cut.parts) {
          q[y] = __ldg(reinterpret_cast<const float2*>(a.ml) + at);
          v[y] = __ldg(reinterpret_cast<const float4*>(a.ws + static_cast<long long>(at) * DP + d));
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) add(q[y], v[y]);
    }
    if (way) {
      acc_of[way][task] = acc;
      ml_of[way][task] = make_float2(m, l);
    }
    __syncthreads();
    if (way == 0) {
      for (int w = 1; w < min(4, cut.parts); ++w) add(ml_of[w][task], acc_of[w][task]);
      const float inv = l == 0.f ? 0.f : (CODES ? exp2_int(L_UNIT) : 1.f) / l;
      const int i = a.by_group.div(row);
      if (x0 + task < rows * dq)
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) +
                                  static_cast<long long>(row0 + i) * a.os[0] +
                                  (cut.kvh * a.group + row - i * a.group) * a.os[1] + d) =
            make_uint2(pack2(acc.x * inv, acc.y * inv, T{}), pack2(acc.z * inv, acc.w * inv, T{}));
    }
    __syncthreads();
  }
}

// One warp per (token, head): joins the parts that went through the workspace, four parts'
// loads in flight.
template <typename T, bool CODES>
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
    const Fall<CODES> fall(m - mn);
    m = mn;
    l = fall.add(l, 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= fall.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (pm[x].x == neg_inf()) continue;  // a part that saw no key
      const Fall<CODES> of_part(pm[x].x - m);
      const float k = of_part.f;
      l = of_part.add(pm[x].y, l);
      acc[0] = fmaf(v[x].x, k, acc[0]);
      acc[1] = fmaf(v[x].y, k, acc[1]);
      acc[2] = fmaf(v[x].z, k, acc[2]);
      acc[3] = fmaf(v[x].w, k, acc[3]);
    }
  }
  const float inv = l == 0.f ? 0.f : (CODES ? exp2_int(L_UNIT) : 1.f) / l;
  if (on)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + t * a.os[0] + h * a.os[1] + lane * 4) =
        make_uint2(pack2(acc[0] * inv, acc[1] * inv, T{}), pack2(acc[2] * inv, acc[3] * inv, T{}));
}

// ---------------------------------------------------------------- launch
Plan plan_step(const srdit_seq_attn_args& u, int sms) {
  Plan p = {};
  p.step = true;
  const int group = u.H / u.Hkv;
  const bool one = u.max_q * group <= 8;
  const long long pairs = static_cast<long long>(u.B) * u.Hkv;
  const int per_sm = one ? 3 : 2, size = u.pages->code == SRDIT_KV_PLAIN ? 16 : 32;
  const long long held = static_cast<long long>(u.pages->table_width) * u.pages->page_size;
  const long long keys = u.max_kv > 0 && u.max_kv < held ? u.max_kv : held;
  const long long blocks = (keys + size - 1) / size;
  p.cluster = p.parts = p.splits = 1;
  // By shares from SHARE_BLOCKS blocks a CTA, two CTAs an SM, three of codes (which take more
  // instructions a byte). The lengths are not known here: shares gain where they differ, and cost where
  // they are equal. us by shares and by clusters, one token, 32 heads over 8 of 128: 32 sequences of up to
  // 4096 keys 52 and 64, e4m3 43 and 61; 8 of up to 32768 105 and 124, e4m3 69 and 110; 128 of up to 1024 56
  // and 52. All of one length: 32 of 4096 90 and 83, e4m3 60 and 63; 32 of 2048 50 and 45; 8 of 32768 167 and
  // 157, e4m3 107 and 118; 16 of 4096 with four tokens 63 and 52. Fewer blocks: 32 of up to 1024 24 and
  // 20.5 (55 blocks a CTA), 8 of 2048 21 and 17 (28). (blocks x sequences in 32 bits)
  const long long ctas = (size == 16 ? 2ll : per_sm) * sms;
  if (u.B <= MAX_SHARED && pairs * blocks >= SHARE_BLOCKS * ctas && u.Hkv <= ctas &&
      u.B * (held / size + 1) < (1ll << 31)) {
    p.shared = true;
    p.ctas = static_cast<int>(ctas / u.Hkv * u.Hkv);
    p.ws_floats = 2 * ctas * (one ? 8 : 16) * ((u.D <= 64 ? 64 : 128) + 2) + 4 * ctas;
    return p;
  }
  // The keys are split until every SM has its CTAs, each with a block per warp at least, within a
  // cluster; more than a cluster's 8 parts go through the workspace, from 8 blocks a warp.
  const long long most = (blocks + WARPS - 1) / WARPS;
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

template <typename T, int DP, int NT, bool CODES>
static int join_shares(const Args& a, const Plan& p, cudaStream_t stream) {
  SRDIT_LAUNCH((join_share_kernel<T, DP, NT, CODES>), p.ctas, 512, 0, stream, a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int DP, int NT, int CODE>
static int launch(const srdit_seq_attn_args& u, const Args& a, const Plan& p, cudaStream_t stream) {
  using C = StepCfg<DP, NT, CODE>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  int rc = set_smem(step_kernel<T, DP, NT, CODE>, C::SMEM, attr_done);
  if (rc) return rc;
  CUtensorMap tk, tv;
  const int cols = C::CODES ? 128 : 64;
  const int rows = u.pages->page_size < C::KB ? u.pages->page_size : C::KB;
  rc = key_map(&tk, u, false, cols, rows);
  if (!rc) rc = key_map(&tv, u, true, cols, rows);
  if (rc) return rc;
  const dim3 grid = p.shared ? dim3(p.ctas)
                             : dim3(static_cast<unsigned>(p.splits),
                                    static_cast<unsigned>(a.B * a.Hkv));
  rc = launch_clusters(p.cluster, step_kernel<T, DP, NT, CODE>, grid, WARPS * 32, C::SMEM, stream, tk,
                       tv, a, p.cluster);
  return rc || !p.shared ? rc : join_shares<T, DP, NT, C::CODES>(a, p, stream);
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
  const unsigned blocks = static_cast<unsigned>((rows + 3) / 4);
  if (u.pages->code == SRDIT_KV_PLAIN)
    SRDIT_LAUNCH((join_step_kernel<T, false>), blocks, 128, 0, stream, a, p.parts);
  else
    SRDIT_LAUNCH((join_step_kernel<T, true>), blocks, 128, 0, stream, a, p.parts);
  return static_cast<int>(cudaGetLastError());
}

int run_step(const srdit_seq_attn_args& u, Args& a, const Plan& p, cudaStream_t stream) {
  a.splits = p.splits;
  a.by_group = Divisor::of(a.group);
  a.shared = p.shared;
  a.ml = a.ws + (p.shared ? 2ll * p.ctas * (u.max_q * a.group <= 8 ? 8 : 16) * (u.D <= 64 ? 64 : 128)
                          : static_cast<long long>(p.parts) * u.T * u.H * u.D);
  if (p.shared) a.cuts = a.ml + 4ll * p.ctas * (u.max_q * a.group <= 8 ? 8 : 16);
  return u.dtype == SRDIT_BF16 ? run_typed<__nv_bfloat16>(u, a, p, stream)
                               : run_typed<__half>(u, a, p, stream);
}

}  // namespace sattn
}  // namespace srdit
