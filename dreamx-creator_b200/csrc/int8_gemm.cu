// int8_gemm.cu -- row-wise scaled int8 GEMM on the tensor cores (sm_100a).
//
//   out[m, n] = a_scale[m] * w_scale[n] * sum_k A[m, k] W[n, k] + bias[n]
//
// The sum is exact in int32 (|A|, |W| <= 128 and K < 131072 keep it below 2^31), so
// neither the order of the products nor a split of K changes a bit of the result.
//
// Two kernels, one for each thing that bounds the product:
//
//   pair_kernel    more than 64 tokens (32 where the weights are small): bounded by the
//                  tensor cores, or by what an SM can load for them. A CTA pair computes a
//                  256 x BN tile with one
//                  tcgen05.mma.cta_group::2.kind::i8 per 32-deep step; two accumulators in
//                  tensor memory let a tile's epilogue run under the next tile's products;
//                  persistent. BN is chosen by the rounds of tiles it leaves (launch).
//   split_kernel   up to 64 tokens: bounded by the weights' bytes. The weights take the
//                  MMA's 128 rows and the tokens its columns (16, 32 or 64), so one token
//                  wastes 15 columns and not 255 rows. K is split over a cluster of up to 8
//                  CTAs, which read one another's int32 partial sums out of shared memory:
//                  no workspace, no atomics, no second launch.
#include <atomic>

#include "elem.cuh"
#include "srdit_internal.h"

namespace srdit {
namespace i8 {

constexpr int BK = 128;  // bytes of K per stage: one 128-byte swizzled row
constexpr int NUM_THREADS = 192;

struct Params {
  const float* a_scale;
  const float* w_scale;
  const void* bias;
  void* out;
  long long ldo;
  int M, N, K;
  int splits;  // split_kernel: CTAs of a cluster along K
  int tile_n;  // split_kernel: weight rows of a tile, up to 128
  int stages;  // split_kernel: blocks of K in flight
  int o_tma;   // pair_kernel: tmO is valid (out, its pitch and its width are 16-byte aligned)
  uint32_t* status;
};

template <typename T>
SRDIT_DEV float bias_at(const Params& p, int n) {
  return p.bias ? to_f(static_cast<const T*>(p.bias)[n]) : 0.f;
}
// acc * sa * sw + bias: the conversion, one product and one fma, a rounding each
SRDIT_DEV float scaled(uint32_t acc, float sa, float sw, float b) {
  return fmaf(static_cast<float>(static_cast<int>(acc)) * sa, sw, b);
}

// ---------------------------------------------------------------- few tokens
// Measured: 1 x 3072 x 14336 10.9 us, 4.1 TB/s; 37 x 4096 x 4096 8.8 us, 2.0 TB/s; a product of
// 1 x 128 x 128, which is launch and latency, takes 3.3. Memory is read at its rate for a few
// microseconds between only. A CTA takes 400 cycles for a block of K, tiles of 32 rows and of
// 112 alike, so without clusters 1 x 14336 x 3072 takes 24 us in place of 9. (Scales
// loaded a token at a time took as long as the sums; 128 tokens a tile in this kernel are slower
// than pair_kernel's 64-column tiles. Bulk copies of the sums into the other CTAs' memory were
// slower, 37 x 4096 x 4096 9.8 us, and not sound: in a process that had run many other products
// 11 x 2832 x 4077 ended in an illegal access, which range checks on every index of the kernel
// did not explain. With loads between two barriers of the cluster it has not been seen in 43000
// products of random sizes.)
//
// Shared memory: a ring of p.stages stages (weight rows, then tokens), barriers. An MMA reads
// 128 weight rows of a stage whatever tile_n is: PAST bytes behind the last stage keep that
// inside this CTA's memory. The partial sums take the ring's place.
constexpr int MAX_STAGES = 16;
template <int BT>
struct SplitCfg {
  static constexpr int PAST = (128 - 64 - BT) * BK;  // tile_n is 64 at least
  static constexpr int BARS = (2 * MAX_STAGES + 1) * 8 + 8;
  static constexpr int MOST = 232448 - 1024 - PAST - BARS;  // for the ring
  static constexpr uint32_t TMEM_COLS = BT < 32 ? 32 : BT;
  static int smem(int stages, int tile_n) {
    return stages * (tile_n + BT) * BK + PAST + BARS + 1024;
  }
};

template <typename T, int BT>
__global__ void __launch_bounds__(NUM_THREADS)
    split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                 const Params p) {
  pdl_begin();
  using C = SplitCfg<BT>;
  const int STAGES = p.stages;
  const int w_bytes = p.tile_n * BK, stage_bytes = w_bytes + BT * BK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * stage_bytes + C::PAST);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* done = empty + MAX_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int n0 = (static_cast<int>(blockIdx.x) / p.splits) * p.tile_n;
  const int num_kb = (p.K + BK - 1) / BK;
  const int kb0 = static_cast<int>(static_cast<long long>(num_kb) * split / p.splits);
  const int kb1 = static_cast<int>(static_cast<long long>(num_kb) * (split + 1) / p.splits);

  auto load = [&](int i, int s) {  // block i of this CTA's K range into stage s
    uint8_t* st = smem + s * stage_bytes;
    mbar_arrive_expect_tx(&full[s], static_cast<uint32_t>(stage_bytes));
    tma_load_2d(st, &tmW, &full[s], (kb0 + i) * BK, n0);
    tma_load_2d(st + w_bytes, &tmA, &full[s], (kb0 + i) * BK, 0);
  };
  const int n_kb = kb1 - kb0;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmA);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0u;
    fence_barrier_init();
    fence_proxy_async_smem();
    // the first loads need none of what the other warps still set up
    for (int i = 0; i < STAGES && i < n_kb; ++i) load(i, i);
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      for (int i = STAGES; i < n_kb; ++i) {
        if (!mbar_wait(&empty[s], ph, p.status, abort_flag)) {
          ok = false;
          break;
        }
        load(i, s);
        if (++s == STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
      // having given up, let the loads in flight land before the CTA exits
      if (!ok)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = idesc_i8(128, BT);
      int s = 0;
      uint32_t ph = 0;
      for (int i = 0; i < n_kb; ++i) {
        if (!mbar_wait(&full[s], ph, p.status, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t w_addr = smem_u32(smem + s * stage_bytes);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k)
          mma_i8_ss(tmem_base, sdesc_sw128(w_addr + k * 32, 16, 1024),
                    sdesc_sw128(w_addr + w_bytes + k * 32, 16, 1024), idesc,
                    (i > 0 || k > 0) ? 1u : 0u);
        tc_commit(&empty[s]);
        if (++s == STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (ok) tc_commit(done);
    }
    __syncwarp();
  }

  // the accumulator: lane = weight row, column = token (rows past tile_n: whatever the
  // buffer held)
  const int sub = warp & 3;
  const uint32_t t_row = tmem_base + (static_cast<uint32_t>(sub * 32) << 16);
  if (p.splits == 1) {
    if (warp >= 2 && mbar_wait_warp(done, 0u, p.status, abort_flag)) {
      tc_fence_after();
      const int n = n0 + sub * 32 + lane;
      const bool n_on = sub * 32 + lane < p.tile_n && n < p.N;
      const float sw = n_on ? p.w_scale[n] : 0.f;
      const float b = n_on ? bias_at<T>(p, n) : 0.f;
      T* out = static_cast<T*>(p.out) + n;
#pragma unroll 1
      for (int c = 0; c < BT && c < p.M; c += 16) {
        uint32_t r[16];
        tmem_ld16(t_row + c, r);
        float sa[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) sa[e] = c + e < p.M ? __ldg(p.a_scale + c + e) : 0.f;
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (c + e < p.M && n_on)
            out[(c + e) * p.ldo] = static_cast<T>(scaled(r[e], sa[e], sw, b));
      }
    }
    __syncwarp();
  } else {
    // Each epilogue warp lays its 32 rows' partial sums out over the ring, which is done with,
    // as [4 tokens][32 rows][4]. After the cluster's barrier 32 rows of 4 tokens are joined by
    // one warp of the cluster, out of all its CTAs' memory. (Stores into the other CTAs'
    // memory, 4 bytes a lane, took 40 ns each.) Both sides are the threads' own accesses, ordered
    // by the barrier.
    const uint32_t sums = smem_u32(smem);
    if (warp >= 2 && mbar_wait_warp(done, 0u, p.status, abort_flag)) {
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < BT && c < p.M; c += 16) {
        uint32_t r[16];
        tmem_ld16(t_row + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<uint4*>(smem + ((sub * (BT / 4) + (c + e) / 4) * 32 + lane) * 16) =
              make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
      }
    }
    __syncwarp();
    cluster_sync();  // every CTA's sums are in its memory
    if (warp >= 2) {
      for (int it = split * 4 + (warp - 2); it < BT; it += p.splits * 4) {
        const int quad = it >> 2, rows = it & 3;
        if (quad * 4 >= p.M) break;
        if (rows * 32 >= p.tile_n) continue;
        uint4 v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          v[x] = make_uint4(0u, 0u, 0u, 0u);
          if (x < p.splits)
            asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v[x].x), "=r"(v[x].y), "=r"(v[x].z), "=r"(v[x].w)
                         : "r"(mapa_shared(sums + ((rows * (BT / 4) + quad) * 32 + lane) * 16,
                                           static_cast<uint32_t>(x)))
                         : "memory");
        }
        const int row = rows * 32 + lane, n = n0 + row;
        const bool n_on = row < p.tile_n && n < p.N;
        const float sw = n_on ? p.w_scale[n] : 0.f;
        const float b = n_on ? bias_at<T>(p, n) : 0.f;
        float sa[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sa[e] = quad * 4 + e < p.M ? __ldg(p.a_scale + quad * 4 + e) : 0.f;
        uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          acc[0] += v[x].x;
          acc[1] += v[x].y;
          acc[2] += v[x].z;
          acc[3] += v[x].w;
        }
        T* out = static_cast<T*>(p.out) + n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (quad * 4 + e < p.M && n_on)
            out[(quad * 4 + e) * p.ldo] = static_cast<T>(scaled(acc[e], sa[e], sw, b));
      }
    }
    __syncwarp();
    cluster_sync();  // no CTA leaves while another reads its memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------- many tokens
// Measured: 6912 x 3072 x 14336 199 us, 3.05 POP/s, the tensor cores' pipe 94% busy;
// 2304 x 3072 x 9216 47 us, 2.75 POP/s; 512 x 4096 x 4096 12.7 us. In tiles of 256 columns
// alone the last was 17.4, and 512 x 1024 x 1024 10.7 in place of 6.1.
constexpr int EPI_WARPS = 4;
constexpr int STG_BYTES = 32 * 128;  // a warp's staging box: 32 rows x 128 bytes

template <int BN>
struct PairCfg {
  static constexpr int A_BYTES = 128 * BK;
  static constexpr int STAGE_BYTES = A_BYTES + (BN / 2) * BK;
  static constexpr int STAGES = BN == 256 ? 5 : BN == 192 ? 6 : 7;
  static constexpr int OFF_STG = STAGES * STAGE_BYTES;
  static constexpr int OFF_COL = OFF_STG + EPI_WARPS * 2 * STG_BYTES;
  static constexpr int OFF_BAR = OFF_COL + 2 * 2 * 256 * 4;  // w_scale, bias
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static_assert(STAGE_BYTES % 1024 == 0, "stages stay 1024-byte aligned");
  static_assert(SMEM <= 232448, "shared memory budget");
};

template <typename T, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NUM_THREADS, 1)
    pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                const __grid_constant__ CUtensorMap tmO, const Params p) {
  pdl_begin();
  using C = PairCfg<BN>;
  constexpr int STAGES = C::STAGES;
  constexpr int CHUNK = 128 / sizeof(T);  // output columns of a staging box
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // completed in the even CTA
  uint64_t* empty = full + STAGES;   // one per CTA
  uint64_t* tfull = empty + STAGES;  // [2]
  uint64_t* tempty = tfull + 2;      // [2], in the even CTA, one arrival per epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  float* col_s = reinterpret_cast<float*>(smem + C::OFF_COL);  // [2][256] w_scale
  float* col_b = col_s + 512;                                  // [2][256] bias

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int num_m = (p.M + 255) / 256;
  const int num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int num_kb = (p.K + BK - 1) / BK;
  const int cid = static_cast<int>(cluster_id_x());
  const int ncl = static_cast<int>(num_clusters_x());

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * EPI_WARPS);
    }
    *abort_flag = 0u;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW);
    if (p.o_tma) tma_prefetch_desc(&tmO);
  }
  if (warp == 1) {
    tmem_alloc_2sm(tmem_slot, 512);
    tmem_relinquish_2sm();
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      const uint32_t full_even = mapa_shared(smem_u32(&full[0]), 0);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = cid; tile < num_tiles && ok; tile += ncl) {
        const int mt = tile / num_n, nt = tile % num_n;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1u, p.status, abort_flag)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2u * C::STAGE_BYTES);
          uint8_t* st = smem + s * C::STAGE_BYTES;
          tma_load_2d_2sm(st, &tmA, full_even + 8u * s, kb * BK, mt * 256 + rank * 128);
          tma_load_2d_2sm(st + C::A_BYTES, &tmW, full_even + 8u * s, kb * BK,
                          nt * BN + rank * (BN / 2));
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // having given up, let the loads in flight land before the CTA exits (their
      // completions are counted on the even CTA's barriers)
      if (!ok)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = idesc_i8(256, BN);
      const uint32_t empty_own = mapa_shared(smem_u32(&empty[0]), 0);
      const uint32_t empty_peer = mapa_shared(smem_u32(&empty[0]), 1);
      const uint32_t tfull_own = mapa_shared(smem_u32(&tfull[0]), 0);
      const uint32_t tfull_peer = mapa_shared(smem_u32(&tfull[0]), 1);
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      int local = 0;
      for (int tile = cid; tile < num_tiles && ok; tile += ncl, ++local) {
        const int acc = local & 1;
        if (!mbar_wait(&tempty[acc], (static_cast<uint32_t>(local >> 1) & 1u) ^ 1u, p.status,
                       abort_flag))
          break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&full[s], ph, p.status, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * C::STAGE_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_i8_ss_2sm(d_tmem, sdesc_sw128(a_addr + k * 32, 16, 1024),
                          sdesc_sw128(a_addr + C::A_BYTES + k * 32, 16, 1024), idesc,
                          (kb > 0 || k > 0) ? 1u : 0u);
          tc_commit_2sm(empty_own + 8u * s);
          tc_commit_2sm(empty_peer + 8u * s);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (ok) {
          tc_commit_2sm(tfull_own + 8u * acc);
          tc_commit_2sm(tfull_peer + 8u * acc);
        }
      }
    }
  } else {
    const int sub = warp & 3;
    const int ep_tid = threadIdx.x - 64;
    uint8_t* stg = smem + C::OFF_STG + sub * 2 * STG_BYTES;
    const uint32_t tempty_even = mapa_shared(smem_u32(&tempty[0]), 0);
    int stores = 0;
    int local = 0;
    bool ok = true;
    for (int tile = cid; tile < num_tiles; tile += ncl, ++local) {
      const int acc = local & 1;
      const int mt = tile / num_n, nt = tile % num_n;
      const int n0 = nt * BN;
      // this tile's column scales and bias (double-buffered; 0 past N)
      for (int c = ep_tid; c < BN; c += 128) {
        const int col = n0 + c;
        col_s[acc * 256 + c] = col < p.N ? __ldg(p.w_scale + col) : 0.f;
        col_b[acc * 256 + c] = col < p.N ? bias_at<T>(p, col) : 0.f;
      }
      if (!named_barrier_all(1, 128, ok)) break;
      ok = mbar_wait_warp(&tfull[acc], static_cast<uint32_t>(local >> 1) & 1u, p.status,
                          abort_flag);
      if (!ok) continue;  // to the barrier, where all four warps learn of it
      tc_fence_after();
      const int row0 = mt * 256 + static_cast<int>(rank) * 128 + sub * 32;
      const float sa = row0 + lane < p.M ? p.a_scale[row0 + lane] : 0.f;
      const float* cs = col_s + acc * 256;
      const float* cb = col_b + acc * 256;
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(sub * 32) << 16) +
                             static_cast<uint32_t>(acc * BN);
      const bool rows_on = row0 < p.M;
#pragma unroll 1
      for (int ch = 0; ch < BN / CHUNK; ++ch) {
        const int col0 = n0 + ch * CHUNK;
        if (!rows_on || col0 >= p.N) break;  // warp-uniform: nothing of the box is stored
        uint8_t* buf = stg + (stores & 1) * STG_BYTES;
        if (p.o_tma && stores >= 2) {
          if (lane == 0) bulk_wait_group_read1();
          __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < CHUNK / 32; ++h) {
          const int c0 = ch * CHUNK + h * 32;
          uint32_t r[32];
          tmem_ld32(t_row + c0, r);
          tmem_ld_wait();
          uint32_t pw[sizeof(T) == 4 ? 32 : 16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float y0 = scaled(r[j], sa, cs[c0 + j], cb[c0 + j]);
            const float y1 = scaled(r[j + 1], sa, cs[c0 + j + 1], cb[c0 + j + 1]);
            if constexpr (sizeof(T) == 4) {
              pw[j] = __float_as_uint(y0);
              pw[j + 1] = __float_as_uint(y1);
            } else {
              pw[j >> 1] = pack2(y0, y1, T{});
            }
          }
          // 16-byte piece q of the box row at q ^ (row & 7): the 128-byte TMA swizzle
#pragma unroll
          for (int q = 0; q < static_cast<int>(sizeof(pw) / 16); ++q)
            *reinterpret_cast<uint4*>(buf + lane * 128 + (((h * 4 + q) ^ (lane & 7)) << 4)) =
                make_uint4(pw[4 * q], pw[4 * q + 1], pw[4 * q + 2], pw[4 * q + 3]);
        }
        if (p.o_tma) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmO, buf, col0, row0);
            bulk_commit_group();
          }
        } else {
          // an output that TMA cannot address: the box row by row, lanes along N
          __syncwarp();
          const int rows = min(32, p.M - row0);
          for (int r = 0; r < rows; ++r) {
            T* o = static_cast<T*>(p.out) + (row0 + r) * p.ldo + col0;
#pragma unroll
            for (int c = lane; c < CHUNK; c += 32) {
              const int byte = c * static_cast<int>(sizeof(T));
              if (col0 + c < p.N)
                o[c] = *reinterpret_cast<const T*>(buf + r * 128 + (((byte >> 4) ^ (r & 7)) << 4) +
                                                   (byte & 15));
            }
          }
          __syncwarp();
        }
        ++stores;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty_even + 8u * acc);
    }
    if (lane == 0) bulk_wait_group_all();
    __syncwarp();
  }

  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_2sm(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- launch
struct Operands {
  const void* a;
  const void* w;
  long long lda, ldw;
};

template <typename T, int BT>
static int launch_split(const Operands& o, Params& p, int dev, cudaStream_t stream) {
  using C = SplitCfg<BT>;
  auto kern = split_kernel<T, BT>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  int rc = set_smem(kern, 232448, attr_done);
  if (rc) return rc;
  // The tile's weight rows and the splits of K with the least time, in cycles: what an SM's
  // CTAs read at 38 bytes a cycle (an SM's share of the memory is 23; the latency of 2000
  // cycles wants 76 KB in flight), each wave's start and end, the cluster's exchange.
  // Clusters of large CTAs do not fill every SM.
  const int sms = num_sms(dev);
  const int num_kb = (p.K + BK - 1) / BK;
  long long best = -1;
  for (int tile = 128; tile >= 64; tile -= 16) {
    for (int splits = 1; splits <= 8 && (splits == 1 || splits * 2 <= num_kb); splits *= 2) {
      const long long ctas = static_cast<long long>((p.N + tile - 1) / tile) * splits;
      const int n_kb = (num_kb + splits - 1) / splits, stage = (tile + BT) * BK;
      int stages = C::MOST / stage < MAX_STAGES ? C::MOST / stage : MAX_STAGES;
      if (stages > n_kb) stages = n_kb;
      int per_sm = C::smem(stages, tile) <= 115712 ? 2 : 1;
      if (ctas > sms && per_sm == 1) {  // two smaller rings on an SM rather than a second wave
        const int half = (115712 - (232448 - C::MOST)) / stage;
        if (half >= 3) {
          stages = half < stages ? half : stages;
          per_sm = 2;
        }
      }
      const long long room = splits > 1 ? sms * per_sm * 7 / 8 : sms * per_sm;
      const long long waves = (ctas + room - 1) / room;
      const long long rounds = (ctas + sms - 1) / sms;
      const long long cost = (rounds > waves ? rounds : waves) * n_kb * stage / 38 + waves * 3000 +
                             (splits > 1 ? 1500 + BT / splits * 20 : 0);
      if (best < 0 || cost < best) {
        best = cost;
        p.tile_n = tile;
        p.splits = splits;
        p.stages = stages;
      }
    }
  }
  const int n_tiles = (p.N + p.tile_n - 1) / p.tile_n;
  CUtensorMap ta, tw;
  rc = make_tmap_2d(&ta, o.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.M, o.lda, BK, BT);
  if (rc) return rc;
  rc = make_tmap_2d(&tw, o.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.N, o.ldw, BK, p.tile_n);
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>(n_tiles * p.splits));
  return launch_clusters(p.splits, kern, grid, NUM_THREADS,
                         static_cast<size_t>(C::smem(p.stages, p.tile_n)), stream, ta, tw, p);
}

template <typename T, int BN>
static int launch_pair(const Operands& o, Params& p, int dev, cudaStream_t stream) {
  using C = PairCfg<BN>;
  auto kern = pair_kernel<T, BN>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  int rc = set_smem(kern, C::SMEM, attr_done);
  if (rc) return rc;
  CUtensorMap ta, tw, to;
  rc = make_tmap_2d(&ta, o.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.M, o.lda, BK, 128);
  if (rc) return rc;
  rc = make_tmap_2d(&tw, o.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K, p.N, o.ldw, BK, BN / 2);
  if (rc) return rc;
  // A TMA store of a box that reaches past column N writes the rest of N's 16-byte piece too:
  // only outputs whose rows end with such a piece are stored by it.
  p.o_tma = (reinterpret_cast<uintptr_t>(p.out) | p.ldo * sizeof(T) | p.N * sizeof(T)) % 16 == 0;
  to = ta;
  if (p.o_tma) {
    const CUtensorMapDataType dt = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                                  : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    rc = make_tmap_2d(&to, p.out, dt, sizeof(T), p.N, p.M, p.ldo, 128 / sizeof(T), 32);
    if (rc) return rc;
  }
  const int tiles = ((p.M + 255) / 256) * ((p.N + BN - 1) / BN);
  const int pairs = num_sms(dev) / 2;
  return launch_plain(kern, 2 * (tiles < pairs ? tiles : pairs), NUM_THREADS, C::SMEM, stream, ta,
                      tw, to, p);
}

// Columns of pair_kernel's tiles for a product, or 0 where split_kernel takes it.
static int pair_columns(int M, int N, int K, int sms) {
  // split_kernel and pair_kernel, K x N = 4096 x 4096: one token 6.7 and 16.2 us, 16 6.9 and
  // 13.6, 48 8.6 and 9.4, 64 8.8 and 9.4.
  // From 33 to 64 tokens the clusters' exchange grows with the tokens, what a pair without a
  // split of K loses grows with K, and large weights want split_kernel's deeper loads: 40 tokens,
  // 1024 x 1024 5.5 and 5.7, 1024 x 4096 6.8 and 6.8, 2048 x 2048 6.9 and 7.3; 64 tokens, 1024 x
  // 1024 6.1 and 5.7, 2048 x 8192 8.7 and 7.6, 3072 x 3072 8.5 and 8.2, 4096 x 1024 7.1 and 9.3,
  // 3072 x 14336 10.5 and 13.1, 16384 x 4096 12.7 and 23.7.
  if (M <= 32 || (M <= 64 && (K > 48 * M || static_cast<long long>(K) * N > 24ll << 20))) return 0;
  // The tile width with the least time: rounds of tiles over the pairs, times the cycles of
  // a block of K, which are the products' (two per column) or the loads' (60 bytes a cycle
  // and SM), whichever is more.
  const int pairs = sms / 2;
  const long long m_tiles = (M + 255) / 256;
  int best = 0;
  long long best_cost = 0;
  for (int bn : {256, 192, 128, 64}) {
    const long long rounds = (m_tiles * ((N + bn - 1) / bn) + pairs - 1) / pairs;
    const int mma = 2 * bn, load = (128 + bn / 2) * BK / 60;
    const long long cost = rounds * (mma > load ? mma : load);
    if (!best || cost < best_cost) {
      best = bn;
      best_cost = cost;
    }
  }
  return best;
}

template <typename T>
static int launch(const Operands& o, Params& p, cudaStream_t stream) {
  const int dev = device_here();
  switch (pair_columns(p.M, p.N, p.K, num_sms(dev))) {
    case 0: break;
    case 256: return launch_pair<T, 256>(o, p, dev, stream);
    case 192: return launch_pair<T, 192>(o, p, dev, stream);
    case 128: return launch_pair<T, 128>(o, p, dev, stream);
    default: return launch_pair<T, 64>(o, p, dev, stream);
  }
  if (p.M <= 16) return launch_split<T, 16>(o, p, dev, stream);
  if (p.M <= 32) return launch_split<T, 32>(o, p, dev, stream);
  return launch_split<T, 64>(o, p, dev, stream);
}

}  // namespace i8
}  // namespace srdit

using namespace srdit;

extern "C" int srdit_int8_gemm_columns(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return i8::pair_columns(M, N, K, num_sms(device_here()));
}

extern "C" int srdit_int8_gemm(const void* a, const float* a_scale, const void* w,
                               const float* w_scale, const void* bias, void* out, int dtype, int M,
                               int N, int K, long long lda, long long ldw, long long ldo,
                               uint32_t* status, cudaStream_t stream) {
  if (M < 0 || N < 0 || K <= 0) return SRDIT_EINVAL;
  if (M == 0 || N == 0) return 0;
  if (!a || !a_scale || !w || !w_scale || !out) return SRDIT_EINVAL;
  // the pitch of one row may be anything
  if (M == 1) {
    lda = (K + 15ll) / 16 * 16;
    ldo = N;
  }
  if (N == 1) ldw = (K + 15ll) / 16 * 16;
  if (lda < K || ldw < K || ldo < N) return SRDIT_EINVAL;
  if (K >= 131072) return SRDIT_EUNSUPPORTED;
  if ((lda % 16) || (ldw % 16) || (reinterpret_cast<uintptr_t>(a) & 15u) ||
      (reinterpret_cast<uintptr_t>(w) & 15u))
    return SRDIT_EALIGN;
  const uintptr_t e = dtype == SRDIT_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(out) % e || reinterpret_cast<uintptr_t>(bias) % e ||
      reinterpret_cast<uintptr_t>(a_scale) % 4 || reinterpret_cast<uintptr_t>(w_scale) % 4)
    return SRDIT_EALIGN;
  const i8::Operands o = {a, w, lda, ldw};
  i8::Params p = {a_scale, w_scale, bias, out, ldo, M, N, K, 1, 128, 1, 0, status};
  switch (dtype) {
    case SRDIT_BF16: return i8::launch<__nv_bfloat16>(o, p, stream);
    case SRDIT_FP16: return i8::launch<__half>(o, p, stream);
    case SRDIT_FP32: return i8::launch<float>(o, p, stream);
    default: return SRDIT_EINVAL;
  }
}
