// cross_attn.cu -- attention of queries over an encoder's keys and values of another
// length, with per-sample key lengths, a key mask and grouped heads (sm_100a).
//
//   o[b, i, h] = sum_j p_j v[b, j, g] / sum_j p_j,   p_j = exp(scale q.k_j - max)
//
// over the keys j < kv_lens[b] with key_mask[b, j]; g = h / (H / Hkv). A row that
// sees no key is 0. A key that is not seen is never used: its score is replaced by
// -inf before anything is computed from it, and its value's row is zeroed on the chip
// (a weight of 0 times a NaN would still be a NaN).
//
// The softmax is one pass over the keys with a running maximum m and sum l, in
// fp32 and base 2: p = 2^(s c - m) with c = scale log2(e). The weights are rounded
// to the inputs' type for the second product (the sum l takes them unrounded).
//
//   tile_kernel   more than 16 query rows per key head: bounded by the tensor cores
//                 and the exponentials. Two tiles of 128 query rows share every key
//                 tile; while one is in its softmax the other has the tensor core.
//   token_kernel  up to 16 query rows per key head (single tokens): bounded by the
//                 bytes of k and v, which go from memory to registers once, in the
//                 layout of the mma operands, without shared memory.
//
// Long contexts with few rows are split over the keys; the parts' (m, l, O) meet in
// shared memory of a cluster (token_kernel) or in the workspace (combine_kernel).
#include <atomic>

#include "sm100.cuh"
#include "srdit_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace srdit {
namespace xattn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int TILE = 128;

struct Args {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  long long qs[3], ks[3], vs[3], os[3];  // {batch, token, head}, elements
  int B, Lq, Lk, H, Hkv, D;
  int group;       // H / Hkv
  int pack;        // tile_kernel: heads of a group side by side in a query tile
  int rt;          // tile_kernel: tokens of a query tile (pack * rt rows)
  int nq, nhp;     // tile_kernel: query-tile pairs per head pack, head packs
  int q_one, k_one, v_one;         // one sample's tensor for all (batch stride 0)
  int k_one_head, v_one_head;      // one key head for all (head stride 0)
  int splits;      // parts of the key range
  int items;       // tile_kernel: work items
  const int32_t* kv_lens;
  const uint8_t* mask;
  long long mask_stride;
  float c;         // scale * log2(e)
  float* ws;       // [parts][rows][D] O, then [parts][rows] {m, l}
  uint32_t* status;
};

SRDIT_DEV float neg_inf() { return -__int_as_float(0x7f800000); }
SRDIT_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
SRDIT_DEV float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
SRDIT_DEV uint32_t pack2(float x, float y, __nv_bfloat16) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(y), "f"(x));
  return d;
}
SRDIT_DEV uint32_t pack2(float x, float y, __half) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(y), "f"(x));
  return d;
}
SRDIT_DEV int key_count(const Args& a, int b) {
  return a.kv_lens ? min(max(__ldg(a.kv_lens + b), 0), a.Lk) : a.Lk;
}

// ---------------------------------------------------------------- tile_kernel
constexpr int TILE_THREADS = 320;  // producer, MMA issuer, 2 x 4 softmax warps

template <int DP>
struct TileCfg {
  static constexpr int SLAB = TILE * 128;  // 128 rows x 64 values
  static constexpr int BYTES = SLAB * (DP / 64);
  static constexpr int STAGES = DP == 128 ? 5 : 10;
  static constexpr int OFF_KV = 2 * BYTES;
  static constexpr int OFF_BAR = OFF_KV + STAGES * BYTES;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static_assert(SMEM <= 232448, "shared memory budget");
};

// One work item: a pair of query tiles of one head pack against one part of a
// sample's keys.
struct Item {
  int b, h0, tok0, part;
  int len;
  int t0, t1;  // key tiles
  bool act1;   // the second query tile has tokens
};
SRDIT_DEV Item item_of(const Args& a, int i) {
  Item o;
  const int qt = i % a.nq;
  i /= a.nq;
  o.h0 = (i % a.nhp) * a.pack;
  i /= a.nhp;
  o.b = i % a.B;
  o.part = i / a.B;
  o.tok0 = qt * 2 * a.rt;
  o.act1 = o.tok0 + a.rt < a.Lq;
  o.len = key_count(a, o.b);
  const int nt = (o.len + TILE - 1) / TILE;
  o.t0 = static_cast<int>(static_cast<long long>(nt) * o.part / a.splits);
  o.t1 = static_cast<int>(static_cast<long long>(nt) * (o.part + 1) / a.splits);
  return o;
}

template <typename T, int DP>
__global__ void __launch_bounds__(TILE_THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Args a) {
  pdl_begin();
  using C = TileCfg<DP>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* q_full = empty + STAGES;  // [2], one per query tile
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_empty + 2;     // scores of a tile ready
  uint64_t* p_full = s_full + 2;      // its weights written (one arrival per warp)
  uint64_t* o_full = p_full + 2;      // its last product done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  static_assert((2 * STAGES + 10) * 8 + 8 <= 256, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    *abort_flag = 0u;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // tensor memory: S0 @0, S1 @128 (weights over the first 64 columns), O0 @256, O1 @384
  const uint32_t tmem_base = *tmem_slot;
  const int step = static_cast<int>(gridDim.x);

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      bool ok = true;
      int idx = 0;              // ring slot uses
      int nq[2] = {0, 0};       // query tiles loaded
      auto load_kv = [&](const CUtensorMap* tm, int tile, int h, int b) {
        const int s = idx % STAGES;
        if (!mbar_wait(&empty[s], (static_cast<uint32_t>(idx / STAGES) & 1u) ^ 1u, a.status,
                       abort_flag))
          return false;
        uint8_t* dst = smem + C::OFF_KV + s * C::BYTES;
        mbar_arrive_expect_tx(&full[s], C::BYTES);
        for (int d = 0; d < DP / 64; ++d)
          tma_load_4d(dst + d * C::SLAB, tm, &full[s], d * 64, h, tile * TILE, b);
        ++idx;
        return true;
      };
      auto load_q = [&](const Item& it, int t) {
        if (!mbar_wait(&q_empty[t], (static_cast<uint32_t>(nq[t]) & 1u) ^ 1u, a.status, abort_flag))
          return false;
        uint8_t* dst = smem + t * C::BYTES;
        mbar_arrive_expect_tx(&q_full[t],
                              static_cast<uint32_t>(a.pack * a.rt * 128 * (DP / 64)));
        for (int d = 0; d < DP / 64; ++d)
          tma_load_4d(dst + d * C::SLAB, &tmQ, &q_full[t], d * 64, it.h0, it.tok0 + t * a.rt,
                      a.q_one ? 0 : it.b);
        ++nq[t];
        return true;
      };
      for (int i = blockIdx.x; i < a.items && ok; i += step) {
        const Item it = item_of(a, i);
        if (it.t0 == it.t1) continue;
        const int g = it.h0 / a.group;
        const int kh = a.k_one_head ? 0 : g, kb = a.k_one ? 0 : it.b;
        const int vh = a.v_one_head ? 0 : g, vb = a.v_one ? 0 : it.b;
        ok = load_q(it, 0) && load_kv(&tmK, it.t0, kh, kb);
        if (ok && it.act1) ok = load_q(it, 1);
        for (int j = it.t0; j < it.t1 && ok; ++j)
          ok = load_kv(&tmV, j, vh, vb) && (j + 1 == it.t1 || load_kv(&tmK, j + 1, kh, kb));
      }
      // having given up, let the loads in flight land before the CTA exits
      if (!ok)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    // S0 S1 | PV0 S0' PV1 S1' | ...: a tile's next scores follow its product, so the
    // weights that share their columns have been read (the tensor core runs in order)
    if (elect_one()) {
      constexpr uint32_t fmt = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
      const uint32_t idesc_s = idesc_make(fmt, fmt, 0u, 0u, 128u, 128u);
      const uint32_t idesc_o = idesc_make(fmt, fmt, 0u, 1u, 128u, static_cast<uint32_t>(DP));
      int idx = 0;
      int nq[2] = {0, 0}, np[2] = {0, 0};
      auto kv_wait = [&](int u) {
        return mbar_wait(&full[u % STAGES], static_cast<uint32_t>(u / STAGES) & 1u, a.status,
                         abort_flag);
      };
      auto scores = [&](int t, int u) {  // S_t = Q_t K^T, K in ring use u
        const uint32_t q_addr = smem_u32(smem + t * C::BYTES);
        const uint32_t k_addr = smem_u32(smem + C::OFF_KV + (u % STAGES) * C::BYTES);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = static_cast<uint32_t>((k >> 2) * C::SLAB + (k & 3) * 32);
          mma_bf16_ss(tmem_base + t * 128u, sdesc_sw128(q_addr + off, 16, 1024),
                      sdesc_sw128(k_addr + off, 16, 1024), idesc_s, k > 0 ? 1u : 0u);
        }
        tc_commit(&s_full[t]);
      };
      auto product = [&](int t, int u, bool first) {  // O_t (+)= P_t V, V in ring use u
        const uint32_t v_addr = smem_u32(smem + C::OFF_KV + (u % STAGES) * C::BYTES);
#pragma unroll
        for (int k = 0; k < TILE / 16; ++k)
          mma_bf16_ts(tmem_base + 256u + t * 128u, tmem_base + t * 128u + k * 8u,
                      sdesc_sw128(v_addr + k * 16 * 128, C::SLAB, 1024), idesc_o,
                      (!first || k > 0) ? 1u : 0u);
      };
      // first item with keys
      int i = blockIdx.x;
      Item it = {};
      auto seek = [&](int from, Item& o) {
        int x = from;
        for (; x < a.items; x += step) {
          o = item_of(a, x);
          if (o.t0 < o.t1) break;
        }
        return x;
      };
      i = seek(i, it);
      bool ok = i < a.items;
      if (ok) {
        ok = mbar_wait(&q_full[0], 0u, a.status, abort_flag) && kv_wait(0);
        if (ok) {
          tc_fence_after();
          scores(0, 0);
          ++nq[0];
          if (it.t1 - it.t0 == 1) tc_commit(&q_empty[0]);
          if (it.act1) {
            ok = mbar_wait(&q_full[1], 0u, a.status, abort_flag);
            if (ok) {
              tc_fence_after();
              scores(1, 0);
              ++nq[1];
              if (it.t1 - it.t0 == 1) tc_commit(&q_empty[1]);
            }
          }
          tc_commit(&empty[0]);
        }
      }
      int j = it.t0;
      while (ok && i < a.items) {
        // the step after (it, j): the item's next key tile, or another item's first
        Item nx = it;
        int ni = i, nj = j + 1;
        const bool last = nj == it.t1;
        if (last) {
          ni = seek(i + step, nx);
          nj = nx.t0;
        }
        const bool more = ni < a.items;
        const int uv = idx + 1, uk = idx + 2;
        ok = kv_wait(uv);
        bool k_ready = false;
        for (int t = 0; t < 2 && ok; ++t) {
          if (t == 0 || it.act1) {
            ok = mbar_wait(&p_full[t], static_cast<uint32_t>(np[t]) & 1u, a.status, abort_flag);
            if (!ok) break;
            tc_fence_after();
            ++np[t];
            product(t, uv, j == it.t0);
            if (last) tc_commit(&o_full[t]);
          }
          if (more && (t == 0 || nx.act1)) {
            if (!k_ready) ok = kv_wait(uk);
            k_ready = true;
            if (ok && last) {
              ok = mbar_wait(&q_full[t], static_cast<uint32_t>(nq[t]) & 1u, a.status, abort_flag);
              ++nq[t];
            }
            if (!ok) break;
            tc_fence_after();
            scores(t, uk);
            if (nj + 1 == nx.t1) tc_commit(&q_empty[t]);
          }
        }
        if (!ok) break;
        tc_commit(&empty[uv % STAGES]);
        if (more) tc_commit(&empty[uk % STAGES]);
        idx += 2;
        it = nx;
        i = ni;
        j = nj;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    const int t = (warp - 2) >> 2;  // query tile
    const int sub = warp & 3;       // tensor-memory lane quarter
    const int row = sub * 32 + lane;
    const uint32_t t_lane = static_cast<uint32_t>(sub * 32) << 16;
    const uint32_t s_tmem = tmem_base + t_lane + t * 128u;
    const uint32_t o_tmem = tmem_base + t_lane + 256u + t * 128u;
    const uint64_t c2 = f2_pack(a.c, a.c);
    const int row_tok = row / a.pack, row_head = row % a.pack;
    const bool row_in = row < a.pack * a.rt;
    int ns = 0, no = 0, idx = 0;
    bool ok = true;
    for (int i = blockIdx.x; i < a.items && ok; i += step) {
      const Item it = item_of(a, i);
      const int n_tiles = it.t1 - it.t0;
      const bool act = t == 0 || it.act1;
      const int tok = it.tok0 + t * a.rt + row_tok;
      const bool row_ok = act && row_in && tok < a.Lq;
      float m = neg_inf(), l = 0.f;
      if (act) {
        for (int j = 0; j < n_tiles; ++j) {
          const int key0 = (it.t0 + j) * TILE;
          const bool masked = a.mask != nullptr || key0 + TILE > it.len;
          uint32_t vis[4];
          if (masked) {
            const uint8_t* mrow = a.mask ? a.mask + it.b * a.mask_stride : nullptr;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int key = key0 + w * 32 + lane;
              vis[w] = __ballot_sync(0xffffffffu,
                                     key < it.len && (!mrow || __ldg(mrow + key) != 0));
            }
            // the values of unseen keys are zeroed: thread r of tile 0 has key r
            if (t == 0) {
              const int u = idx + 2 * j + 1;
              if (!mbar_wait(&full[u % STAGES], static_cast<uint32_t>(u / STAGES) & 1u, a.status,
                             abort_flag)) {
                ok = false;
                break;
              }
              const uint32_t mine = sub == 0 ? vis[0] : sub == 1 ? vis[1] : sub == 2 ? vis[2] : vis[3];
              if (!((mine >> lane) & 1u)) {
                uint8_t* vrow = smem + C::OFF_KV + (u % STAGES) * C::BYTES + row * 128;
                for (int d = 0; d < DP / 64; ++d)
#pragma unroll
                  for (int x = 0; x < 8; ++x)
                    *reinterpret_cast<uint4*>(vrow + d * C::SLAB + x * 16) = make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
            }
          }
          if (!mbar_wait(&s_full[t], static_cast<uint32_t>(ns) & 1u, a.status, abort_flag)) {
            ok = false;
            break;
          }
          ++ns;
          tc_fence_after();
          uint32_t s[4][32];
#pragma unroll
          for (int w = 0; w < 4; ++w) tmem_ld32(s_tmem + w * 32, s[w]);
          tmem_ld_wait();
          if (masked) {
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis[w] >> e) & 1u)) s[w][e] = __float_as_uint(neg_inf());
          }
          float mx[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            mx[w] = __uint_as_float(s[w][0]);
#pragma unroll
            for (int e = 1; e < 31; e += 2)
              mx[w] = max3(mx[w], __uint_as_float(s[w][e]), __uint_as_float(s[w][e + 1]));
            mx[w] = fmaxf(mx[w], __uint_as_float(s[w][31]));
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.c;
          // the maximum moves (and O is rescaled) only when a tile's is 8 above it:
          // weights stay below 2^8 and the quotient is the same
          const bool raise = top > m + 8.f || (m == neg_inf() && top != neg_inf());
          const float m_new = raise ? top : m;
          const float alpha = raise ? ex2(m - m_new) : 1.f;
          m = m_new;
          const float neg_m = m == neg_inf() ? 0.f : -m;
          const uint64_t neg_m2 = f2_pack(neg_m, neg_m);
          if (j > 0 && __any_sync(0xffffffffu, raise)) {
            // scores of this tile are ready, so the product before it is done
#pragma unroll 1
            for (int w = 0; w < DP / 16; ++w) {
              uint32_t o[16];
              tmem_ld16(o_tmem + w * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st16(o_tmem + w * 16, o);
            }
          }
          uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t pw[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 x = f2_split(f2_fma(u64_of(s[w][e], s[w][e + 1]), c2, neg_m2));
              const float p0 = ex2(x.x), p1 = ex2(x.y);
              sum[(e >> 1) & 1] = f2_add(sum[(e >> 1) & 1], f2_pack(p0, p1));
              pw[e >> 1] = pack2(p0, p1, T{});
            }
            tmem_st16(s_tmem + w * 16, pw);
          }
          const float2 sp = f2_split(f2_add(sum[0], sum[1]));
          l = l * alpha + (sp.x + sp.y);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[t]);
        }
        if (!ok) break;
        if (n_tiles > 0) {
          if (!mbar_wait(&o_full[t], static_cast<uint32_t>(no) & 1u, a.status, abort_flag)) {
            ok = false;
            break;
          }
          ++no;
          tc_fence_after();
        }
        // O / l (or, of a part, O, m and l) of this row
        const int head = it.h0 + row_head;
        if (a.splits == 1) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          T* out = static_cast<T*>(a.out) + it.b * a.os[0] + tok * a.os[1] + head * a.os[2];
#pragma unroll 1
          for (int w = 0; w < DP / 16; ++w) {
            uint32_t o[16];
            if (n_tiles > 0) {
              tmem_ld16(o_tmem + w * 16, o);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = 0u;
            }
            uint32_t r[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              r[e] = pack2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv, T{});
            if (row_ok) {
              if (w * 16 < a.D)
                *reinterpret_cast<uint4*>(out + w * 16) = make_uint4(r[0], r[1], r[2], r[3]);
              if (w * 16 + 8 < a.D)
                *reinterpret_cast<uint4*>(out + w * 16 + 8) = make_uint4(r[4], r[5], r[6], r[7]);
            }
          }
        } else {
          const long long rows = static_cast<long long>(a.B) * a.Lq * a.H;
          const long long at = it.part * rows + (static_cast<long long>(it.b) * a.Lq + tok) * a.H + head;
          float* ml = a.ws + a.splits * rows * a.D + at * 2;
          if (row_ok) *reinterpret_cast<float2*>(ml) = make_float2(m, l);
          if (n_tiles > 0) {
            float* po = a.ws + at * a.D;
#pragma unroll 1
            for (int w = 0; w < DP / 16; ++w) {
              uint32_t o[16];
              tmem_ld16(o_tmem + w * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; e += 4)
                if (row_ok && w * 16 + e < a.D)
                  *reinterpret_cast<uint4*>(po + w * 16 + e) =
                      make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            }
          }
        }
        // the next item's first weights, published after this, free O
        tc_fence_before();
      }
      idx += 2 * n_tiles;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- token_kernel
// mma.sync m16n8k16: rows = the query rows of one key head (tokens x grouped
// heads, up to 16). A warp takes blocks of 16 keys. The contraction over the head's
// dims may run in any order, so thread c of a quad holds dims 8c..8c+7 of each 32 (one
// 16-byte load) for both operands; the output's columns may be numbered in any order,
// so lane group g holds value columns 8g..8g+7 of each 64.
constexpr int TOKEN_WARPS = 4;

template <typename T>
SRDIT_DEV void mma16816(float (&d)[4], const uint32_t (&x)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(b0), "r"(b1));
}
SRDIT_DEV uint4 ld16(const void* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}

// blockIdx.x: part of the keys, blockIdx.y: (sample, key head). The parts of a row
// that run as one cluster are joined in its shared memory.
template <typename T, int DP>
__global__ void __launch_bounds__(TOKEN_WARPS * 32)
    token_kernel(const __grid_constant__ Args a, int cluster) {
  pdl_begin();
  constexpr int NC = DP / 32;  // 32-dim pieces of q and k
  constexpr int NV = DP / 64;  // 64-column pieces of v
  __shared__ float so[TOKEN_WARPS][16][DP + 4];
  __shared__ float2 sml[TOKEN_WARPS][16];  // {m, l} of each warp
  __shared__ float co[16][DP + 4];         // the CTA's own part
  __shared__ float2 cml[16];
  if (cluster > 1) cluster_arrive();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int part = blockIdx.x;
  const int b = blockIdx.y / a.Hkv, kvh = blockIdx.y % a.Hkv;
  const int rows = a.Lq * a.group;
  const int len = key_count(a, b);
  const int nblk = (len + 15) / 16;
  const int blk0 = static_cast<int>(static_cast<long long>(nblk) * part / a.splits);
  const int blk1 = static_cast<int>(static_cast<long long>(nblk) * (part + 1) / a.splits);
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + kvh * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + kvh * a.vs[2];
  const uint8_t* mrow = a.mask ? a.mask + b * a.mask_stride : nullptr;

  // row r: token r / group, head kvh * group + r % group
  uint4 qf[2][NC];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = g + 8 * h;
    const T* qp = static_cast<const T*>(a.q) + b * a.qs[0] + (r / a.group) * a.qs[1] +
                  (static_cast<long long>(kvh) * a.group + r % a.group) * a.qs[2];
#pragma unroll
    for (int x = 0; x < NC; ++x)
      qf[h][x] = r < rows && x * 32 + c * 8 < a.D ? ld16(qp + x * 32 + c * 8) : make_uint4(0, 0, 0, 0);
  }
  float o[NV * 8][4];
#pragma unroll
  for (int x = 0; x < NV * 8; ++x)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[x][e] = 0.f;
  float m[2] = {neg_inf(), neg_inf()}, l[2] = {0.f, 0.f};

#pragma unroll 1
  for (int blk = blk0 + warp; blk < blk1; blk += TOKEN_WARPS) {
    const int key0 = blk * 16;
    // k rows g and g + 8 of the block; v rows 2c, 2c + 1, 2c + 8, 2c + 9
    uint4 kf[2][NC], vf[4][NV];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long key = min(key0 + g + 8 * h, len - 1);
#pragma unroll
      for (int x = 0; x < NC; ++x)
        kf[h][x] = x * 32 + c * 8 < a.D ? ld16(kp + key * a.ks[1] + x * 32 + c * 8)
                                        : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long long key = min(key0 + 2 * c + (r & 1) + (r >> 1) * 8, len - 1);
#pragma unroll
      for (int x = 0; x < NV; ++x)
        vf[r][x] = x * 64 + g * 8 < a.D ? ld16(vp + key * a.vs[1] + x * 64 + g * 8)
                                        : make_uint4(0, 0, 0, 0);
    }
    uint32_t vis = 0xffffu;
    if (mrow || key0 + 16 > len) {
      const int key = key0 + (lane & 15);
      vis = __ballot_sync(0xffffffffu, key < len && (!mrow || __ldg(mrow + key) != 0)) & 0xffffu;
      if (vis == 0u) continue;  // warp-uniform
    }
    float s[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[h][e] = 0.f;
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        const uint32_t a0[4] = {qf[0][x].x, qf[1][x].x, qf[0][x].y, qf[1][x].y};
        const uint32_t a1[4] = {qf[0][x].z, qf[1][x].z, qf[0][x].w, qf[1][x].w};
        mma16816<T>(s[h], a0, kf[h][x].x, kf[h][x].y);
        mma16816<T>(s[h], a1, kf[h][x].z, kf[h][x].w);
      }
    }
    if (vis != 0xffffu) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!((vis >> (h * 8 + 2 * c + (e & 1))) & 1u)) s[h][e] = neg_inf();
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!((vis >> (2 * c + (r & 1) + (r >> 1) * 8)) & 1u))
#pragma unroll
          for (int x = 0; x < NV; ++x) vf[r][x] = make_uint4(0, 0, 0, 0);
    }
    // rows g (e = 0, 1) and g + 8 (e = 2, 3), keys 2c, 2c + 1 of both halves
    uint32_t pf[4];
    float alpha[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * a.c;
      const float mn = fmaxf(m[r], top);
      const float neg = mn == neg_inf() ? 0.f : -mn;
      alpha[r] = ex2(m[r] + neg);
      m[r] = mn;
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = ex2(fmaf(s[e >> 1][2 * r + (e & 1)], a.c, neg));
      l[r] = l[r] * alpha[r] + ((p[0] + p[1]) + (p[2] + p[3]));
      pf[r] = pack2(p[0], p[1], T{});
      pf[r + 2] = pack2(p[2], p[3], T{});
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int x = 0; x < NV * 8; ++x) {
        o[x][0] *= alpha[0];
        o[x][1] *= alpha[0];
        o[x][2] *= alpha[1];
        o[x][3] *= alpha[1];
      }
    }
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      const uint32_t r0[4] = {vf[0][x].x, vf[0][x].y, vf[0][x].z, vf[0][x].w};
      const uint32_t r1[4] = {vf[1][x].x, vf[1][x].y, vf[1][x].z, vf[1][x].w};
      const uint32_t r2[4] = {vf[2][x].x, vf[2][x].y, vf[2][x].z, vf[2][x].w};
      const uint32_t r3[4] = {vf[3][x].x, vf[3][x].y, vf[3][x].z, vf[3][x].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // columns 2w (low halves) and 2w + 1 (high halves) of the lane group's eight
        mma16816<T>(o[x * 8 + 2 * w], pf, __byte_perm(r0[w], r1[w], 0x5410),
                    __byte_perm(r2[w], r3[w], 0x5410));
        mma16816<T>(o[x * 8 + 2 * w + 1], pf, __byte_perm(r0[w], r1[w], 0x7632),
                    __byte_perm(r2[w], r3[w], 0x7632));
      }
    }
  }
  // this warp's part to shared memory. Output column n = 2c + (e & 1) of mma x is lane
  // group n's: value column (x / 8) * 64 + n * 8 + x % 8
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = g + 8 * r;
    if (c == 0) sml[warp][row] = make_float2(m[r], l[r]);
    if (row < rows) {
#pragma unroll
      for (int x = 0; x < NV * 8; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          so[warp][row][(x >> 3) * 64 + (2 * c + e) * 8 + (x & 7)] = o[x][2 * r + e];
    }
  }
  __syncthreads();
  // the CTA's part
  for (int x = threadIdx.x; x < rows * DP; x += TOKEN_WARPS * 32) {
    const int row = x / DP, d = x % DP;
    float top = neg_inf();
#pragma unroll
    for (int w = 0; w < TOKEN_WARPS; ++w) top = fmaxf(top, sml[w][row].x);
    float acc = 0.f, sum = 0.f;
    if (top != neg_inf()) {
#pragma unroll
      for (int w = 0; w < TOKEN_WARPS; ++w) {
        const float2 ml = sml[w][row];
        const float f = ex2(ml.x - top);
        acc = fmaf(so[w][row][d], f, acc);
        sum = fmaf(ml.y, f, sum);
      }
    }
    co[row][d] = acc;
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
  // CTA `share` of the cluster joins every shares-th value of the parts
  const long long all_rows = static_cast<long long>(a.B) * a.Lq * a.H;
  const int wparts = a.splits / cluster;
  for (int x = threadIdx.x * shares + share; x < rows * a.D; x += TOKEN_WARPS * 32 * shares) {
    const int row = x / a.D, d = x % a.D;
    float top = neg_inf(), acc = 0.f, sum = 0.f;
    if (cluster > 1) {
      const uint32_t ml0 = smem_u32(&cml[row]), o0 = smem_u32(&co[row][d]);
      float pm[8], pl[8], po[8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        pm[s] = neg_inf();
        pl[s] = po[s] = 0.f;
        if (s < cluster) {
          const uint32_t ra = mapa_shared(ml0, s);
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(pm[s]), "=f"(pl[s]) : "r"(ra));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(po[s]) : "r"(mapa_shared(o0, s)));
        }
        top = fmaxf(top, pm[s]);
      }
      if (top != neg_inf()) {
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          const float f = ex2(pm[s] - top);
          acc = fmaf(po[s], f, acc);
          sum = fmaf(pl[s], f, sum);
        }
      }
    } else {
      top = cml[row].x;
      sum = cml[row].y;
      acc = co[row][d];
    }
    const int tok = row / a.group, head = kvh * a.group + row % a.group;
    if (wparts == 1) {
      static_cast<T*>(a.out)[b * a.os[0] + tok * a.os[1] + head * a.os[2] + d] =
          static_cast<T>(sum == 0.f ? 0.f : acc / sum);
    } else {
      const long long at = (part / cluster) * all_rows + (static_cast<long long>(b) * a.Lq + tok) * a.H + head;
      a.ws[at * a.D + d] = acc;
      if (d == 0)
        *reinterpret_cast<float2*>(a.ws + wparts * all_rows * a.D + at * 2) = make_float2(top, sum);
    }
  }
  if (cluster > 1) {  // no CTA leaves while another reads its shared memory
    cluster_arrive();
    cluster_wait();
  }
}

// ---------------------------------------------------------------- combine_kernel
// One warp per (sample, token, head): joins the parts that went through the workspace.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ Args a, int parts) {
  pdl_begin();
  const long long rows = static_cast<long long>(a.B) * a.Lq * a.H;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const float* ml = a.ws + parts * rows * a.D;
  float top = neg_inf();
  for (int s = lane; s < parts; s += 32) top = fmaxf(top, ml[(s * rows + row) * 2]);
#pragma unroll
  for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.f;
  for (int s = 0; s < parts; ++s) {
    const float2 p = *reinterpret_cast<const float2*>(ml + (s * rows + row) * 2);
    if (p.x == neg_inf()) continue;  // a part that saw no key wrote no O
    const float f = ex2(p.x - top);
    sum = fmaf(p.y, f, sum);
    if (lane * 4 < a.D) {
      const float4 v = *reinterpret_cast<const float4*>(a.ws + (s * rows + row) * a.D + lane * 4);
      acc[0] = fmaf(v.x, f, acc[0]);
      acc[1] = fmaf(v.y, f, acc[1]);
      acc[2] = fmaf(v.z, f, acc[2]);
      acc[3] = fmaf(v.w, f, acc[3]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int h = static_cast<int>(row % a.H);
  const long long bi = row / a.H;
  T* out = static_cast<T*>(a.out) + (bi / a.Lq) * a.os[0] + (bi % a.Lq) * a.os[1] + h * a.os[2];
  if (lane * 4 < a.D)
    *reinterpret_cast<uint2*>(out + lane * 4) =
        make_uint2(pack2(acc[0] * inv, acc[1] * inv, T{}), pack2(acc[2] * inv, acc[3] * inv, T{}));
}

// ---------------------------------------------------------------- launch
// How a call is run: both the launch and the workspace's size go by it.
struct Plan {
  bool token;
  int pack, rt, nq, nhp;
  int splits, cluster, parts;  // parts: partial results per row in the workspace (1: none)
  int items;
};

static Plan make_plan(const srdit_cross_attn_args& a, int sms) {
  Plan p = {};
  const int group = a.H / a.Hkv;
  p.token = static_cast<long long>(a.Lq) * group <= 16;
  p.splits = p.cluster = p.parts = 1;
  if (p.token) {
    // about two CTAs an SM, each with a block of 16 keys per warp at least
    const int pairs = a.B * a.Hkv;
    int want = (2 * sms + pairs - 1) / pairs;
    const int most = (a.Lk + 63) / 64;
    if (want > most) want = most;
    while (p.cluster < 8 && 2 * p.cluster <= want) p.cluster *= 2;
    p.splits = p.cluster;
    if (p.cluster == 8) {
      p.parts = want / 8;
      p.splits = 8 * p.parts;
    }
    return p;
  }
  // as many heads of a group in a tile as fill its rows (94% of them at least)
  p.pack = 1;
  for (int x = group < 128 ? group : 128; x > 1; --x)
    if (group % x == 0 && x * (128 / x) >= 120) {
      p.pack = x;
      break;
    }
  p.rt = 128 / p.pack;
  p.nq = (a.Lq + 2 * p.rt - 1) / (2 * p.rt);
  p.nhp = a.H / p.pack;
  const long long items = static_cast<long long>(p.nq) * p.nhp * a.B;
  const int tiles = (a.Lk + TILE - 1) / TILE;
  if (items * 2 <= sms) {
    long long s = sms / items;
    if (s > tiles / 2) s = tiles / 2;
    if (s > 1) p.splits = p.parts = static_cast<int>(s);
  }
  p.items = static_cast<int>(items * p.splits);
  return p;
}

static int sms_here() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  return num_sms(dev);
}

// a tensor map over [batch, token, head, D] with the given box of heads and tokens;
// dimensions of one entry, and repeated ones (stride 0), have the extent 1
static int map_of(CUtensorMap* m, const void* p, const long long st[3], int B, int L, int H, int D,
                  int box_h, int box_t) {
  const long long row = (D + 7) / 8 * 16;
  const bool ub = B > 1 && st[0] > 0, ut = L > 1 && st[1] > 0, uh = H > 1 && st[2] > 0;
  const long long dims[4] = {D, uh ? H : 1, ut ? L : 1, ub ? B : 1};
  const long long strides[3] = {uh ? st[2] * 2 : row, ut ? st[1] * 2 : row, ub ? st[0] * 2 : row};
  const int box[4] = {64, box_h, box_t, 1};
  return make_tmap_4d(m, p, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, dims, strides, box);
}

template <typename T, int DP>
static int launch_tile(const srdit_cross_attn_args& u, Args& a, const Plan& p, int sms,
                       cudaStream_t stream) {
  using C = TileCfg<DP>;
  auto kern = tile_kernel<T, DP>;
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  if (dev >= kMaxDevices || !attr_done[dev].load(std::memory_order_acquire)) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < kMaxDevices) attr_done[dev].store(true, std::memory_order_release);
  }
  CUtensorMap tq, tk, tv;
  int rc = map_of(&tq, u.q, u.q_stride, u.B, u.Lq, u.H, u.D, p.pack, p.rt);
  // (without keys nothing is loaded: the maps only have to be valid)
  const bool kv = u.Lk > 0;
  if (!rc) rc = map_of(&tk, kv ? u.k : u.q, u.k_stride, kv ? u.B : 1, u.Lk, u.Hkv, u.D, 1, TILE);
  if (!rc) rc = map_of(&tv, kv ? u.v : u.q, u.v_stride, kv ? u.B : 1, u.Lk, u.Hkv, u.D, 1, TILE);
  if (rc) return rc;
  SRDIT_LAUNCH((kern), p.items < sms ? p.items : sms, TILE_THREADS, C::SMEM, stream, tq, tk, tv, a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int DP>
static int launch_token(const Args& a, const Plan& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.B * a.Hkv));
  cfg.blockDim = dim3(TOKEN_WARPS * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, token_kernel<T, DP>, a, p.cluster));
}

template <typename T>
static int run(const srdit_cross_attn_args& u, Args& a, const Plan& p, int sms,
               cudaStream_t stream) {
  int rc;
  if (p.token)
    rc = u.D <= 64 ? launch_token<T, 64>(a, p, stream) : launch_token<T, 128>(a, p, stream);
  else
    rc = u.D <= 64 ? launch_tile<T, 64>(u, a, p, sms, stream)
                   : launch_tile<T, 128>(u, a, p, sms, stream);
  if (rc || p.parts == 1) return rc;
  const long long rows = static_cast<long long>(u.B) * u.Lq * u.H;
  SRDIT_LAUNCH((combine_kernel<T>), static_cast<unsigned>((rows + 7) / 8), 256, 0, stream, a, p.parts);
  return static_cast<int>(cudaGetLastError());
}

// 16-byte rows: base and every stride that is used
static bool check_view(const void* p, const long long st[3], int b, int l, int h) {
  if (reinterpret_cast<uintptr_t>(p) & 15u) return false;
  const int n[3] = {b, l, h};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] < 0 || st[i] % 8)) return false;
  return true;
}

// argument checks; 1: nothing to do
static int check(const srdit_cross_attn_args& a) {
  if (a.B < 0 || a.Lq < 0 || a.Lk < 0 || a.H < 0 || a.Hkv <= 0 || a.H % a.Hkv) return SRDIT_EINVAL;
  if (a.dtype != SRDIT_BF16 && a.dtype != SRDIT_FP16) return SRDIT_EINVAL;
  if (a.B == 0 || a.Lq == 0 || a.H == 0) return 1;
  if (!a.q || !a.out || (a.Lk > 0 && (!a.k || !a.v)) || !(a.scale > 0.f) ||
      a.scale > 3.4028234e38f)
    return SRDIT_EINVAL;
  if (a.D <= 0 || a.D > 128 || a.D % 8) return SRDIT_EUNSUPPORTED;
  if (static_cast<long long>(a.B) * a.Hkv > 65535 ||
      static_cast<long long>(a.B) * a.Lq * a.H > (1ll << 30))
    return SRDIT_EUNSUPPORTED;
  if (!check_view(a.q, a.q_stride, a.B, a.Lq, a.H) || !check_view(a.k, a.k_stride, a.B, a.Lk, a.Hkv) ||
      !check_view(a.v, a.v_stride, a.B, a.Lk, a.Hkv) || !check_view(a.out, a.o_stride, a.B, a.Lq, a.H))
    return SRDIT_EALIGN;
  if (reinterpret_cast<uintptr_t>(a.kv_lens) & 3u) return SRDIT_EALIGN;
  // an output entry is one place; of the inputs, samples and key heads may be repeated
  if ((a.B > 1 && a.o_stride[0] == 0) || (a.Lq > 1 && a.o_stride[1] == 0) ||
      (a.H > 1 && a.o_stride[2] == 0) || (a.Lq > 1 && a.q_stride[1] == 0) ||
      (a.H > 1 && a.q_stride[2] == 0) || (a.Lk > 1 && (a.k_stride[1] == 0 || a.v_stride[1] == 0)))
    return SRDIT_EINVAL;
  return 0;
}

}  // namespace xattn
}  // namespace srdit

using namespace srdit;

extern "C" int srdit_cross_attn_splits(const srdit_cross_attn_args* args) {
  if (!args || xattn::check(*args) != 0) return 1;
  return xattn::make_plan(*args, xattn::sms_here()).parts;
}

extern "C" int srdit_cross_attn(const srdit_cross_attn_args* args, cudaStream_t stream) {
  if (!args) return SRDIT_EINVAL;
  const srdit_cross_attn_args& u = *args;
  const int rc = xattn::check(u);
  if (rc) return rc < 0 ? rc : 0;
  const int sms = xattn::sms_here();
  const xattn::Plan p = xattn::make_plan(u, sms);
  if (p.parts > 1) {
    const long long need = static_cast<long long>(p.parts) * u.B * u.Lq * u.H * (u.D + 2) * 4;
    if (!u.workspace || u.workspace_bytes < need) return SRDIT_EINVAL;
    if (reinterpret_cast<uintptr_t>(u.workspace) & 15u) return SRDIT_EALIGN;
  }
  xattn::Args a = {};
  a.q = u.q;
  a.k = u.k;
  a.v = u.v;
  a.out = u.out;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = u.q_stride[i];
    a.ks[i] = u.k_stride[i];
    a.vs[i] = u.v_stride[i];
    a.os[i] = u.o_stride[i];
  }
  a.B = u.B;
  a.Lq = u.Lq;
  a.Lk = u.Lk;
  a.H = u.H;
  a.Hkv = u.Hkv;
  a.D = u.D;
  a.group = u.H / u.Hkv;
  a.pack = p.pack;
  a.rt = p.rt;
  a.nq = p.nq;
  a.nhp = p.nhp;
  a.splits = p.splits;
  a.items = p.items;
  a.q_one = u.q_stride[0] == 0;
  a.k_one = u.k_stride[0] == 0;
  a.v_one = u.v_stride[0] == 0;
  a.k_one_head = u.k_stride[2] == 0;
  a.v_one_head = u.v_stride[2] == 0;
  a.kv_lens = u.kv_lens;
  a.mask = u.key_mask;
  a.mask_stride = u.mask_stride;
  a.c = u.scale * xattn::kLog2e;
  a.ws = static_cast<float*>(u.workspace);
  a.status = u.status;
  return u.dtype == SRDIT_BF16 ? xattn::run<__nv_bfloat16>(u, a, p, sms, stream)
                               : xattn::run<__half>(u, a, p, sms, stream);
}
