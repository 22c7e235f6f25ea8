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
//                 bytes of k and v, which each warp streams through a ring of its own.
//
// Long contexts with few rows are split over the keys; the parts' (m, l, O) meet in
// shared memory of a cluster (token_kernel) or in the workspace (join_parts_kernel,
// join_ranges_kernel).
#include <atomic>

#include "attn.cuh"
#include "srdit_internal.h"

namespace srdit {
namespace xattn {

constexpr int TILE = 128;

struct Args {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  long long qs[3], os[3];  // {batch, token, head}, elements (k and v go by tensor maps)
  int B, Lq, Lk, H, Hkv, D;
  int group;       // H / Hkv
  int pack;        // tile_kernel: heads of a group side by side in a query tile
  int rt;          // tile_kernel: tokens of a query tile (pack * rt rows)
  int nq, nhp;     // tile_kernel: query-tile pairs per head pack, head packs
  Divisor by_ctas, by_per, by_nq;  // ... by the CTAs, by nq * nhp, by nq
  int q_one, k_one, v_one;         // one sample's tensor for all (batch stride 0)
  int k_one_head, v_one_head;      // one key head for all (head stride 0)
  int ranged;      // tile_kernel: the last round's items are shared out by key tiles
  int splits;      // token_kernel: parts of the key range
  const int32_t* kv_lens;
  const uint8_t* mask;
  long long mask_stride;
  float c;         // scale * log2(e)
  float* ws;       // parts of rows: O
  float* ml;       // ... their {m, l}
  void* cuts;      // tile_kernel: a Cut per CTA
  uint32_t* status;
};

SRDIT_DEV int key_count(const Args& a, int b) {
  return a.kv_lens ? min(max(__ldg(a.kv_lens + b), 0), a.Lk) : a.Lk;
}

// One row of the output from n parts of it in the workspace, by one warp: part p's O at
// row at(p), its {m, l} at ml[at(p)]. Four parts' loads are in flight at a time.
template <typename T, typename At>
SRDIT_DEV void join_rows(const Args& a, int n, At at, const float2* ml, T* out, int lane) {
  float m = neg_inf(), l = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const bool on = lane * 4 < a.D;
  for (int p0 = 0; p0 < n; p0 += 4) {
    float2 pm[4];
    float4 v[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      pm[x] = make_float2(neg_inf(), 0.f);
      v[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p0 + x < n) {
        const long long row = at(p0 + x);
        pm[x] = ml[row];
        if (on) v[x] = *reinterpret_cast<const float4*>(a.ws + row * a.D + lane * 4);
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
      const float g = ex2(pm[x].x - m);
      l = fmaf(pm[x].y, g, l);
      acc[0] = fmaf(v[x].x, g, acc[0]);
      acc[1] = fmaf(v[x].y, g, acc[1]);
      acc[2] = fmaf(v[x].z, g, acc[2]);
      acc[3] = fmaf(v[x].w, g, acc[3]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (on)
    *reinterpret_cast<uint2*>(out + lane * 4) =
        make_uint2(pack2(acc[0] * inv, acc[1] * inv, T{}), pack2(acc[2] * inv, acc[3] * inv, T{}));
}

// ---------------------------------------------------------------- tile_kernel
constexpr int TILE_THREADS = 384;  // producer and MMA issuer, 2 x 4 softmax warps
constexpr int SLOT_ROWS = 2 * TILE;
constexpr int MAX_RANGES = 256;  // CTAs of a launch that may be ranged
constexpr int MAX_LENS = 32;     // samples whose key counts are kept in shared memory

template <int DP>
struct TileCfg {
  static constexpr int SLAB = TILE * 128;  // 128 rows x 64 values
  static constexpr int BYTES = SLAB * (DP / 64);
  static constexpr int STAGES = DP == 128 ? 4 : 10;
  static constexpr int OFF_KV = 2 * BYTES;
  static constexpr int OFF_STG = OFF_KV + STAGES * BYTES;  // 32 rows x 128 bytes per warp
  static constexpr int OFF_LENS = OFF_STG + 8 * 4096;
  static constexpr int OFF_BAR = OFF_LENS + MAX_LENS * 4;
  static constexpr int SMEM = OFF_BAR + 384 + 1024;
  static_assert(SMEM <= 232448, "shared memory budget");
};

// A work item is a pair of query tiles of one head pack against a sample's key tiles
// [t0, t1). Items are ordered by sample, head pack and query tiles, so that items
// which run at the same time share keys.
struct Item {
  int b, h0, tok0, len;
  int t0, t1;
  int slot;   // -1: all of the sample's keys; else where in the workspace the part goes
  int parts;  // of an item that this CTA begins and others end: in how many it is
  bool act1;  // the second query tile has tokens
};

// The items of one CTA: whole items, every gridDim-th one; and (ranged) in place of a last
// round that would leave CTAs idle, an equal share of its items' key-tile steps, whose
// first and last items may be parts of items. Whole rounds come first: their CTAs go through
// a head's keys side by side, out of the same lines of the cache; ranges do not. Parts cost
// a trip through the workspace and a second launch; make_plan compares.
struct Walk {
  const Args& a;
  int cta, ctas;
  int per;              // items per sample
  int b, rest, nt;      // sample, item within it, the sample's key tiles
  int whole;            // items that are taken whole, in rounds of ctas
  int at;               // the next of this CTA's whole items
  int b0, rest0;        // ranged: the first item that is not
  int count;            // ranged: key-tile steps of the ranged items
  int s, s1;            // ranged: this CTA's next step and its end, from the first item's first
  int t0;               // ranged: first key tile of the next item
  bool in_range;

  const int* lens;      // the samples' key counts in shared memory (null: read where needed)

  SRDIT_DEV int keys(int x) const { return lens ? lens[x] : key_count(a, x); }
  SRDIT_DEV int tiles(int x) const { return (keys(x) + TILE - 1) / TILE; }
  // where the ranged steps of a CTA begin (make_plan keeps the product below 2^31)
  SRDIT_DEV int bound(int c) const { return a.by_ctas.div(count * c); }
  // to the n-th item of samples with keys
  SRDIT_DEV void find_item(int n) {
    for (b = 0;; ++b) {
      nt = tiles(b);
      if (nt == 0) continue;
      if (n < per) break;
      n -= per;
    }
    rest = n;
  }
  // to the item and key tile of ranged step x
  SRDIT_DEV void find_step(int x) {
    int r = rest0;
    for (b = b0;; ++b) {
      nt = tiles(b);
      const int n = nt * (per - r);
      if (x < n) break;
      x -= n;
      r = 0;
    }
    rest = r + x / nt;
    t0 = x % nt;
  }
  SRDIT_DEV Walk(const Args& args, int cta_, int ctas_, const int* lens_)
      : a(args), cta(cta_), ctas(ctas_), per(args.nq * args.nhp), b(0), rest(0), nt(0), at(cta_),
        b0(0), rest0(0), count(0), s(0), s1(0), t0(0), in_range(false), lens(lens_) {
    whole = per * a.B;
    if (a.ranged) {  // (make_plan: lens is there)
      int items = 0;
      for (int x = 0; x < a.B; ++x)
        if (keys(x) > 0) items += per;
      whole = items - a.by_ctas.mod(items);
      if (whole < items) {
        find_item(whole);
        b0 = b;
        rest0 = rest;
        count = nt * (per - rest);
        for (int x = b + 1; x < a.B; ++x) count += tiles(x) * per;
      }
      s = bound(cta);
      s1 = bound(cta + 1);
    }
    if (at < whole) {
      if (a.ranged) {
        find_item(at);
      } else {  // of all samples: those without keys are passed over in next()
        b = a.by_per.div(at);
        rest = at - b * per;
        nt = tiles(b);
      }
    }
  }
  SRDIT_DEV void item(Item& o) const {
    o.b = b;
    const int pack = a.by_nq.div(rest);
    o.h0 = pack * a.pack;
    o.tok0 = (rest - pack * a.nq) * 2 * a.rt;
    o.act1 = o.tok0 + a.rt < a.Lq;
    o.len = keys(b);
    o.parts = 0;
  }
  // the next item, or false
  SRDIT_DEV bool next(Item& o) {
    while (at < whole) {
      const bool found = nt > 0;
      if (found) {
        item(o);
        o.t0 = 0;
        o.t1 = nt;
        o.slot = -1;
      }
      at += ctas;
      if (at < whole) {
        rest += ctas;
        if (a.ranged) {
          while (rest >= per || nt == 0) {
            if (nt > 0) rest -= per;
            nt = tiles(++b);
          }
        } else if (rest >= per) {
          const int n = a.by_per.div(rest);
          b += n;
          rest -= n * per;
          nt = tiles(b);
        }
      }
      if (found) return true;
    }
    if (s >= s1) return false;
    if (!in_range) {
      find_step(s);
      in_range = true;
    }
    while (rest >= per || nt == 0) {
      rest = 0;
      nt = tiles(++b);
    }
    item(o);
    o.t0 = t0;
    o.t1 = min(nt, t0 + (s1 - s));
    o.slot = o.t0 > 0 ? 2 * cta : o.t1 < nt ? 2 * cta + 1 : -1;
    if (o.t0 == 0 && o.t1 < nt) {  // this CTA's part and those of the CTAs up to the item's end
      const int end = s + nt;
      o.parts = 2;
      while (bound(cta + o.parts) < end) ++o.parts;
    }
    s += o.t1 - o.t0;
    t0 = 0;
    ++rest;
    return true;
  }
};

// What a CTA leaves for join_ranges_kernel: the item that it begins and does not end, whose
// parts are in its second slot and the first slots of the CTAs after it.
struct Cut {
  int parts, b, h0, tok0;
  int count;  // Walk's, from which the CTAs' ranges follow
  int pad[3];
};

// Warp 0 loads, warp 1 issues the products, warps 4 to 7 and 8 to 11 are the softmax of one
// query tile each, a row a thread, so a row's maximum and sum need no exchange. A key tile of
// a pair is four products of 128 x 128 x DP and 2 x 128 x 128 exponentials: at 128 columns
// 2048 cycles of the tensor core (4096 multiply-adds a cycle) and as many of the unit that
// takes exponentials (16 a cycle); both read 60% busy. What bounds it is the chain of one
// query tile, 3200 cycles a key tile: its scores to registers and their maximum 500, the
// weights 1500 (1160 of a warp that is alone and has no barriers), the second half of its
// product and the next scores 770, and 300 for two barriers between the softmax and the
// tensor core. The other query tile fills in for most of it, but is at the same point.
// Measured: 24 heads of 128, 4096 queries on 8192 keys 324 us, 1.27 PFLOP/s; with the softmax
// left out, the same loads and products take 294 (the clock falls under their power: cuBLAS
// holds 1.39 PFLOP/s in such a loop). 6912 queries on 512 keys 51 us, 0.85 PFLOP/s: an item is
// four key tiles there, and its end (the last product, 64 KB of output through the SM's port)
// 3000 cycles beside their 3400 each; its five rounds are 88% full. 3 x 777 queries on up to
// 1501 masked keys, 16 heads of 64 over 4: 32 us, a masked tile 4000 cycles.
// Slower, or no faster: half of the exponentials as polynomials; two passes over the scores
// (389 us); a warp that applies the mask; a ring of five K or V tiles; ranges in place of whole
// rounds (365); the maximum's comparisons among the exponentials, or none at all, with the
// sum as the test; the two warps of a scheduler taking turns at the exponentials; columns
// of their own for the weights of 64-wide heads, so that scores never wait (336 for 286);
// the mask as bounds from shared memory (77 for 70); rows stored by their threads, 32 bytes
// at a time (53 for 51); a warp's whole rows staged at once with three K or V tiles in place
// of four (50.5 for 51.4, but 332 for 325); the first item found once for all roles (336).
template <typename T, int DP>
__global__ void __launch_bounds__(TILE_THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                const __grid_constant__ Args a) {
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
  uint64_t* p_half = p_full + 2;      // the first half of them
  uint64_t* o_full = p_half + 2;      // its last product done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  int* lens = reinterpret_cast<int*>(smem + C::OFF_LENS);
  static_assert((2 * STAGES + 12) * 8 + 8 <= 384, "barrier area");

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
      mbar_init(&p_half[t], 4);
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
  if (threadIdx.x >= 128 && static_cast<int>(threadIdx.x) - 128 < min(a.B, MAX_LENS))
    lens[threadIdx.x - 128] = key_count(a, threadIdx.x - 128);
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // tensor memory: S0 @0, S1 @128 (weights over the first 64 columns), O0 @256, O1 @384
  const uint32_t tmem_base = *tmem_slot;
  // registers: 104 for the producer's and the issuer's warps, 200 for the softmax's (3 x
  // 128 threads were launched with 168 each)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
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
          if (!mbar_wait(&q_empty[t], (static_cast<uint32_t>(nq[t]) & 1u) ^ 1u, a.status,
                         abort_flag))
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
        Walk walk(a, blockIdx.x, gridDim.x, a.B <= MAX_LENS ? lens : nullptr);
        Item it;
        while (ok && walk.next(it)) {
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
        // O_t (+)= P_t V over the keys 16 k0 to 16 k1, V in ring use u
        auto product = [&](int t, int u, bool first, int k0, int k1) {
          const uint32_t v_addr = smem_u32(smem + C::OFF_KV + (u % STAGES) * C::BYTES);
#pragma unroll
          for (int k = k0; k < k1; ++k)
            mma_bf16_ts(tmem_base + 256u + t * 128u, tmem_base + t * 128u + k * 8u,
                        sdesc_sw128(v_addr + k * 16 * 128, C::SLAB, 1024), idesc_o,
                        (!first || k > 0) ? 1u : 0u);
        };
        Walk walk(a, blockIdx.x, gridDim.x, a.B <= MAX_LENS ? lens : nullptr);
        Item it = {};
        bool on = walk.next(it), ok = on;
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
        while (ok && on) {
          // the step after (it, j): the item's next key tile, or another item's first
          Item nx = it;
          int nj = j + 1;
          const bool last = nj == it.t1;
          bool more = true;
          if (last) {
            more = walk.next(nx);
            nj = nx.t0;
          }
          const int uv = idx + 1, uk = idx + 2;
          ok = kv_wait(uv);
          bool k_ready = false;
          for (int t = 0; t < 2 && ok; ++t) {
            if (t == 0 || it.act1) {
              ok = mbar_wait(&p_half[t], static_cast<uint32_t>(np[t]) & 1u, a.status, abort_flag);
              if (!ok) break;
              tc_fence_after();
              product(t, uv, j == it.t0, 0, 4);
              ok = mbar_wait(&p_full[t], static_cast<uint32_t>(np[t]) & 1u, a.status, abort_flag);
              if (!ok) break;
              tc_fence_after();
              ++np[t];
              product(t, uv, j == it.t0, 4, 8);
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
          on = more;
          j = nj;
        }
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ------------------------------------------------------------ softmax
    const int t = (warp - 4) >> 2;  // query tile
    const int sub = warp & 3;       // tensor-memory lane quarter
    const int row = sub * 32 + lane;
    const uint32_t t_lane = static_cast<uint32_t>(sub * 32) << 16;
    const uint32_t s_tmem = tmem_base + t_lane + t * 128u;
    const uint32_t o_tmem = tmem_base + t_lane + 256u + t * 128u;
    const uint64_t c2 = f2_pack(a.c, a.c);
    uint8_t* stg = smem + C::OFF_STG + (warp - 4) * 4096;
    int ns = 0, no = 0, idx = 0;
    // A wait that runs out sets the abort flag, and those after it end at once: the warp goes
    // through the rest of its item without a branch, so that no lane of it stays behind, and
    // leaves at the item's end. (A vote at every wait: 24 heads of 64, 4096 queries on 8192 keys
    // 296 us in place of 286.)
    Walk walk(a, blockIdx.x, gridDim.x, a.B <= MAX_LENS ? lens : nullptr);
    Item it;
    if (a.ranged && threadIdx.x == 128) reinterpret_cast<Cut*>(a.cuts)[blockIdx.x].parts = 0;
    while (walk.next(it)) {
      const int n_tiles = it.t1 - it.t0;
      const bool act = t == 0 || it.act1;
      float m = neg_inf(), l = 0.f;
      const uint8_t* mrow = a.mask ? a.mask + it.b * a.mask_stride : nullptr;
      // the mask's bytes of this lane's four keys of a tile, read a tile ahead
      uint32_t seen[4];
      auto read_mask = [&](int key0) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int key = key0 + w * 32 + lane;
          seen[w] = key < it.len ? (mrow ? __ldg(mrow + key) : 1u) : 0u;
        }
      };
      if (act) {
        if (mrow) read_mask(it.t0 * TILE);
        for (int j = 0; j < n_tiles; ++j) {
          const int key0 = (it.t0 + j) * TILE;
          const bool masked = a.mask != nullptr || key0 + TILE > it.len;
          uint32_t vis[4];
          if (masked) {
            if (!mrow) read_mask(key0);
#pragma unroll
            for (int w = 0; w < 4; ++w) vis[w] = __ballot_sync(0xffffffffu, seen[w] != 0);
            if (mrow && j + 1 < n_tiles) read_mask(key0 + TILE);
            // the values of unseen keys are zeroed: thread r of tile 0 has key r
            if (t == 0) {
              const int u = idx + 2 * j + 1;
              mbar_wait(&full[u % STAGES], static_cast<uint32_t>(u / STAGES) & 1u, a.status,
                        abort_flag);
              const uint32_t mine =
                  sub == 0 ? vis[0] : sub == 1 ? vis[1] : sub == 2 ? vis[2] : vis[3];
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
          mbar_wait(&s_full[t], static_cast<uint32_t>(ns) & 1u, a.status, abort_flag);
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
            mx[w] = max2(mx[w], __uint_as_float(s[w][31]));
          }
          const float top = max2(max3(mx[0], mx[1], mx[2]), mx[3]) * a.c;
          // the maximum moves (and O is rescaled) only when a tile's is 8 above it:
          // weights stay below 2^8 and the quotient is the same
          // (written so that a NaN raises it too, and stays in l and O)
          const bool raise = !(top <= m + 8.f) && top != neg_inf();
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
          // (all exponents before the first exponential, and the first half published one
          // group late, when its stores are done: 24 heads of 64, 4096 queries on 8192 keys 286
          // us in place of 306; of 128 324 in place of 327)
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 x = f2_split(f2_fma(u64_of(s[w][e], s[w][e + 1]), c2, neg_m2));
              s[w][e] = __float_as_uint(x.x);
              s[w][e + 1] = __float_as_uint(x.y);
            }
          uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t pw[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const uint64_t p2 =
                  f2_pack(ex2(__uint_as_float(s[w][e])), ex2(__uint_as_float(s[w][e + 1])));
              sum[(e >> 1) & 1] = f2_add(sum[(e >> 1) & 1], p2);
              const float2 p = f2_split(p2);
              pw[e >> 1] = pack2(p.x, p.y, T{});
            }
            if (w == 2) {  // the first 64 keys' weights, stored by now: their product can begin
              tmem_st_wait();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&p_half[t]);
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
        mbar_wait(&o_full[t], static_cast<uint32_t>(no) & 1u, a.status, abort_flag);
        if (__any_sync(0xffffffffu, *abort_flag != 0u)) break;
        ++no;
        tc_fence_after();
        // O / l (or, of a part, O, m and l): the warp's 32 rows go through its staging
        // buffer 128 bytes of each at a time
        const float inv = l == 0.f ? 0.f : 1.f / l;
        if (it.slot < 0) {
          // the warp's rows are a box of the output: heads x tokens
          const int tok = it.tok0 + t * a.rt + sub * 32 / a.pack;
          const int head = it.h0 + sub * 32 % a.pack;
#pragma unroll 1
          for (int d = 0; d < DP; d += 64) {
            uint32_t o[2][32];
            tmem_ld32(o_tmem + d, o[0]);
            tmem_ld32(o_tmem + d + 32, o[1]);
            // the box before this one has left the buffer
            if (lane == 0) bulk_wait_group_read0();
            tmem_ld_wait();
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              uint32_t r[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int at = (e & 3) * 8 + y * 2;
                r[y] = pack2(__uint_as_float(o[e >> 2][at]) * inv,
                             __uint_as_float(o[e >> 2][at + 1]) * inv, T{});
              }
              *reinterpret_cast<uint4*>(stg + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                  make_uint4(r[0], r[1], r[2], r[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && tok < a.Lq && d < a.D) {  // boxes start inside the output
              tma_store_4d(&tmO, stg, d, head, tok, it.b);
              bulk_commit_group();
            }
          }
        } else {
          // a part: the slot holds each warp's rows as [D / 32][32 rows][32 values] in the
          // staging buffer's own order, one bulk store per 4 KiB
          const long long box = (static_cast<long long>(it.slot) * 8 + t * 4 + sub) * (DP / 32);
          reinterpret_cast<float2*>(a.ml)[it.slot * SLOT_ROWS + t * TILE + row] = make_float2(m, l);
          if (t == 0 && row == 0 && it.parts) {
            Cut cut = {it.parts, it.b, it.h0, it.tok0, walk.count};
            reinterpret_cast<Cut*>(a.cuts)[blockIdx.x] = cut;
          }
#pragma unroll 1
          for (int d = 0; d < DP / 32; ++d) {
            uint32_t o[32];
            tmem_ld32(o_tmem + d * 32, o);
            if (lane == 0) bulk_wait_group_read0();  // the box before has left the buffer
            tmem_ld_wait();
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 8; ++e)
              *reinterpret_cast<uint4*>(stg + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                  make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                               a.ws + (box + d) * 1024),
                           "r"(smem_u32(stg)), "r"(4096)
                           : "memory");
              bulk_commit_group();
            }
          }
        }
        // the next item's first weights, published after this, free O
        tc_fence_before();
      }
      idx += 2 * n_tiles;
    }
    if (lane == 0) bulk_wait_group_all();
    // samples without keys
    if (a.kv_lens || a.Lk == 0) {
      const int pieces = a.D / 8;
      const int n = a.Lq * a.H * pieces;  // below 2^31: checked at the call
      for (int b = 0; b < a.B; ++b) {
        if (key_count(a, b) > 0) continue;
        for (int x = blockIdx.x * 256 + threadIdx.x - 128; x < n; x += gridDim.x * 256) {
          const int th = x / pieces;
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + b * a.os[0] + (th / a.H) * a.os[1] +
                                    (th % a.H) * a.os[2] + (x - th * pieces) * 8) =
              make_uint4(0, 0, 0, 0);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// One block per JOIN_ROWS rows of the items that the CTAs' ranges cut: joins their parts, two
// rows a warp and four parts' loads in flight. Bounded by their latency: 512 queries on 8192
// keys, 4 heads of 128 take 30.3 us with the join, 256 on 2048, 8 heads of 64 13.9. (Four rows a
// warp, a part at a time: 38.0 and 17.2.)
constexpr int JOIN_ROWS = 16;

template <typename T, int DP>
__global__ void __launch_bounds__(256) join_ranges_kernel(const __grid_constant__ Args a) {
  pdl_begin();
  const Cut cut = reinterpret_cast<const Cut*>(a.cuts)[blockIdx.x];
  if (cut.parts == 0) return;
  constexpr int R = DP / 64;  // rows of a thread: a row of 64 takes half a warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = blockIdx.y >> 1;  // query tile x lane quarter
  const int r0 = (blockIdx.y & 1) * JOIN_ROWS + warp * 2 + (DP == 64 ? lane >> 4 : 0);
  const int quad = lane & 7, d = (lane >> 3) & (DP / 32 - 1);
  float m[R], l[R];
  float4 acc[R];
#pragma unroll
  for (int x = 0; x < R; ++x) {
    m[x] = neg_inf();
    l[x] = 0.f;
    acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int p0 = 0; p0 < cut.parts; p0 += 4) {
    float2 pm[4][R];
    float4 v[4][R];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int cta = static_cast<int>(blockIdx.x) + p0 + y;
      const bool on = p0 + y < cut.parts &&  // and its range is not empty
                      a.by_ctas.div(cut.count * cta) < a.by_ctas.div(cut.count * (cta + 1));
      const int slot = p0 + y == 0 ? 2 * cta + 1 : 2 * cta;
      const float2* ml = reinterpret_cast<const float2*>(a.ml) + slot * SLOT_ROWS + group * 32;
      const float* box = a.ws + (static_cast<long long>(slot) * 8 + group) * (DP / 32) * 1024;
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const int r = r0 + x;
        pm[y][x] = on ? ml[r] : make_float2(neg_inf(), 0.f);
        v[y][x] = on ? *reinterpret_cast<const float4*>(box + (d * 32 + r) * 32 +
                                                        ((quad ^ (r & 7)) << 2))
                     : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int x = 0; x < R; ++x) {
        const float2 q = pm[y][x];
        if (q.x == neg_inf()) continue;  // it saw no key (or the row is none)
        const float mn = max2(m[x], q.x);
        const float f0 = ex2(m[x] - mn), f1 = ex2(q.x - mn);
        m[x] = mn;
        l[x] = l[x] * f0 + q.y * f1;
        acc[x].x = acc[x].x * f0 + v[y][x].x * f1;
        acc[x].y = acc[x].y * f0 + v[y][x].y * f1;
        acc[x].z = acc[x].z * f0 + v[y][x].z * f1;
        acc[x].w = acc[x].w * f0 + v[y][x].w * f1;
      }
  }
  const int col = d * 32 + quad * 4;
#pragma unroll
  for (int x = 0; x < R; ++x) {
    const int r = (group & 3) * 32 + r0 + x, rt = r / a.pack;
    const int tok = cut.tok0 + (group >> 2) * a.rt + rt;
    if (tok >= a.Lq || col >= a.D) continue;
    const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + cut.b * a.os[0] + tok * a.os[1] +
                              (cut.h0 + r % a.pack) * a.os[2] + col) =
        make_uint2(pack2(acc[x].x * inv, acc[x].y * inv, T{}),
                   pack2(acc[x].z * inv, acc[x].w * inv, T{}));
  }
}

// ---------------------------------------------------------------- token_kernel
// mma.sync m16n8k16 with the keys as its rows, S^T = K Q^T and O^T = V^T P^T: the query
// rows of one key head (tokens x grouped heads) are the columns, NT times 8 of them. A warp
// takes blocks of 16 keys. The contraction over the head's dims may run in any order, so
// thread c of a quad holds dims 16c..16c+15 of each 64 (16-byte loads) for both operands;
// O's rows may be numbered in any order, so lane group g holds value columns 8g..8g+7 of
// each 64. The weights change from accumulator to operand layout by movmatrix.
// A warp alone on its scheduler takes 1300 cycles for a block's 230 instructions, nearly all of
// it their latency, so an SM gets three CTAs (168 registers; two of 16 rows), and a warp's
// ring 2 or 3 blocks of 128-wide heads, twice that of 64-wide ones. (Two CTAs with 3 blocks: 4
// x 32768 keys, 32 heads over 8, 86.0 us in place of 80.5, 8 x 512 keys, 24 heads 11.4 in place
// of 10.9; one with 6: 136 and 17.2.)
constexpr int TOKEN_WARPS = 4;

template <int DP, int NT>
struct TokenCfg {
  static constexpr int PER_SM = NT == 1 ? 3 : 2;
  static constexpr int NC = DP / 32;  // 32-dim pieces of q and k
  static constexpr int NV = DP / 64;  // 64-column pieces of v
  static constexpr int SLAB = 16 * 128;         // 16 rows x 64 values, 128-byte swizzle
  static constexpr int BLK = 2 * NV * SLAB;     // a block: k, then v
  static constexpr int STAGES = 6 / PER_SM * (DP == 128 ? 1 : 2);
  static constexpr int RING = TOKEN_WARPS * STAGES * BLK;
  // after the keys: each warp's O [8 NT][DP + 4], then the CTA's, over the ring
  static constexpr int SMEM = RING + 1024;
  static_assert(RING >= (TOKEN_WARPS + 1) * 8 * NT * (DP + 4) * 4, "O fits the ring");
};

// blockIdx.x: part of the keys, blockIdx.y: (sample, key head). The parts of a row
// that run as one cluster are joined in its shared memory.
//
// A warp's ring in shared memory is its own. A block goes to registers whole, and its slot
// is refilled before the block is computed. (Of the ways to fill it, TMA boxes of 16 rows
// keep up with the memory; 16 bytes a lane by cp.async held an SM to 45 GB/s, and a bulk
// copy per row to one row in 8 to 20 cycles.)
// The scores are S^T = K Q^T, 16 keys by 8 rows an instruction, so a row's weights are the
// operand of O^T = V^T P^T as they stand; v is turned in registers, 8 x 8 at a time.
// Measured: 4 x 32768 keys, 32 heads over 8, one token 81 us, 6.63 TB/s (a sum over as many
// bytes reads 5.65); 8 x up to 512 keys, 24 heads 8.2 us: start, one block's latency, join.
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(TOKEN_WARPS * 32, TokenCfg<DP, NT>::PER_SM)
    token_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ Args a, int cluster) {
  pdl_begin();
  using C = TokenCfg<DP, NT>;
  constexpr int NC = C::NC, NV = C::NV, STAGES = C::STAGES, R = 8 * NT;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float(*so)[R][DP + 4] = reinterpret_cast<float(*)[R][DP + 4]>(ring);
  float(*co)[DP + 4] = so[TOKEN_WARPS];   // the CTA's own part
  __shared__ float2 sml[TOKEN_WARPS][R];  // {m, l} of each warp
  __shared__ float2 cml[R];
  __shared__ uint64_t bars[TOKEN_WARPS][STAGES];
  if (cluster > 1) cluster_arrive();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int part = blockIdx.x;
  // samples of different lengths side by side, so that an SM gets some of each
  const int b = blockIdx.y % a.B, kvh = blockIdx.y / a.B;
  const int rows = a.Lq * a.group;
  const int len = key_count(a, b);
  const int nblk = (len + 15) / 16;
  const int blk0 = static_cast<int>(static_cast<long long>(nblk) * part / a.splits);
  const int blk1 = static_cast<int>(static_cast<long long>(nblk) * (part + 1) / a.splits);
  const uint8_t* mrow = a.mask ? a.mask + b * a.mask_stride : nullptr;

  uint64_t* full = bars[warp];
  if (lane == 0) {
    if (warp == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    for (int x = 0; x < STAGES; ++x) mbar_init(&full[x], 1);
    fence_barrier_init();
  }
  uint8_t* mine = ring + warp * STAGES * C::BLK;
  auto fetch = [&](int blk, int slot) {  // by lane 0
    if (blk < blk1) {
      uint8_t* dst = mine + slot * C::BLK;
      mbar_arrive_expect_tx(&full[slot], C::BLK);
#pragma unroll
      for (int x = 0; x < NV; ++x) {
        tma_load_4d(dst + x * C::SLAB, &tmK, &full[slot], x * 64, a.k_one_head ? 0 : kvh, blk * 16,
                    a.k_one ? 0 : b);
        tma_load_4d(dst + (NV + x) * C::SLAB, &tmV, &full[slot], x * 64, a.v_one_head ? 0 : kvh,
                    blk * 16, a.v_one ? 0 : b);
      }
    }
  };
  if (lane == 0) {
#pragma unroll
    for (int x = 0; x < STAGES; ++x) fetch(blk0 + warp + x * TOKEN_WARPS, x);
  }
  __syncwarp();
  // column r: token r / group, head kvh * group + r % group
  uint4 qf[NT][NC];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = g + 8 * n;
    const T* qp = static_cast<const T*>(a.q) + b * a.qs[0] + (r / a.group) * a.qs[1] +
                  (static_cast<long long>(kvh) * a.group + r % a.group) * a.qs[2];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      const int d = (x >> 1) * 64 + c * 16 + (x & 1) * 8;
      qf[n][x] = r < rows && d < a.D ? *reinterpret_cast<const uint4*>(qp + d)
                                     : make_uint4(0, 0, 0, 0);
    }
  }
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

  // a lane's pieces of a swizzled slab: k row g (piece 2c, 2c + 1), v rows 2c and 2c + 1
  // (piece g); every read of 8 lanes meets all banks once
  const uint32_t k_at = static_cast<uint32_t>(g * 128 + (((2 * c) ^ g) << 4));
  const uint32_t v_at = static_cast<uint32_t>(2 * c * 128 + ((g ^ (2 * c)) << 4));
  const uint32_t v_at1 = static_cast<uint32_t>((2 * c + 1) * 128 + ((g ^ (2 * c + 1)) << 4));
  int slot = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (int blk = blk0 + warp; blk < blk1; blk += TOKEN_WARPS) {
    const int key0 = blk * 16;
    uint32_t vis = 0xffffu;
    if (mrow || key0 + 16 > len) {
      const int key = key0 + (lane & 15);
      vis = __ballot_sync(0xffffffffu, key < len && (!mrow || __ldg(mrow + key) != 0)) & 0xffffu;
    }
    if (!mbar_wait_warp(&full[slot], phase, a.status)) {
      // having given up, let the loads in flight land before the ring is used again
      for (int i = 0; i < 200; ++i) __nanosleep(1000);
      break;
    }
    // k rows g and g + 8; v rows 2c, 2c + 1, 2c + 8, 2c + 9
    const uint32_t src = smem_u32(mine) + static_cast<uint32_t>(slot * C::BLK);
    uint4 kf[2][NC], vf[4][NV];
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
    __syncwarp();  // every lane has read the slot
    if (lane == 0) fetch(blk + STAGES * TOKEN_WARPS, slot);
    __syncwarp();
    if (++slot == STAGES) {
      slot = 0;
      phase ^= 1u;
    }
    if (vis != 0xffffu) {  // values of unseen keys: zeros
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!((vis >> (2 * c + (r & 1) + (r >> 1) * 8)) & 1u))
#pragma unroll
          for (int x = 0; x < NV; ++x) vf[r][x] = make_uint4(0, 0, 0, 0);
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
        mma16816<T>(s, kf[0][x].x, kf[1][x].x, kf[0][x].y, kf[1][x].y, qf[n][x].x, qf[n][x].y);
        mma16816<T>(s2, kf[0][x].z, kf[1][x].z, kf[0][x].w, kf[1][x].w, qf[n][x].z, qf[n][x].w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += s2[e];
      if (vis != 0xffffu) {
        if (!((vis >> g) & 1u)) s[0] = s[1] = neg_inf();
        if (!((vis >> (g + 8)) & 1u)) s[2] = s[3] = neg_inf();
      }
      // s[0], s[2]: column 2c, keys g and g + 8; s[1], s[3]: column 2c + 1
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = max2(s[e], s[2 + e]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = max2(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float mn = max2(m[n][e], top * a.c);
        const float neg = mn == neg_inf() ? 0.f : -mn;
        alpha[n][e] = ex2(m[n][e] + neg);
        moved |= mn != m[n][e];
        m[n][e] = mn;
        s[e] = ex2(fmaf(s[e], a.c, neg));
        s[2 + e] = ex2(fmaf(s[2 + e], a.c, neg));
        l[n][e] = fmaf(l[n][e], alpha[n][e], s[e] + s[2 + e]);
      }
      pf[n][0] = transpose8x8(pack2(s[0], s[1], T{}));
      pf[n][1] = transpose8x8(pack2(s[2], s[3], T{}));
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
          mma16816<T>(o[n][x * 4 + w], a0, a1, a2, a3, pf[n][0], pf[n][1]);
      }
    }
  }
  // every warp is done with its ring; O takes its place
  __syncthreads();
  // this warp's part: o[n][x * 4 + w][e] is query column 8n + 2c + (e & 1), value
  // column 64x + 8g + 2w + (e >> 1)
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
        for (int x = 0; x < NV * 4; ++x)
          *reinterpret_cast<float2*>(&so[warp][row][(x >> 2) * 64 + g * 8 + (x & 3) * 2]) =
              make_float2(o[n][x][e], o[n][x][2 + e]);
      }
    }
  }
  __syncthreads();
  // the CTA's part, four columns a thread
  constexpr int DQ = DP / 4;
  for (int x = threadIdx.x; x < rows * DQ; x += TOKEN_WARPS * 32) {
    const int row = x / DQ, d = x % DQ * 4;
    float top = neg_inf();
#pragma unroll
    for (int w = 0; w < TOKEN_WARPS; ++w) top = max2(top, sml[w][row].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    if (top != neg_inf()) {
#pragma unroll
      for (int w = 0; w < TOKEN_WARPS; ++w) {
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
  const long long all_rows = static_cast<long long>(a.B) * a.Lq * a.H;
  const int wparts = a.splits / cluster;
  const int dq = a.D / 4;
  for (int x = threadIdx.x * shares + share; x < rows * dq; x += TOKEN_WARPS * 32 * shares) {
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
    const int tok = row / a.group, head = kvh * a.group + row % a.group;
    if (wparts == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + b * a.os[0] + tok * a.os[1] +
                                head * a.os[2] + d) =
          make_uint2(pack2(acc.x * inv, acc.y * inv, T{}), pack2(acc.z * inv, acc.w * inv, T{}));
    } else {
      const long long at =
          (part / cluster) * all_rows + (static_cast<long long>(b) * a.Lq + tok) * a.H + head;
      *reinterpret_cast<float4*>(a.ws + at * a.D + d) = acc;
      if (d == 0)
        *reinterpret_cast<float2*>(a.ml + at * 2) = make_float2(top, sum);
    }
  }
  if (cluster > 1) {  // no CTA leaves while another reads its shared memory
    cluster_arrive();
    cluster_wait();
  }
}

// One warp per (sample, token, head): joins the parts that went through the workspace.
template <typename T>
__global__ void __launch_bounds__(128)
    join_parts_kernel(const __grid_constant__ Args a, int parts) {
  pdl_begin();
  const long long rows = static_cast<long long>(a.B) * a.Lq * a.H;
  const long long row = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int h = static_cast<int>(row % a.H);
  const long long bi = row / a.H;
  join_rows<T>(a, parts, [&](int p) { return p * rows + row; },
               reinterpret_cast<const float2*>(a.ml),
               static_cast<T*>(a.out) + (bi / a.Lq) * a.os[0] + (bi % a.Lq) * a.os[1] + h * a.os[2],
               threadIdx.x & 31);
}

// ---------------------------------------------------------------- launch
// How a call is run: both the launch and the workspace's size go by it.
struct Plan {
  bool token;
  int pack, rt, nq, nhp;
  int splits, cluster, parts;  // token_kernel; parts in the workspace per row (1: none)
  bool ranged;
  int ctas;                    // tile_kernel
  long long ws_floats(const srdit_cross_attn_args& a) const {
    if (token) return parts > 1 ? static_cast<long long>(parts) * a.B * a.Lq * a.H * (a.D + 2) : 0;
    return ranged ? 2ll * ctas * SLOT_ROWS * ((a.D <= 64 ? 64 : 128) + 2) + 8 * ctas : 0;
  }
};

static Plan make_plan(const srdit_cross_attn_args& a, int sms) {
  Plan p = {};
  const int group = a.H / a.Hkv;
  // 16 rows, token_kernel and tile_kernel: 8 x 512 keys, 24 heads 15.7 and 20.4 us (one row
  // 10.9); 4 x 32768 keys, 8 heads 91 and 118 (four rows 80.7)
  p.token = static_cast<long long>(a.Lq) * group <= 16;
  p.splits = p.cluster = p.parts = 1;
  if (p.token) {
    const int pairs = a.B * a.Hkv;
    const int per_sm = a.Lq * group <= 8 ? TokenCfg<128, 1>::PER_SM : TokenCfg<128, 2>::PER_SM;
    const int blocks = (a.Lk + 15) / 16;
    // The keys are split until every SM has a CTA, each with a block per warp at least (until
    // they have three: 8 x 512 keys, 24 heads 12.5 us in place of 11.7, 8 x 2048 34.4 and 32.7,
    // 8 x 8192 122 and 117; until half of them have one: 4 x 32768, 8 heads 88 and 81), or with
    // samples of different lengths three (8 x up to 2048 22.4 us in place of 27.2, 8 x up to 4096
    // 39.5 and 49.8; six: 26.2 and 42.9).
    const int most = (blocks + TOKEN_WARPS - 1) / TOKEN_WARPS;
    while (p.cluster < 8 && 2 * p.cluster <= most &&
           (pairs * p.cluster < sms || (a.kv_lens && 2 * pairs * p.cluster <= per_sm * sms)))
      p.cluster *= 2;
    p.splits = p.cluster;
    // More than a cluster's 8 parts cost a second launch: from 8 blocks a warp, no more parts
    // than leave it 4, and 1.6 CTAs an SM. (8 heads, 16384 keys: 6 parts 18.8 us, 4 17.4; 3 x
    // 4096, whose clusters have a CTA for each SM: 2 parts 15.6, none 13.1; 1 x 8192: none 15.3,
    // 4 12.9; 2 x 32768: none 52.8, 2 45.2.)
    const int warps = 8 * TOKEN_WARPS;
    if (p.cluster == 8 && blocks >= 8 * warps) {
      p.parts = (sms + 5 * pairs / 2) / (5 * pairs);
      if (p.parts > blocks / (4 * warps)) p.parts = blocks / (4 * warps);
      if (p.parts < 1) p.parts = 1;
      p.splits = 8 * p.parts;
    }
    return p;
  }
  // heads of a group side by side in a query tile, a power of two of them
  p.pack = 1;
  while (p.pack < 128 && group % (2 * p.pack) == 0) p.pack *= 2;
  p.rt = 128 / p.pack;
  p.nq = (a.Lq + 2 * p.rt - 1) / (2 * p.rt);
  p.nhp = a.H / p.pack;
  const long long items = static_cast<long long>(p.nq) * p.nhp * a.B;
  const long long tiles = (a.Lk + TILE - 1) / TILE;
  // A last round of whole items is partly empty (and samples of different lengths, which
  // only the device knows, leave more idle than that); ranges of equal steps are not, but
  // joining their parts costs what 4 steps of the only round do, and 7 of a last one (more
  // CTAs with parts). Ranged and whole: 16 items of 5, 8, 16 key tiles 19.0 and 15.0, 18.3 and
  // 20.5, 23.8 and 34.5 us; 192 items of 8, 12, 16 tiles 42.9 and 39.0, 51.7 and 53.4, 61.6
  // and 67.8 us; 160 items of 8 tiles 39.5 and 38.4.
  if (sms > MAX_RANGES) sms = MAX_RANGES;
  const long long last = items % sms;
  long long ctas = sms;
  if (items < sms) {  // one round
    ctas = last * tiles / 2 < sms ? last * tiles / 2 : sms;
    if (ctas < items) ctas = items;
  }
  const long long idle = last ? tiles - (last * tiles + ctas - 1) / ctas : 0;
  // (the last bound: steps x CTAs in 32 bits)
  p.ranged = a.B <= MAX_LENS && idle > (items < sms ? 4 : 7) && tiles < (1 << 14);
  if (!p.ranged && items < sms) ctas = items;
  p.ctas = static_cast<int>(ctas);
  return p;
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

// k and v in boxes of `rows` keys (without keys nothing is loaded: the maps only have to be
// valid)
static int kv_maps(CUtensorMap* tk, CUtensorMap* tv, const srdit_cross_attn_args& u, int rows) {
  const bool kv = u.Lk > 0;
  const int B = kv ? u.B : 1;
  const int rc = map_of(tk, kv ? u.k : u.q, u.k_stride, B, u.Lk, u.Hkv, u.D, 1, rows);
  return rc ? rc : map_of(tv, kv ? u.v : u.q, u.v_stride, B, u.Lk, u.Hkv, u.D, 1, rows);
}

template <typename T, int DP>
static int launch_tile(const srdit_cross_attn_args& u, Args& a, const Plan& p,
                       cudaStream_t stream) {
  using C = TileCfg<DP>;
  auto kern = tile_kernel<T, DP>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  int rc = set_smem(kern, C::SMEM, attr_done);
  if (rc) return rc;
  CUtensorMap tq, tk, tv, to;
  rc = map_of(&tq, u.q, u.q_stride, u.B, u.Lq, u.H, u.D, p.pack, p.rt);
  if (!rc) rc = kv_maps(&tk, &tv, u, TILE);
  const int box_h = p.pack < 32 ? p.pack : 32;
  if (!rc) rc = map_of(&to, u.out, u.o_stride, u.B, u.Lq, u.H, u.D, box_h, 32 / box_h);
  if (rc) return rc;
  SRDIT_LAUNCH((kern), p.ctas, TILE_THREADS, C::SMEM, stream, tq, tk, tv, to, a);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int DP, int NT>
static int launch_token(const srdit_cross_attn_args& u, const Args& a, const Plan& p,
                        cudaStream_t stream) {
  using C = TokenCfg<DP, NT>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  int rc = set_smem(token_kernel<T, DP, NT>, C::SMEM, attr_done);
  if (rc) return rc;
  CUtensorMap tk, tv;
  rc = kv_maps(&tk, &tv, u, 16);
  if (rc) return rc;
  const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.B * a.Hkv));
  return launch_clusters(p.cluster, token_kernel<T, DP, NT>, grid, TOKEN_WARPS * 32,
                         C::SMEM, stream, tk, tv, a, p.cluster);
}

template <typename T, int DP>
static int launch_token_n(const srdit_cross_attn_args& u, const Args& a, const Plan& p,
                          cudaStream_t stream) {
  return a.Lq * a.group <= 8 ? launch_token<T, DP, 1>(u, a, p, stream)
                             : launch_token<T, DP, 2>(u, a, p, stream);
}

template <typename T>
static int run(const srdit_cross_attn_args& u, Args& a, const Plan& p, cudaStream_t stream) {
  int rc;
  if (p.token)
    rc = u.D <= 64 ? launch_token_n<T, 64>(u, a, p, stream)
                   : launch_token_n<T, 128>(u, a, p, stream);
  else
    rc = u.D <= 64 ? launch_tile<T, 64>(u, a, p, stream) : launch_tile<T, 128>(u, a, p, stream);
  if (rc) return rc;
  if (p.ranged) {
    const dim3 grid(static_cast<unsigned>(p.ctas - 1), SLOT_ROWS / JOIN_ROWS);
    if (u.D <= 64)
      SRDIT_LAUNCH((join_ranges_kernel<T, 64>), grid, 256, 0, stream, a);
    else
      SRDIT_LAUNCH((join_ranges_kernel<T, 128>), grid, 256, 0, stream, a);
    return static_cast<int>(cudaGetLastError());
  }
  if (p.parts == 1) return 0;
  const long long rows = static_cast<long long>(u.B) * u.Lq * u.H;
  SRDIT_LAUNCH((join_parts_kernel<T>), static_cast<unsigned>((rows + 3) / 4), 128, 0, stream, a,
               p.parts);
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
      static_cast<long long>(a.B) * a.Lq * a.H > (1ll << 26))
    return SRDIT_EUNSUPPORTED;
  if (!check_view(a.q, a.q_stride, a.B, a.Lq, a.H) ||
      !check_view(a.k, a.k_stride, a.B, a.Lk, a.Hkv) ||
      !check_view(a.v, a.v_stride, a.B, a.Lk, a.Hkv) ||
      !check_view(a.out, a.o_stride, a.B, a.Lq, a.H))
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

extern "C" int srdit_cross_attn_workspace(const srdit_cross_attn_args* args) {
  if (!args || xattn::check(*args) != 0) return 0;
  const xattn::Plan p = xattn::make_plan(*args, num_sms(device_here()));
  return static_cast<int>((p.ws_floats(*args) + 255) / 256);
}

extern "C" int srdit_cross_attn_items(const srdit_cross_attn_args* args) {
  if (!args || xattn::check(*args) != 0) return 0;
  const xattn::Plan p = xattn::make_plan(*args, num_sms(device_here()));
  return p.token ? 0 : p.nq * p.nhp * args->B;
}

extern "C" int srdit_cross_attn(const srdit_cross_attn_args* args, cudaStream_t stream) {
  if (!args) return SRDIT_EINVAL;
  const srdit_cross_attn_args& u = *args;
  const int rc = xattn::check(u);
  if (rc) return rc < 0 ? rc : 0;
  const xattn::Plan p = xattn::make_plan(u, num_sms(device_here()));
  const long long need = 4 * p.ws_floats(u);
  if (need > 0) {
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
  if (!p.token) {
    a.by_ctas = Divisor::of(p.ctas);
    a.by_per = Divisor::of(p.nq * p.nhp);
    a.by_nq = Divisor::of(p.nq);
  }
  a.splits = p.splits;
  a.ranged = p.ranged;
  a.q_one = u.q_stride[0] == 0;
  a.k_one = u.k_stride[0] == 0;
  a.v_one = u.v_stride[0] == 0;
  a.k_one_head = u.k_stride[2] == 0;
  a.v_one_head = u.v_stride[2] == 0;
  a.kv_lens = u.kv_lens;
  a.mask = u.key_mask;
  a.mask_stride = u.mask_stride;
  a.c = u.scale * kLog2e;
  a.ws = static_cast<float*>(u.workspace);
  if (p.token) {
    a.ml = a.ws + static_cast<long long>(p.parts) * u.B * u.Lq * u.H * u.D;
  } else {
    const long long slots = 2ll * p.ctas * xattn::SLOT_ROWS;
    a.ml = a.ws + slots * (u.D <= 64 ? 64 : 128);
    a.cuts = a.ml + 2 * slots;
  }
  a.status = u.status;
  return u.dtype == SRDIT_BF16 ? xattn::run<__nv_bfloat16>(u, a, p, stream)
                               : xattn::run<__half>(u, a, p, stream);
}
