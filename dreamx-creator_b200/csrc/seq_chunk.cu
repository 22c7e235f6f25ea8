// seq_chunk.cu -- attention of many query rows per key head: whole prompts, and chunks of new
// tokens over the pages of a cache. Bounded by the chain of a query tile, scores, softmax, product:
// 6912 queries on 13824 keys of 24 heads of 128, 16 bits, 970 us at full clocks and 1050 to 1100 in a row,
// where the card's power holds them at 1.6 of 1.97 GHz, 1070 to 1210 TFLOP/s; 2 x 512 on 16384 e4m3 keys,
// 32 heads over 8, 388 us, 700 TFLOP/s.
//
// A work item is up to 2 rt tokens of one sequence with `pack` heads of one group side by side,
// as two query tiles of 128 rows that share every key tile; while one is in its softmax the other
// has the tensor core. A causal item ends at the key tile of its last token, each query tile at
// its own.
//
// Warps: 0 loads keys, values and queries by TMA, 1 issues the products, 2 finds the CTA's items
// and passes them on as records, 3 (16-bit keys) looks over the values of tiles that are partly
// hidden, 4 to 7 and 8 to 11 are the softmax of one query tile each, a row a thread, and with codes
// 12 to 15 widen them in place.
//
// Codes go to the tensor core as fp16, which holds them exactly, and so do the queries.
//   fp16 queries   a key's scale multiplies its scores, a value's its weights, both in fp32
//   bf16 queries   become fp16 times a power of two per row; code times scale is rounded once to
//                  fp16 (an eighth of the answer's rounding), in units that are a power of two per 32
//                  keys
// Either way the running maximum is that of score + exponent of the values' unit, so that the weights
// stay at 2^9 or below, and the sum is of weights in the unit of one. Scales of very different size,
// those of keys that a row does not see among them, are units of their own; where a sum made from
// weights and units would lose a weight beside another's large unit, it is kept with a maximum of its
// own (take_by_key). Scores so large that the rounding of a maximum is more than an exponential takes
// are rounded, with the unit's exponent, before the maximum is taken from them.
#include <atomic>

#include "seq_attn.cuh"

namespace srdit {
namespace sattn {

constexpr int ROWS = 2 * TILE;    // of an item
constexpr int MAX_SLOTS = 192;    // pieces of sequences that are kept in shared memory
constexpr int MIN_SHARE = 4;      // key tiles that a ranged CTA takes at least
constexpr int RECORDS = 4;
constexpr int MAX_SEQS = 64;      // sequences that are kept in shared memory
constexpr int MAX_SORTED = 64;    // pieces that are taken by length
// A weight is 2^(score c - m), its product not rounded and m the rounded one of the largest score:
// from |m| = 2^24 on the two are more than one apart, and that score's weight is any number. So
// where a maximum is FAR or more, products are rounded before m is taken from them. (That branch, not
// taken, costs 1.5% of a long prompt's time over keys in 16 bits, written so; around the exponentials, or
// with the scores taken from tensor memory again, 4% to 7%. Over codes a bound on the scores, or a vote
// on the largest, sends such tiles to code that units of their own need anyway.)
constexpr float FAR = 4194304.f;
// bf16 queries over codes: values' scales that leave every weight that counts in its sum when it is made
// from products of weight and unit: one is lost that is 2^-62 of the largest. With others the sum of
// weights has a maximum of its own.
constexpr float LEAST = 0x1p-44f, MOST = 0x1p20f;

template <int DP, int CODE>
struct ChunkCfg {
  static constexpr bool CODES = CODE != SRDIT_KV_PLAIN;
  static constexpr int THREADS = CODES ? 512 : 384;
  static constexpr int SLAB = TILE * 128;  // 128 rows x 64 values
  static constexpr int BYTES = SLAB * (DP / 64);
  static constexpr int STAGES = DP == 128 ? 4 : CODES ? 6 : 8;
  static constexpr int RAW = BYTES - SLAB;  // where in a stage codes land: its last slab
  static constexpr int OFF_KV = 2 * BYTES;
  static constexpr int OFF_STG = OFF_KV + STAGES * BYTES;  // 32 rows x 64 bytes a warp
  static constexpr int SCALES = 4;         // tiles whose scales are kept: [2][128] each
  static constexpr int OFF_SC = OFF_STG + 8 * 2048;
  static constexpr int OFF_UNITS = OFF_SC + (CODES ? SCALES * 1024 : 0);  // ... and units [3][4]
  static constexpr int OFF_OWN = OFF_UNITS + (CODES ? SCALES * 64 : 0);  // ... or keys' own [2][128]
  static constexpr int OFF_ONE = OFF_OWN + (CODES ? SCALES * 256 : 0);  // units of one: 1, 0, 0
  static constexpr int OFF_MOST = OFF_ONE + (CODES ? 64 : 0);  // queries' largest factors [2][8 warps]
  static constexpr int OFF_Q = OFF_MOST + (CODES ? 64 : 0);    // queries' factors [2][256]
  static constexpr int OFF_REC = OFF_Q + (CODES ? 2048 : 0);
  static constexpr int OFF_PIECES = OFF_REC + RECORDS * 64;
  static constexpr int OFF_STEPS = OFF_PIECES + MAX_SLOTS * 32;  // their first key tiles, order
  static constexpr int OFF_SEQS = OFF_STEPS + (2 * MAX_SLOTS + 4) * 4;
  static constexpr int OFF_GAPS = OFF_SEQS + MAX_SEQS * 16;  // keys without a page, 8 tiles
  static constexpr int GAPS = 8;
  static constexpr int OFF_BAD = OFF_GAPS + GAPS * 16;        // values that are not finite
  static constexpr int OFF_BAR = OFF_BAD + STAGES * 16;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  // What is noted of tile x is written when the stage of its K tile is free. If that was
  // tile y's K tile, the softmax is done with tile y - 1 then, if it was y's V tile, with y.
  static_assert((!CODES || 2 * SCALES >= STAGES + 2) && 2 * GAPS >= STAGES + 2,
                "notes outlive their tile");
  // 16-bit keys: V tiles have stages of their own, whose phases `full` counts
  static_assert(CODES || STAGES % 2 == 0, "K and V tiles alternate");
  static_assert(SMEM <= 232448, "shared memory budget");
};

// Up to 2 rt tokens of a sequence.
struct Piece {
  int row0, tokens;  // first query row; tokens
  int b, pos0;       // sequence; the first token's place in it
  int len, kv0;      // keys; packed: the first one's row
  int e0, e1;        // the ends of the two query tiles' key tiles
  SRDIT_DEV int weight() const { return max(1, max(e0, e1)); }  // key tiles; one without any
};

// What a CTA does next: a piece (tokens 0: nothing more) for a pack of heads, and of its key tiles
// those from t0 on.
struct Record {
  Piece p;
  int h0, g, t0;     // first head, key head
  int part;          // -1: all of the keys; else where in the workspace the part goes
  int parts;         // of an item that this CTA begins and others end: in how many it is
  int pad[3];
  SRDIT_DEV int steps() const { return max(p.e0, p.e1) - t0; }
};

// What a CTA leaves for join_chunk_kernel: the item that it begins and does not end.
struct Cut {
  int parts, row0, tokens, h0;
};

// The pieces of sequences: piece n of sequence b is number begin(b) / (2 rt) + b + n, so that a
// sequence of any length has enough numbers and a search finds it; numbers behind a sequence's
// end are empty.
struct Pieces {
  const Args& a;
  const int4* seqs;  // {begin, end, keys, first key's row} in shared memory, or null

  static SRDIT_DEV int4 sequence(const Args& a, int b) {
    return make_int4(a.rows.begin(b), a.rows.end(b), a.key_count(b),
                     a.paged() ? 0 : a.keys.begin(b));
  }
  SRDIT_DEV int base(int b) const {
    return a.by_piece.div(seqs ? seqs[b].x : a.rows.begin(b)) + b;
  }
  // the last sequence whose base is not above n, by one thread
  SRDIT_DEV int find(int n) const {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (base(mid) <= n) lo = mid; else hi = mid;
    }
    return lo;
  }
  // the same by a warp
  SRDIT_DEV int find_warp(int n) const {
    int lo = 0, count = a.B;
    while (count > 1) {
      const int each = (count + 31) >> 5, at = lo + static_cast<int>(threadIdx.x & 31) * each;
      const unsigned le = __ballot_sync(0xffffffffu, at < lo + count && base(at) <= n);
      const int k = le ? 31 - __clz(le) : 0;
      count = min(each, count - k * each);
      lo += k * each;
    }
    return lo;
  }
  // number n, of sequence b; false: it is empty
  SRDIT_DEV bool piece(int b, int n, Piece& r) const {
    const int4 q = seqs ? seqs[b] : sequence(a, b);
    const int tokens = q.y - q.x;
    const int at = (n - a.by_piece.div(q.x) - b) * 2 * a.rt;
    if (at < 0 || at >= tokens) return false;
    r.b = b;
    r.row0 = q.x + at;
    r.tokens = min(2 * a.rt, tokens - at);
    r.len = q.z;
    r.kv0 = q.w;
    r.pos0 = r.len - tokens + at;
    const int tiles = (r.len + TILE - 1) / TILE;
    auto end = [&](int last) {
      return !a.causal ? tiles : last < 0 ? 0 : min(tiles, last / TILE + 1);
    };
    r.e0 = end(r.pos0 + min(r.tokens, a.rt) - 1);
    r.e1 = r.tokens > a.rt ? end(r.pos0 + r.tokens - 1) : 0;
    return true;
  }
};

// f(first key, scores) of a row's scores, 16 at a time, which may change them: short code, for what is
// not done with every tile.
template <bool kStore, typename F>
SRDIT_DEV void each16(uint32_t s_tmem, F f) {
#pragma unroll 1
  for (int x0 = 0; x0 < TILE; x0 += 16) {
    uint32_t s[16];
    tmem_ld16(s_tmem + x0, s);
    tmem_ld_wait();
    f(x0, s);
    if (kStore) tmem_st16(s_tmem + x0, s);
  }
  if (kStore) tmem_st_wait();
}
// A row's sum of weights apart from O: it is l 2^(base + over) where O's unit is 2^m.
struct Sum {
  float base, over, l;
};
// A row's scores of a tile whose keys and values have units of their own (2^own; or null: the tile's, by
// 32 keys) as those of weights in base 2, rounded, where it sees the key (`seen`); returns the sum of
// the weights in the unit of one, over 2^(the largest score), or adds it to `to`. (Not inlined: hardly
// ever run, and beside the softmax it would displace code that is. Only from kernels that leave the
// warps' registers as they are.)
__device__ __noinline__ float take_by_key(uint32_t s_tmem, uint4 seen, const int8_t* own,
                                          const float* units, float c, Sum* to) {
  auto unit = [&](int x) { return own ? static_cast<float>(own[128 + x]) : units[4 + (x >> 5)]; };
  float top = neg_inf(), sum = 0.f;
  each16<true>(s_tmem, [&](int x0, uint32_t (&s)[16]) {
    const uint32_t vis = (x0 < 32 ? seen.x : x0 < 64 ? seen.y : x0 < 96 ? seen.z : seen.w) >> (x0 & 16);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      const float f = fmaxf(c * (own ? exp2_int(own[x0 + x]) : units[x0 >> 5]), 1.2e-38f);  // (not 0)
      const float y =
          (vis >> x) & 1u ? __fmaf_rn(__uint_as_float(s[x]), f, unit(x0 + x)) : neg_inf();
      top = max2(top, y);
      s[x] = __float_as_uint(y);
    }
  });
  const float neg = top == neg_inf() ? 0.f : -top;
  if (!to) {
    each16<false>(s_tmem, [&](int x0, uint32_t (&s)[16]) {
#pragma unroll
      for (int x = 0; x < 16; ++x)
        sum = fmaf(ex2(__uint_as_float(s[x]) + neg), ex2(-unit(x0 + x)), sum);
    });
    return sum;
  }
  // Scores in two terms, top and the rest, so that large ones keep the units. (The loops are the whole
  // warp's: rows that see no key go through them.)
  float most = neg_inf();
  each16<false>(s_tmem, [&](int x0, uint32_t (&s)[16]) {
#pragma unroll
    for (int x = 0; x < 16; ++x)
      most = max2(most, __uint_as_float(s[x]) + neg - unit(x0 + x));
  });
  if (most == neg_inf()) most = 0.f;
  each16<false>(s_tmem, [&](int x0, uint32_t (&s)[16]) {
#pragma unroll
    for (int x = 0; x < 16; ++x)
      sum += ex2(__uint_as_float(s[x]) + neg - unit(x0 + x) - most);
  });
  if (top != neg_inf()) {
    const float fall = to->base == neg_inf() ? neg_inf() : to->base - top + (to->over - most);
    const bool up = fall <= 0.f;  // (a NaN stays: neither)
    to->l = up ? fmaf(to->l, ex2(fall), sum) : fmaf(sum, ex2(-fall), to->l);
    to->base = up ? top : to->base;
    to->over = up ? most : to->over;
  }
  __syncwarp();
  return 0.f;
}

template <typename T, int DP, int CODE>
__global__ void __launch_bounds__(ChunkCfg<DP, CODE>::THREADS, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Args a,
                 int k_one_head, int v_one_head) {
  pdl_begin();
  using C = ChunkCfg<DP, CODE>;
  using E = typename Compute<T, CODE>::type;
  constexpr int STAGES = C::STAGES;
  constexpr bool CODES = C::CODES;
  // bf16 queries and codes: the queries become fp16, and codes times their scales too
  constexpr bool FOLD = CODES && !__is_same(T, __half);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* loaded = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // by TMA
  uint64_t* full = loaded + STAGES;     // ready for the products
  uint64_t* empty = full + STAGES;
  uint64_t* q_loaded = empty + STAGES;  // [2], one per query tile
  uint64_t* q_full = q_loaded + 2;
  uint64_t* q_empty = q_full + 2;
  uint64_t* s_full = q_empty + 2;     // scores of a tile ready
  uint64_t* p_full = s_full + 2;      // its weights written (one arrival per warp)
  uint64_t* p_half = p_full + 2;      // the first half of them
  uint64_t* o_full = p_half + 2;      // its last product done
  uint64_t* rec_full = o_full + 2;
  uint64_t* rec_empty = rec_full + RECORDS;
  uint64_t* sc_full = rec_empty + RECORDS;  // codes: a tile's scales are there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sc_full + C::SCALES);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  static_assert((3 * STAGES + 14 + 2 * RECORDS + C::SCALES) * 8 + 8 <= 512, "barrier area");
  Record* records = reinterpret_cast<Record*>(smem + C::OFF_REC);
  Piece* kept = reinterpret_cast<Piece*>(smem + C::OFF_PIECES);
  int* starts = reinterpret_cast<int*>(smem + C::OFF_STEPS);  // first key tile of each piece
  int* order = starts + MAX_SLOTS + 4;
  int4* seqs = reinterpret_cast<int4*>(smem + C::OFF_SEQS);
  uint4* gaps = reinterpret_cast<uint4*>(smem + C::OFF_GAPS);  // by tiles, a bit a key
  uint4* bad = reinterpret_cast<uint4*>(smem + C::OFF_BAD);    // by stages

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&loaded[s], 1);
      mbar_init(&full[s], CODES ? 4 : 1);
      mbar_init(&empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_loaded[t], 1);
      mbar_init(&q_full[t], 4);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&p_half[t], 4);
      mbar_init(&o_full[t], 1);
    }
    for (int s = 0; s < RECORDS; ++s) {
      mbar_init(&rec_full[s], 1);
      mbar_init(&rec_empty[s], CODES ? 15 : 11);
    }
    for (int s = 0; s < C::SCALES; ++s) mbar_init(&sc_full[s], 1);
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
  if (FOLD && threadIdx.x < 12)
    reinterpret_cast<float*>(smem + C::OFF_ONE)[threadIdx.x] = threadIdx.x < 4 ? 1.f : 0.f;
  if (warp >= 4 && static_cast<int>(threadIdx.x) - 128 < min(a.B, MAX_SEQS))
    seqs[threadIdx.x - 128] = Pieces::sequence(a, threadIdx.x - 128);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // tensor memory: S0 @0, S1 @128 (weights over the first 64 columns), O0 @256, O1 @384
  const uint32_t tmem_base = *tmem_slot;
  // a tile that some query of the item does not see whole by place
  auto partly = [&](const Record& r, int key0) {
    return key0 + TILE > r.p.len || (a.causal && key0 + TILE - 1 > r.p.pos0);
  };
  if (warp < 4) {
    if constexpr (!CODES)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    else if constexpr (!FOLD)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0) {
      // ------------------------------------------------------------ producer
      // the pages' boxes of a tile side by side: lane l has the box of keys l * box on
      int idx = 0, tiles = 0;   // ring uses, key tiles
      int nq[2] = {0, 0};       // query tiles loaded
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int at = n % RECORDS;
        ok = mbar_wait_warp(&rec_full[at], static_cast<uint32_t>(n / RECORDS) & 1u, a.status,
                            abort_flag);
        if (!ok) break;
        const Record r = records[at];
        __syncwarp();
        if (lane == 0) mbar_arrive(&rec_empty[at]);
        if (r.p.tokens == 0) break;
        if (r.steps() <= 0) continue;
        const int g = r.g;
        const int boxes = TILE >> a.box_log;
        auto load_q = [&](int t) {
          if (!mbar_wait_warp(&q_empty[t], (static_cast<uint32_t>(nq[t]) & 1u) ^ 1u, a.status,
                              abort_flag))
            return false;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_loaded[t], C::BYTES);
            for (int d = 0; d < DP / 64; ++d)
              tma_load_4d(smem + t * C::BYTES + d * C::SLAB, &tmQ, &q_loaded[t], d * 64, r.h0,
                          r.p.row0 + t * a.rt, 0);
          }
          ++nq[t];
          return true;
        };
        // this lane's box of a tile: its page (-1: none) and row; whether keys have no page
        auto place = [&](int tile, int& page, int& row, bool& gap) {
          page = 0;
          row = r.p.kv0 + tile * TILE;
          gap = false;
          if (a.paged()) {
            const int key = tile * TILE + (lane << a.box_log);
            const int p = a.table.by_page.div(key);
            const bool on = lane < boxes && key < r.p.len;
            row = key - p * a.table.page_size;
            page = on ? a.table.page(r.p.b, p) : -1;
            gap = on && page < 0;
          }
        };
        auto load_kv = [&](bool v, int page, int row, bool gap) {
          const CUtensorMap* tm = v ? &tmV : &tmK;
          const int h = (v ? v_one_head : k_one_head) ? 0 : g;
          const int at_page = page >= 0 ? page : max(a.table.pages, 1);  // past the pages: zeros
          const unsigned gap_boxes = __ballot_sync(0xffffffffu, gap);
          const int s = idx % STAGES;
          if (!mbar_wait_warp(&empty[s], (static_cast<uint32_t>(idx / STAGES) & 1u) ^ 1u, a.status,
                              abort_flag))
            return false;
          if (!CODES && !v) {
            if (lane < 4) {
              const uint32_t lo = (gap_boxes >> ((lane * 32) >> a.box_log)) & 1u;
              const uint32_t hi = (gap_boxes >> ((lane * 32 + 16) >> a.box_log)) & 1u;
              reinterpret_cast<uint32_t*>(gaps + tiles % C::GAPS)[lane] =
                  (lo ? 0xffffu : 0u) | (hi ? 0xffff0000u : 0u);
            }
            ++tiles;
            __syncwarp();
          }
          if (lane == 0) mbar_arrive_expect_tx(&loaded[s], CODES ? C::SLAB : C::BYTES);
          __syncwarp();
          uint8_t* dst = smem + C::OFF_KV + s * C::BYTES + (lane << a.box_log) * 128;
          if (lane < boxes) {
            if constexpr (CODES) {
              tma_load_4d(dst + C::RAW, tm, &loaded[s], 0, h, row, at_page);
            } else {
              for (int d = 0; d < DP / 64; ++d)
                tma_load_4d(dst + d * C::SLAB, tm, &loaded[s], d * 64, h, row, at_page);
            }
          }
          ++idx;
          return true;
        };
        int page, row, page1 = 0, row1 = 0;
        bool gap, gap1 = false;
        place(r.t0, page, row, gap);
        ok = (r.p.e0 <= r.t0 || load_q(0)) && load_kv(false, page, row, gap) &&
             (r.p.e1 <= r.t0 || load_q(1));
        const int end = max(r.p.e0, r.p.e1);
        for (int j = r.t0; j < end && ok; ++j) {
          if (j + 1 < end) place(j + 1, page1, row1, gap1);
          ok = load_kv(true, page, row, false) &&
               (j + 1 == end || load_kv(false, page1, row1, gap1));
          page = page1;
          row = row1;
        }
      }
      // having given up, let the loads in flight land before the CTA exits
      if (!ok)
        for (int i = 0; i < 200; ++i) __nanosleep(1000);
    } else if (warp == 1) {
      // ------------------------------------------------------------ MMA issuer
      // S0 S1 | PV0 S0' PV1 S1' | ...: a tile's next scores follow its product, so the
      // weights that share their columns have been read (the tensor core runs in order)
      if (elect_one()) {
        constexpr uint32_t fmt = __is_same(E, __nv_bfloat16) ? 1u : 0u;
        const uint32_t idesc_s = idesc_make(fmt, fmt, 0u, 0u, 128u, 128u);
        const uint32_t idesc_o = idesc_make(fmt, fmt, 0u, 1u, 128u, static_cast<uint32_t>(DP));
        int idx = 0, nrec = 0;
        int nq[2] = {0, 0}, np[2] = {0, 0};
        auto kv_wait = [&](int u, bool v) {
          return mbar_wait((CODES || v ? full : loaded) + u % STAGES,
                           static_cast<uint32_t>(u / STAGES) & 1u, a.status, abort_flag);
        };
        auto q_wait = [&](int t) {
          return mbar_wait((FOLD ? q_full : q_loaded) + t, static_cast<uint32_t>(nq[t]++) & 1u,
                           a.status, abort_flag);
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
        bool ok = true;
        struct Now {
          int t0, e[2], end;
        };
        // The next item with key tiles, of the next `most` records: 1, or 0 if there is none at all, or
        // -1 if it is not among them.
        auto next = [&](Now& r, int most) {
          for (; most > 0; --most) {
            const int at = nrec % RECORDS;
            if (!mbar_wait(&rec_full[at], static_cast<uint32_t>(nrec / RECORDS) & 1u, a.status,
                           abort_flag)) {
              ok = false;
              return 0;
            }
            const int tokens = records[at].p.tokens;
            r.t0 = records[at].t0;
            r.e[0] = records[at].p.e0;
            r.e[1] = records[at].p.e1;
            r.end = max(r.e[0], r.e[1]);
            mbar_arrive(&rec_empty[at]);
            ++nrec;
            if (tokens == 0) return 0;
            if (r.end > r.t0) return 1;
          }
          return -1;
        };
        Now it = {};
        bool begun = false;  // an item's first scores are on their way
        int j = 0;
        while (ok) {
          if (!begun) {
            if (next(it, 0x7fffffff) != 1) break;
            j = it.t0;
            ok = kv_wait(idx, false);
            for (int t = 0; t < 2 && ok; ++t) {
              if (it.e[t] <= it.t0) continue;
              ok = q_wait(t);
              if (!ok) break;
              tc_fence_after();
              scores(t, idx);
              if (it.e[t] - it.t0 == 1) tc_commit(&q_empty[t]);
            }
            if (!ok) break;
            tc_commit(&empty[idx % STAGES]);
            begun = true;
          }
          // The step after (it, j): the item's next key tile, or another item's first. Records come no
          // further than the softmax lets them, which needs this item's products: behind many items
          // without keys the next one is looked for when these are on their way.
          Now nx = it;
          int nj = j + 1;
          const bool last = nj == it.end;
          bool more = true;
          if (last) {
            const int found = next(nx, RECORDS - 1);
            more = found == 1;
            begun = found >= 0;
            nj = nx.t0;
            if (!ok) break;
          }
          const int uv = idx + 1, uk = idx + 2;
          ok = kv_wait(uv, true);
          bool k_ready = false;
          for (int t = 0; t < 2 && ok; ++t) {
            if (j < it.e[t]) {
              ok = mbar_wait(&p_half[t], static_cast<uint32_t>(np[t]) & 1u, a.status, abort_flag);
              if (!ok) break;
              tc_fence_after();
              product(t, uv, j == it.t0, 0, 4);
              ok = mbar_wait(&p_full[t], static_cast<uint32_t>(np[t]) & 1u, a.status, abort_flag);
              if (!ok) break;
              tc_fence_after();
              ++np[t];
              product(t, uv, j == it.t0, 4, 8);
              if (j + 1 == it.e[t]) tc_commit(&o_full[t]);
            }
            if (more && nj < nx.e[t]) {
              if (!k_ready) ok = kv_wait(uk, false);
              k_ready = true;
              if (ok && last) ok = q_wait(t);
              if (!ok) break;
              tc_fence_after();
              scores(t, uk);
              if (nj + 1 == nx.e[t]) tc_commit(&q_empty[t]);
            }
          }
          if (!ok) break;
          tc_commit(&empty[uv % STAGES]);
          if (more) tc_commit(&empty[uk % STAGES]);
          idx += 2;
          if (!begun) continue;
          if (!more) break;
          it = nx;
          j = nj;
        }
      }
      __syncwarp();
    } else if (warp == 2) {
      // ------------------------------------------------------------ items
      // (The code up to the first record is met cold by every CTA, so it is short.)
      const Pieces pieces{a, a.B <= MAX_SEQS ? seqs : nullptr};
      const int cta = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
      int n = 0;
      // piece p for head pack hp, key tiles t0 to t1; by lane 0
      auto pass = [&](const Piece& p, int hp, int t0, int t1, int part, int parts) {
        const int at = n % RECORDS;
        if (!mbar_wait_warp(&rec_empty[at], (static_cast<uint32_t>(n / RECORDS) & 1u) ^ 1u,
                            a.status, abort_flag))
          return false;
        if (lane == 0) {
          Record& r = records[at];
          r.p = p;
          r.p.e0 = max(t0, min(p.e0, t1));
          r.p.e1 = max(t0, min(p.e1, t1));
          r.h0 = hp * a.pack;
          r.g = a.by_packs.div(hp);
          r.t0 = t0;
          r.part = part;
          r.parts = parts;
          mbar_arrive(&rec_full[at]);
        }
        __syncwarp();
        ++n;
        return true;
      };
      bool ok = true;
      constexpr int all_tiles = 0x7fffffff;
      if (a.slots <= MAX_SLOTS) {
        // the pieces that there are
        int total = 0, count = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < a.slots; s0 += 32) {
          const int s = s0 + lane;
          Piece p;
          const bool on = s < a.slots && pieces.piece(pieces.find(s), s, p);
          const int w = on ? p.weight() : 0;
          const unsigned found = __ballot_sync(0xffffffffu, on);
          int sum = w;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
          }
          if (on) {
            const int at = count + __popc(found & ((1u << lane) - 1u));
            kept[at] = p;
            starts[at] = total + sum - w;
          }
          total += __shfl_sync(0xffffffffu, sum, 31);
          count += __popc(found);
        }
        if (lane == 0) starts[count] = total;
        __syncwarp();
        const int items = count * a.nhp;
        if (!a.ranged) {
          // Whole items, one of every gridDim. A few pieces: the longest first; causal: the last ones
          // first; all heads of a piece side by side, in rounds that go forth and back, so that no
          // CTA has the longest of every round. Else a head's pieces, which share its keys, side by
          // side.
          const bool sorted = count <= MAX_SORTED && a.B > 1;
          if (sorted) {
#pragma unroll 1
            for (int k = lane; k < count; k += 32) {
              const int w = starts[k + 1] - starts[k];
              int rank = 0;
              for (int x = 0; x < count; ++x) {
                const int v = starts[x + 1] - starts[x];
                rank += v > w || (v == w && x < k);
              }
              order[rank] = k;
            }
            __syncwarp();
          }
          int step = 2 * (ctas - 1 - cta) + 1;
          for (int x = cta; x < items && ok;) {
            int k, hp;
            if (sorted || a.causal) {
              k = a.by_nhp.div(x);
              hp = x - k * a.nhp;
              k = sorted ? order[k] : count - 1 - k;
              x += step;
              step = 2 * ctas - step;
            } else {
              for (hp = 0, k = x; k >= count; k -= count) ++hp;
              x += ctas;
            }
            ok = pass(kept[k], hp, 0, all_tiles, -1, 0);
          }
        } else {
          // Head pack by head pack. Whole items in rounds as long as every CTA gets one (a.ranged 2),
          // whose CTAs share keys; of the others an equal share of the key tiles.
          // (Loops in place of divisions, which are long code.)
          int whole = 0, hp0 = 0, k0 = 0;
          if (a.ranged == 2) {
            whole = a.by_ctas.div(items) * ctas;
            for (int x = cta, hp = 0, k = cta; x < whole && ok; x += ctas, k += ctas) {
              for (; k >= count; k -= count) ++hp;
              ok = pass(kept[k], hp, 0, all_tiles, -1, 0);
            }
            for (k0 = whole; count > 0 && k0 >= count; k0 -= count) ++hp0;
          }
          const int s0 = hp0 * total + starts[k0];
          const int all = total * a.nhp - s0;
          const int share = max(a.by_ctas.div(all + ctas - 1), MIN_SHARE);
          int s = cta * share;
          const int s1 = min(s + share, all);
          if (lane == 0) static_cast<Cut*>(a.cuts)[cta].parts = 0;
          if (s < s1 && ok) {
            int hp = 0, x = s0 + s;
            for (; x >= total; x -= total) ++hp;
            int k = 0;  // the piece that key tile x is of
            for (int o = 128; o; o >>= 1)
              if (k + o < count && starts[k + o] <= x) k += o;
            while (s < s1 && ok) {
              const int w = starts[k + 1] - starts[k];
              const int t0 = x - starts[k], t1 = min(w, t0 + (s1 - s));
              int parts = 0;
              if (t0 == 0 && t1 < w)
                for (parts = 2; (cta + parts) * share < s + w;) ++parts;
              ok = pass(kept[k], hp, t0, t1, t0 > 0 ? 2 * cta : t1 < w ? 2 * cta + 1 : -1, parts);
              s += t1 - t0;
              x += t1 - t0;
              if (++k == count) {
                k = 0;
                x = 0;
                ++hp;
              }
            }
          }
        }
      } else {
        // more pieces than are kept: whole items, causal the last pieces first, as above
        const int items = a.slots * a.nhp;
        int step = 2 * (ctas - 1 - cta) + 1;
        for (int x = cta; x < items && ok;) {
          int slot, hp;
          if (a.causal) {
            slot = a.by_nhp.div(x);
            hp = x - slot * a.nhp;
            slot = a.slots - 1 - slot;
            x += step;
            step = 2 * ctas - step;
          } else {
            hp = a.by_slots.div(x);
            slot = x - hp * a.slots;
            x += ctas;
          }
          Piece p;
          if (pieces.piece(pieces.find_warp(slot), slot, p)) ok = pass(p, hp, 0, all_tiles, -1, 0);
        }
      }
      if (ok) {
        Piece p = {};
        pass(p, 0, 0, 0, -1, 0);
      }
    } else if constexpr (!CODES) {
      // ------------------------------------------------------------ values of partly hidden tiles
      // Rows behind the sequence become zeros (a weight of 0 times a NaN would be a NaN). Where a
      // causal mask hides some of the tile, so does a row that is not finite, and the queries
      // that see it are told.
      int idx = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int at = n % RECORDS;
        ok = mbar_wait_warp(&rec_full[at], static_cast<uint32_t>(n / RECORDS) & 1u, a.status,
                            abort_flag);
        if (!ok) break;
        const Record r = records[at];
        __syncwarp();
        if (lane == 0) mbar_arrive(&rec_empty[at]);
        if (r.p.tokens == 0) break;
        const int steps = r.steps();
        for (int j = 0; j < steps && ok; ++j) {
          const int u = idx + 2 * j + 1, s = u % STAGES;
          ok = mbar_wait_warp(&loaded[s], static_cast<uint32_t>(u / STAGES) & 1u, a.status,
                              abort_flag);
          if (!ok) break;
          const int key0 = (r.t0 + j) * TILE;
          if (partly(r, key0)) {
#pragma unroll 1
            for (int w = 0; w < 4; ++w) {
              uint8_t* vrow = smem + C::OFF_KV + s * C::BYTES + (w * 32 + lane) * 128;
              const bool behind = key0 + w * 32 + lane >= r.p.len;
              uint32_t m = 0;
              if (!behind && a.causal) {
#pragma unroll
                for (int x = 0; x < DP / 8; ++x) {
                  const uint4 v = *reinterpret_cast<const uint4*>(
                      vrow + (x >> 3) * C::SLAB + (((x + lane) & 7) << 4));
                  m = max_bits(max_bits(max_bits(max_bits(m, v.x), v.y), v.z), v.w);
                }
              }
              const bool off = not_finite<E>(m);
              if (behind || off) {
#pragma unroll
                for (int x = 0; x < DP / 8; ++x)
                  *reinterpret_cast<uint4*>(vrow + (x >> 3) * C::SLAB +
                                            (((x + lane) & 7) << 4)) = make_uint4(0, 0, 0, 0);
              }
              const unsigned all = __ballot_sync(0xffffffffu, off);
              if (lane == 0) reinterpret_cast<uint32_t*>(bad + s)[w] = all;
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&full[s]);
        }
        idx += 2 * max(steps, 0);
      }
    } else {
      // ------------------------------------------------------------ scales of codes
      // The scales of a tile's keys, 0 where there is none, four keys a lane; pages are read two
      // tiles ahead, scales one.
      float* scales = reinterpret_cast<float*>(smem + C::OFF_SC);
      float* units = reinterpret_cast<float*>(smem + C::OFF_UNITS);
      int8_t* own_units = reinterpret_cast<int8_t*>(smem + C::OFF_OWN);
      int idx = 0, tiles = 0;
      bool ok = true;
      for (int n = 0; ok; ++n) {
        const int at = n % RECORDS;
        ok = mbar_wait_warp(&rec_full[at], static_cast<uint32_t>(n / RECORDS) & 1u, a.status,
                            abort_flag);
        if (!ok) break;
        const int t0 = records[at].t0, steps = records[at].steps(), len = records[at].p.len;
        const int b = records[at].p.b, g = records[at].g, tokens = records[at].p.tokens;
        __syncwarp();
        if (lane == 0) mbar_arrive(&rec_empty[at]);
        if (tokens == 0) break;
        const float* ks = a.scale[0] + g * a.ss[0][2];
        const float* vs = a.scale[1] + g * a.ss[1][2];
        auto page_of = [&](int j, int w) {
          const int x = (t0 + j) * TILE + w * 32 + lane;
          return j < steps && x < len ? a.table.page(b, a.table.by_page.div(x)) : -1;
        };
        int page[4], page1[4];
        float k[4], v[4];
        bool apart = false;  // values' scales of the item so far: some beyond LEAST or MOST
        auto fetch = [&](int j) {  // page[]: tile j's
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            k[w] = v[w] = 0.f;
            if (page[w] < 0) continue;
            const int x = (t0 + j) * TILE + w * 32 + lane;
            const long long in = x - a.table.by_page.div(x) * a.table.page_size;
            k[w] = __ldg(ks + page[w] * a.ss[0][0] + in * a.ss[0][1]);
            v[w] = __ldg(vs + page[w] * a.ss[1][0] + in * a.ss[1][1]);
          }
        };
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          page[w] = page_of(0, w);
          page1[w] = page_of(1, w);
        }
        fetch(0);
        for (int j = 0; j < steps && ok; ++j) {
          // the tile's K stage is taken: nobody reads what its place held before
          const int s = idx % STAGES;
          ok = mbar_wait_warp(&loaded[s], static_cast<uint32_t>(idx / STAGES) & 1u, a.status,
                              abort_flag);
          if (!ok) break;
          idx += 2;
          const int place = tiles % C::SCALES;
          float x[8];  // 32 keys' scales, 32 values' scales
          int e[8];
          unsigned gap[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            gap[w] = __ballot_sync(0xffffffffu,
                                   page[w] < 0 && (t0 + j) * TILE + w * 32 + lane < len);
            x[w] = k[w];
            x[4 + w] = v[w];
          }
          bool wide = false;
          if constexpr (FOLD) {
            // 32 keys' scales over 2^e, in [2^6, 2^7) for the largest finite one, so that code times
            // scale, at most 448 x 2^7, is one of fp16. Where one that is not 0 is less than 2^-16 of
            // the largest and would lose bits, every key of the tile has a unit of its own, and from
            // the first value's scale beyond [LEAST, MOST] on every key of the item.
            uint32_t top[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const uint32_t bits = fabsf(x[y]) < 3e38f ? __float_as_uint(fabsf(x[y])) : 0u;
              top[y] = __reduce_max_sync(0xffffffffu, bits);
              const uint32_t least = __reduce_min_sync(0xffffffffu, bits - 1u) + 1u;
              wide |= __uint_as_float(top[y]) > 65536.f * __uint_as_float(least);
              apart |= y >= 4 && (__uint_as_float(top[y]) > MOST ||
                                  (least != 0u && __uint_as_float(least) < LEAST));
            }
            wide |= apart;
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const uint32_t bits = wide ? __float_as_uint(fabsf(x[y])) : top[y];
              e[y] = max(static_cast<int>(bits >> 23) - 133, y < 4 || apart ? -100 : -50);
              x[y] *= exp2_int(-e[y]);
            }
          }
#pragma unroll
          for (int y = 0; y < 8; ++y) scales[place * 256 + y * 32 + lane] = x[y];
          if (lane == 0) gaps[tiles % C::GAPS] = make_uint4(gap[0], gap[1], gap[2], gap[3]);
          if constexpr (FOLD) {
            // units: 2^e of keys; e of values; what makes a sum of weights one in the unit of one; the
            // largest of the first, infinity where keys have their own; whether sums of weights are
            // taken apart from O
            float4* un = reinterpret_cast<float4*>(units + place * 16);
            if (lane == 0) {
              un[0] = make_float4(exp2_int(e[0]), exp2_int(e[1]), exp2_int(e[2]), exp2_int(e[3]));
              un[1] = make_float4(e[4], e[5], e[6], e[7]);
              un[2] = make_float4(exp2_int(-e[4]), exp2_int(-e[5]), exp2_int(-e[6]), exp2_int(-e[7]));
              un[3] = make_float4(wide ? -neg_inf() : exp2_int(max(max(e[0], e[1]), max(e[2], e[3]))),
                                  apart ? 1.f : 0.f, 0.f, 0.f);
            }
            if (wide) {
#pragma unroll
              for (int y = 0; y < 8; ++y)
                own_units[place * 256 + y * 32 + lane] = static_cast<int8_t>(e[y]);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[place]);
          ++tiles;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            page[w] = page1[w];
            page1[w] = page_of(j + 2, w);
          }
          fetch(j + 1);
        }
      }
    }
  } else if (warp < 12) {
    // registers, as 128 threads' shares of what the block was launched with: 104 + 2 x 200 of 3 x
    // 168; fp16 queries over codes 64 + 2 x 192 + 64 of 4 x 128
    if constexpr (!CODES)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    else if constexpr (!FOLD)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ------------------------------------------------------------ softmax
    const int t = (warp - 4) >> 2;  // query tile
    const int sub = warp & 3;       // tensor-memory lane quarter
    const int row = sub * 32 + lane;
    const uint32_t t_lane = static_cast<uint32_t>(sub * 32) << 16;
    const uint32_t s_tmem = tmem_base + t_lane + t * 128u;
    const uint32_t o_tmem = tmem_base + t_lane + 256u + t * 128u;
    uint8_t* stg = smem + C::OFF_STG + (warp - 4) * 2048;
    Sum* own_sum = reinterpret_cast<Sum*>(stg) + lane;  // (until the item's end)
    const float* scales = reinterpret_cast<const float*>(smem + C::OFF_SC);
    const float* q_back = reinterpret_cast<const float*>(smem + C::OFF_Q);
    const float* q_most = reinterpret_cast<const float*>(smem + C::OFF_MOST) + warp - 4;
    const int my_token = t * a.rt + (row >> a.pack_log);
    const int warp_token = t * a.rt + (sub * 32 >> a.pack_log);
    int ns = 0, no = 0, idx = 0, tiles = 0;
    // A wait that runs out sets the abort flag, and those after it end at once: the warp goes
    // through the rest of its item without a branch, so that no lane of it stays behind, and
    // leaves at the item's end.
    for (int n = 0;; ++n) {
      const int at = n % RECORDS;
      if (!mbar_wait_warp(&rec_full[at], static_cast<uint32_t>(n / RECORDS) & 1u, a.status,
                          abort_flag))
        break;
      const Record& rec = records[at];
      const int t0 = rec.t0, e = t ? rec.p.e1 : rec.p.e0, steps = rec.steps();
      const int len = rec.p.len, pos0 = rec.p.pos0, tokens = rec.p.tokens, part = rec.part;
      const int row0 = rec.p.row0, h0 = rec.h0, parts = rec.parts;
      __syncwarp();
      if (lane == 0) mbar_arrive(&rec_empty[at]);
      if (tokens == 0) break;
      const int n_tiles = e - t0;
      float m = neg_inf(), l = 0.f, c = a.c;
      bool far = false;    // a row's maximum is FAR or more
      bool apart = false;  // sums of weights are not in l but in own_sum
      // the last key that this row sees, and the least of its warp's
      const int lim = a.causal ? min(len - 1, pos0 + my_token) : len - 1;
      const int lim0 = a.causal ? min(len - 1, pos0 + warp_token) : len - 1;
      for (int j = 0; j < n_tiles; ++j) {
        const int key0 = (t0 + j) * TILE, u = idx + 2 * j;
        mbar_wait(&s_full[t], static_cast<uint32_t>(ns) & 1u, a.status, abort_flag);
        ++ns;
        tc_fence_after();
        // what was noted before the products that are done now
        if (FOLD && j == 0) c = q_back[(no & 1) * 256 + t * 128 + row];
        const uint4 gap = gaps[tiles % C::GAPS];
        const bool masked = key0 + TILE - 1 > lim0 || (gap.x | gap.y | gap.z | gap.w) != 0u;
        // The maximum moves (and O is rescaled) only when a tile's is 8 above it: weights stay below
        // 2^8 and the quotient is the same. (Written so that a NaN raises it too, and stays in l
        // and O; by the difference, as the sum of a large m and 8 may be m, or far above it.) Scores
        // of this tile are ready, so the product before it is done. Returns the maximum's negative.
        auto new_max = [&](float top) {
          const bool raise = !(top - m <= 8.f) && top != neg_inf();
          const float m_new = raise ? top : m;
          const float alpha = raise ? ex2(m - m_new) : 1.f;
          m = m_new;
          l *= alpha;
          const float neg_m = m == neg_inf() ? 0.f : -m;
          if (__any_sync(0xffffffffu, raise)) {
            if (!CODES) far = __any_sync(0xffffffffu, fabsf(neg_m) >= FAR);
            if (j > 0) {
#pragma unroll 1
            for (int w = 0; w < DP / 16; ++w) {
              uint32_t o[16];
              tmem_ld16(o_tmem + w * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
              tmem_st16(o_tmem + w * 16, o);
            }
            }
          }
          return neg_m;
        };
        // the first 64 keys' weights, stored by now: their product can begin
        auto publish_half = [&] {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[t]);
        };
        // the keys from key0 + 32 w on that this row sees
        auto seen = [&](int w) {
          const int count = lim - key0 + 1 - 32 * w;
          const uint32_t none = w == 0 ? gap.x : w == 1 ? gap.y : w == 2 ? gap.z : gap.w;
          return (count >= 32 ? 0xffffffffu : count <= 0 ? 0u : (1u << count) - 1u) & ~none;
        };
        if constexpr (CODES) {
          // Two passes over the scores, 64 of them at a time, so that the code is short: with all 128
          // in registers at once, as below, it does not fit the instruction caches beside that of the
          // warps that widen codes. (2 x 512 queries on 16384 e4m3 keys, 32 heads over 8 of 128, when this
          // was chosen: 421 us so, 406 in passes of 32, 361 in passes of 64; masks, which few tiles need, as
          // a short loop over the scores before took 3% off. With what large scores and scales far apart
          // need 388; the same keys in 16 bits 264 to 297, by the clocks.)
          const float* sc = scales + (tiles % C::SCALES) * 256;
          const float* units =
              reinterpret_cast<const float*>(smem + C::OFF_UNITS) + tiles % C::SCALES * 16;
          // keys have units of their own, or a score may be 2^25 and more, so that its product with the
          // factor is to be rounded first: one of fp16 queries and codes times scales is below 2^38
          const bool by_key = FOLD && !(units[12] * q_most[(no & 1) * 8] < 0x1p-13f);
          // the scores of keys 64 h on, which have been asked for, as they count
          // (fp16 queries: the scales of 64 keys or values are read while the scores are on their way)
          auto read = [&](const float* from, float4 (&f)[16]) {
#pragma unroll
            for (int x = 0; x < 16; ++x) f[x] = *reinterpret_cast<const float4*>(from + 4 * x);
          };
          auto finish = [&](int h, uint32_t (&s)[2][32]) {
            if constexpr (FOLD) {
              tmem_ld_wait();
            } else {
              float4 k[16];
              read(sc + h * 64, k);
              tmem_ld_wait();
#pragma unroll
              for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int x = 0; x < 32; x += 4) {
                  const float4 f = k[y * 8 + x / 4];
                  const float2 y0 = f2_split(f2_mul(u64_of(s[y][x], s[y][x + 1]), f2_pack(f.x, f.y)));
                  const float2 y1 =
                      f2_split(f2_mul(u64_of(s[y][x + 2], s[y][x + 3]), f2_pack(f.z, f.w)));
                  s[y][x] = __float_as_uint(y0.x);
                  s[y][x + 1] = __float_as_uint(y0.y);
                  s[y][x + 2] = __float_as_uint(y1.x);
                  s[y][x + 3] = __float_as_uint(y1.y);
                }
            }
            if (!FOLD && masked) {
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t vis = seen(2 * h + y);
#pragma unroll
                for (int x = 0; x < 32; ++x)
                  if (!((vis >> x) & 1u)) s[y][x] = __float_as_uint(neg_inf());
              }
            }
          };
          auto ask = [&](int h, uint32_t (&s)[2][32]) {
            tmem_ld32(s_tmem + h * 64, s[0]);
            tmem_ld32(s_tmem + h * 64 + 32, s[1]);
          };
          float sum_of = 0.f;
          if (FOLD && by_key) {
            if (!apart && units[13] != 0.f) {
              apart = true;
              *own_sum = {m, 0.f, l};
              l = 0.f;
            }
            const int8_t* own =
                reinterpret_cast<const int8_t*>(smem) + C::OFF_OWN + tiles % C::SCALES * 256;
            sum_of = take_by_key(s_tmem, make_uint4(seen(0), seen(1), seen(2), seen(3)),
                                 units[12] > 3e38f ? own : nullptr, units, c, apart ? own_sum : nullptr);
            units = reinterpret_cast<const float*>(smem + C::OFF_ONE);
          } else if (FOLD && masked) {
            each16<true>(s_tmem, [&](int x0, uint32_t (&s)[16]) {
              const uint32_t vis = seen(x0 >> 5) >> (x0 & 16);
#pragma unroll
              for (int x = 0; x < 16; ++x)
                if (!((vis >> x) & 1u)) s[x] = __float_as_uint(neg_inf());
            });
          }
          float cj = FOLD && by_key ? 1.f : c;
          // per 32 keys: the scores' factor, and log2 of the unit that the values are in
          auto factor = [&](int w) {
            return FOLD ? fmaxf(cj * units[w], 1.2e-38f) : cj;  // (0 times -inf is NaN)
          };
          float top = neg_inf();
          bool odd = false;  // values of the tile are not finite and hidden from some rows
          // fp16 queries: the exponent of the unit that weights are in, by keys or of all: that of a
          // value's scale (of 2^-100 to 2^100)
          auto exponent = [](float v) {
            v = fminf(fmaxf(v < 3e38f ? v : 0.f, 1e-30f), 1e30f);
            return static_cast<float>(static_cast<int>(__float_as_uint(v) >> 23) - 127);
          };
          bool taken = false;  // m, from scores
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            uint32_t s[2][32];
            ask(h, s);
            finish(h, s);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float mx = __uint_as_float(s[y][0]);
#pragma unroll
              for (int x = 1; x < 31; x += 2)
                mx = max3(mx, __uint_as_float(s[y][x]), __uint_as_float(s[y][x + 1]));
              mx = max2(mx, __uint_as_float(s[y][31]));
              top = max2(top, fmaf(mx, factor(2 * h + y), FOLD ? units[4 + 2 * h + y] : 0.f));
            }
            if constexpr (!FOLD) {  // as they count: the scales are read once
              tmem_st32(s_tmem + h * 64, s[0]);
              tmem_st32(s_tmem + h * 64 + 32, s[1]);
            }
          }
          if constexpr (!FOLD) tmem_st_wait();
          if constexpr (!FOLD) {  // the values' scales are there with the V tile
            mbar_wait(&full[(u + 1) % STAGES], static_cast<uint32_t>((u + 1) / STAGES) & 1u,
                      a.status, abort_flag);
            float most = 0.f, least = 3e38f;  // of the finite ones but 0
            bool not_all = false;             // finite
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float v = fabsf(sc[128 + w * 32 + lane]);
              most = fmaxf(most, v < 3e38f ? v : 0.f);
              least = fminf(least, v > 0.f ? v : 3e38f);
              not_all |= !(v < 3e38f);
            }
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
            least = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(least)));
            const bool large = fabsf(top) >= FAR && fabsf(top) < -neg_inf();
            taken = most > 256.f * least || __any_sync(0xffffffffu, large);
            if (taken) {
              // Products of weights and scales are to be 2^9 at most, but not all far below it, as
              // where the largest scale is one that the row does not see: by key. Scores become
              // exponents, the large ones' products with c rounded before m is taken from them. (Column
              // by column: the shortest code.)
              top = neg_inf();
              auto each = [&](bool store, auto f) {
#pragma unroll 1
                for (int x = 0; x < TILE; ++x) {
                  const float s = __uint_as_float(tmem_ld1(s_tmem + x));
                  tmem_ld_wait();
                  const float in = exponent(fabsf(sc[128 + x])), y = f(__fmaf_rn(s, c, in), in);
                  if (store) tmem_st1(s_tmem + x, __float_as_uint(y));
                }
              };
              each(false, [&](float y, float) {
                top = max2(top, y);
                return y;
              });
              const float m_new = !(top - m <= 8.f) && top != neg_inf() ? top : m;
              const float neg = m_new == neg_inf() ? 0.f : -m_new;
              each(true, [&](float y, float in) { return __fadd_rn(y, neg) - in; });
              tmem_st_wait();
              cj = 1.f;
            } else {
              top += exponent(most);
            }
            odd = masked && __any_sync(0xffffffffu, not_all);
          }
          float neg_m = new_max(top);
          if (taken) neg_m = 0.f;
          if (FOLD) l = fmaf(sum_of, ex2(top + neg_m), l);
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            uint32_t s[2][32];
            ask(h, s);
            if (h) publish_half();
            float4 values[16];
            if constexpr (FOLD) {
              finish(h, s);
            } else {
              read(sc + 128 + h * 64, values);
              tmem_ld_wait();
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              uint32_t pw[16];
              const float lv = FOLD ? units[4 + 2 * h + y] : 0.f, cw = factor(2 * h + y);
              const uint64_t c2 = f2_pack(cw, cw), neg_m2 = f2_pack(neg_m + lv, neg_m + lv);
              uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
              for (int x = 0; x < 32; x += 2) {
                const float2 z = f2_split(f2_fma(u64_of(s[y][x], s[y][x + 1]), c2, neg_m2));
                s[y][x] = __float_as_uint(z.x);
                s[y][x + 1] = __float_as_uint(z.y);
              }
#pragma unroll
              for (int x = 0; x < 32; x += 4) {
                const uint64_t p0 =
                    f2_pack(ex2(__uint_as_float(s[y][x])), ex2(__uint_as_float(s[y][x + 1])));
                const uint64_t p1 =
                    f2_pack(ex2(__uint_as_float(s[y][x + 2])), ex2(__uint_as_float(s[y][x + 3])));
                sum[0] = f2_add(sum[0], p0);
                sum[1] = f2_add(sum[1], p1);
                float2 y0 = f2_split(p0), y1 = f2_split(p1);
                if constexpr (!FOLD) {
                  const float4 v = values[y * 8 + x / 4];
                  y0 = f2_split(f2_mul(p0, f2_pack(v.x, v.y)));
                  y1 = f2_split(f2_mul(p1, f2_pack(v.z, v.w)));
                }
                pw[x >> 1] = pack2(y0.x, y0.y, E{});
                pw[(x >> 1) + 1] = pack2(y1.x, y1.y, E{});
              }
              if (!FOLD && odd) {  // (a scale that is not finite stays with the rows that see its key)
                const uint32_t vis = seen(2 * h + y);
#pragma unroll
                for (int x = 0; x < 16; ++x)
                  pw[x] &= ((vis >> (2 * x)) & 1u ? 0xffffu : 0u) |
                           ((vis >> (2 * x + 1)) & 1u ? 0xffff0000u : 0u);
              }
              const float2 sp = f2_split(f2_add(sum[0], sum[1]));
              l = fmaf(sp.x + sp.y, FOLD ? units[8 + 2 * h + y] : 1.f, l);  // in the unit of one
              tmem_st16(s_tmem + h * 32 + y * 16, pw);
            }
          }
        } else {
          uint32_t s[4][32];
#pragma unroll
          for (int w = 0; w < 4; ++w) tmem_ld32(s_tmem + w * 32, s[w]);
          tmem_ld_wait();
          if (masked) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t vis = seen(w);
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (!((vis >> x) & 1u)) s[w][x] = __float_as_uint(neg_inf());
            }
          }
          float mx[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            mx[w] = __uint_as_float(s[w][0]);
#pragma unroll
            for (int x = 1; x < 31; x += 2)
              mx[w] = max3(mx[w], __uint_as_float(s[w][x]), __uint_as_float(s[w][x + 1]));
            mx[w] = max2(mx[w], __uint_as_float(s[w][31]));
          }
          float neg_m = new_max(max2(max3(mx[0], mx[1], mx[2]), mx[3]) * c);
          if (far) {  // scores that times c are what is to be the exponent
            const float inv = 1.f / c;
#pragma unroll
            for (int w = 0; w < 4; ++w)
#pragma unroll
              for (int x = 0; x < 32; ++x)
                s[w][x] = __float_as_uint(
                    __fadd_rn(__fmul_rn(__uint_as_float(s[w][x]), c), neg_m) * inv);
            neg_m = 0.f;
          }
          const uint64_t c2 = f2_pack(c, c), neg_m2 = f2_pack(neg_m, neg_m);
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const float2 y = f2_split(f2_fma(u64_of(s[w][x], s[w][x + 1]), c2, neg_m2));
              s[w][x] = __float_as_uint(y.x);
              s[w][x + 1] = __float_as_uint(y.y);
            }
          uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t pw[16];
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const uint64_t p2 =
                  f2_pack(ex2(__uint_as_float(s[w][x])), ex2(__uint_as_float(s[w][x + 1])));
              sum[(x >> 1) & 1] = f2_add(sum[(x >> 1) & 1], p2);
              const float2 p = f2_split(p2);
              pw[x >> 1] = pack2(p.x, p.y, E{});
            }
            if (w == 2) publish_half();
            tmem_st16(s_tmem + w * 16, pw);
          }
          const float2 sp = f2_split(f2_add(sum[0], sum[1]));
          l += sp.x + sp.y;
        }
        if constexpr (!CODES || FOLD) {
          // values taken out, as not finite (of 16 bits, only where a causal mask hides some)
          if ((a.causal && key0 + TILE - 1 > pos0) || (FOLD && key0 + TILE > len)) {
            mbar_wait(&full[(u + 1) % STAGES], static_cast<uint32_t>((u + 1) / STAGES) & 1u,
                      a.status, abort_flag);
            uint4 off = bad[(u + 1) % STAGES];
            if (masked)
              off = make_uint4(off.x & seen(0), off.y & seen(1), off.z & seen(2), off.w & seen(3));
            if (off.x | off.y | off.z | off.w) l = __int_as_float(0x7fc00000);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        ++tiles;
      }
      tiles += max(steps, 0) - max(n_tiles, 0);
      if (n_tiles > 0) {
        mbar_wait(&o_full[t], static_cast<uint32_t>(no) & 1u, a.status, abort_flag);
        ++no;
      }
      if (__any_sync(0xffffffffu, *abort_flag != 0u)) break;
      tc_fence_after();
      idx += 2 * max(steps, 0);
      if (CODES) l *= exp2_int(L_UNIT);
      if (FOLD && apart) {  // (l was 0, or NaN where a value seen is not finite)
        const Sum sum = *own_sum;
        __syncwarp();
        l = sum.base == neg_inf() ? 0.f : (l + sum.l) * ex2(sum.base - m + sum.over + L_UNIT);
      }
      const float inv = l == 0.f ? 0.f : (CODES ? exp2_int(L_UNIT) : 1.f) / l;
      if (part < 0) {
        // O / l: the warp's 32 rows go through its staging buffer 64 bytes of each at a time
        const int piece = lane & 3;
        T* to[4];
        bool on[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int r = sub * 32 + y * 8 + (lane >> 2), token = t * a.rt + (r >> a.pack_log);
          on[y] = token < tokens;
          to[y] = static_cast<T*>(a.out) + (row0 + token) * a.os[0] +
                  (h0 + (r & (a.pack - 1))) * a.os[1] + piece * 8;
        }
        const bool any = warp_token < tokens;
#pragma unroll 1
        for (int d = 0; d < DP && any; d += 32) {
          uint32_t o[32];
          if (n_tiles > 0) {
            tmem_ld32(o_tmem + d, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = 0u;
          }
          __syncwarp();  // the rows before have left the buffer
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              w[y] = pack2(__uint_as_float(o[x * 8 + y * 2]) * inv,
                           __uint_as_float(o[x * 8 + y * 2 + 1]) * inv, T{});
            *reinterpret_cast<uint4*>(stg + lane * 64 + ((x ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int r = y * 8 + (lane >> 2);
            if (on[y] && d + piece * 8 < a.D)
              *reinterpret_cast<uint4*>(to[y] + d) =
                  *reinterpret_cast<const uint4*>(stg + r * 64 + ((piece ^ ((r >> 1) & 3)) << 4));
          }
        }
      } else {
        // a part: [D][256 rows], a row a lane
        float* ws = a.ws + static_cast<long long>(part) * DP * ROWS + t * TILE + row;
        reinterpret_cast<float2*>(a.ml)[part * ROWS + t * TILE + row] = make_float2(m, l);
        if (t == 0 && row == 0 && parts) {
          const Cut cut = {parts, row0, tokens, h0};
          static_cast<Cut*>(a.cuts)[blockIdx.x] = cut;
        }
        if (n_tiles > 0) {
#pragma unroll 1
          for (int d = 0; d < DP; d += 32) {
            uint32_t o[32];
            tmem_ld32(o_tmem + d, o);
            tmem_ld_wait();
#pragma unroll
            for (int x = 0; x < 32; ++x) ws[(d + x) * ROWS] = __uint_as_float(o[x]);
          }
        }
      }
      // the next item's first weights, published after this, free O
      tc_fence_before();
    }
  } else if constexpr (CODES) {
    if constexpr (!FOLD) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // ------------------------------------------------------------ codes to fp16
    const int w = warp - 12;
    const int r8 = lane & 7, y0 = lane >> 3;  // a lane's row of 8, its pieces of 16 bytes
    float* scales = reinterpret_cast<float*>(smem + C::OFF_SC);
    float* q_back = reinterpret_cast<float*>(smem + C::OFF_Q);
    float* q_most = reinterpret_cast<float*>(smem + C::OFF_MOST);
    int idx = 0, tiles = 0, nq[2] = {0, 0};
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const int at = n % RECORDS;
      ok = mbar_wait_warp(&rec_full[at], static_cast<uint32_t>(n / RECORDS) & 1u, a.status,
                          abort_flag);
      if (!ok) break;
      const Record r = records[at];
      __syncwarp();
      if (lane == 0) mbar_arrive(&rec_empty[at]);
      if (r.p.tokens == 0) break;
      const int steps = r.steps();
      if (steps <= 0) continue;
      const int end = max(r.p.e0, r.p.e1);
      auto turn_q = [&](int t) {
        if (!mbar_wait_warp(&q_loaded[t], static_cast<uint32_t>(nq[t]) & 1u, a.status, abort_flag))
          return false;
        ++nq[t];
        int least = 120;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          const int row = w * 32 + i * 8 + r8;
          uint8_t* q = smem + t * C::BYTES + row * 128;
          uint4 v[DP / 32];
          uint32_t mx = 0;
#pragma unroll
          for (int x = 0; x < DP / 32; ++x) {
            const int piece = (x & 1) * 4 + y0;
            v[x] = *reinterpret_cast<const uint4*>(q + (x >> 1) * C::SLAB + ((piece ^ r8) << 4));
            mx = max_bits(max_bits(max_bits(max_bits(mx, v[x].x), v[x].y), v[x].z), v[x].w);
          }
          mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = __vmaxu2(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const int k = fp16_exponent(max(mx & 0xffffu, mx >> 16));
          const float f = exp2_int(k);
          least = min(least, k);
#pragma unroll
          for (int x = 0; x < DP / 32; ++x) {
            const int piece = (x & 1) * 4 + y0;
            *reinterpret_cast<uint4*>(q + (x >> 1) * C::SLAB + ((piece ^ r8) << 4)) =
                make_uint4(bf16x2_as_fp16(v[x].x, f), bf16x2_as_fp16(v[x].y, f),
                           bf16x2_as_fp16(v[x].z, f), bf16x2_as_fp16(v[x].w, f));
          }
          // by the uses of this query tile: that of two before has been read, as its weights were
          // there before the last scores of the one before, which freed the queries
          if (y0 == 0) q_back[((nq[t] - 1) & 1) * 256 + t * 128 + row] = a.c * exp2_int(-k);
        }
        least = __reduce_min_sync(0xffffffffu, least);
        if (lane == 0) q_most[((nq[t] - 1) & 1) * 8 + t * 4 + w] = a.c * exp2_int(-least);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);
        return true;
      };
      auto turn = [&](bool v, int tile) {
        const int u = idx, s = u % STAGES;
        ++idx;
        if (!mbar_wait_warp(&loaded[s], static_cast<uint32_t>(u / STAGES) & 1u, a.status,
                            abort_flag))
          return false;
        const int place = tiles % C::SCALES;
        if (!v && !mbar_wait_warp(&sc_full[place], static_cast<uint32_t>(tiles / C::SCALES) & 1u,
                                  a.status, abort_flag))
          return false;
        float* sc = scales + place * 256 + (v ? 128 : 0);
        constexpr int NP = DP / 64;
        // The rows of codes lie where the same rows of the last slab go: a row is read before it is
        // written.
        uint8_t* to = smem + C::OFF_KV + s * C::BYTES + (w * 32 + r8) * 128;
        const uint8_t* from = to + C::RAW;
        const bool look = v && (CODE == SRDIT_Q_E4M3 || FOLD) && partly(r, tile * TILE);
        uint32_t off = 0;  // rows that are not finite, by their scale or a NaN code
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          const int row = w * 32 + i * 8 + r8;
          uint4 c[NP];
#pragma unroll
          for (int k = 0; k < NP; ++k)
            c[k] = *reinterpret_cast<const uint4*>(from + i * 1024 + (((k * 4 + y0) ^ r8) << 4));
          float scale = FOLD ? sc[row] : 1.f;
          if (look) {
            // Zeros in place of rows behind the sequence, and of those that are not finite: the
            // queries that see these are told, or have the scale for it.
            bool nan = FOLD && !(fabsf(scale) < 3e38f);
            if constexpr (CODE == SRDIT_Q_E4M3) {
#pragma unroll
              for (int k = 0; k < NP; ++k)
                nan |= nan_codes(c[k].x) || nan_codes(c[k].y) || nan_codes(c[k].z) ||
                       nan_codes(c[k].w);
            }
            uint32_t rows = __ballot_sync(0xffffffffu, nan);
            rows |= rows >> 16;
            rows = (rows | rows >> 8) & 0xffu;
            off |= rows << (8 * i);
            if (((rows >> r8) & 1u) || tile * TILE + row >= r.p.len) {
#pragma unroll
              for (int k = 0; k < NP; ++k) c[k] = make_uint4(0, 0, 0, 0);
              if (FOLD) scale = 0.f;
              if (!FOLD && tile * TILE + row < r.p.len) sc[row] = __int_as_float(0x7fc00000);
            }
          }
          __syncwarp();
          // the scale in two terms, so that the product is rounded once
          const __half hi = __float2half_rn(scale);
          const __half2 f = __half2half2(hi);
          const __half2 rest = __half2half2(__float2half_rn(scale - __half2float(hi)));
#pragma unroll
          for (int k = 0; k < NP; ++k) {
            uint32_t h[8];
            widen_codes<CODE>(c[k], h);
            if constexpr (FOLD) {
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const __half2 n = *reinterpret_cast<const __half2*>(&h[x]);
                const __half2 y = __hfma2(n, f, __hmul2(n, rest));
                h[x] = *reinterpret_cast<const uint32_t*>(&y);
              }
            }
            uint8_t* slab = to + k * C::SLAB + i * 1024;
            *reinterpret_cast<uint4*>(slab + (((2 * y0) ^ r8) << 4)) =
                make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(slab + (((2 * y0 + 1) ^ r8) << 4)) =
                make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
        if (FOLD && look && lane == 0) reinterpret_cast<uint32_t*>(bad + s)[w] = off;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
        return true;
      };
      for (int j = r.t0; j < end && ok; ++j) {
        // (one copy of the code for keys and values: two are more than the instruction caches hold
        // beside the softmax)
#pragma unroll 1
        for (int x = 0; x < 2 && ok; ++x) {
          if (FOLD && j == r.t0 && (x ? r.p.e1 : r.p.e0) > r.t0) ok = turn_q(x);
          ok = ok && turn(x != 0, j);
        }
        ++tiles;
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

// Joins the parts of the items that the CTAs' shares cut: a block takes 32 columns of 32 rows of
// one, then others, of as many as there are (a block for every CTA's item, rows and columns, most
// of which have nothing to do, took 10 us to launch); a thread four columns of a row, four parts'
// loads in flight: bounded by their latency.
constexpr int JOIN_COLS = 32;
constexpr int JOIN_CTAS = 256;  // of a launch by shares, at most

template <typename T, int DP, bool CODES>
__global__ void __launch_bounds__(JOIN_COLS / 4 * 32)
    join_chunk_kernel(const __grid_constant__ Args a, int ctas) {
  pdl_begin();
  __shared__ int cuts_of[JOIN_CTAS];
  __shared__ int found[JOIN_COLS / 4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Cut* all_cuts = static_cast<const Cut*>(a.cuts);
  const bool mine = static_cast<int>(threadIdx.x) < ctas && all_cuts[threadIdx.x].parts != 0;
  const unsigned bits = __ballot_sync(0xffffffffu, mine);
  if (lane == 0) found[warp] = __popc(bits);
  __syncthreads();
  int count = 0, before = 0;
#pragma unroll
  for (int w = 0; w < JOIN_COLS / 4; ++w) {
    if (w < warp) before += found[w];
    count += found[w];
  }
  if (mine) cuts_of[before + __popc(bits & ((1u << lane) - 1u))] = threadIdx.x;
  __syncthreads();
  const int cols = (a.D + JOIN_COLS - 1) / JOIN_COLS, tasks = count * (ROWS / 32) * cols;
  for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
    const int which = task / ((ROWS / 32) * cols), rest = task - which * ((ROWS / 32) * cols);
    const int first = cuts_of[which];  // the CTA that begins the item
    const Cut cut = all_cuts[first];
    const int row = rest / cols * 32 + lane;
    const int d = rest % cols * JOIN_COLS + warp * 4;
    const int token = row >> a.pack_log, head = cut.h0 + (row & (a.pack - 1));
    if (token >= cut.tokens || d >= a.D) continue;
    float m = neg_inf(), l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < cut.parts; p0 += 4) {
      float2 q[4];
      float v[4][4];
  #pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int p = p0 + y, part = 2 * (first + p) + (p == 0);
        const bool on = p < cut.parts;
        const float* ws = a.ws + (static_cast<long long>(part) * DP + d) * ROWS + row;
        q[y] = on ? __ldg(reinterpret_cast<const float2*>(a.ml) + part * ROWS + row)
                  : make_float2(neg_inf(), 0.f);
  #pragma unroll
        for (int x = 0; x < 4; ++x) v[y][x] = on ? __ldg(ws + x * ROWS) : 0.f;
      }
      float mn = m;
  #pragma unroll
      for (int y = 0; y < 4; ++y) mn = max2(mn, q[y].x);
      if (mn == neg_inf()) continue;  // no key seen yet
      const Fall<CODES> fall(m - mn);
      m = mn;
      l = fall.add(l, 0.f);
  #pragma unroll
      for (int x = 0; x < 4; ++x) acc[x] *= fall.f;
  #pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (q[y].x == neg_inf()) continue;  // it saw no key
        const Fall<CODES> of_part(q[y].x - m);
        l = of_part.add(q[y].y, l);
  #pragma unroll
        for (int x = 0; x < 4; ++x) acc[x] = fmaf(v[y][x], of_part.f, acc[x]);
      }
    }
    const float inv = l == 0.f ? 0.f : (CODES ? exp2_int(L_UNIT) : 1.f) / l;
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (cut.row0 + token) * a.os[0] +
                              head * a.os[1] + d) =
        make_uint2(pack2(acc[0] * inv, acc[1] * inv, T{}), pack2(acc[2] * inv, acc[3] * inv, T{}));
  }
}

// ---------------------------------------------------------------- launch
Plan plan_chunk(const srdit_seq_attn_args& u, int sms) {
  Plan p = {};
  const int group = u.H / u.Hkv;
  // heads of a group side by side in a query tile, a power of two of them
  p.pack = 1;
  while (p.pack < TILE && group % (2 * p.pack) == 0) p.pack *= 2;
  p.rt = TILE / p.pack;
  p.slots = u.T / (2 * p.rt) + u.B;
  p.nhp = u.H / p.pack;
  const long long items = static_cast<long long>(p.slots) * p.nhp;
  long long keys = u.Tk, held = u.Tk;
  if (u.pages) {
    held = static_cast<long long>(u.pages->table_width) * u.pages->page_size;
    keys = u.max_kv > 0 && u.max_kv < held ? u.max_kv : held;
  }
  const long long tiles = (keys + TILE - 1) / TILE;
  // Few items of many key tiles are shared out by key tiles, and so is what a last round of whole
  // items would leave idle (all key tiles in 32 bits, however long the sequences turn out to be);
  // joining the parts costs what several do.
  const long long some =
      (u.B == 1 ? (u.T + 2 * p.rt - 1) / (2 * p.rt) : p.slots - u.B / 2) * static_cast<long long>(p.nhp);
  if (p.slots <= MAX_SLOTS && items * (held / TILE + 1) < (1ll << 30)) {
    // CTAs of shares go through keys at different places and miss what others have fetched: a step
    // takes a quarter more. (us whole and shared out, 32 heads over 8 of 128: 64 queries on 512 keys
    // 16.5 and 18.4, on 1024 24.2 and 20.3, on 32768 511 and 53; 512 on 16384 264 and 148, two of them 299 and
    // 329; a prompt of 1024 24 and 34. The last round of 6912 on 13824, 24 heads: 1148 and 1082, all of it
    // in shares 1323; of 2304 on 6912 223 and 202.)
    const long long rounds = (some + sms - 1) / sms, steps = some * tiles;
    const long long whole = rounds * tiles, shared = steps / sms * 5 / 4 + 7;
    if (some < sms || u.causal) {
      p.ranged = some < 2 * sms && shared < whole;
    } else {
      const long long last = some % sms;
      p.ranged = last && last * tiles / sms * 5 / 4 + 7 < tiles ? 2 : 0;
    }
  }
  if (sms > JOIN_CTAS) sms = JOIN_CTAS;
  p.ctas = static_cast<int>(p.ranged || items > sms ? sms : items);
  p.ws_floats = p.ranged ? 2ll * p.ctas * ROWS * ((u.D <= 64 ? 64 : 128) + 2) + 4 * p.ctas : 0;
  return p;
}

template <typename T, int DP, int CODE>
static int launch(const srdit_seq_attn_args& u, const Args& a, const Plan& p, cudaStream_t stream) {
  using C = ChunkCfg<DP, CODE>;
  auto kern = chunk_kernel<T, DP, CODE>;
  static std::atomic<bool> attr_done[kMaxDevices] = {};
  int rc = set_smem(kern, C::SMEM, attr_done);
  if (rc) return rc;
  CUtensorMap tq, tk, tv;
  {
    const long long row = (u.D + 7) / 8 * 16;
    const bool ut = u.T > 1, uh = u.H > 1 && u.q_stride[1] > 0;
    const long long dims[4] = {u.D, uh ? u.H : 1, u.T, 1};
    const long long strides[3] = {uh ? u.q_stride[1] * 2 : row, ut ? u.q_stride[0] * 2 : row, row};
    const int box[4] = {64, p.pack, p.rt, 1};
    rc = make_tmap_4d(&tq, u.q, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, dims, strides, box);
  }
  const int cols = C::CODES ? 128 : 64;
  if (!rc) rc = key_map(&tk, u, false, cols, 1 << a.box_log);
  if (!rc) rc = key_map(&tv, u, true, cols, 1 << a.box_log);
  if (rc) return rc;
  const bool packed = u.pages == nullptr;
  SRDIT_LAUNCH((kern), p.ctas, C::THREADS, C::SMEM, stream, tq, tk, tv, a,
               packed && u.k_stride[1] == 0, packed && u.v_stride[1] == 0);
  rc = static_cast<int>(cudaGetLastError());
  if (rc || !p.ranged) return rc;
  SRDIT_LAUNCH((join_chunk_kernel<T, DP, C::CODES>), 4 * p.ctas, JOIN_COLS / 4 * 32, 0, stream, a, p.ctas);
  return static_cast<int>(cudaGetLastError());
}

template <typename T, int CODE>
static int launch_size(const srdit_seq_attn_args& u, const Args& a, const Plan& p,
                       cudaStream_t stream) {
  return u.D <= 64 ? launch<T, 64, CODE>(u, a, p, stream) : launch<T, 128, CODE>(u, a, p, stream);
}

template <typename T>
static int run_typed(const srdit_seq_attn_args& u, const Args& a, const Plan& p,
                     cudaStream_t stream) {
  switch (u.pages ? u.pages->code : SRDIT_KV_PLAIN) {
    case SRDIT_Q_INT8: return launch_size<T, SRDIT_Q_INT8>(u, a, p, stream);
    case SRDIT_Q_E4M3: return launch_size<T, SRDIT_Q_E4M3>(u, a, p, stream);
    default: return launch_size<T, SRDIT_KV_PLAIN>(u, a, p, stream);
  }
}

int run_chunk(const srdit_seq_attn_args& u, Args& a, const Plan& p, cudaStream_t stream) {
  a.pack = p.pack;
  a.pack_log = 0;
  while ((1 << a.pack_log) < p.pack) ++a.pack_log;
  a.rt = p.rt;
  a.slots = p.slots;
  a.nhp = p.nhp;
  a.by_nhp = Divisor::of(p.nhp);
  a.by_slots = Divisor::of(p.slots);
  a.by_piece = Divisor::of(2 * p.rt);
  a.by_packs = Divisor::of(a.group / p.pack);
  a.by_ctas = Divisor::of(p.ctas);
  a.ranged = p.ranged;
  const int page = u.pages ? u.pages->page_size : TILE;
  a.box_log = page >= TILE ? 7 : page == 64 ? 6 : page == 32 ? 5 : 4;
  const long long rows = 2ll * p.ctas * ROWS;
  a.ml = a.ws + rows * (u.D <= 64 ? 64 : 128);
  a.cuts = a.ml + 2 * rows;
  return u.dtype == SRDIT_BF16 ? run_typed<__nv_bfloat16>(u, a, p, stream)
                               : run_typed<__half>(u, a, p, stream);
}

}  // namespace sattn
}  // namespace srdit
