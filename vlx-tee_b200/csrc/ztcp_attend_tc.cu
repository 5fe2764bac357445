// ztcp_attend_tc.cu -- attention of the newest tokens over a paged cache (ztcp_attend_pages) on the 5th-generation
// tensor cores, for items of more than one MMA row block: prefill chunks, wide groups.
//
// The mathematics is that of ztcp_attend.cu.  An item is up to 256 (token, head-of-the-group) rows of one sequence
// and KV head, as two row tiles of 128: S = Q K^T (128 x 64 x 16 a step) and O += P V (128 x head_dim x 16) are
// tcgen05.mma, K and V tiles of 64 keys arrive by TMA page by page (boxes of one page's rows, 128-byte swizzle), Q as
// boxes of tokens x group.  S, P and O live in TMEM: per row tile two buffers of 64 scores, each overwritten by its own
// P, and O; the two row tiles fill its 512 columns.
//
// Warps.  0-3 and 4-7: the softmax of row tiles 0 and 1, a thread per row; 8 and 9: one thread each issues the products
// of row tile 0 and 1 (one for both was the limit: an SS product takes 39 cycles to issue, a wait 100); 10: TMA.  A
// CTA's tiles pass through in a row, whatever items they belong to: stage g of the ring holds K of tile g and V of tile
// g - 2, so that with two buffers the scores of the next 64 keys are there when a row tile's softmax has finished with
// these, also where an item ends:
//   tensor core   PV(g) QK(g+2) | PV(g+1) QK(g+3) ...     (for each row tile)
//   softmax       -- S(g+1) ---- -- S(g+2) ------
// (With tiles of 128 keys P and the next S take the same columns, and softmax and products take turns: 3,750 cycles per
// 256 x 128 scores.)  A tile's exponentials are taken under the maximum in use, without looking for a new one first;
// only when a score has grown by more than 2^8 over it (the weights then stay below 2^8, which the 16-bit types hold
// without loss) is the maximum replaced and O rescaled.  m, l and O are fp32.
//
// Bound.  Per 256 x 64 scores the tensor core needs 1,260 cycles (head_dim 128; products of 64 keys read Q at the limit of
// shared memory's 128 bytes a cycle, else they would need 1,024), the exponentials 1,024 of the special-function units'
// 16 a cycle, in a thread's chain of score loads, exponentials and P stores that takes 1,590 when both row tiles are in
// it; together 1,800 were measured.  2,048 new tokens over 32,768 keys, 32 heads of 128: 1,160 to 1,190 us, 900 TFLOP/s (the
// GPU runs at 1.35 to 1.7 GHz then, as its power allows); five ragged chunks of up to 777 tokens over 800 to 8,192 keys:
// 250 to 258 us, 690 TFLOP/s, join included.
//
// Work.  As in ztcp_attend.cu the items form one line that the CTAs (one per SM) share evenly, in units of
// keys x group (Line); attend_merge_kernel joins items that several CTAs share.
//
// Waits are bounded: a wait that runs out (ztcp_tc.cuh) sets the CTA's error word, every role leaves its loop, copies
// and products in flight are waited for (always, and bounded again: a role that has left in time cannot know that another
// one will run out), TMEM is freed, and the merge kernel reports ZTCP_SEQ_TIMEOUT for every sequence.
#include "ztcp_tc.cuh"

namespace ztcp {

namespace {

constexpr int kRowTile = 128;
constexpr int kItemRows = 256;
constexpr int kTileKeys = 64;
constexpr int kThreads = 352;
constexpr int kMmaWarp = 8, kTmaWarp = 10;  // a warp of products for each row tile

struct TcParams {
  AttendParams a;
  PoolBoxes box;
  int32_t item_tokens;  // whole tokens of a group each: at most 256 rows
};

constexpr int kBars = 56;  // barrier slots at the start of shared memory

template <bool BF16, int HALVES, int SLOTS>
__global__ void __launch_bounds__(kThreads, 1)
attend_tc_kernel(const __grid_constant__ TcParams P, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                 const __grid_constant__ CUtensorMap qmap) {
  constexpr int kHalf = kTileKeys * 128;       // 64 columns of a K or V tile,
  constexpr int kTile = HALVES * kHalf;        // the tile,
  constexpr int kStage = 2 * kTile;            // a stage of the ring
  constexpr int kQHalf = kItemRows * 128;      // and 64 columns of Q
  constexpr int kCols = HALVES * 64;           // head_dim rounded up
  extern __shared__ uint8_t smem_raw[];
  __shared__ Waits waits_s;
  __shared__ uint32_t tmem_s;
  __shared__ Job s_jobs[kJobs];
  __shared__ unsigned s_bad[16];
  const CacheParams& c = P.a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile Waits* const waits = &waits_s;

  // barriers first, then the 1,024-byte aligned tiles
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t bars = raw;
  const uint32_t tiles = (raw + kBars * 8 + 1023) & ~1023u;
  const uint32_t qtile = tiles, ring = tiles + HALVES * kQHalf;
  auto full = [&](int s) { return bars + s * 8; };
  auto empty = [&](int s) { return bars + (SLOTS + s) * 8; };
  const uint32_t q_full = bars + 2 * SLOTS * 8, q_empty = q_full + 8, s_full = q_empty + 8, p_full = s_full + 32, pv_last = p_full + 32,
                 pv_prev = pv_last + 16, job_full = pv_prev + 16, job_empty = job_full + 8 * kJobs, drain = job_empty + 8 * kJobs;
  static_assert(2 * SLOTS + 16 + 2 * kJobs <= kBars, "barrier slots");

  if (tid == 0) {
    waits_s.limit = c.wait_cycles;
    waits_s.dead = 0;
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 2);
    }
    for (int q = 0; q < 2; ++q) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(s_full + 16 * q + 8 * b, 1);
        mbar_init(p_full + 16 * q + 8 * b, 4);
      }
      mbar_init(pv_last + 8 * q, 1);
      mbar_init(pv_prev + 8 * q, 1);
    }
    for (int e = 0; e < kJobs; ++e) {
      mbar_init(job_full + 8 * e, 1);
      mbar_init(job_empty + 8 * e, 10);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);
    mbar_init(drain, 1);
    mbar_init(drain + 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_s)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  cudaTriggerProgrammaticLaunchCompletion();  // the joining kernel may be set up meanwhile; it waits for this one's end

  if (warp == kTmaWarp) {
    // ---- TMA: the CTA's tiles in a row, items or not.  Stage g of the ring: K of tile g and V of tile g - 2 ----
    const int per_tile = kTileKeys / P.box.rows, boxes = HALVES * per_tile;
    const int item_rows = P.item_tokens * c.group;
    uint32_t items = 0, pos = 0;
    int64_t at;
    Spot spot;
    const SplitSpan S = locate_warp(c.n_seqs, P.a.grid, lane, [&](int b) { return seq_work(c, item_rows, b); }, &at, &spot);
    Publisher<kTileKeys> pub;
    pub.walk.begin(c, item_rows, 4, spot, at < 0 ? 0 : at, at < 0 ? 0 : S.begin(blockIdx.x + 1));
    pub.cut = Cut{};
    pub.n = 0;
    Job job;
    PageRows pages;
    bool ok = true;
    int32_t row1 = 0, row2 = 0, head1 = 0, head2 = 0;  // pool rows and heads of the last tile and the one before
    // Lane p loads box p of V, of 64 columns and one page each, and lane boxes + p that of K.
    auto stage = [&](bool v_on, bool k_on, int32_t row, int32_t head) {
      const uint32_t slot = pos % SLOTS;
      if (pos >= SLOTS && !warp_wait(empty(slot), (pos / SLOTS - 1) & 1, waits)) return false;
      if (lane == 0) mbar_expect(full(slot), (v_on ? kTile : 0) + (k_on ? kTile : 0));
      __syncwarp();
      const bool isk = lane >= boxes;
      const int p = isk ? lane - boxes : lane;
      if (p < boxes && (isk ? k_on : v_on)) {
        const int x = HALVES > 1 && p >= per_tile;
        tma_load(ring + slot * kStage + (isk ? kTile : 0) + x * kHalf + (p & (per_tile - 1)) * P.box.rows * 128, isk ? &kmap : &vmap, x * 64,
                 isk ? head : head2, isk ? row : row2, full(slot));
      }
      __syncwarp();
      ++pos;
      row2 = row1;
      head2 = head1;
      row1 = row;
      head1 = head;
      return true;
    };
    while (ok && (ok = pub.next(c, S, s_jobs, job_full, job_empty, lane, waits, &job)) && job.ta < job.tb) {
      pages.start(job.ta);
      for (int t = job.ta; t < job.tb; ++t) {
        const int32_t row = pages.at(c, P.box, per_tile, job.b, job.kv_len, t, lane);  // pool_rows: zeros
        // Pages outside the pool count as masked; the softmax warps learn of them here (16 tiles back all have read
        // theirs: the stage that was in this slot, at most 8 tiles back, is spent).
        const unsigned bad = __ballot_sync(0xffffffffu, lane < per_tile && t * kTileKeys + (lane << P.box.shift) < job.kv_len && row == P.box.pool_rows);
        if (lane == 0) s_bad[pos & 15] = bad;
        if (!(ok = stage(pos >= 2, true, row, job.head))) break;
        if (t > job.ta) continue;
        // Q as it lies: tokens x group rows, each half of the columns [256][64] (rows past the item's are other tokens',
        // or left over; nothing of theirs is stored).  The item before needs its own Q for one tile less than V.
        if (items > 0 && !(ok = warp_wait(q_empty, (items - 1) & 1, waits))) break;
        ++items;
        if (lane == 0) mbar_expect(q_full, HALVES * item_rows * 128);
        __syncwarp();
        if (lane < HALVES) tma_load4(qtile + lane * kQHalf, &qmap, lane * 64, 0, job.head, (int)job.row0 + job.row / c.group, q_full);
      }
    }
    if (ok && pos > 0) {  // the last two tiles' V (one tile in all: an empty stage before it)
      ok = stage(pos >= 2, false, 0, 0) && stage(true, false, 0, 0);
    }
    if (lane == 0) P.a.cuts[blockIdx.x] = pub.cut;
    drain_fills(full(0), SLOTS, pos);
    drain_fills(q_full, 1, items);
  } else if (warp >= kMmaWarp) {
    // ---- products of row tile q: one thread ----------------------------------------------------------
    const int q = warp - kMmaWarp;
    if (elect_one()) {
      constexpr uint32_t kHi = desc_hi(1024, kSwizzle128);
      const uint32_t qk = inst_desc(BF16, 128, kTileKeys, false, false), pv = inst_desc(BF16, 128, kCols, false, true);
      const uint32_t v_lo = desc_lo(ring, kHalf), k_lo = desc_lo(ring + kTile, 16), q_lo = desc_lo(qtile + q * kRowTile * 128, 16);
      const uint32_t s_at = tmem + q * 128, o_at = tmem + 256 + q * 128, s_done = s_full + 16 * q, p_there = p_full + 16 * q;
      uint32_t slot = 0, phase = 0;  // of the stage
      uint32_t items = 0, njobs = 0;
      uint32_t qks = 0, pvs = 0;  // scores and products with V so far
      // What tile g, g + 1 and g + 2 of the CTA are, for one stage after the other:
      constexpr int kTile1 = 1, kMine = 2, kFirst = 4, kLast = 8;  // a tile; with rows of this row tile; the item's first, its last
      int now = 0, next = 0, t = 0;
      bool more = true, ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        ok = ok && mbar_wait(bar, parity & 1, waits);
        return ok;
      };
      Job job;
      job.tb = 0;
      while (true) {
        int then = 0;
        if (more && t == job.tb) {
          if (!(ok = take_job_alone(s_jobs, job_full, job_empty, njobs, waits, &job))) break;
          more = job.ta < job.tb;
          t = job.ta;
          then = kFirst;
        }
        if (more) {
          ++t;
          then |= kTile1 | (q == 0 || job.rows > kRowTile ? kMine : 0) | (t == job.tb ? kLast : 0);
        } else {
          then = 0;
        }
        if ((now | next | then) == 0 || !wait(full(slot), phase)) break;
        if (now & kMine) {
          const uint32_t buf = pvs & 1, b = v_lo + slot * (kStage >> 4);
          if (!wait(p_there + 8 * buf, pvs >> 1)) break;
          ++pvs;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; ++k)
            mma_ts(o_at, s_at + buf * 64 + k * 8, b + (k * 2048 >> 4), kHi, pv, !(now & kFirst) || k > 0);
          // Scores that follow say that this product is done; the item's last two have barriers of their own.
          if (now & kLast) tc_commit(pv_last + 8 * q);
          else if ((next & (kFirst | kLast)) == kLast) tc_commit(pv_prev + 8 * q);
        }
        if ((then & kFirst) && !wait(q_full, items++)) break;
        if (then & kMine) {
          // the scores' buffer was last read by a product with V that has been issued, and products run in order
          tc_fence_after();
          const uint32_t buf = qks++ & 1, b = k_lo + slot * (kStage >> 4);
#pragma unroll
          for (int k = 0; k < HALVES * 4; ++k)
            mma_ss(s_at + buf * 64, q_lo + (((k >> 2) * kQHalf + (k & 3) * 32) >> 4), kHi, b + (((k >> 2) * kHalf + (k & 3) * 32) >> 4), kHi, qk, k > 0);
          tc_commit(s_done + 8 * buf);
        }
        tc_commit(empty(slot));
        if (then & kLast) tc_commit(q_empty);
        if (++slot == SLOTS) slot = 0, phase ^= 1;
        now = next;
        next = then;
      }
      drain_products(drain + 8 * q);
    }
    __syncwarp();
  } else {
    // ---- softmax of row tile q: a thread per row -----------------------------------------------------
    const int q = warp >> 2, wg = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t to = tmem + lanes + 256 + q * 128;
    uint32_t step = 0, mine = 0;  // tiles of the CTA, and of this row tile
    uint32_t ends = 0, prevs = 0;  // items of this row tile, and those of more than one tile
    Job job;
    uint32_t njobs = 0;
    auto open = [&] { return take_job(s_jobs, job_full, job_empty, njobs, lane, waits, &job); };
    bool ok = open();
    while (ok && job.ta < job.tb) {
      const Job it = job;
      if (q == 1 && it.rows <= kRowTile) {  // nothing in this row tile
        step += it.tb - it.ta;
        ok = open();
        continue;
      }
      const int r = q * kRowTile + wg;
      // (rows past the item's see what its last row sees: they slow no tile down)
      const int lim = visible_keys(c, Seq{it.kv_len, it.q_len, it.row0}, (it.row + min(r, it.rows - 1)) / c.group);
      const int clear = __reduce_min_sync(0xffffffffu, lim) / kTileKeys;  // tiles that all of the warp's rows see whole
      bool live = false;  // all of them have a maximum
      const bool prev = it.tb - it.ta > 1;
      float m = -INFINITY, l = 0.f;
      for (int t = it.ta; t < it.tb; ++t, ++step, ++mine) {
        const int j0 = t * kTileKeys;
        const uint32_t buf = mine & 1, ts = tmem + lanes + q * 128 + buf * 64;
        if (!(ok = warp_wait(s_full + 16 * q + 8 * buf, (mine >> 1) & 1, waits))) break;
        tc_fence_after();
        const unsigned bad = s_bad[step & 15];
        uint32_t x[64];
        tmem_ld32(ts, x);
        tmem_ld32(ts + 32, x + 32);
        tmem_ready32(x);
        tmem_ready32(x + 32);
        // A tile that every row sees whole, once a maximum is in use: whether a score has outgrown it shows by the way.
        // (A share of the exponentials as a polynomial on the FMA pipes: measured 4 to 11 % slower in all, an eighth to 3/8.)
        bool ready = false;
        if (t < clear && live && !bad) {
          const uint64_t sc2 = pair(c.scale_log2, c.scale_log2), z2 = pair(-m, -m);
          uint64_t sum = pair(0.f, 0.f), sum1 = sum;
          float top = -INFINITY, top1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            top = fmaxf(top, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
            top1 = fmaxf(top1, fmaxf(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])));
            float a, b, d, e;
            unpair(fma2(pair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, z2), a, b);
            unpair(fma2(pair(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), sc2, z2), d, e);
            a = fast_exp2(a);
            b = fast_exp2(b);
            d = fast_exp2(d);
            e = fast_exp2(e);
            sum = add2(sum, pair(a, b));
            sum1 = add2(sum1, pair(d, e));
            x[i / 2] = pack2<BF16>(a, b);
            x[i / 2 + 1] = pack2<BF16>(d, e);
          }
          ready = __all_sync(0xffffffffu, fmaxf(top, top1) * c.scale_log2 <= m + 8.f);
          if (ready) {
            float s0, s1, s2, s3;
            unpair(sum, s0, s1);
            unpair(sum1, s2, s3);
            l += (s0 + s1) + (s2 + s3);
          } else {  // the scores once more
            tmem_ld32(ts, x);
            tmem_ld32(ts + 32, x + 32);
            tmem_ready32(x);
            tmem_ready32(x + 32);
          }
        }
        if (!ready) {
          if (t >= clear || bad) {
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (j0 + i >= lim || (bad >> (i >> P.box.shift) & 1)) x[i] = 0xff800000u;
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 64; i += 2) mx = fmaxf(mx, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
          mx *= c.scale_log2;
          const bool grow = mx > m + 8.f || (m == -INFINITY && mx > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float mn = grow ? mx : m;
            const float f = grow ? fast_exp2(m - mn) : 1.f;  // 0 for the first maximum
            if (t > it.ta) {  // O is this thread's to change between its products
              if (t + 1 < it.tb) ok = warp_wait(s_full + 16 * q + 8 * (buf ^ 1), ((mine + 1) >> 1) & 1, waits);
              else ok = warp_wait(pv_prev + 8 * q, prevs & 1, waits);
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int i = 0; i < kCols; i += 32) {
                uint32_t o[32];
                tmem_ld32(to + i, o);
                tmem_ready32(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st32(to + i, o);
              }
            }
            l *= f;
            m = mn;
            live = __all_sync(0xffffffffu, m > -INFINITY);
          }
          const float z = m == -INFINITY ? 0.f : -m;
          float sum = 0.f, sum1 = 0.f;
#pragma unroll
          for (int i = 0; i < 64; i += 2) {
            const float a = fast_exp2(fmaf(__uint_as_float(x[i]), c.scale_log2, z)), b = fast_exp2(fmaf(__uint_as_float(x[i + 1]), c.scale_log2, z));
            sum += a;
            sum1 += b;
            x[i / 2] = pack2<BF16>(a, b);
          }
          l += sum + sum1;
        }
        tmem_st32(ts, x);
        // rows of V past the sequence's end lie in its last page and may hold anything: zero them for 0 * V (both row
        // tiles' warps do, each for its own product)
        const int end = it.kv_len - j0;
        if (end < kTileKeys && it.kv_len % c.page_tokens != 0) {
          const uint32_t vp = step + 2;
          if (!(ok = warp_wait(full(vp % SLOTS), (vp / SLOTS) & 1, waits))) break;
          if (wg >= end && wg < kTileKeys)
#pragma unroll
            for (int i = 0; i < HALVES * 8; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(ring + (vp % SLOTS) * kStage + (i >> 3) * kHalf + wg * 128 + (i & 7) * 16),
                           "r"(0) : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 16 * q + 8 * buf);
      }
      if (!ok) break;
      if (!(ok = open())) break;

      if (!(ok = warp_wait(pv_last + 8 * q, ends & 1, waits))) break;
      tc_fence_after();
      ++ends;
      prevs += prev;
      const int tok = (it.row + r) / c.group, gh = (it.row + r) - tok * c.group;
      const int64_t o = (it.row0 + tok) * (int64_t)(c.kv_heads * c.group) + it.head * c.group + gh;
      float* const part = P.a.part + (int64_t)(2 * blockIdx.x + (it.inside ? 0 : 1)) * P.a.part_floats;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll 1
      for (int i = 0; i < kCols; i += 32) {
        uint32_t v[32];
        tmem_ld32(to + i, v);
        tmem_ready32(v);
        if (r < it.rows) {
          if (it.whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (i + e < c.v_dim) {
                uint4 w;
                w.x = pack2<BF16>(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv);
                w.y = pack2<BF16>(__uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv);
                w.z = pack2<BF16>(__uint_as_float(v[e + 4]) * inv, __uint_as_float(v[e + 5]) * inv);
                w.w = pack2<BF16>(__uint_as_float(v[e + 6]) * inv, __uint_as_float(v[e + 7]) * inv);
                *reinterpret_cast<uint4*>(P.a.out + o * c.v_dim + i + e) = w;
              }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (i + e < c.v_dim)  // rows contiguous, so that a warp's store is one
                *reinterpret_cast<uint4*>(part + ((i + e) / 4 * P.a.part_rows + r) * 4) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
      }
      tc_fence_before();
      if (r < it.rows) {
        if (!it.whole) {
          part[kItemRows * c.v_dim + r] = m;
          part[kItemRows * (c.v_dim + 1) + r] = l;
        } else if (P.a.lse) {
          P.a.lse[o] = l == 0.f ? -INFINITY : fmaf(m, 0.693147180559945f, logf(l));
        }
      }
    }
    tc_wait_st();  // (a wait that ran out may have left a store of P in flight)
  }
  __syncthreads();
  if (tid == 0 && waits->dead) P.a.cuts[blockIdx.x].error = 1;
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---- host -----------------------------------------------------------------------------------------
template <bool BF16, int HALVES, int SLOTS>
void launch_kernel(const TcParams& P, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, cudaStream_t s) {
  auto* const f = attend_tc_kernel<BF16, HALVES, SLOTS>;
  const int smem = kBars * 8 + 1024 + HALVES * (kItemRows + SLOTS * 2 * kTileKeys) * 128;
  cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  f<<<P.a.grid, kThreads, smem, s>>>(P, k, v, q);
}

}  // namespace

bool attend_tc_fits(const CacheParams& c) { return c.v && c.head_dim <= 128 && c.group <= kItemRows && pages_fit(c, kTileKeys); }

AttendShape attend_tc_shape(const CacheParams& c, int sms) { return {sms, kItemRows, kItemRows * (c.v_dim + 2), 1}; }

bool launch_attend_tc(const AttendParams& A, bool bf16, cudaStream_t s) {
  TcParams P;
  P.a = A;
  P.box = pool_boxes(A.c, kTileKeys);
  P.item_tokens = kItemRows / A.c.group;
  CUtensorMap k, v, q;
  if (!pool_map(&k, A.c.k, A.c, bf16, P.box) || !pool_map(&v, A.c.v, A.c, bf16, P.box) || !query_map(&q, A.c, bf16, P.item_tokens, A.c.group))
    return false;
  if (A.c.head_dim <= 64) bf16 ? launch_kernel<true, 1, 7>(P, k, v, q, s) : launch_kernel<false, 1, 7>(P, k, v, q, s);
  else bf16 ? launch_kernel<true, 2, 5>(P, k, v, q, s) : launch_kernel<false, 2, 5>(P, k, v, q, s);
  return true;
}

}  // namespace ztcp
