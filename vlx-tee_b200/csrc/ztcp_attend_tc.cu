// ztcp_attend_tc.cu -- attention of the newest tokens over a paged cache (ztcp_attend_pages) on the 5th-generation
// tensor cores, for items of more than one MMA row block: prefill chunks, wide groups.
//
// The mathematics is that of ztcp_attend.cu.  An item is up to 256 (token, head-of-the-group) rows of one sequence
// and KV head, as two row tiles of 128: S = Q K^T and O += P V are tcgen05.mma of 128 x 128 x 16, K and V tiles of
// 128 keys arrive by TMA page by page (boxes of one page's rows, 128-byte swizzle), and S, P and O live in TMEM:
// S0 S1 O0 O1 fill its 512 columns, P overwrites the first half of its S.
//
// Warps.  0-3 and 4-7: the softmax of row tiles 0 and 1, a thread per row; 8: one thread issues the products; 9: TMA (10, 11 fill
// the warpgroup).
// The products of one row tile run under the softmax of the other:
//   tensor core   PV0(j-1) QK0(j) | PV1(j-1) QK1(j) | PV0(j) QK0(j+1) | ...
//   softmax 0                       ---- S0(j) ----
//   softmax 1                                         ---- S1(j) ----
// S_q(j) is committed after PV_q(j-1), so whoever sees S_q(j) may also change O_q.  O is rescaled only when a row's
// maximum has grown by more than 2^8 over the one in use (the weights then stay below 2^8, which the 16-bit types
// hold without loss); m, l and O are fp32.
//
// Bound.  Per 128 x 128 scores the tensor core needs 2 x 512 cycles (head_dim 128) and the exponentials 1,024 of the
// 16-per-cycle unit, so the two take turns at being the limit; a share of the exponentials is computed by a
// polynomial on the FMA pipes instead (exp2_poly).
//
// Work.  As in ztcp_attend.cu the items form one line that the CTAs (one per SM) share evenly, in units of
// keys x group (Line); attend_merge_kernel joins items that several CTAs share.
//
// Waits are bounded: a wait that runs out (ztcp_tc.cuh) sets the CTA's error word, every role leaves
// its loop, copies and products in flight are waited for (bounded again), TMEM is freed, and the merge kernel
// reports ZTCP_SEQ_TIMEOUT for every sequence.
#include "ztcp_tc.cuh"

namespace ztcp {

namespace {

constexpr int kRowTile = 128;
constexpr int kItemRows = 256;
constexpr int kThreads = 384;  // three warpgroups: 64,512 registers at launch (168 each)
constexpr int kMmaWarp = 8, kTmaWarp = 9;

struct TcParams {
  AttendParams a;
  PoolBoxes box;
  int32_t item_tokens;  // whole tokens of a group each: at most 256 rows
};

constexpr int kBars = 40;  // barrier slots at the start of shared memory

template <bool BF16, int HALVES, int SLOTS>
__global__ void __launch_bounds__(kThreads, 1)
attend_tc_kernel(const __grid_constant__ TcParams P, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                 const __grid_constant__ CUtensorMap qmap) {
  constexpr int kHalf = kGroupBytes;
  constexpr int kTile = HALVES * kHalf;        // a K or V tile, or a Q row tile
  constexpr int kCols = HALVES * 64;           // head_dim rounded up
  extern __shared__ uint8_t smem_raw[];
  __shared__ int dead_s;
  __shared__ uint32_t tmem_s;
  __shared__ Job s_jobs[kJobs];
  const CacheParams& c = P.a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile int* const dead = &dead_s;

  // barriers first, then the 1,024-byte aligned tiles
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t bars = raw;
  const uint32_t tiles = (raw + kBars * 8 + 1023) & ~1023u;
  const uint32_t qtile = tiles, ring = tiles + 2 * kTile;
  auto full = [&](int s) { return bars + s * 8; };
  auto empty = [&](int s) { return bars + (SLOTS + s) * 8; };
  const uint32_t q_full = bars + 2 * SLOTS * 8, q_empty = q_full + 8, s_full = q_empty + 8, p_full = s_full + 16, o_full = p_full + 16,
                 job_full = o_full + 16, job_empty = job_full + 8 * kJobs, drain = job_empty + 8 * kJobs;
  static_assert(2 * SLOTS + 9 + 2 * kJobs <= kBars, "barrier slots");

  if (tid == 0) {
    dead_s = 0;
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(s_full + 8 * q, 1);
      mbar_init(p_full + 8 * q, 128);
      mbar_init(o_full + 8 * q, 1);
    }
    for (int e = 0; e < kJobs; ++e) {
      mbar_init(job_full + 8 * e, 1);
      mbar_init(job_empty + 8 * e, 9);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(drain, 1);
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

  // The softmax warps hold a row of scores: of the block's registers they take 208 a thread, the others 88 (8 x 32 x 208
  // + 4 x 32 x 88 = 64,512, what the block was launched with).
  if (warp >= kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == kTmaWarp) {
      // ---- TMA: K and V tiles in turn through the ring; lane p fetches page p of the tile ------------
      const int per_tile = kKeys / P.box.rows;
      const int item_rows = P.item_tokens * c.group;
      uint32_t items = 0;
      uint32_t pos = 0;  // tiles so far: K of step t is 2 t, V is 2 t + 1
      int64_t at;
      Spot spot;
      const SplitSpan S = locate_warp(c.n_seqs, P.a.grid, lane, [&](int b) { return seq_work(c, item_rows, b); }, &at, &spot);
      Publisher<kKeys> pub;
      pub.walk.begin(c, item_rows, 2, spot, at < 0 ? 0 : at, at < 0 ? 0 : S.begin(blockIdx.x + 1));
      pub.cut = Cut{};
      pub.n = 0;
      Job job;
      bool ok = true;
      while (ok && (ok = pub.next(c, S, s_jobs, job_full, job_empty, lane, dead, &job)) && job.ta < job.tb) {
        // Q as it lies: tokens x group rows, each half of the columns [256][64] (rows past the item's are other tokens', or
        // left over; nothing of theirs is stored)
        if (items > 0 && !(ok = warp_wait(q_empty, (items - 1) & 1, dead))) break;
        ++items;
        if (lane == 0) mbar_expect(q_full, HALVES * item_rows * 128);
        __syncwarp();
        if (lane < HALVES) tma_load4(qtile + lane * 2 * kHalf, &qmap, lane * 64, 0, job.head, (int)job.row0 + job.row / c.group, q_full);
        for (int t = job.ta; ok && t < job.tb; ++t) {
          const int j = t * kKeys + lane * P.box.rows;
          int32_t row = P.box.pool_rows;  // past the sequence's end, or a bad page: zeros
          if (lane < per_tile && j < job.kv_len) {
            const int64_t r = pool_row(c, job.b, j);
            if (r >= 0) row = (int32_t)r;
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++pos) {
            const int slot = pos % SLOTS;
            ok = ok && (pos < SLOTS || mbar_wait(empty(slot), (pos / SLOTS - 1) & 1, dead));
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
            if (lane == 0) mbar_expect(full(slot), kTile);
            __syncwarp();
            if (lane < per_tile)
#pragma unroll
              for (int x = 0; x < HALVES; ++x)
                tma_load(ring + slot * kTile + x * kHalf + lane * P.box.rows * 128, kv ? &vmap : &kmap, x * 64, job.head, row, full(slot));
          }
        }
      }
      if (lane == 0) P.a.cuts[blockIdx.x] = pub.cut;
      if (*dead) {  // after a timeout: no copy may be in flight when the CTA ends
        int none = 0;
        for (uint32_t p = pos > SLOTS ? pos - SLOTS : 0; p < pos; ++p) mbar_wait(full(p % SLOTS), (p / SLOTS) & 1, &none);
        if (items > 0) mbar_wait(q_full, (items - 1) & 1, &none);
      }
    } else if (warp == kMmaWarp) {
      // ---- products: one thread ------------------------------------------------------------------------
      if (elect_one()) {
        constexpr uint32_t kHi = desc_hi(1024, kSwizzle128);
        const uint32_t qk = inst_desc(BF16, 128, kKeys, false, false), pv = inst_desc(BF16, 128, kCols, false, true);
        const uint32_t k_lo = desc_lo(ring, 16), v_lo = desc_lo(ring, kHalf), q_lo = desc_lo(qtile, 16);
        uint32_t kslot = 0, kphase = 0;    // of the next K tile; V's follows it
        uint32_t vslot = 1, vphase = 0;
        uint32_t items = 0;                // items so far
        uint32_t softs[2] = {0, 0};        // tiles so far, per row tile
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) {
          ok = ok && mbar_wait(bar, parity & 1, dead);
          return ok;
        };
        auto advance = [&](uint32_t& slot, uint32_t& phase) {  // two slots on
          slot += 2;
          if (slot >= SLOTS) slot -= SLOTS, phase ^= 1;
        };
        const uint32_t tm = tmem;
        // Step t multiplies P of tile t - 1 by V and computes the scores of tile t; per row tile in turn, so that each
        // has the other's products to hide its softmax under.
        Job job;
        uint32_t njobs = 0;
        int cur = 0, n = 0;  // row tiles of the step before, and tiles of its item
        int t = 0;           // of the item's tiles, those whose scores are out
        while (ok) {
          const bool fresh = t == n;  // the step's scores are those of the next item
          if (fresh) {  // published once the loads of the item before are out
            if (!(ok = take_job_alone(s_jobs, job_full, job_empty, njobs, dead, &job))) break;
            if (cur == 0 && job.ta == job.tb) break;
          }
          const int nxt = fresh ? (job.ta < job.tb ? (job.rows > kRowTile ? 2 : 1) : 0) : cur;
          if (cur && !wait(full(vslot), vphase)) break;
          bool k_there = false;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (q < cur) {
              if (!wait(p_full + 8 * q, softs[q])) break;
              ++softs[q];
              tc_fence_after();
              const uint32_t b = v_lo + vslot * (kTile >> 4);
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)
                mma_ts(tm + 256 + q * 128, tm + q * 128 + k * 8, b + (k * 2048 >> 4), kHi, pv, t > 1 || k > 0);
              if (fresh) tc_commit(o_full + 8 * q);
            }
            if (q < nxt) {
              if (!k_there && ((fresh && !wait(q_full, items)) || !wait(full(kslot), kphase))) break;
              k_there = true;
              tc_fence_after();
              const uint32_t a = q_lo + q * (kHalf >> 4), b = k_lo + kslot * (kTile >> 4);
#pragma unroll
              for (int k = 0; k < HALVES * 4; ++k) {
                const uint32_t off = ((k >> 2) * kHalf + (k & 3) * 32) >> 4, qoff = ((k >> 2) * 2 * kHalf + (k & 3) * 32) >> 4;
                mma_ss(tm + q * 128, a + qoff, kHi, b + off, kHi, qk, k > 0);
              }
              tc_commit(s_full + 8 * q);
            }
          }
          if (!ok) break;
          if (cur) {
            tc_commit(empty(vslot));
            advance(vslot, vphase);
          }
          if (nxt) {
            tc_commit(empty(kslot));
            advance(kslot, kphase);
          }
          if (fresh) {
            if (nxt == 0) break;
            n = job.tb - job.ta;
            t = 0;
            ++items;
          }
          cur = nxt;
          if (++t == n) tc_commit(q_empty);  // the item's last scores are out
        }
        if (*dead) {  // no product may be in flight when TMEM is freed
          int none = 0;
          tc_commit(drain);
          mbar_wait(drain, 0, &none);
        }
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---- softmax of row tile q: a thread per row -----------------------------------------------------
    const int q = warp >> 2, wg = tid & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const uint32_t ts = tmem + lanes + q * 128, to = tmem + lanes + 256 + q * 128;
    uint32_t step = 0, mine = 0, done = 0;  // tiles of the CTA, tiles and items of this row tile
    Job job;
    uint32_t njobs = 0;
    auto open = [&] { return take_job(s_jobs, job_full, job_empty, njobs, lane, dead, &job); };
    bool ok = open();
    while (ok && job.ta < job.tb) {
      const Job it = job;
      if (q == 1 && it.rows <= kRowTile) {  // nothing in this row tile
        step += it.tb - it.ta;
        ok = open();
        continue;
      }
      const int r = q * kRowTile + wg;
      const int lim = r < it.rows ? visible_keys(c, Seq{it.kv_len, it.q_len, it.row0}, (it.row + r) / c.group) : 0;
      float m = -INFINITY, l = 0.f;
      for (int t = it.ta; t < it.tb; ++t, ++step, ++mine) {
        const int j0 = t * kKeys;
        // pages of this tile outside the pool count as masked
        unsigned bad = 0;
        {
          const int j = j0 + lane * P.box.rows;
          const bool b = lane < kKeys / P.box.rows && j < it.kv_len && pool_row(c, it.b, j) < 0;
          bad = __ballot_sync(0xffffffffu, b);
        }
        if (!(ok = warp_wait(s_full + 8 * q, mine & 1, dead))) break;
        tc_fence_after();
        uint32_t x[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(ts + i * 32, x + i * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ready32(x + i * 32);
        const uint64_t sc2 = pair(c.scale_log2, c.scale_log2);
        // A tile that every row sees whole, once a maximum is in use: its exponentials need no new one unless a score
        // has grown by 2^8, which shows by the way; the scores are then read again below.  Of eight pairs, three
        // exponentials go to the FMA pipes.
        bool done = false;
        if (__all_sync(0xffffffffu, lim >= j0 + kKeys && m > -INFINITY) && !bad) {
          const uint64_t z2 = pair(-m, -m);
          uint64_t sum = pair(0.f, 0.f), sum1 = sum;
          float top = -INFINITY, top1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 128; i += 4) {
            top = fmaxf(top, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
            top1 = fmaxf(top1, fmaxf(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])));
            uint64_t u = fma2(pair(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), sc2, z2);
            uint64_t v = fma2(pair(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), sc2, z2);
            float a, b, d, e;
            if (i % 16 == 4) u = exp2_poly(u), unpair(u, a, b);
            else unpair(u, a, b), a = fast_exp2(a), b = fast_exp2(b), u = pair(a, b);
            if (i % 8 == 0) v = exp2_poly(v), unpair(v, d, e);
            else unpair(v, d, e), d = fast_exp2(d), e = fast_exp2(e), v = pair(d, e);
            sum = add2(sum, u);
            sum1 = add2(sum1, v);
            x[i / 2] = pack2<BF16>(a, b);
            x[i / 2 + 1] = pack2<BF16>(d, e);
          }
          done = __all_sync(0xffffffffu, fmaxf(top, top1) * c.scale_log2 <= m + 8.f);
          if (done) {
            float s0, s1, s2, s3;
            unpair(sum, s0, s1);
            unpair(sum1, s2, s3);
            l += (s0 + s1) + (s2 + s3);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld32(ts + i * 32, x + i * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ready32(x + i * 32);
          }
        }
        if (!done) {
          if (!__all_sync(0xffffffffu, lim >= j0 + kKeys) || bad) {
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (j0 + i >= lim || (bad >> (i >> P.box.shift) & 1)) x[i] = 0xff800000u;
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 128; i += 2) mx = fmaxf(mx, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
          mx *= c.scale_log2;
          const bool grow = mx > m + 8.f || (m == -INFINITY && mx > -INFINITY);
          if (__any_sync(0xffffffffu, grow)) {
            const float mn = grow ? mx : m;
            const float f = grow ? fast_exp2(m - mn) : 1.f;  // 0 for the first maximum
            if (t > it.ta) {
              uint32_t o[32];
#pragma unroll 1
              for (int i = 0; i < HALVES * 2; ++i) {
                tmem_ld32(to + i * 32, o);
                tmem_ready32(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st32(to + i * 32, o);
              }
            }
            l *= f;
            m = mn;
          }
          const float z = m == -INFINITY ? 0.f : -m;
          float sum = 0.f, sum1 = 0.f;
#pragma unroll
          for (int i = 0; i < 128; i += 2) {
            const float a = fast_exp2(fmaf(__uint_as_float(x[i]), c.scale_log2, z)), b = fast_exp2(fmaf(__uint_as_float(x[i + 1]), c.scale_log2, z));
            sum += a;
            sum1 += b;
            x[i / 2] = pack2<BF16>(a, b);
          }
          l += sum + sum1;
        }
        tmem_st32(ts, x);
        tmem_st32(ts + 32, x + 32);
        // rows of V past the sequence's end lie in its last page and may hold anything: zero them for 0 * V
        const int end = it.kv_len - j0;
        if (q == 0 && end < kKeys && it.kv_len % c.page_tokens != 0) {
          const uint32_t vp = 2 * step + 1;
          if (!(ok = warp_wait(full(vp % SLOTS), (vp / SLOTS) & 1, dead))) break;
          if (wg >= end)
#pragma unroll
            for (int i = 0; i < HALVES * 8; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(ring + (vp % SLOTS) * kTile + (i >> 3) * kHalf + wg * 128 + (i & 7) * 16),
                           "r"(0) : "memory");
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tc_wait_st();
        tc_fence_before();
        mbar_arrive(p_full + 8 * q);
      }
      if (!ok) break;
      if (!(ok = open())) break;

      if (!(ok = warp_wait(o_full + 8 * q, done & 1, dead))) break;
      ++done;
      tc_fence_after();
      const bool whole = it.whole;
      const int tok = (it.row + r) / c.group, gh = (it.row + r) - tok * c.group;
      const int64_t o = (it.row0 + tok) * (int64_t)(c.kv_heads * c.group) + it.head * c.group + gh;
      float* const part = P.a.part + (int64_t)(2 * blockIdx.x + (it.inside ? 0 : 1)) * P.a.part_floats;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll 1
      for (int i = 0; i < HALVES * 2; ++i) {
        uint32_t v[32];
        tmem_ld32(to + i * 32, v);
        tmem_ready32(v);
        if (r < it.rows) {
          if (whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (i * 32 + e < c.v_dim) {
                uint4 w;
                w.x = pack2<BF16>(__uint_as_float(v[e]) * inv, __uint_as_float(v[e + 1]) * inv);
                w.y = pack2<BF16>(__uint_as_float(v[e + 2]) * inv, __uint_as_float(v[e + 3]) * inv);
                w.z = pack2<BF16>(__uint_as_float(v[e + 4]) * inv, __uint_as_float(v[e + 5]) * inv);
                w.w = pack2<BF16>(__uint_as_float(v[e + 6]) * inv, __uint_as_float(v[e + 7]) * inv);
                *reinterpret_cast<uint4*>(P.a.out + o * c.v_dim + i * 32 + e) = w;
              }
          } else {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              if (i * 32 + e < c.v_dim)  // rows contiguous, so that a warp's store is one
                *reinterpret_cast<uint4*>(part + ((i * 8 + e / 4) * P.a.part_rows + r) * 4) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
      }
      tc_fence_before();
      if (r < it.rows) {
        if (!whole) {
          part[kItemRows * c.v_dim + r] = m;
          part[kItemRows * (c.v_dim + 1) + r] = l;
        } else if (P.a.lse) {
          P.a.lse[o] = l == 0.f ? -INFINITY : fmaf(m, 0.693147180559945f, logf(l));
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0 && *dead) P.a.cuts[blockIdx.x].error = 1;
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---- host -----------------------------------------------------------------------------------------
template <bool BF16, int HALVES, int SLOTS>
void launch_kernel(const TcParams& P, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, cudaStream_t s) {
  auto* const f = attend_tc_kernel<BF16, HALVES, SLOTS>;
  const int smem = kBars * 8 + 1024 + (2 + SLOTS) * HALVES * kKeys * 128;
  cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  f<<<P.a.grid, kThreads, smem, s>>>(P, k, v, q);
}

}  // namespace

bool attend_tc_fits(const CacheParams& c) { return c.v && c.head_dim <= 128 && c.group <= kItemRows && pages_fit(c, kKeys); }

AttendShape attend_tc_shape(const CacheParams& c, int sms) { return {sms, kItemRows, kItemRows * (c.v_dim + 2), 1}; }

bool launch_attend_tc(const AttendParams& A, bool bf16, cudaStream_t s) {
  TcParams P;
  P.a = A;
  P.box = pool_boxes(A.c, kKeys);
  P.item_tokens = kItemRows / A.c.group;
  CUtensorMap k, v, q;
  if (!pool_map(&k, A.c.k, A.c, bf16, P.box) || !pool_map(&v, A.c.v, A.c, bf16, P.box) || !query_map(&q, A.c, bf16, P.item_tokens, A.c.group))
    return false;
  if (A.c.head_dim <= 64) bf16 ? launch_kernel<true, 1, 8>(P, k, v, q, s) : launch_kernel<false, 1, 8>(P, k, v, q, s);
  else bf16 ? launch_kernel<true, 2, 5>(P, k, v, q, s) : launch_kernel<false, 2, 5>(P, k, v, q, s);
  return true;
}

}  // namespace ztcp
