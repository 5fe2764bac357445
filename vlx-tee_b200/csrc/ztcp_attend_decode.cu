// ztcp_attend_decode.cu -- attention of the newest tokens over a paged cache (ztcp_attend_pages) for items of few
// rows: one token per sequence, or a few, times a group of heads.
//
// The mathematics is that of ztcp_attend.cu.  Bound: a K and V row serves at most N rows here, so the time is that
// of reading K and V once, and the kernel's one job is to keep that many bytes in flight with little else to do.
// The products are turned over, so that the keys fill the tensor core's 128 lanes and the few rows its N columns:
//   S^T[128 keys, N]   = K Q^T        (K, Q K-major)
//   O^T[128 columns, N] += V^T P^T    (V as it lies, MN-major; P^T from shared memory)
// A tile of 128 keys is then one thread per key in the softmax, which touches N scores, and a handful of
// tcgen05.mma by one thread: about 500 instructions per warp where a 16-row mma.sync tile needed 4,000 (measured:
// 359 us for 48 sequences of up to 8,192 tokens, 32/8 heads of 128, against 144 us to read K and V once).
//
// Warps.  0-3: softmax, a thread per key; 4: one thread issues the products; 5: TMA.  K and V tiles pass a ring of
// slots of up to 128 columns, one box per page.  A row's maximum over the tile is a redux per warp and an exchange
// through shared memory; sums stay per thread until the item ends.  O^T is rescaled only when a maximum has grown
// by more than 2^8 over the one in use.  For single-buffer pools V's columns are those of the K tile itself.
//
// Work, joining of shared items and bounded waits as in ztcp_attend_tc.cu.
#include "ztcp_tc.cuh"

namespace ztcp {

namespace {

constexpr int kThreads = 192;
constexpr int kMmaWarp = 4, kTmaWarp = 5;
constexpr int kBars = 40;  // barrier slots at the start of shared memory

struct DecodeParams {
  AttendParams a;
  PoolBoxes box;
};

// KG: 64-column groups of K; MB: 128-column blocks of V; N: rows of an item.
template <int KG, int MB, int N, bool SHARED>
struct Shape {
  static constexpr int kGroups = KG == 1 ? 1 : 2;                       // column groups of a slot
  static constexpr int kSlotBytes = kGroups * kGroupBytes;
  static constexpr int kKSlots = SHARED ? 1 + MB : (KG + 1) / 2;        // slots of a tile's K (shared: group 0, then V's pairs)
  static constexpr int kTileSlots = SHARED ? kKSlots : 2 * kKSlots;
  static constexpr int kQBytes = KG * N * 128;
  static constexpr int kPBytes = N * kKeys * 2;
  static constexpr int kSlots = (232448 - 4096 - kQBytes - kPBytes) / kSlotBytes;
  static constexpr int kSmem = kBars * 8 + 1024 + kSlots * kSlotBytes + kQBytes + kPBytes;
  static constexpr int kCols = (2 + MB) * N <= 64 ? 64 : ((2 + MB) * N <= 128 ? 128 : 256);
  static_assert(kSlots >= kTileSlots && 2 * kSlots + 8 <= kBars && (2 + MB) * N <= kCols, "shape");
  // first column group, and number of groups, of slot s of a tile's K
  static __device__ __forceinline__ int group(int s) { return SHARED ? (s == 0 ? 0 : 2 * s - 1) : s * kGroups; }
  static __device__ __forceinline__ int groups(int s) { return SHARED && s == 0 ? 1 : kGroups; }
};

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t addr, uint32_t* r) {
  if constexpr (N == 32) {
    tmem_ld32(addr, r);
    tmem_ready32(r);
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr) : "memory");
  }
}
template <int N>
__device__ __forceinline__ void tmem_st_cols(uint32_t addr, const uint32_t* r) {
  if constexpr (N == 32) tmem_st32(addr, r);
  else
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
                 "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// P^T, rows of the product contiguous per key: 32-byte swizzle, 8-key groups 256 bytes apart, the next 16 rows one
// block of 128 keys (4,096 bytes) on.
__device__ __forceinline__ uint64_t p_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(kKeys * 32 >> 4) << 16 | (uint64_t)(256 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)6 << 61;
}

template <bool BF16, int KG, int MB, int N, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1)
attend_decode_kernel(const __grid_constant__ DecodeParams P, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using Sh = Shape<KG, MB, N, SHARED>;
  constexpr int kSlots = Sh::kSlots, kTS = Sh::kTileSlots, kKS = Sh::kKSlots;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int dead_s;
  __shared__ uint32_t tmem_s;
  __shared__ float4 s_max[2][N], s_sum[N];  // per row: one value of each softmax warp
  const CacheParams& c = P.a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  volatile int* const dead = &dead_s;

  const uint32_t bars = smem_u32(smem_raw);
  const uint32_t ring = (bars + kBars * 8 + 1023) & ~1023u;
  const uint32_t qbuf = ring + kSlots * Sh::kSlotBytes, pbuf = qbuf + Sh::kQBytes;
  auto full = [&](uint32_t s) { return bars + s * 8; };
  auto empty = [&](uint32_t s) { return bars + (kSlots + s) * 8; };
  const uint32_t q_full = bars + 2 * kSlots * 8, s_full = q_full + 8, p_full = s_full + 16, pv_done = p_full + 8, meet = pv_done + 8,
                 drain = meet + 8;

  int64_t at;
  Spot spot;
  const SplitSpan S = locate(c.n_seqs, P.a.grid, [&](int b) { return seq_work<N>(c, b); },
                             [&](const SplitSpan& s) { return blockIdx.x < s.n ? s.begin(blockIdx.x) : (int64_t)-1; }, &at, &spot);
  if (at < 0) {
    if (tid == 0) P.a.cuts[blockIdx.x] = Cut{};
    return;
  }
  if (tid == 0) {
    dead_s = 0;
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(q_full, 128);
    mbar_init(s_full, 1);
    mbar_init(s_full + 8, 1);
    mbar_init(p_full, 128);
    mbar_init(pv_done, 1);
    mbar_init(meet, 4);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "n"(Sh::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;

  Walk<N> walk;
  walk.begin(c, spot, at, S.begin(blockIdx.x + 1));

  if (warp == kTmaWarp) {
    // ---- TMA: a tile's slots in turn through the ring; lane p fetches page p of the tile ------------
    const int per_tile = kKeys / P.box.rows;
    uint32_t pos = 0;
    bool ok = true;
    while (ok && walk.next(c)) {
      const Item<N>& it = walk.it;
      for (int t = it.ta; ok && t < it.tb; ++t) {
        const int j = t * kKeys + lane * P.box.rows;
        int32_t row = P.box.pool_rows;  // past the sequence's end, or a bad page: zeros
        if (lane < per_tile && j < it.s.kv_len) {
          const int64_t r = pool_row(c, it.b, j);
          if (r >= 0) row = (int32_t)r;
        }
#pragma unroll
        for (int s = 0; s < kTS; ++s, ++pos) {
          const uint32_t slot = pos % kSlots;
          ok = ok && (pos < kSlots || mbar_wait(empty(slot), (pos / kSlots - 1) & 1, dead));
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          const bool isv = !SHARED && s >= kKS;
          const int ks = isv ? s - kKS : s;
          const int g0 = Sh::group(ks), n = Sh::groups(ks);
          if (lane == 0) mbar_expect(full(slot), n * kGroupBytes);
          __syncwarp();
          if (lane < per_tile)
            for (int g = 0; g < n; ++g)
              tma_load(ring + slot * Sh::kSlotBytes + g * kGroupBytes + lane * P.box.rows * 128, isv ? &vmap : &kmap, (g0 + g) * 64, it.h, row,
                       full(slot));
        }
      }
    }
    if (lane == 0) write_cut<N>(P.a, S, c, spot, at, 0);
    if (*dead) {  // after a timeout: no copy may be in flight when the CTA ends
      int none = 0;
      for (uint32_t p = pos > kSlots ? pos - kSlots : 0; p < pos; ++p) mbar_wait(full(p % kSlots), (p / kSlots) & 1, &none);
    }
  } else if (warp == kMmaWarp) {
    // ---- products ----------------------------------------------------------------------------------
    if (lane == 0) {
      const uint32_t qk = inst_desc(BF16, N, false, false), pv = inst_desc(BF16, N, true, true);
      const int ksteps = c.head_dim / 16;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t n) {  // the n-th completion (from 0)
        ok = ok && mbar_wait(bar, n & 1, dead);
        return ok;
      };
      auto scores = [&](uint32_t step) {  // S^T of the CTA's tile `step`
        for (int s = 0; s < kKS; ++s) {
          const uint32_t pos = step * kTS + s, slot = pos % kSlots;
          if (!wait(full(slot), pos / kSlots)) return;
          tc_fence_after();
          const uint32_t kb = ring + slot * Sh::kSlotBytes;
          const int g0 = Sh::group(s), n = Sh::groups(s);
          for (int g = 0; g < n; ++g) {
            const uint32_t qb = qbuf + (g0 + g) * N * 128;
            for (int k = 0; k < 4 && (g0 + g) * 4 + k < ksteps; ++k)
              mma_ss(tmem + (step & 1) * N, smem_desc(kb + g * kGroupBytes + k * 32, 16, 1024), smem_desc(qb + k * 32, 16, 1024), qk,
                     g0 + g > 0 || k > 0);
          }
          if (!SHARED || s == 0) tc_commit(empty(slot));
        }
        tc_commit(s_full + 8 * (step & 1));
      };
      auto values = [&](uint32_t step, bool acc) {  // O^T += V^T P^T
        for (int mb = 0; mb < MB; ++mb) {
          const uint32_t pos = step * kTS + (SHARED ? 1 : kKS) + mb, slot = pos % kSlots;
          if (!wait(full(slot), pos / kSlots)) return;
          tc_fence_after();
          const uint32_t vb = ring + slot * Sh::kSlotBytes;
          // one group of columns only (KG = 1): the block's upper half repeats rows nobody reads
          for (int k = 0; k < kKeys / 16; ++k)
            mma_ss(tmem + (2 + mb) * N, smem_desc(vb + k * 2048, KG == 1 ? 1024 : kGroupBytes, 1024), p_desc(pbuf + k * 512), pv, acc || k > 0);
          tc_commit(empty(slot));
        }
        tc_commit(pv_done);
      };
      uint32_t step = 0, items = 0;
      while (ok && walk.next(c)) {
        const int n = walk.it.tb - walk.it.ta;
        if (!wait(q_full, items)) break;
        ++items;
        tc_fence_after();
        scores(step);
        for (int t = 0; ok && t < n; ++t, ++step) {
          if (!SHARED && t + 1 < n) scores(step + 1);  // under the softmax of this tile
          if (!wait(p_full, step)) break;
          tc_fence_after();
          values(step, t > 0);
          if (SHARED && t + 1 < n && ok) scores(step + 1);
        }
      }
      if (*dead) {  // no product may be in flight when TMEM is freed
        int none = 0;
        tc_commit(drain);
        mbar_wait(drain, 0, &none);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: a thread per key -------------------------------------------------------------------
    const uint32_t lanes = (uint32_t)warp << 21;
    const int chunks = c.head_dim / 8;
    uint32_t step = 0, meets = 0;
    // The four warps meet.  Not a bar.sync, which no bound could end if a warp had left after a timeout.
    auto meet_warps = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(meet);
      return warp_wait(meet, meets++ & 1, dead);
    };
    auto load_q = [&](const Item<N>& it) {
      for (int i = tid; i < it.rows * KG * 8; i += 128) {
        const int r = i / (KG * 8), x = i - r * (KG * 8);
        const int tok = (it.row + r) / c.group, gh = (it.row + r) - tok * c.group;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (x < chunks)
          v = __ldg(reinterpret_cast<const uint4*>(c.q + (it.s.row0 + tok) * c.q_token_stride + (int64_t)(it.h * c.group + gh) * c.q_head_stride) + x);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(qbuf + (x >> 3) * N * 128 + r * 128 + (((x & 7) ^ (r & 7)) << 4)), "r"(v.x),
                     "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_full);
    };
    bool have = walk.next(c), ok = true;
    if (have) load_q(walk.it);
    while (ok && have) {
      const Item<N> it = walk.it;
      const int rows = it.rows;
      float m[N], l[N];
#pragma unroll
      for (int n = 0; n < N; ++n) m[n] = -INFINITY, l[n] = 0.f;
      const int vis0 = visible_keys(c, it.s, it.row / c.group);  // what every row sees
      for (int t = it.ta; t < it.tb; ++t, ++step) {
        const int j0 = t * kKeys, j = j0 + tid;
        const bool there = j < it.s.kv_len && pool_row(c, it.b, j) >= 0;
        if (!(ok = warp_wait(s_full + 8 * (step & 1), (step >> 1) & 1, dead))) break;
        tc_fence_after();
        uint32_t x[N];
        tmem_ld_cols<N>(tmem + lanes + (step & 1) * N, x);
        if (j0 + kKeys > vis0 || !__all_sync(0xffffffffu, there)) {
#pragma unroll
          for (int n = 0; n < N; ++n)
            if (n < rows && !(there && j < visible_keys(c, it.s, (it.row + n) / c.group))) x[n] = 0xff800000u;
        }
        float* const mine = reinterpret_cast<float*>(s_max[step & 1]) + warp;
#pragma unroll
        for (int n = 0; n < N; n += 4)
          if (n < rows) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = warp_max(__uint_as_float(x[n + e]));
              if (lane == n + e) mine[4 * (n + e)] = w;
            }
          }
        if (!(ok = meet_warps())) break;
        float f[N];
        bool grow = false;
#pragma unroll
        for (int n = 0; n < N; n += 4)
          if (n < rows) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 w = s_max[step & 1][n + e];
              const float mx = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)) * c.scale_log2;
              f[n + e] = 1.f;
              if (mx > m[n + e] + 8.f || (m[n + e] == -INFINITY && mx > -INFINITY)) {
                f[n + e] = fast_exp2(m[n + e] - mx);  // 0 for the first maximum
                m[n + e] = mx;
                l[n + e] *= f[n + e];
                grow = grow || n + e < rows;
              }
            }
          }
        if (t > it.ta) {  // the product before has read P and written O
          if (!(ok = warp_wait(pv_done, (step - 1) & 1, dead))) break;
          if (grow) {  // the same in every thread
            tc_fence_after();
#pragma unroll 1
            for (int mb = 0; mb < MB; ++mb) {
              uint32_t o[N];
              tmem_ld_cols<N>(tmem + lanes + (2 + mb) * N, o);
#pragma unroll
              for (int n = 0; n < N; n += 4)
                if (n < rows) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) o[n + e] = __float_as_uint(__uint_as_float(o[n + e]) * f[n + e]);
                }
              tmem_st_cols<N>(tmem + lanes + (2 + mb) * N, o);
            }
            tc_wait_st();
          }
        }
#pragma unroll
        for (int n = 0; n < N; n += 8)
          if (n < rows) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float z = m[n + e] == -INFINITY ? 0.f : m[n + e];
              p[e] = n + e < rows ? fast_exp2(fmaf(__uint_as_float(x[n + e]), c.scale_log2, -z)) : 0.f;
              l[n + e] += p[e];
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(pbuf + (n >> 4) * (kKeys * 32) + tid * 32 +
                                                                        ((((n >> 3) & 1) ^ ((tid >> 2) & 1)) << 4)),
                         "r"(pack2<BF16>(p[0], p[1])), "r"(pack2<BF16>(p[2], p[3])), "r"(pack2<BF16>(p[4], p[5])), "r"(pack2<BF16>(p[6], p[7]))
                         : "memory");
          }
        // rows of V past the sequence's end lie in its last page and may hold anything: zero them for 0 * V
        if (j0 + kKeys > it.s.kv_len && it.s.kv_len % c.page_tokens != 0) {
          for (int s = SHARED ? 1 : kKS; s < kTS; ++s) {
            const uint32_t pos = step * kTS + s, slot = pos % kSlots;
            if (!(ok = warp_wait(full(slot), (pos / kSlots) & 1, dead))) break;
            if (j >= it.s.kv_len)
              for (int i = 0; i < Sh::kGroups * 8; ++i)
                asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(ring + slot * Sh::kSlotBytes + (i >> 3) * kGroupBytes + tid * 128 + (i & 7) * 16),
                             "r"(0) : "memory");
          }
          if (!ok) break;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tc_fence_before();
        mbar_arrive(p_full);
      }
      if (!ok) break;
      have = walk.next(c);
      if (have) load_q(walk.it);  // the item's last QK^T has been seen

#pragma unroll
      for (int n = 0; n < N; ++n)
        if (n < rows) {
          float w = l[n];
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) w += __shfl_xor_sync(0xffffffffu, w, d);
          if (lane == 0) reinterpret_cast<float*>(s_sum)[4 * n + warp] = w;
        }
      if (!(ok = meet_warps())) break;
      if (!(ok = warp_wait(pv_done, (step - 1) & 1, dead))) break;
      tc_fence_after();
      const bool whole = it.ta == 0 && it.tb == it.nt;
      float* const part = P.a.part + (int64_t)(2 * blockIdx.x + (it.inside ? 0 : 1)) * P.a.part_floats;
      const int tok0 = it.row / c.group, gh0 = it.row - tok0 * c.group;
#pragma unroll 1
      for (int mb = 0; mb < MB; ++mb) {
        uint32_t o[N];
        tmem_ld_cols<N>(tmem + lanes + (2 + mb) * N, o);
        const int col = mb * 128 + tid;
        int tok = tok0, gh = gh0;
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (n < rows) {
            const float4 w = s_sum[n];
            const float sum = (w.x + w.y) + (w.z + w.w);
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
            const int64_t r = (it.s.row0 + tok) * (int64_t)(c.kv_heads * c.group) + it.h * c.group + gh;
            const float v = __uint_as_float(o[n]);
            if (col < c.v_dim) {
              if (whole) P.a.out[r * c.v_dim + col] = (uint16_t)(pack2<BF16>(v * inv, 0.f) & 0xffff);
              else part[n * c.v_dim + col] = v;
            }
            if (mb == 0 && tid == n) {
              if (!whole) {
                part[P.a.part_rows * c.v_dim + n] = m[n];
                part[P.a.part_rows * (c.v_dim + 1) + n] = sum;
              } else if (P.a.lse) {
                P.a.lse[r] = sum == 0.f ? -INFINITY : fmaf(m[n], 0.693147180559945f, logf(sum));
              }
            }
            if (++gh == c.group) gh = 0, ++tok;
          }
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (tid == 0 && *dead) P.a.cuts[blockIdx.x].error = 1;
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(Sh::kCols) : "memory");
  }
}

// ---- host -----------------------------------------------------------------------------------------
template <bool BF16, int KG, int MB, int N, bool SHARED>
void launch_kernel(const DecodeParams& P, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  auto* const f = attend_decode_kernel<BF16, KG, MB, N, SHARED>;
  constexpr int smem = Shape<KG, MB, N, SHARED>::kSmem;
  cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  f<<<P.a.grid, kThreads, smem, s>>>(P, k, v);
}

template <bool BF16>
void launch_any(const DecodeParams& P, const CUtensorMap& k, const CUtensorMap& v, cudaStream_t s) {
  const CacheParams& c = P.a.c;
  if (!c.v) P.a.part_rows == 16 ? launch_kernel<BF16, 9, 4, 16, true>(P, k, v, s) : launch_kernel<BF16, 9, 4, 32, true>(P, k, v, s);
  else if (c.head_dim <= 64) launch_kernel<BF16, 1, 1, 16, false>(P, k, v, s);
  else if (c.head_dim <= 128) launch_kernel<BF16, 2, 1, 16, false>(P, k, v, s);
  else launch_kernel<BF16, 4, 2, 16, false>(P, k, v, s);
}

}  // namespace

// Single-buffer pools need V to begin at the second column group.
bool attend_decode_fits(const CacheParams& c) { return (c.v ? c.head_dim <= 256 : c.v_col == 64) && pages_fit(c); }

// Single-buffer pools often have more than 16 heads per KV head: 32 rows an item then, so that K and V are read
// half as often.
AttendShape attend_decode_shape(const CacheParams& c, int sms, int64_t rows) {
  const int n = !c.v && rows > 16 ? 32 : 16;
  return {sms, n, n * (c.v_dim + 2)};
}

bool launch_attend_decode(const AttendParams& A, bool bf16, cudaStream_t s) {
  DecodeParams P;
  P.a = A;
  P.box = pool_boxes(A.c);
  CUtensorMap k, v;
  if (!pool_map(&k, A.c.k, A.c, bf16, P.box)) return false;
  v = k;
  if (A.c.v && !pool_map(&v, A.c.v, A.c, bf16, P.box)) return false;
  if (bf16) launch_any<true>(P, k, v, s);
  else launch_any<false>(P, k, v, s);
  return true;
}

}  // namespace ztcp
