// ztcp_mass.cu -- attention weight per page (ztcp_page_mass), general kernel.
//
// Mathematics.  out[b, p] = decay * mass[b, p] + sum over rows r, heads and tokens j of page p of
// exp(s_rj - lse_r): with the log-sum-exp known, weights need one product and no second pass.  (s - lse is formed by
// one fma and then multiplied by log2 e, so that it is rounded as a small number; a score's products of 64 columns add up
// in the tensor cores' accumulator, which drops its lowest bits, and these parts in fp32.)
//
// Work.  A unit is as many whole pages as fit 64 keys (one, where a page is larger), of one sequence, all KV heads:
// its sums never cross CTAs, so there are no atomics and results repeat bit for bit.  Units of all sequences form
// one line that the CTAs share evenly.  Per step a CTA holds 64 keys of one head and up to 32 rows of its group
// in a ring of cp.async stages; keys are the product's rows, so that a key's weights add up within a thread.
#include "ztcp_kvcache.cuh"

namespace ztcp {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kKeys = 64;
constexpr int kQRows = 32;

__device__ __forceinline__ int seq_pages(const CacheParams& c, const Seq& s) {
  return (int)(((int64_t)s.kv_len + c.page_tokens - 1) / c.page_tokens);
}
__device__ __forceinline__ int seq_units(const MassParams& P, int b) {
  const Seq s = load_seq(P.c, b);
  return (seq_pages(P.c, s) + P.unit_pages - 1) / P.unit_pages;
}

// A step: unit `unit` of sequence b, 64-key part `sub` of it, KV head h, row chunk `rc`.
struct Cursor {
  Seq s;
  int64_t left;  // units to go, this one included
  int32_t b, units, unit, subs, sub, h, rcs, rc;
  __device__ __forceinline__ void load(const MassParams& P, int seq) {
    b = seq;
    s = load_seq(P.c, seq);
    units = (seq_pages(P.c, s) + P.unit_pages - 1) / P.unit_pages;
    rcs = (int)(((int64_t)s.q_len * P.c.group + kQRows - 1) / kQRows);
    if (rcs == 0) rcs = 1;
    subs = (P.unit_pages * P.c.page_tokens + kKeys - 1) / kKeys;
  }
  __device__ __forceinline__ void next(const MassParams& P) {
    if (++rc < rcs) return;
    rc = 0;
    if (++h < P.c.kv_heads) return;
    h = 0;
    if (++sub < subs) return;
    sub = 0;
    if (--left <= 0 || ++unit < units) return;
    unit = 0;
    do load(P, b + 1);
    while (units == 0);  // left > 0: a later sequence has units
  }
};

__device__ __forceinline__ uint32_t chunk_at(uint32_t base, int row, int chunk, int pitch) {
  return base + row * pitch + ((chunk ^ (row & 7)) << 4);
}

template <bool BF16, int STAGES, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM) page_mass_kernel(const __grid_constant__ MassParams P) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_neg[STAGES][kQRows];      // -lse of the stage's rows, -inf where a row adds nothing
  __shared__ int32_t s_lim[STAGES][kQRows];    // keys that the row sees
  __shared__ uint8_t s_there[STAGES][kKeys];   // the key lies in a pool page
  __shared__ float s_key[2][kKeys];
  const CacheParams& c = P.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  const int kb = warp & 3, rg = warp >> 2;  // 16 keys and 16 of the chunk's rows

  for (int b = blockIdx.x * kWarps + warp; b < c.n_seqs; b += gridDim.x * kWarps) {
    write_seq_status(c, b, lane);
    for (int p = seq_pages(c, load_seq(c, b)) + lane; p < c.max_pages; p += 32) P.out[(int64_t)b * c.max_pages + p] = 0.f;
  }
  int64_t at;
  Spot spot;
  const SplitSpan S = locate(c.n_seqs, gridDim.x, [&](int b) { return (int64_t)seq_units(P, b); }, &at, &spot);
  if (at < 0) return;
  Cursor cons;
  cons.load(P, spot.seq);
  cons.unit = (int32_t)(at - spot.first);
  cons.sub = cons.h = cons.rc = 0;
  cons.left = S.begin(blockIdx.x + 1) - at;
  Cursor prod = cons;

  const int pitch = (c.head_dim + 63) / 64 * 128;
  const int chunks = c.head_dim / 8;
  const int sbytes = (kKeys + kQRows) * pitch;
  const uint32_t ring = smem_u32(smem);

  auto issue = [&](int stage) {
    const uint32_t base = ring + stage * sbytes;
    const int u0 = prod.unit * P.unit_pages * c.page_tokens;  // the unit's first key
    const int end = min(prod.s.kv_len - u0, P.unit_pages * c.page_tokens);
    for (int r = tid >> 4; r < kKeys; r += kThreads / 16) {
      const int j = prod.sub * kKeys + r;
      const int64_t row = j < end ? pool_row(c, prod.b, u0 + j) : -1;
      if ((tid & 15) == 0) s_there[stage][r] = row >= 0;
      const int64_t off = row < 0 ? 0 : (row * c.kv_heads + prod.h) * c.head_dim;
      for (int ch = tid & 15; ch < chunks; ch += 16) cp_async16(chunk_at(base, r, ch, pitch), c.k + off + ch * 8, row >= 0);
    }
    const int r0 = prod.rc * kQRows, rows = prod.s.q_len * c.group - r0;
    for (int r = tid >> 4; r < kQRows; r += kThreads / 16) {
      const int tok = (r0 + r) / c.group, gh = (r0 + r) - tok * c.group;
      const int head = prod.h * c.group + gh;
      if (r < rows) {
        const uint16_t* const q = c.q + (prod.s.row0 + tok) * c.q_token_stride + (int64_t)head * c.q_head_stride;
        for (int ch = tid & 15; ch < chunks; ch += 16) cp_async16(chunk_at(base + kKeys * pitch, r, ch, pitch), q + ch * 8, true);
      }
      if ((tid & 15) == 0) {
        float neg = -INFINITY;
        if (r < rows) {
          const float x = __ldg(P.lse + (prod.s.row0 + tok) * (int64_t)(c.kv_heads * c.group) + head);
          if (x != -INFINITY) neg = -x;
        }
        s_neg[stage][r] = neg;
        s_lim[stage][r] = r < rows ? visible_keys(c, prod.s, tok) : 0;
      }
    }
    prod.next(P);
  };

  for (int i = 0; i < STAGES - 1; ++i) {
    if (prod.left > 0) issue(i);
    cp_async_commit();
  }

  const int nks = c.head_dim / 16;
  float k0 = 0.f, k1 = 0.f, page = 0.f;  // weights of keys g and g + 8 of the warp's block; warp 0: of a large page
  int stage = 0;
  while (cons.left > 0) {
    cp_async_wait<STAGES - 2>();
    __syncthreads();
    if (prod.left > 0) issue(stage == 0 ? STAGES - 1 : stage - 1);
    cp_async_commit();

    const int rows = cons.s.q_len * c.group - cons.rc * kQRows;
    if (rg * 16 < rows) {
      const uint32_t kbase = ring + stage * sbytes + kb * 16 * pitch, qbase = ring + stage * sbytes + (kKeys + rg * 16) * pitch;
      float sc[2][4] = {};
      for (int k0 = 0; k0 < nks; k0 += 4) {
        float part[2][4] = {};
        for (int ks = k0; ks < min(k0 + 4, nks); ++ks) {
          uint32_t a[4], b[4];
          ldmatrix4(a, chunk_at(kbase, (lane & 7) + (lane & 8), ks * 2 + (lane >> 4), pitch));
          // rows 0-7 and 8-15 of the row block, both k halves of each
          ldmatrix4(b, chunk_at(qbase, (lane & 7) + ((lane >> 1) & 8), ks * 2 + ((lane >> 3) & 1), pitch));
          mma16816<BF16>(part[0], a, b[0], b[1]);
          mma16816<BF16>(part[1], a, b[2], b[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[0][e] += part[0][e], sc[1][e] += part[1][e];
      }
      const int key = cons.unit * P.unit_pages * c.page_tokens + cons.sub * kKeys + kb * 16 + g;
      const bool ok0 = s_there[stage][kb * 16 + g], ok1 = s_there[stage][kb * 16 + g + 8];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = rg * 16 + n * 8 + 2 * t4 + e;
          const float neg = s_neg[stage][r];
          const int lim = s_lim[stage][r];
          if (ok0 && key < lim) k0 += fast_exp2(fmaf(sc[n][e], c.scale, neg) * 1.44269504088896f);
          if (ok1 && key + 8 < lim) k1 += fast_exp2(fmaf(sc[n][2 + e], c.scale, neg) * 1.44269504088896f);
        }
    }

    if (cons.rc + 1 == cons.rcs && cons.h + 1 == c.kv_heads) {  // the part's last step: sum its pages
      k0 += __shfl_xor_sync(0xffffffffu, k0, 1);
      k0 += __shfl_xor_sync(0xffffffffu, k0, 2);
      k1 += __shfl_xor_sync(0xffffffffu, k1, 1);
      k1 += __shfl_xor_sync(0xffffffffu, k1, 2);
      __syncthreads();  // the sums of the part before have been read
      if (t4 == 0) {
        s_key[rg][kb * 16 + g] = k0;
        s_key[rg][kb * 16 + g + 8] = k1;
      }
      __syncthreads();
      k0 = k1 = 0.f;
      const int T = c.page_tokens;
      const int first = cons.unit * P.unit_pages, pages = min(P.unit_pages, seq_pages(c, cons.s) - first);
      for (int p = warp; p < pages; p += kWarps) {
        const int a = p * T - cons.sub * kKeys, z = min(a + T, kKeys);
        float x = 0.f;
        for (int j = max(a, 0) + lane; j < z; j += 32) x += s_key[0][j] + s_key[1][j];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
        if (cons.subs > 1) x = page += x;  // the unit is one page
        if (cons.sub + 1 == cons.subs) {
          page = 0.f;
          const int64_t o = (int64_t)cons.b * c.max_pages + first + p;
          if (lane == 0) P.out[o] = P.mass ? fmaf(P.decay, P.mass[o], x) : x;
        }
      }
    }
    cons.next(P);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  cp_async_wait<0>();
}

template <bool BF16, int STAGES, int PER_SM>
void launch_kernel(const MassParams& P, int sms, cudaStream_t s) {
  const int smem = STAGES * (kKeys + kQRows) * ((P.c.head_dim + 63) / 64 * 128);
  auto* const k = page_mass_kernel<BF16, STAGES, PER_SM>;
  cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  k<<<sms * PER_SM, kThreads, smem, s>>>(P);
}

}  // namespace

void launch_page_mass(const MassParams& P, bool bf16, cudaStream_t s) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return;
  if (P.c.head_dim <= 128) bf16 ? launch_kernel<true, 4, 2>(P, sms, s) : launch_kernel<false, 4, 2>(P, sms, s);
  else if (P.c.head_dim <= 256) bf16 ? launch_kernel<true, 4, 1>(P, sms, s) : launch_kernel<false, 4, 1>(P, sms, s);
  else bf16 ? launch_kernel<true, 2, 1>(P, sms, s) : launch_kernel<false, 2, 1>(P, sms, s);
}

}  // namespace ztcp
