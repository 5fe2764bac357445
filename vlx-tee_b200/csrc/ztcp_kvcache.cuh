// ztcp_kvcache.cuh -- shared declarations of the kernels behind include/ztcp_kvcache.h.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

namespace ztcp {

int32_t set_last_error(int32_t code, const std::string& msg);  // ztcp_capi.cu

constexpr long long kWaitCycles = 2000000000ll;  // bound of a wait inside a kernel: a second or so

// ------------------------------------------------------------------------------------------------
// Kernel parameters
// ------------------------------------------------------------------------------------------------
// A paged cache and its queries, validated by the host layer (ztcp_kvcache_capi.cu).
struct CacheParams {
  const uint16_t* k;
  const uint16_t* v;      // null: values are columns [v_col, head_dim) of K
  const uint16_t* q;
  int64_t q_token_stride, q_head_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* kv_lens;
  const int32_t* q_starts;  // null: one row per sequence
  int64_t pool_pages, total_rows;
  int32_t n_seqs, max_pages;
  int32_t page_tokens, page_shift;  // page_shift = log2(page_tokens), or -1
  int32_t kv_heads, group;          // group = query heads per KV head
  int32_t head_dim, v_dim, v_col;
  int32_t causal;
  float scale;
  float scale_log2;  // scale * log2(e): scores enter exp2
  int64_t wait_cycles;  // bound of a wait inside a kernel
  int32_t* status;
};

// What a CTA leaves to join.  Its share of the line begins and ends inside items: the part of an item that began
// before the share is its partial 0, the part of one that goes on behind it partial 1.
struct alignas(16) Cut {
  int64_t row0;                    // partial 1's item: the sequence's first row,
  int32_t row, rows, head, last;   // its first packed row, rows (0: no such item), KV head, and last CTA
  int32_t tiles[2];                // tiles in each partial (0: nothing was written)
  int32_t error, reserved[5];      // a wait of the CTA ran out
};

struct AttendParams {
  CacheParams c;
  uint16_t* out;   // [total_rows, kv_heads * group, v_dim]
  float* lse;      // [total_rows, kv_heads * group] or null
  Cut* cuts;       // one per CTA
  float* part;     // two per CTA, part_floats each: o [part_rows][v_dim], m [part_rows], l [part_rows]
  int32_t part_rows, part_floats;
  int32_t tiled;   // o lies as [v_dim / 4][part_rows][4]
  int32_t grid;    // CTAs that share the work
};

// Grid and partials of a kernel.
struct AttendShape {
  int32_t grid, part_rows, part_floats, tiled;
};

struct MassParams {
  CacheParams c;
  const float* lse;
  const float* mass;  // or null
  float decay;
  float* out;
  int32_t unit_pages;  // general kernel: whole pages per unit of work
  int32_t grid;        // tensor-core kernel: CTAs,
  int32_t* errors;     // one word each,
  float* part;         // and segment sums
};

// The attention kernels: whether they can take a call, their shape, and the launch (false: no tensor map could be
// made).  ztcp_attend.cu takes every call; ztcp_attend_tc.cu items of many rows, ztcp_attend_decode.cu of few.
AttendShape attend_shape(const CacheParams& c, int sms);
void launch_attend(const AttendParams& P, bool bf16, cudaStream_t s);
bool attend_tc_fits(const CacheParams& c);
AttendShape attend_tc_shape(const CacheParams& c, int sms);
bool launch_attend_tc(const AttendParams& P, bool bf16, cudaStream_t s);
bool attend_decode_fits(const CacheParams& c);
AttendShape attend_decode_shape(const CacheParams& c, int sms, int64_t rows);
bool launch_attend_decode(const AttendParams& P, bool bf16, cudaStream_t s);
// Joins what the kernel before it left to join, and writes the sequences' status; `rows`: of an item, at most.
void launch_attend_merge(const AttendParams& P, bool bf16, int64_t rows, cudaStream_t s);
void launch_page_mass(const MassParams& P, bool bf16, cudaStream_t s);
// Tensor-core kernel (ztcp_mass_tc.cu): whether it can take a call, workspace bytes, launch (false: no tensor map).
bool page_mass_tc_fits(const CacheParams& c);
int64_t page_mass_tc_workspace(const CacheParams& c, int64_t rows, int sms);
bool launch_page_mass_tc(MassParams m, int64_t rows, int sms, void* workspace, bool bf16, cudaStream_t s);

// ------------------------------------------------------------------------------------------------
// Device helpers
// ------------------------------------------------------------------------------------------------
#if defined(__CUDACC__)

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16-byte asynchronous copy; with `valid` false the destination is filled with zeros and nothing is read.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// D += A (16x16) * B (16x8), fp32 accumulation.
template <bool BF16>
__device__ __forceinline__ void mma16816(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two fp32 values rounded to the 16-bit type, `lo` in the low half.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
  else return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// Arithmetic on pairs of fp32.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x to about 2 ulp; 2^-inf = 0.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sequence b's rows and length, clamped to what the tables and the query buffer hold.
struct Seq {
  int32_t kv_len, q_len;
  int64_t row0;
};
__device__ __forceinline__ Seq load_seq(const CacheParams& c, int b) {
  Seq s;
  // (tiles that end behind the last token have to fit 32 bits)
  const int64_t cap = min((int64_t)c.max_pages * c.page_tokens, (int64_t)INT32_MAX - 4095);
  const int32_t n = __ldg(c.kv_lens + b);
  s.kv_len = n < 0 ? 0 : ((int64_t)n > cap ? (int32_t)cap : n);
  int64_t r0 = b, r1 = b + 1;
  if (c.q_starts) {
    r0 = __ldg(c.q_starts + b);
    r1 = __ldg(c.q_starts + b + 1);
  }
  r0 = r0 < 0 ? 0 : (r0 > c.total_rows ? c.total_rows : r0);
  r1 = r1 < r0 ? r0 : (r1 > c.total_rows ? c.total_rows : r1);
  s.row0 = r0;
  s.q_len = (int32_t)(r1 - r0);
  return s;
}
// Keys that row i (token kv_len - q_len + i) sees: tokens [0, visible).
__device__ __forceinline__ int visible_keys(const CacheParams& c, const Seq& s, int i) {
  if (!c.causal) return s.kv_len;
  const int n = s.kv_len - s.q_len + i + 1;
  return n < 0 ? 0 : (n > s.kv_len ? s.kv_len : n);
}
__device__ __forceinline__ int page_of(const CacheParams& c, int j) {
  return c.page_shift >= 0 ? j >> c.page_shift : j / c.page_tokens;
}
// Pool row (page * page_tokens + row in the page) of token j of sequence b, or -1 when its table entry lies
// outside the pool.
__device__ __forceinline__ int64_t pool_row(const CacheParams& c, int b, int j) {
  const int p = page_of(c, j);
  const int32_t e = __ldg(c.table + (int64_t)b * c.table_stride + p);
  return (e < 0 || e >= c.pool_pages) ? -1 : (int64_t)e * c.page_tokens + (j - p * c.page_tokens);
}

// a / b for non-negative a; most values fit 32 bits, whose division is several times shorter.
__device__ __forceinline__ int64_t div_pos(int64_t a, int64_t b) {
  if (((uint64_t)(a | b) >> 32) == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
  return a / b;
}

// Work laid out on one line -- sequence by sequence, `count(b)` units each -- that a grid's CTAs share evenly.
struct SplitSpan {
  int64_t total;  // units in all
  int64_t share;  // units of a CTA (the last ones may have fewer or none)
  __device__ __forceinline__ int64_t begin(int cta) const { return total < share * cta ? total : share * cta; }
  __device__ __forceinline__ int64_t own_begin() const { return begin(blockIdx.x) < total ? begin(blockIdx.x) : (int64_t)-1; }
  // The CTA whose share holds unit w.
  __device__ __forceinline__ int owner(int64_t w) const { return (int)div_pos(w, share); }
};

struct Spot {
  int32_t seq;
  int64_t first;  // the sequence's first unit on the line
};

// Sums every sequence's units (block-wide, up to 32 warps) and finds the sequence that holds the first unit of this
// CTA's share (-1: it has none).  All threads get the span, that unit and its spot.
template <class Count>
__device__ __forceinline__ SplitSpan locate(int n_seqs, int grid, Count count, int64_t* want, Spot* spot) {
  __shared__ int64_t sm[34];
  const int t = threadIdx.x, nt = blockDim.x;
  const int per = (n_seqs + nt - 1) / nt;
  const int b0 = t * per < n_seqs ? t * per : n_seqs, b1 = b0 + per < n_seqs ? b0 + per : n_seqs;
  int64_t sum = 0;
  for (int b = b0; b < b1; ++b) sum += count(b);
  int64_t inc = sum;  // inclusive scan: within the warp, then over the warps' sums
  const int lane = t & 31, warp = t >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) sm[warp] = inc;
  __syncthreads();
  int64_t base = 0, total = 0;
  for (int w = 0; w < nt / 32; ++w) {
    if (w < warp) base += sm[w];
    total += sm[w];
  }
  SplitSpan S;
  S.total = total;
  S.share = div_pos(total + grid - 1, grid);
  if (S.share == 0) S.share = 1;
  const int64_t target = S.own_begin();
  int64_t at = base + inc - sum;
  if (target >= at && target < at + sum)
    for (int b = b0; b < b1; ++b) {
      const int64_t n = count(b);
      if (target < at + n) {
        sm[32] = b;
        sm[33] = at;
        break;
      }
      at += n;
    }
  __syncthreads();
  *want = target;
  spot->seq = target >= 0 ? (int32_t)sm[32] : 0;
  spot->first = target >= 0 ? sm[33] : 0;
  return S;
}

// One sequence's status: lengths outside the tables, then table entries outside the pool.  Called by one warp.
__device__ __forceinline__ void write_seq_status(const CacheParams& c, int b, int lane) {
  const int32_t raw = c.kv_lens[b];
  const Seq s = load_seq(c, b);
  bool bad_len = raw != s.kv_len;
  if (c.q_starts) {
    const int64_t r0 = c.q_starts[b], r1 = c.q_starts[b + 1];
    bad_len |= r0 != s.row0 || r1 != s.row0 + s.q_len;
  }
  bool bad = false;
  for (int p = lane; (int64_t)p * c.page_tokens < s.kv_len; p += 32) {
    const int32_t e = __ldg(c.table + (int64_t)b * c.table_stride + p);
    bad |= e < 0 || e >= c.pool_pages;
  }
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) c.status[b] = bad ? 6 : (bad_len ? 5 : 0);  // ZTCP_SEQ_*
}

#endif  // __CUDACC__

}  // namespace ztcp
