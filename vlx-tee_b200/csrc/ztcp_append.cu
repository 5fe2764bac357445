// ztcp_append.cu -- norm, rotation and append of new tokens to the paged pool (ztcp_append_tokens).
//
// Mathematics.  Per query and key vector x: y = x * w / sqrt(mean(x^2) + eps) over the normed columns, then the
// leading rope_dim columns turn by the token's angles: (a, b) -> (a cos - b sin, b cos + a sin).  fp32 throughout,
// rounded once.
//
// A pass that is bound by memory: every vector is read once and written once, 16 bytes per lane, by a group of 8, 16 or
// 32 lanes, each with CH chunks of 8 columns, CH * lanes covering head_dim.  A pair's two columns lie in one chunk
// (interleaved) or in chunks rope_dim / 16 lanes apart, which trade values by shuffles; the token's cosines and sines
// stay in registers over its heads.
#include <algorithm>
#include <climits>

#include "ztcp_kvcache.cuh"
#include "../../include/ztcp_kvcache.h"

namespace ztcp {

namespace {

// A lane's part of the token's angles.  Halves paired: a lane of the first half takes its partner's value times -sin.
struct Angles {
  float cs[8], sn[8];
};

// Norm weights of eight columns.
struct Columns {
  uint64_t w[4];
};
__device__ __forceinline__ Columns read_weights(const float* w) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(w)), b = __ldg(reinterpret_cast<const float4*>(w) + 1);
  return {{pair(a.x, a.y), pair(a.z, a.w), pair(b.x, b.y), pair(b.z, b.w)}};
}

// One vector's norm and rotation in a group's registers: x[c] are the columns (lane + c * GROUP) * 8 on, in pairs.  All
// lanes of the warp take part (a shuffle over part of a warp costs several times as much), whatever their vector is.
// `weights(c)`: those of chunk c's columns; normed: whether the lane's vector has any.
template <bool INTER, int GROUP, int CH, class Weights>
__device__ __forceinline__ void norm_rotate(const ztcp_append& A, bool normed, Weights weights, float inv_n, const Angles& g, int lane,
                                            uint64_t x[CH][4]) {
  const int D = (int)A.geom.head_dim, R = (int)A.geom.rope_dim;
  if (A.q_weight || A.k_weight) {
    uint64_t ss = pair(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * GROUP) * 8;
      if (col >= A.norm_from && col < D)
#pragma unroll
        for (int e = 0; e < 4; ++e) ss = fma2(x[c][e], x[c][e], ss);
    }
    float s, s1;
    unpair(ss, s, s1);
    s += s1;
#pragma unroll
    for (int d = GROUP / 2; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float r = rsqrtf(fmaf(s, inv_n, A.eps));
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * GROUP) * 8;
      if (normed && col >= A.norm_from && col < D) {
        const Columns u = weights(c);
        const uint64_t r2 = pair(r, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[c][e] = mul2(mul2(x[c][e], r2), u.w[e]);
      }
    }
  }
  if (R == 0) return;
  const bool turns = lane * 8 < R;  // the lane's rotated columns are in its first chunk: rope_dim <= 8 * GROUP
  if (INTER) {
    if (turns)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float a, b;
        unpair(x[0][e], a, b);
        x[0][e] = pair(a * g.cs[2 * e] - b * g.sn[2 * e], b * g.cs[2 * e] + a * g.sn[2 * e]);
      }
  } else {
    const int half = R / 16;  // lanes to a pair's other half
    const int other = lane < half ? lane + half : (lane < 2 * half ? lane - half : lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float a, b;
      unpair(x[0][e], a, b);
      const uint64_t y = pair(__shfl_sync(0xffffffffu, a, other, GROUP), __shfl_sync(0xffffffffu, b, other, GROUP));
      if (turns) x[0][e] = fma2(x[0][e], pair(g.cs[2 * e], g.cs[2 * e + 1]), mul2(y, pair(g.sn[2 * e], g.sn[2 * e + 1])));
    }
  }
}

// The lane's angles at row `row` of the table: 16-byte pieces 0..3 (cosines, then sines; interleaved: one of each).
__device__ __forceinline__ const float* angle_piece(const ztcp_append& A, const float* row, int lane, int piece) {
  const int R = (int)A.geom.rope_dim, half = R / 16;
  if (A.interleaved) return row + (piece & 1) * (R / 2) + lane * 4;
  return row + (piece >> 1) * (R / 2) + (lane < half ? lane : lane - half) * 8 + (piece & 1) * 4;
}
__device__ __forceinline__ void set_angles(const ztcp_append& A, const float4 p[4], int lane, Angles* g) {
  if (A.interleaved) {
    g->cs[0] = g->cs[1] = p[0].x, g->cs[2] = g->cs[3] = p[0].y, g->cs[4] = g->cs[5] = p[0].z, g->cs[6] = g->cs[7] = p[0].w;
    g->sn[0] = g->sn[1] = p[1].x, g->sn[2] = g->sn[3] = p[1].y, g->sn[4] = g->sn[5] = p[1].z, g->sn[6] = g->sn[7] = p[1].w;
  } else {
    const float s = lane < A.geom.rope_dim / 16 ? -1.f : 1.f;
    g->cs[0] = p[0].x, g->cs[1] = p[0].y, g->cs[2] = p[0].z, g->cs[3] = p[0].w, g->cs[4] = p[1].x, g->cs[5] = p[1].y, g->cs[6] = p[1].z, g->cs[7] = p[1].w;
    g->sn[0] = s * p[2].x, g->sn[1] = s * p[2].y, g->sn[2] = s * p[2].z, g->sn[3] = s * p[2].w;
    g->sn[4] = s * p[3].x, g->sn[5] = s * p[3].y, g->sn[6] = s * p[3].z, g->sn[7] = s * p[3].w;
  }
}

// Where a token's vectors (queries, keys, values in turn) come from and go to: one base each, shifted so that vector i
// lies i strides behind it.
struct Sources {
  const uint16_t *q, *k, *v;
  __device__ __forceinline__ void set(const ztcp_append& A, int64_t tok, int nq, int nk, int lane) {
    q = (const uint16_t*)A.q + tok * A.q_token_stride + lane * 8;
    k = (const uint16_t*)A.k + tok * A.k_token_stride - nq * A.k_head_stride + lane * 8;
    v = (const uint16_t*)A.v + tok * A.v_token_stride - (nq + nk) * A.v_head_stride + lane * 8;
  }
  __device__ __forceinline__ const uint16_t* at(const ztcp_append& A, int i, int nq, int nk) const {
    const uint16_t* const p = i < nq ? q : i < nq + nk ? k : v;
    return p + (int64_t)i * (int32_t)(i < nq ? A.q_head_stride : i < nq + nk ? A.k_head_stride : A.v_head_stride);
  }
};
struct Targets {
  uint16_t *q, *k, *v;
  __device__ __forceinline__ void set(const ztcp_append& A, int64_t tok, int64_t slot, int nq, int nk, int D, int lane) {
    q = (uint16_t*)A.q_out + tok * nq * D + lane * 8;
    k = (uint16_t*)A.k_pool + (slot * nk - nq) * D + lane * 8;
    v = (uint16_t*)A.v_pool + (slot * nk - nq - nk) * D + lane * 8;
  }
  __device__ __forceinline__ uint16_t* at(int i, int nq, int nk, int D) const { return (i < nq ? q : i < nq + nk ? k : v) + i * D; }
};

// A token's position and slot: whether its query and its K/V may be written.
struct Place {
  int64_t slot;
  int32_t pos;
  bool query, keep;
};
__device__ __forceinline__ Place place_of(const ztcp_append& A, int32_t pos, int64_t slot) {
  Place p;
  p.pos = pos;
  p.slot = slot;
  p.query = A.geom.rope_dim == 0 || (pos >= 0 && pos < A.max_pos);
  p.keep = p.query && slot >= 0 && slot < A.pool_pages * A.geom.num_tokens;
  return p;
}
__device__ __forceinline__ int32_t status_of(const ztcp_append& A, const Place& p) { return p.query && (p.keep || p.slot == -1) ? ZTCP_SEQ_OK : ZTCP_SEQ_BAD_BLOCK; }

// A vector in a lane's 16-byte pieces -> arithmetic, if it is a query or a key (`turned`; `any`: a vector of the warp
// is) -> its place.  Called by whole warps, lanes without a vector included.
template <bool BF16, bool INTER, int GROUP, int CH, class Weights>
__device__ __forceinline__ void finish(const ztcp_append& A, uint4 raw[CH], bool any, bool turned, bool normed, Weights weights, bool write,
                                       uint16_t* dst, int D, float inv_n, const Angles& g, int lane) {
  if (any) {
    uint64_t x[CH][4];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const uint32_t w[4] = {raw[c].x, raw[c].y, raw[c].z, raw[c].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<BF16>(w[e]);
        x[c][e] = pair(f.x, f.y);
      }
    }
    norm_rotate<INTER, GROUP, CH>(A, normed, weights, inv_n, g, lane, x);
    if (turned)
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float a, b;
          unpair(x[c][e], a, b);
          w[e] = pack2<BF16>(a, b);
        }
        raw[c] = make_uint4(w[0], w[1], w[2], w[3]);
      }
  }
  if (!write) return;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if ((lane + c * GROUP) * 8 < D) *reinterpret_cast<uint4*>(dst + c * GROUP * 8) = raw[c];
}

// Few tokens: a group per vector, several CTAs per token, so that the vectors are in flight on many SMs at once.
template <bool BF16, bool INTER, int GROUP, int CH>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ ztcp_append A, int32_t* status) {
  const int groups = blockDim.x / GROUP;
  const int tok = blockIdx.x, lane = threadIdx.x % GROUP;
  const int D = (int)A.geom.head_dim, R = (int)A.geom.rope_dim;
  const int nk = (int)A.geom.num_heads, nq = A.q ? (int)A.num_q_heads : 0, total = nq + nk + (A.v ? nk : 0);
  const float inv_n = 1.f / (float)(D - A.norm_from);
  Place p = {};
  Angles g;
  Sources from;
  Targets to;
  from.set(A, tok, nq, nk, lane);
  bool first = true;
  for (int i0 = blockIdx.y * groups + threadIdx.x / 32 * (32 / GROUP); i0 < total; i0 += gridDim.y * groups) {
    const int i = i0 + threadIdx.x % 32 / GROUP;  // i0: the warp's first
    uint4 raw[CH];
    const uint16_t* const src = from.at(A, i, nq, nk);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      raw[c] = make_uint4(0, 0, 0, 0);
      if (i < total && (lane + c * GROUP) * 8 < D) raw[c] = *reinterpret_cast<const uint4*>(src + c * GROUP * 8);
    }
    if (first) {  // after the first vector's loads are out
      first = false;
      p = place_of(A, R > 0 ? __ldg(A.positions + tok) : 0, __ldg(A.slots + tok));
      if (threadIdx.x == 0 && blockIdx.y == 0) status[tok] = status_of(A, p);
      to.set(A, tok, p.slot, nq, nk, D, lane);
      if (p.query && lane * 8 < R) {
        float4 piece[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k < 2 || !A.interleaved) piece[k] = __ldg(reinterpret_cast<const float4*>(angle_piece(A, A.rope_table + (int64_t)p.pos * R, lane, k)));
        set_angles(A, piece, lane, &g);
      }
    }
    const float* const w = i < nq ? A.q_weight : A.k_weight;
    finish<BF16, INTER, GROUP, CH>(A, raw, i0 < nq + nk, i < nq + nk, w && i < nq + nk,
                                   [&](int c) { return read_weights(w + (lane + c * GROUP) * 8 - A.norm_from); },
                                   i < total && (i < nq ? p.query : p.keep), to.at(i, nq, nk, D), D, inv_n, g, lane);
  }
}

// Many tokens: the vectors of all tokens form one line that the warps share evenly; a warp takes 32 / GROUP of them a
// step, STAGES steps ahead by cp.async into its lanes' own 16-byte places in shared memory (no lane reads another's, so
// nothing waits for anything but its own copies).  The next token's angles come the same way, its position and slot
// a token earlier still.  A lane's addresses step from vector to vector and are looked up anew where the kind changes,
// and with one chunk a lane the norm's weights stay in registers: the instructions are the limit.  Measured:
// 8,191 tokens of 32 + 8 + 8 vectors of 128 columns, neighbours paired, half of the columns rotated, in a graph of calls
// 46.6 us (57 with addresses and weights looked up for every vector), as a call in a stream 49.1, 4.1 TB/s; 4,096 of 16 + 1 of
// 576, 36.6 and 38.9 us, 4.2 TB/s; 8,192 of 48 of 128, halves paired, all rotated, 58.
// CTAs per SM: with halves paired a third one's registers were not enough (spilled; 8,192 tokens 75 us, with two 58).
template <bool INTER, int CH>
constexpr int kStreamCtas = CH == 1 && INTER ? 3 : 2;

template <bool BF16, bool INTER, int GROUP, int CH, int STAGES>
__global__ void __launch_bounds__(256, kStreamCtas<INTER, CH>) append_stream_kernel(const __grid_constant__ ztcp_append A, int32_t* status) {
  extern __shared__ uint4 ring[];  // [STAGES][CH][256], then the angles [2][4][256]
  constexpr int kPer = 32 / GROUP;
  const int tid = threadIdx.x, lane = tid % GROUP, sub = tid % 32 / GROUP;
  const int D = (int)A.geom.head_dim, R = (int)A.geom.rope_dim;
  const int nk = (int)A.geom.num_heads, nq = A.q ? (int)A.num_q_heads : 0, total = nq + nk + (A.v ? nk : 0);
  const float inv_n = 1.f / (float)(D - A.norm_from);
  const int steps = (total + kPer - 1) / kPer;  // of a token
  uint4* const angles = ring + STAGES * CH * 256;
  auto slot_at = [&](int stage, int c) { return smem_u32(ring + (stage * CH + c) * 256 + tid); };

  const int64_t units = A.n_tokens * steps, warps = (int64_t)gridDim.x * 8, w = (int64_t)blockIdx.x * 8 + tid / 32;
  const int64_t u0 = units * w / warps, u1 = units * (w + 1) / warps;
  if (u0 >= u1) return;
  int64_t tok = u0 / steps, ptok = tok;             // consumer and producer
  int i = (int)(u0 - tok * steps), pi = i;
  int left = (int)(u1 - u0), pleft = left;
  const int64_t last_tok = (u1 - 1) / steps;

  // the vectors' kinds begin at 0, nq and nq + nk
  auto kind_end = [&](int v) { return v < nq ? nq : v < nq + nk ? nq + nk : INT_MAX; };
  const uint16_t* src;  // the producer's next vector, pv; the next of its kind lies sstep on
  int64_t sstep;
  int pv, pend;
  auto seek_source = [&] {
    Sources from;
    from.set(A, ptok, nq, nk, lane);
    src = from.at(A, pv, nq, nk);
    sstep = kPer * (pv < nq ? A.q_head_stride : pv < nq + nk ? A.k_head_stride : A.v_head_stride);
    pend = kind_end(pv);
  };
  pv = pi * kPer + sub;
  seek_source();
  auto fetch = [&](int stage) {
    if (pv < total) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if ((lane + c * GROUP) * 8 < D) cp_async16(slot_at(stage, c), src + c * GROUP * 8, true);
    }
    --pleft;
    pv += kPer;
    src += sstep;
    if (++pi == steps) {
      pi = 0;
      pv = sub;
      ++ptok;
      seek_source();
    } else if (pv >= pend) {
      seek_source();
    }
  };
  auto fetch_angles = [&](int64_t t, const Place& p) {
    if (p.query && lane * 8 < R)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < 2 || !A.interleaved)
          cp_async16(smem_u32(angles + ((t & 1) * 4 + k) * 256 + tid), angle_piece(A, A.rope_table + (int64_t)p.pos * R, lane, k), true);
  };
  auto read_place = [&](int64_t t) {
    const int64_t at = t <= last_tok ? t : last_tok;
    return place_of(A, R > 0 ? __ldg(A.positions + at) : 0, __ldg(A.slots + at));
  };

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (pleft > 0) fetch(s);
    cp_async_commit();
  }
  Place here = read_place(tok), next = read_place(tok + 1);
  fetch_angles(tok, here);
  cp_async_commit();
  cp_async_wait<0>();  // the pipeline is filled anyhow
  Angles g;
  uint16_t* dst = nullptr;  // the consumer's vector, v
  int v = i * kPer + sub, vend = 0;
  bool write = false, turned = false, normed = false;
  const float* weights = nullptr;
  Columns held = {};
  auto seek_target = [&] {
    Targets to;
    to.set(A, tok, here.slot, nq, nk, D, lane);
    dst = to.at(v, nq, nk, D);
    vend = kind_end(v);
    write = v < nq ? here.query : here.keep;
    turned = v < nq + nk;
    const float* const w = v < nq ? A.q_weight : turned ? A.k_weight : nullptr;
    normed = w != nullptr;
    weights = w + lane * 8 - A.norm_from;
    if (CH == 1 && normed && lane * 8 >= A.norm_from && lane * 8 < D) held = read_weights(weights);
  };
  bool fresh = true;
  int stage = 0, since = 0;  // since: steps of the token so far
  while (left > 0) {
    // this step's copies are STAGES - 1 groups old; the angles, sent with the first step of the token before, are as old
    // only if that token had as many steps here
    if (fresh && since < STAGES) cp_async_wait<0>();
    else cp_async_wait<STAGES - 2>();
    if (fresh) {
      fresh = false;
      since = 0;
      if (lane * 8 < R) {
        float4 piece[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 b = angles[((tok & 1) * 4 + k) * 256 + tid];
          piece[k] = make_float4(__uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w));
        }
        set_angles(A, piece, lane, &g);
      }
      v = i * kPer + sub;
      seek_target();
      fetch_angles(tok + 1, next);
      if (i == 0 && tid % 32 == 0) status[tok] = status_of(A, here);
    }
    if (pleft > 0) fetch(stage == 0 ? STAGES - 1 : stage - 1);
    cp_async_commit();
    uint4 raw[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) raw[c] = ring[(stage * CH + c) * 256 + tid];
    finish<BF16, INTER, GROUP, CH>(A, raw, i * kPer < nq + nk, turned, normed,
                                   [&](int c) { return CH == 1 ? held : read_weights(weights + c * GROUP * 8); }, write && v < total, dst, D, inv_n, g,
                                   lane);
    v += kPer;
    dst += kPer * D;
    if (v >= vend) seek_target();
    --left;
    ++since;
    if (++i == steps) {
      i = 0;
      ++tok;
      here = next;
      next = read_place(tok + 1);
      fresh = true;
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
}

// Streams when every warp of a full grid gets enough steps for its start.  Measured, few against many tokens' kernel: 32 + 8
// + 8 vectors of 128, halves paired, 1,024 tokens 13.7 / 13.9 us, 2,048 24.7 / 20.9 (neighbours paired 10.5 / 10.3 and
// 20.0 / 16.9); 8 + 8 + 8 of 64, 2,048 tokens 8.2 / 9.6, 4,096 17.1 / 15.5; 16 + 1 of 576, 512 tokens 11.8 / 8.6.
template <bool BF16, bool INTER, int GROUP, int CH, int STAGES>
void launch_one(const ztcp_append& A, int32_t* status, int sms, cudaStream_t s) {
  const int64_t vectors = (A.q ? A.num_q_heads : 0) + (A.v ? 2 : 1) * A.geom.num_heads;
  const int64_t steps = A.n_tokens * ((vectors + 32 / GROUP - 1) / (32 / GROUP));
  constexpr int kPerSm = kStreamCtas<INTER, CH>, kDeep = CH == 1 ? 10 : 3;
  if (steps >= (int64_t)sms * kPerSm * 8 * kDeep) {
    constexpr int smem = (STAGES * CH + 8) * 256 * 16;
    auto* const k = append_stream_kernel<BF16, INTER, GROUP, CH, STAGES>;
    cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    k<<<sms * kPerSm, 256, smem, s>>>(A, status);
    return;
  }
  const int64_t groups = std::min<int64_t>((vectors * GROUP + 31) / 32 * 32, 256) / GROUP;
  const int64_t y = std::min((vectors + groups - 1) / groups, (4 * sms + A.n_tokens - 1) / A.n_tokens);
  append_kernel<BF16, INTER, GROUP, CH><<<dim3((unsigned)A.n_tokens, (unsigned)y), (int)groups * GROUP, 0, s>>>(A, status);
}

template <int GROUP, int CH, int STAGES>
void launch_group(const ztcp_append& A, int32_t* status, int sms, cudaStream_t s) {
  if (A.dtype == ZTCP_DTYPE_BF16)
    A.interleaved ? launch_one<true, true, GROUP, CH, STAGES>(A, status, sms, s) : launch_one<true, false, GROUP, CH, STAGES>(A, status, sms, s);
  else
    A.interleaved ? launch_one<false, true, GROUP, CH, STAGES>(A, status, sms, s) : launch_one<false, false, GROUP, CH, STAGES>(A, status, sms, s);
}

}  // namespace

void launch_append(const ztcp_append& A, int32_t* status, cudaStream_t s) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return;
  const int64_t D = A.geom.head_dim;
  if (D <= 64) launch_group<8, 1, 8>(A, status, sms, s);
  else if (D <= 128) launch_group<16, 1, 8>(A, status, sms, s);
  else if (D <= 256) launch_group<32, 1, 8>(A, status, sms, s);
  else if (D <= 768) launch_group<32, 3, 5>(A, status, sms, s);
  else launch_group<32, 4, 4>(A, status, sms, s);
}

}  // namespace ztcp
