// ztcp_kvcache_capi.cu -- host layer of include/ztcp_kvcache.h: validates arguments and launches the kernels on the
// caller's stream.  Nothing here allocates memory or synchronizes.
#include <math.h>
#include <string.h>

#include <atomic>

#include "../../include/ztcp_kvcache.h"
#include "../../include/ztcp_measure.h"
#include "ztcp_kvcache.cuh"

namespace ztcp {
void launch_append(const ztcp_append& A, int32_t* status, cudaStream_t s);
void launch_select(const ztcp_cold_selection& S, cudaStream_t s);
}  // namespace ztcp

namespace {

using ztcp::set_last_error;

int32_t invalid(const char* msg) { return set_last_error(ZTCP_EINVAL, msg); }
bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
constexpr int64_t kInt32Max = 0x7fffffff;
std::atomic<int64_t> g_wait_cycles{ztcp::kWaitCycles};

int32_t check_pool(const ztcp_geometry& g, int32_t dtype, int64_t pool_pages, const void* k, const void* v) {
  if (!k) return invalid("k_pool must not be NULL");
  if (!aligned(k, 16) || !aligned(v, 16)) return invalid("k_pool / v_pool must be 16-byte aligned");
  if (dtype != ZTCP_DTYPE_F16 && dtype != ZTCP_DTYPE_BF16) return invalid("k_pool must be float16 or bfloat16");
  if (!(g.num_tokens > 0 && g.num_heads > 0 && g.head_dim >= 16 && g.head_dim % 16 == 0))
    return invalid("Invalid k_pool dimensions");
  if (!(g.rope_dim >= 0 && g.rope_dim <= g.head_dim && g.rope_dim % 16 == 0)) return invalid("Invalid rope_dim");
  if (pool_pages <= 0 || pool_pages > kInt32Max || g.num_tokens > (1 << 20) || g.num_heads > (1 << 14))
    return invalid("KV pool geometry too large or empty");
  return ZTCP_OK;
}

// A row of 16-bit vectors read 16 bytes at a time.
bool bad_rows(const void* p, int64_t token_stride, int64_t head_stride) {
  return !aligned(p, 16) || token_stride % 8 != 0 || head_stride % 8 != 0;
}

int32_t to_params(const ztcp_kv_cache* k, const ztcp_queries* q, ztcp::CacheParams* c) {
  if (!k || !q) return invalid("cache and queries must not be NULL");
  int32_t rc = check_pool(k->geom, k->dtype, k->pool_pages, k->k_pool, k->v_pool);
  if (rc != ZTCP_OK) return rc;
  const ztcp_geometry& g = k->geom;
  if (g.head_dim > 576) return invalid("head_dim beyond 576");
  if (k->n_seqs <= 0) return invalid("batch must hold at least one sequence");
  // A CTA passes over all sequences to find its place on the line of items, and one by one over sequences without rows,
  // while its other warps wait: 180 ms for 2^20 sequences, of which all but two are empty, and the waits' bound is a second.
  if (k->n_seqs > (1 << 21)) return invalid("more than 2^21 sequences in a batch");
  if (!k->block_tables || !k->kv_lens) return invalid("block_tables and kv_lens must not be NULL");
  if (k->max_pages <= 0 || k->max_pages > k->table_stride || k->max_pages > (1 << 28))
    return invalid("max_pages must be positive and at most the block tables' row length");
  if (!q->q) return invalid("q must not be NULL");
  if (bad_rows(q->q, q->token_stride, q->head_stride))
    return invalid("q must be 16-byte aligned with strides of multiples of 8 elements");
  if (q->total_rows <= 0 || q->total_rows > kInt32Max / 2) return invalid("queries must hold at least one row");
  if (!q->q_starts && q->total_rows != k->n_seqs) return invalid("without q_starts there is one row per sequence");
  if (q->num_heads <= 0 || q->num_heads % g.num_heads != 0 || q->num_heads > (1 << 14))
    return invalid("query heads must be a multiple of the KV heads");
  if (q->total_rows * (q->num_heads / g.num_heads) > kInt32Max)
    return invalid("too many query rows in one call");
  if (q->max_q_len <= 0) return invalid("max_q_len must be positive");
  if (q->max_q_len > kInt32Max) return invalid("max_q_len must be below 2^31");
  if (!(q->scale > 0.f) || isinf(q->scale)) return invalid("scale must be positive and finite");
  memset(c, 0, sizeof(*c));
  c->k = static_cast<const uint16_t*>(k->k_pool);
  c->v = static_cast<const uint16_t*>(k->v_pool);
  c->q = static_cast<const uint16_t*>(q->q);
  c->q_token_stride = q->token_stride;
  c->q_head_stride = q->head_stride;
  c->table = k->block_tables;
  c->table_stride = k->table_stride;
  c->kv_lens = k->kv_lens;
  c->q_starts = q->q_starts;
  c->pool_pages = k->pool_pages;
  c->total_rows = q->total_rows;
  c->n_seqs = (int32_t)k->n_seqs;
  c->max_pages = (int32_t)k->max_pages;
  c->page_tokens = (int32_t)g.num_tokens;
  c->page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (g.num_tokens == (int64_t)1 << i) c->page_shift = i;
  c->kv_heads = (int32_t)g.num_heads;
  c->group = (int32_t)(q->num_heads / g.num_heads);
  c->head_dim = (int32_t)g.head_dim;
  c->v_col = k->v_pool ? 0 : (int32_t)g.rope_dim;
  c->v_dim = c->head_dim - c->v_col;
  c->causal = q->causal != 0;
  c->wait_cycles = g_wait_cycles.load(std::memory_order_relaxed);
  c->scale = q->scale;
  c->scale_log2 = (float)(q->scale * 1.4426950408889634);
  if (isinf(c->scale_log2)) return invalid("scale must be positive and finite, times log2(e) too");
  return ZTCP_OK;
}

// The value columns that an attention output has.
int32_t check_values(const ztcp::CacheParams& c) {
  if (c.v_dim == 0) return invalid("a single-buffer pool needs rope_dim < head_dim");
  if (c.v ? c.head_dim > 256 : c.v_dim > 512)
    return invalid("head_dim beyond 256 (single-buffer pools: 576, with 512 value columns)");
  return ZTCP_OK;
}

int32_t launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_last_error(ZTCP_ECUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return ZTCP_OK;
}

int sm_count() {  // of the current device; 0 without one
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return sms;
}

// The kernel of a call.  Items of few rows (one token or a few, times a group) leave the tensor cores idle whatever is
// done, so the decode kernel turns the products over and reads K and V at memory speed; more rows take the chunk
// kernel's 256-row items.  What their loads cannot take (odd page sizes, other head dims) goes to the general kernel.
// 48 sequences of 1,024 to 8,192 tokens, 8 KV heads of 128, decode against chunk kernel, by rows per KV head: 4 rows 156
// against 174 us, 16 rows 170 against 177, 32 rows 312 against 180 (and so on, a reading of K and V per 16 rows).
enum class Kernel { general, chunk, decode };

Kernel pick_kernel(const ztcp::CacheParams& c, const ztcp_queries* q) {
  const int64_t rows = c.group * q->max_q_len;
  if (ztcp::attend_decode_fits(c) && (rows <= 16 || !ztcp::attend_tc_fits(c))) return Kernel::decode;
  return rows > 16 && ztcp::attend_tc_fits(c) ? Kernel::chunk : Kernel::general;
}

// Fills the workspace-dependent part of P for a workspace at `base`; returns the bytes it takes, 0 without a device.
int64_t plan(Kernel k, const ztcp::CacheParams& c, const ztcp_queries* q, void* base, ztcp::AttendParams* P) {
  const int sms = sm_count();
  if (sms <= 0) return 0;
  const ztcp::AttendShape s = k == Kernel::chunk    ? ztcp::attend_tc_shape(c, sms)
                              : k == Kernel::decode ? ztcp::attend_decode_shape(c, sms, c.group * q->max_q_len)
                                                    : ztcp::attend_shape(c, sms);
  P->c = c;
  P->grid = s.grid;
  P->part_rows = s.part_rows;
  P->part_floats = s.part_floats;
  P->tiled = s.tiled;
  P->cuts = static_cast<ztcp::Cut*>(base);
  P->part = reinterpret_cast<float*>(P->cuts + s.grid);
  return s.grid * ((int64_t)sizeof(ztcp::Cut) + 2 * (int64_t)s.part_floats * (int64_t)sizeof(float));
}

}  // namespace

extern "C" {

int64_t ztcp_wait_limit(int64_t cycles) {
  return g_wait_cycles.exchange(cycles > 0 ? cycles : ztcp::kWaitCycles, std::memory_order_relaxed);
}

int64_t ztcp_attend_workspace_bytes(const ztcp_kv_cache* cache, const ztcp_queries* queries) {
  ztcp::CacheParams c;
  ztcp::AttendParams P;
  if (to_params(cache, queries, &c) != ZTCP_OK || check_values(c) != ZTCP_OK) return -1;
  const int64_t n = plan(pick_kernel(c, queries), c, queries, nullptr, &P);
  if (n <= 0) {
    launched("ztcp_attend_workspace_bytes");
    return -1;
  }
  return n;
}

int32_t ztcp_attend_pages(const ztcp_kv_cache* cache, const ztcp_queries* queries, void* out, float* lse,
                          int32_t* status, void* workspace, int64_t workspace_bytes_given, void* stream) {
  ztcp::CacheParams c;
  ztcp::AttendParams P;
  int32_t rc = to_params(cache, queries, &c);
  if (rc != ZTCP_OK || (rc = check_values(c)) != ZTCP_OK) return rc;
  if (!out || !status || !workspace) return invalid("out, status and workspace must not be NULL");
  if (!aligned(out, 16) || !aligned(workspace, 16)) return invalid("out and workspace must be 16-byte aligned");
  const Kernel kernel = pick_kernel(c, queries);
  const int64_t need = plan(kernel, c, queries, workspace, &P);
  if (need <= 0) return launched("ztcp_attend_pages") != ZTCP_OK ? ZTCP_ECUDA : set_last_error(ZTCP_ECUDA, "no CUDA device");
  if (workspace_bytes_given < need) return invalid("workspace smaller than ztcp_attend_workspace_bytes");
  P.c.status = status;
  P.out = static_cast<uint16_t*>(out);
  P.lse = lse;
  const bool bf16 = cache->dtype == ZTCP_DTYPE_BF16;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  bool made = true;
  if (kernel == Kernel::general) ztcp::launch_attend(P, bf16, s);
  else made = kernel == Kernel::chunk ? ztcp::launch_attend_tc(P, bf16, s) : ztcp::launch_attend_decode(P, bf16, s);
  if (!made) return set_last_error(ZTCP_ECUDA, "cuTensorMapEncodeTiled failed");
  if ((rc = launched("attend_kernel")) != ZTCP_OK) return rc;
  ztcp::launch_attend_merge(P, bf16, c.group * queries->max_q_len, s);
  return launched("attend_merge_kernel");
}

int64_t ztcp_page_mass_workspace_bytes(const ztcp_kv_cache* cache, const ztcp_queries* queries) {
  ztcp::CacheParams c;
  if (to_params(cache, queries, &c) != ZTCP_OK) return -1;
  const int sms = sm_count();
  if (sms <= 0) {
    launched("ztcp_page_mass_workspace_bytes");
    return -1;
  }
  return ztcp::page_mass_tc_fits(c) ? ztcp::page_mass_tc_workspace(c, c.group * queries->max_q_len, sms) : 16;
}

int32_t ztcp_page_mass(const ztcp_kv_cache* cache, const ztcp_queries* queries, const float* lse, const float* mass,
                       float decay, float* out_mass, int32_t* status, void* workspace, int64_t workspace_bytes,
                       void* stream) {
  ztcp::MassParams P = {};
  const int32_t rc = to_params(cache, queries, &P.c);
  if (rc != ZTCP_OK) return rc;
  if (!lse || !out_mass || !status || !workspace) return invalid("lse, out_mass, status and workspace must not be NULL");
  if (!aligned(workspace, 16)) return invalid("workspace must be 16-byte aligned");
  if (!isfinite(decay)) return invalid("decay must be finite");
  const int sms = sm_count();
  if (sms <= 0) return launched("ztcp_page_mass") != ZTCP_OK ? ZTCP_ECUDA : set_last_error(ZTCP_ECUDA, "no CUDA device");
  const bool tc = ztcp::page_mass_tc_fits(P.c);
  if (workspace_bytes < (tc ? ztcp::page_mass_tc_workspace(P.c, P.c.group * queries->max_q_len, sms) : 16)) return invalid("workspace smaller than ztcp_page_mass_workspace_bytes");
  P.c.status = status;
  P.lse = lse;
  P.mass = mass;
  P.decay = decay;
  P.out = out_mass;
  const bool bf16 = cache->dtype == ZTCP_DTYPE_BF16;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!tc) {
    P.unit_pages = P.c.page_tokens >= 64 ? 1 : 64 / P.c.page_tokens;
    ztcp::launch_page_mass(P, bf16, s);
  } else if (!ztcp::launch_page_mass_tc(P, P.c.group * queries->max_q_len, sms, workspace, bf16, s)) {
    return set_last_error(ZTCP_ECUDA, "cuTensorMapEncodeTiled failed");
  }
  return launched("page_mass_kernel");
}

int32_t ztcp_append_tokens(const ztcp_append* a, int32_t* status, void* stream) {
  if (!a || !status) return invalid("append arguments and status must not be NULL");
  const ztcp_geometry& g = a->geom;
  int32_t rc = check_pool(g, a->dtype, a->pool_pages, a->k_pool, a->v_pool);
  if (rc != ZTCP_OK) return rc;
  if (g.head_dim > 1024) return invalid("head_dim beyond 1024");
  if (g.rope_dim > 256) return invalid("rope_dim beyond 256");
  if (!a->k) return invalid("k must not be NULL");
  if ((a->v == nullptr) != (a->v_pool == nullptr)) return invalid("v must be given exactly when v_pool is");
  if (a->q && (!a->q_out || a->num_q_heads <= 0 || a->num_q_heads > (1 << 14)))
    return invalid("q needs q_out and a positive number of heads");
  if ((a->q && bad_rows(a->q, a->q_token_stride, a->q_head_stride)) || bad_rows(a->k, a->k_token_stride, a->k_head_stride) ||
      (a->v && bad_rows(a->v, a->v_token_stride, a->v_head_stride)) || (a->q && !aligned(a->q_out, 16)))
    return invalid("q, k, v and q_out must be 16-byte aligned with strides of multiples of 8 elements");
  for (int64_t st : {a->q_head_stride, a->k_head_stride, a->v_head_stride})
    if (st > kInt32Max || st < 0) return invalid("head strides must be non-negative and below 2^31 elements");
  if (!a->slots) return invalid("slots must not be NULL");
  if (g.rope_dim > 0 && (!a->positions || !a->rope_table || a->max_pos <= 0))
    return invalid("a rotation needs positions and a rope table");
  if (!aligned(a->rope_table, 16) || !aligned(a->q_weight, 16) || !aligned(a->k_weight, 16))
    return invalid("rope_table, q_weight and k_weight must be 16-byte aligned");
  if (a->norm_from < 0 || a->norm_from >= g.head_dim || a->norm_from % 16 != 0)
    return invalid("norm_from must be a multiple of 16 below head_dim");
  if (!(a->eps >= 0.f) || isinf(a->eps)) return invalid("eps must be non-negative and finite");
  if (a->n_tokens <= 0 || a->n_tokens > kInt32Max) return invalid("append must hold at least one token");
  ztcp::launch_append(*a, status, static_cast<cudaStream_t>(stream));
  return launched("append_kernel");
}

int32_t ztcp_select_cold_pages(const ztcp_cold_selection* s, void* stream) {
  if (!s) return invalid("selection must not be NULL");
  if (!s->mass || !s->block_tables || !s->kv_lens) return invalid("mass, block_tables and kv_lens must not be NULL");
  if (!s->cold_blocks || !s->cold_index || !s->cold_starts || !s->kept_tables || !s->kept_mass || !s->kept_lens || !s->status)
    return invalid("selection outputs must not be NULL");
  if (s->n_seqs <= 0 || s->max_pages <= 0 || s->page_tokens <= 0 || s->page_tokens > (1 << 20) || s->n_seqs > kInt32Max ||
      s->max_pages > kInt32Max || s->n_seqs * s->max_pages > kInt32Max)
    return invalid("selection must hold at least one sequence and page, and fewer than 2^31 pages in all");
  // (a CTA's steps through a row end on a multiple of 4,096 pages, which has to fit 32 bits)
  if (s->max_pages > kInt32Max - 4095) return invalid("max_pages beyond 2^31 - 4096");
  if (s->keep < 0 || s->sink < 0 || s->recent < 1) return invalid("keep and sink must be non-negative and recent positive");
  if (s->keep > kInt32Max || s->sink > kInt32Max || s->recent > kInt32Max) return invalid("keep, sink or recent too large");
  ztcp::launch_select(*s, static_cast<cudaStream_t>(stream));
  return launched("select_kernel");
}

}  // extern "C"
