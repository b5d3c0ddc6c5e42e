// Attention over pages and over packed prompts: requests of different lengths in one call.
// Entry points and the choice of kernel.
#include <algorithm>
#include <cmath>

#include "attn_core.h"

#pragma clang fp contract(off)

namespace efh {
namespace {

// One wave per (row, query head).
constexpr int kRowWaves = 4;

template <class T, bool PAGED>
__global__ __launch_bounds__(kRowWaves * kWave) void attention_rows_kernel(RowsArgs a) {
  __shared__ float qs[kRowWaves][256];
  const int row = blockIdx.x, wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int h = blockIdx.y * kRowWaves + wave;
  const int total = min(a.row_start[a.n_seqs], a.max_rows);
  if (row >= total || h >= a.H) return;
  const int r = request_of(a.row_start, a.n_seqs, row), first = a.row_start[r], g = h / (a.H / a.KV);
  int seen;
  long base;
  if constexpr (PAGED) {
    seen = a.kv_len[r] - (a.row_start[r + 1] - row) + 1;
    seen = static_cast<int>(min(static_cast<long>(seen), a.kv.table_ld << a.kv.page_shift));
    base = r * a.kv.table_ld;
  } else {
    seen = row - first + 1;
    base = first;
  }
  for (int d = lane; d < a.hd; d += kWave) qs[wave][d] = a.q[row * a.ldq + static_cast<long>(h) * a.hd + d];
  float sub = -INFINITY, o[4] = {0, 0, 0, 0};
  double l = 0.0;
  wave_attend<T, PAGED>(a.kv, g, a.hd, base, qs[wave], a.c2, 0, seen, &sub, &l, o);
  l = wave_sum_d_dpp(l);
  const float inv = l == 0.0 ? 0.0f : static_cast<float>(1.0 / l);
  float* out = a.out + row * a.ldo + static_cast<long>(h) * a.hd;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + 64 * u < a.hd) out[lane + 64 * u] = o[u] * inv;
}

int check_rows(const RowsArgs& a, size_t heads, size_t KV, size_t n_seqs, size_t max_rows, size_t ldq, size_t ldo,
               float scale, const std::string& w) {
  EFH_CHECK(a.q && a.out && a.row_start, w + "null pointer");
  EFH_CHECK(heads >= 1 && heads <= 65535 && KV >= 1 && heads % KV == 0, w + "heads must be a multiple of the KV heads");
  EFH_CHECK(n_seqs >= 1 && n_seqs <= (size_t(1) << 20), w + "n_seqs must be in [1, 2^20]");
  EFH_CHECK(max_rows <= (size_t(1) << 30), w + "max_rows too large");
  const size_t nq = heads * static_cast<size_t>(a.hd);
  EFH_CHECK(max_rows <= 1 || (ldq >= nq && ldo >= nq), w + "a row stride is shorter than its row");
  EFH_CHECK(ldq % 4 == 0 && ldo % 4 == 0 && aligned16(a.q) && aligned16(a.out),
            w + "strides and addresses must be multiples of 16 bytes");
  EFH_CHECK(scale > 0.0f && std::isfinite(scale), w + "scale must be positive and finite");
  return EF_HIP_OK;
}

template <bool PAGED>
int launch_rows(const RowsArgs& a, int qtype, hipStream_t s) {
  const dim3 grid(a.max_rows, (a.H + kRowWaves - 1) / kRowWaves);
  const int threads = kRowWaves * kWave;
  if (qtype == EF_QTYPE_F32) attention_rows_kernel<float, PAGED><<<grid, threads, 0, s>>>(a);
  else if (qtype == EF_QTYPE_F16) attention_rows_kernel<_Float16, PAGED><<<grid, threads, 0, s>>>(a);
  else attention_rows_kernel<__bf16, PAGED><<<grid, threads, 0, s>>>(a);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

// How a call of paged attention runs.
struct PagedPlan {
  bool few = false;
  int tiles = 1, splits = 1, span = 128;
  size_t bytes = 0;  // workspace
};
constexpr int kFewPairs = 16, kSpanStep = 128, kSpanLeast = 256, kSpanMost = 4096, kSplitWorkgroups = 1024;

PagedPlan plan_paged(size_t H, size_t KV, size_t hd, size_t n_seqs, size_t max_rows, size_t max_new, size_t max_kv) {
  PagedPlan p;
  const size_t pairs = std::max<size_t>(max_new, 1) * (H / KV);
  p.few = pairs <= 64;
  if (!p.few) return p;
  p.tiles = static_cast<int>((pairs + kFewPairs - 1) / kFewPairs);
  const size_t wgs = n_seqs * KV * p.tiles, want = (kSplitWorkgroups + wgs - 1) / wgs;
  const size_t longest = std::max<size_t>(max_kv, 1);
  size_t span = std::min<size_t>(std::max<size_t>((longest + want - 1) / want, kSpanLeast), kSpanMost);
  span = std::max(span, (longest + 1023) / 1024);
  span = (span + kSpanStep - 1) / kSpanStep * kSpanStep;
  p.span = static_cast<int>(span);
  p.splits = static_cast<int>((longest + span - 1) / span);
  if (p.splits > 1) p.bytes = max_rows * H * p.splits * (hd + 2) * sizeof(float);
  return p;
}

}  // namespace
}  // namespace efh

using namespace efh;

extern "C" {

size_t ef_hip_paged_attention_workspace_bytes(size_t heads, const ef_hip_page_pool* pool, size_t n_seqs, size_t max_rows,
                                              size_t max_new, size_t max_kv) {
  if (check_page_pool(pool, "paged_attention") != EF_HIP_OK || heads < 1 || heads > 65535 || heads % pool->KV != 0 ||
      n_seqs < 1 || max_rows > (size_t(1) << 30) || max_kv > 0x7FFFFFFF)
    return 0;
  return plan_paged(heads, pool->KV, pool->hd, n_seqs, max_rows, max_new, max_kv).bytes;
}

int ef_hip_paged_attention(const float* q, size_t ldq, float* out, size_t ldo, size_t heads, const ef_hip_page_pool* pool,
                           const ef_hip_paged_batch* batch, float scale, void* ws, size_t ws_bytes, void* stream) {
  EFH_RC(check_page_pool(pool, "paged_attention"));
  EFH_CHECK(batch != nullptr, "paged_attention: null batch");
  const ef_hip_paged_batch& b = *batch;
  EFH_CHECK(b.kv_len_dev && b.table_dev, "paged_attention: null pointer");
  EFH_CHECK(b.table_ld >= 1 && b.table_ld <= size_t(0x7FFFFFFF) / pool->page_size,
            "paged_attention: table_ld must be at least 1, with a request's positions below 2^31");
  RowsArgs a{};
  a.q = q;
  a.out = out;
  a.ldq = static_cast<long>(ldq);
  a.ldo = static_cast<long>(ldo);
  a.H = static_cast<int>(heads);
  a.KV = static_cast<int>(pool->KV);
  a.hd = static_cast<int>(pool->hd);
  a.row_start = b.row_start_dev;
  a.kv_len = b.kv_len_dev;
  a.n_seqs = static_cast<int>(b.n_seqs);
  a.max_rows = static_cast<int>(b.max_rows);
  EFH_RC(check_rows(a, heads, pool->KV, b.n_seqs, b.max_rows, ldq, ldo, scale, "paged_attention: "));
  a.c2 = scale * 1.44269504088896340736f;
  a.kv = KvSource{pool->k_dev, pool->v_dev, 0, 0, b.table_dev, static_cast<long>(b.table_ld),
                  static_cast<long>(pool_stride(*pool)), log2_of(pool->page_size), static_cast<int>(pool->n_pages)};
  EFH_CHECK(b.max_kv <= 0x7FFFFFFF, "paged_attention: max_kv too large");
  const PagedPlan p = plan_paged(heads, pool->KV, pool->hd, b.n_seqs, b.max_rows, b.max_new, b.max_kv);
  EFH_CHECK(p.bytes == 0 || (ws != nullptr && ws_bytes >= p.bytes && aligned16(ws)),
            "paged_attention: the workspace must have ef_hip_paged_attention_workspace_bytes bytes, at a multiple of 16");
  EFH_CHECK(b.n_seqs * pool->KV <= size_t(0x7FFFFFFF) / p.tiles, "paged_attention: too many requests and heads");
  EFH_RC(require_ready());
  if (b.max_rows == 0) return EF_HIP_OK;
  if (!p.few) return launch_rows<true>(a, pool->qtype, pick(stream));
  AttnTask t{};
  t.r = a;
  t.tiles = p.tiles;
  t.few_most = 0x7FFFFFFF;
  t.s.splits = p.splits;
  t.s.span = p.span;
  t.s.part = static_cast<float*>(ws);
  t.s.stat = reinterpret_cast<f2v*>(t.s.part + b.max_rows * heads * p.splits * pool->hd);
  return launch_attention_few(t, pool->qtype, pick(stream));
}

size_t ef_hip_packed_attention_workspace_bytes(size_t heads, size_t KV, size_t hd, int qtype, size_t n_seqs,
                                               size_t max_rows) {
  (void)heads, (void)KV, (void)hd, (void)qtype, (void)n_seqs, (void)max_rows;
  return 0;
}

int ef_hip_packed_attention(const float* q, size_t ldq, const void* k, size_t ldk, const void* v, size_t ldv, int qtype,
                            float* out, size_t ldo, size_t heads, size_t KV, size_t hd, const int32_t* row_start,
                            size_t n_seqs, size_t max_rows, float scale, void* ws, size_t ws_bytes, void* stream) {
  EFH_CHECK(k && v, "packed_attention: null pointer");
  EFH_CHECK(qtype == EF_QTYPE_F32 || qtype == EF_QTYPE_F16 || qtype == EF_QTYPE_BF16,
            "packed_attention: keys and values are F32, F16 or BF16");
  EFH_CHECK(hd >= 8 && hd <= 256 && hd % 8 == 0, "packed_attention: hd must be a multiple of 8 up to 256");
  RowsArgs a{};
  a.q = q;
  a.out = out;
  a.ldq = static_cast<long>(ldq);
  a.ldo = static_cast<long>(ldo);
  a.H = static_cast<int>(heads);
  a.KV = static_cast<int>(KV);
  a.hd = static_cast<int>(hd);
  a.row_start = row_start;
  a.n_seqs = static_cast<int>(n_seqs);
  a.max_rows = static_cast<int>(max_rows);
  EFH_RC(check_rows(a, heads, KV, n_seqs, max_rows, ldq, ldo, scale, "packed_attention: "));
  const size_t per16 = qtype == EF_QTYPE_F32 ? 4 : 8;
  EFH_CHECK(max_rows <= 1 || (ldk >= KV * hd && ldv >= KV * hd), "packed_attention: a row stride is shorter than its row");
  EFH_CHECK(ldk % per16 == 0 && ldv % per16 == 0 && aligned16(k) && aligned16(v),
            "packed_attention: strides and addresses must be multiples of 16 bytes");
  a.c2 = scale * 1.44269504088896340736f;
  a.kv = KvSource{k, v, static_cast<long>(ldk), static_cast<long>(ldv), nullptr, 0, 0, 0, 0};
  (void)ws, (void)ws_bytes;
  EFH_RC(require_ready());
  if (max_rows == 0) return EF_HIP_OK;
  return launch_rows<false>(a, qtype, pick(stream));
}

}  // extern "C"
