// Attention over pages and over packed prompts: requests of different lengths in one call.
// Entry points and the choice of kernel.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "attn_core.h"

#pragma clang fp contract(off)

namespace efh {
namespace {

int check_rows(const RowsArgs& a, size_t heads, size_t KV, size_t n_seqs, size_t max_rows, size_t ldq, size_t ldo,
               float scale, const char* who) {
  auto w = [who](const char* what) { return std::string(who) + what; };
  EFH_CHECK(a.q && a.out && a.row_start, w("null pointer"));
  EFH_CHECK(heads >= 1 && heads <= 65535 && KV >= 1 && heads % KV == 0, w("heads must be a multiple of the KV heads"));
  EFH_CHECK(n_seqs >= 1 && n_seqs <= (size_t(1) << 20), w("n_seqs must be in [1, 2^20]"));
  EFH_CHECK(max_rows <= (size_t(1) << 30) / heads, w("too many rows and heads"));
  const size_t nq = heads * static_cast<size_t>(a.hd);
  EFH_CHECK(max_rows <= 1 || (ldq >= nq && ldo >= nq), w("a row stride is shorter than its row"));
  EFH_CHECK(ldq % 4 == 0 && ldo % 4 == 0 && aligned16(a.q) && aligned16(a.out),
            w("strides and addresses must be multiples of 16 bytes"));
  EFH_CHECK(scale > 0.0f && std::isfinite(scale), w("scale must be positive and finite"));
  return EF_HIP_OK;
}

AttnTask task_of(const RowsArgs& a) {
  AttnTask t{};
  t.r = a;
  t.few_split = t.tile_split = Split{1, 0x40000000};
  t.group = a.H / a.KV;
  t.magic = static_cast<uint32_t>(((uint64_t(1) << 32) + t.group - 1) / t.group);
  return t;
}

// How a call of paged attention runs: the few-rows kernel for requests of up to few_most (row, head) pairs of a KV
// head, the tiles kernel for those above, either alone where the bounds leave no request to the other.
struct PagedPlan {
  bool few = false, tiles = false, few_wide = false;
  int few_most = 0, few_tiles = 1;
  Split few_split{1, 0x40000000}, tile_split{1, 0x40000000};
  size_t bytes = 0;  // workspace
};
constexpr int kFewPairs = 16, kFewAlone = 64;
constexpr int kFewStep = 128;
constexpr int kTileStep = 64;

// Ranges of positions: as many as make `wgs` workgroups per range about `want` in all, but none shorter than `least`.
Split split_over(size_t wgs, size_t want, size_t longest, size_t least, size_t step) {
  const size_t ranges = std::max<size_t>(want / wgs, 1);
  size_t span = std::max((longest + ranges - 1) / ranges, least);
  span = std::max(span, (longest + 1023) / 1024);
  span = (span + step - 1) / step * step;
  return Split{static_cast<int>((longest + span - 1) / span), static_cast<int>(span)};
}

// Positions are split so that the workgroups fill the GPU once (as many as its CUs hold at the kernels' registers): one
// more than fits costs a second round.  12 x 32k BF16: 5 ranges (480 workgroups of 512) 215 us, 8 (768) 271, 10 (960)
// 237; 64 requests of 2047 FP16: 3 ranges (768 of 768) 26.8 us, 4 (1024) 32.
// The tiles kernel's shortest range is 256 positions, 128 after at most 1536, where that leaves workgroups idle.  FP16, us with
// 256 / 128: 8 requests of 1000 positions (64 dims) 17.5 / 15.6, 200 rows after 200 (128 dims) 22.5 / 19.7, 32 rows after
// 8000 (128 dims) 34.8 / 44.9, 20 requests of 4000 (64 dims) 31.7 / 34.0.
PagedPlan plan_paged(size_t H, size_t KV, size_t hd, int qtype, size_t n_seqs, size_t max_rows, size_t max_new, size_t max_kv) {
  PagedPlan p;
  const size_t cus = ctx().cu_count > 0 ? ctx().cu_count : 256;
  const size_t G = H / KV, pairs = std::max<size_t>(max_new, 1) * G, longest = std::max<size_t>(max_kv, 1);
  p.few = pairs <= kFewAlone || (n_seqs > 1 && G <= kFewAlone);
  p.tiles = pairs > kFewAlone;
  const size_t few_pairs = p.tiles ? std::max<size_t>(kFewPairs, G) : pairs;
  if (p.few) {
    p.few_most = p.tiles ? static_cast<int>(few_pairs) : 0x7FFFFFFF;
    p.few_wide = !p.tiles && few_pairs > kFewPairs && hd <= 128;
    const size_t per = p.few_wide ? 2 * kFewPairs : kFewPairs;
    p.few_tiles = static_cast<int>((few_pairs + per - 1) / per);
    p.few_split = split_over(n_seqs * KV * p.few_tiles, cus * (hd <= 64 ? 3 : hd <= 128 ? 2 : 1), longest, kFewStep, kFewStep);
  }
  if (p.tiles)
    p.tile_split = split_over(std::max<size_t>((max_rows * G + kTilePairs - 1) / kTilePairs * KV, 1),
                              cus * (hd <= 64 && qtype != EF_QTYPE_F32 ? 3 : hd <= 128 ? 2 : 1), longest, longest <= 1536 ? 128 : 256, kTileStep);
  const size_t splits = std::max(p.few_split.splits, p.tile_split.splits);
  if (splits > 1) p.bytes = max_rows * H * (splits * (hd + 2) + 1) * sizeof(float);
  return p;
}

// Whether packed FP32 and BF16 rows go through the prepared tiles: FP32 rows scaled and split
// once instead of by every workgroup, BF16 two products for three; one more launch and pass.  By the
// work, rows times rows of a prompt on average; us from the rows / prepared, 32 heads over 4 of 64 and over 8 of 128:
//   FP32, 64:   100 rows 11.3 / 13.4, 200 rows 16.1 / 16.0, 333 of 9 prompts 11.6 / 14.2, 500 rows 28.3 / 24.1, 1000 of 8
//               23.3 / 22.8, 2000 of 20 32.1 / 31.7, 2000 rows 96.9 / 76.2
//   FP32, 128:  64 rows 15.0 / 15.3, 100 rows 18.8 / 17.0, 333 of 9 22.3 / 20.3, 500 rows 59.7 / 38.0, 2000 of 20 70.4 / 52.7
//   FP32, 80 (12 heads over 4):  64 rows 10.9 / 13.1, 128 rows 16.0 / 15.7, 256 of 4 17.7 / 16.8
//   FP32, 256 (8 over 4):  32 rows 19.7 / 20.8, 64 rows 29.6 / 27.7, 128 rows 42.9 / 35.4
//   FP32, as many KV heads:  16 of 64, 200 rows 16.5 / 16.8, 500 28.0 / 24.7, 6000 297 / 235;  8 of 128, 200 29.8 / 22.3, 6000 630 / 329
//   BF16, 64:   1000 rows 30.4 / 31.3, 1500 of 3 37.1 / 37.1, 2000 rows 60.1 / 56.6, 6000 of 4 168 / 137, 9000 rows 796 / 615
//   BF16, 128:  1000 rows 46.6 / 54.6, 2000 rows 101 / 101, 3000 rows 187 / 159, 9000 rows 1438 / 1169
//   BF16, as many KV heads:  16 of 64, 1000 rows 29.1 / 31.4, 6000 215 / 176;  8 of 128, 1000 43.6 / 51.9, 6000 250 / 242
// The work alone does not know how many workgroups share a tile, nor how full the GPU is: it takes the slower way for many short prompts (FP32,
// 128, 1000 rows of 50: 24.0 / 31.3) and, up to 20% slower, for middle lengths of as many KV heads (FP32, 16 of 64, 6000 of 30:
// 48.5 / 56.1; BF16, 8 of 128, 3000 rows: 116 / 131) or of several BF16 prompts (64, 9000 of 20: 110 / 96).
// EF_HIP_PACKED_ATTENTION=rows|prepared takes one or the other (tests).
bool prepares(size_t hd, int qtype, size_t n_seqs, size_t max_rows) {
  if (qtype == EF_QTYPE_F16 || max_rows == 0) return false;
  if (const char* e = std::getenv("EF_HIP_PACKED_ATTENTION")) {
    if (std::strcmp(e, "rows") == 0) return false;
    if (std::strcmp(e, "prepared") == 0) return true;
  }
  const double work = static_cast<double>(max_rows) * max_rows / n_seqs;
  return work >= (qtype == EF_QTYPE_BF16 ? 4194304.0 : hd <= 64 ? 131072.0 : hd <= 128 ? 8192.0 : 4096.0);
}

size_t prepared_places(size_t hd, int qtype, size_t n_seqs, size_t max_rows) {
  if (!prepares(hd, qtype, n_seqs, max_rows)) return 0;
  const size_t rows = prepared_shape(hd, qtype).rows;
  return (max_rows + rows - 1) / rows + n_seqs;
}
size_t prepared_bytes(size_t KV, size_t hd, int qtype, size_t n_seqs, size_t max_rows) {
  return prepared_places(hd, qtype, n_seqs, max_rows) * KV * (prepared_shape(hd, qtype).bytes + 8);
}

}  // namespace
}  // namespace efh

using namespace efh;

extern "C" {

size_t ef_hip_paged_attention_workspace_bytes(size_t heads, const ef_hip_page_pool* pool, size_t n_seqs, size_t max_rows,
                                              size_t max_new, size_t max_kv) {
  if (check_page_pool(pool, "paged_attention") != EF_HIP_OK || heads < 1 || heads > 65535 || heads % pool->KV != 0 ||
      n_seqs < 1 || n_seqs > (size_t(1) << 20) || max_rows > (size_t(1) << 30) / heads || max_kv > 0x7FFFFFFF)
    return 0;
  return plan_paged(heads, pool->KV, pool->hd, pool->qtype, n_seqs, max_rows, max_new, max_kv).bytes;
}

int ef_hip_paged_attention(const float* q, size_t ldq, float* out, size_t ldo, size_t heads, const ef_hip_page_pool* pool,
                           const ef_hip_paged_batch* batch, float scale, void* ws, size_t ws_bytes, void* stream) {
  EFH_RC(check_page_pool(pool, "paged_attention"));
  EFH_CHECK(batch != nullptr, "paged_attention: null batch");
  const ef_hip_paged_batch& b = *batch;
  EFH_CHECK(b.kv_len_dev && b.table_dev, "paged_attention: null pointer");
  EFH_CHECK(b.table_ld >= 1 && b.table_ld <= kMostPositions / pool->page_size,
            "paged_attention: table_ld must be at least 1, with at most 2^31 - 1024 positions of a request");
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
  const PagedPlan p = plan_paged(heads, pool->KV, pool->hd, pool->qtype, b.n_seqs, b.max_rows, b.max_new, b.max_kv);
  EFH_CHECK(p.bytes == 0 || (ws != nullptr && ws_bytes >= p.bytes && aligned16(ws)),
            "paged_attention: the workspace must have ef_hip_paged_attention_workspace_bytes bytes, at a multiple of 16");
  EFH_CHECK(static_cast<size_t>(p.few_tiles) * p.few_split.splits <= 65535, "paged_attention: too many heads to a KV head");
  // workgroups of a launch: places of tiles and requests, by KV heads and ranges
  const double tiles = (static_cast<double>(b.max_rows) * heads / pool->KV / kTilePairs + 1 + b.n_seqs) * pool->KV;
  const double few = static_cast<double>(b.n_seqs) * pool->KV * p.few_tiles * p.few_split.splits;
  // (the ranges are along x in the launch of both kernels, along y in the tiles kernel's own)
  EFH_CHECK(!p.tiles || (p.few ? tiles * p.tile_split.splits + few : tiles) <= static_cast<double>(kGridMost),
            "paged_attention: too many requests, rows and heads for one launch");
  const size_t ranges = std::max(p.few_split.splits, p.tile_split.splits);
  EFH_CHECK(ranges <= 1 || b.max_rows * heads <= kGridMost * (ranges > kJoinMany ? 1 : 4),
            "paged_attention: too many rows and heads for one launch");
  EFH_RC(require_ready());
  if (b.max_rows == 0) return EF_HIP_OK;
  AttnTask t = task_of(a);
  t.few_split = p.few_split;
  t.tile_split = p.tile_split;
  t.tiles = p.few_tiles;
  t.few_wide = p.few_wide;
  t.few_most = p.few_most;
  const size_t splits = std::max(p.few_split.splits, p.tile_split.splits);
  t.part = static_cast<float*>(ws);
  t.stat = reinterpret_cast<f2v*>(t.part + b.max_rows * heads * splits * pool->hd);
  t.count = splits > 1 ? reinterpret_cast<int*>(t.stat + b.max_rows * heads * splits) : nullptr;
  hipStream_t s = pick(stream);
  if (p.tiles && p.few) EFH_RC(launch_attention_mixed(t, pool->qtype, s));
  else if (p.tiles) EFH_RC(launch_attention_tiles(t, pool->qtype, true, s));
  else EFH_RC(launch_attention_few(t, pool->qtype, s));
  return splits > 1 ? launch_attention_join(t, s) : EF_HIP_OK;
}

size_t ef_hip_packed_attention_workspace_bytes(size_t heads, size_t KV, size_t hd, int qtype, size_t n_seqs,
                                               size_t max_rows) {
  if (heads < 1 || heads > 65535 || KV < 1 || heads % KV != 0 || hd < 8 || hd > 256 || hd % 8 != 0 || n_seqs < 1 ||
      n_seqs > (size_t(1) << 20) || max_rows > (size_t(1) << 30) / heads ||
      (qtype != EF_QTYPE_F32 && qtype != EF_QTYPE_F16 && qtype != EF_QTYPE_BF16))
    return 0;
  return prepared_bytes(KV, hd, qtype, n_seqs, max_rows);
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
  const size_t need = prepared_bytes(KV, hd, qtype, n_seqs, max_rows);
  EFH_CHECK(need == 0 || (ws != nullptr && ws_bytes >= need && aligned16(ws)),
            "packed_attention: the workspace must have ef_hip_packed_attention_workspace_bytes bytes, at a multiple of 16");
  EFH_CHECK((static_cast<double>(max_rows) * heads / KV / kTilePairs + 1 + n_seqs) * KV <= static_cast<double>(kGridMost),
            "packed_attention: too many prompts, rows and heads for one launch");
  EFH_RC(require_ready());
  if (max_rows == 0) return EF_HIP_OK;
  const AttnTask t = task_of(a);
  if (need) return launch_attention_prepared(t, qtype, ws, prepared_places(hd, qtype, n_seqs, max_rows), pick(stream));
  return launch_attention_tiles(t, qtype, false, pick(stream));
}

}  // extern "C"
