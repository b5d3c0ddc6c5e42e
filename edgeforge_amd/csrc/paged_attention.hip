// Attention over pages and over packed prompts: requests of different lengths in one call.
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c2 s_j - sub),  s_j = q . k_j,  c2 = scale log2(e),
// sub the rounded c2 max_j s_j so far (a rescaling is by the difference of two sub, so that it is consistent
// with the terms already summed however large the scores' common part is).
#include <algorithm>
#include <cmath>

#include "paging.h"

#pragma clang fp contract(off)

namespace efh {
namespace {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));

struct RowsArgs {
  const float* q;
  float* out;
  long ldq, ldo;
  int H, KV, hd;
  const int32_t *row_start, *kv_len;  // kv_len null: packed
  int n_seqs, max_rows;
  float c2;
  KvSource kv;
};

// 8 values from a 16-byte boundary (32 bytes in FP32) as FP32.
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f4v a = *reinterpret_cast<const f4v*>(p), b = *reinterpret_cast<const f4v*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else if constexpr (std::is_same_v<T, _Float16>) {
    const h8v a = *reinterpret_cast<const h8v*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
  } else {
    const b8v a = *reinterpret_cast<const b8v*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(a[i]);
  }
}

// What the positions [j0, j1) give one (row, head) pair, by a whole wave: a lane takes every 64th position's
// score and dims lane + 64 u of the output.  q is in LDS.  The sums join (sub, l, o); only seen positions are
// read, so infinities and NaN elsewhere do not matter.
template <class T, bool PAGED>
__device__ void wave_attend(const KvSource& src, int g, int hd, long base, const float* q, float c2, int j0, int j1,
                            float* sub, double* l, float (&o)[4]) {
  const int lane = threadIdx.x & (kWave - 1);
  const T *kp = static_cast<const T*>(src.k), *vp = static_cast<const T*>(src.v);
  for (int c = j0; c < j1; c += kWave) {
    const int j = c + lane;
    long ko = 0, vo = 0;
    const bool seen = j < j1 && kv_offset<PAGED>(src, g, hd, base, j, &ko, &vo);
    float s = -INFINITY;
    if (seen) {
      float part[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      for (int d = 0; d < hd; d += 8) {
        float x[8];
        load8(kp + ko + d, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) part[i] = fmaf(x[i], q[d + i], part[i]);
      }
      s = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
    }
    const float top = wave_max_dpp(s) * c2;
    float al = 1.0f;
    if (top > *sub) {
      al = *sub == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(*sub - top);
      *l *= static_cast<double>(al);
      *sub = top;
    }
    const float from = *sub == -INFINITY ? 0.0f : *sub;
    const float p = seen ? __builtin_amdgcn_exp2f(fmaf(s, c2, -from)) : 0.0f;
    *l += static_cast<double>(p);
    float oc[4] = {0, 0, 0, 0};  // the chunk's own sum: no chain of additions is longer than 64 or the chunks
    for (uint64_t todo = __ballot(seen); todo; todo &= todo - 1) {
      const int at = __ffsll(static_cast<unsigned long long>(todo)) - 1;
      const float pj = __shfl(p, at, kWave);
      const long off = __shfl(vo, at, kWave);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (lane + 64 * u < hd) oc[u] = fmaf(pj, static_cast<float>(vp[off + lane + 64 * u]), oc[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) o[u] = fmaf(o[u], al, oc[u]);
  }
}

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

}  // namespace
}  // namespace efh

using namespace efh;

extern "C" {

size_t ef_hip_paged_attention_workspace_bytes(size_t heads, const ef_hip_page_pool* pool, size_t n_seqs, size_t max_rows,
                                              size_t max_new, size_t max_kv) {
  (void)heads, (void)pool, (void)n_seqs, (void)max_rows, (void)max_new, (void)max_kv;
  return 0;
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
  (void)ws, (void)ws_bytes;
  EFH_RC(require_ready());
  if (b.max_rows == 0) return EF_HIP_OK;
  return launch_rows<true>(a, pool->qtype, pick(stream));
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
