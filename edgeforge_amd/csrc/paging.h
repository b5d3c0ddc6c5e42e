// Pages of the KV cache: what the plan, the append and the attention kernels share (ef_hip_page_pool).
#pragma once

#include <vector>

#include "common.h"

namespace efh {

// cos / sin [n_pos][hd / 2] exactly as kern::RopeTable builds them (src/kernels.cpp:113-131): float pow /
// cos / sin from the host C library, so the device sees the reference's bits.
void rope_tables_host(float theta, size_t hd, size_t n_pos, std::vector<float>* cos_t, std::vector<float>* sin_t);

// The pool's sizes and addresses, checked (EF_HIP_EINVAL with `who` in the message).
int check_page_pool(const ef_hip_page_pool* pool, const char* who);
inline size_t pool_stride(const ef_hip_page_pool& p) { return p.page_stride ? p.page_stride : p.KV * p.page_size * p.hd; }
inline int log2_of(size_t pow2) { return __builtin_ctzll(pow2); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workgroups of 256 threads that one launch takes along x: HIP counts the threads in 32 bits.
constexpr size_t kGridMost = (size_t(1) << 24) - 1;

// The request of row i: the last r with start[r] <= i, for start[0] <= i < start[n] (requests without rows are
// passed over, as the next one starts at the same row).
template <class P>
__host__ __device__ __forceinline__ int request_of(P start, int n, int i) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The last lane of a ballot whose lanes are set from the first one on; 0 where none is.  (Not max(__popcll(lanes) - 1, 0): of an
// unsigned and a signed value that is a double's maximum, 2^32 - 1 for no lane.)
__host__ __device__ __forceinline__ int last_lane(uint64_t lanes) { return lanes ? 63 - __builtin_clzll(lanes) : 0; }

// Where keys and values come from: pages (table != nullptr) or packed rows.
struct KvSource {
  const void *k, *v;
  long ldk, ldv;         // packed: values from one row to the next
  const int32_t* table;  // pages
  long table_ld, page_stride;
  int page_shift, n_pages;
};

// The values of position j of KV head g: their offset from the source's start, in values; false where no page
// holds it.  base: the request's row of the block table, or its first packed row.
template <bool PAGED>
__host__ __device__ __forceinline__ bool kv_offset(const KvSource& s, int g, int hd, long base, int j, long* ko, long* vo) {
  if constexpr (PAGED) {
    const int page = s.table[base + (j >> s.page_shift)];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(s.n_pages)) return false;
    *ko = *vo = page * s.page_stride + ((static_cast<long>(g) << s.page_shift) + (j & ((1 << s.page_shift) - 1))) * hd;
  } else {
    *ko = (base + j) * s.ldk + static_cast<long>(g) * hd;
    *vo = (base + j) * s.ldv + static_cast<long>(g) * hd;
  }
  return true;
}

}  // namespace efh
