// Paged KV cache: one step's block tables and slot maps from the requests' lengths, and RoPE with the
// store of keys and values into their pages.  No counterpart in the reference (one contiguous cache).
#include <cmath>
#include <new>

#include "paging.h"

#pragma clang fp contract(off)

namespace efh {
namespace {

// ---- the plan -------------------------------------------------------------------------------------
// held = ceil(cached / P), total = cached + new, take = ceil(total / P) - held; an ended request gives its held
// pages back.  Three prefix sums over the requests (rows, pages taken, pages given) place everything: the
// free pages are a stack, gives are pushed in order before takes pop in order, so the result does not
// depend on how threads run.
//
// One workgroup: the sums are over at most a few thousand requests, and the stack orders everything.  Bound by latency, a
// launch and about four loads that wait for each other: 64 requests 5.6 us; 700 requests, 25 of them ended with 100 pages each on average and 70
// with a prompt's chunk, 9.4 us and 4.5 for the 21,924 rows' slots in their own launch.
// The sums saturate (a saturating sum is associative), so lengths of any size are compared with the
// bounds without wrapping.
constexpr int kPlanFew = 256, kPlanThreads = 1024, kPlanWaves = kPlanThreads / kWave;

struct PlanArgs {
  const int32_t *cached, *fresh;
  int n_seqs, page_shift, n_pages;
  int32_t* table;
  long table_ld;
  int32_t* free_list;
  const int32_t* n_free;
  int32_t *n_free_out, *kv_len, *row_start, *pos;
  int64_t* slot;
  int max_rows;
  int32_t* status;
};

struct Three {
  uint32_t rows, take, give;
};
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ Three operator+(Three a, Three b) {
  return {add_sat(a.rows, b.rows), add_sat(a.take, b.take), add_sat(a.give, b.give)};
}

// Exclusive prefix of v over the workgroup's threads, on top of *carry, which becomes the total so far.
// The barrier waits for LDS only: nobody reads another thread's stores behind it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
template <int WAVES = kPlanWaves>
__device__ __forceinline__ Three scan_block(Three v, Three* carry, Three (*part)[WAVES]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  Three in = v;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const Three u = {__shfl_up(in.rows, o, kWave), __shfl_up(in.take, o, kWave), __shfl_up(in.give, o, kWave)};
    if (lane >= o) in = in + u;
  }
  if (lane == kWave - 1) (*part)[wave] = in;
  lds_barrier();
  Three before = *carry, all = *carry;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const Three p = (*part)[w];
    if (w < wave) before = before + p;
    all = all + p;
  }
  lds_barrier();
  *carry = all;
  const Three up = {__shfl_up(in.rows, 1, kWave), __shfl_up(in.take, 1, kWave), __shfl_up(in.give, 1, kWave)};
  return lane == 0 ? before : before + up;
}

// A request's share of the sums, and whether its length is bad.
struct Share {
  Three v;
  int cached, held;
  bool bad;
};
__device__ __forceinline__ Share share_of(const PlanArgs& a, int r) {
  Share s = {{0, 0, 0}, 0, 0, false};
  if (r >= a.n_seqs) return s;
  const int c = a.cached[r], x = a.fresh[r];
  const long total = static_cast<long>(c) + max(x, 0), mask = (1L << a.page_shift) - 1;
  s.cached = c;
  s.bad = c < 0 || total > (a.table_ld << a.page_shift);
  if (s.bad) return s;
  s.held = static_cast<int>((c + mask) >> a.page_shift);
  if (x < 0) return s;
  s.v.rows = x;
  s.v.take = static_cast<uint32_t>(((total + mask) >> a.page_shift) - s.held);
  return s;
}
__device__ __forceinline__ bool real_page(const PlanArgs& a, int page) {
  return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.n_pages);
}
// Whole waves walk the table rows of their ended requests, four pieces of 64 entries in flight: how many pages each
// request gives, each given page put(at + i, page).
template <class F>
__device__ __forceinline__ int ended_pages(const PlanArgs& a, int r, int held, int at, F&& put) {
  constexpr int FLIGHT = 4;
  const int lane = threadIdx.x & (kWave - 1);
  uint64_t todo = __ballot(r < a.n_seqs && held > 0 && a.fresh[r] < 0);
  int count = 0, found = 0, j0 = 0;
  while (todo) {
    int page[FLIGHT], who[FLIGHT];
    bool last[FLIGHT];
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      who[i] = todo ? __ffsll(static_cast<unsigned long long>(todo)) - 1 : -1;
      page[i] = -1;
      last[i] = false;
      if (who[i] < 0) continue;
      const int rr = __builtin_amdgcn_readlane(r, who[i]), hh = __builtin_amdgcn_readlane(held, who[i]);
      if (j0 + lane < hh) page[i] = a.table[rr * a.table_ld + j0 + lane];
      j0 += kWave;
      if (j0 >= hh) {
        last[i] = true;
        todo &= todo - 1;
        j0 = 0;
      }
    }
#pragma unroll
    for (int i = 0; i < FLIGHT; ++i) {
      if (who[i] < 0) continue;
      const uint64_t ok = __ballot(real_page(a, page[i]));
      if (real_page(a, page[i])) put(__builtin_amdgcn_readlane(at, who[i]) + found + __popcll(ok & ((1ull << lane) - 1)), page[i]);
      found += __popcll(ok);
      if (last[i]) {
        if (lane == who[i]) count = found;
        found = 0;
      }
    }
  }
  return count;
}
// Pages taken: each growing request's first by its own thread (a decode step takes one or none), the others by whole
// waves.  get(k): the page k places below the top of the stack.
template <class Get>
__device__ __forceinline__ void take_pages(const PlanArgs& a, int r, int held, uint32_t take, uint32_t before, Get&& get) {
  const int lane = threadIdx.x & (kWave - 1);
  if (take > 0) a.table[r * a.table_ld + held] = get(static_cast<int>(before));
  for (uint64_t todo = __ballot(take > 1); todo; todo &= todo - 1) {
    const int who = __ffsll(static_cast<unsigned long long>(todo)) - 1;
    const int rr = __shfl(r, who, kWave), h = __shfl(held, who, kWave), n = __shfl(static_cast<int>(take), who, kWave);
    const int k0 = __shfl(static_cast<int>(before), who, kWave);
    for (int j = 1 + lane; j < n; j += kWave) a.table[rr * a.table_ld + h + j] = get(k0 + j);
  }
}
// Whether the step fits, and what does not: the same for every thread.
struct Verdict {
  bool fits;
  uint32_t n1;  // free pages after the gifts
};
__device__ __forceinline__ Verdict judge(const PlanArgs& a, Three total, int n_bad, int n0) {
  const uint32_t n1 = add_sat(static_cast<uint32_t>(max(n0, 0)), total.give);
  const bool free_bad = n0 < 0 || n0 > a.n_pages || n1 > static_cast<uint32_t>(a.n_pages);
  const uint32_t missing = free_bad || total.take <= n1 ? 0 : total.take - n1;
  const uint32_t over = total.rows > static_cast<uint32_t>(a.max_rows) ? total.rows - a.max_rows : 0;
  const bool fits = !free_bad && missing == 0 && over == 0 && n_bad == 0;
  if (threadIdx.x == 0) {
    a.status[0] = static_cast<int32_t>(min(missing, 0x7FFFFFFFu));
    a.status[1] = n_bad;
    a.status[2] = static_cast<int32_t>(min(over, 0x7FFFFFFFu));
    a.status[3] = free_bad;
    *a.n_free_out = fits ? static_cast<int32_t>(n1 - total.take) : n0;
    a.row_start[a.n_seqs] = fits ? static_cast<int32_t>(total.rows) : 0;
  }
  return {fits, n1};
}

// More requests than threads: every sum again in each pass over them.
__global__ __launch_bounds__(kPlanThreads) void page_plan_kernel(PlanArgs a) {
  __shared__ Three part[kPlanWaves];
  const int t = threadIdx.x, n0 = *a.n_free;
  auto count_only = [](int, int) {};
  Three total = {0, 0, 0};
  int n_bad = 0;
  for (int r0 = 0; r0 < a.n_seqs; r0 += kPlanThreads) {
    Share s = share_of(a, r0 + t);
    n_bad += __syncthreads_count(s.bad);
    s.v.give = ended_pages(a, r0 + t, s.held, 0, count_only);
    scan_block(s.v, &total, &part);
  }
  const Verdict v = judge(a, total, n_bad, n0);
  if (v.fits && total.give > 0) {
    Three carry = {0, 0, 0};
    for (int r0 = 0; r0 < a.n_seqs; r0 += kPlanThreads) {
      Share s = share_of(a, r0 + t);
      s.v.give = ended_pages(a, r0 + t, s.held, 0, count_only);
      const Three before = scan_block(s.v, &carry, &part);
      ended_pages(a, r0 + t, s.held, n0 + static_cast<int>(before.give), [&](int at, int page) { a.free_list[at] = page; });
    }
    __syncthreads();  // what was given is there to be taken
  }
  Three carry = {0, 0, 0};
  for (int r0 = 0; r0 < a.n_seqs; r0 += kPlanThreads) {
    const int r = r0 + t;
    const Share s = share_of(a, r);
    const int x = r < a.n_seqs ? a.fresh[r] : 0;
    const Three before = scan_block(s.v, &carry, &part);
    if (v.fits)
      take_pages(a, r, s.held, s.v.take, before.take, [&](int k) { return a.free_list[static_cast<int>(v.n1) - 1 - k]; });
    if (r >= a.n_seqs) continue;
    a.row_start[r] = v.fits ? static_cast<int>(before.rows) : 0;
    a.kv_len[r] = !v.fits ? s.cached : x < 0 ? 0 : s.cached + static_cast<int>(s.v.rows);
  }
}

// One request to a thread.  The sums are formed once; given pages, taken pages and the requests' starts are kept in LDS
// too, so that a step waits for memory four times (lengths, ended requests' pages, free pages, the table) and for
// none of its own stores.
constexpr int kPlanKept = 4096;  // given and taken pages kept in LDS; beyond, the stores are waited for

template <int THREADS, bool FILL>
__global__ __launch_bounds__(THREADS) void page_plan_once_kernel(PlanArgs a) {
  __shared__ Three part[THREADS / kWave];
  __shared__ int start_s[THREADS + 1], end_s[THREADS], held_s[THREADS], take_s[THREADS], given_s[kPlanKept], taken_s[kPlanKept];
  __shared__ int bad_s;
  const int t = threadIdx.x, n0 = __builtin_amdgcn_readfirstlane(*a.n_free);
  asm volatile("" ::"s"(n0));  // read before the first barrier: n_free_out may be n_free, and is written behind one
  Share s = share_of(a, t);
  const int x = t < a.n_seqs ? a.fresh[t] : 0;
  if (t == 0) bad_s = 0;
  s.v.give = ended_pages(a, t, s.held, 0, [](int, int) {});
  lds_barrier();
  if (s.bad) atomicAdd(&bad_s, 1);
  Three total = {0, 0, 0};
  const Three before = scan_block<THREADS / kWave>(s.v, &total, &part);
  const Verdict v = judge(a, total, bad_s, n0);
  const bool kept = total.give <= kPlanKept && total.take <= kPlanKept;
  if (v.fits && total.give > 0)
    ended_pages(a, t, s.held, static_cast<int>(before.give), [&](int at, int page) {
      a.free_list[n0 + at] = page;
      if (at < kPlanKept) given_s[at] = page;
    });
  start_s[t] = v.fits ? static_cast<int>(before.rows) : 0;
  end_s[t] = s.cached + static_cast<int>(s.v.rows);
  held_s[t] = s.held;
  take_s[t] = static_cast<int>(before.take) - s.held;
  if (t == 0) start_s[a.n_seqs] = v.fits ? static_cast<int>(total.rows) : 0;
  if (kept) lds_barrier();
  else __syncthreads();
  auto top = [&](int k) {  // the page k places below the top of the stack
    const int at = static_cast<int>(v.n1) - 1 - k;
    return kept && at >= n0 ? given_s[at - n0] : a.free_list[at];
  };
  if (kept) {  // every page at once, then the table from LDS
    if (v.fits)
      for (int k = t; k < static_cast<int>(total.take); k += THREADS) taken_s[k] = top(k);
    lds_barrier();
    if (v.fits) take_pages(a, t, s.held, s.v.take, before.take, [&](int k) { return taken_s[k]; });
  } else if (v.fits) {
    take_pages(a, t, s.held, s.v.take, before.take, top);
  }
  if (t < a.n_seqs) {
    a.row_start[t] = v.fits ? static_cast<int>(before.rows) : 0;
    a.kv_len[t] = !v.fits ? s.cached : x < 0 ? 0 : s.cached + static_cast<int>(s.v.rows);
  }
  if constexpr (FILL) {
    if (!kept) __syncthreads();  // the table's new pages
    const int rows = v.fits ? static_cast<int>(total.rows) : 0;
    for (int i = t; i < a.max_rows; i += THREADS) {
      int p = 0;
      int64_t slot = -1;
      if (i < rows) {
        const int r = request_of(start_s, a.n_seqs, i);
        p = end_s[r] - (start_s[r + 1] - i);
        const int b = p >> a.page_shift;
        const int page = kept && b >= held_s[r] ? taken_s[take_s[r] + b] : a.table[r * a.table_ld + b];
        if (real_page(a, page)) slot = (static_cast<int64_t>(page) << a.page_shift) + (p & ((1 << a.page_shift) - 1));
      }
      a.pos[i] = p;
      a.slot[i] = slot;
    }
  }
}

// Each row's position and slot; rows behind the last one get position 0 and slot -1.
__global__ __launch_bounds__(256) void page_rows_kernel(PlanArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.max_rows) return;
  int p = 0;
  int64_t slot = -1;
  if (i < a.row_start[a.n_seqs]) {
    const int r = request_of(a.row_start, a.n_seqs, i);
    p = a.kv_len[r] - (a.row_start[r + 1] - i);
    const int page = a.table[r * a.table_ld + (p >> a.page_shift)];
    if (real_page(a, page)) slot = (static_cast<int64_t>(page) << a.page_shift) + (p & ((1 << a.page_shift) - 1));
  }
  a.pos[i] = p;
  a.slot[i] = slot;
}

// Rows up to which the plan's own workgroup fills positions and slots.
constexpr int kPlanFillRows = 4096;

// ---- RoPE and append --------------------------------------------------------------------------------
// (a, b) -> (a c - b s, b c + a s) on dims j and j + hd / 2.  A thread takes 4 such pairs of one head of one
// row, or 8 values to copy: 16-byte loads and stores in FP32, 8- and 16-byte ones into a 16-bit pool.
// One pass, each value read and written once: bound by memory.  7777 rows of 32 + 2 x 8 heads of 128 into BF16 pages (354 MB)
// 63 us, 5.6 TB/s; 64 rows 3.6 us.
struct AppendArgs {
  const float *q, *k, *v;
  float *q_out, *k_out;
  long ldq, ldqo, ldk, ldko, ldv, rows;
  int heads, KV, hd, n_pos;
  const int32_t* pos;
  const float *cos_t, *sin_t;
  const int64_t* slot;
  void *kp, *vp;
  long stride, n_slots;
  int shift;
};

typedef float f4v __attribute__((ext_vector_type(4)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef __bf16 b4v __attribute__((ext_vector_type(4)));

template <class T>
__device__ __forceinline__ void store4(T* dst, f4v v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<f4v*>(dst) = v;
  else if constexpr (std::is_same_v<T, _Float16>) *reinterpret_cast<h4v*>(dst) = __builtin_convertvector(v, h4v);
  else *reinterpret_cast<b4v*>(dst) = __builtin_convertvector(v, b4v);
}

template <class T>
__global__ __launch_bounds__(256) void rope_append_kernel(AppendArgs a) {
  const int per_head = a.hd / 8, nq = a.heads * per_head, nk = a.KV * per_head, items = nq + 2 * nk, half = a.hd / 2;
  const long id = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  const long row = id / items;
  if (row >= a.rows) return;
  int it = static_cast<int>(id - row * items);
  const int p = a.pos[row];
  const bool known = p >= 0 && p < a.n_pos;
  if (it < nq + nk) {
    const bool is_q = it < nq;
    it -= is_q ? 0 : nq;
    const int head = it / per_head, j = 4 * (it - head * per_head);
    const float* src = (is_q ? a.q + row * a.ldq : a.k + row * a.ldk) + head * a.hd + j;
    const float nan = __int_as_float(0x7FC00000);
    f4v lo = {nan, nan, nan, nan}, hi = lo;
    if (known) {
      const f4v x = *reinterpret_cast<const f4v*>(src), y = *reinterpret_cast<const f4v*>(src + half);
      const f4v c = *reinterpret_cast<const f4v*>(a.cos_t + static_cast<long>(p) * half + j);
      const f4v s = *reinterpret_cast<const f4v*>(a.sin_t + static_cast<long>(p) * half + j);
      lo = x * c - y * s;
      hi = y * c + x * s;
    }
    float* dst = is_q ? a.q_out + row * a.ldqo : a.k_out ? a.k_out + row * a.ldko : nullptr;
    if (dst) {
      dst += head * a.hd + j;
      *reinterpret_cast<f4v*>(dst) = lo;
      *reinterpret_cast<f4v*>(dst + half) = hi;
    }
    if (is_q || !known) return;
    const int64_t at = a.slot[row];
    if (at < 0 || at >= a.n_slots) return;
    T* kp = static_cast<T*>(a.kp) + (at >> a.shift) * a.stride +
            ((static_cast<long>(head) << a.shift) + (at & ((1L << a.shift) - 1))) * a.hd + j;
    store4(kp, lo);
    store4(kp + half, hi);
    return;
  }
  it -= nq + nk;
  const int64_t at = a.slot[row];
  if (!known || at < 0 || at >= a.n_slots) return;
  const int head = it / per_head, j = 8 * (it - head * per_head);
  const float* src = a.v + row * a.ldv + head * a.hd + j;
  const f4v x = *reinterpret_cast<const f4v*>(src), y = *reinterpret_cast<const f4v*>(src + 4);
  T* vp = static_cast<T*>(a.vp) + (at >> a.shift) * a.stride +
          ((static_cast<long>(head) << a.shift) + (at & ((1L << a.shift) - 1))) * a.hd + j;
  store4(vp, x);
  store4(vp + 4, y);
}

}  // namespace

void rope_tables_host(float theta, size_t hd, size_t n_pos, std::vector<float>* cos_t, std::vector<float>* sin_t) {
  const size_t half = hd / 2;
  std::vector<float> inv(half);
  for (size_t i = 0; i < half; ++i) {
    const float expo = static_cast<float>(2 * i) / static_cast<float>(hd);
    inv[i] = 1.0f / std::pow(theta, expo);
  }
  cos_t->resize(n_pos * half);
  sin_t->resize(n_pos * half);
  for (size_t p = 0; p < n_pos; ++p) {
    for (size_t i = 0; i < half; ++i) {
      const float ang = static_cast<float>(p) * inv[i];
      (*cos_t)[p * half + i] = std::cos(ang);
      (*sin_t)[p * half + i] = std::sin(ang);
    }
  }
}

int check_page_pool(const ef_hip_page_pool* p, const char* who) {
  auto w = [who](const char* what) { return std::string(who) + ": " + what; };
  EFH_CHECK(p != nullptr, w("null page pool"));
  EFH_CHECK(p->k_dev && p->v_dev, w("null page memory"));
  EFH_CHECK(p->qtype == EF_QTYPE_F32 || p->qtype == EF_QTYPE_F16 || p->qtype == EF_QTYPE_BF16,
            w("pages hold F32, F16 or BF16 values"));
  EFH_CHECK(p->n_pages >= 1 && p->n_pages <= 0x7FFFFFFF, w("bad page count"));
  EFH_CHECK(p->page_size >= 1 && p->page_size <= 1024 && (p->page_size & (p->page_size - 1)) == 0,
            w("page_size must be a power of two up to 1024"));
  EFH_CHECK(p->hd >= 8 && p->hd <= 256 && p->hd % 8 == 0, w("hd must be a multiple of 8 up to 256"));
  EFH_CHECK(p->KV >= 1 && p->KV <= 65535, w("bad KV head count"));
  const size_t size = p->qtype == EF_QTYPE_F32 ? 4 : 2, least = p->KV * p->page_size * p->hd;
  EFH_CHECK(pool_stride(*p) >= least && pool_stride(*p) * size % 16 == 0 && pool_stride(*p) <= (size_t(1) << 40),
            w("page_stride must hold a page and be a multiple of 16 bytes"));
  EFH_CHECK(pool_stride(*p) <= (size_t(1) << 60) / p->n_pages, w("pool too large"));
  EFH_CHECK(aligned16(p->k_dev) && aligned16(p->v_dev), w("page memory must be aligned to 16 bytes"));
  return EF_HIP_OK;
}

}  // namespace efh

using namespace efh;

extern "C" {

int ef_hip_page_plan(const int32_t* cached, const int32_t* fresh, size_t n_seqs, size_t page_size, size_t n_pages,
                     int32_t* table, size_t table_ld, int32_t* free_list, const int32_t* n_free, int32_t* n_free_out,
                     int32_t* kv_len, int32_t* row_start, int32_t* pos, int64_t* slot, size_t max_rows, int32_t* status,
                     void* stream) {
  EFH_CHECK(cached && fresh && table && free_list && n_free && n_free_out && kv_len && row_start && status,
            "page_plan: null pointer");
  EFH_CHECK(max_rows == 0 || (pos && slot), "page_plan: null pointer");
  EFH_CHECK(n_seqs >= 1 && n_seqs <= (size_t(1) << 20), "page_plan: n_seqs must be in [1, 2^20]");
  EFH_CHECK(page_size >= 1 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
            "page_plan: page_size must be a power of two up to 1024");
  EFH_CHECK(n_pages >= 1 && n_pages <= 0x7FFFFFFF, "page_plan: bad page count");
  EFH_CHECK(max_rows <= 0x7FFFFFFF - 256, "page_plan: max_rows too large");
  EFH_CHECK(table_ld >= 1 && table_ld <= size_t(0x7FFFFFFF) / page_size && table_ld <= size_t(0x7FFFFFFF) / n_seqs,
            "page_plan: table_ld must be at least 1, with a request's positions and the table's entries below 2^31");
  const PlanArgs a{cached,    fresh,      static_cast<int>(n_seqs), log2_of(page_size),         static_cast<int>(n_pages),
                   table,     static_cast<long>(table_ld), free_list, n_free, n_free_out, kv_len, row_start, pos, slot,
                   static_cast<int>(max_rows), status};
  EFH_RC(require_ready());
  hipStream_t s = pick(stream);
  const bool fill = n_seqs <= static_cast<size_t>(kPlanThreads) && max_rows <= static_cast<size_t>(kPlanFillRows);
  if (n_seqs > static_cast<size_t>(kPlanThreads)) page_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
  else if (n_seqs > kPlanFew) fill ? page_plan_once_kernel<kPlanThreads, true><<<1, kPlanThreads, 0, s>>>(a)
                                   : page_plan_once_kernel<kPlanThreads, false><<<1, kPlanThreads, 0, s>>>(a);
  else fill ? page_plan_once_kernel<kPlanFew, true><<<1, kPlanFew, 0, s>>>(a)
            : page_plan_once_kernel<kPlanFew, false><<<1, kPlanFew, 0, s>>>(a);
  if (!fill && max_rows > 0) {
    EFH_HIP(hipGetLastError());
    page_rows_kernel<<<static_cast<unsigned>((max_rows + 255) / 256), 256, 0, s>>>(a);
  }
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

int ef_hip_rope_tables(float theta, size_t hd, size_t n_pos, float* cos_dev, float* sin_dev) {
  EFH_CHECK(cos_dev && sin_dev, "rope_tables: null pointer");
  EFH_CHECK(theta > 0.0f && hd >= 2 && hd % 2 == 0 && hd <= 4096 && n_pos >= 1 && n_pos <= (size_t(1) << 28) / hd,
            "rope_tables: need theta > 0, an even hd up to 4096 and at most 2^28 / hd positions");
  EFH_RC(require_ready());
  std::vector<float> c, s;
  try {
    rope_tables_host(theta, hd, n_pos, &c, &s);
  } catch (const std::bad_alloc&) {
    return fail(EF_HIP_ENOMEM, "rope_tables: no host memory for the tables");
  }
  EFH_RC(ef_hip_memcpy_h2d(cos_dev, c.data(), c.size() * 4, nullptr));
  return ef_hip_memcpy_h2d(sin_dev, s.data(), s.size() * 4, nullptr);
}

int ef_hip_rope_append(const float* q, size_t ldq, float* q_out, size_t ldqo, size_t heads, const float* k, size_t ldk,
                       float* k_out, size_t ldko, const float* v, size_t ldv, size_t rows, const int32_t* pos,
                       const float* cos_dev, const float* sin_dev, size_t n_pos, const int64_t* slot,
                       const ef_hip_page_pool* pool, void* stream) {
  EFH_RC(check_page_pool(pool, "rope_append"));
  EFH_CHECK(q && q_out && k && v && pos && cos_dev && sin_dev && slot, "rope_append: null pointer");
  EFH_CHECK(heads >= 1 && heads <= 65535, "rope_append: bad head count");
  EFH_CHECK(n_pos >= 1 && n_pos <= 0x7FFFFFFF, "rope_append: bad n_pos");
  const size_t nq = heads * pool->hd, nk = pool->KV * pool->hd;
  EFH_CHECK(rows == 1 || (ldq >= nq && ldqo >= nq && ldk >= nk && ldv >= nk && (!k_out || ldko >= nk)),
            "rope_append: a row stride is shorter than its row");
  EFH_CHECK(ldq % 4 == 0 && ldqo % 4 == 0 && ldk % 4 == 0 && ldv % 4 == 0 && (!k_out || ldko % 4 == 0) && aligned16(q) &&
                aligned16(q_out) && aligned16(k) && aligned16(v) && aligned16(cos_dev) && aligned16(sin_dev) &&
                aligned16(k_out),
            "rope_append: strides and addresses must be multiples of 16 bytes");
  EFH_CHECK((q_out != q || ldqo == ldq) && (k_out != k || ldko == ldk),
            "rope_append: rows turned in place need the same stride on both sides");
  const size_t items = (heads + 2 * pool->KV) * (pool->hd / 8);
  EFH_CHECK(rows <= 0x7FFFFFFF && rows <= kGridMost * 256 / items, "rope_append: too many rows");
  const AppendArgs a{q, k, v, q_out, k_out, static_cast<long>(ldq), static_cast<long>(ldqo), static_cast<long>(ldk),
                     static_cast<long>(ldko), static_cast<long>(ldv), static_cast<long>(rows), static_cast<int>(heads),
                     static_cast<int>(pool->KV), static_cast<int>(pool->hd), static_cast<int>(n_pos), pos, cos_dev, sin_dev,
                     slot, pool->k_dev, pool->v_dev, static_cast<long>(pool_stride(*pool)),
                     static_cast<long>(pool->n_pages * pool->page_size), log2_of(pool->page_size)};
  EFH_RC(require_ready());
  if (rows == 0) return EF_HIP_OK;
  const unsigned blocks = static_cast<unsigned>((rows * items + 255) / 256);
  hipStream_t s = pick(stream);
  if (pool->qtype == EF_QTYPE_F32) rope_append_kernel<float><<<blocks, 256, 0, s>>>(a);
  else if (pool->qtype == EF_QTYPE_F16) rope_append_kernel<_Float16><<<blocks, 256, 0, s>>>(a);
  else rope_append_kernel<__bf16><<<blocks, 256, 0, s>>>(a);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

}  // extern "C"
