// Attention of few new rows over pages, and the sum of what ranges of positions gave.
#include <algorithm>

#include "attn_few.h"

namespace efh {
namespace {

// Each (row, head) whose positions were split: its ranges' sums added, by one wave, or by the workgroup's four where there
// are many ranges (one request of 30000 positions: 236 of them).  A lane takes 4 dims of every (waves 64 / (hd / 4))th
// range.  The lengths are not read: the first range's workgroup left their number beside its sums, and the loads of the
// first ranges do not wait for it (what they read beyond it is not used).
constexpr int kJoinFirst = 4;
// Of every range's weight, so that up to 1024 sums near FP32's largest do not pass it together.
constexpr float kJoinRoom = 0x1p-12f;

template <int LANES, bool MANY>  // lanes to a row: 16, 32 or 64; MANY: a workgroup to a row
__global__ __launch_bounds__(256) void attention_join_kernel(AttnTask t) {
  constexpr int WAVES = MANY ? 4 : 1, GROUPS = WAVES * kWave / LANES;
  __shared__ f4v sum_s[MANY ? 4 : 1][MANY ? LANES : 1];
  const RowsArgs& a = t.r;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const long at = MANY ? static_cast<long>(blockIdx.x) : static_cast<long>(blockIdx.x) * 4 + wave, step = static_cast<long>(a.max_rows) * a.H;
  const int group = (MANY ? wave * (kWave / LANES) : 0) + lane / LANES, d = 4 * (lane % LANES);
  const int most = max(t.few_split.splits, t.tile_split.splits);
  const long before = max(a.row_start[0], 0), rows = min(a.row_start[a.n_seqs], a.max_rows);
  if (at >= step) return;
  const bool in = d < a.hd;
  const float* part = t.part + at * a.hd + (in ? d : 0);
  const int ns = min(t.count[at], most);
  f4v first[kJoinFirst];
#pragma unroll
  for (int i = 0; i < kJoinFirst; ++i) first[i] = *reinterpret_cast<const f4v*>(part + min(group + i * GROUPS, most - 1) * step * a.hd);
  f2v st = t.stat[min(lane, most - 1) * step + at];
  if (at < before * a.H || at >= rows * a.H || ns <= 1) return;  // rows of no request have no number either
  float top = lane < ns ? st[0] : -INFINITY;
  for (int s = lane + kWave; s < ns; s += kWave) top = fmaxf(top, t.stat[s * step + at][0]);
  top = wave_max_dpp(top);
  float l = 0.0f;
  f4v o = {0, 0, 0, 0};
  auto add = [&](f4v x, float f) {
#pragma unroll
    for (int u = 0; u < 4; ++u) o[u] = fmaf(x[u], f, o[u]);
  };
  for (int s0 = 0; s0 < ns; s0 += kWave) {
    if (s0 > 0) st = t.stat[min(s0 + lane, ns - 1) * step + at];
    const float w = s0 + lane < ns && st[0] != -INFINITY ? __builtin_amdgcn_exp2f(st[0] - top) * kJoinRoom : 0.0f;
    if (s0 + lane < ns) l = fmaf(st[1], w, l);
    const int end = min(ns - s0, kWave);  // this round's ranges; the trip counts are the same for every group
    for (int b = 0; b < end; b += kJoinFirst * GROUPS) {
      f4v x[kJoinFirst];
#pragma unroll
      for (int i = 0; i < kJoinFirst; ++i) {
        const int s = s0 + b + group + i * GROUPS;
        x[i] = s0 + b == 0 ? first[i] : *reinterpret_cast<const f4v*>(part + min(s, ns - 1) * step * a.hd);
      }
#pragma unroll
      for (int i = 0; i < kJoinFirst; ++i) {
        const int s = b + group + i * GROUPS;
        const float f = __shfl(w, s & 63, kWave);
        if (s < end) add(x[i], f);
      }
    }
  }
  l = wave_sum(l);
#pragma unroll
  for (int off = LANES; off < kWave; off <<= 1) {
#pragma unroll
    for (int u = 0; u < 4; ++u) o[u] += __shfl_xor(o[u], off, kWave);
  }
  if constexpr (MANY) {
    if (lane < LANES) sum_s[wave][lane] = o;
    __syncthreads();
    if (wave != 0) return;
    o = sum_s[0][lane % LANES] + sum_s[1][lane % LANES] + sum_s[2][lane % LANES] + sum_s[3][lane % LANES];
  }
  if (lane >= LANES || !in) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const long row = at / a.H;
  *reinterpret_cast<f4v*>(a.out + row * a.ldo + (at - row * a.H) * a.hd + d) = o * inv;
}

template <int LANES>
void run_join(const AttnTask& t, hipStream_t s) {
  const long pairs = static_cast<long>(t.r.max_rows) * t.r.H;
  if (std::max(t.few_split.splits, t.tile_split.splits) > kJoinMany) attention_join_kernel<LANES, true><<<static_cast<unsigned>(pairs), 256, 0, s>>>(t);
  else attention_join_kernel<LANES, false><<<static_cast<unsigned>((pairs + 3) / 4), 256, 0, s>>>(t);
}

// Workgroups of a CU at the kernel's registers: narrow pages need more of them, but 16 pairs of FP32 heads of 128 still fit twice
// (16 requests of 2000, pages of 8: 45.8 us; once 59.6).
template <class T, int HDP, int NT, bool WIDE>
constexpr int few_occupancy() {
  return HDP == 256 ? 1 : (HDP == 64 && NT == 1 ? 3 : 2) - (WIDE || (sizeof(T) == 4 && HDP == 128 && NT == 1) ? 0 : 1);
}

template <class T, int HDP, int NT, bool WIDE>
__global__ __launch_bounds__(kFewWaves * kWave, (few_occupancy<T, HDP, NT, WIDE>())) void attention_few_kernel(AttnTask t) {
  __shared__ FewLds<HDP, NT> lds;
  const int split = blockIdx.z / t.tiles;
  attention_few<T, HDP, NT, WIDE>(t, lds, blockIdx.x, blockIdx.y, split, blockIdx.z - split * t.tiles);
}

template <class T, int HDP, int NT>
void run_few(const AttnTask& t, hipStream_t s) {
  const dim3 grid(t.r.n_seqs, t.r.KV, t.few_split.splits * t.tiles);
  if (t.r.kv.page_shift >= 4) attention_few_kernel<T, HDP, NT, true><<<grid, kFewWaves * kWave, 0, s>>>(t);
  else attention_few_kernel<T, HDP, NT, false><<<grid, kFewWaves * kWave, 0, s>>>(t);
}

template <class T>
void run_few_of(const AttnTask& t, hipStream_t s) {
  if (t.r.hd <= 64) t.few_wide ? run_few<T, 64, 2>(t, s) : run_few<T, 64, 1>(t, s);
  else if (t.r.hd <= 128) t.few_wide ? run_few<T, 128, 2>(t, s) : run_few<T, 128, 1>(t, s);
  else run_few<T, 256, 1>(t, s);
}

}  // namespace

int launch_attention_few(const AttnTask& t, int qtype, hipStream_t s) {
  if (qtype == EF_QTYPE_F32) run_few_of<float>(t, s);
  else if (qtype == EF_QTYPE_F16) run_few_of<_Float16>(t, s);
  else run_few_of<__bf16>(t, s);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

int launch_attention_join(const AttnTask& t, hipStream_t s) {
  if (t.r.hd <= 64) run_join<16>(t, s);
  else if (t.r.hd <= 128) run_join<32>(t, s);
  else run_join<64>(t, s);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

}  // namespace efh
