// Attention of few new rows over a request's pages (a decode step, a handful of guesses).
//
// A workgroup takes up to 16 NT (row, query head) pairs of one request and KV head and one range of positions; its
// four waves take every fourth step of KT positions and join in LDS at the end, ranges join in
// attention_join_kernel.  S^T = K Q^T puts a pair's scores in its own lanes (D: positions 4 g + r, pair m, lane
// 16 g + m); the k slots of a product may hold positions in any order, so lane 16 g + m loads the V rows
// 4 g + j and the weights feed O^T += V^T P^T from the registers they were computed in.  Keys and values go from
// memory to registers straight: K rows are the A operand as they lie, V is turned in the lane (two halves of
// eight rows to a word by v_perm).  LDS only joins the waves.
//
// Bound by memory: the next step's keys load while this one's weights form, the next values while the next
// scores form.  FP32 pages use v_mfma_f32_16x16x4_f32 on the values as they are.
//
// Masked positions: scores -inf, value rows zero.  A range whose sums come out infinite or NaN is computed again
// by wave_attend, which reads only what each row sees.
#include <algorithm>

#include "attn_core.h"

namespace efh {
namespace {

constexpr int kFewWaves = 4;

template <class T, int HDP, int NT, bool WIDE>
__global__ __launch_bounds__(kFewWaves * kWave, HDP == 256 ? 1 : (HDP == 64 ? 3 : 2) - !WIDE) void attention_few_kernel(AttnTask t) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int KT = F32 ? 16 : 32, TILES = KT / 16, DP = HDP / 16;
  constexpr int KW = F32 ? HDP / 16 : HDP / 32;  // 16-byte pieces of a key row in a lane
  constexpr int VROWS = 4 * TILES, VW = F32 ? DP / 4 : DP * 2 / 16 + (DP == 4);  // value rows of a lane, 16-byte pieces each (8 bytes for 4 halves)
  constexpr float OFFSET = F32 ? 0.0f : Parts<T>::kSubOffset;
  constexpr int PAIRS = 16 * NT, LDO = HDP + 4;
  __shared__ float o_s[kFewWaves][PAIRS * LDO];
  __shared__ f2v stat_s[kFewWaves][PAIRS];

  const RowsArgs& a = t.r;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
  const int m = lane & 15, g4 = lane >> 4;
  const int split = blockIdx.y;
  int id = blockIdx.x;
  const int kvh = id % a.KV;
  id /= a.KV;
  const int tile0 = id % t.tiles, req = id / t.tiles;
  const int hd = a.hd, G = a.H / a.KV;
  const int first = a.row_start[req], n = min(a.row_start[req + 1], a.max_rows) - first;
  const long base = req * a.kv.table_ld;
  const int kv_len = a.kv_len[req];
  const int kv = static_cast<int>(min(static_cast<long>(kv_len), a.kv.table_ld << a.kv.page_shift));
  if (n <= 0 || static_cast<long>(n) * G > t.few_most) return;
  const int ns = splits_of(kv, t.few_split);
  if (split >= ns) return;
  const int j0 = split * t.few_split.span, j1 = split == t.few_split.splits - 1 ? max(kv, 0) : min(max(kv, 0), j0 + t.few_split.span);
  const int before = kv_len - n;  // row i sees positions 0 .. before + i
  const int sh = a.kv.page_shift, pmask = (1 << sh) - 1;
  const T *kp = static_cast<const T*>(a.kv.k), *vp = static_cast<const T*>(a.kv.v);

  // this lane's dims: K pieces (clamped into the row: the query is zero there), V pieces
  int kd[KW], vd[VW];
#pragma unroll
  for (int i = 0; i < KW; ++i) kd[i] = F32 ? min(16 * i + 4 * g4, hd - 4) : min(32 * i + 8 * g4, hd - 8);
#pragma unroll
  for (int i = 0; i < VW; ++i) vd[i] = F32 ? min(m * DP + 4 * i, hd - 4) : DP == 4 ? min(m * DP, hd - 4) : min(m * DP + 8 * i, hd - 8);

  for (int tile = tile0; tile * PAIRS < n * G; tile += t.tiles) {
    // ---- queries -------------------------------------------------------------------------------------
    constexpr int NS = F32 ? 1 : Parts<T>::N;
    f4v qf[F32 ? NT : 1][KW];
    u4v qp[F32 ? 1 : NT][KW][NS];
    float c2[NT];
    int seen[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int pair = tile * PAIRS + 16 * nt + m, row = pair / G, head = kvh * G + pair - row * G;
      const bool active = row < n;
      seen[nt] = active ? min(before + row + 1, kv) : 0;
      const float* q = a.q + (first + (active ? row : 0)) * a.ldq + static_cast<long>(active ? head : kvh * G) * hd;
      c2[nt] = a.c2;
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          qf[nt][i] = *reinterpret_cast<const f4v*>(q + kd[i]);
          if (16 * i + 4 * g4 >= hd) qf[nt][i] = f4v{0, 0, 0, 0};
        }
      } else {
        float x[KW][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          load8(q + kd[i], x[i]);
          if (32 * i + 8 * g4 >= hd) {
#pragma unroll
            for (int u = 0; u < 8; ++u) x[i][u] = 0.0f;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) top = fmaxf(top, fabsf(x[i][u]));
        }
        if constexpr (std::is_same_v<T, _Float16>) {
          const int e = query_exponent(column_max(top));
          c2[nt] = ldexpf(c2[nt], -e);
#pragma unroll
          for (int i = 0; i < KW; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) x[i][u] = ldexpf(x[i][u], e);
        }
#pragma unroll
        for (int i = 0; i < KW; ++i) split8<T>(x[i], qp[nt][i]);
      }
    }
    const int all_see = min(before + tile * PAIRS / G + 1, kv);  // positions that every row of the tile sees

    // ---- one pass over the range's positions -------------------------------------------------------------
    u4v kr[TILES][KW], vr[VROWS][VW];
    bool ok[TILES][WIDE ? 1 : 4];   // whether this lane's value rows have a page
    long koff[TILES], voff[WIDE ? TILES : VROWS];
    bool lost = false, lost_next = false, ok_next[TILES][WIDE ? 1 : 4];
    long koff_next[TILES], voff_next[WIDE ? TILES : VROWS];
    auto place = [&](int c) {  // where the step's rows lie
      lost_next = false;
      if constexpr (WIDE) {
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          const int cu = c + 16 * u;
          int page = -1;
          if (cu < j1) page = a.kv.table[base + (cu >> sh)];
          const bool real = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.kv.n_pages);
          ok_next[u][0] = real;
          lost_next |= !real;
          koff_next[u] = real ? page * a.kv.page_stride + ((static_cast<long>(kvh) << sh) + (cu & pmask)) * hd : 0;
          voff_next[u] = koff_next[u];
        }
      } else {
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          long ko = 0, vo = 0;
          const int jk = c + 16 * u + m;
          if (!(jk < j1 && kv_offset<true>(a.kv, kvh, hd, base, jk, &ko, &vo))) ko = 0;
          koff_next[u] = ko;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int jv = c + 16 * u + 4 * g4 + r;
            ko = vo = 0;
            const bool real = jv < j1 && kv_offset<true>(a.kv, kvh, hd, base, jv, &ko, &vo);
            ok_next[u][r] = real;
            lost_next |= !real;
            voff_next[4 * u + r] = real ? vo : 0;
          }
        }
        lost_next = __any(lost_next);
      }
    };
    auto load_k = [&]() {
#pragma unroll
      for (int u = 0; u < TILES; ++u) {
        const T* row = kp + koff[u] + (WIDE ? m * hd : 0);
#pragma unroll
        for (int i = 0; i < KW; ++i) kr[u][i] = *reinterpret_cast<const u4v*>(row + kd[i]);
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int j = 0; j < VROWS; ++j) {
        const T* row = WIDE ? vp + voff[j / 4] + (4 * g4 + j % 4) * hd : vp + voff[WIDE ? 0 : j];
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          if constexpr (!F32 && DP == 4) {
            const u2v x = *reinterpret_cast<const u2v*>(row + vd[i]);
            vr[j][i] = u4v{x[0], x[1], 0, 0};
          } else {
            vr[j][i] = *reinterpret_cast<const u4v*>(row + vd[i]);
          }
        }
      }
    };
    auto take_place = [&]() {
#pragma unroll
      for (int u = 0; u < TILES; ++u) {
        koff[u] = koff_next[u];
#pragma unroll
        for (int r = 0; r < (WIDE ? 1 : 4); ++r) ok[u][r] = ok_next[u][r];
      }
#pragma unroll
      for (int u = 0; u < (WIDE ? TILES : VROWS); ++u) voff[u] = voff_next[u];
      lost = lost_next;
    };

    f4v o[NT][DP];
    float sub[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int d = 0; d < DP; ++d) o[nt][d] = f4v{0, 0, 0, 0};
      sub[nt] = -INFINITY;
      l[nt] = 0.0f;
    }
    constexpr int STEP = kFewWaves * KT;
    int c = j0 + wave * KT;
    if (c < j1) {
      place(c);
      take_place();
      load_k();
      load_v();
      place(c + STEP);
    }
    for (; c < j1; c += STEP) {
      const bool more = c + STEP < j1;
      const bool partial = lost || c + KT > all_see;
      bool okc[TILES][WIDE ? 1 : 4];
#pragma unroll
      for (int u = 0; u < TILES; ++u)
#pragma unroll
        for (int r = 0; r < (WIDE ? 1 : 4); ++r) okc[u][r] = ok[u][r];
      f4v sc[NT][TILES];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          if constexpr (F32) {
            f4v part[2] = {f4v{0, 0, 0, 0}, f4v{0, 0, 0, 0}};
#pragma unroll
            for (int i = 0; i < KW; ++i)
#pragma unroll
              for (int s = 0; s < 4; ++s)
                part[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[u][i][s]), qf[nt][i][s], part[i & 1], 0, 0, 0);
            sc[nt][u] = part[0] + part[1];
          } else {
            f4v acc = {0, 0, 0, 0};
#pragma unroll
            for (int s = NS - 1; s >= 0; --s)  // the small parts first
#pragma unroll
              for (int i = 0; i < KW; ++i) acc = mfma16<T>(kr[u][i], qp[nt][i][s], acc);
            sc[nt][u] = acc;
          }
        }
      if (more) {
        take_place();
        load_k();
      }
      if (partial) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < TILES; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c + 16 * u + 4 * g4 + r >= min(seen[nt], j1) || !okc[u][WIDE ? 0 : r]) sc[nt][u][r] = -INFINITY;
#pragma unroll
        for (int u = 0; u < TILES; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (c + 16 * u + 4 * g4 + r >= j1 || !okc[u][WIDE ? 0 : r]) {
#pragma unroll
              for (int i = 0; i < VW; ++i) vr[4 * u + r][i] = u4v{0, 0, 0, 0};
            }
      }
      float p[NT][8];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float cm = -INFINITY;
#pragma unroll
        for (int u = 0; u < TILES; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) cm = fmaxf(cm, sc[nt][u][r]);
        cm = column_max(cm);
        const float high = cm * c2[nt] - OFFSET;
        if (__any(high > sub[nt] + kSubSlack)) {
          const float to = fmaxf(sub[nt], high);
          const float al = to == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sub[nt] - to);
          sub[nt] = to;
          l[nt] *= al;
#pragma unroll
          for (int d = 0; d < DP; ++d) o[nt][d] *= al;
        }
        const float from = sub[nt] == -INFINITY ? 0.0f : sub[nt];
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < TILES; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            p[nt][4 * u + r] = __builtin_amdgcn_exp2f(fmaf(sc[nt][u][r], c2[nt], -from));
            sum += p[nt][4 * u + r];
          }
        l[nt] += sum;
      }
      if constexpr (F32) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int d = 0; d < DP; ++d)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[r][d / 4][d % 4]), p[nt][r], o[nt][d], 0, 0, 0);
      } else {
        u4v pp[NT][NS];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) split8<T>(p[nt], pp[nt]);
#pragma unroll
        for (int d = 0; d < DP; ++d) {
          u4v v;  // dim m DP + d of the lane's eight value rows
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[i] = __builtin_amdgcn_perm(vr[(2 * i + 1) % VROWS][d / 8][d % 8 / 2], vr[2 * i % VROWS][d / 8][d % 8 / 2],
                                         d % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int s = NS - 1; s >= 0; --s) o[nt][d] = mfma16<T>(v, pp[nt][s], o[nt][d]);
        }
      }
      if (more) {
        load_v();
        place(c + 2 * STEP);
      }
    }

    // ---- the waves' sums joined ------------------------------------------------------------------------
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float lw = column_sum(l[nt]);
      if (g4 == 0) stat_s[wave][16 * nt + m] = f2v{sub[nt], lw};
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int d = 0; d < DP; ++d) o_s[wave][(16 * nt + m) * LDO + (4 * g4 + r) * DP + d] = o[nt][d][r];
    }
    __syncthreads();
    const int pairs = min(n * G - tile * PAIRS, PAIRS);
    const bool direct = ns == 1;
    auto place_of = [&](int pair, long* out_row, long* part_row) {
      const int p = tile * PAIRS + pair, row = p / G, head = kvh * G + p - row * G;
      *out_row = (first + row) * a.ldo + static_cast<long>(head) * hd;
      *part_row = (static_cast<long>(split) * a.max_rows + first + row) * a.H + head;
    };
    bool bad = false;
    for (int idx = tid; idx < pairs * (hd / 4); idx += kFewWaves * kWave) {
      const int pair = idx / (hd / 4), d = 4 * (idx - pair * (hd / 4));
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) top = fmaxf(top, stat_s[w][pair][0]);
      float sum = 0.0f;
      f4v acc = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) {
        const f2v st = stat_s[w][pair];
        const float f = st[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st[0] - top);
        const f4v x = *reinterpret_cast<const f4v*>(&o_s[w][pair * LDO + d]);
        sum = fmaf(st[1], f, sum);
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] = fmaf(x[u], f, acc[u]);
      }
      bad = bad || !(fabsf(acc[0]) + fabsf(acc[1]) + fabsf(acc[2]) + fabsf(acc[3]) + sum < INFINITY);
      long out_row, part_row;
      place_of(pair, &out_row, &part_row);
      if (direct) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        *reinterpret_cast<f4v*>(a.out + out_row + d) = acc * inv;
      } else {
        *reinterpret_cast<f4v*>(t.part + part_row * hd + d) = acc;
        if (d == 0) t.stat[part_row] = f2v{top, sum};
      }
    }
    if (__syncthreads_or(bad)) {
      // some row sees an infinity or NaN, or has one beside what it sees: each pair again by itself
      float* qs = o_s[wave];
      for (int pair = wave; pair < pairs; pair += kFewWaves) {
        const int p = tile * PAIRS + pair, row = p / G, head = kvh * G + p - row * G;
        const float* q = a.q + (first + row) * a.ldq + static_cast<long>(head) * hd;
        for (int d = lane; d < hd; d += kWave) qs[d] = q[d];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float sb = -INFINITY, ov[4] = {0, 0, 0, 0};
        double ll = 0.0;
        wave_attend<T, true>(a.kv, kvh, hd, base, qs, a.c2, j0, min(j1, min(before + row + 1, kv)), &sb, &ll, ov);
        ll = wave_sum_d_dpp(ll);
        long out_row, part_row;
        place_of(pair, &out_row, &part_row);
        const float inv = ll == 0.0 ? 0.0f : static_cast<float>(1.0 / ll);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int d = lane + 64 * u;
          if (d >= hd) continue;
          if (direct) a.out[out_row + d] = ov[u] * inv;
          else t.part[part_row * hd + d] = ov[u];
        }
        if (!direct && lane == 0) t.stat[part_row] = f2v{sb, static_cast<float>(ll)};
        __builtin_amdgcn_wave_barrier();
      }
    }
    __syncthreads();  // o_s is free for the next tile
  }
}

// Each (row, head) of a request whose positions were split: its ranges' sums added, a wave each.
__global__ __launch_bounds__(256) void attention_join_kernel(AttnTask t) {
  const RowsArgs& a = t.r;
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  const int row = blockIdx.x, h = blockIdx.y * 4 + wave;
  if (row >= min(a.row_start[a.n_seqs], a.max_rows) || h >= a.H) return;
  const int req = request_of(a.row_start, a.n_seqs, row);
  const int kv = static_cast<int>(min(static_cast<long>(a.kv_len[req]), a.kv.table_ld << a.kv.page_shift));
  const long pairs = static_cast<long>(a.row_start[req + 1] - a.row_start[req]) * (a.H / a.KV);
  const int ns = splits_of(kv, pairs <= t.few_most ? t.few_split : t.tile_split);
  if (ns == 1) return;
  const long step = static_cast<long>(a.max_rows) * a.H, at = static_cast<long>(row) * a.H + h;
  float top = -INFINITY;
  for (int s = lane; s < ns; s += kWave) top = fmaxf(top, t.stat[s * step + at][0]);
  top = wave_max_dpp(top);
  float l = 0.0f, o[4] = {0, 0, 0, 0};
  for (int s = 0; s < ns; ++s) {
    const f2v st = t.stat[s * step + at];
    const float f = st[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(st[0] - top);
    l = fmaf(st[1], f, l);
    const float* p = t.part + (s * step + at) * a.hd;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (lane + 64 * u < a.hd) o[u] = fmaf(p[lane + 64 * u], f, o[u]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  float* out = a.out + row * a.ldo + static_cast<long>(h) * a.hd;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + 64 * u < a.hd) out[lane + 64 * u] = o[u] * inv;
}

template <class T, int HDP, int NT>
void run_few(const AttnTask& t, hipStream_t s) {
  const dim3 grid(t.r.n_seqs * t.r.KV * t.tiles, t.few_split.splits);
  if (t.r.kv.page_shift >= 4) attention_few_kernel<T, HDP, NT, true><<<grid, kFewWaves * kWave, 0, s>>>(t);
  else attention_few_kernel<T, HDP, NT, false><<<grid, kFewWaves * kWave, 0, s>>>(t);
}

template <class T>
void run_few_of(const AttnTask& t, hipStream_t s) {
  if (t.r.hd <= 64) run_few<T, 64, 1>(t, s);
  else if (t.r.hd <= 128) run_few<T, 128, 1>(t, s);
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
  attention_join_kernel<<<dim3(t.r.max_rows, (t.r.H + 3) / 4), 256, 0, s>>>(t);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

}  // namespace efh
