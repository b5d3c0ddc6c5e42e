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
// Measured (the kernel, then the join of its ranges): 12 requests of up to 32750 positions, 32 heads over 8 of 128, BF16 (1.17
// GB): 220 + 4.8 us, 5.3 TB/s of the 5.9 that a read of memory reaches; 64 requests of up to 2047, 32 over 4 of 64, FP16
// (103 MB): 19.7 + 4.1 us; one FP32 request of 2047: 6.7 + 3.7 us, bound by latency.  Registers for one more wave per SIMD: 26 -> 34 us at 64 requests.
//
// Masked positions: scores -inf, value rows zero.  A range whose sums come out infinite or NaN is computed again
// by wave_attend, which reads only what each row sees.
#pragma once

#include "attn_core.h"

namespace efh {

constexpr int kFewWaves = 4;

template <int HDP, int NT>
struct FewLds {
  float o[kFewWaves][16 * NT * (HDP + 4)];
  f2v stat[kFewWaves][16 * NT];
};

// One workgroup: request `req`, KV head `kvh`, range `split`, its row tiles tile0, tile0 + t.tiles, ..
template <class T, int HDP, int NT, bool WIDE>
__device__ __forceinline__ void attention_few(const AttnTask& t, FewLds<HDP, NT>& lds, int req, int kvh, int split, int tile0) {
  constexpr bool F32 = sizeof(T) == 4;
  // positions of a step, in matrix tiles of 16 (twice as many, 16 KB a step and wave at hd = 64, cost more occupancy
  // than they gained: 41 requests, 39 of them with one row, 54 -> 61 us)
  constexpr int TILES = F32 ? 1 : 2, KT = 16 * TILES, DP = HDP / 16;
  constexpr int KW = F32 ? HDP / 16 : HDP / 32;  // 16-byte pieces of a key row in a lane
  constexpr int VROWS = 4 * TILES, VW = F32 ? DP / 4 : DP * 2 / 16 + (DP == 4);  // value rows of a lane, 16-byte pieces each (8 bytes for 4 halves)
  constexpr float OFFSET = Parts<T>::kSubOffset, SLACK = Parts<T>::kSubSlack;
  constexpr int PAIRS = 16 * NT, LDO = HDP + 4;
  auto& o_s = lds.o;
  auto& stat_s = lds.stat;

  const RowsArgs& a = t.r;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
  const int m = lane & 15, g4 = lane >> 4;
  const int hd = a.hd, G = t.group;
  const long base = req * a.kv.table_ld;
  const int sh = a.kv.page_shift, pmask = (1 << sh) - 1;
  // the first step's pages, whatever the lengths turn out to be (inside the table, and checked before use)
  int pages[WIDE ? TILES : 1];
  if constexpr (WIDE) {
    const long c0 = static_cast<long>(split) * t.few_split.span + wave * KT, width = (a.kv.table_ld << sh) - 1;
#pragma unroll
    for (int u = 0; u < TILES; ++u) pages[u] = a.kv.table[base + (min(c0 + 16 * u, width) >> sh)];
  }
  const int first = max(a.row_start[req], 0), next = a.row_start[req + 1], n = min(next, a.max_rows) - first;
  const int kv_len = a.kv_len[req];
  const int kv = static_cast<int>(min(static_cast<long>(kv_len), a.kv.table_ld << a.kv.page_shift));
  if (n <= 0 || static_cast<long>(n) * G > t.few_most) return;
  const int ns = splits_of(kv, t.few_split);
  if (split >= ns) return;
  const int j0 = split * t.few_split.span, j1 = split == t.few_split.splits - 1 ? max(kv, 0) : min(max(kv, 0), j0 + t.few_split.span);
  const int before = kv_len - (next - first);  // row i sees positions 0 .. before + i; rows cut by max_rows count
  const T *kp = static_cast<const T*>(a.kv.k), *vp = static_cast<const T*>(a.kv.v);

  // this lane's dims: K pieces (clamped into the row: the query is zero there), V pieces
  int kd[KW], vd[VW];
#pragma unroll
  for (int i = 0; i < KW; ++i) kd[i] = F32 ? min(16 * i + 4 * g4, hd - 4) : min(32 * i + 8 * g4, hd - 8);
#pragma unroll
  for (int i = 0; i < VW; ++i) vd[i] = F32 ? min(m * DP + 4 * i, hd - 4) : DP == 4 ? min(m * DP, hd - 4) : min(m * DP + 8 * i, hd - 8);
  uint32_t kb[KW], vb[VW];  // byte offsets from the first of 16 rows (wide pages: rows of a tile follow each other)
#pragma unroll
  for (int i = 0; i < KW; ++i) kb[i] = (m * hd + kd[i]) * sizeof(T);
#pragma unroll
  for (int i = 0; i < VW; ++i) vb[i] = (4 * g4 * hd + vd[i]) * sizeof(T);

  for (int tile = tile0; tile * PAIRS < n * G; tile += t.tiles) {
    // ---- queries' raw values, then the first step's rows: all in flight together ------------------------------
    constexpr int NS = F32 ? 1 : Parts<T>::N, QW = F32 ? 1 : 2;
    f4v qf[NT][KW][QW];
    int seen[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int pair = tile * PAIRS + 16 * nt + m, row = t.row_of(pair), head = kvh * G + pair - row * G;
      const bool active = row < n;
      seen[nt] = active ? min(before + row + 1, kv) : 0;
      const float* q = a.q + (first + (active ? row : 0)) * a.ldq + static_cast<long>(active ? head : kvh * G) * hd;
#pragma unroll
      for (int i = 0; i < KW; ++i)
#pragma unroll
        for (int w = 0; w < QW; ++w) qf[nt][i][w] = *reinterpret_cast<const f4v*>(q + kd[i] + 4 * w);
    }
    const int all_see = min(before + t.row_of(tile * PAIRS) + 1, kv);  // positions that every row of the tile sees

    // ---- one pass over the range's positions -------------------------------------------------------------
    u4v kr[TILES][KW], vr[VROWS][VW];
    // Where the next step's rows lie: an offset for each tile of 16 rows (wide pages, the same for the whole wave), or
    // for each of the lane's key and value rows; and whether a page holds them, a bit each.
    long off[WIDE ? TILES : 5 * TILES];
    uint32_t held = 0, held_next = 0;
    constexpr uint32_t ALL = WIDE ? (1u << TILES) - 1 : (1u << 4 * TILES) - 1;
    auto look_up = [&](int c) {
      if constexpr (WIDE) {
#pragma unroll
        for (int u = 0; u < TILES; ++u) pages[u] = a.kv.table[base + (min(c + 16 * u, j1 - 1) >> sh)];
      }
    };
    auto place = [&](int c) {
      held_next = 0;
      if constexpr (WIDE) {
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          const int cu = c + 16 * u;
          const bool real = static_cast<uint32_t>(pages[u]) < static_cast<uint32_t>(a.kv.n_pages) && cu < j1;
          held_next |= real ? 1u << u : 0u;
          off[u] = real ? pages[u] * a.kv.page_stride + ((static_cast<long>(kvh) << sh) + (cu & pmask)) * hd : 0;
        }
      } else {
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          long ko = 0, vo = 0;
          const int jk = c + 16 * u + m;
          if (!(jk < j1 && kv_offset<true>(a.kv, kvh, hd, base, jk, &ko, &vo))) ko = 0;
          off[5 * u] = ko;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int jv = c + 16 * u + 4 * g4 + r;
            ko = vo = 0;
            const bool real = jv < j1 && kv_offset<true>(a.kv, kvh, hd, base, jv, &ko, &vo);
            held_next |= real ? 1u << (4 * u + r) : 0u;
            off[5 * u + 1 + r] = real ? vo : 0;
          }
        }
      }
    };
    auto load_k = [&]() {
#pragma unroll
      for (int u = 0; u < TILES; ++u)
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          if constexpr (WIDE) kr[u][i] = *reinterpret_cast<const u4v*>(reinterpret_cast<const char*>(kp + off[u]) + kb[i]);
          else kr[u][i] = *reinterpret_cast<const u4v*>(kp + off[5 * u] + kd[i]);
        }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int j = 0; j < VROWS; ++j)
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const char* at;
          if constexpr (WIDE) at = reinterpret_cast<const char*>(vp + off[j / 4] + j % 4 * hd) + vb[i];
          else at = reinterpret_cast<const char*>(vp + off[5 * (j / 4) + 1 + j % 4] + vd[i]);
          if constexpr (!F32 && DP == 4) {
            const u2v x = *reinterpret_cast<const u2v*>(at);
            vr[j][i] = u4v{x[0], x[1], 0, 0};
          } else {
            vr[j][i] = *reinterpret_cast<const u4v*>(at);
          }
        }
    };

    constexpr int STEP = kFewWaves * KT;
    int c = j0 + wave * KT;
    if (c < j1) {
      if (tile != tile0) look_up(c);
      place(c);
      load_k();
      load_v();
      look_up(c + STEP);
    }
    // ---- queries as operands ------------------------------------------------------------------------------
    u4v qp[F32 ? 1 : NT][KW][NS];
    float c2[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      c2[nt] = a.c2;
#pragma unroll
      for (int i = 0; i < KW; ++i)
        if (F32 ? 16 * i + 4 * g4 >= hd : 32 * i + 8 * g4 >= hd) {
#pragma unroll
          for (int w = 0; w < QW; ++w) qf[nt][i][w] = f4v{0, 0, 0, 0};
        }
      if constexpr (!F32) {
        int e = 0;
        if constexpr (std::is_same_v<T, _Float16>) {
          float top = 0.0f;
#pragma unroll
          for (int i = 0; i < KW; ++i)
#pragma unroll
            for (int u = 0; u < 8; ++u) top = fmaxf(top, fabsf(qf[nt][i][u / 4][u % 4]));
          e = query_exponent(column_max(top));
          c2[nt] = ldexpf(c2[nt], -e);
        }
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          float x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            x[u] = qf[nt][i][u / 4][u % 4];
            if constexpr (std::is_same_v<T, _Float16>) x[u] = ldexpf(x[u], e);
          }
          split8<T>(x, qp[nt][i]);
        }
      }
    }

    f4v o[NT][DP];
    float sub[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int d = 0; d < DP; ++d) o[nt][d] = f4v{0, 0, 0, 0};
      sub[nt] = -INFINITY;
      l[nt] = 0.0f;
    }
    for (; c < j1; c += STEP) {
      const bool more = c + STEP < j1;
      held = held_next;
      const bool partial = (WIDE ? held != ALL : __any(held != ALL)) || c + KT > all_see;
      f4v sc[NT][TILES];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          if constexpr (F32) {
            // a sum for every 16 dims, two at a time: one or two long ones are further from float64 than a plain FP32 sum is
            f4v sum = {0, 0, 0, 0};
#pragma unroll
            for (int two = 0; two < KW; two += 2) {
              f4v part[2] = {f4v{0, 0, 0, 0}, f4v{0, 0, 0, 0}};
              // these products behind the sum before: side by side they take registers (8 rows of 128 dims: 58 -> 92 us)
              if (two) asm volatile("" : "+v"(qf[nt][two][0]), "+v"(qf[nt][two + 1][0]) : "v"(sum));
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                  part[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[u][two + i][s]), qf[nt][two + i][0][s], part[i], 0, 0, 0);
              sum += part[0] + part[1];
              asm volatile("" : "+v"(sum));
            }
            sc[nt][u] = sum;
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
        place(c + STEP);
        load_k();
        look_up(c + 2 * STEP);
      }
      if (partial) {
#pragma unroll
        for (int u = 0; u < TILES; ++u) {
          const int at = c + 16 * u + 4 * g4;  // the lane's first position of the tile
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool real = held >> (WIDE ? u : 4 * u + r) & 1;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if (at + r >= (real ? min(seen[nt], j1) : 0)) sc[nt][u][r] = -INFINITY;
            if (at + r >= (real ? j1 : 0)) {
#pragma unroll
              for (int i = 0; i < VW; ++i) vr[4 * u + r][i] = u4v{0, 0, 0, 0};
            }
          }
        }
      }
      float p[NT][4 * TILES];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float cm = -INFINITY;
#pragma unroll
        for (int u = 0; u < TILES; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) cm = fmaxf(cm, sc[nt][u][r]);
        cm = column_max(cm);
        const float high = cm * c2[nt] - OFFSET;
        if (__any(high > sub[nt] + SLACK)) {
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
        for (int r = 0; r < VROWS; ++r)
#pragma unroll
          for (int d = 0; d < DP; ++d)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              o[nt][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[r][d / 4][d % 4]), p[nt][r], o[nt][d], 0, 0, 0);
      } else {
#pragma unroll
        for (int gr = 0; gr < TILES / 2; ++gr) {  // 32 positions: one product
          u4v pp[NT][NS];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[nt][8 * gr + i];
            split8<T>(x, pp[nt]);
          }
#pragma unroll
          for (int d = 0; d < DP; ++d) {
            u4v v;  // dim m DP + d of the lane's eight value rows
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = __builtin_amdgcn_perm(vr[8 * gr + 2 * i + 1][d / 8][d % 8 / 2], vr[8 * gr + 2 * i][d / 8][d % 8 / 2],
                                           d % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int s = NS - 1; s >= 0; --s) o[nt][d] = mfma16<T>(v, pp[nt][s], o[nt][d]);
          }
        }
      }
      if (more) load_v();
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
      const int p = tile * PAIRS + pair, row = t.row_of(p), head = kvh * G + p - row * G;
      *out_row = (first + row) * a.ldo + static_cast<long>(head) * hd;
      *part_row = (static_cast<long>(split) * a.max_rows + first + row) * a.H + head;
    };
    if (split == 0 && t.count != nullptr) {
      for (int p = tid; p < pairs; p += kFewWaves * kWave) {
        const int row = t.row_of(tile * PAIRS + p);
        t.count[static_cast<long>(first + row) * a.H + kvh * G + tile * PAIRS + p - row * G] = ns;
      }
    }
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
        const int p = tile * PAIRS + pair, row = t.row_of(p), head = kvh * G + p - row * G;
        const float* q = a.q + (first + row) * a.ldq + static_cast<long>(head) * hd;
        for (int d = lane; d < hd; d += kWave) qs[d] = q[d];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float sb = -INFINITY, ov[4] = {0, 0, 0, 0};
        double ll = 0.0;
        wave_attend<T, true>(a.kv, kvh, hd, base, qs, a.c2, j0, min(j1, min(before + row + 1, kv)), kv, &sb, &ll, ov);
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

}  // namespace efh
