// Attention of many new rows: chunks over pages, and packed prompts.
//
// A workgroup takes 128 (row, query head) pairs of one request and KV head, 32 to a wave, and walks the positions
// they see in tiles of BN: a tile's keys and values are staged in LDS once for all pairs, loaded into registers
// while the tile before is used.  S^T = K Q^T by v_mfma_f32_32x32x16 puts a pair's scores in its own two lanes (D:
// positions 8 (i / 4) + 4 h + i % 4, pair lane % 32, h = lane / 32).  The k slots of a product may hold
// positions in any order, so the weights feed O^T += V^T P^T from the registers they were computed in, against
// V read transposed from LDS (ds_read_b64_tr_b16: 16 lanes read four positions' rows of 16 dims and get four
// positions of a dim each).  16-bit parts of the queries and the weights keep FP32's accuracy (attn_core.h): two
// products for FP16 keys and values, three for BF16.  FP32 tiles are scaled by powers of two and split into two
// FP16 parts (three products), as they are staged or, for packed rows with enough work, by a kernel before.
//
// Bound by the matrix cores and, beside them, the vector instructions: 9001 packed FP16 rows (508 GFLOP of attention, twice that in
// products) 873 us, 1165 TFLOP/s of products.  The matrix units are busy 61% of the cycles (70% in a large library product, which
// reaches 1187) and the other vector instructions' issue takes 33% (11%): the two hardly overlap.  The clock falls from 1.8 to
// 1.5 GHz over a few launches of either.  6001 FP32 rows 220 us, with the preparation, 10 to 12 in its traces; 500 rows after 8111 positions of FP16 pages
// 151 us with the join, after 8000 of FP32 pages 155 (hd 64) and 318 (hd 128).  Six products of three BF16 parts took 350 us for the
// 6001 FP32 rows; tiles through registers instead of LDS-DMA 941 us for the 9001 (868 when first changed); sums taken in turn made
// no difference.  Looking for dims that FP16 tiles would lose costs FP32 pages up to 5% (32 rows after 8000, hd 128: 58 -> 61 us); flags of
// every row's dims instead of the first rows' took 3 to 26%.
//
// Masked positions: scores -inf; rows past the last position or without a page are staged as zeros.  Pairs whose
// sums come out infinite or NaN are computed again by wave_attend, which reads only what each row sees.
#pragma once

#include "attn_core.h"

namespace efh {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4v* lds_s4v;

constexpr int kTileWaves = 4, kTileThreads = kTileWaves * kWave;

template <class T>
__device__ __forceinline__ f16v mfma32(u4v a, u4v b, f16v c) {
  if constexpr (std::is_same_v<T, _Float16>)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}

__device__ __forceinline__ float half_max(float v) {  // over lanes l and l + 32
  const u2v b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const u2v b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Tiles have places: request r's are floor(start[r] f / d) + r on (f / d tiles to a row), at least as many as it needs,
// without a sum over the requests before it.  Whose a place is, by a whole wave (64 requests in one round of loads), with
// the request's first row and the next one's.
struct Found {
  int req, first, next;
  long tile;  // the place's number among the request's
};
__device__ __forceinline__ long place_of(int start, int r, int f, int d) { return static_cast<long>(start) * f / d + r; }
__device__ __forceinline__ Found find_request(const int32_t* row_start, int n_seqs, int f, int d, long place) {
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0, len = n_seqs;
  for (;;) {
    const int step = (len + kWave - 1) / kWave, i = lane * step;
    const int start = row_start[min(lo + i, n_seqs)];
    const uint64_t below = __ballot(i < len && place_of(start, lo + i, f, d) <= place);
    const int at = last_lane(below);  // places in front of the first request's: a negative tile of that one
    if (step == 1) {
      const int req = __builtin_amdgcn_readfirstlane(lo + at);
      Found r{req, __builtin_amdgcn_readlane(start, at), 0, 0};
      r.next = at < kWave - 1 ? __builtin_amdgcn_readlane(start, at + 1) : row_start[req + 1];
      r.tile = place - place_of(r.first, req, f, d);
      return r;
    }
    lo += at * step;
    len = min(step, len - at * step);
  }
}

// Where a tile's keys and values come from.
enum Source {
  kPages,     // a request's pages, in their own type
  kRows,      // packed rows, in their own type
  kPrepared,  // packed FP32 or BF16 rows brought to FP16 by attention_prepare_kernel
};

// Heads of up to HC dims (64, 96, 128, 256), in rows of a power of two.
constexpr int row_width(int HC) { return HC == 96 ? 128 : HC; }

template <class T, int HC, int SRC>
struct TileShape {
  static constexpr int HDP = row_width(HC);
  static constexpr bool F32 = sizeof(T) == 4, PREPARED = SRC == kPrepared;
  static constexpr int BN = HDP == 256 || (F32 && HDP >= 128) ? 32 : 64;  // positions of a tile
  static constexpr int PLANES = F32 ? 2 : 1;                              // 16-bit planes of a key or value
  static constexpr int CHUNKS = HDP / 8;                                  // 16-byte chunks of a row
  static constexpr int PLANE = BN * HDP;                                  // 16-bit values of a plane
  static constexpr int BUFFERS = F32 && !PREPARED ? 1 : 2;
  static constexpr int UNITS = PLANE / 8 / kTileThreads;                  // chunks that a thread brings of a plane
};

// Rows lie in LDS without padding (a DMA instruction writes 1 KB in one piece), their 16-byte chunks in another order in
// each row, so that what one LDS cycle serves hits all 64 banks: sixteen lanes that read a chunk of sixteen rows
// (keys), and 32 that read 64 bytes of four rows (values).  Rows of 128 bytes are half the banks wide.
template <int CHUNKS>
__device__ __forceinline__ int k_place(int chunk, int row) {
  return chunk ^ (CHUNKS == 8 ? row >> 1 & 7 : row & (CHUNKS == 16 ? 15 : 7));
}
template <int CHUNKS>
__device__ __forceinline__ int v_place(int chunk, int row) {
  return chunk ^ (CHUNKS == 8 ? (row & 2) << 1 : (row & 3) << 2);
}

// 16 bytes per lane from src to LDS at dst + 16 lane, asynchronously (vmcnt).  As asm because the compiler, seeing
// such a copy, waits for it before every later LDS read; the kernel waits for its tiles itself.  No register is
// written but m0, which the compiler sets anew before each use.
__device__ __forceinline__ void tile_dma16(uint32_t dst, const void* src) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
}
// This wave's copies arrived and its LDS accesses done, then the barrier.
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr int kNoTile = INT32_MIN, kAnyScale = INT32_MAX;

// A tile's exponents, and what the largest value of each of its dims has to reach, from the bits of the largest
// magnitude of its keys and of its values and of the smallest among its rows' largest magnitudes (rows of zeros left
// out).  Keys are brought to 2^14 .. 2^15 (c2 takes each tile's scale back), values to 2^13 .. 2^15, so that neighbouring tiles
// mostly share a scale and the sums keep theirs.
//   What the halves drop of a value is 2^-25 at most or 2^-22 of it: below 2^-24 of (its row's largest) (its dim's largest) /
//   (the tile's largest) as long as that is 1/2 or more for each row and dim.  The tile's largest is below 2^(M + 1), the rows' are
//   2^L or more: a dim's largest has to reach 2^(M - L) (all of them scaled).  Dims of zeros are left out.
struct TileScales {
  int2 e;
  float k_dim, v_dim;
};
__device__ __forceinline__ TileScales tile_scales(uint32_t k_most, uint32_t k_least, uint32_t v_most, uint32_t v_least) {
  auto lead = [](uint32_t most, uint32_t least) {  // subnormal rows: the tile is marked
    return most == 0 ? 0 : least < 0x00800000u ? 15 : static_cast<int>(most >> 23) - static_cast<int>(least >> 23);
  };
  const int lk = lead(k_most, k_least), lv = lead(v_most, v_least);
  const int ek = k_most == 0 ? kAnyScale : 14 + 127 - static_cast<int>(k_most >> 23);
  const int ev = v_most == 0 ? kAnyScale : (14 + 127 - static_cast<int>(v_most >> 23)) & ~1;
  const bool marked = k_most >= 0x7F800000u || v_most >= 0x7F800000u || max(lk, lv) > 14;  // 2^15: no dim would reach it
  return {marked ? int2{kNoTile, kNoTile} : int2{ek, ev}, ldexpf(1.0f, lk - ek), ldexpf(1.0f, lv - ev)};
}

// A thread's 8 dims of a tile's keys or values, over its rows: which hold something else than zero (the low byte), and which a
// value that is large enough (the next one).  The words of all threads of the same dims are joined by OR.
template <class F>
__device__ __forceinline__ uint32_t dim_flags(float least, F&& largest_of) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float most = largest_of(i);
    w |= (most > 0.0f ? 1u << i : 0u) | (most >= least ? 256u << i : 0u);
  }
  return w;
}
// The same in short: a bit for each dim whose value in one row is large enough, put behind those of w.
template <class F>
__device__ __forceinline__ uint32_t large_dims(uint32_t w, float least, F&& value_of) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w = __builtin_amdgcn_alignbit(w, __float_as_uint(least - fabsf(value_of(i))), 31);
  return w;
}
// Whether the joined words of keys (low half) and values have a dim that is neither zero nor large enough.
__device__ __forceinline__ bool dim_too_small(uint32_t w) { return w & ~(w >> 8) & 0x00FF00FFu; }

struct PrepareArgs {
  KvSource kv;
  const int32_t* row_start;
  int n_seqs, max_rows, hd, places;
  uint16_t* blocks;  // [KV][places][2][PLANES][BN][HDP]
  int2* info;        // [KV][places]: exponents of K and V (kNoTile: marked; kAnyScale: all zero)
};

template <class T, int HC, int SRC>
struct TileLds {
  using Sh = TileShape<T, HC, SRC>;
  uint16_t ks[Sh::BUFFERS][Sh::PLANES * Sh::PLANE];
  uint16_t vs[Sh::BUFFERS][Sh::PLANES * Sh::PLANE];
  uint32_t ok[2][Sh::BN / 4];  // a byte per position: whether a page holds it
  int lost;                    // some tile so far had a position without a page
  u4v sizes[2][kTileWaves];    // FP32: each wave's largest and smallest rows of the tile
  uint32_t large[2][Sh::CHUNKS];  // FP32: the tile's large_dims, and its dim_flags
  uint32_t dims[Sh::CHUNKS];
};

// One workgroup: the place `place` of KV head `kvh`, range `split`.
template <class T, int HC, int SRC>
__device__ __forceinline__ void attention_tiles(const AttnTask& t, const PrepareArgs& pre, TileLds<T, HC, SRC>& lds, int kvh, long place,
                                                int split) {
  using Sh = TileShape<T, HC, SRC>;
  constexpr int HDP = Sh::HDP;
  using C = std::conditional_t<SRC == kPrepared || sizeof(T) == 4, _Float16, T>;  // what the products are in
  // F32: tiles go through registers, where they are scaled and split; SCALED: their values are times a power of two
  constexpr bool PAGED = SRC == kPages, PREPARED = SRC == kPrepared, F32 = Sh::F32 && !PREPARED, SCALED = F32 || PREPARED;
  constexpr int BN = Sh::BN, SUB = BN / 32, PLANES = Sh::PLANES, CHUNKS = Sh::CHUNKS, PLANE = Sh::PLANE, UNITS = Sh::UNITS;
  constexpr int KK = HC / 16, DT = HC / 32, NS = Parts<C>::N;
  constexpr float OFFSET = Parts<C>::kSubOffset, SLACK = Parts<C>::kSubSlack;
  auto &ks = lds.ks, &vs = lds.vs;
  auto& ok_s = lds.ok;
  int& lost_s = lds.lost;

  const RowsArgs& a = t.r;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
  const int col = lane & 31, h = lane >> 5;
  const int G = t.group, hd = a.hd;
  const Found who = find_request(a.row_start, a.n_seqs, G, kTilePairs, place);
  const int req = who.req, first = max(who.first, 0), n = min(who.next, a.max_rows) - first;
  const long tile = who.tile;
  if (n <= 0 || tile < 0 || tile * kTilePairs >= static_cast<long>(n) * G || static_cast<long>(n) * G <= t.few_most) return;
  int before, kv;
  long base;
  if constexpr (PAGED) {
    const int kv_len = a.kv_len[req];
    kv = static_cast<int>(min(static_cast<long>(kv_len), a.kv.table_ld << a.kv.page_shift));
    before = kv_len - (who.next - first);  // rows cut by max_rows count
    base = req * a.kv.table_ld;
  } else {
    kv = n;
    before = 0;
    base = first;
  }
  const int ns = splits_of(kv, t.tile_split);
  if (split >= ns) return;

  // ---- this lane's pair --------------------------------------------------------------------------------
  const int pairs = n * G;  // above few_most, and below 2^31 (checked on the host)
  const int pair0 = static_cast<int>(tile) * kTilePairs, pair = pair0 + 32 * wave + col;
  const bool active = pair < pairs;
  const int row = active ? t.row_of(pair) : 0, head = kvh * G + (active ? pair - row * G : 0);
  const int seen = active ? min(before + row + 1, kv) : 0;
  const int tile_last = min(pair0 + kTilePairs, pairs) - 1;
  // positions: those of the split that the tile's last row sees
  const int j0 = split * t.tile_split.span;
  const int j1 = min(split == t.tile_split.splits - 1 ? kv : min(kv, j0 + t.tile_split.span), min(before + t.row_of(tile_last) + 1, kv));
  const bool busy = pair0 + 32 * wave < pairs;  // a wave without a pair only stages
  const int all_see = min(before + t.row_of(pair0 + 32 * wave) + 1, kv);  // positions that every row of the wave sees

  // ---- bringing tiles ------------------------------------------------------------------------------------
  // Unit u of a thread: the chunk at place (tid % CHUNKS) of row tid / CHUNKS + u * 256 / CHUNKS.  16-bit tiles go to
  // LDS by DMA, a tile ahead, in two buffers; FP32 ones through registers, where they are split.  Rows past j1
  // repeat the last one, rows without a page the pool's first, dims past hd the row's last ones: all are masked
  // or multiplied by zero.
  constexpr int ROWS = kTileThreads / CHUNKS, WORDS = F32 ? 2 : 1;
  const int my_place = tid % CHUNKS, my_row = tid / CHUNKS;
  const int k_col = min(8 * k_place<CHUNKS>(my_place, my_row), hd - 8), v_col = min(8 * v_place<CHUNKS>(my_place, my_row), hd - 8);
  const T *kp = static_cast<const T*>(a.kv.k) + k_col, *vp = static_cast<const T*>(a.kv.v) + (F32 ? k_col : v_col);
  static_assert(ROWS % (CHUNKS == 32 ? 8 : 16) == 0, "a thread's rows share their places");
  int page[UNITS];  // of the next tile's rows
  auto look_up = [&](int c) {
    if constexpr (PAGED) {
#pragma unroll
      for (int u = 0; u < UNITS; ++u) page[u] = a.kv.table[base + (min(c + my_row + u * ROWS, j1 - 1) >> a.kv.page_shift)];
    }
  };
  u4v kr[F32 ? UNITS : 1][WORDS], vr[F32 ? UNITS : 1][WORDS];
  uint32_t real_rows = 0;  // FP32: units whose row has a page
  const uint32_t k_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)ks)) + 1024 * wave;
  const uint32_t v_lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void*)vs)) + 1024 * wave;
  int2 info = {0, 0};  // of the tile brought last
  auto bring = [&](int c, int buf, int ok_buf) {
    real_rows = 0;
    if constexpr (PREPARED) {
      const long at = kvh * static_cast<long>(pre.places) + place_of(first, req, 1, BN) + c / BN;
      const uint16_t* block = pre.blocks + at * (2 * PLANES * PLANE) + 8 * tid;
      info = pre.info[at];
#pragma unroll
      for (int u = 0; u < PLANES * UNITS; ++u) {
        tile_dma16(k_lds + (buf * PLANES * PLANE + u * 8 * kTileThreads) * 2, block + u * 8 * kTileThreads);
        tile_dma16(v_lds + (buf * PLANES * PLANE + u * 8 * kTileThreads) * 2, block + PLANES * PLANE + u * 8 * kTileThreads);
      }
      return;
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int r = my_row + u * ROWS, j = min(c + r, j1 - 1);
      long ko, vo;
      if constexpr (PAGED) {
        const bool real = static_cast<uint32_t>(page[u]) < static_cast<uint32_t>(a.kv.n_pages);
        ko = vo = real ? page[u] * a.kv.page_stride + ((static_cast<long>(kvh) << a.kv.page_shift) + (j & ((1 << a.kv.page_shift) - 1))) * hd : 0;
        if (my_place == 0) {
          reinterpret_cast<uint8_t*>(ok_s[ok_buf])[r] = real;
          if (!real) lost_s = 1;
        }
        real_rows |= real ? 1u << u : 0u;
      } else {
        real_rows |= 1u << u;
        ko = (base + j) * a.kv.ldk + static_cast<long>(kvh) * hd;
        vo = (base + j) * a.kv.ldv + static_cast<long>(kvh) * hd;
      }
      if constexpr (F32) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
          kr[u][w] = *reinterpret_cast<const u4v*>(kp + ko + 4 * w);
          vr[u][w] = *reinterpret_cast<const u4v*>(vp + vo + 4 * w);
        }
      } else {
        tile_dma16(k_lds + (buf * PLANE + u * 8 * kTileThreads) * 2, kp + ko);
        tile_dma16(v_lds + (buf * PLANE + u * 8 * kTileThreads) * 2, vp + vo);
      }
    }
  };
  // FP32: the sizes of the tile's rows (as bits: infinities and NaN are the largest), then, behind a barrier, its scales,
  // and the tile into LDS as rounded halves and what they left.
  auto measure = [&](int slot) {
    if constexpr (F32) {
      u4v found;
      if constexpr (PAGED) {  // rows without a page are zeros
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
          if (!(real_rows >> u & 1)) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) kr[u][w] = vr[u][w] = u4v{0, 0, 0, 0};
          }
      }
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint32_t most = 0, least = 0;  // least: of the complements of rows that are not zero
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const u4v(&x)[WORDS] = which ? vr[u] : kr[u];
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) top = max(top, x[i / 4][i % 4] & 0x7FFFFFFFu);
          top = max(top, dpp_self_u<0xB1>(top));
          top = max(top, dpp_self_u<0x4E>(top));
          top = max(top, dpp_self_u<0x141>(top));
          if constexpr (CHUNKS >= 16) top = max(top, dpp_self_u<0x140>(top));
          if constexpr (CHUNKS >= 32) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, kWave)));
          most = max(most, top);
          least = max(least, top ? ~top : 0u);
        }
        found[2 * which] = wave_max_u32_dpp(most);
        found[2 * which + 1] = wave_max_u32_dpp(least);
      }
      if (lane == 0) lds.sizes[slot][wave] = found;
    }
  };
  auto scales = [&](int slot) {
    u4v m = lds.sizes[slot][0];
#pragma unroll
    for (int w = 1; w < kTileWaves; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = max(m[i], lds.sizes[slot][w][i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = __builtin_amdgcn_readfirstlane(m[i]);
    return tile_scales(m[0], ~m[1], m[2], ~m[3]);
  };
  auto put = [&](const TileScales& sc, int slot) {
    if constexpr (F32) {
      const int chunk = k_place<CHUNKS>(my_place, my_row);
      uint32_t large = 0;  // in the first unit's rows: hardly ever less than all of them
#pragma unroll
      for (int which = 0; which < 2; ++which)
        large = large_dims(large, which ? sc.v_dim : sc.k_dim, [&](int i) { return __uint_as_float((which ? vr[0] : kr[0])[i / 4][i % 4]); });
      atomicOr(&lds.large[slot][chunk], large);
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const int own = which ? sc.e.y : sc.e.x, e = own == kAnyScale ? 0 : own;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const u4v(&x)[WORDS] = which ? vr[u] : kr[u];
          const int r = my_row + u * ROWS;
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = ldexpf(__uint_as_float(x[i / 4][i % 4]), e);
          u4v part[2];
          split8<_Float16>(f, part);
          uint16_t* dst = which ? vs[0] + r * HDP + 8 * v_place<CHUNKS>(chunk, r) : ks[0] + r * HDP + 8 * k_place<CHUNKS>(chunk, r);
#pragma unroll
          for (int p = 0; p < 2; ++p) *reinterpret_cast<u4v*>(dst + p * PLANE) = part[p];
        }
      }
    }
  };
  // Whether the tile has a dim too small beside the others: the same for every thread, with a barrier in between where the first
  // units do not answer it.
  auto small_dims = [&](const TileScales& sc, int slot) {
    if constexpr (F32) {
      if (!__any(lds.large[slot][lane % CHUNKS] != 0xFFFFu)) return false;
      uint32_t flags = 0;
#pragma unroll
      for (int which = 0; which < 2; ++which)
        flags |= dim_flags(which ? sc.v_dim : sc.k_dim, [&](int i) {
          float most = 0.0f;
#pragma unroll
          for (int u = 0; u < UNITS; ++u) most = fmaxf(most, fabsf(__uint_as_float((which ? vr[u] : kr[u])[i / 4][i % 4])));
          return most;
        }) << 16 * which;
      atomicOr(&lds.dims[k_place<CHUNKS>(my_place, my_row)], flags);
      tile_barrier();
      return static_cast<bool>(__any(dim_too_small(lds.dims[lane % CHUNKS])));
    }
    return false;
  };
  if (tid == 0) lost_s = 0;
  if (F32 && tid < CHUNKS) lds.large[0][tid] = lds.large[1][tid] = lds.dims[tid] = 0;
  __syncthreads();
  // this lane's reads: keys' row col, chunk 2 k + h; values' rows 4 h + lane % 16 / 4, dims 16 (lane / 16 % 2) + 4 (lane % 4)
  const int vq = (lane & 15) / 4, vchunk = 2 * (lane >> 4 & 1) + (lane & 3) / 2;
  const int k_at = col * HDP, v_at = (4 * h + vq) * HDP + 4 * (lane & 1);

  // ---- queries: their loads and the first tile's in flight together ------------------------------------------
  f4v raw[KK][2];
  {
    const float* q = a.q + static_cast<long>(first + row) * a.ldq + static_cast<long>(head) * hd;
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int w = 0; w < 2; ++w) raw[k][w] = *reinterpret_cast<const f4v*>(q + min(16 * k + 8 * h, hd - 8) + 4 * w);
  }
  if (j0 < j1) {
    look_up(j0);
    bring(j0, 0, 0);
    look_up(j0 + BN);
  }
  u4v qp[KK][NS];
  float c2 = a.c2;
  int e = 0;
  {
    float x[KK][8], top = 0.0f;
#pragma unroll
    for (int k = 0; k < KK; ++k)
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        x[k][u] = 16 * k + 8 * h < hd ? raw[k][u / 4][u % 4] : 0.0f;
        top = fmaxf(top, fabsf(x[k][u]));
      }
    if constexpr (std::is_same_v<C, _Float16>) {
      e = query_exponent(half_max(top));
      c2 = ldexpf(c2, -e);
    }
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      if constexpr (std::is_same_v<C, _Float16>) {
#pragma unroll
        for (int u = 0; u < 8; ++u) x[k][u] = ldexpf(x[k][u], e);
      }
      split8<C>(x[k], qp[k]);
    }
  }

  f16v o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float sub = -INFINITY, l = 0.0f;
  int o_scale = kAnyScale;  // o is times 2^o_scale (scaled tiles)
  int usual = kAnyScale;    // the first scaled tile's
  int turn = 0;
  for (int c = j0; c < j1; c += BN) {
    TileScales scaled{};
    if constexpr (F32) {
      measure(turn);
      tile_barrier();  // the tile before is used, and the sizes are there
      scaled = scales(turn);
      info = scaled.e;
      if (tid < CHUNKS) lds.large[turn ^ 1][tid] = lds.dims[tid] = 0;  // read before that barrier
      if (info.x != kNoTile) put(scaled, turn);
    }
    tile_barrier();  // the tile is there, and the buffer of the tile before is free
    if (F32 && info.x != kNoTile && small_dims(scaled, turn)) info = int2{kNoTile, kNoTile};
    const int now = F32 ? 0 : turn, ok_now = turn;
    turn ^= 1;
    const int2 tile_info = info;
    if (c + BN < j1) {
      bring(c + BN, F32 ? 0 : turn, turn);
      look_up(c + 2 * BN);
    }
    if (!busy) continue;
    const uint16_t *kt = ks[now] + k_at, *vt = vs[now] + v_at;
    float c2t = c2;
    if constexpr (SCALED) {
      const int ek = __builtin_amdgcn_readfirstlane(tile_info.x), ev = __builtin_amdgcn_readfirstlane(tile_info.y);
      // A tile whose values are 2^12 and more from the others' in size is taken from its rows too: a weight's parts are held to 2^-38 of
      // the largest, which is 2^-22 of the output at most as long as no value is more than 2^16 times the others.
      const bool plain = ek == kNoTile || (usual != kAnyScale && ev != kAnyScale && abs(ev - usual) > 12);
      if (!plain && usual == kAnyScale) usual = ev;
      const int to = plain ? 0 : ev == kAnyScale ? o_scale : ev;
      if (to != o_scale) {
        if (o_scale != kAnyScale) {
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = ldexpf(o[d][i], to - o_scale);
        }
        o_scale = to;
      }
      if (plain) {
        // Position by position in FP32, from the rows: both lanes of a pair form its score, each half of the dims.
        const float* q = a.q + static_cast<long>(first + row) * a.ldq + static_cast<long>(head) * hd;
#pragma unroll 1
        for (int j = c; j < min(c + BN, j1); ++j) {
          long ko, vo;
          if (!kv_offset<PAGED>(a.kv, kvh, hd, base, j, &ko, &vo)) continue;
          const T *kj = static_cast<const T*>(a.kv.k) + ko, *vj = static_cast<const T*>(a.kv.v) + vo;
          float part[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
          for (int d = 8 * h; d < hd; d += 16) {
            float x[8], y[8];
            load8(q + d, x);
            load8(kj + d, y);
#pragma unroll
            for (int u = 0; u < 8; ++u) part[u] = fmaf(x[u], y[u], part[u]);
          }
          const float s = half_sum(((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7])));
          const bool sees = j < seen;
          const float high = sees ? s * a.c2 - OFFSET : -INFINITY;
          if (__any(high > sub + SLACK)) {
            const float up = fmaxf(sub, high), al = up == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sub - up);
            sub = up;
            l *= al;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= al;
          }
          if (sees) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s, a.c2, -(sub == -INFINITY ? 0.0f : sub)));
            if (h == 0) l += p;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
              for (int g = 0; g < 4; ++g) {  // dims past hd: the row's last ones, not used
                const T* at = vj + min(32 * d + 8 * g + 4 * h, hd - 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][4 * g + i] = fmaf(p, static_cast<float>(at[i]), o[d][4 * g + i]);
              }
          }
        }
        continue;
      }
      c2t = ldexpf(a.c2, -e - (ek == kAnyScale ? 0 : ek));
    }

    f16v sc[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[s][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < KK; ++k) {
      u4v kf[SUB][PLANES];
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
          kf[s][p] = *reinterpret_cast<const u4v*>(kt + p * PLANE + 32 * s * HDP + 8 * k_place<CHUNKS>(2 * k + h, col));
#pragma unroll
      for (int sum = NS - 1; sum >= 0; --sum)  // the small products first; the sums in turn, as each waits for itself
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
#pragma unroll
          for (int s = 0; s < SUB; ++s)
            if (sum - p >= 0) sc[s] = mfma32<C>(kf[s][p], qp[k][sum - p], sc[s]);
    }
    if (c + BN > all_see) {
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + 32 * s + 8 * (i / 4) + 4 * h + i % 4 >= seen) sc[s][i] = -INFINITY;
    }
    if constexpr (PAGED) {
      if (lost_s) {
#pragma unroll
        for (int s = 0; s < SUB; ++s)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t w = ok_s[ok_now][8 * s + 2 * q + h];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!(w >> (8 * i) & 255)) sc[s][4 * q + i] = -INFINITY;
          }
      }
    }
    float cm = -INFINITY;
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) cm = fmaxf(cm, sc[s][i]);
    const float high = half_max(cm) * c2t - OFFSET;
    if (__any(high > sub + SLACK)) {
      const float to = fmaxf(sub, high);
      const float al = to == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sub - to);
      sub = to;
      l *= al;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= al;
    }
    const float from = sub == -INFINITY ? 0.0f : sub;
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // 16 positions: one step of the products
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(sc[s][8 * half + i], c2t, -from));
          sum += p[i];
        }
        u4v pp[NS];
        split8<C>(p, pp);
        constexpr int TURN = DT < 4 ? DT : 4;  // sums taken in turn
#pragma unroll
        for (int d0 = 0; d0 < DT; d0 += TURN) {
          u4v vf[TURN][PLANES];
#pragma unroll
          for (int d = 0; d < TURN; ++d)
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl) {
              uint16_t* at = const_cast<uint16_t*>(vt) + pl * PLANE + (32 * s + 16 * half) * HDP + 8 * v_place<CHUNKS>(4 * (d0 + d) + vchunk, vq);
              const s4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v)at);
              const s4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v)(at + 8 * HDP));
              const u2v lw = __builtin_bit_cast(u2v, lo), hw = __builtin_bit_cast(u2v, hi);
              vf[d][pl] = u4v{lw[0], lw[1], hw[0], hw[1]};
            }
#pragma unroll
          for (int ps = NS - 1; ps >= 0; --ps)
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl)
#pragma unroll
              for (int d = 0; d < TURN; ++d)
                if (ps - pl >= 0) o[d0 + d] = mfma32<C>(vf[d][pl], pp[ps - pl], o[d0 + d]);
        }
      }
    }
    l += sum;
  }

  // ---- results ---------------------------------------------------------------------------------------------
  l = half_sum(l);
  if constexpr (SCALED) {
    if (o_scale != kAnyScale && o_scale != 0) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = ldexpf(o[d][i], -o_scale);
    }
  }
  bool bad = !(fabsf(l) < INFINITY);
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) bad = bad || !(fabsf(o[d][i]) < INFINITY);
  const bool direct = ns == 1;
  const long out_row = static_cast<long>(first + row) * a.ldo + static_cast<long>(head) * hd;
  const long part_row = (static_cast<long>(split) * a.max_rows + first + row) * a.H + head;
  if (active) {
    const float inv = direct ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
    float* dst = direct ? a.out + out_row : t.part + part_row * hd;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int dim = 32 * d + 8 * q + 4 * h;
        if (dim < hd) *reinterpret_cast<f4v*>(dst + dim) = f4v{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]} * inv;
      }
    if (!direct && h == 0) t.stat[part_row] = f2v{sub, l};
    if (split == 0 && h == 0 && t.count != nullptr) t.count[static_cast<long>(first + row) * a.H + head] = ns;
  }
  uint64_t todo = __ballot(bad && active);
  todo = (todo | todo >> 32) & 0xFFFFFFFFull;
  tile_barrier();  // the last tile is used
  float* qs = reinterpret_cast<float*>(ks[0]) + wave * HDP;
  for (; todo; todo &= todo - 1) {
    const int who = __ffsll(static_cast<unsigned long long>(todo)) - 1;
    const int rr = __shfl(row, who, kWave), hh = __shfl(head, who, kWave), lim = min(j1, __shfl(seen, who, kWave));
    const float* q = a.q + static_cast<long>(first + rr) * a.ldq + static_cast<long>(hh) * hd;
    for (int d = lane; d < hd; d += kWave) qs[d] = q[d];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float sb = -INFINITY, ov[4] = {0, 0, 0, 0};
    double ll = 0.0;
    wave_attend<T, PAGED>(a.kv, kvh, hd, base, qs, a.c2, j0, lim, kv, &sb, &ll, ov);
    ll = wave_sum_d_dpp(ll);
    const float inv = ll == 0.0 ? 0.0f : static_cast<float>(1.0 / ll);
    const long to = direct ? static_cast<long>(first + rr) * a.ldo + static_cast<long>(hh) * hd
                           : (static_cast<long>(split) * a.max_rows + first + rr) * a.H + hh;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int d = lane + 64 * u;
      if (d >= hd) continue;
      if (direct) a.out[to + d] = ov[u] * inv;
      else t.part[to * hd + d] = ov[u];
    }
    if (!direct && lane == 0) t.stat[to] = f2v{sb, static_cast<float>(ll)};
    __builtin_amdgcn_wave_barrier();
  }
}

// Places of the tiles of t's rows.
inline size_t tile_places(const AttnTask& t) {
  return (static_cast<size_t>(t.r.max_rows) * t.group + kTilePairs - 1) / kTilePairs + t.r.n_seqs;
}
// Workgroups of a CU at the kernel's registers and LDS.
template <class T, int HC>
constexpr int tile_occupancy() { return HC == 64 && sizeof(T) == 2 ? 3 : HC <= 128 ? 2 : 1; }

}  // namespace efh
