// Attention of many new rows (attn_tiles.h), and the FP16 tiles of packed FP32 and BF16 rows.
#include "attn_tiles.h"

namespace efh {
namespace {

// ---- packed FP32 and BF16 rows as FP16 ---------------------------------------------------------------------
// A tile of BN rows of one KV head times a power of two (tile_scales): FP32 as two planes, the rounded half and what it
// left, BF16 as one.  Tiles with a row or a dim too small for that beside the others, or with infinities or NaN, are marked;
// the attention kernel takes them from the rows themselves.  Three products (high high, high low, low high) serve
// FP32, two serve BF16, where its rows as they are take three.  The tile is written
// as the kernel's LDS holds it: planes of K, planes of V.
// Read and written once, in one pass: bound by memory and the launch (6001 rows of 4 heads of 64, 12 + 12 MB: 10 to 12 us).
template <class T, int HDP>
__global__ __launch_bounds__(kTileThreads) void attention_prepare_kernel(PrepareArgs a) {
  using Sh = TileShape<T, HDP, kPrepared>;
  constexpr int BN = Sh::BN, CHUNKS = Sh::CHUNKS, UNITS = Sh::UNITS, PLANES = Sh::PLANES, PLANE = Sh::PLANE, ROWS = kTileThreads / CHUNKS;
  __shared__ uint32_t most_s[2], least_s[2], dims_s[CHUNKS];
  const int tid = threadIdx.x, kvh = blockIdx.y, chunk = tid % CHUNKS, my_row = tid / CHUNKS;
  const long place = blockIdx.x;
  const Found who = find_request(a.row_start, a.n_seqs, 1, BN, place);
  const int first = max(who.first, 0), n = min(who.next, a.max_rows) - first;
  const long c = who.tile * BN;
  if (n <= 0 || c < 0 || c >= n) return;
  if (tid < 2) {
    most_s[tid] = 0;
    least_s[tid] = 0xFFFFFFFFu;
  }
  if (tid < CHUNKS) dims_s[tid] = 0;
  float x[2][UNITS][8];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int r = my_row + u * ROWS;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[kv][u][i] = 0.0f;
      if (c + r < n && 8 * chunk < a.hd)
        load8(static_cast<const T*>(kv ? a.kv.v : a.kv.k) + (first + c + r) * (kv ? a.kv.ldv : a.kv.ldk) + static_cast<long>(kvh) * a.hd + 8 * chunk, x[kv][u]);
    }
  __syncthreads();
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t most = 0, least = 0xFFFFFFFFu;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      uint32_t top = 0;  // the row's largest magnitude, as bits (infinities and NaN are the largest)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[kv][u][i]) & 0x7FFFFFFFu);
#pragma unroll
      for (int o = 1; o < CHUNKS; o <<= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), o, kWave)));
      most = max(most, top);
      if (top) least = min(least, top);
    }
#pragma unroll
    for (int o = CHUNKS; o < kWave; o <<= 1) {
      most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o, kWave)));
      least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), o, kWave)));
    }
    if ((tid & (kWave - 1)) == 0) {
      atomicMax(&most_s[kv], most);
      atomicMin(&least_s[kv], least);
    }
  }
  __syncthreads();
  const TileScales sc = tile_scales(most_s[0], least_s[0], most_s[1], least_s[1]);
  const long at = kvh * static_cast<long>(a.places) + place;
  uint32_t flags = 0;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv)
    flags |= dim_flags(kv ? sc.v_dim : sc.k_dim, [&](int i) {
      float most = 0.0f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) most = fmaxf(most, fabsf(x[kv][u][i]));
      return most;
    }) << 16 * kv;
  atomicOr(&dims_s[chunk], flags);
  __syncthreads();
  const bool marked = sc.e.x == kNoTile || __any(dim_too_small(dims_s[(tid & (kWave - 1)) % CHUNKS]));
  if (tid == 0) a.info[at] = marked ? int2{kNoTile, kNoTile} : sc.e;
  if (marked) return;
  uint16_t* block = a.blocks + at * (2 * PLANES * PLANE);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const int own = kv ? sc.e.y : sc.e.x, scale = own == kAnyScale ? 0 : own;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int r = my_row + u * ROWS;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[kv][u][i] = ldexpf(x[kv][u][i], scale);
      u4v part[2];
      split8<_Float16>(x[kv][u], part);
      uint16_t* dst = block + kv * PLANES * PLANE + r * HDP + 8 * (kv ? v_place<CHUNKS>(chunk, r) : k_place<CHUNKS>(chunk, r));
#pragma unroll
      for (int p = 0; p < PLANES; ++p) *reinterpret_cast<u4v*>(dst + p * PLANE) = part[p];
    }
  }
}

template <class T, int HC, int SRC>
__global__ __launch_bounds__(kTileThreads, (tile_occupancy<T, HC>())) void attention_tiles_kernel(AttnTask t, PrepareArgs pre) {
  __shared__ __attribute__((aligned(1024))) TileLds<T, HC, SRC> lds;
  // the last places first: a request's last rows see the most positions
  const int kvh = blockIdx.x % t.r.KV;
  attention_tiles<T, HC, SRC>(t, pre, lds, kvh, static_cast<long>(gridDim.x / t.r.KV) - 1 - blockIdx.x / t.r.KV, blockIdx.y);
}

template <class T, int HC, int SRC>
void run_tiles(const AttnTask& t, const PrepareArgs& pre, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(tile_places(t) * t.r.KV), t.tile_split.splits);
  if constexpr (SRC == kPrepared) attention_prepare_kernel<T, row_width(HC)><<<dim3(pre.places, t.r.KV), kTileThreads, 0, s>>>(pre);
  attention_tiles_kernel<T, HC, SRC><<<grid, kTileThreads, 0, s>>>(t, pre);
}

template <class T, int SRC>
void run_tiles_of(const AttnTask& t, const PrepareArgs& pre, hipStream_t s) {
  if (t.r.hd <= 64) run_tiles<T, 64, SRC>(t, pre, s);
  else if (t.r.hd <= 96) run_tiles<T, 96, SRC>(t, pre, s);
  else if (t.r.hd <= 128) run_tiles<T, 128, SRC>(t, pre, s);
  else run_tiles<T, 256, SRC>(t, pre, s);
}

// Places of prepared tiles, and the bytes of a tile, for `hd` and `qtype`.
template <class T>
PreparedShape shape_of(size_t hd) {
  auto of = [](auto sh) { return PreparedShape{static_cast<size_t>(sh.BN), static_cast<size_t>(2 * sh.PLANES * sh.PLANE * 2)}; };
  return hd <= 64 ? of(TileShape<T, 64, kPrepared>{}) : hd <= 128 ? of(TileShape<T, 128, kPrepared>{}) : of(TileShape<T, 256, kPrepared>{});
}

}  // namespace

PreparedShape prepared_shape(size_t hd, int qtype) {
  return qtype == EF_QTYPE_F32 ? shape_of<float>(hd) : shape_of<__bf16>(hd);
}

int launch_attention_tiles(const AttnTask& t, int qtype, bool paged, hipStream_t s) {
  const PrepareArgs none{};
  if (qtype == EF_QTYPE_F32) paged ? run_tiles_of<float, kPages>(t, none, s) : run_tiles_of<float, kRows>(t, none, s);
  else if (qtype == EF_QTYPE_F16) paged ? run_tiles_of<_Float16, kPages>(t, none, s) : run_tiles_of<_Float16, kRows>(t, none, s);
  else paged ? run_tiles_of<__bf16, kPages>(t, none, s) : run_tiles_of<__bf16, kRows>(t, none, s);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

int launch_attention_prepared(const AttnTask& t, int qtype, void* ws, size_t places, hipStream_t s) {
  PrepareArgs pre{};
  pre.kv = t.r.kv;
  pre.row_start = t.r.row_start;
  pre.n_seqs = t.r.n_seqs;
  pre.max_rows = t.r.max_rows;
  pre.hd = t.r.hd;
  pre.places = static_cast<int>(places);
  pre.blocks = static_cast<uint16_t*>(ws);
  pre.info = reinterpret_cast<int2*>(static_cast<char*>(ws) + places * t.r.KV * prepared_shape(t.r.hd, qtype).bytes);
  if (qtype == EF_QTYPE_F32) run_tiles_of<float, kPrepared>(t, pre, s);
  else run_tiles_of<__bf16, kPrepared>(t, pre, s);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

}  // namespace efh
