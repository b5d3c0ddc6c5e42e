// Attention of requests with few and with many new rows over pages, in one launch: a step of a server that decodes some
// requests while it brings in the prompts of others.  The many-row workgroups come first, the few-row ones fill the CUs
// that they leave.  39 decodes and two chunks of up to 300 rows at 850 to 1700 positions, BF16, with the join: 53.4 us in two
// launches, 39.4 in one.
#include "attn_few.h"
#include "attn_tiles.h"

namespace efh {
namespace {

static_assert(kFewWaves * kWave == kTileThreads, "one launch for both");

template <class T, int HC, bool WIDE>
__global__ __launch_bounds__(kTileThreads, (tile_occupancy<T, HC>())) void attention_mixed_kernel(AttnTask t, unsigned tile_blocks, int places) {
  constexpr int NT = 1, HDP = row_width(HC);
  __shared__ __attribute__((aligned(1024))) union {
    TileLds<T, HC, kPages> tiles;
    FewLds<HDP, NT> few;
  } lds;
  unsigned id = blockIdx.x;
  const int KV = t.r.KV;
  if (id < tile_blocks) {
    const int split = id / (static_cast<unsigned>(places) * KV);
    id -= static_cast<unsigned>(split) * places * KV;
    const PrepareArgs none{};
    attention_tiles<T, HC, kPages>(t, none, lds.tiles, id % KV, places - 1 - static_cast<long>(id / KV), split);
    return;
  }
  id -= tile_blocks;
  const unsigned per = static_cast<unsigned>(t.r.n_seqs) * KV, rest = id / per;  // requests first, then heads, row tiles, ranges
  id -= rest * per;
  const int split = rest / t.tiles;
  attention_few<T, HDP, NT, WIDE>(t, lds.few, id % t.r.n_seqs, id / t.r.n_seqs, split, rest - split * t.tiles);
}

template <class T, int HC>
void run_mixed(const AttnTask& t, hipStream_t s) {
  const size_t places = tile_places(t), tile_blocks = places * t.r.KV * t.tile_split.splits;
  const unsigned blocks = static_cast<unsigned>(tile_blocks + static_cast<size_t>(t.r.n_seqs) * t.r.KV * t.tiles * t.few_split.splits);
  if (t.r.kv.page_shift >= 4)
    attention_mixed_kernel<T, HC, true><<<blocks, kTileThreads, 0, s>>>(t, static_cast<unsigned>(tile_blocks), static_cast<int>(places));
  else
    attention_mixed_kernel<T, HC, false><<<blocks, kTileThreads, 0, s>>>(t, static_cast<unsigned>(tile_blocks), static_cast<int>(places));
}

template <class T>
void run_mixed_of(const AttnTask& t, hipStream_t s) {
  if (t.r.hd <= 64) run_mixed<T, 64>(t, s);
  else if (t.r.hd <= 96) run_mixed<T, 96>(t, s);
  else if (t.r.hd <= 128) run_mixed<T, 128>(t, s);
  else run_mixed<T, 256>(t, s);
}

}  // namespace

int launch_attention_mixed(const AttnTask& t, int qtype, hipStream_t s) {
  if (qtype == EF_QTYPE_F32) run_mixed_of<float>(t, s);
  else if (qtype == EF_QTYPE_F16) run_mixed_of<_Float16>(t, s);
  else run_mixed_of<__bf16>(t, s);
  EFH_HIP(hipGetLastError());
  return EF_HIP_OK;
}

}  // namespace efh
