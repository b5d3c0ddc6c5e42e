// Where the kernels of paged serving look for a position, on the CPU: page numbers outside the pool give no
// address, every other address stays inside it, and rows find their requests.
#include <cstdio>
#include <random>
#include <vector>

#include "paging.h"

using namespace efh;

int main() {
  std::mt19937 rng(11);
  int bad = 0, checked = 0;
  for (int round = 0; round < 200; ++round) {
    const int shift = rng() % 11, KV = 1 + rng() % 8, hd = 8 * (1 + rng() % 32), n_pages = 1 + rng() % 50, ld = 1 + rng() % 20;
    const long stride = (static_cast<long>(KV) << shift) * hd + 8 * (rng() % 3);
    std::vector<int32_t> table(3 * ld);
    for (auto& t : table) t = static_cast<int32_t>(rng() % (n_pages + 6)) - 3;
    table[rng() % table.size()] = 0x7FFFFFFF;
    table[rng() % table.size()] = static_cast<int32_t>(0x80000000u);
    const KvSource s{nullptr, nullptr, 0, 0, table.data(), ld, stride, shift, n_pages};
    for (int r = 0; r < 3; ++r) {
      for (int i = 0; i < 40; ++i) {
        const int j = i == 0 ? (ld << shift) - 1 : static_cast<int>(rng() % (ld << shift)), g = rng() % KV;
        long ko = -1, vo = -1;
        const bool seen = kv_offset<true>(s, g, hd, static_cast<long>(r) * ld, j, &ko, &vo);
        const int page = table[r * ld + (j >> shift)];
        const bool real = page >= 0 && page < n_pages;
        const long want = real ? page * stride + ((static_cast<long>(g) << shift) + (j & ((1 << shift) - 1))) * hd : -1;
        ++checked;
        if (seen != real || ko != want || vo != want || (real && (ko < 0 || ko + hd > n_pages * stride))) ++bad;
      }
    }
  }
  {  // offsets past 32 bits
    const int32_t table[1] = {1000000};
    const KvSource s{nullptr, nullptr, 0, 0, table, 1, 65536, 6, 1000001};
    long ko = 0, vo = 0;
    if (!kv_offset<true>(s, 3, 128, 0, 63, &ko, &vo) || ko != 1000000L * 65536 + (3 * 64 + 63) * 128) ++bad;
    const KvSource p{nullptr, nullptr, 1 << 20, 1 << 19, nullptr, 0, 0, 0, 0};
    if (!kv_offset<false>(p, 1, 64, 5000, 3, &ko, &vo) || ko != 5003L * (1 << 20) + 64 || vo != 5003L * (1 << 19) + 64) ++bad;
  }
  for (int round = 0; round < 200; ++round) {
    const int n = 1 + rng() % 70;
    std::vector<int> start(n + 1, 0), of;
    for (int r = 0; r < n; ++r) {
      const int rows = rng() % 3 == 0 ? 0 : rng() % 5;
      start[r + 1] = start[r] + rows;
      of.insert(of.end(), rows, r);
    }
    for (size_t i = 0; i < of.size(); ++i, ++checked) bad += request_of(start.data(), n, static_cast<int>(i)) != of[i];
  }
  std::printf("%d checked, %d wrong\n", checked, bad);
  return bad ? 1 : 0;
}
