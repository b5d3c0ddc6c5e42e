// What the kernels of attention over pages and packed prompts share (paged_attention.hip, attn_few.hip,
// attn_tiles.hip):
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c2 s_j - sub),  s_j = q . k_j,  c2 = scale log2(e),
// sub the rounded c2 max_j s_j so far (a rescaling is by the difference of two sub, so that it is consistent
// with the terms already summed however large the scores' common part is).
#pragma once

#include "paging.h"

#pragma clang fp contract(off)

namespace efh {

typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

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
// score and dims lane + 64 u of the output.  q is in LDS.  Only seen positions are read, so infinities and NaN elsewhere do not
// matter.  Weights are 2^-room of those of the formula, 2^room being more than twice the request's `kv` positions, so that no
// sum of them times values passes the largest value; sub has the factor.
template <class T, bool PAGED>
__device__ void wave_attend(const KvSource& src, int g, int hd, long base, const float* q, float c2, int j0, int j1, int kv,
                            float* sub, double* l, float (&o)[4]) {
  const int lane = threadIdx.x & (kWave - 1), room = 33 - __clz(max(kv, 1));
  const float weight = ldexpf(1.0f, -room);
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
    const float p = seen ? __builtin_amdgcn_exp2f(fmaf(s, c2, -from)) * weight : 0.0f;
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
  *sub += static_cast<float>(room);
}

// ---- matrix-core operands ------------------------------------------------------------------------------
// FP32 accuracy from 16-bit products: an FP32 operand is split into 16-bit parts whose sum keeps 22 bits or more, and
// the parts' products are summed in FP32 by the matrix cores.
//   FP16 keys and values: 2 parts (11 bits each, both rounded to nearest).  Their small range is met by a power of
//     two: queries are brought to 2^14 .. 2^15 by one that c2 takes back, and p is formed as 2^13 p (the
//     offset stays in sub), so that what the smallest half drops, 2^-25, is below 2^-38 of the largest.
//   BF16: 3 parts (8 bits each, truncated, exact in all 24 bits and FP32's range).
// FP32 keys and values are brought to FP16 by a power of two for a tile and split into 2 parts (attn_tiles.h), or
// multiplied as they are (attn_few.h).
// kSubSlack: a running sub is raised only when a score passes it by this much (in powers of two; the weights then reach 2^8, and
// 2^15 of a half's 2^16 with FP16's offset): with one pass over many positions a new maximum comes often, a much larger one
// hardly ever.
template <class T>
struct Parts;
template <>
struct Parts<float> {
  static constexpr int N = 1;
  static constexpr float kSubOffset = 0.0f, kSubSlack = 8.0f;
};
template <>
struct Parts<_Float16> {
  static constexpr int N = 2;
  static constexpr float kSubOffset = 13.0f, kSubSlack = 2.0f;
  typedef h8v V;
};
template <>
struct Parts<__bf16> {
  static constexpr int N = 3;
  static constexpr float kSubOffset = 0.0f, kSubSlack = 8.0f;
  typedef b8v V;
};

// Two FP32 values' bfloat16 high halves in one word (truncation).
__device__ __forceinline__ uint32_t high_halves(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// x[0..7] as parts: word i of part p holds values 2 i and 2 i + 1.
template <class T>
__device__ __forceinline__ void split8(const float (&x)[8], u4v (&part)[Parts<T>::N]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
    if constexpr (std::is_same_v<T, _Float16>) {
      const uint32_t hi = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v{a, b}), h2v));
      part[0][i] = hi;
      // what the halves left: x - half in one instruction, the half widened on the way (the conversion above has
      // read a and b, so their results are there)
      asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(hi), "v"(a));
      asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(hi), "v"(b));
      part[1][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2v{a, b}), h2v));
    } else {
      part[0][i] = high_halves(a, b);
      a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
      b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
      part[1][i] = high_halves(a, b);
      a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
      b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
      part[2][i] = high_halves(a, b);
    }
  }
}

template <class T>
__device__ __forceinline__ f4v mfma16(u4v a, u4v b, f4v c) {
  if constexpr (std::is_same_v<T, _Float16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}

// Over the lanes that differ in bit 4 and bit 5 (one column of a 16-wide matrix tile).
__device__ __forceinline__ float column_max(float v) {
  const u2v a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const u2v b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
  const u2v a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const u2v b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The power of two that brings a row of FP16 queries whose largest magnitude is `top` to 2^14 .. 2^15 (1 for a row of
// zeros, infinities or NaN), as its exponent.
__device__ __forceinline__ int query_exponent(float top) {
  const int e = static_cast<int>(__float_as_uint(top) >> 23 & 255);
  return top == 0.0f || e == 255 ? 0 : min(141 - e, 127);
}

// ---- the split over positions ----------------------------------------------------------------------------
// A request's positions are cut into `splits` ranges of `span` (the last one takes the rest, whatever the length);
// each range's (sub, l) and unnormalised sums go to the workspace, and attention_join_kernel adds them.
struct Split {
  int splits, span;
};
__host__ __device__ __forceinline__ int splits_of(int kv, Split s) {
  const int need = kv <= 0 ? 1 : (kv - 1) / s.span + 1;
  return need < s.splits ? need : s.splits;
}

struct AttnTask {
  RowsArgs r;
  Split few_split, tile_split;
  float* part;  // [splits][rows * H][hd]
  f2v* stat;    // [splits][rows * H]: sub, l
  int* count;   // [rows * H]: ranges that hold sums (one: the output is already there); null where nothing is split
  int group;       // H / KV
  uint32_t magic;  // ceil(2^32 / group)
  // pair / group: the product's high half is the quotient or one more (its error is below pair group / 2^32 < group)
  __device__ __forceinline__ int row_of(int pair) const {
    if (group == 1) return pair;
    const int q = static_cast<int>(__umulhi(static_cast<uint32_t>(pair), magic));
    return q - (static_cast<int64_t>(q) * group > pair);
  }
  int tiles;     // few-rows kernel: workgroups per (request, KV head) along its rows
  bool few_wide; // few-rows kernel: 32 (row, head) pairs to a workgroup, not 16
  int few_most;  // (row, head) pairs of a KV head up to which a request is the few-rows kernel's, not the tiles kernel's
};

// Positions of a request: the kernels count two steps (of 128 positions at most) past the last in 32 bits.
constexpr size_t kMostPositions = (size_t(1) << 31) - 1024;
// Ranges from which on a (row, head) pair's join has a workgroup of its own, not a wave.
constexpr int kJoinMany = 16;
// (row, head) pairs of a KV head in a workgroup of the tiles kernel
constexpr int kTilePairs = 128;

// Packed FP32 and BF16 rows prepared as FP16 tiles of `rows` rows and `bytes` bytes; the workspace holds KV tiles of
// each of the places (ceil(max_rows / rows) + n_seqs of them), then 8 bytes for each.
struct PreparedShape {
  size_t rows, bytes;
};
PreparedShape prepared_shape(size_t hd, int qtype);
int launch_attention_prepared(const AttnTask& t, int qtype, void* ws, size_t places, hipStream_t s);
int launch_attention_tiles(const AttnTask& t, int qtype, bool paged, hipStream_t s);
// few and tiles in one launch (t.few_wide is not used: 16 pairs to a workgroup)
int launch_attention_mixed(const AttnTask& t, int qtype, hipStream_t s);
int launch_attention_join(const AttnTask& t, hipStream_t s);
int launch_attention_few(const AttnTask& t, int qtype, hipStream_t s);

}  // namespace efh
