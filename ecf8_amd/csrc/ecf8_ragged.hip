// Attention of a ragged batch on gfx950: sequences of different lengths, new
// tokens packed one sequence after the other, keys and values in the pages of
// a cache (bf16 or e4m3) or packed like the queries.  Head dimension 128,
// fp32 scores, softmax statistics and sums.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "ecf8.h"
#include "ecf8_dev.h"
#include "ecf8_draft_layout.h"
#include "ecf8_paged.h"
#include "ecf8_paged_layout.h"

namespace {

using namespace ecf8::paged;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.0e38f;  // stands for the maximum of no keys
constexpr float kNone = -0x1p100f;   // and for the exponents' while all scores are -inf

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// two fp32 -> packed bf16, round to nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const v2bf v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}

// The maximum of the lanes of the same number mod 16.
__device__ __forceinline__ float max_of_groups(float x) {
  uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  u = __float_as_uint(x);
  const auto b = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Eight bf16 with their infinities and NaNs replaced by zeros.  Values of steps
// with masked positions are staged like this: what a masked position holds
// must not enter the sums, not even as 0 x inf.
__device__ __forceinline__ u32x4 finite_or_zero(u32x4 v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if ((v[j] & 0x7f80u) == 0x7f80u) v[j] &= 0xffff0000u;
    if ((v[j] & 0x7f800000u) == 0x7f800000u) v[j] &= 0xffffu;
  }
  return v;
}

__device__ __forceinline__ bool differ(u32x4 a, u32x4 b) {
  return ((a[0] ^ b[0]) | (a[1] ^ b[1]) | (a[2] ^ b[2]) | (a[3] ^ b[3])) != 0;
}

// 16 e4m3 codes -> bf16, exact.
__device__ __forceinline__ void widen16(u32x4 c, u32x4 (&out)[2]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], false);
    const v2f hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[j], true);
    out[j >> 1][2 * (j & 1)] =
        __builtin_amdgcn_perm(__float_as_uint(lo[1]), __float_as_uint(lo[0]), 0x07060302u);
    out[j >> 1][2 * (j & 1) + 1] =
        __builtin_amdgcn_perm(__float_as_uint(hi[1]), __float_as_uint(hi[0]), 0x07060302u);
  }
}

// The same by the conversion that gives bf16 at once: half of the instructions.
__device__ __forceinline__ void widen16_pairs(u32x4 c, u32x4 (&out)[2]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    out[j >> 1][2 * (j & 1)] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[j], 1.f, false));
    out[j >> 1][2 * (j & 1) + 1] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[j], 1.f, true));
  }
}

// Keys and values lie in LDS as rows of 128 bf16, 272 and 288 bytes apart: the
// key operand reads 16 bytes of 16 rows, the transposing value read 32 bytes
// of eight rows each half wave, and both find all 64 banks, at addresses that
// differ by constants.
constexpr int kKeyRow = 17, kValueRow = 18;  // in units of 16 bytes

// Orders this wave's LDS accesses (the hardware runs them in order): one
// lane's writes before another's reads.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Lane n of each 16 lanes, in all of them.
template <int n>
__device__ __forceinline__ uint32_t row_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x150 + n, 0xF, 0xF, true);
}

struct Attn {
  const uint16_t *q;
  uint16_t *out;
  const void *k, *v;                       // pools, or packed rows
  int64_t q_stride, out_stride, k_stride, v_stride;
  const float *ks, *vs;                    // scales of e4m3 pools
  const int *starts, *table;               // of the batch; packed rows: starts alone
  const int *n_items, *others;             // others: items of a class that is not launched
  const Item *items;
  const uint64_t *stamp;                   // of the schedule, and what it has to be
  uint64_t want_stamp;
  int *refused;
  float2 *stats;                           // partial maxima and sums
  float *sums;
  int Hkv, group, rows, seqs, width, shift;
  uint32_t pages;
  int grid;                                // item slots launched per KV head
  int max_new;                             // new tokens of a sequence
  float scale;                             // of the scores, times log2(e)
  const uint64_t *masks;                   // trees: of the packed rows
  const uint64_t *planned, *step;          // their step, and the batch's
};

enum Source { kPages, kPagesFp8, kPacked };

typedef __attribute__((address_space(3))) const uint8_t lds_u8;
typedef const __attribute__((address_space(1))) uint8_t global_u8;

// Where a lane finds its operands in 32 keys' rows at an LDS address: the
// keys' dims 32 kk + 8 (lane / 16) + {0..7} of row 16 tile + lane mod 16, and
// (transposed) the values' dim 16 d + lane mod 16 of keys 16 half + 4 (lane /
// 16) + {0..3}.  ds_read_b64_tr_b16: 16 lanes read 4 rows x 16 columns, lane i
// gets column i.
struct Operands {
  uint32_t k, v;
  __device__ __forceinline__ explicit Operands(int lane) {
    const int i = lane & 15, g = lane >> 4;
    k = (uint32_t)(i * (16 * kKeyRow) + 16 * g);
    v = (uint32_t)((4 * g + (i >> 2)) * (16 * kValueRow) + 8 * (i & 3));
  }
  static __device__ __forceinline__ v8bf key(lds_u8 *p, int tile, int kk) {
    return *reinterpret_cast<__attribute__((address_space(3))) const v8bf *>(
        p + 64 * kk + 256 * kKeyRow * tile);
  }
  static __device__ __forceinline__ u32x4 values(lds_u8 *p, int d) {
    const u32x2 a = __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p + 32 * d)));
    const u32x2 b = __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p + 32 * d + 256 * kValueRow)));
    return u32x4{a[0], a[1], b[0], b[1]};
  }
};

// T groups of 16 queries (rows) against 32 keys a step.  Scores are computed
// transposed (S^T = K Q^T, v_mfma_f32_16x16x32_bf16), so a lane holds scores of
// one query of each group, lane mod 16, and the probabilities are the second
// product's B operand (O^T += V^T P^T) as they stand.  kFine: they enter in two
// parts of bf16, where the matrix unit has nothing better to do; the error
// against 64 bits is then the output's rounding, and else 1.4 times that.
// kAhead: operands are read from LDS this many ahead of their products (and not all
// at once, which would take registers that the other operands live in).  kFirst: the
// wave goes before the SIMD's other one while it mixes products and softmax, and
// after it in the scores, which are products alone (16 trees of 64 after 8192: 95 us,
// 100 without).
template <int T, bool kFine = false, int kAhead = 1, bool kFirst = false>
struct Rows {
  v4f o[T][8];
  // of the lane's query (alike in its four lanes): the whole number that its
  // base-2 exponents are taken from, and the sum of its probabilities, as a
  // product with ones (four times the same)
  float m[T];
  v4f l[T];
  // kFine: what the last probabilities lost when they were cut off to bf16, in
  // bf16: a second product adds it, and 2^-15 of them is lost
  u32x4 low[kFine ? T : 1];

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int t = 0; t < T; ++t) {
#pragma unroll
      for (int d = 0; d < 8; ++d) o[t][d] = v4f{0.f, 0.f, 0.f, 0.f};
      m[t] = 0.f, l[t] = v4f{0.f, 0.f, 0.f, 0.f};
    }
  }

  static __device__ __forceinline__ void scores(const Operands &at, lds_u8 *k,
                                                const v8bf (&q)[T][4], v4f (&s)[T][2]) {
#pragma unroll
    for (int t = 0; t < T; ++t) s[t][0] = s[t][1] = v4f{0.f, 0.f, 0.f, 0.f};
    lds_u8 *p = k + at.k;
    v8bf f[kAhead + 1];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = at.key(p, i & 1, i >> 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = i + kAhead;
      if (n < 8) f[n % (kAhead + 1)] = at.key(p, n & 1, n >> 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < T; ++t)
        s[t][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[i % (kAhead + 1)], q[t][i >> 1],
                                                              s[t][i & 1], 0, 0, 0);
    }
  }

  __device__ __forceinline__ void second(const Operands &at, lds_u8 *v, const u32x4 (&p)[T]) {
    v = v + at.v;
    u32x4 f[kAhead + 1];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) f[d] = at.values(v, d);
    sum(p);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      if (d + kAhead < 8) f[(d + kAhead) % (kAhead + 1)] = at.values(v, d + kAhead);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const v8bf vd = __builtin_bit_cast(v8bf, f[d % (kAhead + 1)]);
        o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vd, __builtin_bit_cast(v8bf, p[t]),
                                                          o[t][d], 0, 0, 0);
        if constexpr (kFine)
          o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vd, __builtin_bit_cast(v8bf, low[t]),
                                                            o[t][d], 0, 0, 0);
      }
    }
  }

  // Scores -> probabilities, powers of two from m rounded to bf16 (at most 2^-8
  // of each, like the output's own rounding): the second product then runs at
  // the bf16 rate.  At first, and where a probability reaches 2 (uniform,
  // rare), m goes to 6 above the query's largest exponent so far.  Otherwise it
  // stays: nothing overflows, and the quotient of the sums is the same.  m is a
  // whole number, so sums are scaled by powers of two: exactly.
  __device__ __forceinline__ void weigh(const v4f (&s)[T][2], float c, u32x4 (&p)[T], bool first) {
    powers(s, c, p);
    uint32_t bits = 0;
#pragma unroll
    for (int t = 0; t < T; ++t) bits |= (p[t][0] | p[t][1]) | (p[t][2] | p[t][3]);
    if (first || __any((bits & 0x40004000u) != 0)) raise(s, c, p, first);
  }
  __device__ __forceinline__ void raise(const v4f (&s)[T][2], float c, u32x4 (&p)[T], bool first) {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const v4f a = s[t][0], b = s[t][1];
      float top = fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])),
                        fmaxf(fmaxf(b[0], b[1]), fmaxf(b[2], b[3])));
      top = max_of_groups(top);
      // (kNone, below any exponent, while there was no score above -inf)
      float to = fmaxf(ceilf(top * c) + 6.f, kNone);
      if (!first) to = fmaxf(to, m[t]);
      const float f = first ? 1.f : __builtin_amdgcn_exp2f(m[t] - to);
      m[t] = to;
      l[t] *= f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[t][d] *= f;
    }
    powers(s, c, p);
  }
  __device__ __forceinline__ void powers(const v4f (&s)[T][2], float c, u32x4 (&p)[T]) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        v4f e;
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(fmaf(s[t][x][i], c, -m[t]));
        if constexpr (kFine) {
          // cut off, not rounded; the rest is above zero unless all is zero, so
          // that an infinite value stays what it is
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float e0 = e[2 * h], e1 = e[2 * h + 1];
            const uint32_t u0 = __float_as_uint(e0), u1 = __float_as_uint(e1) & 0xffff0000u;
            p[t][2 * x + h] = u1 | u0 >> 16;
            low[t][2 * x + h] = pack_bf16(
                fmaf(e0, 0x1p-24f, e0 - __uint_as_float(u0 & 0xffff0000u)),
                fmaf(e1, 0x1p-24f, e1 - __uint_as_float(u1)));
          }
        } else {
          p[t][2 * x] = pack_bf16(e[0], e[1]);
          p[t][2 * x + 1] = pack_bf16(e[2], e[3]);
        }
      }
  }
  // Two probabilities: cut off to bf16, and what they lost (see powers).
  static __device__ __forceinline__ u32x2 cut(float e0, float e1) {
    const uint32_t u0 = __float_as_uint(e0), u1 = __float_as_uint(e1) & 0xffff0000u;
    return u32x2{u1 | u0 >> 16,
                 pack_bf16(fmaf(e0, 0x1p-24f, e0 - __uint_as_float(u0 & 0xffff0000u)),
                           fmaf(e1, 0x1p-24f, e1 - __uint_as_float(u1)))};
  }
  __device__ __forceinline__ void sum(const u32x4 (&p)[T]) {
    constexpr uint32_t one = 0x3f803f80u;
    const v8bf ones = __builtin_bit_cast(v8bf, u32x4{one, one, one, one});
#pragma unroll
    for (int t = 0; t < T; ++t) {
      l[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(v8bf, p[t]), l[t], 0,
                                                     0, 0);
      if constexpr (kFine)
        l[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(v8bf, low[t]), l[t],
                                                       0, 0, 0);
    }
  }

  // One step j of a run of steps without masked positions, as one stream: the
  // second product of step j - 1 (its probabilities `was`) with the softmax of
  // step j between its instructions, then the scores of step j + 1.  A product
  // takes half of its time from the vector unit, so the two have to be mixed
  // finely to run beside each other: 3 products, 3 exponents and exponentials at
  // a time.  Operands are read from LDS kAhead products' operands ahead.
  // between(i), i < 8: other work beside the scores.
  static __device__ __forceinline__ u32x4 operand(lds_u8 *v, lds_u8 *k, int i) {
    if (i < 8) return Operands::values(v, i);
    return __builtin_bit_cast(u32x4, Operands::key(k, i & 1, (i - 8) >> 1));
  }
  template <class Between>
  __device__ __forceinline__ void stream(lds_u8 *v, lds_u8 *k, u32x4 (&was)[T],
                                         const v8bf (&q)[T][4], v4f (&s)[T][2], float c,
                                         Between between) {
    if constexpr (kFirst) __builtin_amdgcn_s_setprio(1);
    u32x4 f[kAhead + 1], p[T], rest[kFine ? T : 1];
    if constexpr (kFine) {
#pragma unroll
      for (int t = 0; t < T; ++t) rest[t] = low[t];
    }
    float e[T][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) f[i] = operand(v, k, i);
    __builtin_amdgcn_sched_barrier(0);
    sum(was);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[(i + kAhead) % (kAhead + 1)] = operand(v, k, i + kAhead);
#pragma unroll
      for (int t = 0; t < T; ++t) {
        e[t][i & 1] = __builtin_amdgcn_exp2f(fmaf(s[t][i >> 2][i & 3], c, -m[t]));
        if (i & 1) {
          if constexpr (kFine) {
            const u32x2 two = cut(e[t][0], e[t][1]);
            p[t][i >> 1] = two[0], low[t][i >> 1] = two[1];
          } else {
            p[t][i >> 1] = pack_bf16(e[t][0], e[t][1]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < T; ++t) {
        o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(v8bf, f[i % (kAhead + 1)]), __builtin_bit_cast(v8bf, was[t]),
            o[t][i], 0, 0, 0);
        if constexpr (kFine)
          o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(v8bf, f[i % (kAhead + 1)]), __builtin_bit_cast(v8bf, rest[t]),
              o[t][i], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    uint32_t bits = 0;
#pragma unroll
    for (int t = 0; t < T; ++t) bits |= (p[t][0] | p[t][1]) | (p[t][2] | p[t][3]);
    if (__any((bits & 0x40004000u) != 0)) raise(s, c, p, false);
#pragma unroll
    for (int t = 0; t < T; ++t) was[t] = p[t];
    if constexpr (kFirst) __builtin_amdgcn_s_setprio(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i + kAhead < 8) f[(8 + i + kAhead) % (kAhead + 1)] = operand(v, k, 8 + i + kAhead);
      between(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < T; ++t)
        s[t][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(v8bf, f[(8 + i) % (kAhead + 1)]), q[t][i >> 1],
            i < 2 ? v4f{0.f, 0.f, 0.f, 0.f} : s[t][i & 1], 0, 0, 0);
    }
  }

  // The lane's query of group t reads keys up to limit[t] only.
  static __device__ __forceinline__ void mask(v4f (&s)[T][2], int key0, const int (&limit)[T],
                                              int lane) {
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (key0 + 16 * x + 4 * (lane >> 4) + i > limit[t]) s[t][x][i] = -INFINITY;
  }

  // The lane's query of group t reads the keys of the set bits of word[t] only.
  static __device__ __forceinline__ void mask_words(v4f (&s)[T][2], const uint32_t (&word)[T],
                                                    int lane) {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const uint32_t w = word[t] >> (4 * (lane >> 4));
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(w >> (16 * x + i) & 1)) s[t][x][i] = -INFINITY;
    }
  }

  // Adds the infinities and NaNs of keys [first, end), whose values were
  // staged without them: each reaches the queries that read its position.
  // value(key, dim): four values of a key from dim on.  Rare.
  template <class Value>
  __device__ __forceinline__ void add_odd(int first, int end, const int (&limit)[T], int lane,
                                          Value value) {
#pragma unroll 1
    for (int key = first; key < end; ++key)
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const u32x2 v = value(key, 16 * d + 4 * (lane >> 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x =
              __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
          const bool odd = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
#pragma unroll
          for (int t = 0; t < T; ++t)
            if (odd && key <= limit[t]) o[t][d][i] += x;
        }
      }
  }
  // The same of trees: reads(t, key) says which queries do.
  template <class Value, class Reads>
  __device__ __forceinline__ void add_odd_if(int first, int end, int lane, Value value,
                                             Reads reads) {
#pragma unroll 1
    for (int key = first; key < end; ++key)
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const u32x2 v = value(key, 16 * d + 4 * (lane >> 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x =
              __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
          const bool odd = (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
#pragma unroll
          for (int t = 0; t < T; ++t)
            if (odd && reads(t, key)) o[t][d][i] += x;
        }
      }
  }
};

// The queries' operands: group t's rows are row0 + 16 t + lane mod 16, rows
// from `end` on repeat the last; limit: the last position each reads.
template <int T>
__device__ __forceinline__ void query_limits(const Attn &a, int cached, int row0, int end, int lane,
                                             int (&limit)[T]) {
#pragma unroll
  for (int t = 0; t < T; ++t)
    limit[t] = cached + min(row0 + 16 * t + (lane & 15), end - 1) / a.group;
}
template <int T>
__device__ __forceinline__ void load_queries(const Attn &a, int kvh, int start, int row0, int end,
                                             int lane, v8bf (&q)[T][4]) {
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int row = min(row0 + 16 * t + (lane & 15), end - 1);
    const int tok = row / a.group, head = kvh * a.group + row % a.group;
    const uint16_t *p = a.q + (int64_t)min(start + tok, a.rows - 1) * a.q_stride + head * kD +
                        8 * (lane >> 4);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) q[t][kk] = *reinterpret_cast<const v8bf *>(p + 32 * kk);
  }
}

// What an item needs to know of its sequence.
struct Place {
  int seq, row0, k0, k1, part;
  int start, n, cached;  // first packed row, new tokens, tokens before them
};

// The item-th tile of packed prompts, the ones that read the most keys first:
// i-th tiles of all sequences before (i - 1)-th ones.  Up to kSorted sequences:
// bisection for the level i, of which every lane counts kSorted / 64
// sequences' tiles.  24 prompts of 8192 rows: 78 us, 82 us in packed order; with
// 512 sequences the search costs more than it gains (95 us, 83 us).
constexpr int kSorted = 128;
__device__ __forceinline__ bool sorted_tile(const Attn &a, int tile_rows, int item, Place &p,
                                            int lane) {
  int here[kSorted / 64], n[kSorted / 64], tiles[kSorted / 64], most = 0;
#pragma unroll
  for (int i = 0; i < kSorted / 64; ++i) {
    const int s = 64 * i + lane;
    here[i] = n[i] = tiles[i] = 0;
    if (64 * i >= a.seqs) continue;  // uniform
    if (s < a.seqs) {
      here[i] = min(max(a.starts[s], 0), a.rows);
      n[i] = max(min(a.starts[s + 1], a.rows), here[i]) - here[i];
    }
    tiles[i] = (int)((uint32_t)(n[i] * a.group + tile_rows - 1) / (uint32_t)tile_rows);
    most = max(most, tiles[i]);
  }
  auto above = [&](int level) {  // tiles of this level or a higher one
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kSorted / 64; ++i)
      if (64 * i < a.seqs) sum += max(tiles[i] - level, 0);
    return __builtin_amdgcn_readlane(ecf8::dev::wave_inclusive_scan(sum), 63);
  };
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o));
  int lo = 0, hi = __builtin_amdgcn_readfirstlane(most), next = 0;  // next = above(hi)
  if (item >= above(0)) return false;
  while (hi - lo > 1) {  // above(lo) > item >= above(hi)
    const int mid = (lo + hi) >> 1, t = above(mid);
    if (t > item) lo = mid;
    else hi = mid, next = t;
  }
  int rank = item - next;
#pragma unroll
  for (int i = 0; i < kSorted / 64; ++i) {
    if (64 * i >= a.seqs) continue;
    const uint64_t has = __ballot(tiles[i] > lo);
    const int before = __popcll(has & ((1ull << lane) - 1));
    const uint64_t is = __ballot(tiles[i] > lo && before == rank);
    if (is) {  // uniform
      const int k = __builtin_ctzll(is);
      p.seq = 64 * i + k;
      p.start = __builtin_amdgcn_readlane(here[i], k), p.n = __builtin_amdgcn_readlane(n[i], k);
    }
    rank -= __popcll(has);
  }
  p.row0 = lo * tile_rows;
  return true;
}

// The same of more sequences, the last in memory first: sequence s has places
// floor(starts[s] G / R) + s on, which is room for its ceil(n G / R) tiles
// whatever the other lengths are.  64 probes a round.
__device__ __forceinline__ bool packed_tile(const Attn &a, int tile_rows, int item, Place &p,
                                            int lane) {
  const int vt = a.grid - 1 - item;
  int lo = 0, hi = a.seqs, here = 0, next = 0;
  auto first = [&](int start, int s) {
    return (int)((uint32_t)(start * a.group) / (uint32_t)tile_rows) + s;
  };
  for (;;) {
    const int step = (hi - lo + 63) / 64;
    const int s = min(lo + lane * step, a.seqs - 1);
    here = min(max(a.starts[s], 0), a.rows), next = min(a.starts[s + 1], a.rows);
    const uint64_t below = __ballot(lo + lane * step < hi && first(here, s) <= vt);
    const int k = below ? 63 - __builtin_clzll(below) : 0;
    here = __builtin_amdgcn_readlane(here, k), next = __builtin_amdgcn_readlane(next, k);
    lo += k * step;
    hi = min(hi, lo + step);
    if (step == 1) break;
  }
  p.seq = lo;
  p.start = here;
  p.n = max(next, here) - here;
  p.row0 = (vt - first(here, lo)) * tile_rows;
  return p.row0 >= 0 && p.row0 < p.n * a.group;
}

__device__ __forceinline__ bool find_tile(const Attn &a, int tile_rows, int item, Place &p,
                                          int lane) {
  if (item >= a.grid || !(a.seqs <= kSorted ? sorted_tile(a, tile_rows, item, p, lane)
                                            : packed_tile(a, tile_rows, item, p, lane)))
    return false;
  p.cached = 0;
  p.k0 = 0;
  p.k1 = min(p.n, (p.row0 + tile_rows - 1) / a.group + 1);
  p.part = -1;
  return true;
}

// The item of slot `item`; false past the last.
template <Source kSrc>
__device__ __forceinline__ bool get_item(const Attn &a, int tile_rows, int item, Place &p,
                                         int lane) {
  if constexpr (kSrc == kPacked) {
    // (the last workgroup, which has no tile or one of the last)
    if (a.refused && blockIdx.x == gridDim.x - 1) {
      bool bad = false;
      for (int s = threadIdx.x; s < a.seqs; s += 256) {
        const int from = a.starts[s], to = a.starts[s + 1];
        bad |= from < 0 || from > to || to > a.rows;
      }
      if (bad) *a.refused = 1;
    }
    return find_tile(a, tile_rows, item, p, lane);
  } else {
    // (the last workgroup, which has no item or a short one)
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0 && a.refused &&
        (a.starts[a.seqs] > a.rows ||
         (*a.stamp == a.want_stamp ? a.others && *a.others > 0 : *a.stamp != 0)))
      *a.refused = 1;
    const Item it = a.items[item];  // item < a.grid: in the list, filled or not
    asm volatile("" ::"s"(it.seq), "s"(it.start));  // not after the wait for n_items
    if (*a.stamp != a.want_stamp || item >= *a.n_items) return false;
    p.seq = it.seq, p.row0 = it.row0, p.k0 = it.k0, p.k1 = it.k1, p.part = it.part;
    p.start = it.start, p.n = it.n, p.cached = it.cached;
    if (p.n > a.max_new && threadIdx.x == 0 && a.refused) *a.refused = 1;
    return true;
  }
}

// The item of slot `item` of a step's trees; false past the last, and of trees that
// were planned for another step or sizes.
__device__ __forceinline__ bool get_tree_item(const Attn &a, int item, Place &p) {
  const Item it = a.items[item];  // item < a.grid: in the list, filled or not
  const uint64_t stamp = *a.stamp, planned = *a.planned, step = *a.step;
  const int n_items = *a.n_items, step_rows = a.starts[a.seqs];
  // (all before the first wait)
  asm volatile("" ::"s"(it.seq), "s"(it.start), "s"(n_items), "s"(stamp), "s"(planned), "s"(step),
               "s"(step_rows));
  const bool ours = stamp == a.want_stamp && planned == step;
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0 && a.refused && (!ours || step_rows > a.rows))
    *a.refused = 1;
  if (!ours || item >= n_items) return false;
  p.seq = it.seq, p.row0 = it.row0, p.k0 = it.k0, p.k1 = it.k1, p.part = it.part;
  p.start = it.start, p.n = it.n, p.cached = it.cached;
  return true;
}

// The masks of the lane's queries, as load_queries has them.
template <int T>
__device__ __forceinline__ void load_masks(const Attn &a, int start, int row0, int end, int lane,
                                           uint64_t (&bits)[T]) {
#pragma unroll
  for (int t = 0; t < T; ++t)
    bits[t] = a.masks[min(start + min(row0 + 16 * t + (lane & 15), end - 1) / a.group, a.rows - 1)];
}

// Which of the 32 keys from key0 < end on a query of mask `bits` reads: the cached
// ones, and the mask's of the rows after them.
__device__ __forceinline__ uint32_t tree_word(uint64_t bits, int key0, int cached, int end) {
  const int off = key0 - cached;
  uint64_t w;
  if (off <= -32) w = ~0ull;
  else if (off <= 0) w = bits << -off | ((1ull << -off) - 1);
  else w = off < 64 ? bits >> off : 0;
  if (end - key0 < 32) w &= (1ull << (end - key0)) - 1;
  return (uint32_t)w;
}

// Four bf16 of a sequence's value rows at (key, dim), as they lie in memory.
template <Source kSrc>
__device__ __forceinline__ u32x2 value4(const Attn &a, const Place &p, int kvh, int key, int dim) {
  if constexpr (kSrc == kPacked)
    return *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(a.v) +
                                            (int64_t)(p.start + key) * a.v_stride + kvh * kD + dim);
  const uint32_t page =
      min((uint32_t)a.table[(size_t)p.seq * a.width + (key >> a.shift)], a.pages - 1);
  const size_t at =
      (((page * a.Hkv + kvh) << a.shift) + (key & ((1 << a.shift) - 1))) * (size_t)kD + dim;
  if constexpr (kSrc == kPages)
    return *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(a.v) + at);
  const uint32_t codes =
      *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.v) + at);
  u32x4 w[2];
  widen16(u32x4{codes, 0, 0, 0}, w);
  return u32x2{w[0][0], w[0][1]};
}

// Workgroup barrier that waits for LDS only (a __syncthreads would also
// wait for the prefetched global loads).
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt((0x3F & 15) | (0x3 << 14) | (0x7 << 4) | (0x0 << 8));  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Workgroup of four waves: up to 16 T rows (token, head of the group) of one
// KV head against positions [k0, k1), 128 a round, 32 a wave; the waves' sums
// are joined in LDS.  A wave stages its keys and values through registers into
// LDS of its own, a round ahead, so the loop has no barrier.
//
// Bound by the pages' bytes: 64 sequences of up to 8192 keys, 8 heads (1.11 GB),
// 169 us, 6.6 TB/s; six of 100000 keys in e4m3, 4 heads (390 MB), 68 us, 5.7
// TB/s.  The matrix unit is busy for a tenth of that, so probabilities enter in
// two parts (kFine) at no cost.  With the join, these take 172 and 72 us; 195 and 82
// if page loads go through the caches, which a page, read once, gains nothing from;
// 173 and 78 with T = 2 where the step's rows allow 1.
//
// kTree: the step's trees (rows read the cached positions and their masks'), up to 32
// rows.  64 chains of 5 in groups of four after up to 8192 keys, 1.1 GB: 178 us, 6.1
// TB/s.  T = 1 up to 16 rows: one tree of 4 after 4096 10.5 us, 11.5 with T = 2.
template <Source kSrc, int T, bool kTree = false>
__global__ __launch_bounds__(256, 2) void few_kernel(Attn a) {
  __shared__ u32x4 s_kv[4][32 * (kKeyRow + kValueRow)];  // a wave's keys and values
  __shared__ float s_m[4][16 * T], s_l[4][16 * T];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = (int)blockIdx.x % a.Hkv;
  u32x4 *s_k = s_kv[wave], *s_v = s_kv[wave] + 32 * kKeyRow;
  constexpr bool kFp8 = kSrc == kPagesFp8;
  constexpr int kUnits = kFp8 ? 8 : 16;      // 16-byte units of a row in memory
  constexpr int kLoads = kUnits / 2;         // per lane and 32 rows
  const int unit = lane % kUnits;
  const Operands ops(lane);

  Place p;
  if constexpr (kTree) {
    if (!get_tree_item(a, (int)blockIdx.x / a.Hkv, p)) return;
  } else {
    if (!get_item<kSrc>(a, 16 * T, (int)blockIdx.x / a.Hkv, p, lane)) return;
  }
  const int n_rows = min(p.n * a.group - p.row0, 16 * T);
  // the first query's limit, or what all read
  const int low = kTree ? p.cached - 1 : p.cached + p.row0 / a.group;
  float c = a.scale, vscale = 1.f;
  if constexpr (kFp8) c *= a.ks[kvh], vscale = a.vs[kvh];

  // the row (page, head, offset) of key key0 + 8 (lane / 16) + lane mod 8; keys
  // past the last repeat it
  const int *table = kSrc == kPacked ? nullptr : a.table + (size_t)p.seq * a.width;
  auto locate = [&](int key0) -> uint32_t {
    const int key = min(key0 + 8 * (lane >> 4) + (lane & 7), p.k1 - 1);
    if constexpr (kSrc == kPacked) return (uint32_t)(p.start + key);
    const uint32_t page = min((uint32_t)table[key >> a.shift], a.pages - 1);
    return ((page * a.Hkv + kvh) << a.shift) + (key & ((1 << a.shift) - 1));
  };
  int key0 = p.k0 + 32 * wave;
  uint32_t at = locate(key0), next = locate(key0 + 128);
  v8bf q[T][4];
  int limit[T];
  uint64_t bits[T];
  load_queries<T>(a, kvh, p.start, p.row0, p.row0 + n_rows, lane, q);
  if constexpr (kTree) load_masks<T>(a, p.start, p.row0, p.row0 + n_rows, lane, bits);
  else query_limits<T>(a, p.cached, p.row0, p.row0 + n_rows, lane, limit);
  u32x4 kr[kLoads], vr[kLoads];
  bool odd = false;
  auto load = [&](uint32_t at) {
    const uint32_t rows[8] = {row_lane<0>(at), row_lane<1>(at), row_lane<2>(at),
                              row_lane<3>(at), row_lane<4>(at), row_lane<5>(at),
                              row_lane<6>(at), row_lane<7>(at)};
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t even = rows[kFp8 ? 2 * i : i], odd = rows[kFp8 ? 2 * i + 1 : i];
      const uint32_t w = lane & (kFp8 ? 8 : 0) ? odd : even;
      if constexpr (kSrc == kPacked) {
        kr[i] = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.k) +
                                                 (int64_t)w * a.k_stride + kvh * kD + 8 * unit);
        vr[i] = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.v) +
                                                 (int64_t)w * a.v_stride + kvh * kD + 8 * unit);
      } else {  // (read once)
        kr[i] = __builtin_nontemporal_load(static_cast<const u32x4 *>(a.k) +
                                            (size_t)w * kUnits + unit);
        vr[i] = __builtin_nontemporal_load(static_cast<const u32x4 *>(a.v) +
                                            (size_t)w * kUnits + unit);
      }
    }
  };
  auto store = [&](bool masked) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = 8 * (lane >> 4) + (kFp8 ? 2 * i + ((lane >> 3) & 1) : i);
      if constexpr (kFp8) {
        u32x4 w[2];
        widen16(kr[i], w);
        s_k[row * kKeyRow + 2 * unit] = w[0];
        s_k[row * kKeyRow + 2 * unit + 1] = w[1];
        widen16(vr[i], w);
        if (masked) {
          const u32x4 f0 = finite_or_zero(w[0]), f1 = finite_or_zero(w[1]);
          odd |= differ(f0, w[0]) || differ(f1, w[1]);
          w[0] = f0, w[1] = f1;
        }
        s_v[row * kValueRow + 2 * unit] = w[0];
        s_v[row * kValueRow + 2 * unit + 1] = w[1];
      } else {
        s_k[row * kKeyRow + unit] = kr[i];
        if (masked) {
          const u32x4 f = finite_or_zero(vr[i]);
          odd |= differ(f, vr[i]);
          vr[i] = f;
        }
        s_v[row * kValueRow + unit] = vr[i];
      }
    }
  };

  Rows<T, true> w;
  w.init();
  if (key0 < p.k1) {  // uniform
    load(at);
    at = next;
    for (; key0 < p.k1; key0 += 128) {
      const bool masked = key0 + 31 > low;  // uniform
      wave_fence();
      store(masked);
      wave_fence();
      if (key0 + 128 < p.k1) {
        load(at);
        at = locate(key0 + 256);
      }
      lds_u8 *k = (lds_u8 *)s_k, *v = (lds_u8 *)s_v;
      v4f s[T][2];
      u32x4 pr[T];
      w.scores(ops, k, q, s);
      if (masked) {
        if constexpr (kTree) {
          uint32_t word[T];
#pragma unroll
          for (int t = 0; t < T; ++t) word[t] = tree_word(bits[t], key0, p.cached, p.k1);
          w.mask_words(s, word, lane);
        } else {
          w.mask(s, key0, limit, lane);
        }
      }
      w.weigh(s, c, pr, key0 == p.k0 + 32 * wave);
      w.second(ops, v, pr);
    }
    if (__any(odd))
      for (key0 = p.k0 + 32 * wave; key0 < p.k1; key0 += 128)
        if (key0 + 31 > low) {
          if constexpr (kTree)
            w.add_odd_if(
                key0, min(key0 + 32, p.k1), lane,
                [&](int key, int dim) { return value4<kSrc>(a, p, kvh, key, dim); },
                [&](int t, int key) {
                  return (tree_word(bits[t], key, p.cached, p.k1) & 1) != 0;
                });
          else
            w.add_odd(key0, min(key0 + 32, p.k1), limit, lane,
                      [&](int key, int dim) { return value4<kSrc>(a, p, kvh, key, dim); });
        }
  }

  // join the waves
  float l[T];
#pragma unroll
  for (int t = 0; t < T; ++t) {
    l[t] = w.l[t][0];
    if (l[t] == 0.f) w.m[t] = kLowest;
    if (lane < 16) s_m[wave][16 * t + lane] = w.m[t], s_l[wave][16 * t + lane] = l[t];
  }
  __syncthreads();
  // rows of 32 units of 4 sums, unit u of row r at u ^ r; over the wave's own
  // keys and values, which it has read
  float4 *so = reinterpret_cast<float4 *>(s_kv[wave]);
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const int r = 16 * t + (lane & 15);
    const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float f = __builtin_amdgcn_exp2f(w.m[t] - top);
#pragma unroll
    for (int d = 0; d < 8; ++d)
      so[r * 32 + ((4 * d + (lane >> 4)) ^ r)] =
          make_float4(w.o[t][d][0] * f, w.o[t][d][1] * f, w.o[t][d][2] * f, w.o[t][d][3] * f);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * n_rows; i += 256) {
    const int row = i >> 5, u = i & 31;
    float4 t[4];
    float sum = 0.f, mt = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      t[x] = reinterpret_cast<const float4 *>(s_kv[x])[row * 32 + (u ^ row)];
      sum += s_l[x][row] * __builtin_amdgcn_exp2f(s_m[x][row] - mt);
    }
    const float4 all = make_float4((t[0].x + t[1].x) + (t[2].x + t[3].x),
                                   (t[0].y + t[1].y) + (t[2].y + t[3].y),
                                   (t[0].z + t[1].z) + (t[2].z + t[3].z),
                                   (t[0].w + t[1].w) + (t[2].w + t[3].w));
    if (p.part >= 0) {
      const size_t at = ((size_t)p.part * a.Hkv + kvh) * kFewRows + row;
      reinterpret_cast<float4 *>(a.sums)[at * 32 + u] = all;
      if (u == 0) a.stats[at] = make_float2(mt, sum);
    } else {
      const int g = p.row0 + row;
      const int tk = p.start + g / a.group;
      const float inv = kTree && sum == 0.f ? 0.f : vscale / sum;  // (a mask can be empty)
      if (tk < a.rows)
        *reinterpret_cast<u32x2 *>(a.out + (int64_t)tk * a.out_stride +
                                   (kvh * a.group + g % a.group) * kD + 4 * u) =
            u32x2{pack_bf16(all.x * inv, all.y * inv), pack_bf16(all.z * inv, all.w * inv)};
    }
  }
}

constexpr int kT = 3;  // groups of 16 rows a wave of the tile kernel
constexpr int kTileWaves = kTileRows / (16 * kT);

// Workgroup of four waves, one a SIMD, two workgroups a CU: 192 rows (token,
// head of the group) of one KV head, 48 a wave, against positions [k0, k1).
// 48 rows share every operand that a wave reads from LDS: at 32 the reads
// alone would take as long as the products.
//
// A wave's softmax of a step of 32 keys runs beside the second product of the
// step before (Rows::stream).  Keys and values go through registers to a ring
// of LDS stages.  Steps without masked positions have a loop of their own: with
// the masks' branches in it a step took 8% longer.
//
// Bound by the products (51 MFMA of 16 cycles a wave and step) and the vector
// instructions beside them (140): 1.25 PFLOP/s in the loop of unmasked steps,
// where a large library product reaches 1.34.  One prompt of 8192 tokens, 32
// heads: 485 to 505 us by card, of which the loop takes 440; 24 prompts of 8192
// tokens together: 80 us, mostly the first loads and the last steps of ~100 short
// tiles.  Tiles of 384 rows and eight waves reach the same rate in the loop, but take
// 1.04 and 1.3 times as long: fewer tiles fill the card less evenly.  Pages of fewer
// than 8 positions (not kWhole): 6 registers spilled in bf16.
template <Source kSrc, bool kWhole>
__global__ __launch_bounds__(64 * kTileWaves, 2) void tile_kernel(Attn a) {
  // Stages of a step's keys and values each: after the barrier before step j
  // the waves read steps j - 1 to j + 1 and write j + 2.
  constexpr int kRing = 4;
  __shared__ u32x4 s_kv[kRing][32 * (kKeyRow + kValueRow)];
  __shared__ int s_odd;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = (int)blockIdx.x % a.Hkv;
  const Operands ops(lane);
  constexpr bool kFp8 = kSrc == kPagesFp8;
  // A wave loads 1 KB pieces: kRows rows of a step, kLoads of them for the keys
  // and as many for the values.
  constexpr int kUnits = kFp8 ? 8 : 16;      // 16-byte units of a row in memory
  constexpr int kRows = 64 / kUnits, kPieces = 32 / kRows;
  constexpr int kLoads = kPieces / kTileWaves;
  const int unit = lane % kUnits, sub = lane / kUnits;

  Place p;
  if (!get_item<kSrc>(a, kTileRows, (int)blockIdx.x / a.Hkv, p, lane)) return;
  const int all_rows = min(p.n * a.group - p.row0, kTileRows);
  const int first_row = 16 * kT * wave, n_rows = min(all_rows - first_row, 16 * kT);
  // the last position that all rows of the wave read, and of the workgroup
  const int low = p.cached + (p.row0 + min(first_row, all_rows - 1)) / a.group;
  const int low0 = p.cached + p.row0 / a.group;
  float c = a.scale, vscale = 1.f;
  if constexpr (kFp8) c *= a.ks[kvh], vscale = a.vs[kvh];

  const int steps = (p.k1 - p.k0 + 31) / 32;
  // the steps that all rows read in full
  const int full = max(0, (min(low0 + 1, p.k1) - p.k0) / 32);
  const int *table = kSrc == kPacked ? nullptr : a.table + (size_t)p.seq * a.width;
  // the first key of this wave's piece i of step j; (kTail: past the end the
  // last piece, and its last row)
  auto piece = [&](auto tail, int j, int i) {
    const int key = p.k0 + 32 * j + (32 / kLoads) * i + kRows * wave;
    return decltype(tail)::value ? min(key, (p.k1 - 1) & -kRows) : key;
  };
  // Pages of the pieces to be loaded next.  kWhole: a page has kRows positions
  // or more, so a piece lies in one, and lane i looks up that of piece i;
  // otherwise a lane looks up its own rows.
  constexpr int kEntries = kWhole ? 1 : kLoads;
  int entry[kEntries];
  auto look = [&](auto tail, int j, int (&entry)[kEntries]) {
    if constexpr (kSrc != kPacked) {
#pragma unroll
      for (int i = 0; i < kEntries; ++i) {
        // (never a scalar load: it would make every wait for LDS wait for all
        // of LDS)
        int key = kWhole ? piece(tail, j, 0) : piece(tail, j, i) + sub;
        if constexpr (kWhole && kLoads > 1) key += (32 / kLoads) * (lane & (kLoads - 1));
        if (decltype(tail)::value) key = min(key, p.k1 - 1);
        uint32_t at = (uint32_t)(key >> a.shift) * 4u;
        asm volatile("" : "+v"(at));
        entry[i] = *reinterpret_cast<const int *>(reinterpret_cast<const uint8_t *>(table) + at);
      }
    }
  };
  int first[3][kEntries];
#pragma unroll
  for (int x = 0; x <= 2; ++x) look(std::true_type(), x, first[x]);
  v8bf q[kT][4];
  load_queries<kT>(a, kvh, p.start, p.row0 + first_row, p.row0 + all_rows, lane, q);
  u32x4 kr[kLoads], vr[kLoads];
  auto load_piece = [&](auto tail, int j, int i, int entry, u32x4 &kr, u32x4 &vr) {
    // a piece's base is scalar, a lane's offset has 32 bits
    const int key = piece(tail, j, i);
    const int row = decltype(tail)::value ? min(sub, p.k1 - 1 - key) : sub;
    const uint8_t *kb, *vb;
    uint32_t ko, vo;
    if constexpr (kSrc == kPacked) {
      const int64_t at = p.start + key;
      kb = static_cast<const uint8_t *>(a.k) + 2 * (at * a.k_stride + kvh * kD);
      vb = static_cast<const uint8_t *>(a.v) + 2 * (at * a.v_stride + kvh * kD);
      ko = __umul24(row, 2 * (uint32_t)a.k_stride) + 16 * unit;
      vo = __umul24(row, 2 * (uint32_t)a.v_stride) + 16 * unit;
    } else {
      const uint32_t mask = (1u << a.shift) - 1;
      if constexpr (kWhole) {
        const uint32_t page = min((uint32_t)__builtin_amdgcn_readlane(entry, i), a.pages - 1);
        const size_t at = (size_t)(((page * a.Hkv + kvh) << a.shift) + (key & mask)) *
                          (16 * kUnits);
        kb = static_cast<const uint8_t *>(a.k) + at;
        vb = static_cast<const uint8_t *>(a.v) + at;
        ko = vo = (uint32_t)row * (16 * kUnits) + 16 * unit;
      } else {
        const uint32_t page = min((uint32_t)entry, a.pages - 1);
        const size_t at = (size_t)(((page * a.Hkv + kvh) << a.shift) + ((key + row) & mask)) *
                          (16 * kUnits);
        kr = *reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(a.k) + at + 16 * unit);
        vr = *reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(a.v) + at + 16 * unit);
        return;
      }
    }
    global_u8 *kg = (global_u8 *)kb, *vg = (global_u8 *)vb;
    asm volatile("" : "+s"(kg), "+s"(vg));  // (else 64-bit offsets stay in vector registers)
    kr = *(const __attribute__((address_space(1))) u32x4 *)(kg + ko);
    vr = *(const __attribute__((address_space(1))) u32x4 *)(vg + vo);
  };
  // piece i of step j to its stage (kTail: it may have masked positions)
  auto store_piece = [&](auto tail, int j, int i, u32x4 kr, u32x4 vr) {
    constexpr bool kTail = decltype(tail)::value;
    u32x4 *s_k = s_kv[j % kRing], *s_v = s_kv[j % kRing] + 32 * kKeyRow;
    const int row = (32 / kLoads) * i + kRows * wave + sub;
    if constexpr (kFp8) {
      u32x4 w[2];
      widen16(kr, w);
      s_k[row * kKeyRow + 2 * unit] = w[0];
      s_k[row * kKeyRow + 2 * unit + 1] = w[1];
      widen16(vr, w);
      if (kTail && j >= full) {  // uniform
        const u32x4 f0 = finite_or_zero(w[0]), f1 = finite_or_zero(w[1]);
        if (differ(f0, w[0]) || differ(f1, w[1])) s_odd = 1;
        w[0] = f0, w[1] = f1;
      }
      s_v[row * kValueRow + 2 * unit] = w[0];
      s_v[row * kValueRow + 2 * unit + 1] = w[1];
    } else {
      s_k[row * kKeyRow + unit] = kr;
      if (kTail && j >= full) {  // uniform
        const u32x4 f = finite_or_zero(vr);
        if (differ(f, vr)) s_odd = 1;
        vr = f;
      }
      s_v[row * kValueRow + unit] = vr;
    }
  };
  auto load = [&](int j, const int (&entry)[kEntries], u32x4 (&kr)[kLoads], u32x4 (&vr)[kLoads]) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_piece(std::true_type(), j, i, entry[kWhole ? 0 : i], kr[i], vr[i]);
  };
  auto store = [&](int j, const u32x4 (&kr)[kLoads], const u32x4 (&vr)[kLoads]) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) store_piece(std::true_type(), j, i, kr[i], vr[i]);
  };
  auto barrier = [] {
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto keys = [&](int j) { return (lds_u8 *)s_kv[j % kRing]; };
  auto values = [&](int j) { return (lds_u8 *)(s_kv[j % kRing] + 32 * kKeyRow); };

  Rows<kT> w;
  w.init();
  v4f s[kT][2];
  u32x4 pr[kT];
  {
    u32x4 k1[2][kLoads], v1[2][kLoads];
    if (threadIdx.x == 0) s_odd = 0;
#pragma unroll
    for (int x = 0; x < 2; ++x) load(x, first[x], k1[x], v1[x]);
    load(2, first[2], kr, vr);
    look(std::true_type(), 3, entry);
    __syncthreads();  // s_odd
#pragma unroll
    for (int x = 0; x < 2; ++x) store(x, k1[x], v1[x]);
    lds_barrier();
  }
  // (a step past the last is the last again, and never read)
  auto between = [&](auto tail, int j, int i) {
    if (i == 0 || i == 1) {
      if (i < kLoads) store_piece(tail, j + 2, i, kr[i], vr[i]);
    } else if (i == 2 || i == 4) {
      const int x = i == 4;
      if (x < kLoads) load_piece(tail, j + 3, x, entry[kWhole ? 0 : x], kr[x], vr[x]);
    } else if (i == 6) {
      look(tail, j + 4, entry);
    }
  };
  if (n_rows <= 0) {  // uniform: a wave without rows stages its share
#pragma unroll 1
    for (int j = 0; j < steps; ++j) {
      barrier();
#pragma unroll
      for (int i = 0; i < 8; ++i) between(std::true_type(), j, i);
    }
    return;
  }
  // The lane and the limits are formed where they are needed, not kept in
  // registers through the loops.
  auto late_lane = [] {
    uint32_t none = 0;
    asm volatile("" : "+v"(none));
    return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none));
  };
  auto mask = [&](int j) {
    const int late = late_lane();
    int limit[kT];
    query_limits<kT>(a, p.cached, p.row0 + first_row, p.row0 + all_rows, late, limit);
    w.mask(s, p.k0 + 32 * j, limit, late);
  };
  w.scores(ops, keys(0), q, s);
  barrier();
  if (p.k0 + 31 > low) mask(0);
  w.weigh(s, c, pr, true);
#pragma unroll
  for (int i = 0; i < 8; ++i) between(std::true_type(), 0, i);
  w.scores(ops, keys(1), q, s);
  int j = 1;
#pragma unroll 1
  for (; j < full - 4; ++j) {
    barrier();
    w.stream(values(j - 1) + ops.v, keys(j + 1) + ops.k, pr, q, s, c,
             [&](int i) { between(std::false_type(), j, i); });
  }
#pragma unroll 1
  for (; j < steps; ++j) {
    barrier();
    if (p.k0 + 32 * j + 31 > low) mask(j);  // uniform
    w.stream(values(j - 1) + ops.v, keys(j + 1) + ops.k, pr, q, s, c,
             [&](int i) { between(std::true_type(), j, i); });
  }
  w.second(ops, values(steps - 1), pr);
  const int late = late_lane();
  if (s_odd) {  // (written before the last barrier)
    int limit[kT];
    query_limits<kT>(a, p.cached, p.row0 + first_row, p.row0 + all_rows, late, limit);
    w.add_odd(p.k0 + 32 * full, p.k1, limit, late,
              [&](int key, int dim) { return value4<kSrc>(a, p, kvh, key, dim); });
  }
#pragma unroll
  for (int t = 0; t < kT; ++t) {
    const float l = w.l[t][0];
    const int row = first_row + 16 * t + (late & 15), g = late >> 4;
    if (row >= all_rows) continue;
    if (p.part >= 0) {
      const size_t at = ((size_t)p.part * a.Hkv + kvh) * kTileRows + row;
      v4f *sums = reinterpret_cast<v4f *>(a.sums) + at * 32 + g;
#pragma unroll
      for (int d = 0; d < 8; ++d) sums[4 * d] = w.o[t][d];
      if (g == 0) a.stats[at] = make_float2(l == 0.f ? kLowest : w.m[t], l);
    } else {
      const int at = p.row0 + row, tk = p.start + at / a.group;
      const float inv = vscale / l;
      if (tk < a.rows) {
        uint16_t *op = a.out + (int64_t)tk * a.out_stride +
                       (kvh * a.group + at % a.group) * kD + 4 * g;
#pragma unroll
        for (int d = 0; d < 8; ++d)
          *reinterpret_cast<u32x2 *>(op + 16 * d) =
              u32x2{pack_bf16(w.o[t][d][0] * inv, w.o[t][d][1] * inv),
                    pack_bf16(w.o[t][d][2] * inv, w.o[t][d][3] * inv)};
      }
    }
  }
}

// One class's joins: the plan's list, and the workgroups of a join (over the
// rows) and of all of them.
struct Joins {
  const int *n;
  const Join *list;
  const float *sums;
  const float2 *stats;
  int rows_groups, groups;
};

// The parts of split rows, joined: four dims a lane, kSplit halves of a wave a
// row (each every kSplit-th part), four parts' loads at a time.
template <int kSplit, int kPartRows>
__device__ __forceinline__ void join_parts(const Attn &a, const Joins &o, int group) {
  __shared__ float s_top[8], s_l[8];
  __shared__ v4f s_sum[8][32];
  const int lane = threadIdx.x & 31, half = threadIdx.x >> 5;
  const int y = group % o.rows_groups, kvh = group / o.rows_groups % a.Hkv;
  const int j = group / o.rows_groups / a.Hkv;
  const Join jn = o.list[j];  // j: in the list, filled or not
  asm volatile("" ::"s"(jn.row0), "s"(jn.start));  // not after the wait for the count
  if (*a.stamp != a.want_stamp || j >= *o.n) return;
  constexpr int part_rows = kPartRows;
  const int n_rows = min(jn.tokens * a.group - jn.row0, part_rows);
  const float vscale = a.vs ? a.vs[kvh] : 1.f;
  constexpr int kRows = 8 / kSplit;  // at a time
  for (int row0 = kRows * y; row0 < n_rows; row0 += kRows * o.rows_groups) {
    const int row = min(row0 + half / kSplit, n_rows - 1);
    const size_t at = ((size_t)jn.part * a.Hkv + kvh) * part_rows + row;
    const size_t step = (size_t)a.Hkv * part_rows;
    // (maxima of parts without a key are below every other's)
    float top = kLowest, l = 0.f;
    v4f sum = {};
    for (int x0 = half % kSplit; x0 < jn.n; x0 += 4 * kSplit) {
      v4f v[4];
      float2 st[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const size_t p = at + min(x0 + u * kSplit, jn.n - 1) * step;
        v[u] = reinterpret_cast<const v4f *>(o.sums)[p * 32 + lane];
        st[u] = o.stats[p];
      }
      float to = top;
#pragma unroll
      for (int u = 0; u < 4; ++u) to = fmaxf(to, st[u].x);  // (past the last: that again)
      const float f0 = __builtin_amdgcn_exp2f(top - to);
      l *= f0, sum *= f0;
      top = to;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (x0 + u * kSplit >= jn.n) break;
        const float f = __builtin_amdgcn_exp2f(st[u].x - top);
        l = fmaf(f, st[u].y, l);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = fmaf(f, v[u][i], sum[i]);
      }
    }
    if constexpr (kSplit > 1) {
      if (lane == 0) s_top[half] = top, s_l[half] = l;
      s_sum[half][lane] = sum;
      __syncthreads();
      if (half == 0) {
        float to = s_top[0];
#pragma unroll
        for (int x = 1; x < 8; ++x) to = fmaxf(to, s_top[x]);
        l = 0.f, sum = v4f{};
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const float f = __builtin_amdgcn_exp2f(s_top[x] - to);
          l = fmaf(f, s_l[x], l);
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = fmaf(f, s_sum[x][lane][i], sum[i]);
        }
      }
    }
    const int g = jn.row0 + row, tk = jn.start + g / a.group;
    const float inv = vscale / l;
    if ((kSplit == 1 ? row0 + half < n_rows : half == 0) && tk < a.rows)
      *reinterpret_cast<u32x2 *>(a.out + (int64_t)tk * a.out_stride +
                                 (kvh * a.group + g % a.group) * kD + 4 * lane) =
          u32x2{pack_bf16(sum[0] * inv, sum[1] * inv), pack_bf16(sum[2] * inv, sum[3] * inv)};
    if constexpr (kSplit > 1) __syncthreads();
  }
}

// Both classes in one launch.  Latency: two joins of 85 parts, 3 us; 22 tiles in
// 86 parts, 8 heads (67 MB), 13 us.
__global__ __launch_bounds__(256) void join_kernel(Attn a, Joins few, Joins tiles) {
  const int i = (int)blockIdx.x;
  if (i < few.groups) join_parts<8, kFewRows>(a, few, i);
  else join_parts<1, kTileRows>(a, tiles, i - few.groups);
}

// ------------------------------------------------------------ drafted trees

// Workgroup: 16 T rows (token, head of the group) a wave of one KV head, against
// positions [k0, k1), 32 a step: 64 and 128 rows in four waves, two workgroups a CU,
// or 256 in eight, one a CU.  As in tile_kernel a wave's softmax of a step runs
// beside the second product of the step before.  Keys and values go through
// registers, two steps ahead, to a ring of LDS stages.  kGroups = 2: eight waves, two
// groups with a ring each, which take half of the keys and join over LDS.
//
// A step's 32 keys cost 16 T rows 17 T products (kFine 25 T) and some 45 T vector
// instructions, which in the loop take 0.8 to 1.0 of the sum of their times, whatever
// their order.  256 rows and long contexts are bound by them: eight trees of 64 with 8
// heads a group (two tiles of 256) after 32768 e4m3 keys, 175 us with the join, 870
// TFLOP/s of the 1240 that a large library product reaches beside it; the two units'
// cycles add up to 71% of the launch.  Of smaller trees, 24 of up to 26 after up to 6000
// bf16 keys, 57 to 62 us by card, 3.7 TB/s, they are two thirds: the rest is the pieces'
// first loads and last sums, and a barrier every 32 keys.
// kOnce, pages past the caches, where a sequence's pages are read by one workgroup:
// those take 61 us, 63 through the caches; of two tiles (16 trees of 64 with 8
// heads a group, after 8192) 92 us, and 95 past the caches.
// Not faster: 128 rows in eight waves, 192 in four (registers spill), half of the
// waves for the staging alone (bf16 5% faster where contexts are long, e4m3 and short
// ones 10% slower), loads three steps ahead.
template <Source kSrc, int kGroups, int kWaves, int T, bool kFine, bool kOnce>
__global__ __launch_bounds__(64 * kGroups * kWaves, 2) void tree_kernel(Attn a) {
  constexpr int kDepth = 2;
  constexpr int kRows = 16 * T * kWaves, kThreads = 64 * kWaves;  // of a group
  constexpr bool kFp8 = kSrc == kPagesFp8;
  constexpr int kUnits = kFp8 ? 8 : 16;               // 16-byte units of a row in memory
  // rows a pass of the threads; twice a step's: keys and values have half of them each
  constexpr int kPass = kThreads / kUnits;
  constexpr bool kHalves = kPass > 32;
  constexpr int kLoads = kHalves ? 1 : 32 / kPass;
  // after the barrier before step j the waves read steps j - 1 to j + 1 and write j + 2
  constexpr int kRing = 4;
  // steps that two groups share: one tree of 32 after 4096 (pieces of 13 steps) 20.5 us,
  // 21.5 from eight on; 32 of 8, 8 heads a group, after up to 512 19.7 and 18.8
  constexpr int kBoth = 16;
  __shared__ u32x4 s_rings[kGroups][kRing][32 * (kKeyRow + kValueRow)];
  __shared__ int s_odds[kGroups];
  const int lane = threadIdx.x & 63;
  const int tid = kGroups > 1 ? (int)threadIdx.x % kThreads : (int)threadIdx.x;
  const int group = kGroups > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads) : 0;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = (int)blockIdx.x % a.Hkv;
  const Operands ops(lane);
  auto &s_kv = s_rings[group];
  int &s_odd = s_odds[group];

  Place p;
  if (!get_tree_item(a, (int)blockIdx.x / a.Hkv, p)) return;
  const int all_rows = min(p.n * a.group - p.row0, kRows);
  const int first_row = 16 * T * wave;
  const int n_rows = min(all_rows - first_row, 16 * T);
  int most = (p.k1 - p.k0 + 31) / 32;  // steps of a group
  const bool both = kGroups > 1 && most >= kBoth;
  if (both) {
    most = (most + 1) / 2;
    const int middle = p.k0 + 32 * most;
    if (group) p.k0 = middle;
    else p.k1 = middle;
  } else if (group) {
    return;  // (barriers wait for the waves that are left)
  }
  float c = a.scale, vscale = 1.f;
  if constexpr (kFp8) c *= a.ks[kvh], vscale = a.vs[kvh];

  // load i of a step: row kPass i + sub of its keys and values.  kTail: past the
  // end the last row again.
  const int unit = tid % kUnits;
  const int sub = tid / kUnits % (kHalves ? 32 : kPass);
  const bool key_half = !kHalves || tid < kThreads / 2;
  const int *table = a.table + (size_t)p.seq * a.width;
  const int steps = (p.k1 - p.k0 + 31) / 32;
  auto key_of = [&](auto tail, int j, int i) {
    const int key = p.k0 + 32 * j + kPass * i + sub;
    return decltype(tail)::value ? min(key, p.k1 - 1) : key;
  };
  struct Staged {
    u32x4 k[kLoads], v[kHalves ? 1 : kLoads];  // (kHalves: k alone, a key or a value)
    int entry[kLoads];                         // pages of the step kDepth later
  };
  auto look = [&](auto tail, int j, Staged &r) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) r.entry[i] = table[key_of(tail, j, i) >> a.shift];
  };
  auto place = [&](auto tail, int j, const Staged &r, size_t (&at)[kLoads]) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t page = min((uint32_t)r.entry[i], a.pages - 1);
      at[i] = (size_t)(((page * a.Hkv + kvh) << a.shift) +
                       (key_of(tail, j, i) & ((1 << a.shift) - 1))) * kUnits + unit;
    }
  };
  auto load = [&](const size_t (&at)[kLoads], Staged &r) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      auto get = [&](const void *pool) {
        const u32x4 *x = static_cast<const u32x4 *>(pool) + at[i];
        return kOnce ? __builtin_nontemporal_load(x) : *x;
      };
      r.k[i] = get(key_half ? a.k : a.v);
      if constexpr (!kHalves) r.v[i] = get(a.v);
    }
  };
  auto store = [&](auto tail, int j, const Staged &r) {
    u32x4 *s_k = s_kv[j % kRing], *s_v = s_k + 32 * kKeyRow;
    const bool masked = decltype(tail)::value && p.k0 + 32 * j + 31 >= p.cached;  // uniform
    auto finite = [&](u32x4 v) {
      if (!masked) return v;
      const u32x4 f = finite_or_zero(v);
      if (differ(f, v)) s_odd = 1;
      return f;
    };
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = kPass * i + sub;
      if constexpr (kFp8) {
        u32x4 w[2];
        widen16_pairs(r.k[i], w);
        if (key_half) {
          s_k[row * kKeyRow + 2 * unit] = w[0];
          s_k[row * kKeyRow + 2 * unit + 1] = w[1];
        }
        if constexpr (!kHalves) widen16_pairs(r.v[i], w);
        if (!kHalves || !key_half) {
          s_v[row * kValueRow + 2 * unit] = finite(w[0]);
          s_v[row * kValueRow + 2 * unit + 1] = finite(w[1]);
        }
      } else {
        s_k[row * kKeyRow + unit] = r.k[i];
        s_v[row * kValueRow + unit] = finite(r.v[i]);
      }
    }
  };
  auto barrier = [] {
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto keys = [&](int j) { return (lds_u8 *)s_kv[j % kRing]; };
  auto values = [&](int j) { return (lds_u8 *)(s_kv[j % kRing] + 32 * kKeyRow); };

  // r[x]: the next steps j of j mod kDepth = (x + 2) mod kDepth; the first two are
  // staged before the loop
  constexpr std::true_type kTail;
  Staged r[kDepth], lead[2];
  look(kTail, 0, lead[0]), look(kTail, 1, lead[1]);
#pragma unroll
  for (int x = 0; x < kDepth; ++x) look(kTail, 2 + x, r[x]);
  v8bf q[T][4];
  const int row0 = p.row0 + min(first_row, all_rows - 1), row_end = p.row0 + all_rows;
  load_queries<T>(a, kvh, p.start, row0, row_end, lane, q);
  if (tid == 0) s_odd = 0;
  size_t at[kLoads];
#pragma unroll
  for (int x = 0; x < 2; ++x) place(kTail, x, lead[x], at), load(at, lead[x]);
#pragma unroll
  for (int x = 0; x < kDepth; ++x) {
    place(kTail, 2 + x, r[x], at);
    look(kTail, 2 + kDepth + x, r[x]);
    load(at, r[x]);
  }
  __syncthreads();  // s_odd
  store(kTail, 0, lead[0]), store(kTail, 1, lead[1]);
  lds_barrier();

  // Beside the scores of step j + 1: step j + 2 to its stage, and the loads of the
  // step kDepth later.  Loads past the end are the last row again, never read: a
  // load that may not be there makes every wait one for all loads.
  auto between = [&](auto tail, int j, int i, Staged &r) {
    if (i == 0) {
      // (in the end the stage of the last step's values is read once more)
      if (!decltype(tail)::value || j + 2 < steps) store(tail, j + 2, r);
    } else if (i == 2) {
      // (pages before the rows: what waits for them must not wait for these rows)
      place(tail, j + 2 + kDepth, r, at);
      look(tail, j + 2 + 2 * kDepth, r);
    } else if (i == 4) {
      load(at, r);
    }
  };
  // all waves pass as many barriers: one for step 0, kDepth a turn
  const int turns = (most - 1 + kDepth - 1) / kDepth;
  if (n_rows <= 0) {  // uniform: a wave without rows stages its share
    barrier();
#pragma unroll
    for (int i = 0; i < 8; ++i) between(kTail, 0, i, r[0]);
#pragma unroll 1
    for (int turn = 0; turn < turns; ++turn)
#pragma unroll
      for (int x = 1; x <= kDepth; ++x) {
        barrier();
#pragma unroll
        for (int i = 0; i < 8; ++i) between(kTail, turn * kDepth + x, i, r[x % kDepth]);
      }
    if (both) barrier(), barrier();  // (the groups' join)
    return;
  }
  Rows<T, kFine, 2, true> w;
  w.init();
  v4f s[T][2];
  u32x4 pr[T];
  auto mask = [&](int j) {
    const int key0 = p.k0 + 32 * j;
    if (key0 + 31 < p.cached) return;  // uniform
    uint64_t bits[T];  // (not kept in registers through the loops)
    load_masks<T>(a, p.start, row0, row_end, lane, bits);
    uint32_t word[T];
#pragma unroll
    for (int t = 0; t < T; ++t) word[t] = tree_word(bits[t], key0, p.cached, p.k1);
    w.mask_words(s, word, lane);
  };
  w.scores(ops, keys(0), q, s);
  barrier();
  mask(0);
  w.weigh(s, c, pr, true);
#pragma unroll
  for (int i = 0; i < 8; ++i) between(kTail, 0, i, r[0]);
  w.scores(ops, keys(1), q, s);
  // Turns whose steps, and those that they load, have no masks and no end: a loop of
  // their own, without a branch.
  const int full = max(0, (min(p.cached, p.k1) - p.k0) / 32);
  const int clear = min(turns, max(0, full - 3 - 2 * kDepth) / kDepth);
  int turn = 0;
#pragma unroll 1
  for (; turn < clear; ++turn) {
#pragma unroll
    for (int x = 1; x <= kDepth; ++x) {
      const int j = turn * kDepth + x;
      barrier();
      w.stream(values(j - 1) + ops.v, keys(j + 1) + ops.k, pr, q, s, c,
               [&](int i) { between(std::false_type(), j, i, r[x % kDepth]); });
    }
  }
#pragma unroll 1
  for (; turn < turns; ++turn) {
#pragma unroll
    for (int x = 1; x <= kDepth; ++x) {
      const int j = turn * kDepth + x;
      barrier();
      if (j < steps) {  // uniform
        mask(j);
        w.stream(values(j - 1) + ops.v, keys(j + 1) + ops.k, pr, q, s, c,
                 [&](int i) { between(kTail, j, i, r[x % kDepth]); });
      }
    }
  }
  w.second(ops, values(steps - 1), pr);
  if (s_odd) {  // (written before the last barrier)
    uint64_t bits[T];
    load_masks<T>(a, p.start, row0, row_end, lane, bits);
    for (int key0 = p.k0 + 32 * max(0, (p.cached - p.k0) / 32); key0 < p.k1; key0 += 32)
      w.add_odd_if(
          key0, min(key0 + 32, p.k1), lane,
          [&](int key, int dim) { return value4<kSrc>(a, p, kvh, key, dim); },
          [&](int t, int key) { return (tree_word(bits[t], key, p.cached, p.k1) & 1) != 0; });
  }
#pragma unroll
  for (int t = 0; t < T; ++t)
    if (w.l[t][0] == 0.f) w.m[t] = kLowest;
  if (both) {  // the second group's sums over LDS (its ring) to the first
    v4f *sums = reinterpret_cast<v4f *>(s_rings[kGroups - 1]) + wave * (T * 8 * 64) + lane;
    float2 *stats = reinterpret_cast<float2 *>(reinterpret_cast<v4f *>(s_rings[kGroups - 1]) +
                                               kWaves * T * 8 * 64) + wave * (T * 64) + lane;
    barrier();
    if (group) {
#pragma unroll
      for (int t = 0; t < T; ++t) {
        stats[64 * t] = make_float2(w.m[t], w.l[t][0]);
#pragma unroll
        for (int d = 0; d < 8; ++d) sums[64 * (8 * t + d)] = w.o[t][d];
      }
    }
    barrier();
    if (group) return;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const float2 st = stats[64 * t];
      const float top = fmaxf(w.m[t], st.x);
      const float f0 = __builtin_amdgcn_exp2f(w.m[t] - top);
      const float f1 = __builtin_amdgcn_exp2f(st.x - top);
      w.m[t] = top;
      w.l[t][0] = fmaf(f1, st.y, w.l[t][0] * f0);
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const v4f v = sums[64 * (8 * t + d)];
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[t][d][i] = fmaf(f1, v[i], w.o[t][d][i] * f0);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const float l = w.l[t][0];
    const int row = first_row + 16 * t + (lane & 15), g = lane >> 4;
    if (row >= all_rows) continue;
    if (p.part >= 0) {
      const size_t at = ((size_t)p.part * a.Hkv + kvh) * kRows + row;
      v4f *sums = reinterpret_cast<v4f *>(a.sums) + at * 32 + g;
#pragma unroll
      for (int d = 0; d < 8; ++d) sums[4 * d] = w.o[t][d];
      if (g == 0) a.stats[at] = make_float2(w.m[t], l);
    } else {
      const int at = p.row0 + row, tk = p.start + at / a.group;
      const float inv = l == 0.f ? 0.f : vscale / l;  // (a mask can be empty)
      if (tk < a.rows) {
        uint16_t *op = a.out + (int64_t)tk * a.out_stride +
                       (kvh * a.group + at % a.group) * kD + 4 * g;
#pragma unroll
        for (int d = 0; d < 8; ++d)
          *reinterpret_cast<u32x2 *>(op + 16 * d) =
              u32x2{pack_bf16(w.o[t][d][0] * inv, w.o[t][d][1] * inv),
                    pack_bf16(w.o[t][d][2] * inv, w.o[t][d][3] * inv)};
      }
    }
  }
}

// Joins the parts of split rows: workgroup of `per` rows of a tile and KV head, four
// dims a lane, eight parts' loads at a time.  Half a wave a row, or, for many parts
// of few rows, a row at a time, its parts dealt to the eight half waves.  Latency of
// three loads in a row: 3 us of one tree, 6 to 11 of many.
__global__ __launch_bounds__(256) void tree_join_kernel(Attn a, Joins o, int part_rows, int per) {
  __shared__ float s_top[8], s_l[8];
  __shared__ v4f s_sum[8][32];
  const int lane = threadIdx.x & 31, half = threadIdx.x >> 5;
  const int kvh = (int)blockIdx.x % a.Hkv, group = (int)blockIdx.x / a.Hkv;
  const int y = group % o.rows_groups, j = group / o.rows_groups;
  const Join jn = o.list[j];  // j: in the list, filled or not
  const uint64_t stamp = *a.stamp, planned = *a.planned, step_now = *a.step;
  const int n_joins = *o.n;
  asm volatile("" ::"s"(jn.row0), "s"(jn.start), "s"(stamp), "s"(planned), "s"(step_now),
               "s"(n_joins));
  // (as in get_tree_item)
  if (stamp != a.want_stamp || planned != step_now || j >= n_joins) return;
  const int end = min(min(jn.tokens * a.group - jn.row0, part_rows), (y + 1) * per);
  const float vscale = a.vs ? a.vs[kvh] : 1.f;
  const size_t step = (size_t)a.Hkv * part_rows;
  const size_t at0 = ((size_t)jn.part * a.Hkv + kvh) * part_rows;
  float top, l;
  v4f sum;
  // parts x0, x0 + every, ... of a row (maxima of parts without a key are below
  // every other's)
  auto gather = [&](int row, int x0, int every) {
    top = kLowest, l = 0.f, sum = v4f{};
    for (; x0 < jn.n; x0 += 8 * every) {
      v4f v[8];
      float2 st[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const size_t p = at0 + row + min(x0 + u * every, jn.n - 1) * step;
        v[u] = reinterpret_cast<const v4f *>(o.sums)[p * 32 + lane];
        st[u] = o.stats[p];
      }
      float to = top;
#pragma unroll
      for (int u = 0; u < 8; ++u) to = fmaxf(to, st[u].x);  // (past the last: that again)
      const float f0 = __builtin_amdgcn_exp2f(top - to);
      l *= f0, sum *= f0;
      top = to;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (x0 + u * every >= jn.n) break;
        const float f = __builtin_amdgcn_exp2f(st[u].x - top);
        l = fmaf(f, st[u].y, l);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = fmaf(f, v[u][i], sum[i]);
      }
    }
  };
  auto put = [&](int row) {
    const int g = jn.row0 + row, tk = jn.start + g / a.group;
    const float inv = l == 0.f ? 0.f : vscale / l;  // (a mask can be empty)
    if (tk < a.rows)
      *reinterpret_cast<u32x2 *>(a.out + (int64_t)tk * a.out_stride +
                                 (kvh * a.group + g % a.group) * kD + 4 * lane) =
          u32x2{pack_bf16(sum[0] * inv, sum[1] * inv), pack_bf16(sum[2] * inv, sum[3] * inv)};
  };
  if ((jn.n + 7) / 8 <= per * ((jn.n + 63) / 64)) {  // whichever takes fewer batches
    for (int row = y * per + half; row < end; row += 8) gather(row, 0, 1), put(row);
    return;
  }
  for (int row = y * per; row < end; ++row) {
    gather(row, half, 8);
    if (lane == 0) s_top[half] = top, s_l[half] = l;
    s_sum[half][lane] = sum;
    __syncthreads();
    if (half == 0) {
      float to = s_top[0];
#pragma unroll
      for (int x = 1; x < 8; ++x) to = fmaxf(to, s_top[x]);
      l = 0.f, sum = v4f{};
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float f = __builtin_amdgcn_exp2f(s_top[x] - to);
        l = fmaf(f, s_l[x], l);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = fmaf(f, s_sum[x][lane][i], sum[i]);
      }
      put(row);
    }
    __syncthreads();
  }
}

inline hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }
inline bool aligned(const void *p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}
inline int launched() { return hipGetLastError() == hipSuccess ? ECF8_OK : ECF8_ERR_HIP; }

}  // namespace

extern "C" int ecf8_paged_attention(const void *q, int64_t q_stride, int64_t rows,
                                    const ecf8_paged_batch *b, const void *k_pool,
                                    const void *v_pool, int fp8, const float *k_scale,
                                    const float *v_scale, int64_t max_new, void *out,
                                    int64_t out_stride, void *stream) {
  if (!q || !k_pool || !v_pool || !out || rows <= 0 || max_new <= 0 ||
      (fp8 && (!k_scale || !v_scale)))
    return ECF8_ERR_INVALID_ARG;
  if (const int rc = check_batch(b)) return rc;
  if (rows > b->rows) return ECF8_ERR_CAPACITY;
  if (max_new > rows) max_new = rows;  // (and its products fit)
  const int64_t wide = (int64_t)b->Hq * kD;
  if (q_stride % 8 || out_stride % 4 || (rows > 1 && (q_stride < wide || out_stride < wide)))
    return ECF8_ERR_UNSUPPORTED;
  if (!aligned(q, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(out, 8) ||
      !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return ECF8_ERR_MISALIGNED;
  const Work w = work_layout(b->seqs, b->rows, b->Hq, b->Hkv);
  auto *base = static_cast<uint8_t *>(b->work);
  auto *counts = reinterpret_cast<Counts *>(base);
  const int G = b->Hq / b->Hkv;
  Attn a{};
  a.q = static_cast<const uint16_t *>(q), a.out = static_cast<uint16_t *>(out);
  a.k = k_pool, a.v = v_pool;
  a.q_stride = q_stride, a.out_stride = out_stride;
  a.ks = fp8 ? k_scale : nullptr, a.vs = fp8 ? v_scale : nullptr;
  a.starts = b->starts, a.table = b->table, a.refused = b->refused;
  a.stamp = &counts->stamp, a.want_stamp = schedule_stamp(b);
  a.Hkv = b->Hkv, a.group = G, a.rows = (int)rows, a.seqs = b->seqs, a.width = b->width;
  a.shift = __builtin_ctz((unsigned)b->page_size), a.pages = (uint32_t)b->pages;
  a.max_new = (int)max_new;
  a.scale = kLog2e / sqrtf((float)kD);
  const bool many = max_new * G > kFewRows;
  Joins few{}, tiles{};
  if (G <= kFewRows) {
    a.n_items = &counts->few, a.others = many ? nullptr : &counts->tiles;
    a.items = reinterpret_cast<const Item *>(base + w.few_at);
    a.stats = reinterpret_cast<float2 *>(base + w.few_stats);
    a.sums = reinterpret_cast<float *>(base + w.few_sums);
    // items that the parts' target and the longest sequence allow
    const int64_t seqs = rows < b->seqs ? rows : b->seqs;
    const int64_t most = seqs * (((int64_t)b->width * b->page_size + kFewKeys - 1) / kFewKeys);
    a.grid = (int)(w.few_parts / 2 + seqs < most ? w.few_parts / 2 + seqs : most);
    const unsigned grid = (unsigned)(a.grid * a.Hkv);
#define ECF8_FEW(S, T) few_kernel<S, T><<<grid, 256, 0, as_stream(stream)>>>(a)
    if (max_new * G <= 16) {
      if (fp8) ECF8_FEW(kPagesFp8, 1);
      else ECF8_FEW(kPages, 1);
    } else {
      if (fp8) ECF8_FEW(kPagesFp8, 2);
      else ECF8_FEW(kPages, 2);
    }
    if (most > seqs) {  // something may be split
      few.rows_groups = (int)(max_new * G < 8 ? max_new * G : 8);
      few.groups = (int)(seqs < w.few_parts / 2 ? seqs : w.few_parts / 2) * a.Hkv * few.rows_groups;
      few.n = &counts->few_joins;
      few.list = reinterpret_cast<const Join *>(base + w.few_joins_at);
      few.stats = a.stats, few.sums = a.sums;
    }
  }
  if (many) {
    a.n_items = &counts->tiles, a.others = nullptr;
    a.items = reinterpret_cast<const Item *>(base + w.tiles_at);
    a.stats = reinterpret_cast<float2 *>(base + w.tile_stats);
    a.sums = reinterpret_cast<float *>(base + w.tile_sums);
    const int64_t most = rows * G / kTileRows + (rows < b->seqs ? rows : b->seqs);  // tiles
    const int64_t joins = most < w.tile_parts / 2 ? most : w.tile_parts / 2;
    a.grid = (int)most + w.tile_parts / 2;  // a cut adds an item
    const unsigned grid = (unsigned)(a.grid * a.Hkv);
#define ECF8_TILES(S, W) tile_kernel<S, W><<<grid, 64 * kTileWaves, 0, as_stream(stream)>>>(a)
    if (b->page_size >= 8) {
      if (fp8) ECF8_TILES(kPagesFp8, true);
      else ECF8_TILES(kPages, true);
    } else {
      if (fp8) ECF8_TILES(kPagesFp8, false);
      else ECF8_TILES(kPages, false);
    }
    tiles.rows_groups = kTileRows / 8, tiles.groups = (int)joins * a.Hkv * tiles.rows_groups;
    tiles.n = &counts->tile_joins;
    tiles.list = reinterpret_cast<const Join *>(base + w.tile_joins_at);
    tiles.stats = a.stats, tiles.sums = a.sums;
  }
  if (const int groups = few.groups + tiles.groups)
    join_kernel<<<(unsigned)groups, 256, 0, as_stream(stream)>>>(a, few, tiles);
  return launched();
}

extern "C" int ecf8_draft_attention(const void *q, int64_t q_stride, int64_t rows,
                                    const ecf8_paged_batch *b, const ecf8_draft_trees *trees,
                                    const void *k_pool, const void *v_pool, int fp8,
                                    const float *k_scale, const float *v_scale, void *out,
                                    int64_t out_stride, void *stream) {
  if (!q || !k_pool || !v_pool || !out || rows <= 0 || (fp8 && (!k_scale || !v_scale)))
    return ECF8_ERR_INVALID_ARG;
  if (const int rc = ecf8::draft::check_trees(b, trees)) return rc;
  if (rows > b->rows) return ECF8_ERR_CAPACITY;
  const int64_t wide = (int64_t)b->Hq * kD;
  if (q_stride % 8 || out_stride % 4 || (rows > 1 && (q_stride < wide || out_stride < wide)))
    return ECF8_ERR_UNSUPPORTED;
  if (!aligned(q, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(out, 8) ||
      !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return ECF8_ERR_MISALIGNED;
  const ecf8::draft::Work w = ecf8::draft::work_layout(b->seqs, b->rows, b->Hq, b->Hkv,
                                                       trees->max_nodes, trees->max_children);
  auto *base = static_cast<uint8_t *>(trees->work);
  auto *counts = reinterpret_cast<ecf8::draft::Counts *>(base);
  Attn a{};
  a.q = static_cast<const uint16_t *>(q), a.out = static_cast<uint16_t *>(out);
  a.k = k_pool, a.v = v_pool;
  a.q_stride = q_stride, a.out_stride = out_stride;
  a.ks = fp8 ? k_scale : nullptr, a.vs = fp8 ? v_scale : nullptr;
  a.starts = b->starts, a.table = b->table, a.refused = b->refused;
  a.masks = trees->masks, a.planned = &counts->step, a.step = ecf8::draft::step_of(b);
  a.stamp = &counts->stamp, a.want_stamp = ecf8::draft::schedule_stamp(b, trees);
  a.Hkv = b->Hkv, a.group = b->Hq / b->Hkv, a.rows = (int)rows, a.seqs = b->seqs;
  a.width = b->width;
  a.shift = __builtin_ctz((unsigned)b->page_size), a.pages = (uint32_t)b->pages;
  a.scale = kLog2e / sqrtf((float)kD);
  a.n_items = &counts->items;
  a.items = reinterpret_cast<const Item *>(base + w.items_at);
  a.stats = reinterpret_cast<float2 *>(base + w.stats);
  a.sums = reinterpret_cast<float *>(base + w.sums);
  // tiles of the step, and the pieces that their cuts add
  const int64_t seqs = rows < b->seqs ? rows : b->seqs;
  const int64_t tiles = (rows < w.nodes ? rows : w.nodes) * a.group / w.tile + seqs;
  const int64_t units =
      ((int64_t)b->width * b->page_size + ecf8::draft::kUnitKeys - 1) / ecf8::draft::kUnitKeys;
  const int64_t cuts = w.target < tiles * (units - 1) ? w.target : tiles * (units - 1);
  a.grid = (int)(tiles + cuts);
  const unsigned grid = (unsigned)(a.grid * a.Hkv);
  Joins j{};
  j.n = &counts->joins, j.list = reinterpret_cast<const Join *>(base + w.joins_at);
  j.stats = a.stats, j.sums = a.sums;
  // rows a workgroup: eight, fewer while there are not a thousand workgroups (one tree
  // of 8 after 4096: 12.5 us, 14.2 with eight; 16 of 32 after 8192: 87, 97 with one)
  const int most_rows = trees->max_nodes * a.group < w.tile ? trees->max_nodes * a.group : w.tile;
  const int64_t splits = (tiles < cuts ? tiles : cuts) * a.Hkv;
  int per = 8;
  while (per > 1 && splits * ((most_rows + per - 1) / per) < 1024) per /= 2;
  j.rows_groups = (most_rows + per - 1) / per;
  j.groups = (int)(splits * j.rows_groups);
#define ECF8_TREE_FEW(T)                                                                  \
  do {                                                                                    \
    if (fp8) few_kernel<kPagesFp8, T, true><<<grid, 256, 0, as_stream(stream)>>>(a);      \
    else few_kernel<kPages, T, true><<<grid, 256, 0, as_stream(stream)>>>(a);             \
  } while (0)
#define ECF8_TREE(G, W, T, F, O)                                                                \
  do {                                                                                          \
    constexpr unsigned threads = 64 * G * W;                                                    \
    if (fp8) tree_kernel<kPagesFp8, G, W, T, F, O><<<grid, threads, 0, as_stream(stream)>>>(a); \
    else tree_kernel<kPages, G, W, T, F, O><<<grid, threads, 0, as_stream(stream)>>>(a);        \
  } while (0)
  const bool halves = ecf8::draft::in_halves(w.tile, b->seqs, b->Hkv);
  switch (w.tile) {
    case 16:
      ECF8_TREE_FEW(1);
      break;
    case 32:
      ECF8_TREE_FEW(2);
      break;
    case 64:  // (two parts cost up to 3% in bf16, a tenth in e4m3)
      if (halves) ECF8_TREE(2, 4, 1, true, true);
      else ECF8_TREE(1, 4, 1, true, true);
      break;
    case 128:  // (16 trees of 26 after 8192: 78 us, 65 in one)
      if (halves) ECF8_TREE(2, 4, 2, true, true);
      else ECF8_TREE(1, 4, 2, true, true);
      break;
    // (see kOnce.  Rounded to bf16 once, as in tile_kernel, since the products bound these:
    // eight trees of 64 with 8 heads a group after 32768 e4m3 keys 179 us, 228 in two
    // parts; 16 of 64 after 8192 bf16 ones 95 and 121)
    default:
      if (trees->max_nodes * a.group <= 256) ECF8_TREE(1, 8, 2, false, true);
      else ECF8_TREE(1, 8, 2, false, false);
  }
#undef ECF8_TREE_FEW
#undef ECF8_TREE
  if (j.groups)
    tree_join_kernel<<<(unsigned)j.groups, 256, 0, as_stream(stream)>>>(
        a, j, w.tile < kFewRows ? kFewRows : w.tile, per);
  return launched();
}

extern "C" int ecf8_ragged_attention_checked(const void *q, int64_t q_stride, const void *k,
                                             int64_t k_stride, const void *v, int64_t v_stride,
                                             int64_t rows, const int *starts, int64_t seqs, int Hq,
                                             int Hkv, void *out, int64_t out_stride, int *refused,
                                             void *stream) {
  if (!q || !k || !v || !starts || !out || rows <= 0 || seqs <= 0 || Hq <= 0 || Hkv <= 0)
    return ECF8_ERR_INVALID_ARG;
  const int64_t wide = (int64_t)Hq * kD, kv = (int64_t)Hkv * kD;
  if (!sizes_ok(seqs, rows, Hq, Hkv) || q_stride % 8 || k_stride % 8 || v_stride % 8 ||
      out_stride % 4 || k_stride > (1 << 22) || v_stride > (1 << 22) ||
      (rows > 1 && (q_stride < wide || out_stride < wide || k_stride < kv ||
                                      v_stride < kv)))
    return ECF8_ERR_UNSUPPORTED;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 8) ||
      !aligned(starts, 4) || !aligned(refused, 4))
    return ECF8_ERR_MISALIGNED;
  Attn a{};
  a.q = static_cast<const uint16_t *>(q), a.out = static_cast<uint16_t *>(out);
  a.k = k, a.v = v;
  a.q_stride = q_stride, a.out_stride = out_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.starts = starts, a.refused = refused;
  a.Hkv = Hkv, a.group = Hq / Hkv, a.rows = (int)rows, a.seqs = (int)seqs;
  a.scale = kLog2e / sqrtf((float)kD);
  // Tiles once they make up a workgroup for every CU: one prompt of 512 / 1024 / 1536
  // / 2048 rows of 32 heads takes 22 / 36 / 49 / 64 us in tiles and 16 / 34 / 57 / 87
  // us in 32 rows a workgroup; 2048 rows in 16 / 64 prompts 17 / 13 and 33 / 29 us,
  // 8192 in 512 73 and 108 us.
  const bool tiles = rows * Hq / kTileRows >= kTileSlots / 2;
  a.grid = (int)(rows * a.group / (tiles ? kTileRows : kFewRows) + seqs);
  const unsigned grid = (unsigned)((int64_t)a.grid * Hkv);
  if (tiles) ECF8_TILES(kPacked, true);
  else ECF8_FEW(kPacked, 2);
#undef ECF8_FEW
#undef ECF8_TILES
  return launched();
}

extern "C" int ecf8_ragged_attention(const void *q, int64_t q_stride, const void *k,
                                     int64_t k_stride, const void *v, int64_t v_stride,
                                     int64_t rows, const int *starts, int64_t seqs, int Hq,
                                     int Hkv, void *out, int64_t out_stride, void *stream) {
  return ecf8_ragged_attention_checked(q, q_stride, k, k_stride, v, v_stride, rows, starts, seqs,
                                       Hq, Hkv, out, out_stride, nullptr, stream);
}
