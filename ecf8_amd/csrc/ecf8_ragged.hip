// Attention of a ragged batch on gfx950: sequences of different lengths, new
// tokens packed one sequence after the other, keys and values in the pages of
// a cache (bf16 or e4m3) or packed like the queries.  Head dimension 128,
// fp32 scores, softmax statistics and sums.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "ecf8.h"
#include "ecf8_paged.h"
#include "ecf8_paged_layout.h"

namespace {

using namespace ecf8::paged;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.0e38f;  // running maximum before any score

typedef float v16f __attribute__((ext_vector_type(16)));
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

// Eight bf16 with their infinities and NaNs replaced by zeros.
__device__ __forceinline__ u32x4 finite_or_zero(u32x4 v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if ((v[j] & 0x7f80u) == 0x7f80u) v[j] &= 0xffff0000u;
    if ((v[j] & 0x7f800000u) == 0x7f800000u) v[j] &= 0xffffu;
  }
  return v;
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

// Keys and values lie in LDS as rows of 16 units of 16 bytes, unit c of row
// `row` at c ^ turn(row).  The key operand reads one unit of 32 rows, the
// transposing value reads four units of four rows each half wave: both find
// all 64 banks.
__device__ __forceinline__ int turn(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }

// Orders this wave's LDS accesses (the hardware runs them in order): one
// lane's writes before another's reads.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

struct Attn {
  const uint16_t *q;
  uint16_t *out;
  const void *k, *v;                       // pools, or packed rows
  int64_t q_stride, out_stride, k_stride, v_stride;
  const float *ks, *vs;                    // scales of e4m3 pools
  const int *starts, *lengths, *table;     // of the batch; packed rows: starts alone
  const int *n_items, *others;             // other: items of a class that is not launched
  const Item *items;
  int *refused;
  float2 *stats;                           // partial maxima and sums
  float *sums;
  int Hkv, group, rows, seqs, width, shift;
  uint32_t pages;
  int grid;                                // item slots launched per KV head
  float scale;                             // of the scores, times log2(e)
};

enum Source { kPages, kPagesFp8, kPacked };

// 32 rows of queries against 32 keys a step: the scores of one step, their
// softmax and the second product.  Scores are computed transposed (S^T = K
// Q^T), so a lane holds its query's scores of 16 keys: the running maximum
// takes one exchange with lane ^ 32, and the probabilities are the second
// product's B operand (O^T += V^T P^T) as they stand.  V^T comes from V's
// rows in LDS by the transposing reads (ds_read_b64_tr_b16: 16 lanes read 4
// keys x 16 dims, lane i gets dim i of the four keys).
struct Wave {
  v16f o[4];
  float m, l;  // of query lane & 31; both halves hold the same m, each its own l

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    m = kLowest, l = 0.f;
  }

  static __device__ __forceinline__ v16f scores(const u32x4 *s_k, const v8bf (&qf)[8], int lane) {
    const int r = lane & 31, h = lane >> 5;
    v16f s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      const v8bf kf = *reinterpret_cast<const v8bf *>(&s_k[r * 16 + ((2 * kk + h) ^ turn(r))]);
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[kk], s, 0, 0, 0);
    }
    return s;
  }

  // Four keys' values of this lane's dim 32 d + (lane & 31): keys 16 g + 8 half
  // + 4 (lane >> 5) + {0..3}.
  static __device__ __forceinline__ u32x2 values(const u32x4 *s_v, int d, int g, int half,
                                                 int lane) {
    const int i = lane & 15, key = 16 * g + 8 * half + 4 * (lane >> 5) + (i >> 2);
    const int unit = 4 * d + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
    const uint8_t *p = reinterpret_cast<const uint8_t *>(&s_v[key * 16 + (unit ^ turn(key))]) +
                       8 * (i & 1);
    const v4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_v4s *)(v4s *)const_cast<uint8_t *>(p));
    return __builtin_bit_cast(u32x2, v);
  }
  static __device__ __forceinline__ u32x4 values8(const u32x4 *s_v, int d, int g, int lane) {
    const u32x2 a = values(s_v, d, g, 0, lane), b = values(s_v, d, g, 1, lane);
    return u32x4{a[0], a[1], b[0], b[1]};
  }

  // One step of 32 keys from key0 on; kMasked: this lane's query reads keys
  // up to `limit` only.
  template <bool kMasked>
  __device__ __forceinline__ void step(v16f s, const u32x4 *s_v, int key0, int limit, float c,
                                       int lane) {
    const int h = lane >> 5;
    if constexpr (kMasked) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 8 * (i >> 2) + 4 * h + (i & 3) > limit) s[i] = -INFINITY;
    }
    float bm = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) bm = fmaxf(bm, s[i]);
    const auto hm = __builtin_amdgcn_permlane32_swap(__float_as_uint(bm), __float_as_uint(bm),
                                                     false, false);
    const float mn = fmaxf(m, fmaxf(__uint_as_float(hm[0]), __uint_as_float(hm[1])));
    // uniform: some query's maximum moved by more than a factor 2^8 of its
    // exponentials.  Below that m stays: nothing overflows, and the quotient
    // of the sums is the same.
    if (__any((mn - m) * c > 8.f)) {
      const float f = __builtin_amdgcn_exp2f((m - mn) * c);
      l *= f;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= f;
      m = mn;
    }
    const float mc = m * c;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -mc));
      l += s[i];
    }
    // Probabilities rounded to bf16 (at most 2^-8 of each, like the output's
    // own rounding): the second product then runs at the bf16 rate.
    u32x4 p[2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j) p[g][j] = pack_bf16(s[8 * g + 2 * j], s[8 * g + 2 * j + 1]);
    uint32_t odd = 0;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        u32x4 v = values8(s_v, d, g, lane);
        if constexpr (kMasked) {
          // what a masked position holds must not enter, not even as 0 x inf
          const u32x4 f = finite_or_zero(v);
#pragma unroll
          for (int j = 0; j < 4; ++j) odd |= f[j] ^ v[j];
          v = f;
        }
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, v),
                                                       __builtin_bit_cast(v8bf, p[g]), o[d], 0, 0,
                                                       0);
      }
    if constexpr (kMasked) {
      if (__any(odd != 0)) not_finite(s, s_v, lane);  // uniform, rare
    }
  }

  // The infinities and NaNs among a masked step's values, for the queries that
  // give their keys a probability above zero: counted by products of zeros
  // and ones, then added.
  __device__ __forceinline__ void not_finite(const v16f &s, const u32x4 *s_v, int lane) {
    u32x4 p[2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p[g][j] = (s[8 * g + 2 * j] > 0.f ? 0x3f80u : 0u) |
                  (s[8 * g + 2 * j + 1] > 0.f ? 0x3f800000u : 0u);
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll 1
      for (int kind = 0; kind < 3; ++kind) {  // +inf, -inf, NaN
        const uint32_t want = kind == 0 ? 0x7f80u : 0xff80u;
        v16f n;
#pragma unroll
        for (int i = 0; i < 16; ++i) n[i] = 0.f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          u32x4 v = values8(s_v, d, g, lane);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = v[j] & 0xffffu, hi = v[j] >> 16;
            const bool a = kind == 2 ? (lo & 0x7fffu) > 0x7f80u : lo == want;
            const bool b = kind == 2 ? (hi & 0x7fffu) > 0x7f80u : hi == want;
            v[j] = (a ? 0x3f80u : 0u) | (b ? 0x3f800000u : 0u);
          }
          n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, v),
                                                      __builtin_bit_cast(v8bf, p[g]), n, 0, 0, 0);
        }
        const float add = kind == 0 ? INFINITY : kind == 1 ? -INFINITY : NAN;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (n[i] > 0.f) o[d][i] += add;
      }
  }
};

// What an item needs to know of its sequence.
struct Place {
  int seq, row0, k0, k1, part;
  int start, n, cached;  // first packed row, new tokens, tokens before them
};

// Sequence and tile of virtual tile `vt` of packed prompts: sequence s has
// tiles floor(starts[s] G / R) + s on, which is room for its ceil(n G / R)
// ones whatever the other lengths are.  64 probes a round.
__device__ __forceinline__ bool find_tile(const Attn &a, int tile_rows, int vt, Place &p,
                                          int lane) {
  int lo = 0, hi = a.seqs;
  auto first = [&](int s) {
    return (int)((int64_t)min(max(a.starts[s], 0), a.rows) * a.group / tile_rows) + s;
  };
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, s = lo + lane * step;
    const uint64_t below = __ballot(s < hi && first(s) <= vt);
    const int k = below ? 63 - __builtin_clzll(below) : 0;
    lo += k * step;
    hi = min(hi, lo + step);
  }
  p.seq = lo;
  p.start = min(max(a.starts[lo], 0), a.rows);
  p.n = max(min(a.starts[lo + 1], a.rows) - p.start, 0);
  p.cached = 0;
  p.row0 = (vt - first(lo)) * tile_rows;
  if (p.row0 < 0 || p.row0 >= p.n * a.group) return false;
  p.k0 = 0;
  p.k1 = min(p.n, (p.row0 + tile_rows - 1) / a.group + 1);
  p.part = -1;
  return true;
}

// Workgroup of four waves: 32 rows (token, head of the group) of one KV head
// against positions [k0, k1), 128 a round, 32 a wave; the waves' sums are
// joined in LDS.  A wave stages its keys and values through registers into
// LDS of its own, a round ahead, so the loop has no barrier.
template <Source kSrc>
__global__ __launch_bounds__(256, 2) void attend32_kernel(Attn a) {
  __shared__ u32x4 s_kv[4][2][32 * 16];  // a wave's keys and values
  __shared__ float s_m[4][32], s_l[4][32];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, h = lane >> 5;
  const int kvh = (int)blockIdx.x % a.Hkv;
  u32x4 *s_k = s_kv[wave][0], *s_v = s_kv[wave][1];
  constexpr bool kFp8 = kSrc == kPagesFp8;
  constexpr int kUnits = kFp8 ? 8 : 16;      // 16-byte units of a row in memory
  constexpr int kLoads = kUnits / 2;         // per lane and 32 rows
  constexpr int kRowsPer = 64 / kUnits;      // rows per load

  for (int item = (int)blockIdx.x / a.Hkv;; item += a.grid) {
    Place p;
    if constexpr (kSrc == kPacked) {
      if (item >= a.grid) return;
      if (!find_tile(a, kFewRows, a.grid - 1 - item, p, lane)) return;
    } else {
      const int count = *a.n_items;
      if (blockIdx.x == 0 && threadIdx.x == 0 && a.refused &&
          (a.starts[a.seqs] > a.rows || (a.others && *a.others > 0)))
        *a.refused = 1;
      if (item >= count) return;
      const Item &it = a.items[item];
      p.seq = it.seq, p.row0 = it.row0, p.k0 = it.k0, p.k1 = it.k1, p.part = it.part;
      p.start = a.starts[p.seq];
      p.n = a.starts[p.seq + 1] - p.start;
      p.cached = a.lengths[p.seq] - p.n;
    }
    const int n_rows = min(p.n * a.group - p.row0, 32);
    if (n_rows <= 0 || p.start < 0 || p.cached < 0) continue;  // not the planned step's lengths
    // this lane's query: rows past the last repeat it, unstored
    const int row = p.row0 + min(r, n_rows - 1);
    const int tok = row / a.group, head = kvh * a.group + row % a.group;
    const int limit = p.cached + tok;
    const int low = p.cached + p.row0 / a.group;  // the first query's limit
    const int token = min(p.start + tok, a.rows - 1);

    v8bf qf[8];
    const uint16_t *qp = a.q + (int64_t)token * a.q_stride + head * kD + 8 * h;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) qf[kk] = *reinterpret_cast<const v8bf *>(qp + 16 * kk);
    float c = a.scale, vscale = 1.f;
    if constexpr (kFp8) c *= a.ks[kvh], vscale = a.vs[kvh];

    // the row (page, head, offset) of key key0 + (lane & 31); keys past the
    // last repeat it
    const int *table = kSrc == kPacked ? nullptr : a.table + (size_t)p.seq * a.width;
    auto locate = [&](int key0) -> uint32_t {
      const int key = min(key0 + r, p.k1 - 1);
      if constexpr (kSrc == kPacked) return (uint32_t)(p.start + key);
      const uint32_t page = min((uint32_t)table[key >> a.shift], a.pages - 1);
      return ((page * a.Hkv + kvh) << a.shift) + (key & ((1 << a.shift) - 1));
    };
    u32x4 kr[kLoads], vr[kLoads];
    auto load = [&](uint32_t at) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int src = (lane / kUnits) + kRowsPer * i, unit = lane % kUnits;
        const uint32_t w = (uint32_t)__shfl((int)at, src);
        if constexpr (kSrc == kPacked) {
          kr[i] = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.k) +
                                                   (int64_t)w * a.k_stride + kvh * kD + 8 * unit);
          vr[i] = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.v) +
                                                   (int64_t)w * a.v_stride + kvh * kD + 8 * unit);
        } else {
          kr[i] = static_cast<const u32x4 *>(a.k)[(size_t)w * kUnits + unit];
          vr[i] = static_cast<const u32x4 *>(a.v)[(size_t)w * kUnits + unit];
        }
      }
    };
    auto store = [&]() {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int row = (lane / kUnits) + kRowsPer * i, unit = lane % kUnits;
        if constexpr (kFp8) {
          u32x4 w[2];
          widen16(kr[i], w);
          s_k[row * 16 + ((2 * unit) ^ turn(row))] = w[0];
          s_k[row * 16 + ((2 * unit + 1) ^ turn(row))] = w[1];
          widen16(vr[i], w);
          s_v[row * 16 + ((2 * unit) ^ turn(row))] = w[0];
          s_v[row * 16 + ((2 * unit + 1) ^ turn(row))] = w[1];
        } else {
          s_k[row * 16 + (unit ^ turn(row))] = kr[i];
          s_v[row * 16 + (unit ^ turn(row))] = vr[i];
        }
      }
    };

    Wave w;
    w.init();
    int key0 = p.k0 + 32 * wave;
    if (key0 < p.k1) {  // uniform
      uint32_t at = locate(key0);
      load(at);
      at = locate(key0 + 128);
      for (; key0 < p.k1; key0 += 128) {
        wave_fence();
        store();
        wave_fence();
        if (key0 + 128 < p.k1) {
          load(at);
          at = locate(key0 + 256);
        }
        const v16f s = Wave::scores(s_k, qf, lane);
        if (key0 + 31 > low) w.step<true>(s, s_v, key0, limit, c, lane);  // uniform
        else w.step<false>(s, s_v, key0, limit, c, lane);
      }
    }
    float l = w.l + __shfl_xor(w.l, 32);

    // join the waves
    if (h == 0) s_m[wave][r] = w.m, s_l[wave][r] = l;
    __syncthreads();
    const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float f = __builtin_amdgcn_exp2f((w.m - top) * c);
    // 32 rows of 32 units of 4 sums, unit u of row r at u ^ r; over the wave's
    // own keys and values, which it has read
    float4 *so = reinterpret_cast<float4 *>(s_kv[wave]);
    wave_fence();
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        so[r * 32 + ((8 * d + 2 * j + h) ^ r)] =
            make_float4(w.o[d][4 * j] * f, w.o[d][4 * j + 1] * f, w.o[d][4 * j + 2] * f,
                        w.o[d][4 * j + 3] * f);
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * n_rows; i += 256) {
      const int row = i >> 5, u = i & 31;
      float4 t[4];
      float sum = 0.f, mt = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        t[x] = reinterpret_cast<const float4 *>(s_kv[x])[row * 32 + (u ^ row)];
        sum += s_l[x][row] * __builtin_amdgcn_exp2f((s_m[x][row] - mt) * c);
      }
      const float4 all = make_float4((t[0].x + t[1].x) + (t[2].x + t[3].x),
                                     (t[0].y + t[1].y) + (t[2].y + t[3].y),
                                     (t[0].z + t[1].z) + (t[2].z + t[3].z),
                                     (t[0].w + t[1].w) + (t[2].w + t[3].w));
      if (p.part >= 0) {
        const size_t at = ((size_t)p.part * a.Hkv + kvh) * 32 + row;
        reinterpret_cast<float4 *>(a.sums)[at * 32 + u] = all;
        if (u == 0) a.stats[at] = make_float2(mt * c, sum);
      } else {
        const int g = p.row0 + row;
        const int tk = p.start + g / a.group;
        const float inv = vscale / sum;
        if (tk < a.rows)
          *reinterpret_cast<u32x2 *>(a.out + (int64_t)tk * a.out_stride +
                                     (kvh * a.group + g % a.group) * kD + 4 * u) =
              u32x2{pack_bf16(all.x * inv, all.y * inv), pack_bf16(all.z * inv, all.w * inv)};
      }
    }
    __syncthreads();  // the next item's stores come after
  }
}

// The parts of split rows, joined: a wave per row, two dims a lane.
__global__ __launch_bounds__(256) void join_kernel(Attn a, const int *n_joins, const Join *joins,
                                                   int part_rows) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = (int)blockIdx.x % a.Hkv, j = (int)blockIdx.x / a.Hkv;
  if (j >= *n_joins) return;
  const Join jn = joins[j];
  const int start = a.starts[jn.seq], n = a.starts[jn.seq + 1] - start;
  const int n_rows = min(n * a.group - jn.row0, part_rows);
  const float vscale = a.vs ? a.vs[kvh] : 1.f;
  for (int row = 4 * (int)blockIdx.y + wave; row < n_rows; row += 4 * (int)gridDim.y) {
    const size_t at = ((size_t)jn.part * a.Hkv + kvh) * part_rows + row;
    const size_t step = (size_t)a.Hkv * part_rows;
    float top = -INFINITY;
    for (int x = lane; x < jn.n; x += 64) top = fmaxf(top, a.stats[at + x * step].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    float l = 0.f, s0 = 0.f, s1 = 0.f;
    for (int x0 = 0; x0 < jn.n; x0 += 8) {
      float2 v[8], st[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const size_t p = at + min(x0 + u, jn.n - 1) * step;
        v[u] = reinterpret_cast<const float2 *>(a.sums)[p * 64 + lane];
        st[u] = a.stats[p];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (x0 + u >= jn.n) break;
        const float f = __builtin_amdgcn_exp2f(st[u].x - top);
        l = fmaf(f, st[u].y, l);
        s0 = fmaf(f, v[u].x, s0);
        s1 = fmaf(f, v[u].y, s1);
      }
    }
    const int g = jn.row0 + row, tk = start + g / a.group;
    const float inv = vscale / l;
    if (tk < a.rows)
      *reinterpret_cast<uint32_t *>(a.out + (int64_t)tk * a.out_stride +
                                    (kvh * a.group + g % a.group) * kD + 2 * lane) =
          pack_bf16(s0 * inv, s1 * inv);
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
  a.starts = b->starts, a.lengths = b->lengths, a.table = b->table, a.refused = b->refused;
  a.Hkv = b->Hkv, a.group = G, a.rows = (int)rows, a.seqs = b->seqs, a.width = b->width;
  a.shift = __builtin_ctz((unsigned)b->page_size), a.pages = (uint32_t)b->pages;
  a.scale = kLog2e / sqrtf((float)kD);
  const bool many = max_new * G > kFewRows;
  if (G <= kFewRows) {
    a.n_items = &counts->few, a.others = many ? nullptr : &counts->tiles;
    a.items = reinterpret_cast<const Item *>(base + w.few_at);
    a.stats = reinterpret_cast<float2 *>(base + w.few_stats);
    a.sums = reinterpret_cast<float *>(base + w.few_sums);
    a.grid = w.few_parts / 2 + (int)(rows < b->seqs ? rows : b->seqs);
    const unsigned grid = (unsigned)(a.grid * a.Hkv);
    if (fp8) attend32_kernel<kPagesFp8><<<grid, 256, 0, as_stream(stream)>>>(a);
    else attend32_kernel<kPages><<<grid, 256, 0, as_stream(stream)>>>(a);
    join_kernel<<<dim3((unsigned)(w.few_parts / 2 * a.Hkv), 1), 256, 0, as_stream(stream)>>>(
        a, &counts->few_joins, reinterpret_cast<const Join *>(base + w.few_joins_at), kFewRows);
  }
  if (many) {
    a.n_items = &counts->tiles, a.others = nullptr;
    a.items = reinterpret_cast<const Item *>(base + w.tiles_at);
    a.stats = reinterpret_cast<float2 *>(base + w.tile_stats);
    a.sums = reinterpret_cast<float *>(base + w.tile_sums);
    const int64_t items = rows * G / kTileRows + (rows < b->seqs ? rows : b->seqs) + w.tile_parts;
    a.grid = (int)(items < w.tile_items ? items : w.tile_items);
    const unsigned grid = (unsigned)(a.grid * a.Hkv);
    if (fp8) attend32_kernel<kPagesFp8><<<grid, 256, 0, as_stream(stream)>>>(a);
    else attend32_kernel<kPages><<<grid, 256, 0, as_stream(stream)>>>(a);
    join_kernel<<<dim3((unsigned)(w.tile_parts / 2 * a.Hkv), kTileRows / 32), 256, 0,
                  as_stream(stream)>>>(
        a, &counts->tile_joins, reinterpret_cast<const Join *>(base + w.tile_joins_at), kTileRows);
  }
  return launched();
}

extern "C" int ecf8_ragged_attention(const void *q, int64_t q_stride, const void *k,
                                     int64_t k_stride, const void *v, int64_t v_stride,
                                     int64_t rows, const int *starts, int64_t seqs, int Hq,
                                     int Hkv, void *out, int64_t out_stride, void *stream) {
  if (!q || !k || !v || !starts || !out || rows <= 0 || seqs <= 0 || Hq <= 0 || Hkv <= 0)
    return ECF8_ERR_INVALID_ARG;
  const int64_t wide = (int64_t)Hq * kD, kv = (int64_t)Hkv * kD;
  if (!sizes_ok(seqs, rows, Hq, Hkv) || q_stride % 8 || k_stride % 8 || v_stride % 8 ||
      out_stride % 4 || (rows > 1 && (q_stride < wide || out_stride < wide || k_stride < kv ||
                                      v_stride < kv)))
    return ECF8_ERR_UNSUPPORTED;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 8) ||
      !aligned(starts, 4))
    return ECF8_ERR_MISALIGNED;
  Attn a{};
  a.q = static_cast<const uint16_t *>(q), a.out = static_cast<uint16_t *>(out);
  a.k = k, a.v = v;
  a.q_stride = q_stride, a.out_stride = out_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.starts = starts;
  a.Hkv = Hkv, a.group = Hq / Hkv, a.rows = (int)rows, a.seqs = (int)seqs;
  a.scale = kLog2e / sqrtf((float)kD);
  a.grid = (int)(rows * a.group / kFewRows + seqs);
  attend32_kernel<kPacked><<<(unsigned)((int64_t)a.grid * Hkv), 256, 0, as_stream(stream)>>>(a);
  return launched();
}
