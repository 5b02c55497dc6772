// Speculative decoding on gfx950, but for the trees' attention: the trees' masks,
// positions and schedule, the target's probabilities, their verification and
// the move of the accepted rows in the cache.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ecf8.h"
#include "ecf8_dev.h"
#include "ecf8_draft.h"
#include "ecf8_draft_layout.h"

namespace {

using namespace ecf8::draft;
using ecf8::paged::kMaxSeqs;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
// the same at any address of their elements
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef v4f v4f_any __attribute__((aligned(4)));

__device__ __forceinline__ float bf16_f32(uint32_t h16) { return __uint_as_float(h16 << 16); }

// --------------------------------------------------------------- the plan

struct Plan {
  const int *starts, *lengths, *parents;
  uint64_t *masks;
  int *out_parents, *positions, *refused;
  Counts *counts;
  Item *items;
  Join *joins;
  int seqs, rows, all_rows, group, max_nodes, max_children, tile, target;
  uint64_t stamp;
  const uint64_t *step;  // the batch's
};

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kPer = kMaxSeqs / kPlanThreads;
constexpr int kLeast = 1;  // units on both sides of a cut
// What a workgroup's first loads and last sums take, in units.  64 trees after 512
// keys: of 8 tokens 25 us, 28.5 with one; of 32 42 and 50; few long ones alike.
constexpr int kBegin = 5;

// The exclusive prefix sums of N values over the workgroup, and their totals.
// Calls in a row alternate between two halves of `waves`.
template <int N>
__device__ __forceinline__ void block_scan(const int (&v)[N], int (*waves)[kPlanWaves],
                                           int (&before)[N], int (&total)[N]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int inc[N];
#pragma unroll
  for (int x = 0; x < N; ++x) {
    inc[x] = ecf8::dev::wave_inclusive_scan(v[x]);
    if (lane == 63) waves[x][wave] = inc[x];
  }
  __syncthreads();
#pragma unroll
  for (int x = 0; x < N; ++x) {
    before[x] = inc[x] - v[x], total[x] = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
      const int t = waves[x][w];
      if (w < wave) before[x] += t;
      total[x] += t;
    }
  }
}

// A wave's tree: lane t is row t.  A row's mask is the union of the parents' on
// the way up, in six doublings.
__device__ __forceinline__ void plan_tree(const Plan &a, int s) {
  const int lane = threadIdx.x & 63;
  const int start = a.starts[s], n = a.starts[s + 1] - start;
  if (n <= 0) return;
  const int cached = a.lengths[s] - n;
  if (n > a.max_nodes || start < 0 || start > a.rows - n || cached < 0) {
    for (int t = lane; t < n; t += 64)
      if (start >= 0 && start + t < a.all_rows) {
        a.masks[start + t] = 0;
        a.out_parents[start + t] = -1;
      }
    if (lane == 0 && a.refused) *a.refused = 1;
    return;
  }
  int up = lane < n ? a.parents[start + lane] : -1;
  bool bad = lane < n && (lane ? up < 0 || up >= lane : up != -1);
  int before = 0;  // earlier rows of the same parent
  for (int k = 0; k < n; ++k) before += k < lane && __builtin_amdgcn_readlane(up, k) == up;
  bad |= lane > 0 && lane < n && before >= a.max_children;
  if (__any(bad)) {
    up = -1;
    if (lane == 0 && a.refused) *a.refused = 1;
  }
  const int parent = up;
  uint64_t bits = 1ull << lane;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const uint64_t above = __shfl(bits, up & 63);
    const int next = __shfl(up, up & 63);
    if (up >= 0) bits |= above, up = next;
  }
  if (lane < n) {
    a.masks[start + lane] = bits;
    a.out_parents[start + lane] = parent;
    a.positions[start + lane] = cached + __popcll(bits) - 1;
  }
}

// Buckets of lengths, the longest first.
constexpr int kBuckets = 64;
__device__ __forceinline__ int bucket_of(int length, int share) {
  return kBuckets - 1 - min(kBuckets - 1, (int)(48ll * length / share));
}

// The attention's schedule, by one workgroup.  Every (sequence, tile of rows)
// has ceil(length / kUnitKeys) units, and kBegin for its first loads and last
// sums; laid end to end they are cut at the multiples of a workgroup's share, and
// the pieces listed from the longest on.
__device__ __forceinline__ void plan_schedule(const Plan &a) {
  __shared__ int s_first[kMaxSeqs + 1];  // tiles before a sequence's
  __shared__ int s_waves[2][2][kPlanWaves];
  __shared__ int s_bucket[kBuckets];
  const int tid = threadIdx.x, S = a.seqs;
  const int step = (S + kPlanThreads - 1) / kPlanThreads;
  if (tid < kBuckets) s_bucket[tid] = 0;
  int tiles[kPer], sum = 0, units = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = step * tid + i;
    tiles[i] = 0;
    if (i >= step || s >= S) continue;
    const int start = a.starts[s], n = a.starts[s + 1] - start, len = a.lengths[s];
    if (n < 1 || n > a.max_nodes || start < 0 || start > a.rows - n || len < n) continue;
    tiles[i] = (n * a.group + a.tile - 1) / a.tile;
    sum += tiles[i];
    units += tiles[i] * ((len + kUnitKeys - 1) / kUnitKeys + kBegin);
  }
  // (the sum of all can pass 32 bits, a thread's cannot)
  const int one[1] = {sum}, halves[2] = {units & 0xffff, units >> 16};
  int at[1], n_tiles[1], skip[2], all[2];
  block_scan(one, s_waves[0], at, n_tiles);
  block_scan(halves, s_waves[1], skip, all);
  const int64_t exact = (((int64_t)all[1] << 16) + all[0] + a.target - 1) / a.target;
  const int share = (int)min(max(exact, (int64_t)2 * kLeast), (int64_t)1 << 29);
  {
    int first = at[0];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int s = step * tid + i;
      if (i < step && s < S) s_first[s] = first;
      first += tiles[i];
    }
    if (tid == 0) s_first[S] = n_tiles[0];
  }
  __syncthreads();
  int n_items = 0, n_joins = 0, parts = 0, from0 = 0;  // from0: mod share
  // This thread's tile of a thousand, its units before it, pieces and their places.
  struct Tile {
    Item it;
    int len, units, f, c0, k, part, join;
  } mine{};
  auto take = [&](int i0) {
    const int i = i0 + tid;
    Tile t{};
    if (i < n_tiles[0]) {
      int lo = 0, hi = S;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_first[mid] <= i) lo = mid;
        else hi = mid;
      }
      t.it.seq = lo, t.it.row0 = (i - s_first[lo]) * a.tile;
      t.it.start = a.starts[lo], t.it.n = a.starts[lo + 1] - t.it.start;
      t.len = a.lengths[lo], t.it.cached = t.len - t.it.n;
      t.units = (t.len + kUnitKeys - 1) / kUnitKeys;
    }
    const int all_units[1] = {t.units ? t.units + kBegin : 0};
    int from[1], total[1];
    block_scan(all_units, s_waves[0], from, total);
    t.f = from0 + from[0] + kBegin;
    t.c0 = (t.f + kLeast + share - 1) / share;
    const int c1 = (t.f + t.units - kLeast) / share;
    t.k = t.units ? max(0, c1 - t.c0 + 1) + 1 : 0;
    const int cut[2] = {t.k > 1 ? t.k : 0, t.k > 1};
    int before[2], all_cut[2];
    block_scan(cut, s_waves[1], before, all_cut);
    t.part = parts + before[0], t.join = n_joins + before[1];
    parts += all_cut[0], n_joins += all_cut[1];
    from0 = (from0 + total[0]) % share;
    mine = t;
  };
  // Twice over the tiles: count the pieces of each length, then write them.
  for (int write = 0; write < 2; ++write) {
    if (n_tiles[0] > kPlanThreads) from0 = parts = n_joins = 0;
    for (int i0 = 0; i0 < n_tiles[0]; i0 += kPlanThreads) {  // uniform
      if (!write || n_tiles[0] > kPlanThreads) take(i0);  // (a thousand are kept)
      for (int j = 0; j < mine.k; ++j) {
        const int u0 = j ? (mine.c0 + j - 1) * share - mine.f : 0;
        const int u1 = j + 1 < mine.k ? (mine.c0 + j) * share - mine.f : mine.units;
        const int to = atomicAdd(&s_bucket[bucket_of(u1 - u0, share)], 1);
        if (write) {
          Item it = mine.it;
          it.k0 = u0 * kUnitKeys, it.k1 = min(u1 * kUnitKeys, mine.len);
          it.part = mine.k > 1 ? mine.part + j : -1;
          a.items[to] = it;
        }
      }
      if (write && mine.k > 1)
        a.joins[mine.join] =
            Join{mine.it.row0, mine.part, mine.k, mine.it.start, mine.it.n, {0, 0, 0}};
    }
    __syncthreads();
    if (!write) {
      const int count[1] = {tid < kBuckets ? s_bucket[tid] : 0};
      int first[1], total[1];
      block_scan(count, s_waves[0], first, total);
      if (tid < kBuckets) s_bucket[tid] = first[0];
      n_items = total[0];
      __syncthreads();
    }
  }
  if (tid == 0) a.counts->items = n_items, a.counts->joins = n_joins, a.counts->stamp = a.stamp;
}

// The first workgroup schedules, the others take 16 sequences' trees each.  Latency of
// loads, scans and barriers in a row: 6.6 us of 16 trees, 6.7 of 512.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(Plan a) {
  if (blockIdx.x == 0) {
    plan_schedule(a);
  } else {
    if (blockIdx.x == 1 && threadIdx.x == 0) a.counts->step = *a.step;  // (6.9 us in the first)
    const int s = ((int)blockIdx.x - 1) * kPlanWaves + (int)(threadIdx.x >> 6);
    if (s < a.seqs) plan_tree(a, s);
  }
}

// -------------------------------------------------------- probabilities

constexpr double kLog2e = 1.4426950408889634;

struct Probs {
  const uint16_t *logits;
  float *out;
  const float *temperature;
  int64_t ld, ldo;
  uint2 *work;  // [rows, kChunks]
  float common;
  int V, chunks;
};

// log2(e) / temperature in two parts, hi cut off and lo above zero, so that both
// products of -inf are -inf.
struct Scale {
  float hi, lo;
  bool greedy;
  __device__ __forceinline__ explicit Scale(float t) {
    greedy = t <= 0.f;
    // (finite and above zero, so that -inf times it is -inf)
    const double c = fmin(fmax(kLog2e / (double)t, 0x1p-100), 0x1p100);
    hi = (float)c;
    if ((double)hi >= c) hi = __uint_as_float(__float_as_uint(hi) - 1);
    lo = fmaxf((float)(c - (double)hi), 0x1p-126f);
    if (t != t) hi = t;
  }
  // exp(x / temperature), x <= 0; NaN of NaN.  The first part alone would leave all
  // terms of a row, and so their sum, off by up to 2^-24 of their exponents, more than
  // all else together: 5 rows of 151936 1.8e-7 from 64 bits, 0.9e-7 with both.
  __device__ __forceinline__ float exp(float x) const {
    return __builtin_amdgcn_exp2f(fmaf(x, hi, x * lo));
  }
};

// Sort key of a logit at index i as in ecf8_greedy_emit: larger is better, NaN
// above everything, equal values to the lower index.
__device__ __forceinline__ uint64_t logit_key(uint32_t h, uint32_t i) {
  uint32_t k;
  if ((h & 0x7fffu) > 0x7f80u) k = 0x1ffffu;
  else if ((h & 0x7fffu) == 0) k = 0x8000u;
  else k = h & 0x8000u ? 0x8000u - (h & 0x7fffu) : 0x8000u + h;
  return ((uint64_t)k << 32) | (uint32_t)~i;
}

template <class Vec>
__device__ __forceinline__ float logit(Vec v, int j) {
  return j & 1 ? __uint_as_float(v[j >> 1] & 0xffff0000u) : bf16_f32(v[j >> 1] & 0xffffu);
}

// A thread's part of a run of a row: units of kUnit logits, kAtOnce of them in
// flight; units(u, n, v): n units from u on, 256 apart.  The row's last V mod
// kUnit come one each to the first threads of the last run: single(i, logit).
constexpr int kAtOnce = 4;
template <int kUnit, class VecAny, class Vec, class Units, class Single>
__device__ __forceinline__ void for_run(const Probs &a, int row, Vec, Units units,
                                        Single single) {
  const uint16_t *x = a.logits + (int64_t)row * a.ld;
  const int whole = a.V / kUnit, per = (whole + a.chunks - 1) / a.chunks;
  const int u0 = blockIdx.x * per, u1 = min(u0 + per, whole);
  for (int u = u0 + (int)threadIdx.x; u < u1; u += 256 * kAtOnce) {
    Vec v[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      v[i] = *reinterpret_cast<const VecAny *>(x + kUnit * (int64_t)min(u + 256 * i, u1 - 1));
    units(u, min(kAtOnce, (u1 - u + 255) / 256), v);
  }
  if (blockIdx.x == a.chunks - 1 && (int)threadIdx.x < a.V % kUnit) {
    const int i = kUnit * whole + (int)threadIdx.x;
    single(i, x[i]);
  }
}

// The largest logit of a run of a row and the sum of the exponentials below it;
// greedy rows: the best key.  Bound by HBM: 416 rows of 151936 (126 MB) 28.5 us, 4.4
// TB/s; the second kernel (253 MB written) 46 us, 5.5 TB/s.
__global__ __launch_bounds__(256) void probability_stats_kernel(Probs a) {
  __shared__ uint64_t s_k[4];
  __shared__ float s_m[4], s_l[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = blockIdx.y;
  const Scale c(a.temperature ? a.temperature[row] : a.common);
  uint2 *out = a.work + (size_t)row * ECF8_PROBABILITY_CHUNKS + blockIdx.x;
  if (c.greedy) {  // uniform
    uint64_t best = 0;
    auto take = [&](uint32_t h, int i) {
      const uint64_t k = logit_key(h, i);
      best = k > best ? k : best;
    };
    for_run<8, u32x4_any>(
        a, row, u32x4{},
        [&](int u, int n, const u32x4(&v)[kAtOnce]) {
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i)
            if (i < n)
#pragma unroll
              for (int j = 0; j < 8; ++j)
                take((v[i][j >> 1] >> (16 * (j & 1))) & 0xffffu, 8 * (u + 256 * i) + j);
        },
        [&](int i, uint32_t h) { take(h, i); });
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t k = __shfl_xor(best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) s_k[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 4; ++i) best = s_k[i] > best ? s_k[i] : best;
      *out = make_uint2((uint32_t)best, (uint32_t)(best >> 32));
    }
    return;
  }
  // m: -inf while nothing else was there; sums from it count from 0 then, which
  // -inf leaves at 0 and NaN makes NaN
  float m = -INFINITY, l = 0.f;
  auto raise = [&](float top) {
    if (top > m) l *= m == -INFINITY ? 1.f : c.exp(m - top), m = top;
    return m == -INFINITY ? 0.f : m;
  };
  for_run<8, u32x4_any>(
      a, row, u32x4{},
      [&](int u, int n, const u32x4(&v)[kAtOnce]) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) top = fmaxf(top, logit(v[i], j));
        const float from = raise(top);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (i < n)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j & 1] += c.exp(logit(v[i], j) - from);
        l += sum[0] + sum[1];
      },
      [&](int i, uint32_t h) {
        const float y = bf16_f32(h);
        l += c.exp(y - raise(y));
      });
  auto join = [&](float m2, float l2) {
    const float top = fmaxf(m, m2);
    l = (m == -INFINITY ? l : l * c.exp(m - top)) + (m2 == -INFINITY ? l2 : l2 * c.exp(m2 - top));
    m = top;
  };
  for (int o = 32; o > 0; o >>= 1) {
    const float m2 = __shfl_xor(m, o), l2 = __shfl_xor(l, o);
    join(m2, l2);
  }
  if (lane == 0) s_m[wave] = m, s_l[wave] = l;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 4; ++i) join(s_m[i], s_l[i]);
    *out = make_uint2(__float_as_uint(m), __float_as_uint(l));
  }
}

// kPast: stores go past the caches, so that the logits, read twice, stay there.
template <bool kPast>
__global__ __launch_bounds__(256) void probability_kernel(Probs a) {
  const int lane = threadIdx.x & 63, row = blockIdx.y;
  float *out = a.out + (int64_t)row * a.ldo;
  const Scale c(a.temperature ? a.temperature[row] : a.common);
  const uint2 st = a.work[(size_t)row * ECF8_PROBABILITY_CHUNKS + min(lane, a.chunks - 1)];
  auto put = [&](int i, v4f p) {
    v4f_any *to = reinterpret_cast<v4f_any *>(out + i);
    if constexpr (kPast) __builtin_nontemporal_store(p, to);
    else *to = p;
  };
  if (c.greedy) {  // uniform
    uint64_t best = ((uint64_t)st.y << 32) | st.x;
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t k = __shfl_xor(best, o);
      best = k > best ? k : best;
    }
    const int at = (int)~(uint32_t)best;
    const int whole = a.V / 4, per = (whole + a.chunks - 1) / a.chunks;
    const int u1 = min((int)(blockIdx.x + 1) * per, whole);
    for (int u = blockIdx.x * per + (int)threadIdx.x; u < u1; u += 256) {
      const int i = at - 4 * u;
      put(4 * u, v4f{i == 0 ? 1.f : 0.f, i == 1 ? 1.f : 0.f, i == 2 ? 1.f : 0.f,
                     i == 3 ? 1.f : 0.f});
    }
    if (blockIdx.x == a.chunks - 1 && (int)threadIdx.x < a.V % 4) {
      const int i = 4 * whole + (int)threadIdx.x;
      out[i] = i == at ? 1.f : 0.f;
    }
    return;
  }
  const float m0 = __uint_as_float(st.x);
  float m = m0;
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  // (lanes past the last run: nothing)
  float l = lane >= a.chunks ? 0.f : __uint_as_float(st.y);
  if (m0 != -INFINITY) l *= c.exp(m0 - m);
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  // a row with a NaN, an infinity or nothing but -inf is NaN throughout
  const float inv = l > 0.f && l < INFINITY ? 1.f / l : NAN;
  for_run<4, u32x2_any>(
      a, row, u32x2{},
      [&](int u, int n, const u32x2(&v)[kAtOnce]) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (i < n) {
            v4f p;
#pragma unroll
            for (int j = 0; j < 4; ++j) p[j] = c.exp(logit(v[i], j) - m) * inv;
            put(4 * (u + 256 * i), p);
          }
      },
      [&](int i, uint32_t h) { out[i] = c.exp(bf16_f32(h) - m) * inv; });
}

// --------------------------------------------------------- verification

// What says whether trees were planned for the batch's step.
struct Planned {
  const Counts *counts;
  const uint64_t *step;
  uint64_t stamp;
  __device__ __forceinline__ bool now() const {
    return (int)(counts->stamp == stamp) & (int)(counts->step == *step);
  }
  // (neither, of trees that never were planned)
  __device__ __forceinline__ bool other() const { return !now() && counts->stamp != 0; }
};

// Where a sequence's walk ended, for the kernel that draws its next token.
struct Ended {
  int64_t row;                // packed row whose w is drawn from, -1: none
  int kept, gone, n_tokens, pad;
  int64_t tokens[kMaxNodes];  // that are gone from w
  double inv[kMaxNodes];      // 1 / Z of the levels that are gone
};
static_assert(sizeof(Ended) <= kEndedBytes, "the layout has room for it");

struct Verify {
  const int *starts, *parents;
  const int64_t *tokens;
  const float *target, *draft, *accept, *sample;
  int64_t ld_target, ld_draft;
  int *kept, *path, *refused;
  int64_t *emitted, *next_token;
  double *runs, *mass;  // [2, seqs, kRuns], [max_children - 1, nodes, kRuns]
  Ended *ended;         // [seqs]
  int64_t nodes;
  int seqs, rows, V, max_nodes, max_children, packed;
  int per, lanes;  // runs a workgroup, threads a run
  Planned planned;
};

// Lane i's value, for an i that is the same in all lanes (a read of a scalar
// register's worth, where a shuffle goes through LDS).
__device__ __forceinline__ int lane_of(int v, int i) {
  return __builtin_amdgcn_readlane(v, __builtin_amdgcn_readfirstlane(i));
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int i) {
  return (uint64_t)(uint32_t)lane_of((int)(v >> 32), i) << 32 | (uint32_t)lane_of((int)v, i);
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int i) {
  return (int64_t)lane_of((uint64_t)v, i);
}
__device__ __forceinline__ double lane_of(double v, int i) {
  return __longlong_as_double((long long)lane_of((uint64_t)__double_as_longlong(v), i));
}

// The inclusive prefix sum over the wave (see ecf8::dev::wave_inclusive_scan), and
// the sum.
template <int kCtrl, int kRows>
__device__ __forceinline__ double dpp_or_zero(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)u, kCtrl, kRows, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), kCtrl, kRows, 0xF, false);
  return __longlong_as_double((long long)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo));
}
__device__ __forceinline__ double wave_scan(double v) {
  v += dpp_or_zero<0x111, 0xF>(v);  // row_shr:1
  v += dpp_or_zero<0x112, 0xF>(v);  // row_shr:2
  v += dpp_or_zero<0x114, 0xF>(v);  // row_shr:4
  v += dpp_or_zero<0x118, 0xF>(v);  // row_shr:8
  v += dpp_or_zero<0x142, 0xA>(v);  // row_bcast:15
  v += dpp_or_zero<0x143, 0xC>(v);  // row_bcast:31
  return v;
}
__device__ __forceinline__ double wave_sum(double v) { return lane_of(wave_scan(v), 63); }

// What a wave knows of a sequence's tree, lane t of row t.
struct Tree {
  int start, n, up, rank;  // rank: earlier rows of the same parent
  int64_t token;
  bool in;                 // the token is one of the vocabulary
  double u, p, q;          // q, p: of the token, after the parent
  uint64_t kids, above;    // children; ancestors and itself
};

// false: nothing to verify.
template <bool kDrawn>
__device__ __forceinline__ bool load_tree(const Verify &a, int s, Tree &t) {
  const int lane = threadIdx.x & 63;
  t.start = a.starts[s], t.n = a.starts[s + 1] - t.start;
  const bool planned = a.planned.now();
  if (!planned || t.n < 1 || t.n > a.max_nodes || t.start < 0 || t.start > a.rows - t.n)
    return false;
  const int row = t.start + min(lane, t.n - 1);
  t.up = lane < t.n ? a.parents[row] : -1;
  if (t.up >= lane) t.up = -1;  // (of parents that were written over)
  t.token = a.tokens[row];
  t.in = t.token >= 0 && t.token < a.V;
  t.u = (double)a.accept[row];
  const int64_t after = t.start + max(t.up, 0), c = t.in ? t.token : 0;
  t.p = t.in ? (double)a.target[after * a.ld_target + c] : 0.0;
  t.q = kDrawn && t.in ? (double)a.draft[after * a.ld_draft + c] : 0.0;
  t.kids = 0;
  for (int k = 1; k < t.n; ++k)
    if (__builtin_amdgcn_readlane(t.up, k) == lane) t.kids |= 1ull << k;
  t.rank = __popcll(__shfl(t.kids, t.up & 63) & ((1ull << lane) - 1));
  t.above = 1ull << lane;
  int up = t.up;
#pragma unroll
  for (int i = 0; i < 6; ++i) {
    const uint64_t more = __shfl(t.above, up & 63);
    const int next = __shfl(up, up & 63);
    if (up >= 0) t.above |= more, up = next;
  }
  return true;
}

// Where the walk ends: the last accepted row and its rejected children.
struct End {
  int last;
  uint64_t gone;
};

// Drafts that are different tokens: what is left of w is Z less the rejected.
__device__ __forceinline__ End walk_top(const Tree &t) {
  End e{0, 0};
  for (;;) {
    uint64_t kids = lane_of(t.kids, e.last);
    double mass = 1.0;
    e.gone = 0;
    int next = -1;
    while (kids) {
      const int j = __builtin_ctzll(kids);
      kids &= kids - 1;
      const int64_t c = lane_of(t.token, j);
      // (a token that was rejected is not left)
      const bool twice = __any(((e.gone >> (threadIdx.x & 63)) & 1) && t.token == c);
      const double w = twice ? 0.0 : lane_of(t.p, j), u = lane_of(t.u, j);
      if (u * mass < w) {
        next = j;
        break;
      }
      mass -= w;
      e.gone |= 1ull << j;
    }
    if (next < 0) return e;
    e.last = next;
  }
}

// Drafts that were drawn.  Lane t tries row t's children as far as the sums Z of
// `known` levels allow; s_inv[l][t]: 1 / Z after l rejections (l = 0: 1).  Sums
// exist of rows that the walk could still reach when they were taken.  Returns
// the rows that need the next level's, of those the walk can reach.
struct Tried {
  int next, gone;  // accepted child or -1; rejected children
  bool open;       // children are left to be tried
  bool reached;
};
__device__ __forceinline__ uint64_t try_drawn(const Verify &a, int s, const Tree &t, int known,
                                              double (*s_inv)[64], Tried &r) {
  const int lane = threadIdx.x & 63;
  r = Tried{-1, 0, lane < t.n && t.kids != 0, false};
  uint64_t left = t.kids;
  double z = 1.0;
  s_inv[0][lane] = 1.0;
  for (int l = 0;; ++l) {
    // child l of the rows that rejected all before it; all lanes take part in the
    // exchange
    const int j = left ? __builtin_ctzll(left) : 0;
    const double u = __shfl(t.u, j), q = __shfl(t.q, j);
    double w = __shfl(t.p, j);
    if (r.open) {
      for (int x = 0; x < l; ++x) w = fmax(fma(w, s_inv[x][lane], -q), 0.0);
      if (u * q * z < w) {
        r.next = j, r.open = false;
      } else {
        left &= left - 1, ++r.gone;
        r.open = left != 0;
      }
    }
    const bool up_open = __shfl((int)r.open, t.up & 63);
    const int up_next = __shfl(r.next, t.up & 63), up_gone = __shfl(r.gone, t.up & 63);
    const bool ok = lane == 0 || (lane < t.n && t.up >= 0 &&
                                  (up_open ? t.rank >= up_gone : up_next == lane));
    r.reached = lane < t.n && (t.above & ~__ballot(ok)) == 0;
    const uint64_t need = __ballot(r.open && r.reached);
    if (l == known || !need) return need;
    for (uint64_t m = need; m; m &= m - 1) {
      const int i = __builtin_ctzll(m);
      const int64_t node = a.packed ? t.start + i : (int64_t)s * a.max_nodes + i;
      const double sum = wave_sum(a.mass[(l * a.nodes + node) * kRuns + lane]);
      if (lane == i) z = sum;
    }
    s_inv[l + 1][lane] = 1.0 / z;
    if (r.open && !r.reached) r.open = false;  // nobody asks any more
  }
}

__device__ __forceinline__ int run_length(int V) { return ((V + kRuns - 1) / kRuns + 3) / 4 * 4; }

// What is left of the target's row p after `gone` drawn drafts of row q, or without
// some tokens.
struct Row {
  const float *p, *q;
  int gone, n_tokens;
  const double *inv;
  const int64_t *tokens;

  // four elements from v on; those at or past `end` are zero
  __device__ __forceinline__ void load(int v, int end, v4f &pv, v4f &qv) const {
    pv = qv = v4f{};
    if (v + 4 <= end) {
      pv = *reinterpret_cast<const v4f_any *>(p + v);
      if (gone) qv = *reinterpret_cast<const v4f_any *>(q + v);
    } else {
      for (int j = 0; j < 4; ++j)
        if (v + j < end) {
          pv[j] = p[v + j];
          if (gone) qv[j] = q[v + j];
        }
    }
  }
  __device__ __forceinline__ void left(int v, v4f pv, v4f qv, bool some, double (&w)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (double)pv[j];
    for (int x = 0; x < gone; ++x) {
      const double f = inv[x];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = fmax(fma(w[j], f, -(double)qv[j]), 0.0);
    }
    if (some)
      for (int x = 0; x < n_tokens; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (tokens[x] == v + j) w[j] = 0.0;
  }
  // is a token of [lo, end) gone?
  __device__ __forceinline__ bool any_token(int64_t lo, int64_t end) const {
    bool some = false;
    for (int x = 0; x < n_tokens; ++x) some |= tokens[x] >= lo && tokens[x] < end;
    return some;
  }
};

// The sums over a workgroup's runs of w and, kWhole, of p: done(run, w, p) is called
// by the first of a run's threads.  One or all four waves take a run, kUnits units of
// four elements in flight.
constexpr int kUnits = 2;
template <bool kWhole, class Done>
__device__ __forceinline__ void sum_runs(const Verify &a, const Row &r, Done done) {
  __shared__ double s_sum[2][4];
  const int len = run_length(a.V), l = (int)threadIdx.x % a.lanes;
  for (int x = (int)threadIdx.x / a.lanes; x < a.per; x += 256 / a.lanes) {
    const int run = blockIdx.x * a.per + x;
    const int64_t lo = min((int64_t)run * len, (int64_t)a.V);
    const int end = (int)min(lo + len, (int64_t)a.V);
    const bool some = r.any_token(lo, end);
    double sum = 0.0, whole = 0.0;
    const int step = 4 * a.lanes;
    for (int64_t v = lo + 4 * l; v < end; v += kUnits * step) {
      v4f pv[kUnits], qv[kUnits];
#pragma unroll
      for (int i = 0; i < kUnits; ++i)
        r.load((int)min(v + i * step, (int64_t)end), end, pv[i], qv[i]);
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        double w[4];
        r.left((int)v + i * step, pv[i], qv[i], some, w);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
        if constexpr (kWhole)
          whole += ((double)pv[i][0] + (double)pv[i][1]) + ((double)pv[i][2] + (double)pv[i][3]);
      }
    }
    sum = wave_sum(sum);
    if constexpr (kWhole) whole = wave_sum(whole);
    if (a.lanes > 64) {  // uniform
      __syncthreads();
      if ((threadIdx.x & 63) == 0)
        s_sum[0][threadIdx.x >> 6] = sum, s_sum[1][threadIdx.x >> 6] = whole;
      __syncthreads();
      sum = (s_sum[0][0] + s_sum[0][1]) + (s_sum[0][2] + s_sum[0][3]);
      whole = (s_sum[1][0] + s_sum[1][1]) + (s_sum[1][2] + s_sum[1][3]);
    }
    if (l == 0 && run < kRuns) done(run, sum, whole);
  }
}

// Level `level`: the sums of what `level` rejected children leave, by runs of
// the vocabulary, of every row whose next child needs it.
__global__ __launch_bounds__(256) void mass_kernel(Verify a, int level) {
  extern __shared__ double s_dyn[];  // [level][64]
  double(*s_inv)[64] = reinterpret_cast<double(*)[64]>(s_dyn);
  __shared__ double s_f[kMaxNodes];
  __shared__ uint64_t s_need;
  const int s = blockIdx.y;
  Tree t;
  if (!load_tree<true>(a, s, t)) return;
  if (threadIdx.x < 64) {
    Tried r;
    const uint64_t need = try_drawn(a, s, t, level - 1, s_inv, r);
    if (threadIdx.x == 0) s_need = need;
  }
  __syncthreads();
  for (uint64_t need = s_need; need; need &= need - 1) {
    const int i = __builtin_ctzll(need);
    __syncthreads();
    if ((int)threadIdx.x < level) s_f[threadIdx.x] = s_inv[threadIdx.x][i];
    __syncthreads();
    const int64_t row = t.start + i;
    const int64_t node = a.packed ? row : (int64_t)s * a.max_nodes + i;
    const Row r{a.target + row * a.ld_target, a.draft + row * a.ld_draft, level, 0, s_f, nullptr};
    sum_runs<false>(a, r, [&](int run, double sum, double) {
      a.mass[((level - 1) * a.nodes + node) * kRuns + run] = sum;
    });
  }
}

// The end of each walk: what was accepted, and the sums of the last row's w and of
// its target probabilities by runs.  Latency, of loads that wait for each other: starts,
// the tree, its tokens' probabilities, the row.  (A launch of its own for the draw
// that follows takes 6 us; drawing in the last of a sequence's workgroups to finish
// needs each of them to write back L2: 36 us for 16 sequences instead of 17.)
template <bool kDrawn>
__global__ __launch_bounds__(256) void last_kernel(Verify a) {
  extern __shared__ double s_dyn[];  // [max_children][64]
  __shared__ Ended s_end;
  const int s = blockIdx.y, lane = threadIdx.x & 63;
  const bool first = blockIdx.x == 0;  // writes what was accepted
  int *path = a.path + (size_t)s * a.max_nodes;
  int64_t *emitted = a.emitted + (size_t)s * a.max_nodes;
  Tree t;
  if (!load_tree<kDrawn>(a, s, t)) {  // uniform, and in all workgroups alike
    if (first && (int)threadIdx.x < a.max_nodes) path[threadIdx.x] = -1, emitted[threadIdx.x] = -1;
    if (first && threadIdx.x == 0) {
      a.kept[s] = 0, a.next_token[s] = -1, a.ended[s].row = -1;
      if (a.refused && (t.n != 0 || (s == 0 && a.starts[a.seqs] > a.rows))) *a.refused = 1;
    }
    return;
  }
  if (threadIdx.x < 64) {
    int last, gone = 0, n_tokens = 0;
    if constexpr (kDrawn) {
      double(*s_inv)[64] = reinterpret_cast<double(*)[64]>(s_dyn);
      Tried r;
      try_drawn(a, s, t, a.max_children - 1, s_inv, r);
      const uint64_t ends = __ballot(r.reached && r.next < 0);
      last = ends ? __builtin_ctzll(ends) : 0;
      gone = lane_of(r.gone, last);
      if (lane < gone) s_end.inv[lane] = s_inv[lane][last];
    } else {
      const End w = walk_top(t);
      last = w.last, n_tokens = __popcll(w.gone);
      if ((w.gone >> lane) & 1) s_end.tokens[__popcll(w.gone & ((1ull << lane) - 1))] = t.token;
    }
    const uint64_t way = lane_of(t.above, last);
    const int kept = __popcll(way);
    if (lane == 0)
      s_end.row = t.start + last, s_end.kept = kept, s_end.gone = gone, s_end.n_tokens = n_tokens;
    if (first) {
      const int place = __popcll(way & ((1ull << lane) - 1));
      if ((way >> lane) & 1) {
        path[place] = lane;
        if (place > 0) emitted[place - 1] = t.token;
      }
      if (lane >= kept && lane < a.max_nodes) path[lane] = -1, emitted[lane] = -1;
      const bool strange = __any(lane > 0 && lane < t.n && !t.in);
      if (lane == 0) {
        a.kept[s] = kept;
        if (a.refused && (strange || (s == 0 && a.starts[a.seqs] > a.rows))) *a.refused = 1;
      }
    }
  }
  __syncthreads();
  const Row r{a.target + s_end.row * a.ld_target,
              kDrawn ? a.draft + s_end.row * a.ld_draft : nullptr, s_end.gone, s_end.n_tokens,
              s_end.inv, s_end.tokens};
  sum_runs<true>(a, r, [&](int run, double sum, double whole) {
    a.runs[(size_t)s * kRuns + run] = sum;
    a.runs[(size_t)(a.seqs + s) * kRuns + run] = whole;
  });
  if (first) {  // for the next kernel
    const int words = (int)(sizeof(Ended) / 8);
    for (int i = threadIdx.x; i < words; i += 256)
      reinterpret_cast<uint64_t *>(a.ended + s)[i] = reinterpret_cast<const uint64_t *>(&s_end)[i];
  }
}

// The next token: the run that holds it, then the thread's elements, then the
// element.  Two dependent loads and three scans.
constexpr int kHeld = 4;  // units of four elements that stay in registers
template <bool kDrawn>
__global__ __launch_bounds__(256) void pick_kernel(Verify a) {
  __shared__ Ended s_end;
  __shared__ double s_sum[4], s_before, s_goal;
  __shared__ int s_run, s_whole, s_first, s_last;
  const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Ended *ended = a.ended + s;
  const int64_t row = ended->row;
  if (threadIdx.x < 64) {
    const double sum_w = a.runs[(size_t)s * kRuns + lane];
    const double sum_p = a.runs[(size_t)(a.seqs + s) * kRuns + lane];
    const double sample = (double)a.sample[s];
    double upto = wave_scan(sum_w);
    double total = lane_of(upto, 63), mine = sum_w;
    const bool whole = !(total > 0.0);
    if (whole) upto = wave_scan(sum_p), total = lane_of(upto, 63), mine = sum_p;
    const double goal = fmax(sample, 0.0) * total;
    // (a run of nothing can pass the goal too: lanes add in orders of their own, and
    // their sums differ by roundings)
    const uint64_t some = __ballot(mine > 0.0), over = some & __ballot(upto > goal);
    // (a sample of one or more: the last that there is)
    const int run = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
    const double before = lane_of(upto, max(run - 1, 0));
    if (lane == 0) {
      s_run = total > 0.0 && total < INFINITY ? run : -1;
      s_whole = whole, s_goal = goal, s_before = run > 0 ? before : 0.0;
      s_first = 0x7fffffff, s_last = -1;
    }
  } else if (threadIdx.x < 128) {
    s_end.tokens[lane] = ended->tokens[lane];  // (some were never written, nor are read)
    s_end.inv[lane] = ended->inv[lane];
    if (lane == 0)
      s_end.kept = ended->kept, s_end.gone = ended->gone, s_end.n_tokens = ended->n_tokens;
  }
  if (row < 0) return;  // uniform
  __syncthreads();
  const int run = s_run;
  int64_t *next = a.emitted + (size_t)s * a.max_nodes + s_end.kept - 1;
  if (run < 0) {  // uniform
    if (threadIdx.x == 0) {
      *next = a.next_token[s] = -1;
      if (a.refused) *a.refused = 1;
    }
    return;
  }
  const int len = run_length(a.V), lo = run * len;  // (run has elements)
  const int end = min(lo + len, a.V);
  const int each = ((end - lo + 255) / 256 + 3) / 4 * 4;
  const int v0 = min(lo + each * (int)threadIdx.x, end), v1 = min(v0 + each, end);
  const Row r{a.target + row * a.ld_target, kDrawn ? a.draft + row * a.ld_draft : nullptr,
              s_whole ? 0 : s_end.gone, s_whole ? 0 : s_end.n_tokens, s_end.inv, s_end.tokens};
  const bool some = r.any_token(lo, end);
  v4f pv[kHeld], qv[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) r.load(min(v0 + 4 * i, v1), v1, pv[i], qv[i]);
  auto each_unit = [&](auto use) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      double w[4];
      r.left(v0 + 4 * i, pv[i], qv[i], some, w);
      use(v0 + 4 * i, w);
    }
    for (int v = v0 + 4 * kHeld; v < v1; v += 4) {
      v4f p, q;
      double w[4];
      r.load(v, v1, p, q);
      r.left(v, p, q, some, w);
      use(v, w);
    }
  };
  double sum = 0.0;
  each_unit([&](int, const double(&w)[4]) { sum += (w[0] + w[1]) + (w[2] + w[3]); });
  const double upto = wave_scan(sum);
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  double before = s_before + (upto - sum);
  for (int x = 0; x < wave; ++x) before += s_sum[x];
  // The first element that passes the goal; where rounding leaves none, the last
  // above zero.
  int first = 0x7fffffff, last = -1;
  each_unit([&](int v, const double(&w)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      before += w[j];
      if (w[j] > 0.0) {
        if (before > s_goal) first = min(first, v + j);
        last = v + j;
      }
    }
  });
  if (first != 0x7fffffff) atomicMin(&s_first, first);
  if (last >= 0) atomicMax(&s_last, last);
  __syncthreads();
  if (threadIdx.x == 0) {
    const int at = s_first != 0x7fffffff ? s_first : s_last;
    *next = a.next_token[s] = at;
    if (at < 0 && a.refused) *a.refused = 1;
  }
}

// ------------------------------------------------------- the cache's rows

constexpr int kKeepPools = 128, kKeepAtOnce = 8;
struct Keep {
  const int *starts, *lengths, *table, *kept, *path;
  int *refused;
  Planned planned;
  int width, shift, Hkv, max_nodes, units, n, per;  // units: of 16 bytes a row
  uint32_t pages;
  uint8_t *pool[kKeepPools];
};

// Workgroup: one sequence, `per` (pool, head) pairs, a wave kKeepAtOnce of them at a
// time.  Rows move to earlier places and no further than the row before them, so a
// wave that takes a pair's rows in order, 64 / units at a time, never reads what it
// has written.  Latency of small moves: 64 sequences' paths in 36 layers (some 3 rows
// each, 44 MB) 12 us, 15 with a pair at a time.
__global__ __launch_bounds__(256) void keep_kernel(Keep a) {
  __shared__ uint32_t s_from[kMaxNodes], s_to[kMaxNodes];
  const int s = blockIdx.y, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int start = a.starts[s], n = a.starts[s + 1] - start, cached = a.lengths[s] - n;
  int kept = a.kept[s];
  const bool other = a.planned.other();
  if (kept < 1) return;
  if (other) {
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.refused) *a.refused = 1;
    return;
  }
  const int row = lane < a.max_nodes ? a.path[(size_t)s * a.max_nodes + lane] : -1;
  const int before = __shfl_up(row, 1);
  const bool bad = lane < kept && (lane == 0 ? row != 0 : row <= before || row >= n);
  const uint64_t wrong = __ballot(bad) | (kept > a.max_nodes ? 1ull << (a.max_nodes - 1) : 0) |
                         (cached < 0 || n < 1 ? 1ull : 0);
  if (wrong) {
    kept = min(kept, (int)__builtin_ctzll(wrong));
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.refused) *a.refused = 1;
  }
  const uint64_t moves = __ballot(lane < kept && row != lane);
  if (!moves) return;
  const int first = __builtin_ctzll(moves), moved = kept - first;  // (and all after it)
  if (threadIdx.x < 64 && lane >= first && lane < kept) {
    auto slot = [&](int pos) {
      const int at = min(pos >> a.shift, a.width - 1);
      const uint32_t page = min((uint32_t)a.table[(size_t)s * a.width + at], a.pages - 1);
      return ((page * a.Hkv) << a.shift) + (uint32_t)(pos & ((1 << a.shift) - 1));
    };
    s_from[lane - first] = slot(cached + row);
    s_to[lane - first] = slot(cached + lane);
  }
  __syncthreads();
  const int unit = lane % a.units, sub = lane / a.units, step = 64 / a.units;
  const int end = min((int)(blockIdx.x + 1) * a.per, a.n * a.Hkv);
  for (int i0 = blockIdx.x * a.per + wave; i0 < end; i0 += 4 * kKeepAtOnce) {
    u32x4 *pool[kKeepAtOnce];  // of the pair, at its head
#pragma unroll
    for (int x = 0; x < kKeepAtOnce; ++x) {
      const int i = min(i0 + 4 * x, end - 1);
      pool[x] = reinterpret_cast<u32x4 *>(a.pool[i / a.Hkv]) +
                (((size_t)(i % a.Hkv) << a.shift) * a.units + unit);
    }
    for (int r = sub; r - sub < moved; r += step) {  // uniform
      const int row = min(r, moved - 1);
      const size_t from = (size_t)s_from[row] * a.units, to = (size_t)s_to[row] * a.units;
      u32x4 v[kKeepAtOnce];
#pragma unroll
      for (int x = 0; x < kKeepAtOnce; ++x) v[x] = pool[x][from];
#pragma unroll
      for (int x = 0; x < kKeepAtOnce; ++x)
        if (r < moved && i0 + 4 * x < end) pool[x][to] = v[x];
    }
  }
}

inline hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }
inline bool aligned(const void *p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}
inline int launched() { return hipGetLastError() == hipSuccess ? ECF8_OK : ECF8_ERR_HIP; }

Work layout_of(const ecf8_paged_batch *b, const ecf8_draft_trees *t) {
  return work_layout(b->seqs, b->rows, b->Hq, b->Hkv, t->max_nodes, t->max_children);
}

}  // namespace

extern "C" int64_t ecf8_draft_work_bytes(int64_t seqs, int64_t rows, int Hq, int Hkv,
                                         int max_nodes, int max_children) {
  return sizes_ok(seqs, rows, Hq, Hkv, max_nodes, max_children)
             ? work_layout(seqs, rows, Hq, Hkv, max_nodes, max_children).bytes
             : -1;
}

extern "C" int ecf8_draft_plan(const ecf8_paged_batch *b, const ecf8_draft_trees *t,
                               const int *parents, int64_t rows, void *stream) {
  if (!parents || rows <= 0) return ECF8_ERR_INVALID_ARG;
  if (const int rc = check_trees(b, t)) return rc;
  if (rows > b->rows) return ECF8_ERR_CAPACITY;
  if (!aligned(parents, 4)) return ECF8_ERR_MISALIGNED;
  const Work w = layout_of(b, t);
  auto *base = static_cast<uint8_t *>(t->work);
  const Plan a{b->starts, b->lengths, parents, t->masks, t->parents, b->positions, b->refused,
               reinterpret_cast<Counts *>(base), reinterpret_cast<Item *>(base + w.items_at),
               reinterpret_cast<Join *>(base + w.joins_at), b->seqs, (int)rows, b->rows,
               b->Hq / b->Hkv, t->max_nodes, t->max_children, w.tile, w.target,
               schedule_stamp(b, t), step_of(b)};
  const unsigned grid = 1 + (unsigned)((b->seqs + kPlanWaves - 1) / kPlanWaves);
  plan_kernel<<<grid, kPlanThreads, 0, as_stream(stream)>>>(a);
  return launched();
}

extern "C" int64_t ecf8_probability_work_bytes(int64_t rows) {
  return rows <= 0 || rows > 65535 ? -1 : rows * ECF8_PROBABILITY_CHUNKS * 8;
}

extern "C" int ecf8_token_probabilities(const void *logits, int64_t ld, int64_t rows, int64_t V,
                                        const float *temperature, float common, float *out,
                                        int64_t ldo, void *work, int64_t work_bytes,
                                        void *stream) {
  if (!logits || !out || !work || rows <= 0 || V <= 0) return ECF8_ERR_INVALID_ARG;
  if (rows > 65535 || V > (1 << 30) || (rows > 1 && ld < V)) return ECF8_ERR_UNSUPPORTED;
  if ((rows > 1 && ldo < V) || work_bytes < ecf8_probability_work_bytes(rows))
    return ECF8_ERR_CAPACITY;
  if (!aligned(logits, 2) || !aligned(out, 4) || !aligned(temperature, 4) || !aligned(work, 8))
    return ECF8_ERR_MISALIGNED;
  // A run is what a workgroup has in flight at once, 1024 units of eight, or, while
  // the workgroups are few, less.  416 rows of 151936 in 8 / 19 runs: 78 / 75 us.
  const int64_t units = (V + 7) / 8;
  int64_t chunks = 2048 / rows < (units + 255) / 256 ? 2048 / rows : (units + 255) / 256;
  if (chunks < (units + 1023) / 1024) chunks = (units + 1023) / 1024;
  if (chunks > ECF8_PROBABILITY_CHUNKS) chunks = ECF8_PROBABILITY_CHUNKS;
  const Probs a{static_cast<const uint16_t *>(logits), out, temperature, ld, ldo,
                static_cast<uint2 *>(work), common, (int)V, (int)chunks};
  const dim3 grid((unsigned)chunks, (unsigned)rows);
  probability_stats_kernel<<<grid, 256, 0, as_stream(stream)>>>(a);
  // (64 rows of 151936, 39 MB: 17.4 us, 18.5 past the caches; 416, 253 MB: 108 and 78)
  if (rows * V >= 1 << 24) probability_kernel<true><<<grid, 256, 0, as_stream(stream)>>>(a);
  else probability_kernel<false><<<grid, 256, 0, as_stream(stream)>>>(a);
  return launched();
}

extern "C" int ecf8_draft_verify(const ecf8_paged_batch *b, const ecf8_draft_trees *t,
                                 const int64_t *tokens, int64_t rows, const float *target,
                                 int64_t ld_target, const float *draft, int64_t ld_draft,
                                 int64_t V, const float *accept, const float *sample,
                                 void *stream) {
  if (!tokens || !target || !accept || !sample || rows <= 0 || V <= 0) return ECF8_ERR_INVALID_ARG;
  if (const int rc = check_trees(b, t)) return rc;
  if (rows > b->rows) return ECF8_ERR_CAPACITY;
  if (V > (1 << 30) || (rows > 1 && (ld_target < V || (draft && ld_draft < V))))
    return ECF8_ERR_UNSUPPORTED;
  if (!aligned(tokens, 8) || !aligned(target, 4) || !aligned(draft, 4) || !aligned(accept, 4) ||
      !aligned(sample, 4))
    return ECF8_ERR_MISALIGNED;
  const Work w = layout_of(b, t);
  auto *base = static_cast<uint8_t *>(t->work);
  Verify a{b->starts, t->parents, tokens, target, draft, accept, sample, ld_target, ld_draft,
           t->kept, t->path, b->refused, t->emitted, t->next_token,
           reinterpret_cast<double *>(base + w.runs), reinterpret_cast<double *>(base + w.mass),
           reinterpret_cast<Ended *>(base + w.ended), w.nodes, b->seqs, (int)rows, (int)V,
           t->max_nodes, t->max_children, w.packed, 1, 256,
           {reinterpret_cast<const Counts *>(base), step_of(b), schedule_stamp(b, t)}};
  // A wave a run once that leaves four workgroups a CU.  64 chains of 5 drawn from 32000:
  // 15 us, 22 with four waves; 8 trees of 32 from 151936: 32 with four, 39 with one.
  if (b->seqs * (kRuns / 4) >= 1024) a.per = 4, a.lanes = 64;
  const dim3 grid((unsigned)(kRuns / a.per), (unsigned)b->seqs);
  const unsigned lds = draft ? (unsigned)(t->max_children * 64 * sizeof(double)) : 0;
  if (draft) {
    for (int level = 1; level < t->max_children; ++level)
      mass_kernel<<<grid, 256, lds, as_stream(stream)>>>(a, level);
    last_kernel<true><<<grid, 256, lds, as_stream(stream)>>>(a);
    pick_kernel<true><<<(unsigned)b->seqs, 256, 0, as_stream(stream)>>>(a);
  } else {
    last_kernel<false><<<grid, 256, 0, as_stream(stream)>>>(a);
    pick_kernel<false><<<(unsigned)b->seqs, 256, 0, as_stream(stream)>>>(a);
  }
  return launched();
}

extern "C" int ecf8_draft_keep(const ecf8_paged_batch *b, const ecf8_draft_trees *t,
                               void *const *pools, int n_pools, int fp8, void *stream) {
  if (!pools || n_pools <= 0) return ECF8_ERR_INVALID_ARG;
  if (const int rc = check_trees(b, t)) return rc;
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i]) return ECF8_ERR_INVALID_ARG;
    if (!aligned(pools[i], 16)) return ECF8_ERR_MISALIGNED;
  }
  Keep a{};
  a.starts = b->starts, a.lengths = b->lengths, a.table = b->table;
  a.kept = t->kept, a.path = t->path, a.refused = b->refused;
  a.planned = {static_cast<const Counts *>(t->work), step_of(b), schedule_stamp(b, t)};
  a.width = b->width, a.shift = __builtin_ctz((unsigned)b->page_size), a.Hkv = b->Hkv;
  a.max_nodes = t->max_nodes, a.units = fp8 ? kD / 16 : kD / 8, a.pages = (uint32_t)b->pages;
  for (int i0 = 0; i0 < n_pools; i0 += kKeepPools) {
    a.n = n_pools - i0 < kKeepPools ? n_pools - i0 : kKeepPools;
    for (int i = 0; i < a.n; ++i) a.pool[i] = static_cast<uint8_t *>(pools[i0 + i]);
    // a thousand workgroups, and whole turns of their waves
    const int64_t pairs = (int64_t)a.n * a.Hkv, each = pairs * b->seqs / 1024;
    constexpr int kTurn = 4 * kKeepAtOnce;
    a.per = each < 4 ? 4 : each < kTurn ? (int)each : (int)(each / kTurn * kTurn);
    const dim3 grid((unsigned)((pairs + a.per - 1) / a.per), (unsigned)b->seqs);
    keep_kernel<<<grid, 256, 0, as_stream(stream)>>>(a);
  }
  return launched();
}
