// The bookkeeping of a paged KV cache on gfx950: block tables, slot maps and
// the attention's schedule from request lengths, and the cache write of a
// step's rows (head norms, rotary embedding, optional e4m3 codes).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ecf8.h"
#include "ecf8_dev.h"
#include "ecf8_paged.h"
#include "ecf8_paged_layout.h"

namespace {

using namespace ecf8::paged;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr float kFp8Max = 448.f;

// --------------------------------------------------------------- the plan

struct Plan {
  int *table, *owned, *free_pages, *n_free, *starts, *lengths, *slots, *positions;
  const int *cached, *new_tokens, *release;
  int *refused;
  Counts *counts;
  Item *few, *tiles;
  Join *few_joins, *tile_joins;
  int seqs, rows, pages, shift, width, group;  // page size 1 << shift
  int few_target, tile_target, fill_rows;
  uint64_t stamp;
};

constexpr int kPlanThreads = 1024;
constexpr int kPer = kMaxSeqs / kPlanThreads;  // most sequences per thread

// The i-th sequence of this thread: seqs / kPlanThreads consecutive ones
// each, rounded up; -1 past its last.
__device__ __forceinline__ int seq_of(int i, int seqs) {
  const int step = (seqs + kPlanThreads - 1) / kPlanThreads;
  const int s = step * (int)threadIdx.x + i;
  return i < step && s < seqs ? s : -1;
}

// The exclusive prefix sums of N values over the workgroup, and their totals.
// Calls in a row alternate between the two halves of `waves`.
constexpr int kPlanWaves = kPlanThreads / 64;
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

// Writes exclusive prefix sums of the threads' sequences' values, of which
// `at` come before this thread's.
__device__ __forceinline__ void put_firsts(const int (&v)[kPer], int at, int total, int seqs,
                                           int *out) {
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = seq_of(i, seqs);
    if (s >= 0) out[s] = at;
    at += v[i];
  }
  if (threadIdx.x == 0) out[seqs] = total;
}
__device__ __forceinline__ int sum_of(const int (&v)[kPer]) {
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += v[i];
  return sum;
}

// Buckets of lengths, the longest first, for an order that tells lengths apart
// by a 48th of a share.
constexpr int kBuckets = 64;
__device__ __forceinline__ int bucket_of(int length, int share) {
  return kBuckets - 1 - min(kBuckets - 1, (int)(48ll * length / share));
}
// Counts become first places; the total.
__device__ __forceinline__ int start_buckets(int *bucket, int (*waves)[kPlanWaves]) {
  const int tid = threadIdx.x, count[1] = {tid < kBuckets ? bucket[tid] : 0};
  int first[1], all[1];
  block_scan(count, waves, first, all);
  if (tid < kBuckets) bucket[tid] = first[0];
  __syncthreads();
  return all[0];
}

// The last s < seqs with first[s] <= i: the sequence that element i of a
// flattened ragged list belongs to (first: exclusive prefix sums).
__device__ __forceinline__ int find_seq(const int *first, int seqs, int i) {
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void fill_row(const Plan &a, const int *first, int i) {
  int slot = -1, pos = -1;
  if (i < first[a.seqs]) {
    const int s = find_seq(first, a.seqs, i);
    pos = a.lengths[s] - (first[s + 1] - first[s]) + (i - first[s]);
    slot = (a.table[(size_t)s * a.width + (pos >> a.shift)] << a.shift) |
           (pos & ((1 << a.shift) - 1));
  }
  a.slots[i] = slot;
  a.positions[i] = pos;
}

// One workgroup plans the step: prefix sums over the sequences (rows,
// pages to take, pages to give back) say where everything goes, then pages,
// items and rows are written element by element, each finding its sequence by
// bisection in LDS.  All of it is latency, of three scans and some ten dependent
// loads: 64 sequences 8.8 us, 512 that leave and 512 that come 18.8 us.  (Scans of
// one value each, nine of them: 11.2 us.)
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(Plan a) {
  __shared__ int s_start[kMaxSeqs + 1], s_take[kMaxSeqs + 1], s_back[kMaxSeqs + 1];
  __shared__ int s_waves[2][3][kPlanWaves];  // (of two scans in a row)
  __shared__ int s_bad, s_part[kMaxSeqs], s_bucket[2][kBuckets];
  const int tid = threadIdx.x, S = a.seqs;
  const int page = 1 << a.shift;
  if (tid == 0) s_bad = 0;
  if (tid < 2 * kBuckets) s_bucket[tid / kBuckets][tid % kBuckets] = 0;
  __syncthreads();
  const int n_free = a.n_free[0];
  uint64_t planned = 0;  // (here: its load waits for nothing)
  if (tid == 0) planned = a.counts->step + 1;
  int c[kPer], n[kPer], own[kPer], take[kPer], back[kPer];
  bool bad = n_free < 0 || n_free > a.pages;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = seq_of(i, S);
    c[i] = n[i] = own[i] = take[i] = back[i] = 0;
    if (s < 0) continue;
    c[i] = a.cached[s];
    n[i] = a.new_tokens[s];
    own[i] = a.owned[s];
    if (own[i] < 0 || own[i] > a.width) bad = true, own[i] = 0;
    if (a.release && a.release[s]) back[i] = own[i], own[i] = 0;
    const int most = a.width << a.shift;
    if (c[i] < 0 || n[i] < 0 || n[i] > a.rows || c[i] > most - n[i]) bad = true, c[i] = n[i] = 0;
    take[i] = max(0, ((c[i] + n[i] + page - 1) >> a.shift) - own[i]);
  }
  if (bad) s_bad = 1;
  const int sums[3] = {sum_of(n), sum_of(take), sum_of(back)};
  int at0[3], all0[3];
  block_scan(sums, s_waves[0], at0, all0);
  const int rows = all0[0], taken = all0[1], given = all0[2];
  put_firsts(n, at0[0], rows, S, s_start);
  put_firsts(take, at0[1], taken, S, s_take);
  put_firsts(back, at0[2], given, S, s_back);
  __syncthreads();
  if (s_bad || rows > a.rows || taken > n_free + given || given > a.pages - n_free) {
    for (int s = tid; s <= S; s += kPlanThreads) {
      s_start[s] = 0;
      a.starts[s] = 0;
      if (s < S) a.lengths[s] = 0;
    }
    __syncthreads();
    if (tid == 0) {
      *a.counts = Counts{0, 0, 0, 0, a.stamp, planned};
      if (a.refused) *a.refused = 1;
    }
    if (a.fill_rows)
      for (int i = tid; i < a.rows; i += kPlanThreads) fill_row(a, s_start, i);
    return;
  }
  // pages given back, then pages taken
  for (int i = tid; i < given; i += kPlanThreads) {
    const int s = find_seq(s_back, S, i);
    int *e = a.table + (size_t)s * a.width + (i - s_back[s]);
    a.free_pages[n_free + i] = *e;
    *e = -1;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int s = seq_of(i, S);
    if (s < 0) continue;
    a.owned[s] = own[i] + take[i];
    a.starts[s] = s_start[s];
    a.lengths[s] = c[i] + n[i];
  }
  if (tid == 0) {
    a.n_free[0] = n_free + given - taken;
    a.starts[S] = rows;
  }
  __threadfence_block();
  __syncthreads();
  for (int i = tid; i < taken; i += kPlanThreads) {
    const int s = find_seq(s_take, S, i), j = i - s_take[s];
    const int held = a.owned[s] - (s_take[s + 1] - s_take[s]);
    a.table[(size_t)s * a.width + held + j] = a.free_pages[n_free + given - 1 - i];
  }
  // The attention's schedule.  Sequences of few rows, in units of kFewKeys keys:
  // laid end to end they are cut at the multiples of a workgroup's share, and
  // the pieces listed from the longest on.  Against as many equal parts, 64
  // sequences of 8 to 8192 keys take 0.89 of the time, 6 of 100000 keys 0.84.
  int units[kPer], items[kPer], joins[kPer], tiles[kPer], cut0[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = n[i] * a.group;
    units[i] = r > 0 && r <= kFewRows ? (c[i] + n[i] + kFewKeys - 1) / kFewKeys : 0;
    tiles[i] = r > kFewRows ? (r + kTileRows - 1) / kTileRows : 0;
  }
  const int sums1[2] = {sum_of(units), sum_of(tiles)};
  int at1[2], all1[2];
  block_scan(sums1, s_waves[1], at1, all1);
  const int few_share = max(1, (all1[0] + a.few_target - 1) / a.few_target);
  const int n_tiles = all1[1];
  {
    int from = at1[0];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      // cuts inside the sequence, from number cut0 on
      cut0[i] = from / few_share + 1;
      const int cuts = units[i] ? (from + units[i] - 1) / few_share - cut0[i] + 1 : 0;
      items[i] = units[i] ? cuts + 1 : 0;
      joins[i] = cuts > 0;
      from += units[i];
    }
  }
  const int sums2[2] = {sum_of(items), sum_of(joins)};
  int at2[2], all2[2];
  block_scan(sums2, s_waves[0], at2, all2);
  const int n_items = all2[0], n_joins = all2[1];
  put_firsts(units, at1[0], all1[0], S, s_take);
  put_firsts(items, at2[0], n_items, S, s_back);
  {
    int join = at2[1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int s = seq_of(i, S);
      if (s < 0) continue;
      // parts: one number a cut, and one more a sequence that is cut
      s_part[s] = joins[i] ? cut0[i] - 1 + join : -1;
      if (joins[i]) a.few_joins[join] = Join{0, s_part[s], items[i], s_start[s], n[i], {0, 0, 0}};
      join += joins[i];
    }
  }
  __syncthreads();
  for (int write = 0; write < 2; ++write) {
    for (int i = tid; i < n_items; i += kPlanThreads) {
      const int s = find_seq(s_back, S, i), j = i - s_back[s], from = s_take[s];
      const int end = s_take[s + 1] - from, cut = from / few_share + j;
      const int u0 = j ? cut * few_share - from : 0, u1 = min((cut + 1) * few_share - from, end);
      const int at = atomicAdd(&s_bucket[0][bucket_of(u1 - u0, few_share)], 1);
      if (write) {
        const int tokens = s_start[s + 1] - s_start[s], length = a.lengths[s];
        a.few[at] = Item{s, 0, u0 * kFewKeys, min(u1 * kFewKeys, length),
                         s_part[s] < 0 ? -1 : s_part[s] + j, s_start[s], tokens, length - tokens};
      }
    }
    __syncthreads();
    if (!write) start_buckets(s_bucket[0], s_waves[1]);
  }
  // Tiles of the others, in units of kTileKeys keys.  A tile of more than half
  // a workgroup's share is long: the long ones, laid end to end, are cut at
  // the multiples of the share.  Items are listed from the longest on: that
  // way a tile's last piece and the next one's first follow each other on a CU,
  // and short tiles fill up what is left.  (A step of 1024 rows after 8192 keys beside
  // 8 single tokens: 0.73 of the time of equal parts, of which 33 met 32 CUs.)
  int t_items = 0, t_joins = 0;
  if (n_tiles > 0) {  // uniform
    put_firsts(tiles, at1[1], n_tiles, S, s_back);
    __syncthreads();
    struct Tile {
      int seq, row0, end, units, n, cached;
    };
    auto tile_at = [&](int i) {
      Tile t{};
      if (i >= n_tiles) return t;
      t.seq = find_seq(s_back, S, i);
      t.row0 = (i - s_back[t.seq]) * kTileRows;
      t.n = s_start[t.seq + 1] - s_start[t.seq];
      t.cached = a.lengths[t.seq] - t.n;
      t.end = t.cached + min(t.n, (t.row0 + kTileRows - 1) / a.group + 1);
      t.units = (t.end + kTileKeys - 1) / kTileKeys;
      return t;
    };
    // A share of all units, to the unit: rounded up a thread, 1036 tiles of which two
    // have 1564 units were all one piece (2590 us of attention, now 720).  The
    // total can pass 32 bits (a thread's cannot: at most 1370 tiles of 2^18), so low
    // and high parts are summed apart.
    int mine = 0;
    for (int i = tid; i < n_tiles; i += kPlanThreads) mine += tile_at(i).units + kTileStart;
    const int halves[2] = {mine & 0xffff, mine >> 16};
    int skip[2], all[2];
    block_scan(halves, s_waves[1], skip, all);
    const int64_t all_units = ((int64_t)all[1] << 16) + all[0];
    // (more units than a tile can have are as good as any)
    const int64_t exact = (all_units + a.tile_target - 1) / a.tile_target;
    const int share = __builtin_amdgcn_readfirstlane(
        (int)min(max(exact, (int64_t)(2 * kTileMinUnits)), (int64_t)1 << 20));
    // Twice over the tiles: count the items of each length, then write them.
    for (int write = 0; write < 2; ++write) {
      int from0 = 0, t_parts = 0;
      for (int i0 = 0; i0 < n_tiles; i0 += kPlanThreads) {  // uniform
        const Tile t = tile_at(i0 + tid);
        const bool is_long = 2 * t.units > share;
        const int units_long[1] = {is_long ? kTileStart + t.units : 0};
        int from[1], all_long[1];
        block_scan(units_long, s_waves[0], from, all_long);
        from[0] += from0 + kTileStart;
        // cuts that leave kTileMinUnits on both sides
        const int c0 = (from[0] + kTileMinUnits + share - 1) / share;
        const int c1 = (from[0] + t.units - kTileMinUnits) / share;
        const int k = t.units ? (is_long ? max(0, c1 - c0 + 1) : 0) + 1 : 0;
        const int cut[2] = {k > 1 ? k : 0, k > 1};
        int p[2], all_cut[2];
        block_scan(cut, s_waves[1], p, all_cut);
        p[0] += t_parts, p[1] += t_joins;
        for (int j = 0; j < k; ++j) {
          const int u0 = j ? (c0 + j - 1) * share - from[0] : 0;
          const int u1 = j + 1 < k ? (c0 + j) * share - from[0] : t.units;
          const int at = atomicAdd(&s_bucket[1][bucket_of(u1 - u0, share)], 1);
          if (write)
            a.tiles[at] = Item{t.seq, t.row0, u0 * kTileKeys, min(u1 * kTileKeys, t.end),
                               k > 1 ? p[0] + j : -1, s_start[t.seq], t.n, t.cached};
        }
        if (write) {
          if (k > 1) a.tile_joins[p[1]] = Join{t.row0, p[0], k, s_start[t.seq], t.n, {0, 0, 0}};
          t_parts += all_cut[0], t_joins += all_cut[1];
        }
        from0 += all_long[0];
      }
      __syncthreads();
      if (!write) t_items = start_buckets(s_bucket[1], s_waves[0]);
    }
  }
  if (tid == 0) *a.counts = Counts{n_items, t_items, n_joins, t_joins, a.stamp, planned};
  if (a.fill_rows) {
    __threadfence_block();
    __syncthreads();
    for (int i = tid; i < a.rows; i += kPlanThreads) fill_row(a, s_start, i);
  }
}

// The rows of a large step, on workgroups of their own.
constexpr int kFillThreads = 256;
__global__ __launch_bounds__(kFillThreads) void fill_kernel(Plan a) {
  __shared__ int s_start[kMaxSeqs + 1];
  for (int s = threadIdx.x; s <= a.seqs; s += kFillThreads) s_start[s] = a.starts[s];
  __syncthreads();
  const int i = blockIdx.x * kFillThreads + threadIdx.x;
  if (i < a.rows) fill_row(a, s_start, i);
}

// -------------------------------------------------------- the cache write

__device__ __forceinline__ float bf16_f32(uint32_t h16) { return __uint_as_float(h16 << 16); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const v2bf v = {(__bf16)lo, (__bf16)hi};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ void unpack8(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = bf16_f32(v[j] & 0xffffu);
    f[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8f(const float *p, float (&f)[8]) {
  const float4 a = *reinterpret_cast<const float4 *>(p);
  const float4 b = *reinterpret_cast<const float4 *>(p + 4);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), kCtrl,
                                                               0xF, 0xF, true));
}

// Four values / scale, clamped to +-448, as e4m3fn codes.  NaN stays NaN.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float scale) {
  auto clamped = [scale](float x) {
    const float y = x / scale;
    return y != y ? y : fminf(fmaxf(y, -kFp8Max), kFp8Max);
  };
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(clamped(a), clamped(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamped(c), clamped(d), lo, true);
}

struct Write {
  const uint16_t *qkv, *qn, *kn;
  const float *cosv, *sinv;
  const int *slots, *positions, *step_rows;
  int *refused;
  uint16_t *q_out;
  void *kp, *vp;
  const float *ks, *vs;
  float eps;
  int Hq, Hkv, shift, table_len, rows, parts;  // parts: workgroups a row
  uint32_t slots_end;                    // pages * page size
};

// 16 lanes a head, 8 dims a lane (16-byte loads); dims d and d +- 64 lie 8
// lanes apart, the norm's sum and the rotary partner are row rotations.
// Workgroup: one row, 16 kU heads, all loads before the arithmetic.
// HBM-bound: 8192 rows of 32 + 16 heads (202 MB) 31 us, 6.5 TB/s; a step of 16
// rows 2.3 us back to back, two memory round trips.
template <int kU, bool kFp8>
__global__ __launch_bounds__(256) void write_kernel(Write a) {
  const int row = (int)blockIdx.x / a.parts, part = (int)blockIdx.x % a.parts;
  const int H = a.Hq + 2 * a.Hkv;
  const int l = threadIdx.x & 15;
  const int h0 = part * 16 * kU + (int)(threadIdx.x >> 4);
  const int slot = a.slots[row], pos = a.positions[row];
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.refused && *a.step_rows > a.rows) *a.refused = 1;
  u32x4 x[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u)
    x[u] = *reinterpret_cast<const u32x4 *>(
        a.qkv + ((size_t)row * H + min(h0 + 16 * u, H - 1)) * kD + 8 * l);
  const u32x4 qw = *reinterpret_cast<const u32x4 *>(a.qn + 8 * l);
  const u32x4 kw = *reinterpret_cast<const u32x4 *>(a.kn + 8 * l);
  if ((uint32_t)slot >= a.slots_end || (uint32_t)pos >= (uint32_t)a.table_len) return;
  float c[8], s[8];
  load8f(a.cosv + (size_t)pos * 64 + 8 * (l & 7), c);
  load8f(a.sinv + (size_t)pos * 64 + 8 * (l & 7), s);
  if (l < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = -s[j];
  }
  const uint32_t page = (uint32_t)slot >> a.shift, off = (uint32_t)slot & ((1u << a.shift) - 1);
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const int h = h0 + 16 * u;
    if (h >= H) break;
    float v[8];
    unpack8(x[u], v);
    if (h < a.Hq + a.Hkv) {
      float w[8];
      unpack8(h < a.Hq ? qw : kw, w);
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
      ss += dpp<0x128>(ss);  // row_ror:8
      ss += dpp<0x124>(ss);  // row_ror:4
      ss += dpp<0x4E>(ss);   // quad_perm 2, 3, 0, 1
      ss += dpp<0xB1>(ss);   // quad_perm 1, 0, 3, 2
      const float rs = rsqrtf(ss / (float)kD + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = v[j] * rs * w[j];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = fmaf(v[j], c[j], dpp<0x128>(v[j]) * s[j]);
    }
    if (h < a.Hq) {
      *reinterpret_cast<u32x4 *>(a.q_out + ((size_t)row * a.Hq + h) * kD + 8 * l) =
          u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                pack_bf16(v[6], v[7])};
      continue;
    }
    const bool key = h < a.Hq + a.Hkv;
    const int kh = h - a.Hq - (key ? 0 : a.Hkv);
    const size_t at = ((((size_t)page * a.Hkv + kh) << a.shift) + off) * kD + 8 * l;
    if constexpr (kFp8) {
      const float sc = (key ? a.ks : a.vs)[kh];
      *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(key ? a.kp : a.vp) + at) =
          u32x2{codes4(v[0], v[1], v[2], v[3], sc), codes4(v[4], v[5], v[6], v[7], sc)};
    } else {
      *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(key ? a.kp : a.vp) + at) =
          u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                pack_bf16(v[6], v[7])};
    }
  }
}

inline hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }
inline bool aligned(const void *p, uintptr_t a) {
  return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0;
}
inline int launched() { return hipGetLastError() == hipSuccess ? ECF8_OK : ECF8_ERR_HIP; }

}  // namespace

extern "C" int64_t ecf8_paged_work_bytes(int64_t seqs, int64_t rows, int Hq, int Hkv) {
  return sizes_ok(seqs, rows, Hq, Hkv) ? work_layout(seqs, rows, Hq, Hkv).bytes : -1;
}

extern "C" int ecf8_paged_plan(const ecf8_paged_batch *b, const int *cached,
                               const int *new_tokens, const int *release, void *stream) {
  if (!cached || !new_tokens) return ECF8_ERR_INVALID_ARG;
  if (const int rc = ecf8::paged::check_batch(b)) return rc;
  if (!aligned(cached, 4) || !aligned(new_tokens, 4) || !aligned(release, 4))
    return ECF8_ERR_MISALIGNED;
  const Work w = work_layout(b->seqs, b->rows, b->Hq, b->Hkv);
  auto *base = static_cast<uint8_t *>(b->work);
  // one launch while the rows are few enough for one workgroup
  const bool one = b->rows <= 4 * kPlanThreads;
  const Plan a{b->table, b->owned, b->free_pages, b->n_free, b->starts, b->lengths, b->slots,
               b->positions, cached, new_tokens, release, b->refused,
               reinterpret_cast<Counts *>(base), reinterpret_cast<Item *>(base + w.few_at),
               reinterpret_cast<Item *>(base + w.tiles_at),
               reinterpret_cast<Join *>(base + w.few_joins_at),
               reinterpret_cast<Join *>(base + w.tile_joins_at), b->seqs, b->rows, b->pages,
               __builtin_ctz((unsigned)b->page_size), b->width, b->Hq / b->Hkv, w.few_parts / 2,
               w.tile_parts / 2, one, ecf8::paged::schedule_stamp(b)};
  plan_kernel<<<1, kPlanThreads, 0, as_stream(stream)>>>(a);
  if (!one)
    fill_kernel<<<(unsigned)((b->rows + kFillThreads - 1) / kFillThreads), kFillThreads, 0,
                  as_stream(stream)>>>(a);
  return launched();
}

extern "C" int ecf8_paged_qk_norm_rope(const void *qkv, int64_t rows, const ecf8_paged_batch *b,
                                       const void *q_norm, const void *k_norm, float eps,
                                       const float *cos_t, const float *sin_t, int64_t table_len,
                                       void *q_out, void *k_pool, void *v_pool, int fp8,
                                       const float *k_scale, const float *v_scale, void *stream) {
  if (!qkv || !q_norm || !k_norm || !cos_t || !sin_t || !q_out || !k_pool || !v_pool ||
      rows <= 0 || table_len <= 0 || (fp8 && (!k_scale || !v_scale)))
    return ECF8_ERR_INVALID_ARG;
  if (const int rc = ecf8::paged::check_batch(b)) return rc;
  if (rows > b->rows) return ECF8_ERR_CAPACITY;
  if (table_len > kMaxLen) return ECF8_ERR_UNSUPPORTED;
  if (!aligned(qkv, 16) || !aligned(q_norm, 16) || !aligned(k_norm, 16) || !aligned(cos_t, 16) ||
      !aligned(sin_t, 16) || !aligned(q_out, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) ||
      !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return ECF8_ERR_MISALIGNED;
  const int H = b->Hq + 2 * b->Hkv;
  // Three heads a lane, 48 a workgroup, once there are workgroups enough either
  // way (48 heads, 16 / 512 / 1024 / 8192 rows 2.3 / 4.0 / 5.9 / 32.7 us with one and
  // 3.0 / 4.1 / 5.9 / 30.5 us with three), where that makes one workgroup of two or
  // three, or fills two thirds of its lanes.  8192 rows of 12 / 20 / 24 / 32 / 52 /
  // 60 / 64 / 72 / 144 heads: 11.3 / 21.1 / 21.9 / 23.8 / 39.3 / 42.0 / 48.6 / 62.2 / 124 us
  // with one, 12.8 / 15.3 / 17.0 / 21.3 / 42.5 / 44.0 / 47.6 / 54.2 / 103 us with three.
  // (The rule's worst: 64 heads, 1024 rows in e4m3, 10.1 us with three, 8.4 with one.)
  const bool fills = H <= 48 ? H > 16 : 3 * H >= 2 * 48 * ((H + 47) / 48);
  const bool wide = fills && rows * ((H + 15) / 16) > 2048;
  const int per = wide ? 48 : 16, parts = (H + per - 1) / per;
  const Write a{static_cast<const uint16_t *>(qkv), static_cast<const uint16_t *>(q_norm),
                static_cast<const uint16_t *>(k_norm), cos_t, sin_t, b->slots, b->positions,
                b->starts + b->seqs, b->refused, static_cast<uint16_t *>(q_out), k_pool, v_pool,
                k_scale, v_scale, eps, b->Hq, b->Hkv, __builtin_ctz((unsigned)b->page_size),
                (int)table_len, (int)rows, parts,
                (uint32_t)b->pages * (uint32_t)b->page_size};
  const unsigned grid = (unsigned)(rows * parts);
#define ECF8_WRITE(U, F) write_kernel<U, F><<<grid, 256, 0, as_stream(stream)>>>(a)
  if (wide) {
    if (fp8) ECF8_WRITE(3, true);
    else ECF8_WRITE(3, false);
  } else {
    if (fp8) ECF8_WRITE(1, true);
    else ECF8_WRITE(1, false);
  }
#undef ECF8_WRITE
  return launched();
}
