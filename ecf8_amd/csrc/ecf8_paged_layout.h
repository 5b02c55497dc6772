// What the step's plan (ecf8_paged.hip) and the attention that follows it
// (ecf8_ragged.hip) share: the work buffer of a batch.
#ifndef ECF8_PAGED_LAYOUT_H
#define ECF8_PAGED_LAYOUT_H

#include <stdint.h>

#include "ecf8.h"
#include "ecf8_paged.h"

namespace ecf8 {
namespace paged {

constexpr int kD = 128;            // head dimension
constexpr int kMaxSeqs = 4096;
constexpr int kMaxRows = 1 << 18;
constexpr int kMaxLen = 1 << 24;   // positions of a sequence

// A "row" of the attention is a (new token, query head of the group) pair:
// row t * G + g of a sequence and KV head.  Sequences of up to kFewRows rows
// are split along their keys at multiples of kFewKeys, the others also into
// tiles of kTileRows rows, split at multiples of kTileKeys.
constexpr int kFewRows = 32, kFewKeys = 128;
constexpr int kTileRows = 192, kTileKeys = 64;
constexpr int kTileMinUnits = 4;  // a part of a tile is at least this long
constexpr int kTileStart = 4;     // what a tile costs beside its keys, in the same units
// workgroups that a split aims at, over all KV heads: two a CU
constexpr int kFewSlots = 512, kTileSlots = 512;

// One workgroup's part of the attention, per KV head.
struct Item {
  int seq, row0;  // rows [row0, row0 + kFewRows or kTileRows)
  int k0, k1;     // positions
  int part;       // index of the partial sums, -1: the only part, final
  int start, n, cached;  // first packed row, new tokens, tokens before them
};
// Rows whose parts [part, part + n) are to be joined.
struct Join {
  int row0, part, n;
  int start, tokens;  // of the sequence: first packed row, new tokens
  int pad[3];
};

// At the start of the work buffer.  stamp: of the sizes that the plan wrote the
// lists for (schedule_stamp), zero before the first plan.  The attention reads no
// item under another: a list of anything else would send it out of its buffers.
struct Counts {
  int few, tiles, few_joins, tile_joins;
  uint64_t stamp;
};

// Byte offsets of the work buffer's parts.
struct Work {
  int few_parts, tile_parts;    // parts each class has room for
  int few_items, tile_items;    // items
  int64_t few_at, tiles_at, few_joins_at, tile_joins_at;
  int64_t few_stats, few_sums, tile_stats, tile_sums, bytes;
};

inline Work work_layout(int64_t seqs, int64_t rows, int Hq, int Hkv) {
  Work w;
  const int64_t few = kFewSlots / Hkv > 1 ? kFewSlots / Hkv : 1;
  const int64_t tiles = kTileSlots / Hkv > 1 ? kTileSlots / Hkv : 1;
  const int64_t G = Hq / Hkv;
  w.few_parts = (int)(2 * few);
  w.tile_parts = (int)(2 * tiles);
  w.few_items = (int)(few + seqs);
  w.tile_items = (int)(rows * G / kTileRows + seqs + 2 * tiles);
  int64_t at = 256;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  w.few_at = take(w.few_items * (int64_t)sizeof(Item));
  w.tiles_at = take(w.tile_items * (int64_t)sizeof(Item));
  w.few_joins_at = take(few * (int64_t)sizeof(Join));
  w.tile_joins_at = take(tiles * (int64_t)sizeof(Join));
  w.few_stats = take(w.few_parts * (int64_t)Hkv * kFewRows * 8);
  w.few_sums = take(w.few_parts * (int64_t)Hkv * kFewRows * kD * 4);
  w.tile_stats = take(w.tile_parts * (int64_t)Hkv * kTileRows * 8);
  w.tile_sums = take(w.tile_parts * (int64_t)Hkv * kTileRows * kD * 4);
  w.bytes = at;
  return w;
}

// FNV-1a over the sizes that items and the buffer's parts depend on; never zero.
inline uint64_t schedule_stamp(const ecf8_paged_batch *b) {
  uint64_t h = 0xcbf29ce484222325ull;
  for (const int x : {b->seqs, b->rows, b->pages, b->page_size, b->width, b->Hq, b->Hkv})
    for (int byte = 0; byte < 4; ++byte)
      h = (h ^ (((uint32_t)x >> (8 * byte)) & 0xff)) * 0x100000001b3ull;
  return h | 1;
}

inline bool sizes_ok(int64_t seqs, int64_t rows, int Hq, int Hkv) {
  return seqs >= 1 && seqs <= kMaxSeqs && rows >= 1 && rows <= kMaxRows && Hkv >= 1 &&
         Hq >= Hkv && Hq % Hkv == 0 && Hq <= 1024;
}

// A batch's sizes and pointers, as every entry point that takes one needs
// them.
inline int check_batch(const ecf8_paged_batch *b) {
  if (!b || !b->table || !b->owned || !b->free_pages || !b->n_free || !b->starts ||
      !b->lengths || !b->slots || !b->positions || !b->work || b->seqs <= 0 || b->rows <= 0 ||
      b->pages <= 0 || b->page_size <= 0 || b->width <= 0 || b->Hq <= 0 || b->Hkv <= 0)
    return ECF8_ERR_INVALID_ARG;
  const int64_t page = b->page_size;
  if (!sizes_ok(b->seqs, b->rows, b->Hq, b->Hkv) || page > 1024 || (page & (page - 1)) ||
      b->width * page > kMaxLen || (int64_t)b->seqs * b->width > INT32_MAX ||
      (int64_t)b->pages * page > INT32_MAX || b->pages * page * b->Hkv > INT32_MAX)
    return ECF8_ERR_UNSUPPORTED;
  const uintptr_t ints = (uintptr_t)b->table | (uintptr_t)b->owned | (uintptr_t)b->free_pages |
                         (uintptr_t)b->n_free | (uintptr_t)b->starts | (uintptr_t)b->lengths |
                         (uintptr_t)b->slots | (uintptr_t)b->positions | (uintptr_t)b->refused;
  if ((ints & 3) || ((uintptr_t)b->work & 15)) return ECF8_ERR_MISALIGNED;
  if (b->work_bytes < work_layout(b->seqs, b->rows, b->Hq, b->Hkv).bytes)
    return ECF8_ERR_CAPACITY;
  return ECF8_OK;
}

}  // namespace paged
}  // namespace ecf8

#endif  // ECF8_PAGED_LAYOUT_H
