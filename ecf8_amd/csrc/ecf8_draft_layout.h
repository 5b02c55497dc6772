// What the trees' plan and verification (ecf8_draft.hip) and their attention
// (ecf8_ragged.hip) share: the work buffer of a batch's trees.
#ifndef ECF8_DRAFT_LAYOUT_H
#define ECF8_DRAFT_LAYOUT_H

#include <stdint.h>

#include "ecf8_draft.h"
#include "ecf8_paged_layout.h"

namespace ecf8 {
namespace draft {

using paged::Item;
using paged::Join;
using paged::kD;

constexpr int kMaxNodes = 64;  // a row's mask is 64 bits
constexpr int kUnitKeys = 128; // key ranges are cut at multiples
// Runs of the vocabulary that a row's probabilities are summed by.
constexpr int kRuns = 64;
constexpr int kEndedBytes = 1056;  // of where a sequence's walk ended

// Rows (token, head of the group) of a workgroup of the attention: what a sequence
// has, in as few workgroups as registers allow, since each reads the sequence's pages.
// One tree of 8 in groups of four after 4096: 12.5 us in 32 rows, 13.2 in 64; 16 trees
// of 64 after 8192 bf16 keys 94 in 256, 132 in two of 128.  (Of 32 they take 87 in 128
// and 74 in 256, since probabilities of 256 rows are rounded once.)
inline int tile_rows(int max_nodes, int group) {
  const int r = max_nodes * group;
  return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : r <= 128 ? 128 : 256;
}
// Does a workgroup of 64 or 128 rows have a second group of waves, for half of its keys?
// Where every sequence and head can have a CU of its own: half as many pieces to join.
// Eight trees of 26 after 8192: 38 us, 43 without; 32 of 32 after 512 29.5 and 35; 64
// (two rounds of CUs) of 32 after 512 49 and 42; some 2 to 3 us more: 16 of 32 after 1024
// 33 and 30, 32 of 8 with 8 heads a group after 512 19.7 and 17.7.
inline bool in_halves(int tile, int64_t seqs, int Hkv) {
  return (tile == 64 || tile == 128) && seqs * Hkv <= 256;
}
// Workgroups that a split aims at, over all KV heads: two a CU, one of eight waves.  64
// chains of 5 after up to 8192: 177 us, 205 with 256; 16 trees of 64 after 8192: 95,
// 109 with 512.
inline int slots(int tile, int64_t seqs, int Hkv) {
  return tile > 128 || in_halves(tile, seqs, Hkv) ? 256 : 512;
}

// At the start of the work buffer.  stamp: as in the batch's; step: the batch's that
// the trees were planned for.
struct Counts {
  int items, joins;
  uint64_t stamp, step;
};

// Byte offsets of the work buffer's parts.
struct Work {
  int tile, target, parts, items;
  int64_t items_at, joins_at, stats, sums;  // of the attention
  int64_t runs, ended, mass, bytes;         // of the verification
  int64_t nodes;                            // rows that a step of trees can have
  bool packed;  // they are the step's rows (else max_nodes a sequence)
};

inline Work work_layout(int64_t seqs, int64_t rows, int Hq, int Hkv, int max_nodes,
                        int max_children) {
  Work w;
  const int G = Hq / Hkv;
  w.tile = tile_rows(max_nodes, G);
  w.target = slots(w.tile, seqs, Hkv) / Hkv > 1 ? slots(w.tile, seqs, Hkv) / Hkv : 1;
  w.parts = 2 * w.target;
  w.packed = rows <= seqs * max_nodes;
  w.nodes = w.packed ? rows : seqs * max_nodes;
  w.items = (int)(w.nodes * G / w.tile + seqs + w.target);
  int64_t at = 256;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  w.items_at = take(w.items * (int64_t)sizeof(Item));
  w.joins_at = take(w.target * (int64_t)sizeof(Join));
  const int part_rows = w.tile < paged::kFewRows ? paged::kFewRows : w.tile;
  w.stats = take(w.parts * (int64_t)Hkv * part_rows * 8);
  w.sums = take(w.parts * (int64_t)Hkv * part_rows * kD * 4);
  // sums of what is left and of the target's own, by runs
  w.runs = take(2 * seqs * kRuns * 8);
  w.ended = take(seqs * kEndedBytes);
  // of each row with children, what is left after one, two, ... of them
  w.mass = take(max_children > 1 ? (max_children - 1) * w.nodes * kRuns * 8 : 0);
  w.bytes = at;
  return w;
}

inline uint64_t schedule_stamp(const ecf8_paged_batch *b, const ecf8_draft_trees *t) {
  uint64_t h = paged::schedule_stamp(b);
  for (const int x : {t->max_nodes, t->max_children})
    for (int byte = 0; byte < 4; ++byte)
      h = (h ^ (((uint32_t)x >> (8 * byte)) & 0xff)) * 0x100000001b3ull;
  return h | 1;
}

inline bool sizes_ok(int64_t seqs, int64_t rows, int Hq, int Hkv, int max_nodes,
                     int max_children) {
  return paged::sizes_ok(seqs, rows, Hq, Hkv) && max_nodes >= 1 && max_nodes <= kMaxNodes &&
         max_children >= 1 && max_children <= kMaxNodes;
}

// How many steps of a batch were planned.
inline const uint64_t *step_of(const ecf8_paged_batch *b) {
  return &static_cast<const paged::Counts *>(b->work)->step;
}

// A batch's and its trees' sizes and pointers.
inline int check_trees(const ecf8_paged_batch *b, const ecf8_draft_trees *t) {
  if (const int rc = paged::check_batch(b)) return rc;
  if (!t || !t->masks || !t->parents || !t->kept || !t->path || !t->emitted || !t->next_token ||
      !t->work || t->max_nodes <= 0 || t->max_children <= 0)
    return ECF8_ERR_INVALID_ARG;
  if (!sizes_ok(b->seqs, b->rows, b->Hq, b->Hkv, t->max_nodes, t->max_children))
    return ECF8_ERR_UNSUPPORTED;
  const uintptr_t longs =
      (uintptr_t)t->masks | (uintptr_t)t->emitted | (uintptr_t)t->next_token;
  const uintptr_t ints = (uintptr_t)t->parents | (uintptr_t)t->kept | (uintptr_t)t->path;
  if ((longs & 7) || (ints & 3) || ((uintptr_t)t->work & 15)) return ECF8_ERR_MISALIGNED;
  if (t->work_bytes <
      work_layout(b->seqs, b->rows, b->Hq, b->Hkv, t->max_nodes, t->max_children).bytes)
    return ECF8_ERR_CAPACITY;
  return ECF8_OK;
}

}  // namespace draft
}  // namespace ecf8

#endif  // ECF8_DRAFT_LAYOUT_H
