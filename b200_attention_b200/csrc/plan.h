// The schedule of a planned attention call (packed sequences, shared prefixes): what the host-side
// planner writes and the kernels read. Plain integers, no CUDA types.
#pragma once

#include <cstdint>
#include <string>
#include <vector>

namespace b200attn {

// A piece: one or two Q tiles of packed rows against a run of 128-key K/V tiles of one K/V head.
// Query heads that share a K/V head are packed into the rows of a tile: row r of a tile is token
// r / group, head r % group of the group, so a tile holds floor(128 / group) tokens.
// A CTA has two lanes, each with a Q tile, scores and an accumulator of its own. A piece of two Q
// tiles takes both, and they share every K/V tile. Pieces of one Q tile are walked two at a time,
// one on each lane, with K/V tiles fetched for the lanes in turn.
struct alignas(16) PlanPiece {
  int32_t token;     // first token (row of q and o)
  int32_t n_tokens;  // tokens of this block, 1 .. 2 * floor(128 / group)
  int32_t kv_row;    // first key: row of k and v (of the prefix's, if source == 1)
  int32_t n_keys;    // keys from kv_row on that belong to this piece
  int32_t tiles[2];  // K/V tiles that each Q tile visits; [0] >= 1, [1] >= [0], or 0: one Q tile
  int32_t diag;      // token i of the block sees keys j <= diag + i, j counted from kv_row
  int32_t kv_head;
  int32_t source;    // 0: k and v, 1: the prefix's
  int32_t slot_row;  // first row of this piece's partial result, or -1: it writes o and lse itself
  int32_t pad[2];
};
static_assert(sizeof(PlanPiece) == 48, "read as three 16-byte words");

// A join unit: a few tokens of one K/V head whose partial results sit in the same pieces.
struct alignas(16) PlanUnit {
  int32_t token, n_tokens, kv_head;
  int32_t part0, parts;  // entries part0 .. part0 + parts - 1 of the part list; none: no key is visible
  int32_t pad[3];
};
static_assert(sizeof(PlanUnit) == 32, "table layout");

// The table as the kernels see it, in 32-bit words: header, the pieces of every CTA as four bounds
// (pieces of two Q tiles, then lane 0's, then lane 1's, end) with its first piece beside them, so that the loads of
// that can start after one look at the table, pieces, units, parts (the row of the partials that holds the unit's first token, head 0 of the group).
constexpr int kPlanMaxCtas = 160;
constexpr int kPlanMagic = 0x62706c33;
enum PlanHeader : int { kPlanHdrMagic = 0, kPlanHdrPieces, kPlanHdrUnits, kPlanHdrUnitAt, kPlanHdrPartAt, kPlanHeaderWords = 16 };
constexpr int kPlanCtaAt = kPlanHeaderWords;
constexpr int kPlanCtaWords = 16;  // the bounds, and a copy of the CTA's first piece
constexpr int kPlanPieceAt = kPlanCtaAt + kPlanCtaWords * kPlanMaxCtas;

constexpr int kPlanJoinRows = 32;  // most rows of a join unit (one token at least)
constexpr int32_t kPlanNoDiag = 1 << 30;

struct PlanInput {
  int32_t sequences;
  const int32_t* len_q;
  const int32_t* len_kv;
  const int64_t* start_kv;  // or nullptr: back to back
  int32_t len_prefix;
  int32_t heads, heads_kv;
  bool causal;
  int32_t sm_count;
};

struct Plan {
  std::vector<int32_t> table;
  int32_t grid = 0;       // CTAs that have a piece
  int32_t pieces = 0;
  int32_t units = 0;
  int32_t wide_pieces = 0;  // of two Q tiles
  int64_t slot_rows = 0;  // rows of fp32 partials that the pieces write
  int64_t rows_q = 0;     // rows of q and o that the plan covers
  int64_t rows_kv = 0;    // rows of k and v that it may read: past the last key of any sequence
};

// Fills `plan`; returns "" or what is wrong with the input.
std::string plan_build(const PlanInput& in, Plan* plan);

inline int32_t plan_tile_tokens(int32_t group) { return 128 / group; }
inline int32_t plan_small_tokens(int32_t group) { return 32 / group; }

}  // namespace b200attn
