// Planned attention for sm_100a: packed sequences of different lengths, grouped heads, causal masks, and
// requests that share a prefix, in one persistent kernel that walks a schedule made on the host
// (plan.cpp), and a second small kernel that joins partial results.
//
//   O_i = sum_j p_ij V_j,  p_ij = 2^(c s_ij - m_i) / sum_j 2^(c s_ij - m_i),  s = Q K^T,  c = scale * log2(e)
//   joining two runs of keys a and b of a row:  lse = log(e^lse_a + e^lse_b),
//   O = O_a e^(lse_a - lse) + O_b e^(lse_b - lse)
//
// The kernel is built like attn_fwd_ws_kernel (same tiles, descriptors, TMEM layout and softmax):
//   warps 0-3, 4-7  softmax of Q tile 0 / 1, a row per thread
//   warps 8-11      epilogue: bf16 O and LSE, or an fp32 partial (a lane's last piece: its softmax warps)
//   warp 12         tcgen05.mma     warp 13  TMA loads
//   warp 14         clears the rows of a V tile behind the last key: they belong to another sequence or to
//                   memory nobody wrote, and 0 * NaN is NaN in the product P V
// What differs is where work comes from. Query heads that share a K/V head are packed into the rows of a
// tile (row = token * group + head of the group, which is one TMA box of floor(128 / group) tokens x group
// heads), so a K/V tile is read once for the whole group, a single token fills `group` rows instead of one,
// and a block of rows spans fewer tokens and so fewer tiles that the causal diagonal cuts.
//
// Pieces of two Q tiles (long prompts, wide batches on a prefix) share every K/V tile, as in the kernel above, and are
// bound like it by the chain scores -> softmax -> PV of two tiles that fill each other's gaps. A piece of one Q tile
// (single tokens, short prompts) would run that chain without a partner; so two such pieces run side by side, one on
// each of the CTA's two lanes, and the K/V ring serves the lanes in turn (LaneWalk). Where such pieces have at most
// 32 rows, a lane's Q buffer holds four of them and their loads run ahead, so that a lane goes from piece to piece
// without waiting for Q. (The tensor cores read 128 rows from there: rows that are not the piece's own give scores
// that nobody looks at.)
//
// Measured on a B200 (calls back to back; a plain copy reaches 6.4 TB/s, a cuBLAS bf16 product 1658 TFLOPS in a burst and
// 1400 under the power cap):
//   one prompt of 16384 tokens, 16 heads, causal    0.84 ms in a burst (1300 TFLOPS), 0.99 ms under the power cap (1110);
//       1.47 M cycles, tensor pipe busy 62 % of them: bound by the chain, as attn_fwd_ws_kernel (1.45 M) is
//   64 single tokens, 32 + 8 heads, 100-12000 keys  0.23 to 0.25 ms from GPU to GPU in a burst (5.6 to 6.1 TB/s), 0.26 for
//       long (5.3): bound by memory
//   64 tokens behind 32768 shared rows, 32 + 8 heads, up to 1024 keys of their own    72 to 81 us, 3.3 to 3.7 TB/s: half
//       the CTAs work on the prefix (chain), half on short runs of keys, which each have a start, a hand-over and a partial
//       result of their own
//   one token, 128 keys                             5 us: load, scores, softmax, product, store one after the other
// Asked for and not kept, being slower: K/V tiles prefetched into the L2 two to six ahead (single tokens 235 -> 289 us and
// more), a third slot in the K/V ring for CTAs of small pieces (228 -> 232 us), boxes of 32 rows for the tile in which a
// sequence ends (single tokens 1 % faster, prompts 1.5 % slower).

#include "attn_device_sm100.cuh"
#include "launch_overlap.cuh"
#include "plan_kernels.cuh"

namespace b200attn {

namespace {

constexpr int kPairSlotsP = 2;
constexpr int kPairBytesP = 2 * kTileBytes;
constexpr int kPlanThreads = 512;
// Registers per thread of the three kinds of warps (128 in the mean). Against 184 / 64 / 80: 3 % at 8 prompts of 1 to
// 8192 tokens; against 192 / 56 / 72: 2 %.
constexpr int kPlanRegsSoftmax = 192;
constexpr int kPlanRegsEpilogue = 48;
constexpr int kPlanRegsOther = 80;
constexpr int kQSlots = 4;        // small Q tiles that a lane's buffer holds
constexpr int kQSlotRows = 32;    // rows of each
constexpr int kPieceCache = 192;  // pieces of a CTA kept in shared memory; further ones are read from the table

enum PlanBarrier : int {
  kPbQFull = 0,       // +lane * kQSlots + slot   TMA -> MMA
  kPbQEmpty = 8,      // +lane * kQSlots + slot   MMA -> TMA
  kPbSFull = 16,      // +lane  MMA -> softmax
  kPbPReady = 18,     // +lane  softmax (4 warps) -> MMA
  kPbPvDone = 20,     // +lane  MMA -> epilogue
  kPbFin = 22,        // +lane  softmax (4 warps) -> epilogue
  kPbFinFree = 24,    // +lane  epilogue (4 warps) -> softmax
  kPbOFree = 26,      // +lane  epilogue (4 warps) -> MMA
  kPbPairFull = 28,   // +slot  TMA -> MMA, warp 14
  kPbPairEmpty = 30,  // +slot  MMA and warp 14 -> TMA
  kPbTailClean = 32,  // +slot  warp 14 -> MMA: the rows of a V tile behind the last key are zero
  kPbDrain = 34,
  kNumPlanBarriers = 35
};

__device__ __forceinline__ uint32_t plan_barrier_count(int i) {
  if ((i >= kPbPReady && i < kPbPvDone) || (i >= kPbFin && i < kPbPairFull)) return 4;  // a warpgroup's four warps
  return i >= kPbPairEmpty && i < kPbTailClean ? 2 : 1;
}

struct alignas(16) PlanAux {
  uint64_t bar[kNumPlanBarriers];
  float row_max[kQTilesPerItem][kBlockM];
  float row_sum[kQTilesPerItem][kBlockM];
  uint32_t tmem_base;
  alignas(16) uint32_t abort_flag;  // NotedWait: where the wait was that ran out,
  uint32_t timeout[3];              // warp * 2 + parity, piece, tile
  int32_t first[4];  // pieces of two Q tiles, lane 0's, lane 1's, end; counted in the whole table
  PlanPiece cache[kPieceCache];
};

constexpr int kPlanSmemBytes = kQTilesPerItem * kTileBytes + kPairSlotsP * kPairBytesP + int(sizeof(PlanAux));
static_assert(kPlanSmemBytes <= 227 * 1024, "shared memory of a CTA");

// Waits of short code: one loop, and a timeout is noted in shared memory (from the abort flag on), for the CTA to report
// when it ends. For launches without pieces of two Q tiles. There a round of two short pieces runs through more code than
// an SM's instruction cache holds (137 requests to the GPC's cache for each piece of one K/V tile, 33 for a second tile), the
// caches behind it serve the SMs of a GPC together, and CTAs in larger GPCs take longer for the same work (148 tokens of
// 128 keys: 17 us with 12 SMs to a GPC, 25 us with 20). With these waits in the place of WaitCtx's:
//   148 tokens, 32 + 8 heads, of 128 / 256 / 300 keys   29.0 / 38.7 / 49.9 -> 27.4 / 35.4 / 47.1 us
//   100 tokens of 5-600 keys                            44.8 -> 42.4 us
//   64 tokens of 100-12000 keys                         238 -> 236 us
// Prompts are 3 to 6 % slower with them (16384 tokens, 16 heads: 956 -> 1013 us). WaitCtx's build spills 24 bytes a
// thread, which are loaded 368 bytes' worth; without its constants in registers that falls to 76 and prompts take 1 to
// 3 % longer. Scores taken 32 at a time in a loop (half the code of a tile) cost 6 % at 64
// tokens of 100-12000 keys, MMAs issued in loops 2 %.
struct NotedWait : WaitCtx {
  __device__ __forceinline__ void note(int site, uint32_t parity) const {
    const uint32_t who = (threadIdx.x >> 5) * 2 + parity;
    asm volatile("st.volatile.shared::cta.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(abort_addr), "r"(site), "r"(who),
                 "r"(item), "r"(tile)
                 : "memory");
  }
  __device__ __forceinline__ bool wait_issue(uint32_t bar, uint32_t parity, int site) const {
    return wait_warp(bar, parity, site);
  }
  __device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int site) const {
    bool ok = false;
    uint64_t t0 = 0;
    uint32_t n = 0;
    while (true) {
      ok = ok || mbar_try_wait(bar, parity, 0);  // a lane that has seen the phase end does not look again
      if (__all_sync(0xffffffffu, ok)) return true;
      if (__builtin_expect((++n & 63u) == 0, 0)) {
        const uint64_t now = global_timer_ns();
        if (t0 == 0) t0 = now;
        bool over = aborted();
        if (!over && now - t0 > limit_ns) {
          note(site, parity);
          over = true;
        }
        if (__any_sync(0xffffffffu, over)) return false;
      }
    }
  }
};

__device__ __forceinline__ void pass_on(const WaitCtx&, const PlanAux*) {}
// By one thread, after every role has ended.
__device__ __forceinline__ void pass_on(const NotedWait& w, const PlanAux* aux) {
  if (aux->abort_flag == 0 || w.status == nullptr || atomicCAS(w.status, 0, kDevWaitTimeout) != 0) return;
  w.status[1] = int(aux->abort_flag);
  w.status[2] = int(blockIdx.x);
  w.status[3] = int(aux->timeout[0] >> 1);
  w.status[4] = int(aux->timeout[0] & 1u);
  w.status[5] = int(aux->timeout[1]);
  w.status[6] = int(aux->timeout[2]);
  __threadfence_system();
}

// The CTA's pieces, counted from its first one: [0, pairs) take both lanes, [pairs, lane1) are lane 0's, [lane1, end)
// lane 1's. Every role walks them in the same order: the first kind one by one, the others with LaneWalk.
struct Pieces {
  const PlanAux* aux;
  const PlanPiece* table;
  int pairs, lane1, end;
  __device__ __forceinline__ Pieces(const PlanParams& p, const PlanAux* a)
      : aux(a), table(reinterpret_cast<const PlanPiece*>(p.table + kPlanPieceAt) + a->first[0]),
        pairs(a->first[1] - a->first[0]), lane1(a->first[2] - a->first[0]), end(a->first[3] - a->first[0]) {}
  __device__ __forceinline__ int last_of(int lane) const {  // -1: none
    return lane ? (end > lane1 ? end - 1 : pairs - 1) : (lane1 > pairs ? lane1 - 1 : pairs - 1);
  }
  __device__ __forceinline__ const PlanPiece* at(int i) const { return i < kPieceCache ? &aux->cache[i] : table + i; }
};

__device__ __forceinline__ PlanPiece piece_of(int4 a, int4 b, int4 c) {
  PlanPiece p;
  p.token = a.x;
  p.n_tokens = a.y;
  p.kv_row = a.z;
  p.n_keys = a.w;
  p.tiles[0] = b.x;
  p.tiles[1] = b.y;
  p.diag = b.z;
  p.kv_head = b.w;
  p.source = c.x;
  p.slot_row = c.y;
  return p;
}

// Steps of the pieces of one Q tile: a K/V tile of lane 0, one of lane 1, and so on; a lane that has run out leaves
// the turns to the other.
struct LaneWalk {
  int next[2], end[2], tile[2], tiles[2];
  int turn;
  __device__ __forceinline__ explicit LaneWalk(const Pieces& ps) : turn(0) {
    next[0] = ps.pairs;
    end[0] = next[1] = ps.lane1;
    end[1] = ps.end;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      tile[q] = 0;
      tiles[q] = next[q] < end[q] ? ps.at(next[q])->tiles[0] : 0;
    }
  }
  struct Step {
    int lane, piece, tile;
    bool last;  // of its piece
  };
  __device__ __forceinline__ bool more() const { return next[0] < end[0] || next[1] < end[1]; }
  __device__ __forceinline__ bool take(const Pieces& ps, Step& s) {
    if (!more()) return false;
    const bool other = turn ? next[1] >= end[1] : next[0] >= end[0];
    s.lane = other ? turn ^ 1 : turn;
    turn = s.lane ^ 1;
    if (s.lane == 0)
      advance<0>(ps, s);
    else
      advance<1>(ps, s);
    return true;
  }
  template <int q>
  __device__ __forceinline__ void advance(const Pieces& ps, Step& s) {
    s.piece = next[q];
    s.tile = tile[q];
    s.last = ++tile[q] == tiles[q];
    if (s.last) {
      tile[q] = 0;
      if (++next[q] < end[q]) tiles[q] = ps.at(next[q])->tiles[0];
    }
  }
  // the piece that follows on a lane whose piece has just had its last step, or null
  __device__ __forceinline__ const PlanPiece* following(const Pieces& ps, int lane) const {
    const int n = lane ? next[1] : next[0];
    return n < (lane ? end[1] : end[0]) ? ps.at(n) : nullptr;
  }
};

__device__ __forceinline__ int piece_tiles(const PlanPiece* pc) { return max(pc->tiles[0], pc->tiles[1]); }

// Keys in the last tile that the piece visits, if its keys end inside it; 0 otherwise.
__device__ __forceinline__ int piece_tail(const PlanPiece* pc) {
  const int in_last = pc->n_keys - (piece_tiles(pc) - 1) * kBlockN;
  return in_last < kBlockN ? in_last : 0;
}

// Pieces of one Q tile with few rows; on every lane they come after the larger ones.
__device__ __forceinline__ bool is_small(const PlanParams& p, const PlanPiece* pc) {
  return pc->tiles[1] == 0 && pc->n_tokens <= p.small_tokens;
}

// ---- TMA producer: K/V in pairs (V of one tile, K of the next), as in attn_fwd_ws_kernel -----------------
template <class Wait>
struct Loader {
  const PlanParams& p;
  const PlanMaps& maps;
  uint32_t smem_q, smem_kv, bar0, lead;
  uint32_t slot = 0, empty_parity = 1;   // parity 1 passes on a fresh barrier
  uint32_t q_empty_parity = 0xff;        // bit per Q slot
  uint32_t small_loaded[2] = {0, 0};     // small pieces of each lane: the next one goes to slot small_loaded % 4
  uint32_t armed = 0, armed_parity = 0;  // for the early-exit path: "full" barriers armed, last parity of each

  __device__ __forceinline__ Loader(const PlanParams& p_, const PlanMaps& m_, uint32_t q_, uint32_t kv_, uint32_t b_,
                                    uint32_t lead_)
      : p(p_), maps(m_), smem_q(q_), smem_kv(kv_), bar0(b_), lead(lead_) {}
  __device__ __forceinline__ uint32_t bar(int i) const { return bar0 + 8u * uint32_t(i); }

  // V tile of one piece (or none) and K tile of one (or none) to the next slot of the ring.
  template <bool kFresh = false>  // on barriers that nobody has used yet
  __device__ __forceinline__ bool push_pair(const PlanPiece* v_pc, int v_tile, const PlanPiece* k_pc, int k_tile, int site,
                                            const Wait& w) {
    if (!kFresh && !w.wait_issue(bar(kPbPairEmpty + slot), empty_parity, site)) return false;
    const uint32_t full_parity = empty_parity ^ 1u;
    armed |= 1u << slot;
    armed_parity = (armed_parity & ~(1u << slot)) | (full_parity << slot);
    const uint32_t full = bar(kPbPairFull + slot);
    const uint32_t dst = smem_kv + slot * kPairBytesP;
    mbar_arrive_expect_tx_lead(lead, full, (v_pc != nullptr ? kTileBytes : 0) + (k_pc != nullptr ? kTileBytes : 0));
    if (v_pc != nullptr) {
      const CUtensorMap* tv = v_pc->source ? &maps.v_prefix : &maps.v;
      const int row = v_pc->kv_row + v_tile * kBlockN, h = v_pc->kv_head;
      tma_load_4d_lead(lead, dst, tv, 0, row, h, 0, full);
      tma_load_4d_lead(lead, dst + kBoxBytes, tv, 64, row, h, 0, full);
    }
    if (k_pc != nullptr) {
      const CUtensorMap* tk = k_pc->source ? &maps.k_prefix : &maps.k;
      const int row = k_pc->kv_row + k_tile * kBlockN, h = k_pc->kv_head;
      tma_load_4d_lead(lead, dst + kTileBytes, tk, 0, row, h, 0, full);
      tma_load_4d_lead(lead, dst + kTileBytes + kBoxBytes, tk, 64, row, h, 0, full);
    }
    slot ^= 1u;
    if (slot == 0) empty_parity ^= 1u;
    return true;
  }

  // Q tile `tile` of a piece to a lane: a box of 64 columns x group heads x tokens lands as rows
  // token * group + head.
  template <bool kFresh = false>
  __device__ __forceinline__ bool load_q(const PlanPiece* pc, int lane, int tile, const Wait& w) {
    const bool small = is_small(p, pc);
    uint32_t n = 0;  // slot
    if (small) n = (lane ? small_loaded[1]++ : small_loaded[0]++) % kQSlots;
    const int s = lane * kQSlots + int(n);
    if (!kFresh && !w.wait_issue(bar(kPbQEmpty + s), (q_empty_parity >> s) & 1u, 100 + s)) return false;
    q_empty_parity ^= 1u << s;
    armed |= 1u << (kPairSlotsP + s);
    armed_parity = (armed_parity & ~(1u << (kPairSlotsP + s))) | (((q_empty_parity >> s) & 1u) << (kPairSlotsP + s));
    const uint32_t full = bar(kPbQFull + s), dst = smem_q + lane * kTileBytes + n * (kQSlotRows * 128);
    const CUtensorMap* tq = small ? &maps.q_small : &maps.q;
    const int token = pc->token + tile * p.tile_tokens;
    mbar_arrive_expect_tx_lead(lead, full, uint32_t((small ? p.small_tokens * p.group : p.tile_rows) * kHeadDim * 2));
    tma_load_4d_lead(lead, dst, tq, 0, 0, pc->kv_head, token, full);
    tma_load_4d_lead(lead, dst + kBoxBytes, tq, 64, 0, pc->kv_head, token, full);
    return true;
  }

  // Q and the first K tile (which travels alone) of the CTA's first piece.
  __device__ __forceinline__ void begin(const PlanPiece* pc, const Wait& w) {
    load_q<true>(pc, 0, 0, w);
    push_pair<true>(nullptr, 0, pc, 0, 110, w);
    if (pc->tiles[1] > 0) load_q<true>(pc, 1, 1, w);
  }

  __device__ void run(const PlanAux* aux, Wait& w) {
    const Pieces ps(p, aux);
    bool ok = true;
    for (int n = 0; ok && n < ps.pairs; ++n) {
      const PlanPiece* pc = ps.at(n);
      const int T = pc->tiles[1];
      w.item = n;
      w.tile = 0;
      for (int q = 0; ok && n > 0 && q < kQTilesPerItem; ++q) ok = load_q(pc, q, q, w);
      for (int i = 0; ok && i < T; ++i) {
        w.tile = i;
        // the last V with the first K of the CTA's next piece, if any (it is lane 0's, if the pairs end here)
        const bool last = i + 1 == T;
        ok = push_pair(pc, i, !last ? pc : n + 1 < ps.end ? ps.at(n + 1) : nullptr, last ? 0 : i + 1, 111, w);
      }
    }
    if (ok && ps.end > ps.pairs) {
      // Q of a lane's pieces up to three ahead of piece `done`, or one ahead while pieces fill the whole buffer. The
      // first small piece goes to slot 0 and so waits for the last large one; the others then find theirs free.
      int next_q[2] = {ps.pairs, ps.lane1};
      auto load_ahead = [&](int lane, int done, int most) -> bool {
        int n = lane ? next_q[1] : next_q[0];
        const int end = min(lane ? ps.end : ps.lane1, n + most);
        while (n < end && (n == done + 1 || (n < done + kQSlots && is_small(p, ps.at(done + 1))))) {
          if (!load_q(ps.at(n), lane, 0, w)) return false;
          ++n;
        }
        if (lane) next_q[1] = n; else next_q[0] = n;
        return true;
      };
      LaneWalk walk(ps);
      if (ps.pairs == 0) next_q[0] = 1; else ok = load_ahead(0, ps.pairs - 1, 1);
      if (ok && ps.lane1 < ps.end)
        ok = load_ahead(1, ps.lane1 - 1, 1) && push_pair(nullptr, 0, ps.at(ps.lane1), 0, 114, w);
      LaneWalk::Step st;
      while (ok && walk.take(ps, st)) {
        const PlanPiece* pc = ps.at(st.piece);
        w.item = st.piece;
        w.tile = st.tile;
        const PlanPiece* k_pc = st.last ? walk.following(ps, st.lane) : pc;
        ok = push_pair(pc, st.tile, k_pc, st.last ? 0 : st.tile + 1, 115, w);
        // a piece's first step fetches ahead; so does its last, in case the next piece had to wait for the buffer
        if (ok && (st.last || st.tile == 0)) ok = load_ahead(st.lane, st.last ? st.piece : st.piece - 1, kQSlots);
      }
    }

    if (!ok || w.aborted()) {
      for (int s = 0; s < kPairSlotsP + 2 * kQSlots; ++s) {
        if (!((armed >> s) & 1u)) continue;
        const uint32_t b = (s < kPairSlotsP) ? bar(kPbPairFull + s) : bar(kPbQFull + (s - kPairSlotsP));
        const uint64_t t0 = global_timer_ns();
        while (!mbar_try_wait(b, (armed_parity >> s) & 1u, 1000)) {
          if (global_timer_ns() - t0 > w.limit_ns) break;
        }
      }
    }
  }
};

// ---- V tails ------------------------------------------------------------------------------------------
// Sees every pair (it takes part in handing pairs back, so it can never miss a phase). Where the V tile holds
// the end of a piece's keys inside it, the rows behind are set to zero before the MMA warp may use the tile.
template <class Wait>
__device__ void plan_tail_role(const PlanParams& p, const PlanAux* aux, uint8_t* kv, uint32_t bar0, int lane,
                               Wait& w) {
  auto bar = [&](int i) { return bar0 + 8u * uint32_t(i); };
  uint32_t slot = 0, full_parity = 0;
  auto next_pair = [&](int tail) -> bool {  // tail: keys in the V tile, 0 = all of them (or no V tile)
    if (!w.wait_warp(bar(kPbPairFull + slot), full_parity, 600)) return false;
    if (tail > 0) {
      for (int box = 0; box < 2; ++box) {
        uint4* row = reinterpret_cast<uint4*>(kv + slot * kPairBytesP + box * kBoxBytes + tail * 128);
        const int words = (kBlockN - tail) * 8;
        for (int j = lane; j < words; j += 32) row[j] = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
    }
    __syncwarp();
    if (lane == 0) {
      if (tail > 0) mbar_arrive(bar(kPbTailClean + slot));
      mbar_arrive(bar(kPbPairEmpty + slot));
    }
    slot ^= 1u;
    if (slot == 0) full_parity ^= 1u;
    return true;
  };
  const Pieces ps(p, aux);
  if (ps.pairs > 0 && !next_pair(0)) return;
  for (int n = 0; n < ps.pairs; ++n) {
    const PlanPiece* pc = ps.at(n);
    const int T = pc->tiles[1];
    w.item = n;
    for (int i = 0; i < T; ++i) {
      w.tile = i;
      if (!next_pair(i + 1 == T ? piece_tail(pc) : 0)) return;
    }
  }
  if (ps.end > ps.pairs) {
    if (ps.pairs == 0 && !next_pair(0)) return;
    if (ps.lane1 < ps.end && !next_pair(0)) return;
    LaneWalk walk(ps);
    LaneWalk::Step st;
    while (walk.take(ps, st)) {
      w.item = st.piece;
      w.tile = st.tile;
      if (!next_pair(st.last ? piece_tail(ps.at(st.piece)) : 0)) return;
    }
  }
}

// ---- MMA issuer ---------------------------------------------------------------------------------------
template <class Wait>
__device__ void plan_mma_role(const PlanParams& p, const PlanAux* aux, uint32_t smem_q, uint32_t smem_kv,
                              uint32_t bar0, uint32_t tmem_base, uint32_t lead, Wait& w) {
  auto bar = [&](int i) { return bar0 + 8u * uint32_t(i); };
  uint32_t slot = 0, full_parity = 0;
  uint32_t tail_parity = 0;      // bit per slot
  uint32_t p_parity = 0;         // bit per lane
  uint32_t q_full_parity = 0;    // bit per Q slot
  uint32_t small_used[2] = {0, 0};
  uint32_t q_slot[2] = {0, kQSlots};  // of the piece on each lane
  uint32_t o_free_parity = 3;    // passes on the fresh barrier: both accumulators start out free
  bool ok = true, k_ready = false;

  auto wait_pair = [&](int site) -> bool {
    if (!w.wait_issue(bar(kPbPairFull + slot), full_parity, site)) return false;
    slot ^= 1u;
    if (slot == 0) full_parity ^= 1u;
    return true;  // the pair is the one in slot ^ 1
  };
  // Scores of a lane's piece with a K tile; after its last one the Q slot is free.
  auto scores = [&](int lane, uint32_t k_smem, bool last) {
    const uint32_t s = lane ? q_slot[1] : q_slot[0];
    const uint32_t q = smem_q + lane * kTileBytes + (s % kQSlots) * (kQSlotRows * 128);
    issue_qk(lead, tmem_base + lane * kBlockN, q, k_smem);
    umma_commit_lead(lead, bar(kPbSFull + lane));
    if (last) umma_commit_lead(lead, bar(kPbQEmpty + s));
  };
  // First scores of a piece on a lane, K in the pair waited for last.
  auto first_scores = [&](int lane, const PlanPiece* pc, int tiles) -> bool {
    const uint32_t s = lane * kQSlots + (is_small(p, pc) ? (lane ? small_used[1]++ : small_used[0]++) % kQSlots : 0u);
    if (!w.wait_issue(bar(kPbQFull + s), (q_full_parity >> s) & 1u, 201 + lane)) return false;
    q_full_parity ^= 1u << s;
    if (lane) q_slot[1] = s; else q_slot[0] = s;
    tc_fence_after_sync();
    scores(lane, smem_kv + (slot ^ 1u) * kPairBytesP + kTileBytes, tiles == 1);
    return true;
  };
  // The V tile of the pair waited for last, if a piece's keys end inside it, once its other rows are zero.
  auto wait_tail = [&]() -> bool {
    const uint32_t s = slot ^ 1u;
    if (!w.wait_issue(bar(kPbTailClean + s), (tail_parity >> s) & 1u, 211)) return false;
    tail_parity ^= 1u << s;
    return true;
  };
  // PV of tile i on a lane, once its probabilities are there and, for the first tile, its accumulator has been read
  // out by the epilogue of the piece before.
  auto weighted_sum = [&](int lane, int i, uint32_t v_smem) -> bool {
    if (i == 0) {
      if (!w.wait_issue(bar(kPbOFree + lane), (o_free_parity >> lane) & 1u, 240 + lane)) return false;
      o_free_parity ^= 1u << lane;
    }
    if (!w.wait_issue(bar(kPbPReady + lane), (p_parity >> lane) & 1u, 220 + lane)) return false;
    p_parity ^= 1u << lane;
    tc_fence_after_sync();
    issue_pv(lead, tmem_base + kQTilesPerItem * kBlockN + lane * kHeadDim, tmem_base + lane * kBlockN, v_smem, i > 0);
    return true;
  };

  const Pieces ps(p, aux);
  for (int n = 0; ok && n < ps.pairs; ++n) {
    const PlanPiece* pc = ps.at(n);
    const int Tq[kQTilesPerItem] = {pc->tiles[0], pc->tiles[1]};
    const int T = Tq[1];
    const bool tail = piece_tail(pc) > 0;
    w.item = n;
    w.tile = 0;
    if (!k_ready) {
      if (!(ok = wait_pair(200))) break;
      k_ready = true;
    }
#pragma unroll
    for (int q = 0; q < kQTilesPerItem; ++q) ok = ok && first_scores(q, pc, Tq[q]);
    if (!ok) break;
    // also covers the PV of the previous piece that read the V half of this pair
    umma_commit_lead(lead, bar(kPbPairEmpty + (slot ^ 1u)));

    for (int i = 0; ok && i < T; ++i) {
      w.tile = i;
      // V_i and K_{i+1} (or K_0 of this CTA's next piece) in one phase
      if (!(ok = wait_pair(210))) break;
      const uint32_t v_smem = smem_kv + (slot ^ 1u) * kPairBytesP;
      const uint32_t k_smem = v_smem + kTileBytes;
      if (tail && i + 1 == T && !(ok = wait_tail())) break;
#pragma unroll
      for (int q = 0; q < kQTilesPerItem; ++q) {
        if (i < Tq[q]) {
          if (!(ok = weighted_sum(q, i, v_smem))) break;
          if (i + 1 < Tq[q]) {
            scores(q, k_smem, i + 2 == Tq[q]);
          } else {
            umma_commit_lead(lead, bar(kPbPvDone + q));
          }
        }
      }
      if (ok && i + 1 < T) umma_commit_lead(lead, bar(kPbPairEmpty + (slot ^ 1u)));
    }
  }
  if (ok && ps.end > ps.pairs) {
    LaneWalk walk(ps);
    if (!k_ready) ok = wait_pair(203);
    ok = ok && first_scores(0, ps.at(ps.pairs), walk.tiles[0]);
    if (ok) umma_commit_lead(lead, bar(kPbPairEmpty + (slot ^ 1u)));
    if (ok && ps.lane1 < ps.end) {
      ok = wait_pair(204) && first_scores(1, ps.at(ps.lane1), walk.tiles[1]);
      if (ok) umma_commit_lead(lead, bar(kPbPairEmpty + (slot ^ 1u)));
    }
    LaneWalk::Step st;
    while (ok && walk.take(ps, st)) {
      w.item = st.piece;
      w.tile = st.tile;
      const int lane = st.lane;
      if (!(ok = wait_pair(212))) break;
      const uint32_t v_smem = smem_kv + (slot ^ 1u) * kPairBytesP;
      if (st.last && piece_tail(ps.at(st.piece)) > 0 && !(ok = wait_tail())) break;
      if (!(ok = weighted_sum(lane, st.tile, v_smem))) break;
      if (!st.last) {
        scores(lane, v_smem + kTileBytes, st.tile + 2 == (lane ? walk.tiles[1] : walk.tiles[0]));
      } else {
        umma_commit_lead(lead, bar(kPbPvDone + lane));
        const PlanPiece* following = walk.following(ps, lane);
        if (following != nullptr && !(ok = first_scores(lane, following, following->tiles[0]))) break;
      }
      // nobody waits for the last pair to be handed back, and the CTA may be gone by then
      if (walk.more()) umma_commit_lead(lead, bar(kPbPairEmpty + (slot ^ 1u)));
    }
  }

  if (!ok || w.aborted()) {
    // Leaving early: make sure nothing this warp issued is still running before TMEM goes.
    umma_commit_lead(lead, bar(kPbDrain));
    const uint64_t t0 = global_timer_ns();
    while (!mbar_try_wait(bar(kPbDrain), 0, 1000)) {
      if (global_timer_ns() - t0 > w.limit_ns) break;
    }
  }
}

// ---- the result of a row ---------------------------------------------------------------------------------------
// The calling thread's row r of a Q tile: normalised O (from TMEM, `o_row`) and LSE, to o and lse or to the piece's
// partial result. Called by whole warps; kLoads x 16 columns are read at a time.
template <int kLoads>
__device__ __forceinline__ void store_result(const PlanParams& p, const PlanPiece* pc, int tile, int r, float m, float l,
                                             uint32_t o_row) {
  const int token_in_tile = r / p.group, head_in_group = r - token_in_tile * p.group;
  const int token = tile * p.tile_tokens + token_in_tile;  // of the block
  const bool live = r < p.tile_rows && token < pc->n_tokens;
  if (!__any_sync(0xffffffffu, live)) return;
  const bool seen = l != 0.0f;  // false: the row saw no key (a NaN sum counts as seen)
  const float weight = 1.0f / l;
  const float lse = seen ? (m + log2f(l)) * kLn2 : kNegInf;
  const int slot_row = pc->slot_row;
  const int head = pc->kv_head * p.group + head_in_group;
  const int64_t row = int64_t(pc->token) + token;
  float* part = nullptr;
  __nv_bfloat16* out = nullptr;
  if (live) {
    if (slot_row >= 0) {
      const int64_t at = int64_t(slot_row) + token * p.group + head_in_group;
      part = p.part_o + at * kHeadDim;
      p.part_lse[at] = lse;
    } else {
      out = p.o + row * p.o_stride_t + int64_t(head) * p.o_stride_h;
      if (p.lse != nullptr) p.lse[int64_t(head) * p.lse_stride_h + row] = lse;
    }
  }
  constexpr int kChunk = 16;
#pragma unroll 1
  for (int c = 0; c < kHeadDim / kChunk; c += kLoads) {
    __syncwarp();
    uint32_t acc[kLoads][kChunk];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) tmem_ld16(o_row + (c + u) * kChunk, acc[u]);
    tmem_wait_ld();
    if (live) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        float v[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; ++j) v[j] = seen ? __uint_as_float(acc[u][j]) * weight : 0.0f;
        if (slot_row >= 0) {
          char* dst = reinterpret_cast<char*>(part + (c + u) * kChunk);
#pragma unroll
          for (int j = 0; j < kChunk; j += 8)
            st_global_32b(dst + 4 * j, make_uint4(__float_as_uint(v[j]), __float_as_uint(v[j + 1]), __float_as_uint(v[j + 2]), __float_as_uint(v[j + 3])),
                          make_uint4(__float_as_uint(v[j + 4]), __float_as_uint(v[j + 5]), __float_as_uint(v[j + 6]), __float_as_uint(v[j + 7])));
        } else {
          uint4* dst = reinterpret_cast<uint4*>(out + (c + u) * kChunk);
          uint4 w[kChunk / 8];
#pragma unroll
          for (int j = 0; j < kChunk / 8; ++j)
            w[j] = make_uint4(pack_bf16x2(v[8 * j + 0], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                              pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
          if (p.o_aligned) {
            st_global_32b(dst, w[0], w[1]);
          } else {
            dst[0] = w[0];
            dst[1] = w[1];
          }
        }
      }
    }
  }
  __syncwarp();
}

// ---- softmax: one row per thread -------------------------------------------------------------------------
// As in attn_fwd_ws_kernel: the first tile is taken with its maximum, later ones speculate against the row's reference
// and go the exact way where the tile's sum says that it has to move. The maximum comes first because the largest
// probability of a row is then 2^0 = 1 and loses nothing when it is rounded to bf16: where one key of the first tile
// outweighs the others (its score 9 to 15, theirs about N(0, 1)) a reference of 0 rounds all of the row's result once
// more, by up to 2^-8 (error against 64 bits, of the norm: single tokens of 128 keys 0.0021 -> 0.0013, of 1024 0.0024 ->
// 0.0016, of 4096 0.0024 -> 0.0017, prompts of 1024 0.0021 -> 0.0015), and with a few keys it does so for any scores. It
// costs a part of one tile's time per piece: 148 tokens of 128 keys 26.2 -> 27.3 us, of 256 34.5 -> 35.3, of 300 46.2 ->
// 46.9, 64 of 100-2000 53.1 -> 53.4, 64 of 100-12000 230 either way, whole prompts no more (16384 tokens 850 -> 843).
// One difference: rows that see no key of a tile, or of the whole piece. Their m becomes -inf, which sends them down the
// exact path, where it is subtracted as 0 so that every probability is 2^-inf = 0.
template <class Wait>
__device__ void plan_softmax_role(const PlanParams& p, PlanAux* aux, uint32_t bar0, uint32_t tmem_base, int q,
                                  int warp_in_group, int lane, Wait& w) {
  auto bar = [&](int i) { return bar0 + 8u * uint32_t(i); };
  const float sum_limit = exp2f(B200ATTN_REBASE_LOG2);
  const uint32_t lane_field = uint32_t(warp_in_group * 32) << 16;
  const uint32_t s_tmem = tmem_base + q * kBlockN + lane_field;
  const uint32_t p_tmem = s_tmem;  // bf16 P overwrites S columns 0..63
  const uint32_t o_tmem = tmem_base + kQTilesPerItem * kBlockN + q * kHeadDim + lane_field;
  const int r = warp_in_group * 32 + lane;
  const float scale_log2 = p.scale_log2;
  const f2 scale2 = f2_splat(scale_log2);
  uint32_t s_parity = 0, fin_free_parity = 1;
  uint32_t pieces = 0;  // of this lane, so far

  for (int n = 0;; ++n) {
    int T, tile_limit, row_limit, rows;
    {
      // (Looked up anew for every piece: the loop over its tiles needs the registers.)
      const Pieces ps(p, aux);
      if (q && n == ps.pairs) n = ps.lane1;  // over lane 0's pieces
      if (n >= (q ? ps.end : ps.lane1)) break;
      const PlanPiece* pc = ps.at(n);
      const int tile = n < ps.pairs ? q : 0;  // which of the piece's Q tiles
      T = pc->tiles[tile];
      const int n_keys = pc->n_keys, diag = pc->diag + tile * p.tile_tokens;
      const int token_in_tile = min(r, p.tile_rows - 1) / p.group;  // idle rows go with the last
      tile_limit = min(n_keys - 1, diag);                 // last key that the tile's first row sees
      row_limit = min(n_keys - 1, diag + token_in_tile);  // last key that this row sees
      // rows of this tile that exist; a warp without one only keeps the protocol going
      rows = (min(pc->n_tokens - tile * p.tile_tokens, p.tile_tokens)) * p.group;
    }
    const bool row_live = r < rows;
    const bool warp_live = warp_in_group * 32 < rows;
    w.item = n;
    w.tile = 0;
    if (!w.wait_warp(bar(kPbFinFree + q), fin_free_parity, 310 + q)) return;
    fin_free_parity ^= 1u;
    float m = 0.0f;  // reference maximum, log2 units
    float l = 0.0f;  // running sum of 2^(s - m)
    for (int i = 0; i < T; ++i) {
      w.tile = i;
      if (!w.wait_warp(bar(kPbSFull + q), s_parity, 300 + q)) return;
      s_parity ^= 1u;
      tc_fence_after_sync();
      if (warp_live) {
        uint32_t s[4][32];
        tmem_ld32(s_tmem + 0, s[0]);
        tmem_wait_ld();  // chunk 0 alone, so that its exponentials overlap the other three loads
        tmem_ld32(s_tmem + 32, s[1]);
        tmem_ld32(s_tmem + 64, s[2]);
        tmem_ld32(s_tmem + 96, s[3]);
        const bool tail = i * kBlockN + kBlockN - 1 > tile_limit;  // uniform across the warp
        const int valid = row_limit - i * kBlockN + 1;             // keys of this tile that the row sees
        if (tail || i == 0) {
          tmem_wait_ld();
          if (tail) mask_tail(s, valid);
          if (i == 0) m = row_max(s) * scale_log2;
        }

        uint32_t packed[4][16];
        f2 sum_a = f2_splat(0.0f), sum_b = f2_splat(0.0f);
        {
          const f2 neg_m2 = f2_splat(-m);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            exp_chunk(s[c], scale2, neg_m2, packed[c], sum_a, sum_b);
            if (c == 0) tmem_wait_ld();
          }
        }
        float tile_sum = f2_hsum(sum_a, sum_b);
        // written so that a NaN sum also lands on the exact path
        const bool stands = tile_sum < sum_limit;
        if (__builtin_expect(__any_sync(0xffffffffu, row_live && !stands), 0)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(s_tmem + c * 32, s[c]);
          tmem_wait_ld();
          if (tail) mask_tail(s, valid);
          const float tile_max = row_max(s) * scale_log2;
          const float m_new = i == 0 ? tile_max : fmaxf(m, tile_max);
          if (i > 0) {
            const float f = m_new == kNegInf ? 1.0f : ex2_approx(m - m_new);
            l *= f;
            if (__any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll 1
              for (int c = 0; c < kHeadDim / 16; ++c) {
                uint32_t acc[16];
                tmem_ld16(o_tmem + c * 16, acc);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[j] = __float_as_uint(__uint_as_float(acc[j]) * f);
                tmem_st16(o_tmem + c * 16, acc);
              }
              tmem_wait_st();
            }
          }
          m = m_new;
          const f2 neg_m2 = f2_splat(m == kNegInf ? 0.0f : -m);
          sum_a = f2_splat(0.0f);
          sum_b = f2_splat(0.0f);
#pragma unroll
          for (int c = 0; c < 4; ++c) exp_chunk(s[c], scale2, neg_m2, packed[c], sum_a, sum_b);
          tile_sum = f2_hsum(sum_a, sum_b);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_st16(p_tmem + c * 16, packed[c]);
        tmem_wait_st();
        l += tile_sum;
      }
      tc_fence_before_sync();
      __syncwarp();
#ifdef B200ATTN_TEST_DROP_P_READY
      // Test builds only (never the shipped library): see attn_fwd_ws_kernel.
      const bool withheld = (q == 0 && warp_in_group == 0 && n == 0 && i == 1);
      mbar_arrive_lead((lane == 0 && !withheld) ? 1u : 0u, bar(kPbPReady + q));
#else
      mbar_arrive_lead(lane == 0 ? 1u : 0u, bar(kPbPReady + q));
#endif
    }
    const Pieces ps(p, aux);
    if (n != ps.last_of(q)) {
      aux->row_max[q][r] = m;
      aux->row_sum[q][r] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kPbFin + q));
    } else {
      // This lane's last piece: these warps have nothing left to do, so they store its result themselves, both lanes at
      // the same time. (The piece before it is through: its epilogue handed kPbFinFree back after its last PV, so the
      // phase waited for here is the next one.)
      if (!w.wait_warp(bar(kPbPvDone + q), pieces & 1u, 430 + q)) return;
      tc_fence_after_sync();
      store_result<2>(p, ps.at(n), n < ps.pairs ? q : 0, r, m, l, o_tmem);
    }
    ++pieces;
  }
}

// ---- epilogue -----------------------------------------------------------------------------------------------
// Warps 8 to 11, for all but the last piece of each lane (see above).
template <class Wait>
__device__ void plan_epilogue_role(const PlanParams& p, const PlanAux* aux, uint32_t bar0, uint32_t tmem_base,
                                   int warp_in_group, int lane, Wait& w) {
  auto bar = [&](int i) { return bar0 + 8u * uint32_t(i); };
  const uint32_t lane_field = uint32_t(warp_in_group * 32) << 16;
  const int r = warp_in_group * 32 + lane;
  uint32_t fin_parity = 0;  // bit per lane
  const Pieces ps(p, aux);

  // The result of piece n on lane q: its Q tile `tile`.
  auto finish = [&](int n, int q, int tile) -> bool {
    if (n == ps.last_of(q)) return true;
    if (!w.wait_warp(bar(kPbFin + q), (fin_parity >> q) & 1u, 410 + q)) return false;
    if (!w.wait_warp(bar(kPbPvDone + q), (fin_parity >> q) & 1u, 420 + q)) return false;
    fin_parity ^= 1u << q;
    tc_fence_after_sync();
    const float m = aux->row_max[q][r];
    const float l = aux->row_sum[q][r];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(kPbFinFree + q));
    store_result<1>(p, ps.at(n), tile, r, m, l, tmem_base + kQTilesPerItem * kBlockN + q * kHeadDim + lane_field);
    // O_q has been read: the next piece's first PV may overwrite it
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(kPbOFree + q));
    return true;
  };

  for (int n = 0; n < ps.pairs; ++n) {
    w.item = n;
    for (int q = 0; q < kQTilesPerItem; ++q) {
      w.tile = ps.at(n)->tiles[q];
      if (!finish(n, q, q)) return;
    }
  }
  LaneWalk walk(ps);  // pieces end in the order of their last steps
  LaneWalk::Step st;
  while (walk.take(ps, st)) {
    if (!st.last) continue;
    w.item = st.piece;
    w.tile = st.tile;
    if (!finish(st.piece, st.lane, 0)) return;
  }
}

template <class Wait>
__global__ void __launch_bounds__(kPlanThreads, 1)
attn_plan_kernel(const __grid_constant__ PlanMaps maps, const PlanParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint8_t* kv = smem + kQTilesPerItem * kTileBytes;
  PlanAux* aux = reinterpret_cast<PlanAux*>(kv + kPairSlotsP * kPairBytesP);
  const uint32_t smem_q = smem_u32(smem), smem_kv = smem_u32(kv);
  const uint32_t bar0 = smem_u32(&aux->bar[0]);

  Wait w;
  w.abort_addr = smem_u32(&aux->abort_flag);
  w.status = p.status;
  w.limit_ns = uint64_t(p.wait_limit_ms) * 1000000ull;
  w.item = -1;
  w.tile = -1;

  // The next kernel of the stream may be brought up from here on; it waits for the end of this one before it touches
  // anything that this one writes, as this one does below (also where it has nothing to do, so that whoever waits for
  // this kernel has waited for the ones before it).
  launch_dependents();
  const bool misaligned = (smem_q & 1023u) != 0;  // uniform across the CTA
  const int4* record = reinterpret_cast<const int4*>(p.table + kPlanCtaAt + kPlanCtaWords * blockIdx.x);
  if (warp == 13 && lane < 6) tma_prefetch_desc(&maps.q + lane);
  const int4 first = record[0];
  const int piece0 = first.x, piece1 = first.w;
  const bool no_plan = p.table[kPlanHdrMagic] != kPlanMagic;  // freed memory, say, under a captured call
  if (misaligned || no_plan || piece0 >= piece1) {  // uniform across the CTA; the last: fewer CTAs than the grid
    if (threadIdx.x == 0 && (misaligned || no_plan)) {
      aux->abort_flag = 0;
      w.raise(misaligned ? kDevSmemMisaligned : kDevNoPlan, 3, 0);
    }
    wait_for_previous();
    return;
  }
  const uint32_t lead = (lane == 0) ? 1u : 0u;
  Loader<Wait> loader(p, maps, smem_q, smem_kv, bar0, lead);
  if (warp == 13) {
    const PlanPiece piece = piece_of(record[1], record[2], record[3]);
    for (int i = lane; i < kNumPlanBarriers; i += 32) mbar_init(bar0 + 8u * i, plan_barrier_count(i));
    mbar_init_fence();
    fence_proxy_async_smem();
    if (lane == 0) {
      aux->abort_flag = 0;
      aux->first[0] = first.x;
      aux->first[1] = first.y;
      aux->first[2] = first.z;
      aux->first[3] = first.w;
    }
    __syncwarp();
    // The whole CTA waits here (at the barrier below), before any of its bounded waits begin.
    wait_for_previous();
    loader.begin(&piece, w);  // under way while the rest of the CTA sets itself up
  } else {
    const int4* src = reinterpret_cast<const int4*>(p.table + kPlanPieceAt) + size_t(piece0) * 3;
    int4* dst = reinterpret_cast<int4*>(aux->cache);
    const int words = min(piece1 - piece0, kPieceCache) * 3;
    if (threadIdx.x < 384)  // warps 0 to 11
      for (int j = threadIdx.x; j < words; j += 384) dst[j] = src[j];
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(&aux->tmem_base), 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = aux->tmem_base;

  if (warp < 8) {
    reg_grow<kPlanRegsSoftmax>();
    plan_softmax_role(p, aux, bar0, tmem_base, warp >> 2, warp & 3, lane, w);
  } else if (warp < 12) {
    reg_shrink<kPlanRegsEpilogue>();
    plan_epilogue_role(p, aux, bar0, tmem_base, warp & 3, lane, w);
  } else {
    reg_shrink<kPlanRegsOther>();
    if (warp == 12) {
      plan_mma_role(p, aux, smem_q, smem_kv, bar0, tmem_base, lead, w);
    } else if (warp == 13) {
      loader.run(aux, w);
    } else if (warp == 14) {
      plan_tail_role(p, aux, kv, bar0, lane, w);
    }
    __syncwarp();
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
    if (lane == 0) pass_on(w, aux);
  }
}

// ---- join ---------------------------------------------------------------------------------------------------
// A block per unit (at most 32 rows, or one token), lane l of a warp holding columns 4l .. 4l + 3 of a row. Parts are
// taken with a running reference and sum, so that LSEs and partial rows are on their way together and nothing waits for
// a pass over the LSEs first. A warp has the parts of two rows in flight where there are at most two, else four parts
// of one row, and a unit of fewer than eight rows spreads the parts of a row over several warps. 64 registers: the
// blocks of 512 units are then resident together (eight parts in flight took 79 registers and twice as long there).
// Rows without a part, and rows whose parts saw no key, get O = 0 and LSE = -inf. Bound by latency for few rows
// (64 tokens x 32 heads, 9 parts: 5.1 us), else by reading 516 bytes per part and row (82 thousand: 12.3 us).
constexpr int kJoinWarps = 8;

struct JoinState {
  float m, sum;
  float4 acc;
  __device__ __forceinline__ void clear() {
    m = kNegInf;
    sum = 0.0f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void rebase(float top) {  // top >= m
    const float f = m == top ? 1.0f : expf(m - top);
    m = top;
    sum *= f;
    acc.x *= f;
    acc.y *= f;
    acc.z *= f;
    acc.w *= f;
  }
  __device__ __forceinline__ void add(float weight, const float4& a, float s) {
    sum = fmaf(weight, s, sum);
    acc.x = fmaf(a.x, weight, acc.x);
    acc.y = fmaf(a.y, weight, acc.y);
    acc.z = fmaf(a.z, weight, acc.z);
    acc.w = fmaf(a.w, weight, acc.w);
  }
};

// Weight of something with LSE or reference `of` against `top` >= of: 0 where it saw no key.
__device__ __forceinline__ float join_weight(float of, float top) { return expf(of - (top == kNegInf ? 0.0f : top)); }

__device__ __forceinline__ void join_store(const PlanParams& p, const PlanUnit& un, int r, int lane, const JoinState& s) {
  const int token = r / p.group;
  const int head = un.kv_head * p.group + (r - token * p.group);
  const int64_t row = int64_t(un.token) + token;
  const bool seen = s.sum != 0.0f;  // a NaN sum counts as seen
  const float inv = seen ? 1.0f / s.sum : 0.0f;
  uint2 out;
  out.x = pack_bf16x2(s.acc.x * inv, s.acc.y * inv);
  out.y = pack_bf16x2(s.acc.z * inv, s.acc.w * inv);
  *reinterpret_cast<uint2*>(p.o + row * p.o_stride_t + int64_t(head) * p.o_stride_h + lane * 4) = out;
  if (p.lse != nullptr && lane == 0)
    p.lse[int64_t(head) * p.lse_stride_h + row] = seen ? s.m + logf(s.sum) : kNegInf;
}

// Parts k0, k0 + step, .. of rows r0 .. r0 + kRows - 1 (those below `rows`), kParts of them at a time.
template <int kRows, int kParts>
__device__ __forceinline__ void join_rows(const PlanParams& p, const int32_t* parts, int n_parts, int k0, int step, int r0,
                                          int rows, int lane, JoinState (&s)[kRows]) {
#pragma unroll
  for (int i = 0; i < kRows; ++i) s[i].clear();
  for (int k = k0; k < n_parts; k += step * kParts) {
    float lse[kRows][kParts];
    float4 a[kRows][kParts];
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      const bool there = k + j * step < n_parts;
      const int at = (there ? parts[k + j * step] : 0) + r0;
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        lse[i][j] = kNegInf;
        a[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there && r0 + i < rows) {
          lse[i][j] = __ldcg(p.part_lse + at + i);
          a[i][j] = __ldcg(reinterpret_cast<const float4*>(p.part_o + int64_t(at + i) * kHeadDim) + lane);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float top = s[i].m;
#pragma unroll
      for (int j = 0; j < kParts; ++j) top = fmaxf(top, lse[i][j]);
      s[i].rebase(top);
#pragma unroll
      for (int j = 0; j < kParts; ++j) s[i].add(join_weight(lse[i][j], top), a[i][j], 1.0f);
    }
  }
}

template <int kRows, int kParts>
__device__ __forceinline__ void join_unit(const PlanParams& p, const PlanUnit& un, const int32_t* parts, int rows, int warp,
                                          int lane) {
  for (int r0 = warp * kRows; r0 < rows; r0 += kJoinWarps * kRows) {
    JoinState s[kRows];
    join_rows<kRows, kParts>(p, parts, un.parts, 0, 1, r0, rows, lane, s);
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (r0 + i < rows) join_store(p, un, r0 + i, lane, s[i]);
  }
}

__global__ void __launch_bounds__(kJoinWarps * 32, 4)
attn_plan_join_kernel(const PlanParams p) {
  __shared__ float4 shared_acc[kJoinWarps][32];
  __shared__ float shared_m[kJoinWarps], shared_sum[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = p.table[kPlanHdrMagic] == kPlanMagic ? p.table[kPlanHdrUnits] : 0;
  const PlanUnit* unit = reinterpret_cast<const PlanUnit*>(p.table + p.table[kPlanHdrUnitAt]);
  const int32_t* part_list = p.table + p.table[kPlanHdrPartAt];
  // (This kernel does not let the next one be brought up before its own end: with 512 units that left the next call's
  // CTAs waiting on SMs of their own and cost 25 us of 75.)
  bool waited = false;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const PlanUnit un = unit[u];
    const int32_t* parts = part_list + un.part0;
    if (!waited) {
      if (lane < un.parts) asm volatile("prefetch.global.L1 [%0];" ::"l"(parts + lane));
      wait_for_previous();
    }
    waited = true;
    const int rows = un.n_tokens * p.group;
    if (rows <= kJoinWarps / 2 && un.parts > 2) {  // uniform across the block
      const int per_row = rows == 1 ? 8 : rows == 2 ? 4 : 2;  // warps of a row
      const int r = warp / per_row, share = warp - r * per_row;
      JoinState s[1];
      if (r < rows) {
        join_rows<1, 4>(p, parts, un.parts, share, per_row, r, rows, lane, s);
        shared_acc[warp][lane] = s[0].acc;
        if (lane == 0) {
          shared_m[warp] = s[0].m;
          shared_sum[warp] = s[0].sum;
        }
      }
      __syncthreads();
      if (r < rows && share == 0) {
        for (int j = 1; j < per_row; ++j) {
          const float m = shared_m[warp + j], top = fmaxf(s[0].m, m);
          s[0].rebase(top);
          s[0].add(join_weight(m, top), shared_acc[warp + j][lane], shared_sum[warp + j]);
        }
        join_store(p, un, r, lane, s[0]);
      }
      __syncthreads();
    } else if (un.parts <= 2) {
      join_unit<2, 2>(p, un, parts, rows, warp, lane);
    } else {
      join_unit<1, 4>(p, un, parts, rows, warp, lane);
    }
  }
  if (!waited) wait_for_previous();
}

}  // namespace

cudaError_t prepare_plan_kernels() {
  constexpr int kPoolNeeded = 128 * (2 * kPlanRegsSoftmax + kPlanRegsEpilogue + kPlanRegsOther);
  for (const auto kernel : {attn_plan_kernel<WaitCtx>, attn_plan_kernel<NotedWait>}) {
    cudaFuncAttributes fa;
    cudaError_t e = cudaFuncGetAttributes(&fa, kernel);
    if (e != cudaSuccess) return e;
    // a growing role would block in hardware if the launch did not reserve what the roles ask for
    if (fa.numRegs * kPlanThreads < kPoolNeeded) return cudaErrorLaunchOutOfResources;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPlanSmemBytes);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t launch_plan(const PlanMaps& maps, const PlanParams& p, int grid, bool wide, cudaStream_t stream) {
  return launch_overlapped(wide ? attn_plan_kernel<WaitCtx> : attn_plan_kernel<NotedWait>, grid, kPlanThreads,
                           kPlanSmemBytes, stream, maps, p);
}

cudaError_t launch_plan_join(const PlanParams& p, int grid, cudaStream_t stream) {
  return launch_overlapped(attn_plan_join_kernel, grid, kJoinWarps * 32, 0, stream, p);
}

}  // namespace b200attn
