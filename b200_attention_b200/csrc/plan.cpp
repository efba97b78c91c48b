// Host-side planner of the packed and shared-prefix attention calls: cuts the work into pieces,
// deals them to CTAs and lists what has to be joined afterwards. No CUDA.
//
// An item is a block of 2 * floor(128 / group) tokens of one sequence and one K/V head with every
// key it sees (for a shared prefix: a block of tokens of all sequences with the prefix). Items are
// dealt to the CTA that is free first, longest first. Where that leaves CTAs idle at the end, cutting helps, at the
// price of the pieces' own starts and of the join of their partial results. Two ways of cutting are tried, and the
// schedule that finishes first by the costs below is taken: long items into pieces of equal length, for a
// handful of lengths (few items, single tokens with many keys); and, of a schedule with more items than CTAs, only
// what the busiest CTAs have too much, which goes to those that have least.
#include "plan.h"

#include <algorithm>
#include <queue>
#include <utility>

namespace b200attn {

namespace {

constexpr int kTile = 128;

// Costs in thousandths of the time of a K/V tile against two Q tiles (1.6 us), as measured with pieces of equal length.
// A piece of one Q tile runs on one of a CTA's two lanes: alone it is bound by its chain of steps, beside another lane
// by what the two share, which is above all memory (64 KB per tile). Next to a prefix, whose pieces load memory on
// every CTA, a tile costs more of that; without one a CTA that has more tiles than others gets more of the memory's
// rate, and a piece's start weighs more. Two pairs of figures are worth little on average and much at some shapes: over
// 26 decode and prefix shapes, measured twice, 2.0 and 1.1 % in the mean, from -16 % (10 tokens of 4000 keys, 40 heads:
// 48.8 us with the first pair everywhere, 41.1 as it is) to +6 % (16 tokens of 1000-8000 keys: 49.2 -> 52.2); the second
// pair everywhere costs 90 tokens on a prefix of 3000 41.0 -> 45.4 us.
constexpr int64_t kTilePair = 1000;
constexpr int64_t kTilePairPrefix = 1250;  // the same, with every CTA on keys of its own, which come from memory
constexpr int64_t kPairStart = 2200;    // Q load, first scores, last PV, stores
constexpr int64_t kTileSharedPrefix = 930;
constexpr int64_t kSharedStartPrefix = 750;
constexpr int64_t kTileShared = 600;
constexpr int64_t kSharedStart = 1800;
constexpr int64_t kTileChain = 950;     // scores, softmax, PV of one tile after the other
constexpr int64_t kChainStart = 1300;
constexpr int64_t kTilesMemory = 13;    // two tiles of one Q tile, of all CTAs' time together: 128 KB at 6.3 TB/s
constexpr int64_t kJoin = 2500;         // the second kernel, once,
constexpr int64_t kJoinRows = 14;       // and per row of partial results, divided by this
// A piece is walked without a look at the other CTAs, under waits of limited length: keep it below a tenth of a second.
constexpr int32_t kLongestPiece = 1 << 15;
constexpr int32_t kShortestCut = 3;     // tiles of what is left, and of what is taken, where an item is trimmed

struct Item {
  int32_t token, n_tokens, kv_row, n_keys, tiles0, tiles1, diag, kv_head, source;
  int32_t sequence;  // -1: prefix
  int32_t longest() const { return tiles1 > 0 ? tiles1 : tiles0; }
};

struct Cost {
  int32_t kind;    // 2: two Q tiles, 1: one, 0: one with few rows; in this order on every CTA
  int64_t shared;  // of the CTA's time
  int64_t chain;   // of a lane's time, for one Q tile
};
Cost cost_of(const PlanPiece& p, int32_t small_tokens, bool has_prefix) {
  if (p.tiles[1] > 0) return {2, kPairStart + p.tiles[1] * (p.source == 1 ? kTilePairPrefix : kTilePair), 0};
  return {p.n_tokens <= small_tokens ? 0 : 1,
          has_prefix ? kSharedStartPrefix + p.tiles[0] * kTileSharedPrefix : kSharedStart + p.tiles[0] * kTileShared,
          kChainStart + p.tiles[0] * kTileChain};
}

// Tiles [from, from + len) of an item.
PlanPiece cut_piece(const Item& it, int32_t from, int32_t len) {
  PlanPiece p{};
  p.token = it.token;
  p.n_tokens = it.n_tokens;
  p.kv_row = it.kv_row + from * kTile;
  p.n_keys = int32_t(std::min<int64_t>(it.n_keys - int64_t(from) * kTile, int64_t(len) * kTile));
  p.tiles[0] = std::max(0, std::min(it.tiles0 - from, len));
  p.tiles[1] = std::max(0, std::min(it.tiles1 - from, len));
  if (p.tiles[0] == 0) p.tiles[0] = 1;  // a fully masked tile: leaves an empty partial result
  p.diag = it.diag == kPlanNoDiag ? kPlanNoDiag : it.diag - from * kTile;
  p.kv_head = it.kv_head;
  p.source = it.source;
  p.slot_row = -1;
  return p;
}

struct Cta {
  int64_t pairs = 0, shared = 0, lane[2] = {0, 0};
  int64_t end() const { return pairs + std::max(shared, std::max(lane[0], lane[1])); }
  // by the shared time: a CTA with one busy lane takes a second piece almost for nothing
  int64_t free_at() const { return pairs + std::max(shared, std::min(lane[0], lane[1])); }
};

// Tiles [from, from + len) of an item.
struct Run {
  int32_t item, from, len;
  Cost cost;
};

// Runs and where they go.
struct Deal {
  std::vector<Run> runs;
  std::vector<Cta> cta;
  std::vector<std::vector<int32_t>> dealt;  // of each CTA: runs of two Q tiles, of lane 0, of lane 1

  // Hands out runs (indices, longest first) to the CTA that is free first, and those of one Q tile to its lane that is.
  void hand_out(const std::vector<int32_t>& order) {
    using Load = std::pair<int64_t, int32_t>;  // (free at, CTA)
    std::vector<Load> loads(cta.size());
    for (size_t c = 0; c < cta.size(); ++c) loads[c] = {cta[c].free_at(), int32_t(c)};
    std::priority_queue<Load, std::vector<Load>, std::greater<Load>> next(std::greater<Load>(), std::move(loads));
    for (const int32_t i : order) {
      const Cost& c = runs[size_t(i)].cost;
      const int32_t at = next.top().second;
      next.pop();
      Cta& t = cta[size_t(at)];
      int32_t list = 0;
      if (c.kind == 2) {
        t.pairs += c.shared;
      } else {
        const int32_t lane = t.lane[1] < t.lane[0] ? 1 : 0;
        t.lane[lane] += c.chain;
        t.shared += c.shared;
        list = 1 + lane;
      }
      dealt[size_t(at) * 3 + size_t(list)].push_back(i);
      next.push({t.free_at(), at});
    }
  }
  int64_t end() const {
    int64_t e = 0;
    for (const Cta& t : cta) e = std::max(e, t.end());
    return e;
  }
  int64_t mean() const {
    int64_t sum = 0;
    for (const Run& r : runs) sum += r.cost.shared;
    return sum / int64_t(cta.size());
  }
};

struct Planner {
  const std::vector<Item>& items;
  int32_t sm_count, group, small_tokens;
  bool has_prefix;  // every piece leaves a partial result
  bool by_groups;   // K/V of sixteen heads at a time, where all of it would not stay in L2 (see CausalWalk's groups)

  Cost cost(const Run& r) const {
    return cost_of(cut_piece(items[size_t(r.item)], r.from, r.len), small_tokens, has_prefix);
  }

  // Items cut into pieces of at most `len` tiles, not dealt yet.
  Deal uniform(int32_t len) const {
    Deal d;
    d.cta.resize(size_t(sm_count));
    d.dealt.resize(size_t(sm_count) * 3);
    for (size_t i = 0; i < items.size(); ++i) {
      const int32_t longest = items[i].longest(), n = (longest + len - 1) / len, l = (longest + n - 1) / n;
      for (int32_t from = 0; from < longest; from += l) {
        Run r{int32_t(i), from, std::min(l, longest - from), {}};
        r.cost = cost(r);
        d.runs.push_back(r);
      }
    }
    return d;
  }

  void deal(Deal* d) const {
    // by kind, then by group of heads, then longest first
    std::vector<std::pair<uint64_t, int32_t>> keys(d->runs.size());
    for (size_t i = 0; i < keys.size(); ++i) {
      const Run& r = d->runs[i];
      const uint64_t head_group = by_groups ? uint64_t(items[size_t(r.item)].kv_head / 16) & 0x3ffffu : 0;
      keys[i] = {(uint64_t(2 - r.cost.kind) << 62) | (head_group << 44) | ((uint64_t(1) << 44) - 1 - uint64_t(r.cost.shared)),
                 int32_t(i)};
    }
    std::sort(keys.begin(), keys.end());
    std::vector<int32_t> order(keys.size());
    for (size_t i = 0; i < order.size(); ++i) order[i] = keys[i].second;
    d->hand_out(order);
  }

  // Takes from every CTA that ends after `limit` the end of its longest run, and hands that out again.
  Deal trimmed(const Deal& from, int64_t limit) const {
    Deal d = from;
    std::vector<int32_t> loose;
    for (size_t c = 0; c < d.cta.size(); ++c) {
      const int64_t excess = d.cta[c].end() - limit;
      if (excess <= 0 || d.dealt[c * 3].empty()) continue;
      const size_t at = size_t(d.dealt[c * 3].front());
      const int32_t tiles = std::max<int32_t>(kShortestCut, int32_t((excess + kTilePair - 1) / kTilePair));
      if (d.runs[at].len - tiles < kShortestCut) continue;
      Run rest{d.runs[at].item, d.runs[at].from + d.runs[at].len - tiles, tiles, {}};
      d.runs[at].len -= tiles;
      rest.cost = cost(rest);
      const Cost shorter = cost(d.runs[at]);
      d.cta[c].pairs -= d.runs[at].cost.shared - shorter.shared;
      d.runs[at].cost = shorter;
      loose.push_back(int32_t(d.runs.size()));
      d.runs.push_back(rest);
    }
    std::stable_sort(loose.begin(), loose.end(), [&](int32_t a, int32_t b) {
      return d.runs[size_t(a)].cost.shared > d.runs[size_t(b)].cost.shared;
    });
    d.hand_out(loose);
    return d;
  }

  // What the join adds.
  int64_t join(const Deal& d) const {
    std::vector<int32_t> runs_of(items.size(), 0);
    for (const Run& r : d.runs) ++runs_of[size_t(r.item)];
    int64_t rows = 0;
    for (const Run& r : d.runs)
      if (has_prefix || runs_of[size_t(r.item)] > 1) rows += int64_t(items[size_t(r.item)].n_tokens) * group;
    return rows > 0 ? kJoin + rows / kJoinRows : 0;
  }

  Deal best() const {
    int64_t total_tiles = 0, long_items = 0;
    int32_t longest = 1;
    bool pairs = false;
    for (const Item& it : items) {
      total_tiles += it.longest();
      longest = std::max(longest, it.longest());
      pairs = pairs || it.tiles1 > 0;
    }
    for (const Item& it : items) long_items += 2 * it.longest() > longest ? 1 : 0;
    const int32_t uncut = std::min(longest, kLongestPiece);  // what is left whole where it can be
    std::vector<int32_t> lens;
    auto consider = [&](int64_t len) {
      len = std::max<int64_t>(1, len);
      if (len < uncut && std::find(lens.begin(), lens.end(), int32_t(len)) == lens.end()) lens.push_back(int32_t(len));
    };
    const int64_t even = (total_tiles + sm_count - 1) / sm_count;
    for (const int64_t parts : {1, 2, 4, 8}) consider((even + parts - 1) / parts);
    consider((longest + 1) / 2);
    consider((3 * int64_t(longest) + 3) / 4);
    // as many pieces of the longest items as fill the CTAs, or their lanes, a whole number of times
    for (const int64_t rounds : {1, 2, 4}) {
      const int64_t n = long_items > 0 ? rounds * sm_count / long_items : 0;
      if (n > 1) consider((longest + n - 1) / n);
    }

    Deal found = uniform(uncut);
    deal(&found);
    int64_t end = found.end() + join(found);
    const Deal whole = found;
    auto offer = [&](Deal&& d) {
      const int64_t e = d.end() + join(d);
      if (e >= end) return;
      end = e;
      found = std::move(d);
    };
    // Close to what no schedule can beat: not worth the time of looking for another (a decode step plans anew each time).
    if (!pairs && end <= std::max(whole.mean() * 107 / 100, total_tiles * kTilesMemory / 2)) return found;
    // What a few CTAs have too much. With fewer items than CTAs there is nothing to even out.
    if (pairs && items.size() > size_t(sm_count))
      for (const int64_t percent : {101, 102, 104, 107})
        if (whole.mean() * percent / 100 + kJoin < end) offer(trimmed(whole, whole.mean() * percent / 100 + kPairStart));
    if (end <= whole.mean() * 104 / 100) return found;
    for (const int32_t len : lens) {
      Deal d = uniform(len);
      if (d.mean() + join(d) >= end - end / 100) continue;  // no better to speak of, however it is dealt
      deal(&d);
      offer(std::move(d));
    }
    return found;
  }
};

}  // namespace

std::string plan_build(const PlanInput& in, Plan* plan) {
  if (in.sequences < 1) return "there must be at least one sequence";
  if (in.heads < 1 || in.heads_kv < 1 || in.heads % in.heads_kv != 0)
    return "heads must be a positive multiple of heads_kv";
  const int32_t group = in.heads / in.heads_kv;
  if (group > 128) return "more than 128 query heads per K/V head";
  if (in.sm_count < 1 || in.sm_count > kPlanMaxCtas) return "sm_count must be 1 .. 160";
  if (in.len_prefix < 0 || in.len_prefix >= (1 << 30)) return "len_prefix must be 0 .. 2^30 - 1";

  const int32_t tile_tokens = plan_tile_tokens(group);
  const int32_t block = 2 * tile_tokens, small_tokens = plan_small_tokens(group);
  std::vector<int64_t> first_token(size_t(in.sequences) + 1, 0), first_key(size_t(in.sequences), 0);
  int64_t at = 0;
  plan->rows_kv = 0;
  for (int32_t s = 0; s < in.sequences; ++s) {
    const int64_t n = in.len_q[s], m = in.len_kv[s];
    if (n < 0 || m < 0 || n >= (1 << 30) || m >= (1 << 30)) return "lengths must be 0 .. 2^30 - 1";
    if (in.causal && in.len_prefix > 0 && m < n)
      return "with a prefix and a causal mask a sequence needs at least as many keys of its own as queries";
    first_token[size_t(s) + 1] = first_token[size_t(s)] + n;
    const int64_t start = in.start_kv != nullptr ? in.start_kv[s] : at;
    if (start < 0 || start + m >= (int64_t(1) << 31) - 256) return "K/V rows must be 0 .. 2^31 - 257";
    first_key[size_t(s)] = start;
    at += m;
    if (m > 0) plan->rows_kv = std::max(plan->rows_kv, start + m);
  }
  plan->rows_q = first_token.back();
  if (plan->rows_q >= (int64_t(1) << 31) - 256) return "too many query rows";

  const bool has_prefix = in.len_prefix > 0;

  // ---- items
  std::vector<Item> items;
  int64_t kv_bytes = int64_t(in.len_prefix) * in.heads_kv * 512;
  for (int32_t s = 0; s < in.sequences; ++s) {
    const int32_t n = in.len_q[s], m = in.len_kv[s];
    kv_bytes += int64_t(m) * in.heads_kv * 512;
    if (m == 0) continue;
    for (int32_t t = 0; t < n; t += block) {
      Item it{};
      it.sequence = s;
      it.token = int32_t(first_token[size_t(s)]) + t;
      it.n_tokens = std::min(block, n - t);
      it.kv_row = int32_t(first_key[size_t(s)]);
      it.n_keys = m;
      it.diag = in.causal ? m - n + t : kPlanNoDiag;
      int32_t tiles[2];
      for (int32_t q = 0; q < 2; ++q) {
        const int32_t here = std::min(tile_tokens, it.n_tokens - q * tile_tokens);  // tokens of Q tile q
        if (here <= 0) {
          tiles[q] = 0;
          continue;
        }
        const int64_t keys = in.causal ? std::min<int64_t>(m, int64_t(it.diag) + q * tile_tokens + here) : m;
        tiles[q] = keys <= 0 ? 0 : int32_t((keys + kTile - 1) / kTile);
      }
      if (tiles[0] == 0 && tiles[1] == 0) continue;  // no row of the block sees a key
      it.tiles0 = std::max(1, tiles[0]);
      it.tiles1 = tiles[1];
      for (int32_t h = 0; h < in.heads_kv; ++h) {
        it.kv_head = h;
        items.push_back(it);
      }
    }
  }
  if (in.len_prefix > 0) {
    const int32_t tiles = (in.len_prefix + kTile - 1) / kTile;
    for (int64_t t = 0; t < plan->rows_q; t += block) {
      Item it{};
      it.sequence = -1;
      it.token = int32_t(t);
      it.n_tokens = int32_t(std::min<int64_t>(block, plan->rows_q - t));
      it.kv_row = 0;
      it.n_keys = in.len_prefix;
      it.diag = kPlanNoDiag;
      it.tiles0 = tiles;
      it.tiles1 = it.n_tokens > tile_tokens ? tiles : 0;
      it.source = 1;
      for (int32_t h = 0; h < in.heads_kv; ++h) {
        it.kv_head = h;
        items.push_back(it);
      }
    }
  }
  // ---- pieces, with the rows of their partial results
  const bool by_groups = kv_bytes > (int64_t(64) << 20);
  const Deal deal = Planner{items, in.sm_count, group, small_tokens, has_prefix, by_groups}.best();
  std::vector<int32_t> by_item(deal.runs.size());  // runs in the order of items and keys
  for (size_t i = 0; i < by_item.size(); ++i) by_item[i] = int32_t(i);
  std::sort(by_item.begin(), by_item.end(), [&](int32_t a, int32_t b) {
    const Run &x = deal.runs[size_t(a)], &y = deal.runs[size_t(b)];
    return x.item != y.item ? x.item < y.item : x.from < y.from;
  });
  std::vector<PlanPiece> pieces(deal.runs.size());  // of each run
  std::vector<int32_t> item_piece0(items.size() + 1, 0);
  int64_t slots = 0;
  for (size_t k = 0, i = 0; i < items.size(); ++i) {
    item_piece0[i] = int32_t(k);
    size_t last = k;
    while (last < by_item.size() && deal.runs[size_t(by_item[last])].item == int32_t(i)) ++last;
    const bool partial = has_prefix || last - k > 1;
    for (; k < last; ++k) {
      const Run& r = deal.runs[size_t(by_item[k])];
      PlanPiece& p = pieces[size_t(by_item[k])];
      p = cut_piece(items[i], r.from, r.len);
      plan->wide_pieces += p.tiles[1] > 0 ? 1 : 0;
      if (!partial) continue;
      p.slot_row = int32_t(slots);
      slots += int64_t(items[i].n_tokens) * group;
      if (slots >= (int64_t(1) << 31) - 512) return "too many partial rows";
    }
  }
  item_piece0[items.size()] = int32_t(pieces.size());
  if (pieces.size() >= (size_t(1) << 24)) return "too many pieces";
  plan->slot_rows = slots;
  plan->pieces = int32_t(pieces.size());
  auto slot_of = [&](int32_t k) { return pieces[size_t(by_item[size_t(k)])].slot_row; };

  // ---- join units
  std::vector<PlanUnit> units;
  std::vector<int32_t> parts;
  const int32_t unit_tokens = std::max(1, kPlanJoinRows / group);
  const int32_t heads_kv = in.heads_kv;
  // items of a (sequence, block) are heads_kv consecutive entries, in the order they were made
  size_t next_own = 0;
  size_t prefix_at = items.size();
  if (has_prefix) prefix_at = items.size() - size_t((plan->rows_q + block - 1) / block) * size_t(heads_kv);
  for (int32_t s = 0; s < in.sequences; ++s) {
    const int32_t n = in.len_q[s];
    for (int32_t t = 0; t < n; t += block) {
      const int32_t token = int32_t(first_token[size_t(s)]) + t;
      const int32_t here = std::min(block, n - t);
      const bool own = next_own < prefix_at && items[next_own].sequence == s && items[next_own].token == token;
      for (int32_t h = 0; h < heads_kv; ++h) {
        const size_t own_item = next_own + size_t(h);
        if (own && !has_prefix && item_piece0[own_item + 1] - item_piece0[own_item] == 1) continue;  // wrote o itself
        for (int32_t i = 0; i < here;) {
          int32_t count = std::min(unit_tokens, here - i);
          PlanUnit u{};
          u.token = token + i;
          u.part0 = int32_t(parts.size());
          u.kv_head = h;
          if (has_prefix) {
            const int32_t b = u.token / block;  // a unit stays inside one block of the prefix's items
            count = std::min(count, (b + 1) * block - u.token);
            const size_t item = prefix_at + size_t(b) * size_t(heads_kv) + size_t(h);
            for (int32_t p = item_piece0[item]; p < item_piece0[item + 1]; ++p)
              parts.push_back(slot_of(p) + (u.token - b * block) * group);
          }
          if (own)
            for (int32_t p = item_piece0[own_item]; p < item_piece0[own_item + 1]; ++p)
              parts.push_back(slot_of(p) + i * group);
          u.n_tokens = count;
          u.parts = int32_t(parts.size()) - u.part0;
          units.push_back(u);
          i += count;
        }
      }
      if (own) next_own += size_t(heads_kv);
    }
  }
  if (units.size() >= (size_t(1) << 28) || parts.size() >= (size_t(1) << 28)) return "too many rows to join";
  plan->units = int32_t(units.size());

  plan->grid = 0;
  for (int32_t c = 0; c < in.sm_count; ++c)
    for (int32_t k = 0; k < 3; ++k)
      if (!deal.dealt[size_t(c) * 3 + size_t(k)].empty()) plan->grid = c + 1;

  // ---- table
  const size_t unit_at = size_t(kPlanPieceAt) + pieces.size() * (sizeof(PlanPiece) / 4);
  const size_t part_at = unit_at + units.size() * (sizeof(PlanUnit) / 4);
  plan->table.assign((part_at + parts.size() + 3) / 4 * 4, 0);
  int32_t* t = plan->table.data();
  t[kPlanHdrMagic] = kPlanMagic;
  t[kPlanHdrPieces] = plan->pieces;
  t[kPlanHdrUnits] = plan->units;
  t[kPlanHdrUnitAt] = int32_t(unit_at);
  t[kPlanHdrPartAt] = int32_t(part_at);
  PlanPiece* out = reinterpret_cast<PlanPiece*>(t + kPlanPieceAt);
  int32_t k = 0;
  for (int32_t c = 0; c < kPlanMaxCtas; ++c) {
    for (int32_t part = 0; part < 3; ++part) {
      t[kPlanCtaAt + kPlanCtaWords * c + part] = k;
      if (c < in.sm_count)
        for (const int32_t i : deal.dealt[size_t(c) * 3 + size_t(part)]) out[k++] = pieces[size_t(i)];
    }
    const int32_t begin = t[kPlanCtaAt + kPlanCtaWords * c];
    t[kPlanCtaAt + kPlanCtaWords * c + 3] = k;
    if (begin < k) *reinterpret_cast<PlanPiece*>(t + kPlanCtaAt + kPlanCtaWords * c + 4) = out[begin];
  }
  std::copy(units.begin(), units.end(), reinterpret_cast<PlanUnit*>(t + unit_at));
  std::copy(parts.begin(), parts.end(), t + part_at);
  return "";
}

}  // namespace b200attn
