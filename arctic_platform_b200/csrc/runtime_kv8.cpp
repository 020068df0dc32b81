// Work items of chunk attention over the 8-bit cache (csrc/kv_fp8_chunk.cu), host side.
//
// A tile holds `hp` query heads of one key head for `tp` = 128 / hp tokens; an item is one or two tiles (tokens of one sequence, side by
// side) over the 128-token blocks that they see.  Items are dealt out to the CTAs in one of two ways, by the estimated time of the
// slowest CTA: whole, the longest first to whoever has least; or in a row that is cut into equal shares, where an item that crosses
// a border is cut along the keys into parts that leave their results to a join.
#include <algorithm>
#include <cstdint>
#include <functional>
#include <queue>
#include <vector>

namespace {
constexpr int kBlock = 128;
// Estimated times, in microseconds: a block of two tiles, of one where the other items have two, of one where none has; an item besides its
// blocks; what a part takes longer than an item; the join of the parts.
constexpr double kTwoTiles = 2.7, kOneOfTwo = 2.5, kOneTile = 1.4, kItem = 4.0, kPart = 1.5, kJoin = 4.0;
constexpr int kLeast = 2;          // blocks of a part

struct Work {
  int32_t row0, tokens, seq, kvh, head0, heads, pos0, len, blocks;
  double block;                    // time of one
};
struct Piece {
  int work, from, blocks, part;    // part: number among its item's pieces, -1: whole
};

// Items in a row over `ctas` shares of `share`; false: they do not fit.
bool cut(const std::vector<Work>& work, double share, int ctas, std::vector<std::vector<Piece>>* out) {
  int c = 0;
  double load = 0;
  for (int i = 0; i < static_cast<int>(work.size()); ++i) {
    const Work& w = work[i];
    int at = 0, part = 0;
    for (;;) {
      const int left = w.blocks - at;
      const double whole = kItem + (part ? kPart : 0.0) + left * w.block;
      if (load + whole <= share * (1 + 1e-9)) {
        if (out) (*out)[c].push_back({i, at, left, part ? part : -1});
        load += whole;
        break;
      }
      const int fit = std::min(static_cast<int>((share - load - kItem - kPart) / w.block), left - kLeast);
      if (fit >= kLeast) {
        if (out) (*out)[c].push_back({i, at, fit, part});
        ++part;
        at += fit;
      } else if (load == 0) {
        return false;
      }
      load = 0;
      if (++c == ctas) return false;
    }
  }
  return true;
}
}  // namespace

extern "C" {

// new_tokens, lengths [n]; items [..][12], joins [..][8] (first call with cap 0 for the sizes), first [sms + 1]: items of CTA c are
// [first[c], first[c + 1]); counts {items, joins, scratch tiles, CTAs, 1 where no item has two tiles}.
int32_t apb_rt_kv8_plan(const int32_t* new_tokens, const int32_t* lengths, int32_t n, int32_t Hq, int32_t Hkv, int32_t sms, int32_t* items,
                        int64_t items_cap, int32_t* first, int32_t* joins, int64_t joins_cap, int64_t* counts) {
  if (n < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv || sms < 1) return -1;
  const int R = Hq / Hkv, hp = std::min(R, 128), tp = 128 / hp;
  bool one_tile = true;
  for (int s = 0; s < n; ++s) one_tile = one_tile && new_tokens[s] <= tp;
  std::vector<Work> work;
  int32_t row = 0;
  for (int s = 0; s < n; ++s) {
    const int m = new_tokens[s], len = lengths[s];
    for (int t0 = 0; t0 < m; t0 += 2 * tp) {
      const int tokens = std::min(2 * tp, m - t0), pos0 = len - m + t0;
      const int end = std::max(0, std::min(len, pos0 + tokens));
      for (int kvh = 0; kvh < Hkv; ++kvh)
        for (int h = 0; h < R; h += hp)
          work.push_back({row + t0, tokens, s, kvh, kvh * R + h, std::min(hp, R - h), pos0, len, (end + kBlock - 1) / kBlock,
                          one_tile ? kOneTile : tokens > tp ? kTwoTiles : kOneOfTwo});
    }
    row += m;
  }
  std::vector<std::vector<Piece>> ctas(sms);
  // whole items, longest first
  std::vector<int> order(work.size());
  double all = 0;
  for (size_t i = 0; i < work.size(); ++i) order[i] = static_cast<int>(i), all += kItem + work[i].blocks * work[i].block;
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return work[a].blocks * work[a].block > work[b].blocks * work[b].block; });
  using Load = std::pair<double, int>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> least;
  for (int c = 0; c < sms; ++c) least.push({0.0, c});
  double whole = 0;
  for (int i : order) {
    Load l = least.top();
    least.pop();
    ctas[l.second].push_back({i, 0, work[i].blocks, -1});
    l.first += kItem + work[i].blocks * work[i].block;
    whole = std::max(whole, l.first);
    least.push(l);
  }
  // the smallest share with which cut ones fit
  double lo = all / sms, hi = whole - kJoin;
  if (hi > lo && cut(work, hi, sms, nullptr)) {
    for (int i = 0; i < 24 && hi - lo > 0.002 * hi; ++i) {
      const double mid = (lo + hi) / 2;
      (cut(work, mid, sms, nullptr) ? hi : lo) = mid;
    }
    if (hi + kJoin < 0.98 * whole) {
      for (auto& c : ctas) c.clear();
      cut(work, hi, sms, &ctas);
    }
  }
  // parts of an item are numbered in the order of their keys
  std::vector<int> parts(work.size(), 1), base(work.size(), 0);
  for (const auto& c : ctas)
    for (const Piece& p : c)
      if (p.part >= 0) parts[p.work] = std::max(parts[p.work], p.part + 1);
  int64_t n_items = 0, n_joins = 0, tiles_used = 0, used = 0;
  for (size_t i = 0; i < work.size(); ++i) {
    if (parts[i] == 1) continue;
    const Work& w = work[i];
    const int tiles = w.tokens > tp ? 2 : 1;
    base[i] = static_cast<int>(tiles_used);
    for (int g = 0; g < tiles; ++g, ++n_joins)
      if (n_joins < joins_cap) {
        const int32_t j[8] = {w.row0 + g * tp, std::min(tp, w.tokens - g * tp), w.head0, w.heads, base[i] + g, parts[i], tiles, 0};
        std::copy(j, j + 8, joins + n_joins * 8);
      }
    tiles_used += static_cast<int64_t>(parts[i]) * tiles;
  }
  for (int c = 0; c < sms; ++c) {
    if (first) first[c] = static_cast<int32_t>(n_items);
    if (!ctas[c].empty()) used = c + 1;
    for (const Piece& p : ctas[c]) {
      const Work& w = work[p.work];
      if (n_items < items_cap) {
        const int32_t v[12] = {w.row0, w.tokens, w.seq, w.kvh, w.head0, w.heads, w.pos0, w.len, p.from, p.blocks,
                               parts[p.work] > 1 ? base[p.work] + p.part * (w.tokens > tp ? 2 : 1) : -1, 0};
        std::copy(v, v + 12, items + n_items * 12);
      }
      ++n_items;
    }
  }
  if (first) first[sms] = static_cast<int32_t>(n_items);
  counts[0] = n_items;
  counts[1] = n_joins;
  counts[2] = tiles_used;
  counts[3] = used;
  counts[4] = one_tile;
  return 0;
}
}
