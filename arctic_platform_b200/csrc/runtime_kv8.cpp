// Work items of chunk attention over the 8-bit cache (csrc/kv_fp8_chunk.cu), host side.
//
// A tile holds `hp` query heads of one key head for `tp` = 128 / hp tokens; an item is one or two tiles (tokens of one sequence, side by
// side) over the 128-token blocks that they see.  Items are dealt out to the CTAs in one of two ways, by the estimated time of the
// slowest CTA: whole, the longest first to whoever has least; or in a row that is cut into equal shares, where an item that crosses
// a border is cut along the keys into parts that leave their results to a join.  Where some sequence has more than one tile, the same is
// done for pairs of CTAs with tiles of twice the tokens, and the form that is sooner done is taken.
#include <algorithm>
#include <cstdint>
#include <functional>
#include <queue>
#include <vector>

namespace {
constexpr int kBlock = 128;
// How items are taken (kv8_chunk_kernel's forms): of one or two tiles by a CTA, of one by a CTA, of one or two of 256 rows by two CTAs.
enum Form : int { kTwo, kDual, kPair };
// Estimated times of a form, in microseconds (measured at head dimension 128, with 74 or 148 equal items over 1024 to 8192 tokens): a block
// of two tiles, of one; an item besides its blocks.
struct Cost {
  double two, one, item;
};
constexpr Cost kCost[3] = {{2.6, 2.2, 6.0}, {1.7, 1.7, 5.0}, {2.4, 2.2, 7.0}};
constexpr double kPart = 1.5, kJoin = 4.0;          // what a part takes longer than an item; the join of the parts
constexpr int kLeast = 2;          // blocks of a part

struct Work {
  int32_t row0, tokens, seq, kvh, head0, heads, pos0, len, blocks;
  double block, item;              // time of one, and of the item besides
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
      const double whole = w.item + (part ? kPart : 0.0) + left * w.block;
      if (load + whole <= share * (1 + 1e-9)) {
        if (out) (*out)[c].push_back({i, at, left, part ? part : -1});
        load += whole;
        break;
      }
      const int fit = std::min(static_cast<int>((share - load - w.item - kPart) / w.block), left - kLeast);
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

struct Deal {
  Form form = kTwo;
  int tile = 0;                    // tokens of a tile
  std::vector<Work> work;
  std::vector<std::vector<Piece>> workers;
  double time = 0;
};

Deal deal(Form form, const int32_t* new_tokens, const int32_t* lengths, int n, int R, int Hkv, int sms) {
  const int hp = std::min(R, 128), ctas = form == kPair ? 2 : 1, tp = 128 / hp * ctas, step = form == kDual ? tp : 2 * tp;
  const int workers = std::max(1, sms / ctas);
  const Cost& cost = kCost[form];
  Deal d;
  d.form = form;
  d.tile = tp;
  std::vector<Work>& work = d.work;
  int32_t row = 0;
  for (int s = 0; s < n; ++s) {
    const int m = new_tokens[s], len = lengths[s];
    for (int t0 = 0; t0 < m; t0 += step) {
      const int tokens = std::min(step, m - t0), pos0 = len - m + t0;
      const int end = std::max(0, std::min(len, pos0 + tokens));
      for (int kvh = 0; kvh < Hkv; ++kvh)
        for (int h = 0; h < R; h += hp)
          work.push_back({row + t0, tokens, s, kvh, kvh * R + h, std::min(hp, R - h), pos0, len, (end + kBlock - 1) / kBlock,
                          tokens > tp ? cost.two : cost.one, cost.item});
    }
    row += m;
  }
  d.workers.resize(workers);
  // whole items, longest first
  std::vector<int> order(work.size());
  double all = 0;
  for (size_t i = 0; i < work.size(); ++i) order[i] = static_cast<int>(i), all += work[i].item + work[i].blocks * work[i].block;
  std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return work[a].blocks * work[a].block > work[b].blocks * work[b].block; });
  using Load = std::pair<double, int>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> least;
  for (int c = 0; c < workers; ++c) least.push({0.0, c});
  for (int i : order) {
    Load l = least.top();
    least.pop();
    d.workers[l.second].push_back({i, 0, work[i].blocks, -1});
    l.first += work[i].item + work[i].blocks * work[i].block;
    d.time = std::max(d.time, l.first);
    least.push(l);
  }
  // the smallest share with which cut ones fit
  double lo = all / workers, hi = d.time - kJoin;
  if (hi > lo && cut(work, hi, workers, nullptr)) {
    for (int i = 0; i < 24 && hi - lo > 0.002 * hi; ++i) {
      const double mid = (lo + hi) / 2;
      (cut(work, mid, workers, nullptr) ? hi : lo) = mid;
    }
    if (hi + kJoin < 0.98 * d.time) {
      for (auto& c : d.workers) c.clear();
      cut(work, hi, workers, &d.workers);
      d.time = hi + kJoin;
    }
  }
  return d;
}

// Estimated time of apb_kv8_few, in microseconds: rounds in which the four warps of a CTA take two pages each, in waves where CTAs do not
// all have a place, and what it takes besides.  Measured, few / items of one tile, 32 / 8 heads of 128: 8 rows 1 x 300 tokens 9 / 13 us, 16 x
// 1500 18 / 27, 128 x 6000 207 / 417, 1 x 30000 37 / 34; 16 rows 16 x 300 19 / 13, 4 x 6000 23 / 26, 16 x 6000 55 / 68, 1 x 30000 48 / 35.
double few_time(const int32_t* lengths, int n, int rows, int Hkv, int D, int sms) {
  int64_t longest = 0;
  for (int s = 0; s < n; ++s) longest = std::max<int64_t>(longest, (lengths[s] + 15) / 16);
  const int64_t units = static_cast<int64_t>(n) * Hkv;
  const int places = rows > 8 && D == 128 ? 2 : 3;          // CTAs of an SM, as kv8_splits has them
  int64_t splits = 1;
  while (splits < 8 && units * splits * 2 <= places * sms && splits * 8 < longest) splits *= 2;
  const double waves = units * splits / (static_cast<double>(sms) * places);
  return (rows > 8 ? 12.0 : 7.0) + (longest / (8.0 * splits)) * (waves > 1 ? waves + 0.25 : 1.0) * (rows > 8 ? 1.5 : 1.2);
}
}  // namespace

extern "C" {

// 1 where attention of few tokens of each sequence is sooner done without items, the way of decode attention (apb_kv8_few).
int32_t apb_rt_kv8_few(const int32_t* new_tokens, const int32_t* lengths, int32_t n, int32_t Hq, int32_t Hkv, int32_t D, int32_t sms) {
  if (n < 1 || Hkv < 1 || Hq < 1 || Hq % Hkv || sms < 1) return 0;
  const int R = Hq / Hkv;
  for (int s = 0; s < n; ++s)
    if (static_cast<int64_t>(new_tokens[s]) * R > 16) return 0;
  const int rows = n ? *std::max_element(new_tokens, new_tokens + n) * R : 0;
  return few_time(lengths, n, rows, Hkv, D, sms) < deal(kDual, new_tokens, lengths, n, R, Hkv, sms).time;
}

// new_tokens, lengths [n]; form: -1 the one that is sooner done (kDual where no sequence has two tiles, whatever is asked for); items [..][12],
// joins [..][8] (first call with cap 0 for the sizes), first [sms + 1]: items of CTA (or pair) c are [first[c], first[c + 1]); counts {items,
// joins, scratch tiles of 128 rows, CTAs or pairs, form}.
int32_t apb_rt_kv8_plan(const int32_t* new_tokens, const int32_t* lengths, int32_t n, int32_t Hq, int32_t Hkv, int32_t D, int32_t sms,
                        int32_t form, int32_t* items, int64_t items_cap, int32_t* first, int32_t* joins, int64_t joins_cap, int64_t* counts) {
  if (n < 0 || Hkv < 1 || Hq < 1 || Hq % Hkv || sms < 1) return -1;
  const int R = Hq / Hkv, hp = std::min(R, 128), tp = 128 / hp;
  bool one_tile = true;
  for (int s = 0; s < n; ++s) one_tile = one_tile && new_tokens[s] <= tp;
  Deal d = deal(one_tile ? kDual : kTwo, new_tokens, lengths, n, R, Hkv, sms);
  const bool pairs_open = !one_tile && D == 128 && sms > 1;       // of 64 columns a half would have another swizzle
  if (form == kPair && !pairs_open) return -1;
  if (pairs_open && form != kTwo) {
    Deal pairs = deal(kPair, new_tokens, lengths, n, R, Hkv, sms);
    if (form == kPair || pairs.time < d.time) d = std::move(pairs);
  }
  const std::vector<Work>& work = d.work;
  // parts of an item are numbered in the order of their keys
  std::vector<int> parts(work.size(), 1), base(work.size(), 0);
  for (const auto& c : d.workers)
    for (const Piece& p : c)
      if (p.part >= 0) parts[p.work] = std::max(parts[p.work], p.part + 1);
  auto tiles_of = [&](const Work& w) { return (w.tokens > d.tile ? 2 : 1) * (d.form == kPair ? 2 : 1); };       // of 128 rows, in the scratch
  int64_t n_items = 0, n_joins = 0, tiles_used = 0, used = 0;
  for (size_t i = 0; i < work.size(); ++i) {
    if (parts[i] == 1) continue;
    const Work& w = work[i];
    const int tiles = tiles_of(w);
    base[i] = static_cast<int>(tiles_used);
    for (int g = 0; g * tp < w.tokens; ++g, ++n_joins)
      if (n_joins < joins_cap) {
        const int32_t j[8] = {w.row0 + g * tp, std::min(tp, w.tokens - g * tp), w.head0, w.heads, base[i] + g, parts[i], tiles, 0};
        std::copy(j, j + 8, joins + n_joins * 8);
      }
    tiles_used += static_cast<int64_t>(parts[i]) * tiles;
  }
  const int workers = static_cast<int>(d.workers.size());
  for (int c = 0; c < workers; ++c) {
    if (first) first[c] = static_cast<int32_t>(n_items);
    if (!d.workers[c].empty()) used = c + 1;
    for (const Piece& p : d.workers[c]) {
      const Work& w = work[p.work];
      if (n_items < items_cap) {
        const int32_t v[12] = {w.row0, w.tokens, w.seq, w.kvh, w.head0, w.heads, w.pos0, w.len, p.from, p.blocks,
                               parts[p.work] > 1 ? base[p.work] + p.part * tiles_of(w) : -1, 0};
        std::copy(v, v + 12, items + n_items * 12);
      }
      ++n_items;
    }
  }
  if (first) std::fill(first + workers, first + sms + 1, static_cast<int32_t>(n_items));
  counts[0] = n_items;
  counts[1] = n_joins;
  counts[2] = tiles_used;
  counts[3] = used;
  counts[4] = d.form;
  return 0;
}
}
