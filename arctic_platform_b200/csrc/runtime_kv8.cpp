// Work items of chunk attention over the 8-bit cache (csrc/kv_fp8_chunk.cu), host side.
//
// A tile holds `hp` query heads of one key head for `tp` = 128 / hp tokens; an item is one or two tiles (tokens of one sequence, side by
// side) over the 128-token blocks that they see.  Where there are fewer items than it takes to keep the GPU busy evenly, they are cut
// along the keys into parts of `limit` blocks at most, each an item of its own that leaves its result to a join.
#include <algorithm>
#include <cstdint>
#include <queue>
#include <vector>

namespace {
constexpr int kBlock = 128;
// Time of an item in blocks of two tiles: set-up and output, and what one tile takes of two.
constexpr double kItem = 2.0, kPart = 1.0, kOneTile = 0.6;

struct Work {
  int32_t row0, tokens, seq, kvh, head0, heads, pos0, len, blocks;
};

int parts_of(int blocks, int limit) { return std::max(1, (blocks + limit - 1) / limit); }

// Time until all items are through, longest first, on `sms` machines.
double makespan(const std::vector<Work>& work, int limit, int tp, int sms) {
  std::vector<double> cost;
  for (const Work& w : work) {
    const int n = parts_of(w.blocks, limit);
    const double each = (w.blocks / static_cast<double>(n)) * (w.tokens > tp ? 1.0 : kOneTile) + kItem + (n > 1 ? kPart : 0.0);
    cost.insert(cost.end(), n, each);
  }
  std::sort(cost.begin(), cost.end(), [](double a, double b) { return a > b; });
  // the kernel deals the items out forth and back
  std::vector<double> load(sms, 0.0);
  for (size_t i = 0; i < cost.size(); ++i) {
    const size_t round = i / sms, k = i % sms;
    load[(round & 1) ? sms - 1 - k : k] += cost[i];
  }
  return *std::max_element(load.begin(), load.end());
}
}  // namespace

extern "C" {

// new_tokens, lengths [n]; out: items [..][12], joins [..][8] (first call with cap 0 for the sizes), counts {items, joins, scratch tiles}.
int32_t apb_rt_kv8_plan(const int32_t* new_tokens, const int32_t* lengths, int32_t n, int32_t Hq, int32_t Hkv, int32_t sms, int32_t* items,
                        int64_t items_cap, int32_t* joins, int64_t joins_cap, int64_t* counts) {
  if (n < 0 || Hkv < 1 || Hq % Hkv || sms < 1) return -1;
  const int R = Hq / Hkv, hp = std::min(R, 128), tp = 128 / hp;
  std::vector<Work> work;
  int32_t row = 0;
  for (int s = 0; s < n; ++s) {
    const int m = new_tokens[s], len = lengths[s];
    for (int t0 = 0; t0 < m; t0 += 2 * tp) {
      const int tokens = std::min(2 * tp, m - t0), pos0 = len - m + t0;
      const int end = std::max(0, std::min(len, pos0 + tokens));
      for (int kvh = 0; kvh < Hkv; ++kvh)
        for (int h = 0; h < R; h += hp)
          work.push_back({row + t0, tokens, s, kvh, kvh * R + h, std::min(hp, R - h), pos0, len, (end + kBlock - 1) / kBlock});
    }
    row += m;
  }
  int most = 0;
  for (const Work& w : work) most = std::max(most, w.blocks);
  int limit = std::max(1, most);
  double best = makespan(work.empty() ? std::vector<Work>{{0, 0, 0, 0, 0, 0, 0, 0, 0}} : work, limit, tp, sms);
  if (static_cast<int64_t>(work.size()) < 8ll * sms)         // more are even enough
    for (int parts = 2; parts <= 64 && (most + parts - 1) / parts >= 2; ++parts) {
      const int l = (most + parts - 1) / parts;
      const double t = makespan(work, l, tp, sms);
      if (t < 0.97 * best) best = t, limit = l;
    }
  struct Item {
    int32_t v[12];
    double cost;
  };
  std::vector<Item> out;
  int64_t n_joins = 0, tiles_used = 0;
  for (const Work& w : work) {
    const int parts = parts_of(w.blocks, limit), tiles = w.tokens > tp ? 2 : 1;
    for (int k = 0; k < parts; ++k) {
      const int b0 = static_cast<int>(static_cast<int64_t>(w.blocks) * k / parts), b1 = static_cast<int>(static_cast<int64_t>(w.blocks) * (k + 1) / parts);
      Item it = {{w.row0, w.tokens, w.seq, w.kvh, w.head0, w.heads, w.pos0, w.len, b0, b1 - b0,
                  parts > 1 ? static_cast<int32_t>(tiles_used + k * tiles) : -1, 0},
                 (b1 - b0) * (tiles > 1 ? 1.0 : kOneTile)};
      out.push_back(it);
    }
    if (parts > 1) {
      for (int g = 0; g < tiles; ++g, ++n_joins)
        if (n_joins < joins_cap) {
          const int32_t j[8] = {w.row0 + g * tp, std::min(tp, w.tokens - g * tp), w.head0, w.heads, static_cast<int32_t>(tiles_used + g), parts, tiles, 0};
          std::copy(j, j + 8, joins + n_joins * 8);
        }
      tiles_used += static_cast<int64_t>(parts) * tiles;
    }
  }
  std::stable_sort(out.begin(), out.end(), [](const Item& a, const Item& b) { return a.cost > b.cost; });
  for (size_t i = 0; i < out.size() && static_cast<int64_t>(i) < items_cap; ++i) std::copy(out[i].v, out[i].v + 12, items + i * 12);
  counts[0] = static_cast<int64_t>(out.size());
  counts[1] = n_joins;
  counts[2] = tiles_used;
  return 0;
}
}
