// Runs the plan of an attention launch (csrc/attention_plan.h) on the CPU, every workgroup's, and checks that the tiles, their
// parts and the merge's units come out once each. Plans come on stdin, one a line:
//   tokens seqs hq hk d causal max_keys cu[0 .. seqs] [paged lengths[0 .. seqs - 1]]
// and each is answered by a line: "ok" and the number of items, or what is wrong.

#include "wave.h"

#include "attention_plan.h"

#include <iostream>
#include <map>
#include <set>
#include <sstream>
#include <string>
#include <tuple>

using namespace bp::attn;

namespace {

struct Wanted {
  int rows, keys, end, splits_seen = 0;
};

template <bool MERGE>
Item item_of(const Args& a, int index, bool& uniform) {
  static Item lanes[wave::kLanes];
  wave::run([&](int lane) { lanes[lane] = find_item<MERGE>(a, index); });
  for (int l = 1; l < wave::kLanes; ++l) {
    const Item &x = lanes[0], &y = lanes[l];
    if (x.b != y.b) uniform = false;
    else if (x.b < 0) uniform &= x.extra == y.extra;
    else uniform &= std::tie(x.row0, x.rows, x.key0, x.key1, x.split, x.splits, x.slot, x.small, x.divided, x.first, x.keys) ==
                    std::tie(y.row0, y.rows, y.key0, y.key1, y.split, y.splits, y.slot, y.small, y.divided, y.first, y.keys);
  }
  return lanes[0];
}

std::string check(Args a, const std::vector<int>& cu, const std::vector<int>& lengths, bool paged) {
  a.cu = cu.data();
  a.lengths = paged ? lengths.data() : nullptr;
  Launch n;
  if (!plan_launch(a, n)) return "no launch";
  std::vector<float> none(1);
  a.ws = n.workspace > 0 ? none.data() : nullptr;  // (never read: only whether there is one counts)
  std::ostringstream out;

  std::map<std::pair<int, int>, Wanted> tiles;  // by sequence and first row
  const int group = a.group.d;
  for (int b = 0; b < a.seqs; ++b) {
    const int begin = min(max(cu[b], 0), a.tokens), end = min(max(cu[b + 1], begin), a.tokens);
    const int count = end - begin, rows = count * group, keys = paged ? min(max(lengths[b], 0), a.max_keys) : count;
    const int tile = rows <= 64 ? 32 : 128;
    for (int r = 0; r < rows; r += tile) {
      Wanted w;
      w.rows = min(tile, rows - r);
      w.keys = keys;
      w.end = a.causal ? min(keys, max(0, keys - count + (r + w.rows - 1) / group + 1)) : keys;
      tiles[{b, r}] = w;
    }
  }

  // every part of every tile once, its keys whole and apart, its slot its own
  std::map<std::pair<int, int>, std::map<int, Item>> seen;
  std::set<int> slots;
  int items = 0, extras = 0;
  bool uniform = true;
  for (int index = 0; index < n.index; ++index) {
    const Item it = item_of<false>(a, index, uniform);
    if (!uniform) return "lanes that disagree";
    if (it.b < 0) {
      if (it.extra != extras++) return "places past the last tile out of order";
      continue;
    }
    if (extras > 0) return "a tile past the last";
    ++items;
    const auto w = tiles.find({it.b, it.row0});
    if (w == tiles.end()) {
      out << "index " << index << ": no tile at row " << it.row0 << " of sequence " << it.b;
      return out.str();
    }
    if (it.rows != w->second.rows || it.keys != w->second.keys || it.begin != min(max(cu[it.b], 0), a.tokens))
      return "a tile of wrong size";
    if (!seen[{it.b, it.row0}].emplace(it.split, it).second) {
      out << "sequence " << it.b << " row " << it.row0 << " part " << it.split << " twice";
      return out.str();
    }
    if (it.divided) {
      if (it.slot + it.split >= a.slots) return "a slot past the workspace";
      if (!slots.insert(it.slot + it.split).second) return "a slot of two parts";
    }
  }
  if (extras < 1) return "no workgroup for the rows of no sequence";
  int divided_rows = 0;
  std::map<std::pair<int, int>, int> live;  // parts of a tile that have keys
  for (const auto& [key, w] : tiles) {
    const auto s = seen.find(key);
    if (s == seen.end()) {
      out << "sequence " << key.first << " row " << key.second << " never";
      return out.str();
    }
    int at = 0, count = 0;
    for (const auto& [split, it] : s->second) {
      if (split != count++ || it.splits != s->second.begin()->second.splits) return "parts that do not belong together";
      if (it.key0 != at || it.key1 < at) return "keys left out or twice";
      at = it.key1;
      if (it.key1 > it.key0 || split == 0) live[key] = split + 1;
    }
    if (at != w.end) return "keys left out at the end";
    if (count != s->second.begin()->second.splits) return "parts left out";
    if (s->second.begin()->second.divided) divided_rows += w.rows;
  }

  // every row of the divided tiles in one unit of the merge, with its tile's slots and live parts
  if (n.merges > 0) {
    std::set<std::pair<int, int>> rows;
    for (int unit = 0;; ++unit) {
      const Item it = item_of<true>(a, unit, uniform);
      if (!uniform) return "lanes that disagree";
      if (it.b < 0) break;
      const auto s = seen.find({it.b, it.row0});
      if (s == seen.end() || !s->second.begin()->second.divided) return "a unit of no divided tile";
      if (it.slot != s->second.begin()->second.slot || it.splits != live[{it.b, it.row0}]) return "a unit with other parts";
      for (int r = 0; r < it.rows; ++r)
        if (!rows.emplace(it.b, it.row0 + it.split + r).second) return "a row of two units";
    }
    if (static_cast<int>(rows.size()) != divided_rows) return "divided rows in no unit";
  } else if (divided_rows > 0) {
    return "divided rows without a merge";
  }
  out << "ok " << items << " of them ordered " << a.order << " divided " << slots.size();
  return out.str();
}

}  // namespace

int main() {
  std::string line;
  while (std::getline(std::cin, line)) {
    std::istringstream in(line);
    Args a = {};
    in >> a.tokens >> a.seqs >> a.hq >> a.hk.d >> a.d >> a.causal >> a.max_keys;
    std::vector<int> cu(a.seqs + 1), lengths(a.seqs);
    for (int& x : cu) in >> x;
    std::string paged;
    in >> paged;
    for (int& x : lengths) in >> x;
    a.page = Div::of(1);
    std::cout << check(a, cu, lengths, paged == "paged") << std::endl;
  }
}
