// attn_plan.cu — sj_attn_plan: which keys the query rows of a batch see (host code).
//
// A row's visible keys are at most two intervals of packed rows: the segment's
// prefix, and the part of the row's document that causality, the window and
// kv_lens leave.  The plan holds
//   rows   8 words for each query row: its packed position, the two disjoint
//          intervals [a0, a1) and [b0, b1) (a1 <= b0; the first empty only when
//          both are), 3 words of padding;
//   items  4 words for each tile of up to 128 consecutive query rows: first
//          row, rows, first key tile, key tiles; most key tiles first, so that
//          the longest work starts first;
//   tiles  for each item its key tiles: the first key row k0 of 64, greedily
//          from the first key that a row of the item sees and no earlier tile
//          covers; ~k0 when every row of the item sees all 64 keys (no mask).
// For few query rows also
//   parts   8 words each: first row, rows, first key tile, key tiles of a run of a
//           group's tiles, the workspace row of its first row (-1: the group has
//           one part), and, in the k-th part's words, the k-th group's first part
//           and number of parts, 1 word of padding; a group is up to 16 query rows
//           of one segment;
//   splits  4 words for each group of several parts: first row, rows, parts, first
//           workspace row;
//   few     the groups' key tiles, as above.
#include <algorithm>
#include <array>
#include <cstdlib>
#include <new>
#include <vector>

#include "../../include/snapjudge_b200.h"
#include "kernels.h"

namespace {

int bad(const char* m) {
  sjb::set_last_error(m);
  return SJ_ERR_INVALID;
}

struct Iv {
  int a, b;
};
// Above this many query rows the tile kernel fills the GPU.
constexpr int kFewMostRows = 4096;
// Parts that the warps of one block compute and join.
constexpr int kJoinMost = 8;

// The rows' keys as tiles: `next` tiles greedily over the union of the intervals.
struct Row {
  int pos, a0, a1, b0, b1, seg;
};
void cover(const Row* rows, int r0, int r1, std::vector<Iv>& iv, std::vector<int32_t>& tiles) {
  iv.clear();
  Iv ca{0, 0x7fffffff}, cb{0, 0x7fffffff};  // keys that every row sees, by its intervals
  for (int r = r0; r < r1; ++r) {
    const Row& w = rows[r];
    // (neighbours mostly have the same intervals)
    if (w.a1 > w.a0 && (r == r0 || w.a0 != rows[r - 1].a0 || w.a1 != rows[r - 1].a1)) iv.push_back({w.a0, w.a1});
    if (w.b1 > w.b0 && (r == r0 || w.b0 != rows[r - 1].b0 || w.b1 != rows[r - 1].b1)) iv.push_back({w.b0, w.b1});
    ca.a = std::max(ca.a, w.a0), ca.b = std::min(ca.b, w.a1);
    cb.a = std::max(cb.a, w.b0), cb.b = std::min(cb.b, w.b1);
  }
  std::sort(iv.begin(), iv.end(), [](const Iv& x, const Iv& y) { return x.a < y.a; });
  long long next = 0;  // first key that no tile covers yet
  for (const Iv& v : iv) {
    for (long long k = std::max<long long>(v.a, next); k < v.b; k = next) {
      next = k + 64;
      const int k0 = (int)k;
      const bool full = (k0 >= ca.a && next <= ca.b) || (k0 >= cb.a && next <= cb.b);
      tiles.push_back(full ? ~k0 : k0);
    }
  }
}

int make_plan(const sj_attn_plan_args& p, int32_t* plan, int64_t plan_len,
              sj_attn_plan_info* info) {
  const int32_t* cu = p.cu_seqlens;
  if (p.B < 0) return bad("negative batch");
  if (p.window < 0) return bad("negative window");
  if (p.form < SJ_ATTN_AUTO || p.form > SJ_ATTN_FEW) return bad("bad form");
  if (!cu) return bad("cu_seqlens is null");
  if (cu[0] != 0) return bad("cu_seqlens[0] must be 0");
  for (int b = 0; b < p.B; ++b) {
    const int n = cu[b + 1] - cu[b];
    if (cu[b + 1] < cu[b]) return bad("cu_seqlens must be non-decreasing");
    if (p.prefix && (p.prefix[b] < 0 || p.prefix[b] > n))
      return bad("a prefix must be between 0 and its segment's length");
    if (p.kv_lens && p.kv_lens[b] < 0) return bad("kv_lens must not be negative");
  }
  const int T = cu[p.B];
  if (p.docs) {
    if (p.n_docs < 0) return bad("negative number of documents");
    if (p.docs[0] != 0 || p.docs[p.n_docs] != T)
      return bad("documents must start at row 0 and end at the last row");
    for (int d = 0; d < p.n_docs; ++d)
      if (p.docs[d + 1] < p.docs[d]) return bad("documents must be non-decreasing");
    for (int b = 0, d = 0; b <= p.B; ++b) {
      while (d < p.n_docs && p.docs[d] < cu[b]) ++d;
      if (p.docs[d] != cu[b]) return bad("every segment boundary must be a document boundary");
    }
  }
  if (p.n_q < 0) return bad("negative number of query rows");
  if (p.q_rows)
    for (int r = 0; r < p.n_q; ++r)
      if (p.q_rows[r] < 0 || p.q_rows[r] >= T || (r > 0 && p.q_rows[r] <= p.q_rows[r - 1]))
        return bad("q_rows must be strictly increasing rows of the batch");
  const int nr = p.q_rows ? p.n_q : T;

  // the rows' intervals
  std::vector<Row> rows((size_t)nr);
  for (int r = 0, b = 0, d = 0; r < nr; ++r) {
    const int i = p.q_rows ? p.q_rows[r] : r;
    while (cu[b + 1] <= i) ++b;
    int lo = cu[b], hi = cu[b + 1];
    if (p.docs) {
      while (p.docs[d + 1] <= i) ++d;
      lo = p.docs[d];
      hi = p.docs[d + 1];
    }
    if (p.causal) hi = std::min(hi, i + 1);
    if (p.window > 0) {
      lo = std::max(lo, i - std::min(p.window, i));
      if (p.window < hi - i) hi = i + p.window + 1;
    }
    const int n = cu[b + 1] - cu[b];
    const int end = cu[b] + (p.kv_lens ? std::min(p.kv_lens[b], n) : n);
    hi = std::min(hi, end);
    const int a0 = cu[b];
    const int a1 = p.prefix ? std::min(a0 + p.prefix[b], end) : a0;
    lo = std::max(lo, a1);
    hi = std::max(hi, lo);
    Row& w = rows[r];
    w.pos = i;
    w.seg = b;
    if (a1 == a0) {  // no prefix
      w.a0 = lo, w.a1 = hi, w.b0 = w.b1 = hi;
    } else if (lo == a1) {  // one interval
      w.a0 = a0, w.a1 = hi, w.b0 = w.b1 = hi;
    } else {
      w.a0 = a0, w.a1 = a1, w.b0 = lo, w.b1 = hi;
    }
  }

  // query tiles and the key tiles that they need
  struct Item {
    int row0, rows, tile0, tiles;
  };
  std::vector<Item> items;
  std::vector<int32_t> tiles;
  std::vector<Iv> iv;
  for (int r0 = 0; r0 < nr; r0 += 128) {
    const int r1 = std::min(nr, r0 + 128);
    Item it{r0, r1 - r0, (int)tiles.size(), 0};
    cover(rows.data(), r0, r1, iv, tiles);
    // nearest first: where scores fall with the distance, the maximum is found at once
    const int mid = rows[(r0 + r1) / 2].pos;
    auto away = [&](int e) { return std::abs((e < 0 ? ~e : e) + 32 - mid); };
    std::stable_sort(tiles.begin() + it.tile0, tiles.end(),
                     [&](int x, int y) { return away(x) < away(y); });
    if (tiles.size() > 0x7fffffff) return bad("the batch needs too many key tiles");
    it.tiles = (int)tiles.size() - it.tile0;
    items.push_back(it);
  }
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& x, const Item& y) { return x.tiles > y.tiles; });

  // few query rows: groups of up to 16 rows of one segment, split into parts
  struct Part {
    int row0, rows, tile0, tiles, ws;
  };
  std::vector<Part> parts;
  std::vector<std::array<int, 4>> splits;
  std::vector<int32_t> few;
  std::vector<std::array<int, 2>> first;  // each group's first part and parts
  int max_rows = 0, join = 0;
  long long ws_rows = 0;
  if (nr > 0 && (p.form == SJ_ATTN_FEW || (p.form == SJ_ATTN_AUTO && nr <= kFewMostRows))) {
    std::vector<Item> groups;
    for (int r0 = 0, r1; r0 < nr; r0 = r1) {
      for (r1 = r0 + 1; r1 < nr && r1 < r0 + 16 && rows[r1].seg == rows[r0].seg;) ++r1;
      Item g{r0, r1 - r0, (int)few.size(), 0};
      cover(rows.data(), r0, r1, iv, few);
      g.tiles = (int)few.size() - g.tile0;
      groups.push_back(g);
    }
    // parts short enough to spread over the SMs, long enough not to be joined often
    const int most = (int)std::min<long long>(8, 1 + (long long)few.size() * 8 / (148 * 8));
    int widest = 0;
    for (const Item& g : groups) {
      const int n = std::max(1, (g.tiles + most - 1) / most), per = (g.tiles + n - 1) / n;
      widest = std::max(widest, n);
      first.push_back({(int)parts.size(), n});
      max_rows = std::max(max_rows, g.rows);
      if (n > 1) splits.push_back({g.row0, g.rows, n, (int)ws_rows});
      for (int k = 0; k < n; ++k) {
        const int t0 = std::min(g.tiles, k * per), t1 = std::min(g.tiles, t0 + per);
        parts.push_back({g.row0, g.rows, g.tile0 + t0, t1 - t0, n > 1 ? (int)ws_rows : -1});
        if (n > 1) ws_rows += g.rows;
      }
    }
    // at most half of the joining blocks' warps without a part
    if (widest > 1 && widest <= kJoinMost && (size_t)widest * groups.size() <= 2 * parts.size())
      join = widest;
  }

  if (few.size() > 0x7fffffff || ws_rows > 0x7fffffff) return bad("the batch needs too many key tiles");
  info->n_rows = nr;
  info->n_keys = T;
  info->n_items = (int)items.size();
  info->n_tiles = (int)tiles.size();
  info->off_items = 8ll * nr;
  info->off_tiles = info->off_items + 4ll * (long long)items.size();
  info->n_parts = (int)parts.size();
  info->n_splits = (int)splits.size();
  info->n_groups = (int)first.size();
  info->join = join;
  info->n_few_tiles = (int)few.size();
  info->longest = items.empty() ? 0 : items[0].tiles;
  info->form = p.form;
  info->max_group_rows = max_rows;
  info->ws_rows = (int)ws_rows;
  info->off_parts = info->off_tiles + ((long long)tiles.size() + 3) / 4 * 4;  // 16-byte words
  info->off_splits = info->off_parts + 8ll * (long long)parts.size();
  info->off_few_tiles = info->off_splits + 4ll * (long long)splits.size();
  info->plan_len = parts.empty() ? info->off_tiles + (long long)tiles.size()
                                 : info->off_few_tiles + (long long)few.size();
  if (!plan) return SJ_OK;
  if (plan_len < info->plan_len) return bad("the plan's memory is too small");
  for (int r = 0; r < nr; ++r) {
    const Row& w = rows[r];
    const int32_t v[8] = {w.pos, w.a0, w.a1, w.b0, w.b1, 0, 0, 0};
    std::copy(v, v + 8, plan + 8ll * r);
  }
  for (size_t k = 0; k < items.size(); ++k) {
    const int32_t v[4] = {items[k].row0, items[k].rows, items[k].tile0, items[k].tiles};
    std::copy(v, v + 4, plan + info->off_items + 4 * (long long)k);
  }
  std::copy(tiles.begin(), tiles.end(), plan + info->off_tiles);
  if (parts.empty()) return SJ_OK;
  std::fill(plan + info->off_tiles + (long long)tiles.size(), plan + info->off_parts, 0);
  for (size_t k = 0; k < parts.size(); ++k) {
    const Part& q = parts[k];
    const bool g = k < first.size();
    const int32_t v[8] = {q.row0, q.rows, q.tile0, q.tiles, q.ws, g ? first[k][0] : 0,
                          g ? first[k][1] : 0, 0};
    std::copy(v, v + 8, plan + info->off_parts + 8 * (long long)k);
  }
  for (size_t k = 0; k < splits.size(); ++k)
    std::copy(splits[k].begin(), splits[k].end(), plan + info->off_splits + 4 * (long long)k);
  std::copy(few.begin(), few.end(), plan + info->off_few_tiles);
  return SJ_OK;
}

}  // namespace

extern "C" int sj_attn_plan(const sj_attn_plan_args* args, int32_t* plan, int64_t plan_len,
                            sj_attn_plan_info* info) {
  if (!args || !info) return bad("null plan argument");
  try {
    return make_plan(*args, plan, plan_len, info);
  } catch (const std::bad_alloc&) {
    return bad("out of host memory for the plan");
  }
}
