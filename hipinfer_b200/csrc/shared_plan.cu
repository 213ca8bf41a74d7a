// The plan of a step's shared-prefix attention, made on the host from the lengths alone and used by every layer of the step.
//
// A group's shared range and a request's own range are SEGMENTS: some rows against a range of keys. A segment's keys are cut into equal
// chunks, an item is (chunk, kv head, up to tile_tokens rows), and each CTA gets a list of items: the shared items in the order of their keys,
// so that the CTAs at work at one time read the same tiles (once from memory, then from L2), each to the CTA with the least work so
// far, then the requests' own, longest first. A chunk is the one among a few fractions of an even share of the work whose longest CTA, and whose partial
// results, cost least.
#include "common.cuh"
#include "shared_plan.h"

#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

namespace {

struct Segment {
  int table, token, tokens, pos, lo, hi;   // as in SharedItem; SP_NO_MASK or the first token's position
  int tiles, chunks, parts, base;          // key tiles; what a chunk length makes of it
  bool shared;
};
struct Cut {
  long parts = 0;      // part rows
  double cost = 0;     // in key tiles of one CTA
};

struct Planner {
  int Hkv, G, key_tile, n_ctas, narrow_tokens, few_tokens;
  double item_cost, wide_cost, few_cost, part_cost;
  static constexpr double row_cost = 0.02;               // of a part of the row that has most of them (they are joined one after another)
  std::vector<Segment> segs;
  std::vector<std::vector<std::pair<int, int>>> lists;   // a CTA's (segment, head * chunks + chunk)

  bool narrow(const Segment& s) const { return s.tokens <= narrow_tokens; }
  double tile_cost(const Segment& s) const { return s.tokens <= few_tokens ? few_cost : narrow(s) ? 1.0 : wide_cost; }
  // What chunks of about `cost` come to: the longest CTA, if the shared items fill rounds of all CTAs and the requests' own ones what is left of the
  // last of them, and the partial results.
  Cut cut(double cost) {
    Cut c;
    double sum[2] = {0, 0}, most[2] = {0, 0};
    long items[2] = {0, 0};
    int parts[2] = {0, 0};
    for (Segment& s : segs) {
      const int len = std::max(1, (int)(cost / tile_cost(s) + 0.999));
      s.chunks = (s.tiles + len - 1) / len;
      s.parts = s.chunks * (narrow(s) ? 2 : 1);
      s.base = (int)std::min<long>(c.parts, 0x7fffffff);
      c.parts += (long)Hkv * s.parts * s.tokens * G;
      const int k = s.shared ? 0 : 1;
      const double all = item_cost * s.chunks + tile_cost(s) * s.tiles;
      sum[k] += Hkv * all;
      most[k] = std::max(most[k], all / s.chunks);
      items[k] += (long)Hkv * s.chunks;
      parts[k] = std::max(parts[k], s.parts);
    }
    auto rounds = [&](int k) { return items[k] ? (items[k] + n_ctas - 1) / n_ctas * (sum[k] / items[k]) : 0.0; };
    const double even = (sum[0] + sum[1]) / n_ctas;
    double longest = std::max(even, rounds(0));
    if (!items[0]) longest = std::max(even, rounds(1));
    if (items[1] && even >= rounds(0)) longest = std::max(longest, even + most[1] / 2);
    c.cost = std::max(longest, std::max(most[0], most[1])) + part_cost * c.parts + row_cost * (parts[0] + parts[1]);
    return c;
  }
  // Gives the items to the CTAs.
  void deal() {
    // the CTAs as a heap, the one with the least work (of these the lowest) on top
    std::vector<std::pair<float, int>> load(n_ctas);
    for (int i = 0; i < n_ctas; i++) load[i] = {0.f, i};
    lists.assign(n_ctas, {});
    auto give = [&](int s, int item) {
      std::pair<float, int> l = load[0];
      l.first += (float)(item_cost + tile_cost(segs[s]) * segs[s].tiles / segs[s].chunks);
      lists[l.second].push_back({s, item});
      int at = 0;
      for (int child; (child = 2 * at + 1) < n_ctas; at = child) {
        if (child + 1 < n_ctas && load[child + 1] < load[child]) child++;
        if (!(load[child] < l)) break;
        load[at] = load[child];
      }
      load[at] = l;
    };
    std::vector<int> own, shared;
    int most = 0;
    for (size_t i = 0; i < segs.size(); i++) {
      (segs[i].shared ? shared : own).push_back((int)i);
      if (segs[i].shared) most = std::max(most, segs[i].chunks);
    }
    for (int k = 0; k < most; k++)
      for (int h = 0; h < Hkv; h++)
        for (int i : shared)
          if (k < segs[i].chunks) give(i, h * segs[i].chunks + k);
    std::stable_sort(own.begin(), own.end(), [&](int a, int b) { return (long)segs[a].tiles * segs[b].chunks > (long)segs[b].tiles * segs[a].chunks; });
    for (int i : own)
      for (int u = 0; u < Hkv * segs[i].chunks; u++) give(i, u);
  }
};

}  // namespace

// q_len, ctx_len [R]; groups [n_groups][3]: first request, requests, shared tokens. out: SP_HEADER ints, then items, each CTA's first item (one more
// for the end), tokens; returns the ints that were written, or, where `cap` is too small, minus the number that is needed; 0 with a message in
// hb_last_error for lengths that make no plan. tile_tokens: rows of q in an item; narrow_tokens: items of at most so many rows leave two
// parts (two chains share their keys), 0: none do. Costs are in key tiles of a narrow item: an item's beginning and end, a tile of another
// item, a part row; a tile of an item of up to few_tokens rows (0: as another).
HB_EXPORT int hb_shared_plan(const int* q_len, const int* ctx_len, int R, const int* groups, int n_groups, int Hq, int Hkv, int tile_tokens,
                             int narrow_tokens, int key_tile, int n_ctas, float item_cost, float wide_cost, float part_cost, int few_tokens, float few_cost,
                             int* out, int cap) {
  try {
    if (R < 0 || n_groups < 0 || Hkv < 1 || Hq < Hkv || Hq % Hkv || tile_tokens < 1 || key_tile < 1 || n_ctas < 1) {
      hb_set_error("hb_shared_plan: bad sizes (%d requests, %d groups, %d/%d heads, %d rows an item)", R, n_groups, Hq, Hkv, tile_tokens);
      return 0;
    }
    std::vector<int> start(R + 1, 0), group_of(R, -1), shared(R, 0);
    long rows = 0;
    for (int r = 0; r < R; r++) {
      if (q_len[r] < 0 || ctx_len[r] < 0 || (long)q_len[r] + ctx_len[r] >= SP_NO_MASK) {
        hb_set_error("hb_shared_plan: request %d has %d rows behind %d tokens", r, q_len[r], ctx_len[r]);
        return 0;
      }
      rows += q_len[r];
      if (rows > (1 << 28)) {
        hb_set_error("hb_shared_plan: too many rows");
        return 0;
      }
      start[r + 1] = (int)rows;
    }
    for (int g = 0; g < n_groups; g++) {
      const int first = groups[3 * g], n = groups[3 * g + 1], s = groups[3 * g + 2];
      if (first < 0 || n < 0 || (long)first + n > R || s < 0) {
        hb_set_error("hb_shared_plan: group %d (requests %d to %ld, %d tokens) is outside the %d requests", g, first, (long)first + n - 1, s, R);
        return 0;
      }
      for (int r = first; r < first + n; r++) {
        if (group_of[r] >= 0) {
          hb_set_error("hb_shared_plan: request %d is in groups %d and %d", r, group_of[r], g);
          return 0;
        }
        if (s > ctx_len[r]) {
          hb_set_error("hb_shared_plan: group %d shares %d tokens, request %d holds %d", g, s, r, ctx_len[r]);
          return 0;
        }
        group_of[r] = g;
        shared[r] = s;
      }
    }
    Planner p;
    p.Hkv = Hkv;
    p.G = Hq / Hkv;
    p.key_tile = key_tile;
    p.n_ctas = n_ctas;
    p.narrow_tokens = narrow_tokens;
    p.item_cost = item_cost;
    p.wide_cost = wide_cost;
    p.part_cost = part_cost;
    p.few_tokens = few_tokens;
    p.few_cost = few_cost;
    const int T = start[R];
    std::vector<SharedToken> tokens(T);
    std::vector<int> pre_seg(T, -1), own_seg(T, -1), pre_row(T, 0), own_row(T, 0);
    auto add = [&](int table, int token, int n, int pos, int lo, int hi, bool is_shared, std::vector<int>& seg, std::vector<int>& row) {
      for (int at = 0; at < n; at += tile_tokens) {
        Segment s = {};
        s.table = table;
        s.token = token + at;
        s.tokens = std::min(tile_tokens, n - at);
        s.pos = pos == SP_NO_MASK ? pos : pos + at;
        s.lo = lo;
        s.hi = pos == SP_NO_MASK ? hi : std::min(hi, s.pos + s.tokens);
        s.shared = is_shared;
        s.tiles = (s.hi - 1) / key_tile - s.lo / key_tile + 1;
        for (int i = 0; i < s.tokens; i++) {
          seg[s.token + i] = (int)p.segs.size();
          row[s.token + i] = i * p.G;
        }
        p.segs.push_back(s);
      }
    };
    for (int g = 0; g < n_groups; g++) {
      const int first = groups[3 * g], n = groups[3 * g + 1], s = groups[3 * g + 2];
      int with = 0;                                          // requests that bring rows
      for (int r = first; r < first + n; r++) with += q_len[r] > 0;
      if (with < 2 || s == 0) {                              // nothing is shared by two: the keys are the requests' own
        for (int r = first; r < first + n; r++) shared[r] = 0;
        continue;
      }
      add(first, start[first], start[first + n] - start[first], SP_NO_MASK, 0, s, true, pre_seg, pre_row);
    }
    for (int r = 0; r < R; r++) {
      const bool fresh = q_len[r] <= SP_FRESH;
      const int hi = fresh ? ctx_len[r] : ctx_len[r] + q_len[r];
      if (q_len[r] > 0 && hi > shared[r]) add(r, start[r], q_len[r], fresh ? SP_NO_MASK : ctx_len[r], shared[r], hi, false, own_seg, own_row);
      for (int i = 0; i < q_len[r]; i++) {
        SharedToken& t = tokens[start[r] + i];
        t = {};
        t.table = r;
        t.first = ctx_len[r];
        t.fresh = fresh ? i + 1 : 0;
      }
    }
    double all = 0;
    for (const Segment& s : p.segs) all += (p.item_cost + p.tile_cost(s) * s.tiles) * Hkv;
    const double share = std::max(1.0, all / n_ctas);
    double best = 1, cost = -1;
    for (double f = 2.0; f > 0.1; f *= 0.93) {
      const double chunk = std::max(1.0, share * f - p.item_cost);
      const Cut c = p.cut(chunk);
      if (c.parts < 0x7fffffff && (cost < 0 || c.cost < cost)) {
        cost = c.cost;
        best = chunk;
      }
    }
    if (cost < 0) {
      hb_set_error("hb_shared_plan: the partial results of %d rows are too many", T);
      return 0;
    }
    const Cut c = p.cut(best);
    p.deal();
    std::vector<SharedItem> items;
    std::vector<int> ctas;
    int max_rows = 0, masked = 0;
    for (auto& list : p.lists) {
      if (list.empty()) continue;
      ctas.push_back((int)items.size());
      for (auto& it : list) {
        const Segment& s = p.segs[it.first];
        const int h = it.second / s.chunks, k = it.second % s.chunks, rows_of = s.tokens * p.G;
        const int t0 = s.lo / key_tile, a = t0 + (int)((long)s.tiles * k / s.chunks), b = t0 + (int)((long)s.tiles * (k + 1) / s.chunks);
        SharedItem x;
        x.table = s.table;
        x.token = s.token;
        x.tokens = s.tokens;
        x.pos = s.pos;
        x.lo = std::max(s.lo, a * key_tile);
        x.hi = std::min(s.hi, b * key_tile);
        x.head = h;
        x.part = s.base + (h * s.parts + k * (s.parts / s.chunks)) * rows_of;
        items.push_back(x);
        max_rows = std::max(max_rows, rows_of);
        masked |= s.pos != SP_NO_MASK;
      }
    }
    const int n_cta = (int)ctas.size();
    ctas.push_back((int)items.size());
    for (int t = 0; t < T; t++) {
      SharedToken& x = tokens[t];
      if (pre_seg[t] >= 0) {
        const Segment& s = p.segs[pre_seg[t]];
        x.pre_base = s.base + pre_row[t];
        x.pre_n = s.parts;
        x.pre_rows = s.tokens * p.G;
      }
      if (own_seg[t] >= 0) {
        const Segment& s = p.segs[own_seg[t]];
        x.own_base = s.base + own_row[t];
        x.own_n = s.parts;
        x.own_rows = s.tokens * p.G;
      }
    }
    const long off_items = SP_HEADER, off_ctas = off_items + (long)items.size() * 8, off_tokens = (off_ctas + (long)ctas.size() + 3) / 4 * 4,
               ints = off_tokens + (long)T * 12;
    if (ints > 0x7fffffff) {
      hb_set_error("hb_shared_plan: a plan of %ld numbers", ints);
      return 0;
    }
    if (ints > cap) return (int)-ints;
    std::fill(out, out + SP_HEADER, 0);
    out[SP_ITEMS] = (int)items.size();
    out[SP_CTAS] = n_cta;
    out[SP_PARTS] = (int)c.parts;
    out[SP_TOKENS] = T;
    out[SP_MAX_ROWS] = max_rows;
    out[SP_OFF_ITEMS] = (int)off_items;
    out[SP_OFF_CTAS] = (int)off_ctas;
    out[SP_OFF_TOKENS] = (int)off_tokens;
    out[SP_INTS] = (int)ints;
    out[SP_MASKED] = masked;
    static_assert(sizeof(SharedItem) == 32 && sizeof(SharedToken) == 48, "as the offsets have it");
    std::copy(items.begin(), items.end(), (SharedItem*)(out + off_items));
    std::copy(ctas.begin(), ctas.end(), out + off_ctas);
    std::copy(tokens.begin(), tokens.end(), (SharedToken*)(out + off_tokens));
    return (int)ints;
  } catch (const std::exception& e) {
    hb_set_error("hb_shared_plan: %s", e.what());
    return 0;
  }
}
