// The plan of a step's shared-prefix attention, made on the host from the lengths alone and used by every layer of the step.
//
// A group's shared range and a request's own range are SEGMENTS: some rows against a range of keys. A segment's keys are cut into equal
// chunks, an item is (chunk, kv head, up to tile_tokens rows), and each CTA gets a list of items: the shared items in the order of their keys,
// so that the CTAs at work at one time read the same tiles (once from memory, then from L2), each to the CTA with the least work so
// far, then the requests' own, longest first. The number of keys in a chunk is the one among a few multiples of an even share whose longest CTA, and whose
// partial results, cost least.
#include "common.cuh"
#include "shared_plan.h"

#include <algorithm>
#include <exception>
#include <queue>
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
  int Hkv, G, key_tile, n_ctas, narrow_tokens;
  double item_cost, part_cost;
  std::vector<Segment> segs;
  std::vector<std::vector<std::pair<int, int>>> lists;   // a CTA's (segment, head * chunks + chunk)

  int parts_of(const Segment& s, int chunks) const { return chunks * (s.tokens <= narrow_tokens ? 2 : 1); }
  // Cuts the segments into chunks of at most `len` tiles and gives the items to the CTAs.
  Cut cut(int len, bool keep) {
    Cut c;
    typedef std::pair<double, int> Load;
    std::priority_queue<Load, std::vector<Load>, std::greater<Load>> q;
    for (int i = 0; i < n_ctas; i++) q.push(Load(0.0, i));
    if (keep) lists.assign(n_ctas, {});
    double longest = 0;
    auto give = [&](int s, int item, double cost) {
      Load l = q.top();
      q.pop();
      l.first += cost;
      longest = std::max(longest, l.first);
      if (keep) lists[l.second].push_back({s, item});
      q.push(l);
    };
    std::vector<int> own, shared;
    int most = 0;
    for (size_t i = 0; i < segs.size(); i++) {
      Segment& s = segs[i];
      s.chunks = (s.tiles + len - 1) / len;
      s.parts = parts_of(s, s.chunks);
      s.base = (int)std::min<long>(c.parts, 0x7fffffff);
      c.parts += (long)Hkv * s.parts * s.tokens * G;
      (s.shared ? shared : own).push_back((int)i);
      if (s.shared) most = std::max(most, s.chunks);
    }
    for (int k = 0; k < most; k++)
      for (int h = 0; h < Hkv; h++)
        for (int i : shared)
          if (k < segs[i].chunks) give(i, h * segs[i].chunks + k, item_cost + double(segs[i].tiles) / segs[i].chunks);
    std::stable_sort(own.begin(), own.end(), [&](int a, int b) { return (long)segs[a].tiles * segs[b].chunks > (long)segs[b].tiles * segs[a].chunks; });
    for (int i : own)
      for (int u = 0; u < Hkv * segs[i].chunks; u++) give(i, u, item_cost + double(segs[i].tiles) / segs[i].chunks);
    c.cost = longest + part_cost * c.parts;
    return c;
  }
};

}  // namespace

// q_len, ctx_len [R]; groups [n_groups][3]: first request, requests, shared tokens. out: SP_HEADER ints, then items, each CTA's first item (one more
// for the end), tokens; returns the ints that were written, or, where `cap` is too small, minus the number that is needed; 0 with a message in
// hb_last_error for lengths that make no plan. tile_tokens: rows of q in an item; narrow_tokens: items of at most so many rows leave two
// parts (their key tiles go to two chains in turn), 0: none do.
HB_EXPORT int hb_shared_plan(const int* q_len, const int* ctx_len, int R, const int* groups, int n_groups, int Hq, int Hkv, int tile_tokens,
                             int narrow_tokens, int key_tile, int n_ctas, float item_cost, float part_cost, int* out, int cap) {
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
    p.part_cost = part_cost;
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
    long tiles = 0, longest = 1;
    for (const Segment& s : p.segs) {
      tiles += (long)s.tiles * Hkv;
      longest = std::max<long>(longest, s.tiles);
    }
    const double share = std::max(1.0, double(tiles) / n_ctas);
    int best = 1;
    double cost = -1;
    for (double f : {1.0, 1.1, 1.25, 2.0, 0.75, 0.5, 0.4, 0.34, 0.25, 4.0}) {
      const int len = (int)std::max(1.0, std::min(double(longest), share * f + 0.999));
      const Cut c = p.cut(len, false);
      if (c.parts < 0x7fffffff && (cost < 0 || c.cost < cost)) {
        cost = c.cost;
        best = len;
      }
    }
    if (cost < 0) {
      hb_set_error("hb_shared_plan: the partial results of %d rows are too many", T);
      return 0;
    }
    const Cut c = p.cut(best, true);
    std::vector<SharedItem> items;
    std::vector<int> ctas;
    int max_rows = 0;
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
