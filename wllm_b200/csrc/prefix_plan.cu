// The plan of attention over shared prefixes, worked out on the host from the step's block tables: no kernels here.
//
// Requests that hold the same page at the same place of their tables have the same tokens up to its end.  So the tables are walked as a tree: the requests that agree on
// the next page stay together, and every stretch of pages on which a set of two or more agrees is one *segment*, attended to by the rows of all of them; what is left of a
// request's keys is its own segment.  Segments are cut into items, (tile of rows) x (range of keys), one CTA each and key/value head.  How long the ranges are decides
// between SMs without work (long ranges) and results that have to be written and merged (short ones): of a few bounds on what an item may cost the one with the earliest
// estimated end is taken.  The caller says what its kernel takes for a tile of keys, for an item beside them and for a row of results.  Items are listed dearest first, those that read
// the same keys side by side (for the L2).
#include "common.cuh"
#include "prefix_plan.cuh"

#include <algorithm>
#include <cstring>
#include <new>
#include <vector>

namespace {

enum { OUT_TOO_SMALL = 4, PAGES_OUT_OF_RANGE = 7 };

struct Segment { int first, count, key_lo, key_hi; bool own; };       // first, count: its requests in `members`

struct Planner {
    const int* tables;
    long long width;
    int R, ps, align, min_keys;
    std::vector<int> share, cover, members;
    std::vector<Segment> segments;

    int page(int r, int i) const { return tables[r * width + i]; }

    // `set`: requests that agree on all pages in front of `from`; their keys in front of `key` belong to segments.  Beyond DEEPEST branchings requests go on alone (the stack is the caller's).
    static constexpr int DEEPEST = 256;
    void walk(const std::vector<int>& set, int from, int key, int depth) {
        std::vector<int> next;
        for (int r : set)
            if (share[r] > from) next.push_back(r);
        std::stable_sort(next.begin(), next.end(), [&](int a, int b) { return page(a, from) < page(b, from); });
        for (size_t i = 0; i < next.size();) {
            size_t j = i + 1;
            while (j < next.size() && page(next[j], from) == page(next[i], from)) ++j;
            if (j - i >= 2) {
                std::vector<int> group(next.begin() + i, next.begin() + j);
                std::sort(group.begin(), group.end());
                int p = share[group[0]];                   // the first page on which they do not agree, row by row of the tables
                const int* first = tables + group[0] * width;
                for (size_t m = 1; m < group.size(); ++m) {
                    const int* other = tables + group[m] * width;
                    const int most = std::min(p, share[group[m]]);
                    if (most <= from) { p = from; break; }
                    const bool same = memcmp(first + from, other + from, (size_t)(most - from) * sizeof(int)) == 0;
                    p = same ? most : (int)(std::mismatch(first + from, first + most, other + from).first - first);
                }
                int hi = (int)((long long)p * ps / align * align);
                if (hi - key >= min_keys) {
                    segments.push_back({(int)members.size(), (int)group.size(), key, hi, false});
                    members.insert(members.end(), group.begin(), group.end());
                    for (int r : group) cover[r] = hi;
                } else hi = key;
                if (depth < DEEPEST) walk(group, p, hi, depth + 1);
            }
            i = j;
        }
    }
};

struct Tile { int token, tokens, key_lo, key_hi, request; bool own; };
struct Item { int tile, key_lo, key_hi, row, sides, cost; };

long long padded(long long n) { return (n + 3) & ~3ll; }

}  // namespace

// tables [R][width] (pages that hold no key of a request are not looked at), q_len, ctx_len [R] on the host.  rep: query heads a key/value head; tile_rows: rows of an item at
// most; key_tile: keys of a tile, whole tiles make an item's range; align: segments end at multiples of it; min_keys: no shared segment is shorter; pool_pages: one past the largest
// page number; ctas: CTAs that run at once; costs: {a tile of keys, an item beside its tiles; the same two for items of at most `thin` rows; thin; a thousand rows of results and
// kv heads; results that a thin item of several tiles leaves}, in the caller's units; caps: {items, tokens, results, tokens of the batch} that the array is laid out for, zeros: what this plan needs (a captured
// step's array lies at fixed places whatever the batch holds).  out [room]; info [10]: ints used, items, rows, shared keys saved (keys x further holders), most results of a
// token, tiles of rows, tokens of items, results, tiles of rows by tiles of keys, the largest page number (-1: none).
// Returns 0; 2: sizes that make no sense, or more than the caps hold; 4: `room` is too small (info[0] says what is needed); 7: a page number outside the pool.
WLLM_API int wllm_prefix_plan(const int* tables, long long width, int R, const int* q_len, const int* ctx_len, int page_size, int rep, int nkv, int tile_rows, int key_tile, int align,
                              int min_keys, int pool_pages, int ctas, const int* costs, const int* caps, int* out, long long room, long long* info) {
    try {
        if (R < 0 || R > (1 << 20) || width < 0 || page_size < 1 || rep < 1 || nkv < 1 || tile_rows < rep || key_tile < 1 || align < 1 || ctas < 1 || pool_pages < 1) return WLLM_BAD_SIZE;
        Planner p{tables, width, R, page_size, align, min_keys, {}, {}, {}, {}};
        p.share.assign(R, 0);
        p.cover.assign(R, 0);
        std::vector<int> start(R + 1, 0), all;
        long long total = 0;
        for (int r = 0; r < R; ++r) {
            if (q_len[r] < 0 || (q_len[r] > 0 && (ctx_len[r] < q_len[r] || ctx_len[r] > width * page_size))) return WLLM_BAD_SIZE;
            start[r] = (int)total;
            total += q_len[r];
            if (total > (1 << 26)) return WLLM_BAD_SIZE;
            if (q_len[r] == 0) continue;
            p.share[r] = (ctx_len[r] - q_len[r]) / page_size;
            all.push_back(r);
        }
        start[R] = (int)total;
        p.walk(all, 0, 0, 0);
        long long saved = 0;
        for (const Segment& s : p.segments) saved += (long long)(s.count - 1) * (s.key_hi - s.key_lo);
        for (int r : all) {
            p.segments.push_back({(int)p.members.size(), 1, p.cover[r], ctx_len[r], true});
            p.members.push_back(r);
        }
        long long last_page = -1;
        for (const Segment& s : p.segments) {             // (shared pages are looked at once)
            const int* held = tables + p.members[s.first] * width;
            const int end = (int)((s.key_hi + (long long)page_size - 1) / page_size);
            unsigned top = 0;                             // (a number below zero is a large one)
            for (int i = s.key_lo / page_size; i < end; ++i) top = std::max(top, (unsigned)held[i]);
            if (top >= (unsigned)pool_pages) return PAGES_OUT_OF_RANGE;
            if (s.key_hi > s.key_lo) last_page = std::max<long long>(last_page, top);
        }
        // tiles of rows: whole tokens of a segment's requests, one behind the other
        const int per_tile = tile_rows / rep;
        std::vector<Tile> tiles;
        std::vector<int> tokens, at;              // of all segments, and their positions
        for (const Segment& s : p.segments) {
            const int first = (int)tokens.size();
            for (int m = 0; m < s.count; ++m) {
                const int r = p.members[s.first + m];
                for (int t = 0; t < q_len[r]; ++t) {
                    tokens.push_back(start[r] + t);
                    at.push_back(ctx_len[r] - q_len[r] + t);
                }
            }
            const int n = (int)tokens.size() - first;
            for (int t = 0; t < n; t += per_tile) {
                const int count = std::min(per_tile, n - t);
                tiles.push_back({first + t, count, s.key_lo, s.own ? at[first + t + count - 1] + 1 : s.key_hi, p.members[s.first], s.own});
            }
            if (tokens.size() > (1u << 28)) return WLLM_BAD_SIZE;
        }
        // what an item may cost at most: tiles by their keys, thin ones apart
        auto keys_of = [&](const Tile& t) { return (t.key_hi - t.key_lo + key_tile - 1) / key_tile; };
        auto is_thin = [&](const Tile& t) { return t.tokens * rep <= costs[4] ? 1 : 0; };
        struct Alike { int keys, thin, count; long long rows; };
        std::vector<Alike> alike;
        {
            int longest = 0;
            for (const Tile& t : tiles) longest = std::max(longest, keys_of(t));
            std::vector<int> place(2 * (longest + 1), -1);
            for (const Tile& t : tiles) {
                int& at = place[2 * keys_of(t) + is_thin(t)];
                if (at < 0) {
                    at = (int)alike.size();
                    alike.push_back({keys_of(t), is_thin(t), 0, 0});
                }
                ++alike[at].count;
                alike[at].rows += (long long)t.tokens * rep;
            }
        }
        auto parts_of = [&](int keys, int thin, int most) { return std::min(keys, std::max(1, (int)(((long long)keys * costs[2 * thin] + most - 1) / most))); };
        const long long most_items = caps[0] > 0 ? caps[0] : (1 << 22), most_results = caps[2] > 0 ? caps[2] : (1 << 28);
        int dearest = 1;
        for (const Alike& a : alike) dearest = (int)std::min<long long>(std::max<long long>(dearest, (long long)a.keys * costs[2 * a.thin]), 1 << 30);
        // The CTAs take pairs off the sorted list to and fro: CTA b gets the b-th of the first `ctas`, the b-th from behind of the next, and so on.  The end is that of the first CTA, of the last, or of
        // those where the list's last round begins or stops; with many rounds none is far from the mean.  (With the mean and half of the dearest item in its place for any number of rounds, 24 portions on
        // 6,000 keys became 208 long items for 148 SMs, 64.9 us a layer; 57.0 so, and 96 tokens on 32,768 keys 58.9 and 55.4.)
        struct Run { int tiles_cost; double cost; long long count; };
        std::vector<Run> runs;
        auto end_of = [&](long long pairs, double all, double top) {
            const long long rounds = (pairs + ctas - 1) / ctas, rest = pairs % ctas;
            if (rounds <= 1) return top;
            if (rounds > 24) return all / ctas + 0.5 * top;
            std::sort(runs.begin(), runs.end(), [](const Run& a, const Run& b) { return a.tiles_cost > b.tiles_cost; });
            const bool back = !(rounds & 1);               // the last round runs from the last CTA to the first
            const long long edges[4] = {0, ctas - 1, back ? ctas - rest : rest - 1, back ? ctas - rest - 1 : rest};
            double end = 0;
            for (int e = 0; e < (rest ? 4 : 2); ++e) {
                const long long b = edges[e];
                double load = 0;
                long long before = 0;
                size_t run = 0;
                for (long long r = 0; r < rounds; ++r) {
                    const long long rank = r * ctas + ((r & 1) ? ctas - 1 - b : b);
                    while (run < runs.size() && rank >= before + runs[run].count) before += runs[run++].count;
                    if (run == runs.size()) break;
                    load += runs[run].cost;
                }
                end = std::max(end, load);
            }
            return end;
        };
        double best = 0;
        int most = 0;
        for (long long m = std::max(1, std::min(costs[0], costs[2]));; m = m * 6 / 5 + 1) {
            const int bound = (int)std::min<long long>(m, dearest);
            long long n = 0, results_rows = 0;
            double all = 0, top = 0;
            runs.clear();
            for (const Alike& a : alike) {
                const int parts = parts_of(a.keys, a.thin, bound), least = a.keys / parts, longer = a.keys % parts, tile = costs[2 * a.thin], item = costs[2 * a.thin + 1];
                if (longer) runs.push_back({(least + 1) * tile, (double)(least + 1) * tile + item, (long long)longer * a.count * nkv});
                runs.push_back({least * tile, (double)least * tile + item, (long long)(parts - longer) * a.count * nkv});
                n += (long long)parts * a.count;
                results_rows += parts * a.rows * (a.thin && a.keys > parts ? costs[6] : 1);
                all += ((double)a.keys * costs[2 * a.thin] + (double)parts * costs[2 * a.thin + 1]) * a.count;
                top = std::max(top, (double)((a.keys + parts - 1) / parts) * costs[2 * a.thin] + costs[2 * a.thin + 1]);
            }
            const double end = end_of(n * nkv, all * nkv, top) + (double)results_rows * nkv * costs[5] / 1000;
            if (n <= most_items && results_rows / rep <= most_results && (most == 0 || end < best * 0.99)) {
                best = end;
                most = bound;
            }
            if (bound == dearest) break;
        }
        if (most == 0 && !tiles.empty()) return WLLM_BAD_SIZE;
        // items: of the tiles that follow one another with the same keys, range by range
        std::vector<Item> items;
        long long rows = 0, results = 0;
        for (size_t i = 0; i < tiles.size();) {
            size_t j = i + 1;
            while (j < tiles.size() && !tiles[i].own && !tiles[j].own && is_thin(tiles[j]) == is_thin(tiles[i]) && tiles[j].request == tiles[i].request && tiles[j].key_lo == tiles[i].key_lo && tiles[j].key_hi == tiles[i].key_hi) ++j;
            const int k = keys_of(tiles[i]), parts = parts_of(k, is_thin(tiles[i]), most);
            for (int s = 0; s < parts; ++s) {
                const int from = (int)((long long)k * s / parts), to = (int)((long long)k * (s + 1) / parts);
                for (size_t t = i; t < j; ++t) {
                    const int sides = is_thin(tiles[t]) && to - from > 1 ? costs[6] : 1;
                    items.push_back({(int)t, tiles[i].key_lo + from * key_tile, std::min(tiles[i].key_hi, tiles[i].key_lo + to * key_tile), (int)rows, sides, (to - from) * costs[2 * is_thin(tiles[t])]});
                    rows += (long long)tiles[t].tokens * rep * sides;
                    results += tiles[t].tokens * sides;
                    if (rows > 0x7fffffff / nkv) return WLLM_BAD_SIZE;
                }
            }
            i = j;
        }
        // results by token, in the order in which segments were found: ascending keys
        std::vector<int> starts(total + 1, 0), listed(results);
        for (const Item& it : items)
            for (int t = 0; t < tiles[it.tile].tokens; ++t) starts[tokens[tiles[it.tile].token + t] + 1] += it.sides;
        int most_listed = 0;
        for (long long t = 0; t < total; ++t) {
            most_listed = std::max(most_listed, starts[t + 1]);
            starts[t + 1] += starts[t];
        }
        {
            std::vector<int> next(starts.begin(), starts.end() - 1);
            for (const Item& it : items)
                for (int t = 0; t < tiles[it.tile].tokens; ++t)
                    for (int side = 0; side < it.sides; ++side) listed[next[tokens[tiles[it.tile].token + t]]++] = it.row + (side * tiles[it.tile].tokens + t) * rep;
        }
        std::stable_sort(items.begin(), items.end(), [](const Item& a, const Item& b) { return a.cost > b.cost; });

        const long long need[4] = {(long long)items.size(), (long long)tokens.size(), results, total};
        long long cap[4];
        for (int i = 0; i < 4; ++i) {
            cap[i] = caps[i] > 0 ? caps[i] : need[i];
            if (need[i] > cap[i]) return WLLM_BAD_SIZE;
        }
        const long long at_items = PLAN_HEADER, at_tokens = at_items + padded(cap[0] * PLAN_ITEM), at_starts = at_tokens + padded(cap[1] * 2), at_results = at_starts + padded(cap[3] + 1),
                        at_positions = at_results + padded(cap[2]), used = at_positions + padded(cap[3]);
        info[0] = used; info[1] = need[0]; info[2] = rows; info[3] = saved; info[4] = most_listed; info[5] = (long long)tiles.size(); info[6] = need[1]; info[7] = results;
        info[8] = 0;
        for (const Alike& a : alike) info[8] += (long long)a.keys * a.count;
        info[9] = last_page;
        if (used > 0x7fffffff) return WLLM_BAD_SIZE;
        if (used > room) return OUT_TOO_SMALL;
        std::fill(out, out + used, 0);
        std::fill(out + at_positions + total, out + at_positions + cap[3], -1);      // rows behind the last token: passed by
        out[PLAN_ITEMS] = (int)need[0]; out[PLAN_TOKENS] = (int)total; out[PLAN_AT_ITEMS] = (int)at_items; out[PLAN_AT_TOKENS] = (int)at_tokens;
        out[PLAN_AT_STARTS] = (int)at_starts; out[PLAN_AT_RESULTS] = (int)at_results; out[PLAN_AT_POSITIONS] = (int)at_positions; out[PLAN_ROWS] = (int)rows;
        for (size_t i = 0; i < items.size(); ++i) {
            const Tile& t = tiles[items[i].tile];
            int* o = out + at_items + i * PLAN_ITEM;
            o[ITEM_TOKEN] = t.token; o[ITEM_TOKENS] = t.tokens; o[ITEM_KEY_LO] = items[i].key_lo; o[ITEM_KEY_HI] = items[i].key_hi;
            o[ITEM_REQUEST] = t.request; o[ITEM_OWN] = t.own ? 1 : 0; o[ITEM_ROW] = items[i].row;
            bool follow = true;
            for (int j = 1; j < t.tokens && follow; ++j) follow = tokens[t.token + j] == tokens[t.token] + j;
            o[ITEM_FIRST] = follow ? tokens[t.token] : -1;
        }
        for (size_t i = 0; i < tokens.size(); ++i) {
            out[at_tokens + 2 * i] = tokens[i];
            out[at_tokens + 2 * i + 1] = at[i];
        }
        for (long long t = 0; t <= cap[3]; ++t) out[at_starts + t] = starts[std::min(t, total)];     // (tokens past the last have no results)
        std::copy(listed.begin(), listed.end(), out + at_results);
        for (int r = 0; r < R; ++r)
            for (int t = 0; t < q_len[r]; ++t) out[at_positions + start[r] + t] = ctx_len[r] - q_len[r] + t;
        return WLLM_OK;
    } catch (const std::bad_alloc&) {
        return WLLM_BAD_SIZE;
    }
}
