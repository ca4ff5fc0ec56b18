// Host-side check of how tt_shared_prefix_attention is cut into CTAs (tt_prefix_plan.cuh): over the CTAs of the
// prefix pass every (kv head, row tile) meets every key tile exactly once, in spans that are not empty, each span has
// partial slots of its own inside the workspace, and the join finds for each row exactly the slots that hold its
// partials.  Shapes come on stdin (rows, query heads, kv heads, head_dim, prefix_len, page size, table width); a line
// with each shape's plan goes out, then random shapes are checked.  Built with nvcc as a host program by
// tests/test_prefix_plan_cpu.py (no GPU needed).
#include <cstdio>
#include <map>
#include <set>
#include <vector>

#include "../tritiercache_b200/csrc/tt_prefix_plan.cuh"

using namespace tt;

static unsigned long long rng_state = 88172645463325252ull;
static int rnd(int n) {  // xorshift64, [0, n)
    rng_state ^= rng_state << 13;
    rng_state ^= rng_state >> 7;
    rng_state ^= rng_state << 17;
    return (int)(rng_state % (unsigned long long)(n > 0 ? n : 1));
}

struct Seen {
    int spans = 0, units = 0;  // most spans and most kv heads or row tiles of a CTA
};

static const char* check(const PrefixParams& p, Seen* seen) {
    const tt_shared_prefix_args& a = p.a;
    if (p.splits < 1 || (p.walk_prefix && p.join != (p.splits > 1)) || (!p.walk_prefix && !p.join)) return "splits or join";
    if (p.walk_prefix) return nullptr;
    if (p.tile_rows != 128 && p.tile_rows != 256) return "tile rows";
    if (p.tile_rows == 128 && p.row_tiles != 1) return "several row tiles of 128";
    const int groups = prefix_groups(p);
    const bool pair = p.tile_rows == 256;
    if ((long long)groups * p.lanes > kSms) return "more CTAs than SMs";
    std::vector<char> met((size_t)a.num_kv_heads * p.row_tiles * p.kv_tiles, 0);
    std::map<long long, std::pair<int, int>> slots;  // slot pair -> kv head, row tile
    const char* bad = nullptr;
    for (int g = 0; g < groups && !bad; ++g)
        for (int l = 0; l < p.lanes && !bad; ++l) {
            int spans = 0;
            std::set<int> units;
            prefix_spans(p, g, l, [&](int kvh, int tile, long long at, int k0, int n) {
                ++spans;
                units.insert(kvh * p.row_tiles + tile);
                if (kvh < 0 || kvh >= a.num_kv_heads || tile < 0 || tile >= p.row_tiles || n < 1 || k0 < 0 || k0 + n > p.kv_tiles)
                    bad = "a span outside the problem";
                else if (at < 0 || 2 * at + 1 >= (long long)prefix_slots(p)) bad = "a slot outside the workspace";
                else if (!slots.emplace(at, std::make_pair(kvh, tile)).second) bad = "two spans in one slot";
                for (int k = k0; k < k0 + n && !bad; ++k)
                    if (met[((size_t)kvh * p.row_tiles + tile) * p.kv_tiles + k]++) bad = "a key tile met twice";
                return !bad;
            });
            if (!spans) bad = "a CTA without work";
            if (spans > seen->spans) seen->spans = spans;
            if ((int)units.size() > seen->units) seen->units = (int)units.size();
        }
    if (bad) return bad;
    for (char m : met)
        if (!m) return "a key tile not met";
    std::map<std::pair<int, int>, int> spans_of;
    for (const auto& s : slots) ++spans_of[s.second];
    for (int i = 0; i < 400; ++i) {
        const int r = i == 0 ? 0 : i == 1 ? a.num_rows - 1 : rnd(a.num_rows), head = i == 0 ? 0 : i == 1 ? a.num_q_heads - 1 : rnd(a.num_q_heads);
        const int kvh = head / p.group, m = r * p.group + head % p.group, tile = m / p.tile_rows;
        const PrefixPartials got = prefix_partials(p, r, head);
        // a 128-row tile's partials lie in both slots of a span, a 256-row tile's in the half's
        if (got.n != spans_of[{kvh, tile}] * (pair ? 1 : 2)) return "the join misses partials";
        for (int k = 0; k < got.n; ++k) {
            const long long row = got.first + k * got.step, slot = row / 128;
            if (row % 128 != m % 128 || (pair && slot % 2 != (m % 256) / 128)) return "the join reads another row";
            const auto s = slots.find(slot / 2);
            if (s == slots.end() || s->second != std::make_pair(kvh, tile)) return "the join reads another tile";
        }
    }
    return nullptr;
}

static PrefixParams plan(int R, int nq, int nkv, int hd, int prefix, int P, int W) {
    tt_shared_prefix_args a = {};
    a.num_rows = R, a.num_q_heads = nq, a.num_kv_heads = nkv, a.head_dim = hd, a.prefix_len = prefix, a.page_size = P, a.table_width = W;
    a.scale = 0.1f;
    return plan_prefix(a);
}

int main() {
    int s[7];
    while (std::scanf("%d %d %d %d %d %d %d", s, s + 1, s + 2, s + 3, s + 4, s + 5, s + 6) == 7) {
        const PrefixParams p = plan(s[0], s[1], s[2], s[3], s[4], s[5], s[6]);
        Seen seen;
        if (const char* bad = check(p, &seen)) {
            std::printf("FAIL %s: %d %d %d %d %d\n", bad, s[0], s[1], s[2], s[3], s[4]);
            return 1;
        }
        std::printf("plan %d %d %d %d %d %d %d %d %zu\n", p.walk_prefix, p.tile_rows, p.row_tiles, p.lanes, p.spans, p.per, seen.spans,
                    seen.units, prefix_workspace(p));
    }
    int crossed[2] = {0, 0};
    for (int it = 0; it < 6000; ++it) {
        const int nkv = 1 + rnd(it % 3 ? 8 : 160), group = 1 + rnd(12), R = 1 + rnd(it % 2 ? 40 : 700), hd = rnd(2) ? 64 : 128;
        const int prefix = 1 + rnd(it % 5 ? 3000 : 40000), P = 16 << rnd(4), W = rnd(50);
        const PrefixParams p = plan(R, nkv * group, nkv, hd, prefix, P, W);
        Seen seen;
        if (const char* bad = check(p, &seen)) {
            std::printf("FAIL %s: %d %d %d %d %d\n", bad, R, nkv * group, nkv, hd, prefix);
            return 1;
        }
        if (seen.units > 1) ++crossed[p.tile_rows == 256];
    }
    std::printf("ok %d %d\n", crossed[0], crossed[1]);
    return crossed[0] && crossed[1] ? 0 : 1;
}
