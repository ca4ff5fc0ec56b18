// tt_prefix_plan.cuh -- how tt_shared_prefix_attention is cut into CTAs: the plan of a call, the spans of key
// tiles of each CTA of the prefix pass, and the partials that the join finds for a row.  Host and device.
#pragma once
#include <limits.h>

#include "tt_common.cuh"

namespace tt {

constexpr int kRowWarps = 4;     // warps of a CTA of the rows' pass
constexpr int kGroup = 16;       // tokens per warp step
constexpr int kPsTile = 128;     // prefix pass: keys per tile, rows per accumulator
constexpr float kLog2e = 1.4426950408889634f;

struct PrefixParams {
    tt_shared_prefix_args a;
    float scale_log2;            // scale * log2(e)
    long long patience;          // clocks that a wait may take before the CTA gives up
    int page_shift;
    int group;                   // query heads per kv head
    int head_tiles;              // tiles of 8*NB query heads per kv head
    int splits;                  // CTAs per row and head tile in the rows' pass
    // prefix pass: a unit is a kv head and one tile of tile_rows rows of its (row, head of the group) matrix, or
    // with lanes = row_tiles all its tiles at once, one CTA of a group of `lanes` each.  The flattened (unit, key
    // tile) list is cut into spans of `per` for the groups: `spans` a unit, or, with spans = 0, across units.
    // A span's partials are in slots 2 ((group + unit) lanes + lane) + t of 128 rows: t is the half of a 256-row
    // tile, or even and odd key tiles of a 128-row one
    int walk_prefix;             // 1: no prefix pass, the rows' pass reads the prefix too
    int tile_rows, row_tiles, lanes, units, kv_tiles, per, spans;
    float* part_o;               // [slot][128][hd]
    float2* part_ml;             // [slot][128] (m in log2 units, l)
    int join;                    // 1: the rows' pass leaves partials [splits][num_rows][num_q_heads] for k_prefix_join; 0: outputs
    float* own_o;
    float2* own_ml;
};

constexpr int kSms = 148;
constexpr long long kWalk = 1 << 23;
constexpr int kCross = 4;  // measured: 7 tiles in 30 us, 7 in two spans in 40 (384 rows of heads on 8k)

inline int prefix_groups(const PrefixParams& p) {
    return p.spans ? p.units * p.spans : (int)(((long long)p.units * p.kv_tiles + p.per - 1) / p.per);
}
inline size_t prefix_slots(const PrefixParams& p) {
    return p.walk_prefix ? 0 : 2 * ((size_t)prefix_groups(p) + (size_t)p.units) * p.lanes;
}
inline size_t own_slots(const PrefixParams& p) { return p.join ? (size_t)p.splits * p.a.num_rows * p.a.num_q_heads : 0; }

inline PrefixParams plan_prefix(const tt_shared_prefix_args& a) {
    PrefixParams p = {};
    p.a = a;
    p.scale_log2 = a.scale * kLog2e;
    p.group = a.num_q_heads / a.num_kv_heads;
    while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
    p.head_tiles = p.group <= 8 ? 1 : (p.group + 15) / 16;
    // One row has nobody to share with, and reading a short prefix again for each of a few rows, from L2, costs less
    // than a pass of its own and its partials (32/8 heads of 128: 8 rows on 512 tokens 9.5 against 12.5 us, on 1024
    // 11.5 against 12.7, on 2048 15.2 against 13.0; 2 rows on 4096 11.4 against 12.6; 16 rows on 512 10.9 against 14.0).
    // The prefix pass takes its maxima before the scale, so the scale must not turn them round.
    const long long again = (long long)a.num_rows * a.prefix_len * a.num_kv_heads * p.head_tiles * a.head_dim;
    p.walk_prefix = a.num_rows < 2 || again <= kWalk || !(a.scale > 0.f);
    if (!p.walk_prefix) {
        const int rows = a.num_rows * p.group;
        p.tile_rows = rows > kPsTile ? 2 * kPsTile : kPsTile;
        p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
        p.kv_tiles = (a.prefix_len + kPsTile - 1) / kPsTile;
        // CTA groups over all row tiles of a kv head, unless they would leave more than a tenth of the SMs idle
        p.lanes = kSms / p.row_tiles * p.row_tiles * 10 >= kSms * 9 ? p.row_tiles : 1;
        p.units = a.num_kv_heads * (p.row_tiles / p.lanes);
        const int groups = kSms / p.lanes;
        // Equal spans across units use every SM, but a CTA whose span crosses a unit's border starts and ends twice,
        // which costs it about kCross key tiles; whole spans per unit may leave SMs idle.
        p.per = (int)(((long long)p.units * p.kv_tiles + groups - 1) / groups);
        if (p.units <= groups) {
            const int whole = (p.kv_tiles + groups / p.units - 1) / (groups / p.units);
            if (whole <= p.per + kCross) p.per = whole, p.spans = 1;
        }
        // A span of one key tile leaves as many bytes of partials as two, and a 128-row tile's second accumulator
        // without work (64 rows of 32 heads on 2k: 27.8 -> 23.2 us; at least four tiles: 25.5).
        if (p.per < 2) p.per = 2;
        if (p.spans) p.spans = (p.kv_tiles + p.per - 1) / p.per;
    }
    // CTAs of the rows' pass per row and head tile: two for each SM in all, if that leaves a warp two groups
    const long long tokens = (long long)a.table_width * a.page_size + (p.walk_prefix ? a.prefix_len : 0);
    const long long units = (long long)a.num_rows * a.num_kv_heads * p.head_tiles;
    const long long most = tokens / (kRowWarps * kGroup * 2), fit = 2 * kSms / units;
    p.splits = (int)(most < fit ? most : fit);
    if (p.splits < 1) p.splits = 1;
    p.join = p.splits > 1 || !p.walk_prefix;
    return p;
}

inline size_t prefix_workspace(const PrefixParams& p) {
    return (prefix_slots(p) * kPsTile + own_slots(p)) * (p.a.head_dim * sizeof(float) + sizeof(float2));
}

// The spans of a CTA of the prefix pass (CTA `lane` of `group`): fn(kv head, row tile, slot, first key tile, key tiles)
// for each, until fn returns false.
// p.spans > 0: so many spans a unit, none crosses units; else the flattened list in spans of p.per.
template <typename F>
__host__ __device__ __forceinline__ void prefix_spans(const PrefixParams& p, int group, int lane, F fn) {
    long long f, end;
    if (p.spans) {
        const long long u = group / p.spans;
        f = u * p.kv_tiles + (long long)(group % p.spans) * p.per;
        end = f + p.per < (u + 1) * p.kv_tiles ? f + p.per : (u + 1) * p.kv_tiles;
    } else {
        f = (long long)group * p.per;
        const long long all = (long long)p.units * p.kv_tiles;
        end = f + p.per < all ? f + p.per : all;
    }
    while (f < end) {
        const int u = (int)(f / p.kv_tiles), k0 = (int)(f % p.kv_tiles);
        const int n = end - f < p.kv_tiles - k0 ? (int)(end - f) : p.kv_tiles - k0;
        const int kvh = p.lanes > 1 ? u : u / p.row_tiles, tile = p.lanes > 1 ? lane : u % p.row_tiles;
        if (!fn(kvh, tile, (long long)(group + u) * p.lanes + lane, k0, n)) return;
        f += n;
    }
}

// The prefix pass's partials of row r and query head `head`: n of them, `step` rows apart from row `first` of the
// partials (slots of 128 rows).
struct PrefixPartials {
    long long first, step;
    int n;
};
__host__ __device__ __forceinline__ PrefixPartials prefix_partials(const PrefixParams& p, int r, int head) {
    const int kvh = head / p.group, row = r * p.group + head % p.group;
    const int tile = row / p.tile_rows, in = row % p.tile_rows, lane = p.lanes > 1 ? tile : 0;
    const bool pair = p.tile_rows == 256;
    const int u = p.lanes > 1 ? kvh : kvh * p.row_tiles + tile;
    const int g0 = p.spans ? u * p.spans : u * p.kv_tiles / p.per;
    const int g1 = p.spans ? g0 + p.spans - 1 : ((u + 1) * p.kv_tiles - 1) / p.per;
    // even and odd key tiles are neighbours (!pair has one row tile, so one lane)
    const long long first = (2 * ((long long)(g0 + u) * p.lanes + lane) + (pair ? in >> 7 : 0)) * 128 + (in & 127);
    const long long step = (pair ? 2 * p.lanes : 1) * 128;
    const int n = (g1 - g0 + 1) * (pair ? 1 : 2);
    return PrefixPartials{first, step, n};
}

}  // namespace tt
