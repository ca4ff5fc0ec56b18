// tt_prefix_rows.cuh -- the pass of tt_shared_prefix_attention over each row's own pages, which also
// joins what the prefix pass left.
//
// One cluster of C CTAs per (row, kv head, tile of up to 8*NB query heads).  Its 4*C warps take the row's
// tokens in groups of 16 (a group never crosses a page), warp w groups w, w+4C, ...; each warp keeps its
// own cp.async pipeline of K and V groups, so no warp waits for another before the end.  Per group, with
// mma.sync m16n8k16 and tokens along M, because a row has few query heads and 16 tokens:
//   S^T[16 x 8] = K[16 x hd] Q^T[hd x 8]         (K by ldmatrix, Q^T in registers)
//   P^T = 2^(S^T - m), transposed in registers (movmatrix) into the second product's B operand
//   O^T[hd x 8] += V^T[hd x 16] P^T[16 x 8]       (V by transposing ldmatrix)
// m is a reference, not the maximum: it is raised (and O, l rescaled) only when a logit exceeds it by
// kSlack, so the cross-lane maximum and the rescale run once or twice a row instead of once a group;
// weights stay below 2^kSlack and every sum is float32.
// At the end the warps' (m, l, O) meet in shared memory, the CTAs' through the cluster's, and the prefix
// pass's partials from the workspace: one output, no further launch.
//
// Bound: HBM (the row's K and V are read once, by one cluster).
#pragma once
#include <cuda_bf16.h>

#include "tt_common.cuh"
#include "tt_launch.cuh"

namespace tt {

constexpr float kSlack = 8.f;    // log2 units a logit may exceed the reference before it is raised
constexpr int kRowWarps = 4;
constexpr int kGroup = 16;       // tokens per warp step

struct PrefixParams {
    tt_shared_prefix_args a;
    float scale_log2;            // scale * log2(e)
    int page_shift;
    int group;                   // query heads per kv head
    int head_tiles;              // tiles of 8*NB query heads per kv head
    // prefix pass: units of (kv head, tile of tile_rows rows of (row, head of the group)), the flattened
    // (unit, key tile) list cut into spans of `per` for the CTAs; a span's partials are in slots
    // 2 (cta + unit) + t of 128 rows: t the half of a 256-row tile, or even and odd key tiles of a 128-row one
    int walk_prefix;             // 1: no prefix pass, the rows' pass reads the prefix too
    int tile_rows, row_tiles, kv_tiles, per;
    float* part_o;               // [slot][128][hd]
    float2* part_ml;             // [slot][128] (m in log2 units, l)
};

template <typename T> __device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two floats rounded to T, and the rounded values.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 16 bytes to shared memory, zeros when !live (nothing is read then).
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// A running join of partials (m, l, O): adds one of weight 2^(m - M).
struct Join {
    float M = -INFINITY, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(float2 ml, float4 x) {
        // an empty partial (m = -inf) has l = 0 and must not bring 2^(-inf + inf); a NaN l passes through
        if (ml.x == -INFINITY && ml.y == 0.f) return;
        const float n = fmaxf(M, ml.x), f = M == -INFINITY ? 0.f : fast_exp2(M - n);
        const float w = ml.x == -INFINITY ? 1.f : fast_exp2(ml.x - n);
        L = L * f + ml.y * w;
        o.x = o.x * f + x.x * w;
        o.y = o.y * f + x.y * w;
        o.z = o.z * f + x.z * w;
        o.w = o.w * f + x.w * w;
        M = n;
    }
};

template <int HD, int NB> constexpr int row_out_bytes() { return 8 * NB * HD * 4 + 8 * NB * 8; }  // one warp's O and (m, l)
template <int HD, int NB, int ST> constexpr int row_warp_bytes() {
    return ST * 2 * kGroup * HD * 2 > row_out_bytes<HD, NB>() ? ST * 2 * kGroup * HD * 2 : row_out_bytes<HD, NB>();
}

template <typename T, int HD, int NB, int ST>
__global__ void __launch_bounds__(kRowWarps * 32) k_prefix_rows(const PrefixParams p) {
    extern __shared__ __align__(128) unsigned char sm[];
    constexpr int KS = HD / 16, CH = HD / 8;          // k-steps, 16-byte chunks of a token's row
    constexpr int kTile = kGroup * HD * 2;            // bytes of a K (or V) group
    constexpr int kWarp = row_warp_bytes<HD, NB, ST>();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), C = cluster_size();
    const int r = blockIdx.x / C;
    const int kvh = blockIdx.y / p.head_tiles, h0 = (blockIdx.y % p.head_tiles) * 8 * NB;
    const int heads = min(8 * NB, p.group - h0);      // query heads of this tile
    const tt_shared_prefix_args& a = p.a;

    const int seq = a.row_seq ? a.row_seq[r] : r;
    if (seq < 0) {  // padding; the wait keeps this grid from ending before the prefix pass
        pdl_wait();
        return;
    }
    int len = a.row_lens[r];
    bool bad = false;
    if (seq >= a.num_tables || len < 0 || ((long long)len + a.page_size - 1) >> p.page_shift > a.table_width) {
        bad = true;
        len = 0;
    }
    const int pre_groups = p.walk_prefix ? (a.prefix_len + kGroup - 1) / kGroup : 0;
    const int groups = pre_groups + (len + kGroup - 1) / kGroup;
    const int* own = a.tables + (long long)(bad ? 0 : seq) * a.table_stride;
    const int step = kRowWarps * C, g0 = rank * kRowWarps + warp;
    const int gpp = p.page_shift - 4;                 // log2 groups per page

    // first token of group g, its page (-1 none) and the tokens that count
    const auto page_of = [&](int g) {
        if (g >= groups) return -1;
        return g < pre_groups ? a.prefix_table[g >> gpp] : own[(g - pre_groups) >> gpp];
    };
    const uint32_t base = smem_addr(sm) + warp * kWarp;
    const T* kp = static_cast<const T*>(a.k) + (long long)kvh * a.k_head_stride;
    const T* vp = static_cast<const T*>(a.v) + (long long)kvh * a.v_head_stride;
    const auto issue = [&](int g, int page, int stage) {
        if (g < groups) {
            const int t0 = (g < pre_groups ? g : g - pre_groups) * kGroup;
            const int n = (g < pre_groups ? a.prefix_len : len) - t0;
            const bool ok = page >= 0 && page < a.num_pages;
            bad |= !ok;
            const long long pg = ok ? page : 0;
            const int in_page = t0 & (a.page_size - 1);
            const T* ks = kp + pg * a.k_page_stride + in_page * a.k_token_stride;
            const T* vs = vp + pg * a.v_page_stride + in_page * a.v_token_stride;
            const uint32_t kd = base + stage * 2 * kTile, vd = kd + kTile;
#pragma unroll
            for (int i = 0; i < kGroup * CH / 32; ++i) {
                const int t = (i * 32 + lane) / CH, c = (i * 32 + lane) % CH;
                const bool live = ok && t < n;
                const uint32_t off = t * HD * 2 + ((c ^ (t & 7)) << 4);
                cp16(kd + off, ks + (live ? t * a.k_token_stride + c * 8 : 0), live);
                cp16(vd + off, vs + (live ? t * a.v_token_stride + c * 8 : 0), live);
            }
        }
        cp_commit();
    };

    int g_issue = g0, page = page_of(g0);
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        const int nextp = page_of(g_issue + step);
        issue(g_issue, page, s);
        g_issue += step;
        page = nextp;
    }

    // Q^T fragments: head n = lane / 4, channels 2 * (lane % 4) and + 8 of each k-step
    uint32_t qf[NB][KS][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int h = nb * 8 + (lane >> 2);
        const T* q = static_cast<const T*>(a.q) + r * a.q_row_stride + (long long)(kvh * p.group + h0 + h) * a.q_head_stride;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                qf[nb][k][j] = h < heads ? *reinterpret_cast<const uint32_t*>(q + k * 16 + j * 8 + 2 * (lane & 3)) : 0u;
    }

    float o[NB][KS][4];
    float m[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        m[nb][0] = m[nb][1] = -INFINITY;
        l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nb][k][i] = 0.f;
    }

    int stage = 0;
    for (int g = g0; g < groups; g += step) {
        cp_wait<ST - 1>();
        __syncwarp();
        const uint32_t kd = base + stage * 2 * kTile, vd = kd + kTile;
        float s[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nb][i] = 0.f;
        {
            const int t = lane & 15;
            const uint32_t row = kd + t * HD * 2;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t af[4];
                ldsm4(af, row + (((2 * k + (lane >> 4)) ^ (t & 7)) << 4));
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16816<T>(s[nb], af, qf[nb][k][0], qf[nb][k][1]);
            }
        }
        const int n = (g < pre_groups ? a.prefix_len - g * kGroup : len - (g - pre_groups) * kGroup);
        const bool lo = (lane >> 2) < n, hi = (lane >> 2) + 8 < n;
        bool raise = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            s[nb][0] = lo ? s[nb][0] * p.scale_log2 : -INFINITY;
            s[nb][1] = lo ? s[nb][1] * p.scale_log2 : -INFINITY;
            s[nb][2] = hi ? s[nb][2] * p.scale_log2 : -INFINITY;
            s[nb][3] = hi ? s[nb][3] * p.scale_log2 : -INFINITY;
            raise |= fmaxf(s[nb][0], s[nb][2]) > m[nb][0] + kSlack || fmaxf(s[nb][1], s[nb][3]) > m[nb][1] + kSlack;
        }
        if (__any_sync(~0u, raise)) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float x = fmaxf(s[nb][j], s[nb][j + 2]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
                    x = fmaxf(x, m[nb][j]);
                    const float f = m[nb][j] == x ? 1.f : m[nb][j] == -INFINITY ? 0.f : fast_exp2(m[nb][j] - x);
                    m[nb][j] = x;
                    l[nb][j] *= f;
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        o[nb][k][j] *= f;
                        o[nb][k][j + 2] *= f;
                    }
                }
        }
        uint32_t pb[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float m0 = m[nb][0] == -INFINITY ? 0.f : m[nb][0], m1 = m[nb][1] == -INFINITY ? 0.f : m[nb][1];
            const float p0 = fast_exp2(s[nb][0] - m0), p1 = fast_exp2(s[nb][1] - m1);
            const float p2 = fast_exp2(s[nb][2] - m0), p3 = fast_exp2(s[nb][3] - m1);
            l[nb][0] += p0 + p2;
            l[nb][1] += p1 + p3;
            pb[nb][0] = movm_t(pack2<T>(p0, p1));
            pb[nb][1] = movm_t(pack2<T>(p2, p3));
        }
        {
            const int t = (lane & 7) + ((lane >> 4) << 3);
            const uint32_t row = vd + t * HD * 2;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t af[4];
                ldsm4_t(af, row + (((2 * k + ((lane >> 3) & 1)) ^ (t & 7)) << 4));
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16816<T>(o[nb][k], af, pb[nb][0], pb[nb][1]);
            }
        }
        __syncwarp();
        const int nextp = page_of(g_issue + step);
        issue(g_issue, page, stage);
        g_issue += step;
        page = nextp;
        stage = stage + 1 == ST ? 0 : stage + 1;
    }
    cp_wait<0>();
    __syncwarp();

    // this warp's partial to its part of shared memory: O [8*NB][HD], then (m, l) [8*NB]
    float* wo = reinterpret_cast<float*>(sm + warp * kWarp);
    float2* wml = reinterpret_cast<float2*>(wo + 8 * NB * HD);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        const int h = nb * 8 + 2 * (lane & 3);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[nb][j] += __shfl_xor_sync(~0u, l[nb][j], d);
            if ((lane >> 2) == 0) wml[h + j] = make_float2(m[nb][j], bad ? NAN : l[nb][j]);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                wo[(h + (i & 1)) * HD + k * 16 + (lane >> 2) + ((i >> 1) << 3)] = o[nb][k][i];
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    pdl_wait();  // the prefix pass's partials

    // the join: each CTA of the cluster takes its share of the outputs, four channels a thread
    const uint32_t local = smem_addr(sm);
    const int quads = heads * (HD / 4);
    for (int x = rank * blockDim.x + threadIdx.x; x < quads; x += C * blockDim.x) {
        const int h = x / (HD / 4), c = (x % (HD / 4)) * 4;
        Join jn;
        for (uint32_t k = 0; k < C; ++k) {
            const uint32_t at = C > 1 ? map_rank(local, k) : local;
            for (int w = 0; w < kRowWarps; ++w) {
                const uint32_t wb = at + w * kWarp;
                jn.add(ld_cluster2(wb + 8 * NB * HD * 4 + h * 8), ld_cluster4(wb + (h * HD + c) * 4));
            }
        }
        if (!p.walk_prefix && a.prefix_len > 0) {
            const int row = r * p.group + h0 + h, tile = row / p.tile_rows, in = row % p.tile_rows;
            const long long u = (long long)kvh * p.row_tiles + tile;
            const long long c0 = u * p.kv_tiles / p.per, c1 = ((u + 1) * p.kv_tiles - 1) / p.per;
            const bool pair = p.tile_rows == 256;
            const long long first = 2 * (c0 + u) + (pair ? in >> 7 : 0), past = 2 * (c1 + u) + 2;
#pragma unroll 4
            for (long long s = first; s < past; s += pair ? 2 : 1) {
                const long long at = s * 128 + (in & 127);
                jn.add(p.part_ml[at], *reinterpret_cast<const float4*>(p.part_o + at * HD + c));
            }
        }
        const float inv = jn.L == 0.f ? 0.f : 1.f / jn.L;
        T res[4] = {from_f32<T>(jn.o.x * inv), from_f32<T>(jn.o.y * inv), from_f32<T>(jn.o.z * inv), from_f32<T>(jn.o.w * inv)};
        T* out = static_cast<T*>(a.out) + r * a.out_row_stride + (long long)(kvh * p.group + h0 + h) * a.out_head_stride + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = res[i];
    }
    if (C > 1) cluster_sync();  // the others may still read this CTA's shared memory
}

}  // namespace tt
