// tt_prefix_rows.cuh -- the pass of tt_shared_prefix_attention over each row's own pages, and the join of
// both passes.
//
// `splits` CTAs per (row, kv head, tile of up to 8*NB query heads).  Their 4*splits warps take the row's
// tokens in groups of 16 (a group never crosses a page), warp w groups w, w+4*splits, ...; each warp keeps its
// own pipeline of K and V groups, so no warp waits for another before the end.  Per group, with
// mma.sync m16n8k16 and tokens along M, because a row has few query heads and 16 tokens:
//   S^T[16 x 8] = K[16 x hd] Q^T[hd x 8]         (K by ldmatrix, Q^T in registers)
//   P^T = 2^(S^T - m), transposed in registers (movmatrix) into the second product's B operand
//   O^T[hd x 8] += V^T[hd x 16] P^T[16 x 8]       (V by transposing ldmatrix)
// m is a reference, not the maximum: it is raised (and O, l rescaled) only when a logit exceeds it by
// kSlack, so the cross-lane maximum and the rescale run once or twice a row instead of once a group;
// weights stay below 2^kSlack and every sum is float32.
// At the end the warps' (m, l, O) meet in shared memory, and k_prefix_join joins what the splits and the prefix
// pass left.  (A row's splits as a thread-block cluster joined through distributed shared memory, and the rows'
// CTAs joining the prefix pass's partials themselves, cost more: the CTAs wait for the prefix pass, where they
// could run beside it, its time being the tensor cores' and theirs the memory's.)
//
// Loads are TMA boxes of 16 tokens (cp.async by the lanes instead cost the warps a third of their instructions,
// and beside the prefix pass more: 282 against 257 us for 256 rows on 32k).  Weights are rounded to the pages'
// type for the second product, as in the prefix pass; logits, exponentials and sums are float32 (a product below
// 2^-25 of its sum is dropped by the tensor cores, while its weight counts in l).
//
// Bound: HBM (each row's K and V are read once).  Alone, 256 rows of up to 2048 tokens (1.08 GB): 170 us,
// 6.3 TB/s.  More than eight query heads a kv head take two fragments of everything and spill 44 bytes at 128
// registers a thread: 256 rows of up to 2048 tokens in 2 kv heads 62 us with 12 or 16 heads each, 52 with 8.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "tt_common.cuh"
#include "tt_launch.cuh"
#include "tt_prefix_plan.cuh"

namespace tt {

constexpr float kSlack = 8.f;    // log2 units a logit may exceed the reference before it is raised

constexpr long long kPatience = 4000000000LL;  // clocks that a wait may take (about two seconds)

__device__ int g_prefix_error = 0;  // a wait that ran out (TT_ERR_TIMEOUT); reported by tt_device_error

struct WaitState {           // in shared memory, of those that give up together: a warp here, a CTA in the prefix pass
    long long limit;         // clocks that a wait may take (in constant memory it cost 0.3 us of every call)
    int abort;
    int pad;
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
// Barriers in shared memory
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint32_t b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(b) : "memory"); }
__device__ __forceinline__ void bar_expect(uint32_t b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(b), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                 : "=r"(ok) : "r"(b), "r"(parity) : "memory");
    return ok != 0;
}
// Bounded: false when it took too long here (recorded) or elsewhere.
__device__ __noinline__ bool bar_wait_slow(uint32_t b, uint32_t parity, volatile WaitState* w) {
    const long long t0 = clock64(), limit = w->limit;
    while (clock64() - t0 < limit) {
        if (bar_try(b, parity)) return true;
        if (w->abort) return false;
    }
    w->abort = 1;
    atomicCAS(&g_prefix_error, 0, (int)TT_ERR_TIMEOUT);
    return false;
}
__device__ __forceinline__ bool bar_wait(uint32_t b, uint32_t parity, volatile WaitState* w) {
    return bar_try(b, parity) || bar_wait_slow(b, parity, w);
}
// The wait for copies or products in flight, before their memory is given back: whatever the limit, kPatience.
__device__ __noinline__ void bar_drain(uint32_t b, uint32_t parity) {
    const long long t0 = clock64();
    while (!bar_try(b, parity))
        if (clock64() - t0 > kPatience) {
            atomicCAS(&g_prefix_error, 0, (int)TT_ERR_TIMEOUT);
            return;
        }
}

// The same by a whole warp, with one answer.
__device__ __forceinline__ bool bar_wait_warp(uint32_t b, uint32_t parity, volatile WaitState* w) {
    return __all_sync(~0u, bar_wait(b, parity, w));
}

// A box of the pool: channel, head, token in page, page.  Outside the pool it is zeros.
__device__ __forceinline__ void tma_load4(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar,
                                          uint64_t policy) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, "
                 "%3, %4, %5}], [%6], %7;"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ uint64_t policy_evict_first() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ uint64_t policy_evict_last() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
    return p;
}

// A warp's join of n partials (m, l, O) of one row and query head, lane i taking channels i*HD/32 on: the
// weights first (a lane a partial), then the O rows, whose loads wait for nothing.  ml(i) gives (m, l), o(i)
// the address of O.  An empty partial (m = -inf, l = 0) has no O; l = NaN marks a failed one and stays.
template <int HD, typename ML, typename O>
__device__ __forceinline__ void join_partials(int n, ML ml, O o, float& M, float& L, float* acc) {
    constexpr int C = HD / 32;
    const int lane = threadIdx.x & 31;
    M = -INFINITY;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, ml(i).x);
#pragma unroll
    for (int d = 16; d; d >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, d));
    L = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    for (int base = 0; base < n; base += 32) {
        float w = 0.f;
        if (base + lane < n) {
            const float2 x = ml(base + lane);
            w = M == -INFINITY ? 0.f : fast_exp2(x.x - M);
            L += w * x.y;
        }
        const int m = min(32, n - base);
#pragma unroll 8
        for (int j = 0; j < m; ++j) {
            const float f = __shfl_sync(~0u, w, j);
            const float* p = o(base + j) + lane * C;
            float x[C];
            if constexpr (C == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
            else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(p);
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] += f != 0.f ? f * x[c] : 0.f;
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) L += __shfl_xor_sync(~0u, L, d);
}

template <typename T, int HD>
__device__ __forceinline__ void store_out(const PrefixParams& p, float L, const float* acc, int r, int head) {
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* out = static_cast<T*>(p.a.out) + r * p.a.out_row_stride + (long long)head * p.a.out_head_stride + (threadIdx.x & 31) * (HD / 32);
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) out[c] = from_f32<T>(acc[c] * inv);
}

// The join of the two passes: W warps a (row, query head), each a W-th of its partials, so that their loads
// are in flight together.
constexpr int kJoinWarps = 8;

template <typename T, int HD, int W>
__global__ void __launch_bounds__(kJoinWarps * 32) k_prefix_join(const PrefixParams p) {
    __shared__ __align__(16) float so[kJoinWarps][HD];
    __shared__ float2 sml[kJoinWarps];
    const tt_shared_prefix_args& a = p.a;
    const int warp = threadIdx.x >> 5, sub = warp % W;
    const long long rh = (long long)blockIdx.x * (kJoinWarps / W) + warp / W, all = (long long)a.num_rows * a.num_q_heads;
    const int r = (int)(rh / a.num_q_heads), head = (int)(rh % a.num_q_heads);
    const bool on = rh < all && !(a.row_seq && a.row_seq[r] < 0);
    const PrefixPartials pre = on && !p.walk_prefix ? prefix_partials(p, r, head) : PrefixPartials{0, 0, 0};
    const int n = on ? (p.splits + pre.n - sub + W - 1) / W : 0;
    pdl_wait();
    float M, L, acc[HD / 32];
    join_partials<HD>(n,
                      [&](int k) {
                          const int i = k * W + sub;
                          return *(i < p.splits ? p.own_ml + (i * all + rh) : p.part_ml + (pre.first + (i - p.splits) * pre.step));
                      },
                      [&](int k) {
                          const int i = k * W + sub;
                          return i < p.splits ? p.own_o + (i * all + rh) * HD : p.part_o + (pre.first + (i - p.splits) * pre.step) * HD;
                      },
                      M, L, acc);
    if constexpr (W > 1) {
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) so[warp][(threadIdx.x & 31) * (HD / 32) + c] = acc[c];
        if ((threadIdx.x & 31) == 0) sml[warp] = make_float2(M, L);
        __syncthreads();
        if (sub) return;
        join_partials<HD>(W, [&](int k) { return sml[warp + k]; }, [&](int k) { return so[warp + k]; }, M, L, acc);
    }
    if (on) store_out<T, HD>(p, L, acc, r, head);
}

template <int HD, int NB> constexpr int row_out_bytes() { return 8 * NB * HD * 4 + 8 * NB * 8; }  // one warp's O and (m, l)
template <int HD, int NB, int ST> constexpr int row_warp_bytes() {
    static_assert(ST * 2 * kGroup * HD * 2 >= row_out_bytes<HD, NB>(), "the partials take the stages' place");
    return ST * 2 * kGroup * HD * 2;
}
template <int HD, int NB, int ST> constexpr int row_smem() {
    return kRowWarps * (row_warp_bytes<HD, NB, ST>() + 2 * ST * 8 + (int)sizeof(WaitState));
}

template <typename T, int HD, int NB, int ST>
__global__ void __launch_bounds__(kRowWarps * 32, 4)
k_prefix_rows(const PrefixParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    extern __shared__ __align__(1024) unsigned char sm[];
    constexpr int KS = HD / 16;                       // k-steps of the first product
    constexpr int kTile = kGroup * HD * 2;            // bytes of a K (or V) group: HD / 64 boxes of 16 x 128
    constexpr int kWarp = row_warp_bytes<HD, NB, ST>();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
    const int kvh = blockIdx.y / p.head_tiles, h0 = (blockIdx.y % p.head_tiles) * 8 * NB;
    const int heads = min(8 * NB, p.group - h0);      // query heads of this tile
    const tt_shared_prefix_args& a = p.a;

    // This grid runs beside the prefix pass and waits for nothing of it, but must not end before it does, for the
    // join waits for this grid alone: the last CTA sees to that.
    const bool last = blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
    pdl_trigger();

    const int seq = a.row_seq ? a.row_seq[r] : r;
    if (seq < 0) {  // padding
        if (last) pdl_wait();
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
    const int step = kRowWarps * p.splits, g0 = split * kRowWarps + warp;
    const int gpp = p.page_shift - 4;                 // log2 groups per page

    const uint32_t base = smem_addr(sm) + warp * kWarp;
    const uint32_t bars = smem_addr(sm) + kRowWarps * kWarp + warp * 2 * ST * 8;  // K of each stage, V of each stage
    volatile WaitState* wait = reinterpret_cast<WaitState*>(sm + kRowWarps * (kWarp + 2 * ST * 8)) + warp;
    if (lane == 0) {
        wait->limit = p.patience;
        wait->abort = 0;
        for (int i = 0; i < 2 * ST; ++i) bar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\nfence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    // Evict first: a row's own pages are read once.  A prefix that the rows read themselves is read again, but from L2
    // all the same, and the normal policy costs more than it saves (32/8 heads of 128: one row on 32k 26.7 against
    // 28.8 us, 8 rows on 1024 11.5 against 11.7, 64 rows on 8k with a negative scale 231 against 251; 256 rows of up to
    // 2000 own tokens on 4k with a negative scale 520 against 406).
    const uint64_t once = policy_evict_first();

    const auto page_of = [&](int g) {
        if (g >= groups) return 0;
        const int pg = g < pre_groups ? a.prefix_table[g >> gpp] : own[(g - pre_groups) >> gpp];
        if (pg >= 0 && pg < a.num_pages) return pg;
        bad = true;
        return a.num_pages;  // outside the pool: the load gives zeros
    };
    // K or V of group g into its half of a stage
    const auto issue = [&](int g, int page, int stage, int is_v) {
        if (g < groups && lane == 0) {
            const int in_page = ((g < pre_groups ? g : g - pre_groups) * kGroup) & (a.page_size - 1);
            const uint32_t bar = bars + 8 * (is_v * ST + stage), dst = base + (stage * 2 + is_v) * kTile;
            bar_expect(bar, kTile);
#pragma unroll
            for (int h = 0; h < HD / 64; ++h)
                tma_load4(dst + h * (kGroup * 128), is_v ? &vmap : &kmap, h * 64, kvh, in_page, page, bar, once);
        }
    };

    // K of a group is asked for as soon as the first product has used the K before it, V after the second
    int g_issue = g0, page = page_of(g0);
#pragma unroll
    for (int s = 0; s < ST; ++s) {
        const int nextp = page_of(g_issue + step);
        issue(g_issue, page, s, 0);
        issue(g_issue, page, s, 1);
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
    uint32_t phase = 0;
    bool lost = false, at_v = false;  // a wait ran out; it was for V, with K used and the stage's next one asked for
    int g = g0;
    for (; g < groups; g += step) {
        const uint32_t kd = base + stage * 2 * kTile, vd = kd + kTile;
        if (!bar_wait_warp(bars + 8 * stage, phase, wait)) {
            lost = true;
            break;
        }
        float s[NB][4], s1[NB][4];  // two chains of products
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nb][i] = s1[nb][i] = 0.f;
        {
            const int t = lane & 15;
            const uint32_t row = kd + t * 128;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t af[4];
                ldsm4(af, row + (k / 4) * (kGroup * 128) + (((2 * (k % 4) + (lane >> 4)) ^ (t & 7)) << 4));
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16816<T>(k & 1 ? s1[nb] : s[nb], af, qf[nb][k][0], qf[nb][k][1]);
            }
        }
        __syncwarp();
        issue(g_issue, page, stage, 0);
        const int n = (g < pre_groups ? a.prefix_len - g * kGroup : len - (g - pre_groups) * kGroup);
        const bool lo = (lane >> 2) < n, hi = (lane >> 2) + 8 < n;
        bool raise = false;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[nb][i] = (i < 2 ? lo : hi) ? (s[nb][i] + s1[nb][i]) * p.scale_log2 : -INFINITY;
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
        if (!bar_wait_warp(bars + 8 * (ST + stage), phase, wait)) {
            lost = true;
            at_v = true;
            break;
        }
        if (n < kGroup) {
            // what lies behind the last token may be NaN, and 0 * NaN is not 0
            for (int x = n * 8 + lane; x < kGroup * 8; x += 32)
#pragma unroll
                for (int h = 0; h < HD / 64; ++h)
                    *reinterpret_cast<uint4*>(sm + (vd - smem_addr(sm)) + h * (kGroup * 128) + x * 16) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
        }
        {
            const int t = (lane & 7) + ((lane >> 4) << 3);
            const uint32_t row = vd + t * 128;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t af[4];
                ldsm4_t(af, row + (k / 4) * (kGroup * 128) + (((2 * (k % 4) + ((lane >> 3) & 1)) ^ (t & 7)) << 4));
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) mma16816<T>(o[nb][k], af, pb[nb][0], pb[nb][1]);
            }
        }
        __syncwarp();
        const int nextp = page_of(g_issue + step);
        issue(g_issue, page, stage, 1);
        g_issue += step;
        page = nextp;
        if (++stage == ST) {
            stage = 0;
            phase ^= 1;
        }
    }
    if (lost) {
        // the result is lost; no copy may be in flight when the stages are used again: the oldest is at `stage`
        bad = true;
        for (int i = 0; i < 2 * ST; ++i) {
            const int st = (stage + i / 2) % ST;
            const bool next = at_v && i == 0;  // a phase that is long past would be waited for in vain
            if (next ? g_issue < groups : g + (i / 2) * step < groups)
                bar_drain(bars + 8 * ((i & 1) * ST + st), phase ^ (next || st < stage));
        }
        __syncwarp();
    }

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
    __syncthreads();

    // the join of the warps, a warp a query head
    for (int h = warp; h < heads; h += kRowWarps) {
        const int head = kvh * p.group + h0 + h;
        const auto warp_o = [&](int w) { return reinterpret_cast<const float*>(sm + w * kWarp); };
        float M, L, acc[HD / 32];
        join_partials<HD>(kRowWarps, [&](int w) { return reinterpret_cast<const float2*>(warp_o(w) + 8 * NB * HD)[h]; },
                          [&](int w) { return warp_o(w) + h * HD; }, M, L, acc);
        if (p.join) {
            const long long at = ((long long)split * a.num_rows + r) * a.num_q_heads + head;
            if (lane == 0) p.own_ml[at] = make_float2(M, L);
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) p.own_o[at * HD + lane * (HD / 32) + c] = acc[c];
        } else {
            store_out<T, HD>(p, L, acc, r, head);
        }
    }
    if (last) pdl_wait();
}

}  // namespace tt
