// tt_prefix_shared.cuh -- the pass of tt_shared_prefix_attention over the prefix that all rows share.
//
// For one kv head the rows of all requests' query heads form one matrix of num_rows * group rows, so the
// prefix is a dense attention of that matrix over prefix_len keys: GEMM-shaped work, on the tensor cores
// (tcgen05), each K and V page read once per tile of rows.  A CTA holds two 128-row accumulators at once,
// so that the tensor cores work for one while the softmax warps work for the other:
//   PAIR   (more than 128 rows per kv head)  the two halves of a 256-row tile, over the same keys
//   !PAIR  (at most 128)                     one 128-row tile, over the even and the odd key tiles
// Per key tile of 128 tokens and accumulator t:  S_t = Q K^T (both from shared memory, into tensor memory),
// the softmax warps read S_t (a thread a row), write P_t = 2^(S_t scale - m) over it in the pages' type,
// and O_t += P_t V (P from tensor memory, V from shared memory).  m is a reference that is raised, and O
// rescaled, only when a logit exceeds it by kSlack, as in the rows' pass.
//
// Work: units of (kv head, row tile), each kv_tiles key tiles.  Each unit is cut into the same number of equal spans,
// one per CTA; where that would leave too many SMs idle the flattened list of all units' tiles is cut instead, and a
// CTA's span may cross into the next unit (tt_prefix_plan.cuh).  Where the row tiles of a
// kv head fill the SMs in whole groups, a group of CTAs takes the same span for all of them, so that each K
// and V page comes from HBM once and from L2 for the rest of the group.  A span inside a unit leaves one
// partial (m, l, O) per accumulator in the workspace, in a slot that no other span has; the join adds them.
//
// Warps: 0 loads K and V (TMA, one box per page and 64 channels, 128-byte swizzle), 1 issues the matrix
// instructions, 2 clears the V rows behind the prefix's end (what lies there may be NaN, and 0 * NaN is not
// 0), 4-7 and 8-11 are the softmax of the two accumulators and load their queries.
//
// Bound: 256 rows of 32 heads on 32k take 144 us (950 TFLOP/s; 83 us at the measured GEMM rate), 2.5 us a key
// tile of 256 rows.  Neither the exponentials (16 a clock: half of that), nor the products alone, nor the loads
// set it: removing any one gains under a tenth.  It is the chain S -> weights -> products through barriers, with
// the two softmax warps that share a scheduler with the warp issuing the products slower than the others by
// half.  Measured beside it and no faster: the tile as a pair of CTAs (cta_group::2; 161 us, the arrivals
// between the CTAs cost more than the shared K and V save), steps of 64 keys with two S an accumulator
// (146-168 us; a product of 64 columns takes as long as one of 128), a quarter of the exponentials as
// polynomials (139 against 143), five K/V slots (143 us, but no rows' CTA beside them).
#pragma once
#include "tt_prefix_rows.cuh"

namespace tt {

constexpr int kPsThreads = 384;

template <int HD, bool PAIR> struct PsShape {
    static constexpr int kSlot = kPsTile * HD * 2;                 // a K or V tile
    static constexpr int kHalf = kPsTile * 64 * 2;                 // 64 of its channels: 128-byte rows
    static constexpr int kQ = (PAIR ? 2 : 1) * kSlot;
    static constexpr int kSlots = HD == 128 ? (PAIR ? 3 : 4) : 8;  // 160 KB with Q: leaves room for a CTA of the rows' pass
    static constexpr int kSmem = kQ + kSlots * kSlot + 256;        // tiles, barriers
    static constexpr uint32_t kTmemO = 256;                        // S_0 S_1 in columns 0, 128; O_t behind
};

struct PsBars {  // in shared memory
    uint64_t full[8], empty[8], q_full, s_full[2], p_ready[4], v_cut, v_fixed, drain;
    WaitState wait;
    uint32_t tmem, loads;
    int bad;
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc) : "memory");
}
#define TT_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define TT_W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
// 32 columns of the warp's 32 lanes: v[c] is column c of this thread's lane.
__device__ __forceinline__ void tc_ld32(uint32_t* v, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
                 "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : TT_R4(v, 0), TT_R4(v, 4), TT_R4(v, 8), TT_R4(v, 12), TT_R4(v, 16), TT_R4(v, 20), TT_R4(v, 24), TT_R4(v, 28)
                 : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::TT_W4(v, 0), TT_W4(v, 4), TT_W4(v, 8), TT_W4(v, 12), TT_W4(v, 16), TT_W4(v, 20), TT_W4(v, 24), TT_W4(v, 28),
                   "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::TT_W4(v, 0), TT_W4(v, 4), TT_W4(v, 8), TT_W4(v, 12), "r"(addr) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// One thread of the warp, known as such to the compiler: operands of the tcgen05 instructions it issues are
// uniform.  (With `lane == 0` instead each product took about 70 clocks to issue.)
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok));
    return ok != 0;
}

// Two float32 at a time, as the FMA pipe takes them; the larger of three.
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b) {  // x = x a + b, y = y a + b
    asm("{\n.reg .b64 v, a, b;\nmov.b64 v, {%0, %1};\nmov.b64 a, {%2, %2};\nmov.b64 b, {%3, %3};\n"
        "fma.rn.f32x2 v, v, a, b;\nmov.b64 {%0, %1}, v;\n}" : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {  // x += a, y += b
    asm("{\n.reg .b64 v, a;\nmov.b64 v, {%0, %1};\nmov.b64 a, {%2, %3};\nadd.rn.f32x2 v, v, a;\nmov.b64 {%0, %1}, v;\n}"
        : "+f"(x), "+f"(y) : "f"(a), "f"(b));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Shared-memory operand descriptors, 128-byte swizzle.  K-major (rows of 64 channels, groups of eight rows
// 1024 bytes apart) and MN-major (V: a token's 64 channels contiguous; groups of eight tokens 1024 bytes
// apart, the next 64 channels `lbo` bytes on).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
template <typename T> constexpr uint32_t ps_idesc(int n, bool b_mn) {
    const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return 1u << 4 | fmt << 7 | fmt << 10 | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kPsTile >> 4) << 24;
}

// The spans of this CTA.
template <typename F>
__device__ __forceinline__ void ps_spans(const PrefixParams& p, F fn) {
    prefix_spans(p, blockIdx.x / p.lanes, blockIdx.x % p.lanes, fn);
}

template <typename T, int HD, bool PAIR>
__global__ void __launch_bounds__(512, 1)  // 128 registers a thread, not the 168 that 384 threads could have
k_prefix_shared(const PrefixParams p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using S = PsShape<HD, PAIR>;
    constexpr int kLook = PAIR ? 1 : 2;  // key tiles whose first product is issued ahead
    extern __shared__ __align__(1024) unsigned char sm[];
    PsBars* bars = reinterpret_cast<PsBars*>(sm + S::kQ + S::kSlots * S::kSlot);
    const uint32_t q_s = smem_addr(sm), ring = q_s + S::kQ;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const tt_shared_prefix_args& a = p.a;
    volatile WaitState* wait = &bars->wait;
    const uint32_t full = smem_addr(bars->full), empty = smem_addr(bars->empty), q_full = smem_addr(&bars->q_full),
                   s_full = smem_addr(bars->s_full), p_ready = smem_addr(bars->p_ready), v_cut = smem_addr(&bars->v_cut),
                   v_fixed = smem_addr(&bars->v_fixed), drain = smem_addr(&bars->drain);

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kSlots; ++i) {
            bar_init(full + 8 * i, 1);
            bar_init(empty + 8 * i, 1);
        }
        bar_init(q_full, 256);
        for (int t = 0; t < 2; ++t) {
            bar_init(s_full + 8 * t, 1);
            bar_init(p_ready + 16 * t, 128);
            bar_init(p_ready + 16 * t + 8, 128);
        }
        bar_init(v_cut, 1);
        bar_init(v_fixed, 32);
        bar_init(drain, 1);
        bars->wait.limit = p.patience;
        bars->wait.abort = 0;
        bars->bad = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&bars->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem;
    pdl_trigger();

    if (warp == 0) {
        // ---- K and V tiles into the ring, in the order the products take them
        const int box = a.page_size < kPsTile ? a.page_size : kPsTile;  // tokens per load
        const int boxes = kPsTile / box;
        const uint64_t again = policy_evict_last();  // the other row tiles read it too
        uint32_t it = 0;
        ps_spans(p, [&](int kvh, int tile, long long slot_at, int k0, int n) {
            const auto load = [&](const CUtensorMap* map, int kt) {
                const int t0 = (k0 + kt) * kPsTile;
                const int left = a.prefix_len - t0, use = left < kPsTile ? (left + box - 1) / box : boxes;
                int page = a.num_pages;  // outside the pool: the load gives zeros
                if (lane < use) {
                    page = a.prefix_table[(t0 + lane * box) >> p.page_shift];
                    if (page < 0 || page >= a.num_pages) {
                        page = a.num_pages;
                        *(volatile int*)&bars->bad = 1;  // before the arrival below, seen by all that depends on it
                    }
                }
                const uint32_t slot = it % S::kSlots, phase = (it / S::kSlots) & 1;
                if (!bar_wait_warp(empty + 8 * slot, phase ^ 1, wait)) return false;
                if (lane == 0) bar_expect(full + 8 * slot, use * box * HD * 2);
                __syncwarp();
                if (lane < use) {
                    const uint32_t dst = ring + slot * S::kSlot + lane * box * 128;
                    const int row = (t0 + lane * box) & (a.page_size - 1);
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h) tma_load4(dst + h * S::kHalf, map, h * 64, kvh, row, page, full + 8 * slot, again);
                }
                ++it;
                return true;
            };
            for (int i = 0; i < kLook && i < n; ++i)
                if (!load(&kmap, i)) return false;
            for (int j = 0; j < n; ++j) {
                if (!load(&vmap, j)) return false;
                if (j + kLook < n && !load(&kmap, j + kLook)) return false;
            }
            return true;
        });
        bars->loads = it;
    } else if (warp == 1) {
        // ---- the matrix instructions, from one thread
        if (elect_one()) {
            constexpr uint32_t id_qk = ps_idesc<T>(kPsTile, false), id_pv = ps_idesc<T>(HD, true);
            uint32_t it = 0, q_phase = 0, fix_phase = 0, p_phase[2] = {0, 0};
            const auto slot_of = [&](uint32_t i) { return ring + (i % S::kSlots) * S::kSlot; };
            const auto slot_full = [&](uint32_t i) { return bar_wait(full + 8 * (i % S::kSlots), (i / S::kSlots) & 1, wait); };
            const auto qk = [&](int t, uint32_t i) {
                const uint64_t q = smem_desc(q_s + (PAIR ? t * S::kSlot : 0), 16, 1024), k = smem_desc(slot_of(i), 16, 1024);
#pragma unroll
                for (int s = 0; s < HD / 16; ++s) {
                    const int off = ((s / 4) * S::kHalf + (s % 4) * 32) / 16;  // addresses in units of 16 bytes
                    tc_mma_ss(tmem + t * 128, q + off, k + off, id_qk, s > 0);
                }
            };
            const auto pv = [&](int t, uint32_t i, int half, bool acc) {  // 64 of the tile's keys
                const uint64_t v = smem_desc(slot_of(i), S::kHalf, 1024);
#pragma unroll
                for (int k = 0; k < kPsTile / 32; ++k) {
                    const int s = half * (kPsTile / 32) + k;
                    tc_mma_ts(tmem + S::kTmemO + t * HD, tmem + t * 128 + s * 8, v + s * 2048 / 16, id_pv, acc || k > 0);
                }
            };
            ps_spans(p, [&](int kvh, int tile, long long slot_at, int k0, int n) {
                if (!bar_wait(q_full, q_phase, wait)) return false;
                q_phase ^= 1;
                tc_fence_after();
                const bool cut = k0 + n == p.kv_tiles && a.prefix_len % kPsTile;
                for (int i = 0; i < kLook && i < n; ++i) {
                    if (!slot_full(it)) return false;
                    tc_fence_after();
                    for (int t = PAIR ? 0 : i; t < (PAIR ? 2 : i + 1); ++t) {
                        qk(t, it);
                        tc_commit(s_full + 8 * t);
                    }
                    tc_commit(empty + 8 * (it % S::kSlots));
                    ++it;
                }
                for (int j = 0; j < n; ++j) {
                    const uint32_t vi = it++, ki = it;
                    const bool more = j + kLook < n;
                    if (more) ++it;
                    if (!slot_full(vi)) return false;
                    if (cut && j == n - 1) {
                        bar_arrive(v_cut);
                        if (!bar_wait(v_fixed, fix_phase, wait)) return false;
                        fix_phase ^= 1;
                    }
                    for (int t = PAIR ? 0 : j & 1; t < (PAIR ? 2 : (j & 1) + 1); ++t) {
                        if (!bar_wait(p_ready + 16 * t, p_phase[t], wait)) return false;
                        tc_fence_after();
                        pv(t, vi, 0, PAIR ? j > 0 : j > 1);
                        if (!bar_wait(p_ready + 16 * t + 8, p_phase[t], wait)) return false;
                        p_phase[t] ^= 1;
                        tc_fence_after();
                        pv(t, vi, 1, true);
                        if (!PAIR || t == 1) tc_commit(empty + 8 * (vi % S::kSlots));
                        if (more) {
                            if ((!PAIR || t == 0) && !slot_full(ki)) return false;
                            tc_fence_after();
                            qk(t, ki);
                            if (!PAIR || t == 1) tc_commit(empty + 8 * (ki % S::kSlots));
                        }
                        tc_commit(s_full + 8 * t);  // the next S_t, or the last O_t
                    }
                }
                return true;
            });
            // every product and every arrival above has happened before the CTA gives its memory back
            tc_commit(drain);
            bar_drain(drain, 0);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---- V rows behind the end of the prefix
        if (a.prefix_len % kPsTile) {
            uint32_t loads = 0, phase = 0;
            ps_spans(p, [&](int kvh, int tile, long long slot_at, int k0, int n) {
                loads += 2 * n;
                if (k0 + n != p.kv_tiles) return true;
                if (!bar_wait_warp(v_cut, phase, wait)) return false;
                phase ^= 1;
                const int from = a.prefix_len % kPsTile * 8;
                unsigned char* v = sm + S::kQ + (loads - 1) % S::kSlots * S::kSlot;  // the span's last load
                for (int x = from + lane; x < kPsTile * 8; x += 32)
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h) *reinterpret_cast<uint4*>(v + h * S::kHalf + x * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(v_fixed);
                return true;
            });
        }
    } else if (warp >= 4) {
        // ---- softmax: thread = row of accumulator t
        const int t = (warp - 4) >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = tmem + ((uint32_t)(row & 96) << 16), s_col = lanes + t * 128, o_col = lanes + S::kTmemO + t * HD;
        const int rows_all = a.num_rows * p.group;
        const bool q16 = !(((uintptr_t)a.q & 15) | ((a.q_row_stride | a.q_head_stride) & 7));
        uint32_t phase = 0, q_phase = 0;
        ps_spans(p, [&](int kvh, int tile, long long slot_at, int k0, int n) {
            const int mine = PAIR ? n : (n - t + 1) / 2;
            const int mrow = tile * p.tile_rows + (PAIR ? t * kPsTile : 0) + row;
            const bool warp_on = mrow - lane < rows_all;  // any row of this warp
            if (PAIR || t == 0) {
                // this row's query into the swizzled layout of the first product
                const int r = mrow / p.group, h = kvh * p.group + mrow % p.group;
                const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + r * a.q_row_stride + h * a.q_head_stride);
                unsigned char* dst = sm + (PAIR ? t * S::kSlot : 0) + row * 128;
#pragma unroll 4
                for (int c = 0; c < HD / 8; ++c) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (mrow < rows_all) {
                        if (q16) x = src[c];
                        else {
                            const uint32_t* s4 = reinterpret_cast<const uint32_t*>(src + c);
                            x = make_uint4(s4[0], s4[1], s4[2], s4[3]);
                        }
                    }
                    *reinterpret_cast<uint4*>(dst + (c / 8) * S::kHalf + (((c % 8) ^ (row & 7)) << 4)) = x;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            // Accumulator 1 of !PAIR has loaded nothing, but arrives too: it has seen the last O_1 of the span before.
            // Without that s_full[1] could complete twice before a late warp looks once, and the warp would wait for a
            // phase that itself waits for the warp.  With no tile in this span it waits for the others' arrivals, lest
            // it arrive twice in one phase.
            bar_arrive(q_full);
            if (!PAIR && mine == 0 && !bar_wait_warp(q_full, q_phase, wait)) return false;
            q_phase ^= 1;
            float m = -INFINITY, l = 0.f;
            for (int i = 0; i < mine; ++i) {
                if (!bar_wait_warp(s_full + 8 * t, phase, wait)) return false;
                phase ^= 1;
                tc_fence_after();
                // The upper half of S goes through the registers for its maximum only; the lower half stays in them,
                // becomes weights first (its P lies over S columns that have been read) and the upper half is read
                // again: 64 registers of S instead of 128, and the second product starts on the lower half.
                float s[64];
                uint32_t* su = reinterpret_cast<uint32_t*>(s);
                const int left = a.prefix_len - (k0 + (PAIR ? i : 2 * i + t)) * kPsTile;
                const auto get = [&](int from) {
                    tc_ld32(su, s_col + from);
                    tc_ld32(su + 32, s_col + from + 32);
                    tc_wait_ld();
                    if (left < kPsTile) {
#pragma unroll
                        for (int c = 0; c < 64; ++c) s[c] = from + c < left ? s[c] : -INFINITY;
                    }
                };
                float lsum[2] = {0.f, 0.f};
                float neg = 0.f;
                const auto put = [&](int from) {  // weights of the 64 columns in s
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        uint32_t w[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float x = s[c + 2 * k], y = s[c + 2 * k + 1];
                            fma2(x, y, p.scale_log2, neg);
                            x = fast_exp2(x);
                            y = fast_exp2(y);
                            add2(lsum[0], lsum[1], x, y);
                            w[k] = pack2<T>(x, y);
                        }
                        tc_st16(s_col + (from + c) / 2, w);
                    }
                };
                if (warp_on) {
                    get(64);
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int c = 4; c < 64; c += 2) mx[c / 2 & 3] = max3(mx[c / 2 & 3], s[c], s[c + 1]);
                    get(0);
#pragma unroll
                    for (int c = 0; c < 64; c += 2) mx[c / 2 & 3] = max3(mx[c / 2 & 3], s[c], s[c + 1]);
                    const float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2;
                    if (__any_sync(~0u, top > m + kSlack)) {
                        const float nm = fmaxf(m, top);
                        const float f = nm == m ? 1.f : m == -INFINITY ? 0.f : fast_exp2(m - nm);
                        m = nm;
                        l *= f;
                        if (i > 0) {  // the arrival on s_full says that O has every step before this one
#pragma unroll 1
                            for (int c = 0; c < HD / 32; ++c) {
                                uint32_t* o = su;  // S is read again afterwards
                                tc_ld32(o, o_col + 32 * c);
                                tc_wait_ld();
#pragma unroll
                                for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                                tc_st32(o_col + 32 * c, o);
                            }
                            get(0);
                        }
                    }
                    neg = m == -INFINITY ? 0.f : -m;
                    put(0);
                    tc_wait_st();
                }
                tc_fence_before();
                bar_arrive(p_ready + 16 * t);
                if (warp_on) {
                    get(64);
                    put(64);
                    l += lsum[0] + lsum[1];
                    tc_wait_st();
                }
                tc_fence_before();
                bar_arrive(p_ready + 16 * t + 8);
            }
            // the span's partial
            const long long slot = 2 * slot_at + t;
            if (mine > 0) {
                if (!bar_wait_warp(s_full + 8 * t, phase, wait)) return false;
                phase ^= 1;
                tc_fence_after();
                if (warp_on) {
                    float* dst = p.part_o + (slot * kPsTile + row) * HD;
#pragma unroll
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tc_ld32(o, o_col + 32 * c);
                        tc_wait_ld();
                        if (mrow < rows_all) {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                *reinterpret_cast<uint4*>(dst + 32 * c + 4 * k) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
                        }
                    }
                }
                tc_fence_before();
            }
            if (mrow < rows_all) p.part_ml[slot * kPsTile + row] = make_float2(m, *(volatile int*)&bars->bad ? NAN : l);
            return true;
        });
        if (wait->abort) {
            // a wait ran out: nothing that this CTA was to leave may be taken for a result
            ps_spans(p, [&](int kvh, int tile, long long slot_at, int k0, int n) {
                p.part_ml[(2 * slot_at + t) * kPsTile + row] = make_float2(-INFINITY, NAN);
                return true;
            });
        }
    }
    __syncthreads();
    if (warp == 0 && wait->abort) {
        // whichever warp gave up, no copy may be in flight when the CTA ends: the last load of each slot
        const uint32_t it = bars->loads;
        for (uint32_t i = it > S::kSlots ? it - S::kSlots : 0; i < it; ++i)
            bar_drain(full + 8 * (i % S::kSlots), (i / S::kSlots) & 1);
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace tt
