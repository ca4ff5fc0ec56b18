// tt_paged.cu -- page tables from request lengths, and the norm / rotation / placing of a step's
// queries, keys and values (C ABI: tt_page_tables, tt_qk_norm_rope).
#include <cuda_bf16.h>
#include <limits.h>

#include "tt_common.cuh"
#include "tt_launch.cuh"

namespace tt {

static_assert(sizeof(tt_page_tables_args) == 144 && sizeof(tt_qk_norm_rope_args) == 296, "packed by paged.py");

// ---------------------------------------------------------------------------
// Page tables
//
// Two exclusive scans over the requests: first of the pages that ended requests give back and of the
// rows that the others bring, then of the pages the others need (which needs to know whose rows fit).
// One CTA does both: the data are 8 bytes a request, so latency is all there is to lose, and a second
// CTA would only add a wait.  What is proportional to the rows is done by the same CTA while it is
// small (one launch) and by a grid in a second launch when it is not.
// ---------------------------------------------------------------------------
constexpr int kPtThreads = 1024;
constexpr int kPtItems = 4;                    // requests per thread and tile
constexpr int kPtSmallSeqs = 2048;             // one-launch form: requests held in shared memory
constexpr int kPtSmallRows = 8192;             // and rows written by one CTA

struct PtWorkspace {                           // of the two-launch form: header, then first[num_seqs], ctx[num_seqs]
    int top;
    int pad;
};

static bool pt_small(int num_seqs, int num_rows) { return num_seqs <= kPtSmallSeqs && num_rows <= kPtSmallRows; }

struct Pair64 {
    long long a, b;
};

// Exclusive scan of one pair per thread over the block; totals in *tot.
__device__ __forceinline__ Pair64 block_scan2(Pair64 v, Pair64* tot, Pair64* sm) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    Pair64 x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long ya = __shfl_up_sync(~0u, x.a, d), yb = __shfl_up_sync(~0u, x.b, d);
        if (lane >= d) x.a += ya, x.b += yb;
    }
    if (lane == 31) sm[w] = x;
    __syncthreads();
    if (w == 0) {
        Pair64 t = lane < nw ? sm[lane] : Pair64{0, 0};
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long ya = __shfl_up_sync(~0u, t.a, d), yb = __shfl_up_sync(~0u, t.b, d);
            if (lane >= d) t.a += ya, t.b += yb;
        }
        if (lane < nw) sm[lane] = t;
    }
    __syncthreads();
    const Pair64 base = w ? sm[w - 1] : Pair64{0, 0};
    *tot = sm[nw - 1];
    __syncthreads();  // sm is used again
    return Pair64{base.a + x.a - v.a, base.b + x.b - v.b};
}

__device__ __forceinline__ int clamp_i32(long long x) { return x > INT_MAX ? INT_MAX : (int)x; }

struct PtReq {
    long long ctx, held, n;  // tokens held, pages held, new tokens
    bool ended;
};
__device__ __forceinline__ PtReq pt_req(const tt_page_tables_args& p, int b) {
    PtReq r{0, 0, 0, false};
    if (b < p.num_seqs) {
        const int c = p.ctx_lens[b], n = p.new_lens[b];
        r.ctx = c > 0 ? c : 0;
        r.held = (r.ctx + p.page_size - 1) / p.page_size;
        r.ended = n < 0;
        r.n = n > 0 ? n : 0;
    }
    return r;
}

// Row t of the step, of request b: ctx tokens held, first row cu, first popped entry `first` (-1: deferred).
struct PtRow {
    long long slot;
    int pos, seq, len;
};
__device__ __forceinline__ PtRow pt_row(const tt_page_tables_args& p, int b, int ctx, int cu, int first, int top,
                                        int t) {
    if (first < 0) return PtRow{-1, 0, -1, 0};
    const int held = (int)(((long long)ctx + p.page_size - 1) / p.page_size);
    const int pos = ctx + (t - cu), pg = pos / p.page_size;
    const int page = pg < held ? p.tables[b * p.table_stride + pg] : p.free_pages[top - 1 - first - (pg - held)];
    return PtRow{(long long)page * p.page_size + pos % p.page_size, pos + p.position_offset, b, pos + 1};
}
__device__ __forceinline__ void pt_store(const tt_page_tables_args& p, int t, const PtRow& r) {
    p.slots[t] = r.slot;
    p.positions[t] = r.pos;
    p.row_seq[t] = r.seq;
    p.row_lens[t] = r.len;
}

// First b in [0, n) with cu[b + 1] > t, n when there is none.
template <typename F>
__device__ __forceinline__ int pt_find(F cu, int n, int t) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int m = (lo + hi) >> 1;
        if (cu(m + 1) > t) hi = m;
        else lo = m + 1;
    }
    return lo;
}

// SMALL: one launch; per-request results in shared memory, tables and rows written here.
template <bool SMALL>
__global__ void __launch_bounds__(kPtThreads) k_page_scan(const tt_page_tables_args p) {
    extern __shared__ int sm_dyn[];
    int* cu_s = sm_dyn;                      // [num_seqs + 1] when SMALL
    int* first_s = sm_dyn + p.num_seqs + 1;  // [num_seqs] when SMALL
    int* ctx_s = first_s + p.num_seqs;       // [num_seqs] when SMALL
    __shared__ Pair64 sm[32];
    __shared__ int late_s;
    const int tid = threadIdx.x, tile = blockDim.x * kPtItems, B = p.num_seqs;
    if (tid == 0) late_s = 0;
    int fc = *p.free_count;
    fc = fc < 0 ? 0 : fc > p.free_capacity ? p.free_capacity : fc;

    // pages given back, first rows
    Pair64 carry{0, 0};
    for (int base = 0; base < B; base += tile) {
        PtReq r[kPtItems];
        Pair64 s{0, 0};
        int back[kPtItems];
#pragma unroll
        for (int i = 0; i < kPtItems; ++i) {
            r[i] = pt_req(p, base + tid * kPtItems + i);
            back[i] = r[i].ended ? (int)(r[i].held < p.table_width ? r[i].held : p.table_width) : 0;
            s.a += back[i];
            s.b += r[i].n;
        }
        Pair64 tot;
        Pair64 at = block_scan2(s, &tot, sm);
        at.a += carry.a + fc;
        at.b += carry.b;
#pragma unroll
        for (int i = 0; i < kPtItems; ++i) {
            const int b = base + tid * kPtItems + i;
            if (b < B) {
                p.cu_new[b] = clamp_i32(at.b);
                if (SMALL) cu_s[b] = clamp_i32(at.b);
            }
            // the warp copies the pages of each of its ended requests together
            unsigned todo = __ballot_sync(~0u, back[i] > 0);
            while (todo) {
                const int l = __ffs(todo) - 1;
                todo &= todo - 1;
                const int bb = base + ((tid & ~31) + l) * kPtItems + i, cnt = __shfl_sync(~0u, back[i], l);
                const long long dst = __shfl_sync(~0u, at.a, l);
                for (int j = tid & 31; j < cnt; j += 32)
                    if (dst + j < p.free_capacity) p.free_pages[dst + j] = p.tables[bb * p.table_stride + j];
            }
            at.a += back[i];
            at.b += r[i].n;
        }
        carry.a += tot.a;
        carry.b += tot.b;
    }
    const int top = (int)(fc + carry.a > p.free_capacity ? (long long)p.free_capacity : fc + carry.a);
    if (tid == 0) {
        p.cu_new[B] = clamp_i32(carry.b);
        if (SMALL) cu_s[B] = clamp_i32(carry.b);
        if (!SMALL) static_cast<PtWorkspace*>(p.workspace)->top = top;
    }
    __syncthreads();  // the pushed pages are visible to the block

    // pages needed
    int* first_g = reinterpret_cast<int*>(static_cast<PtWorkspace*>(p.workspace) + 1);
    int* ctx_g = first_g + B;
    long long need_carry = 0;
    int late_n = 0;
    long long given_n = 0;
    for (int base = 0; base < B; base += tile) {
        PtReq r[kPtItems];
        int need[kPtItems];
        bool late[kPtItems];
        Pair64 s{0, 0};
#pragma unroll
        for (int i = 0; i < kPtItems; ++i) {
            const int b = base + tid * kPtItems + i;
            r[i] = pt_req(p, b);
            const long long last = (r[i].ctx + r[i].n + p.page_size - 1) / p.page_size;
            const long long end = b < B ? (long long)(SMALL ? cu_s[b] : p.cu_new[b]) + r[i].n : 0;
            late[i] = r[i].n > 0 && (last > p.table_width || end > p.num_rows);
            need[i] = r[i].n > 0 && !late[i] ? (int)(last - r[i].held) : 0;
            s.a += need[i];
        }
        Pair64 tot;
        long long at = need_carry + block_scan2(s, &tot, sm).a;
#pragma unroll
        for (int i = 0; i < kPtItems; ++i) {
            const int b = base + tid * kPtItems + i;
            late[i] = late[i] || (need[i] > 0 && at + need[i] > top);
            const int given = late[i] ? 0 : need[i];
            const int first = late[i] ? -1 : clamp_i32(at);
            if (b < B) {
                // seq_lens may be ctx_lens: this thread alone reads and writes entry b, the rows use the copy
                (SMALL ? first_s : first_g)[b] = first;
                (SMALL ? ctx_s : ctx_g)[b] = (int)r[i].ctx;
                p.seq_lens[b] = r[i].ended ? 0 : (int)(late[i] ? r[i].ctx : r[i].ctx + r[i].n);
                late_n += late[i];
                given_n += given;
            }
            if (SMALL) {
                if (given > 0) p.tables[b * p.table_stride + r[i].held] = p.free_pages[top - 1 - first];
                unsigned todo = __ballot_sync(~0u, given > 1);
                while (todo) {
                    const int l = __ffs(todo) - 1;
                    todo &= todo - 1;
                    const int bb = base + ((tid & ~31) + l) * kPtItems + i, cnt = __shfl_sync(~0u, given, l);
                    const int f = __shfl_sync(~0u, first, l), h = (int)__shfl_sync(~0u, r[i].held, l);
                    for (int j = 1 + (tid & 31); j < cnt; j += 32)
                        p.tables[bb * p.table_stride + h + j] = p.free_pages[top - 1 - f - j];
                }
            }
            at += need[i];
        }
        need_carry += tot.a;
    }
    if (late_n) atomicAdd(&late_s, late_n);
    Pair64 tot;
    block_scan2(Pair64{given_n, 0}, &tot, sm);  // also the barrier before the rows and late_s
    if (tid == 0) {
        *p.free_count_out = top - (int)tot.a;
        *p.deferred = late_s;
    }
    if (SMALL) {
        for (int t = tid; t < p.num_rows; t += blockDim.x) {
            const int b = pt_find([&](int i) { return cu_s[i]; }, B, t);
            pt_store(p, t, b < B ? pt_row(p, b, ctx_s[b], cu_s[b], first_s[b], top, t) : PtRow{-1, 0, -1, 0});
        }
    }
}

// The second launch: rows and new table entries of the two-launch form.
constexpr int kPrThreads = 256;
constexpr int kPrRows = 4;  // consecutive rows per thread: one search, 16- and 32-byte stores

__global__ void __launch_bounds__(kPrThreads) k_page_rows(const tt_page_tables_args p, int row_blocks) {
    pdl_wait();
    const int B = p.num_seqs, top = static_cast<const PtWorkspace*>(p.workspace)->top;
    const int* first = reinterpret_cast<const int*>(static_cast<const PtWorkspace*>(p.workspace) + 1);
    const int* ctx = first + B;
    if ((int)blockIdx.x < row_blocks) {
        const long long t0 = ((long long)blockIdx.x * kPrThreads + threadIdx.x) * kPrRows;
        if (t0 >= p.num_rows) return;
        int b = pt_find([&](int i) { return p.cu_new[i]; }, B, (int)t0);
        for (int i = 0; i < kPrRows; ++i) {
            const long long t = t0 + i;
            if (t >= p.num_rows) break;
            while (b < B && p.cu_new[b + 1] <= t) ++b;
            pt_store(p, (int)t, b < B ? pt_row(p, b, ctx[b], p.cu_new[b], first[b], top, (int)t) : PtRow{-1, 0, -1, 0});
        }
    } else {
        const int w = ((blockIdx.x - row_blocks) * kPrThreads + threadIdx.x) >> 5, lane = threadIdx.x & 31;
        const int nw = (gridDim.x - row_blocks) * (kPrThreads / 32);
        for (int b = w; b < B; b += nw) {
            const int n = p.new_lens[b];
            if (first[b] < 0 || n <= 0) continue;
            const int held = (int)(((long long)ctx[b] + p.page_size - 1) / p.page_size);
            const int given = (int)(((long long)ctx[b] + n + p.page_size - 1) / p.page_size) - held;
            for (int j = lane; j < given; j += 32)
                p.tables[b * p.table_stride + held + j] = p.free_pages[top - 1 - first[b] - j];
        }
    }
}

// ---------------------------------------------------------------------------
// Norm of queries and keys per head, rotation by position, placing
//
// A head's hd/2 channel pairs (c, c + rot/2), or (c, c + (hd-rot)/2) behind rot, are spread over G lanes,
// VEC consecutive pairs a lane and step, so both channels of a pair meet in one lane, loads are 2 x VEC
// contiguous elements, and the sum of squares is one butterfly over G lanes.  A group of G lanes keeps the
// cos, sin and weights of its channels in registers and walks `chunk` heads of one row, so the tables are
// read once a row and chunk, not once a head.  Bytes of q, k, v in and out are the floor.
// ---------------------------------------------------------------------------
template <typename T> struct Elem;
template <> struct Elem<float> {
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};

template <typename T, int N>
struct alignas(sizeof(T) * N <= 16 ? sizeof(T) * N : 16) Pack {
    T x[N];
};

template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, float* f) {
    const Pack<T, VEC> v = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = Elem<T>::up(v.x[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float* f) {
    Pack<T, VEC> v;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v.x[i] = Elem<T>::down(f[i]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = v;
}
template <typename T>
__device__ __forceinline__ float load_any(const void* p, long long i, bool f32) {
    return f32 ? static_cast<const float*>(p)[i] : Elem<T>::up(static_cast<const T*>(p)[i]);
}

template <typename T, typename TQ, typename TKV, int VEC, int STEPS>
__global__ void __launch_bounds__(256) k_norm_rope(const tt_qk_norm_rope_args p, int glog, int chunk, int chunks) {
    const int G = 1 << glog, lane = threadIdx.x & (G - 1);
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> glog;
    const long long row = item / chunks;
    // groups past the end keep running (the butterflies are warp-wide) without loads or stores
    const bool in = row < p.num_rows;
    const int h0 = (int)(item % chunks) * chunk;
    const int heads = p.num_q_heads + (p.v ? 2 : 1) * p.num_kv_heads;
    const int hd = p.head_dim, half = p.rot_dim >> 1, rest = (hd - p.rot_dim) >> 1;

    bool live = in;
    long long page = row;
    int tok = 0;
    if (in && p.slots) {
        const long long s = p.slots[row];
        live = s >= 0 && s < p.num_pages * p.page_size;
        page = s / p.page_size;
        tok = (int)(s % p.page_size);
    }
    long long pos = row;
    if (in && p.positions) pos = p.positions_i64 ? static_cast<const long long*>(p.positions)[row]
                                                 : (long long)static_cast<const int*>(p.positions)[row];
    const bool pos_ok = pos >= 0 && pos < p.table_rows;

    int ca[STEPS], cb[STEPS];  // first channels of this lane's runs of pairs, -1: none
    float co[STEPS][VEC], si[STEPS][VEC], wq[2][STEPS][VEC], wk[2][STEPS][VEC];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int pr = (lane + s * G) * VEC;
        ca[s] = pr < half ? pr : pr < half + rest ? pr + half : -1;
        cb[s] = pr < half ? pr + half : ca[s] + rest;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            co[s][i] = 1.f;
            si[s][i] = 0.f;
            if (live && pr < half) {
                co[s][i] = pos_ok ? load_any<T>(p.cos, pos * p.cos_stride + pr + i, p.table_dtype == TT_DTYPE_F32) : NAN;
                si[s][i] = pos_ok ? load_any<T>(p.sin, pos * p.sin_stride + pr + i, p.table_dtype == TT_DTYPE_F32) : NAN;
            }
            const bool use = live && ca[s] >= 0, f = p.weight_dtype == TT_DTYPE_F32;
            wq[0][s][i] = use && p.q_weight ? load_any<T>(p.q_weight, ca[s] + i, f) : 1.f;
            wq[1][s][i] = use && p.q_weight ? load_any<T>(p.q_weight, cb[s] + i, f) : 1.f;
            wk[0][s][i] = use && p.k_weight ? load_any<T>(p.k_weight, ca[s] + i, f) : 1.f;
            wk[1][s][i] = use && p.k_weight ? load_any<T>(p.k_weight, cb[s] + i, f) : 1.f;
        }
    }
    const float inv = 1.f / (float)hd;

#pragma unroll 2
    for (int hh = 0; hh < chunk; ++hh) {
        const int h = h0 + hh;
        const bool is_q = h < p.num_q_heads, is_k = !is_q && h < p.num_q_heads + p.num_kv_heads;
        const bool on = live && h < heads;
        const int kh = is_q ? h : is_k ? h - p.num_q_heads : h - p.num_q_heads - p.num_kv_heads;
        const T* src = is_q ? static_cast<const T*>(p.q) + row * p.q_row_stride + kh * p.q_head_stride
                     : is_k ? static_cast<const T*>(p.k) + row * p.k_row_stride + kh * p.k_head_stride
                            : static_cast<const T*>(p.v) + row * p.v_row_stride + kh * p.v_head_stride;
        float a[STEPS][VEC], b[STEPS][VEC];
        float ss = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (on && ca[s] >= 0) {
                load_pack<T, VEC>(src + ca[s], a[s]);
                load_pack<T, VEC>(src + cb[s], b[s]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) a[s][i] = b[s][i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss += a[s][i] * a[s][i] + b[s][i] * b[s][i];
        }
        // groups of one warp may be at heads of different kinds: all lanes take the butterfly
        for (int d = G >> 1; d; d >>= 1) ss += __shfl_xor_sync(~0u, ss, d);
        if (is_q ? p.q_weight != nullptr : is_k && p.k_weight != nullptr) {
            const float r = rsqrtf(ss * inv + p.eps);
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a[s][i] *= r * (is_q ? wq[0][s][i] : wk[0][s][i]);
                    b[s][i] *= r * (is_q ? wq[1][s][i] : wk[1][s][i]);
                }
        }
        if (!on) continue;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (ca[s] < 0) continue;
            float x[VEC], y[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const bool turn = (is_q || is_k) && ca[s] < half;
                x[i] = turn ? a[s][i] * co[s][i] - b[s][i] * si[s][i] : a[s][i];
                y[i] = turn ? b[s][i] * co[s][i] + a[s][i] * si[s][i] : b[s][i];
            }
            if (is_q) {
                TQ* d = static_cast<TQ*>(p.q_out) + row * p.q_out_row_stride + kh * p.q_out_head_stride;
                store_pack<TQ, VEC>(d + ca[s], x);
                store_pack<TQ, VEC>(d + cb[s], y);
            } else {
                TKV* d = is_k ? static_cast<TKV*>(p.k_dst) + page * p.k_page_stride + tok * p.k_token_stride + kh * p.k_dst_head_stride
                              : static_cast<TKV*>(p.v_dst) + page * p.v_page_stride + tok * p.v_token_stride + kh * p.v_dst_head_stride;
                store_pack<TKV, VEC>(d + ca[s], x);
                store_pack<TKV, VEC>(d + cb[s], y);
            }
        }
    }
}

template <typename T, typename TQ, typename TKV>
static cudaError_t launch_norm_rope(const tt_qk_norm_rope_args& a, bool vec, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int pairs = a.head_dim / 2, width = vec ? V : 1;
    int glog = 0;
    while (glog < 5 && (1 << glog) * width < pairs) ++glog;
    const int G = 1 << glog, steps = (pairs + G * width - 1) / (G * width);
    // Heads a group walks: as many as leave about four warps an SM partition, so that tables and weights
    // are read seldom in a long prompt and a single token still uses a group per head.
    const int heads = a.num_q_heads + (a.v ? 2 : 1) * a.num_kv_heads;
    int chunk = heads;
    while (chunk > 1 && (long long)a.num_rows * ((heads + chunk - 1) / chunk) * G < 148LL * 512) chunk = (chunk + 1) / 2;
    const int chunks = (heads + chunk - 1) / chunk;
    const long long threads = (long long)a.num_rows * chunks * G;
    const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
#define TT_NR(VV, SS) launch(k_norm_rope<T, TQ, TKV, VV, SS>, grid, block, 0, st, false, a, glog, chunk, chunks)
    if (vec) return steps <= 1 ? TT_NR(V, 1) : TT_NR(V, 2);
    return steps <= 2 ? TT_NR(1, 2) : TT_NR(1, 8);
#undef TT_NR
}

template <typename T>
static cudaError_t launch_norm_rope_out(const tt_qk_norm_rope_args& a, bool vec, cudaStream_t st) {
    const bool qf = a.q_dtype == TT_DTYPE_F32, kf = a.kv_dtype == TT_DTYPE_F32;
    if (qf) return kf ? launch_norm_rope<T, float, float>(a, vec, st) : launch_norm_rope<T, float, T>(a, vec, st);
    return kf ? launch_norm_rope<T, T, float>(a, vec, st) : launch_norm_rope<T, T, T>(a, vec, st);
}

static bool dtype_ok(int d) { return d == TT_DTYPE_F32 || d == TT_DTYPE_BF16 || d == TT_DTYPE_F16; }
static int dtype_bytes(int d) { return d == TT_DTYPE_F32 ? 4 : 2; }

}  // namespace tt

using namespace tt;

extern "C" {

size_t tt_page_tables_workspace(int num_seqs, int num_rows) {
    if (num_seqs < 0 || num_rows < 0 || pt_small(num_seqs, num_rows)) return 0;
    return sizeof(PtWorkspace) + 2 * sizeof(int) * (size_t)num_seqs;
}

tt_status tt_page_tables(const tt_page_tables_args* args, void* stream) {
    if (!args) return set_error(TT_ERR_INVALID_ARGUMENT, "page_tables: null pointer argument.");
    const tt_page_tables_args& a = *args;
    if (a.num_seqs < 0 || a.num_rows < 0 || a.free_capacity < 0 || a.table_width < 0)
        return set_error(TT_ERR_INVALID_ARGUMENT, "page_tables: sizes must be non-negative.");
    if (a.page_size <= 0) return set_error(TT_ERR_INVALID_ARGUMENT, "page_tables: page_size must be positive.");
    if ((long long)a.table_width * a.page_size > INT_MAX)
        return set_error(TT_ERR_UNSUPPORTED, "page_tables: table_width * page_size must not exceed 2^31 - 1.");
    if (a.num_seqs > 0 && a.table_stride < a.table_width)
        return set_error(TT_ERR_INVALID_ARGUMENT, "page_tables: table_stride is below table_width.");
    if (!a.free_count || !a.free_count_out || !a.cu_new || !a.deferred ||
        (a.num_seqs > 0 && (!a.ctx_lens || !a.new_lens || !a.seq_lens || (a.table_width > 0 && !a.tables))) ||
        (a.free_capacity > 0 && !a.free_pages) ||
        (a.num_rows > 0 && (!a.slots || !a.positions || !a.row_seq || !a.row_lens)))
        return set_error(TT_ERR_INVALID_ARGUMENT, "page_tables: null pointer argument.");
    const cudaStream_t st = (cudaStream_t)stream;
    if (pt_small(a.num_seqs, a.num_rows)) {
        const int threads = a.num_seqs <= 256 * kPtItems && a.num_rows <= 1024 ? 256 : kPtThreads;
        return check_cuda(launch(k_page_scan<true>, dim3(1), dim3(threads), (3 * (size_t)a.num_seqs + 1) * sizeof(int),
                                 st, false, a), "page_tables");
    }
    if (!a.workspace || ((uintptr_t)a.workspace & 7))
        return set_error(TT_ERR_INVALID_ARGUMENT, "page_tables: workspace is missing or not 8-byte aligned.");
    tt_status s = check_cuda(launch(k_page_scan<false>, dim3(1), dim3(kPtThreads), 0, st, false, a), "page_tables");
    if (s != TT_OK) return s;
    const int row_blocks = (int)(((long long)a.num_rows + kPrThreads * kPrRows - 1) / (kPrThreads * kPrRows));
    int seq_blocks = (a.num_seqs + kPrThreads / 32 - 1) / (kPrThreads / 32);
    seq_blocks = seq_blocks > 148 * 8 ? 148 * 8 : seq_blocks;
    return check_cuda(launch(k_page_rows, dim3((unsigned)(row_blocks + seq_blocks)), dim3(kPrThreads), 0, st, true, a,
                             row_blocks), "page_tables");
}

tt_status tt_qk_norm_rope(const tt_qk_norm_rope_args* args, void* stream) {
    if (!args) return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: null pointer argument.");
    const tt_qk_norm_rope_args& a = *args;
    if (a.num_rows < 0 || a.num_q_heads <= 0 || a.num_kv_heads <= 0)
        return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: num_rows must be non-negative, the head counts positive.");
    if (a.head_dim <= 0 || (a.head_dim & 1) || a.head_dim > 512)
        return set_error(TT_ERR_UNSUPPORTED, "qk_norm_rope: head_dim must be even and at most 512.");
    if (a.rot_dim < 0 || (a.rot_dim & 1) || a.rot_dim > a.head_dim)
        return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: rot_dim must be even and within head_dim.");
    if (!dtype_ok(a.dtype) || (a.q_dtype != a.dtype && a.q_dtype != TT_DTYPE_F32) ||
        (a.kv_dtype != a.dtype && a.kv_dtype != TT_DTYPE_F32) ||
        (a.weight_dtype != a.dtype && a.weight_dtype != TT_DTYPE_F32) ||
        (a.table_dtype != a.dtype && a.table_dtype != TT_DTYPE_F32))
        return set_error(TT_ERR_UNSUPPORTED, "qk_norm_rope: unsupported data type combination.");
    if (a.slots && (a.page_size <= 0 || a.num_pages < 0))
        return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: page_size must be positive, num_pages non-negative.");
    if (a.table_rows < 0) return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: table_rows must be non-negative.");
    if ((a.v == nullptr) != (a.v_dst == nullptr))
        return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: v and v_dst come together.");
    if (a.num_rows == 0) return TT_OK;
    if (!a.q || !a.k || !a.q_out || !a.k_dst || (a.rot_dim > 0 && (!a.cos || !a.sin)))
        return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: null pointer argument.");
    if (a.rot_dim > 0 && !a.positions && a.table_rows < a.num_rows)
        return set_error(TT_ERR_INVALID_ARGUMENT, "qk_norm_rope: without positions the tables need a row for each row.");
    if ((long long)a.num_rows * (a.num_q_heads + 2LL * a.num_kv_heads) > (1LL << 31))
        return set_error(TT_ERR_UNSUPPORTED, "qk_norm_rope: more than 2^31 heads in one call.");
    // 16-byte loads need runs of pairs that fill them, on both sides of the rotation's border
    const int es = dtype_bytes(a.dtype), V = 16 / es;
    bool vec = (a.rot_dim / 2) % V == 0 && ((a.head_dim - a.rot_dim) / 2) % V == 0 && a.head_dim % V == 0;
    const auto fits = [&](const void* ptr, int dt, long long s0, long long s1, long long s2) {
        const int w = dtype_bytes(dt) * V > 16 ? 16 / dtype_bytes(dt) : V;
        return ((uintptr_t)ptr & 15) == 0 && s0 % w == 0 && s1 % w == 0 && s2 % w == 0;
    };
    vec = vec && fits(a.q, a.dtype, a.q_row_stride, a.q_head_stride, 0) && fits(a.k, a.dtype, a.k_row_stride, a.k_head_stride, 0) &&
          fits(a.q_out, a.q_dtype, a.q_out_row_stride, a.q_out_head_stride, 0) &&
          fits(a.k_dst, a.kv_dtype, a.k_page_stride, a.k_token_stride, a.k_dst_head_stride);
    if (a.v)
        vec = vec && fits(a.v, a.dtype, a.v_row_stride, a.v_head_stride, 0) &&
              fits(a.v_dst, a.kv_dtype, a.v_page_stride, a.v_token_stride, a.v_dst_head_stride);
    const cudaStream_t st = (cudaStream_t)stream;
    cudaError_t e;
    if (a.dtype == TT_DTYPE_F32) e = launch_norm_rope<float, float, float>(a, vec, st);
    else if (a.dtype == TT_DTYPE_BF16) e = launch_norm_rope_out<__nv_bfloat16>(a, vec, st);
    else e = launch_norm_rope_out<__half>(a, vec, st);
    return check_cuda(e, "qk_norm_rope");
}

}  // extern "C"
