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

// Pages that hold x tokens (x below 2^32: so may be the pages, where a page is one token).
__device__ __forceinline__ long long pt_pages(const tt_page_tables_args& p, long long x) {
    const uint32_t u = (uint32_t)x, P = (uint32_t)p.page_size;
    return (long long)(u / P) + (u % P != 0);
}

struct PtReq {
    long long ctx, held, n;  // tokens held, pages held, new tokens
    bool ended;
};
__device__ __forceinline__ PtReq pt_req(const tt_page_tables_args& p, int b) {
    PtReq r{0, 0, 0, false};
    if (b < p.num_seqs) {
        const int c = p.ctx_lens[b], n = p.new_lens[b];
        r.ctx = c > 0 ? c : 0;
        r.held = pt_pages(p, r.ctx);
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
    const int held = (int)pt_pages(p, ctx);
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
            // the warp copies the pages of its ended requests, four requests at a time, eight lanes each (their
            // table rows are not written in this call)
            unsigned todo = __ballot_sync(~0u, back[i] > 0);
            while (todo) {
                unsigned rest = todo;
                for (int k = (tid & 31) >> 3; k && rest; --k) rest &= rest - 1;
                const int l = rest ? __ffs(rest) - 1 : 0;
                const int bb = base + ((tid & ~31) + l) * kPtItems + i, cnt = __shfl_sync(~0u, back[i], l);
                const long long dst = __shfl_sync(~0u, at.a, l);
                const int32_t* row = p.tables + bb * p.table_stride;
                if (rest) {
#pragma unroll 4
                    for (int j = tid & 7; j < cnt; j += 8) {
                        const int page = __ldg(row + j);
                        if (dst + j < p.free_capacity) p.free_pages[dst + j] = page;
                    }
                }
                for (int k = 0; k < 4; ++k) todo &= todo - 1;
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
            const long long last = pt_pages(p, r[i].ctx + r[i].n);
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

__global__ void __launch_bounds__(kPrThreads) k_page_rows(const tt_page_tables_args p, int row_blocks, int wide) {
    pdl_wait();
    const int B = p.num_seqs, top = static_cast<const PtWorkspace*>(p.workspace)->top;
    const int* first = reinterpret_cast<const int*>(static_cast<const PtWorkspace*>(p.workspace) + 1);
    const int* ctx = first + B;
    if ((int)blockIdx.x < row_blocks) {
        const long long t0 = ((long long)blockIdx.x * kPrThreads + threadIdx.x) * kPrRows;
        if (t0 >= p.num_rows) return;
        int b = pt_find([&](int i) { return p.cu_new[i]; }, B, (int)t0);
        PtRow r[kPrRows];
#pragma unroll
        for (int i = 0; i < kPrRows; ++i) {
            const long long t = t0 + i;
            while (b < B && p.cu_new[b + 1] <= t) ++b;
            r[i] = b < B ? pt_row(p, b, ctx[b], p.cu_new[b], first[b], top, (int)t) : PtRow{-1, 0, -1, 0};
        }
        if (t0 + kPrRows <= p.num_rows && wide) {
            reinterpret_cast<longlong2*>(p.slots + t0)[0] = make_longlong2(r[0].slot, r[1].slot);
            reinterpret_cast<longlong2*>(p.slots + t0)[1] = make_longlong2(r[2].slot, r[3].slot);
            *reinterpret_cast<int4*>(p.positions + t0) = make_int4(r[0].pos, r[1].pos, r[2].pos, r[3].pos);
            *reinterpret_cast<int4*>(p.row_seq + t0) = make_int4(r[0].seq, r[1].seq, r[2].seq, r[3].seq);
            *reinterpret_cast<int4*>(p.row_lens + t0) = make_int4(r[0].len, r[1].len, r[2].len, r[3].len);
        } else {
#pragma unroll
            for (int i = 0; i < kPrRows; ++i)
                if (t0 + i < p.num_rows) pt_store(p, (int)(t0 + i), r[i]);
        }
    } else {
        const int w = ((blockIdx.x - row_blocks) * kPrThreads + threadIdx.x) >> 5, lane = threadIdx.x & 31;
        const int nw = (gridDim.x - row_blocks) * (kPrThreads / 32);
        for (int b = w; b < B; b += nw) {
            const int n = p.new_lens[b];
            if (first[b] < 0 || n <= 0) continue;
            const int held = (int)pt_pages(p, ctx[b]), given = (int)(pt_pages(p, (long long)ctx[b] + n) - held);
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
// cos, sin and weights of its channels in registers and walks up to `chunk` heads of one kind (query, key or
// value) of one row, so the tables are read once a row and chunk, not once a head, and it asks for `kBatch`
// heads before it works on the first.  Bytes of q, k, v in and out are the floor.
// ---------------------------------------------------------------------------
template <typename T> struct Elem;  // float32 of a value and back, one at a time and as the halves of a word
template <> struct Elem<float> {
    static __device__ __forceinline__ float up(float x) { return x; }
    static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
    static __device__ __forceinline__ float2 up2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t down2(float x, float y) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
        return r;
    }
};
template <> struct Elem<__half> {
    static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
    static __device__ __forceinline__ float2 up2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t down2(float x, float y) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
        return r;
    }
};

// N values of T as the 16-byte words that memory moves them in (arrays of 16-bit classes are moved one by one);
// N = 1 is the unaligned form.
template <typename T, int N> struct Pack {
    static constexpr int kWords = N * (int)sizeof(T) / 16;
    uint4 w[kWords];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = reinterpret_cast<const uint4*>(p)[k];
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int k = 0; k < kWords; ++k) reinterpret_cast<uint4*>(p)[k] = w[k];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[k] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void up(float* f) const {
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
            const uint32_t v[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    f[4 * k + i] = __uint_as_float(v[i]);
                } else {
                    const float2 x = Elem<T>::up2(v[i]);
                    f[8 * k + 2 * i] = x.x;
                    f[8 * k + 2 * i + 1] = x.y;
                }
            }
        }
    }
    __device__ __forceinline__ void down(const float* f) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) v[i] = __float_as_uint(f[4 * k + i]);
                else v[i] = Elem<T>::down2(f[8 * k + 2 * i], f[8 * k + 2 * i + 1]);
            }
            w[k] = make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
};
template <typename T> struct Pack<T, 1> {
    T x;
    __device__ __forceinline__ void load(const T* p) { x = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = x; }
    __device__ __forceinline__ void zero() { x = Elem<T>::down(0.f); }
    __device__ __forceinline__ void up(float* f) const { *f = Elem<T>::up(x); }
    __device__ __forceinline__ void down(const float* f) { x = Elem<T>::down(*f); }
};

// x += a b, y += c d in one instruction
__device__ __forceinline__ void fma2(float& x, float& y, float a, float c, float b, float d) {
    asm("{\n.reg .b64 v, a, b;\nmov.b64 v, {%0, %1};\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\n"
        "fma.rn.f32x2 v, a, b, v;\nmov.b64 {%0, %1}, v;\n}" : "+f"(x), "+f"(y) : "f"(a), "f"(c), "f"(b), "f"(d));
}

template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, float* f) {
    Pack<T, VEC> v;
    v.load(p);
    v.up(f);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float* f) {
    Pack<T, VEC> v;
    v.down(f);
    v.store(p);
}
template <typename T>
__device__ __forceinline__ float load_any(const void* p, long long i, bool f32) {
    return f32 ? static_cast<const float*>(p)[i] : Elem<T>::up(static_cast<const T*>(p)[i]);
}

// N values of T or float32 from p[i] on; `aligned` when 16-byte loads may be used.
template <typename T, int N>
__device__ __forceinline__ void load_row(const void* p, long long i, bool f32, bool aligned, float* f) {
    if (N > 1 && aligned) {
        if (f32) load_pack<float, N>(static_cast<const float*>(p) + i, f);
        else load_pack<T, N>(static_cast<const T*>(p) + i, f);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = load_any<T>(p, i + k, f32);
    }
}

// Measured for 32k rows of 32 + 8 + 8 heads of 128 (floor 125 us at the copy rate): batches of 1, 2, 4, 8 heads
// 240, 200, 177, 280 us (one head leaves too little in flight, eight spend the registers that warps need);
// 4, 8, 16 heads a group 230 (batch 2), 177, 187; blocks of 256 and 128 threads 177, 172.
constexpr int kNrChunk = 8, kNrBatch = 4, kNrThreads = 1024, kNrBlock = 128;

// Groups of a row: cq for the queries, then ck for the keys, then (with v) ck for the values; group c of a kind
// takes heads c, c + cq (or ck), ..., so that the groups of a warp are at neighbouring heads together.
struct NrShape {
    int glog, chunk, cq, ck, chunks;
    int table_aligned, weight_aligned;
};

// With a row's cos, sin and a head's weights, x' = r (A x - B y) and y' = r (C y + D x) for each pair, where
// A = w_x cos, B = w_y sin, C = w_y cos, D = w_x sin and r = rsqrt(mean square + eps).  FULL: every channel is
// rotated (else the others take x' = r A x, without the partner, which may be infinite).
template <typename T, typename TQ, typename TKV, int VEC, int STEPS, int kBatch, bool FULL>
__global__ void __launch_bounds__(kNrBlock) k_norm_rope(const tt_qk_norm_rope_args p, const NrShape sh) {
    const int G = 1 << sh.glog, lane = threadIdx.x & (G - 1);
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> sh.glog;
    const long long row = item / sh.chunks;
    const int ch = (int)(item % sh.chunks);
    const int kind = ch < sh.cq ? 0 : ch < sh.cq + sh.ck ? 1 : 2;
    const int h0 = kind == 0 ? ch : kind == 1 ? ch - sh.cq : ch - sh.cq - sh.ck, hstep = kind == 0 ? sh.cq : sh.ck;
    const int hd = p.head_dim, half = p.rot_dim >> 1, rest = (hd - p.rot_dim) >> 1;

    // groups past the end keep running (the butterflies are warp-wide) without loads or stores
    bool live = row < p.num_rows;
    long long page = row;
    int tok = 0;
    if (live && p.slots) {
        const long long s = p.slots[row];
        live = s >= 0 && s < p.num_pages * p.page_size;
        page = s / p.page_size;
        tok = (int)(s % p.page_size);
    }
    // this group's heads: h0, h0 + hstep, ...
    const int mine = live ? ((kind == 0 ? p.num_q_heads : p.num_kv_heads) - h0 + hstep - 1) / hstep : 0;
    const T* src = kind == 0 ? static_cast<const T*>(p.q) + row * p.q_row_stride + h0 * p.q_head_stride
                 : kind == 1 ? static_cast<const T*>(p.k) + row * p.k_row_stride + h0 * p.k_head_stride
                             : static_cast<const T*>(p.v) + row * p.v_row_stride + h0 * p.v_head_stride;
    const long long src_step = hstep * (kind == 0 ? p.q_head_stride : kind == 1 ? p.k_head_stride : p.v_head_stride);
    TQ* dq = static_cast<TQ*>(p.q_out) + row * p.q_out_row_stride + h0 * p.q_out_head_stride;
    TKV* dkv = kind == 1 ? static_cast<TKV*>(p.k_dst) + page * p.k_page_stride + tok * p.k_token_stride + h0 * p.k_dst_head_stride
                         : static_cast<TKV*>(p.v_dst) + page * p.v_page_stride + tok * p.v_token_stride + h0 * p.v_dst_head_stride;
    const long long dst_step = hstep * (kind == 0 ? p.q_out_head_stride : kind == 1 ? p.k_dst_head_stride : p.v_dst_head_stride);

    int ca[STEPS], cb[STEPS];  // first channels of this lane's runs of pairs, -1: none
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int pr = (lane + s * G) * VEC;
        ca[s] = pr < half ? pr : pr < half + rest ? pr + half : -1;
        cb[s] = pr < half ? pr + half : ca[s] + rest;
    }
    // the first heads are on their way before the tables are asked for
    Pack<T, VEC> ra[kBatch][STEPS], rb[kBatch][STEPS];
    const auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                if (i + u < mine && ca[s] >= 0) {
                    ra[u][s].load(src + ca[s]);
                    rb[u][s].load(src + cb[s]);
                } else {
                    ra[u][s].zero();
                    rb[u][s].zero();
                }
            }
            src += src_step;
        }
    };
    fetch(0);

    const void* weight = kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr;
    float A[STEPS][VEC], B[STEPS][VEC], C[STEPS][VEC], D[STEPS][VEC];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        float co[VEC], si[VEC], wa[VEC], wb[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) co[i] = wa[i] = wb[i] = 1.f, si[i] = 0.f;
        const int pr = (lane + s * G) * VEC;
        if (mine > 0 && kind < 2 && pr < half) {
            long long pos = row;
            if (p.positions) pos = p.positions_i64 ? static_cast<const long long*>(p.positions)[row]
                                                   : (long long)static_cast<const int*>(p.positions)[row];
            const bool f32 = p.table_dtype == TT_DTYPE_F32;
            if (pos >= 0 && pos < p.table_rows) {
                load_row<T, VEC>(p.cos, pos * p.cos_stride + pr, f32, sh.table_aligned, co);
                load_row<T, VEC>(p.sin, pos * p.sin_stride + pr, f32, sh.table_aligned, si);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) co[i] = si[i] = NAN;
            }
        }
        if (mine > 0 && weight && ca[s] >= 0) {
            const bool f32 = p.weight_dtype == TT_DTYPE_F32;
            load_row<T, VEC>(weight, ca[s], f32, sh.weight_aligned, wa);
            load_row<T, VEC>(weight, cb[s], f32, sh.weight_aligned, wb);
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            A[s][i] = wa[i] * co[i];
            B[s][i] = wb[i] * si[i];
            C[s][i] = wb[i] * co[i];
            D[s][i] = wa[i] * si[i];
        }
    }
    const float inv = 1.f / (float)hd;

    for (int i = 0; i < sh.chunk; i += kBatch) {
        if (i) fetch(i);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            float a[STEPS][VEC], b[STEPS][VEC], s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                ra[u][s].up(a[s]);
                rb[u][s].up(b[s]);
#pragma unroll
                for (int k = 0; k < VEC; ++k) fma2(s0, s1, a[s][k], b[s][k], a[s][k], b[s][k]);
            }
            // groups of one warp may be at heads of different kinds: all lanes take the butterfly
            float ss = s0 + s1;
            for (int d = G >> 1; d; d >>= 1) ss += __shfl_xor_sync(~0u, ss, d);
            const float r = weight ? rsqrtf(ss * inv + p.eps) : 1.f;
            if (i + u < mine) {
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    if (ca[s] < 0) continue;
                    float x[VEC], y[VEC];
                    if (kind < 2) {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) {
                            x[k] = A[s][k] * a[s][k];
                            y[k] = C[s][k] * b[s][k];
                            if (FULL || ca[s] < half) {
                                x[k] = fmaf(-B[s][k], b[s][k], x[k]);
                                y[k] = fmaf(D[s][k], a[s][k], y[k]);
                            }
                            x[k] *= r;
                            y[k] *= r;
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) x[k] = a[s][k], y[k] = b[s][k];
                    }
                    if (kind == 0) {
                        store_pack<TQ, VEC>(dq + ca[s], x);
                        store_pack<TQ, VEC>(dq + cb[s], y);
                    } else {
                        store_pack<TKV, VEC>(dkv + ca[s], x);
                        store_pack<TKV, VEC>(dkv + cb[s], y);
                    }
                }
            }
            dq += dst_step;
            dkv += dst_step;
        }
    }
}

template <typename T, typename TQ, typename TKV>
static cudaError_t launch_norm_rope(const tt_qk_norm_rope_args& a, bool vec, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const int pairs = a.head_dim / 2, width = vec ? V : 1;
    NrShape sh = {};
    while (sh.glog < 5 && (1 << sh.glog) * width < pairs) ++sh.glog;
    const int G = 1 << sh.glog, steps = (pairs + G * width - 1) / (G * width);
    // Heads a group walks: up to kNrChunk, fewer while the groups would not fill the GPU, so that a single token
    // uses a group per head.
    const auto chunks = [&](int c) { return (a.num_q_heads + c - 1) / c + (a.v ? 2 : 1) * ((a.num_kv_heads + c - 1) / c); };
    sh.chunk = kNrChunk;
    while (sh.chunk > 1 && (long long)a.num_rows * chunks(sh.chunk) * G < 148LL * kNrThreads) sh.chunk /= 2;
    sh.cq = (a.num_q_heads + sh.chunk - 1) / sh.chunk;
    sh.ck = (a.num_kv_heads + sh.chunk - 1) / sh.chunk;
    sh.chunks = chunks(sh.chunk);
    const int te = a.table_dtype == TT_DTYPE_F32 ? 4 : V;  // elements of a 16-byte load
    sh.table_aligned = !(((uintptr_t)a.cos | (uintptr_t)a.sin) & 15) && a.cos_stride % te == 0 && a.sin_stride % te == 0;
    sh.weight_aligned = !(((uintptr_t)a.q_weight | (uintptr_t)a.k_weight) & 15);
    const long long threads = (long long)a.num_rows * sh.chunks * G;
    const dim3 grid((unsigned)((threads + kNrBlock - 1) / kNrBlock)), block(kNrBlock);
#define TT_NR(VV, SS, BB, FF) launch(k_norm_rope<T, TQ, TKV, VV, SS, BB, FF>, grid, block, 0, st, false, a, sh)
    if (vec && steps == 1 && a.rot_dim == a.head_dim) return sh.chunk == 1 ? TT_NR(V, 1, 1, true) : TT_NR(V, 1, kNrBatch, true);
    if (vec) return steps > 1 ? TT_NR(V, 2, 1, false) : TT_NR(V, 1, kNrBatch, false);
    return steps <= 2 ? TT_NR(1, 2, 1, false) : TT_NR(1, 8, 1, false);
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
    const int wide = !(((uintptr_t)a.slots | (uintptr_t)a.positions | (uintptr_t)a.row_seq | (uintptr_t)a.row_lens) & 15);
    int seq_blocks = (a.num_seqs + kPrThreads / 32 - 1) / (kPrThreads / 32);
    seq_blocks = seq_blocks > 148 * 8 ? 148 * 8 : seq_blocks;
    return check_cuda(launch(k_page_rows, dim3((unsigned)(row_blocks + seq_blocks)), dim3(kPrThreads), 0, st, true, a,
                             row_blocks, wide), "page_tables");
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
