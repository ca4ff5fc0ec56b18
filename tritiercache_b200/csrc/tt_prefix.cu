// tt_prefix.cu -- attention of a batch over a shared prefix and each row's own pages (C ABI:
// tt_shared_prefix_attention).
#include <limits.h>

#include <atomic>

#include "tt_prefix_shared.cuh"

namespace tt {

static_assert(sizeof(tt_shared_prefix_args) == 208, "packed by paged.py");

constexpr int kSms = 148;
constexpr long long kWalk = 1 << 23;
constexpr int kCross = 4;  // measured: 7 tiles in 30 us, 7 in two spans in 40 (384 rows of heads on 8k)

// All kernels ask for the whole of an SM's shared memory: the passes' CTAs share one, and an SM that has to
// divide its memory anew between two kernels has to run dry first.  Once per kernel and device.
template <auto Kern>
static cudaError_t set_smem(size_t bytes) {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
    if (e != cudaSuccess || (done.load(std::memory_order_acquire) & bit)) return e;
    e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(Kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
}

template <typename T, int HD, int NB>
static cudaError_t launch_rows(const PrefixParams& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    constexpr int ST = HD == 64 ? 4 : 2;
    constexpr size_t smem = row_smem<HD, NB, ST>();
    auto* kern = k_prefix_rows<T, HD, NB, ST>;
    const cudaError_t e = set_smem<k_prefix_rows<T, HD, NB, ST>>(smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(p.a.num_rows * p.splits), (unsigned)(p.a.num_kv_heads * p.head_tiles));
    return launch(kern, grid, dim3(kRowWarps * 32), smem, st, !p.walk_prefix, p, km, vm);
}

template <typename T>
static cudaError_t launch_rows_t(const PrefixParams& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    const bool one = p.group <= 8;
    if (p.a.head_dim == 64) return one ? launch_rows<T, 64, 1>(p, km, vm, st) : launch_rows<T, 64, 2>(p, km, vm, st);
    return one ? launch_rows<T, 128, 1>(p, km, vm, st) : launch_rows<T, 128, 2>(p, km, vm, st);
}

template <typename T, int HD, int W>
static cudaError_t launch_join_w(const PrefixParams& p, cudaStream_t st) {
    const cudaError_t e = set_smem<k_prefix_join<T, HD, W>>(0);
    if (e != cudaSuccess) return e;
    const long long warps = (long long)p.a.num_rows * p.a.num_q_heads * W;
    return launch(k_prefix_join<T, HD, W>, dim3((unsigned)((warps + kJoinWarps - 1) / kJoinWarps)), dim3(kJoinWarps * 32), 0, st, true, p);
}
template <typename T, int HD>
static cudaError_t launch_join(const PrefixParams& p, cudaStream_t st) {
    // a warp loads eight partials at once
    const int n = p.splits + (p.walk_prefix ? 0 : (p.kv_tiles / p.per + 1) * (p.tile_rows == kPsTile ? 2 : 1));
    return n <= 8 ? launch_join_w<T, HD, 1>(p, st) : n <= 16 ? launch_join_w<T, HD, 2>(p, st)
         : n <= 32 ? launch_join_w<T, HD, 4>(p, st) : launch_join_w<T, HD, 8>(p, st);
}
template <typename T>
static cudaError_t launch_join_t(const PrefixParams& p, cudaStream_t st) {
    return p.a.head_dim == 64 ? launch_join<T, 64>(p, st) : launch_join<T, 128>(p, st);
}

static tt_status check_prefix(const tt_shared_prefix_args* args) {
    if (!args) return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: null pointer argument.");
    const tt_shared_prefix_args& a = *args;
    if (a.num_rows < 0 || a.num_q_heads <= 0 || a.num_kv_heads <= 0 || a.num_q_heads % a.num_kv_heads)
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: num_rows must be non-negative and num_q_heads a "
                         "positive multiple of num_kv_heads.");
    if (a.head_dim != 64 && a.head_dim != 128)
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: head_dim must be 64 or 128.");
    if (a.dtype != TT_DTYPE_BF16 && a.dtype != TT_DTYPE_F16)
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: dtype must be bf16 or f16.");
    if (a.page_size < 16 || a.page_size > 32768 || (a.page_size & (a.page_size - 1)))
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: page_size must be a power of two from 16 to 32768.");
    if (a.num_pages <= 0 || a.prefix_len < 0 || a.table_width < 0 || a.num_tables < 0)
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: sizes must be non-negative, num_pages positive.");
    if ((long long)a.table_width * a.page_size > INT_MAX)
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: table_width * page_size must not exceed 2^31 - 1.");
    if (!a.row_seq && a.num_tables < a.num_rows)
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: without row_seq the tables need a row for each row.");
    if ((long long)a.num_rows * a.num_q_heads > (1 << 26))
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: more than 2^26 query heads in one call.");
    if (a.num_q_heads > 65535) return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: more than 65535 query heads.");
    if (!(a.scale > -INFINITY && a.scale < INFINITY))
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: scale must be finite.");
    if ((a.k_page_stride | a.k_token_stride | a.k_head_stride | a.v_page_stride | a.v_token_stride | a.v_head_stride) & 7)
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: strides of k and v must be multiples of 8 elements.");
    if ((a.q_row_stride | a.q_head_stride) & 1)
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: strides of q must be multiples of 2 elements.");
    if (((long long)a.num_rows * a.num_q_heads / kPsTile + a.num_q_heads) * (a.prefix_len / kPsTile + 1) > INT_MAX)
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: rows times prefix_len too large for one call.");
    if (a.num_rows == 0) return TT_OK;
    if (!a.q || !a.out || !a.row_lens || (a.prefix_len > 0 && !a.prefix_table) ||
        (a.num_tables > 0 && a.table_width > 0 && !a.tables) || !a.k || !a.v)
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: null pointer argument.");
    if (((uintptr_t)a.k & 15) || ((uintptr_t)a.v & 15) || ((uintptr_t)a.q & 3))
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: k and v must be 16-byte aligned, q 4-byte aligned.");
    return TT_OK;
}

static int prefix_groups(const PrefixParams& p) {
    return p.spans ? p.units * p.spans : (int)(((long long)p.units * p.kv_tiles + p.per - 1) / p.per);
}
static size_t prefix_slots(const PrefixParams& p) {
    return p.walk_prefix ? 0 : 2 * ((size_t)prefix_groups(p) + (size_t)p.units) * p.lanes;
}
static size_t own_slots(const PrefixParams& p) { return p.join ? (size_t)p.splits * p.a.num_rows * p.a.num_q_heads : 0; }

static PrefixParams plan_prefix(const tt_shared_prefix_args& a) {
    PrefixParams p = {};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
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

static size_t prefix_workspace(const PrefixParams& p) {
    return (prefix_slots(p) * kPsTile + own_slots(p)) * (p.a.head_dim * sizeof(float) + sizeof(float2));
}

// The pool in boxes of 64 channels and `tokens` tokens of one head.
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
    static const EncodeFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}
static bool encode_pool(CUtensorMap* map, const tt_shared_prefix_args& a, const void* base, int64_t page, int64_t token,
                        int64_t head, int tokens) {
    const EncodeFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.num_kv_heads, (cuuint64_t)a.page_size, (cuuint64_t)a.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)head * 2, (cuuint64_t)token * 2, (cuuint64_t)page * 2};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)tokens, 1};
    const cuuint32_t one[4] = {1, 1, 1, 1};
    return fn(map, a.dtype == TT_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
              const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD, bool PAIR>
static cudaError_t launch_shared(const PrefixParams& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    using S = PsShape<HD, PAIR>;
    static_assert(sizeof(PsBars) <= 256 && S::kSmem <= 227 * 1024 && S::kSlots <= 8, "shared memory of the prefix pass");
    auto* kern = k_prefix_shared<T, HD, PAIR>;
    const cudaError_t e = set_smem<k_prefix_shared<T, HD, PAIR>>(S::kSmem);
    if (e != cudaSuccess) return e;
    return launch(kern, dim3((unsigned)(prefix_groups(p) * p.lanes)), dim3(kPsThreads), S::kSmem, st, false, p, km, vm);
}
template <typename T>
static cudaError_t launch_shared_t(const PrefixParams& p, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t st) {
    const bool pair = p.tile_rows == 2 * kPsTile;
    if (p.a.head_dim == 64) return pair ? launch_shared<T, 64, true>(p, km, vm, st) : launch_shared<T, 64, false>(p, km, vm, st);
    return pair ? launch_shared<T, 128, true>(p, km, vm, st) : launch_shared<T, 128, false>(p, km, vm, st);
}

cudaError_t prefix_device_error(int clear, int* out) {
    cudaError_t e = cudaMemcpyFromSymbol(out, g_prefix_error, sizeof(int));
    if (e == cudaSuccess && clear) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_prefix_error, &zero, sizeof(int));
    }
    return e;
}

}  // namespace tt

using namespace tt;

extern "C" {

tt_status tt_shared_prefix_attention_workspace(const tt_shared_prefix_args* args, size_t* bytes) {
    const tt_status s = check_prefix(args);
    if (s != TT_OK) return s;
    if (!bytes) return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: null pointer argument.");
    *bytes = args->num_rows ? prefix_workspace(plan_prefix(*args)) : 0;
    return TT_OK;
}

tt_status tt_shared_prefix_attention(const tt_shared_prefix_args* args, void* stream) {
    const tt_status s = check_prefix(args);
    if (s != TT_OK) return s;
    if (args->num_rows == 0) return TT_OK;
    PrefixParams p = plan_prefix(*args);
    const tt_shared_prefix_args& a = p.a;
    const bool bf = a.dtype == TT_DTYPE_BF16;
    const cudaStream_t st = (cudaStream_t)stream;
    const auto encode = [&](CUtensorMap* km, CUtensorMap* vm, int tokens) {
        return encode_pool(km, a, a.k, a.k_page_stride, a.k_token_stride, a.k_head_stride, tokens) &&
               encode_pool(vm, a, a.v, a.v_page_stride, a.v_token_stride, a.v_head_stride, tokens);
    };
    if (prefix_workspace(p)) {
        if (!a.workspace || ((uintptr_t)a.workspace & 15))
            return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: workspace is missing or not 16-byte aligned.");
        const size_t slots = prefix_slots(p) * kPsTile;
        p.part_o = static_cast<float*>(a.workspace);
        p.own_o = p.part_o + slots * a.head_dim;
        p.part_ml = reinterpret_cast<float2*>(p.own_o + own_slots(p) * a.head_dim);
        p.own_ml = p.part_ml + slots;
    }
    CUtensorMap km, vm;
    if (!p.walk_prefix) {
        if (!encode(&km, &vm, a.page_size < kPsTile ? a.page_size : kPsTile))
            return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: no tensor map takes the strides of k and v.");
        const tt_status e = check_cuda(bf ? launch_shared_t<__nv_bfloat16>(p, km, vm, st) : launch_shared_t<__half>(p, km, vm, st),
                                       "shared_prefix_attention");
        if (e != TT_OK) return e;
    }
    if (!encode(&km, &vm, kGroup))
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: no tensor map takes the strides of k and v.");
    const tt_status e = check_cuda(bf ? launch_rows_t<__nv_bfloat16>(p, km, vm, st) : launch_rows_t<__half>(p, km, vm, st),
                                   "shared_prefix_attention");
    if (e != TT_OK || !p.join) return e;
    return check_cuda(bf ? launch_join_t<__nv_bfloat16>(p, st) : launch_join_t<__half>(p, st), "shared_prefix_attention");
}

}  // extern "C"
