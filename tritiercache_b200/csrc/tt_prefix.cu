// tt_prefix.cu -- attention of a batch over a shared prefix and each row's own pages (C ABI:
// tt_shared_prefix_attention).
#include <limits.h>

#include "tt_prefix_shared.cuh"

namespace tt {

static_assert(sizeof(tt_shared_prefix_args) == 208, "packed by paged.py");

constexpr int kSms = 148;

template <typename T, int HD, int NB>
static cudaError_t launch_rows(const PrefixParams& p, int cluster, bool dependent, cudaStream_t st) {
    constexpr int ST = HD == 64 ? 4 : 2;
    const size_t smem = (size_t)kRowWarps * row_warp_bytes<HD, NB, ST>();
    auto* kern = k_prefix_rows<T, HD, NB, ST>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)(p.a.num_rows * cluster), (unsigned)(p.a.num_kv_heads * p.head_tiles));
    return launch(kern, grid, dim3(kRowWarps * 32), smem, st, dependent, cluster, p);
}

template <typename T>
static cudaError_t launch_rows_t(const PrefixParams& p, int nb, int cluster, bool dependent, cudaStream_t st) {
    if (p.a.head_dim == 64) return nb == 1 ? launch_rows<T, 64, 1>(p, cluster, dependent, st) : launch_rows<T, 64, 2>(p, cluster, dependent, st);
    return nb == 1 ? launch_rows<T, 128, 1>(p, cluster, dependent, st) : launch_rows<T, 128, 2>(p, cluster, dependent, st);
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
    if (a.num_pages < 0 || a.prefix_len < 0 || a.table_width < 0 || a.num_tables < 0)
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: sizes must be non-negative.");
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
    if (a.num_rows == 0) return TT_OK;
    if (!a.q || !a.out || !a.row_lens || (a.prefix_len > 0 && !a.prefix_table) ||
        (a.num_tables > 0 && a.table_width > 0 && !a.tables) || (a.num_pages > 0 && (!a.k || !a.v)))
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: null pointer argument.");
    if (((uintptr_t)a.k & 15) || ((uintptr_t)a.v & 15) || ((uintptr_t)a.q & 3))
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: k and v must be 16-byte aligned, q 4-byte aligned.");
    return TT_OK;
}

static int prefix_ctas(const PrefixParams& p) {
    const long long total = (long long)p.a.num_kv_heads * p.row_tiles * p.kv_tiles;
    return (int)((total + p.per - 1) / p.per);
}

static PrefixParams plan_prefix(const tt_shared_prefix_args& a) {
    PrefixParams p = {};
    p.a = a;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    p.group = a.num_q_heads / a.num_kv_heads;
    while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
    p.head_tiles = p.group <= 8 ? 1 : (p.group + 15) / 16;
    // One row has nobody to share with.  The prefix pass takes its maxima before the scale, so the scale must
    // not turn them round.
    p.walk_prefix = a.num_rows < 2 || a.prefix_len == 0 || !(a.scale > 0.f) || a.num_pages == 0;
    if (!p.walk_prefix) {
        const int rows = a.num_rows * p.group;
        p.tile_rows = rows > kPsTile ? 2 * kPsTile : kPsTile;
        p.row_tiles = (rows + p.tile_rows - 1) / p.tile_rows;
        p.kv_tiles = (a.prefix_len + kPsTile - 1) / kPsTile;
        const long long total = (long long)a.num_kv_heads * p.row_tiles * p.kv_tiles;
        p.per = (int)((total + kSms - 1) / kSms);
    }
    return p;
}

static size_t prefix_workspace(const PrefixParams& p) {
    if (p.walk_prefix) return 0;
    const size_t slots = 2 * ((size_t)prefix_ctas(p) + (size_t)p.a.num_kv_heads * p.row_tiles);
    return slots * kPsTile * (p.a.head_dim * sizeof(float) + sizeof(float2));
}

// The pool as [page][token][head][channel] boxes of 64 channels and up to 128 tokens of one head.
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
                        int64_t head) {
    const EncodeFn fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.num_kv_heads, (cuuint64_t)a.page_size, (cuuint64_t)a.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)head * 2, (cuuint64_t)token * 2, (cuuint64_t)page * 2};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)(a.page_size < kPsTile ? a.page_size : kPsTile), 1};
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
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return e;
    return launch(kern, dim3((unsigned)prefix_ctas(p)), dim3(kPsThreads), S::kSmem, st, false, 1, p, km, vm);
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
    const bool bf = args->dtype == TT_DTYPE_BF16;
    const cudaStream_t st = (cudaStream_t)stream;
    if (!p.walk_prefix) {
        if (!args->workspace || ((uintptr_t)args->workspace & 15))
            return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: workspace is missing or not 16-byte aligned.");
        const tt_shared_prefix_args& a = p.a;
        CUtensorMap km, vm;
        // strides that a tensor map does not take (an expanded pool): the rows' pass reads the prefix itself
        if (!encode_pool(&km, a, a.k, a.k_page_stride, a.k_token_stride, a.k_head_stride) ||
            !encode_pool(&vm, a, a.v, a.v_page_stride, a.v_token_stride, a.v_head_stride)) {
            p.walk_prefix = 1;
        } else {
            p.part_o = static_cast<float*>(args->workspace);
            const size_t slots = 2 * ((size_t)prefix_ctas(p) + (size_t)a.num_kv_heads * p.row_tiles);
            p.part_ml = reinterpret_cast<float2*>(p.part_o + slots * kPsTile * a.head_dim);
            const tt_status e = check_cuda(bf ? launch_shared_t<__nv_bfloat16>(p, km, vm, st) : launch_shared_t<__half>(p, km, vm, st),
                                           "shared_prefix_attention");
            if (e != TT_OK) return e;
        }
    }
    // CTAs per row and head tile: enough for the GPU, and no more than leaves a warp a few groups
    const long long tokens = (long long)args->table_width * args->page_size + (p.walk_prefix ? args->prefix_len : 0);
    const long long units = (long long)args->num_rows * args->num_kv_heads * p.head_tiles;
    int cluster = 1;
    while (cluster < 8 && units * cluster < 2 * kSms && tokens > (long long)cluster * kRowWarps * kGroup * 2) cluster *= 2;
    const int nb = p.group <= 8 ? 1 : 2;
    return check_cuda(bf ? launch_rows_t<__nv_bfloat16>(p, nb, cluster, !p.walk_prefix, st)
                         : launch_rows_t<__half>(p, nb, cluster, !p.walk_prefix, st), "shared_prefix_attention");
}

}  // extern "C"
