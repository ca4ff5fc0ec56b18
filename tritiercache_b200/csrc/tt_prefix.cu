// tt_prefix.cu -- attention of a batch over a shared prefix and each row's own pages (C ABI:
// tt_shared_prefix_attention).
#include <limits.h>

#include <atomic>

#include "tt_prefix_shared.cuh"

namespace tt {

static_assert(sizeof(tt_shared_prefix_args) == 208, "packed by paged.py");

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
    if (a.prefix_len > INT_MAX - kPsTile + 1)  // it is rounded up to whole key tiles
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: prefix_len must not exceed 2^31 - 128.");
    if (!a.row_seq && a.num_tables < a.num_rows)
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: without row_seq the tables need a row for each row.");
    if ((long long)a.num_rows * a.num_q_heads > (1 << 26))
        return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: more than 2^26 query heads in one call.");
    if (a.num_q_heads > 65535) return set_error(TT_ERR_UNSUPPORTED, "shared_prefix_attention: more than 65535 query heads.");
    // scores are kept in log2 units
    if (!(a.scale * kLog2e > -INFINITY && a.scale * kLog2e < INFINITY))
        return set_error(TT_ERR_INVALID_ARGUMENT, "shared_prefix_attention: scale and scale * log2(e) must be finite.");
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

static std::atomic<long long> g_wait_limit{kPatience};

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

tt_status tt_shared_prefix_wait_limit(int64_t clocks) {
    g_wait_limit.store(clocks < 0 || clocks > kPatience ? kPatience : (long long)clocks, std::memory_order_relaxed);
    return TT_OK;
}

tt_status tt_shared_prefix_attention(const tt_shared_prefix_args* args, void* stream) {
    const tt_status s = check_prefix(args);
    if (s != TT_OK) return s;
    if (args->num_rows == 0) return TT_OK;
    PrefixParams p = plan_prefix(*args);
    p.patience = g_wait_limit.load(std::memory_order_relaxed);
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
