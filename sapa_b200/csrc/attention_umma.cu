// attention_umma.cu — launches of the tensor-core kernels of attention over sequences.
#include "attention.cuh"
#include "tma_util.cuh"

namespace sapa {
namespace attn {

__device__ int g_wait_timeout = 0;

}  // namespace attn
}  // namespace sapa

#include "attention_umma.cuh"
#include "attention_umma_grad.cuh"

namespace sapa {
namespace attn {

namespace um {

// rows of 64 channels: dims and strides (in elements) of the axes behind the channels
static bool encode(CUtensorMap *map, const void *base, int dim, int rank, const long long *dims, const long long *strides, const int *boxes, bool half) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return false;
    cuuint64_t d[4] = {(cuuint64_t)dim}, st[3];
    cuuint32_t box[4] = {64u}, one[4] = {1u, 1u, 1u, 1u};
    for (int i = 0; i < rank; ++i) {
        d[i + 1] = (cuuint64_t)dims[i];
        st[i] = (cuuint64_t)strides[i] * 2;
        box[i + 1] = (cuuint32_t)boxes[i];
    }
    const CUtensorMapDataType type = half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    auto call = [&]() {
        return fn(map, type, (cuuint32_t)rank + 1, const_cast<void *>(base), d, st, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = call();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {                            // a thread without a context: the runtime's no-op binds the device's
        cudaFree(nullptr);
        r = call();
    }
    last_encode_result() = (int)r;
    return r == CUDA_SUCCESS;
}

// The warps take registers from one another by numbers that go by those at launch: with others they would wait for ever.
template <auto *KERNEL, int REGISTERS> static int check_registers(const char *name) {
    static const int regs = [] {
        cudaFuncAttributes f;
        return cudaFuncGetAttributes(&f, (const void *)KERNEL) == cudaSuccess ? f.numRegs : -1;
    }();
    SAPA_REQUIRE(regs == REGISTERS, SAPA_ERR_LAUNCH, "%s: built with %d registers a thread, not %d", name, regs, REGISTERS);
    return SAPA_OK;
}

template <typename T, int D, bool WIDE, bool PAGED, bool LOW>
static int launch(const Args &p, const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, long long items, cudaStream_t st) {
    using L = um::Lay<D, WIDE>;
    int sms = 0;
    if (int e = prepare_launch((const void *)sapa_attention_umma_kernel<T, D, WIDE, PAGED, LOW>, L::SMEM, "sapa_attention_umma_kernel", sms)) return e;
    if (int e = check_registers<sapa_attention_umma_kernel<T, D, WIDE, PAGED, LOW>, REGS>("sapa_attention_umma_kernel")) return e;
    launch_next(sapa_attention_umma_kernel<T, D, WIDE, PAGED, LOW>, dim3((unsigned)(items < sms ? items : sms)), dim3(um::NT), L::SMEM, st, q, k, v, p, (int)items);
    return check_launch(WIDE ? "sapa_attention_umma_kernel<wide>" : "sapa_attention_umma_kernel<narrow>");
}

}  // namespace um

bool umma_takes(const sapa_attention &a, int dtype) {
    if (dtype == SAPA_F32) return false;
    if (a.page_table == nullptr) return a.keys > 0;
    return a.page >= 8 && (a.page & (a.page - 1)) == 0;               // pages that a tile of 128 keys holds whole, or that hold it
}

int umma_forward(const Args &p, bool wide, long long items, int dtype, cudaStream_t st) {
    using namespace um;
    const sapa_attention &a = p.a;
    const bool half = dtype == SAPA_F16, paged = a.page_table != nullptr;
    CUtensorMap q, k, v;
    const int tok = ROWS / p.share;
    const long long qd[2] = {a.heads, a.tokens}, qs[2] = {a.query_strides[1], a.query_strides[0]};
    const int qb[2] = {p.share, tok};
    bool good = encode(&q, a.query, a.dim, 2, qd, qs, qb, half);
    const int rows = a.page < KT ? a.page : KT;
    const long long kd[3] = {a.groups, paged ? a.page : a.keys, a.pages}, ks[3] = {a.key_strides[1], a.key_strides[0], a.key_strides[2]},
                    vs[3] = {a.value_strides[1], a.value_strides[0], a.value_strides[2]};
    const int kb[3] = {1, paged ? rows : KT, 1};
    good = good && encode(&k, a.key, a.dim, paged ? 3 : 2, kd, ks, kb, half) && encode(&v, a.value, a.dim, paged ? 3 : 2, kd, vs, kb, half);
    SAPA_REQUIRE(good, SAPA_ERR_LAUNCH, "sapa_attention_forward: cuTensorMapEncodeTiled failed (%d)", last_encode_result());
    auto run = [&](auto t, auto d, auto w) -> int {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        constexpr bool W = decltype(w)::value;
        if (paged) return launch<T, D, W, true, false>(p, q, k, v, items, st);
        return a.low != nullptr ? launch<T, D, W, false, true>(p, q, k, v, items, st) : launch<T, D, W, false, false>(p, q, k, v, items, st);
    };
    auto pick = [&](auto t) -> int {
        using Narrow = std::integral_constant<int, 64>;
        using Wide = std::integral_constant<int, 128>;
        if (a.dim <= 64) return wide ? run(t, Narrow(), std::true_type()) : run(t, Narrow(), std::false_type());
        return wide ? run(t, Wide(), std::true_type()) : run(t, Wide(), std::false_type());
    };
    return half ? pick(__half()) : pick(__nv_bfloat16());
}

namespace umg {

template <typename T, int D, bool KEYS>
static int launch(const Args &p, const Grads &g, const CUtensorMap &own0, const CUtensorMap &own1, const CUtensorMap &over0, const CUtensorMap &over1, long long items,
                  cudaStream_t st) {
    int sms = 0;
    constexpr int SMEM = umg::Lay<D, KEYS>::SMEM;
    if (int e = prepare_launch((const void *)sapa_attention_umma_grad_kernel<T, D, KEYS>, SMEM, "sapa_attention_umma_grad_kernel", sms)) return e;
    if (int e = um::check_registers<sapa_attention_umma_grad_kernel<T, D, KEYS>, umg::GRAD_REGS>("sapa_attention_umma_grad_kernel")) return e;
    launch_next(sapa_attention_umma_grad_kernel<T, D, KEYS>, dim3((unsigned)(items < sms ? items : sms)), dim3(umg::THREADS), SMEM, st, own0, own1, over0, over1, p, g, (int)items);
    return check_launch(KEYS ? "sapa_attention_umma_grad_kernel<keys>" : "sapa_attention_umma_grad_kernel<queries>");
}

}  // namespace umg

int umma_backward(const Args &p, const Grads &g, int dtype, cudaStream_t st) {
    using namespace um;
    const sapa_attention &a = p.a;
    const bool half = dtype == SAPA_F16;
    const int tok = ROWS / p.share, over_rows = a.dim <= 64 ? umg::Lay<64, true>::TN : umg::Lay<128, true>::TN;      // that keys' items go over
    const int at_once = p.share < over_rows ? p.share : over_rows, few = over_rows / at_once;
    const long long qd[2] = {a.heads, a.tokens}, qs[2] = {a.query_strides[1], a.query_strides[0]}, os[2] = {g.go_strides[1], g.go_strides[0]};
    const long long kd[2] = {a.groups, a.keys}, ks[2] = {a.key_strides[1], a.key_strides[0]}, vs[2] = {a.value_strides[1], a.value_strides[0]};
    const long long key_items = most_blocks(a, a.keys, KT) * a.groups, query_items = most_blocks(a, a.tokens, tok) * a.groups;
    SAPA_REQUIRE(key_items < 0x3fffffffll && query_items < 0x3fffffffll, SAPA_ERR_UNSUPPORTED, "sapa_attention_backward: too many blocks");
    if (key_items == 0 || query_items == 0) return SAPA_OK;           // no sequence
    // the operands as an item holds them (128 rows) and as another goes over them
    CUtensorMap q[2], o[2], k[2], v[2];
    bool good = true;
    for (int i = 0; i < 2; ++i) {
        const int qb[2] = {i == 0 ? p.share : at_once, i == 0 ? tok : few}, kb[2] = {1, i == 0 ? KT : umg::Lay<64, false>::TN};
        good = good && encode(&q[i], a.query, a.dim, 2, qd, qs, qb, half) && encode(&o[i], g.go, a.dim, 2, qd, os, qb, half) &&
               encode(&k[i], a.key, a.dim, 2, kd, ks, kb, half) && encode(&v[i], a.value, a.dim, 2, kd, vs, kb, half);
    }
    SAPA_REQUIRE(good, SAPA_ERR_LAUNCH, "sapa_attention_backward: cuTensorMapEncodeTiled failed (%d)", last_encode_result());
    auto run = [&](auto t, auto d) -> int {
        using T = decltype(t);
        constexpr int D = decltype(d)::value;
        if (int e = umg::launch<T, D, true>(p, g, k[0], v[0], q[1], o[1], key_items, st)) return e;
        return umg::launch<T, D, false>(p, g, q[0], o[0], k[1], v[1], query_items, st);
    };
    using Narrow = std::integral_constant<int, 64>;
    using Wide = std::integral_constant<int, 128>;
    if (half) return a.dim <= 64 ? run(__half(), Narrow()) : run(__half(), Wide());
    return a.dim <= 64 ? run(__nv_bfloat16(), Narrow()) : run(__nv_bfloat16(), Wide());
}

// Flag of this family's bounded waits on the current device, cleared when it was raised; -1: it cannot be read.
int wait_timeout_flag() {
    int flag = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&flag, g_wait_timeout, sizeof(int)) != cudaSuccess) return -1;
    if (flag != 0 && cudaMemcpyToSymbol(g_wait_timeout, &zero, sizeof(int)) != cudaSuccess) return -1;
    return flag;
}

}  // namespace attn
}  // namespace sapa
