// attention.cu — attention over sequences of tokens: the entry points, and the kernels on the FP32 pipe, which serve float32 and the pages that
// the tensor-core kernels (attention_umma.cu) do not take.
//
// One pass over the keys with the running maximum m and sum l of the softmax: a tile's scores s change m to m', l to
// l 2^(m - m') + sum 2^(s - m') and the output sum the same way (base 2, with log2(e) in the scale).  The query heads that share a key head
// are rows of one block (row = token x head), so that a key is read once for all of them.
#include "attention.cuh"
#include "tma_util.cuh"

#include <cmath>

namespace sapa {
namespace attn {

namespace rows {

constexpr int NT = 256, KT = 64;              // threads; keys of a tile
template <int RI, int DP> struct Lay {
    static constexpr int BM = 16 * RI, QS = DP + 4, PS = KT + 4;
    static constexpr int Q0 = 0, K0 = Q0 + BM * QS, V0 = K0 + KT * QS, P0 = V0 + KT * DP, END = P0 + BM * PS;
    static constexpr size_t SMEM = (size_t)END * sizeof(float);
};

template <typename T> __device__ __forceinline__ float4 load4(const T *p);
template <> __device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 widen(__half2 a, __half2 b) { const float2 x = __half22float2(a), y = __half22float2(b); return make_float4(x.x, x.y, y.x, y.y); }
__device__ __forceinline__ float4 widen(__nv_bfloat162 a, __nv_bfloat162 b) {
    const float2 x = __bfloat1622float2(a), y = __bfloat1622float2(b);
    return make_float4(x.x, x.y, y.x, y.y);
}
template <> __device__ __forceinline__ float4 load4(const __half *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return widen(*reinterpret_cast<const __half2 *>(&u.x), *reinterpret_cast<const __half2 *>(&u.y));
}
template <> __device__ __forceinline__ float4 load4(const __nv_bfloat16 *p) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    return widen(*reinterpret_cast<const __nv_bfloat162 *>(&u.x), *reinterpret_cast<const __nv_bfloat162 *>(&u.y));
}
// 8 elements, 0 where they are not `there`
__device__ __forceinline__ void load8(const float *p, bool there, float4 (&v)[2]) {
    v[0] = v[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (there) { v[0] = load4(p); v[1] = load4(p + 4); }
}
template <typename T> __device__ __forceinline__ void load8(const T *p, bool there, float4 (&v)[2]) {
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (there) raw = *reinterpret_cast<const uint4 *>(p);
    using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    v[0] = widen(*reinterpret_cast<const P *>(&raw.x), *reinterpret_cast<const P *>(&raw.y));
    v[1] = widen(*reinterpret_cast<const P *>(&raw.z), *reinterpret_cast<const P *>(&raw.w));
}
__device__ __forceinline__ void store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ bool finite4(float4 v) { return isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w); }
__device__ __forceinline__ float at(const float4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
template <typename T> __device__ __forceinline__ void put4(T *p, float4 v);
template <> __device__ __forceinline__ void put4(float *p, float4 v) { store4(p, v); }
template <typename T> __device__ __forceinline__ void put4(T *p, float4 v) {
    T e[4] = {from_acc<T>(v.x), from_acc<T>(v.y), from_acc<T>(v.z), from_acc<T>(v.w)};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(e);
}

// scale * s - base in base 2.  The product is not rounded by itself, nor the scale: with scores of 20 either would put a weight 1e-6 off.
__device__ __forceinline__ float exponent(const Args &p, float s, float base) {
    const float x = fmaf(s, p.scale_log2, -base);
    return isfinite(x) ? fmaf(s, p.scale_rest, x) : x;
}
// lse of a row from the maximum and the sum of its softmax in base 2, and in float32 what its rounding leaves out: that of the logarithm too, which would
// put all weights of the row off by up to 3e-7
__device__ __forceinline__ void put_lse(const sapa_attention &a, long long row, bool none, bool lost, float m, float sum, bool rest = true) {
    const double lse = ((double)m + (rest ? log2((double)sum) : (double)log2f(sum))) * 0.6931471805599453;
    const float high = none ? -INFINITY : lost ? __int_as_float(0x7fffffff) : (float)lse;
    a.lse[row] = high;
    if (rest && a.low != nullptr) static_cast<float *>(a.low)[row] = isfinite(high) ? (float)(lse - high) : 0.f;
}

}  // namespace rows

// RI: rows of a thread (a block has 16 of them across), DP: channels in shared memory.  256 threads as 16 x 16: rows ty + 16 i, of the scores
// the keys tx + 16 j, of the output the channels 4 tx + 64 j.  What bounds it: the FP32 pipe and the shared-memory reads that feed it (12 wide loads
// to 128 FMAs for the scores); with one row a thread (single tokens) reading the keys.
template <typename T, int RI, int DP>
__global__ void __launch_bounds__(rows::NT) sapa_attention_rows_kernel(const __grid_constant__ Args p) {
    using namespace rows;
    using L = Lay<RI, DP>;
    extern __shared__ __align__(16) float sm[];
    __shared__ Plan plan;
    __shared__ int bad_page;
    const sapa_attention &a = p.a;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int group = blockIdx.x % a.groups, tok = L::BM / p.share, D = a.dim;
    begin_after_previous();
    if (tid < 32) {
        const Plan r = ForwardPlans(p, tok, tid).at(blockIdx.x / a.groups);
        if (tid == 0) { plan = r; bad_page = 0x7fffffff; }
    }
    clear_outside(static_cast<T *>(a.out), a.offsets, a.B, a.tokens, a.heads * D, blockIdx.x, gridDim.x, tid, NT);
    if (a.lse != nullptr) clear_outside(a.lse, a.offsets, a.B, a.tokens, a.heads, blockIdx.x, gridDim.x, tid, NT);
    if (a.low != nullptr && std::is_same<T, float>::value) clear_outside(static_cast<float *>(a.low), a.offsets, a.B, a.tokens, a.heads, blockIdx.x, gridDim.x, tid, NT);
    __syncthreads();
    const Item it = plan.it;
    if (!it.there) return;
    const Sequence s = sequence_at(a, it.b);
    const int first = it.block * tok, used = min(tok, s.nq - first) * p.share;          // first token, rows in use
    int lim[RI];
    float m[RI], l[RI], o[RI][DP / 16];
#pragma unroll
    for (int i = 0; i < RI; ++i) {
        const int r = ty + 16 * i;
        lim[i] = r < used ? sees(s, first + r / p.share, a.causal) : 0;
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) o[i][c] = 0.f;
    }
    const int least = sees(s, first, a.causal), most = sees(s, first + used / p.share - 1, a.causal);      // of the block's tokens
    const int room = min(most, s.bad);                                                   // positions that are there to be read
    const long long from = (long long)it.part * plan.tiles * TILE, upto = min((long long)room, from + (long long)plan.tiles * TILE);
    if (tid == 0 && s.bad < most) atomicMin(&bad_page, s.bad);       // other threads may have found an earlier one

    for (int e = tid; e < L::BM * (DP / 4); e += NT) {
        const int r = e / (DP / 4), c = e % (DP / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < used && c < D)
            v = load4(static_cast<const T *>(a.query) + (long long)(s.q0 + first + r / p.share) * a.query_strides[0] +
                      (long long)(group * p.share + r % p.share) * a.query_strides[1] + c);
        store4(sm + L::Q0 + r * L::QS + c, v);
    }
    // a tile's keys and values, by way of registers: all pages first, then all rows; of narrow blocks while the tile before is at work
    constexpr int EACH = KT * (DP / 4) / NT;
    constexpr bool AHEAD = RI <= 2;
    float4 kr[EACH], vr[EACH];
    auto fetch = [&](int k0) {
        const int n = min(KT, (int)upto - k0);
        long long key_at[EACH], value_at[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int e = tid + i * NT, r = e / (DP / 4), position = k0 + r;
            key_at[i] = -1;
            if (r >= n || e % (DP / 4) * 4 >= D) continue;
            long long row = s.k0 + position, page = 0;
            if (a.page_table != nullptr) {
                const unsigned at = (unsigned)position / (unsigned)a.page;
                page = a.page_table[(long long)it.b * a.max_pages + at];
                row = position - (int)(at * a.page);
                if ((unsigned long long)page >= (unsigned)a.pages) { atomicMin(&bad_page, position); continue; }
            }
            key_at[i] = row * a.key_strides[0] + page * a.key_strides[2];
            value_at[i] = row * a.value_strides[0] + page * a.value_strides[2];
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            kr[i] = vr[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (key_at[i] < 0) continue;
            const int c = (tid + i * NT) % (DP / 4) * 4;
            kr[i] = load4(static_cast<const T *>(a.key) + key_at[i] + group * a.key_strides[1] + c);
            vr[i] = load4(static_cast<const T *>(a.value) + value_at[i] + group * a.value_strides[1] + c);
        }
    };
    if (AHEAD && from < upto) fetch((int)from);
    for (int k0 = (int)from; k0 < upto; k0 += KT) {
        const int n = min(KT, (int)upto - k0);
        bool odd = false;
        if (!AHEAD) fetch(k0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int e = tid + i * NT, r = e / (DP / 4), c = e % (DP / 4) * 4;
            odd = odd || !finite4(vr[i]);
            store4(sm + L::K0 + r * L::QS + c, kr[i]);
            store4(sm + L::V0 + r * DP + c, vr[i]);
        }
        if (AHEAD && k0 + KT < upto) fetch(k0 + KT);
        // a value that a row does not see must not reach it, not even as 0 * infinity
        const bool careful = __syncthreads_or(odd && k0 + KT > least);
        float sc[RI][4];
#pragma unroll
        for (int i = 0; i < RI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[i][j] = 0.f;
#pragma unroll 2
        for (int c = 0; c < DP; c += 4) {
            float4 k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = *reinterpret_cast<const float4 *>(sm + L::K0 + (tx + 16 * j) * L::QS + c);
#pragma unroll
            for (int i = 0; i < RI; ++i) {
                const float4 q = *reinterpret_cast<const float4 *>(sm + L::Q0 + (ty + 16 * i) * L::QS + c);
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[i][j] = fmaf(q.w, k[j].w, fmaf(q.z, k[j].z, fmaf(q.y, k[j].y, fmaf(q.x, k[j].x, sc[i][j]))));
            }
        }
#pragma unroll
        for (int i = 0; i < RI; ++i) {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (k0 + tx + 16 * j < lim[i] && tx + 16 * j < n) top = fmaxf(top, sc[i][j] * p.scale_log2);
            }
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float now = fmaxf(m[i], top), base = now == -INFINITY ? 0.f : now, old = exp2f(m[i] - base);
            m[i] = now;
            l[i] *= old;
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) o[i][c] *= old;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool seen = k0 + tx + 16 * j < lim[i] && tx + 16 * j < n;
                const float w = seen ? exp2f(exponent(p, sc[i][j], base)) : 0.f;
                l[i] += w;
                sm[L::P0 + (ty + 16 * i) * L::PS + tx + 16 * j] = w;
            }
        }
        __syncwarp();                          // the 16 threads that share a row are in one warp
        if (!careful) {
#pragma unroll
            for (int j = 0; j < DP / 64; ++j) {      // a tile by itself and then to the sum: fewer roundings at the sum's size (over 1500 keys half the error)
                float4 t[RI];
#pragma unroll
                for (int i = 0; i < RI; ++i) t[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
                for (int k = 0; k < KT; k += 4) {
                    float4 w[RI];
#pragma unroll
                    for (int i = 0; i < RI; ++i) w[i] = *reinterpret_cast<const float4 *>(sm + L::P0 + (ty + 16 * i) * L::PS + k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 v = *reinterpret_cast<const float4 *>(sm + L::V0 + (k + e) * DP + 4 * tx + 64 * j);
#pragma unroll
                        for (int i = 0; i < RI; ++i) {
                            const float x = at(w[i], e);
                            t[i].x = fmaf(x, v.x, t[i].x); t[i].y = fmaf(x, v.y, t[i].y); t[i].z = fmaf(x, v.z, t[i].z); t[i].w = fmaf(x, v.w, t[i].w);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < RI; ++i) { o[i][4 * j] += t[i].x; o[i][4 * j + 1] += t[i].y; o[i][4 * j + 2] += t[i].z; o[i][4 * j + 3] += t[i].w; }
            }
        } else {
#pragma unroll 1
            for (int c = 0; c < DP / 16; ++c) {
                const int at = 4 * tx + 64 * (c >> 2) + (c & 3);
#pragma unroll
                for (int i = 0; i < RI; ++i) {
                    float t = 0.f;
                    for (int k = 0; k < n; ++k)
                        if (k0 + k < lim[i]) t = fmaf(sm[L::P0 + (ty + 16 * i) * L::PS + k], sm[L::V0 + k * DP + at], t);
#pragma unroll
                    for (int e = 0; e < DP / 16; ++e) o[i][e] += e == c ? t : 0.f;
                }
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RI; ++i) {
        const int r = ty + 16 * i;
        float sum = l[i];
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (r >= used) continue;
        const bool none = lim[i] <= from, lost = lim[i] > bad_page;       // no key seen here; one that cannot be read
        const float nan = __int_as_float(0x7fffffff);
        const int head = group * p.share + r % p.share;
        const long long row = (long long)(s.q0 + first + r / p.share) * a.heads + head;
        if (it.parts == 1) {
            const float inv = none ? 0.f : lost ? nan : 1.f / sum;        // 0 / 0 where every score is -infinity, as the formula has it
            T *out = static_cast<T *>(a.out) + row * D;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j)
                if (4 * tx + 64 * j < D)
                    put4(out + 4 * tx + 64 * j, none ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(o[i][4 * j] * inv, o[i][4 * j + 1] * inv, o[i][4 * j + 2] * inv, o[i][4 * j + 3] * inv));
            if (a.lse != nullptr && tx == 0) put_lse(a, row, none, lost || sum == 0.f, m[i], sum, std::is_same<T, float>::value);
        } else {
            const float inv = sum == 0.f ? 0.f : lost ? nan : 1.f / sum;
            const long long at = ((long long)blockIdx.x * L::BM + r);
#pragma unroll
            for (int j = 0; j < DP / 64; ++j)
                if (4 * tx + 64 * j < D)
                    store4(p.part + at * D + 4 * tx + 64 * j, make_float4(o[i][4 * j] * inv, o[i][4 * j + 1] * inv, o[i][4 * j + 2] * inv, o[i][4 * j + 3] * inv));
            if (tx == 0) p.part_sums[at] = make_float2(sum == 0.f ? -INFINITY : m[i], lost ? nan : sum);
        }
    }
}

// Joins the parts of the split sequences: out = sum w_p out_p / sum w_p, w_p = 2^(m_p - max m) times the part's sum (lse_p as one number would be rounded).  Grid: a block and group, 16 of its rows; a warp per row, whose
// lanes first weigh the parts and then take 4 channels each, of every part or (up to 64 channels) of every other one.  Bound by the latency of its few
// loads: eight parts are on their way at once.
template <typename T>
__global__ void __launch_bounds__(256) sapa_attention_join_kernel(const __grid_constant__ Args p, int bm, int tok) {
    const sapa_attention &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = blockIdx.x % a.groups, D = a.dim;
    const int ways = D <= 64 ? 2 : 1, way = D <= 64 ? lane >> 4 : 0, c = 4 * (D <= 64 ? lane & 15 : lane);
    begin_after_previous();
    const Plan plan = split_at<false>(p, blockIdx.x / a.groups, tok, part_tiles(p, tok, lane), lane);
    if (!plan.it.there || plan.it.parts == 1) return;
    const Sequence s = sequence_at(a, plan.it.b);
    const int first = plan.it.block * tok, used = min(tok, s.nq - first) * p.share, parts = plan.it.parts;
    const long long step = (long long)a.groups * bm;                                  // from a part to the next
    for (int r = blockIdx.y * 16 + warp; r < min(used, (int)blockIdx.y * 16 + 16); r += 8) {
        const long long at = ((long long)plan.first * a.groups + group) * bm + r;
        const int lim = sees(s, first + r / p.share, a.causal);
        float top = -INFINITY;
        bool lost = false;
        for (int q = lane; q < parts; q += 32) { const float2 e = p.part_sums[at + q * step]; top = fmaxf(top, e.x); lost = lost || e.y != e.y; }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        lost = __any_sync(0xffffffffu, lost) || (lim > 0 && top == -INFINITY);
        float sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        const float *from = p.part + at * D + c;
        for (int q0 = 0; q0 < parts; q0 += 32) {
            const float2 e = q0 + lane < parts ? p.part_sums[at + (q0 + lane) * step] : make_float2(-INFINITY, 0.f);
            const float mine = e.x == -INFINITY ? 0.f : exp2f(e.x - top) * e.y;
            const int n = min(32, parts - q0);
            for (int q = 0; q < n; q += 8 * ways) {
                float4 v[8];
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {                                         // a part that a row sees nothing of counts 0, and holds 0
                    const int k = q + i * ways + way;
                    w[i] = __shfl_sync(0xffffffffu, mine, k & 31);
                    if (k >= n) w[i] = 0.f;
                    v[i] = k < n && c < D ? *reinterpret_cast<const float4 *>(from + (q0 + k) * step * D) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum += w[i];
                    acc.x = fmaf(w[i], v[i].x, acc.x); acc.y = fmaf(w[i], v[i].y, acc.y); acc.z = fmaf(w[i], v[i].z, acc.z); acc.w = fmaf(w[i], v[i].w, acc.w);
                }
            }
        }
        if (ways == 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16); acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
            acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16); acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
        }
        const float inv = lost ? __int_as_float(0x7fffffff) : lim <= 0 ? 0.f : 1.f / sum;
        const long long row = (long long)(s.q0 + first + r / p.share) * a.heads + group * p.share + r % p.share;
        if (c < D && way == 0) {
            const float4 v = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            rows::put4(static_cast<T *>(a.out) + row * D + c, v);
            if (a.low != nullptr && !std::is_same<T, float>::value)
                rows::put4(static_cast<T *>(a.low) + row * D + c, make_float4(left_out<T>(v.x), left_out<T>(v.y), left_out<T>(v.z), left_out<T>(v.w)));
        }
        if (a.lse != nullptr && lane == 0) rows::put_lse(a, row, lim <= 0, lost, top, sum, std::is_same<T, float>::value);
    }
}

// ---------------------------------------------------------------------------------- backward
// delta, and what lies outside the sequences: 8 or 16 lanes (up to 64 or 128 channels) per token and head, 8 channels each.  Reads grad_out, out and what its
// rounding left out once, which bounds it (8262 tokens x 16 heads x 128 channels, bfloat16: 28 us, 3.6 TB/s; with two rows to a thread 29, with four 44).  In
// float16 also sums of squares, for which blocks behind those of the queries read the values.
template <typename T, int LANES>
__global__ void __launch_bounds__(256, 8) sapa_attention_delta_kernel(const __grid_constant__ Args p, const __grid_constant__ Grads g) {
    const sapa_attention &a = p.a;
    constexpr bool SQUARES = std::is_same<T, __half>::value;
    constexpr bool RESTS = !std::is_same<T, float>::value;            // `out` before its rounding: by itself that would make the gradients a third less exact
    constexpr int ROWS = 256 / LANES;                                 // of a block
    const int lane = threadIdx.x % LANES, c = 8 * lane, D = a.dim;
    auto squares = [](const float4 (&x)[2]) {
        return fmaf(x[1].w, x[1].w, fmaf(x[1].z, x[1].z, fmaf(x[1].y, x[1].y, fmaf(x[1].x, x[1].x, fmaf(x[0].w, x[0].w, fmaf(x[0].z, x[0].z, fmaf(x[0].y, x[0].y, x[0].x * x[0].x)))))));
    };
    begin_after_previous();
    const long long n = (long long)a.tokens * a.heads, query_blocks = (n + ROWS - 1) / ROWS, m = SQUARES ? (long long)a.keys * a.groups : 0;
    const int begin = a.B > 0 ? a.offsets[0] : 0, end = a.B > 0 ? a.offsets[a.B] : 0;
    for (long long block = blockIdx.x; block < query_blocks + (m + ROWS - 1) / ROWS; block += gridDim.x) {
        if (SQUARES && block >= query_blocks) {
            const long long row = (block - query_blocks) * ROWS + threadIdx.x / LANES;
            const unsigned t = m <= 0x7fffffff ? (unsigned)row / (unsigned)a.groups : (unsigned)(row / a.groups), group = (unsigned)(row - (long long)t * a.groups);
            float4 v[2];
            rows::load8(static_cast<const T *>(a.value) + t * a.value_strides[0] + group * a.value_strides[1] + c, row < m && c < D, v);
            float square = squares(v);
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) square += __shfl_xor_sync(0xffffffffu, square, o);
            if (lane == 0 && row < m) g.value_squares[(long long)group * a.keys + t] = square;
            continue;
        }
        const long long row = block * ROWS + threadIdx.x / LANES;
        const unsigned t = n <= 0x7fffffff ? (unsigned)row / (unsigned)a.heads : (unsigned)(row / a.heads), h = (unsigned)(row - (long long)t * a.heads);
        const bool there = row < n && c < D;
        float4 u[2], v[2], low[2];
        rows::load8(static_cast<const T *>(a.out) + row * D + c, there, u);
        rows::load8(static_cast<const T *>(g.go) + t * g.go_strides[0] + h * g.go_strides[1] + c, there, v);
        rows::load8(static_cast<const T *>(a.low) + row * D + c, there && RESTS, low);
        float sum = 0.f, square = SQUARES ? squares(v) : 0.f;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            sum = fmaf(u[e].w + low[e].w, v[e].w, fmaf(u[e].z + low[e].z, v[e].z, fmaf(u[e].y + low[e].y, v[e].y, fmaf(u[e].x + low[e].x, v[e].x, sum))));
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (SQUARES) square += __shfl_xor_sync(0xffffffffu, square, o);
        }
        if (lane != 0 || row >= n) continue;
        if (g.nlse != nullptr) {
            const long long at = ((long long)(h / p.share) * a.tokens + t) * p.share + h % p.share;
            g.delta[at] = sum;
            if (SQUARES) g.squares[at] = square;
            // of no sequence: +infinity, as of a row that sees no key, for what such a row of the query holds shows in nothing else
            g.nlse[at] = (int)t >= begin && (int)t < end ? -1.4426950408889634f * a.lse[row] : INFINITY;
        } else {
            g.delta[row] = sum;
        }
    }
    clear_outside(static_cast<T *>(g.gq), a.offsets, a.B, a.tokens, a.heads * D, blockIdx.x, gridDim.x, threadIdx.x, 256);
    clear_outside(static_cast<T *>(g.gk), a.key_offsets, a.B, a.keys, a.groups * D, blockIdx.x, gridDim.x, threadIdx.x, 256);
    clear_outside(static_cast<T *>(g.gv), a.key_offsets, a.B, a.keys, a.groups * D, blockIdx.x, gridDim.x, threadIdx.x, 256);
}

// float16.  The power of two that dS of a sequence and key head is multiplied with to be held in 16 bits: |dS| = |P_j sum_k P_k (dP_j - dP_k)| is at most a quarter
// of the range of dP, that is half the product of the longest rows of grad_out and of value, and comes to 2^14 at most.  The scores' weights, around
// 1 / keys, leave it among the normal numbers then, whatever size the gradients have.  Rows that are not finite do not count.  A block of 1024 threads to each,
// or a warp where there are more than two rounds of blocks (2000 sequences of up to 20 tokens, 12 heads: forward and gradients 1874 us with blocks, 1727 with warps;
// 8 sequences of up to 1024 tokens: 172 and 175).
template <bool WARPS>
__global__ void __launch_bounds__(WARPS ? 256 : 1024) sapa_attention_factor_kernel(const __grid_constant__ Args p, const __grid_constant__ Grads g) {
    const sapa_attention &a = p.a;
    __shared__ float most[2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int STEP = WARPS ? 32 : 1024;
    const long long index = WARPS ? (long long)blockIdx.x * 8 + warp : blockIdx.x;
    begin_after_previous();
    if (index >= (long long)a.B * a.groups) return;                   // a whole warp
    const int b = (int)(index / a.groups), group = (int)(index % a.groups);
    const Sequence s = sequence_at(a, b);
    auto largest = [&](const float *x, long long n) {
        float top[4] = {0.f, 0.f, 0.f, 0.f};
        for (long long i = WARPS ? lane : threadIdx.x; i < n; i += 4 * STEP)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = i + STEP * e < n ? x[i + STEP * e] : 0.f;
                top[e] = isfinite(v) ? fmaxf(top[e], v) : top[e];
            }
        return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    };
    auto of_warp = [](float r) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, o));
        return r;
    };
    float x = of_warp(largest(g.squares + ((long long)group * a.tokens + s.q0) * p.share, (long long)s.nq * p.share));
    float y = of_warp(largest(g.value_squares + (long long)group * a.keys + s.k0, s.nk));
    if (!WARPS) {
        if (lane == 0) { most[0][warp] = x; most[1][warp] = y; }
        __syncthreads();
        if (warp != 0) return;
        x = of_warp(most[0][lane]);
        y = of_warp(most[1][lane]);
    }
    const int j = (int)(__float_as_uint(x) >> 23), k = (int)(__float_as_uint(y) >> 23);      // sums below 2^(j - 126), 2^(k - 126); none is subnormal, as squares of float16
    if (lane == 0) g.factor[index] = j == 0 || k == 0 ? 1.f : __int_as_float((127 + 15 - ((j + k - 252 + 1) >> 1)) << 23);
}

namespace grad {
using namespace rows;
constexpr int OWN = 32, OVER = 32, TEAM = 128, TEAMS = 4, THREADS = TEAM * TEAMS, WS = OWN + 4;      // rows or keys of a block, of a tile that it goes over
template <int DP> struct Lay {
    static constexpr int XS = DP + 4;
    static constexpr int A0 = 0, A1 = OWN * XS, LA = 2 * OWN * XS, TEAM0 = LA + 3 * OWN;
    static constexpr int B0 = 0, B1 = OVER * XS, P0 = 2 * OVER * XS, S0 = P0 + OVER * WS, LB = S0 + OVER * WS, EACH = LB + 3 * OVER;      // of a team
    static constexpr size_t SMEM = (size_t)(TEAM0 + TEAMS * EACH) * sizeof(float);
    static_assert(EACH >= 2 * 4 * (DP / 16) * TEAM, "a team's sums are handed over in its tile");
};
__device__ __forceinline__ void team_sync(int team) { asm volatile("bar.sync %0, 128;\n" ::"r"(1 + team) : "memory"); }
__device__ __forceinline__ bool team_or(int team, bool v) {
    unsigned any;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n barrier.cta.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(any) : "r"(1 + team), "r"((unsigned)v) : "memory");
    return any != 0;
}
// all threads of the blocks of a cluster; what they wrote before is seen after it, in each other's shared memory too
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// shared memory of another block of the cluster, at the place of `own` here
__device__ __forceinline__ unsigned in_block(const float *own, int rank) {
    unsigned at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(own)), "r"(rank));
    return at;
}
__device__ __forceinline__ float load_far(unsigned at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(at) : "memory");
    return v;
}
}  // namespace grad

// float32.  KEYS: gradients of 32 keys and values, over the rows (token x head of a key head) that see them; otherwise those of 32 query rows, over the keys
// that they see.  P and dS of a tile of 32 are formed again from the scores, lse and delta: P = 2^(s - lse), dS = P (dP - delta); no atomics.  Four teams of
// 128 threads take the tiles in turn and add up at the end: a team by itself waits most of the time (1342 tokens, 8 heads of 64 channels: keys 164 us).
// Threads of a team as 8 x 16: of S and dP the rows ty + 8 i and the columns tx + 16 j, of the sums the rows 4 ty + i and the channels 4 tx + 64 j.
// What bounds it: the FP32 pipe and the shared-memory reads beside it, in small problems the longest item: with SHARED the blocks of a cluster take its tiles in turn.
template <int DP, bool KEYS, bool SHARED>
__global__ void __launch_bounds__(grad::THREADS, 1) sapa_attention_rows_grad_kernel(const __grid_constant__ Args p, const __grid_constant__ Grads g) {
    using namespace grad;
    using T = float;
    using L = grad::Lay<DP>;
    extern __shared__ __align__(16) float sm[];
    __shared__ Item item;
    const sapa_attention &a = p.a;
    const int team = threadIdx.x / TEAM, tid = threadIdx.x % TEAM, tx = tid & 15, ty = tid >> 4, D = a.dim;
    float *const mine = sm + L::TEAM0 + team * L::EACH;               // this team's tile
    constexpr int ROWS = KEYS ? OVER : OWN;                                                   // of a tile of rows
    const int share = p.share, at_once = min(share, ROWS), tok = ROWS / at_once, turns = (share + at_once - 1) / at_once;      // more heads than rows: in turns
    const int slots = KEYS ? a.groups : a.groups * turns, slot = blockIdx.x % slots, group = slot % a.groups;
    const int rank = SHARED ? blockIdx.y : 0, ranks = SHARED ? gridDim.y : 1;      // SHARED: the blocks of a cluster share an item's tiles
    begin_after_previous();
    if (threadIdx.x < 32) {
        const Item r = KEYS ? InOrder<false, KeyBlocks>(a, KeyBlocks{a.causal != 0, tok, OWN}, tid).at(blockIdx.x / slots)
                            : InOrder<true, QueryBlocks>(a, QueryBlocks{a.causal != 0, tok, OVER}, tid).at(blockIdx.x / slots);
        if (tid == 0) item = r;
    }
    __syncthreads();
    if (!item.there) return;
    const Sequence s = sequence_at(a, item.b);

    // rows of tokens from i0, heads from h0: r -> token i0 + r / at_once, head h0 + r % at_once
    auto load = [&](float *to0, float *to1, float *lse, int rows, int me, int threads, bool keys, int k0, int i0, int h0, int used) {      // returns whether something is not finite
        bool odd = false;
        constexpr int AT_ONCE = 4;
        float4 u[AT_ONCE], v[AT_ONCE];
#pragma unroll 1
        for (int e0 = 0; e0 < rows * (DP / 4); e0 += AT_ONCE * threads) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int e = e0 + me + i * threads, r = e / (DP / 4), c = e % (DP / 4) * 4;
                u[i] = v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r >= rows || c >= D) continue;
                if (keys) {
                    if (k0 + r >= s.nk) continue;
                    u[i] = load4(static_cast<const T *>(a.key) + (long long)(s.k0 + k0 + r) * a.key_strides[0] + group * a.key_strides[1] + c);
                    v[i] = load4(static_cast<const T *>(a.value) + (long long)(s.k0 + k0 + r) * a.value_strides[0] + group * a.value_strides[1] + c);
                } else {
                    if (r >= used || h0 + r % at_once >= share) continue;
                    const long long t = s.q0 + i0 + r / at_once, h = group * share + h0 + r % at_once;
                    u[i] = load4(static_cast<const T *>(a.query) + t * a.query_strides[0] + h * a.query_strides[1] + c);
                    v[i] = load4(static_cast<const T *>(g.go) + t * g.go_strides[0] + h * g.go_strides[1] + c);
                }
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const int e = e0 + me + i * threads, r = e / (DP / 4), c = e % (DP / 4) * 4;
                if (r >= rows) continue;
                odd = odd || !finite4(u[i]) || (!keys && !finite4(v[i]));
                store4(to0 + r * L::XS + c, u[i]);
                store4(to1 + r * L::XS + c, v[i]);
            }
        }
        if (!keys)
            for (int r = me; r < rows; r += threads) {
                float e = 0.f, rest = 0.f, d = 0.f;
                if (r < used && h0 + r % at_once < share) {
                    const long long at = (long long)(s.q0 + i0 + r / at_once) * a.heads + group * share + h0 + r % at_once;
                    const double both = ((double)a.lse[at] + static_cast<const float *>(a.low)[at]) * 1.4426950408889634;
                    e = (float)both;
                    rest = isfinite(e) ? (float)(both - e) : 0.f;
                    d = g.delta[at];
                }
                lse[r] = e;
                lse[rows + r] = d;
                lse[2 * rows + r] = rest;
            }
        return odd;
    };
    float x[4][DP / 16], y[4][DP / 16];        // KEYS: of values, of keys; otherwise y: of queries
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) x[i][c] = y[i][c] = 0.f;

    // a tile: rows of tokens from i0, heads from h0; keys from k0
    auto tile = [&](int i0, int h0, int used, int k0, bool odd) {
        auto limit = [&](int r) { return r < used && h0 + r % at_once < share ? sees(s, i0 + r / at_once, a.causal) - k0 : 0; };      // keys of the tile that a row sees
        const bool careful = team_or(team, odd);
        float sc[4][2], dp[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) sc[i][j] = dp[i][j] = 0.f;
#pragma unroll 2
        for (int c = 0; c < DP; c += 4) {
            float4 u[2], v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                u[j] = *reinterpret_cast<const float4 *>(mine + L::B0 + (tx + 16 * j) * L::XS + c);
                v[j] = *reinterpret_cast<const float4 *>(mine + L::B1 + (tx + 16 * j) * L::XS + c);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 m = *reinterpret_cast<const float4 *>(sm + L::A0 + (ty + 8 * i) * L::XS + c);
                const float4 n = *reinterpret_cast<const float4 *>(sm + L::A1 + (ty + 8 * i) * L::XS + c);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    sc[i][j] = fmaf(m.w, u[j].w, fmaf(m.z, u[j].z, fmaf(m.y, u[j].y, fmaf(m.x, u[j].x, sc[i][j]))));
                    dp[i][j] = fmaf(n.w, v[j].w, fmaf(n.z, v[j].z, fmaf(n.y, v[j].y, fmaf(n.x, v[j].x, dp[i][j]))));
                }
            }
        }
        constexpr int HAS = KEYS ? 2 : 4;      // rows that this thread has
        int lim[HAS];
        const float *const lse = KEYS ? mine + L::LB : sm + L::LA;
#pragma unroll
        for (int i = 0; i < HAS; ++i) lim[i] = limit(KEYS ? tx + 16 * i : ty + 8 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int own = ty + 8 * i, over = tx + 16 * j, r = KEYS ? over : own, k = KEYS ? own : over;
                const bool seen = k < lim[KEYS ? j : i];
                const float w = seen ? exp2f(exponent(p, sc[i][j], lse[r]) - lse[2 * ROWS + r]) : 0.f;
                if (KEYS) mine[L::P0 + over * WS + own] = w;
                mine[L::S0 + over * WS + own] = seen ? w * (dp[i][j] - lse[ROWS + r]) : 0.f;
            }
        team_sync(team);
        if (!careful) {
#pragma unroll 4
            for (int n = 0; n < OVER; ++n) {
                const float4 w = KEYS ? *reinterpret_cast<const float4 *>(mine + L::P0 + n * WS + 4 * ty) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 ds = *reinterpret_cast<const float4 *>(mine + L::S0 + n * WS + 4 * ty);
#pragma unroll
                for (int j = 0; j < DP / 64; ++j) {
                    const float4 f = *reinterpret_cast<const float4 *>(mine + L::B0 + n * L::XS + 4 * tx + 64 * j);
                    const float4 o = KEYS ? *reinterpret_cast<const float4 *>(mine + L::B1 + n * L::XS + 4 * tx + 64 * j) : f;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (KEYS) x[i][4 * j + e] = fmaf(at(w, i), at(o, e), x[i][4 * j + e]);
                            y[i][4 * j + e] = fmaf(at(ds, i), at(f, e), y[i][4 * j + e]);
                        }
                }
            }
        } else {                               // what is not seen must not reach a gradient, not even as 0 * infinity
            for (int n = 0; n < OVER; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if ((KEYS ? 4 * ty + i : n) >= limit(KEYS ? n : 4 * ty + i)) continue;
#pragma unroll
                    for (int c = 0; c < DP / 16; ++c) {
                        const int col = 4 * tx + 64 * (c >> 2) + (c & 3);
                        if (KEYS) x[i][c] = fmaf(mine[L::P0 + n * WS + 4 * ty + i], mine[L::B1 + n * L::XS + col], x[i][c]);
                        y[i][c] = fmaf(mine[L::S0 + n * WS + 4 * ty + i], mine[L::B0 + n * L::XS + col], y[i][c]);
                    }
                }
        }
    };

    const int first = item.block * (KEYS ? OWN : tok);                // key or token
    if (KEYS) {
        load(sm + L::A0, sm + L::A1, nullptr, OWN, threadIdx.x, THREADS, true, first, 0, 0, 0);
        __syncthreads();
        const int from = a.causal ? (int)max(0ll, (long long)first - s.nk + s.nq) : 0;      // the first token that sees one of them
        const int tiles = from < s.nq ? tiles_of(s.nq - from, tok) * turns : 0;
        for (int i = rank * TEAMS + team; i < tiles; i += ranks * TEAMS) {
            const int i0 = from + i / turns * tok, h0 = i % turns * at_once, used = min(tok, s.nq - i0) * at_once;
            team_sync(team);
            const bool odd = load(mine + L::B0, mine + L::B1, mine + L::LB, OVER, tid, TEAM, false, 0, i0, h0, used);
            tile(i0, h0, used, first, odd);
        }
    } else {
        const int h0 = slot / a.groups * at_once, used = min(tok, s.nq - first) * at_once;
        const int tiles = tiles_of(sees(s, first + used / at_once - 1, a.causal), OVER);
        load(sm + L::A0, sm + L::A1, sm + L::LA, OWN, threadIdx.x, THREADS, false, 0, first, h0, used);
        __syncthreads();
        for (int i = rank * TEAMS + team; i < tiles; i += ranks * TEAMS) {
            team_sync(team);
            const bool odd = load(mine + L::B0, mine + L::B1, nullptr, OVER, tid, TEAM, true, i * OVER, 0, 0, 0);
            tile(first, h0, used, i * OVER, odd);
        }
    }
    // the teams' sums, in their order, through their tiles; then those of the cluster's blocks
    auto hand_over = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                mine[(i * (DP / 16) + c) * TEAM + tid] = y[i][c];
                if (KEYS) mine[(4 * (DP / 16) + i * (DP / 16) + c) * TEAM + tid] = x[i][c];
            }
    };
    auto add = [&](auto sum_of) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
                y[i][c] += sum_of(i * (DP / 16) + c);
                if (KEYS) x[i][c] += sum_of(4 * (DP / 16) + i * (DP / 16) + c);
            }
    };
    team_sync(team);
    if (team != 0) hand_over();
    __syncthreads();
    if (!SHARED && team != 0) return;
    if (!SHARED || team == 0) {
#pragma unroll 1
        for (int q = 1; q < TEAMS; ++q) {
            const float *const other = sm + L::TEAM0 + q * L::EACH + tid;
            add([&](int i) { return other[i * TEAM]; });
        }
        if (SHARED && rank != 0) hand_over();
    }
    if (SHARED) {
        cluster_sync();
        if (team + rank == 0) {
#pragma unroll 1
            for (int q = 1; q < ranks; ++q) {
                const unsigned other = in_block(mine + tid, q);
                add([&](int i) { return load_far(other + 4u * TEAM * i); });
            }
        }
        cluster_sync();                        // the other blocks' memory is there until it has been read
        if (team + rank != 0) return;
    }
    // the scores' scale is in the gradients of queries and keys
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = 4 * ty + i;
        long long row;
        if (KEYS) {
            if (first + n >= s.nk) continue;
            row = (long long)(s.k0 + first + n) * a.groups + group;
        } else {
            const int h = slot / a.groups * at_once + n % at_once;
            if (n >= min(tok, s.nq - first) * at_once || h >= share) continue;
            row = (long long)(s.q0 + first + n / at_once) * a.heads + group * share + h;
        }
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            const int c = 4 * tx + 64 * j;
            if (c >= D) continue;
            const float f = a.scale;
            put4(static_cast<T *>(KEYS ? g.gk : g.gq) + row * D + c, make_float4(y[i][4 * j] * f, y[i][4 * j + 1] * f, y[i][4 * j + 2] * f, y[i][4 * j + 3] * f));
            if (KEYS) put4(static_cast<T *>(g.gv) + row * D + c, make_float4(x[i][4 * j], x[i][4 * j + 1], x[i][4 * j + 2], x[i][4 * j + 3]));
        }
    }
}

// ---------------------------------------------------------------------------------- writing into a paged cache
// A warp takes 2 KB of a token's keys and of its values, all on their way at once: where they go is found once for them.  What bounds it: reading and writing
// them once; for single tokens the launch.
__global__ void __launch_bounds__(256) sapa_paged_write_kernel(const __grid_constant__ sapa_paged_rows a, int esize) {
    constexpr int EACH = 4;
    begin_after_previous();
    const int chunks = a.dim * esize / 16, per_row = a.groups * chunks, lane = threadIdx.x & 31, parts = (per_row + 32 * EACH - 1) / (32 * EACH);
    const long long n = (long long)a.tokens * parts;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (long long)gridDim.x * 8) {
        const int t = (int)(i / parts), part = (int)(i % parts);
        // the first sequence whose end lies behind the token
        int lo = 0, hi = a.B;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.offsets[mid + 1] > t) hi = mid; else lo = mid + 1;
        }
        if (lo == a.B || t < a.offsets[lo]) continue;
        const long long at = (long long)a.key_lengths[lo] - min(a.offsets[lo + 1], a.tokens) + t;
        if (at < 0 || at >= (long long)a.max_pages * a.page) continue;
        const int page = a.page_table[(long long)lo * a.max_pages + at / a.page], slot = (int)(at % a.page);
        if ((unsigned)page >= (unsigned)a.pages) continue;
        auto from = [&](const void *x, const long long (&st)[2], int group, int c) {
            return reinterpret_cast<const uint4 *>(static_cast<const char *>(x) + ((long long)t * st[0] + group * st[1]) * esize + 16 * c);
        };
        auto to = [&](void *x, const long long (&st)[3], int group, int c) {
            return reinterpret_cast<uint4 *>(static_cast<char *>(x) + (page * st[2] + slot * st[0] + group * st[1]) * esize + 16 * c);
        };
        uint4 k[EACH], v[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int x = (part * EACH + e) * 32 + lane, group = x / chunks, c = x - group * chunks;
            if (x >= per_row) continue;
            k[e] = *from(a.key, a.key_strides, group, c);
            v[e] = *from(a.value, a.value_strides, group, c);
        }
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            const int x = (part * EACH + e) * 32 + lane, group = x / chunks, c = x - group * chunks;
            if (x >= per_row) continue;
            *to(a.key_pages, a.key_page_strides, group, c) = k[e];
            *to(a.value_pages, a.value_page_strides, group, c) = v[e];
        }
    }
}

// ---------------------------------------------------------------------------------- host side
constexpr int MOST_ROWS = 0x7fffff00;
static int check(const sapa_attention *a, int dtype, const char *fn) {
    SAPA_REQUIRE(a != nullptr, SAPA_ERR_ARGUMENT, "%s: the arguments are NULL", fn);
    SAPA_REQUIRE(dtype == SAPA_F32 || dtype == SAPA_F16 || dtype == SAPA_BF16, SAPA_ERR_DTYPE, "%s: dtype code %d is not supported", fn, dtype);
    SAPA_REQUIRE(a->B >= 0 && a->tokens >= 0 && a->keys >= 0, SAPA_ERR_ARGUMENT, "%s: negative size", fn);
    // a tile may begin at the last row: its end has to be a number too
    SAPA_REQUIRE(a->tokens < MOST_ROWS && a->keys < MOST_ROWS, SAPA_ERR_UNSUPPORTED, "%s: more than 2^31 - 256 tokens or keys", fn);
    SAPA_REQUIRE(a->heads > 0 && a->groups > 0 && a->heads % a->groups == 0, SAPA_ERR_ARGUMENT, "%s: %d heads do not share %d key heads evenly", fn, a->heads, a->groups);
    SAPA_REQUIRE(a->heads / a->groups <= 128, SAPA_ERR_UNSUPPORTED, "%s: more than 128 heads share a key head", fn);
    SAPA_REQUIRE(a->dim > 0 && a->dim <= 128 && a->dim % 8 == 0, SAPA_ERR_UNSUPPORTED, "%s: dim %d is not a multiple of 8 up to 128", fn, a->dim);
    SAPA_REQUIRE(std::isfinite(a->scale), SAPA_ERR_ARGUMENT, "%s: the scale is not finite", fn);
    SAPA_REQUIRE(a->offsets != nullptr, SAPA_ERR_ARGUMENT, "%s: offsets is NULL", fn);
    if (a->page_table != nullptr) {
        SAPA_REQUIRE(a->key_lengths != nullptr, SAPA_ERR_ARGUMENT, "%s: key_lengths is NULL", fn);
        SAPA_REQUIRE(a->pages > 0 && a->page > 0 && a->max_pages > 0, SAPA_ERR_ARGUMENT, "%s: pages, page and max_pages must be positive", fn);
        SAPA_REQUIRE((long long)a->max_pages * a->page < MOST_ROWS, SAPA_ERR_UNSUPPORTED, "%s: more than 2^31 positions", fn);
    } else {
        SAPA_REQUIRE(a->key_offsets != nullptr, SAPA_ERR_ARGUMENT, "%s: key_offsets is NULL", fn);
    }
    const long long quantum = 16 / (long long)dtype_size(dtype);
    for (long long s : {a->query_strides[0], a->query_strides[1], a->key_strides[0], a->key_strides[1], a->value_strides[0], a->value_strides[1]})
        SAPA_REQUIRE(s >= 0 && s % quantum == 0, SAPA_ERR_ALIGNMENT, "%s: strides must be multiples of 16 bytes", fn);
    if (a->page_table != nullptr)
        SAPA_REQUIRE(a->key_strides[2] >= 0 && a->value_strides[2] >= 0 && a->key_strides[2] % quantum == 0 && a->value_strides[2] % quantum == 0, SAPA_ERR_ALIGNMENT,
                     "%s: strides must be multiples of 16 bytes", fn);
    if (a->tokens == 0) return SAPA_OK;
    SAPA_REQUIRE(a->query != nullptr && a->out != nullptr, SAPA_ERR_ARGUMENT, "%s: query or out is NULL", fn);
    SAPA_REQUIRE(a->keys == 0 || (a->key != nullptr && a->value != nullptr), SAPA_ERR_ARGUMENT, "%s: key or value is NULL", fn);
    SAPA_REQUIRE(all_aligned16(a->query, a->key, a->value, a->out, a->low), SAPA_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", fn);
    return SAPA_OK;
}

static Args args_of(const sapa_attention *a) {
    Args p{};
    p.a = *a;
    const double scale = (double)a->scale * 1.4426950408889634;
    p.scale_log2 = (float)scale;
    p.scale_rest = (float)(scale - p.scale_log2);
    p.share = a->heads / a->groups;
    return p;
}

// A forward of this call: rows of a block, whether its keys are split, and the room that takes.
struct Shape {
    bool umma, narrow;
    int bm, tok, split, rows;      // rows: of a block that can be in use
    long long blocks, grid;        // blocks x groups at most; items at most
    size_t part, lse, bytes;       // of the workspace
};
static Shape shape_of(const Args &p, int dtype, int sms) {
    const sapa_attention &a = p.a;
    Shape s{};
    s.umma = umma_takes(a, dtype);
    if (s.umma) {
        // short sequences: a row tile a block, as long as an average sequence has no more rows
        s.narrow = (long long)a.tokens * p.share <= 128ll * a.B;
        s.tok = 128 / p.share * (s.narrow ? 1 : 2);
        s.bm = s.tok * p.share;
    } else {
        // single tokens and short chunks: 16 rows a block, as long as an average sequence has no more
        s.narrow = p.share <= 16 && (long long)a.tokens * p.share <= 16ll * a.B;
        s.bm = s.narrow ? 16 : 128;
        // few blocks of 128 rows: of 32, before keys are split (1342 tokens of 515-token sequences, 8 heads of 64 channels, float32: 80 us with 128 and split keys)
        if (!s.narrow && p.share <= 32 && most_blocks(a, a.tokens, 128 / p.share) * a.groups < 2ll * sms) s.bm = 32;
        s.tok = s.bm / p.share;
    }
    s.blocks = most_blocks(a, a.tokens, s.tok) * a.groups;
    s.rows = (a.tokens < s.tok ? a.tokens : s.tok) * p.share;
    s.grid = s.blocks;
    if (a.B == 0) return s;                          // no sequence: nothing to split
    // few blocks: their keys are split so that every SM has items
    const long long keys = a.page_table != nullptr ? (long long)a.max_pages * a.page : a.keys;
    if (s.blocks < 2ll * sms && keys > (s.umma ? 8 : 2) * TILE) {
        s.split = (s.umma ? (s.narrow ? 2 : 3) : 4) * sms;
        s.grid = s.blocks + s.split;
        s.part = (size_t)s.grid * s.bm * a.dim * sizeof(float);
        s.lse = (size_t)s.grid * s.bm * sizeof(float2);
        s.bytes = (s.part + s.lse + 255) / 256 * 256;
    }
    return s;
}

static int sm_count(const char *fn, int &sms) { return tmau::device_sms(fn, sms); }

template <typename T, int RI, int DP> static int run_rows(const Args &p, const Shape &s, cudaStream_t st) {
    using L = rows::Lay<RI, DP>;
    int sms = 0;
    if (int e = tmau::prepare_launch((const void *)sapa_attention_rows_kernel<T, RI, DP>, (int)L::SMEM, "sapa_attention_rows_kernel", sms)) return e;
    launch_next(sapa_attention_rows_kernel<T, RI, DP>, dim3((unsigned)s.grid), dim3(rows::NT), L::SMEM, st, p);
    return check_launch("sapa_attention_rows_kernel");
}

template <int DP, bool KEYS, bool SHARED> static int run_grad_by(const Args &p, const Grads &g, long long blocks, int ranks, cudaStream_t st) {
    using L = grad::Lay<DP>;
    int sms = 0;
    const auto kernel = sapa_attention_rows_grad_kernel<DP, KEYS, SHARED>;
    if (int e = tmau::prepare_launch((const void *)kernel, (int)L::SMEM, "sapa_attention_rows_grad_kernel", sms)) return e;
    if (SHARED) {                                    // launch_next, with a cluster
        cudaLaunchAttribute attributes[2];
        attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[0].val.programmaticStreamSerializationAllowed = 1;
        attributes[1].id = cudaLaunchAttributeClusterDimension;
        attributes[1].val.clusterDim.x = attributes[1].val.clusterDim.z = 1;
        attributes[1].val.clusterDim.y = (unsigned)ranks;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3((unsigned)blocks, (unsigned)ranks); config.blockDim = dim3(grad::THREADS); config.dynamicSmemBytes = L::SMEM; config.stream = st;
        config.attrs = attributes; config.numAttrs = 2;
        (void)cudaLaunchKernelEx(&config, kernel, p, g);      // a failure is what check_launch reads
    } else {
        launch_next(kernel, dim3((unsigned)blocks), dim3(grad::THREADS), L::SMEM, st, p, g);
    }
    return check_launch(KEYS ? "sapa_attention_rows_grad_kernel<keys>" : "sapa_attention_rows_grad_kernel<queries>");
}
// Hardly more blocks than SMs (the longest decide), and a team's turn of an average sequence more than two tiles: clusters of 2 or 4 blocks share the tiles of
// one.  Forward and gradients without and with that: one sequence of 1000 tokens, 4 heads of 128 channels, 398 and 290 us; of 500, 4 / 2 heads of 64, 164 and
// 89; 1342 tokens of three sequences, 8 / 4 heads (176 blocks of keys) 217 and 203.  Where it does not pay: 220 blocks of keys (sequences of some 200
// tokens, 16 / 8 heads) 148 and 170; sequences of some 260 tokens with a head to each key head (two tiles a turn) 119 and 122; 344 blocks of queries beside those
// 176 of keys 209 and 241.
template <int DP, bool KEYS> static int run_grad(const Args &p, const Grads &g, long long blocks, int sms, cudaStream_t st) {
    const sapa_attention &a = p.a;
    if (blocks == 0) return SAPA_OK;
    const long long tiles = (KEYS ? (long long)a.tokens * p.share : a.keys) / grad::OVER / (a.B > 0 ? a.B : 1);
    int ranks = 1;
    while (ranks < 4 && blocks * ranks <= (KEYS ? sms + sms / 4 : sms) && tiles > 2 * ranks * grad::TEAMS) ranks *= 2;
    return ranks > 1 ? run_grad_by<DP, KEYS, true>(p, g, blocks, ranks, st) : run_grad_by<DP, KEYS, false>(p, g, blocks, 1, st);
}

}  // namespace attn
}  // namespace sapa

using namespace sapa;
using namespace sapa::attn;

extern "C" size_t sapa_attention_workspace(const sapa_attention *a, int dtype) {
    int sms = 0;
    if (check(a, dtype, "sapa_attention_workspace") != SAPA_OK || a->tokens == 0 || sm_count("sapa_attention_workspace", sms) != SAPA_OK) return 0;
    return shape_of(args_of(a), dtype, sms).bytes;
}

extern "C" int sapa_attention_forward(const sapa_attention *a, void *workspace, size_t workspace_bytes, int dtype, void *stream) {
    const char *fn = "sapa_attention_forward";
    trace_reset();
    if (int e = check(a, dtype, fn)) return e;
    if (a->tokens == 0) return SAPA_OK;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int sms = 0;
    if (int e = sm_count(fn, sms)) return e;
    Args p = args_of(a);
    Shape s = shape_of(p, dtype, sms);
    if (s.grid == 0) s.grid = 1;                     // no sequence: every row is cleared
    SAPA_REQUIRE(s.grid < 0x3fffffffll, SAPA_ERR_UNSUPPORTED, "%s: too many blocks", fn);
    if (s.split > 0) {
        SAPA_REQUIRE(workspace != nullptr && workspace_bytes >= s.bytes, SAPA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", fn, s.bytes, workspace_bytes);
        SAPA_REQUIRE(aligned16(workspace), SAPA_ERR_ALIGNMENT, "%s: the workspace must be 256-byte aligned", fn);
        p.split = s.split;
        p.least = s.umma ? 4 : 1;
        p.part = static_cast<float *>(workspace);
        p.part_sums = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + s.part);
    }
    return SAPA_DISPATCH_FAST(dtype, [&]() -> int {
        int e;
        if (s.umma) e = umma_forward(p, !s.narrow, s.grid, dtype, st);
        else if (s.narrow) e = a->dim <= 64 ? run_rows<scalar_t, 1, 64>(p, s, st) : run_rows<scalar_t, 1, 128>(p, s, st);
        else if (s.bm == 32) e = a->dim <= 64 ? run_rows<scalar_t, 2, 64>(p, s, st) : run_rows<scalar_t, 2, 128>(p, s, st);
        else e = a->dim <= 64 ? run_rows<scalar_t, 8, 64>(p, s, st) : run_rows<scalar_t, 8, 128>(p, s, st);
        if (e != SAPA_OK || s.split == 0) return e;
        launch_next(sapa_attention_join_kernel<scalar_t>, dim3((unsigned)s.blocks, (unsigned)ceil_div(s.rows, 16)), dim3(256), 0, st, p, s.bm, s.tok);
        return check_launch("sapa_attention_join_kernel");
    });
}

// floats in a workspace: delta, in 16 bits lse in another order, in float16 the squares and factors too
static size_t floats(size_t n) { return (n * sizeof(float) + 255) / 256 * 256; }
static size_t row_floats(const sapa_attention *a) { return floats((size_t)a->tokens * a->heads); }
static size_t value_floats(const sapa_attention *a) { return floats((size_t)a->keys * a->groups); }

extern "C" size_t sapa_attention_backward_workspace(const sapa_attention *a, int dtype) {
    if (check(a, dtype, "sapa_attention_backward_workspace") != SAPA_OK) return 0;
    if (dtype == SAPA_F16) return 3 * row_floats(a) + value_floats(a) + floats((size_t)a->B * a->groups);
    return row_floats(a) * (dtype == SAPA_F32 ? 1 : 2);
}

extern "C" int sapa_attention_backward(const sapa_attention *a, const void *grad_out, long long grad_token_stride, long long grad_head_stride,
                                       void *grad_query, void *grad_key, void *grad_value, void *workspace, size_t workspace_bytes, int dtype,
                                       void *stream) {
    const char *fn = "sapa_attention_backward";
    trace_reset();
    if (int e = check(a, dtype, fn)) return e;
    SAPA_REQUIRE(a->page_table == nullptr, SAPA_ERR_UNSUPPORTED, "%s: the paged form has no gradients", fn);
    if (a->tokens == 0 && a->keys == 0) return SAPA_OK;
    const long long quantum = 16 / (long long)dtype_size(dtype);
    SAPA_REQUIRE(a->tokens == 0 || (grad_out != nullptr && grad_query != nullptr && a->lse != nullptr && a->low != nullptr), SAPA_ERR_ARGUMENT,
                 "%s: grad_out, grad_query, lse or low is NULL", fn);
    SAPA_REQUIRE(a->keys == 0 || (grad_key != nullptr && grad_value != nullptr), SAPA_ERR_ARGUMENT, "%s: grad_key or grad_value is NULL", fn);
    SAPA_REQUIRE(all_aligned16(grad_out, grad_query, grad_key, grad_value, workspace) && grad_token_stride >= 0 && grad_head_stride >= 0 &&
                     grad_token_stride % quantum == 0 && grad_head_stride % quantum == 0,
                 SAPA_ERR_ALIGNMENT, "%s: tensors and strides must be 16-byte aligned", fn);
    const size_t need = sapa_attention_backward_workspace(a, dtype);
    SAPA_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), SAPA_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", fn, need, workspace_bytes);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const Args p = args_of(a);
    if (a->tokens == 0 || a->keys == 0) {            // nothing is seen: every gradient is zero
        const size_t row = (size_t)a->dim * dtype_size(dtype), queries = (size_t)a->tokens * a->heads * row, keys = (size_t)a->keys * a->groups * row;
        if (queries != 0) cudaMemsetAsync(grad_query, 0, queries, st);
        if (keys != 0) { cudaMemsetAsync(grad_key, 0, keys, st); cudaMemsetAsync(grad_value, 0, keys, st); }
        return check_launch("memset");
    }
    const bool umma = dtype != SAPA_F32;
    char *const ws = static_cast<char *>(workspace);
    Grads g{grad_out, {grad_token_stride, grad_head_stride}, grad_query, grad_key, grad_value, reinterpret_cast<float *>(ws), nullptr, nullptr, nullptr, nullptr};
    if (umma) g.nlse = reinterpret_cast<float *>(ws + row_floats(a));
    if (dtype == SAPA_F16) {
        g.squares = reinterpret_cast<float *>(ws + 2 * row_floats(a));
        g.value_squares = reinterpret_cast<float *>(ws + 3 * row_floats(a));
        g.factor = reinterpret_cast<float *>(ws + 3 * row_floats(a) + value_floats(a));
    }
    int sms = 0;
    if (int e = sm_count(fn, sms)) return e;
    const int delta_rows = a->dim <= 64 ? 32 : 16;                    // of a block
    const long long delta_blocks = ((long long)a->tokens * a->heads + delta_rows - 1) / delta_rows + (dtype == SAPA_F16 ? ((long long)a->keys * a->groups + delta_rows - 1) / delta_rows : 0);
    const dim3 delta_grid((unsigned)(delta_blocks < (1ll << 20) ? delta_blocks : 1ll << 20));
    const int at_once = p.share < grad::OWN ? p.share : grad::OWN, slots = (p.share + at_once - 1) / at_once, tok = grad::OWN / at_once;
    const long long key_blocks = most_blocks(*a, a->keys, grad::OWN) * a->groups, query_blocks = most_blocks(*a, a->tokens, tok) * a->groups * slots;
    SAPA_REQUIRE(key_blocks < 0x7fffffffll && query_blocks < 0x7fffffffll && (long long)a->B * a->groups < 0x7fffffffll, SAPA_ERR_UNSUPPORTED, "%s: too many blocks", fn);
    return SAPA_DISPATCH_FAST(dtype, [&]() -> int {
        if (a->dim <= 64) launch_next(sapa_attention_delta_kernel<scalar_t, 8>, delta_grid, dim3(256), 0, st, p, g);
        else launch_next(sapa_attention_delta_kernel<scalar_t, 16>, delta_grid, dim3(256), 0, st, p, g);
        if (int e = check_launch("sapa_attention_delta_kernel")) return e;
        if (dtype == SAPA_F16 && a->B > 0) {
            const unsigned factors = (unsigned)(a->B * a->groups);
            if (factors > 4u * (unsigned)sms) launch_next(sapa_attention_factor_kernel<true>, dim3((factors + 7) / 8), dim3(256), 0, st, p, g);
            else launch_next(sapa_attention_factor_kernel<false>, dim3(factors), dim3(1024), 0, st, p, g);
            if (int e = check_launch("sapa_attention_factor_kernel")) return e;
        }
        if (umma) return umma_backward(p, g, dtype, st);
        if (a->dim <= 64) {
            if (int e = run_grad<64, true>(p, g, key_blocks, sms, st)) return e;
            return run_grad<64, false>(p, g, query_blocks, sms, st);
        }
        if (int e = run_grad<128, true>(p, g, key_blocks, sms, st)) return e;
        return run_grad<128, false>(p, g, query_blocks, sms, st);
    });
}

extern "C" int sapa_paged_write(const sapa_paged_rows *a, int dtype, void *stream) {
    const char *fn = "sapa_paged_write";
    trace_reset();
    SAPA_REQUIRE(a != nullptr, SAPA_ERR_ARGUMENT, "%s: the arguments are NULL", fn);
    const long long esize = (long long)dtype_size(dtype);
    SAPA_REQUIRE(esize != 0, SAPA_ERR_DTYPE, "%s: dtype code %d is not supported", fn, dtype);
    SAPA_REQUIRE(a->B >= 0 && a->tokens >= 0 && a->groups > 0 && a->dim > 0 && a->pages > 0 && a->page > 0 && a->max_pages > 0, SAPA_ERR_ARGUMENT, "%s: sizes must be positive", fn);
    SAPA_REQUIRE(a->dim * esize % 16 == 0, SAPA_ERR_UNSUPPORTED, "%s: rows must be multiples of 16 bytes", fn);
    for (long long s : {a->key_strides[0], a->key_strides[1], a->value_strides[0], a->value_strides[1], a->key_page_strides[0], a->key_page_strides[1],
                        a->key_page_strides[2], a->value_page_strides[0], a->value_page_strides[1], a->value_page_strides[2]})
        SAPA_REQUIRE(s >= 0 && s * esize % 16 == 0, SAPA_ERR_ALIGNMENT, "%s: strides must be multiples of 16 bytes", fn);
    if (a->tokens == 0 || a->B == 0) return SAPA_OK;
    SAPA_REQUIRE(a->key != nullptr && a->value != nullptr && a->key_pages != nullptr && a->value_pages != nullptr, SAPA_ERR_ARGUMENT, "%s: a tensor is NULL", fn);
    SAPA_REQUIRE(a->offsets != nullptr && a->page_table != nullptr && a->key_lengths != nullptr, SAPA_ERR_ARGUMENT, "%s: offsets, page_table or key_lengths is NULL", fn);
    SAPA_REQUIRE(all_aligned16(a->key, a->value, a->key_pages, a->value_pages), SAPA_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", fn);
    int sms = 0;
    if (int e = sm_count(fn, sms)) return e;
    const long long warps = (long long)a->tokens * ((a->groups * (a->dim * esize / 16) + 127) / 128), blocks = (warps + 7) / 8;
    launch_next(sapa_paged_write_kernel, dim3((unsigned)(blocks < 16ll * sms ? blocks : 16ll * sms)), dim3(256), 0, static_cast<cudaStream_t>(stream), *a, (int)esize);
    return check_launch("sapa_paged_write_kernel");
}
