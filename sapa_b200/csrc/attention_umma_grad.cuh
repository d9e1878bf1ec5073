// attention_umma_grad.cuh — the gradients of attention over sequences in 16 bits on the 5th-generation tensor cores.  Included by
// attention_umma.cu behind attention_umma.cuh.
//
// P and dS of a tile are formed again: P = 2^(scale s - lse), dS = P (dP - delta), rounded to the inputs' type for the products that take them from
// tensor memory; the sums are float32.  Two kernels without atomics, so that results do not depend on the order of anything:
//   * keys: a block holds 128 keys and values and goes over the row tiles (token x query head) that see them.  S^T = K Q^T and dP^T = V dO^T have the keys in
//     the lanes of tensor memory, so that P^T and dS^T are first operands of dV += P^T dO and dK += dS^T Q as they are;
//   * queries: a block holds a row tile and goes over the key tiles: S = Q K^T, dP = dO V^T, dQ += dS K.
// Seven products where five would do with dQ summed by atomics; each operand is in shared memory once, K-major for one product and MN-major for another.
// Two warpgroups take half of a tile's columns each.
// What a row does not see: P and dS are 0 there, and 0 * infinity must not reach a gradient.  In tiles that are not seen whole, what is not finite in the
// operand behind P or dS is replaced with 0 once the products that need it as it is have read it.  Values that are not finite in a row of dO are
// added to the gradients of the values that it sees; those of keys that a row sees make its gradient NaN; a row of Q makes its P NaN by itself.
#pragma once

#include "attention_umma.cuh"

namespace sapa {
namespace attn {
namespace umg {

using namespace um;

constexpr int THREADS = 10 * 32;

template <int D> struct KeyLay {
    static constexpr int TILE_BYTES = D / 64 * BLOCK_BYTES, NST = D == 64 ? 3 : 2;
    static constexpr int K0 = 0, V0 = TILE_BYTES, Q0 = 2 * TILE_BYTES, O0 = Q0 + NST * TILE_BYTES, END = O0 + NST * TILE_BYTES;
    static constexpr int NEED = END + 1024, SMEM = NEED < 120 * 1024 ? 120 * 1024 : NEED;
    static constexpr int S_COL = 0, P_COL = 128, V_COL = 256, K_COL = 256 + D, TMEM_COLS = 512;      // S^T, dP^T, dV, dK
};
template <int D> struct QueryLay {
    static constexpr int TILE_BYTES = D / 64 * BLOCK_BYTES, NK = D == 64 ? 4 : 3, NV = D == 64 ? 3 : 2;
    static constexpr int Q0 = 0, O0 = TILE_BYTES, K0 = 2 * TILE_BYTES, V0 = K0 + NK * TILE_BYTES, END = V0 + NV * TILE_BYTES;
    static constexpr int NEED = END + 1024, SMEM = NEED < 120 * 1024 ? 120 * 1024 : NEED;
    static constexpr int S_COL = 0, P_COL = 256, Q_COL = 384, TMEM_COLS = 512;                       // S twice, dP, dQ
};

// D[128 x N] (+)= A[128 x 16 KSTEPS] B, A and B K-major in shared memory
template <typename T, int D> __device__ __forceinline__ void mma_rows(unsigned leader, unsigned d, unsigned a, unsigned b) {
    constexpr unsigned IDESC = IDESC_M128<T> | idesc_n(128);
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
        tc_mma<false>(leader, d, a + (c >> 2) * (BLOCK_BYTES >> 4) + (c & 3) * 2, b + (c >> 2) * (BLOCK_BYTES >> 4) + (c & 3) * 2, HI, IDESC, c > 0 ? 1u : 0u);
}
// D[128 x D] (+)= A[128 x 128] B: A in tensor memory as the two warpgroups leave it (64 columns' 32 words each, 64 apart), B MN-major
template <typename T, int D> __device__ __forceinline__ void mma_columns(unsigned leader, unsigned d, unsigned a, unsigned b, bool add) {
    constexpr unsigned IDESC = IDESC_M128<T> | (1u << 16) | idesc_n(D);
#pragma unroll
    for (int c = 0; c < 8; ++c)
        tc_mma_ta<false>(leader, d, a + (c >> 2) * 64 + (c & 3) * 8, b + c * (2048 >> 4), HI, IDESC, add || c > 0 ? 1u : 0u);
}
template <typename T> __device__ __forceinline__ void store_packed(unsigned taddr, const float *v) {
#pragma unroll
    for (int c = 0; c < 64; c += 32) {
        unsigned w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pack_pair(T(), v[c + 2 * e], v[c + 2 * e + 1]);
        tc_st16(taddr + c / 2, w);
    }
}

}  // namespace umg

template <typename T, int D>
__global__ void __launch_bounds__(umg::THREADS, 1) sapa_attention_umma_keys_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap omap,
                                                                             const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                             const __grid_constant__ Args p, const __grid_constant__ Grads g) {
    using namespace umg;
    using L = KeyLay<D>;
    constexpr int NST = L::NST;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(16) float row_lse[NST][ROWS], row_delta[NST][ROWS];
    __shared__ __align__(8) unsigned long long bars[1 + 5 * NST + 5];
    __shared__ unsigned tmem_slot;
    __shared__ Item item;
    __shared__ int odd_first, odd_last;
    const sapa_attention &a = p.a;
    const unsigned base = ((unsigned)__cvta_generic_to_shared(smem_dyn) + 1023u) & ~1023u;
    const unsigned kvfull = (unsigned)__cvta_generic_to_shared(bars), qfull = kvfull + 8, qempty = qfull + 8 * NST, ofull = qempty + 8 * NST, oempty = ofull + 8 * NST;
    const unsigned lfull = oempty + 8 * NST, sfull = lfull + 8 * NST, pfull = sfull + 8, dpfull = pfull + 8, dsfull = dpfull + 8, done = dsfull + 8;
    const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
    const int group = blockIdx.x % a.groups, tok = ROWS / p.share, rows = tok * p.share;

    if (warp == MMA_WARP) {
        if (lane == 0) {
            mbar_init(kvfull, 1);
            for (int i = 0; i < NST; ++i) {
                mbar_init(qfull + 8 * i, 1); mbar_init(qempty + 8 * i, 1); mbar_init(ofull + 8 * i, 1); mbar_init(oempty + 8 * i, 1);
                mbar_init(lfull + 8 * i, 32);
            }
            mbar_init(sfull, 1); mbar_init(dpfull, 1); mbar_init(done, 1); mbar_init(pfull, 256); mbar_init(dsfull, 256);
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            odd_first = 0x7fffffff; odd_last = -1;
        }
        __syncwarp();
        tc_alloc((unsigned)__cvta_generic_to_shared(&tmem_slot), L::TMEM_COLS);
        tc_relinquish();
    }
    // rows that no copy fills: they are behind P and dS, which are 0 there
    for (int i = tid; i < (ROWS - rows) * 8 * (D / 64) * 2 * NST; i += THREADS) {
        const int tile = i / ((ROWS - rows) * 8), e = i % ((ROWS - rows) * 8);
        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(base + L::Q0 + tile * BLOCK_BYTES + (rows + e / 8) * 128 + (e % 8) * 16), "r"(0u) : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    begin_after_previous();
    if (warp == 0) {
        const Item r = InOrder<false, KeyBlocks>(a, KeyBlocks{a.causal != 0, tok, KT}, lane).at(blockIdx.x / a.groups);
        if (lane == 0) item = r;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = warp_uniform(*reinterpret_cast<volatile unsigned *>(&tmem_slot));
    bool ok = true;
    if (item.there) {
        const Sequence s = sequence_at(a, item.b);
        const int k0 = item.block * KT;
        const int from = a.causal ? (int)max(0ll, (long long)k0 - s.nk + s.nq) : 0;      // the first token that sees one of the keys
        const int n = (int)warp_uniform(from < s.nq ? (s.nq - from + tok - 1) / tok : 0);
        if (warp == LOAD_WARP) {
            int st = 0, ph = 0;
            if (lane == 0) {
                mbar_expect_tx(kvfull, 2 * L::TILE_BYTES);
                for (int b = 0; b < D / 64; ++b) {
                    tma_load_3d(base + L::K0 + b * BLOCK_BYTES, &kmap, kvfull, 64 * b, group, s.k0 + k0);
                    tma_load_3d(base + L::V0 + b * BLOCK_BYTES, &vmap, kvfull, 64 * b, group, s.k0 + k0);
                }
            }
            const long long at0 = ((long long)group * a.tokens + s.q0 + from) * p.share, end = (long long)a.tokens * a.heads;
            float e[4], d[4];
            auto fetch = [&](int i) {                                 // a tile's lse and delta, ahead of their use
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const long long at = at0 + (long long)i * rows + lane + 32 * r;
                    e[r] = at < end ? g.nlse[at] : 0.f;
                    d[r] = at < end ? g.delta[at] : 0.f;
                }
            };
            if (n > 0) fetch(0);
            for (int i = 0; i < n && ok; ++i) {
                if (lane == 0) {
                    ok = mbar_wait_bounded(qempty + 8 * st, ph ^ 1);
                    if (ok) {
                        mbar_expect_tx(qfull + 8 * st, (D / 64) * 128 * rows);
                        for (int b = 0; b < D / 64; ++b)
                            tma_load_3d(base + L::Q0 + st * L::TILE_BYTES + b * BLOCK_BYTES, &qmap, qfull + 8 * st, 64 * b, group * p.share, s.q0 + from + i * tok);
                        ok = mbar_wait_bounded(oempty + 8 * st, ph ^ 1);
                        if (!ok) (void)mbar_wait_bounded(qfull + 8 * st, ph);
                    }
                    if (ok) {
                        mbar_expect_tx(ofull + 8 * st, (D / 64) * 128 * rows);
                        for (int b = 0; b < D / 64; ++b)
                            tma_load_3d(base + L::O0 + st * L::TILE_BYTES + b * BLOCK_BYTES, &omap, ofull + 8 * st, 64 * b, group * p.share, s.q0 + from + i * tok);
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
                if (!ok) break;
#pragma unroll
                for (int r = 0; r < 4; ++r) { row_lse[st][lane + 32 * r] = e[r]; row_delta[st][lane + 32 * r] = d[r]; }
                mbar_arrive(lfull + 8 * st);
                if (i + 1 < n) fetch(i + 1);
                if (++st == NST) { st = 0; ph ^= 1; }
            }
            if (lane == 0) {
                ok = mbar_wait_bounded(kvfull, 0) && ok;
                if (!ok) {                                            // none of its loads may land after it has left
                    (void)drain_loads<NST>(qfull, st, ph);
                    (void)drain_loads<NST>(ofull, st, ph);
                }
            }
        } else if (warp == MMA_WARP) {
            const unsigned leader = elect_leader();
            const unsigned k_rows = warp_uniform(desc_lo(base + L::K0, 16)), v_rows = warp_uniform(desc_lo(base + L::V0, 16));
            const unsigned q_rows = warp_uniform(desc_lo(base + L::Q0, 16)), o_rows = warp_uniform(desc_lo(base + L::O0, 16));
            const unsigned q_cols = warp_uniform(desc_lo(base + L::Q0, BLOCK_BYTES)), o_cols = warp_uniform(desc_lo(base + L::O0, BLOCK_BYTES));
            constexpr unsigned STEP = L::TILE_BYTES >> 4;
            ok = mbar_wait_warp(kvfull, 0);
            if (n > 0 && ok) {
                ok = mbar_wait_warp(qfull, 0);
                if (ok) { tc_fence_after(); mma_rows<T, D>(leader, tmem + L::S_COL, k_rows, q_rows); tc_commit_by(leader, sfull); }
                ok = ok && mbar_wait_warp(ofull, 0);
                if (ok) { mma_rows<T, D>(leader, tmem + L::P_COL, v_rows, o_rows); tc_commit_by(leader, dpfull); }
            }
            int st = 0, next = 1 % NST, next_ph = NST == 1 ? 1 : 0;
            for (int i = 0; i < n && ok; ++i) {
                ok = mbar_wait_warp(pfull, i & 1);
                if (!ok) break;
                tc_fence_after();
                mma_columns<T, D>(leader, tmem + L::V_COL, tmem + L::S_COL, o_cols + st * STEP, i > 0);
                tc_commit_by(leader, oempty + 8 * st);
                if (i + 1 < n) {
                    ok = mbar_wait_warp(qfull + 8 * next, next_ph);
                    if (!ok) break;
                    mma_rows<T, D>(leader, tmem + L::S_COL, k_rows, q_rows + next * STEP);
                    tc_commit_by(leader, sfull);
                }
                ok = mbar_wait_warp(dsfull, i & 1);
                if (!ok) break;
                tc_fence_after();
                mma_columns<T, D>(leader, tmem + L::K_COL, tmem + L::P_COL, q_cols + st * STEP, i > 0);
                tc_commit_by(leader, qempty + 8 * st);
                if (i + 1 < n) {
                    ok = mbar_wait_warp(ofull + 8 * next, next_ph);
                    if (!ok) break;
                    mma_rows<T, D>(leader, tmem + L::P_COL, v_rows, o_rows + next * STEP);
                    tc_commit_by(leader, dpfull);
                }
                st = next;
                if (++next == NST) { next = 0; next_ph ^= 1; }
            }
            if (n > 0 && ok) tc_commit_by(leader, done);
        } else {
            const int half = warp >> 2, r = tid & 127, key = k0 + r;      // columns [64 half, 64 half + 64) of this thread's key
            const unsigned quarter = (unsigned)((warp & 3) * 32) << 16;
            const unsigned s_at = tmem + quarter + L::S_COL + 64 * half, d_at = tmem + quarter + L::P_COL + 64 * half;
            int st = 0, ph = 0;
            for (int i = 0; i < n; ++i) {
                const int token = from + i * tok, used = min(rows, (s.nq - token) * p.share);
                // rows from `low` on see the key
                const long long before = (long long)key - s.nk + s.nq - token;
                const int low = a.causal && before > 0 ? (int)min(before * p.share, 1ll << 20) : 0;
                const bool part = used < ROWS || (a.causal && (long long)k0 + KT - 1 - s.nk + s.nq - token > 0);
                if (!mbar_wait_warp(lfull + 8 * st, ph) || !mbar_wait_warp(sfull, i & 1)) { ok = false; break; }
                tc_fence_after();
                float x[64], y[64];
                tc_ld32(s_at, x);
                tc_ld32(s_at + 32, x + 32);
                tc_wait_ld();
                const float2 scale = make_float2(p.scale_log2, p.scale_log2);
                const float4 *lse = reinterpret_cast<const float4 *>(&row_lse[st][64 * half]), *delta = reinterpret_cast<const float4 *>(&row_delta[st][64 * half]);
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    const float4 e = lse[c >> 2];
                    const float2 u = fma2(make_float2(x[c], x[c + 1]), scale, make_float2(e.x, e.y)), w = fma2(make_float2(x[c + 2], x[c + 3]), scale, make_float2(e.z, e.w));
                    x[c] = ex2_ftz(u.x); x[c + 1] = ex2_ftz(u.y); x[c + 2] = ex2_ftz(w.x); x[c + 3] = ex2_ftz(w.y);
                }
                const int lo = low - 64 * half, hi = used - 64 * half;
                if (part) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) x[c] = c >= lo && c < hi ? x[c] : 0.f;
                }
                store_packed<T>(s_at, x);
                if (part) {                                           // dP has been computed from dO as it is, S from Q
                    if (!mbar_wait_warp(dpfull, i & 1)) { ok = false; break; }
                    if (half == 0) {
                        if (clean_row<T, D>(base + L::O0 + st * L::TILE_BYTES, r) && r < used) { atomicMin(&odd_first, i * rows + r); atomicMax(&odd_last, i * rows + r); }
                    } else {
                        (void)clean_row<T, D>(base + L::Q0 + st * L::TILE_BYTES, r);
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(pfull);
                if (!mbar_wait_warp(dpfull, i & 1)) { ok = false; break; }
                tc_fence_after();
                tc_ld32(d_at, y);
                tc_ld32(d_at + 32, y + 32);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 64; c += 4) {
                    const float4 e = delta[c >> 2];
                    const float2 u = mul2(make_float2(x[c], x[c + 1]), add2(make_float2(y[c], y[c + 1]), make_float2(-e.x, -e.y)));
                    const float2 w = mul2(make_float2(x[c + 2], x[c + 3]), add2(make_float2(y[c + 2], y[c + 3]), make_float2(-e.z, -e.w)));
                    y[c] = u.x; y[c + 1] = u.y; y[c + 2] = w.x; y[c + 3] = w.y;
                }
                if (part) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) y[c] = c >= lo && c < hi ? y[c] : 0.f;
                }
                store_packed<T>(d_at, y);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(dsfull);
                if (++st == NST) { st = 0; ph ^= 1; }
            }
            if (ok && n > 0) ok = mbar_wait_warp(done, 0);
            tc_fence_after();
            // the first warpgroup stores the gradients of the values, the second those of the keys
            const unsigned at = tmem + quarter + (half == 0 ? L::V_COL : L::K_COL);
            const float factor = half == 0 ? 1.f : a.scale;
            T *const to = static_cast<T *>(half == 0 ? g.gv : g.gk) + ((long long)(s.k0 + key) * a.groups + group) * a.dim;
            const int odd0 = odd_first, odd1 = odd_last;
#pragma unroll 1
            for (int c = 0; c < D && c < a.dim && ok; c += 32) {
                float o[32];
                if (n > 0) {
                    tc_ld32(at + c, o);
                    tc_wait_ld();
                }
                if (key >= s.nk) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = n > 0 ? o[e] * factor : 0.f;
                if (half == 0 && odd1 >= 0) {                         // rare: rows of dO with something not finite that see this value
                    for (int row = odd0; row <= odd1; ++row) {
                        const int i = from + row / p.share;
                        if (key >= sees(s, i, a.causal)) continue;
                        const T *v = static_cast<const T *>(g.go) + (long long)(s.q0 + i) * g.go_strides[0] + (long long)(group * p.share + row % p.share) * g.go_strides[1] + c;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float f = c + e < a.dim ? to_acc(v[e]) : 0.f;
                            if (!isfinite(f)) o[e] += f;
                        }
                    }
                }
                store_row(to + c, o, a.dim - c);
            }
        }
    }
    if (!ok) atomicExch(&g_wait_timeout, 1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP) tc_dealloc(tmem, L::TMEM_COLS);
}

template <typename T, int D>
__global__ void __launch_bounds__(umg::THREADS, 1) sapa_attention_umma_queries_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap omap,
                                                                                const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                                const __grid_constant__ Args p, const __grid_constant__ Grads g) {
    using namespace umg;
    using L = QueryLay<D>;
    constexpr int NK = L::NK, NV = L::NV;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) unsigned long long bars[1 + 2 * NK + 2 * NV + 5];
    __shared__ unsigned tmem_slot;
    __shared__ Item item;
    __shared__ int odd_first, odd_last;
    const sapa_attention &a = p.a;
    const unsigned base = ((unsigned)__cvta_generic_to_shared(smem_dyn) + 1023u) & ~1023u;
    const unsigned qofull = (unsigned)__cvta_generic_to_shared(bars), kfull = qofull + 8, kempty = kfull + 8 * NK, vfull = kempty + 8 * NK, vempty = vfull + 8 * NV;
    const unsigned sfull = vempty + 8 * NV, dpfull = sfull + 16, dsfull = dpfull + 8, done = dsfull + 8;
    const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
    const int group = blockIdx.x % a.groups, tok = ROWS / p.share, rows = tok * p.share;

    if (warp == MMA_WARP) {
        if (lane == 0) {
            mbar_init(qofull, 1);
            for (int i = 0; i < NK; ++i) { mbar_init(kfull + 8 * i, 1); mbar_init(kempty + 8 * i, 1); }
            for (int i = 0; i < NV; ++i) { mbar_init(vfull + 8 * i, 1); mbar_init(vempty + 8 * i, 1); }
            mbar_init(sfull, 1); mbar_init(sfull + 8, 1); mbar_init(dpfull, 1); mbar_init(done, 1); mbar_init(dsfull, 256);
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            odd_first = 0x7fffffff; odd_last = -1;
        }
        __syncwarp();
        tc_alloc((unsigned)__cvta_generic_to_shared(&tmem_slot), L::TMEM_COLS);
        tc_relinquish();
    }
    begin_after_previous();
    if (warp == 0) {
        const Item r = InOrder<true, QueryBlocks>(a, QueryBlocks{a.causal != 0, tok, KT}, lane).at(blockIdx.x / a.groups);
        if (lane == 0) item = r;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = warp_uniform(*reinterpret_cast<volatile unsigned *>(&tmem_slot));
    bool ok = true;
    if (item.there) {
        const Sequence s = sequence_at(a, item.b);
        const int first = item.block * tok, used = min(tok, s.nq - first) * p.share;
        const int n = (int)warp_uniform((sees(s, first + used / p.share - 1, a.causal) + KT - 1) / KT);
        if (warp == LOAD_WARP) {
            if (lane == 0) {
                mbar_expect_tx(qofull, 2 * (D / 64) * 128 * rows);
                for (int b = 0; b < D / 64; ++b) {
                    tma_load_3d(base + L::Q0 + b * BLOCK_BYTES, &qmap, qofull, 64 * b, group * p.share, s.q0 + first);
                    tma_load_3d(base + L::O0 + b * BLOCK_BYTES, &omap, qofull, 64 * b, group * p.share, s.q0 + first);
                }
                int ks = 0, kph = 0, vs = 0, vph = 0;
                for (int i = 0; i < n && ok; ++i) {
                    ok = mbar_wait_bounded(kempty + 8 * ks, kph ^ 1);
                    if (!ok) break;
                    mbar_expect_tx(kfull + 8 * ks, L::TILE_BYTES);
                    for (int b = 0; b < D / 64; ++b) tma_load_3d(base + L::K0 + ks * L::TILE_BYTES + b * BLOCK_BYTES, &kmap, kfull + 8 * ks, 64 * b, group, s.k0 + i * KT);
                    if (++ks == NK) { ks = 0; kph ^= 1; }
                    ok = mbar_wait_bounded(vempty + 8 * vs, vph ^ 1);
                    if (!ok) break;
                    mbar_expect_tx(vfull + 8 * vs, L::TILE_BYTES);
                    for (int b = 0; b < D / 64; ++b) tma_load_3d(base + L::V0 + vs * L::TILE_BYTES + b * BLOCK_BYTES, &vmap, vfull + 8 * vs, 64 * b, group, s.k0 + i * KT);
                    if (++vs == NV) { vs = 0; vph ^= 1; }
                }
                ok = mbar_wait_bounded(qofull, 0) && ok;
                if (!ok) {
                    (void)drain_loads<NK>(kfull, ks, kph);
                    (void)drain_loads<NV>(vfull, vs, vph);
                }
            }
        } else if (warp == MMA_WARP) {
            const unsigned leader = elect_leader();
            const unsigned q_rows = warp_uniform(desc_lo(base + L::Q0, 16)), o_rows = warp_uniform(desc_lo(base + L::O0, 16));
            const unsigned k_rows = warp_uniform(desc_lo(base + L::K0, 16)), v_rows = warp_uniform(desc_lo(base + L::V0, 16));
            const unsigned k_cols = warp_uniform(desc_lo(base + L::K0, BLOCK_BYTES));
            constexpr unsigned STEP = L::TILE_BYTES >> 4;
            int ks = 0, kph = 0, vs = 0, vph = 0, used_k = 0;         // next to wait for; stage of the keys of the tile in turn
            auto scores = [&](int i) {
                ok = ok && mbar_wait_warp(kfull + 8 * ks, kph);
                if (!ok) return;
                mma_rows<T, D>(leader, tmem + L::S_COL + 128 * (i & 1), q_rows, k_rows + ks * STEP);
                tc_commit_by(leader, sfull + 8 * (i & 1));
                if (++ks == NK) { ks = 0; kph ^= 1; }
            };
            auto products = [&]() {                                   // dP
                ok = ok && mbar_wait_warp(vfull + 8 * vs, vph);
                if (!ok) return;
                mma_rows<T, D>(leader, tmem + L::P_COL, o_rows, v_rows + vs * STEP);
                tc_commit_by(leader, dpfull);
                tc_commit_by(leader, vempty + 8 * vs);
                if (++vs == NV) { vs = 0; vph ^= 1; }
            };
            ok = mbar_wait_warp(qofull, 0);
            tc_fence_after();
            if (n > 0) { scores(0); products(); }
            if (n > 1) scores(1);
            for (int i = 0; i < n && ok; ++i) {
                ok = mbar_wait_warp(dsfull, i & 1);
                if (!ok) break;
                tc_fence_after();
                mma_columns<T, D>(leader, tmem + L::Q_COL, tmem + L::P_COL, k_cols + used_k * STEP, i > 0);
                tc_commit_by(leader, kempty + 8 * used_k);
                if (++used_k == NK) used_k = 0;
                if (i + 1 < n) products();
                if (i + 2 < n) scores(i + 2);
            }
            if (n > 0 && ok) tc_commit_by(leader, done);
        } else {
            const int half = warp >> 2, r = tid & 127, token = first + r / p.share;
            const bool mine = r < used;
            const unsigned quarter = (unsigned)((warp & 3) * 32) << 16;
            const unsigned d_at = tmem + quarter + L::P_COL + 64 * half;
            const int lim = mine ? sees(s, token, a.causal) : 0, least = sees(s, first, a.causal);
            const long long row = ((long long)group * a.tokens + s.q0 + first) * p.share + r;
            const float nlse = mine ? g.nlse[row] : 0.f, delta = mine ? g.delta[row] : 0.f;
            int st = 0;
            for (int i = 0; i < n; ++i) {
                const int k0 = i * KT, left = lim - k0 - 64 * half;
                const bool part = k0 + KT > least;
                const unsigned s_at = tmem + quarter + L::S_COL + 128 * (i & 1) + 64 * half;
                if (!mbar_wait_warp(sfull + 8 * (i & 1), (i >> 1) & 1)) { ok = false; break; }
                tc_fence_after();
                float x[64], y[64];
                tc_ld32(s_at, x);
                tc_ld32(s_at + 32, x + 32);
                tc_wait_ld();
                const float2 scale = make_float2(p.scale_log2, p.scale_log2), e = make_float2(nlse, nlse), d = make_float2(-delta, -delta);
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float2 u = fma2(make_float2(x[c], x[c + 1]), scale, e);
                    x[c] = ex2_ftz(u.x); x[c + 1] = ex2_ftz(u.y);
                }
                if (part && half == 0) {                              // the scores have been computed from the keys as they are
                    if (clean_row<T, D>(base + L::K0 + st * L::TILE_BYTES, r) && k0 + r < s.nk) { atomicMin(&odd_first, k0 + r); atomicMax(&odd_last, k0 + r); }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                if (!mbar_wait_warp(dpfull, i & 1)) { ok = false; break; }
                tc_fence_after();
                tc_ld32(d_at, y);
                tc_ld32(d_at + 32, y + 32);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 64; c += 2) {
                    const float2 u = mul2(make_float2(x[c], x[c + 1]), add2(make_float2(y[c], y[c + 1]), d));
                    y[c] = u.x; y[c + 1] = u.y;
                }
                if (part) {
#pragma unroll
                    for (int c = 0; c < 64; ++c) y[c] = c < left ? y[c] : 0.f;
                }
                store_packed<T>(d_at, y);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(dsfull);
                if (++st == NK) st = 0;
            }
            if (ok && n > 0) ok = mbar_wait_warp(done, 0);
            tc_fence_after();
            // each warpgroup stores half of the channels
            T *const to = static_cast<T *>(g.gq) + ((long long)(s.q0 + token) * a.heads + group * p.share + r % p.share) * a.dim;
            const int odd0 = odd_first, odd1 = odd_last;
#pragma unroll 1
            for (int c = half * (D / 2); c < (half + 1) * (D / 2) && c < a.dim && ok; c += 32) {
                float o[32];
                if (n > 0) {
                    tc_ld32(tmem + quarter + L::Q_COL + c, o);
                    tc_wait_ld();
                }
                if (!mine) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = n > 0 && lim > 0 ? o[e] * a.scale : 0.f;
                if (odd1 >= 0) {                                      // rare: keys with something not finite that this row sees
                    for (int k = odd0; k <= min(lim - 1, odd1); ++k) {
                        const T *v = static_cast<const T *>(a.key) + (long long)(s.k0 + k) * a.key_strides[0] + group * a.key_strides[1] + c;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float f = c + e < a.dim ? to_acc(v[e]) : 0.f;
                            if (!isfinite(f)) o[e] = __int_as_float(0x7fffffff);
                        }
                    }
                }
                store_row(to + c, o, a.dim - c);
            }
        }
    }
    if (!ok) atomicExch(&g_wait_timeout, 1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP) tc_dealloc(tmem, L::TMEM_COLS);
}

}  // namespace attn
}  // namespace sapa
