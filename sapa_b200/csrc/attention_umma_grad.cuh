// attention_umma_grad.cuh — the gradients of attention over sequences in 16 bits on the 5th-generation tensor cores.  Included by
// attention_umma.cu behind attention_umma.cuh.
//
// P and dS of a tile are formed again: P = 2^(scale s - lse), dS = P (dP - delta), rounded to the inputs' type for the products that take them from
// tensor memory; the sums are float32.  Two launches of one kernel, without atomics, so that results do not depend on the order of anything:
//   * KEYS: an item holds 128 keys and values and goes over the rows (token x query head) that see them.  S^T = K Q^T and dP^T = V dO^T have the keys in
//     the lanes of tensor memory, so that P^T and dS^T are first operands of dV += P^T dO and dK += dS^T Q as they are;
//   * otherwise an item holds 128 rows and goes over the keys that they see: S = Q K^T, dP = dO V^T, dQ += dS K.
// Seven products where five would do with dQ summed by atomics; each operand is in shared memory once, K-major for one product and MN-major for another.
// What is gone over comes in tiles of 64, so that tensor memory holds S and dP of two: a warpgroup each takes every other tile (a thread a lane, 64 columns) while
// the products of the other one run.  (Tiles of 128 shared by both warpgroups, with one S and dP: 3100 clocks a 128 x 128 tile of keys' gradients in
// 128 channels, of which the products are 2048.)  A block an SM goes through its items, as the forward does.
// What a row does not see: P and dS are 0 there, and 0 * infinity must not reach a gradient.  In tiles that are not seen whole, what is not finite in the
// operand behind P or dS is replaced with 0 once the products that need it as it is have read it.  Values that are not finite in a row of dO are
// added to the gradients of the values that it sees; those of keys that a row sees make its gradient NaN; a row of Q makes its P NaN by itself.
#pragma once

#include "attention_umma.cuh"

namespace sapa {
namespace attn {
namespace umg {

using namespace um;

constexpr int N = 64, BOX_BYTES = N * 128;                            // rows of a tile that is gone over
constexpr int ROW_WARP = VALUE_WARP;                                  // loads lse and delta

template <int D> struct Lay {
    static constexpr int OWN = D / 64 * BLOCK_BYTES, HALF = D / 64 * BOX_BYTES, STAGE = 2 * HALF, NST = D == 64 ? 8 : 4;
    static constexpr int OWN0 = 0, ST0 = 2 * OWN, NEED = ST0 + NST * STAGE + 1024, SMEM = NEED < 120 * 1024 ? 120 * 1024 : NEED;
    static constexpr int S_COL = 0, P_COL = 2 * N, ACC_COL = 4 * N, TMEM_COLS = 512;      // S twice, dP twice, dV and dK or dQ
    static_assert(SMEM <= 222 * 1024 && ACC_COL + 2 * D <= TMEM_COLS, "shared memory, with lse and delta; tensor memory");
};

// An item of a block
struct Work {
    bool there;
    int b, group, n;               // tiles to go over
    int first;                     // KEYS: first key; otherwise first token
    int from, turns;               // KEYS: the first token that sees a key; tiles that the heads of a token take
    Sequence s;
    int odd_first, odd_last;       // rows or keys with something not finite, of tiles that are not seen whole
};

// S[128 x 64] = A B^T, both K-major in shared memory
template <typename T, int D> __device__ __forceinline__ void mma_rows(unsigned leader, unsigned d, unsigned a, unsigned b) {
    constexpr unsigned IDESC = IDESC_M128<T> | idesc_n(N);
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
        tc_mma<false>(leader, d, a + (c >> 2) * (BLOCK_BYTES >> 4) + (c & 3) * 2, b + (c >> 2) * (BOX_BYTES >> 4) + (c & 3) * 2, HI, IDESC, c > 0 ? 1u : 0u);
}
// acc[128 x D] (+)= A[128 x 64] B: A in tensor memory, B MN-major
template <typename T, int D> __device__ __forceinline__ void mma_columns(unsigned leader, unsigned d, unsigned a, unsigned b, bool add) {
    constexpr unsigned IDESC = IDESC_M128<T> | (1u << 16) | idesc_n(D);
#pragma unroll
    for (int c = 0; c < N / 16; ++c) tc_mma_ta<false>(leader, d, a + c * 8, b + c * (2048 >> 4), HI, IDESC, add || c > 0 ? 1u : 0u);
}
template <typename T> __device__ __forceinline__ void store_packed(unsigned taddr, const float *v) {
#pragma unroll
    for (int c = 0; c < N; c += 32) {
        unsigned w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pack_pair(T(), v[c + 2 * e], v[c + 2 * e + 1]);
        tc_st16(taddr + c / 2, w);
    }
}
// a row of a tile of 64
template <typename T, int D> __device__ __forceinline__ bool clean_box(unsigned tile, int row) {
    bool any = false;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) any = clean_line<T>(tile + b * BOX_BYTES + row * 128, row) || any;
    return any;
}

}  // namespace umg

template <typename T, int D, bool KEYS>
__global__ void __launch_bounds__(um::NT, 1) sapa_attention_umma_grad_kernel(const __grid_constant__ CUtensorMap own0, const __grid_constant__ CUtensorMap own1,
                                                                             const __grid_constant__ CUtensorMap over0, const __grid_constant__ CUtensorMap over1,
                                                                             const __grid_constant__ Args p, const __grid_constant__ Grads g, const int most_items) {
    using namespace umg;
    using L = umg::Lay<D>;
    using Work = umg::Work;
    constexpr int NST = L::NST;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(16) float row_lse[KEYS ? NST : 1][N], row_delta[KEYS ? NST : 1][N];
    __shared__ __align__(8) unsigned long long bars[2 + 2 * NST + 8 + 4 + 2];
    __shared__ unsigned tmem_slot;
    __shared__ Work queue[2];
    const sapa_attention &a = p.a;
    const unsigned base = ((unsigned)__cvta_generic_to_shared(smem_dyn) + 1023u) & ~1023u;
    const unsigned ownfull = (unsigned)__cvta_generic_to_shared(bars), ownempty = ownfull + 8, full = ownempty + 8, empty = full + 8 * NST, sfull = empty + 8 * NST;
    const unsigned pfull = sfull + 16, dpfull = pfull + 16, dsfull = dpfull + 16, posted = dsfull + 16, taken = posted + 16, done = taken + 16, accfree = done + 8;
    const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
    // KEYS: rows of a tile are `tok` tokens x `at_once` heads of a key head, which take `turns` tiles if they are more than 64; otherwise an item is `tok` tokens
    const int at_once = KEYS ? min(p.share, N) : p.share, tok = (KEYS ? N : ROWS) / at_once, rows = tok * at_once;

    if (warp == MMA_WARP) {
        if (lane == 0) {
            mbar_init(ownfull, 1); mbar_init(ownempty, 1); mbar_init(done, 1); mbar_init(accfree, 256);
            for (int i = 0; i < NST; ++i) { mbar_init(full + 8 * i, KEYS ? 33 : 1); mbar_init(empty + 8 * i, 1); }
            for (int i = 0; i < 2; ++i) {
                mbar_init(sfull + 8 * i, 1); mbar_init(dpfull + 8 * i, 1); mbar_init(pfull + 8 * i, 128); mbar_init(dsfull + 8 * i, 128);
                mbar_init(posted + 8 * i, 1); mbar_init(taken + 8 * i, KEYS ? 11 : 10);
            }
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
        tc_alloc((unsigned)__cvta_generic_to_shared(&tmem_slot), L::TMEM_COLS);
        tc_relinquish();
    }
    if (KEYS)                                                         // rows that no copy fills: they are behind P and dS, which are 0 there
        for (int i = tid; i < (N - rows) * 8 * (D / 64) * 2 * NST; i += NT) {
            const int tile = i / ((N - rows) * 8), e = i % ((N - rows) * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(base + L::ST0 + tile * BOX_BYTES + (rows + e / 8) * 128 + (e % 8) * 16), "r"(0u) : "memory");
        }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    begin_after_previous();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = warp_uniform(*reinterpret_cast<volatile unsigned *>(&tmem_slot));
    bool ok = true;
    int turn = 0;
    auto next_work = [&]() {                                          // nullptr behind the last one, or where a wait gave up
        ok = ok && mbar_wait_warp(posted + 8 * (turn & 1), (turn >> 1) & 1);
        return ok && queue[turn & 1].there ? &queue[turn & 1] : nullptr;
    };
    auto work_done = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(taken + 8 * (turn & 1));
        ++turn;
    };

    if (warp == PLAN_WARP) {
        typename std::conditional<KEYS, InOrder<false, KeyBlocks>, InOrder<true, QueryBlocks>>::type order(a, {a.causal != 0, tok, KT}, lane);
        for (int round = 0;; ++round) {
            const int index = round * (int)gridDim.x + (round & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
            Work w{};
            if (index < most_items) {
                const Item it = order.at(index / a.groups);
                w.there = it.there;
                if (w.there) {
                    w.b = it.b; w.group = index % a.groups;
                    w.s = sequence_at(a, it.b);
                    if (KEYS) {
                        w.first = it.block * KT;
                        w.from = a.causal ? (int)max(0ll, (long long)w.first - w.s.nk + w.s.nq) : 0;
                        w.turns = tiles_of(p.share, at_once);
                        w.n = w.from < w.s.nq ? tiles_of(w.s.nq - w.from, tok) * w.turns : 0;
                    } else {
                        w.first = it.block * tok;
                        w.n = tiles_of(sees(w.s, min(w.first + tok, w.s.nq) - 1, a.causal), N);
                    }
                }
            }
            w.odd_first = 0x7fffffff; w.odd_last = -1;
            ok = mbar_wait_warp(taken + 8 * (round & 1), ((round >> 1) & 1) ^ 1);
            if (!ok) break;
            if (lane == 0) { queue[round & 1] = w; mbar_arrive(posted + 8 * (round & 1)); }
            __syncwarp();
            if (!w.there) break;
        }
    } else if (warp == LOAD_WARP) {
        int st = 0, ph = 0, own_ph = 0;
        while (Work *w = next_work()) {
            const int n = w->n, first = w->first, group = w->group;
            const Sequence s = w->s;
            if (lane == 0 && n > 0) {
                ok = mbar_wait_bounded(ownempty, own_ph ^ 1);
                if (ok) {
                    mbar_expect_tx(ownfull, 2 * (D / 64) * 128 * (KEYS ? KT : rows));
                    for (int c = 0; c < D / 64; ++c) {
                        const int head = KEYS ? group : group * p.share, token = (KEYS ? s.k0 : s.q0) + first;
                        tma_load_3d(base + L::OWN0 + c * BLOCK_BYTES, &own0, ownfull, 64 * c, head, token);
                        tma_load_3d(base + L::OWN0 + L::OWN + c * BLOCK_BYTES, &own1, ownfull, 64 * c, head, token);
                    }
                    own_ph ^= 1;
                }
                int token = KEYS ? s.q0 + w->from : s.k0, head = KEYS ? group * p.share : group, part = 0;
                for (int i = 0; i < n && ok; ++i) {
                    ok = mbar_wait_bounded(empty + 8 * st, ph ^ 1);
                    if (!ok) break;
                    mbar_expect_tx(full + 8 * st, 2 * (D / 64) * 128 * (KEYS ? rows : N));
                    for (int c = 0; c < D / 64; ++c) {
                        const unsigned dst = base + L::ST0 + st * L::STAGE + c * BOX_BYTES;
                        tma_load_3d(dst, &over0, full + 8 * st, 64 * c, head + part * at_once, token);
                        tma_load_3d(dst + L::HALF, &over1, full + 8 * st, 64 * c, head + part * at_once, token);
                    }
                    if (!KEYS) token += N;
                    else if (++part == w->turns) { part = 0; token += tok; }
                    if (++st == NST) { st = 0; ph ^= 1; }
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
            if (!ok) break;
            work_done();
        }
        if (!ok && lane == 0) {                                       // none of its loads may land after it has left
            (void)drain_loads<NST>(full, st, ph);
            (void)mbar_wait_bounded(ownfull, own_ph ^ 1);
        }
    } else if (warp == ROW_WARP) {
        if (KEYS) {                                                   // lse and delta of a tile's rows, two a lane, read a tile ahead
            int st = 0, ph = 0;
            while (Work *w = next_work()) {
                const int n = w->n;
                const long long at0 = ((long long)w->group * a.tokens + w->s.q0 + w->from) * p.share, end = (long long)a.tokens * a.heads;
                float e[2], d[2];
                int part = 0;
                long long token = 0;
                auto fetch = [&]() {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int row = lane + 32 * r;
                        const long long at = at0 + (token + row / at_once) * p.share + part * at_once + row % at_once;
                        e[r] = row < rows && at < end ? g.nlse[at] : -INFINITY;      // P = 0 where no row is
                        d[r] = row < rows && at < end ? g.delta[at] : 0.f;
                    }
                    if (++part == w->turns) { part = 0; token += tok; }
                };
                if (n > 0) fetch();
                for (int i = 0; i < n; ++i) {
                    ok = mbar_wait_warp(empty + 8 * st, ph ^ 1);
                    if (!ok) break;
#pragma unroll
                    for (int r = 0; r < 2; ++r) { row_lse[st][lane + 32 * r] = e[r]; row_delta[st][lane + 32 * r] = d[r]; }
                    mbar_arrive(full + 8 * st);
                    if (i + 1 < n) fetch();
                    if (++st == NST) { st = 0; ph ^= 1; }
                }
                if (!ok) break;
                work_done();
            }
        }
    } else if (warp == MMA_WARP) {
        const unsigned leader = elect_leader();
        const unsigned a0 = warp_uniform(desc_lo(base + L::OWN0, 16)), a1 = warp_uniform(desc_lo(base + L::OWN0 + L::OWN, 16));
        const unsigned b_rows = warp_uniform(desc_lo(base + L::ST0, 16)), b_cols = warp_uniform(desc_lo(base + L::ST0, BOX_BYTES));
        constexpr unsigned STEP = L::STAGE >> 4, SECOND = L::HALF >> 4;
        int st = 0, ph = 0, own_ph = 0, free_ph = 1, tph[2] = {0, 0}, now = 0;      // next stage to wait for; stage of the tile in turn
        auto scores = [&](int t, bool wait) {
            if (wait) ok = ok && mbar_wait_warp(full + 8 * st, ph);
            if (!ok) return;
            mma_rows<T, D>(leader, tmem + L::S_COL + t * N, a0, b_rows + st * STEP);
            tc_commit_by(leader, sfull + 8 * t);
        };
        auto products = [&](int t) {                                  // dP, of the stage that scores() has waited for
            mma_rows<T, D>(leader, tmem + L::P_COL + t * N, a1, b_rows + st * STEP + SECOND);
            tc_commit_by(leader, dpfull + 8 * t);
            if (++st == NST) { st = 0; ph ^= 1; }
        };
        while (Work *w = next_work()) {
            const int n = (int)warp_uniform(w->n);
            if (n > 0) {
                ok = mbar_wait_warp(ownfull, own_ph);
                own_ph ^= 1;
                tc_fence_after();
            }
            for (int t = 0; t < 2 && t < n && ok; ++t) {
                scores(t, true);
                if (ok) products(t);
                if (t + 1 == n && ok) tc_commit_by(leader, ownempty);
            }
            ok = ok && mbar_wait_warp(accfree, free_ph);              // the item before has been stored
            free_ph ^= 1;
            for (int i = 0; i < n && ok; ++i) {
                const int t = i & 1;
                ok = mbar_wait_warp(pfull + 8 * t, t == 0 ? tph[0] : tph[1]);
                if (!ok) break;
                tc_fence_after();
                if (KEYS) mma_columns<T, D>(leader, tmem + L::ACC_COL, tmem + L::S_COL + t * N, b_cols + now * STEP + SECOND, i > 0);
                if (i + 2 < n) scores(t, true);
                ok = ok && mbar_wait_warp(dsfull + 8 * t, t == 0 ? tph[0] : tph[1]);
                if (!ok) break;
                tc_fence_after();
                mma_columns<T, D>(leader, tmem + L::ACC_COL + (KEYS ? D : 0), tmem + L::P_COL + t * N, b_cols + now * STEP, i > 0);
                tc_commit_by(leader, empty + 8 * now);
                if (++now == NST) now = 0;
                if (i + 2 < n) {
                    products(t);
                    if (i + 3 == n) tc_commit_by(leader, ownempty);
                }
                if (t == 0) tph[0] ^= 1; else tph[1] ^= 1;
            }
            if (!ok) break;
            tc_commit_by(leader, done);
            work_done();
        }
    } else {
        const int t = warp >> 2, r = tid & 127;
        const unsigned quarter = (unsigned)((warp & 3) * 32) << 16;
        const unsigned s_at = tmem + quarter + L::S_COL + t * N, d_at = tmem + quarter + L::P_COL + t * N;
        const float2 scale = make_float2(p.scale_log2, p.scale_log2);
        const int row_token = r / p.share;
        int sph = 0;
        unsigned loads = 0;                                           // stages that the items before took
        while (Work *w = next_work()) {
            const Sequence s = w->s;
            const int n = w->n, first = w->first;
            const int key = first + r, token = first + row_token;     // of this thread's lane, KEYS or otherwise
            const bool mine = KEYS ? key < s.nk : r < rows && token < s.nq;
            const int lim = !KEYS && mine ? sees(s, token, a.causal) : 0, least = KEYS ? 0 : sees(s, first, a.causal);
            float nlse = 0.f, delta = 0.f;
            if (!KEYS && mine) {
                const long long row = ((long long)w->group * a.tokens + s.q0 + first) * p.share + r;
                nlse = g.nlse[row]; delta = g.delta[row];
            }
            for (int i = t; i < n; i += 2) {
                const unsigned load = loads + i, st = load % NST, stage = base + L::ST0 + st * L::STAGE;
                // columns [lo, hi) are what the lane sees, or is seen by; part: not all 64 for every lane
                int lo = 0, hi;
                bool part;
                if (KEYS) {
                    const int tile = i / w->turns, heads = min(p.share - (i - tile * w->turns) * at_once, at_once), first_token = w->from + tile * tok;
                    const long long ahead = (long long)key - s.nk + s.nq - first_token, farthest = (long long)first + KT - 1 - s.nk + s.nq - first_token;
                    if (a.causal && ahead > 0) lo = (int)min(ahead * at_once, (long long)N);
                    hi = min(tok, s.nq - first_token) * at_once;
                    if (heads < at_once) hi = heads;                  // one token, the last of its heads
                    part = hi < rows || (a.causal && farthest > 0);
                } else {
                    hi = lim - i * N;
                    part = (i + 1) * N > least;
                }
                if (!mbar_wait_warp(sfull + 8 * t, sph)) { ok = false; break; }
                if (KEYS && !mbar_wait_warp(full + 8 * st, (load / NST) & 1)) { ok = false; break; }      // has come: makes lse and delta visible
                tc_fence_after();
                float x[N], y[N];
                tc_ld32(s_at, x);
                tc_ld32(s_at + 32, x + 32);
                tc_wait_ld();
                if (!KEYS) {                                          // the next scores may come
                    tc_fence_before();
                    mbar_arrive(pfull + 8 * t);
                }
                const float4 *lses = reinterpret_cast<const float4 *>(row_lse[KEYS ? st : 0]), *deltas = reinterpret_cast<const float4 *>(row_delta[KEYS ? st : 0]);
#pragma unroll
                for (int c = 0; c < N; c += 4) {
                    const float4 e = KEYS ? lses[c >> 2] : make_float4(nlse, nlse, nlse, nlse);
                    float2 u = fma2(make_float2(x[c], x[c + 1]), scale, make_float2(e.x, e.y)), v = fma2(make_float2(x[c + 2], x[c + 3]), scale, make_float2(e.z, e.w));
                    x[c] = ex2_ftz(u.x); x[c + 1] = ex2_ftz(u.y); x[c + 2] = ex2_ftz(v.x); x[c + 3] = ex2_ftz(v.y);
                }
                if (KEYS) {
                    if (part) {
#pragma unroll
                        for (int c = 0; c < N; ++c) x[c] = c >= lo && c < hi ? x[c] : 0.f;
                    }
                    store_packed<T>(s_at, x);
                }
                if (part) {                                           // behind the products that take the tiles as they are
                    if (!mbar_wait_warp(dpfull + 8 * t, sph)) { ok = false; break; }
                    if (KEYS) {
                        const bool odd = clean_box<T, D>(stage + (r >> 6) * L::HALF, r & 63);
                        if (odd && r >= 64 && (r & 63) < hi) { atomicMin(&w->odd_first, i); atomicMax(&w->odd_last, i); }
                    } else if (r < N) {
                        if (clean_box<T, D>(stage, r) && i * N + r < s.nk) { atomicMin(&w->odd_first, i * N + r); atomicMax(&w->odd_last, i * N + r); }
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                if (KEYS) {
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive(pfull + 8 * t);
                }
                if (!mbar_wait_warp(dpfull + 8 * t, sph)) { ok = false; break; }
                sph ^= 1;
                tc_fence_after();
                tc_ld32(d_at, y);
                tc_ld32(d_at + 32, y + 32);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < N; c += 4) {
                    const float4 e = KEYS ? deltas[c >> 2] : make_float4(delta, delta, delta, delta);
                    const float2 u = mul2(make_float2(x[c], x[c + 1]), add2(make_float2(y[c], y[c + 1]), make_float2(-e.x, -e.y)));
                    const float2 v = mul2(make_float2(x[c + 2], x[c + 3]), add2(make_float2(y[c + 2], y[c + 3]), make_float2(-e.z, -e.w)));
                    y[c] = u.x; y[c + 1] = u.y; y[c + 2] = v.x; y[c + 3] = v.y;
                }
                if (part) {
#pragma unroll
                    for (int c = 0; c < N; ++c) y[c] = c >= lo && c < hi ? y[c] : 0.f;
                }
                store_packed<T>(d_at, y);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(dsfull + 8 * t);
            }
            loads += n;
            ok = ok && mbar_wait_warp(done, turn & 1);
            tc_fence_after();
            // KEYS: the first warpgroup stores the gradients of the values, the second those of the keys; otherwise each half of the channels
            const bool values = KEYS && t == 0;
            const unsigned at = tmem + quarter + L::ACC_COL + (KEYS ? t * D : 0);
            const float factor = values ? 1.f : a.scale;
            T *const to = KEYS ? static_cast<T *>(values ? g.gv : g.gk) + ((long long)(s.k0 + key) * a.groups + w->group) * a.dim
                               : static_cast<T *>(g.gq) + ((long long)(s.q0 + token) * a.heads + w->group * p.share + r % p.share) * a.dim;
            const int odd0 = w->odd_first, odd1 = w->odd_last;
#pragma unroll 1
            for (int c = KEYS ? 0 : t * (D / 2); c < (KEYS ? D : (t + 1) * (D / 2)) && c < a.dim && ok; c += 32) {
                float o[32];
                if (n > 0) {
                    tc_ld32(at + c, o);
                    tc_wait_ld();
                }
                if (!mine) continue;
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = n > 0 && (KEYS || lim > 0) ? o[e] * factor : 0.f;
                if (odd1 >= 0 && (values || !KEYS)) {                 // rare: what is not finite and was taken out of the products
                    for (int i = odd0; i <= odd1; ++i)
                        for (int k = 0; k < (KEYS ? rows : 1); ++k) {
                            const T *v;
                            if (KEYS) {                               // row k of tile i
                                const int tile = i / w->turns, row = w->from + tile * tok + k / at_once, head = (i - tile * w->turns) * at_once + k % at_once;
                                if (row >= s.nq || head >= p.share || key >= sees(s, row, a.causal)) continue;
                                v = static_cast<const T *>(g.go) + (long long)(s.q0 + row) * g.go_strides[0] + (long long)(w->group * p.share + head) * g.go_strides[1] + c;
                            } else {
                                if (i >= lim) continue;
                                v = static_cast<const T *>(a.key) + (long long)(s.k0 + i) * a.key_strides[0] + w->group * a.key_strides[1] + c;
                            }
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float f = c + e < a.dim ? to_acc(v[e]) : 0.f;
                                if (!isfinite(f)) o[e] = KEYS ? o[e] + f : __int_as_float(0x7fffffff);
                            }
                        }
                }
                store_row(to + c, o, a.dim - c);
            }
            tc_fence_before();
            mbar_arrive(accfree);
            if (!ok) break;
            work_done();
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
