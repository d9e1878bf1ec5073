// attention_umma_grad.cuh — the gradients of attention over sequences in 16 bits on the 5th-generation tensor cores.  Included by
// attention_umma.cu behind attention_umma.cuh.
//
// P and dS of a tile are formed again: P = 2^(scale s - lse), dS = P (dP - delta), rounded to the inputs' type for the products that take them from
// tensor memory (dS in float16 by a power of two, see sapa_attention_factor_kernel); the sums are float32.  Two launches of one kernel, without atomics, so that results do not depend on the order of anything:
//   * KEYS: an item holds 128 keys and values and goes over the rows (token x query head) that see them.  S^T = K Q^T and dP^T = V dO^T have the keys in
//     the lanes of tensor memory, so that P^T and dS^T are first operands of dV += P^T dO and dK += dS^T Q as they are;
//   * otherwise an item holds 128 rows and goes over the keys that they see: S = Q K^T, dP = dO V^T, dQ += dS K.
// Seven products where five would do with dQ summed by atomics; each operand is in shared memory once, K-major for one product and MN-major for another.
// What is gone over comes in tiles of 64, so that tensor memory holds S and dP of two: two warpgroups take every other tile (a thread a lane, 32 columns) while
// the products of the other one run, and the item's own operands are in tensor memory.  Those of keys in 128 channels find no room there, and products of
// 128 x 64 that read both operands from shared memory take 6 KB of it every 32 clocks, more than it gives (128 bytes a clock): there the tiles are of 128, and
// the four warpgroups take a quarter of the columns each (BOTH).  A block an SM goes through its items, as the forward does.
// What a row does not see: P and dS are 0 there, and 0 * infinity must not reach a gradient.  In tiles that are not seen whole, what is not finite in the
// operand behind P or dS is replaced with 0 once the products that need it as it is have read it.  Values that are not finite in a row of dO are
// added to the gradients of the values that it sees; those of keys that a row sees make its gradient NaN; a row of Q makes its P NaN by itself.
#pragma once

#include "attention_umma.cuh"

namespace sapa {
namespace attn {
namespace umg {

using namespace um;

// Of sequences up to so long dS goes into its product with what its rounding to the inputs' type leaves out: between few tokens its errors do not average out, and
// made gradients up to 1.65 times as far from the exact ones as their own rounding does (1.5 from some 40 tokens on, 1.4 over long sequences).
constexpr int FINE = 64;
constexpr int N = 32, GROUPS = 4;                                     // columns of a thread; warpgroups that form P and dS
constexpr int MMA = 4 * GROUPS, LOAD = MMA + 1, PLANS = MMA + 2, ROW = MMA + 3, THREADS = (4 * GROUPS + 4) * 32;      // warps; ROW loads lse and delta
// registers a thread: 96 at launch
constexpr int GRAD_REGS = 96, FORM_REGS = 104, REST_REGS = 64;
static_assert(GROUPS * 128 * FORM_REGS + 128 * REST_REGS <= THREADS * GRAD_REGS, "a block draws on what it was launched with");

template <int D, bool KEYS> struct Lay {
    static constexpr bool BOTH = KEYS && D == 128;
    static constexpr int TN = BOTH ? 128 : 64, SLOTS = BOTH ? 1 : 2, FORM = GROUPS * 128 / SLOTS;      // rows of a tile that is gone over, tiles at once, threads that take one
    static constexpr int OWN = D / 64 * BLOCK_BYTES, BOX = TN * 128, HALF = D / 64 * BOX, NST = BOTH ? 2 : D == 64 ? 8 : 4;      // stages of each operand
    static constexpr int OWN0 = 0, ST0 = 2 * OWN, NEED = ST0 + 2 * NST * HALF + 1024, SMEM = NEED < 120 * 1024 ? 120 * 1024 : NEED;
    // S and dP of what is at work, dV and dK or dQ, and where there is room the item's own two operands
    static constexpr int S_COL = 0, P_COL = 128, ACC_COL = 256, OWN_COL = ACC_COL + (KEYS ? 2 : 1) * D, TMEM_COLS = 512;
    static constexpr bool IN_TMEM = OWN_COL + D <= TMEM_COLS;
    static_assert(SMEM <= 222 * 1024 && OWN_COL <= TMEM_COLS, "shared memory, with lse and delta; tensor memory");
};
// An item of a block
struct Work {
    bool there, fine;              // fine: dS with what its rounding leaves out
    int b, group, n;               // tiles to go over
    int first;                     // KEYS: first key; otherwise first token
    int from, turns;               // KEYS: the first token that sees a key; tiles that the heads of a token take
    Sequence s;
    int odd_first, odd_last;       // rows or keys with something not finite, of tiles that are not seen whole
    float factor, rescale;         // of dS; of the gradients of queries and keys
};

// S[128 x TN] = A B^T, both K-major in shared memory, or A in tensor memory
template <typename T, int D, int TN, bool IN_TMEM> __device__ __forceinline__ void mma_rows(unsigned leader, unsigned d, unsigned a, unsigned b) {
    constexpr unsigned IDESC = IDESC_M128<T> | idesc_n(TN);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        const unsigned at = b + (c >> 2) * (TN * 128 >> 4) + (c & 3) * 2;
        if (IN_TMEM) tc_mma_ta<false>(leader, d, a + c * 8, at, HI, IDESC, c > 0 ? 1u : 0u);
        else tc_mma<false>(leader, d, a + (c >> 2) * (BLOCK_BYTES >> 4) + (c & 3) * 2, at, HI, IDESC, c > 0 ? 1u : 0u);
    }
}
// acc[128 x D] (+)= A[128 x TN] B: A in tensor memory, the 16 words of a thread's 32 columns in 32, B MN-major
template <typename T, int D, int TN> __device__ __forceinline__ void mma_columns(unsigned leader, unsigned d, unsigned a, unsigned b, bool add) {
    constexpr unsigned IDESC = IDESC_M128<T> | (1u << 16) | idesc_n(D);
#pragma unroll
    for (int c = 0; c < TN / 16; ++c) tc_mma_ta<false>(leader, d, a + (c >> 1) * N + (c & 1) * 8, b + c * (2048 >> 4), HI, IDESC, add || c > 0 ? 1u : 0u);
}
template <typename T> __device__ __forceinline__ void store_packed(unsigned taddr, const float *v) {
    unsigned w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = pack_pair(T(), v[2 * e], v[2 * e + 1]);
    tc_st16(taddr, w);
}
// Replaces what is not finite in a row of a tile of TN rows; whether there was any.
template <typename T, int D, int TN> __device__ __forceinline__ bool clean_box(unsigned tile, int row) {
    bool any = false;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) any = clean_line<T>(tile + b * TN * 128 + row * 128, row) || any;
    return any;
}

}  // namespace umg

template <typename T, int D, bool KEYS>
__global__ void __launch_bounds__(umg::THREADS, 1) sapa_attention_umma_grad_kernel(const __grid_constant__ CUtensorMap own0, const __grid_constant__ CUtensorMap own1,
                                                                             const __grid_constant__ CUtensorMap over0, const __grid_constant__ CUtensorMap over1,
                                                                             const __grid_constant__ Args p, const __grid_constant__ Grads g, const int most_items) {
    using namespace umg;
    using L = umg::Lay<D, KEYS>;
    using Work = umg::Work;
    constexpr int NST = L::NST, TN = L::TN, SLOTS = L::SLOTS;
    constexpr bool SCALED = std::is_same<T, __half>::value;           // dS by a power of two: float16 holds neither the small nor the large ones
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(16) float row_lse[KEYS ? NST : 1][TN], row_delta[KEYS ? NST : 1][TN];      // as nlse, -delta
    __shared__ __align__(8) unsigned long long bars[2 + 4 * NST + 8 + 4 + 3];
    __shared__ unsigned tmem_slot;
    __shared__ bool row_odd[NST];                                     // KEYS: whether a row of the stage may hold something not finite
    __shared__ Work queue[2];
    const sapa_attention &a = p.a;
    const unsigned base = ((unsigned)__cvta_generic_to_shared(smem_dyn) + 1023u) & ~1023u;
    const unsigned ownfull = (unsigned)__cvta_generic_to_shared(bars), ownempty = ownfull + 8, full = ownempty + 8, empty = full + 8 * NST, full1 = empty + 8 * NST, empty1 = full1 + 8 * NST, sfull = empty1 + 8 * NST;
    const unsigned pfull = sfull + 16, dpfull = pfull + 16, dsfull = dpfull + 16, posted = dsfull + 16, taken = posted + 16, done = taken + 16, accfree = done + 8, ownready = accfree + 8;
    const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
    // KEYS: rows of a tile are `tok` tokens x `at_once` heads of a key head, which take `turns` tiles if they are more; otherwise an item is `tok` tokens
    const int at_once = KEYS ? min(p.share, TN) : p.share, tok = (KEYS ? TN : ROWS) / at_once, rows = tok * at_once;

    if (warp == MMA) {
        if (lane == 0) {
            mbar_init(ownfull, 1); mbar_init(ownempty, L::IN_TMEM ? GROUPS * 128 : 1); mbar_init(done, 1); mbar_init(accfree, GROUPS * 128); mbar_init(ownready, GROUPS * 128);
            for (int i = 0; i < NST; ++i) { mbar_init(full + 8 * i, KEYS ? 33 : 1); mbar_init(empty + 8 * i, 1); mbar_init(full1 + 8 * i, 1); mbar_init(empty1 + 8 * i, 1); }
            for (int i = 0; i < 2; ++i) {
                mbar_init(sfull + 8 * i, 1); mbar_init(dpfull + 8 * i, 1); mbar_init(pfull + 8 * i, L::FORM); mbar_init(dsfull + 8 * i, L::FORM);
                mbar_init(posted + 8 * i, 1); mbar_init(taken + 8 * i, 4 * GROUPS + (KEYS ? 3 : 2));
            }
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
        tc_alloc((unsigned)__cvta_generic_to_shared(&tmem_slot), L::TMEM_COLS);
        tc_relinquish();
    }
    if (KEYS)                                                         // rows that no copy fills: they are behind P and dS, which are 0 there
        for (int i = tid; i < (TN - rows) * 8 * (D / 64) * 2 * NST; i += umg::THREADS) {
            const int tile = i / ((TN - rows) * 8), e = i % ((TN - rows) * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(base + L::ST0 + tile * L::BOX + (rows + e / 8) * 128 + (e % 8) * 16), "r"(0u) : "memory");
        }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    begin_after_previous();
    auto meet = [&]() {
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    };
    if (warp != PLANS) meet();                                    // that one looks for the first item meanwhile
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

    if (warp >= MMA) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(REST_REGS));
        if (warp == PLANS) {
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
                        w.fine = max(w.s.nq, w.s.nk) <= FINE;
                        w.factor = SCALED ? g.factor[(long long)w.b * a.groups + w.group] : 1.f;
                        w.rescale = a.scale / w.factor;               // exact: by a power of two
                        if (KEYS) {
                            w.first = it.block * KT;
                            w.from = a.causal ? (int)max(0ll, (long long)w.first - w.s.nk + w.s.nq) : 0;
                            w.turns = tiles_of(p.share, at_once);
                            w.n = w.from < w.s.nq ? tiles_of(w.s.nq - w.from, tok) * w.turns : 0;
                        } else {
                            w.first = it.block * tok;
                            w.n = tiles_of(sees(w.s, min(w.first + tok, w.s.nq) - 1, a.causal), TN);
                        }
                    }
                }
                w.odd_first = 0x7fffffff; w.odd_last = -1;
                if (round == 0) meet();
                ok = mbar_wait_warp(taken + 8 * (round & 1), ((round >> 1) & 1) ^ 1);
                if (!ok) break;
                if (lane == 0) { queue[round & 1] = w; mbar_arrive(posted + 8 * (round & 1)); }
                __syncwarp();
                if (!w.there) break;
            }
        } else if (warp == LOAD) {
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
                    // keys' items from the last token down: those of a sequence begin at the same place and find there what another has just read
                    const int tiles = KEYS ? n / w->turns : n;
                    int token = KEYS ? s.q0 + w->from + (tiles - 1) * tok : s.k0, head = KEYS ? group * p.share : group, part = 0;
                    for (int i = 0; i < n && ok; ++i) {
                        for (int o = 0; o < 2; ++o) {                 // the two operands: the second is done with sooner
                            const unsigned here = (o == 0 ? full : full1) + 8 * st;
                            ok = mbar_wait_bounded((o == 0 ? empty : empty1) + 8 * st, ph ^ 1);
                            if (!ok) {
                                if (o == 1) (void)mbar_wait_bounded(full + 8 * st, ph);
                                break;
                            }
                            mbar_expect_tx(here, (D / 64) * 128 * (KEYS ? rows : TN));
                            for (int c = 0; c < D / 64; ++c)
                                tma_load_3d(base + L::ST0 + (o * NST + st) * L::HALF + c * L::BOX, o == 0 ? &over0 : &over1, here, 64 * c, head + part * at_once, token);
                        }
                        if (!ok) break;
                        if (!KEYS) token += TN;
                        else if (++part == w->turns) { part = 0; token -= tok; }
                        if (++st == NST) { st = 0; ph ^= 1; }
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
                if (!ok) break;
                work_done();
            }
            if (!ok && lane == 0) {                                       // none of its loads may land after it has left
                (void)drain_loads<NST>(full, st, ph);
                (void)drain_loads<NST>(full1, st, ph);
                (void)mbar_wait_bounded(ownfull, own_ph ^ 1);
            }
        } else if (warp == ROW) {
            if (KEYS) {                                                   // lse and delta of a tile's rows, read a tile ahead
                int st = 0, ph = 0;
                while (Work *w = next_work()) {
                    const int n = w->n;
                    const long long at0 = ((long long)w->group * a.tokens + w->s.q0 + w->from) * p.share, end = (long long)a.tokens * a.heads;
                    const float factor = SCALED ? w->factor : 1.f;
                    float e[TN / 32], d[TN / 32];
                    int part = 0;
                    long long token = (long long)(n / max(w->turns, 1) - 1) * tok;
                    auto fetch = [&]() {
#pragma unroll
                        for (int r = 0; r < TN / 32; ++r) {
                            const int row = lane + 32 * r, head = part * at_once + row % at_once;
                            const long long at = at0 + (token + row / at_once) * p.share + head;
                            const bool mine = row < rows && at < end && head < p.share;
                            e[r] = mine ? g.nlse[at] : -INFINITY;                       // P = 0 where no row is
                            d[r] = mine ? g.delta[at] : 0.f;
                            if (row < rows && head >= p.share) e[r] = INFINITY;         // heads of the next key head, whatever they hold
                        }
                        if (++part == w->turns) { part = 0; token -= tok; }
                    };
                    if (n > 0) fetch();
                    for (int i = 0; i < n; ++i) {
                        ok = mbar_wait_warp(empty + 8 * st, ph ^ 1);
                        if (!ok) break;
#pragma unroll
                        for (int r = 0; r < TN / 32; ++r) { row_lse[st][lane + 32 * r] = e[r]; row_delta[st][lane + 32 * r] = SCALED ? -d[r] * factor : -d[r]; }
                        // what is not finite in a row of dO is in its delta, and in a row of Q in its lse, if it sees a key; nlse of the others is +infinity
                        bool odd = false;
#pragma unroll
                        for (int r = 0; r < TN / 32; ++r) odd = odd || !isfinite(d[r]) || !(e[r] < INFINITY);
                        odd = __any_sync(0xffffffffu, odd);
                        if (lane == 0) row_odd[st] = odd;
                        mbar_arrive(full + 8 * st);
                        if (i + 1 < n) fetch();
                        if (++st == NST) { st = 0; ph ^= 1; }
                    }
                    if (!ok) break;
                    work_done();
                }
            }
        } else if (warp == MMA) {
            const unsigned leader = elect_leader();
            const unsigned a0 = L::IN_TMEM ? tmem + L::OWN_COL : warp_uniform(desc_lo(base + L::OWN0, 16));
            const unsigned a1 = L::IN_TMEM ? tmem + L::OWN_COL + D / 2 : warp_uniform(desc_lo(base + L::OWN0 + L::OWN, 16));
            const unsigned b_rows = warp_uniform(desc_lo(base + L::ST0, 16)), b_cols = warp_uniform(desc_lo(base + L::ST0, L::BOX));
            constexpr unsigned STEP = L::HALF >> 4, SECOND = NST * STEP;
            int st = 0, ph = 0, own_ph = 0, free_ph = 1, tph0 = 0, tph1 = 0, now = 0;      // next stage to wait for; stage of the tile in turn
            auto scores = [&](int t) {
                ok = ok && mbar_wait_warp(full + 8 * st, ph);
                if (!ok) return;
                mma_rows<T, D, TN, L::IN_TMEM>(leader, tmem + L::S_COL + t * 64, a0, b_rows + st * STEP);
                tc_commit_by(leader, sfull + 8 * t);
            };
            auto products = [&](int t) {                              // dP, of the stage that scores() has waited for
                ok = ok && mbar_wait_warp(full1 + 8 * st, ph);
                if (!ok) return;
                mma_rows<T, D, TN, L::IN_TMEM>(leader, tmem + L::P_COL + t * 64, a1, b_rows + st * STEP + SECOND);
                tc_commit_by(leader, dpfull + 8 * t);
                if (!KEYS) tc_commit_by(leader, empty1 + 8 * st);
                if (++st == NST) { st = 0; ph ^= 1; }
            };
            while (Work *w = next_work()) {
                const int n = (int)warp_uniform(w->n), fine = (int)warp_uniform(w->fine);
                if (n > 0) {
                    ok = mbar_wait_warp(L::IN_TMEM ? ownready : ownfull, own_ph);
                    own_ph ^= 1;
                    tc_fence_after();
                }
                for (int t = 0; t < SLOTS && t < n && ok; ++t) {
                    scores(t);
                    products(t);
                    if (t + 1 == n && ok && !L::IN_TMEM) tc_commit_by(leader, ownempty);
                }
                ok = ok && mbar_wait_warp(accfree, free_ph);          // the item before has been stored
                free_ph ^= 1;
                for (int i = 0; i < n && ok; ++i) {
                    const int t = SLOTS == 1 ? 0 : i & 1;
                    ok = mbar_wait_warp(pfull + 8 * t, t == 0 ? tph0 : tph1);
                    if (!ok) break;
                    tc_fence_after();
                    if (KEYS) {
                        mma_columns<T, D, TN>(leader, tmem + L::ACC_COL, tmem + L::S_COL + t * 64, b_cols + now * STEP + SECOND, i > 0);
                        tc_commit_by(leader, empty1 + 8 * now);
                    }
                    if (i + SLOTS < n) scores(t);
                    ok = ok && mbar_wait_warp(dsfull + 8 * t, t == 0 ? tph0 : tph1);
                    if (!ok) break;
                    tc_fence_after();
                    mma_columns<T, D, TN>(leader, tmem + L::ACC_COL + (KEYS ? D : 0), tmem + L::P_COL + t * 64, b_cols + now * STEP, i > 0);
                    if (fine) mma_columns<T, D, TN>(leader, tmem + L::ACC_COL + (KEYS ? D : 0), tmem + L::P_COL + t * 64 + N / 2, b_cols + now * STEP, true);
                    tc_commit_by(leader, empty + 8 * now);
                    if (++now == NST) now = 0;
                    if (i + SLOTS < n) {
                        products(t);
                        if (i + SLOTS + 1 == n && ok && !L::IN_TMEM) tc_commit_by(leader, ownempty);
                    }
                    if (t == 0) tph0 ^= 1; else tph1 ^= 1;
                }
                if (!ok) break;
                tc_commit_by(leader, done);
                work_done();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(FORM_REGS));
        // warpgroup, the tile that it takes (BOTH: all take every tile, otherwise two each every other one), its part of the columns
        const int wg = warp >> 2, t = L::BOTH ? 0 : wg >> 1, part_of = L::BOTH ? wg : wg & 1, r = tid & 127, bar = 8 * t, col0 = N * part_of;
        const unsigned quarter = (unsigned)((warp & 3) * 32) << 16;
        const unsigned s_at = tmem + quarter + L::S_COL + wg * N, d_at = tmem + quarter + L::P_COL + wg * N;
        const float2 scale = make_float2(p.scale_log2, p.scale_log2);
        const int row_token = r / p.share;
        int sph = 0, own_ph = 0;
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
            const float2 factor = SCALED ? make_float2(w->factor, w->factor) : make_float2(1.f, 1.f);
            if (SCALED) delta *= factor.x;
            auto less = [&](float2 dp, float2 minus_delta) { return SCALED ? fma2(dp, factor, minus_delta) : add2(dp, minus_delta); };
            if (L::IN_TMEM && n > 0) {                                // the item's own operands, half of one by each warpgroup; what was there has been used: `done`
                if (!mbar_wait_warp(ownfull, own_ph)) { ok = false; break; }
                own_ph ^= 1;
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < D / 64; ++h) {
                    unsigned v[16];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int chunk = (wg & 1) * (D / 16) + 4 * h + e;
                        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[4 * e]), "=r"(v[4 * e + 1]), "=r"(v[4 * e + 2]), "=r"(v[4 * e + 3])
                                     : "r"(base + L::OWN0 + (wg >> 1) * L::OWN + (chunk >> 3) * BLOCK_BYTES + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) : "memory");
                    }
                    tc_st16(tmem + quarter + L::OWN_COL + (wg >> 1) * (D / 2) + (wg & 1) * (D / 4) + 16 * h, v);
                }
                mbar_arrive(ownempty);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(ownready);
            }
            for (int i = L::BOTH ? 0 : t; i < n; i += SLOTS) {
                const unsigned load = loads + i, st = load % NST, stage = base + L::ST0 + st * L::HALF;
                // columns [lo, hi) of the tile are what the lane sees, or is seen by; part: not all for every lane; masked: of this warpgroup's, or some are of no row
                // (0, but 0 * infinity is not)
                int lo = 0, hi;
                bool part;
                if (KEYS) {
                    const int turns = w->turns, tile = i / turns, heads = min(p.share - (i - tile * turns) * at_once, at_once), first_token = w->from + (n / turns - 1 - tile) * tok;
                    const long long ahead = (long long)key - s.nk + s.nq - first_token, farthest = (long long)first + KT - 1 - s.nk + s.nq - first_token;
                    if (a.causal && ahead > 0) lo = (int)min(ahead * at_once, (long long)TN);
                    hi = min(tok, s.nq - first_token) * at_once;
                    if (heads < at_once) hi = heads;                  // one token, the last of its heads
                    part = hi < rows || (a.causal && farthest > 0);
                } else {
                    hi = lim - i * TN;
                    part = (i + 1) * TN > least;
                }
                const bool masked = part || (KEYS && col0 + N > rows);
                float x[N], y[N];
                if (KEYS) {                                           // lse, ahead of the scores
                    if (!mbar_wait_warp(full + 8 * st, (load / NST) & 1)) { ok = false; break; }
#pragma unroll
                    for (int c = 0; c < N; c += 4) *reinterpret_cast<float4 *>(&y[c]) = *reinterpret_cast<const float4 *>(&row_lse[KEYS ? st : 0][col0 + c]);
                }
                if (!mbar_wait_warp(sfull + bar, sph)) { ok = false; break; }
                tc_fence_after();
                tc_ld32(s_at, x);
                tc_wait_ld();
                if (!KEYS) {                                          // the next scores may come
                    tc_fence_before();
                    mbar_arrive(pfull + bar);
                }
#pragma unroll
                for (int c = 0; c < N; c += 2) {
                    const float2 u = fma2(make_float2(x[c], x[c + 1]), scale, KEYS ? make_float2(y[c], y[c + 1]) : make_float2(nlse, nlse));
                    x[c] = ex2_ftz(u.x); x[c + 1] = ex2_ftz(u.y);
                }
                if (KEYS) {
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < N; ++c) x[c] = col0 + c >= lo && col0 + c < hi ? x[c] : 0.f;
                    }
                    store_packed<T>(s_at, x);
                }
                if (part && (!KEYS || row_odd[st])) {                 // behind the products that take the tiles as they are
                    if (!mbar_wait_warp(dpfull + bar, sph)) { ok = false; break; }
                    if (KEYS) {                                       // rows of dO by the first warpgroup of the tile's, of Q by the second
                        if (part_of < 2 && r < TN) {
                            const bool odd = clean_box<T, D, TN>(stage + (part_of == 0 ? NST * L::HALF : 0), r);
                            if (odd && part_of == 0 && r < hi) { atomicMin(&w->odd_first, i); atomicMax(&w->odd_last, i); }
                        }
                    } else if (part_of == 0 && r < TN) {
                        if (clean_box<T, D, TN>(stage, r) && i * TN + r < s.nk) { atomicMin(&w->odd_first, i * TN + r); atomicMax(&w->odd_last, i * TN + r); }
                    }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();                                     // lanes that found something went another way: tensor memory is used by whole warps
                }
                if (KEYS) {
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive(pfull + bar);
                }
                if (!mbar_wait_warp(dpfull + bar, sph)) { ok = false; break; }
                sph ^= 1;
                tc_fence_after();
                tc_ld32(d_at, y);
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < N; c += 4) {
                    const float4 d = KEYS ? *reinterpret_cast<const float4 *>(&row_delta[KEYS ? st : 0][col0 + c]) : make_float4(-delta, -delta, -delta, -delta);
                    const float2 u = mul2(make_float2(x[c], x[c + 1]), less(make_float2(y[c], y[c + 1]), make_float2(d.x, d.y)));
                    const float2 v = mul2(make_float2(x[c + 2], x[c + 3]), less(make_float2(y[c + 2], y[c + 3]), make_float2(d.z, d.w)));
                    y[c] = u.x; y[c + 1] = u.y; y[c + 2] = v.x; y[c + 3] = v.y;
                }
                if (masked) {
#pragma unroll
                    for (int c = 0; c < N; ++c) y[c] = col0 + c >= lo && col0 + c < hi ? y[c] : 0.f;
                }
                store_packed<T>(d_at, y);
                if (w->fine) {
#pragma unroll
                    for (int c = 0; c < N; ++c) y[c] = left_out<T>(y[c]);
                    store_packed<T>(d_at + N / 2, y);
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(dsfull + bar);
            }
            loads += n;
            ok = ok && mbar_wait_warp(done, turn & 1);
            tc_fence_after();
            // 32 channels a warpgroup at a time: of the gradients of values, of keys; or of queries
            const int odd0 = w->odd_first, odd1 = w->odd_last;
            const bool whole = whole_rows(KEYS ? g.gk : g.gq, a.dim) && (!KEYS || whole_rows(g.gv, a.dim));
#pragma unroll 1
            for (int unit = wg; unit < (KEYS ? 2 : 1) * (D / 32) && ok; unit += GROUPS) {
                const bool values = KEYS && unit < D / 32;
                const int c = unit % (D / 32) * 32;
                if (c >= a.dim) continue;
                const unsigned at = tmem + quarter + L::ACC_COL + unit * 32 - c;
                const float by = values ? 1.f : w->rescale;
                T *const to = KEYS ? static_cast<T *>(values ? g.gv : g.gk) + ((long long)(s.k0 + key) * a.groups + w->group) * a.dim
                                   : static_cast<T *>(g.gq) + ((long long)(s.q0 + token) * a.heads + w->group * p.share + r % p.share) * a.dim;
                float o[32];
                __syncwarp();                                         // behind the stores of the unit before, which not every lane makes
                if (n > 0) {
                    tc_ld32(at + c, o);
                    tc_wait_ld();
                }
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = n > 0 && (KEYS || lim > 0) ? o[e] * by : 0.f;
                if (odd1 >= 0 && mine && (values || !KEYS)) {         // rare: what is not finite and was taken out of the products
                    for (int i = odd0; i <= odd1; ++i)
                        for (int k = 0; k < (KEYS ? rows : 1); ++k) {
                            const T *v;
                            if (KEYS) {                               // row k of tile i
                                const int tile = i / w->turns, row = w->from + (n / w->turns - 1 - tile) * tok + k / at_once, head = (i - tile * w->turns) * at_once + k % at_once;
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
                __syncwarp();
                store_rows(to + c, mine, o, a.dim - c, whole);
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
    if (warp == MMA) tc_dealloc(tmem, L::TMEM_COLS);
}

}  // namespace attn
}  // namespace sapa
