// attention_umma.cuh — attention over sequences in 16 bits on the 5th-generation tensor cores, forward.  Included by attention_umma.cu.
//
// A block takes 128-row tiles (row = token x query head of one key head) against tiles of 128 keys:
//   * a warp loads queries, keys and values with TMA (rows of 64 channels, 128-byte swizzle; of a paged cache a box a page);
//   * a warp issues S = Q K^T (both operands K-major in shared memory) and O += P V (P in tensor memory, V as TMA lands it, MN-major);
//   * a warpgroup for each of two S / O accumulators: a thread holds a row, 128 scores in registers, so maximum and sum need no shuffles; it writes P,
//     rounded to the type of V as the second product takes it, over S.  The sum is of the weights before that rounding.
// The two accumulators are two row tiles over the same keys (WIDE: long prompts; each key tile is used twice), or one row tile over the even and the
// odd key tiles, joined at the end (single tokens and short chunks): while one's softmax runs, the other's products do.
// O is scaled again only when a row's maximum has grown by more than 2^8 since it last was: weights stay below 2^8 and the sums exact enough, and
// the warpgroup that owns S owns O too at that time, for S was computed behind the product that last added to O.
// What a row does not see: its scores are set to -infinity; a value that is not finite would still reach its output as 0 * infinity.  So in tiles that not
// every row sees whole, what is not finite among the values is replaced with 0 in front of the product, and added to the outputs of the rows that see it.
#pragma once

#include "attention.cuh"
#include "finite.cuh"
#include "umma_util.cuh"

namespace sapa {
namespace attn {
namespace um {

using namespace ummau;

constexpr int KT = TILE, ROWS = 128, BLOCK_BYTES = 128 * 128;         // keys of a tile, rows of a tile; 128 rows of 64 channels
constexpr int MMA_WARP = 8, LOAD_WARP = 9, NT = 10 * 32;
constexpr unsigned HI = (1024u >> 4) | (1u << 14) | (2u << 29);       // 8 rows of 128 bytes, descriptor version 1, 128-byte swizzle
constexpr float GROWTH = 8.f;                                         // powers of two

// 2 row tiles: as many stages as fit beside them
template <int D, bool WIDE> struct Lay {
    static constexpr int STAGE = D / 64 * BLOCK_BYTES, Q_BYTES = (WIDE ? 2 : 1) * STAGE, NST = (224 * 1024 - Q_BYTES) / STAGE > 8 ? 8 : (224 * 1024 - Q_BYTES) / STAGE;
    static constexpr int Q0 = 0, KV0 = Q_BYTES;
    static constexpr int NEED = KV0 + NST * STAGE + 1024, SMEM = NEED < 120 * 1024 ? 120 * 1024 : NEED;      // one block an SM: tensor memory
    static constexpr int S_COL = 0, O_COL = 256, TMEM_COLS = 512;
    static_assert(SMEM <= 227 * 1024 && NST * STAGE >= ROWS * D * 4, "shared memory");      // the odd tiles' sums are handed over in it
};

__device__ __forceinline__ void tc_ld32(unsigned taddr, float *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]),
                   "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]),
                   "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st32(unsigned taddr, const float *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};\n"
                 ::"f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]), "f"(r[10]), "f"(r[11]),
                 "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]), "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]),
                 "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]), "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31]), "r"(taddr) : "memory");
}
// two floats at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ void tma_load_3d(unsigned dst, const CUtensorMap *map, unsigned bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// Replaces what is not finite in a row of a landed tile (128 rows of D channels) with 0; whether there was any.
template <typename T, int D> __device__ __forceinline__ bool clean_row(unsigned tile, int row) {
    bool any = false;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
        const unsigned line = tile + b * BLOCK_BYTES + row * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) {                                 // in another order in every row: no two on the same banks
            const unsigned at = line + ((c ^ (row & 7)) << 4);
            unsigned v[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
            if (!finite::all_finite<T, 4>(v)) {
                any = true;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = finite::or_zero<T>(v[e]);
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
            }
        }
    }
    return any;
}
// 32 channels of a row of the output from float32, those below `left`
template <typename T> __device__ __forceinline__ void store_row(T *to, const float *v, int left) {
#pragma unroll
    for (int c = 0; c < 32; c += 8)
        if (c < left)
            *reinterpret_cast<uint4 *>(to + c) = make_uint4(pack_pair(T(), v[c], v[c + 1]), pack_pair(T(), v[c + 2], v[c + 3]), pack_pair(T(), v[c + 4], v[c + 5]),
                                                            pack_pair(T(), v[c + 6], v[c + 7]));
}

}  // namespace um

template <typename T, int D, bool WIDE, bool PAGED>
__global__ void __launch_bounds__(um::NT, 1) sapa_attention_umma_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                                                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args p) {
    using namespace um;
    using L = um::Lay<D, WIDE>;
    constexpr int NST = L::NST;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) unsigned long long bars[1 + 2 * NST + 4];
    __shared__ unsigned tmem_slot;
    __shared__ Plan plan;
    __shared__ int bad_page, odd_first, odd_last;
    __shared__ float2 handed[WIDE ? 1 : ROWS];                        // maximum and sum of the odd tiles
    const sapa_attention &a = p.a;
    const unsigned base = ((unsigned)__cvta_generic_to_shared(smem_dyn) + 1023u) & ~1023u;
    const unsigned qfull = (unsigned)__cvta_generic_to_shared(bars), full = qfull + 8, empty = full + 8 * NST, sfull = empty + 8 * NST, pfull = sfull + 16;
    const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
    const int group = blockIdx.x % a.groups, tile_tok = ROWS / p.share, tok = WIDE ? 2 * tile_tok : tile_tok;

    if (warp == MMA_WARP) {
        if (lane == 0) {
            mbar_init(qfull, 1);
            for (int i = 0; i < NST; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
            for (int i = 0; i < 2; ++i) { mbar_init(sfull + 8 * i, 1); mbar_init(pfull + 8 * i, 128); }
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
            bad_page = 0x7fffffff; odd_first = 0x7fffffff; odd_last = -1;
        }
        __syncwarp();
        tc_alloc((unsigned)__cvta_generic_to_shared(&tmem_slot), L::TMEM_COLS);
        tc_relinquish();
    }
    begin_after_previous();
    if (warp == 0) {
        const Plan r = plan_at(p, blockIdx.x / a.groups, tok, lane);
        if (lane == 0) plan = r;
    }
    clear_outside(static_cast<T *>(a.out), a.offsets, a.B, a.tokens, a.heads * a.dim, blockIdx.x, gridDim.x, tid, NT);
    if (a.lse != nullptr) clear_outside(a.lse, a.offsets, a.B, a.tokens, a.heads, blockIdx.x, gridDim.x, tid, NT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = warp_uniform(*reinterpret_cast<volatile unsigned *>(&tmem_slot));
    const Item it = plan.it;
    bool ok = true;
    if (it.there) {
        const Sequence s = sequence_at(a, it.b);
        const int first = it.block * tok;                             // first token
        // key tiles of the two accumulators: [j0, j0 + n[t]) each (WIDE), or every other one of n
        const int j0 = (int)min((long long)it.part * plan.tiles, 0x7fffffffll / KT);
        int n[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int last = min(first + (WIDE ? (t + 1) * tile_tok : tile_tok), s.nq) - 1;      // its last token
            const bool some = last >= first + (WIDE ? t * tile_tok : 0);
            const int tiles = some ? (min(sees(s, last, a.causal), s.bad) + KT - 1) / KT : 0;
            n[t] = max(0, (int)min((long long)tiles, (long long)j0 + plan.tiles) - j0);
        }
        const int all = (int)warp_uniform(max(n[0], n[1]));           // the block's
        if (!WIDE) { n[0] = (all + 1) / 2; n[1] = all / 2; }
        const int n0 = (int)warp_uniform(n[0]), n1 = (int)warp_uniform(n[1]);

        if (warp == LOAD_WARP) {
            int st = 0, ph = 0;
            const int boxes = PAGED ? max(1, KT / a.page) : 1, box_rows = KT / boxes;
            if (lane == 0) {
                mbar_expect_tx(qfull, (WIDE ? 2 : 1) * (D / 64) * 128 * p.share * tile_tok);
                for (int t = 0; t < (WIDE ? 2 : 1); ++t)
                    for (int b = 0; b < D / 64; ++b)
                        tma_load_3d(base + L::Q0 + t * L::STAGE + b * BLOCK_BYTES, &qmap, qfull, 64 * b, group * p.share, s.q0 + first + t * tile_tok);
            }
            const int used = min(s.bad, s.nk);                        // positions that the table has pages for
            // pages of a tile, each lane one: the page, -1 behind the keys
            auto page_of = [&](int j) {
                const int at = j * KT + lane * box_rows;
                if (!PAGED || lane >= boxes || j >= j0 + all || at >= used) return -1;
                int page = a.page_table[(long long)it.b * a.max_pages + at / a.page];
                if ((unsigned)page >= (unsigned)a.pages) { atomicMin(&bad_page, at); page = 0; }
                return page;
            };
            auto load = [&](const CUtensorMap *map, int j, int page) {
                const unsigned there = PAGED ? __ballot_sync(0xffffffffu, page >= 0) : 1u;
                bool can = true;
                if (lane == 0) {
                    can = mbar_wait_bounded(empty + 8 * st, ph ^ 1);
                    if (can) mbar_expect_tx(full + 8 * st, __popc(there) * box_rows * (D / 64) * 128);
                }
                ok = __shfl_sync(0xffffffffu, can, 0) != 0;
                if (!ok) return;
                const unsigned dst = base + L::KV0 + st * L::STAGE;
                if (PAGED) {
                    if (page >= 0)
                        for (int b = 0; b < D / 64; ++b)
                            tma_load_4d(dst + b * BLOCK_BYTES + lane * box_rows * 128, map, full + 8 * st, 64 * b, group, a.page >= KT ? (j * KT) % a.page : 0, page);
                } else if (lane == 0) {
                    for (int b = 0; b < D / 64; ++b) tma_load_3d(dst + b * BLOCK_BYTES, map, full + 8 * st, 64 * b, group, s.k0 + j * KT);
                }
                if (++st == NST) { st = 0; ph ^= 1; }
            };
            if (WIDE) {
                int page = page_of(j0);
                for (int j = j0; j < j0 + all && ok; ++j) {
                    const int next = page_of(j + 1);
                    load(&kmap, j, page);
                    if (ok) load(&vmap, j, page);
                    page = next;
                }
            } else {                                                  // K0, K1, V0, K2, V1, ...
                int before = page_of(j0), page = page_of(j0 + 1);
                if (all > 0) load(&kmap, j0, before);
                for (int j = j0; j < j0 + all && ok; ++j) {
                    const int next = page_of(j + 2);
                    if (j + 1 < j0 + all) load(&kmap, j + 1, page);
                    if (ok) load(&vmap, j, before);
                    before = page; page = next;
                }
            }
            if (lane == 0) ok = mbar_wait_bounded(qfull, 0) && ok;
            if (!ok && lane == 0) (void)drain_loads<NST>(full, st, ph);
        } else if (warp == MMA_WARP) {
            constexpr unsigned IDESC_S = IDESC_M128<T> | idesc_n(KT), IDESC_O = IDESC_M128<T> | (1u << 16) | idesc_n(D);
            const unsigned leader = elect_leader();
            const unsigned q_base = warp_uniform(desc_lo(base + L::Q0, 16)), k_base = warp_uniform(desc_lo(base + L::KV0, 16)), v_base = warp_uniform(desc_lo(base + L::KV0, BLOCK_BYTES));
            constexpr unsigned STEP = L::STAGE >> 4;
            int st = 0, ph = 0;                                       // next stage to wait for
            auto wait_full = [&]() {                                  // the stage, once it has landed
                ok = ok && mbar_wait_warp(full + 8 * st, ph);
                const int now = st;
                if (++st == NST) { st = 0; ph ^= 1; }
                return now;
            };
            auto scores = [&](int t, int stage) {
                const unsigned q = q_base + (WIDE ? t : 0) * STEP, k = k_base + stage * STEP;
#pragma unroll
                for (int c = 0; c < D / 16; ++c)
                    tc_mma<false>(leader, tmem + L::S_COL + t * KT, q + (c >> 2) * (BLOCK_BYTES >> 4) + (c & 3) * 2, k + (c >> 2) * (BLOCK_BYTES >> 4) + (c & 3) * 2, HI, IDESC_S, c > 0 ? 1u : 0u);
            };
            auto outputs = [&](int t, int stage, bool add) {
                const unsigned v = v_base + stage * STEP;
#pragma unroll
                for (int c = 0; c < KT / 16; ++c)
                    tc_mma_ta<false>(leader, tmem + L::O_COL + t * D, tmem + L::S_COL + t * KT + c * 8, v + c * (2048 >> 4), HI, IDESC_O, add || c > 0 ? 1u : 0u);
            };
            ok = mbar_wait_warp(qfull, 0);
            if (WIDE) {
                if (all > 0 && ok) {
                    const int k = wait_full();
                    if (ok) {
                        tc_fence_after();
                        if (n0 > 0) { scores(0, k); tc_commit_by(leader, sfull); }
                        if (n1 > 0) { scores(1, k); tc_commit_by(leader, sfull + 8); }
                        tc_commit_by(leader, empty + 8 * k);
                    }
                }
                for (int j = 0; j < all && ok; ++j) {
                    const int v = wait_full();
                    int k = -1;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int nt = t == 0 ? n0 : n1;
                        if (j >= nt || !ok) continue;
                        ok = mbar_wait_warp(pfull + 8 * t, j & 1);
                        if (!ok) break;
                        tc_fence_after();
                        outputs(t, v, j > 0);
                        if (j + 1 < nt) {
                            if (k < 0) k = wait_full();
                            if (!ok) break;
                            scores(t, k);
                        }
                        tc_commit_by(leader, sfull + 8 * t);
                    }
                    if (!ok) break;
                    tc_commit_by(leader, empty + 8 * v);
                    if (k >= 0) tc_commit_by(leader, empty + 8 * k);
                }
            } else {
                for (int t = 0; t < 2 && t < all && ok; ++t) {
                    const int k = wait_full();
                    if (!ok) break;
                    scores(t, k);
                    tc_commit_by(leader, sfull + 8 * t);
                    tc_commit_by(leader, empty + 8 * k);
                }
                for (int i = 0; i < all && ok; ++i) {
                    const int t = i & 1, v = wait_full();
                    ok = ok && mbar_wait_warp(pfull + 8 * t, (i >> 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    outputs(t, v, i > 1);
                    tc_commit_by(leader, empty + 8 * v);
                    if (i + 2 < all) {
                        const int k = wait_full();
                        if (!ok) break;
                        scores(t, k);
                        tc_commit_by(leader, empty + 8 * k);
                    }
                    tc_commit_by(leader, sfull + 8 * t);
                }
            }
        } else {
            const int t = warp >> 2, r = tid & 127, steps = t == 0 ? n0 : n1;
            const unsigned quarter = (unsigned)((warp & 3) * 32) << 16;
            const unsigned s_at = tmem + quarter + L::S_COL + t * KT, o_at = tmem + quarter + L::O_COL + t * D;
            const int head0 = r % p.share, token = first + (WIDE ? t * tile_tok : 0) + r / p.share;      // of this thread's row
            const int tile_first = first + (WIDE ? t * tile_tok : 0);
            const bool mine = r < tile_tok * p.share && token < s.nq;
            const int lim = mine ? sees(s, token, a.causal) : 0;
            const int least = tile_first < s.nq ? min(sees(s, tile_first, a.causal), min(s.bad, s.nk)) : 0;      // keys that all its rows see
            const int seen = min(s.nk, s.bad);                        // what lies behind is nobody's
            const bool busy = __any_sync(0xffffffffu, mine);
            const bool turned = p.scale_log2 <= 0.f;                  // the largest score is not the largest product
            const float scale = turned ? 1.f : p.scale_log2;
            float m = -INFINITY, sum = 0.f;
            for (int i = 0; i < steps; ++i) {
                const int j = j0 + (WIDE ? i : 2 * i + t), k0 = j * KT;
                const bool part = k0 + KT > least;
                if (!mbar_wait_warp(sfull + 8 * t, i & 1)) { ok = false; break; }
                tc_fence_after();
                // the values of a tile that not every row sees; behind the scores, which came behind the last use of the stage before this one
                if (part) {
                    const int rel = j - j0, load = WIDE ? 2 * rel + 1 : rel == all - 1 ? 2 * all - 1 : 2 * rel + 2, stage = load % NST;
                    if (!mbar_wait_warp(full + 8 * stage, (load / NST) & 1)) { ok = false; break; }
                    if (clean_row<T, D>(base + L::KV0 + stage * L::STAGE, r) && k0 + r < seen) { atomicMin(&odd_first, k0 + r); atomicMax(&odd_last, k0 + r); }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                }
                if (busy) {
                    float x[KT];
#pragma unroll
                    for (int c = 0; c < KT; c += 32) tc_ld32(s_at + c, x + c);
                    tc_wait_ld();
                    if (turned) {
#pragma unroll
                        for (int c = 0; c < KT; ++c) x[c] *= p.scale_log2;
                    }
                    if (part) {
                        const int left = lim - k0;
#pragma unroll
                        for (int c = 0; c < KT; ++c) x[c] = c < left ? x[c] : -INFINITY;
                    }
                    float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int c = 4; c < KT; c += 4)
#pragma unroll
                        for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], x[c + e]);
                    const float now = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale);
                    const bool grown = mine && now > m + GROWTH;      // each row by itself: its bits do not depend on its neighbours
                    if (i == 0) {
                        m = now;
                    } else if (__any_sync(0xffffffffu, grown)) {
                        const float old = grown ? ex2_ftz(m - now) : 1.f;
                        m = grown ? now : m;
                        sum *= old;
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            tc_ld32(o_at + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] *= old;
                            tc_st32(o_at + c, o);
                        }
                    }
                    const float off = m == -INFINITY ? 0.f : -m;
                    const float2 scale2 = make_float2(scale, scale), off2 = make_float2(off, off);
                    float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < KT; c += 32) {
                        unsigned w[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float2 y = fma2(make_float2(x[c + e], x[c + e + 1]), scale2, off2);
                            y.x = ex2_ftz(y.x); y.y = ex2_ftz(y.y);
                            sums[(e >> 1) & 1] = add2(sums[(e >> 1) & 1], y);
                            w[e >> 1] = pack_pair(T(), y.x, y.y);
                        }
                        tc_st16(s_at + c / 2, w);
                    }
                    sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                    tc_wait_st();
                }
                tc_fence_before();
                mbar_arrive(pfull + 8 * t);
            }
            if (ok && steps > 0) ok = mbar_wait_warp(sfull + 8 * t, steps & 1);      // the outputs are complete
            tc_fence_after();
            float *const handover = reinterpret_cast<float *>(smem_dyn + (base + L::KV0 - (unsigned)__cvta_generic_to_shared(smem_dyn)));
            float other = 0.f, own = 1.f;                             // what the two halves' sums count
            bool join = false;
            if (!WIDE) {
                asm volatile("bar.sync 1, 256;\n" ::: "memory");      // the other half's products have read the stages too
                if (t == 1) {
                    if (busy && steps > 0) {
                        handed[r] = make_float2(m, sum);
#pragma unroll 1
                        for (int c = 0; c < D; c += 32) {
                            float o[32];
                            tc_ld32(o_at + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) handover[(c + e) * ROWS + r] = o[e];
                        }
                    }
                    asm volatile("bar.sync 1, 256;\n" ::: "memory");
                } else {
                    asm volatile("bar.sync 1, 256;\n" ::: "memory");
                    join = n1 > 0;
                    if (join && busy) {
                        const float2 h = handed[r];
                        const float now = fmaxf(m, h.x), from = now == -INFINITY ? 0.f : now;
                        own = exp2f(m - from); other = exp2f(h.x - from);
                        sum = sum * own + h.y * other;
                        m = now;
                    }
                }
            }
            if ((WIDE || t == 0) && busy && ok) {
                const int head = group * p.share + head0, from = j0 * KT;
                const bool none = lim <= from, lost = lim > min(bad_page, s.bad);
                const float nan = __int_as_float(0x7fffffff);
                const long long row = (long long)(s.q0 + token) * a.heads + head;
                const long long at = (long long)blockIdx.x * (tok * p.share) + (WIDE ? t * tile_tok * p.share : 0) + r;
                const float inv = none ? 0.f : lost ? nan : it.parts > 1 && sum == 0.f ? 0.f : 1.f / sum;
                const int odd0 = odd_first, odd1 = odd_last;
#pragma unroll 1
                for (int c = 0; c < D && c < a.dim; c += 32) {
                    float o[32];
                    if (steps > 0) {
                        tc_ld32(o_at + c, o);
                        tc_wait_ld();
                    }
                    if (!mine) continue;
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        o[e] = none || steps == 0 ? 0.f : o[e] * own;
                        if (!WIDE && join && !none) o[e] = fmaf(handover[(c + e) * ROWS + r], other, o[e]);
                        o[e] = none ? 0.f : o[e] * inv;
                    }
                    if (odd1 >= 0 && !none && sum != 0.f) {           // rare: values that are not finite and that this row sees
                        for (int k = odd0; k <= min(lim - 1, odd1); ++k) {
                            const T *v = key_row<T>(a, s, it.b, k, a.value, a.value_strides);
                            if (v == nullptr) continue;
                            v += group * a.value_strides[1] + c;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float f = c + e < a.dim ? to_acc(v[e]) : 0.f;
                                if (!isfinite(f)) o[e] += f;
                            }
                        }
                    }
                    if (it.parts == 1) {
                        store_row(static_cast<T *>(a.out) + row * a.dim + c, o, a.dim - c);
                    } else {
                        float *to = p.part + at * a.dim + c;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            if (e < a.dim - c) *reinterpret_cast<float4 *>(to + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                if (mine) {
                    const float log = none || (it.parts > 1 && sum == 0.f) ? -INFINITY : lost || sum == 0.f ? nan : m + log2f(sum);
                    if (it.parts > 1) p.part_lse[at] = lost ? nan : log;
                    else if (a.lse != nullptr) a.lse[row] = log * 0.6931471805599453f;
                }
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
