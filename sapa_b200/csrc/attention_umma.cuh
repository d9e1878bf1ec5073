// attention_umma.cuh — attention over sequences in 16 bits on the 5th-generation tensor cores, forward.  Included by attention_umma.cu.
//
// A block an SM, items in turn: 128-row tiles (row = token x query head of one key head) against tiles of 128 keys.
//   * a warp finds the items, one ahead (they follow from lengths that only the device knows);
//   * a warp loads queries and keys, another the values, with TMA (rows of 64 channels, 128-byte swizzle; of a paged cache a box a page);
//   * a warp issues S = Q K^T (both operands K-major in shared memory) and O += P V (P in tensor memory, V as TMA lands it, MN-major);
//   * a warpgroup for each of two S / O accumulators: a thread holds a row, 128 scores in registers, so maximum and sum need no shuffles; it writes P,
//     rounded to the type of V as the second product takes it, over S.  The sum is of the weights before that rounding.
// The two accumulators are two row tiles over the same keys (WIDE: long prompts; each key tile is used twice), or one row tile over the even and the
// odd key tiles, joined at the end (single tokens and short chunks): while one's softmax runs, the other's products do.
// O is scaled again only when a row's maximum has grown by more than 2^8 since it last was: weights stay below 2^8 and the sums exact enough, and
// the warpgroup that owns S owns O too at that time, for S was computed behind the product that last added to O.
// What bounds it: of long prompts the tensor pipe between the two softmaxes, the exponentials (a quarter of them by FMA units) and
// the power limit (8192 tokens, 32 heads of 128 channels, causal, bfloat16: 412 us, 1.33 PFLOP/s); of short ones an item's start and end and how
// evenly the items share the SMs; of single tokens reading the cache (209 thousand keys, 8 key heads of 128 channels: 131 us at the copy rate, 150 warm).
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
constexpr int MMA_WARP = 8, LOAD_WARP = 9, PLAN_WARP = 10, VALUE_WARP = 11, NT = 12 * 32;
constexpr int REGS = 168;                                             // a thread's at launch
constexpr unsigned HI = (1024u >> 4) | (1u << 14) | (2u << 29);       // 8 rows of 128 bytes, descriptor version 1, 128-byte swizzle
constexpr int BY_FMA = 1, BY_FMA_OF = 4;                              // exponentials that the FMA units take over
constexpr float GROWTH = 8.f;                                         // powers of two

// 2 row tiles: as many stages as fit beside them
template <int D, bool WIDE> struct Lay {
    static constexpr int STAGE = D / 64 * BLOCK_BYTES, Q_BYTES = (WIDE ? 2 : 1) * STAGE, NST = (224 * 1024 - Q_BYTES) / STAGE > 8 ? 8 : (224 * 1024 - Q_BYTES) / STAGE;
    static constexpr int Q0 = 0, KV0 = Q_BYTES;
    static constexpr int NEED = KV0 + NST * STAGE + 1024, SMEM = NEED < 120 * 1024 ? 120 * 1024 : NEED;      // one block an SM: tensor memory
    static constexpr int S_COL = 0, O_COL = 256, TMEM_COLS = 512;
    // registers a thread: what the softmax needs for a row of scores (with 208 narrow blocks keep 500 bytes of it in memory: single tokens over 209 thousand keys
    // 157 us, 150 with 224; four prompts of up to 100 tokens, in wide blocks, 8.8 us with 208, 9.5 with 224), the rest for the other four warps; multiples of 8
    static constexpr int SOFTMAX_REGS = WIDE ? 208 : 224, OTHER_REGS = WIDE ? 88 : 56;
    static_assert(8 * 32 * SOFTMAX_REGS + 4 * 32 * OTHER_REGS <= NT * REGS, "a block draws on what it was launched with");
    // whether the second product begins with half of a tile's weights.  In 64 channels it is short, and waiting for the stores twice costs more than that
    // gains: one prompt of 8192 tokens, 32 heads, bfloat16: 64 channels 374 us with halves, 358 without; 128 channels 414 and 436.
    static constexpr bool HALVES = D == 128;
    // place in the order of loads of an item's tile, of `all`
    static __device__ __forceinline__ unsigned stage_of(int tile, int all, bool keys) {
        if (WIDE) return 2 * tile + (keys ? 0 : 1);
        return keys ? (tile == 0 ? 0 : 2 * tile - 1) : (tile == all - 1 ? 2 * all - 1 : 2 * tile + 2);
    }
    static_assert(SMEM <= 225 * 1024 && NST >= 3, "shared memory");      // with the 2 KB that a block holds besides
};

// An item of a block: `tok` tokens of a sequence, one key head, key tiles from j0
struct Work {
    bool there;
    int b, group, index, parts;    // index: of the item among all
    int first, j0, all, n0, n1;    // first token; key tiles, of all and of each accumulator
    Sequence s;
    int bad_page, odd_first, odd_last;      // first position without a page; keys with a value that is not finite and not seen by every row
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
// the largest of three, NaN if one of them is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max2(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// 2^x without the unit that ex2 keeps busy: x = n + f with n the nearest whole number, 2^f by a polynomial with the least relative error over [-1/2, 1/2]
// (1.0e-4 in degree 3, a fortieth of bfloat16's half step; 2.8e-6 in degree 4 for float16) that is 1 at 0, and n added to its exponent.  0 from 2^-127 down.
// What a NaN gives is a number: a row with a NaN has to be found by its maximum.
template <typename T> __device__ __forceinline__ float2 ex2_by_fma(float2 x) {
    constexpr float ROUND = 12582912.f;                               // 1.5 * 2^23: adding it leaves whole numbers
    x.x = fmaxf(x.x, -127.f); x.y = fmaxf(x.y, -127.f);
    const float2 t = add2(x, make_float2(ROUND, ROUND)), n = add2(t, make_float2(-ROUND, -ROUND)), f = fma2(n, make_float2(-1.f, -1.f), x);
    float2 y;
    if constexpr (std::is_same<T, __half>::value) {
        y = fma2(f, make_float2(0.009582843631505966f, 0.009582843631505966f), make_float2(0.055906426161527634f, 0.055906426161527634f));
        y = fma2(f, y, make_float2(0.24024099111557007f, 0.24024099111557007f));
        y = fma2(f, y, make_float2(0.6931241750717163f, 0.6931241750717163f));
    } else {
        y = fma2(f, make_float2(0.055008865892887115f, 0.055008865892887115f), make_float2(0.2422109693288803f, 0.2422109693288803f));
        y = fma2(f, y, make_float2(0.693282961845398f, 0.693282961845398f));
    }
    y = fma2(f, y, make_float2(1.f, 1.f));
    return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(t.x) << 23)), __int_as_float(__float_as_int(y.y) + (__float_as_int(t.y) << 23)));
}
__device__ __forceinline__ void tma_load_3d(unsigned dst, const CUtensorMap *map, unsigned bar, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// Replaces what is not finite in 128 bytes of a row of a landed tile with 0; whether there was any.  All are read before they are looked at.
template <typename T> __device__ __forceinline__ bool clean_line(unsigned line, int row) {
    unsigned v[32];
#pragma unroll
    for (int c = 0; c < 8; ++c)                                       // in another order in every row: no two on the same banks
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[4 * c]), "=r"(v[4 * c + 1]), "=r"(v[4 * c + 2]), "=r"(v[4 * c + 3])
                     : "r"(line + ((c ^ (row & 7)) << 4)) : "memory");
    if (finite::all_finite<T, 32>(v)) return false;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(line + ((c ^ (row & 7)) << 4)), "r"(finite::or_zero<T>(v[4 * c])),
                     "r"(finite::or_zero<T>(v[4 * c + 1])), "r"(finite::or_zero<T>(v[4 * c + 2])), "r"(finite::or_zero<T>(v[4 * c + 3])) : "memory");
    return true;
}
// The same for a row of a tile of 128 rows
template <typename T, int D> __device__ __forceinline__ bool clean_row(unsigned tile, int row) {
    bool any = false;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) any = clean_line<T>(tile + b * BLOCK_BYTES + row * 128, row) || any;
    return any;
}
// 32 channels of a row each of a warp's lanes, from float32, those below `left`; `mine`: whether the lane has one.  A row in every lane is a line in every
// lane, and a store takes a cycle for each: so two lanes write halves of one row and then of the other, 32 bytes each (`whole`: rows begin on 32
// bytes).  One prompt of 8192 tokens spent 5800 of an item's 100 thousand clocks on 16-byte stores of a row a lane.
__device__ __forceinline__ void store32(void *to, const unsigned *w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
                 ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
template <typename T> __device__ __forceinline__ void store_rows(T *to, bool mine, const float *v, int left, bool whole) {
    unsigned w[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = pack_pair(T(), v[2 * e], v[2 * e + 1]);
    if (whole && left >= 32) {
        const bool odd = threadIdx.x & 1;
        T *const peer = reinterpret_cast<T *>(__shfl_xor_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), 1));
        const bool peers = __shfl_xor_sync(0xffffffffu, mine, 1);
        unsigned got[8], own[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            own[e] = odd ? w[8 + e] : w[e];
            got[e] = __shfl_xor_sync(0xffffffffu, odd ? w[e] : w[8 + e], 1);
        }
        if (odd ? peers : mine) {                                     // the even lane's row
            unsigned x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = odd ? got[e] : own[e];
            store32(odd ? peer + 16 : to, x);
        }
        if (odd ? mine : peers) {                                     // the odd lane's
            unsigned x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = odd ? own[e] : got[e];
            store32(odd ? to + 16 : peer, x);
        }
    } else if (mine) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (8 * c < left) *reinterpret_cast<uint4 *>(to + 8 * c) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
    }
}
// whether rows of `dim` 16-bit channels from `base` begin on 32 bytes
__device__ __forceinline__ bool whole_rows(const void *base, int dim) { return dim % 16 == 0 && reinterpret_cast<unsigned long long>(base) % 32 == 0; }

}  // namespace um

// LOW: stores what the rounding of the outputs leaves out too.
template <typename T, int D, bool WIDE, bool PAGED, bool LOW>
__global__ void __launch_bounds__(um::NT, 1) sapa_attention_umma_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                                                        const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args p, const int most_items) {
    using namespace um;
    using L = um::Lay<D, WIDE>;
    constexpr int NST = L::NST;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) unsigned long long bars[2 + 2 * NST + 6 + 4 + 4 + 2];
    __shared__ unsigned tmem_slot;
    __shared__ Work queue[2];
    __shared__ float handed[WIDE ? 1 : 2][ROWS];                      // maximum, then sum, of the even and the odd tiles
    const sapa_attention &a = p.a;
    const unsigned base = ((unsigned)__cvta_generic_to_shared(smem_dyn) + 1023u) & ~1023u;
    const unsigned qfull = (unsigned)__cvta_generic_to_shared(bars), qempty = qfull + 8, full = qempty + 8, empty = full + 8 * NST, sfull = empty + 8 * NST, pfull = sfull + 16;
    const unsigned posted = pfull + 32, taken = posted + 16, pair = taken + 16, done = pair + 32;
    const int tid = threadIdx.x, warp = (int)warp_uniform(tid >> 5), lane = tid & 31;
    const int tile_tok = ROWS / p.share, tok = WIDE ? 2 * tile_tok : tile_tok;

    if (warp == MMA_WARP) {
        if (lane == 0) {
            mbar_init(qfull, 1); mbar_init(qempty, 1);
            for (int i = 0; i < NST; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
            for (int i = 0; i < 2; ++i) { mbar_init(sfull + 8 * i, 1); mbar_init(done + 8 * i, 1); mbar_init(pfull + 16 * i, 128); mbar_init(pfull + 16 * i + 8, 128); mbar_init(posted + 8 * i, 1); mbar_init(taken + 8 * i, 11); }
            for (int i = 0; i < 4; ++i) mbar_init(pair + 8 * i, 256);
            asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        }
        __syncwarp();
        tc_alloc((unsigned)__cvta_generic_to_shared(&tmem_slot), L::TMEM_COLS);
        tc_relinquish();
    }
    begin_after_previous();
    clear_outside(static_cast<T *>(a.out), a.offsets, a.B, a.tokens, a.heads * a.dim, blockIdx.x, gridDim.x, tid, NT);
    if (a.lse != nullptr) clear_outside(a.lse, a.offsets, a.B, a.tokens, a.heads, blockIdx.x, gridDim.x, tid, NT);
    if (LOW) clear_outside(static_cast<T *>(a.low), a.offsets, a.B, a.tokens, a.heads * a.dim, blockIdx.x, gridDim.x, tid, NT);
    auto meet = [&]() {
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
    };
    if (warp != PLAN_WARP) meet();                                    // that one looks for the first item meanwhile
    const unsigned tmem = warp_uniform(*reinterpret_cast<volatile unsigned *>(&tmem_slot));
    bool ok = true;
    // the block's items one after the other: what all warps but the plans' go through
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

    if (warp >= MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(L::OTHER_REGS));
        if (warp == PLAN_WARP) {
            ForwardPlans plans(p, tok, lane);
            for (int round = 0;; ++round) {
                // item numbers go there and back over the grid: the work of a block's items evens out
                const int index = round * (int)gridDim.x + (round & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
                Work w{};
                if (index < most_items) {
                    const Plan r = plans.at(index / a.groups);
                    w.there = r.it.there;
                    if (w.there) {
                        w.b = r.it.b; w.parts = r.it.parts; w.group = index % a.groups; w.index = index;
                        w.s = sequence_at(a, w.b);
                        w.first = r.it.block * tok;
                        // key tiles of the two accumulators: [j0, j0 + n[t]) each (WIDE), or every other one
                        w.j0 = r.it.part * (r.it.parts > 1 ? r.tiles : 0);
                        int n[2];
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int last = min(w.first + (WIDE ? (t + 1) * tile_tok : tile_tok), w.s.nq) - 1;      // its last token
                            const bool some = last >= w.first + (WIDE ? t * tile_tok : 0);
                            const int tiles = some ? tiles_of(min(sees(w.s, last, a.causal), w.s.bad), KT) : 0;
                            n[t] = max(0, min(tiles - w.j0, r.tiles));
                        }
                        w.all = max(n[0], n[1]);
                        w.n0 = WIDE ? n[0] : (w.all + 1) / 2;
                        w.n1 = WIDE ? n[1] : w.all / 2;
                    }
                }
                w.bad_page = 0x7fffffff; w.odd_first = 0x7fffffff; w.odd_last = -1;
                if (round == 0) meet();
                ok = mbar_wait_warp(taken + 8 * (round & 1), ((round >> 1) & 1) ^ 1);
                if (!ok) break;
                if (lane == 0) { queue[round & 1] = w; mbar_arrive(posted + 8 * (round & 1)); }
                __syncwarp();
                if (!w.there) break;
            }
        } else if (warp == LOAD_WARP || warp == VALUE_WARP) {
            // keys (and queries) by one warp, values by the other: a box a page takes its time.  They share the ring of stages in the order in which the products
            // take them.  WIDE: K0, V0, K1, V1, ...; otherwise K0, K1, V0, K2, V1, ...: the scores are a tile further ahead.
            const bool keys = warp == LOAD_WARP;
            const CUtensorMap *const map = keys ? &kmap : &vmap;
            int qph = 0;
            unsigned loads = 0;                                       // stages that the items before took
            const int boxes = PAGED ? max(1, KT / a.page) : 1, box_rows = KT / boxes;
            unsigned last = 0;                                        // the last stage of this warp's, and one
            while (Work *w = next_work()) {
                const int j0 = w->j0, all = w->all, b = w->b, group = w->group;
                const Sequence s = w->s;
                const int used = min(s.bad, s.nk);                    // positions that the table has pages for
                // entries of the table for a tile, each lane one.  Looked at only when they are used, so that they are on their way till then.
                auto page_of = [&](int j) {
                    const int at = j * KT + lane * box_rows;
                    return !PAGED || lane >= boxes || j >= j0 + all || at >= used ? -1 : a.page_table[(long long)b * a.max_pages + (unsigned)at / (unsigned)a.page];
                };
                int page = page_of(j0), next = page_of(j0 + 1);
                if (keys && all > 0) {
                    if (lane == 0) {
                        ok = mbar_wait_bounded(qempty, qph ^ 1);
                        if (ok) {
                            mbar_expect_tx(qfull, (WIDE ? 2 : 1) * (D / 64) * 128 * p.share * tile_tok);
                            for (int t = 0; t < (WIDE ? 2 : 1); ++t)
                                for (int c = 0; c < D / 64; ++c)
                                    tma_load_3d(base + L::Q0 + t * L::STAGE + c * BLOCK_BYTES, &qmap, qfull, 64 * c, group * p.share, s.q0 + w->first + t * tile_tok);
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
                    if (!ok) break;
                    qph ^= 1;
                }
                for (int j = j0; j < j0 + all && ok; ++j) {
                    const int behind = page_of(j + 2), at = j * KT + lane * box_rows, rel = j - j0;
                    const unsigned load = loads + L::stage_of(rel, all, keys), st = load % NST, dst = base + L::KV0 + st * L::STAGE;
                    const bool mine = PAGED && lane < boxes && at < used;
                    const unsigned there = PAGED ? __ballot_sync(0xffffffffu, mine) : 1u;
                    if (mine && (unsigned)page >= (unsigned)a.pages) { atomicMin(&w->bad_page, at); page = 0; }
                    __syncwarp();
                    if (lane == 0) {
                        ok = mbar_wait_bounded(empty + 8 * st, ((load / NST) & 1) ^ 1);
                        if (ok) mbar_expect_tx(full + 8 * st, __popc(there) * box_rows * (D / 64) * 128);
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0) != 0;
                    if (!ok) break;
                    if (PAGED) {
                        if (mine)
                            for (int c = 0; c < D / 64; ++c)
                                tma_load_4d(dst + c * BLOCK_BYTES + lane * box_rows * 128, map, full + 8 * st, 64 * c, group, a.page >= KT ? (unsigned)(j * KT) % (unsigned)a.page : 0, page);
                    } else if (lane == 0) {
                        for (int c = 0; c < D / 64; ++c) tma_load_3d(dst + c * BLOCK_BYTES, map, full + 8 * st, 64 * c, group, s.k0 + j * KT);
                    }
                    last = load + 1;
                    page = next; next = behind;
                }
                if (!ok) break;
                loads += 2 * all;
                work_done();
            }
            if (!ok && lane == 0) {                                   // none of its loads may land after it has left: each, while its stage is waited for again
                for (unsigned load = last > NST ? last - NST : 0; load < last; ++load) (void)mbar_wait_bounded(full + 8 * (load % NST), (load / NST) & 1);
                if (keys) (void)mbar_wait_bounded(qfull, qph ^ 1);
            }
        } else if (warp == MMA_WARP) {
            constexpr unsigned IDESC_S = IDESC_M128<T> | idesc_n(KT), IDESC_O = IDESC_M128<T> | (1u << 16) | idesc_n(D);
            const unsigned leader = elect_leader();
            const unsigned q_base = warp_uniform(desc_lo(base + L::Q0, 16)), k_base = warp_uniform(desc_lo(base + L::KV0, 16)), v_base = warp_uniform(desc_lo(base + L::KV0, BLOCK_BYTES));
            constexpr unsigned STEP = L::STAGE >> 4;
            int st = 0, ph = 0, qph = 0, pph0 = 0, pph1 = 0;              // next stage to wait for
            auto wait_full = [&]() {                                      // the stage, once it has landed
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
            auto outputs = [&](int t, int stage, bool add) {              // as its weights come, half a tile at a time
                const unsigned v = v_base + stage * STEP, parity = t == 0 ? pph0 : pph1;
#pragma unroll
                for (int c = 0; c < KT / 16; ++c) {
                    if (c % (KT / 32) == 0) {
                        ok = ok && mbar_wait_warp(pfull + 16 * t + 8 * (c / (KT / 32)), parity);
                        if (!ok) return;
                        tc_fence_after();
                    }
                    tc_mma_ta<false>(leader, tmem + L::O_COL + t * D, tmem + L::S_COL + t * KT + c * 8, v + c * (2048 >> 4), HI, IDESC_O, add || c > 0 ? 1u : 0u);
                }
                if (t == 0) pph0 ^= 1; else pph1 ^= 1;
            };
            // An item's last outputs have a barrier of their own: the next item's first scores come right behind them, and a warp that has not yet seen one phase
            // of a barrier end when the next one does waits for ever.  Everything else is behind weights (pfull) that come from who has seen it.
            while (Work *w = next_work()) {
                const int all = (int)warp_uniform(w->all), n0 = (int)warp_uniform(w->n0), n1 = (int)warp_uniform(w->n1);
                if (all > 0) {
                    ok = mbar_wait_warp(qfull, qph);
                    qph ^= 1;
                }
                if (WIDE) {
                    if (all > 0 && ok) {
                        const int k = wait_full();
                        if (ok) {
                            tc_fence_after();
                            if (n0 > 0) { scores(0, k); tc_commit_by(leader, sfull); }
                            if (n1 > 0) { scores(1, k); tc_commit_by(leader, sfull + 8); }
                            tc_commit_by(leader, empty + 8 * k);
                            if (all == 1) tc_commit_by(leader, qempty);
                        }
                    }
                    for (int j = 0; j < all && ok; ++j) {
                        const int v = wait_full();
                        int k = -1;
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const int nt = t == 0 ? n0 : n1;
                            if (j >= nt || !ok) continue;
                            outputs(t, v, j > 0);
                            if (!ok) break;
                            if (j + 1 < nt) {
                                if (k < 0) k = wait_full();
                                if (!ok) break;
                                scores(t, k);
                            }
                            tc_commit_by(leader, (j + 1 < nt ? sfull : done) + 8 * t);
                        }
                        if (!ok) break;
                        tc_commit_by(leader, empty + 8 * v);
                        if (k >= 0) tc_commit_by(leader, empty + 8 * k);
                        if (j + 2 == all) tc_commit_by(leader, qempty);   // the queries have been read
                    }
                } else {
                    for (int t = 0; t < 2 && t < all && ok; ++t) {
                        const int k = wait_full();
                        if (!ok) break;
                        tc_fence_after();
                        scores(t, k);
                        tc_commit_by(leader, sfull + 8 * t);
                        tc_commit_by(leader, empty + 8 * k);
                        if (t + 1 == all) tc_commit_by(leader, qempty);
                    }
                    for (int i = 0; i < all && ok; ++i) {
                        const int t = i & 1, v = wait_full();
                        if (ok) outputs(t, v, i > 1);
                        if (!ok) break;
                        tc_commit_by(leader, empty + 8 * v);
                        if (i + 2 < all) {
                            const int k = wait_full();
                            if (!ok) break;
                            scores(t, k);
                            tc_commit_by(leader, empty + 8 * k);
                            if (i + 3 == all) tc_commit_by(leader, qempty);
                        }
                        tc_commit_by(leader, (i + 2 < all ? sfull : done) + 8 * t);
                    }
                }
                if (!ok) break;
                work_done();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(L::SOFTMAX_REGS));
        const int t = warp >> 2, r = tid & 127;
        const unsigned quarter = (unsigned)((warp & 3) * 32) << 16;
        const unsigned s_at = tmem + quarter + L::S_COL + t * KT, o_at = tmem + quarter + L::O_COL + t * D;
        const int head0 = r % p.share, row_token = r / p.share;
        const bool in_tile = r < tile_tok * p.share;
        const bool turned = p.scale_log2 <= 0.f;                      // the largest score is not the largest product
        const float scale = turned ? 1.f : p.scale_log2;
        int sph = 0, done_ph = 0;
        unsigned loads = 0;                                           // stages that the items before took
        while (Work *w = next_work()) {
            const Sequence s = w->s;
            const int j0 = w->j0, all = w->all, n0 = w->n0, n1 = w->n1, steps = t == 0 ? n0 : n1;
            const int tile_first = w->first + (WIDE ? t * tile_tok : 0), token = tile_first + row_token;      // of this thread's row
            const bool mine = in_tile && token < s.nq;
            const int lim = mine ? sees(s, token, a.causal) : 0;
            const int seen = min(s.nk, s.bad);                        // what lies behind is nobody's
            const int least = tile_first < s.nq ? min(sees(s, tile_first, a.causal), seen) : 0;      // keys that all its rows see
            const bool busy = __any_sync(0xffffffffu, mine);
            float m = -INFINITY, sum = 0.f;
            for (int i = 0; i < steps; ++i) {
                const int j = j0 + (WIDE ? i : 2 * i + t), k0 = j * KT;
                const bool part = k0 + KT > least;
                if (!mbar_wait_warp(sfull + 8 * t, sph)) { ok = false; break; }
                sph ^= 1;
                tc_fence_after();
                // the values of a tile that not every row sees; behind the scores, which came behind the last use of the stage before this one.  One row tile
                // cleans a tile of keys: the products of the second come behind those of the first, which sees fewer keys and so has cleaned all that it takes.
                if (part && (!WIDE || t == 0 || i >= *const_cast<volatile int *>(&w->n0))) {      // read here: no register for it
                    const unsigned load = loads + L::stage_of(j - j0, all, false), stage = load % NST;
                    if (!mbar_wait_warp(full + 8 * stage, (load / NST) & 1)) { ok = false; break; }
                    if (clean_row<T, D>(base + L::KV0 + stage * L::STAGE, r) && k0 + r < seen) { atomicMin(&w->odd_first, k0 + r); atomicMax(&w->odd_last, k0 + r); }
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    __syncwarp();                                     // lanes that found something went another way: tensor memory is read by whole warps
                }
                if (busy) {
                    float x[KT];
#pragma unroll
                    for (int c = 0; c < KT; c += 32) {
                        tc_ld32(s_at + c, x + c);
                        if (!L::HALVES || c == KT - 32) tc_wait_ld();      // each by itself: what has come is looked at meanwhile
                    }
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
                    for (int c = 4; c + 8 <= KT; c += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e) top[e] = max3(top[e], x[c + e], x[c + 4 + e]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = max2(top[e], x[KT - 4 + e]);
                    const float now = max2(m, max2(max2(top[0], top[1]), max2(top[2], top[3])) * scale);
                    // each row by itself: its bits do not depend on its neighbours.  A NaN goes on into all its weights.
                    const bool grown = mine && !(now <= m + GROWTH);
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
                        unsigned v[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float2 y = fma2(make_float2(x[c + e], x[c + e + 1]), scale2, off2);
                            if ((e >> 1) % BY_FMA_OF < BY_FMA) y = ex2_by_fma<T>(y);
                            else y = make_float2(ex2_ftz(y.x), ex2_ftz(y.y));
                            sums[(e >> 1) & 1] = add2(sums[(e >> 1) & 1], y);
                            v[e >> 1] = pack_pair(T(), y.x, y.y);
                        }
                        tc_st16(s_at + c / 2, v);
                        if (c == (L::HALVES ? KT / 2 : KT) - 32) {    // the second product can begin
                            tc_wait_st();
                            tc_fence_before();
                            mbar_arrive(pfull + 16 * t);
                        }
                    }
                    sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
                    tc_wait_st();
                } else {
                    mbar_arrive(pfull + 16 * t);
                }
                tc_fence_before();
                mbar_arrive(pfull + 16 * t + 8);
            }
            loads += 2 * all;
            if (ok && steps > 0) {                                    // the outputs are complete
                ok = mbar_wait_warp(done + 8 * t, done_ph);
                done_ph ^= 1;
            }
            tc_fence_after();
            if (!(m < INFINITY)) sum = __int_as_float(0x7fffffff);    // infinity less infinity, or a NaN
            float own = 1.f, other = 0.f;                             // what the accumulators' sums count: this row tile's, or the even and the odd key tiles'
            if (!WIDE) {
                auto meet = [&](int i) {                              // of all 256 threads, bounded like every wait
                    mbar_arrive(pair + 8 * i);
                    ok = mbar_wait_warp(pair + 8 * i, turn & 1) && ok;
                };
                handed[t][r] = m;
                tc_fence_before();
                meet(0);                                              // both are complete
                tc_fence_after();
                const float even = handed[0][r], odd = n1 > 0 ? handed[1][r] : -INFINITY;
                m = fmaxf(even, odd);
                const float from = m == -INFINITY ? 0.f : m;
                own = exp2f(even - from); other = n1 > 0 ? exp2f(odd - from) : 0.f;
                meet(1);
                handed[t][r] = sum;
                meet(2);
                sum = handed[0][r] * own + (n1 > 0 ? handed[1][r] * other : 0.f);
            }
            if (busy && ok) {
                const int head = w->group * p.share + head0;
                const bool none = lim <= j0 * KT, lost = lim > min(w->bad_page, s.bad), split = w->parts > 1;
                const float nan = __int_as_float(0x7fffffff);
                const long long row = (long long)(s.q0 + token) * a.heads + head;
                const long long at = (long long)w->index * (tok * p.share) + (WIDE ? t * tile_tok * p.share : 0) + r;
                const float inv = none ? 0.f : lost ? nan : split && sum == 0.f ? 0.f : 1.f / sum;
                const int odd0 = w->odd_first, odd1 = w->odd_last;
                const bool whole = whole_rows(a.out, a.dim) && (!LOW || whole_rows(a.low, a.dim));
                // WIDE: all channels of this tile's row; otherwise each warpgroup half of them
                constexpr int WIDTH = WIDE ? D : D / 2;
#pragma unroll 1
                for (int c = WIDE ? 0 : t * WIDTH; c < (WIDE ? D : (t + 1) * WIDTH) && c < a.dim; c += 32) {
                    float o[32];
                    __syncwarp();                                     // behind the stores of the channels before, which not every lane makes
                    if (all > 0) tc_ld32(WIDE ? o_at + c : tmem + quarter + L::O_COL + c, o);
                    tc_wait_ld();
                    if (!WIDE) {
                        if (n1 > 0) {
                            float q[32];
                            tc_ld32(tmem + quarter + L::O_COL + D + c, q);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = fmaf(q[e], other, o[e] * own);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] *= own;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = none || (WIDE ? steps : all) == 0 ? (none ? 0.f : inv) : o[e] * inv;
                    if (odd1 >= 0 && mine && !none && sum != 0.f) {   // rare: values that are not finite and that this row sees
                        for (int k = odd0; k <= min(lim - 1, odd1); ++k) {
                            const T *v = key_row<T>(a, s, w->b, k, a.value, a.value_strides);
                            if (v == nullptr) continue;
                            v += w->group * a.value_strides[1] + c;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                const float f = c + e < a.dim ? to_acc(v[e]) : 0.f;
                                if (!isfinite(f)) o[e] += f;
                            }
                        }
                    }
                    __syncwarp();
                    if (!split) {
                        store_rows(static_cast<T *>(a.out) + row * a.dim + c, mine, o, a.dim - c, whole);
                        if (LOW) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = left_out<T>(o[e]);
                            store_rows(static_cast<T *>(a.low) + row * a.dim + c, mine, o, a.dim - c, whole);
                        }
                    } else if (mine) {
                        float *to = p.part + at * a.dim + c;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            if (e < a.dim - c) *reinterpret_cast<float4 *>(to + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
                if (mine && (WIDE || t == 0)) {
                    const float log = none || (split && sum == 0.f) ? -INFINITY : lost || sum == 0.f ? nan : m + log2f(sum);
                    if (split) p.part_sums[at] = make_float2(none || sum == 0.f ? -INFINITY : m, none ? 0.f : lost ? nan : sum);
                    else if (a.lse != nullptr) a.lse[row] = log * 0.6931471805599453f;
                }
            }
            tc_fence_before();
            if (!WIDE) {
                mbar_arrive(pair + 24);
                ok = mbar_wait_warp(pair + 24, turn & 1) && ok;       // both accumulators, and what was handed, have been read
            }
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
