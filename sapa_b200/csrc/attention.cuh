// attention.cuh — what the kernels of attention over sequences share: the call's arguments on the device, where a sequence's tokens and keys
// are, and which of them a block of the grid takes.
#pragma once

#include "common.cuh"

namespace sapa {
namespace attn {

struct Args {
    sapa_attention a;
    float scale_log2, scale_rest;  // scale * log2(e): the softmax runs in base 2; what its rounding left out
    int share;                     // query heads of a key head
    int split, least;              // > 0: items that the keys of all sequences are spread over, and tiles of an item at least, see Plan
    float *part;                   // outputs of the parts of split sequences, float32
    float2 *part_sums;             // their maxima and sums, in base 2
};

// Tokens and keys of a sequence, within the tensors whatever the offsets say.
struct Sequence {
    int q0, nq;                    // first token, tokens
    int k0, nk;                    // first key (packed), keys
    int bad;                       // paged: first position that the table has no page for
};
__device__ __forceinline__ int within(int v, int lo, int hi) { return min(max(v, lo), hi); }
__device__ __forceinline__ Sequence sequence_at(const sapa_attention &a, int b) {
    Sequence s;
    s.q0 = within(a.offsets[b], 0, a.tokens);
    s.nq = within(a.offsets[b + 1], s.q0, a.tokens) - s.q0;
    s.k0 = 0;
    s.bad = 0x7fffffff;
    if (a.page_table != nullptr) {
        s.nk = max(a.key_lengths[b], 0);
        const long long room = (long long)a.max_pages * a.page;
        if (s.nk > room) s.bad = (int)room;
    } else {
        s.k0 = within(a.key_offsets[b], 0, a.keys);
        s.nk = within(a.key_offsets[b + 1], s.k0, a.keys) - s.k0;
    }
    return s;
}
// keys that token i of the sequence sees
__device__ __forceinline__ int sees(const Sequence &s, int i, bool causal) {
    return causal ? max(0, s.nk - s.nq + i + 1) : s.nk;      // i < nq
}

// A block's work: `rows` rows (tokens x query heads of one key head, the heads of a token next to each other) of a sequence.
struct Item {
    int b, block, part, parts;     // sequence, block of `tok` tokens in it, part of its keys
    bool there;
};
__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ int warp_scan(int v, int lane) {      // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// The blocks of all sequences in the order of their work, found by a whole warp: those with the most first, so that short ones fill the end.
// `Blocks::at_least(s, w)`: blocks of a sequence with at least w units of work, all for w = 0; `units(s)`: the most that one of its blocks has.  LAST: a
// sequence's blocks have the more work the later they come (a causal token sees the more keys), otherwise the less.  The amount of work is searched
// for by halving, each time adding up the sequences' counts; each lane keeps the first of its sequences in registers.  A block of the grid asks for
// growing indices, so the search goes on from the last one's: mostly nothing is added up again, and no sequence is looked at twice.
// Of more than SORTED sequences the order is theirs: adding up so many again and again would take longer than it gains.
template <bool LAST, typename Blocks> struct InOrder {
    const sapa_attention &a;
    const Blocks kind;
    const int lane;
    Sequence own;
    static constexpr int SORTED = 512;
    int total, lo, hi, upto, behind;                    // all(lo) = upto > index >= behind = all(hi)
    int chunk, passed;                                  // sequences below `chunk` have their blocks of just lo units among the first `passed` ones
    __device__ __forceinline__ InOrder(const sapa_attention &args, const Blocks &k, int l, bool wanted = true)
        : a(args), kind(k), lane(l), own{0, 0, 0, 0, 0}, total(0), lo(0), hi(0), upto(0), behind(0), chunk(0), passed(0) {
        if (!wanted) return;
        if (lane < a.B) own = sequence_at(a, lane);
        int most = kind.units(own);
        for (int b = lane + 32; b < a.B; b += 32) most = max(most, kind.units(sequence_at(a, b)));
        total = all(0);
        hi = (int)__reduce_max_sync(0xffffffffu, (unsigned)most) + 1;
        lo = a.B > SORTED ? 0 : hi;
        upto = a.B > SORTED ? total : 0;
    }
    __device__ __forceinline__ int all(int w) const {
        int n = kind.at_least(own, w);
        for (int b = lane + 32; b < a.B; b += 32) n += kind.at_least(sequence_at(a, b), w);
        return warp_sum(n);
    }
    __device__ __forceinline__ Item at(int index) {
        Item it{0, 0, 0, 1, false};
        if (index >= total) return it;
        if (index >= upto) {
            hi = lo;
            behind = upto;
            lo = 0;
            upto = total;
            while (hi - lo > 1) {
                const int mid = lo + (hi - lo) / 2, n = all(mid);
                if (n > index) { lo = mid; upto = n; } else { hi = mid; behind = n; }
            }
            chunk = 0;
            passed = behind;
        }
        for (int b0 = chunk; b0 < a.B; b0 += 32) {      // among the blocks with just lo units
            const int b = b0 + lane;
            const Sequence s = b0 == 0 ? own : b < a.B ? sequence_at(a, b) : Sequence{0, 0, 0, 0, 0};
            const int more = kind.at_least(s, hi), here = kind.at_least(s, lo) - more, end = warp_scan(here, lane);
            const int left = index - passed;
            const unsigned hit = __ballot_sync(0xffffffffu, left < end);
            if (hit != 0u) {
                const int from = __ffs(hit) - 1, before = more + left - (end - here);      // blocks of the sequence with no less work in front of it
                it.b = b0 + from;
                it.block = __shfl_sync(0xffffffffu, LAST ? kind.at_least(s, 0) - 1 - before : before, from);
                it.there = true;
                return it;
            }
            passed += __shfl_sync(0xffffffffu, end, 31);
            chunk = b0 + 32;
        }
        return it;
    }
};
__device__ __forceinline__ int tiles_of(int n, int tile) { return (int)(((unsigned)n + (unsigned)tile - 1) / (unsigned)tile); }
// Blocks of `tok` tokens, by the tiles of `tile` keys that they go over (what a block's last token sees)
struct QueryBlocks {
    bool causal;
    int tok, tile;
    __device__ __forceinline__ int units(const Sequence &s) const { return tiles_of(min(s.nk, s.bad), tile); }
    __device__ __forceinline__ int at_least(const Sequence &s, int w) const {
        const int n = tiles_of(s.nq, tok), seen = (w - 1) * tile;                     // one key more is needed
        if (w == 0) return n;
        if (min(s.nk, s.bad) <= seen) return 0;
        const int token = seen - s.nk + s.nq;                                         // the first that sees so many
        return !causal || token <= 0 ? n : token >= s.nq ? 0 : n - (int)((unsigned)token / (unsigned)tok);
    }
};
// Blocks of `tile` keys, by the tiles of `tok` tokens that see them
struct KeyBlocks {
    bool causal;
    int tok, tile;
    __device__ __forceinline__ int units(const Sequence &s) const { return tiles_of(s.nq, tok); }
    __device__ __forceinline__ int at_least(const Sequence &s, int w) const {
        const int n = tiles_of(s.nk, tile), last = s.nq - (w - 1) * tok - 1;          // the last token that a block may begin with
        if (w == 0) return n;
        if (last < 0) return 0;
        const int key = last - s.nq + s.nk;                                           // the last key that it sees
        return !causal ? n : key < 0 ? 0 : min(n, (int)((unsigned)key / (unsigned)tile) + 1);
    }
};
// Where a block that is split finds its part: the keys of every sequence are cut into parts of even lengths, tiles of TILE keys,
// so many that all sequences together make about `split` items (their lengths are known on the device alone).  A sequence's blocks all have as many parts as its
// whole length gives; of a causal block the last ones may see nothing and are empty.
constexpr int TILE = 128;
struct Plan {
    Item it;
    int tiles;                     // TILEs of a part
    int first;                     // number of the block's first part among all
};
// Tiles of a part at most, for all sequences
__device__ __forceinline__ int part_tiles(const Args &p, int tok, int lane) {
    unsigned long long work = 0;
    for (int b = lane; b < p.a.B; b += 32) {
        const Sequence s = sequence_at(p.a, b);
        work += (unsigned long long)((s.nq + tok - 1) / tok) * (unsigned)((min(s.nk, s.bad) + TILE - 1) / TILE);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
    return (int)max((work * p.a.groups + p.split - 1) / (unsigned)p.split, (unsigned long long)p.least);
}
// The index-th item (PARTS) or block (!PARTS) of all sequences, by a whole warp.  tok: tokens of a block; most: of part_tiles.
template <bool PARTS>
__device__ __forceinline__ Plan split_at(const Args &p, int index, int tok, int most, int lane) {
    const sapa_attention &a = p.a;
    Plan r{{0, 0, 0, 1, false}, 0x7fffffff / TILE, 0};
    int before = 0, items = 0;     // blocks or items of the sequences before; their items
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int b = b0 + lane;
        int blocks = 0, parts = 1, tiles = 0;
        if (b < a.B) {
            const Sequence s = sequence_at(a, b);
            blocks = (s.nq + tok - 1) / tok;
            tiles = (min(s.nk, s.bad) + TILE - 1) / TILE;
            parts = max(1, (tiles + most - 1) / most);
            tiles = (tiles + parts - 1) / parts;
        }
        const int mine = PARTS ? blocks * parts : blocks, upto = warp_scan(mine, lane), ends = warp_scan(blocks * parts, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, index < before + upto);
        if (hit != 0u) {
            const int from = __ffs(hit) - 1;
            const int at = index - before - __shfl_sync(0xffffffffu, upto - mine, from);
            r.it.parts = __shfl_sync(0xffffffffu, parts, from);
            r.tiles = __shfl_sync(0xffffffffu, tiles, from);
            r.it.b = b0 + from;
            r.it.block = PARTS ? at / r.it.parts : at;
            r.it.part = PARTS ? at % r.it.parts : 0;
            r.it.there = true;
            r.first = items + __shfl_sync(0xffffffffu, ends - blocks * parts, from) + r.it.block * r.it.parts;
            return r;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
        items += __shfl_sync(0xffffffffu, ends, 31);
    }
    return r;
}
// The work of a forward kernel's blocks (group apart), by a whole warp, for growing indices.
struct ForwardPlans {
    const Args &p;
    const int tok, lane, most;
    InOrder<true, QueryBlocks> order;
    __device__ __forceinline__ ForwardPlans(const Args &args, int t, int l)
        : p(args), tok(t), lane(l), most(args.split > 0 ? part_tiles(args, t, l) : 0), order(args.a, QueryBlocks{args.a.causal != 0, t, TILE}, l, args.split == 0) {}
    __device__ __forceinline__ Plan at(int index) {
        if (p.split > 0) return split_at<true>(p, index, tok, most, lane);
        return Plan{order.at(index), 0x7fffffff / TILE, 0};
    }
};

// what rounding to T leaves out of a finite number
template <typename T> __device__ __forceinline__ float left_out(float v) { return isfinite(v) ? v - to_acc(from_acc<T>(v)) : 0.f; }

// Of a backward pass
struct Grads {
    const void *go;                // grad_out
    long long go_strides[2];
    void *gq, *gk, *gv;
    float *delta;                  // sum over channels of grad_out * out: [tokens, heads], or like nlse where that is there
    float *nlse;                   // -log2(e) lse as the tensor-core kernels read it: [groups, tokens, heads of a group]; or NULL
    // float16, otherwise NULL: sums of squares of the rows of grad_out (like nlse) and of value ([groups, keys]), and from them the factor of dS of each
    // sequence and key head ([B, groups])
    float *squares, *value_squares, *factor;
};

// Tensor-core forward (attention_umma.cu): what it takes, and its launch; wide: two row tiles a block.
bool umma_takes(const sapa_attention &a, int dtype);
int umma_forward(const Args &p, bool wide, long long items, int dtype, cudaStream_t st);
int umma_backward(const Args &p, const Grads &g, int dtype, cudaStream_t st);
// Blocks of `tok` tokens that all sequences together can have.
inline long long most_blocks(const sapa_attention &a, long long total, int tok) {
    const long long n = total / tok + a.B;
    return n < total ? n : total;
}

// First element of the row at a position of a sequence's keys; nullptr where the table has no page for it.
template <typename T>
__device__ __forceinline__ const T *key_row(const sapa_attention &a, const Sequence &s, int b, int position, const void *base, const long long (&strides)[3]) {
    if (a.page_table == nullptr) return static_cast<const T *>(base) + (long long)(s.k0 + position) * strides[0];
    const int n = position / a.page;
    if (n >= a.max_pages) return nullptr;
    const int page = a.page_table[(long long)b * a.max_pages + n];
    if ((unsigned)page >= (unsigned)a.pages) return nullptr;
    return static_cast<const T *>(base) + (long long)page * strides[2] + (long long)(position % a.page) * strides[0];
}

// Rows of no sequence (before the first, behind the last) of a dense [rows, width] tensor: zeros, each block of the grid a share, 16 bytes at a time where
// the range allows.
template <typename T>
__device__ __forceinline__ void clear_range(T *x, long long from, long long to, long long at, long long step) {
    constexpr int VEC = 16 / sizeof(T);
    if (((from | to) % VEC) == 0 && (reinterpret_cast<unsigned long long>(x) & 15) == 0) {
        for (long long i = from / VEC + at; i < to / VEC; i += step) reinterpret_cast<uint4 *>(x)[i] = make_uint4(0u, 0u, 0u, 0u);
    } else {
        for (long long i = from + at; i < to; i += step) x[i] = from_acc<T>(0.f);
    }
}
template <typename T>
__device__ __forceinline__ void clear_outside(T *x, const int *offsets, int B, int rows, int width, long long block, long long blocks, int tid, int threads) {
    const int begin = B > 0 ? within(offsets[0], 0, rows) : 0, end = B > 0 ? within(offsets[B], begin, rows) : 0;
    if (begin > 0) clear_range(x, 0, (long long)begin * width, block * threads + tid, blocks * threads);
    if (end < rows) clear_range(x, (long long)end * width, (long long)rows * width, block * threads + tid, blocks * threads);
}

}  // namespace attn
}  // namespace sapa
