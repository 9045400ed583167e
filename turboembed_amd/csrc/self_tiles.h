// The kernel of attention of a call's own tokens: each to the states of its
// sequence up to its own, over the rows of the call (a whole prompt) or over
// the pages of a cache.
//
// The rows of a (sequence, key head) are its tokens' heads that read it, row r
// token r / share, head kv * share + r % share: its keys and values are read
// once for all of them. M of them, 32 or 16, are a wave's; a block is one wave's
// or four waves', or the same rows are four waves', each with every fourth tile
// of the keys. A block's keys pass through LDS in tiles of KB. Scores are
// computed transposed, S^T = K Q^T, so that a lane holds one row (lane % M) and
// M / 2 of 32 keys, the others in the lanes M apart; O^T += V^T P^T then takes P
// as the score registers hold it, against V's columns for the same keys in that
// order (16-bit values by LDS reads that transpose, F32 values one by one). The
// softmax is the running one, in base 2 and F32: what it takes for a row's
// maximum moves only when a score is 2^8 above the one that it was set by.
//
// Int8 states' codes are numbers of every type, so they go into the products
// unscaled: a key's scale is a factor of its scores, a value's one of its
// weights. Four waves get them through registers, a tile ahead, and as numbers
// into LDS; a wave alone has the codes themselves in LDS.
//
// What it reaches, and what bounds it: single tokens the states' bytes (64 over
// 200-8192 BF16 states, 32 heads over 8 of 128: 194 us, 5.7 TB/s; 96 over 100-6000
// int8 states, 12 heads of 64: 125 us, 3.8 TB/s); long 16-bit prompts the
// softmax's vector instructions beside the products (8 x 2048-8192 tokens, 32
// heads over 8 of 128: 2.11-2.15 ms, 920-940 TFLOP/s); F32 prompts how evenly
// blocks of one to 16 tiles fall on the SIMDs (24 x 20-500 tokens, 12 heads of 64:
// 65-71 us, in which matrix instructions, 64 cycles each, are busy a third).
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attention_tile.h"
#include "cache_find.h"
#include "launch.h"

namespace rocm {

template <typename T, Held HELD, int DP, int WAVES, int M, int SPLIT> struct SelfTile {
    static constexpr bool F32 = std::is_same<T, float>::value;
    static constexpr bool BYTES = HELD == Held::Bytes, CODES = HELD == Held::Codes || BYTES;
    static constexpr int ROWS = M * WAVES;
    static constexpr int KB = WAVES == 1 || F32 ? 32 : 64;
    static constexpr int PITCH = DP * (BYTES ? 1 : (int)sizeof(T)), CPR = PITCH / 16;   // a row's bytes and chunks in LDS
    static constexpr int BUF = KB * PITCH;
    // (A wave alone writes a tile of codes' numbers once it has read the one before.
    // While one of F32 or of those that share rows waits for its tile, another of
    // its SIMD computes: more of them fit.)
    static constexpr int BUFS = WAVES == 1 && (SPLIT > 1 || F32 || HELD == Held::Codes) ? 1 : 2;
    static constexpr int TILES = BUFS * 2 * BUF;
    // Behind the tiles: of codes, each buffer's scales of K and V, those of V that
    // are added apart, and the largest of V's; then a word a wave.
    static constexpr int SIDE = (3 * KB + 4) * 4;
    static constexpr int FLAGS = TILES + (CODES ? BUFS * SIDE : 0);
    // Of waves that share rows each has an area, where it leaves its results.
    static constexpr int RESULTS = M * DP * 4 + 1024, AREA = FLAGS > RESULTS ? FLAGS : RESULTS;
    static constexpr int LDS = SPLIT > 1 ? SPLIT * AREA : FLAGS + (WAVES > 1 ? 4 * WAVES : 0);
    static constexpr int OCC = F32 ? (DP <= (HELD == Held::Chunks ? 96 : 64) || WAVES == 4 ? 2 : 1) : DP <= 64 ? 3 : 2;
    // Workgroups of a call over a cache: as many as the card's 256 compute units
    // hold at once, of 160 KiB of LDS each, given in steps of 1280 bytes: their
    // work is equal, and a second turn would be a short one. us at 0.75, 1, 1.34
    // and 2 times as many:
    //   256 tokens over 256 BF16 states each, 4 heads of 64                     33  33  40  41
    //   64 tokens over 200-8192 BF16 states, 32 heads over 8 of 128 (no nt)     263 241 279 245
    //   96 F16 tokens over 100-6000 int8 states, 12 heads of 64                 154 149 166 150
    //   8 x 512 tokens over 1024-8192 int8 states, 32 heads over 8 of 128       589 481 586 484
    static constexpr int BY_LDS = 163840 / ((LDS + 1279) / 1280 * 1280), BY_WAVES = OCC * 4 / WAVES;
    static constexpr int GROUPS = 256 * (BY_LDS < BY_WAVES ? BY_LDS : BY_WAVES);
    static_assert(GROUPS <= (WAVES > 1 ? MOST_TILED : MOST_ALONE), "a workspace holds their parts");
    // LDS serves 256 bytes a cycle, and rows' chunks are swapped so that what it
    // serves at once lies in different banks: 16 keys of one chunk of K; of V what
    // 32 lanes read, 8 bytes each, to transpose.
    static constexpr int PERIOD = CPR % 16 == 0 ? 1 : CPR % 8 == 0 ? 2 : CPR % 4 == 0 ? 4 : 8;   // keys until the banks repeat
    static __device__ __forceinline__ int swap_k(int key) { return CPR == 6 ? 0 : key / PERIOD % (16 / PERIOD); }
    static __device__ __forceinline__ int swap_v(int key) {
        const int k1 = key >> 1 & 1, k2 = key >> 2 & 1, k3 = key >> 3 & 1, k4 = key >> 4 & 1;
        if (BYTES && M == 32) return CPR == 8 ? 2 * (k1 | k3 << 1) : CPR == 4 ? 2 * k3 : 0;      // 0-3, 8-11 by two chunks
        if (BYTES) return CPR == 8 ? k1 | k2 << 1 | k4 << 2 : CPR == 4 ? k2 | k4 << 1 : k4;       // 0-7, 16-23 by one
        if (F32) return CPR % 16 == 0 ? k2 * 8 : 0;
        if (M == 16) return 2 * (key / PERIOD % (8 / PERIOD));                                    // 0-7 by two
        return PERIOD == 1 ? (key & 3) * 4 : PERIOD == 2 ? k1 * 4 : 0;                            // 0-3 by four
    }
    // Codes that a lane moves at once: the most of which a tile is whole loads.
    static constexpr int unit() {
        for (int u = 16; u > 4; u /= 2)
            if (KB * (DP / u) % (64 * WAVES) == 0 && DP % u == 0) return u;
        return 4;
    }
};

// ---- which rows and keys a workgroup takes ---------------------------------------

// A block: rows row0 .. of a (sequence, key head), their keys in tiles first ..
// first + tiles - 1.
struct Block {
    int q0;             // the sequence's first token
    int kv, row0, rows;
    int at0, last;      // the first and the last row's tokens' positions
    int hi;             // keys from hi on are past every row, or the pages
    int first, tiles;
};

// A sequence's blocks of ROWS rows, and what they cost: a block's keys and a
// fixed OVERHEAD, times share (so that row r of them is at r), in closed form.
struct Blocks {
    uint64_t a, most, slope;
    int n, linear;      // blocks; those below `most`
};
constexpr int OVERHEAD = 96;   // keys that a block's start and end are worth

__device__ __forceinline__ int blocks_of(const Seq &s, int share, int rows) {
    return (int)(((uint32_t)s.rows * (uint32_t)share + rows - 1) / (uint32_t)rows);
}

// a / b where it is below 2^52, by F64.
__device__ __forceinline__ uint64_t quotient(uint64_t a, uint64_t b) {
    uint64_t q = (uint64_t)((double)a / (double)b);
    if (q * b > a) --q;
    if ((q + 1) * b <= a) ++q;
    return q;
}

__device__ __forceinline__ Blocks cost_of(const SelfArgs &a, const Seq &s, int rows) {
    Blocks b;
    b.n = blocks_of(s, a.share, rows);
    const int past = within(s.first(), 0, room(a.c));
    b.a = (uint64_t)a.share * (uint64_t)(past + OVERHEAD);
    b.slope = (uint64_t)rows;
    b.linear = b.n;
    b.most = 0;
    if (a.window < room(a.c)) {
        b.most = (uint64_t)a.share * (uint64_t)(a.window + OVERHEAD) + rows;
        b.linear = b.most < b.a ? 0 : (int)min((uint64_t)b.n, quotient(b.most - b.a, b.slope));
    }
    return b;
}
// The cost of the first n blocks.
__device__ __forceinline__ uint64_t cost_to(const Blocks &b, int n) {
    const uint64_t l = (uint64_t)min(n, b.linear);
    return l * b.a + b.slope * (l * (l + 1) / 2) + (uint64_t)(n - (int)l) * b.most;
}

template <int ROWS, int KB> __device__ __forceinline__ Block block_of(const SelfArgs &a, const Seq &s, int kv, int b) {
    Block k;
    const int all = s.rows * a.share;
    k.q0 = s.row0, k.kv = kv, k.row0 = b * ROWS;
    k.rows = min(ROWS, all - k.row0);
    k.at0 = s.first() + k.row0 / a.share;
    k.last = s.first() + (k.row0 + k.rows - 1) / a.share;
    k.hi = a.c.paged ? (k.last < room(a.c) ? k.last + 1 : room(a.c)) : k.last + 1;
    const int lo = a.window > k.at0 ? 0 : k.at0 - a.window + 1;
    k.first = lo / KB;
    k.tiles = max(0, (k.hi + KB - 1) / KB - k.first);
    return k;
}

// The sum of a wave's values up to and with each lane's.
__device__ __forceinline__ uint64_t prefix_sum(uint64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)v, o, 64), hi = (uint32_t)__shfl_up((int)(v >> 32), o, 64);
        if (lane >= o) v += (uint64_t)hi << 32 | lo;
    }
    return v;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

// A place in the order of a key head's tiles: sequence, block, tile.
struct Place {
    int seq, block, tile;
    __device__ bool operator==(const Place &o) const { return seq == o.seq && block == o.block && tile == o.tile; }
};

// The first sequence from i on that has rows, or how many there are: found by a
// wave, 64 a step, as idle ones may be many.
__device__ __forceinline__ int with_rows(const CacheArgs &a, int i) {
    const int lane = threadIdx.x & 63;
    for (; i < a.seqs; i += 64) {
        const uint64_t has = __ballot(i + lane < a.seqs && seq_of(a, i + lane).rows > 0);
        if (has) return i + __ffsll((unsigned long long)has) - 1;
    }
    return a.seqs;
}

// A call over a cache is cut into pieces of equal cost, wherever the cuts fall:
// its lengths are on the device, and one token's sequences may be as different
// as they like. A piece is a workgroup of each key head: those go to one XCD, at
// about one time, as a slot's heads lie next to each other in the cache's lines
// (96 tokens over 100-6000 int8 states, 12 heads of 64: cut across the heads 200
// us, 152 so when that was tried). from .. to are the places of piece g.
template <int ROWS, int KB> struct Cuts {
    Place from, to;
    bool any;
    __device__ __forceinline__ Cuts(const SelfArgs &a, int g, int pieces, uint64_t least) {
        const int lane = threadIdx.x & 63, n = a.c.seqs;
        const auto cost = [&](int i) {
            const Blocks b = cost_of(a, seq_of(a.c, i), ROWS);
            return cost_to(b, b.n);
        };
        // Lane l adds up sequences l * per and on: one sum over the wave, however
        // many sequences there are.
        const int per = (n + 63) / 64;
        uint64_t upto = 0;
#pragma unroll 4
        for (int j = 0; j < per; ++j)
            if (lane * per + j < n) upto += cost(lane * per + j);
        upto = prefix_sum(upto);
        const uint64_t total = lane_of(upto, 63);
        // (No more pieces than their least work makes worth while.)
        const uint64_t worth = quotient(total + least - 1, least);
        if (worth < (uint64_t)pieces) pieces = max(1, (int)worth);
        any = total > 0 && g < pieces;
        if (!any) return;
        // Lane 0 finds the piece's first place, lane 1 the next one's.
        const uint64_t each = quotient(total, (uint64_t)pieces), rest = total - each * (uint64_t)pieces;
        const auto cut = [&](uint64_t i) { return each * i + min(i, rest); };
        const uint64_t f = cut((uint64_t)g + (lane & 1));
        const uint64_t f0 = lane_of(f, 0), f1 = lane_of(f, 1);
        // The sequences of both, and their costs' start.
        int at0 = n, at1 = n;
        uint64_t before0 = total, before1 = total;
        const auto find = [&](uint64_t f, int &at, uint64_t &before) {
            const uint64_t past = __ballot(upto > f);
            if (past == 0) return;
            const int l = __ffsll((unsigned long long)past) - 1;
            at = l * per;
            before = l ? lane_of(upto, l - 1) : 0;
            for (int j = 0; per > 1 && j < per; j += 64) {
                const uint64_t sum = prefix_sum(j + lane < per && at + lane < n ? cost(at + lane) : 0);
                const uint64_t here = __ballot(before + sum > f);
                const int k = here ? __ffsll((unsigned long long)here) - 1 : 64;
                at += k;
                before += k ? lane_of(sum, k - 1) : 0;
                if (here) return;
            }
        };
        find(f0, at0, before0);
        find(f1, at1, before1);
        const int at = lane & 1 ? at1 : at0;
        const uint64_t before = lane & 1 ? before1 : before0;
        Place p{at, 0, 0};
        if (at < n) {
            const Seq s = seq_of(a.c, at);
            const Blocks m = cost_of(a, s, ROWS);
            const uint64_t rest = f - before;
            int lo = 0, hi = m.n;      // cost_to(lo) <= rest < cost_to(hi)
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (cost_to(m, mid) <= rest) lo = mid;
                else hi = mid;
            }
            p.block = lo;
            const uint64_t c0 = cost_to(m, lo), c = cost_to(m, lo + 1) - c0;
            const Block b = block_of<ROWS, KB>(a, s, 0, lo);
            p.tile = min(b.tiles, (int)((double)(rest - c0) / (double)c * (double)b.tiles));
            // (A cut next to a block's end goes there: a part costs its way to memory.)
            const int near = (int)min((uint64_t)b.tiles, quotient(each, (uint64_t)a.share * KB * 8));
            if (p.tile <= near && p.tile * 2 < b.tiles) p.tile = 0;
            else if (b.tiles - p.tile <= near) p.tile = b.tiles;
            if (p.tile == b.tiles) {
                p.tile = 0;
                if (b.tiles > 0 && ++p.block == m.n) p.block = 0, ++p.seq;
            }
        }
        const auto one = [&](int v, int l) { return __builtin_amdgcn_readlane(v, l); };
        from = Place{one(p.seq, 0), one(p.block, 0), one(p.tile, 0)};
        to = Place{one(p.seq, 1), one(p.block, 1), one(p.tile, 1)};
        // (A sequence without rows has no place.)
        from.seq = with_rows(a.c, from.seq), to.seq = with_rows(a.c, to.seq);
    }
};

// Workgroup x's (sequence, key head, block) of a prompt: the blocks with the
// most keys first, over all sequences, so that the last to run are short; of one
// number, the key heads next to each other (8 of them go to as many XCDs). Of
// more than MOST_COUNTED sequences: one after another.
template <int ROWS> struct Turn {
    int seq, kv, block;
    bool any;
    __device__ __forceinline__ Turn(const SelfArgs &a, uint32_t x, char *lds, int threads) {
        const int lane = threadIdx.x & 63, n = a.c.seqs, kv_heads = a.c.kv;
        int *count = (int *)lds;
        const auto blocks = [&](int i) { return i < n ? blocks_of(seq_of(a.c, i), a.share, ROWS) : 0; };
        any = false;
        const int item = (int)(x / (uint32_t)kv_heads);
        kv = (int)(x - (uint32_t)item * (uint32_t)kv_heads);
        if (n > MOST_COUNTED) {
            // (Sequence i's blocks from place i + its first row / ROWS on: they end
            // before the next one's, and a search finds whose a place is.)
            const auto place = [&](int i) {
                return (uint32_t)within(a.c.starts[i], 0, a.c.tokens) * (uint32_t)a.share / ROWS + (uint32_t)i;
            };
            int lo = 0, count = n;
            for (;;) {
                const int step = (count + 63) / 64, at = lane * step;
                const int hits = __popcll(__ballot(at < count && place(lo + at) <= (uint32_t)item));
                if (hits == 0) return;
                const int found = (hits - 1) * step;
                lo += found, count = min(step, count - found);
                if (step == 1) break;
            }
            seq = lo;
            const uint32_t at = (uint32_t)item - place(lo);
            any = at < (uint32_t)blocks(lo);
            block = (int)at;
            return;
        }
        int own = 0;    // the first 64 sequences' in registers
        if (n <= 64) {
            own = blocks(lane);
        } else {
            for (int i = threadIdx.x; i < n; i += threads) count[i] = blocks(i);
            __syncthreads();
        }
        const auto at = [&](int i0) { return n <= 64 ? own : i0 + lane < n ? count[i0 + lane] : 0; };
        // The blocks numbered b or more of all sequences.
        const auto from = [&](int b) {
            int sum = 0;
            for (int i0 = 0; i0 < n; i0 += 64) {
                const uint32_t v = (uint32_t)max(0, at(i0) - b);
                for (int k = 0; __ballot(v >> k) != 0; ++k) sum += __popcll(__ballot(v >> k & 1)) << k;
            }
            return sum;
        };
        if (item >= from(0)) return;
        int lo = 0, hi = a.c.tokens;   // from(hi) <= item < from(lo)
        hi = (int)(((uint64_t)hi * a.share + ROWS - 1) / ROWS);
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (from(mid) > item) lo = mid;
            else hi = mid;
        }
        block = lo;
        int left = item - from(lo + 1);      // of the sequences with more than lo blocks, in order
        for (int i0 = 0; i0 < n; i0 += 64) {
            uint64_t has = __ballot(at(i0) > lo);
            if (left >= __popcll(has)) {
                left -= __popcll(has);
                continue;
            }
            for (; left > 0; --left) has &= has - 1;
            seq = i0 + __ffsll((unsigned long long)has) - 1;
            any = true;
            break;
        }
        if (n > 64) __syncthreads();   // (count lies where tiles will)
    }
};

// ---- parts ---------------------------------------------------------------------------

// The marks of piece p and key head h, u = p kv + h, then their parts: 2 u of the
// block that they start inside of, 2 u + 1 of the one that they leave unfinished.
struct SelfParts {
    SelfMark *marks;
    float *parts;
    uint64_t pitch;
    int pieces;
    uint64_t least;      // cost
    // Workgroup x: eight pieces of a head, then of the next, so that a piece's
    // heads go to one XCD.
    __device__ __forceinline__ void whose(uint32_t x, int kv, int &piece, int &head) const {
        const uint32_t eight = 8u * (uint32_t)kv, q = x / eight, rest = x - q * eight;
        head = (int)(rest / 8), piece = (int)(q * 8 + rest % 8);
    }
    __device__ __forceinline__ float *part(int i) const { return parts + (uint64_t)i * pitch; }
};

// ---- the kernel ------------------------------------------------------------------------

// The largest of a wave's numbers of 0 or more.
__device__ __forceinline__ float wave_max(float v) {
    const auto with = [&](int other) { v = fmaxf(v, __uint_as_float((uint32_t)other)); };
    with(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x128, 0xf, 0xf, true));   // 8 lanes on, of 16
    with(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x124, 0xf, 0xf, true));
    with(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x122, 0xf, 0xf, true));
    with(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x121, 0xf, 0xf, true));
    return four_max(v);
}

// 1 / v of a power of 2 from 2^-126 to 2^126.
__device__ __forceinline__ float inverse(float v) { return __uint_as_float((254u << 23) - __float_as_uint(v)); }

// v, as one that the compiler knows nothing of: what is made of it in a path
// that is rarely taken is made there, and no register holds it meanwhile.
__device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

template <typename T>
__device__ __forceinline__ void two_of(float w0, float w1, T (&hi)[2], T (&lo)[2], bool positive) {
    if (positive) {
        const auto b = below<T>(w0, w1);
        hi[0] = b[0], hi[1] = b[1];
        lo[0] = from_f32<T>(w0 - to_f32(hi[0])), lo[1] = from_f32<T>(w1 - to_f32(hi[1]));
    } else {
        // (Of w0 and w1 as they are in F32: made of a product's exact value, the first
        // number may be another one than that which is taken off.)
        asm("" : "+v"(w0), "+v"(w1));
        hi[0] = from_f32<T>(w0), hi[1] = from_f32<T>(w1);
        lo[0] = from_f32<T>(w0 - to_f32(hi[0])), lo[1] = from_f32<T>(w1 - to_f32(hi[1]));
    }
}

template <typename T, Held HELD, bool PAGED, int DP, int WAVES, int M, int SPLIT>
__global__ void __launch_bounds__(64 * WAVES * SPLIT)
__attribute__((amdgpu_waves_per_eu(SelfTile<T, HELD, DP, WAVES, M, SPLIT>::OCC)))
self_tiles(SelfArgs a, SelfParts parts) {
    using C = SelfTile<T, HELD, DP, WAVES, M, SPLIT>;
    static_assert(WAVES == 1 || SPLIT == 1, "waves share a tile or rows");
    constexpr int THREADS = 64 * WAVES * SPLIT;
    using Mul = Product<T, M>;
    constexpr bool F32 = C::F32, CODES = C::CODES, F16 = std::is_same<T, _Float16>::value;
    // 16-bit weights for the products with V: the sum of two numbers, so that the
    // output's rounding alone shows; but rounded once where four waves share a tile:
    // the matrix cores bound those calls, and a second product with V takes 31% longer
    // (8 x 2048-8192 tokens, 32 heads over 8 of 128: 2.11 to 2.78 ms; 8 x 512 over
    // int8 states: 490 to 600 us). Waves that share rows wait for what comes before:
    // 2000 tokens, 12 heads of 64, 26.5 us with one, 28.6 with two.
    constexpr bool TWO = WAVES == 1 && !F32;
    constexpr int KB = C::KB, SUB = KB / 32, PITCH = C::PITCH, BUF = C::BUF, CPR = C::CPR;
    constexpr int E = Chunk<T>::N, ROWS = C::ROWS;
    static_assert(PAGED || C::LDS >= 4 * MOST_COUNTED, "LDS holds the sequences' numbers of blocks");
    // Lanes of a row; a lane's scores of 32 keys; the results of the product with
    // V, and a lane's registers of one. Register i: key or column 4 H (i / 4) + 4 h
    // + i % 4 (h: which of the row's lanes).
    constexpr int H = 64 / M, NS = M / 2, DT = DP / M, NR = M * M / 64;
    // m is LEAD above the maximum (base 2) that it was set by, and is set again
    // by one that is LAG above that. With a LEAD of LAG weights are 1 at most, so
    // that values of F32's size add up to finite sums. F16's need no such room,
    // and its weights have no range to give away: there they reach 2^LAG.
    constexpr float LAG = 8.0f, LEAD = F16 ? 0.0f : LAG;
    constexpr uint64_t FULL = KB == 64 ? ~0ull : 0xffffffffull;
    typedef typename Chunk<T>::vec vec;
    typedef typename Mul::frag frag;
    typedef typename Mul::acc acc;
    typedef float scores_t __attribute__((ext_vector_type(M / 2)));
    extern __shared__ __attribute__((aligned(1024))) char smem[];

    const int tid = threadIdx.x, lane = tid & 63, number = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Which of the waves that share a tile, or the keys.
    const int wave = WAVES > 1 ? number : 0, own = SPLIT > 1 ? number : 0;
    char *const area = smem + (SPLIT > 1 ? own * C::AREA : 0);
    // What the waves of a tile, or this one alone, wait for each other with.
    const auto sync = [] {
        if constexpr (SPLIT > 1) asm volatile("" ::: "memory");
        else __syncthreads();
    };
    const int r = lane % M, h = lane / M, d = a.c.width;
    const CacheArgs &c = a.c;

    // ---- a tile's way to LDS
    // Of chunks, load j of a wave fills 64 in order; of codes that come through
    // registers, 64 units.
    constexpr bool STAGED = HELD == Held::Codes, BYTES = C::BYTES, DIRECT = HELD == Held::Chunks || BYTES;
    typedef typename std::conditional<CODES, int8_t, T>::type Kept;
    constexpr int UN = STAGED ? C::unit() : 16 / (int)sizeof(Kept), UPR = DP / UN;
    constexpr int NL = KB * UPR / 64 / WAVES;
    static_assert(NL * 64 * WAVES == KB * UPR, "whole loads a wave");
    // A wave alone reads the states of a sequence of one block once: where their rows
    // are whole lines of 128 bytes, past the caches (nt), which have nobody to keep them
    // for. (64 tokens over 200-8192 BF16 states, 32 heads over 8 of 128: 235 us, 212 so;
    // over int8 heads of 64, two of which share a line, 149 and 168. A chunk among
    // many single tokens has more such blocks, each of which reads them again: 200
    // tokens 645 us, 512 of one sequence 133, both in one call 1390.)
    constexpr int ONCE = PAGED && WAVES == 1 && PITCH % 128 == 0 ? 2 : 0;
    constexpr int GROUP = 16;                 // keys that lie in one page, where pages are whole groups
    const auto group_at = [&](int j) { return (wave * NL + j) * 64 / CPR / GROUP * GROUP; };
    const auto unit_at = [&](int j, int l) { return (wave * NL + j) * 64 + l; };
    const auto key_at = [&](int j, int l) { return unit_at(j, l) / UPR; };
    const auto col_k_at = [&](int j, int l) {
        return (STAGED ? unit_at(j, l) % UPR : unit_at(j, l) % CPR ^ C::swap_k(key_at(j, l))) * UN;
    };
    const auto col_v_at = [&](int j, int l) {
        return (STAGED ? unit_at(j, l) % UPR : unit_at(j, l) % CPR ^ C::swap_v(key_at(j, l))) * UN;
    };
    // (Chunks: bytes from a tile's or a group's first key, which 31 bits hold.)
    uint32_t ko[NL], vo[NL];
    if constexpr (DIRECT)
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            const uint32_t key = PAGED ? key_at(j, lane) % GROUP : key_at(j, lane);
            ko[j] = (key * (uint32_t)c.ks[0] + col_k_at(j, lane)) * (uint32_t)sizeof(Kept);
            vo[j] = (key * (uint32_t)c.vs[0] + col_v_at(j, lane)) * (uint32_t)sizeof(Kept);
        }
    // (uniform; where a load has keys of two groups, a lane takes its own)
    const bool groups_whole = PAGED && GROUP * CPR % 64 == 0 && c.page_tokens % GROUP == 0;

    // (Columns past the width keep these zeros. Behind Turn, whose last barrier
    // follows its last look at what it counts in the same bytes.)
    const auto clear = [&] {
        if (HELD == Held::Chunks && d < DP)   // uniform
            for (int i = tid; i < C::LDS / 16; i += THREADS) *(vec *)(smem + i * 16) = vec{};
    };

    Place at{}, end{};
    bool front = false;    // this workgroup starts inside of a block
    int kv, unit_id = 0;   // its key head; of its parts
    if constexpr (PAGED) {
        int piece;
        parts.whose(blockIdx.x, c.kv, piece, kv);
        if (piece >= parts.pieces) return;
        unit_id = piece * c.kv + kv;
        const Cuts<ROWS, KB> cuts(a, piece, parts.pieces, parts.least);
        if (cuts.any) at = cuts.from, end = cuts.to, front = at.tile > 0;
        else at = end = Place{c.seqs, 0, 0};
        if (!front && tid == 0) parts.marks[unit_id] = SelfMark{};
    } else {
        const Turn<ROWS> turn(a, blockIdx.x, smem, THREADS);
        if (!turn.any) return;
        at = Place{turn.seq, turn.block, 0}, kv = turn.kv;
    }
    clear();
    // (A workgroup that begins where it ends, inside of a block, leaves a part
    // without keys.)
    bool more = !PAGED || !(at == end) || front;
    while (more) {
        const Seq seq = seq_of(c, at.seq);
        const Block b = block_of<ROWS, KB>(a, seq, kv, at.block);
        const bool last_here = PAGED && at.seq == end.seq && at.block == end.block;
        const bool begun = at.tile > 0, ends = !last_here || end.tile == b.tiles;
        const int t0 = b.first + at.tile, t1 = b.first + (last_here ? end.tile : b.tiles);
        __syncthreads();    // every wave has read the block before

        const bool work = M * wave < b.rows;   // this wave has rows
        const int row = b.row0 + min(M * wave + r, b.rows - 1);
        const int of_token = a.share == 1 ? row : row / a.share;
        const uint64_t token = (uint64_t)b.q0 + of_token, head = (uint64_t)b.kv * a.share + (row - of_token * a.share);
        // The keys that this lane's row sees, and those that every row of the
        // block does.
        const int pos = seq.first() + of_token;
        const int low = a.window > pos ? 0 : pos - a.window + 1;
        // ...and those that any of this wave's rows does.
        const int ahead = ROWS == M ? b.last : seq.first() + (b.row0 + min(M * wave + M, b.rows) - 1) / a.share;
        const int behind = ROWS == M ? 0 : uniform(__builtin_amdgcn_readlane(low, 0));
        const int all_hi = b.at0, all_lo = a.window > b.last ? 0 : b.last - a.window + 1;
        const Kept *K0 = (const Kept *)c.k + b.kv * c.ks[1], *V0 = (const Kept *)c.v + b.kv * c.vs[1];

        // The slot of key `lane` of a tile, or -1: no state.
        const auto slot_at = [&](int t) {
            const int p = t * KB + lane;
            if (!PAGED) return lane < KB && p < b.hi ? b.q0 + p : -1;
            return t < t1 && lane < KB && p < b.hi ? slot_of(c, at.seq, p) : -1;
        };
        int slot = -1, next_slot = -1;
        bool alive = false;             // of the tile on its way: key `lane` is a state
        // Codes on their way, and their scales (a lane a key).
        typedef uint32_t codes_t __attribute__((ext_vector_type(UN >= 16 ? 4 : UN >= 8 ? 2 : 1), aligned(1)));
        codes_t kq[STAGED ? NL : 1], vq[STAGED ? NL : 1];
        float sk = 0.0f, sv = 0.0f;
        bool apart = false;             // some values are to be added apart

        // n of a unit's codes, a word at a time.
        const auto some_codes = [&](const int8_t *p, int n) {
            typedef uint32_t loose __attribute__((aligned(1)));
            codes_t q{};
#pragma unroll
            for (int w = 0; w < UN / 4; ++w) {
                uint32_t x = 0;
                if (n >= 4 * w + 4) {
                    x = *(const loose *)(p + 4 * w);
                } else {
#pragma unroll
                    for (int i = 0; i < 3; ++i)
                        if (4 * w + i < n) x |= (uint32_t)(uint8_t)p[4 * w + i] << (8 * i);
                }
                q[w] = x;
                __builtin_amdgcn_sched_barrier(0);
            }
            return q;
        };
        // Starts the tile of `slot` on its way; without pages, tile t.
        const auto load = [&](int t, int buf) {
            char *K = area + buf * 2 * BUF, *V = K + BUF;
            alive = slot >= 0;
            if constexpr (CODES)
                if (wave == 0) {
                    sk = alive ? c.k_scales[(uint64_t)slot * c.kss + b.kv] : 0.0f;
                    sv = alive ? c.v_scales[(uint64_t)slot * c.vss + b.kv] : 0.0f;
                }
            if constexpr (DIRECT) {
                // (As buffer loads where a base is common to the lanes: those
                // take 32-bit offsets.)
                typedef __attribute__((address_space(3))) void *to;
                typedef __attribute__((address_space(3))) char *lds;
                typedef __attribute__((address_space(1))) const void *from;
                const auto rsrc = [](const Kept *p) {
                    return __builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, -1, 0x00020000);
                };
                const auto send = [&](__amdgpu_buffer_rsrc_t tile, uint32_t at, char *dst) {
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(tile, (to)((lds)smem + (dst - smem)), 16, (int)at, 0, 0, ONCE);
                };
                const auto base = [&](int j) {
                    // (Without a page: slot 0, whose keys are not looked at.)
                    if constexpr (PAGED)
                        return (uint64_t)max(0, __builtin_amdgcn_readlane(slot, group_at(j)));
                    return (uint64_t)b.q0 + (uint64_t)t * KB;
                };
                const int last = b.hi - 1 - t * KB;
                if ((PAGED ? groups_whole : last >= KB - 1) && d == DP) {   // uniform
#pragma unroll
                    for (int j = 0; j < NL; ++j) {
                        const uint64_t s = base(j);
                        send(rsrc(K0 + s * c.ks[0]), ko[j], K + (wave * NL + j) * 1024);
                        send(rsrc(V0 + s * c.vs[0]), vo[j], V + (wave * NL + j) * 1024);
                    }
                } else if (!PAGED || groups_whole) {   // uniform
                    const int lane = fresh(tid & 63);
#pragma unroll
                    for (int j = 0; j < NL; ++j) {
                        const uint64_t s = base(j);
                        const uint32_t back = PAGED ? 0 : (uint32_t)max(0, key_at(j, lane) - last) * (uint32_t)sizeof(Kept);
                        if (col_k_at(j, lane) < d)
                            send(rsrc(K0 + s * c.ks[0]), ko[j] - back * (uint32_t)c.ks[0], K + (wave * NL + j) * 1024);
                        if (col_v_at(j, lane) < d)
                            send(rsrc(V0 + s * c.vs[0]), vo[j] - back * (uint32_t)c.vs[0], V + (wave * NL + j) * 1024);
                    }
                } else {
                    const int lane = fresh(tid & 63);
#pragma unroll
                    for (int j = 0; j < NL; ++j) {
                        const uint64_t s = (uint64_t)max(0, __shfl(slot, key_at(j, lane), 64));
                        const int ck = col_k_at(j, lane), cv = col_v_at(j, lane);
                        if (ck < d)
                            __builtin_amdgcn_global_load_lds((from)(K0 + s * c.ks[0] + ck), (to)((lds)smem + (K - smem) + (wave * NL + j) * 1024),
                                                             16, 0, ONCE);
                        if (cv < d)
                            __builtin_amdgcn_global_load_lds((from)(V0 + s * c.vs[0] + cv), (to)((lds)smem + (V - smem) + (wave * NL + j) * 1024),
                                                             16, 0, ONCE);
                    }
                }
            } else if constexpr (HELD == Held::Loose) {
                const int lane = fresh(tid & 63);
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    const int s = __shfl(slot, key_at(j, lane), 64), at = unit_at(j, lane) * 16;
                    const int ck = col_k_at(j, lane), cv = col_v_at(j, lane), nk = d - ck, nv = d - cv;
                    *(vec *)(K + at) = s >= 0 && nk > 0 ? read_chunk(K0 + (uint64_t)s * c.ks[0] + ck, nk) : vec{};
                    *(vec *)(V + at) = s >= 0 && nv > 0 ? read_chunk(V0 + (uint64_t)s * c.vs[0] + cv, nv) : vec{};
                }
            } else {
                if (d % UN == 0) {   // uniform
#pragma unroll
                    for (int j = 0; j < NL; ++j) {
                        // (Without a state: slot 0's; past the width: the first
                        // ones again. Neither counts: their weights are 0, the
                        // sums of those columns nobody's, and codes are numbers.)
                        const uint64_t s = (uint64_t)max(0, __shfl(slot, key_at(j, lane), 64));
                        const int col = d == DP || col_k_at(j, lane) < d ? col_k_at(j, lane) : 0;
                        kq[j] = *(const codes_t *)(K0 + s * c.ks[0] + col);
                        vq[j] = *(const codes_t *)(V0 + s * c.vs[0] + col);
                    }
                } else {
                    const int lane = fresh(tid & 63);
#pragma unroll
                    for (int j = 0; j < NL; ++j) {
                        const uint64_t s = (uint64_t)max(0, __shfl(slot, key_at(j, lane), 64));
                        const int col = col_k_at(j, lane);
                        kq[j] = some_codes(K0 + s * c.ks[0] + col, d - col);
                        vq[j] = some_codes(V0 + s * c.vs[0] + col, d - col);
                    }
                }
            }
        };
        // Codes that have come through registers, as numbers of T, into LDS, and the
        // scales of all codes.
        const auto put = [&](int t, int buf) {
            if constexpr (CODES) {
                char *K = area + buf * 2 * BUF, *V = K + BUF;
                float *side = (float *)(area + C::TILES + buf * C::SIDE);
                const auto spread = [&](const codes_t &q, char *row, int col, int swap) {
#pragma unroll
                    for (int e0 = 0; e0 < UN; e0 += E) {
                        T x[E];
#pragma unroll
                        for (int e = 0; e < E; e += 4) numbers_of(q[(e0 + e) / 4], x + e);
                        vec y;
#pragma unroll
                        for (int e = 0; e < E; ++e) y[e] = x[e];
                        *(vec *)(row + (((col + e0) / E) ^ swap) * 16) = y;
                    }
                };
                if constexpr (STAGED)
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    const int key = key_at(j, lane), col = col_k_at(j, lane);
                    spread(kq[j], K + key * PITCH, col, C::swap_k(key));
                    __builtin_amdgcn_sched_barrier(0);   // (one unit's numbers in registers at a time)
                    spread(vq[j], V + key * PITCH, col, C::swap_v(key));
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (wave == 0) {
                    // Values that some rows do not see, and that those cannot have
                    // next to theirs, are added apart.
                    const bool common = t * KB + lane <= all_hi && t * KB + lane >= all_lo;
                    const bool alone = lane < KB && !common && !(fabsf(sv) < INFINITY);
                    apart |= alone;
                    if (lane < KB) {
                        side[lane] = sk;
                        side[KB + lane] = alone ? 0.0f : sv;
                        side[2 * KB + lane] = alone ? sv : 0.0f;
                    }
                    if constexpr (F16) {
                        const float top = wave_max(alone ? 0.0f : fabsf(sv));
                        if (lane == 0) side[3 * KB] = top;
                    }
                }
            }
        };

        // ---- the tiles
        if (t0 + own < t1) {
            slot = slot_at(t0 + own);
            load(t0 + own, 0);
            next_slot = slot_at(t0 + own + SPLIT);
        }
        // This row's q: of each H E columns the lane's E. Of codes as they are, whose
        // chunks are 2 E columns, of each 2 H E the lane's chunk, if they are so many.
        constexpr int NQ = DP / (H * E);
        constexpr bool PAIRS = BYTES && NQ % 2 == 0;
        vec q[NQ];
        {
            const int h = fresh(lane) / M;   // (else its comparisons are kept from block to block)
            const T *p = (const T *)a.q + token * a.qs[0] + head * a.qs[1];
#pragma unroll
            for (int s = 0; s < NQ; ++s) {
                const int col = PAIRS ? (H * (s >> 1) + h) * 2 * E + (s & 1) * E : (H * s + h) * E;
                q[s] = read_chunk(p + col, d - col);
            }
            if (a.turn != 1.0f)   // uniform
#pragma unroll
                for (int s = 0; s < NQ; ++s)
#pragma unroll
                    for (int e = 0; e < E; ++e) q[s][e] = from_f32<T>(to_f32(q[s][e]) * a.turn);
        }

        acc o[DT];
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = acc{};
        float m = -INFINITY, l = 0.0f;
        bool any = false, far = false;   // this row has seen a state; a maximum past 2^24
        // Weights of F16 have no range for a value's scale beside their own: they are
        // of its size against a power of 2 that is at least this row's largest so far,
        // and twice to four times it when that sets it (from 2^-40 on, of which 127
        // halves are nothing in F16). Those of rows that see other states differ, and
        // nothing of a row depends on what it does not see.
        float unit = __uint_as_float((127 - 40) << 23);

        // S^T of the tile's keys, 32 of them a scores_t.
        const int kr = r * PITCH, ks = C::swap_k(r);
        const auto scores = [&](const char *K, scores_t (&s)[SUB]) {
            // M keys at a time, from m0 of tile part u: their results go next to each other.
            constexpr int BLOCKS = 32 / M;
            acc part[SUB][BLOCKS];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int v = 0; v < BLOCKS; ++v) part[u][v] = acc{};
            // (32 keys on, the swap is the same; 16 on it may not be.)
            const auto row = [&](int u, int v) { return K + (32 * u + M * v) * PITCH + kr; };
            const auto swap = [&](int v) { return M == 32 ? ks : C::swap_k(r + M * v); };
            if constexpr (BYTES) {
                typedef uint32_t words __attribute__((ext_vector_type(PAIRS ? 4 : 2)));
#pragma unroll
                for (int x = 0; x < (PAIRS ? NQ / 2 : NQ); ++x)
#pragma unroll
                    for (int v = 0; v < BLOCKS; ++v) {
                        const words w = PAIRS ? *(const words *)(row(0, v) + ((H * x + h) ^ swap(v)) * 16)
                                              : *(const words *)(row(0, v) + ((H / 2 * x + h / 2) ^ swap(v)) * 16 + h % 2 * 8);
#pragma unroll
                        for (int z = 0; z < (PAIRS ? 2 : 1); ++z) {
                            T n[8];
                            numbers_of(w[2 * z], n), numbers_of(w[2 * z + 1], n + 4);
                            frag f;
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] = n[e];
                            part[0][v] = Mul::run(f, q[PAIRS ? 2 * x + z : x], part[0][v]);
                        }
                    }
            } else if constexpr (F32) {
                // (A chunk read two ahead of its products, which are slow enough to hide it.)
                const auto chunk = [&](int x) { return *(const vec *)(row(0, 0) + ((2 * x + h) ^ ks) * 16); };
                vec k[3] = {chunk(0), chunk(1)};
#pragma unroll
                for (int x = 0; x < NQ; ++x) {
                    if (x + 2 < NQ) k[(x + 2) % 3] = chunk(x + 2);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < E; ++e) part[0][0] = Mul::run(k[x % 3][e], q[x][e], part[0][0]);
                }
            } else {
                // (Chunks read two steps ahead of their products: an LDS read takes
                // longer than the products of one.)
                constexpr int AHEAD = NQ < 3 ? NQ : 3;
                vec k[AHEAD][SUB][BLOCKS];
                const auto ahead = [&](int x) {
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int v = 0; v < BLOCKS; ++v)
                            k[x % AHEAD][u][v] = *(const vec *)(row(u, v) + ((H * x + h) ^ swap(v)) * 16);
                };
#pragma unroll
                for (int x = 0; x < AHEAD - 1; ++x) ahead(x);
#pragma unroll
                for (int x = 0; x < NQ; ++x) {
                    if (x + AHEAD - 1 < NQ) ahead(x + AHEAD - 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int v = 0; v < BLOCKS; ++v) part[u][v] = Mul::run(k[x % AHEAD][u][v], q[x], part[u][v]);
                }
            }
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < NS; ++i) s[u][i] = part[u][i / NR][i % NR];
        };
        // O^T += V^T P^T over 32 keys; weight(i) is register i's, in order.
        const auto add_values = [&](const char *V, auto weight) {
            if constexpr (F32) {
                // (Values and weights two keys ahead of their products.)
                float v[3][DT], p[3];
                const auto ahead = [&](int i) {
                    const int key = 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
                    for (int t = 0; t < DT; ++t)
                        v[i % 3][t] =
                            *(const float *)(V + key * PITCH + (((r >> 2) + 8 * t) ^ C::swap_v(key)) * 16 + (r & 3) * 4);
                    p[i % 3] = weight(i);
                };
                ahead(0), ahead(1);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (i + 2 < 16) ahead(i + 2);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int t = 0; t < DT; ++t) o[t] = Mul::run(v[i % 3][t], p[i % 3], o[t]);
                }
            } else {
                // 8 H keys a product: registers 8 j .. 8 j + 7. A group of 16 lanes
                // reads 4 keys by 16 columns, and a lane gets its column's 4; of
                // codes 8 keys.
                const int n = lane & 15, half = r >> 4;    // which 16 of the product's columns
                // (4 H keys on, and 8 H, the swap is the same.)
                constexpr int AT = DT < 4 ? DT : DT % 4 == 0 ? 4 : 3;   // results at a time
                uint32_t place[DT];
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const int k = BYTES ? 4 * H * (n >> 3) + 4 * h + ((n >> 1) & 3) : 4 * h + (n >> 2);
                    const int x = BYTES ? M / 16 * t + half : M / 8 * t + 2 * half + ((n >> 1) & 1);
                    place[t] = (uint32_t)(uintptr_t)(lds_ptr)smem + (uint32_t)(V - smem) + k * PITCH + (x ^ C::swap_v(k)) * 16 + (n & 1) * 8;
                }
                const auto product = [&](auto jj) {
                    constexpr int j = decltype(jj)::value;
                    frag f, rest;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float w0 = weight(8 * j + e), w1 = weight(8 * j + e + 1);
                        if constexpr (TWO) {
                            T hi[2], lo[2];
                            two_of<T>(w0, w1, hi, lo, !CODES);
                            f[e] = hi[0], f[e + 1] = hi[1], rest[e] = lo[0], rest[e + 1] = lo[1];
                        } else {
                            f[e] = from_f32<T>(w0), f[e + 1] = from_f32<T>(w1);
                        }
                    }
#pragma unroll
                    for (int t0 = 0; t0 < DT; t0 += AT) {
                        uint32_t at[4];
#pragma unroll
                        for (int t = 0; t < 4; ++t) at[t] = place[t0 + (t < AT ? t : 0)];
                        frag v[AT];
                        if constexpr (BYTES) {
                            words2 w[4];
                            read_tr8<8 * H * j * PITCH>(w, at);
#pragma unroll
                            for (int t = 0; t < AT; ++t) {
                                T y[8];
                                numbers_of(w[t][0], y), numbers_of(w[t][1], y + 4);
#pragma unroll
                                for (int e = 0; e < 8; ++e) v[t][e] = y[e];
                            }
                        } else {
                            words2 w[8];
                            read_tr16<8 * H * j * PITCH, 4 * H * PITCH>(w, at);
#pragma unroll
                            for (int t = 0; t < AT; ++t) {
                                struct {
                                    words2 lo, hi;
                                } both{w[2 * t], w[2 * t + 1]};
                                v[t] = __builtin_bit_cast(frag, both);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < AT; ++t) o[t0 + t] = Mul::run(v[t], f, o[t0 + t]);
                        if constexpr (TWO)
#pragma unroll
                            for (int t = 0; t < AT; ++t) o[t0 + t] = Mul::run(v[t], rest, o[t0 + t]);
                    }
                };
                product(std::integral_constant<int, 0>());
                if constexpr (NS / 8 > 1) product(std::integral_constant<int, 1>());
            }
        };
        const auto raise = [&](float mx) {   // m, for scores of up to mx
            if (__ballot(mx > m + (LAG - LEAD)) == 0) return;
            const float mn = fmaxf(m, mx + LEAD);
            // (Equal: both infinite, of one sign.)
            const float f = __builtin_amdgcn_exp2f(m == mn ? 0.0f : m - mn);
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= f;
            l *= f;
            m = mn;
            far = __ballot(fabsf(m) > 16777216.0f && m != -INFINITY) != 0;
        };
        // The keys of a tile that this lane's row sees.
        const auto seen_of = [&](uint64_t live, int t) -> uint64_t {
            if (t * KB + KB - 1 <= all_hi && t * KB >= all_lo) return live;   // uniform
            const int lo = max(0, low - t * KB), hi = min(KB - 1, pos - t * KB);
            return lo > hi ? 0 : live & (~0ull << lo) & (~0ull >> (63 - hi));
        };
        const auto scaled_scores = [&](const char *K, const float *side, scores_t (&s)[SUB]) {
            scores(K, s);
            if constexpr (CODES)
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int g = 0; g < NS / 4; ++g) {
                        const f32x4 f = *(const f32x4 *)(side + 32 * u + 4 * H * g + 4 * h);
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[u][4 * g + e] *= f[e];
                    }
        };
        // `unit`, for a tile with a value's scale above it. (Rarely: in a loop, before
        // there are scores, for the registers.)
        const auto raise_unit = [&](const float *side, uint64_t live, int t) {
            if (__ballot(side[3 * KB] > unit) == 0) return;
            const uint64_t seen = seen_of(live, t);
            float top = 0.0f;
#pragma nounroll
            for (int key = 4 * (fresh(lane) / M); key < KB; key += 4 * H) {
                const f32x4 v = *(const f32x4 *)(side + KB + key);
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, seen >> (key + e) & 1 ? fabsf(v[e]) : 0.0f);
            }
            top = M == 32 ? both_max(top) : four_max(top);
            const uint32_t e = min(253u, (__float_as_uint(top) >> 23) + 2);
            const float now = top > unit ? __uint_as_float(e << 23) : unit, f = unit * inverse(now);
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= f;
            unit = now;
        };
        const auto tile = [&](const char *K, const float *side, uint64_t live, int t) {
            if constexpr (CODES && F16) raise_unit(side, live, t);
            scores_t s[SUB];
            scaled_scores(K, side, s);
            const uint64_t seen = seen_of(live, t);
            any |= seen != 0;
            if (__ballot(seen != FULL) != 0) {
#pragma unroll
                for (int u = 0; u < SUB; ++u) {
                    const uint32_t word = (uint32_t)(seen >> (32 * u)) >> (4 * h);
#pragma unroll
                    for (int i = 0; i < NS; ++i)
                        s[u][i] = (word >> (4 * H * (i >> 2) + (i & 3))) & 1u ? s[u][i] : -INFINITY;
                }
            }
            // Waves that share a tile or rows: a product's values are on their way while
            // the one before runs, and two of its weights are made behind each of that
            // one's instructions (8 x 2048-8192 tokens, 32 heads over 8 of 128: 2068 to
            // 2021 us).
            constexpr bool EARLY = !F32 && !CODES && (WAVES > 1 || SPLIT > 1);
            constexpr int STEP = 8 * H, STEPS = KB / STEP;   // keys of a product
            frag v[2][EARLY ? DT : 1];
            const auto fetch = [&](int x) {
                typedef short s4 __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) char *lds;
                typedef __attribute__((address_space(3))) s4 *from;
                const int n = lane & 15, half = r >> 4, k = 4 * h + (n >> 2);
                if constexpr (EARLY)
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const lds at = (lds)smem + (K - smem) + k * PITCH + ((M / 8 * t + 2 * half + ((n >> 1) & 1)) ^ C::swap_v(k)) * 16 +
                                   (n & 1) * 8 + BUF + x * STEP * PITCH;
                    struct {
                        s4 lo, hi;
                    } both{__builtin_amdgcn_ds_read_tr16_b64_v4i16((from)at),
                           __builtin_amdgcn_ds_read_tr16_b64_v4i16((from)(at + 4 * H * PITCH))};
                    v[x % 2][t] = __builtin_bit_cast(frag, both);
                }
            };
            if constexpr (EARLY) {
                fetch(0);
                __builtin_amdgcn_sched_barrier(0);
            }
            float mx = s[0][0];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < NS; ++i) mx = fmaxf(mx, s[u][i]);
            raise((M == 32 ? both_max(mx) : four_max(mx)) * a.scale);
            const float base = m == -INFINITY ? 0.0f : m;
            // A score's distance from the maximum in one rounding; where the
            // maximum is so large that its own rounding shows, from the rounded
            // score, which is no larger.
            float scale = a.scale;
            if (far) {   // uniform
#pragma unroll
                for (int u = 0; u < SUB; ++u) s[u] *= scale;
                scale = 1.0f;
            }
            if constexpr (EARLY) {
                // Two weights of the next product behind each of this one's.
                float sum[2] = {};
                const auto pair = [&](int x, int e, frag &f, frag &rest) {
                    const int u = x * STEP / 32, i = x * STEP % 32 / STEP * 8 + e;
                    const float w0 = __builtin_amdgcn_exp2f(fmaf(s[u][i], scale, -base));
                    const float w1 = __builtin_amdgcn_exp2f(fmaf(s[u][i + 1], scale, -base));
                    sum[0] += w0, sum[1] += w1;
                    if constexpr (TWO) {
                        T hi[2], lo[2];
                        two_of<T>(w0, w1, hi, lo, true);
                        f[e] = hi[0], f[e + 1] = hi[1], rest[e] = lo[0], rest[e + 1] = lo[1];
                    } else {
                        f[e] = from_f32<T>(w0), f[e + 1] = from_f32<T>(w1);
                    }
                };
                frag f, rest, f2, rest2;
#pragma unroll
                for (int e = 0; e < 8; e += 2) pair(0, e, f, rest);
#pragma unroll
                for (int x = 0; x < STEPS; ++x) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (x + 1 < STEPS) fetch(x + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int t = 0; t < (DT > 4 ? DT : 4); ++t) {
                        if (t < DT) o[t] = Mul::run(v[x % 2][t], f, o[t]);
                        __builtin_amdgcn_sched_barrier(0);
                        if (x + 1 < STEPS && t < 4) pair(x + 1, 2 * t, f2, rest2);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if constexpr (TWO)
#pragma unroll
                        for (int t = 0; t < DT; ++t) o[t] = Mul::run(v[x % 2][t], rest, o[t]);
                    f = f2;
                    if constexpr (TWO) rest = rest2;
                }
                l += sum[0] + sum[1];
                return;
            }
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                float sum = 0.0f;
                f32x4 sv[NS / 4];
                if constexpr (CODES)
#pragma unroll
                    for (int g = 0; g < NS / 4; ++g) sv[g] = *(const f32x4 *)(side + KB + 32 * u + 4 * H * g + 4 * h);
                const float inv = inverse(unit);
                add_values(K + BUF + 32 * u * PITCH, [&](int i) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(s[u][i], scale, -base));
                    sum += w;
                    if constexpr (CODES && F16) return w * inv * sv[i >> 2][i & 3];
                    if constexpr (CODES) return w * sv[i >> 2][i & 3];
                    return w;
                });
                l += sum;
            }
        };
        // Values that are no numbers weigh nothing for the rows that do not see
        // them, but 0 times them is no number: where some row does not see them,
        // they are 0 for the products, and are added here, once the maxima are
        // known. (Slowly: this is as good as never.)
        const auto add_apart = [&](const char *K, const float *side, uint64_t live, int t) {
            scores_t s[SUB];
            scaled_scores(K, side, s);
            const int h = fresh(lane) / M;
            const uint64_t seen = seen_of(live, t);
            const float base = m == -INFINITY ? 0.0f : m;
            for (int key = 0; key < KB; ++key) {
                const bool see = seen >> key & 1;
                if (__ballot(see) == 0) continue;
                float extra = 1.0f;
                if constexpr (CODES) {
                    extra = side[2 * KB + key];
                    if (__ballot(extra != 0.0f) == 0) continue;
                }
                const int i = (key & 31) / (4 * H) * 4 + (key & 3), from = (key >> 2) % H;
                float x = 0.0f;
#pragma unroll
                for (int v = 0; v < SUB; ++v)
#pragma unroll
                    for (int n = 0; n < NS; ++n) x = key >> 5 == v && i == n ? s[v][n] : x;
                x = __shfl(x, r + M * from, 64);
                const float w = (far ? __builtin_amdgcn_exp2f(x * a.scale - base)
                                     : __builtin_amdgcn_exp2f(fmaf(x, a.scale, -base))) * extra;
                typedef T four __attribute__((ext_vector_type(4)));
                const char *row = K + BUF + key * PITCH;
                const int swap = C::swap_v(key);
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int g = 0; g < NR / 4; ++g) {
                        const int at = (M * t + 4 * H * g + 4 * h) * (BYTES ? 1 : (int)sizeof(T));
                        const char *p = row + ((at >> 4) ^ swap) * 16 + (at & 15);
                        four v;
                        if constexpr (BYTES) {
                            T n[4];
                            numbers_of(*(const uint32_t *)p, n);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = n[e];
                        } else {
                            v = *(const four *)p;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float f = to_f32(v[e]);
                            o[t][4 * g + e] = see && (CODES || !(fabsf(f) < INFINITY)) ? fmaf(w, f, o[t][4 * g + e]) : o[t][4 * g + e];
                        }
                        __builtin_amdgcn_sched_barrier(0);   // (this path is to cost no registers)
                    }
            }
        };
        const auto is_partial = [&](int t) { return t * KB + KB - 1 > all_hi || t * KB < all_lo; };   // uniform

        for (int t = t0 + own, buf = 0; t < t1; t += SPLIT, buf ^= C::BUFS - 1) {
            char *K = area + buf * 2 * BUF, *V = K + BUF;
            const float *side = (const float *)(area + C::TILES + buf * C::SIDE);
            if constexpr (!STAGED) __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's loads are in LDS
            if constexpr (CODES) put(t, buf);
            const uint64_t live = __ballot(alive);
            if (!CODES && live != FULL) {   // uniform
                // A value that is no state's weighs 0, but not if it is no number.
                const int lane = fresh(tid & 63);
#pragma unroll
                for (int j = 0; j < NL; ++j)
                    if (!((live >> key_at(j, lane)) & 1)) *(vec *)(V + unit_at(j, lane) * 16) = vec{};
            }
            if (!CODES && is_partial(t)) {
                const int lane = fresh(tid & 63);
#pragma unroll
                for (int j = 0; j < NL; ++j) {
                    vec x = *(const vec *)(V + unit_at(j, lane) * 16);
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < E; ++e) sum = fmaf(to_f32(x[e]), 0.0f, sum);
                    if (sum != 0.0f) {   // (0 times a number is 0)
#pragma unroll
                        for (int e = 0; e < E; ++e) x[e] = fabsf(to_f32(x[e])) < INFINITY ? x[e] : (T)0.0f;
                        *(vec *)(V + unit_at(j, lane) * 16) = x;
                        apart = true;
                    }
                }
            }
            sync();   // the tile is there, and the other one read
            const auto next = [&] {
                if (t + SPLIT < t1) {
                    slot = next_slot;
                    load(t + SPLIT, buf ^ (C::BUFS - 1));
                    next_slot = slot_at(t + 2 * SPLIT);
                }
            };
            // (Into the buffer that is being read, once it has been.)
            constexpr bool LATE = C::BUFS == 1 && !STAGED;
            if constexpr (!LATE) next();
            if (work && live != 0 && t * KB <= ahead && t * KB + KB > behind) tile(K, side, live, t);   // (uniform)
            if constexpr (LATE) {
                __builtin_amdgcn_sched_barrier(0);
                next();
            }
        }
        bool again = __ballot(apart) != 0;
        if constexpr (WAVES > 1) {
            int *flags = (int *)(smem + C::FLAGS);
            if (lane == 0) flags[wave] = again;
            __syncthreads();
            int sum = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) sum |= flags[w];
            again = uniform(sum) != 0;
        }
        if (again) {   // uniform over the workgroup
            for (int t = t0 + own; t < t1; t += SPLIT) {
                if (!is_partial(t)) continue;
                sync();
                slot = slot_at(t);
                load(t, 0);
                __builtin_amdgcn_s_waitcnt(0x0f70);
                if constexpr (CODES) put(t, 0);
                const uint64_t live = __ballot(alive);
                sync();
                if (work) add_apart(area, (const float *)(area + C::TILES), live, t);
            }
        }

        if (work) {
            const int h = fresh(lane) / M;
            l = M == 32 ? both_sum(l) : four_sum(l);
            if constexpr (CODES && F16)
#pragma unroll
                for (int t = 0; t < DT; ++t) o[t] *= unit;
            // Four of a row's sums, from column col on: divided into the output, or
            // into a part.
            const int at = M * wave + r, groups = (d + 3) / 4;
            const bool there = at < b.rows, direct = !PAGED || (!begun && ends);
            f32x4 *const part = (f32x4 *)parts.part(2 * unit_id + (begun ? 0 : 1));
            T *const out = (T *)a.out + token * a.os[0] + head * a.os[1];
            const auto leave = [&](int col, const f32x4 &v, float inv) {
                if (!there) return;
                if (!direct) {
                    // (Four columns of every row, then the next four.)
                    if (col / 4 < groups) part[col / 4 * b.rows + at] = v;
                    return;
                }
                typedef T loose4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
                const loose4 y{from_f32<T>(v[0] * inv), from_f32<T>(v[1] * inv), from_f32<T>(v[2] * inv), from_f32<T>(v[3] * inv)};
                if (col + 4 <= d) {
                    *(loose4 *)(out + col) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (col + e < d) out[col + e] = y[e];
                }
            };
            if constexpr (SPLIT > 1) {
                // The waves' results, each from its own maximum, together.
                f32x4 *const mine = (f32x4 *)area;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int g = 0; g < NR / 4; ++g)
                        mine[(t * (NR / 4) + g) * 64 + lane] = f32x4{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]};
                constexpr int LAST = M * DP * 4 / 16;
                mine[LAST + lane] = f32x4{m, l, any ? 1.0f : 0.0f, 0.0f};
                __syncthreads();
                const auto of = [&](int w) { return (const f32x4 *)(smem + w * C::AREA); };
                f32x4 each[SPLIT];
                m = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < SPLIT; ++w) each[w] = of(w)[LAST + lane], m = fmaxf(m, each[w][0]);
#pragma unroll
                for (int w = 0; w < SPLIT; ++w) {
                    // (Equal: both infinite, of one sign.)
                    each[w][0] = __builtin_amdgcn_exp2f(each[w][0] == m ? 0.0f : each[w][0] - m);
                    l = fmaf(each[w][0], each[w][1], l);
                    any |= each[w][2] != 0.0f;
                }
                const float inv = any ? 1.0f / l : 0.0f;
                for (int x = own; x < DT * (NR / 4); x += SPLIT) {
                    f32x4 v{};
#pragma unroll
                    for (int w = 0; w < SPLIT; ++w) {
                        const f32x4 u = of(w)[x * 64 + lane];
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = fmaf(each[w][0], u[e], v[e]);
                    }
                    leave(M * (x / (NR / 4)) + 4 * H * (x % (NR / 4)) + 4 * h, v, inv);
                }
            } else {
                const float inv = any ? 1.0f / l : 0.0f;   // (all scores minus infinity: 0 times infinity)
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int g = 0; g < NR / 4; ++g)
                        leave(M * t + 4 * H * g + 4 * h, f32x4{o[t][4 * g], o[t][4 * g + 1], o[t][4 * g + 2], o[t][4 * g + 3]}, inv);
            }
            // ...and behind a part's sums the maxima and sums of weights.
            if (there && !direct && h == 0 && own == 0)
                ((float2 *)(part + groups * b.rows))[at] = float2{m, any && m == -INFINITY && l == 0.0f ? 1.0f : l};
        }
        if constexpr (!PAGED) {
            more = false;
        } else {
            if (begun && tid == 0) parts.marks[unit_id] = SelfMark{1, ends, b.q0, b.kv, b.row0, b.rows, {0, 0}};
            // On to the next block.
            if (last_here) {
                more = false;
            } else {
                at.tile = 0;
                if (++at.block == blocks_of(seq, a.share, ROWS)) {
                    at.block = 0;
                    at.seq = with_rows(c, at.seq + 1);
                }
                more = at.seq < c.seqs && !(at == end);
            }
        }
    }
}

// The parts of blocks that were cut: a lane four columns of a row, of every
// part, or, where there are many, a few lanes, each of some of them.
template <typename T> __global__ void __launch_bounds__(256) self_join(SelfArgs a, SelfParts parts) {
    const int lane = threadIdx.x & 63, d = a.c.width, kv = a.c.kv;
    int x, head;
    parts.whose(blockIdx.x, kv, x, head);
    if (x >= parts.pieces) return;
    const SelfMark mark = parts.marks[x * kv + head];
    if (!(mark.front && mark.done)) return;
    // The pieces before it that lie inside of the block, and the one that began it.
    int inside = 0;
    for (int g = x - 1;; g -= 64) {
        const SelfMark *before = parts.marks + (g - lane) * kv + head;
        const bool in = g - lane >= 0 && before->front && !before->done;
        const uint64_t not_in = ~__ballot(in);
        if (not_in) {
            inside += __ffsll((unsigned long long)not_in) - 1;
            break;
        }
        inside += 64;
    }
    const int n = inside + 2, first = x - inside - 1;
    const auto part = [&](int p) { return (const f32x4 *)parts.part(2 * ((first + p) * kv + head) + (p == 0)); };
    const int groups = (d + 3) / 4, rows = mark.rows;
    constexpr int AT = 8;     // parts on their way at a time
    int lanes = 1;            // of four columns: an eighth of the parts, up to 16
    while (lanes < 16 && lanes * AT < n) lanes *= 2;
    const int items = 64 / lanes, sub = lane / items;
    const int waves = (rows * groups + items - 1) / items;
    for (int w = blockIdx.y * 4 + (threadIdx.x >> 6); w < waves; w += gridDim.y * 4) {
        const int item = w * items + lane % items, i = min(item / groups, rows - 1), col = item % groups;
        float m = -INFINITY, l = 0.0f;
        f32x4 o{};
        for (int p0 = sub; p0 < n; p0 += AT * lanes) {
            float2 q[AT];
            f32x4 v[AT];
            float top = m;
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                q[k] = float2{-INFINITY, 0.0f}, v[k] = f32x4{};
                const int p = p0 + k * lanes;
                if (p < n) q[k] = ((const float2 *)(part(p) + groups * rows))[i], v[k] = part(p)[col * rows + i];
            }
#pragma unroll
            for (int k = 0; k < AT; ++k) top = fmaxf(top, q[k].x);
            // (Equal: both infinite, of one sign.)
            const float f = __builtin_amdgcn_exp2f(m == top ? 0.0f : m - top);
            l *= f, o *= f, m = top;
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                const float wk = __builtin_amdgcn_exp2f(q[k].x == m ? 0.0f : q[k].x - m);
                l = fmaf(wk, q[k].y, l);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fmaf(wk, v[k][e], o[e]);
            }
        }
        for (int s = items; s < 64; s *= 2) {   // the lanes of the same columns
            const float m2 = __shfl_xor(m, s, 64), l2 = __shfl_xor(l, s, 64), top = fmaxf(m, m2);
            const float f = __builtin_amdgcn_exp2f(m == top ? 0.0f : m - top), f2 = __builtin_amdgcn_exp2f(m2 == top ? 0.0f : m2 - top);
            l = fmaf(f, l, f2 * l2);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(f, o[e], f2 * __shfl_xor(o[e], s, 64));
            m = top;
        }
        if (sub != 0 || item >= rows * groups) continue;
        // No maximum: no state (0), or scores of minus infinity alone.
        const float inv = m == -INFINITY ? (l == 0.0f ? 0.0f : __builtin_nanf("")) : 1.0f / l;
        const int row = mark.row0 + i;
        T *out = (T *)a.out + ((uint64_t)mark.q0 + row / a.share) * a.os[0] +
                 ((uint64_t)mark.kv * a.share + row % a.share) * a.os[1];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * col + e < d) out[4 * col + e] = from_f32<T>(o[e] * inv);
    }
}

// ---- launches --------------------------------------------------------------------------

template <typename T, Held HELD, bool PAGED, int DP, int WAVES, int M = 32, int SPLIT = 1>
static hipError_t launch_tiles(hipStream_t s, const SelfArgs &a, const SelfLaunch &f) {
    using C = SelfTile<T, HELD, DP, WAVES, M, SPLIT>;
    SelfParts parts{};
    uint32_t groups = f.groups;
    if (PAGED) {
        parts.pieces = std::min(f.pieces, std::max(1, C::GROUPS / a.c.kv));
        groups = (uint32_t)(parts.pieces + 7) / 8 * 8 * a.c.kv;
        parts.marks = (SelfMark *)a.ws;
        parts.parts = (float *)(parts.marks + (uint64_t)parts.pieces * a.c.kv);
        parts.pitch = self_part_floats(f.part_rows, a.c.width);
        parts.least = (uint64_t)a.share * 4 * C::KB;
    }
    const hipError_t e = enqueue(self_tiles<T, HELD, PAGED, DP, WAVES, M, SPLIT>, dim3(groups), dim3(64 * WAVES * SPLIT),
                                 C::LDS, s, a, parts);
    // (Blocks of one tile are not cut.)
    if (e != hipSuccess || !PAGED || room(a.c) <= C::KB) return e;
    return enqueue(self_join<T>, dim3(groups, f.part_rows <= 16 ? 2 : (f.part_rows * DP / 4 + 511) / 512), dim3(256), 0, s, a, parts);
}

template <typename T, bool PAGED, int DP> static hipError_t launch_held(hipStream_t s, const SelfArgs &a, const SelfLaunch &f) {
    constexpr bool F32 = std::is_same<T, float>::value;
    // (Blocks of 16 rows: 16-bit tokens over a cache.)
    if constexpr (PAGED && !F32) {
        if (f.rows == 16)
            return f.held == Held::Bytes    ? launch_tiles<T, Held::Bytes, true, DP, 1, 16>(s, a, f)
                   : f.held == Held::Chunks ? launch_tiles<T, Held::Chunks, true, DP, 1, 16>(s, a, f)
                                            : hipErrorInvalidValue;
        if (f.held == Held::Bytes) return launch_tiles<T, Held::Bytes, true, DP, 1>(s, a, f);
    }
    if constexpr (PAGED)
        if (f.held == Held::Codes)
            return f.rows == 32 ? launch_tiles<T, Held::Codes, true, DP, 1>(s, a, f)
                                : launch_tiles<T, Held::Codes, true, DP, 4>(s, a, f);
    if (f.held == Held::Loose) return launch_tiles<T, Held::Loose, PAGED, DP, 1>(s, a, f);
    // (A wave alone has F32 prompts and a cache's tokens, four share the rows of
    // prompts alone, or, but for F32 prompts, a tile.)
    if constexpr (!PAGED)
        if (f.split) return launch_tiles<T, Held::Chunks, false, DP, 1, 32, 4>(s, a, f);
    if constexpr (PAGED || F32)
        if (f.rows == 32) return launch_tiles<T, Held::Chunks, PAGED, DP, 1>(s, a, f);
    if constexpr (PAGED || !F32) return launch_tiles<T, Held::Chunks, PAGED, DP, 4>(s, a, f);
    return hipErrorInvalidValue;
}

template <typename T> static hipError_t launch_self(hipStream_t s, const SelfArgs &a, const SelfLaunch &f) {
    const auto go = [&](auto paged) {
        constexpr bool PAGED = decltype(paged)::value;
        if (a.c.width <= 32) return launch_held<T, PAGED, 32>(s, a, f);
        if (a.c.width <= 64) return launch_held<T, PAGED, 64>(s, a, f);
        if (a.c.width <= 96) return launch_held<T, PAGED, 96>(s, a, f);
        return launch_held<T, PAGED, 128>(s, a, f);
    };
    return a.c.paged ? go(std::true_type()) : go(std::false_type());
}

}  // namespace rocm
