// How attention of a call's own tokens is launched (its kernels: self_tiles.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "array_checks.h"
#include "cache.h"

namespace rocm {

namespace {

constexpr uint64_t MOST_THREADS = 1ull << 31;   // of a launch

// The most pieces of a call over a cache, by its blocks' rows.
uint64_t most_pieces(int rows, int kv) {
    return std::max<uint64_t>(1, (rows == 128 ? MOST_TILED : MOST_ALONE) / kv);
}

uint64_t parts_bytes(int rows, uint64_t all_rows, int kv, int width) {
    return most_pieces(rows, kv) * kv *
           (sizeof(SelfMark) + 2 * 4 * self_part_floats((int)std::min<uint64_t>(rows, all_rows), width));
}

}  // namespace

SelfLaunch self_plan(const SelfArgs &a) {
    SelfLaunch f{};
    const uint64_t tokens = a.c.tokens, rows = tokens * a.share;   // (of a key head)
    const uint64_t seqs = std::min<uint64_t>(a.c.seqs, tokens), size = a.i8 ? 1 : dt_bytes(a.dt);
    const auto whole = [&](const void *p, const uint64_t (&stride)[2]) {
        return (reinterpret_cast<uintptr_t>(p) | stride[0] * size | stride[1] * size) % 16 == 0;
    };
    // (Keys and values in aligned whole chunks, a tile of them within 31 bits.)
    const bool chunks = a.c.width * size % 16 == 0 && whole(a.c.k, a.c.ks) && whole(a.c.v, a.c.vs) &&
                        std::max(a.c.ks[0], a.c.vs[0]) < (1u << 31) / 64 / 4;
    f.held = a.i8 ? Held::Codes : chunks ? Held::Chunks : Held::Loose;
    const bool f32 = a.dt == Dt::F32;
    f.rows = 32;
    if (f.held == Held::Chunks && !a.c.paged) {
        // Prompts: blocks of 128 rows, where there are enough of them for every
        // compute unit; else four waves a block of 32. F32, whose products take long:
        // a wave a block of 32, if those are enough. us of 12 heads of 64, by how many
        // blocks there are of that size:
        //   F32, waves of 32 rows, and four of 32    2184  20 x 20-500 tokens    63   74
        //                                            1752  16 x 20-500           59   60
        //                                             984  8 x 100-500           54   38
        //                                            1128  3000                 262  148
        //   BF16, four of 128, and four of 32         636  16 x 100-500          21   32
        //                                             516  5400                 101  116
        //                                             384  4000                  78   74
        //                                             192  2000                  43   30
        // (Not in order: a long sequence's last blocks run alone. 6000 F32 tokens, of
        // 2256 blocks, would take 486 for 650, 12 x 100-500 BF16, of 480, 21 for 25.)
        if (!f32 && a.c.kv * (rows / 128 + seqs) >= 512 && rows > 32 * seqs) f.rows = 128;
        else f.split = !f32 || a.c.kv * (rows / 32 + seqs) < 2048;
    } else if (f.held != Held::Loose && rows > 32 * seqs) {
        f.rows = 128;
    }
    // A wave alone makes numbers of codes as it reads them, four of them once.
    // (F32's slow products leave it no need to.)
    if (a.i8 && f.rows == 32 && chunks && !f32) f.held = Held::Bytes;
    // Tokens of few heads: blocks of 16 rows.
    if (a.c.paged && !f32 && rows <= 16 * seqs && (f.held == Held::Bytes || f.held == Held::Chunks)) f.rows = 16;
    // At most. (Of many sequences, an empty one has a place too.)
    const uint64_t blocks = a.c.kv * (rows / f.rows + (!a.c.paged && a.c.seqs > MOST_COUNTED ? a.c.seqs : seqs));
    if (!a.c.paged) {
        if (blocks * (f.rows == 128 || f.split ? 256 : 64) > MOST_THREADS)
            fail(TURBO_E_CAPACITY, "rocm: a prompt of " + std::to_string(blocks) + " workgroups");
        f.groups = (uint32_t)blocks;
        return f;
    }
    // (No more than there can be tiles.)
    const uint64_t tiles = blocks / a.c.kv * std::max<uint64_t>(1, ((uint64_t)room(a.c) + 31) / 32);
    f.pieces = (int)std::min<uint64_t>(most_pieces(f.rows, a.c.kv), std::max<uint64_t>(1, tiles));
    // (Eight pieces of each key head at least, of 256 threads where they are joined.)
    if ((uint64_t)(f.pieces + 7) / 8 * 8 * a.c.kv * 256 > MOST_THREADS)
        fail(TURBO_E_CAPACITY, "rocm: cache attention of " + std::to_string(a.c.kv) + " key heads");
    // (The device adds up the blocks' costs in 64 bits and shares them out in F64: a
    // piece's has to stay below 2^52, 2^48 for these, of which a kernel may run a
    // sixteenth.)
    const u128 cost = (u128)(blocks / a.c.kv) * ((u128)a.share * ((uint64_t)room(a.c) + 96) + rows + 128);
    if (cost >> 48 >= (uint64_t)f.pieces)
        fail(TURBO_E_CAPACITY, "rocm: cache attention of " + std::to_string(a.share) + " heads to a key head over " +
                                   std::to_string(room(a.c)) + " positions");
    f.part_rows = (int)std::min<uint64_t>(f.rows, rows);
    return f;
}

uint64_t self_workspace(uint64_t tokens, uint64_t seqs, int heads, int kv, int width) {
    if (tokens == 0 || seqs == 0) return 0;
    const uint64_t rows = tokens * (heads / kv);
    return std::max(parts_bytes(32, rows, kv, width), parts_bytes(128, rows, kv, width));
}

hipError_t self_attention(hipStream_t s, const SelfArgs &a, const SelfLaunch &f) {
    if (a.c.tokens == 0 || a.c.seqs == 0) return hipSuccess;
    return a.dt == Dt::F32 ? self_f32(s, a, f) : a.dt == Dt::F16 ? self_f16(s, a, f) : self_bf16(s, a, f);
}

}  // namespace rocm
