// States in the pages of a cache, and the sequences that own them: how the
// kernels of cache_rows.hip and self_tiles.h find a token's sequence,
// its position and a position's slot. What the arrays hold is the caller's
// and may be anything: whatever they hold, no index leaves its array.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace rocm {

// Strides are in elements. Without pages position p of sequence i is row
// starts[i] + p of k and v, and its length its rows.
struct CacheArgs {
    void *k, *v;
    float *k_scales, *v_scales;             // with int8 states
    uint64_t ks[2], vs[2];                  // of slots and heads
    uint64_t kss, vss;                      // of the scales' slots
    const int32_t *starts, *lengths, *pages;
    uint64_t page_row;                      // of a sequence's pages
    int seqs, columns, page_tokens, page_count;
    int tokens;                             // rows of the call
    int kv, width;
    bool paged;
};

// A sequence's rows of the call, and the states it has with them.
struct Seq {
    int row0, rows, length;
    __host__ __device__ int first() const { return length - rows; }   // the first row's position; below 0: no state
};

inline __host__ __device__ int within(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Sequence i of the call: rows outside of 0 .. tokens are nobody's.
inline __host__ __device__ Seq seq_of(const CacheArgs &a, int i) {
    Seq s;
    s.row0 = within(a.starts[i], 0, a.tokens);
    s.rows = within(a.starts[i + 1], s.row0, a.tokens) - s.row0;
    s.length = a.paged ? (a.lengths[i] < 0 ? 0 : a.lengths[i]) : s.rows;
    return s;
}

// Positions that a sequence's pages have room for.
inline __host__ __device__ int room(const CacheArgs &a) {
    const uint64_t n = (uint64_t)a.columns * a.page_tokens;
    return n > INT32_MAX ? INT32_MAX : (int)n;
}

// The slot of sequence i's position p (0 or more), or -1: past the table, or
// on a page that the cache does not have.
inline __host__ __device__ int slot_of(const CacheArgs &a, int i, int p) {
    const uint32_t column = (uint32_t)p / (uint32_t)a.page_tokens;
    if (column >= (uint32_t)a.columns) return -1;
    const int32_t page = a.pages[(uint64_t)i * a.page_row + column];
    if ((uint32_t)page >= (uint32_t)a.page_count) return -1;
    return page * a.page_tokens + (int)((uint32_t)p - column * (uint32_t)a.page_tokens);
}

hipError_t cache_write(hipStream_t s, const CacheArgs &a, Dt rows, bool i8, const void *k, const void *v,
                       const uint64_t (&ks)[2], const uint64_t (&vs)[2]);
hipError_t cache_read(hipStream_t s, const CacheArgs &a, Dt rows, bool i8, void *k, void *v, const uint64_t (&ks)[2],
                      const uint64_t (&vs)[2]);

// Attention of the call's rows to their sequences' states, up to their own.
struct SelfArgs {
    CacheArgs c;
    const void *q;
    void *out;
    uint64_t qs[2], os[2];   // strides of tokens and heads
    float *ws;
    Dt dt;
    bool i8;
    int share;               // query heads that read one key head
    int window;              // states that a row sees, its own last (INT32_MAX: all)
    float scale;             // of a score, times log2(e); positive...
    float turn;              // ...with 1, -1 or 0 times q
};

// How keys and values reach LDS: in aligned whole chunks, by themselves;
// through registers, at any alignment; int8 states as numbers, through
// registers; or as they are, in aligned whole chunks, by themselves.
enum class Held : int { Chunks, Loose, Codes, Bytes };

// How a call is launched, from what the host knows of it: its rows and
// sequences, not their lengths.
constexpr int MOST_COUNTED = 2048;   // sequences of a prompt whose blocks are ordered
constexpr int MOST_ALONE = 256 * 12, MOST_TILED = 256 * 3;   // workgroups of a call over a cache, of a wave and of four
struct SelfLaunch {
    Held held;
    int rows;            // of a block: 16 or 32 (a wave's), or 128 (four waves')
    bool split;          // 32 rows are four waves', each with every fourth tile of the keys
    uint32_t groups;     // of a prompt: workgroups, the most blocks that there can be
    int pieces;          // of a call over a cache, at most, each a workgroup of every key head
    int part_rows;       // the most rows of a part
};
SelfLaunch self_plan(const SelfArgs &a);
// The bytes of workspace that calls of up to so many tokens and sequences need.
uint64_t self_workspace(uint64_t tokens, uint64_t seqs, int heads, int kv, int width);
hipError_t self_attention(hipStream_t s, const SelfArgs &a, const SelfLaunch &f);
hipError_t self_f32(hipStream_t s, const SelfArgs &a, const SelfLaunch &f);
hipError_t self_f16(hipStream_t s, const SelfArgs &a, const SelfLaunch &f);
hipError_t self_bf16(hipStream_t s, const SelfArgs &a, const SelfLaunch &f);

// A block whose tiles are cut over workgroups: each leaves a part, and says so
// here. front: it starts inside of a block; done: it ends that block.
struct SelfMark {
    int front, done;
    int q0, kv, row0, rows;
    int pad[2];
};
// A part's floats, of up to `rows` rows: their sums, four columns of every row
// after another, then each row's maximum (base 2) and sum of weights; a row
// without a finite maximum leaves 1 for that sum if it had a state.
inline __host__ __device__ uint64_t self_part_floats(int rows, int width) {
    return ((uint64_t)rows * ((width + 3) / 4 * 4 + 2) + 3) / 4 * 4;
}

}  // namespace rocm
