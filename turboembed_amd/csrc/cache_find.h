// The sequence and the position of a call's token, on the device.
#pragma once

#include "cache.h"

namespace rocm {

// The last sequence that starts at or before token t (-1: none does), found by
// a wave, 64 sequences a step.
__device__ __forceinline__ int seq_before(const CacheArgs &a, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, count = a.seqs + 1, found = -1;
    while (count > 0) {
        const int step = (count + 63) / 64;
        const int at = lane * step;
        const int hits = __popcll(__ballot(at < count && a.starts[lo + at] <= t));
        if (hits == 0) break;
        found = lo + (hits - 1) * step;
        if (step == 1) break;
        count = min(step, count - (found - lo));
        lo = found;
    }
    return found;
}

// The position of token t of sequence i, from seq_before(t' <= t) on; i is
// moved to t's own sequence. Below 0: it has none, or no state.
__device__ __forceinline__ int position_of(const CacheArgs &a, int t, int &i) {
    // (Doubled steps: the sequences between two tokens may be many empty ones.)
    const auto past = [&](uint32_t n) { return n <= (uint32_t)(a.seqs - i) && a.starts[i + (int)n] <= t; };
    uint32_t step = 1;
    for (; past(step); step *= 2) i += (int)step;
    while ((step /= 2) > 0)
        if (past(step)) i += (int)step;
    if (i < 0 || i >= a.seqs) return -1;
    const Seq s = seq_of(a, i);
    return t < s.row0 ? -1 : s.first() + (t - s.row0);
}

}  // namespace rocm
