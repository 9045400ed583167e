// The int8 product on the caller's codes and scales: out[m, n] =
// (sum_k a[m, k] w[n, k]) as[m] ws[n] + bias[n].
//
// The sum is whole, so how it is cut over waves and steps changes nothing, and
// an inner width that no vector divides costs no copy: the inner width is read
// in 16-byte chunks, the last of them ending at the row's end and so
// overlapping the one before; a's bytes that were already counted there are
// taken as 0 (and all of them in chunks past the end), w's are left as they
// are. Rows past M or N repeat the last.
//
// Every kernel multiplies w by a transposed, so that a lane holds four
// consecutive columns of one output row.
#include <hip/hip_runtime.h>

#include <cmath>

#include "devmath.h"
#include "launch.h"
#include "operators.h"

namespace rocm {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int loose4 __attribute__((ext_vector_type(4), aligned(1)));

// An output from its exact sum: both scales and the bias in F32 (the sum's
// conversion and its product with a's scale round, then the rest once).
__device__ __forceinline__ float scaled(int sum, float as, float ws, float bias) {
    return fmaf((float)sum * as, ws, bias);
}

__device__ __forceinline__ void put(void *out, Dt t, uint64_t at, float v) {
    if (t == Dt::F32) ((float *)out)[at] = v;
    else if (t == Dt::F16) ((_Float16 *)out)[at] = (_Float16)v;
    else ((__bf16 *)out)[at] = (__bf16)v;
}

// The bytes of a's 16-byte chunk c that count, of an inner width k >= 16.
__device__ __forceinline__ i32x4 counted(i32x4 v, int c, int k) {
    const int z = 16 * c - (k - 16);   // bytes from the front that do not
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int zi = z - 4 * i;
        v[i] = zi <= 0 ? v[i] : zi >= 4 ? 0 : v[i] & (int)(0xffffffffu << (8 * zi));
    }
    return v;
}

// ---- Inner widths below 16: an output a lane, its products one by one ------------

__global__ void __launch_bounds__(256) linear_i8_narrow(LinearArgs a) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < (uint64_t)a.m * a.n; i += (uint64_t)gridDim.x * 256) {
        const uint64_t m = i / a.n, n = i % a.n;
        int sum = 0;
        for (int k = 0; k < a.k; ++k) sum += (int)a.a[m * a.lda + k] * a.w[n * a.ldw + k];
        put(a.out, a.ot, m * a.ldo + n, scaled(sum, a.as[m], a.ws[n], a.bias ? a.bias[n] : 0.0f));
    }
}

// ---- Few rows: 16 columns a workgroup, its waves cutting the inner width ---------
//
// Bound by w's bytes, each read once, straight into the matrix instruction's
// registers: a lane 16 bytes of a column's row, four lanes 64 consecutive ones.
// The waves' sums meet in LDS. One row by 4096 x 4096 takes 5.7 us (2.9 TB/s,
// a launch's start and end among it), 48 rows by 1024 x 4096 7.0.
template <int WAVES, int MT> __global__ void __launch_bounds__(64 * WAVES) linear_i8_rows(LinearArgs a, uint64_t blocks) {
    __shared__ __attribute__((aligned(16))) i32x4 part[WAVES][MT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, h = lane >> 4;
    const int chunks = (a.k + 15) / 16, full = a.k / 16;
    const uint32_t tiles = (a.n - 1) / 16 + 1;
    for (uint64_t i = blockIdx.x; i < blocks; i += gridDim.x) {
        const int tile = (int)(i % tiles), m0 = (int)(i / tiles) * 16 * MT;
        const int8_t *ap[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) ap[t] = a.a + (uint64_t)min(m0 + 16 * t + r, a.m - 1) * a.lda;
        const int8_t *wp = a.w + (uint64_t)min(16 * tile + r, a.n - 1) * a.ldw;
        i32x4 acc[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = i32x4{0, 0, 0, 0};
        // A step is 8 chunks of each row (128 bytes), two products; the next
        // step's reads go out before this one's products.
        struct Step {
            i32x4 w[2], x[2][MT];
        };
        const auto read = [&](Step &f, int c0) {
            if (c0 >= chunks) return;   // uniform
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int k = min(16 * (c0 + 4 * u + h), a.k - 16);
                f.w[u] = *(const loose4 *)(wp + k);
#pragma unroll
                for (int t = 0; t < MT; ++t) f.x[u][t] = *(const loose4 *)(ap[t] + k);
            }
        };
        const auto multiply = [&](Step &f, int c0) {
            if (c0 >= chunks) return;
            if (c0 + 8 > full)
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int t = 0; t < MT; ++t) f.x[u][t] = counted(f.x[u][t], c0 + 4 * u + h, a.k);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[u], f.x[u][t], acc[t], 0, 0, 0);
        };
        Step f0, f1;
        constexpr int STEP = 8 * WAVES;
        read(f0, 8 * wave);
        for (int c0 = 8 * wave; c0 < chunks; c0 += 2 * STEP) {
            read(f1, c0 + STEP);
            multiply(f0, c0);
            read(f0, c0 + 2 * STEP);
            multiply(f1, c0 + STEP);
        }
        if (i != blockIdx.x) __syncthreads();   // the last block's sums are read
#pragma unroll
        for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
        __syncthreads();
        for (int e = tid; e < 64 * MT; e += 64 * WAVES) {
            const int t = e >> 6, l = e & 63;
            i32x4 s = part[0][t][l];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) s += part[w][t][l];
            // Columns 4 (l / 16) .. + 3 of row l % 16.
            const int m = m0 + 16 * t + (l & 15), n = 16 * tile + 4 * (l >> 4);
            if (m >= a.m) continue;
            const float as = a.as[m];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < a.n)
                    put(a.out, a.ot, (uint64_t)m * a.ldo + n + j,
                        scaled(s[j], as, a.ws[n + j], a.bias ? a.bias[n + j] : 0.0f));
        }
    }
}

// ---- Tiles: both operands through LDS ----------------------------------------------
//
// BM rows of a by BN of w a workgroup, WM x WN waves, 128 bytes of the inner
// width a stage, two stages: the next one is on its way while one is computed.
// (Three and four stages were no faster: a compute unit reads some 20 to 27
// bytes a clock, and the stages wait for that. A 256 x 256 tile asks for 32;
// on random operands the chip's power holds the clock at 1.9 GHz besides:
// 32768 x 4096 x 4096 takes 537 us (2.05 POP/s), 436 on zeros.)
// LDS rows are 128 bytes, chunk c of row r at place c ^ (r / 2 % 8), so that
// the 16 rows of a read's pass (256 bytes, two rows a bank round) lie in
// different banks. DIRECT (16-byte aligned operands and strides, K a multiple
// of 16): memory to LDS without registers; without it 1111 x 1001 x 1537 takes
// 13.7 us, 8.1 at K = 1536.
template <int BM, int BN, int WM, int WN, bool DIRECT>
__global__ void __launch_bounds__(64 * WM * WN) linear_i8_tiles(LinearArgs a, int grid_n) {
    constexpr int WAVES = WM * WN, ROWS = BM + BN, STAGE = ROWS * 128;
    constexpr int TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int LOADS = ROWS / 8 / WAVES;   // a wave's, 8 rows each
    static_assert(LOADS * 8 * WAVES == ROWS, "whole loads a wave");
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    // XCD-aware numbering: workgroups go to the 8 XCDs in turn, and each XCD
    // takes tiles that follow one another.
    const int per = gridDim.x / 8;
    int b = blockIdx.x;
    if (b < per * 8) b = (b % 8) * per + b / 8;
    // GROUP rows of tiles at a time, column by column: the tiles at work in an
    // XCD share more of a and w than a row of them would.
    constexpr int GROUP = 4;
    const int grid_m = gridDim.x / grid_n, g0 = b / (GROUP * grid_n) * GROUP, gm = min(GROUP, grid_m - g0);
    const int in = b - g0 * grid_n;
    const int m0 = (g0 + in % gm) * BM, n0 = in / gm * BN;

    // This lane's place in each load: row (of a, then of w) and chunk.
    const int8_t *src[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const int row = (wave * LOADS + j) * 8 + (lane >> 3);
        src[j] = row < BM ? a.a + (uint64_t)min(m0 + row, a.m - 1) * a.lda
                          : a.w + (uint64_t)min(n0 + row - BM, a.n - 1) * a.ldw;
    }
    // (Half the row's number: 4 for every other load, and lane / 16.)
    static_assert(LOADS % 2 == 0, "a load's parity is its number's");
    const int chunk[2] = {(lane & 7) ^ (lane >> 4), (lane & 7) ^ (4 + (lane >> 4))};
    i32x4 held[DIRECT ? 1 : LOADS];
    auto load = [&](int stage) {
        const int at[2] = {min(128 * stage + 16 * chunk[0], a.k - 16), min(128 * stage + 16 * chunk[1], a.k - 16)};
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int k = at[j & 1];
            if constexpr (DIRECT) {
                char *dst = smem + stage % 2 * STAGE + (wave * LOADS + j) * 1024;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src[j] + k),
                                                 (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
            } else {
                held[j] = *(const loose4 *)(src[j] + k);
            }
        }
    };
    const int stages = (a.k + 127) / 128, r = lane & 31, h = lane >> 5;
    // A stage's loads are over and in LDS, and every wave is done with the
    // stage before; where the inner width ends in it, a's bytes that do not
    // count are 0.
    auto arrive = [&](int stage) {
        char *at = smem + stage % 2 * STAGE + wave * LOADS * 1024 + lane * 16;
        const bool tail = 128 * (stage + 1) > a.k;   // uniform
        if constexpr (DIRECT) __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const bool rows = (wave * LOADS + j) * 8 < BM;   // (uniform: of a)
            if constexpr (DIRECT) {
                if (tail && rows) *(i32x4 *)(at + j * 1024) = counted(*(i32x4 *)(at + j * 1024), 8 * stage + chunk[j & 1], a.k);
            } else {
                *(i32x4 *)(at + j * 1024) = tail && rows ? counted(held[j], 8 * stage + chunk[j & 1], a.k) : held[j];
            }
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): this wave's reads and writes of LDS
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    // What the epilogue multiplies by, read now: this lane's rows' scales, and
    // columns 64 i + lane of the wave's.
    constexpr int COLS = BN / WN, PITCH = COLS * 4 + 16;   // bytes of a staged row, F32's
    static_assert(WAVES * (32 * PITCH + 8 * COLS) <= 2 * STAGE, "staging fits the stages");
    const int nw = n0 + wn * COLS, mw = m0 + wm * (BM / WM);
    float ascale[TM], wscale[(COLS + 63) / 64], wbias[(COLS + 63) / 64];
#pragma unroll
    for (int j = 0; j < TM; ++j) ascale[j] = a.as[min(mw + 32 * j + r, a.m - 1)];
#pragma unroll
    for (int i = 0; i < (COLS + 63) / 64; ++i) {
        const int n = min(nw + 64 * i + lane, a.n - 1);
        wscale[i] = a.ws[n], wbias[i] = a.bias ? a.bias[n] : 0.0f;
    }
    i32x16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = i32x16{};
    // A quarter of a stage (32 bytes of the inner width) as the matrix
    // instruction takes it, read while the quarter before is multiplied.
    struct Quarter {
        i32x4 x[TM], w[TN];
    };
    const auto read = [&](Quarter &f, int stage, int ks) {
        const char *A = smem + stage % 2 * STAGE + wm * (BM / WM) * 128,
                   *W = smem + stage % 2 * STAGE + (BM + wn * (BN / WN)) * 128;
        const int at = r * 128 + (((2 * ks + h) ^ (r >> 1 & 7)) * 16);
        // lgkmcnt(0): the quarter read before the last products; so the next
        // ones wait for it alone, not for this one.
        __builtin_amdgcn_s_waitcnt(0xc07f);
#pragma unroll
        for (int i = 0; i < TN; ++i) f.w[i] = *(const i32x4 *)(W + i * 4096 + at);
#pragma unroll
        for (int j = 0; j < TM; ++j) f.x[j] = *(const i32x4 *)(A + j * 4096 + at);
    };
    const auto multiply = [&](const Quarter &f) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    Quarter f0, f1;
    load(0);
    arrive(0);
    if (stages > 1) load(1);
    read(f0, 0, 0);
    for (int s = 0; s + 1 < stages; ++s) {
        read(f1, s, 1);
        multiply(f0);
        read(f0, s, 2);
        multiply(f1);
        read(f1, s, 3);
        multiply(f0);
        arrive(s + 1);
        if (s + 2 < stages) load(s + 2);
        read(f0, s + 1, 0);
        multiply(f1);
    }
    read(f1, stages - 1, 1);
    multiply(f0);
    read(f0, stages - 1, 2);
    multiply(f1);
    read(f1, stages - 1, 3);
    multiply(f0);
    multiply(f1);

    // Epilogue: a lane's row is m = lane % 32, its columns 8 g + 4 h .. + 3 of
    // each tile. Staged through LDS 32 rows at a time in the output's type, so
    // that a store writes a row's columns one after another.
    __syncthreads();
    char *mine = smem + wave * (32 * PITCH + 8 * COLS);
    float *cols = (float *)(mine + 32 * PITCH);   // the wave's columns' scales, then their biases
#pragma unroll
    for (int i = 0; i < (COLS + 63) / 64; ++i)
        if (COLS >= 64 || lane < COLS) cols[64 * i + lane] = wscale[i], cols[COLS + 64 * i + lane] = wbias[i];
    const auto finish = [&](auto zero) {
        typedef decltype(zero) O;
        typedef O out4 __attribute__((ext_vector_type(4)));
        constexpr int PER = 16 / sizeof(O), LANES = COLS / PER;   // a store's columns, a row's stores
#pragma unroll
        for (int j = 0; j < TM; ++j) {
#pragma unroll
            for (int i = 0; i < TN; ++i) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int c = 32 * i + 8 * g + 4 * h;
                    const f32x4 ws = *(const f32x4 *)(cols + c), bias = *(const f32x4 *)(cols + COLS + c);
                    out4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[e] = from_f32<O>(scaled(acc[i][j][4 * g + e], ascale[j], ws[e], bias[e]));
                    *(out4 *)(mine + r * PITCH + c * sizeof(O)) = y;
                }
                __builtin_amdgcn_sched_barrier(0);   // (one tile's sums out of the accumulators at a time)
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0): the wave's rows are in LDS
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 32 * LANES / 64; ++q) {
                const int at = 64 * q + lane, row = at / LANES, c = at % LANES * PER;
                const int m = mw + 32 * j + row, n = nw + c;
                const i32x4 v = *(const i32x4 *)(mine + row * PITCH + c * sizeof(O));
                if (m >= a.m || n >= a.n) continue;
                O *o = (O *)a.out + (uint64_t)m * a.ldo + n;
                if (n + PER <= a.n) {
                    *(loose4 *)o = v;
                } else {
#pragma unroll
                    for (int e = 0; e < PER - 1; ++e)
                        if (n + e < a.n) o[e] = *(const O *)(mine + row * PITCH + (c + e) * sizeof(O));
                }
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);   // read before the next rows overwrite them
            __builtin_amdgcn_wave_barrier();
        }
    };
    if (a.ot == Dt::F32) finish(0.0f);
    else if (a.ot == Dt::F16) finish((_Float16)0.0f);
    else finish((__bf16)0.0f);
}

template <int BM, int BN, int WM, int WN> static hipError_t launch_tiles(hipStream_t s, const LinearArgs &a, bool direct) {
    const int gn = (a.n - 1) / BN + 1, gm = (a.m - 1) / BM + 1;
    const dim3 grid((uint32_t)gn * gm), block(64 * WM * WN);
    constexpr int lds = 2 * (BM + BN) * 128;
    if (direct) return enqueue(linear_i8_tiles<BM, BN, WM, WN, true>, grid, block, lds, s, a, gn);
    if constexpr (BM < 256) return enqueue(linear_i8_tiles<BM, BN, WM, WN, false>, grid, block, lds, s, a, gn);
    return hipErrorInvalidValue;
}

template <int MT> static hipError_t launch_rows(hipStream_t s, const LinearArgs &a) {
    constexpr int WAVES = 8;   // (4 to 16 take the same time within 5%)
    const uint64_t blocks = ((uint64_t)(a.n - 1) / 16 + 1) * ((a.m - 1) / (16 * MT) + 1);
    // (A launch holds less than 2^32 threads; past a bound workgroups take several blocks.)
    const dim3 grid((uint32_t)(blocks < (1 << 16) ? blocks : 1 << 16));
    return enqueue(linear_i8_rows<WAVES, MT>, grid, dim3(64 * WAVES), 0, s, a, blocks);
}

int linear_i8_kernel(int m, int n, int k, bool aligned) {
    // By the estimated time in us, fitted to 52 shapes of 1 to 30000 rows, N of
    // 100 to 30000 and K of 32 to 8192 (its choice is the fastest measured or
    // within 10% of it). What a compute unit reads sets the pace: 36 KB/us of
    // 16-row pieces and 0.4 us for each one's sums, or a stage of a tile in 0.25
    // to 1.75 us (64 x 64: 16 KB; 128 x 128: 32 KB, slower with every unit at
    // work; 256 x 256: 64 KB) and its start and end.
    // us measured, rows kernel / 64 / 128 / 256: 48 x 1024 x 4096 6.6, 11.3,
    // 23.7, 51; 256 x 1024 x 1024 6.1, 5.2, 10.0, 19; 2048 x 4096 x 1024 -,
    // 18.8, 16.2, 21.9; 6532 x 7168 x 64 312, 39, 42, 33.
    const double stages = (k + 127) / 128;
    const auto blocks = [&](double bm, double bn) { return std::ceil(m / bm) * std::ceil(n / bn); };
    const auto rounds = [](double n) { return std::ceil(n / 256); };
    double least = INFINITY;
    int best = 0;
    const auto offer = [&](int which, double time) {
        if (time < least) least = time, best = which;
    };
    for (int mt = 1; mt <= 4; ++mt)
        if (m > 16 * (mt - 1)) {
            const double n = blocks(16.0 * mt, 16);
            offer(mt, rounds(n) * k * (1 + mt) * 16 / 36000 + n / 256 * mt * 0.4);
        }
    offer(64, std::fmax(1, blocks(64, 64) / 256) * (stages * 0.25 + 0.8));
    const double n128 = blocks(128, 128);
    offer(128, rounds(n128) * (stages * (n128 < 256 ? 0.63 : 0.83) + 4));
    if (aligned) offer(256, rounds(blocks(256, 256)) * (stages * 1.75 + 8));   // (no registers to hold a stage)
    return best;
}

hipError_t linear_i8(hipStream_t s, const LinearArgs &a) {
    if (a.m <= 0 || a.n <= 0) return hipSuccess;
    if (a.k < 16) {
        const uint64_t blocks = ((uint64_t)a.m * a.n + 255) / 256;
        return enqueue(linear_i8_narrow, dim3((uint32_t)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, s, a);
    }
    // A launch holds less than 2^32 threads: a product of more than 2^22 of the
    // smallest tiles goes by halves.
    if (((uint64_t)(a.m - 1) / 64 + 1) * ((a.n - 1) / 64 + 1) > 1 << 22) {
        LinearArgs first = a, second = a;
        const uint64_t size = dt_bytes(a.ot);
        if (a.m >= a.n) {
            first.m = (a.m / 2 + 255) / 256 * 256, second.m = a.m - first.m;
            second.a += first.m * a.lda, second.as += first.m;
            second.out = (char *)a.out + first.m * a.ldo * size;
        } else {
            first.n = (a.n / 2 + 255) / 256 * 256, second.n = a.n - first.n;
            second.w += first.n * a.ldw, second.ws += first.n;
            if (a.bias) second.bias += first.n;
            second.out = (char *)a.out + first.n * size;
        }
        const hipError_t e = linear_i8(s, first);
        return e != hipSuccess ? e : linear_i8(s, second);
    }
    const auto whole = [](const void *p, uint64_t ld) { return (reinterpret_cast<uintptr_t>(p) | ld) % 16 == 0; };
    const bool direct = whole(a.a, a.lda) && whole(a.w, a.ldw) && a.k % 16 == 0;
    switch (linear_i8_kernel(a.m, a.n, a.k, direct)) {
    case 1: return launch_rows<1>(s, a);
    case 2: return launch_rows<2>(s, a);
    case 3: return launch_rows<3>(s, a);
    case 4: return launch_rows<4>(s, a);
    case 64: return launch_tiles<64, 64, 2, 2>(s, a, direct);
    case 128: return launch_tiles<128, 128, 2, 2>(s, a, direct);
    default: return launch_tiles<256, 256, 2, 4>(s, a, direct);
    }
}

}  // namespace rocm
