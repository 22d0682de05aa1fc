// Product of int8 codes with scales for each token and each channel.
//
//   y[t][n] = T( float(sum_k c[t][k] * w[n][k]) * (s[t] * u[n]) + b[n] )
//
// The sum is exact: 32-bit integers, and at most 2^17 - 1 products of at most 2^14.  The weight's rows go in as the matrix
// instruction's first operand and the codes' as its second, so that a lane ends with four neighbouring channels of one token.
#include "tde_int8_linear.h"

#include <type_traits>

namespace tde {
namespace block {

namespace {

template <class T>
__device__ __forceinline__ void store4(char *out, const float (&y)[4], int count, bool whole) {
    if (whole) {
        if constexpr (T::kBytes == 4)
            store_words<16>(out, Words<16>{{__builtin_bit_cast(uint32_t, y[0]), __builtin_bit_cast(uint32_t, y[1]),
                                            __builtin_bit_cast(uint32_t, y[2]), __builtin_bit_cast(uint32_t, y[3])}});
        else store_words<8>(out, Words<8>{{T::narrow(y[0], y[1]), T::narrow(y[2], y[3])}});
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < count) store_element<T>(out + i * T::kBytes, y[i]);
}

// 16 bytes of a row from byte k on; zeros beyond the row and for rows that do not exist.
__device__ __forceinline__ u32x4 load16(const int8_t *base, int64_t row, int64_t rows, int64_t k, int64_t length) {
    u32x4 v = {0, 0, 0, 0};
    if (row >= rows || k >= length) return v;
    const int8_t *p = base + row * length + k;
    if (k + 16 <= length) {
        typedef u32x4 __attribute__((aligned(1))) loose;
        return *(const __attribute__((address_space(1))) loose *)p;
    }
    const int left = (int)(length - k);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (i < left) v[i / 4] |= (uint32_t)(uint8_t)((const __attribute__((address_space(1))) int8_t *)p)[i] << (8 * (i % 4));
    return v;
}

// A wavefront's sums, scaled: WT tokens from t0 on, WN channels from n0 on.  INSIDE: all of them exist.
template <class T, int WT, int WN, bool INSIDE>
__device__ __forceinline__ void store_sums(const LinearArgs &a, const i32x16 (&acc)[WN / 32][WT / 32], int64_t t0, int64_t n0, int lane) {
    const bool biased = a.bias != nullptr;
    float s[WT / 32];
#pragma unroll
    for (int j = 0; j < WT / 32; ++j) {
        const int64_t t = t0 + j * 32 + (lane & 31);
        s[j] = INSIDE || t < a.tokens ? a.scales[t] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < WN / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int64_t n = n0 + i * 32 + g * 8 + (lane >> 5) * 4;
            const int count = INSIDE ? 4 : (int)(a.n - n < 4 ? a.n - n : 4);
            float u[4], b[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u[r] = INSIDE || r < count ? a.weight_scales[n + r] : 0.0f;
                b[r] = biased && (INSIDE || r < count) ? a.bias[n + r] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < WT / 32; ++j) {
                const int64_t t = t0 + j * 32 + (lane & 31);
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    y[r] = (float)acc[i][j][g * 4 + r] * (s[j] * u[r]);
                    if (biased) y[r] += b[r];
                }
                if (INSIDE || (t < a.tokens && count > 0)) store4<T>(a.out + (t * a.n + n) * T::kBytes, y, count, count >= 4);
            }
        }
}
template <class T, int WT, int WN>
__device__ __forceinline__ void store_tile(const LinearArgs &a, const i32x16 (&acc)[WN / 32][WT / 32], int64_t t0, int64_t n0, int lane) {
    if (t0 + WT <= a.tokens && n0 + WN <= a.n) store_sums<T, WT, WN, true>(a, acc, t0, n0, lane);
    else store_sums<T, WT, WN, false>(a, acc, t0, n0, lane);
}

// BT tokens x BN channels a workgroup, WT x WN of them a wavefront; 128 bytes of both operands' rows at a time, double-buffered.
template <class T, int BT, int BN, int WT, int WN>
__global__ void __launch_bounds__((BT / WT) * (BN / WN) * 64) linear_tile_kernel(const LinearArgs a, int32_t token_tiles) {
    constexpr int THREADS = (BT / WT) * (BN / WN) * 64;
    constexpr int KB = 128, CH = KB / 16;
    constexpr int C_LOADS = BT * CH / THREADS, W_LOADS = BN * CH / THREADS;
    static_assert(C_LOADS >= 1 && W_LOADS >= 1, "a thread loads whole chunks");
    __shared__ __align__(16) char lds[2][(BT + BN) * KB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wave_t = wave % (BT / WT), wave_n = wave / (BT / WT);
    const int64_t t0 = (int64_t)(blockIdx.x % token_tiles) * BT, n0 = (int64_t)(blockIdx.x / token_tiles) * BN;
    // 16 rows of one chunk are read together: their places cover the banks
    const auto place = [](int row, int chunk) { return row * KB + ((chunk ^ (row >> 1)) & 7) * 16; };

    u32x4 c_reg[C_LOADS], w_reg[W_LOADS];
    const int chunk = threadIdx.x % CH, row0 = threadIdx.x / CH;
    const auto load = [&](int64_t k) {
#pragma unroll
        for (int i = 0; i < C_LOADS; ++i) c_reg[i] = load16(a.codes, t0 + row0 + i * (THREADS / CH), a.tokens, k + chunk * 16, a.k);
#pragma unroll
        for (int i = 0; i < W_LOADS; ++i) w_reg[i] = load16(a.weight, n0 + row0 + i * (THREADS / CH), a.n, k + chunk * 16, a.k);
    };
    const auto store = [&](char *to) {
#pragma unroll
        for (int i = 0; i < C_LOADS; ++i) *(u32x4 *)(to + place(row0 + i * (THREADS / CH), chunk)) = c_reg[i];
#pragma unroll
        for (int i = 0; i < W_LOADS; ++i) *(u32x4 *)(to + BT * KB + place(row0 + i * (THREADS / CH), chunk)) = w_reg[i];
    };

    i32x16 acc[WN / 32][WT / 32];
#pragma unroll
    for (int i = 0; i < WN / 32; ++i)
#pragma unroll
        for (int j = 0; j < WT / 32; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    load(0);
    store(lds[0]);
    __syncthreads();
    int at = 0;
    for (int64_t k = 0; k < a.k; k += KB) {
        const bool more = k + KB < a.k;
        if (more) load(k + KB);
        const char *const codes = lds[at] + 0, *const weight = lds[at] + BT * KB;
#pragma unroll
        for (int s = 0; s < KB / 32; ++s) {
            i32x4 cf[WT / 32], wf[WN / 32];
#pragma unroll
            for (int j = 0; j < WT / 32; ++j) cf[j] = *(const i32x4 *)(codes + place(wave_t * WT + j * 32 + (lane & 31), s * 2 + (lane >> 5)));
#pragma unroll
            for (int i = 0; i < WN / 32; ++i) wf[i] = *(const i32x4 *)(weight + place(wave_n * WN + i * 32 + (lane & 31), s * 2 + (lane >> 5)));
#pragma unroll
            for (int i = 0; i < WN / 32; ++i)
#pragma unroll
                for (int j = 0; j < WT / 32; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[i], cf[j], acc[i][j], 0, 0, 0);
        }
        if (more) store(lds[at ^ 1]);
        __syncthreads();
        at ^= 1;
    }

    store_tile<T, WT, WN>(a, acc, t0 + wave_t * WT, n0 + wave_n * WN, lane);
}

// ---- tiles through LDS without registers ----

// 16 bytes a lane from a buffer to LDS: lane l's go to lds + 16 * l.  Written in assembly because the compiler, which cannot tell one
// stage of a tile from the next, waits for every such load before any read from LDS; it returns nothing in registers.  It counts
// like any load, so a wait that the compiler places only becomes longer.  wait_for_stage() is the wait that the data needs.
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t lane_offset, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(lane_offset), "s"(rsrc), "s"(offset), "s"(lds)
                 : "memory", "m0");
}
// Until at most N loads are outstanding.
template <int N>
__device__ __forceinline__ void wait_for_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Block b -> tile: neighbouring blocks go to the eight dies in turn, so each die gets a contiguous run of tiles; runs
// go down the token tiles of a group of eight, then on to the next channels, so that a die's workgroups share operands in its cache.
struct TileOrder {
    uint32_t tiles, token_tiles, channel_tiles;
    __device__ __forceinline__ void tile(uint32_t block, uint32_t &t, uint32_t &n) const {
        const uint32_t run = tiles / 8, more = tiles % 8, die = block % 8;
        const uint32_t at = die * run + (die < more ? die : more) + block / 8;
        const uint32_t group = at / (8 * channel_tiles), first = group * 8;
        const uint32_t high = token_tiles - first < 8 ? token_tiles - first : 8, in = at - group * 8 * channel_tiles;
        n = in / high;
        t = first + in % high;
    }
};

// As linear_tile_kernel, for rows of whole 4 bytes: STAGES tiles in LDS, loaded STAGES - 1 ahead.  A stage is complete when every
// wavefront has waited for its own loads and passed the barrier, which also says that the stage before has been read.
template <class T, int BT, int BN, int WT, int WN, int STAGES>
__global__ void __launch_bounds__((BT / WT) * (BN / WN) * 64) linear_staged_kernel(const LinearArgs a, const TileOrder order) {
    constexpr int WAVES = (BT / WT) * (BN / WN);
    constexpr int KB = 128, CH = KB / 16;
    constexpr int C_LOADS = BT * CH / 64 / WAVES, W_LOADS = BN * CH / 64 / WAVES, LOADS = C_LOADS + W_LOADS;
    static_assert(C_LOADS * 64 * WAVES == BT * CH && W_LOADS * 64 * WAVES == BN * CH, "a wavefront loads whole groups of 8 rows");
    static_assert((STAGES - 2) * LOADS < 64, "the counter of outstanding loads has six bits");
    constexpr int STAGE = (BT + BN) * KB;
    __shared__ __align__(16) char lds[STAGES * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave_t = wave % (BT / WT), wave_n = wave / (BT / WT);
    uint32_t t_tile, n_tile;
    order.tile(blockIdx.x, t_tile, n_tile);
    const int64_t t0 = (int64_t)t_tile * BT, n0 = (int64_t)n_tile * BN;
    const auto place = [](int row, int chunk) { return row * KB + ((chunk ^ (row >> 1)) & 7) * 16; };

    // a load moves 8 rows of 128 bytes; which chunk a lane takes follows from the place that it fills
    const auto resource = [&](const int8_t *base, int64_t row, int64_t rows) {
        const int64_t left = (rows - row) * a.k; // what lies behind the last row is not read
        const uint64_t address = reinterpret_cast<uint64_t>(base + row * a.k);
        return i32x4{__builtin_amdgcn_readfirstlane((int)address), __builtin_amdgcn_readfirstlane((int)((address >> 32) & 0xffff)),
                     __builtin_amdgcn_readfirstlane((int)(left < 0x7fffffff ? left : 0x7fffffff)), 0x00020000};
    };
    const i32x4 codes = resource(a.codes, t0, a.tokens), weight = resource(a.weight, n0, a.n);
    uint32_t c_off[C_LOADS], w_off[W_LOADS];
    const auto lane_offset = [&](int group) { // 8 rows from 8 * group on
        const int row = group * 8 + (lane >> 3);
        return (uint32_t)row * (uint32_t)a.k + (uint32_t)(((lane & 7) ^ (row >> 1)) & 7) * 16u;
    };
#pragma unroll
    for (int i = 0; i < C_LOADS; ++i) c_off[i] = lane_offset(wave * C_LOADS + i);
#pragma unroll
    for (int i = 0; i < W_LOADS; ++i) w_off[i] = lane_offset(wave * W_LOADS + i);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const int blocks = (int)((a.k + KB - 1) / KB);
    const auto issue = [&](int block, int stage) {
        const uint32_t at = lds0 + stage * STAGE;
#pragma unroll
        for (int i = 0; i < C_LOADS; ++i) load_to_lds(codes, c_off[i], block * KB, at + (wave * C_LOADS + i) * 1024);
#pragma unroll
        for (int i = 0; i < W_LOADS; ++i) load_to_lds(weight, w_off[i], block * KB, at + BT * KB + (wave * W_LOADS + i) * 1024);
    };

    i32x16 acc[WN / 32][WT / 32];
#pragma unroll
    for (int i = 0; i < WN / 32; ++i)
#pragma unroll
        for (int j = 0; j < WT / 32; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

    const int c_row = wave_t * WT + (lane & 31), w_row = wave_n * WN + (lane & 31);
    const auto multiply = [&](const char *stage, int left, auto ends) {
        i32x4 cf[2][WT / 32], wf[2][WN / 32]; // of two steps of 32 bytes: the next one's reads go ahead of this one's products
        const auto read = [&](int s) {
#pragma unroll
            for (int j = 0; j < WT / 32; ++j) cf[s & 1][j] = *(const i32x4 *)(stage + place(c_row + j * 32, s * 2 + (lane >> 5)));
#pragma unroll
            for (int i = 0; i < WN / 32; ++i) {
                wf[s & 1][i] = *(const i32x4 *)(stage + BT * KB + place(w_row + i * 32, s * 2 + (lane >> 5)));
                if constexpr (decltype(ends)::value) { // what lies behind the row's end counts as zero
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        if (s * 32 + (lane >> 5) * 16 + w * 4 >= left) wf[s & 1][i][w] = 0;
                }
            }
        };
        read(0);
#pragma unroll
        for (int s = 0; s < KB / 32; ++s) {
            if (s + 1 < KB / 32) read(s + 1);
            __builtin_amdgcn_sched_barrier(0); // left alone the reads sink to the end of the products that are to cover them
#pragma unroll
            for (int i = 0; i < WN / 32; ++i)
#pragma unroll
                for (int j = 0; j < WT / 32; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[s & 1][i], cf[s & 1][j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (i < blocks) issue(i, i);
    int stage = 0;
    const int whole = (int)(a.k / KB);
    for (int block = 0; block < whole; ++block) {
        if (block + STAGES - 2 < blocks) wait_for_loads<(STAGES - 2) * LOADS>();
        else wait_for_loads<0>();
        __syncthreads();
        if (block + STAGES - 1 < blocks) issue(block + STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);
        multiply(lds + stage * STAGE, KB, std::false_type{});
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    if (whole < blocks) {
        wait_for_loads<0>();
        __syncthreads();
        multiply(lds + stage * STAGE, (int)(a.k - (int64_t)whole * KB), std::true_type{});
    }

    store_tile<T, WT, WN>(a, acc, t0 + wave_t * WT, n0 + wave_n * WN, lane);
}

// ---- few tokens: bound by the weight's bytes ----

__device__ __forceinline__ u32x4 load16_inside(const int8_t *p) {
    typedef u32x4 __attribute__((aligned(1))) loose;
    return *(const __attribute__((address_space(1))) loose *)p;
}

// Up to M tokens by dot products of four bytes: a wavefront has R channels and goes along their rows, 1 KiB of each at a time.
template <class T, int M, int R, int AHEAD>
__global__ void __launch_bounds__(256) linear_dot_kernel(const LinearArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * R;
    if (n0 >= a.n) return;
    const int8_t *w[R], *c[M]; // rows that do not exist repeat the last one
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = a.weight + (n0 + r < a.n ? n0 + r : a.n - 1) * a.k;
#pragma unroll
    for (int m = 0; m < M; ++m) c[m] = a.codes + (m < a.tokens ? m : a.tokens - 1) * a.k;
    int sum[R][M] = {};
    const auto add = [&](const u32x4 (&wv)[R], const u32x4 (&cv)[M]) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[r][m] = __builtin_amdgcn_sdot4((int)wv[r][i], (int)cv[m][i], sum[r][m], false);
    };
    int64_t k = 0;
    for (; k + AHEAD * 1024 <= a.k; k += AHEAD * 1024) {
        u32x4 wv[AHEAD][R], cv[AHEAD][M];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
#pragma unroll
            for (int r = 0; r < R; ++r) wv[h][r] = load16_inside(w[r] + k + h * 1024 + lane * 16);
#pragma unroll
            for (int m = 0; m < M; ++m) cv[h][m] = load16_inside(c[m] + k + h * 1024 + lane * 16);
        }
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) add(wv[h], cv[h]);
    }
    for (; k < a.k; k += 1024) {
        u32x4 wv[R], cv[M];
#pragma unroll
        for (int r = 0; r < R; ++r) wv[r] = load16(w[r], 0, 1, k + lane * 16, a.k);
#pragma unroll
        for (int m = 0; m < M; ++m) cv[m] = load16(c[m], 0, 1, k + lane * 16, a.k);
        add(wv, cv);
    }
    // sums over the lanes; lane r * M + m keeps that one
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            int x = sum[r][m];
            x += __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, false);
            x += __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, false);
            x += __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, false);
            x += __builtin_amdgcn_update_dpp(0, x, 0x140, 0xf, 0xf, false);
            x = __builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16) + __builtin_amdgcn_readlane(x, 32) + __builtin_amdgcn_readlane(x, 48);
            if (lane == r * M + m) mine = x;
        }
    const int64_t n = n0 + lane / M, t = lane % M;
    if (lane >= R * M || n >= a.n || t >= a.tokens) return;
    float y = (float)mine * (a.scales[t] * a.weight_scales[n]);
    if (a.bias != nullptr) y += a.bias[n];
    store_element<T>(a.out + (t * a.n + n) * T::kBytes, y);
}

// MB x 16 tokens and NB x 16 channels a workgroup; its wavefronts take pieces of 128 bytes of the rows in turn, with operands straight
// from memory (a lane's 16 bytes are its part of an instruction's operand), and are added up in LDS at the end.
template <class T, int MB, int NB, int WAVES, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) linear_skinny_kernel(const LinearArgs a, int32_t token_tiles) {
    constexpr int TOKENS = 16 * MB, CHANNELS = 16 * NB;
    __shared__ __align__(16) int32_t part[WAVES][TOKENS][CHANNELS + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int64_t t0 = (int64_t)(blockIdx.x % token_tiles) * TOKENS, n0 = (int64_t)(blockIdx.x / token_tiles) * CHANNELS;
    const int8_t *c[MB], *w[NB];
#pragma unroll
    for (int m = 0; m < MB; ++m) {
        const int64_t t = t0 + m * 16 + col;
        c[m] = a.codes + (t < a.tokens ? t : a.tokens - 1) * a.k;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int64_t at = n0 + n * 16 + col;
        w[n] = a.weight + (at < a.n ? at : a.n - 1) * a.k;
    }
    i32x4 acc[NB][MB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[n][m] = i32x4{0, 0, 0, 0};
    const auto multiply = [&](const u32x4 (&wv)[2][NB], const u32x4 (&cv)[2][MB]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int m = 0; m < MB; ++m)
                    acc[n][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, wv[h][n]), __builtin_bit_cast(i32x4, cv[h][m]), acc[n][m], 0, 0, 0);
    };
    int64_t k = (int64_t)wave * AHEAD * 128;
    for (; k + AHEAD * 128 <= a.k; k += WAVES * AHEAD * 128) {
        u32x4 wv[AHEAD][2][NB], cv[AHEAD][2][MB];
#pragma unroll
        for (int x = 0; x < AHEAD; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int n = 0; n < NB; ++n) wv[x][h][n] = load16_inside(w[n] + k + x * 128 + h * 64 + quad * 16);
#pragma unroll
                for (int m = 0; m < MB; ++m) cv[x][h][m] = load16_inside(c[m] + k + x * 128 + h * 64 + quad * 16);
            }
#pragma unroll
        for (int x = 0; x < AHEAD; ++x) multiply(wv[x], cv[x]);
    }
    for (int x = 0; x < AHEAD && k < a.k; ++x, k += 128) { // the last piece of all, in one wavefront
        u32x4 wv[2][NB], cv[2][MB];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int n = 0; n < NB; ++n) wv[h][n] = load16(w[n], 0, 1, k + h * 64 + quad * 16, a.k);
#pragma unroll
            for (int m = 0; m < MB; ++m) cv[h][m] = load16(c[m], 0, 1, k + h * 64 + quad * 16, a.k);
        }
        multiply(wv, cv);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int m = 0; m < MB; ++m) *(i32x4 *)&part[wave][m * 16 + col][n * 16 + quad * 4] = acc[n][m];
    __syncthreads();
    for (int at = threadIdx.x; at < TOKENS * CHANNELS / 4; at += 64 * WAVES) {
        const int64_t t = t0 + at / (CHANNELS / 4), n = n0 + at % (CHANNELS / 4) * 4;
        if (t >= a.tokens || n >= a.n) continue;
        i32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int v = 0; v < WAVES; ++v) sum += *(const i32x4 *)&part[v][at / (CHANNELS / 4)][at % (CHANNELS / 4) * 4];
        const int count = (int)(a.n - n < 4 ? a.n - n : 4);
        const float s = a.scales[t];
        float y[4] = {};
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < count) {
                y[r] = (float)sum[r] * (s * a.weight_scales[n + r]);
                if (a.bias != nullptr) y[r] += a.bias[n + r];
            }
        store4<T>(a.out + (t * a.n + n) * T::kBytes, y, count, count == 4);
    }
}

template <class T, int BT, int BN, int WT, int WN, int STAGES>
int launch_staged(const LinearArgs &a, hipStream_t s) {
    const int64_t token_tiles = (a.tokens + BT - 1) / BT, channel_tiles = (a.n + BN - 1) / BN;
    if (token_tiles * channel_tiles > 0x7fffffff / 8) return TDE_ETOOBIG;
    const TileOrder order{(uint32_t)(token_tiles * channel_tiles), (uint32_t)token_tiles, (uint32_t)channel_tiles};
    linear_staged_kernel<T, BT, BN, WT, WN, STAGES><<<order.tiles, (BT / WT) * (BN / WN) * 64, 0, s>>>(a, order);
    return TDE_OK;
}

template <class T, int M>
void launch_dot(const LinearArgs &a, hipStream_t s) {
    if (a.n >= 8192) linear_dot_kernel<T, M, 4, 2><<<(uint32_t)((a.n + 15) / 16), 256, 0, s>>>(a);
    else linear_dot_kernel<T, M, 1, 4><<<(uint32_t)((a.n + 3) / 4), 256, 0, s>>>(a);
}

template <class T, int MB, int NB, int WAVES, int AHEAD>
int launch_skinny(const LinearArgs &a, hipStream_t s) {
    const int64_t token_tiles = (a.tokens + 16 * MB - 1) / (16 * MB), blocks = token_tiles * ((a.n + 16 * NB - 1) / (16 * NB));
    if (blocks > 0x7fffffff) return TDE_ETOOBIG;
    linear_skinny_kernel<T, MB, NB, WAVES, AHEAD><<<(uint32_t)blocks, 64 * WAVES, 0, s>>>(a, (int32_t)token_tiles);
    return TDE_OK;
}

#ifndef FORCE
#define FORCE 0
#endif
template <class T>
int launch_typed(const LinearArgs &a, hipStream_t s) {
    int st = TDE_OK;
    const bool words = a.k % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.codes) | reinterpret_cast<uintptr_t>(a.weight)) & 3u) == 0;
    if (a.tokens <= 4 && FORCE != 5) {
        if (a.tokens == 1) launch_dot<T, 1>(a, s);
        else if (a.tokens == 2) launch_dot<T, 2>(a, s);
        else launch_dot<T, 4>(a, s);
    } else if (a.tokens <= 16) {
        st = a.n >= 8192 ? launch_skinny<T, 1, 2, 8, 2>(a, s) : launch_skinny<T, 1, 1, 16, 2>(a, s);
    } else if (a.tokens <= 32) {
        st = a.n >= 8192 ? launch_skinny<T, 2, 2, 8, 2>(a, s) : launch_skinny<T, 2, 1, 16, 2>(a, s);
    } else if (a.tokens <= 64) {
        st = launch_skinny<T, 4, 2, 8, 2>(a, s);
    } else if (words) {
        const int64_t tiles256 = ((a.tokens + 255) / 256) * ((a.n + 255) / 256), tiles128 = ((a.tokens + 127) / 128) * ((a.n + 127) / 128);
        if (FORCE == 1 || (FORCE == 0 && tiles256 >= 128)) st = launch_staged<T, 256, 256, 128, 64, 2>(a, s);
        else if (FORCE == 2 || (FORCE == 0 && tiles128 >= 200)) st = launch_staged<T, 128, 128, 64, 64, 2>(a, s);
        else st = launch_staged<T, 64, 64, 32, 32, 4>(a, s);
    } else {
        const int64_t token_tiles = (a.tokens + 127) / 128, blocks = token_tiles * ((a.n + 127) / 128);
        if (blocks > 0x7fffffff) return TDE_ETOOBIG;
        linear_tile_kernel<T, 128, 128, 64, 64><<<(uint32_t)blocks, 256, 0, s>>>(a, (int32_t)token_tiles);
    }
    if (st != TDE_OK) return st;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace

int launch_int8_linear(const LinearArgs &a, int out_dtype, hipStream_t s) {
    switch (out_dtype) {
    case TDE_BF16: return launch_typed<Bf16>(a, s);
    case TDE_F16: return launch_typed<F16>(a, s);
    case TDE_F32: return launch_typed<F32>(a, s);
    }
    return TDE_EDTYPE;
}

} // namespace block
} // namespace tde
