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

// A wavefront's sums, scaled: WT tokens from t0 on, WN channels from n0 on, as many as there are.
template <class T, int WT, int WN>
__device__ __forceinline__ void store_sums(const LinearArgs &a, const i32x16 (&acc)[WN / 32][WT / 32], int64_t t0, int64_t n0, int lane) {
    const bool biased = a.bias != nullptr;
    float s[WT / 32];
#pragma unroll
    for (int j = 0; j < WT / 32; ++j) {
        const int64_t t = t0 + j * 32 + (lane & 31);
        s[j] = t < a.tokens ? a.scales[t] : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < WN / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int64_t n = n0 + i * 32 + g * 8 + (lane >> 5) * 4;
            const int count = (int)(a.n - n < 4 ? a.n - n : 4);
            float u[4], b[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u[r] = r < count ? a.weight_scales[n + r] : 0.0f;
                b[r] = biased && r < count ? a.bias[n + r] : 0.0f;
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
                if (t < a.tokens && count > 0) store4<T>(a.out + (t * a.n + n) * T::kBytes, y, count, count >= 4);
            }
        }
}
// The same for a tile whose tokens and channels all exist, by way of LDS (`room`, kStoreRoom bytes of the wavefront's own): a lane
// has 4 channels of 32 different tokens' rows, and leaves with 16 bytes next to its neighbours'.  (Stored as they are, 8 bytes a row,
// the results of 4096 x 4096 x 4096 take 30 us of 85.)
template <class T, int WN>
constexpr int kStoreRoom = 32 * (WN * T::kBytes + 16);
template <class T, int WT, int WN>
__device__ __forceinline__ void store_rows(const LinearArgs &a, const i32x16 (&acc)[WN / 32][WT / 32], int64_t t0, int64_t n0, int lane, char *room) {
    const bool biased = a.bias != nullptr;
    constexpr int PITCH = WN * T::kBytes + 16, LANES = WN * T::kBytes / 16, ROWS = 64 / LANES; // lanes of a row, rows of a store
    const int row = lane & 31, from = (lane >> 5) * 4;
#pragma unroll
    for (int j = 0; j < WT / 32; ++j) {
        const float s = a.scales[t0 + j * 32 + row];
#pragma unroll
        for (int i = 0; i < WN / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int n = i * 32 + g * 8 + from;
                float y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    y[r] = (float)acc[i][j][g * 4 + r] * (s * a.weight_scales[n0 + n + r]);
                    if (biased) y[r] += a.bias[n0 + n + r];
                }
                const Words<4 * T::kBytes> w = narrow_all<T, 4>(y);
                char *const to = room + row * PITCH + n * T::kBytes;
                if constexpr (T::kBytes == 4) *(u32x4 *)to = u32x4{w.w[0], w.w[1], w.w[2], w.w[3]};
                else *(u32x2 *)to = u32x2{w.w[0], w.w[1]};
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int x = 0; x < 32 / ROWS; ++x) {
            const int at = x * ROWS + lane / LANES;
            const u32x4 v = *(const u32x4 *)(room + at * PITCH + lane % LANES * 16);
            store_words<16>(a.out + ((t0 + j * 32 + at) * a.n + n0) * T::kBytes + lane % LANES * 16, Words<16>{{v[0], v[1], v[2], v[3]}});
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}
template <class T, int WT, int WN>
__device__ __forceinline__ void store_tile(const LinearArgs &a, const i32x16 (&acc)[WN / 32][WT / 32], int64_t t0, int64_t n0, int lane, char *room) {
    if (t0 + WT <= a.tokens && n0 + WN <= a.n) store_rows<T, WT, WN>(a, acc, t0, n0, lane, room);
    else store_sums<T, WT, WN>(a, acc, t0, n0, lane);
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

    static_assert(kStoreRoom<T, WN> * THREADS / 64 <= (int)sizeof(lds));
    store_tile<T, WT, WN>(a, acc, t0 + wave_t * WT, n0 + wave_n * WN, lane, lds[0] + wave * kStoreRoom<T, WN>);
}

// ---- tiles through LDS without registers ----

// 16 bytes a lane from a buffer to LDS: lane l's go to lds + 16 * l.  Written in assembly because the compiler, which cannot tell one
// stage of a tile from the next, waits for every such load before any read from LDS; it returns nothing in registers.  It counts
// like any load, so a wait that the compiler places only becomes longer.  wait_for_stage() is the wait that the data needs.
// STREAM: read once, not to be kept in the caches.
template <bool STREAM = false>
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t lane_offset, uint32_t offset, uint32_t lds) {
    if constexpr (STREAM)
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen nt lds"
                     :
                     : "v"(lane_offset), "s"(rsrc), "s"(offset), "s"(lds)
                     : "memory", "m0");
    else
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

// As linear_tile_kernel, for rows of whole 4 bytes: STAGES blocks of 128 bytes of the rows in LDS, loaded STAGES - 1 ahead.  A stage
// is complete when every wavefront has waited for its own loads and passed the barrier, which also says that the stage before has
// been read.
template <class T, int BT, int BN, int WT, int WN, int STAGES>
__global__ void __launch_bounds__((BT / WT) * (BN / WN) * 64) linear_staged_kernel(const LinearArgs a, const TileOrder order) {
    constexpr int WAVES = (BT / WT) * (BN / WN);
    constexpr int KB = 128, CH = KB / 16;
    constexpr int C_LOADS = BT / 8 / WAVES, W_LOADS = BN / 8 / WAVES, LOADS = C_LOADS + W_LOADS;
    static_assert(C_LOADS * 8 * WAVES == BT && W_LOADS * 8 * WAVES == BN, "a wavefront loads whole groups of 8 rows");
    static_assert((STAGES - 2) * LOADS < 64, "the counter of outstanding loads has six bits");
    constexpr int STAGE = (BT + BN) * KB;
    __shared__ __align__(16) char lds[STAGES * STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wave_t = wave % (BT / WT), wave_n = wave / (BT / WT);
    uint32_t t_tile, n_tile;
    order.tile(blockIdx.x, t_tile, n_tile);
    const int64_t t0 = (int64_t)t_tile * BT, n0 = (int64_t)n_tile * BN;
    // 16 rows of one chunk are read together: their places cover the banks
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
    const auto lane_offset = [&](int rows8) { // rows from 8 * rows8 on
        const int row = rows8 * 8 + (lane >> 3);
        return (uint32_t)row * (uint32_t)a.k + (uint32_t)((lane ^ (row >> 1)) & (CH - 1)) * 16u;
    };
#pragma unroll
    for (int i = 0; i < C_LOADS; ++i) c_off[i] = lane_offset(wave * C_LOADS + i);
#pragma unroll
    for (int i = 0; i < W_LOADS; ++i) w_off[i] = lane_offset(wave * W_LOADS + i);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
    const int blocks = (int)((a.k + KB - 1) / KB), whole = (int)(a.k / KB);
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
    __syncthreads(); // the stages have been read
    static_assert(kStoreRoom<T, WN> * WAVES <= STAGES * STAGE);
    store_tile<T, WT, WN>(a, acc, t0 + wave_t * WT, n0 + wave_n * WN, lane, lds + wave * kStoreRoom<T, WN>);
}

// ---- few tokens: bound by the weight's bytes ----

template <bool STREAM>
__device__ __forceinline__ u32x4 load16_inside(const int8_t *p) {
    typedef u32x4 __attribute__((aligned(1))) loose;
    const auto *const from = (const __attribute__((address_space(1))) loose *)p;
    return STREAM ? __builtin_nontemporal_load(from) : *from;
}

// Up to M tokens by dot products of four bytes: a wavefront has R channels and goes along their rows, 1 KiB of each at a time.
template <class T, int M, int R, int AHEAD, bool STREAM>
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
    // wavefronts begin at different places: see linear_pieces_kernel
    constexpr int STEP = AHEAD * 1024;
    const uint32_t steps = (uint32_t)(a.k / STEP), first = steps == 0 ? 0 : (uint32_t)(n0 / R) % steps;
    for (uint32_t i = 0; i < steps; ++i) {
        const int64_t k = (int64_t)(i + first < steps ? i + first : i + first - steps) * STEP;
        u32x4 wv[AHEAD][R], cv[AHEAD][M];
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) {
#pragma unroll
            for (int r = 0; r < R; ++r) wv[h][r] = load16_inside<STREAM>(w[r] + k + h * 1024 + lane * 16);
#pragma unroll
            for (int m = 0; m < M; ++m) cv[h][m] = load16_inside<false>(c[m] + k + h * 1024 + lane * 16);
        }
#pragma unroll
        for (int h = 0; h < AHEAD; ++h) add(wv[h], cv[h]);
    }
    for (int64_t k = (int64_t)steps * STEP; k < a.k; k += 1024) {
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

// MB x 16 tokens and NB x 16 channels a workgroup; its wavefronts take pieces of 128 bytes of the rows in turn, each through LDS of its
// own (STAGES pieces, no barrier), and are added up at the end.
template <class T, int MB, int NB, int WAVES, int STAGES, bool STREAM>
__global__ void __launch_bounds__(64 * WAVES) linear_pieces_kernel(const LinearArgs a, int32_t token_tiles) {
    constexpr int TOKENS = 16 * MB, CHANNELS = 16 * NB, KB = 128;
    constexpr int LOADS = 2 * (MB + NB), STAGE = (TOKENS + CHANNELS) * KB, RING = STAGES * STAGE;
    constexpr int PART = TOKENS * (CHANNELS + 4); // sums of a wavefront
    constexpr int LDS = WAVES * (RING > PART * 4 ? RING : PART * 4);
    static_assert(STAGES * LOADS < 64, "the counter of outstanding loads has six bits");
    __shared__ __align__(16) char lds[LDS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int64_t t0 = (int64_t)(blockIdx.x % token_tiles) * TOKENS, n0 = (int64_t)(blockIdx.x / token_tiles) * CHANNELS;
    const auto place = [](int row, int chunk) { return row * KB + ((chunk ^ (row >> 1)) & 7) * 16; };
    // rows that do not exist lie behind the resources' ends, as pieces behind the last do: they are not read
    const auto resource = [&](const int8_t *base, int64_t row, int64_t rows, int most) {
        const int64_t left = rows - row < most ? rows - row : most;
        const uint64_t address = reinterpret_cast<uint64_t>(base + row * a.k);
        return i32x4{__builtin_amdgcn_readfirstlane((int)address), __builtin_amdgcn_readfirstlane((int)((address >> 32) & 0xffff)),
                     __builtin_amdgcn_readfirstlane((int)(left * a.k)), 0x00020000};
    };
    const i32x4 codes = resource(a.codes, t0, a.tokens, TOKENS), weight = resource(a.weight, n0, a.n, CHANNELS);
    constexpr uint32_t kBehind = 0x40000000;
    const int pieces = (int)((a.k + KB - 1) / KB);
    const uint32_t row_off = (uint32_t)(lane >> 3) * (uint32_t)a.k, step = 8u * (uint32_t)a.k;
    // rows 8 apart take chunks four places apart
    const uint32_t chunk_even = (uint32_t)((lane ^ (lane >> 4)) & 7) * 16u, chunk_odd = chunk_even ^ 64u;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds + wave * RING;
    // workgroups begin at different pieces: rows that lie a power of two apart share memory channels, piece by piece
    // (8 x 8192 x 8192: 19.5 us beginning together, 13.8 like this; 8 x 8320 x 8192 14 either way)
    const int first = (int)(blockIdx.x * 13 % (uint32_t)pieces);
    const auto turned = [&](int piece) { return piece + first >= pieces ? piece + first - pieces : piece + first; };
    const auto issue = [&](int piece, int stage) {
        const uint32_t at = row_off + (piece < pieces ? (uint32_t)turned(piece) * KB : kBehind);
#pragma unroll
        for (int i = 0; i < 2 * MB; ++i) load_to_lds(codes, at + i * step + (i & 1 ? chunk_odd : chunk_even), 0, lds0 + stage * STAGE + i * 1024);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i)
            load_to_lds<STREAM>(weight, at + i * step + (i & 1 ? chunk_odd : chunk_even), 0, lds0 + stage * STAGE + TOKENS * KB + i * 1024);
    };
    i32x4 acc[NB][MB];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[n][m] = i32x4{0, 0, 0, 0};
    const auto multiply = [&](int stage, int left) {
        const char *const from = lds + wave * RING + stage * STAGE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4 w[NB], c[MB];
#pragma unroll
            for (int m = 0; m < MB; ++m) c[m] = *(const i32x4 *)(from + place(m * 16 + col, h * 4 + quad));
#pragma unroll
            for (int n = 0; n < NB; ++n) w[n] = *(const i32x4 *)(from + TOKENS * KB + place(n * 16 + col, h * 4 + quad));
            if (left < KB) { // what lies behind the row's end counts as zero
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (h * 64 + quad * 16 + i * 4 >= left) w[n][i] = 0;
            }
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int m = 0; m < MB; ++m) acc[n][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[n], c[m], acc[n][m], 0, 0, 0);
        }
    };
#pragma unroll
    for (int x = 0; x < STAGES; ++x) issue(wave + x * WAVES, x);
    int stage = 0;
    for (int piece = wave; piece < pieces; piece += WAVES) {
        wait_for_loads<(STAGES - 1) * LOADS>();
        multiply(stage, (int)(a.k - (int64_t)turned(piece) * KB));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the stage has been read
        issue(piece + STAGES * WAVES, stage);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    wait_for_loads<0>();
    __syncthreads();
    int32_t(*const part)[TOKENS][CHANNELS + 4] = reinterpret_cast<int32_t(*)[TOKENS][CHANNELS + 4]>(lds);
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

// The same for rows that begin anywhere: operands come straight from memory to registers (a lane's 16 bytes are its part of an
// instruction's operand), which takes loads of 16 bytes from 16 rows at once.  Bound by those loads, which the hardware splits where
// they do not begin on words: 10 x 5121 x 7168 takes 32 us (tiles by way of registers and LDS 49, rows of whole words 9), 24 x 4099 x 4096 18
// (29), 32 x 1001 x 2000 7 (11); with 7168 channels 32 tokens would be faster in tiles (56 and 45), from 33 on all are.
template <class T, int MB, int NB, int WAVES, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) linear_loose_kernel(const LinearArgs a, int32_t token_tiles) {
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
                for (int n = 0; n < NB; ++n) wv[x][h][n] = load16_inside<false>(w[n] + k + x * 128 + h * 64 + quad * 16);
#pragma unroll
                for (int m = 0; m < MB; ++m) cv[x][h][m] = load16_inside<false>(c[m] + k + x * 128 + h * 64 + quad * 16);
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

// Weights from 32 MB on pass by the caches: they would push out what fits there, and come faster (one token x 8192 x 8192 12.0 us, by way
// of the caches 13.7).  A smaller one may still be there from the last call (one token x 8192 x 1280 3.7 us, streamed 4.1).
bool streams(const LinearArgs &a) { return a.n * a.k >= (int64_t)32 << 20; }

template <class T, int M>
int launch_dot(const LinearArgs &a, hipStream_t s) {
    if (!fits_launch((a.n + (a.n >= 8192 ? 15 : 3)) / (a.n >= 8192 ? 16 : 4), 256)) return TDE_ETOOBIG;
    // Four channels a wavefront share the codes' loads; one where that leaves few wavefronts.  With rows of 8192 bytes, in us: four tokens x 8192
    // channels 17.9 (one channel a wavefront 22.5), x 4096 13.5 (12.3), x 1280 8.9 (5.4); two x 8192 14.1 (16.2), x 4096 11.2 (9.2); one token has no
    // codes to share: x 8192 12.5 (12.4), x 10240 17.0 (14.9), but 28672 channels of 2048 bytes 10.6 (12.0).
    if (a.n >= 8192 && streams(a)) linear_dot_kernel<T, M, 4, 2, true><<<(uint32_t)((a.n + 15) / 16), 256, 0, s>>>(a);
    else if (a.n >= 8192) linear_dot_kernel<T, M, 4, 2, false><<<(uint32_t)((a.n + 15) / 16), 256, 0, s>>>(a);
    else if (streams(a)) linear_dot_kernel<T, M, 1, 4, true><<<(uint32_t)((a.n + 3) / 4), 256, 0, s>>>(a);
    else linear_dot_kernel<T, M, 1, 4, false><<<(uint32_t)((a.n + 3) / 4), 256, 0, s>>>(a);
    return TDE_OK;
}

template <class T, int BT, int BN, int WT, int WN, int STAGES>
int launch_staged(const LinearArgs &a, hipStream_t s) {
    const int64_t token_tiles = (a.tokens + BT - 1) / BT, channel_tiles = (a.n + BN - 1) / BN;
    if (!fits_launch(token_tiles * channel_tiles, (BT / WT) * (BN / WN) * 64)) return TDE_ETOOBIG;
    const TileOrder order{(uint32_t)(token_tiles * channel_tiles), (uint32_t)token_tiles, (uint32_t)channel_tiles};
    linear_staged_kernel<T, BT, BN, WT, WN, STAGES><<<order.tiles, (BT / WT) * (BN / WN) * 64, 0, s>>>(a, order);
    return TDE_OK;
}

template <class T, int MB, int NB, int WAVES, int STAGES>
int launch_pieces(const LinearArgs &a, hipStream_t s) {
    const int64_t token_tiles = (a.tokens + 16 * MB - 1) / (16 * MB), blocks = token_tiles * ((a.n + 16 * NB - 1) / (16 * NB));
    if (!fits_launch(blocks, 64 * WAVES)) return TDE_ETOOBIG;
    if (streams(a) && token_tiles == 1)
        linear_pieces_kernel<T, MB, NB, WAVES, STAGES, true><<<(uint32_t)blocks, 64 * WAVES, 0, s>>>(a, (int32_t)token_tiles);
    else linear_pieces_kernel<T, MB, NB, WAVES, STAGES, false><<<(uint32_t)blocks, 64 * WAVES, 0, s>>>(a, (int32_t)token_tiles);
    return TDE_OK;
}

template <class T, int BT, int BN, int WT, int WN>
int launch_tile(const LinearArgs &a, hipStream_t s) {
    const int64_t token_tiles = (a.tokens + BT - 1) / BT, blocks = token_tiles * ((a.n + BN - 1) / BN);
    if (!fits_launch(blocks, (BT / WT) * (BN / WN) * 64)) return TDE_ETOOBIG;
    linear_tile_kernel<T, BT, BN, WT, WN><<<(uint32_t)blocks, (BT / WT) * (BN / WN) * 64, 0, s>>>(a, (int32_t)token_tiles);
    return TDE_OK;
}

template <class T, int MB>
int launch_loose(const LinearArgs &a, hipStream_t s) {
    const int64_t token_tiles = (a.tokens + 16 * MB - 1) / (16 * MB), blocks = token_tiles * ((a.n + 15) / 16);
    if (!fits_launch(blocks, 512)) return TDE_ETOOBIG;
    linear_loose_kernel<T, MB, 1, 8, 2><<<(uint32_t)blocks, 512, 0, s>>>(a, (int32_t)token_tiles);
    return TDE_OK;
}

// ---- which kernel ----

// From 65 tokens on every kernel works on tiles, and which one is best follows from how many rounds its tiles need on the units and
// what 128 bytes of the rows cost in a round (microseconds, measured with every unit busy) beside what a launch costs at all:
//
//   tokens x channels  a round's 128 bytes  launch   e.g. (us, against the next best)
//   256 x 256          1.9                  5        8192 x 8192 x 8192 487 (256 x 128: 553)
//   256 x 128          1.17                 4        2048 x 4096 x 4096 41 (128 x 128: 49)
//   128 x 128          0.66                 4        512 x 8192 x 8192 46 (256 x 128: 61)
//   64 x 128           0.55                 3.5      1257 x 5000 x 1100 22.8 (64 x 64: 26.0)
//   64 x 64            0.37 one a unit, 0.62 two a unit at once
//                                           3.5      128 x 5120 x 7168 18.3 (64 x 32: 22.2)
//   64 x 32 in pieces  0.25, 0.11 where fewer than half of the units are busy
//                                           5.5      100 x 8192 x 1280 9.7 (64 x 64: 19.0)
enum Tile { k256x256, k256x128, k128x128, k64x128, k64x64, kPieces };
Tile best_tile(int64_t tokens, int64_t n, int64_t k) {
    const int64_t cus = device_compute_units();
    const auto tiles = [&](int64_t bt, int64_t bn) { return ((tokens + bt - 1) / bt) * ((n + bn - 1) / bn); };
    const auto rounds = [&](int64_t t, int64_t at_once) { return (double)((t + at_once - 1) / at_once); };
    const double blocks = (double)((k + 127) / 128);
    const int64_t small = tiles(64, 64), pieces = tiles(64, 32);
    const double cost[] = {
        5.0 + blocks * 1.9 * rounds(tiles(256, 256), cus),
        4.0 + blocks * 1.17 * rounds(tiles(256, 128), cus),
        4.0 + blocks * 0.66 * rounds(tiles(128, 128), cus),
        3.5 + blocks * 0.55 * rounds(tiles(64, 128), cus),
        3.5 + blocks * (small <= cus ? 0.37 : 0.62 * rounds(small, 2 * cus)),
        5.5 + blocks * (pieces * 2 <= cus ? 0.11 : 0.25 * rounds(pieces, cus)),
    };
    int best = 0;
    for (int i = 1; i <= kPieces; ++i)
        if (cost[i] < cost[best]) best = i;
    return (Tile)best;
}

template <class T>
int launch_typed(const LinearArgs &a, hipStream_t s) {
    int st = TDE_OK;
    const bool words = a.k % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.codes) | reinterpret_cast<uintptr_t>(a.weight)) & 3u) == 0;
    if (a.tokens <= 4) {
        if (a.tokens == 1) st = launch_dot<T, 1>(a, s);
        else if (a.tokens == 2) st = launch_dot<T, 2>(a, s);
        else st = launch_dot<T, 4>(a, s);
    } else if (words && a.tokens <= 64) {
        // channels of a workgroup: two blocks of 16 where that leaves a workgroup for half of the units at least (16 x 5120 x 7168 9.0
        // us, with one block 12.0; 16 x 8192 x 1280 6.7 and 5.9)
        const bool two = (a.n + 31) / 32 >= device_compute_units() / 2;
        if (a.tokens <= 16) st = two ? launch_pieces<T, 1, 2, 4, 3>(a, s) : launch_pieces<T, 1, 1, 8, 4>(a, s);
        else if (a.tokens <= 32) st = two ? launch_pieces<T, 2, 2, 8, 2>(a, s) : launch_pieces<T, 2, 1, 8, 3>(a, s);
        else st = two ? launch_pieces<T, 4, 2, 8, 1>(a, s) : launch_pieces<T, 4, 1, 4, 3>(a, s);
    } else if (words) {
        switch (best_tile(a.tokens, a.n, a.k)) {
        case k256x256: st = launch_staged<T, 256, 256, 128, 64, 2>(a, s); break;
        case k256x128: st = launch_staged<T, 256, 128, 64, 64, 3>(a, s); break;
        case k128x128: st = launch_staged<T, 128, 128, 64, 32, 4>(a, s); break;
        case k64x128: st = launch_staged<T, 64, 128, 32, 32, 5>(a, s); break;
        case k64x64: st = launch_staged<T, 64, 64, 32, 32, 4>(a, s); break;
        case kPieces: st = launch_pieces<T, 4, 2, 8, 1>(a, s); break;
        }
    } else if (a.tokens <= 32) {
        st = a.tokens <= 16 ? launch_loose<T, 1>(a, s) : launch_loose<T, 2>(a, s);
    } else {
        // 128 x 128 by eight wavefronts where such tiles occupy two thirds of the units (1000 x 4099 x 4096, 256 of them, 49 us; 64 x 64
        // 61), else 64 x 64 (600 x 3001 x 3000, 120 of the larger ones, 32 us against 40; 64 x 5121 x 7168 49 against 62)
        const int64_t large = ((a.tokens + 127) / 128) * ((a.n + 127) / 128);
        st = large * 3 >= (int64_t)device_compute_units() * 2 ? launch_tile<T, 128, 128, 64, 32>(a, s) : launch_tile<T, 64, 64, 32, 32>(a, s);
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
