// Product of int8 codes with scales for each token and each channel.
//
//   y[t][n] = T( float(sum_k c[t][k] * w[n][k]) * (s[t] * u[n]) + b[n] )
//
// The sum is exact: 32-bit integers, and at most 2^17 - 1 products of at most 2^14.  The weight's rows go in as the matrix
// instruction's first operand and the codes' as its second, so that a lane ends with four neighbouring channels of one token.
#include "tde_int8_linear.h"

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

#pragma unroll
    for (int j = 0; j < WT / 32; ++j) {
        const int64_t t = t0 + wave_t * WT + j * 32 + (lane & 31);
        if (t >= a.tokens) continue;
        const float s = a.scales[t];
#pragma unroll
        for (int i = 0; i < WN / 32; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int64_t n = n0 + wave_n * WN + i * 32 + g * 8 + (lane >> 5) * 4;
                const int count = (int)(a.n - n < 4 ? a.n - n : 4);
                if (count <= 0) continue;
                float y[4] = {};
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (r < count) {
                        y[r] = (float)acc[i][j][g * 4 + r] * (s * a.weight_scales[n + r]);
                        if (a.bias != nullptr) y[r] += a.bias[n + r];
                    }
                store4<T>(a.out + (t * a.n + n) * T::kBytes, y, count, count == 4);
            }
    }
}

template <class T>
int launch_typed(const LinearArgs &a, hipStream_t s) {
    const int64_t bt = a.tokens <= 32 ? 32 : 128;
    const int64_t token_tiles = (a.tokens + bt - 1) / bt, blocks = token_tiles * ((a.n + 127) / 128);
    if (blocks > 0x7fffffff) return TDE_ETOOBIG;
    if (bt == 32) linear_tile_kernel<T, 32, 128, 32, 32><<<(uint32_t)blocks, 256, 0, s>>>(a, (int32_t)token_tiles);
    else linear_tile_kernel<T, 128, 128, 64, 64><<<(uint32_t)blocks, 256, 0, s>>>(a, (int32_t)token_tiles);
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
