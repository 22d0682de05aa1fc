// What the operators of an attention block share: element types, small-vector access, sums across lanes, and the place of a token in
// a ragged batch over a paged cache.  Internal to libtde_hip.so.
#ifndef TDE_BLOCK_H
#define TDE_BLOCK_H

#include <hip/hip_runtime.h>

#include <cstdint>

#include "tde_abi.h"

namespace tde {

int hip_failed(hipError_t e); // records the code for tde_last_hip_error and returns TDE_EHIP (tde_abi.hip)
int device_compute_units();   // of the current device; 256 where none can be asked (tde_abi.hip)

namespace block {

// Whether a launch holds that many threads: the packet that starts it counts them in 32 bits.
inline bool fits_launch(int64_t blocks, int threads) { return blocks <= (int64_t)0xffffffff / threads; }

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Bf16 {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ void widen(uint32_t w, float &lo, float &hi) {
        lo = __builtin_bit_cast(float, w << 16);
        hi = __builtin_bit_cast(float, w & 0xffff0000u);
    }
    static __device__ __forceinline__ float widen1(uint16_t h) { return __builtin_bit_cast(float, (uint32_t)h << 16); }
    static __device__ __forceinline__ uint32_t narrow(float lo, float hi) { // to nearest even
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
    }
    static __device__ __forceinline__ uint16_t narrow1(float x) { return (uint16_t)narrow(x, 0.0f); }
};
struct F16 {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ void widen(uint32_t w, float &lo, float &hi) {
        const f16x2 h = __builtin_bit_cast(f16x2, w);
        lo = (float)h[0];
        hi = (float)h[1];
    }
    static __device__ __forceinline__ float widen1(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
    static __device__ __forceinline__ uint32_t narrow(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2));
    }
    static __device__ __forceinline__ uint16_t narrow1(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
};
struct F32 {
    static constexpr int kBytes = 4;
};

// N elements of T between registers and memory; the address need only be a multiple of the element's size (global accesses of any
// width take such addresses on this hardware).
template <int BYTES>
struct Words {
    uint32_t w[BYTES / 4];
};
// STREAM: passed by the caches, for what is read or written once.
template <int BYTES, bool STREAM = false>
__device__ __forceinline__ Words<BYTES> load_words(const void *p) {
    Words<BYTES> r;
    if constexpr (BYTES % 16 == 0) {
        typedef u32x4 __attribute__((aligned(2))) loose;
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const auto *const from = (const __attribute__((address_space(1))) loose *)p + i;
            const u32x4 v = STREAM ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
        }
    } else if constexpr (BYTES == 8) {
        typedef u32x2 __attribute__((aligned(2))) loose;
        const u32x2 v = *(const __attribute__((address_space(1))) loose *)p;
        r.w[0] = v[0];
        r.w[1] = v[1];
    } else {
        static_assert(BYTES == 4, "4, 8 or whole 16 bytes");
        typedef uint32_t __attribute__((aligned(2))) loose;
        r.w[0] = *(const __attribute__((address_space(1))) loose *)p;
    }
    return r;
}
template <int BYTES, bool STREAM = false>
__device__ __forceinline__ void store_words(void *p, const Words<BYTES> &r) {
    if constexpr (BYTES % 16 == 0) {
        typedef u32x4 __attribute__((aligned(2))) loose;
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            auto *const to = (__attribute__((address_space(1))) loose *)p + i;
            const loose v = u32x4{r.w[4 * i], r.w[4 * i + 1], r.w[4 * i + 2], r.w[4 * i + 3]};
            if constexpr (STREAM) __builtin_nontemporal_store(v, to);
            else *to = v;
        }
    } else if constexpr (BYTES == 8) {
        typedef u32x2 __attribute__((aligned(2))) loose;
        *(__attribute__((address_space(1))) loose *)p = u32x2{r.w[0], r.w[1]};
    } else {
        static_assert(BYTES == 4, "4, 8 or whole 16 bytes");
        typedef uint32_t __attribute__((aligned(2))) loose;
        *(__attribute__((address_space(1))) loose *)p = r.w[0];
    }
}

template <class T, int N>
__device__ __forceinline__ void widen_all(const Words<N * T::kBytes> &raw, float (&x)[N]) {
    if constexpr (T::kBytes == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = __builtin_bit_cast(float, raw.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) T::widen(raw.w[i], x[2 * i], x[2 * i + 1]);
    }
}
template <class T, int N>
__device__ __forceinline__ Words<N * T::kBytes> narrow_all(const float (&x)[N]) {
    Words<N * T::kBytes> raw;
    if constexpr (T::kBytes == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) raw.w[i] = __builtin_bit_cast(uint32_t, x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) raw.w[i] = T::narrow(x[2 * i], x[2 * i + 1]);
    }
    return raw;
}
template <class T>
__device__ __forceinline__ float load_element(const char *p) {
    if constexpr (T::kBytes == 4) return *(const __attribute__((address_space(1))) float *)p;
    else return T::widen1(*(const __attribute__((address_space(1))) uint16_t *)p);
}
template <class T>
__device__ __forceinline__ void store_element(char *p, float x) {
    if constexpr (T::kBytes == 4) *(__attribute__((address_space(1))) float *)p = x;
    else *(__attribute__((address_space(1))) uint16_t *)p = T::narrow1(x);
}

template <int CONTROL>
__device__ __forceinline__ float lanes_moved(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CONTROL, 0xf, 0xf, false));
}
// Sum over aligned groups of 2^log2 lanes, the same bits in each of the group's lanes.  Lanes change partners inside rows of 16 by
// data-parallel moves (a mirror reaches the other half where both halves already agree), beyond them by the half-swaps.
__device__ __forceinline__ float sum_over_lanes(float x, int log2) {
    if (log2 >= 1) x += lanes_moved<0xB1>(x);
    if (log2 >= 2) x += lanes_moved<0x4E>(x);
    if (log2 >= 3) x += lanes_moved<0x141>(x);
    if (log2 >= 4) x += lanes_moved<0x140>(x);
    if (log2 >= 5) x += __shfl_xor(x, 16);
    if (log2 >= 6) x += __shfl_xor(x, 32);
    return x;
}

// n / d for n < 2^31 and 1 <= d < 2^31.  With r = floor(2^32 / d), n * r / 2^32 is below n / d by less than n / 2^32 < 1/2, so its
// floor is the quotient or one less, and one comparison tells which.
struct Divisor32 {
    uint32_t d, reciprocal; // floor(2^32 / d), or 2^32 - 1 for d == 1
    __host__ __device__ Divisor32() : d(1), reciprocal(0xffffffffu) {}
    __host__ __device__ explicit Divisor32(uint32_t divisor)
        : d(divisor), reciprocal(divisor == 1 ? 0xffffffffu : (uint32_t)(0x100000000ull / divisor)) {}
    __host__ __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
        const uint32_t q = (uint32_t)(((uint64_t)n * reciprocal) >> 32); // the quotient or one less
        return n - q * d >= d ? q + 1 : q;
    }
};

// A ragged batch over a paged cache, as the device sees it.
struct PagedBatch {
    const int32_t *table;  // [seqs, table_pages]
    const int32_t *starts; // [seqs + 1]
    const int32_t *lens;   // [seqs]
    int64_t table_stride;
    int32_t seqs, table_pages, cache_pages;
    Divisor32 page; // tokens a page
};

// The page with number `at` in a sequence's row of the table, or -1 where the table or the cache has none.
__host__ __device__ __forceinline__ int32_t page_number(const PagedBatch &b, const int32_t *row, uint32_t at) {
    if (at >= (uint32_t)b.table_pages) return -1;
    const int32_t page = row[at];
    return page >= 0 && page < b.cache_pages ? page : -1;
}

// The sequence of row `token` for a whole wavefront (`token` the same in all lanes): the number of sequences that end at or before
// it, seqs for a row behind the last.  64 probes a step, so up to 64 sequences take one load and 4096 two.  Whatever the array
// holds, the result lies in [0, seqs] and the number of steps is fixed by seqs.
__device__ __forceinline__ int sequence_of(const PagedBatch &b, int64_t token, int lane) {
    int base = 0, width = b.seqs;
    while (width > 0) {
        const int step = (width + 63) >> 6;
        const int64_t at = (int64_t)base + (int64_t)(lane + 1) * step;
        const bool ends = at <= base + width && at <= b.seqs && b.starts[at] <= token;
        const int passed = __builtin_popcountll(__builtin_amdgcn_ballot_w64(ends));
        const int skipped = passed * step;
        if (step == 1) return base + passed;
        base += skipped;
        width = width - skipped < step ? width - skipped : step;
    }
    return base;
}

} // namespace block
} // namespace tde

#endif // TDE_BLOCK_H
