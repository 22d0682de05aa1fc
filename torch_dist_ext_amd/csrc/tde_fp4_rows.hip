// Codes and scales of a cache in 4 bits as numbers of T: T(code * 2^(e - 127)), one rounding (none in bf16 and fp32 but among subnormal numbers).
//
// Bound by memory, by what is written: a lane turns 4 bytes of codes into 8 numbers, so that a wavefront's stores are whole lines, and past the caches:
// 131072 rows of 8 heads of 128 channels take 51 us, 6.7 TB/s, and 63 with stores that stay in the caches.  (Four such pieces a lane: 51 us, and 512 rows of
// a head 2.8 and not 2.2.)
#include "tde_fp4_rows.h"

namespace tde {
namespace block {

namespace {

template <class T>
__device__ __forceinline__ Words<8 * T::kBytes> numbers(uint32_t codes, float scale) {
    Words<8 * T::kBytes> y;
#define TDE_PAIR(CONVERT, BYTE) __builtin_bit_cast(uint32_t, CONVERT(codes, scale, BYTE))
    if constexpr (T::kBytes == 4) {
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
        const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
        const float all[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
        y = narrow_all<F32, 8>(all);
    } else if constexpr (__is_same(T, Bf16)) {
        y = {{TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, 0), TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, 1),
              TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, 2), TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, 3)}};
    } else {
        y = {{TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, 0), TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, 1),
              TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, 2), TDE_PAIR(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, 3)}};
    }
#undef TDE_PAIR
    return y;
}

} // namespace

template <class T>
__global__ void __launch_bounds__(256) unpack_fp4_kernel(const UnpackArgs a) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.total) return;
    const uint32_t row = a.pieces.quotient(i), piece = i - row * a.pieces.d;
    const uint32_t outer = a.inner.quotient(row), n2 = row - outer * a.inner.d, n0 = a.middle.quotient(outer), n1 = outer - n0 * a.middle.d;
    const Words<4> codes = load_words<4>(a.codes + n0 * a.code_stride[0] + n1 * a.code_stride[1] + n2 * a.code_stride[2] + piece * 4);
    const uint32_t scale = *(const __attribute__((address_space(1))) uint8_t *)(a.scales + n0 * a.scale_stride[0] + n1 * a.scale_stride[1] +
                                                                               n2 * a.scale_stride[2] + piece / 4);
    store_words<8 * T::kBytes, true>(a.out + (uint64_t)i * (8 * T::kBytes), numbers<T>(codes.w[0], __builtin_bit_cast(float, scale << 23)));
}

int launch_unpack_fp4(const UnpackArgs &a, int out_dtype, hipStream_t s) {
    const uint32_t blocks = ((uint32_t)a.total + 255) / 256;
    if (out_dtype == TDE_BF16) unpack_fp4_kernel<Bf16><<<blocks, 256, 0, s>>>(a);
    else if (out_dtype == TDE_F16) unpack_fp4_kernel<F16><<<blocks, 256, 0, s>>>(a);
    else unpack_fp4_kernel<F32><<<blocks, 256, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace block
} // namespace tde
