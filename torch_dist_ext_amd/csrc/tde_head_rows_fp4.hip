// Rows of one head each into a paged cache in 4 bits: norm and rotation as in tde_head_rows.hip, then for every 32 channels of a key or a value
//
//   e = exponent of (the largest magnitude rounded to two significant bits) - 2      clamped; a power of two that the codes are multiplied by
//   code = e2m1(x / 2^e)                                                             to nearest even, 6 at most
//
// The rounded exponent lets a block's largest value be 3.5 to 7 of its units: from 7 on the next unit's 4 is as near as 6 is.  (Blocks of normally distributed
// numbers: error 0.112 relative, 0.115 with a unit that is never too small or that the largest value's power of two gives by itself.)
//
// A code is the one nearest to the exact value only if that is known to which side of a border between two codes it lies, and a border can be missed by any
// rounding on the way.  Keys are therefore normed and rotated in doubles (vector instructions on doubles run at half the rate of floats' here, and memory sets the time), and
// what is left is cut to 32 bits with its last bit set where anything was cut off: no border of codes, which have three significant bits, lies between.  The
// hardware's conversion then rounds once.
//
// Bound by memory: a row is read once, 16 bytes a lane, with its partner in the rotation, which comes from the nearest cache.
#include "tde_block.h"
#include "tde_head_rows.h"

namespace tde {
namespace block {

namespace {

__device__ __forceinline__ double sum_over_lanes(double x, int log2) {
    for (int m = 0; m < log2; ++m) x += __shfl_xor(x, 1 << m);
    return x;
}

// x cut to 32 bits, the last bit set if that took anything off.
__device__ __forceinline__ float cut(double x) {
    const float near = (float)x;
    const double back = near;
    uint32_t bits = __builtin_bit_cast(uint32_t, near);
    if (back != x) bits = (bits - (uint32_t)(__builtin_fabs(back) > __builtin_fabs(x))) | 1u;
    return __builtin_bit_cast(float, bits);
}

__device__ __forceinline__ float multiply_add(float x, float y, float z) { return __builtin_fmaf(x, y, z); }
__device__ __forceinline__ double multiply_add(double x, double y, double z) { return __builtin_fma(x, y, z); }

// Norm and rotation of a lane's eight channels x; y are their partners in the rotation, c and s (with the sign that the channel takes it) theirs.
template <class A>
struct Channels {
    A x[8], y[8];
};
template <class A>
__device__ __forceinline__ void norm_and_turn(Channels<A> &v, bool normed, const float (&gx)[8], const float (&gy)[8], int dim, float eps, int lanes_log2,
                                              uint32_t turned, const float (&c)[8], const float (&s)[8]) {
    if (normed) {
        A sq = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += v.x[i] * v.x[i];
        sq = sum_over_lanes(sq, lanes_log2);
        const A scale = (A)1 / (sizeof(A) == 8 ? (A)__builtin_sqrt((double)(sq / (A)dim + (A)eps)) : (A)__builtin_sqrtf((float)(sq / (A)dim + (A)eps)));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v.x[i] = v.x[i] * scale * (A)gx[i];
            v.y[i] = v.y[i] * scale * (A)gy[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if ((turned >> i) & 1) v.x[i] = multiply_add(v.x[i], (A)c[i], v.y[i] * (A)s[i]);
}

} // namespace

// A lane has eight channels, four neighbouring lanes a block; rows of a token share a wavefront.
// WHOLE: chunks of eight channels lie in one half of the rotation, or behind it.
template <class T, bool INTERLEAVED, bool WHOLE>
__global__ void __launch_bounds__(256) head_rows_fp4_kernel(const HeadRowsFp4Args a) {
    constexpr int BYTES = 8 * T::kBytes;
    const int lane = threadIdx.x & 63;
    const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = a.waves_per_token.quotient(wave);
    const int64_t token = row;
    if (token >= a.tokens) return;
    const int part = (int)(wave - row * a.waves_per_token.d);
    const int place = lane & ((1 << a.lanes_log2) - 1), d0 = place * 8;
    const bool has = d0 < a.dim;
    int h = part * (64 >> a.lanes_log2) + (lane >> a.lanes_log2);
    const bool there = h < a.heads[0] + a.heads[1] + a.heads[2];
    const int cls = h < a.heads[0] ? 0 : (h < a.heads[0] + a.heads[1] ? 1 : 2);
    h -= cls == 0 ? 0 : (cls == 1 ? a.heads[0] : a.heads[0] + a.heads[1]);
    const char *src = cls == 0 ? a.in[0] : (cls == 1 ? a.in[1] : a.in[2]);
    src += token * (cls == 0 ? a.in_token[0] : (cls == 1 ? a.in_token[1] : a.in_token[2]));
    src += h * (cls == 0 ? a.in_head[0] : (cls == 1 ? a.in_head[1] : a.in_head[2]));

    // Partners.  Not interleaved: the same channels of the rotation's other half, which are one chunk where halves are whole ones.
    const int rot = 2 * a.half;
    const bool apart = !INTERLEAVED && cls != 2 && there && has && d0 < rot;
    const int to_partner = d0 < a.half ? a.half : -a.half;
    Words<BYTES> own{}, other{};
    if (there && has) own = load_words<BYTES>(src + d0 * T::kBytes);
    if (WHOLE && apart) other = load_words<BYTES>(src + (d0 + to_partner) * T::kBytes);

    const Place where = place_of(a.batch, token, lane);
    const int64_t position = a.positions != nullptr ? explicit_position(a, token) : where.position;
    const bool known = position >= 0 && position < a.table_rows;
    const float *const row_of = a.cos_sin + (known ? position : 0) * a.table_stride;
    const char *const gamma = cls == 2 ? nullptr : (cls == 0 ? a.gamma[0] : a.gamma[1]);

    float x[8], y[8], gx[8] = {}, gy[8] = {}, c[8] = {}, s[8] = {};
    widen_all<T, 8>(own, x);
    widen_all<T, 8>(other, y);
    uint32_t turned = 0; // channels that are rotated, a bit each
    if (there && has && cls != 2) {
        if (gamma != nullptr) widen_all<T, 8>(load_words<BYTES>(gamma + d0 * T::kBytes), gx);
        if constexpr (!WHOLE) { // channel by channel
            for (int i = 0; i < 8; ++i) {
                const int d = d0 + i;
                if (d >= rot) break;
                const bool first = INTERLEAVED ? (d & 1) == 0 : d < a.half;
                const int j = INTERLEAVED ? d >> 1 : (first ? d : d - a.half), partner = INTERLEAVED ? d ^ 1 : (first ? d + a.half : d - a.half);
                const float sine = known ? row_of[a.half + j] : __builtin_nanf("");
                y[i] = load_element<T>(src + partner * T::kBytes);
                if (gamma != nullptr) gy[i] = load_element<T>(gamma + partner * T::kBytes);
                c[i] = known ? row_of[j] : __builtin_nanf("");
                s[i] = first ? -sine : sine;
                turned |= 1u << i;
            }
        } else if (d0 < rot) {
            turned = 0xff;
            if constexpr (INTERLEAVED) {
                float cosines[4], sines[4];
                load_floats(row_of + d0 / 2, known, cosines);
                load_floats(row_of + a.half + d0 / 2, known, sines);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[i] = x[i ^ 1];
                    gy[i] = gx[i ^ 1];
                    c[i] = cosines[i >> 1];
                    s[i] = (i & 1) == 0 ? -sines[i >> 1] : sines[i >> 1];
                }
            } else {
                if (gamma != nullptr) widen_all<T, 8>(load_words<BYTES>(gamma + (d0 + to_partner) * T::kBytes), gy);
                const int j = d0 < a.half ? d0 : d0 - a.half;
                load_floats(row_of + j, known, c);
                load_floats(row_of + a.half + j, known, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] = d0 < a.half ? -s[i] : s[i];
            }
        }
    }

    if (cls == 0) {
        Channels<float> v;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v.x[i] = x[i];
            v.y[i] = y[i];
        }
        norm_and_turn(v, gamma != nullptr, gx, gy, a.dim, a.eps, a.lanes_log2, turned, c, s);
        if (!there || !has) return;
        Words<BYTES> out = narrow_all<T, 8>(v.x);
        if (where.position < 0) out = Words<BYTES>{};
        store_words<BYTES>(a.out[0] + token * a.out_token[0] + h * a.out_head[0] + d0 * T::kBytes, out);
        return;
    }
    if (cls == 1) {
        Channels<double> v;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v.x[i] = x[i];
            v.y[i] = y[i];
        }
        norm_and_turn(v, gamma != nullptr, gx, gy, a.dim, a.eps, a.lanes_log2, turned, c, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = cut(v.x[i]);
    }
    uint32_t largest = 0; // magnitudes compare as whole numbers, infinities and NaN above all
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, __builtin_bit_cast(uint32_t, x[i]) & 0x7fffffffu);
    largest = max(largest, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)largest, 0xB1, 0xf, 0xf, false));
    largest = max(largest, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)largest, 0x4E, 0xf, 0xf, false));
    const bool finite = largest < 0x7f800000u;
    const int exponent = (int)((largest + 0x00200000u) >> 23) - 2;
    const uint32_t scale = finite ? (uint32_t)min(max(exponent, 2), a.most_exponent + 127) : 255u;
    const float unit = __builtin_bit_cast(float, scale << 23);
    uint32_t codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], unit, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], unit, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], unit, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], unit, 3);
    if (!there || !has || where.page < 0) return;
    const auto &late = arguments_again<HeadRowsFp4Args>();
    const int i = cls - 1;
    char *const to = (i == 0 ? late.out[1] : late.out[2]) + where.page * (i == 0 ? late.out_page[1] : late.out_page[2]) +
                     where.slot * (i == 0 ? late.out_token[1] : late.out_token[2]) + h * (i == 0 ? late.out_head[1] : late.out_head[2]);
    store_words<4>(to + d0 / 2, Words<4>{{finite ? codes : 0u}});
    if ((place & 3) == 0) {
        char *const scale_to = (i == 0 ? late.scales[0] : late.scales[1]) + where.page * (i == 0 ? late.scale_page[0] : late.scale_page[1]) +
                               where.slot * (i == 0 ? late.scale_slot[0] : late.scale_slot[1]) + h * (i == 0 ? late.scale_head[0] : late.scale_head[1]);
        *(__attribute__((address_space(1))) uint8_t *)(scale_to + place / 4) = (uint8_t)scale;
    }
}

int launch_head_rows_fp4(HeadRowsFp4Args &a, int dtype, hipStream_t s) {
    const int64_t heads_all = (int64_t)a.heads[0] + a.heads[1] + a.heads[2];
    if (a.tokens == 0 || heads_all == 0) return TDE_OK;
    a.lanes_log2 = 2;
    while ((8 << a.lanes_log2) < a.dim) ++a.lanes_log2;
    const int64_t at_once = 64 >> a.lanes_log2, waves = (heads_all + at_once - 1) / at_once;
    if (a.tokens > (int64_t)0x7ffffff0 / waves) return TDE_ETOOBIG;
    const uint32_t blocks = (uint32_t)((a.tokens * waves + 3) / 4);
    if (!fits_launch(blocks, 256)) return TDE_ETOOBIG;
    a.waves_per_token = Divisor32((uint32_t)waves);
    const bool whole = (a.interleaved ? 2 * a.half : a.half) % 8 == 0;
    const auto launch = [&](auto type) {
        using T = decltype(type);
        if (a.interleaved && whole) head_rows_fp4_kernel<T, true, true><<<blocks, 256, 0, s>>>(a);
        else if (a.interleaved) head_rows_fp4_kernel<T, true, false><<<blocks, 256, 0, s>>>(a);
        else if (whole) head_rows_fp4_kernel<T, false, true><<<blocks, 256, 0, s>>>(a);
        else head_rows_fp4_kernel<T, false, false><<<blocks, 256, 0, s>>>(a);
    };
    if (dtype == TDE_BF16) launch(Bf16{});
    else if (dtype == TDE_F16) launch(F16{});
    else if (dtype == TDE_F32) launch(F32{});
    else return TDE_EDTYPE;
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace block
} // namespace tde
