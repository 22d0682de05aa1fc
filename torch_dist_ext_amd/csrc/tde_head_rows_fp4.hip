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
// A row is read once, 16 bytes a lane, with its partner in the rotation, which comes from the nearest cache.  8192 tokens of 32 + 2 * 8 heads of 128
// fp16 channels, a half of them rotated, take 38 us, 4.6 TB/s: vector instructions take 21 us of it, and the waits for rows, a token's sequence and place the
// rest.  Rows of one kind to an instruction, queries written past the caches and doubles of one channel at a time brought it there from 60.
#include "tde_block.h"
#include "tde_head_rows.h"

#include <type_traits>

namespace tde {
namespace block {

namespace {

template <int CONTROL>
__device__ __forceinline__ float from_lane(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CONTROL, 0xf, 0xf, false));
}
template <int CONTROL>
__device__ __forceinline__ double from_lane(double x) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, x);
    const uint32_t low = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, CONTROL, 0xf, 0xf, false);
    const uint32_t high = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), CONTROL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)high << 32 | low);
}
// Over 4, 8, 16 or 32 neighbouring lanes, the same sum in each.
template <class A>
__device__ __forceinline__ A sum_over_lanes(A x, int log2) {
    x += from_lane<0xb1>(x);               // the neighbour's
    x += from_lane<0x4e>(x);               // the other two's of four
    if (log2 > 2) x += from_lane<0x141>(x); // mirrored in eight
    if (log2 > 3) x += from_lane<0x140>(x); // in sixteen
    if (log2 > 4) x += __shfl_xor(x, 16);
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

typedef float f32x8 __attribute__((ext_vector_type(8)));

// x as if it were new here, behind what was new before: what follows from it is not computed any earlier.
__device__ __forceinline__ float in_turn(float x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Norm and rotation of a lane's eight channels x; y are their partners in the rotation, c and s (with the sign that the channel takes it) theirs.
template <bool WHOLE>
__device__ __forceinline__ void norm_and_turn(float (&x)[8], const float (&y)[8], bool normed, const float (&gx)[8], const float (&gy)[8], int dim, float eps,
                                              int lanes_log2, uint32_t turned, f32x8 c, f32x8 s) {
    float scale = 1.0f;
    if (normed) {
        float sq = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
        scale = 1.0f / __builtin_sqrtf(sum_over_lanes(sq, lanes_log2) / (float)dim + eps);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float other = y[i];
        if (normed) {
            x[i] = x[i] * scale * gx[i];
            other = other * scale * gy[i];
        }
        // (partners are taken from y: x's own are those of other channels)
        if (WHOLE ? turned != 0 : ((turned >> i) & 1) != 0) x[i] = __builtin_fmaf(x[i], c[i], other * s[i]);
    }
}
// The same in doubles, cut: one channel after the other, as all at once they would take the registers of twice as many wavefronts.
template <bool WHOLE>
__device__ __forceinline__ void norm_and_turn_exactly(float (&x)[8], const float (&y)[8], bool normed, const float (&gx)[8], const float (&gy)[8], int dim, float eps,
                                                      int lanes_log2, uint32_t turned, f32x8 c, f32x8 s) {
    double scale = 1.0;
    if (normed) {
        double sq = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const double own = in_turn(x[i]);
            sq += own * own;
        }
        scale = 1.0 / __builtin_sqrt(sum_over_lanes(sq, lanes_log2) / (double)dim + (double)eps);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        double own = in_turn(x[i]), other = in_turn(y[i]);
        if (normed) {
            own = own * scale * (double)in_turn(gx[i]);
            other = other * scale * (double)in_turn(gy[i]);
        }
        if (WHOLE ? turned != 0 : ((turned >> i) & 1) != 0) own = __builtin_fma(own, (double)in_turn(c[i]), other * (double)in_turn(s[i]));
        x[i] = in_turn(cut(own));
    }
}

// place_of, whose chain of loads is one shorter where a lane has a sequence of its own.
__device__ __forceinline__ Place place_at_once(const PagedBatch &b, int64_t token, int lane) {
    if (b.seqs > 64) return place_of(b, token, lane);
    const int mine = min(lane, b.seqs - 1);
    int32_t begin = 0, end = 0, len = 0;
    if (mine >= 0) {
        begin = b.starts[mine];
        end = b.starts[mine + 1];
        len = b.lens[mine];
    }
    Place p{-1, -1, 0};
    const int seq = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < b.seqs && end <= token));
    if (seq >= b.seqs) return p;
    const int64_t first = __builtin_amdgcn_readlane(begin, seq);
    if (token < first) return p;
    p.position = (int64_t)__builtin_amdgcn_readlane(len, seq) - (__builtin_amdgcn_readlane(end, seq) - first) + (token - first);
    if (p.position < 0 || p.position > 0x7fffffff) return p; // the latter only where starts do not ascend
    const uint32_t at = b.page.quotient((uint32_t)p.position);
    p.slot = (int32_t)((uint32_t)p.position - at * b.page.d);
    p.page = page_number(b, b.table + seq * b.table_stride, at);
    return p;
}

} // namespace

// A lane has eight channels of R rows of one token, which share their cosines, sines, gammas and place; four neighbouring lanes have a block.  As many
// rows as a wavefront has at once are of one kind: queries, keys or values, so that nothing but the row's head differs between lanes.
// WHOLE: chunks of eight channels lie in one half of the rotation, or behind it.
template <class T, bool INTERLEAVED, bool WHOLE, int R>
__global__ void __launch_bounds__(256) head_rows_fp4_kernel(const HeadRowsFp4Args a) {
    constexpr int BYTES = 8 * T::kBytes;
    const int lane = threadIdx.x & 63;
    const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = a.waves_per_token.quotient(wave);
    const int64_t token = row;
    if (token >= a.tokens) return;
    int round = (int)(wave - row * a.waves_per_token.d) * (R > 1 ? R * a.turns : 1);
    const int place = lane & ((1 << a.lanes_log2) - 1), d0 = place * 8;
    const bool has = d0 < a.dim;
    const int rot = 2 * a.half;
    // Partners.  Not interleaved: the same channels of the rotation's other half, which are one chunk where halves are whole ones.
    const bool turned_apart = !INTERLEAVED && WHOLE && d0 < rot;
    const int to_partner = d0 < a.half ? a.half : -a.half;

    Words<BYTES> own[R], other[R];
    const char *source[R];
    int cls[R], head[R]; // query, key, value; -1: no row
    const auto load = [&] { // the rows from `round` on
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int of_q = a.rounds[0], of_k = a.rounds[1];
            cls[r] = round + r < of_q ? 0 : (round + r < of_q + of_k ? 1 : 2);
            const int h = ((round + r - (cls[r] == 0 ? 0 : (cls[r] == 1 ? of_q : of_q + of_k))) << (6 - a.lanes_log2)) + (lane >> a.lanes_log2);
            const bool there = h < (cls[r] == 0 ? a.heads[0] : (cls[r] == 1 ? a.heads[1] : a.heads[2])) && has;
            head[r] = there ? h : -1;
            const auto &late = arguments_again<HeadRowsFp4Args>();
            source[r] = late.in[cls[r]] + token * late.in_token[cls[r]] + h * late.in_head[cls[r]];
            own[r] = Words<BYTES>{};
            if (there) own[r] = load_words<BYTES, (R > 1)>(source[r] + d0 * T::kBytes);
            if constexpr (!INTERLEAVED && WHOLE) {
                other[r] = Words<BYTES>{};
                if (there && turned_apart && cls[r] != 2) other[r] = load_words<BYTES>(source[r] + (d0 + to_partner) * T::kBytes);
            }
        }
    };
    load();

    const Place where = place_at_once(a.batch, token, lane);
    const int64_t position = a.positions != nullptr ? explicit_position(a, token) : where.position;
    const bool known = position >= 0 && position < a.table_rows;
    const float *const row_of = a.cos_sin + (known ? position : 0) * a.table_stride;

    // Cosines and sines (with the sign that the channel takes them) of the lane's channels.
    f32x8 c = {}, s = {};
    uint32_t turned = 0; // channels that are rotated, a bit each
    if constexpr (!WHOLE) {
        for (int i = 0; i < 8; ++i) {
            const int d = d0 + i;
            if (d >= rot) break;
            const bool first = INTERLEAVED ? (d & 1) == 0 : d < a.half;
            const int j = INTERLEAVED ? d >> 1 : (first ? d : d - a.half);
            const float sine = known ? row_of[a.half + j] : __builtin_nanf("");
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
                c[i] = cosines[i >> 1];
                s[i] = (i & 1) == 0 ? -sines[i >> 1] : sines[i >> 1];
            }
        } else {
            const int j = d0 < a.half ? d0 : d0 - a.half;
            float cosines[8], sines[8];
            load_floats(row_of + j, known, cosines);
            load_floats(row_of + a.half + j, known, sines);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                c[i] = cosines[i];
                s[i] = d0 < a.half ? -sines[i] : sines[i];
            }
        }
    }
    const auto gammas_at = [&](const char *from, int d, bool wanted) {
        Words<BYTES> w{};
        if (from != nullptr && has && wanted) w = load_words<BYTES>(from + d * T::kBytes);
        return w;
    };
    constexpr int K = R > 1 ? 1 : 0; // gammas of queries and of keys, or of the only row
    Words<BYTES> gamma[K + 1], other_gamma[K + 1];
#pragma unroll
    for (int i = 0; i <= K; ++i) {
        const char *const of = R > 1 ? a.gamma[i] : (cls[0] == 0 ? a.gamma[0] : (cls[0] == 1 ? a.gamma[1] : nullptr));
        gamma[i] = gammas_at(of, d0, true);
        other_gamma[i] = gammas_at(of, d0 + to_partner, turned_apart);
    }

    for (int turn = 0;;) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x[8];
            widen_all<T, 8>(own[r], x);
            const auto norm_and_turn_row = [&](auto exactly, const char *from, const Words<BYTES> &own_gamma, const Words<BYTES> &other_gamma) {
                float y[8] = {}, gx[8], gy[8];
                if constexpr (!INTERLEAVED && WHOLE) widen_all<T, 8>(other[r], y);
                widen_all<T, 8>(own_gamma, gx);
                widen_all<T, 8>(other_gamma, gy);
                if constexpr (INTERLEAVED) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        y[i] = x[i ^ 1];
                        gy[i] = gx[i ^ 1];
                    }
                } else if constexpr (!WHOLE) { // one by one
                    if (head[r] >= 0)
                        for (int i = 0; i < 8; ++i) {
                            if (((turned >> i) & 1) == 0) break;
                            const int partner = d0 + i < a.half ? d0 + i + a.half : d0 + i - a.half;
                            y[i] = load_element<T>(source[r] + partner * T::kBytes);
                            if (from != nullptr) gy[i] = load_element<T>(from + partner * T::kBytes);
                        }
                }
                if constexpr (decltype(exactly)::value) norm_and_turn_exactly<WHOLE>(x, y, from != nullptr, gx, gy, a.dim, a.eps, a.lanes_log2, turned, c, s);
                else norm_and_turn<WHOLE>(x, y, from != nullptr, gx, gy, a.dim, a.eps, a.lanes_log2, turned, c, s);
            };
            if (cls[r] == 0) {
                norm_and_turn_row(std::false_type{}, a.gamma[0], gamma[0], other_gamma[0]);
                if (head[r] >= 0) {
                    Words<BYTES> out = narrow_all<T, 8>(x);
                    if (where.position < 0) out = Words<BYTES>{};
                    store_words<BYTES, (R > 1)>(a.out[0] + token * a.out_token[0] + head[r] * a.out_head[0] + d0 * T::kBytes, out);
                }
                continue;
            }
            if (cls[r] == 1) norm_and_turn_row(std::true_type{}, a.gamma[1], gamma[K], other_gamma[K]);
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
            if (head[r] < 0 || where.page < 0) continue;
            const auto &late = arguments_again<HeadRowsFp4Args>();
            char *const to = late.out[cls[r]] + where.page * late.out_page[cls[r]] + where.slot * late.out_token[cls[r]] + head[r] * late.out_head[cls[r]];
            store_words<4>(to + d0 / 2, Words<4>{{finite ? codes : 0u}});
            if ((place & 3) == 0) {
                const int i = cls[r] - 1;
                char *const scale_to = late.scales[i] + where.page * late.scale_page[i] + where.slot * late.scale_slot[i] + head[r] * late.scale_head[i];
                *(__attribute__((address_space(1))) uint8_t *)(scale_to + place / 4) = (uint8_t)scale;
            }
        }
        if (R == 1 || ++turn == a.turns) break;
        round += R;
        load();
    }
}

int launch_head_rows_fp4(HeadRowsFp4Args &a, int dtype, hipStream_t s) {
    const int64_t heads_all = (int64_t)a.heads[0] + a.heads[1] + a.heads[2];
    if (a.tokens == 0 || heads_all == 0) return TDE_OK;
    a.lanes_log2 = 2;
    while ((8 << a.lanes_log2) < a.dim) ++a.lanes_log2;
    for (int i = 0; i < 3; ++i) a.rounds[i] = (a.heads[i] + (64 >> a.lanes_log2) - 1) >> (6 - a.lanes_log2);
    const int64_t rounds = (int64_t)a.rounds[0] + a.rounds[1] + a.rounds[2];
    const auto waves_of = [&](int rows) { return (rounds + rows - 1) / rows; };
    const bool whole = (a.interleaved ? 2 * a.half : a.half) % 8 == 0;
    // Rows of a lane, and how often it takes as many, which then share what a token has in common.  8192 tokens of 32 + 2 * 8 heads of 128 bf16 channels, and the
    // caches' unpacking behind them, take 63 us with four rows three times, 74 with four once and 85 with one; 2048 tokens 27, 29 and 28; fp32 rows take 63 with one and 77 with four (4096 tokens), whose registers are too many.  Few rows are for all units.
    const int rows = whole && dtype != TDE_F32 && a.tokens * waves_of(4) >= 1024 ? 4 : 1;
    const int64_t all = waves_of(rows), least = rows == 1 ? all : std::min(all, std::max<int64_t>(1, 4096 / a.tokens)); // wavefronts of a token
    a.turns = (int32_t)((all + least - 1) / least);
    const int64_t waves = (all + a.turns - 1) / a.turns;
    if (a.tokens > (int64_t)0x7ffffff0 / waves) return TDE_ETOOBIG;
    const uint32_t blocks = (uint32_t)((a.tokens * waves + 3) / 4);
    if (!fits_launch(blocks, 256)) return TDE_ETOOBIG;
    a.waves_per_token = Divisor32((uint32_t)waves);
    const auto launch = [&](auto type) {
        using T = decltype(type);
        if (!whole && a.interleaved) head_rows_fp4_kernel<T, true, false, 1><<<blocks, 256, 0, s>>>(a);
        else if (!whole) head_rows_fp4_kernel<T, false, false, 1><<<blocks, 256, 0, s>>>(a);
        else if (rows == 1 && a.interleaved) head_rows_fp4_kernel<T, true, true, 1><<<blocks, 256, 0, s>>>(a);
        else if (rows == 1) head_rows_fp4_kernel<T, false, true, 1><<<blocks, 256, 0, s>>>(a);
        else if constexpr (T::kBytes == 2) {
            if (a.interleaved) head_rows_fp4_kernel<T, true, true, 4><<<blocks, 256, 0, s>>>(a);
            else head_rows_fp4_kernel<T, false, true, 4><<<blocks, 256, 0, s>>>(a);
        }
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
