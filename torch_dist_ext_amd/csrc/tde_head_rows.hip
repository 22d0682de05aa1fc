// Rows of one head each: RMSNorm over the head's channels, the position rotation, and where the row goes -- a dense output or a slot
// of a paged cache.  One kernel family serves tde_qk_norm_rope and tde_append_kv.
//
//   u = x * 1/sqrt(mean(x^2) + eps) * gamma       in fp32 (left out without a gamma)
//   (a, b) -> (a cos - b sin, b cos + a sin)      for the rotated channels' pairs: (d, d + rot/2), or (2d, 2d + 1) if interleaved
//   T(.)                                          one rounding, at the end; the sum of squares is held in fp32
//
// Bound by memory: every row is read and written once.  A lane has two chunks of 16 bytes of a row (8 where the head's length or the
// rotation's halves need it), so several rows share a wavefront.  All rows of a wavefront belong to one token: its position, its row of the
// rotation's table and its page are looked up once, with scalar or shared loads, while the rows are on their way.
#include "tde_block.h"
#include "tde_head_rows.h"

namespace tde {
namespace block {

// The token's place: its sequence's cache position and the slot's page.  position < 0: the row belongs to no sequence's range (it
// lies in front of the first one or behind the last, or its sequence is shorter than its new tokens).
struct Place {
    int64_t position;
    int32_t page, slot; // page < 0: not in the cache
};

__device__ __forceinline__ Place place_of(const PagedBatch &b, int64_t token, int lane) {
    Place p{-1, -1, 0};
    const int seq = __builtin_amdgcn_readfirstlane(sequence_of(b, token, lane));
    if (seq >= b.seqs) return p;
    const int64_t begin = b.starts[seq], end = b.starts[seq + 1], len = b.lens[seq];
    if (token < begin) return p;
    p.position = len - (end - begin) + (token - begin);
    if (p.position < 0) return p;
    if (p.position > 0x7fffffff) return p; // only where starts do not ascend
    const uint32_t at = b.page.quotient((uint32_t)p.position);
    p.slot = (int32_t)((uint32_t)p.position - at * b.page.d);
    p.page = page_number(b, b.table + seq * b.table_stride, at);
    return p;
}

__device__ __forceinline__ int64_t explicit_position(const HeadRowsArgs &a, int64_t token) {
    return a.positions_wide ? ((const int64_t *)a.positions)[token] : (int64_t)((const int32_t *)a.positions)[token];
}

// Address of head `h` of class `cls` (0 query, 1 key, 2 value) in the outputs; null where the row is not stored.
template <bool PAGED>
__device__ __forceinline__ char *destination(const HeadRowsArgs &a, const Place &place, int64_t token, int cls, int h) {
    if (!PAGED || cls == 0) return a.out[cls] + token * a.out_token[cls] + h * a.out_head[cls];
    if (place.page < 0) return nullptr;
    return a.out[cls] + place.page * a.out_page[cls] + place.slot * a.out_token[cls] + h * a.out_head[cls];
}

// VE floats of the table; NaN where the position is not in it.
template <int N>
__device__ __forceinline__ void load_floats(const float *p, bool known, float (&x)[N]) {
    Words<N * 4> w;
#pragma unroll
    for (int i = 0; i < N; ++i) w.w[i] = 0x7fc00000u;
    if (known) w = load_words<N * 4>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __builtin_bit_cast(float, w.w[i]);
}

// A lane has two chunks of VE channels of a row: chunk p and its partner in the other half of the rotation, or, behind the rotated
// channels and with interleaved pairs, one in each half of what there is (neighbouring lanes then load neighbouring chunks; with two
// neighbours a lane, a chunk of 8192 rows took 53 us in place of 40).  Rotating needs no other lane, and R rows of a token share
// the lane's cosines, sines and gammas.
template <class T, int VE, int R, bool INTERLEAVED, bool PAGED, bool STREAM>
__global__ void __launch_bounds__(256) head_rows_kernel(const HeadRowsArgs a) {
    constexpr int BYTES = VE * T::kBytes;
    const int lane = threadIdx.x & 63;
    const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = a.waves_per_token.quotient(wave);
    const int64_t token = row;
    if (token >= a.tokens) return;
    const int part = (int)(wave - row * a.waves_per_token.d);
    const int rows_at_once = 64 >> a.lanes_log2;
    const int place = lane & ((1 << a.lanes_log2) - 1);
    const int pairs = a.half / VE; // lanes with a partner in the other half
    const int chunks = a.dim / VE;
    const int rest = INTERLEAVED ? 0 : 2 * pairs; // first of the chunks without a partner, in halves of `apart`
    const int apart = (chunks - rest + 1) / 2;
    int c0 = place, c1 = place + pairs;
    if (INTERLEAVED || place >= pairs) {
        const int u = place - (INTERLEAVED ? 0 : pairs);
        c0 = u < apart ? rest + u : chunks;
        c1 = u < apart ? rest + u + apart : chunks;
    }
    const bool has0 = c0 < chunks, has1 = c1 < chunks;
    const int at0 = c0 * BYTES, at1 = c1 * BYTES;
    const int heads = a.heads[0] + a.heads[1] + a.heads[2];

    Words<BYTES> raw[R][2];
    int cls[R], head[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        int h = (part * R + r) * rows_at_once + (lane >> a.lanes_log2);
        const bool there = h < heads;
        cls[r] = h < a.heads[0] ? 0 : (h < a.heads[0] + a.heads[1] ? 1 : 2);
        h -= cls[r] == 0 ? 0 : (cls[r] == 1 ? a.heads[0] : a.heads[0] + a.heads[1]);
        head[r] = there ? h : -1;
        const char *src = cls[r] == 0 ? a.in[0] : (cls[r] == 1 ? a.in[1] : a.in[2]);
        const int64_t per_token = cls[r] == 0 ? a.in_token[0] : (cls[r] == 1 ? a.in_token[1] : a.in_token[2]);
        const int64_t per_head = cls[r] == 0 ? a.in_head[0] : (cls[r] == 1 ? a.in_head[1] : a.in_head[2]);
        src += token * per_token + h * per_head;
        raw[r][0] = raw[r][1] = Words<BYTES>{};
        if (there && has0) raw[r][0] = load_words<BYTES, STREAM>(src + at0);
        if (there && has1) raw[r][1] = load_words<BYTES, STREAM>(src + at1);
    }

    Place where{0, -1, 0};
    if (PAGED) where = place_of(a.batch, token, lane);
    const bool placed = !PAGED || where.position >= 0;
    const int64_t position = a.positions != nullptr ? explicit_position(a, token) : where.position;

    // Cosines and sines of the lane's pairs.  Interleaved: the first half of them belongs to the first chunk.
    const int rot = 2 * a.half;
    const bool turned0 = c0 * VE < rot, turned1 = has1 && c1 * VE < rot;
    float cs[VE], sn[VE];
    {
        const bool known = position >= 0 && position < a.table_rows;
        const float *const row_of = a.cos_sin + (known ? position : 0) * a.table_stride;
#pragma unroll
        for (int i = 0; i < VE; ++i) cs[i] = sn[i] = 0.0f;
        if constexpr (!INTERLEAVED) {
            if (turned0) {
                load_floats(row_of + place * VE, known, cs);
                load_floats(row_of + a.half + place * VE, known, sn);
            }
        } else {
            constexpr int N = VE / 2;
            const auto load_half = [&](int chunk, int from) {
                float c[N], s[N];
                load_floats(row_of + chunk * N, known, c);
                load_floats(row_of + a.half + chunk * N, known, s);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    cs[from + i] = c[i];
                    sn[from + i] = s[i];
                }
            };
            if (turned0) load_half(c0, 0);
            if (turned1) load_half(c1, N);
        }
    }
    Words<BYTES> gamma[2][2]{}; // of queries and keys
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        if (a.gamma[g] != nullptr && has0) gamma[g][0] = load_words<BYTES>(a.gamma[g] + at0);
        if (a.gamma[g] != nullptr && has1) gamma[g][1] = load_words<BYTES>(a.gamma[g] + at1);
    }

#pragma unroll
    for (int r = 0; r < R; ++r) {
        float x0[VE], x1[VE];
        widen_all<T, VE>(raw[r][0], x0);
        widen_all<T, VE>(raw[r][1], x1);
        if (a.gamma[0] != nullptr || a.gamma[1] != nullptr) {
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < VE; ++i) sq = __builtin_fmaf(x0[i], x0[i], sq);
#pragma unroll
            for (int i = 0; i < VE; ++i) sq = __builtin_fmaf(x1[i], x1[i], sq);
            sq = sum_over_lanes(sq, a.lanes_log2);
            const float scale = 1.0f / __builtin_sqrtf(sq / (float)a.dim + a.eps);
            const bool normed = cls[r] == 0 ? a.gamma[0] != nullptr : (cls[r] == 1 && a.gamma[1] != nullptr);
            float g0[VE], g1[VE];
            {
                Words<BYTES> w0, w1;
#pragma unroll
                for (int i = 0; i < BYTES / 4; ++i) {
                    w0.w[i] = cls[r] == 0 ? gamma[0][0].w[i] : gamma[1][0].w[i];
                    w1.w[i] = cls[r] == 0 ? gamma[0][1].w[i] : gamma[1][1].w[i];
                }
                widen_all<T, VE>(w0, g0);
                widen_all<T, VE>(w1, g1);
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                x0[i] = normed ? x0[i] * scale * g0[i] : x0[i];
                x1[i] = normed ? x1[i] * scale * g1[i] : x1[i];
            }
        }
        if constexpr (!INTERLEAVED) {
            if (turned0) {
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float u = x0[i], v = x1[i];
                    x0[i] = __builtin_fmaf(u, cs[i], -(v * sn[i]));
                    x1[i] = __builtin_fmaf(v, cs[i], u * sn[i]);
                }
            }
        } else {
            const auto turn = [&](float (&x)[VE], int from) {
#pragma unroll
                for (int i = 0; i < VE / 2; ++i) {
                    const float u = x[2 * i], v = x[2 * i + 1], c = cs[from + i], s = sn[from + i];
                    x[2 * i] = __builtin_fmaf(u, c, -(v * s));
                    x[2 * i + 1] = __builtin_fmaf(v, c, u * s);
                }
            };
            if (turned0) turn(x0, 0);
            if (turned1) turn(x1, VE / 2);
        }
        if (head[r] < 0) continue;
        Words<BYTES> y0 = narrow_all<T, VE>(x0), y1 = narrow_all<T, VE>(x1);
        if (cls[r] == 2) { // values go as they are
            y0 = raw[r][0];
            y1 = raw[r][1];
        }
        if (!placed) {
            if (cls[r] != 0) continue;
            y0 = y1 = Words<BYTES>{};
        }
        char *to = destination<PAGED>(a, where, token, cls[r], head[r]);
        if (to == nullptr) continue;
        if (has0) store_words<BYTES, STREAM>(to + at0, y0);
        if (has1) store_words<BYTES, STREAM>(to + at1, y1);
    }
}

// Any head length and rotation: a wavefront for each row, one element a lane at a time; the partner is read again (from the cache
// nearest to the unit).  Taken where no chunk of 8 bytes divides the head and the rotation's halves, and where a wavefront's lanes do not hold
// a row with two chunks each: more than 512 channels in fp32, or in 2-byte types where only chunks of 8 bytes divide them.
template <class T, bool INTERLEAVED, bool PAGED>
__global__ void __launch_bounds__(256) head_elements_kernel(const HeadRowsArgs a) {
    const int lane = threadIdx.x & 63;
    const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row = a.waves_per_token.quotient(wave); // one wavefront a head here
    const int64_t token = row;
    if (token >= a.tokens) return;
    int h = (int)(wave - row * a.waves_per_token.d);
    const int cls = h < a.heads[0] ? 0 : (h < a.heads[0] + a.heads[1] ? 1 : 2);
    h -= cls == 0 ? 0 : (cls == 1 ? a.heads[0] : a.heads[0] + a.heads[1]);
    const char *src = a.in[cls] + token * a.in_token[cls] + h * a.in_head[cls];

    Place place{0, -1, 0};
    if (PAGED) place = place_of(a.batch, token, lane);
    const bool placed = !PAGED || place.position >= 0;
    const int64_t position = a.positions != nullptr ? explicit_position(a, token) : place.position;
    const bool known = position >= 0 && position < a.table_rows;
    const float *row_of = a.cos_sin + (known ? position : 0) * a.table_stride;
    if (!placed && cls != 0) return;
    char *to = destination<PAGED>(a, place, token, cls, h);
    if (to == nullptr) return;

    const char *gamma = cls == 2 ? nullptr : a.gamma[cls];
    float scale = 1.0f;
    if (gamma != nullptr) {
        float sq = 0.0f;
        for (int d = lane; d < a.dim; d += 64) {
            const float x = load_element<T>(src + d * T::kBytes);
            sq = __builtin_fmaf(x, x, sq);
        }
        scale = 1.0f / __builtin_sqrtf(sum_over_lanes(sq, 6) / (float)a.dim + a.eps);
    }
    const auto normed = [&](int d) {
        const float x = load_element<T>(src + d * T::kBytes);
        return gamma != nullptr ? x * scale * load_element<T>(gamma + d * T::kBytes) : x;
    };
    for (int d = lane; d < a.dim; d += 64) {
        float y = normed(d);
        if (cls != 2 && d < 2 * a.half) {
            const bool first = INTERLEAVED ? (d & 1) == 0 : d < a.half;
            const int j = INTERLEAVED ? d >> 1 : (first ? d : d - a.half);
            const int other = INTERLEAVED ? d ^ 1 : (first ? d + a.half : d - a.half);
            const float c = known ? row_of[j] : __builtin_nanf(""), s = known ? row_of[a.half + j] : __builtin_nanf("");
            const float t = normed(other) * s;
            y = __builtin_fmaf(y, c, first ? -t : t);
        }
        if (!placed) y = 0.0f;
        store_element<T>(to + d * T::kBytes, y);
    }
}

namespace {

template <class T, int VE, int R, bool STREAM>
void launch_rows(const HeadRowsArgs &a, uint32_t blocks, hipStream_t s) {
    if (a.paged) {
        if (a.interleaved) head_rows_kernel<T, VE, R, true, true, STREAM><<<blocks, 256, 0, s>>>(a);
        else head_rows_kernel<T, VE, R, false, true, STREAM><<<blocks, 256, 0, s>>>(a);
    } else {
        if (a.interleaved) head_rows_kernel<T, VE, R, true, false, STREAM><<<blocks, 256, 0, s>>>(a);
        else head_rows_kernel<T, VE, R, false, false, STREAM><<<blocks, 256, 0, s>>>(a);
    }
}

template <class T>
void launch_elements(const HeadRowsArgs &a, uint32_t blocks, hipStream_t s) {
    if (a.paged) {
        if (a.interleaved) head_elements_kernel<T, true, true><<<blocks, 256, 0, s>>>(a);
        else head_elements_kernel<T, false, true><<<blocks, 256, 0, s>>>(a);
    } else {
        if (a.interleaved) head_elements_kernel<T, true, false><<<blocks, 256, 0, s>>>(a);
        else head_elements_kernel<T, false, false><<<blocks, 256, 0, s>>>(a);
    }
}

template <class T>
int launch_typed(HeadRowsArgs &a, const HeadRowsPlan &plan, hipStream_t s) {
    constexpr int V = 16 / T::kBytes;
    if (plan.chunk_bytes == 16) {
        switch (plan.rows) {
        case 1: launch_rows<T, V, 1, false>(a, plan.blocks, s); break;
        case 2: launch_rows<T, V, 2, true>(a, plan.blocks, s); break;
        case 3: launch_rows<T, V, 3, true>(a, plan.blocks, s); break;
        default: launch_rows<T, V, 5, true>(a, plan.blocks, s); break;
        }
    } else if (plan.chunk_bytes == 8) {
        launch_rows<T, V / 2, 1, false>(a, plan.blocks, s);
    } else {
        launch_elements<T>(a, plan.blocks, s);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace

// Which kernel, and its launch.  heads_all: rows a token has.
int plan_head_rows(int elem, int dim, int half, bool interleaved, int64_t tokens, int64_t heads_all, HeadRowsPlan *p) {
    p->chunk_bytes = 0;
    for (int bytes = 16; bytes >= 8; bytes /= 2) {
        const int ve = bytes / elem;
        if (dim % ve == 0 && (interleaved ? 2 * half : half) % ve == 0 && (dim / ve + 1) / 2 <= 64) {
            p->chunk_bytes = bytes;
            break;
        }
    }
    int64_t waves = heads_all; // a token
    p->lanes_log2 = 6;
    p->rows = 1;
    if (p->chunk_bytes != 0) {
        const int lanes = (dim * elem / p->chunk_bytes + 1) / 2;
        p->lanes_log2 = 0;
        while ((1 << p->lanes_log2) < lanes) ++p->lanes_log2;
        const int64_t at_once = 64 >> p->lanes_log2;
        const auto waves_of = [&](int rows) { return (heads_all + rows * at_once - 1) / (rows * at_once); };
        // Rows that share a lane's cosines and sines: as many as make the fewest wavefronts' work, counting those loads as two rows,
        // once there is work for every unit at least four times over; before that one, and more wavefronts.  (8192 tokens x 40 heads of 128: by 5
        // rows 35.0 us, 2 38.3, 3 38.0, 4 41.0; x 20 heads by 3 21.1, 2 23.5, 5 23.3.  4 is not built: where it would be taken, with 32 heads, it
        // is 31.1, 5 32.4.)
        if (p->chunk_bytes == 16 && tokens * waves_of(5) >= 4096) {
            int64_t best = 0;
            for (int rows : {2, 3, 5}) {
                const int64_t cost = waves_of(rows) * (rows + 2);
                if (best == 0 || cost < best) {
                    best = cost;
                    p->rows = rows;
                }
            }
        }
        waves = waves_of(p->rows);
    }
    p->waves_per_token = (uint32_t)waves;
    if (waves != 0 && tokens > (int64_t)0x7ffffff0 / waves) return TDE_ETOOBIG;
    p->blocks = (uint32_t)((tokens * waves + 3) / 4);
    if (!fits_launch(p->blocks, 256)) return TDE_ETOOBIG;
    return TDE_OK;
}

int launch_head_rows(HeadRowsArgs &a, int dtype, hipStream_t s) {
    const int64_t heads_all = (int64_t)a.heads[0] + a.heads[1] + a.heads[2];
    if (a.tokens == 0 || heads_all == 0) return TDE_OK;
    HeadRowsPlan plan;
    const int st = plan_head_rows(dtype == TDE_F32 ? 4 : 2, a.dim, a.half, a.interleaved, a.tokens, heads_all, &plan);
    if (st != TDE_OK) return st;
    a.lanes_log2 = plan.lanes_log2;
    a.waves_per_token = Divisor32(plan.waves_per_token);
    switch (dtype) {
    case TDE_BF16: return launch_typed<Bf16>(a, plan, s);
    case TDE_F16: return launch_typed<F16>(a, plan, s);
    case TDE_F32: return launch_typed<F32>(a, plan, s);
    }
    return TDE_EDTYPE;
}

} // namespace block
} // namespace tde
