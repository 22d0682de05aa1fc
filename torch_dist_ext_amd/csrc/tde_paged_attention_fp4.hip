// Attention over paged caches in 4 bits: e2m1 codes with a power of two for 32 channels.
//
// Chunks take the kernel of the 16-bit caches, whose tiles' numbers the wavefronts make of codes on their way to LDS: a number is made once a workgroup and
// enters 128 rows' products.
//
// Decode rows (16 a tile at most) have a kernel of their own, below.  A number enters few products there, and what a call waits for is the codes' bytes.
#include "tde_paged_attention_kernel.h"

namespace tde {
namespace block {

namespace {

// An address that the whole wavefront shares, kept apart from what lanes add to it.
__device__ __forceinline__ const char *scalar(const char *p) {
    asm volatile("" : "+s"(p));
    return p;
}

// Bytes BYTES at a wavefront's address plus the lane's offset; read once, not to be kept in the caches.
template <int BYTES>
__device__ __forceinline__ Words<BYTES> load_at(const char *base, uint32_t lane_offset) {
    Words<BYTES> r;
    const char *const p = base + lane_offset;
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const u32x4 v = __builtin_nontemporal_load((const __attribute__((address_space(1))) u32x4 *)p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * i + j] = v[j];
        }
    } else if constexpr (BYTES == 8) {
        const u32x2 v = __builtin_nontemporal_load((const __attribute__((address_space(1))) u32x2 *)p);
        r.w[0] = v[0];
        r.w[1] = v[1];
    } else {
        r.w[0] = __builtin_nontemporal_load((const __attribute__((address_space(1))) uint32_t *)p);
    }
    return r;
}
__device__ __forceinline__ uint32_t load_two_bytes(const char *base, uint32_t lane_offset) {
    return __builtin_nontemporal_load((const __attribute__((address_space(1))) uint16_t *)(base + lane_offset));
}
__device__ __forceinline__ uint32_t load_scale(const char *base, uint32_t lane_offset) {
    return *(const __attribute__((address_space(1))) uint8_t *)(base + lane_offset);
}

// Lane J of every four's x, in all of the four.
template <int J>
__device__ __forceinline__ uint32_t of_quad(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, J * 0x55, 0xf, 0xf, false);
}

// The codes of 32 keys and values, as a lane holds them.
template <int D>
struct Step {
    static constexpr int kKeyBytes = D / 8, kValueBytes = D / 32, kScales = D == 256 ? 2 : 1; // of a key, of a value, of both's scales
    Words<kKeyBytes> k[2];
    Words<kValueBytes < 4 ? 4 : kValueBytes> v[8];
    uint32_t k_scale[2][kScales], v_scale[2][kScales];
};

} // namespace

// 16 rows (token x query head of one key head's group) a workgroup, WAVES wavefronts with keys of their own, 32 a step: no wavefront waits for another before
// the end, and nothing goes by way of LDS.
//
//   S' = K Q'   a lane has a quarter of a key's channels: 16 bytes of codes are its operands of four products (heads of 128)
//   O' = V' P'  a product's rows are 16 channels, its depth 32 keys; a lane has eight keys of D/16 neighbouring channels, one of each product
//
// so codes are loaded as they lie, by 16 lanes a row, and a lane makes operands of them without any other lane: the two numbers that an instruction makes of a
// byte belong to two products, and a permutation pairs them with the next key's.  (By way of LDS and transposing loads: twice the instructions.)  Keys are
// taken in an order in which a load's four rows are neighbours: product row 4q + r is key 4r + q of 16.
//
// Two steps are on their way while one is worked on.  Loads are never left out, so that the compiler knows how many are outstanding: where a key has no
// page, or lies behind the last one, they take what lies in a page that exists, and the key's weight is NaN or 0.
// SPAN: keys in a row that are known to lie in one page, 16 or 8; their address is scalar.
template <class T, int D, int WAVES, int SPAN, bool SPLIT>
__global__ void __launch_bounds__(64 * WAVES, 2) decode_fp4_kernel(const AttentionFp4Args a) {
    constexpr int KT = 32, E = D / 16;         // keys a step; channels of a value that a lane has
    constexpr int SPANS = KT / SPAN;           // of a step
    __shared__ __align__(16) float joined[WAVES * 16 * (D + 4)];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t item_index = a.kv_heads.quotient(blockIdx.x);
    const int kv_head = (int)(blockIdx.x - item_index * a.kv_heads.d);
    const Item it = locate<16, SPLIT>(a, (int32_t)item_index, lane);
    const bool parts = SPLIT && it.chunks > 1; // this item's rows go to the second launch
    if (SPLIT && kv_head == 0 && threadIdx.x == 0 && (it.seq < 0 || it.chunk == 0) && (uint32_t)it.tile_of_call < (uint32_t)a.tiles) {
        JoinItem *const j = a.joins + it.tile_of_call; // as attention_kernel
        j->chunks = parts ? it.chunks : 0;
        j->item = (int32_t)item_index;
        j->tile = it.tile;
        j->begin = it.begin;
        j->count = it.count;
        j->len = it.len;
    }
    if (it.seq < 0) return;
    const int group = (int)a.group.d;
    const int col = lane & 15, quad = lane >> 4;

    // this lane's row: the token, the head, the last key that it sees
    const int64_t rows_all = (int64_t)it.count * group;
    const int64_t r_of_lane = (int64_t)it.tile * 16 + col;
    const bool row_there = r_of_lane < rows_all;
    const uint32_t row_token = a.group.quotient((uint32_t)(row_there ? r_of_lane : 0));
    const int head = kv_head * group + (int)((uint32_t)(row_there ? r_of_lane : 0) - row_token * a.group.d);
    const int32_t token = row_there ? it.begin + (int32_t)row_token : -1;
    const int32_t last = row_there ? it.len - it.count + (int32_t)row_token : -1;
    if (it.seq >= a.batch.seqs) { // rows of no sequence
        if (!a.zero_tail || wave != 0 || token < 0) return;
        for (int d = quad * 8; d < a.dim; d += 32) store_words<16>(a.out + token * a.out_token + head * a.out_head + d * 2, Words<16>{});
        return;
    }

    // keys that the tile's rows see, of this item's chunk, and of them the wavefront's
    const int64_t top_row = std::min<int64_t>((int64_t)(it.tile + 1) * 16, rows_all) - 1;
    const int32_t top = it.len - it.count + (int32_t)a.group.quotient((uint32_t)top_row) + 1; // keys that the tile's last row sees
    const int32_t lowest = it.len - it.count + (int32_t)a.group.quotient((uint32_t)((int64_t)it.tile * 16)) + 1; // and its first
    const int64_t from64 = SPLIT ? (int64_t)it.chunk * it.keys : 0;
    const int32_t from = __builtin_amdgcn_readfirstlane((int32_t)std::min<int64_t>(from64, 0x7fffffc0));
    const int32_t until = __builtin_amdgcn_readfirstlane((int32_t)std::min<int64_t>(SPLIT ? from64 + it.keys : 0x7fffffc0, std::min(top, walked(a, it.len))));
    const int32_t pairs_all = until > from ? (int32_t)(((int64_t)until - from + 2 * KT - 1) / (2 * KT)) : 0;
    const int32_t pairs_each = (pairs_all + WAVES - 1) / WAVES;
    int32_t pairs = std::max(0, std::min(pairs_each, pairs_all - wave * pairs_each));
    int32_t key0 = from + wave * pairs_each * 2 * KT;

    // What the end needs, in vector registers: scalar ones are few.
    const int32_t end_tile = in_place(it.tile), end_begin = in_place(it.begin), end_count = in_place(it.count), end_len = in_place(it.len);
    const int32_t end_item = in_place((int32_t)item_index), end_parts = in_place(parts), end_kv_head = in_place(kv_head);

    // ---- loading ----
    const auto *const table = (const __attribute__((address_space(4))) int32_t *)(a.batch.table + it.seq * a.batch.table_stride);
    uint32_t next_at = a.batch.page.quotient((uint32_t)key0), next_slot = (uint32_t)key0 - next_at * a.batch.page.d;
    // entries of the next step's spans, where they lie in their pages
    int32_t entry[SPANS];
    uint32_t slot[SPANS];
    const auto look_up = [&] {
#pragma unroll
        for (int i = 0; i < SPANS; ++i) {
            entry[i] = table[std::min(next_at, (uint32_t)a.batch.table_pages - 1)];
            if (next_at >= (uint32_t)a.batch.table_pages) entry[i] = -1;
            slot[i] = next_slot;
            next_slot += SPAN;
            if (next_slot == a.batch.page.d) {
                next_slot = 0;
                ++next_at;
            }
        }
    };
    // Offsets of the lane.  Channels that the head does not have repeat others; queries have zeros there.
    const int key_of_lane = (col & 3) * 4 + (col >> 2); // of 16
    const bool channels_there = quad * (D / 4) < a.dim;
    const uint32_t key_in_span = (uint32_t)(key_of_lane & (SPAN - 1)), value_at = (uint32_t)(col * E < a.dim ? col * E : 0);
    const uint32_t k_lane = key_in_span * a.k_slot + (channels_there ? quad * (D / 8) : 0);
    const uint32_t k_second = D == 256 && quad * 64 + 32 < a.dim ? 1 : 0; // heads of 256: whether the lane has the second of its blocks
    const uint32_t k_scale_lane = key_in_span * a.k_scale_slot + (channels_there ? quad * (D / 4) / 32 : 0);
    const uint32_t v_lane = (uint32_t)quad * a.v_slot + value_at / 2;
    // a scale for each of 16 keys and 4 blocks: every lane loads another one, that of key 4 (lane mod 4) + quad for the four lanes' block
    const uint32_t v_scale_lane = (uint32_t)(((col & 3) * 4 + quad) & (SPAN - 1)) * a.v_scale_slot + value_at / 32;
    const uint32_t v_scale_first = (uint32_t)(((col & 3) * 4 + quad) & (SPAN - 1)) * a.v_scale_slot + (uint32_t)std::min(((col & ~3) * E) / 32, a.dim / 32 - 1);
    const uint32_t v_scale_second = (uint32_t)(((col & 3) * 4 + quad) & (SPAN - 1)) * a.v_scale_slot + (uint32_t)std::min(((col & ~3) * E) / 32 + 1, a.dim / 32 - 1);
    const char *const k_base = a.k + kv_head * a.k_head, *const v_base = a.v + kv_head * a.v_head;
    const char *const k_scale_base = a.k_scales + kv_head * a.k_scale_head, *const v_scale_base = a.v_scales + kv_head * a.v_scale_head;
    const bool key_in_second = SPAN == 8 && key_of_lane >= 8, scale_in_second = SPAN == 8 && (col & 3) >= 2;
    // Codes of the step that was looked up; lost: bits of spans without a page.
    const auto fetch = [&](Step<D> &s, uint32_t &lost) {
        lost = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) { // 16 keys
            const char *k_at[16 / SPAN], *v_at[16 / SPAN], *k_scale_at[16 / SPAN], *v_scale_at[16 / SPAN];
#pragma unroll
            for (int i = 0; i < 16 / SPAN; ++i) {
                const int of = t * (16 / SPAN) + i;
                const bool none = (uint32_t)entry[of] >= (uint32_t)a.batch.cache_pages;
                lost |= (uint32_t)none << of;
                const uint32_t page = none ? 0 : (uint32_t)entry[of];
                k_at[i] = scalar(k_base + ((uint64_t)page * a.k_page + (uint64_t)slot[of] * a.k_slot));
                v_at[i] = scalar(v_base + ((uint64_t)page * a.v_page + (uint64_t)slot[of] * a.v_slot));
                k_scale_at[i] = scalar(k_scale_base + ((uint64_t)page * a.k_scale_page + (uint64_t)slot[of] * a.k_scale_slot));
                v_scale_at[i] = scalar(v_scale_base + ((uint64_t)page * a.v_scale_page + (uint64_t)slot[of] * a.v_scale_slot));
            }
            if constexpr (SPAN == 16) {
                s.k[t] = load_at<Step<D>::kKeyBytes>(k_at[0], k_lane);
                s.k_scale[t][0] = load_scale(k_scale_at[0], k_scale_lane);
                if constexpr (D == 256) {
                    s.k_scale[t][1] = load_scale(k_scale_at[0], k_scale_lane + k_second);
                    s.v_scale[t][0] = load_scale(v_scale_at[0], v_scale_first);
                    s.v_scale[t][1] = load_scale(v_scale_at[0], v_scale_second);
                } else {
                    s.v_scale[t][0] = load_scale(v_scale_at[0], v_scale_lane);
                }
            } else {
                s.k[t] = load_at<Step<D>::kKeyBytes>(key_in_second ? k_at[1] : k_at[0], k_lane);
                s.k_scale[t][0] = load_scale(key_in_second ? k_scale_at[1] : k_scale_at[0], k_scale_lane);
                const char *const from_span = scale_in_second ? v_scale_at[1] : v_scale_at[0];
                if constexpr (D == 256) {
                    s.k_scale[t][1] = load_scale(key_in_second ? k_scale_at[1] : k_scale_at[0], k_scale_lane + k_second);
                    s.v_scale[t][0] = load_scale(from_span, v_scale_first);
                    s.v_scale[t][1] = load_scale(from_span, v_scale_second);
                } else {
                    s.v_scale[t][0] = load_scale(from_span, v_scale_lane);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) { // keys 4j + quad
                const int span = j * 4 / SPAN;
                const char *const from_row = scalar(v_at[span] + (uint64_t)(uint32_t)(j * 4 - span * SPAN) * a.v_slot);
                if constexpr (D == 64) s.v[t * 4 + j].w[0] = load_two_bytes(from_row, v_lane);
                else s.v[t * 4 + j] = load_at<Step<D>::kValueBytes>(from_row, v_lane);
            }
            if constexpr (SPAN == 8) __builtin_amdgcn_sched_barrier(0); // scalar registers for one half's addresses at a time
        }
    };

    u32x4 q[D / 32]; // channels quad * D/4 + 8 i
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int d = quad * (D / 4) + i * 8;
        q[i] = u32x4{0, 0, 0, 0};
        if (token >= 0 && d < a.dim) {
            const Words<16> w = load_words<16>(a.q + token * a.q_token + head * a.q_head + d * 2);
            q[i] = u32x4{w.w[0], w.w[1], w.w[2], w.w[3]};
        }
    }

    f32x4 o[E], l = {0, 0, 0, 0}; // o[c][r]: channel (4 quad + r) E + c; l: sums of weights
    float m = -__builtin_inff(), shift = 0.0f, away = 0.0f; // as attention_kernel
#pragma unroll
    for (int c = 0; c < E; ++c) o[c] = f32x4{0, 0, 0, 0};

    const auto work = [&](const Step<D> &s, int32_t key0, uint32_t lost) {
        // ---- scores ----
        f32x4 score[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            uint32_t scale[Step<D>::kScales]; // of channels that the head does not have: 0, which a NaN would not be
#pragma unroll
            for (int i = 0; i < Step<D>::kScales; ++i)
                scale[i] = (D == 256 ? quad * 64 + i * 32 < a.dim : channels_there) ? read_scale<T>(s.k_scale[t][i]) : 0;
            score[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < D / 32; ++i) score[t] = Mfma<T>::mul(from_fp4<T>(s.k[t].w[i], scale[D == 256 ? i / 4 : 0]), q[i], score[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (__builtin_expect(lost != 0, 0)) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if ((lost >> ((t * 16 + r * 4) / SPAN)) & 1) score[t][r] = __builtin_nanf("");
        }
        const bool partly = (int64_t)key0 + KT > std::min(lowest, until); // not all rows see all keys
        if (partly) {
            const int32_t see = std::min(last, until - 1) - key0 - quad;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (t * 16 + r * 4 > see) score[t][r] = -__builtin_inff();
        }

        // ---- softmax, as attention_kernel's ----
        float top_score = score[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) top_score = __builtin_fmaxf(top_score, score[t][r]);
        top_score = __builtin_fmaxf(m, max_of_row(top_score));
        if (__builtin_amdgcn_ballot_w64((top_score - m) * a.scale_log2 > Mfma<T>::kLag) != 0) {
            const float top = seen_or_zero(top_score), octaves = top * a.scale_log2;
            const float alpha = __builtin_amdgcn_exp2f((m - top) * a.scale_log2);
            m = top_score;
            const bool near = __builtin_fabsf(octaves) < kFarOctaves;
            shift = (near ? octaves : 0.0f) - Mfma<T>::kRaise;
            away = near ? 0.0f : top;
            l *= alpha;
#pragma unroll
            for (int c = 0; c < E; ++c) o[c] *= alpha;
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(away != 0.0f) != 0, 0)) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) score[t][r] -= away;
        }
        u32x4 p, rest; // weights of keys 4r + quad of the first 16 and of the second, and what rounding left of them
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) score[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[t][r], a.scale_log2, -shift));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f32x4 x = score[w >> 1];
            const float x0 = x[(w & 1) * 2], x1 = x[(w & 1) * 2 + 1];
            p[w] = Mfma<T>::part(x0, x1);
            float lo, hi;
            T::widen(p[w], lo, hi);
            rest[w] = Mfma<T>::part(x0 - lo, x1 - hi);
        }
        const uint32_t ones = T::narrow(1.0f, 1.0f);
        l = Mfma<T>::mul(u32x4{ones, ones, ones, ones}, p, l);
        l = Mfma<T>::mul(u32x4{ones, ones, ones, ones}, rest, l);

        __builtin_amdgcn_sched_barrier(0);
        // ---- values ----
        uint32_t scale[8]; // of the lane's block, of each of its keys
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const auto spread = [&](uint32_t x, uint32_t(&to)[4]) {
                to[0] = of_quad<0>(x), to[1] = of_quad<1>(x), to[2] = of_quad<2>(x), to[3] = of_quad<3>(x);
            };
            uint32_t first[4];
            spread(read_scale<T>(s.v_scale[t][0]), first);
            if constexpr (D == 256) {
                uint32_t second[4];
                spread(read_scale<T>(s.v_scale[t][1]), second);
#pragma unroll
                for (int j = 0; j < 4; ++j) first[j] = (col & 2) != 0 ? second[j] : first[j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) scale[t * 4 + j] = first[j];
        }
        // Two channels: a byte of each of the lane's values, as operands of two products.
        const auto operands = [&](int b, u32x4(&vf)[2]) {
            uint32_t pair[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float unit = __builtin_bit_cast(float, scale[i] << 23);
                const uint32_t w = s.v[i].w[b / 4];
                pair[i] = b % 4 == 0 ? Mfma<T>::template from_fp4<0>(w, unit)
                                     : (b % 4 == 1 ? Mfma<T>::template from_fp4<1>(w, unit)
                                                   : (b % 4 == 2 ? Mfma<T>::template from_fp4<2>(w, unit) : Mfma<T>::template from_fp4<3>(w, unit)));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vf[0][i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100u);
                vf[1][i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302u);
            }
        };
        // A NaN block that not all rows see: a weight of zero would not keep it from the sums.  Its scale is replaced, and rows that see it get a NaN by way of a
        // product of their own (a block has all channels of a lane).
        if (partly) {
            uint32_t largest = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) largest = std::max(largest, scale[i]);
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(largest == 255) != 0, 0)) {
                const int32_t see = std::min(last, until - 1) - key0 - quad;
                const uint32_t one = T::narrow1(1.0f);
                u32x4 seen, mark; // 1 where the row sees the key, where the key's block is NaN
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const int key = (w >> 1) * 16 + (w & 1) * 8;
                    seen[w] = (one & ~(uint32_t)((see - key) >> 31)) | ((one & ~(uint32_t)((see - key - 4) >> 31)) << 16);
                    mark[w] = one * ((scale[2 * w] + 1) >> 8) | (one * ((scale[2 * w + 1] + 1) >> 8)) << 16;
                }
                const f32x4 found = Mfma<T>::mul(mark, seen, f32x4{0, 0, 0, 0});
#pragma unroll
                for (int c = 0; c < E; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[c][r] += found[r] != 0.0f ? __builtin_nanf("") : 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) scale[i] &= ((scale[i] + 1) >> 8) - 1; // 255: 0
            }
        }
#pragma unroll
        for (int b = 0; b < E / 2; ++b) {
            u32x4 vf[2];
            operands(b, vf);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                o[b * 2 + h] = Mfma<T>::mul(vf[h], p, o[b * 2 + h]);
                o[b * 2 + h] = Mfma<T>::mul(vf[h], rest, o[b * 2 + h]);
            }
        }
    };

    if (pairs > 0) {
        Step<D> s0, s1;
        uint32_t lost0, lost1;
        look_up();
        fetch(s0, lost0);
        look_up();
        fetch(s1, lost1);
        look_up();
        for (; pairs > 1; --pairs) {
            work(s0, key0, lost0);
            fetch(s0, lost0);
            look_up();
            work(s1, key0 + KT, lost1);
            fetch(s1, lost1);
            look_up();
            key0 += 2 * KT;
        }
        work(s0, key0, lost0);
        work(s1, key0 + KT, lost1);
    }

    // ---- join the wavefronts: [wave][row][D + 4] ----
    const auto &late = arguments_again<AttentionFp4Args>();
    {
        float *const part = joined + (wave * 16 + col) * (D + 4);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < E; c += 4) *(f32x4 *)(part + (quad * 4 + r) * E + c) = f32x4{o[c][r], o[c + 1][r], o[c + 2][r], o[c + 3][r]};
        if (quad == 0) *(f32x2 *)(part + D) = f32x2{m, l[0]};
    }
    __syncthreads();
    const int64_t at_part = ((int64_t)end_item * late.kv_heads.d + end_kv_head) * 16; // of the partial results
    // thread -> row and four channels
    for (int at = threadIdx.x; at < 16 * (D / 4); at += 64 * WAVES) {
        const int row = at / (D / 4), d = at % (D / 4) * 4;
        const int64_t r = (int64_t)end_tile * 16 + row;
        if (r >= (int64_t)end_count * late.group.d) continue;
        float top_m = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top_m = __builtin_fmaxf(top_m, joined[(w * 16 + row) * (D + 4) + D]);
        const float top = seen_or_zero(top_m);
        f32x4 sum = {0, 0, 0, 0};
        float all = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float *const part = joined + (w * 16 + row) * (D + 4);
            const float weight = __builtin_amdgcn_exp2f((part[D] - top) * late.scale_log2);
            sum += *(const f32x4 *)(part + d) * weight;
            all += part[D + 1] * weight;
        }
        if (end_parts != 0) {
            float *const part = late.partial + (at_part + row) * (D + 4);
            *(f32x4 *)(part + d) = sum;
            if (d == 0) *(f32x2 *)(part + D) = f32x2{top_m, all};
        } else if (d < late.dim) {
            const uint32_t t = late.group.quotient((uint32_t)r);
            const int h = end_kv_head * (int)late.group.d + (int)((uint32_t)r - t * late.group.d);
            f32x4 y = sum * (1.0f / all);
            if (end_len - end_count + (int32_t)t < 0) y = f32x4{0, 0, 0, 0}; // sees no key
            store_words<8>(late.out + (end_begin + (int32_t)t) * late.out_token + h * late.out_head + d * 2,
                           Words<8>{{T::narrow(y[0], y[1]), T::narrow(y[2], y[3])}});
        }
    }
}

namespace {

template <class T, int D, int SPAN>
void launch_decode(const AttentionFp4Args &a, const AttentionPlan &p, uint32_t blocks, hipStream_t s) {
    constexpr int WAVES = 4;
    if (!p.split) {
        decode_fp4_kernel<T, D, WAVES, SPAN, false><<<blocks, 64 * WAVES, 0, s>>>(a);
        return;
    }
    decode_fp4_kernel<T, D, WAVES, SPAN, true><<<blocks, 64 * WAVES, 0, s>>>(a);
    const uint32_t joins = (uint32_t)a.tiles * a.kv_heads.d;
    if (p.join_waves == 16) attention_join_kernel<T, HeldFp4, D, 16, 1, 16><<<joins * 16, 1024, 0, s>>>(a);
    else attention_join_kernel<T, HeldFp4, D, 16, 4, 1><<<joins * 4, 256, 0, s>>>(a);
}

template <class T, int D>
void launch_decode_of(const AttentionFp4Args &a, const AttentionPlan &p, uint32_t blocks, hipStream_t s) {
    if (a.batch.page.d % 16 == 0) launch_decode<T, D, 16>(a, p, blocks, s);
    else launch_decode<T, D, 8>(a, p, blocks, s);
}

template <class T>
void launch_decode_type(const AttentionFp4Args &a, const AttentionPlan &p, uint32_t blocks, hipStream_t s) {
    if (p.wide_dim == 64) launch_decode_of<T, 64>(a, p, blocks, s);
    else if (p.wide_dim == 128) launch_decode_of<T, 128>(a, p, blocks, s);
    else launch_decode_of<T, 256>(a, p, blocks, s);
}

} // namespace

// As plan_attention.  The decode kernel takes pages of whole 8 keys, tables and caches that have any.
int plan_attention_fp4(int dim, int64_t tokens, int q_heads, int kv_heads, const tde_paged_batch &b, AttentionPlan *p) {
    const bool spans = b.page_size % 8 == 0 && b.table_pages > 0 && b.cache_pages > 0;
    return plan_attention_rows(dim, tokens, q_heads, kv_heads, b.seqs, (int64_t)b.table_pages * b.page_size, spans ? 16 : 64, p);
}

int launch_attention_fp4(AttentionFp4Args &a, const AttentionPlan &p, int dtype, hipStream_t s) {
    if (p.rows != 16) return launch_planned<HeldFp4>(a, p, dtype, s);
    const uint32_t blocks = set_sizes(a, p);
    if (dtype == TDE_BF16) launch_decode_type<Bf16>(a, p, blocks, s);
    else launch_decode_type<F16>(a, p, blocks, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace block
} // namespace tde
