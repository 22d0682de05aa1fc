// Attention of new tokens over a paged cache: o_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys j <= the token's position.
//
// One pass over the keys with a running maximum m and sum l for each row, in fp32.  A tile's rows are (new token, query head of one
// key head's group), so every key and value is loaded once for the whole group.  Both products run on the matrix units, transposed:
//
//   S' = K Q'   16 keys x 16 rows an instruction, 32 channels deep
//   O' = V' P'  16 channels x 16 rows, 32 keys deep
//
// An instruction's result has its 16 columns -- the rows -- along the lanes, so a row's maximum, sum and rescaling factor are one value
// a lane, and a lane's scores of two key blocks are, converted to T, its operand of the second product without any exchange: the
// product's keys only need the same order on both sides, and V' is read from LDS with transposing loads in just that order.
// The weights go into the second product, whose operands are T, rounded to T, and their sum is that of the rounded ones: one more product, with
// a row of ones.  In calls of 16 rows a sequence and less, which wait for the caches' bytes, what the rounding leaves goes in as a second operand, into sums of
// its own: the result is then off by its own rounding alone (error against doubles 0.0017 in place of 0.0022 in bf16; 64 rows over up to 8192
// keys 195.9 us and 194.8, one over 131072 24.5 and 23.9).  Chunks wait for their instructions, and stay with one: 4096 rows behind 4096
// take 406 us, with two operands 540.
//
// Where the rows of a call fill few workgroups the keys are split as well (see locate) and a second launch joins the parts.
#ifndef TDE_PAGED_ATTENTION_KERNEL_H
#define TDE_PAGED_ATTENTION_KERNEL_H

#include "tde_paged_attention.h"

#include <algorithm>
#include <type_traits>

namespace tde {
namespace block {

#define TDE_LDS __attribute__((address_space(3)))

namespace {

template <class T>
struct Mfma;
template <>
struct Mfma<Bf16> {
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static constexpr uint32_t kExponent = 0x7f80u, kMantissa = 0x007fu;
    static constexpr uint32_t kMostExponent = 125; // of a scale with which all codes are finite
    static constexpr float kLag = 8.0f, kRaise = 0.0f; // see where weights are computed
    // Two numbers within a step of x0 and x1, where another operand takes what is left.
    static __device__ __forceinline__ uint32_t part(float x0, float x1) { return Bf16::narrow(x0, x1); }
    // Byte BYTE of eight codes as two numbers, exact but for subnormal ones.
    template <int BYTE>
    static __device__ __forceinline__ uint32_t from_fp4(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
    }
};
template <>
struct Mfma<F16> {
    static __device__ __forceinline__ f32x4 mul(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static constexpr uint32_t kExponent = 0x7c00u, kMantissa = 0x03ffu;
    static constexpr uint32_t kMostExponent = 13;
    static constexpr float kLag = 4.0f, kRaise = 11.0f;
    static __device__ __forceinline__ uint32_t part(float x0, float x1) { // towards zero: one instruction for both, to nearest it is three
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    }
    template <int BYTE>
    static __device__ __forceinline__ uint32_t from_fp4(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, BYTE));
    }
};
// What a scale's byte counts as where codes become numbers of T: blocks whose 6 is no number of fp16 are NaN there.
template <class T>
__device__ __forceinline__ uint32_t read_scale(uint32_t e) {
    return __is_same(T, F16) && e > 127 + Mfma<F16>::kMostExponent ? 255 : e;
}

__device__ __forceinline__ uint32_t load_byte(const char *p) { return *(const __attribute__((address_space(1))) uint8_t *)p; }
// Eight codes as numbers of T; `scale` is a scale's byte.
template <class T>
__device__ __forceinline__ u32x4 from_fp4(uint32_t codes, uint32_t scale) {
    const float factor = __builtin_bit_cast(float, scale << 23); // the conversion takes the exponent alone: 0 for 2^-127, 255 for NaN
    return u32x4{Mfma<T>::template from_fp4<0>(codes, factor), Mfma<T>::template from_fp4<1>(codes, factor), Mfma<T>::template from_fp4<2>(codes, factor),
                 Mfma<T>::template from_fp4<3>(codes, factor)};
}

// Maximum over the four lanes that hold a row (lane, lane ^ 16, lane ^ 32, lane ^ 48): swaps of rows of 16 lanes and of halves, of a value
// with itself, leave a pair's two values side by side.
// (Elements of a pair by way of variables: a bit_cast of the second one reads the first.)
__device__ __forceinline__ float max_of_row(float x) {
    const auto rows = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t r0 = rows[0], r1 = rows[1];
    x = __builtin_fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
    const auto halves = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t h0 = halves[0], h1 = halves[1];
    return __builtin_fmaxf(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
}

// The exponent of a weight is x * scale_log2 - m * scale_log2, one instruction that has the second product rounded.  What the rounding
// leaves is the same for all weights that refer to one maximum, and cancels, but it grows with the product: up to 2^-15 of an octave below 2^10
// octaves (which is also how far two maxima's weights may be off when they meet), up to 2^7 octaves below 2^32, where a row's largest weight is
// 0 or no number of T any more.  From 2^10 octaves on the distance from the maximum is taken first, which is exact next to it.
constexpr float kFarOctaves = 1024.0f;

// What maximum m takes off the maxima that are compared with it; nothing where no key has been seen, for all of them are -inf then.
__device__ __forceinline__ float seen_or_zero(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// What a workgroup works on.  The items of a call: for every sequence its tiles of rows, for every tile its chunks of keys, in that
// order; the rows of no sequence, behind the last one and in front of the first, are two more "sequences" without keys.
struct Item {
    int32_t seq;      // from seqs on: rows of no sequence; -1: none
    int32_t tile;     // of the sequence
    int32_t chunk, chunks;
    int32_t tile_of_call; // number of its tile among the call's; for an item that is none the number of tiles and how many too far it is
    int32_t begin, count; // its rows of the call
    int32_t len;      // its keys
    int32_t keys;     // of a chunk
};

__device__ __forceinline__ int64_t clamped(int64_t x, int64_t low, int64_t high) { return x < low ? low : (x > high ? high : x); }

// The rows and keys of sequence i, whatever the arrays hold: rows inside the call's, lengths not negative.
__device__ __forceinline__ void extent(const AttentionArgs &a, int i, int32_t &begin, int32_t &count, int32_t &len) {
    begin = count = len = 0;
    if (i > a.batch.seqs + 1) return;
    const bool front = i == a.batch.seqs + 1;
    const int64_t s = front ? 0 : clamped(a.batch.starts[i], 0, a.tokens);
    const int64_t e = i == a.batch.seqs ? a.tokens : clamped(a.batch.starts[front ? 0 : i + 1], 0, a.tokens);
    begin = (int32_t)s;
    count = (int32_t)(e > s ? e - s : 0);
    if (i < a.batch.seqs) len = a.batch.lens[i] > 0 ? a.batch.lens[i] : 0;
}

template <int ROWS>
__device__ __forceinline__ int32_t tiles_of(const AttentionArgs &a, int32_t count) {
    return (int32_t)(((int64_t)count * a.group.d + ROWS - 1) / ROWS);
}

// Keys that are walked through: a length beyond the page table's row needs one key of it to make the rows that see it NaN.
__device__ __forceinline__ int32_t walked(const AttentionArgs &a, int32_t len) { return len > a.capacity ? a.capacity + 1 : len; }

// Keys of a chunk: all keys that the tiles have between them, over the number of items aimed at, in whole blocks of 64; sequences
// of any lengths then give chunks of one size, and the number of items is at most target + tiles.
__device__ __forceinline__ int32_t keys_of_chunk(const AttentionArgs &a, int64_t total) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) total += __shfl_xor((long long)total, m);
    int64_t keys = (total + a.target - 1) / a.target;
    keys = (keys + 63) & ~(int64_t)63;
    return (int32_t)clamped(keys, a.min_chunk, 0x7fffffc0);
}

// The item with number `want`; one wavefront, 64 sequences at a time.
template <int ROWS, bool SPLIT>
__device__ __forceinline__ Item locate(const AttentionArgs &a, int32_t want, int lane) {
    Item it{-1, 0, 0, 1, 0, 0, 0, 0, 0x7fffffc0};
    int32_t begin, count, len;
    extent(a, lane, begin, count, len);
    if (SPLIT) {
        int64_t total = (int64_t)tiles_of<ROWS>(a, count) * walked(a, len);
        for (int i = lane + 64; i < a.batch.seqs; i += 64) {
            int32_t other, n, keys;
            extent(a, i, other, n, keys);
            total += (int64_t)tiles_of<ROWS>(a, n) * walked(a, keys);
        }
        it.keys = keys_of_chunk(a, total);
    }
    int32_t passed = 0, tiles_passed = 0;
    for (int base = 0;;) {
        int32_t tiles = tiles_of<ROWS>(a, count);
        const int32_t chunks = SPLIT && walked(a, len) > it.keys ? (walked(a, len) - 1) / it.keys + 1 : 1;
        int32_t upto = 0, tiles_upto = 0; // inclusive sums over the lanes, of items and tiles
        const auto add_up = [&] {
            upto = tiles * chunks;
            tiles_upto = tiles;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const int32_t below = __shfl_up(upto, m), tiles_below = SPLIT ? __shfl_up(tiles_upto, m) : 0;
                if (lane >= m) {
                    upto += below;
                    tiles_upto += tiles_below;
                }
            }
            return __builtin_popcountll(__builtin_amdgcn_ballot_w64(passed + upto <= want));
        };
        int at = add_up();
        if (at < 64) {
            int32_t place = lane; // of the sequence among these
            if (!SPLIT) {
                // Unsplit, what sees most keys goes first: the longest of these sequences, and (below) a sequence's last tiles; short
                // items then fill the units that are free early (20 sequences of up to 700 tokens behind 3000: 154 us in the call's
                // order, 132 in this one; 100 of up to 60 tokens, where counting takes its share: 96 and 100).
                const int32_t there = std::min(64, a.batch.seqs + 2 - base);
                int32_t rank = 0;
                for (int i = 0; i < there; ++i) {
                    const int32_t other = __builtin_amdgcn_readlane(len, i);
                    rank += (int32_t)(other > len) | ((int32_t)(other == len) & (int32_t)(i < lane));
                }
                place = __builtin_amdgcn_ds_permute((lane < there ? rank : lane) * 4, lane);
                begin = __shfl(begin, place);
                count = __shfl(count, place);
                len = __shfl(len, place);
                tiles = __shfl(tiles, place);
                at = add_up();
            }
            it.seq = base + __builtin_amdgcn_readlane(place, at);
            it.begin = __builtin_amdgcn_readlane(begin, at);
            it.count = __builtin_amdgcn_readlane(count, at);
            it.len = __builtin_amdgcn_readlane(len, at);
            it.chunks = __builtin_amdgcn_readlane(chunks, at);
            const int32_t local = want - passed - __builtin_amdgcn_readlane(upto - tiles * chunks, at);
            it.tile = local / it.chunks;
            it.chunk = local - it.tile * it.chunks;
            it.tile_of_call = tiles_passed + __builtin_amdgcn_readlane(tiles_upto - tiles, at) + it.tile;
            // sums that overflow, which only overlapping sequences can give, name no tile
            if ((uint32_t)it.tile >= (uint32_t)__builtin_amdgcn_readlane(tiles, at)) it.seq = -1;
            if (!SPLIT) it.tile = __builtin_amdgcn_readlane(tiles, at) - 1 - it.tile;
            return it;
        }
        passed += __builtin_amdgcn_readlane(upto, 63);
        tiles_passed += __builtin_amdgcn_readlane(tiles_upto, 63);
        base += 64;
        if (base > a.batch.seqs + 1) {
            it.tile_of_call = tiles_passed + (want - passed);
            return it;
        }
        extent(a, base + lane, begin, count, len);
    }
}

// x as if it were new here: what follows from it is computed in this place and not, as what never changes, before a loop through which
// there is no register to keep it.
__device__ __forceinline__ int in_place(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// 16 bytes a lane from memory to LDS: lane l's go to lds + 16 * l, lanes that are switched off leave their place as it is.  In assembly
// because the compiler waits for every such load before any read from LDS; nothing returns in registers.  wait_for_loads() is the
// wait that the data needs.
// STREAM: read once, not to be kept in the caches.
template <bool STREAM>
__device__ __forceinline__ void load_to_lds(const char *p, uint32_t lds) {
    if constexpr (STREAM) asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" : : "v"(p), "s"(lds) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(lds) : "memory", "m0");
}
template <bool STREAM>
__device__ __forceinline__ void load_to_lds(uint64_t base, uint32_t lane_offset, uint32_t lds) {
    base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)base) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(base >> 32)) << 32;
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    if constexpr (STREAM) asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" : : "v"(lane_offset), "s"(base), "s"(lds) : "memory", "m0");
    else asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(lane_offset), "s"(base), "s"(lds) : "memory", "m0");
}
// Whether 16 keys lie in one page and lanes' offsets from the first of them hold 32 bits.
template <class C>
__device__ __forceinline__ bool scalar_rows_of([[maybe_unused]] const typename C::Args &a) {
    if constexpr (C::kFp4) return a.batch.page.d % 16 == 0 && (a.k_slot | a.v_slot | a.k_scale_slot | a.v_scale_slot) < (uint32_t)kNearSlots && a.batch.cache_pages > 0;
    return false;
}

// The kernel's arguments, for what is done at its end: those of caches in 4 bits are too many for the scalar registers.
template <class C>
__device__ __forceinline__ const typename C::Args &late_arguments([[maybe_unused]] const typename C::Args &a) {
    if constexpr (C::kFp4) return arguments_again<typename C::Args>();
    else return a;
}

// What values that are not finite add up to, 0 where there is none; found: 1 for each +inf, 128 for each -inf, 16384 for each NaN, of 64 keys at most.
__device__ __forceinline__ float found_adds(float found) {
    const uint32_t f = (uint32_t)found;
    float add = (f & 127u) != 0 ? __builtin_inff() : 0.0f;
    add -= (f & (16384u - 128u)) != 0 ? __builtin_inff() : 0.0f;
    return f >= 16384u ? __builtin_nanf("") : add;
}

// Until at most N loads are outstanding.
template <int N>
__device__ __forceinline__ void wait_for_loads() {
    static_assert(N < 64, "the counter has six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

} // namespace

// NB blocks of 16 rows a wavefront.  SHARED: the wavefronts have rows of their own and share tiles of keys, double-buffered in LDS;
// otherwise all have the same rows and take the tiles in turn, each through LDS of its own, and are joined at the end.
// (Heads of 64: four workgroups a unit hide the loads, with the registers of three 8 rows over 16000 keys take 24.0 us in place of 20.2, and 24 sequences
// of up to 512 rows over a cache in 4 bits 78 in place of 61.)
constexpr int workgroups_a_unit(bool fp4, int dim, int nb, bool shared, bool split, bool rest) {
    return dim == 256 ? 1 : (dim == 64 && (!shared || (fp4 && nb == 1 && !split && !rest)) ? 4 : 2);
}

// REST: weights as two numbers of T.
template <class T, class C, int D, int NB, int WAVES, bool SHARED, bool SPLIT, bool REST = !SHARED>
__global__ void __launch_bounds__(64 * WAVES, workgroups_a_unit(C::kFp4, D, NB, SHARED, SPLIT, REST)) attention_kernel(const typename C::Args a) {
    constexpr bool FP4 = C::kFp4;
    constexpr int KT = SHARED && D <= 128 ? 64 : 32; // keys a tile
    constexpr int CH = D / 8;                        // chunks of 16 bytes a row
    constexpr int ROWS = 16 * NB * (SHARED ? WAVES : 1);
    constexpr int LOADERS = SHARED ? WAVES : 1;
    constexpr int AT_ONCE = 64 / CH;                  // rows of a load
    constexpr int LOADS = KT / AT_ONCE / LOADERS;     // a wavefront, of keys and of values
    constexpr int TILE = KT * D * 2;
    constexpr int BUFFERS = SHARED ? 2 : WAVES;
    constexpr int JOIN = SHARED ? 0 : WAVES * 16 * NB * (D + 4) * 4;
    constexpr int LDS = 2 * TILE * BUFFERS > JOIN ? 2 * TILE * BUFFERS : JOIN;
    __shared__ __align__(16) char lds[LDS];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t item_index = a.kv_heads.quotient(blockIdx.x);
    const int kv_head = (int)(blockIdx.x - item_index * a.kv_heads.d);
    const Item it = locate<ROWS, SPLIT>(a, (int32_t)item_index, lane);
    const bool parts = SPLIT && it.chunks > 1; // this item's rows go to the second launch
    if (SPLIT && kv_head == 0 && threadIdx.x == 0 && (it.seq < 0 || it.chunk == 0) && (uint32_t)it.tile_of_call < (uint32_t)a.tiles) {
        // What the second launch has to know of each tile that there may be.  Items are at most a.target more than tiles, so the
        // items that are none are enough for the tiles that are none.
        JoinItem *const j = a.joins + it.tile_of_call;
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

    // this lane's row in each of its blocks: the token, the head, the last key that it sees
    int32_t token[NB], last[NB];
    int head[NB];
    const int64_t rows_all = (int64_t)it.count * group;
    const int row0 = SHARED ? wave * 16 * NB : 0;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int64_t r = (int64_t)it.tile * ROWS + row0 + n * 16 + col;
        const bool there = r < rows_all;
        const uint32_t t = a.group.quotient((uint32_t)(there ? r : 0));
        head[n] = kv_head * group + (int)((uint32_t)(there ? r : 0) - t * a.group.d);
        token[n] = there ? it.begin + (int32_t)t : -1;
        last[n] = there ? it.len - it.count + (int32_t)t : -1;
    }
    if (it.seq >= a.batch.seqs) { // rows of no sequence
        if (!a.zero_tail || (!SHARED && wave != 0)) return;
#pragma unroll
        for (int n = 0; n < NB; ++n)
            if (token[n] >= 0)
                for (int d = quad * 8; d < a.dim; d += 32)
                    store_words<16>(a.out + token[n] * a.out_token + head[n] * a.out_head + d * 2, Words<16>{});
        return;
    }

    // keys that the tile's rows see, of this item's chunk
    const int64_t top_row = std::min<int64_t>((int64_t)(it.tile + 1) * ROWS, rows_all) - 1;
    const int32_t top = it.len - it.count + (int32_t)a.group.quotient((uint32_t)top_row) + 1; // keys that the tile's last row sees
    const int32_t lowest = it.len - it.count + (int32_t)a.group.quotient((uint32_t)((int64_t)it.tile * ROWS)) + 1; // and its first
    const int64_t from64 = SPLIT ? (int64_t)it.chunk * it.keys : 0;
    const int32_t from = (int32_t)std::min<int64_t>(from64, 0x7fffffc0);
    const int32_t until = (int32_t)std::min<int64_t>(SPLIT ? from64 + it.keys : 0x7fffffc0, std::min(top, walked(a, it.len)));

    // ---- loading ----
    const int32_t *const table = a.batch.table + it.seq * a.batch.table_stride;
    const char *const k_base = a.k + kv_head * a.k_head, *const v_base = a.v + kv_head * a.v_head;
    constexpr int TILE_STEP = SHARED ? KT : KT * WAVES;
    // Keys up to two tiles behind the last one: there are 2^31 - 255 at most, so 32 bits hold them, which scalar instructions compare.
    using Key = std::conditional_t<FP4, int32_t, int64_t>;
    static_assert(!FP4 || TILE_STEP <= 64, "");
    const int32_t first_key = from + (SHARED ? 0 : wave * KT);
    // Lane l holds the table's entry window + l: 64 pages, and a tile needs no more.  Nothing else in the loop is loaded by way of
    // registers: the compiler would wait for it, and with it for every load to LDS that was issued before.
    int32_t window = -64, entries = -1;
    uint64_t missing = 0; // entries that are no page
    const auto look_up = [&](int32_t key0) { // before offsets_of(key0)
        const uint32_t first = a.batch.page.quotient((uint32_t)key0);
        const uint32_t end = a.batch.page.quotient((uint32_t)std::min<Key>((Key)key0 + KT, until) - 1);
        if (end - (uint32_t)window < 64) return;
        window = (int32_t)first;
        entries = page_number(a.batch, table, first + lane);
        asm volatile("" : "+v"(entries)); // waited for here
        missing = __builtin_amdgcn_ballot_w64(entries < 0);
    };
    // Where key `tile key + lane` lies in the caches, from their heads' first channels on: not there (kNoKey) from `until` on,
    // lost (kNoPage) where the table or the cache has no page for it.
    constexpr int64_t kNoKey = -1, kNoPage = -2;
    struct Offsets {
        int64_t k, v;
    };
    const auto offsets_of = [&](int64_t key0) -> Offsets {
        const int64_t key = key0 + lane;
        const bool there = (KT == 64 || lane < KT) && key < until;
        const uint32_t at = a.batch.page.quotient((uint32_t)(there ? key : key0)), slot = (uint32_t)key - at * a.batch.page.d;
        const int32_t page = __shfl(entries, (int)(at - (uint32_t)window));
        if (!there) return {kNoKey, kNoKey};
        if (page < 0) return {kNoPage, kNoPage};
        return {(int64_t)((uint64_t)(uint32_t)page * a.k_page + (uint64_t)slot * a.k_slot),
                (int64_t)((uint64_t)(uint32_t)page * a.v_page + (uint64_t)slot * a.v_slot)};
    };
    const auto of_lane = [](int64_t x, int from) { return (int64_t)__shfl((long long)x, from); };
    // Chunks are stored at places that spread over the banks what is read together: 16 keys of one chunk (keys), 8 keys of two
    // neighbouring chunks (values).  A load fills places in order, so a lane's place says which chunk it takes.
    const auto k_turn = [](int row) { return D == 64 ? (row >> 1) & 7 : row & 15; };
    const auto v_turn = [](int row) { return D == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1; };
    // Turns reach M + 1 chunks; what lies beyond is written apart, so that it stays a constant.
    constexpr int M = CH < 16 ? CH - 1 : 15;
    const auto k_place = [&](int row, int first, int more) { return (row * CH + (first & ~M) + (((first & M) + more) ^ k_turn(row))) * 16; };
    const auto v_place = [&](int row, int first, int more) { return (row * CH + (first & ~M) + (((first & M) + more) ^ v_turn(row))) * 16; };
    const uint32_t lds0 = (uint32_t)(uintptr_t)(TDE_LDS char *)lds;
    const int load_row = SHARED ? wave * LOADS * AT_ONCE : 0; // the wavefront's first
    // The rows of a load lie in one page wherever pages hold whole numbers of them: then a load is a scalar address and an offset of the
    // lane that never changes but for its turn.  Where 16 rows lie in one page the address is looked up once for them.  (Lanes'
    // offsets have 32 bits: slots far apart go the other way.  Two blocks of rows leave no scalar registers for loads one by one.)
    constexpr int SPAN = 16;
    const bool whole_spans = NB == 2 || a.batch.page.d % SPAN == 0;
    const bool whole_pages = a.batch.page.d % (NB == 2 ? SPAN : AT_ONCE) == 0 && (a.k_slot | a.v_slot) < 1u << 27;
    const uint32_t k_lane = (uint32_t)(lane / CH) * a.k_slot, v_lane = (uint32_t)(lane / CH) * a.v_slot;
    const uint32_t k_chunk = (uint32_t)((lane % CH) ^ k_turn(lane / CH)) * 16, v_chunk = (uint32_t)((lane % CH) ^ v_turn(lane / CH)) * 16;
    const uint32_t dim_bytes = (uint32_t)in_place(a.dim * 2);
    // Loads the keys and/or values of a tile (look_up has been called for it) to `to` from the start of lds.  Returns whether exactly
    // LOADS loads were issued for each; lost: keys without a page.
    const auto load = [&](int32_t key0, uint32_t to, uint64_t &lost, auto keys, auto values) -> bool {
        constexpr bool KEYS = decltype(keys)::value, VALUES = decltype(values)::value;
        const uint32_t at = to + load_row * CH * 16;
        const uint32_t first = a.batch.page.quotient((uint32_t)key0) - (uint32_t)window;
        const uint32_t end = a.batch.page.quotient((uint32_t)key0 + KT - 1) - (uint32_t)window;
        if (whole_pages && until - key0 >= KT && (missing >> first << first << (63 - end)) == 0) {
            uint64_t k_at = 0, v_at = 0;
            uint32_t k_row = 0, v_row = 0;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int row = load_row + i * AT_ONCE;
                if (i % (SPAN / AT_ONCE) == 0 || !whole_spans) {
                    const uint32_t key = (uint32_t)(key0 + row), page = a.batch.page.quotient(key), slot = key - page * a.batch.page.d;
                    const uint32_t number = (uint32_t)__builtin_amdgcn_readlane(entries, (int)(page - (uint32_t)window));
                    if constexpr (KEYS) k_at = (uint64_t)k_base + (uint64_t)number * a.k_page + (uint64_t)slot * a.k_slot;
                    if constexpr (VALUES) v_at = (uint64_t)v_base + (uint64_t)number * a.v_page + (uint64_t)slot * a.v_slot;
                    k_row = k_lane;
                    v_row = v_lane;
                } else {
                    k_row += AT_ONCE * a.k_slot;
                    v_row += AT_ONCE * a.v_slot;
                }
                // Channels that the head does not have: the keys' stay zeros (every load has lanes with channels, so none is left out),
                // the values', which no output takes, repeat the first ones.
                const uint32_t kc = k_chunk ^ (uint32_t)k_turn(row) * 16, vc = v_chunk ^ (uint32_t)v_turn(row) * 16;
                if (KEYS && kc < dim_bytes) load_to_lds<!SHARED>(k_at, kc + k_row, lds0 + at + i * 1024);
                if (VALUES) load_to_lds<!SHARED>(v_at, (vc < dim_bytes ? vc : 0) + v_row, lds0 + at + TILE + i * 1024);
            }
            lost = 0;
            return true;
        }
        const Offsets where = offsets_of(key0);
        const int l = in_place(lane);
#pragma unroll 2
        for (int i = 0; i < LOADS; ++i) {
            const int row = load_row + l / CH + i * AT_ONCE;
            const int64_t k_at = of_lane(where.k, row), v_at = of_lane(where.v, row);
            const int kc = (l % CH) ^ k_turn(row), vc = (l % CH) ^ v_turn(row);
            if (k_at >= 0) {
                if (KEYS && kc * 8 < a.dim) load_to_lds<!SHARED>(k_base + k_at + kc * 16, lds0 + at + i * 1024);
                if (VALUES && vc * 8 < a.dim) load_to_lds<!SHARED>(v_base + v_at + vc * 16, lds0 + at + TILE + i * 1024);
            } else if (VALUES) { // a weight of zero would not keep what lies there from the sums; scores are replaced
                *(u32x4 *)(lds + at + TILE + i * 1024 + l * 16) = u32x4{0, 0, 0, 0};
            }
        }
        lost = __builtin_amdgcn_ballot_w64(where.k == kNoPage);
        return false;
    };
    // A cache in 4 bits goes by way of registers: a lane takes 32 channels of a key and of its value, or of one of the two where lanes are enough for both, which are
    // numbers of T once they are in LDS.  The next tile's codes are on their way while a tile is worked on.
    static_assert(!FP4 || SHARED, "wavefronts with keys of their own take codes another way");
    constexpr int PIECES = D / 32;                                  // of a row
    constexpr bool HALVES = FP4 && KT * PIECES * 2 <= 64 * WAVES;   // keys are the first half of the wavefronts', values the second's
    static_assert(!FP4 || KT * PIECES == 64 * WAVES / (HALVES ? 2 : 1), "one piece a lane");
    struct Codes {
        u32x4 k, v; // HALVES: k alone
        uint32_t k_scale, v_scale;
    };
    [[maybe_unused]] Codes codes{};
    [[maybe_unused]] const bool takes_values = HALVES && wave >= WAVES / 2;
    constexpr int WAVE_ROWS = 64 / PIECES;
    const int piece_row0 = (HALVES ? wave % (WAVES / 2) : wave) * WAVE_ROWS, piece_row = piece_row0 + lane / PIECES, piece = lane % PIECES;
    [[maybe_unused]] const bool piece_there = piece * 32 < a.dim;
    // What a wavefront loads from: keys' codes or, with HALVES, its own kind's; values' codes; their scales.
    struct Held {
        const char *codes, *scales;
        uint32_t page, slot, scale_page, scale_slot;
    };
    const auto held = [&]([[maybe_unused]] bool values) -> Held {
        if constexpr (FP4) {
            return values ? Held{v_base, a.v_scales + kv_head * a.v_scale_head, a.v_page, a.v_slot, a.v_scale_page, a.v_scale_slot}
                          : Held{k_base, a.k_scales + kv_head * a.k_scale_head, a.k_page, a.k_slot, a.k_scale_page, a.k_scale_slot};
        }
        return {};
    };
    [[maybe_unused]] Held mine{};
    if constexpr (HALVES) { // kept: loaded anew for each tile they are waited for (24 sequences of up to 512 rows: 64 us, and 61)
        mine = held(takes_values);
        asm volatile("" : "+s"(mine.codes), "+s"(mine.scales), "+s"(mine.page), "+s"(mine.slot), "+s"(mine.scale_page), "+s"(mine.scale_slot));
    }
    // A wavefront's rows (8, 16 or twice 16) then have scalar addresses.
    [[maybe_unused]] const bool scalar_rows = scalar_rows_of<C>(a);
    const auto fetch = [&]([[maybe_unused]] int32_t key0, [[maybe_unused]] uint64_t &lost) { // look_up has been called for the tile
        if constexpr (FP4) {
            const uint32_t first = a.batch.page.quotient((uint32_t)key0) - (uint32_t)window;
            const uint32_t end = a.batch.page.quotient((uint32_t)key0 + KT - 1) - (uint32_t)window;
            uint32_t of_page = 0, of_slot = 0; // of the lane's row
            bool there = true;
            lost = 0;
            const bool all_there = scalar_rows && end < 64 && (missing >> first << first << (63 - end)) == 0;
            if (!all_there) {
                const int64_t key = (int64_t)key0 + lane;
                const bool key_there = (KT == 64 || lane < KT) && key < until;
                const uint32_t at = a.batch.page.quotient((uint32_t)(key_there ? key : key0));
                const int32_t entry = __shfl(entries, (int)(at - (uint32_t)window));
                const int32_t page = key_there ? entry : -1;
                lost = __builtin_amdgcn_ballot_w64(key_there && page < 0);
                of_page = (uint32_t)__shfl(page, piece_row);
                of_slot = (uint32_t)key0 + piece_row - (uint32_t)__shfl((int)at, piece_row) * a.batch.page.d;
                there = (int32_t)of_page >= 0;
                codes = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}, 0, 0}; // zeros where there is no key: no weight would keep what lies there from the sums
            }
            const auto one = [&](const Held &h, u32x4 &to, uint32_t &to_scale) {
                const char *from, *scale_from;
                if (all_there) {
                    // keys behind the last one may be there, whatever they hold: their weights are 0, and where they are not finite they are taken out as
                    // values are that not all rows see
                    const auto at_key = [&](uint32_t key, const char *&codes_at, const char *&scales_at) {
                        const uint32_t page = a.batch.page.quotient(key), slot = key - page * a.batch.page.d;
                        const uint32_t number = (uint32_t)__builtin_amdgcn_readlane(entries, (int)(page - (uint32_t)window));
                        codes_at = h.codes + ((uint64_t)number * h.page + (uint64_t)slot * h.slot);
                        scales_at = h.scales + ((uint64_t)number * h.scale_page + (uint64_t)slot * h.scale_slot);
                    };
                    at_key((uint32_t)key0 + piece_row0, from, scale_from);
                    if constexpr (WAVE_ROWS > 16) {
                        const char *second, *scale_second;
                        at_key((uint32_t)key0 + piece_row0 + 16, second, scale_second);
                        from = lane < 32 ? from : second;
                        scale_from = lane < 32 ? scale_from : scale_second;
                    }
                    const uint32_t row = (uint32_t)(lane / PIECES) & 15u;
                    from += row * h.slot + (piece_there ? piece : 0) * 16;
                    scale_from += row * h.scale_slot + (piece_there ? piece : 0);
                } else {
                    from = h.codes + ((uint64_t)of_page * h.page + (uint64_t)of_slot * h.slot + piece * 16);
                    scale_from = h.scales + ((uint64_t)of_page * h.scale_page + (uint64_t)of_slot * h.scale_slot + piece);
                }
                if (all_there || (there && piece_there)) {
                    const Words<16> w = load_words<16>(from);
                    to = u32x4{w.w[0], w.w[1], w.w[2], w.w[3]};
                    to_scale = load_byte(scale_from);
                }
            };
            if constexpr (HALVES) {
                one(mine, codes.k, codes.k_scale);
            } else {
                one(held(false), codes.k, codes.k_scale);
                one(held(true), codes.v, codes.v_scale);
            }
        }
    };
    // Part `i` of PARTS of the codes that were fetched into LDS as numbers.
    constexpr int PARTS = HALVES ? 4 : 8;
    // When: while the matrix units work on the tile's scores (4096 rows behind 4096 in heads of 128: 433 us, ahead of them 449; 24 sequences of up to 512
    // rows in heads of 64 60.5 and 61).
    const auto put = [&]([[maybe_unused]] uint32_t to, [[maybe_unused]] int i) {
        if constexpr (FP4) {
            const bool second = !HALVES && i >= 4;
            const u32x4 from = second ? codes.v : codes.k;
            const uint32_t scale = second ? codes.v_scale : codes.k_scale;
            const bool values = HALVES ? takes_values : second;
            const int at = values ? TILE + v_place(piece_row, piece * 4, i & 3) : k_place(piece_row, piece * 4, i & 3);
            // channels that the head does not have are zeros
            *(u32x4 *)(lds + to + at) = from_fp4<T>(piece_there ? from[i & 3] : 0, piece_there ? read_scale<T>(scale) : 0);
        }
    };
    constexpr std::true_type kYes{};
    constexpr std::false_type kNo{};
    uint32_t buf = SHARED ? 0 : wave * 2 * TILE;
    if (!FP4 && a.dim < D) { // channels that the head does not have stay zeros
        for (int i = threadIdx.x * 16; i < 2 * TILE * BUFFERS; i += 64 * WAVES * 16) *(u32x4 *)(lds + i) = u32x4{0, 0, 0, 0};
        __syncthreads();
    }
    uint64_t lost_next = 0;
    [[maybe_unused]] uint64_t lost_fetched = 0;
    [[maybe_unused]] bool keys_exact = false, values_exact = false; // of the loads that are outstanding
    if (first_key < until) {
        look_up(first_key);
        if constexpr (FP4) {
            fetch(first_key, lost_next);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) put(buf, i);
            if ((Key)first_key + TILE_STEP < until) {
                look_up(first_key + TILE_STEP);
                fetch(first_key + TILE_STEP, lost_fetched);
            }
        } else if constexpr (SHARED) load(first_key, buf, lost_next, kYes, kYes);
        else {
            keys_exact = load(first_key, buf, lost_next, kYes, kNo);
            values_exact = load(first_key, buf, lost_next, kNo, kYes);
        }
    }

    u32x4 q[NB][D / 32];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const int d = s * 32 + quad * 8;
            q[n][s] = u32x4{0, 0, 0, 0};
            if (token[n] >= 0 && d < a.dim) {
                const Words<16> w = load_words<16>(a.q + token[n] * a.q_token + head[n] * a.q_head + d * 2);
                q[n][s] = u32x4{w.w[0], w.w[1], w.w[2], w.w[3]};
            }
        }

    f32x4 o[NB][D / 16], l[NB]; // l: sums of weights, each of the four elements the whole row's
    f32x4 o_rest[NB][REST ? D / 16 : 1]; // apart: a rest of 0, or of the other sign, would make an infinite value's sum NaN
    float m[NB], shift[NB], away[NB]; // the maximum; what is taken off exponents; off scores that are far from zero
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        m[n] = -__builtin_inff();
        shift[n] = away[n] = 0.0f; // nothing seen yet: every weight is 0
        l[n] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            o[n][d] = f32x4{0, 0, 0, 0};
            if constexpr (REST) o_rest[n][d] = f32x4{0, 0, 0, 0};
        }
    }

    const auto sync = [] { // between what a tile's readers and writers do in LDS
        if constexpr (SHARED) __syncthreads();
        else {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    Key next = (Key)first_key + TILE_STEP;
    for (int32_t key0 = first_key; key0 < until;) {
        const bool more = next < until;
        const uint64_t lost = lost_next; // keys without a page
        if constexpr (FP4) {
            sync();
            lost_next = lost_fetched;
        } else if constexpr (SHARED) {
            wait_for_loads<0>();
            sync();
            if (more) {
                look_up((int32_t)next);
                load((int32_t)next, buf ^ (2 * TILE), lost_next, kYes, kYes);
            }
        } else {
            // the keys are there; the values that were issued behind them may come later
            if (values_exact) wait_for_loads<LOADS>();
            else wait_for_loads<0>();
            sync();
        }

        __builtin_amdgcn_sched_barrier(0);
        // ---- scores ----
        // Operands come in units of two: the next unit's reads go ahead of this one's products, and no further, which
        // registers would have to pay for.
        f32x4 s[NB][KT / 16];
        {
            constexpr int U = 2, UNITS = KT / 16 * (D / 32 / U);
            u32x4 kf[2][U];
            const auto read = [&](int unit) {
                const int kb = unit / (D / 32 / U), st = unit % (D / 32 / U) * U;
#pragma unroll
                for (int u = 0; u < U; ++u) // 16 rows on, turns are the same
                    kf[unit & 1][u] = *(const u32x4 *)(lds + (buf + k_place(col, (st + u) * 4, quad)) + kb * 16 * CH * 16);
            };
            read(0);
#pragma unroll
            for (int unit = 0; unit < UNITS; ++unit) {
                const int kb = unit / (D / 32 / U), st = unit % (D / 32 / U) * U;
                if (unit + 1 < UNITS) read(unit + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    if (st == 0) s[n][kb] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int u = 0; u < U; ++u) s[n][kb] = Mfma<T>::mul(kf[unit & 1][u], q[n][st + u], s[n][kb]);
                }
                // the next tile's numbers, which the products leave time for (behind the last tile old ones, which nothing reads)
                if constexpr (FP4) {
#pragma unroll
                    for (int i = unit * PARTS / UNITS; i < (unit + 1) * PARTS / UNITS; ++i) put(buf ^ (2 * TILE), i);
                }
            }
        }
        if constexpr (FP4) {
            if (next + TILE_STEP < until) {
                look_up((int32_t)next + TILE_STEP);
                fetch((int32_t)next + TILE_STEP, lost_fetched);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (FP4 ? __builtin_expect(lost != 0, 0) : lost != 0) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int kb = 0; kb < KT / 16; ++kb)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if ((lost >> (quad * 4) >> (kb * 16 + r)) & 1) s[n][kb][r] = __builtin_nanf("");
        }
        if ((Key)key0 + KT > std::min(lowest, until)) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int32_t see = std::min(last[n], until - 1) - key0 - quad * 4;
#pragma unroll
                for (int kb = 0; kb < KT / 16; ++kb)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (kb * 16 + r > see) s[n][kb][r] = -__builtin_inff();
            }
        }

        if (!SHARED && more) { // the keys have been read: the next ones take their place
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            look_up((int32_t)next);
            keys_exact = load((int32_t)next, buf, lost_next, kYes, kNo);
        }

        // ---- softmax ----
        // The maximum that weights refer to only moves once a score exceeds it by kLag octaves, so that sums are rarely rescaled.
        // Weights and sums alike are raised by kRaise octaves: weights reach 2^(kRaise + kLag), the largest of a row 2^kRaise at least, and sums
        // are fp32.  In bf16 neither matters.  Of fp16's 40 octaves 2^-24 .. 2^16 the raised ones leave weights of 2^-25 of the
        // largest all their bits and lose those below 2^-36; unraised, 16 octaves would lie idle above and a row whose one key takes nearly
        // all would lose what the others add up to (20000 keys at 2^-25 each: nothing of 6e-4).
        float top_score[NB];
        bool grown = false;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float t = s[n][0][0];
#pragma unroll
            for (int kb = 0; kb < KT / 16; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) t = __builtin_fmaxf(t, s[n][kb][r]);
            top_score[n] = __builtin_fmaxf(m[n], max_of_row(t));
            grown = grown || (top_score[n] - m[n]) * a.scale_log2 > Mfma<T>::kLag;
        }
        if (__builtin_amdgcn_ballot_w64(grown) != 0) {
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const float top = seen_or_zero(top_score[n]), octaves = top * a.scale_log2;
                const float alpha = __builtin_amdgcn_exp2f((m[n] - top) * a.scale_log2);
                m[n] = top_score[n];
                const bool near = __builtin_fabsf(octaves) < kFarOctaves;
                shift[n] = (near ? octaves : 0.0f) - Mfma<T>::kRaise;
                away[n] = near ? 0.0f : top;
                l[n] *= alpha;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    o[n][d] *= alpha;
                    if constexpr (REST) o_rest[n][d] *= alpha;
                }
            }
        }
        bool far = false;
#pragma unroll
        for (int n = 0; n < NB; ++n) far = far || away[n] != 0.0f;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(far) != 0, 0)) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int kb = 0; kb < KT / 16; ++kb)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[n][kb][r] -= away[n];
        }
        u32x4 p[NB][KT / 32], rest[NB][REST ? KT / 32 : 1];
        // Over caches in 4 bits weights are made two by two, those of the second 32 keys only while the matrix units are at the first's values (4096 rows behind
        // 4096 in heads of 128: 382 us, and 395 all ahead; heads of 64 have no registers for it: 60.1 and 58.9).
        constexpr bool LATE = FP4 && D == 128 && !REST;
        [[maybe_unused]] const auto weigh = [&](int n, int ks, int w) {
            const f32x4 x = s[n][2 * ks + (w >> 1)];
            const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[(w & 1) * 2], a.scale_log2, -shift[n]));
            const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[(w & 1) * 2 + 1], a.scale_log2, -shift[n]));
            p[n][ks][w] = T::narrow(x0, x1);
        };
        if constexpr (LATE) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int w = 0; w < 4; ++w) weigh(n, 0, w);
        }
#pragma unroll
        for (int n = 0; n < (LATE ? 0 : NB); ++n) {
#pragma unroll
            for (int kb = 0; kb < KT / 16; ++kb)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[n][kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][kb][r], a.scale_log2, -shift[n]));
#pragma unroll
            for (int ks = 0; ks < KT / 32; ++ks)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const f32x4 x = s[n][2 * ks + (w >> 1)];
                    const float x0 = x[(w & 1) * 2], x1 = x[(w & 1) * 2 + 1];
                    if constexpr (REST) p[n][ks][w] = Mfma<T>::part(x0, x1);
                    else p[n][ks][w] = T::narrow(x0, x1);
                }
            if constexpr (REST) {
#pragma unroll
                for (int ks = 0; ks < KT / 32; ++ks)
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        float lo, hi;
                        T::widen(p[n][ks][w], lo, hi);
                        const f32x4 x = s[n][2 * ks + (w >> 1)];
                        rest[n][ks][w] = Mfma<T>::part(x[(w & 1) * 2] - lo, x[(w & 1) * 2 + 1] - hi);
                    }
            }
        }

        __builtin_amdgcn_sched_barrier(0);
        // ---- values ----
        if constexpr (!SHARED) {
            if (more && keys_exact) wait_for_loads<LOADS>();
            else wait_for_loads<0>();
            sync();
        }
        // whether values that not all rows see hold an infinity or a NaN
        bool poisoned = false;
        if ((FP4 ? (Key)key0 + KT : std::min<Key>((Key)key0 + KT, until)) > lowest) { // (of 4 bits, what lies behind the last key is there)
            // an exponent of ones plus one at its lowest bit carries out of its field; the field's neighbours are masked off before
            constexpr uint32_t E = Mfma<T>::kExponent, LOW = E & (~E + 1u);
            uint32_t carried = 0;
            const char *const mine = lds + buf + TILE + in_place(SHARED ? (int)threadIdx.x : lane) * 16;
#pragma unroll 4
            for (int i = 0; i < TILE; i += 64 * LOADERS * 16) {
                const u32x4 v = *(const u32x4 *)(mine + i);
#pragma unroll
                for (int w = 0; w < 4; ++w) carried |= (v[w] & (E | E << 16)) + (LOW | LOW << 16);
            }
            if constexpr (SHARED) poisoned = __syncthreads_or((carried & 0x80008000u) != 0);
            else poisoned = __builtin_amdgcn_ballot_w64((carried & 0x80008000u) != 0) != 0;
        }

        // 4 keys x 16 channels for each 16 lanes, transposed on the way: a lane gets one channel of the keys 4 * quad ... + 3 and,
        // 16 keys on, of as many again
        const auto value_operand = [&](uint32_t tile, int quad, int col, int ks, int d) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            const uint32_t at = tile + v_place(quad * 4 + (col >> 2), d * 2, (col & 3) >> 1) + (col & 1) * 8; // 16 rows on, turns are the same
            const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TDE_LDS s16x4 *)(lds + at + ks * 32 * CH * 16));
            const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((TDE_LDS s16x4 *)(lds + at + (ks * 32 + 16) * CH * 16));
            const u32x2 xu = __builtin_bit_cast(u32x2, x), yu = __builtin_bit_cast(u32x2, y);
            return u32x4{xu[0], xu[1], yu[0], yu[1]};
        };
        if (__builtin_expect(poisoned, 0)) {
            // A weight of zero does not keep an infinity or NaN from the product.  Such values are taken out of the tile, and which
            // of them a row sees is counted by a product of its own (found_adds).
            constexpr uint32_t E = Mfma<T>::kExponent, M = Mfma<T>::kMantissa;
#pragma unroll 1
            for (int ks = 0; ks < KT / 32; ++ks) {
                const int here_quad = in_place(quad), here_col = in_place(col);
                u32x4 seen[NB]; // 1.0 where the row sees the key
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const int32_t see = std::min(last[n], until - 1) - key0 - ks * 32;
                    const uint32_t one = T::narrow1(1.0f);
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int key = (w >> 1) * 16 + here_quad * 4 + (w & 1) * 2;
                        seen[n][w] = (one & ~(uint32_t)((see - key) >> 31)) | ((one & ~(uint32_t)((see - key - 1) >> 31)) << 16);
                    }
                }
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    __builtin_amdgcn_sched_barrier(0); // one after the other: interleaved they take too many registers
                    const u32x4 vf = value_operand(buf + TILE, here_quad, here_col, ks, d);
                    u32x4 mark;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t marks = 0;
#pragma unroll
                        for (int hi = 0; hi < 32; hi += 16) {
                            const uint32_t h = (vf[w] >> hi) & 0xffffu;
                            const uint32_t code = (h & M) != 0 ? T::narrow1(16384.0f) : ((h & 0x8000u) != 0 ? T::narrow1(128.0f) : T::narrow1(1.0f));
                            marks |= ((h & E) == E ? code : 0u) << hi;
                        }
                        mark[w] = marks;
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        const f32x4 found = Mfma<T>::mul(mark, seen[n], f32x4{0, 0, 0, 0});
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[n][d][r] += found_adds(found[r]);
                        asm volatile("" : "+v"(o[n][d])); // now, not once all channels' marks have been found
                    }
                }
            }
            sync();
            char *const mine = lds + buf + TILE + in_place(SHARED ? (int)threadIdx.x : lane) * 16;
#pragma unroll 1
            for (int i = 0; i < TILE; i += 64 * LOADERS * 16) {
                u32x4 v = *(const u32x4 *)(mine + i);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    if ((v[w] & E) == E) v[w] &= 0xffff0000u;
                    if ((v[w] >> 16 & E) == E) v[w] &= 0x0000ffffu;
                }
                *(u32x4 *)(mine + i) = v;
            }
            sync();
        }
        const uint32_t ones = T::narrow(1.0f, 1.0f);
#pragma unroll
        for (int ks = 0; ks < (LATE ? 1 : KT / 32); ++ks)
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                l[n] = Mfma<T>::mul(u32x4{ones, ones, ones, ones}, p[n][ks], l[n]);
                if constexpr (REST) l[n] = Mfma<T>::mul(u32x4{ones, ones, ones, ones}, rest[n][ks], l[n]);
            }
        {
            constexpr int U = 4, UNITS = KT / 32 * (D / 16 / U);
            u32x4 vf[2][U];
            const auto read = [&](int unit) {
                const int ks = unit / (D / 16 / U), d = unit % (D / 16 / U) * U;
#pragma unroll
                for (int u = 0; u < U; ++u) vf[unit & 1][u] = value_operand(buf + TILE, quad, col, ks, d + u);
            };
            read(0);
#pragma unroll
            for (int unit = 0; unit < UNITS; ++unit) {
                const int ks = unit / (D / 16 / U), d = unit % (D / 16 / U) * U;
                if (unit + 1 < UNITS) read(unit + 1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (LATE) {
                    if (unit == UNITS / 2) {
#pragma unroll
                        for (int n = 0; n < NB; ++n) l[n] = Mfma<T>::mul(u32x4{ones, ones, ones, ones}, p[n][1], l[n]);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        o[n][d + u] = Mfma<T>::mul(vf[unit & 1][u], p[n][ks], o[n][d + u]);
                        if constexpr (REST) o_rest[n][d + u] = Mfma<T>::mul(vf[unit & 1][u], rest[n][ks], o_rest[n][d + u]);
                    }
                    if constexpr (LATE) {
                        constexpr int SLOTS = UNITS / 2 * U, EACH = (NB * 4 + SLOTS - 1) / SLOTS;
                        const int slot = unit * U + u;
#pragma unroll
                        for (int i = slot * EACH; i < (slot + 1) * EACH; ++i)
                            if (slot < SLOTS && i < NB * 4) weigh(i / 4, 1, i % 4);
                        if (slot < SLOTS) __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }

        if constexpr (SHARED) buf ^= 2 * TILE;
        else if (more) { // and so do the next values
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            values_exact = load((int32_t)next, buf, lost_next, kNo, kYes);
        }
        key0 = (int32_t)std::min<Key>(next, 0x7fffffff);
        next += TILE_STEP;
    }

    if constexpr (REST) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[n][d][r] += __builtin_fabsf(o[n][d][r]) < __builtin_inff() ? o_rest[n][d][r] : 0.0f;
    }

    // ---- what is left ----
    const auto &late = late_arguments<C>(a);
    const int64_t slot = ((int64_t)item_index * a.kv_heads.d + kv_head) * ROWS; // of the partial results
    if constexpr (SHARED) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            if (token[n] < 0) continue;
            if (parts) {
                float *const part = late.partial + (slot + row0 + n * 16 + col) * (D + 4);
#pragma unroll
                for (int d = 0; d < D / 16; ++d) *(f32x4 *)(part + d * 16 + quad * 4) = o[n][d];
                if (quad == 0) *(f32x2 *)(part + D) = f32x2{m[n], l[n][0]};
            } else {
                const float inverse = 1.0f / l[n][0];
                char *const to = late.out + token[n] * late.out_token + head[n] * late.out_head;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    const int at = d * 16 + quad * 4;
                    if (at >= a.dim) continue;
                    f32x4 y = o[n][d] * inverse;
                    if (last[n] < 0) y = f32x4{0, 0, 0, 0}; // sees no key
                    store_words<8>(to + at * 2, Words<8>{{T::narrow(y[0], y[1]), T::narrow(y[2], y[3])}});
                }
            }
        }
    } else {
        // join the wavefronts: [wave][row][D + 4]
        float *const mine = (float *)lds + wave * 16 * NB * (D + 4);
        __syncthreads(); // every wavefront is done with its tiles
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            float *const part = mine + (n * 16 + col) * (D + 4);
#pragma unroll
            for (int d = 0; d < D / 16; ++d) *(f32x4 *)(part + d * 16 + quad * 4) = o[n][d];
            if (quad == 0) *(f32x2 *)(part + D) = f32x2{m[n], l[n][0]};
        }
        __syncthreads();
        // thread -> row and four channels
        for (int at = threadIdx.x; at < 16 * NB * (D / 4); at += 64 * WAVES) {
            const int row = at / (D / 4), d = at % (D / 4) * 4;
            const int64_t r = (int64_t)it.tile * ROWS + row;
            if (r >= rows_all) continue;
            float top_m = -__builtin_inff();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) top_m = __builtin_fmaxf(top_m, ((float *)lds)[(w * 16 * NB + row) * (D + 4) + D]);
            const float top = seen_or_zero(top_m);
            f32x4 sum = {0, 0, 0, 0};
            float all = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float *const part = (const float *)lds + (w * 16 * NB + row) * (D + 4);
                const float weight = __builtin_amdgcn_exp2f((part[D] - top) * a.scale_log2);
                sum += *(const f32x4 *)(part + d) * weight;
                all += part[D + 1] * weight;
            }
            if (parts) {
                float *const part = late.partial + (slot + row) * (D + 4);
                *(f32x4 *)(part + d) = sum;
                if (d == 0) *(f32x2 *)(part + D) = f32x2{top_m, all};
            } else {
                if (d >= a.dim) continue;
                const uint32_t t = a.group.quotient((uint32_t)r);
                const int h = kv_head * group + (int)((uint32_t)r - t * a.group.d);
                f32x4 y = sum * (1.0f / all);
                if (it.len - it.count + (int32_t)t < 0) y = f32x4{0, 0, 0, 0};
                store_words<8>(late.out + (it.begin + (int32_t)t) * late.out_token + h * late.out_head + d * 2,
                               Words<8>{{T::narrow(y[0], y[1]), T::narrow(y[2], y[3])}});
            }
        }
    }
}

// Joins the chunks of a tile's rows: RW rows a workgroup, WAVES wavefronts a row, which take chunks in turn, eight at once.
template <class T, class C, int D, int ROWS, int RW, int WAVES>
__global__ void __launch_bounds__(64 * RW * WAVES) attention_join_kernel(const typename C::Args a) {
    constexpr int E = D / 64; // channels a lane
    constexpr int AHEAD = 8;
    __shared__ float joined[RW * WAVES][D + 4];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t at = blockIdx.x / (ROWS / RW), tile = a.kv_heads.quotient(at);
    const int kv_head = (int)(at - tile * a.kv_heads.d);
    const JoinItem j = a.joins[tile];
    if (j.chunks <= 0) return;
    // Where starts do not ascend an entry may never have been written; whatever it holds, what follows stays inside the call's arrays.
    if (j.item < 0 || j.item >= a.items || j.tile < 0 || j.begin < 0 || j.count < 0 || j.count > a.tokens - j.begin) return;
    const int32_t item = j.item;
    const int row = (int)(blockIdx.x % (ROWS / RW)) * RW + wave / WAVES;
    const int64_t r = (int64_t)j.tile * ROWS + row;
    const bool there = r < (int64_t)j.count * a.group.d;
    if (WAVES == 1 && !there) return;
    if (!(RW > 1 && WAVES > 1) && !there) return; // a workgroup of one row, or wavefronts of one each
    float best = -__builtin_inff(), sum[E] = {}, all = 0.0f;
    const int64_t step = (int64_t)a.kv_heads.d * ROWS * (D + 4); // from one item's partial results to the next one's
    const float *const parts = a.partial + (((int64_t)item * a.kv_heads.d + kv_head) * ROWS + row) * (int64_t)(D + 4);
    // of those that are items of this call: all of them where starts ascend
    const int chunks = there ? (int)std::min<int64_t>(j.chunks, a.items - (int64_t)item) : 0;
    for (int c0 = wave % WAVES; c0 < chunks; c0 += WAVES * AHEAD) {
        float pm[AHEAD], pl[AHEAD], x[AHEAD][E];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int c = c0 + i * WAVES;
            const float *const part = parts + (c < chunks ? c : c0) * step;
            pm[i] = c < chunks ? part[D] : -__builtin_inff();
            pl[i] = part[D + 1];
#pragma unroll
            for (int e = 0; e < E; ++e) x[i][e] = part[lane * E + e];
        }
        float top = best;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) top = __builtin_fmaxf(top, pm[i]);
        const float from = seen_or_zero(top);
        const float old = __builtin_amdgcn_exp2f((best - from) * a.scale_log2);
        all *= old;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] *= old;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float weight = __builtin_amdgcn_exp2f((pm[i] - from) * a.scale_log2);
            const bool counts = c0 + i * WAVES < chunks; // what a repeated chunk holds may not be finite
            all += counts ? pl[i] * weight : 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += counts ? x[i][e] * weight : 0.0f;
        }
        best = top;
    }
    const uint32_t t = a.group.quotient((uint32_t)r);
    const int head = kv_head * (int)a.group.d + (int)((uint32_t)r - t * a.group.d);
    char *const to = a.out + (j.begin + (int32_t)t) * a.out_token + head * a.out_head;
    const bool sees = j.len - j.count + (int32_t)t >= 0;
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) joined[wave][lane * E + e] = sum[e];
        if (lane == 0) {
            joined[wave][D] = best;
            joined[wave][D + 1] = all;
        }
        __syncthreads();
        if (wave % WAVES != 0 || !there) return;
        float top = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = __builtin_fmaxf(top, joined[wave + w][D]);
        const float from = seen_or_zero(top);
        all = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float weight = __builtin_amdgcn_exp2f((joined[wave + w][D] - from) * a.scale_log2);
            all += joined[wave + w][D + 1] * weight;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += joined[wave + w][lane * E + e] * weight;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane * E + e < a.dim) store_element<T>(to + (lane * E + e) * 2, sees ? sum[e] / all : 0.0f);
}
namespace {

template <class T, class C, int D, int NB, int WAVES, bool SHARED, bool REST = !SHARED>
void launch_one(const typename C::Args &a, const AttentionPlan &p, uint32_t blocks, hipStream_t s) {
    constexpr int ROWS = 16 * NB * (SHARED ? WAVES : 1);
    if (!p.split) {
        attention_kernel<T, C, D, NB, WAVES, SHARED, false, REST><<<blocks, 64 * WAVES, 0, s>>>(a);
        return;
    }
    attention_kernel<T, C, D, NB, WAVES, SHARED, true, REST><<<blocks, 64 * WAVES, 0, s>>>(a);
    const uint32_t joins = (uint32_t)a.tiles * a.kv_heads.d;
    if (p.join_waves == 16) attention_join_kernel<T, C, D, ROWS, 1, 16><<<joins * ROWS, 1024, 0, s>>>(a);
    else attention_join_kernel<T, C, D, ROWS, 4, 1><<<joins * (ROWS / 4), 256, 0, s>>>(a);
}

template <class T, class C, int D>
void launch_dim(const typename C::Args &a, const AttentionPlan &p, uint32_t blocks, hipStream_t s) {
    [[maybe_unused]] constexpr int ALONE = D == 256 ? 2 : 4; // wavefronts that each hold tiles of their own in LDS
    if constexpr (!C::kFp4) {
        if (p.rows == 16) return launch_one<T, C, D, 1, ALONE, false>(a, p, blocks, s);
    }
    if constexpr (C::kFp4 && D == 128) {
        if (p.rows == 256) {
            attention_kernel<T, C, D, 2, 8, true, false><<<blocks, 512, 0, s>>>(a);
            return;
        }
    }
    if constexpr (C::kFp4) {
        if (p.two_numbers) return launch_one<T, C, D, 1, 4, true, true>(a, p, blocks, s);
    }
    if (p.rows == 64) launch_one<T, C, D, 1, 4, true>(a, p, blocks, s);
    else attention_kernel<T, C, D, D <= 128 ? 2 : 1, D <= 128 ? 4 : 8, true, false><<<blocks, D <= 128 ? 256 : 512, 0, s>>>(a); // 128, never split
}

template <class T, class C>
void launch_type(const typename C::Args &a, const AttentionPlan &p, uint32_t blocks, hipStream_t s) {
    if (p.wide_dim == 64) launch_dim<T, C, 64>(a, p, blocks, s);
    else if (p.wide_dim == 128) launch_dim<T, C, 128>(a, p, blocks, s);
    else launch_dim<T, C, 256>(a, p, blocks, s);
}

// A plan's sizes into the arguments; returns the number of workgroups.
[[maybe_unused]] uint32_t set_sizes(AttentionArgs &a, const AttentionPlan &p) {
    a.items = (int32_t)p.items;
    a.tiles = (int32_t)p.tiles;
    a.target = p.target;
    a.min_chunk = p.min_chunk;
    a.capacity = (int32_t)std::min<int64_t>((int64_t)a.batch.table_pages * a.batch.page.d, 0x7fffff00);
    // the joins' items behind the partial results, which want 16-byte boundaries
    a.joins = reinterpret_cast<JoinItem *>(a.partial + p.items * a.kv_heads.d * p.rows * (p.wide_dim + 4));
    return (uint32_t)(p.items * a.kv_heads.d);
}

template <class C>
int launch_planned(typename C::Args &a, const AttentionPlan &p, int dtype, hipStream_t s) {
    const uint32_t blocks = set_sizes(a, p);
    if (dtype == TDE_BF16) launch_type<Bf16, C>(a, p, blocks, s);
    else launch_type<F16, C>(a, p, blocks, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace

} // namespace block
} // namespace tde

#endif // TDE_PAGED_ATTENTION_KERNEL_H
