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

// A lane's offset as if it were new here, so that it stays 32 bits wide and the address it goes with scalar.
__device__ __forceinline__ uint32_t here(uint32_t offset) {
    asm volatile("" : "+v"(offset));
    return offset;
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

// Workgroups that a unit holds, by their registers.
constexpr int resident_workgroups(int dim, int span) { return dim <= 64 && span == 16 ? 4 : (dim <= 128 ? 3 : 2); }

// Keys are shared out in units, a pair of a wavefront's steps.  A tile counts as a unit for each wavefront at least, and so does a runner's part.
constexpr int kUnit = 64, kDecodeWaves = 4;

__device__ __forceinline__ int32_t units_of_tile(const AttentionFp4Args &a, int i, int32_t len) { // of sequence i
    const int32_t units = (int32_t)(((int64_t)walked(a, len) + kUnit - 1) / kUnit);
    return i < a.batch.seqs ? std::max(kDecodeWaves, units) : kDecodeWaves;
}
// Of sequence i; rows of no sequence are no tiles where they are left as they are.
__device__ __forceinline__ int32_t tiles_to_do(const AttentionFp4Args &a, int i, int32_t count) { return i < a.batch.seqs || a.zero_tail ? tiles_of<16>(a, count) : 0; }

// Sums over the lanes up to each one, without LDS.
__device__ __forceinline__ int32_t sums_upto(int32_t x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false); // from 1, 2, 4, 8 lanes below, of rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false); // a row's last lane to the next row, the second one's to the upper half
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}

// How a call's tiles go to its runners, in units: `each` a runner, and tiles padded to multiples of `pad`.
struct Shares {
    int32_t each, pad;
    __device__ __forceinline__ int32_t padded(int32_t units) const { return pad == 1 ? units : (units + pad - 1) / pad * pad; }
};

} // namespace

// 16 rows (token x query head of one key head's group) a workgroup, WAVES wavefronts with keys of their own, 32 a step: no wavefront waits for another before
// the end, and nothing goes by way of LDS.
//
//   S' = K Q'   a lane has a quarter of a key's channels: 16 bytes of codes are its operands of four products (heads of 128)
//   O' = V' P'  a product's rows are 16 channels, its depth 32 keys; a lane has eight keys of D/16 neighbouring channels, one of each product
//
// so codes are loaded as they lie, by 16 lanes a row, and a lane makes operands of them without any other lane: the two numbers that an instruction makes of a
// value's byte belong to two products, and a permutation pairs them with the next key's.  Keys are taken in an order in which a load's four rows are
// neighbours: product row 4q + r is key 4r + q of 16.  (The products that take codes and scales as they are, with queries as sums of two e4m3 numbers, save 34 of
// some 200 vector instructions a step, but what prepares the queries costs more than that: 64 rows over up to 8192 keys 80 us in place of 73.)
//
// Two steps are on their way while one is worked on.  Loads are never left out, so that the compiler knows how many are outstanding: where a key has no
// page, or lies behind the last one, they take what lies in a page that exists, and the key's weight is NaN or 0.
// SPAN: keys in a row that are known to lie in one page, 16 or 8; their address is scalar.
//
// All units of all tiles, in order, go to as many workgroups as the device holds at once, the same number to each: whatever the lengths, none has more than
// another, and none begins when others have ended.  (A workgroup for each tile, long ones cut at one length: 64 rows over up to 8192 keys 72 us.)  Only where
// tiles alone fill the device twice is each a workgroup's, however long it is (plan_attention_fp4).  A workgroup
// has the end of one tile, whole ones, and the beginning of another; where runners are many and tiles few, tiles begin where a runner does, which has one part then
// (48 sequences of 3 rows over up to 6000 keys 27.9 us, and 31.2 without; one row over 262144 19.2 and 22.4; 64 over up to 8192 66, and 86 if they did).
// What is cut is joined by a second launch.  Parts go to places of the workgroup's own: 2r for the tile that others began, 2r + 1 for the one that others end.
template <class T, int D, int WAVES, int SPAN>
__global__ void __launch_bounds__(64 * WAVES, resident_workgroups(D, SPAN)) decode_fp4_kernel(const AttentionFp4Args args) {
    constexpr int KT = 32, E = D / 16;         // keys a step; channels of a value that a lane has
    __shared__ __align__(16) float joined[WAVES * 16 * (D + 4)];
    __shared__ i32x4 kept[WAVES][3]; // what a wavefront knows of the next part: in registers it would be there throughout

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const AttentionFp4Args &a = args;
    // a runner's key heads are on one die, where their neighbouring bytes meet in its cache
    uint32_t runner, kv_head;
    if (a.runners.d % 8 == 0) {
        const uint32_t at = blockIdx.x >> 3, of_die = a.kv_heads.quotient(at);
        kv_head = at - of_die * a.kv_heads.d;
        runner = of_die * 8 + (blockIdx.x & 7);
    } else {
        runner = a.kv_heads.quotient(blockIdx.x);
        kv_head = blockIdx.x - runner * a.kv_heads.d;
    }

    // ---- what is this runner's ----
    // Units are counted in 32 bits: there are fewer than 2^31 where starts ascend, and where they do not, whatever comes of it stays inside the arrays.
    int base = 0; // 64 sequences a time, one a lane
    int32_t begins, counts, lens, tiles_all = 0, units_all = 0;
    extent(a, lane, begins, counts, lens);
    for (int at = 0; !a.whole_tiles;) {
        const int32_t tiles = tiles_to_do(a, at + lane, counts);
        tiles_all += __builtin_amdgcn_readlane(sums_upto(tiles), 63);
        units_all += __builtin_amdgcn_readlane(sums_upto(tiles * units_of_tile(a, at + lane, lens)), 63);
        at += 64;
        if (at > a.batch.seqs + 1) break;
        extent(a, at + lane, begins, counts, lens);
    }
    Shares shares{1, 1};
    if (a.whole_tiles) {
        shares.pad = 0;
    } else {
        const int32_t runners = (int32_t)a.runners.d;
        const bool aligned = tiles_all <= runners / 4;
        const uint32_t over = (uint32_t)(aligned ? runners - tiles_all : runners);
        shares.each = std::max(kDecodeWaves, (int32_t)((uint32_t)(units_all + (int32_t)over - 1) / over));
        if (aligned || a.joins == nullptr) shares.each = (shares.each + kDecodeWaves - 1) & -kDecodeWaves; // (without joins all tiles have as many)
        shares.each = std::min(shares.each, a.most_each); // which sums of sequences that overlap could exceed
        if (aligned) shares.pad = shares.each;
    }
    const auto units_here = [&](int i, int32_t len) { return shares.pad == 0 ? 1 : shares.padded(units_of_tile(a, i, len)); }; // of a tile
    const uint32_t first = runner * (uint32_t)shares.each;
    if (a.joins != nullptr && kv_head == 0 && threadIdx.x == 0) a.joins[runner].chunks = 0;
    if (!a.whole_tiles && a.batch.seqs + 1 >= 64) extent(a, lane, begins, counts, lens);
    int at_seq;
    int32_t tile, unit;
    for (uint32_t passed = 0;;) {
        const int32_t n = units_here(base + lane, lens), units = tiles_to_do(a, base + lane, counts) * n, upto = sums_upto(units);
        at_seq = __builtin_popcountll(__builtin_amdgcn_ballot_w64(passed + (uint32_t)upto <= first));
        if (at_seq < 64) {
            const uint32_t local = first - passed - (uint32_t)__builtin_amdgcn_readlane(upto - units, at_seq), of_tile = (uint32_t)__builtin_amdgcn_readlane(n, at_seq);
            tile = __builtin_amdgcn_readfirstlane((int32_t)(local / of_tile));
            unit = (int32_t)(local - (uint32_t)tile * of_tile);
            break;
        }
        passed += (uint32_t)__builtin_amdgcn_readlane(upto, 63);
        base += 64;
        if (base > a.batch.seqs + 1) return; // nothing
        extent(a, base + lane, begins, counts, lens);
    }
    struct Part { // of a tile, the next that is to be done
        int32_t seq, begin, count, len, tile, unit, left, each, pad;
        uint32_t runner, kv_head;
    };
    const auto keep = [&](const Part &p) {
        i32x4 *const to = kept[wave];
        to[0] = i32x4{p.seq, p.begin, p.count, p.len};
        to[1] = i32x4{p.tile, p.unit, p.left, p.each};
        to[2] = i32x4{p.pad, (int32_t)p.runner, (int32_t)p.kv_head, 0};
    };
    keep({base + at_seq, __builtin_amdgcn_readlane(begins, at_seq), __builtin_amdgcn_readlane(counts, at_seq), __builtin_amdgcn_readlane(lens, at_seq), tile, unit,
          shares.each, shares.each, shares.pad, runner, kv_head});

    for (;;) { // the runner's part of one tile after the other
        const AttentionFp4Args &a = arguments_again<AttentionFp4Args>(); // for this part: kept over all of them they would fill the scalar registers
        const int thread = in_place((int)threadIdx.x), lane = thread & 63, col = lane & 15, quad = lane >> 4, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
        const auto kept_part = [&]() -> Part {
            const i32x4 x = kept[wave][0], y = kept[wave][1], z = kept[wave][2];
            const auto one = [](int32_t v) { return __builtin_amdgcn_readfirstlane(v); };
            return {one(x[0]), one(x[1]), one(x[2]), one(x[3]), one(y[0]), one(y[1]), one(y[2]), one(y[3]), one(z[0]), (uint32_t)one(z[1]), (uint32_t)one(z[2])};
        };
        const Part part = kept_part();
        const int group = (int)a.group.d;
        const int32_t seq = part.seq, tile = part.tile, seq_begin = part.begin, seq_count = part.count, seq_len = part.len;
        const uint32_t kv_head = part.kv_head;
        const int32_t of_tile = part.pad == 0 ? 1 : Shares{part.each, part.pad}.padded(units_of_tile(a, seq, seq_len));
        const int32_t taken = std::min(part.left, of_tile - part.unit);
        const bool whole = taken == of_tile;
        if (a.joins != nullptr && kv_head == 0 && thread == 0 && part.unit == 0 && !whole) {
            JoinItem *const join = a.joins + part.runner;
            join->tile = tile;
            join->begin = seq_begin;
            join->count = seq_count;
            join->len = seq_len;
            join->chunks = 1 + (int32_t)((uint32_t)(of_tile - taken + part.each - 1) / (uint32_t)part.each);
        }

        // this lane's row: the token, the head, the last key that it sees
        const int64_t rows_all = (int64_t)seq_count * group;
        const int64_t r_of_lane = (int64_t)tile * 16 + col;
        const bool row_there = r_of_lane < rows_all;
        const uint32_t row_token = a.group.quotient((uint32_t)(row_there ? r_of_lane : 0));
        const int head = (int)kv_head * group + (int)((uint32_t)(row_there ? r_of_lane : 0) - row_token * a.group.d);
        const int32_t token = row_there ? seq_begin + (int32_t)row_token : -1;
        const int32_t last = row_there ? seq_len - seq_count + (int32_t)row_token : -1;
        if (seq >= a.batch.seqs) { // rows of no sequence
            if (wave == 0 && token >= 0)
                for (int d = quad * 8; d < a.dim; d += 32) store_words<16>(a.out + token * a.out_token + head * a.out_head + d * 2, Words<16>{});
        } else {

            // keys that the tile's rows see, of this runner's part, and of them the wavefront's
            const int64_t top_row = std::min<int64_t>((int64_t)(tile + 1) * 16, rows_all) - 1;
            const int32_t top = seq_len - seq_count + (int32_t)a.group.quotient((uint32_t)top_row) + 1; // keys that the tile's last row sees
            const int32_t lowest = seq_len - seq_count + (int32_t)a.group.quotient((uint32_t)((int64_t)tile * 16)) + 1; // and its first
            const int32_t from = (int32_t)std::min<int64_t>((int64_t)part.unit * kUnit, 0x7fffffc0);
            const int64_t to = part.pad == 0 ? 0x7fffffc0 : (int64_t)from + (int64_t)taken * kUnit;
            const int32_t until = __builtin_amdgcn_readfirstlane((int32_t)std::min<int64_t>(to, std::min(top, walked(a, seq_len))));
            const int32_t pairs_all = until > from ? (int32_t)(((int64_t)until - from + 2 * KT - 1) / (2 * KT)) : 0;
            const int32_t pairs_each = (pairs_all + WAVES - 1) / WAVES;
            int32_t pairs = std::max(0, std::min(pairs_each, pairs_all - wave * pairs_each));
            int32_t key0 = from + wave * pairs_each * 2 * KT;

            // What the end needs, in vector registers: scalar ones are few.
            const int32_t end_tile = in_place(tile), end_begin = in_place(seq_begin), end_count = in_place(seq_count), end_len = in_place(seq_len);
            const int32_t end_place = in_place((int32_t)(part.runner * 2 + (part.unit == 0))), end_parts = in_place(!whole), end_kv_head = in_place((int)kv_head);

            // ---- loading ----
            const auto *const table = (const __attribute__((address_space(4))) int32_t *)(a.batch.table + seq * a.batch.table_stride);
            // Where the next span lies, and the page behind its own.
            uint32_t slot = (uint32_t)key0, at = a.batch.page.quotient((uint32_t)key0);
            slot -= at * a.batch.page.d;
            // The table's entry, of which nothing is asked, so that nothing waits for it, before its page is entered.
            const auto entry_of = [&](uint32_t at) { return table[std::min(at, (uint32_t)a.batch.table_pages - 1)]; };
            const char *k_at, *v_at, *k_scale_at, *v_scale_at;
            bool missing;
            // (Heads' addresses and pages' strides in vector registers where two spans' addresses fill the scalar ones.)
            const auto stored = [](auto x) {
                if constexpr (SPAN == 8) asm volatile("" : "+v"(x));
                return x;
            };
            const auto taken_up = [](uint32_t x) { return SPAN == 8 ? (uint32_t)__builtin_amdgcn_readfirstlane((int)x) : x; };
            const auto address = [&](const char *p) {
                return SPAN == 8 ? (const char *)((uint64_t)taken_up((uint32_t)(uintptr_t)p) | (uint64_t)taken_up((uint32_t)((uintptr_t)p >> 32)) << 32) : p;
            };
            const char *const k_head = stored(a.k + kv_head * a.k_head), *const v_head = stored(a.v + kv_head * a.v_head);
            const char *const k_scale_head = stored(a.k_scales + kv_head * a.k_scale_head), *const v_scale_head = stored(a.v_scales + kv_head * a.v_scale_head);
            const uint32_t cache_pages = stored((uint32_t)a.batch.cache_pages), k_page = stored(a.k_page), v_page = stored(a.v_page), k_scale_page = stored(a.k_scale_page), v_scale_page = stored(a.v_scale_page);
            const auto enter = [&](int32_t entry) { // a page, at slot `slot`
                missing = (uint32_t)entry >= taken_up(cache_pages) || at >= (uint32_t)a.batch.table_pages;
                const uint32_t page = missing ? 0 : (uint32_t)entry;
                k_at = address(k_head) + ((uint64_t)page * taken_up(k_page) + (uint64_t)slot * a.k_slot);
                v_at = address(v_head) + ((uint64_t)page * taken_up(v_page) + (uint64_t)slot * a.v_slot);
                k_scale_at = address(k_scale_head) + ((uint64_t)page * taken_up(k_scale_page) + (uint64_t)slot * a.k_scale_slot);
                v_scale_at = address(v_scale_head) + ((uint64_t)page * taken_up(v_scale_page) + (uint64_t)slot * a.v_scale_slot);
            };
            int32_t entry_behind = 0;
            const auto advance = [&] { // by a span
                slot += SPAN;
                if (slot == a.batch.page.d) {
                    slot = 0;
                    ++at;
                    enter(entry_behind);
                    entry_behind = entry_of(at + 1);
                } else {
                    k_at += SPAN * a.k_slot;
                    v_at += SPAN * a.v_slot;
                    k_scale_at += SPAN * a.k_scale_slot;
                    v_scale_at += SPAN * a.v_scale_slot;
                }
            };
            // Offsets of the lane.  Channels that the head does not have repeat others; their keys' scales become 0.
            const int key_of_lane = (col & 3) * 4 + (col >> 2), scale_key = (col & 3) * 4 + quad; // of 16
            const uint32_t key_in_span = (uint32_t)(key_of_lane & (SPAN - 1)), scale_in_span = (uint32_t)(scale_key & (SPAN - 1));
            const bool has_channels = quad * (D / 4) < a.dim, has_second = D == 256 && quad * 64 + 32 < a.dim; // heads of 256: a lane has two blocks
            const uint32_t k_lane = key_in_span * a.k_slot + (has_channels ? quad * (D / 8) : 0);
            const uint32_t k_scale_lane = key_in_span * a.k_scale_slot + (has_channels ? quad * (D / 4) / 32 : 0);
            const uint32_t k_second = has_second ? 16 : 0, k_scale_second = has_second ? 1 : 0;
            const int value_channel = col * E < a.dim ? col * E : 0;
            uint32_t v_lane[SPAN / 4]; // of keys 4j + quad of a span
#pragma unroll
            for (int j = 0; j < SPAN / 4; ++j) v_lane[j] = (uint32_t)(j * 4 + quad) * a.v_slot + value_channel / 2;
            // A scale for each of 16 keys and 4 blocks: every lane loads another one, that of key 4 (lane mod 4) + quad for the block of its four lanes (heads of 256:
            // the blocks, two).
            const uint32_t v_scale_lane = scale_in_span * a.v_scale_slot + (D == 256 ? std::min((col & ~3) * E / 32, a.dim / 32 - 1) : value_channel / 32);
            const uint32_t v_scale_next = D == 256 && ((col & ~3) * E / 32 + 1) * 32 < a.dim ? 1 : 0;
            const bool key_in_second = SPAN == 8 && key_of_lane >= 8, scale_in_second = SPAN == 8 && scale_key >= 8;
            // Codes of a step; lost: bits of spans without a page.
            const auto fetch = [&](Step<D> &s, uint32_t &lost) {
                lost = 0;
#pragma unroll
                for (int t = 0; t < 2; ++t) { // 16 keys
                    const char *k_of[16 / SPAN], *v_of[16 / SPAN], *k_scale_of[16 / SPAN], *v_scale_of[16 / SPAN];
#pragma unroll
                    for (int i = 0; i < 16 / SPAN; ++i) {
                        k_of[i] = scalar(k_at);
                        v_of[i] = scalar(v_at);
                        k_scale_of[i] = scalar(k_scale_at);
                        v_scale_of[i] = scalar(v_scale_at);
                        lost |= (uint32_t)missing << (t * (16 / SPAN) + i);
                        advance();
                    }
                    const char *const k_from = SPAN == 8 && key_in_second ? k_of[16 / SPAN - 1] : k_of[0];
                    const char *const k_scale_from = SPAN == 8 && key_in_second ? k_scale_of[16 / SPAN - 1] : k_scale_of[0];
                    const char *const v_scale_from = SPAN == 8 && scale_in_second ? v_scale_of[16 / SPAN - 1] : v_scale_of[0];
                    if constexpr (D == 256) {
                        const Words<16> low = load_at<16>(k_from, here(k_lane)), high = load_at<16>(k_from, here(k_lane + k_second));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s.k[t].w[i] = low.w[i];
                            s.k[t].w[4 + i] = high.w[i];
                        }
                    } else {
                        s.k[t] = load_at<Step<D>::kKeyBytes>(k_from, here(k_lane));
                    }
                    s.k_scale[t][0] = load_scale(k_scale_from, here(k_scale_lane));
                    s.v_scale[t][0] = load_scale(v_scale_from, here(v_scale_lane));
                    if constexpr (D == 256) {
                        s.k_scale[t][1] = load_scale(k_scale_from, here(k_scale_lane + k_scale_second));
                        s.v_scale[t][1] = load_scale(v_scale_from, here(v_scale_lane + v_scale_next));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) { // keys 4j + quad
                        const char *const from = v_of[j * 4 / SPAN];
                        if constexpr (D == 64) s.v[t * 4 + j].w[0] = load_two_bytes(from, here(v_lane[j % (SPAN / 4)]));
                        else s.v[t * 4 + j] = load_at<Step<D>::kValueBytes>(from, here(v_lane[j % (SPAN / 4)]));
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

            const auto work = [&](Step<D> &s, int32_t key0, uint32_t lost) {
                // ---- scores ----
                f32x4 score[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    uint32_t scale[Step<D>::kScales]; // of channels that the head does not have: 0, which a NaN would not be
                    scale[0] = has_channels ? read_scale<T>(s.k_scale[t][0]) : 0;
                    if constexpr (D == 256) scale[1] = has_second ? read_scale<T>(s.k_scale[t][1]) : 0;
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
                uint32_t unit[8]; // scales of the lane's block, of each of its keys, as fp32's bits (255: an infinity's)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const auto spread = [&](uint32_t x, uint32_t *to) {
                        to[0] = of_quad<0>(x), to[1] = of_quad<1>(x), to[2] = of_quad<2>(x), to[3] = of_quad<3>(x);
                    };
                    spread(read_scale<T>(s.v_scale[t][0]) << 23, unit + t * 4);
                    if constexpr (D == 256) {
                        uint32_t second[4];
                        spread(read_scale<T>(s.v_scale[t][1]) << 23, second);
#pragma unroll
                        for (int j = 0; j < 4; ++j) unit[t * 4 + j] = (col & 2) != 0 ? second[j] : unit[t * 4 + j];
                    }
                }
                // Two channels: a byte of each of the lane's values, as operands of two products.
                const auto operands = [&](int b, u32x4(&vf)[2]) {
                    uint32_t pair[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float factor = __builtin_bit_cast(float, unit[i]);
                        const uint32_t w = s.v[i].w[b / 4];
                        pair[i] = b % 4 == 0 ? Mfma<T>::template from_fp4<0>(w, factor)
                                             : (b % 4 == 1 ? Mfma<T>::template from_fp4<1>(w, factor)
                                                           : (b % 4 == 2 ? Mfma<T>::template from_fp4<2>(w, factor) : Mfma<T>::template from_fp4<3>(w, factor)));
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        vf[0][i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x05040100u);
                        vf[1][i] = __builtin_amdgcn_perm(pair[2 * i + 1], pair[2 * i], 0x07060302u);
                    }
                };
                // Values that are no finite numbers: a weight of zero would not keep them from the sums of rows that do not see them, nor a second number of the other sign
                // leave an infinity what it is.  They are taken out, and which of them a row sees is counted by a product of its own, as attention_kernel does.
                uint32_t largest = 0; // scale
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < Step<D>::kScales; ++i) largest = std::max(largest, s.v_scale[t][i]);
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(largest > 127 + Mfma<T>::kMostExponent) != 0, 0)) {
                    constexpr uint32_t X = Mfma<T>::kExponent, M = Mfma<T>::kMantissa;
                    const int32_t see = std::min(last, until - 1) - key0 - quad;
                    const uint32_t one = T::narrow1(1.0f);
                    u32x4 seen; // 1 where the row sees the key
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int key = (w >> 1) * 16 + (w & 1) * 8;
                        seen[w] = (one & ~(uint32_t)((see - key) >> 31)) | ((one & ~(uint32_t)((see - key - 4) >> 31)) << 16);
                    }
                    if constexpr (__is_same(T, F16)) { // whole blocks are NaN, and a lane's channels are of one block
                        u32x4 mark;
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            mark[w] = one * ((unit[2 * w] + 0x00800000u) >> 31) | (one * ((unit[2 * w + 1] + 0x00800000u) >> 31)) << 16;
                        const f32x4 found = Mfma<T>::mul(mark, seen, f32x4{0, 0, 0, 0});
#pragma unroll
                        for (int c = 0; c < E; ++c)
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[c][r] += found[r] != 0.0f ? __builtin_nanf("") : 0.0f;
                    } else {
#pragma unroll
                        for (int b = 0; b < E / 2; ++b) {
                            u32x4 vf[2];
                            operands(b, vf);
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                __builtin_amdgcn_sched_barrier(0); // one after the other: interleaved they take too many registers
                                u32x4 mark;
#pragma unroll
                                for (int w = 0; w < 4; ++w) {
                                    uint32_t marks = 0;
#pragma unroll
                                    for (int half = 0; half < 32; half += 16) {
                                        const uint32_t x = (vf[h][w] >> half) & 0xffffu;
                                        const uint32_t code = (x & M) != 0 ? T::narrow1(16384.0f) : ((x & 0x8000u) != 0 ? T::narrow1(128.0f) : T::narrow1(1.0f));
                                        marks |= ((x & X) == X ? code : 0u) << half;
                                    }
                                    mark[w] = marks;
                                }
                                const f32x4 found = Mfma<T>::mul(mark, seen, f32x4{0, 0, 0, 0});
#pragma unroll
                                for (int r = 0; r < 4; ++r) o[b * 2 + h][r] += found_adds(found[r]);
                                asm volatile("" : "+v"(o[b * 2 + h])); // now, not once all channels' marks have been found
                            }
                        }
                    }
                    // codes that are infinities become 0, and so do NaN blocks' scales
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (__is_same(T, Bf16)) {
#pragma unroll
                            for (int j = 0; j < (E + 7) / 8; ++j) {
                                const uint32_t two = s.v[i].w[j] >> 2 & 0x11111111u, four = two & s.v[i].w[j] >> 1; // from there on, a bit for each
                                s.v[i].w[j] &= ~((unit[i] == 0x7f000000u ? two : (unit[i] == 0x7e800000u ? four : 0u)) * 15u);
                            }
                        }
                        unit[i] &= ((unit[i] + 0x00800000u) >> 31) - 1;
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
                enter(entry_of(at));
                entry_behind = entry_of(at + 1);
                fetch(s0, lost0);
                fetch(s1, lost1);
                for (; pairs > 1; --pairs) {
                    work(s0, key0, lost0);
                    fetch(s0, lost0);
                    work(s1, key0 + KT, lost1);
                    fetch(s1, lost1);
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
            const int64_t at_part = ((int64_t)end_place * late.kv_heads.d + end_kv_head) * 16; // of the partial results
            // thread -> row and four channels
            for (int at = thread; at < 16 * (D / 4); at += 64 * WAVES) {
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

        // ---- the next part ----
        const AttentionFp4Args &again = arguments_again<AttentionFp4Args>();
        Part next = kept_part();
        const auto units_again = [&](int i, int32_t len) { return next.pad == 0 ? 1 : Shares{next.each, next.pad}.padded(units_of_tile(again, i, len)); };
        next.left -= units_again(next.seq, next.len) - next.unit;
        if (next.left <= 0) return;
        next.unit = 0;
        if (++next.tile >= tiles_of<16>(again, next.count)) { // the next sequence with tiles
            next.tile = 0;
            ++next.seq;
            for (;; next.seq += 64) {
                if (next.seq > again.batch.seqs + 1) return;
                int32_t begins, counts, lens;
                extent(again, next.seq + lane, begins, counts, lens);
                const uint64_t there = __builtin_amdgcn_ballot_w64(tiles_to_do(again, next.seq + lane, counts) > 0);
                if (there == 0) continue;
                const int at = __builtin_ctzll(there);
                next.seq += at;
                next.begin = __builtin_amdgcn_readlane(begins, at), next.count = __builtin_amdgcn_readlane(counts, at), next.len = __builtin_amdgcn_readlane(lens, at);
                break;
            }
        }
        keep(next);
        __syncthreads(); // the wavefronts' results have been read
    }
}

namespace {

// Where a runner's cut tile has its parts: the first in the runner's second place, the others in the following runners' first ones.
__device__ __forceinline__ const float *part_of(const AttentionFp4Args &a, int row_floats, uint32_t runner, uint32_t kv_head, int row, int part) {
    const int64_t place = part == 0 ? 2 * (int64_t)runner + 1 : 2 * ((int64_t)runner + part);
    return a.partial + ((place * a.kv_heads.d + kv_head) * 16 + row) * (int64_t)row_floats;
}

// A row of a cut tile: the token, its place in the output; false: there is none.
struct JoinedRow {
    char *to;
    int64_t r; // among the sequence's
    bool there, sees;
};
__device__ __forceinline__ JoinedRow joined_row(const AttentionFp4Args &a, const JoinItem &j, uint32_t kv_head, int row) {
    JoinedRow o;
    o.r = (int64_t)j.tile * 16 + row;
    o.there = o.r < (int64_t)j.count * a.group.d;
    const uint32_t t = a.group.quotient((uint32_t)(o.there ? o.r : 0));
    const int head = (int)(kv_head * a.group.d) + (int)((uint32_t)(o.there ? o.r : 0) - t * a.group.d);
    o.to = a.out + (j.begin + (int64_t)t) * a.out_token + head * a.out_head;
    o.sees = j.len - j.count + (int64_t)t >= 0;
    return o;
}

// Parts of a row, one after the other, to a running maximum: each lane E neighbouring channels.
template <int E>
struct Joined {
    float best = -__builtin_inff(), all = 0.0f, sum[E] = {};
    __device__ __forceinline__ void scale_to(float top, float scale_log2) {
        const float old = __builtin_amdgcn_exp2f((best - seen_or_zero(top)) * scale_log2);
        all *= old;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] *= old;
        best = top;
    }
    // AT parts that are there where `counts`.
    template <int AT>
    __device__ __forceinline__ void add(const float (&m)[AT], const float (&l)[AT], const float (&x)[AT][E], const bool (&counts)[AT], float scale_log2) {
        float top = best;
#pragma unroll
        for (int i = 0; i < AT; ++i) top = counts[i] ? __builtin_fmaxf(top, m[i]) : top;
        scale_to(top, scale_log2);
        const float from = seen_or_zero(top);
#pragma unroll
        for (int i = 0; i < AT; ++i) {
            const float weight = __builtin_amdgcn_exp2f((m[i] - from) * scale_log2);
            all += counts[i] ? l[i] * weight : 0.0f; // what a place holds that does not count may not be finite
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += counts[i] ? x[i][e] * weight : 0.0f;
        }
    }
};

} // namespace

// Joins the parts of tiles that were cut: a wavefront a row, eight parts at once.
template <class T, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(const AttentionFp4Args a) {
    constexpr int E = D / 64, AHEAD = 8;
    const int lane = threadIdx.x & 63;
    const uint32_t at = blockIdx.x / 4, runner = a.kv_heads.quotient(at), kv_head = at - runner * a.kv_heads.d;
    const JoinItem j = a.joins[runner];
    if (j.chunks <= 0) return;
    const int row = (int)(blockIdx.x % 4) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const JoinedRow o = joined_row(a, j, kv_head, row);
    if (!o.there) return;
    const int parts = (int)std::min<int64_t>(j.chunks, a.runners.d - runner);
    Joined<E> all;
    for (int c0 = 0; c0 < parts; c0 += AHEAD) {
        float m[AHEAD], l[AHEAD], x[AHEAD][E];
        bool counts[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            counts[i] = c0 + i < parts;
            const float *const part = part_of(a, D + 4, runner, kv_head, row, counts[i] ? c0 + i : c0);
            m[i] = part[D];
            l[i] = part[D + 1];
#pragma unroll
            for (int e = 0; e < E; ++e) x[i][e] = part[lane * E + e];
        }
        all.add(m, l, x, counts, a.scale_log2);
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (lane * E + e < a.dim) store_element<T>(o.to + (lane * E + e) * 2, o.sees ? all.sum[e] / all.all : 0.0f);
}

// The same where few tiles have very many parts: a workgroup 32 channels of a row, 8 lanes a part, 128 parts at once, and again.  (One row over 262144 keys, 512 parts:
// a workgroup a row took 12 us.)
constexpr int kMostRunners = 1024;
template <class T, int D>
__global__ void __launch_bounds__(1024) decode_join_many_kernel(const AttentionFp4Args a) {
    constexpr int SLICES = D / 32, AHEAD = 4;
    __shared__ int cut_of_wave[16], found;
    __shared__ __align__(16) float joined[16][32 + 2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t tile = blockIdx.x / (SLICES * 16), of_tile = blockIdx.x - tile * (SLICES * 16), cut = a.kv_heads.quotient(tile);
    const uint32_t kv_head = tile - cut * a.kv_heads.d;
    const int row = (int)(of_tile / SLICES), slice = (int)(of_tile % SLICES);
    // the runner that began the tile with number `cut` of those that were cut
    const bool begins = threadIdx.x < a.runners.d && a.joins[threadIdx.x].chunks > 0;
    const uint64_t of_wave = __builtin_amdgcn_ballot_w64(begins);
    if (threadIdx.x == 0) found = -1;
    if (lane == 0) cut_of_wave[wave] = __builtin_popcountll(of_wave);
    __syncthreads();
    uint32_t number = __builtin_popcountll(of_wave & (((uint64_t)1 << lane) - 1));
    for (int w = 0; w < wave; ++w) number += cut_of_wave[w];
    if (begins && number == cut) found = (int)threadIdx.x;
    __syncthreads();
    const int runner = found;
    if (runner < 0) return;
    const JoinItem j = a.joins[runner];
    const JoinedRow o = joined_row(a, j, kv_head, row);
    if (!o.there) return;
    const int parts = (int)std::min<int64_t>(j.chunks, (int64_t)a.runners.d - runner);
    Joined<4> all;
    for (int c0 = wave * 8 + (lane >> 3); c0 < parts; c0 += 128 * AHEAD) {
        float m[AHEAD], l[AHEAD], x[AHEAD][4];
        bool counts[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            counts[i] = c0 + i * 128 < parts;
            const float *const part = part_of(a, D + 4, runner, kv_head, row, counts[i] ? c0 + i * 128 : c0);
            m[i] = part[D];
            l[i] = part[D + 1];
            const f32x4 four = *(const f32x4 *)(part + slice * 32 + (lane & 7) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = four[e];
        }
        all.add(m, l, x, counts, a.scale_log2);
    }
    // over the wavefront's parts, then over the wavefronts
    float top = all.best;
#pragma unroll
    for (int s = 8; s < 64; s <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, s));
    all.scale_to(top, a.scale_log2);
#pragma unroll
    for (int s = 8; s < 64; s <<= 1) {
        all.all += __shfl_xor(all.all, s);
#pragma unroll
        for (int e = 0; e < 4; ++e) all.sum[e] += __shfl_xor(all.sum[e], s);
    }
    if (lane < 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) joined[wave][lane * 4 + e] = all.sum[e];
        if (lane == 0) {
            joined[wave][32] = top;
            joined[wave][33] = all.all;
        }
    }
    __syncthreads();
    if (threadIdx.x >= 32) return;
    float m[16], l[16], x[16][1];
    bool counts[16];
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        counts[w] = true;
        m[w] = joined[w][32];
        l[w] = joined[w][33];
        x[w][0] = joined[w][lane];
    }
    Joined<1> last;
    last.add(m, l, x, counts, a.scale_log2);
    const int d = slice * 32 + lane;
    if (d < a.dim) store_element<T>(o.to + d * 2, o.sees ? last.sum[0] / last.all : 0.0f);
}

namespace {

template <class T, int D>
void launch_decode(const AttentionFp4Args &a, const AttentionPlan &p, hipStream_t s) {
    const uint32_t blocks = a.runners.d * a.kv_heads.d;
    if (a.batch.page.d % 16 == 0) decode_fp4_kernel<T, D, kDecodeWaves, 16><<<blocks, 64 * kDecodeWaves, 0, s>>>(a);
    else decode_fp4_kernel<T, D, kDecodeWaves, 8><<<blocks, 64 * kDecodeWaves, 0, s>>>(a);
    if (!p.split) return;
    if (p.join_waves == 16) decode_join_many_kernel<T, D><<<(uint32_t)p.tiles * a.kv_heads.d * (D / 2), 1024, 0, s>>>(a);
    else decode_join_kernel<T, D><<<blocks * 4, 256, 0, s>>>(a);
}

template <class T>
void launch_decode_type(const AttentionFp4Args &a, const AttentionPlan &p, hipStream_t s) {
    if (p.wide_dim == 64) launch_decode<T, 64>(a, p, s);
    else if (p.wide_dim == 128) launch_decode<T, 128>(a, p, s);
    else launch_decode<T, 256>(a, p, s);
}

} // namespace

namespace {

// Which kernel.  Calls whose sequences have few rows on average go to the decode kernel, tiles of 16 rows; the others to tiles of 64 and more.  How many are few:
// 16; with heads of up to 64 channels 32 where tiles of 64 would leave units idle (48 sequences of 6 x 4 rows over 6000 keys 55 us, tiles of 64 69; but 300 over
// 600 85 and 76), of up to 128 32 (64 sequences of 8 x 4 over 4000 115 and 120, of up to as many 69 and 94; with 48 153 and 121), of more 96, as tiles of 64
// leave them one wavefront a SIMD (20 of 8 x 6 over 6000 97 and 155, of 24 x 4 over 6000 171 and 351; 64 of up to 30 x 4 over 500 57 and 52).  The average decides for all
// rows: a chunk beside many single rows goes to tiles of 16 as well, single rows beside a long chunk to large ones (4 heads a key head, up to 2000 keys, the chunk behind
// 1000: 255 rows and 1500 206 us, in two calls 82 and 98; 60 and 400 62, 36 and 41; 63 and 4000, large tiles, 268, 36 and 204; in heads of 256 60 and 1500 276, 54 and 161).
int64_t few_rows(int wide_dim, int64_t tiles) {
    return wide_dim == 256 ? 96 : (wide_dim == 128 || tiles < device_compute_units() ? 32 : 16);
}

// Tiles that share keys.  Heads of 65 to 128 take 256 rows where those are two workgroups a unit at most and sequences are long (128 rows, two workgroups
// at once, make numbers of all codes twice): 4096 rows behind 4096 382 us and 415, 3700 behind 8000 582 and 644, 2 x 2048 behind 2048 206 and 236, 3100 by
// themselves 101 and 103.  Elsewhere a unit that gets one tile more than others costs what that saves: 5000 rows behind 2000 413 and 399, 8192 by themselves 526
// and 545, 20 sequences of up to 700 behind 3000 129 and 117.
//
// Heads of more than 128 take 128 rows, two wavefronts a SIMD, where those give three units of eight a tile, of two sequences at most two of eight; fewer are split,
// in tiles of 64 rows, whose one wavefront a SIMD is slow: 1200 rows x 4 on 4 key heads behind 4000 243 us and 432, 600 214 and 260, 450 208 and 155; of 8 sequences of
// up to 200 behind 8000 300 and 320, of 12 of up to 120 336 and 249.
//
// Calls of 16 rows a sequence and less that the decode kernel does not take have their weights as two numbers, as it has, in tiles of 64 rows, of which they fill few (64
// rows over up to 8192 keys in pages of 12 tokens 201 us, one number 183; 48 x 3 over up to 6000 in heads of 64 60 and 42; 20 over up to 6000 in heads of 256 238 and 197).
int plan_tiles(int dim, int64_t tokens, int q_heads, int kv_heads, int seqs, int64_t capacity, AttentionPlan *p) {
    const int64_t rows_all = tokens * (q_heads / kv_heads), cus = device_compute_units();
    const bool two_numbers = rows_all <= (int64_t)seqs * 16;
    const int status = plan_attention_rows(dim, tokens, q_heads, kv_heads, seqs, capacity, 64, two_numbers ? 64 : 128, p);
    p->two_numbers = two_numbers;
    if (status != TDE_OK || two_numbers) return status;
    if (p->wide_dim == 256 && p->rows == 64 && rows_all / 128 * kv_heads >= cus * (seqs <= 2 ? 2 : 3) / 8) {
        *p = AttentionPlan{};
        p->wide_dim = 256;
        p->rows = 128;
        p->join_waves = 1;
    } else if (p->wide_dim == 128 && p->rows == 128 && rows_all >= (int64_t)seqs * 8192 && rows_all / 256 * kv_heads <= 2 * cus) {
        p->rows = 256;
    } else {
        return TDE_OK;
    }
    p->tiles = p->items = rows_all / p->rows + seqs + 2;
    return fits_launch(p->items * kv_heads, 512) ? TDE_OK : TDE_ETOOBIG;
}

} // namespace

int plan_attention_fp4(int dim, int64_t tokens, int q_heads, int kv_heads, const tde_paged_batch &b, bool near, AttentionPlan *p) {
    const int64_t rows_all = tokens * (q_heads / kv_heads), capacity = (int64_t)b.table_pages * b.page_size;
    const int wide_dim = dim <= 64 ? 64 : (dim <= 128 ? 128 : 256);
    // (It takes pages of whole 8 keys, and a table and caches that have any.)
    if (!near || b.page_size % 8 != 0 || b.table_pages == 0 || b.cache_pages == 0 || rows_all > b.seqs * few_rows(wide_dim, (int64_t)b.seqs * kv_heads))
        return plan_tiles(dim, tokens, q_heads, kv_heads, b.seqs, capacity, p);
    *p = AttentionPlan{};
    p->wide_dim = wide_dim;
    p->rows = 16;
    // As many runners as the device holds workgroups, by their registers; every die the same number.
    const int64_t tiles = rows_all / 16 + b.seqs + 2;
    const int64_t most = std::max<int64_t>(kDecodeWaves, (capacity + kUnit) / kUnit); // units of a tile
    if (tiles > 0x7fffff00 / most) return plan_tiles(dim, tokens, q_heads, kv_heads, b.seqs, capacity, p); // units are counted in 32 bits
    const int64_t at_once = std::max<int64_t>(1, std::min<int64_t>((int64_t)resident_workgroups(p->wide_dim, b.page_size % 16 == 0 ? 16 : 8) * device_compute_units() / kv_heads, kMostRunners));
    const int64_t likely = std::max<int64_t>({1, std::min<int64_t>(b.seqs, tokens), rows_all / 16}); // tiles
    // Where tiles alone fill the device more than twice each is a runner's, and nothing is cut (200 rows over 1500 keys 52 us and 61, 512 over 2047 216 and 225).
    // Lengths, which are the device's, do not count: one that is far longer than the others is walked by a workgroup for each key head (200 rows over 500 keys 35 us,
    // with 131072 keys in one of them 943; 191 rows, which are shared out, 34 and 75).
    p->whole_tiles = likely >= 2 * at_once;
    p->runners = p->whole_tiles ? tiles : std::min(at_once >= 8 ? at_once & ~(int64_t)7 : at_once, (tiles * most + kDecodeWaves - 1) / kDecodeWaves);
    p->split = !p->whole_tiles && most > kDecodeWaves;
    p->tiles = std::min(tiles, p->runners); // that can be cut, or more
    const int64_t runners = p->runners;
    // of a runner, with the few that are left over where tiles begin at runners (a third more) and the rounding
    p->most_each = std::min<int64_t>((tiles * most / runners + kDecodeWaves) * 2, 0x7fffff00);
    if (runners > 0x7fffff00 / kv_heads || !fits_launch(runners * kv_heads * 4, 256)) return TDE_ETOOBIG;
    // few tiles of very many parts
    p->join_waves = runners / likely >= 32 && fits_launch(p->tiles * kv_heads * (p->wide_dim / 2), 1024) ? 16 : 1;
    if (p->split) p->workspace_bytes = runners * (int64_t)sizeof(JoinItem) + 2 * runners * kv_heads * 16 * (int64_t)(p->wide_dim + 4) * 4;
    return TDE_OK;
}

int launch_attention_fp4(AttentionFp4Args &a, const AttentionPlan &p, int dtype, hipStream_t s) {
    if (p.rows != 16) return launch_planned<HeldFp4>(a, p, dtype, s);
    a.runners = Divisor32((uint32_t)p.runners);
    a.whole_tiles = p.whole_tiles;
    a.most_each = (int32_t)p.most_each;
    a.capacity = (int32_t)std::min<int64_t>((int64_t)a.batch.table_pages * a.batch.page.d, 0x7fffff00);
    a.joins = p.split ? reinterpret_cast<JoinItem *>(a.partial + 2 * p.runners * a.kv_heads.d * 16 * (p.wide_dim + 4)) : nullptr;
    if (dtype == TDE_BF16) launch_decode_type<Bf16>(a, p, s);
    else launch_decode_type<F16>(a, p, s);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace block
} // namespace tde
