// A step's lengths, page tables and slot maps: sequences shrink, their pages go back on the stack, sequences grow with pages from it.
//
// All of it is sums over the sequences in order: a page that goes back or comes has a number among the call's, and with it its place on the stack; a row has
// its number among the rows.  One workgroup does it, a sequence a thread, with sums over the threads; pages and rows, of which a sequence has any number,
// are then shared out evenly, and each looks up whose it is in the sums.  A workgroup sees what it has written behind a barrier, so nothing has to wait
// for another launch; only the maps of many rows are a launch of their own, over all units.
//
// Bound by latency: loads of the lengths, a sum over the workgroup (a second one if something is missing), a load from the stack, one from the table.  64
// sequences of 4 rows take 4.2 us in a captured graph, where an empty kernel takes 1.6.
#include "tde_page_update.h"

#include <type_traits>

namespace tde {
namespace block {

namespace {

template <int N>
using Is = std::integral_constant<int, N>;

// x + y, most at most, whatever they are: the addition ends at 2^32 - 1.
__device__ __forceinline__ uint32_t add_up_to(uint32_t x, uint32_t y, uint32_t most) { return min(__builtin_elementwise_add_sat(x, y), most); }

struct Sums {
    uint32_t upto[2], all[2]; // inclusive, and over the workgroup
};
// Sums of two numbers over the threads, each up to a most that no sum exceeds; `parts` is free again at the next barrier.
template <int THREADS>
__device__ __forceinline__ Sums sums_over_threads(uint32_t x0, uint32_t x1, uint32_t most0, uint32_t most1, uint32_t (*parts)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t y0 = __shfl_up(x0, m), y1 = __shfl_up(x1, m);
        if (lane >= m) {
            x0 = add_up_to(x0, y0, most0);
            x1 = add_up_to(x1, y1, most1);
        }
    }
    __syncthreads(); // the sums before have been read
    if (lane == 63) {
        parts[wave][0] = x0;
        parts[wave][1] = x1;
    }
    __syncthreads();
    Sums s{{x0, x1}, {0, 0}};
    for (int w = 0; w < THREADS / 64; ++w) {
        const uint32_t p0 = parts[w][0], p1 = parts[w][1];
        if (w < wave) {
            s.upto[0] = add_up_to(s.upto[0], p0, most0);
            s.upto[1] = add_up_to(s.upto[1], p1, most1);
        }
        s.all[0] = add_up_to(s.all[0], p0, most0);
        s.all[1] = add_up_to(s.all[1], p1, most1);
    }
    return s;
}

// The first of n ascending sums that exceeds e, which the last one does.
__device__ __forceinline__ int owner_of(const uint32_t *sums, int n, uint32_t e) { // n >= 1
    int low = 0;
    while (n > 1) {
        const int half = n >> 1;
        if (sums[low + half - 1] <= e) {
            low += half;
            n -= half;
        } else {
            n = half;
        }
    }
    return low;
}

struct Lengths {
    uint32_t keep, had_pages, kept_pages; // pages that the table's row has
};
__device__ __forceinline__ uint32_t pages_of(const PageUpdateArgs &a, uint32_t tokens) {
    const uint32_t whole = a.page.quotient(tokens);
    return whole + (uint32_t)(whole * a.page.d < tokens);
}
__device__ __forceinline__ Lengths lengths_of(const PageUpdateArgs &a, int seq) {
    const int32_t len = max(a.lens[seq], 0);
    const int32_t keep = a.kept == nullptr ? len : min(max(a.kept[seq], 0), len);
    const uint32_t width = (uint32_t)a.width;
    return {(uint32_t)keep, min(pages_of(a, (uint32_t)len), width), min(pages_of(a, (uint32_t)keep), width)};
}

} // namespace

// Any number of sequences, THREADS at a time.
template <bool MAPS>
__global__ void __launch_bounds__(1024) page_update_kernel(const PageUpdateArgs a) {
    constexpr int THREADS = 1024;
    __shared__ uint32_t parts[THREADS / 64][2], pages_upto[THREADS], rows_upto[THREADS], first_page[THREADS], keep_of[THREADS];
    constexpr uint32_t kAny = 0x80000000u;
    const int tid = threadIdx.x;
    const uint32_t before = (uint32_t)min(max(*a.count, 0), a.capacity);

    // ---- pages back on the stack ----
    uint32_t returned = 0; // of all sequences: the first one's first page ends up on top
    if (a.kept != nullptr) {
        uint32_t mine = 0;
        for (int seq = tid; seq < a.seqs; seq += THREADS) {
            const Lengths l = lengths_of(a, seq);
            mine += l.had_pages - l.kept_pages;
        }
        returned = sums_over_threads<THREADS>(mine, 0, kAny, kAny, parts).all[0];
        uint32_t passed = 0;
        for (int base = 0; base < a.seqs && returned != 0; base += THREADS) {
            const int seq = base + tid;
            const Lengths l = seq < a.seqs ? lengths_of(a, seq) : Lengths{};
            const Sums s = sums_over_threads<THREADS>(l.had_pages - l.kept_pages, 0, kAny, kAny, parts);
            pages_upto[tid] = s.upto[0];
            first_page[tid] = l.kept_pages;
            __syncthreads();
            for (uint32_t e = tid; e < s.all[0]; e += THREADS) {
                const int at = owner_of(pages_upto, THREADS, e);
                const uint32_t page = first_page[at] + (e - (at == 0 ? 0 : pages_upto[at - 1])), place = before + returned - 1 - (passed + e);
                if (place < (uint32_t)a.capacity) a.stack[place] = a.table[(base + at) * a.table_stride + page];
            }
            passed += s.all[0];
            __syncthreads();
        }
    }
    const uint32_t there = min(before + returned, (uint32_t)a.capacity);

    // ---- sequences grow ----
    uint32_t asked_pages = 0, asked_rows = 0, taken = 0, rows = 0;
    for (int base = 0; base < a.seqs; base += THREADS) {
        const int seq = base + tid;
        const Lengths l = seq < a.seqs ? lengths_of(a, seq) : Lengths{};
        const uint32_t more = seq < a.seqs ? (uint32_t)max(a.added[seq], 0) : 0;
        const uint32_t then = l.keep + more; // below 2^32
        const uint32_t need_pages = then <= 0x7fffffffu ? pages_of(a, then) : 0x80000000u; // which no row of the table has
        const bool fits = need_pages <= (uint32_t)a.width;
        const uint32_t need = fits && more != 0 ? need_pages - l.kept_pages : 0;
        const uint32_t most_pages = there + 1, most_rows = (uint32_t)a.tokens + 1;
        const Sums asked = sums_over_threads<THREADS>(min(need, most_pages), fits ? min(more, most_rows) : 0, most_pages, most_rows, parts);
        const bool served = fits && (need == 0 || add_up_to(asked_pages, asked.upto[0], most_pages) <= there) &&
                            add_up_to(asked_rows, asked.upto[1], most_rows) <= (uint32_t)a.tokens;
        asked_pages = add_up_to(asked_pages, asked.all[0], most_pages);
        asked_rows = add_up_to(asked_rows, asked.all[1], most_rows);
        const Sums s = sums_over_threads<THREADS>(served ? need : 0, served ? more : 0, kAny, kAny, parts);
        pages_upto[tid] = s.upto[0];
        rows_upto[tid] = s.upto[1];
        first_page[tid] = l.kept_pages;
        keep_of[tid] = l.keep;
        if (seq < a.seqs) {
            a.lens[seq] = (int32_t)(l.keep + (served ? more : 0));
            a.starts[seq + 1] = (int32_t)(rows + s.upto[1]);
        }
        __syncthreads();
        for (uint32_t e = tid; e < s.all[0]; e += THREADS) {
            const int at = owner_of(pages_upto, THREADS, e);
            const uint32_t page = first_page[at] + (e - (at == 0 ? 0 : pages_upto[at - 1]));
            a.table[(base + at) * a.table_stride + page] = a.stack[there - 1 - (taken + e)];
        }
        __syncthreads();
        if (MAPS) {
            for (uint32_t e = tid; e < s.all[1]; e += THREADS) {
                const int at = owner_of(rows_upto, THREADS, e);
                const uint32_t position = keep_of[at] + (e - (at == 0 ? 0 : rows_upto[at - 1])), page = a.page.quotient(position);
                a.positions[rows + e] = (int32_t)position;
                a.slots[rows + e] = (int64_t)a.table[(base + at) * a.table_stride + page] * a.page.d + (position - page * a.page.d);
            }
        }
        taken += s.all[0];
        rows += s.all[1];
    }
    if (tid == 0) {
        a.starts[0] = 0;
        *a.count = (int32_t)(there - taken);
    }
    if (MAPS)
        for (uint32_t t = rows + tid; t < (uint32_t)a.tokens; t += THREADS) {
            a.positions[t] = -1;
            a.slots[t] = -1;
        }
}

// The same for no more sequences than threads: one sum over them says what goes back, what is asked for and, unless something is missing, what is given.
template <int THREADS, bool MAPS>
__global__ void __launch_bounds__(THREADS) page_update_once_kernel(const PageUpdateArgs a) {
    constexpr int WAVES = THREADS / 64;
    constexpr uint32_t kAny = 0x7fffffffu;
    __shared__ uint32_t parts[2][WAVES][3], back_upto[THREADS], pages_upto[THREADS], rows_upto[THREADS], first_page[THREADS], keep_of[THREADS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool there_is = tid < a.seqs;
    const Lengths l = there_is ? lengths_of(a, tid) : Lengths{};
    const uint32_t more = there_is ? (uint32_t)max(a.added[tid], 0) : 0;
    const uint32_t before = (uint32_t)min(max(*a.count, 0), a.capacity);
    const uint32_t then = l.keep + more; // below 2^32
    const uint32_t need_pages = then <= 0x7fffffffu ? pages_of(a, then) : 0x80000000u; // which no row of the table has
    const bool fits = need_pages <= (uint32_t)a.width;
    const uint32_t need = fits && more != 0 ? need_pages - l.kept_pages : 0;

    // Sums over the threads up to each one and of all, no more than kAny.
    struct Three {
        uint32_t v[3];
    };
    const auto sums = [&](Three &upto, Three &all, uint32_t(&of_waves)[WAVES][3]) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const auto add = [&](auto control, auto rows) {
                upto.v[k] = add_up_to(upto.v[k], (uint32_t)__builtin_amdgcn_update_dpp(0, (int)upto.v[k], decltype(control)::value, decltype(rows)::value, 0xf, false), kAny);
            };
            // from 1, 2, 4, 8 lanes below, of rows of 16; a row's last lane to the next row, the second one's to the upper half
            add(Is<0x111>{}, Is<0xf>{}), add(Is<0x112>{}, Is<0xf>{}), add(Is<0x114>{}, Is<0xf>{}), add(Is<0x118>{}, Is<0xf>{});
            add(Is<0x142>{}, Is<0xa>{}), add(Is<0x143>{}, Is<0xc>{});
            if (lane == 63) of_waves[wave][k] = upto.v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            uint32_t below = 0, sum = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                below = w == wave ? sum : below;
                sum = add_up_to(sum, of_waves[w][k], kAny);
            }
            upto.v[k] = add_up_to(upto.v[k], below, kAny);
            all.v[k] = sum;
        }
    };
    Three upto{{l.had_pages - l.kept_pages, need, fits ? more : 0}}, all;
    sums(upto, all, parts[0]);
    const uint32_t returned = all.v[0], back = upto.v[0], there = min(before + returned, (uint32_t)a.capacity);
    bool served = fits;
    if (all.v[1] > there || all.v[2] > (uint32_t)a.tokens) { // some wait
        served = fits && (need == 0 || upto.v[1] <= there) && upto.v[2] <= (uint32_t)a.tokens;
        upto = Three{{0, served ? need : 0, served ? more : 0}};
        sums(upto, all, parts[1]);
    }
    back_upto[tid] = back;
    pages_upto[tid] = upto.v[1];
    rows_upto[tid] = upto.v[2];
    first_page[tid] = l.kept_pages;
    keep_of[tid] = l.keep;
    if (there_is) {
        a.lens[tid] = (int32_t)(l.keep + (served ? more : 0));
        a.starts[tid + 1] = (int32_t)upto.v[2];
    }
    const uint32_t taken = all.v[1], rows = all.v[2];
    if (tid == 0) {
        a.starts[0] = 0;
        *a.count = (int32_t)(there - taken);
    }
    __syncthreads();
    for (uint32_t e = tid; e < returned; e += THREADS) {
        const int at = owner_of(back_upto, a.seqs, e);
        const uint32_t page = first_page[at] + (e - (at == 0 ? 0 : back_upto[at - 1])), place = before + returned - 1 - e;
        if (place < (uint32_t)a.capacity) a.stack[place] = a.table[at * a.table_stride + page];
    }
    __syncthreads();
    for (uint32_t e = tid; e < taken; e += THREADS) {
        const int at = owner_of(pages_upto, a.seqs, e);
        const uint32_t page = first_page[at] + (e - (at == 0 ? 0 : pages_upto[at - 1]));
        a.table[at * a.table_stride + page] = a.stack[there - 1 - e];
    }
    if constexpr (MAPS) {
        __syncthreads();
        for (uint32_t t = tid; t < (uint32_t)a.tokens; t += THREADS) {
            int32_t position = -1;
            int64_t slot = -1;
            if (t < rows) {
                const int at = owner_of(rows_upto, a.seqs, t);
                const uint32_t p = keep_of[at] + (t - (at == 0 ? 0 : rows_upto[at - 1])), page = a.page.quotient(p);
                position = (int32_t)p;
                slot = (int64_t)a.table[at * a.table_stride + page] * a.page.d + (p - page * a.page.d);
            }
            a.positions[t] = position;
            a.slots[t] = slot;
        }
    }
}

// Positions and slots of many rows, after the tables: a row a thread.
__global__ void __launch_bounds__(256) page_maps_kernel(const PageUpdateArgs a) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t >= (uint32_t)a.tokens) return;
    int32_t position = -1;
    int64_t slot = -1;
    if (t < (uint32_t)a.starts[a.seqs]) {
        int low = 0; // sequences that end at or before the row
        for (int n = a.seqs; n > 1;) {
            const int half = n >> 1;
            if ((uint32_t)a.starts[low + half] <= t) {
                low += half;
                n -= half;
            } else {
                n = half;
            }
        }
        position = a.lens[low] - (a.starts[low + 1] - (int32_t)t);
        const uint32_t page = a.page.quotient((uint32_t)position);
        slot = (int64_t)a.table[low * a.table_stride + page] * a.page.d + ((uint32_t)position - page * a.page.d);
    }
    a.positions[t] = position;
    a.slots[t] = slot;
}

int launch_page_update(const PageUpdateArgs &a, hipStream_t s) {
    // Threads: 64 sequences with 4 rows each take 4.2 us with 256 and 5.3 with 1024; 200 with 16 take 9.0 and 6.6.  Maps in a launch of their own: 64
    // sequences with 128 rows take 8.1 us, 7.8 without; 16 with 1024 take 7.4, 8.7 without.
    const bool maps = a.tokens > 4096;
    if (a.seqs <= 256 && a.tokens <= 512) page_update_once_kernel<256, true><<<1, 256, 0, s>>>(a);
    else if (a.seqs <= 1024 && !maps) page_update_once_kernel<1024, true><<<1, 1024, 0, s>>>(a);
    else if (a.seqs <= 1024) page_update_once_kernel<1024, false><<<1, 1024, 0, s>>>(a);
    else if (!maps) page_update_kernel<true><<<1, 1024, 0, s>>>(a);
    else page_update_kernel<false><<<1, 1024, 0, s>>>(a);
    if (maps) page_maps_kernel<<<((uint32_t)a.tokens + 255) / 256, 256, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? TDE_OK : hip_failed(e);
}

} // namespace block
} // namespace tde
