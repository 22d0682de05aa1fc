// Host check of what the paged kernels compute addresses from (csrc/tde_block.h): quotients for every kind of divisor, and page
// numbers from tables that hold anything.  Exit status 0: everything right.
#include "tde_block.h"

#include <cstdio>
#include <vector>

using namespace tde::block;

int main() {
    long wrong = 0;
    std::vector<uint32_t> divisors = {1, 2, 3, 5, 7, 16, 24, 33, 64, 100, 127, 128, 1000, 4096, 65535, 65536, 65537, 1u << 20, (1u << 30) - 1, 1u << 30, 0x7fffffffu};
    for (uint32_t i = 1; i < 3000; ++i) divisors.push_back(i);
    for (uint32_t d : divisors) {
        const Divisor32 div(d);
        const auto check = [&](uint64_t n) {
            if (n < (1ull << 31) && div.quotient((uint32_t)n) != (uint32_t)n / d) ++wrong;
        };
        for (uint64_t n = 0; n < 300; ++n) check(n), check(0x7fffffffull - n);
        for (uint64_t m = d; m < (1ull << 31); m += d + m / 3) check(m - 1), check(m), check(m + 1);
        for (uint64_t k = 1; k < 60; ++k) check(k * d - 1), check(k * d), check(((1ull << 31) / d - (k < (1ull << 31) / d ? k : 0)) * d - 1);
    }
    const Divisor32 unset;
    for (uint32_t n = 0; n < 100; ++n) wrong += unset.quotient(n) != n;

    // rows of three entries inside a larger array: the neighbours hold valid pages that must not be taken
    const int32_t table[] = {1, 1, 1, /**/ 0, -1, 4, /**/ 1, 1, 1};
    PagedBatch b{};
    b.table_pages = 3;
    b.cache_pages = 4;
    wrong += page_number(b, table + 3, 0) != 0;
    wrong += page_number(b, table + 3, 1) != -1;
    wrong += page_number(b, table + 3, 2) != -1;
    for (uint32_t at : {3u, 4u, 0x7fffffffu, 0x80000000u, 0xffffffffu}) wrong += page_number(b, table + 3, at) != -1;
    const int32_t odd[] = {3, (int32_t)0x80000000, 0x7fffffff};
    wrong += page_number(b, odd, 0) != 3 || page_number(b, odd, 1) != -1 || page_number(b, odd, 2) != -1;
    b.cache_pages = 0;
    wrong += page_number(b, odd, 0) != -1;
    b.table_pages = 0;
    wrong += page_number(b, nullptr, 0) != -1;
    std::printf("%ld wrong\n", wrong);
    return wrong == 0 ? 0 : 1;
}
