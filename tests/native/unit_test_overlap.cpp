// Host check of csrc/tde_overlap.h against sets of bytes: random slices, permutations and expansions of small buffers.  What is said to be
// apart is apart; within one order of strides what is said to share does.  Exit status 0: everything right.
#include "tde_overlap.h"

#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

using tde::Region;

struct View {
    std::vector<int64_t> size, stride;
    int64_t at, element;
    Region region() const { return Region((const void *)(uintptr_t)at, (int)size.size(), size.data(), stride.data(), element); }
    // bytes, and whether one is taken twice
    std::set<int64_t> bytes(bool *twice) const {
        std::set<int64_t> all;
        std::vector<int64_t> index(size.size(), 0);
        *twice = false;
        for (int64_t n : size)
            if (n == 0) return all;
        for (;;) {
            int64_t p = at;
            for (size_t i = 0; i < size.size(); ++i) p += index[i] * stride[i] * element;
            for (int64_t b = 0; b < element; ++b) *twice |= !all.insert(p + b).second;
            size_t i = 0;
            while (i < size.size() && ++index[i] == size[i]) index[i++] = 0;
            if (i == size.size()) return all;
        }
    }
};

static int below(int n) { return std::rand() % n; }

// A slice of a contiguous tensor of the given sizes, its dimensions in any order.
static View slice(const std::vector<int64_t> &whole, int64_t base, int64_t element, bool permute, bool expand) {
    View v;
    v.at = base;
    v.element = element;
    int64_t stride = 1;
    for (size_t i = whole.size(); i-- > 0;) {
        const int64_t from = below((int)whole[i]), n = 1 + below((int)(whole[i] - from));
        v.at += from * stride * element;
        v.size.push_back(n);
        v.stride.push_back(n == 1 && below(2) ? below(100) : stride); // a single element's stride may be anything
        stride *= whole[i];
    }
    if (expand && below(3) == 0) {
        const int i = below((int)v.size.size());
        v.size[i] = 1 + below(3);
        v.stride[i] = 0;
    }
    for (size_t i = v.size.size(); permute && i > 1; --i) {
        const int j = below((int)i);
        std::swap(v.size[i - 1], v.size[j]);
        std::swap(v.stride[i - 1], v.stride[j]);
    }
    if (below(60) == 0) v.size[0] = 0;
    return v;
}

int main() {
    std::srand(1);
    long wrong = 0, shared = 0, apart = 0;
    for (int round = 0; round < 200000; ++round) {
        std::vector<int64_t> whole;
        for (int i = 0, n = 1 + below(4); i < n; ++i) whole.push_back(1 + below(4));
        const int64_t element = 1 << below(3);
        const bool permute = below(2);
        const View a = slice(whole, 1000, element, permute, false), b = slice(whole, 1000, element, permute, false);
        bool a_twice, b_twice;
        const auto in_a = a.bytes(&a_twice), in_b = b.bytes(&b_twice);
        bool common = false;
        for (int64_t x : in_a) common |= in_b.count(x) != 0;
        wrong += a_twice || tde::overlaps_itself(a.region());
        wrong += tde::overlap(a.region(), b.region()) != common || tde::overlap(b.region(), a.region()) != common;
        (common ? shared : apart) += 1;
        // another tensor's slice in the same memory, with an element of its own: nothing that shares may be missed
        std::vector<int64_t> other;
        for (int i = 0, n = 1 + below(4); i < n; ++i) other.push_back(1 + below(4));
        const View c = slice(other, 990 + below(60), 1 << below(3), true, true);
        bool c_twice;
        const auto in_c = c.bytes(&c_twice);
        common = false;
        for (int64_t x : in_a) common |= in_c.count(x) != 0;
        wrong += common && !(tde::overlap(a.region(), c.region()) && tde::overlap(c.region(), a.region()));
        wrong += c_twice != tde::overlaps_itself(c.region());
    }
    std::printf("%ld wrong, %ld pairs that share and %ld that do not\n", wrong, shared, apart);
    return wrong == 0 && shared > 1000 && apart > 1000 ? 0 : 1;
}
