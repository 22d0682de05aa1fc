// Which bytes a strided tensor occupies, and whether two of them, or two elements of one, share any.  Host only.
#ifndef TDE_OVERLAP_H
#define TDE_OVERLAP_H

#include <algorithm>
#include <cstdint>

namespace tde {

// Runs of `width` bytes at `at` plus any multiple below sizes[i] of strides[i] bytes; strides descend, sizes are 2 at least.
struct Region {
    static constexpr int kMostDims = 4;
    int64_t at = 0, width = 0, sizes[kMostDims], strides[kMostDims]; // width 0: no bytes
    int dims = 0;

    // Of `n` dimensions (kMostDims at most), strides in elements and not negative.
    Region(const void *data, int n, const int64_t *size, const int64_t *stride, int64_t element) : at((int64_t)(uintptr_t)data), width(element) {
        for (int i = 0; i < n; ++i) {
            if (size[i] == 0) width = 0;
            if (size[i] <= 1) continue;
            int to = dims++;
            for (; to > 0 && strides[to - 1] < stride[i] * element; --to) {
                sizes[to] = sizes[to - 1];
                strides[to] = strides[to - 1];
            }
            sizes[to] = size[i];
            strides[to] = stride[i] * element;
        }
        for (; width > 0 && dims > 0 && strides[dims - 1] == width; --dims) width *= sizes[dims - 1]; // neighbouring runs are one
    }
    // Bytes from the first one to behind the last, of the dimensions from `from` on.
    int64_t reach(int from = 0) const {
        int64_t r = width;
        for (int i = from; i < dims; ++i) r += (sizes[i] - 1) * strides[i];
        return r;
    }
};

// Whether elements share bytes.  Exact where every stride spans what lies inside it, as slices, permutations and expansions of contiguous
// tensors have it; other orders count as overlapping.
inline bool overlaps_itself(const Region &r) {
    if (r.width == 0) return false;
    for (int i = 0; i < r.dims; ++i)
        if (r.strides[i] < r.reach(i + 1)) return true;
    return false;
}

// Whether b's run of dimensions from j on, `offset` bytes behind a's from i on, meets it.
inline bool meet(const Region &a, int i, const Region &b, int j, int64_t offset) {
    if (offset >= a.reach(i) || -offset >= b.reach(j)) return false;
    const int64_t sa = i < a.dims ? a.strides[i] : 0, sb = j < b.dims ? b.strides[j] : 0, s = std::max(sa, sb);
    if (s == 0) return true;
    // The larger stride's dimension; the other region has it once, unless it has the same.  Within it, places repeat: of all pairs of indexes
    // only the two whose distance is nearest to the offset can meet.
    const int64_t na = sa == s ? a.sizes[i] : 1, nb = sb == s ? b.sizes[j] : 1;
    const int ia = sa == s ? i + 1 : i, jb = sb == s ? j + 1 : j;
    if (a.reach(ia) > s || b.reach(jb) > s) return true; // no such order: taken as meeting
    const int64_t steps = offset >= 0 ? offset / s : -((-offset + s - 1) / s); // floor
    for (const int64_t apart : {steps, steps + 1}) // index in a less index in b
        if (apart < na && -apart < nb && meet(a, ia, b, jb, offset - apart * s)) return true;
    return false;
}

// Whether the two share bytes.  Exact for regions whose strides are the same and span what lies inside them (heads or channels of one tensor,
// keys beside values); where their orders differ, interleaved regions count as sharing.
inline bool overlap(const Region &a, const Region &b) { return a.width != 0 && b.width != 0 && meet(a, 0, b, 0, b.at - a.at); }

} // namespace tde

#endif // TDE_OVERLAP_H
