// Where a sequence's rows and positions lie, from what a call's tables say of it. Plain arithmetic, so that the host can run it too.
#pragma once
#ifdef __CUDACC__
#define PAGED_HD __host__ __device__ __forceinline__
#else
#define PAGED_HD inline
#endif

namespace b200i {

// One sequence's part of a call.
struct PagedSeq {
    int first, n;  // its rows
    int length;    // positions in its cache, the new ones among them
    int pos0;      // position of its first row (negative where a table says that fewer are cached than are new)
};

// Rows lo .. hi - 1 of `rows` in all and `length` positions, of `capacity` that the page table has room for. Whatever the tables say, the rows lie
// within the call's and the length within the capacity.
PAGED_HD PagedSeq paged_place(int lo, int hi, int length, int rows, int capacity) {
    PagedSeq s;
    s.first = lo < 0 ? 0 : (lo > rows ? rows : lo);
    hi = hi < rows ? hi : rows;
    s.n = hi > s.first ? hi - s.first : 0; // compared first: a difference of any two words leaves 32 bits
    s.length = length < 0 ? 0 : (length > capacity ? capacity : length);
    s.pos0 = s.length - s.n;
    return s;
}

} // namespace b200i
