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

// Whether rows lo .. hi - 1 lie within the call's `rows` and, where there are any, `length` positions within the `capacity` of the page table.
PAGED_HD bool paged_holds(int lo, int hi, int length, int rows, int capacity) { return 0 <= lo && lo <= hi && hi <= rows && (lo == hi || length <= capacity); }

// Where they are. A sequence that is not held has no rows: to move its positions to where there is room would put new keys over old ones.
PAGED_HD PagedSeq paged_place(int lo, int hi, int length, int rows, int capacity) {
    PagedSeq s;
    const bool held = paged_holds(lo, hi, length, rows, capacity);
    s.first = held ? lo : 0;
    s.n = held ? hi - lo : 0;
    s.length = length < 0 ? 0 : (length > capacity ? capacity : length);
    s.pos0 = s.length - s.n;
    return s;
}

} // namespace b200i
