/* paged_index.h — where a position of a sequence lies in the paged pool.  Plain functions, compiled for the card by the
 * kernels and for the host by the test that walks them over bad tables. */
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define SV_HD __host__ __device__ __forceinline__
#else
#define SV_HD inline
#endif

namespace sv {

/* The page that column `col` of a sequence's page-table row names, or -1: no such column, or no such page in the pool. */
SV_HD int32_t paged_page(const int32_t* row, uint32_t stride, uint32_t pool_pages, uint32_t col) {
    if (col >= stride) return -1;
    const int32_t page = row[col];
    return (page < 0 || (uint32_t)page >= pool_pages) ? -1 : page;
}

/* Division by a number that stays the same through a launch: a multiply and a shift, for numerators below 2^31. */
struct PagedDiv { uint32_t d, mul, shift; };
SV_HD PagedDiv paged_div(uint32_t d) {
    PagedDiv x;
    x.d = d; x.shift = 0;
    while (x.shift < 31u && (1u << x.shift) < d) ++x.shift;
    x.mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << x.shift) - d)) / d + 1u);
    return x;
}
SV_HD uint32_t paged_quot(uint32_t n, const PagedDiv& x) { return ((uint32_t)(((uint64_t)n * x.mul) >> 32) + n) >> x.shift; }

/* The number in the pool of block `block` of a sequence (a page holds per.d of them), or -1. */
SV_HD int32_t paged_block(const int32_t* row, uint32_t stride, uint32_t pool_pages, const PagedDiv& per, uint32_t block) {
    const uint32_t col = paged_quot(block, per);
    const int32_t page = paged_page(row, stride, pool_pages, col);
    return page < 0 ? -1 : (int32_t)((uint32_t)page * per.d + (block - col * per.d));
}

/* How a row at position p splits its n = p / B + 1 blocks: the first `lo` and those from `hi` on are always attended, and of
 * those between, when there are any, `take` are chosen by score. */
struct PagedChoice { uint32_t n, lo, hi, take, count; };
SV_HD PagedChoice paged_choice(uint32_t p, uint32_t block_pos, uint32_t first, uint32_t last, uint32_t top) {
    PagedChoice c;
    c.n = p / block_pos + 1u;
    if (c.n <= first + last + top) { c.lo = c.hi = c.n; c.take = 0u; c.count = c.n; }
    else { c.lo = first; c.hi = c.n - last; c.take = top; c.count = first + last + top; }
    return c;
}

}  // namespace sv
