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

/* The first pool position of block `block` of a sequence (`block_pos` positions, a divisor of a page's), or -1. */
SV_HD int32_t paged_block_slot(const int32_t* row, uint32_t stride, uint32_t pool_pages, uint32_t page_pos, uint32_t block_pos, uint32_t block) {
    const uint32_t per = page_pos / block_pos, col = block / per;
    const int32_t page = paged_page(row, stride, pool_pages, col);
    return page < 0 ? -1 : (int32_t)((uint32_t)page * page_pos + (block - col * per) * block_pos);
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
