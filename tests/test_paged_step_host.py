"""The paged step's operators without a GPU: what their entry points refuse before anything is enqueued, and the page
arithmetic walked over bad tables."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import paged_reference as ref
from silvann_b200 import ext

CSRC = Path(__file__).resolve().parents[1] / "silvann_b200" / "csrc"
A = 1 << 20        # an address nothing is read from: every call here is refused on the host


def refused(fn, args, **change):
    args = {**args, **change}
    with pytest.raises(ext.B200Error) as e:
        fn(**args)
    assert e.value.code == ext.E_ARGUMENT
    return str(e.value)


TABLES = dict(new_lens=A, page_table=A, row_start=A, row_seq=A, row_pos=A, row_slot=A, free_out=A, free_pages=A, free_at=A, lens=A, counts=A, seqs=4, table_stride=8, rows=16,
              free_total=64, pool_pages=64, page_positions=64)
WRITE = dict(k_pool=A, v_pool=A, k_means=A, k_rows=A, v_rows=A, row_slot=A, rows=4, kv_heads=2, head_dim=128, pool_pages=64, page_positions=64, block_positions=64)
SPARSE = dict(o=A, res=None, chosen=A, q=A, k_pool=A, v_pool=A, k_means=A, row_seq=A, row_pos=A, rows=4, page_table=A, seqs=4, table_stride=8, pool_pages=64, page_positions=64,
              block_positions=64, q_heads=16, kv_heads=2, head_dim=128, first=1, last=2, top=13)


@pytest.mark.parametrize("change", [
    *[{k: None} for k in list(TABLES)[:11]], {"lens": A + 2}, {"seqs": 0}, {"seqs": 8193}, {"table_stride": 0}, {"rows": 0}, {"rows": 1 << 31}, {"free_total": 0},
    {"pool_pages": 0}, {"page_positions": 0}, {"pool_pages": 1 << 25}, {"pool_pages": 1 << 40}])
def test_tables_refuses(change):
    assert "paged_tables" in refused(ext.paged_tables, TABLES, **change)


@pytest.mark.parametrize("change", [
    {"k_pool": None}, {"v_pool": None}, {"k_means": None}, {"k_rows": None}, {"v_rows": None}, {"row_slot": None}, {"dtype": 2}, {"rows": 0}, {"kv_heads": 0}, {"head_dim": 0},
    {"kv_heads": 1, "head_dim": 12}, {"k_stride": 128}, {"v_stride": 260}, {"pool_pages": 0}, {"pool_pages": 1 << 26}, {"block_positions": 48}, {"block_positions": 128},
    {"block_positions": 8}, {"k_pool": A + 8}, {"v_rows": A + 2}, {"k_means": A + 4}, {"row_slot": A + 2}])
def test_write_refuses(change):
    assert "paged_write" in refused(ext.paged_write, WRITE, **change)


@pytest.mark.parametrize("change", [
    {"o": None}, {"q": None}, {"k_pool": None}, {"v_pool": None}, {"k_means": None}, {"row_seq": None}, {"row_pos": None}, {"page_table": None}, {"dtype": -1}, {"head_dim": 96},
    {"head_dim": 512}, {"kv_heads": 0}, {"q_heads": 0}, {"q_heads": 15}, {"q_heads": 130}, {"rows": 0}, {"seqs": 0}, {"table_stride": 0}, {"pool_pages": 0}, {"pool_pages": 1 << 26},
    {"block_positions": 0}, {"block_positions": 48}, {"block_positions": 128}, {"last": 0}, {"first": 1000, "top": 23}, {"top": 0xFFFFFFFF}, {"first": 0xFFFFFFFF, "top": 0xFFFFFFFF},
    {"q_stride": 16 * 128 - 8}, {"q_stride": 16 * 128 + 4}, {"q": A + 8}, {"k_pool": A + 8}, {"v_pool": A + 2}, {"k_means": A + 8}, {"res": A + 2}, {"page_table": A + 1},
    {"o": A + 1}, {"rows": (1 << 23) + 1}, {"kv_heads": 8192, "q_heads": 8192}, {"chosen": A + 2}, {"row_pos": A + 1}])
def test_sparse_refuses(change):
    assert "paged_sparse" in refused(ext.paged_sparse, SPARSE, **change)


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_no_table_entry_becomes_an_address_outside_the_pool(tmp_path):
    """Every block of every row of a table of good, missing and stale entries: the kernels' own page arithmetic answers a
    place whose whole block lies in the pool, or -1."""
    src = tmp_path / "walk.cpp"
    src.write_text(r"""
#include "paged_index.h"
#include <cstdio>
#include <climits>
#include <initializer_list>
int main() {
    const int32_t entries[] = {0, 6, 3, -1, 7, INT_MIN, INT_MAX, 100, 1};
    for (uint32_t B : {16u, 32u, 64u, 128u})
        for (uint32_t per : {1u, 2u, 3u, 5u}) {
            const uint32_t P = B * per, pool = 7;
            for (uint32_t stride : {1u, 4u, 9u})
                for (uint32_t b = 0; b < 60; ++b) {
                    const int32_t at = sv::paged_block(entries, stride, pool, sv::paged_div(per), b);
                    const long got = at < 0 ? -1 : (long)at * B;
                    const uint32_t col = b * B / P;
                    const bool good = col < stride && entries[col] >= 0 && entries[col] < (int32_t)pool;
                    const long want = good ? (long)entries[col] * P + (long)b * B % P : -1;
                    if (got != want || (got >= 0 && got + B > pool * P)) { printf("B %u P %u stride %u block %u: %ld, not %ld\n", B, P, stride, b, got, want); return 1; }
                }
        }
    // a block far along a long table, where the column alone needs 27 bits, and the last block of the largest pool
    if (sv::paged_block(entries, 4, 7, sv::paged_div(1), 0x7FFFFFFFu / 16) != -1) return 2;
    const int32_t last[] = {(1 << 27) - 2};
    if (sv::paged_block(last, 1, (1u << 27) - 1, sv::paged_div(1), 0) != (1 << 27) - 2) return 3;
    for (uint32_t d : {1u, 2u, 3u, 5u, 7u, 48u, 64u, 641u, 65535u, 65536u, 1000003u, 0x3FFFFFFFu, 0x40000000u, 0x40000001u, 0x7FFFFFFFu}) {
        const sv::PagedDiv x = sv::paged_div(d);
        for (uint64_t k = 0; k < 4000; ++k)
            for (int64_t j = -2; j <= 2; ++j) {
                const int64_t n = (k < 2000 ? (int64_t)(k * d) : (int64_t)(0x7FFFFFFF - (k - 2000) * 1000003)) + j;
                if (n >= 0 && n <= 0x7FFFFFFF && sv::paged_quot((uint32_t)n, x) != (uint32_t)n / d) { printf("%ld / %u\n", (long)n, d); return 6; }
            }
    }
    for (uint32_t p = 0; p < 3000; ++p)
        for (uint32_t B : {16u, 64u, 128u})
            for (uint32_t first : {0u, 1u, 3u}) for (uint32_t last_ : {1u, 2u}) for (uint32_t top : {0u, 1u, 7u}) {
                const sv::PagedChoice c = sv::paged_choice(p, B, first, last_, top);
                const uint32_t n = p / B + 1, keep = first + last_ + top;
                if (c.n != n || c.count != (n < keep ? n : keep) || c.lo + c.take + (c.n - c.hi) != c.count) return 4;
                if (c.take && !(c.hi - c.lo > c.take)) return 5;
            }
    return 0;
}
""")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined,address", "-I", str(CSRC), str(src), "-o", str(tmp_path / "walk")], check=True)
    r = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-2000:])


def test_the_reference_of_the_tables():
    """A step by hand: sequence 0 grows across a page, 1 ends, 2 is new and takes what 1 gave back."""
    t = ref.tables([3, 5, 0, 4], [2, -1, 6, 0], [[9, -1], [4, 7], [-1, -1], [2, -1]], [0, 0, 0, 1, 3, 5], 3, 10, 10, 4)
    assert t["status"] == 0 and t["free_at"] == 4 and list(t["free"]) == [0, 4, 7, 1, 3, 5]
    assert t["new_lens"].tolist() == [5, 0, 6, 4] and t["row_start"].tolist() == [0, 2, 2, 8, 8]
    assert t["table"].tolist() == [[9, 4], [4, 7], [7, 1], [2, -1]]
    assert t["slot"].tolist() == [39, 16, 28, 29, 30, 31, 4, 5, -1, -1]
    full = ref.tables([4], [1], [[0, 1]], [0, 1], 2, 4, 2, 4)
    assert full["status"] == ref.NO_PAGES and full["slot"].tolist() == [-1] * 4 and full["new_lens"].tolist() == [4]


def test_the_reference_of_the_choice():
    q, means = np.ones((2, 4)), np.array([[0.0], [5], [1], [5], [np.nan], [7], [0], [0]]) * np.ones((8, 4))
    k = v = np.ones((8 * 16, 4))
    pick = lambda p, first, last, top: ref.sparse_row(q, k, v, means, [0, 1, 2, 3, 4, 5, 6, 7], p, 16, 16, first, last, top)[0]
    assert pick(127, 1, 1, 2) == [0, 1, 5, 7] and pick(127, 0, 1, 3) == [1, 3, 5, 7] and pick(127, 0, 2, 0) == [6, 7] and pick(40, 2, 1, 9) == [0, 1, 2]
    assert pick(127, 0, 1, 6) == [0, 1, 2, 3, 5, 6, 7]
