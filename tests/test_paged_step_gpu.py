"""The paged step's operators on a B200 — a step's tables, rows into the pool with the blocks' mean keys, attention over
selected blocks — against their definitions in plain Python and 64 bits (tests/paged_reference.py).

Tolerances, from arithmetic.  Tables, slots, copied rows and chosen blocks: equal.  A block's mean: half a step of the type
plus the fp32 sum's error, (B + 1) roundings of at most 2^-24 of the mean magnitude.  Attention: a score is a sum of d
products in fp32, off by at most (d + 3) 2^-24 of the sum of their magnitudes |s|, and takes a factor exp with it, so a weight is
off by (1 + e)^2 with e that error (its own maximum moves as well); weights are kept to 2^-16 or better, exp to 2^-21, and n of them are
summed in fp32: together an output is off by at most ((2 (d + 3) 2^-24 |s| + 2^-16 + 2^-20 + n 2^-24) max|v|), twice over for
numerator and normaliser, and half a step of the type."""
import numpy as np
import pytest

import oracle
import paged_reference as ref
from oracle import from_bits, to_bits
from silvann_b200 import ext
from util import dev, host_bits

pytestmark = pytest.mark.gpu

STEP = {0: 2.0 ** -11, 1: 2.0 ** -8}          # half a step of the type, relative
FLOOR = {0: 2.0 ** -25, 1: 2.0 ** -133}       # half a step below the smallest normal


def i32(cuda, *shape, fill=-77):
    return cuda.full(shape, fill, dtype=cuda.int32, device="cuda")


def random_tables(rng, lens, page, extra, stride=None):
    """(table [seqs][stride], order, used): distinct pages for what is held, the rest of `order` free."""
    held = [-(-int(n) // page) for n in lens]
    stride = stride or max(1, max(held)) + 3
    pool = sum(held) + extra
    order = rng.permutation(pool).astype(np.int32)
    table, at = np.full((len(lens), stride), -1, np.int32), 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    return table, order, at


# ---------------------------------------------------------------------------------------------------------------------
# the step's tables


def run_tables(cuda, lens, counts, table, free, free_at, rows, pool_pages, page, in_place=False):
    L, C, T, F = dev(cuda, np.array(lens, np.int32)), dev(cuda, np.array(counts, np.int32)), dev(cuda, np.array(table, np.int32)), dev(cuda, np.array(free, np.int32))
    at = i32(cuda, 1, fill=int(free_at))
    new, out = (L, at) if in_place else (i32(cuda, len(lens)), i32(cuda, 1))
    start, seq, pos, slot = i32(cuda, len(lens) + 1), i32(cuda, rows + 5), i32(cuda, rows + 5), i32(cuda, rows + 5)
    ext.paged_tables(new, T, start, seq, pos, slot, out, F, at, L, C, len(lens), T.shape[1], rows, F.numel(), pool_pages, page)
    cuda.cuda.synchronize()
    for x in (seq, pos, slot):
        assert (x[rows:] == -77).all()
    n = lambda t: t.cpu().numpy()
    return dict(new_lens=n(new), table=n(T), row_start=n(start), seq=n(seq)[:rows], pos=n(pos)[:rows], slot=n(slot)[:rows], free_at=int(out), free=n(F), status=ext.device_status())


def same(got, want):
    for k in want:
        assert np.array_equal(got[k], want[k]), (k, got[k], want[k])


@pytest.mark.parametrize("seqs,page,lo,hi,c_hi,ended,pad", [
    (1, 64, 0, 0, 1, 0, 0), (1, 16, 15, 15, 1, 0, 3), (1, 256, 255, 255, 70000, 0, 0), (3, 1, 0, 9, 4, 2, 5), (32, 256, 0, 3000, 1, 0, 0), (33, 48, 0, 500, 97, 4, 100),
    (1024, 64, 0, 200, 3, 7, 11), (1025, 64, 0, 200, 3, 3, 11), (8192, 16, 0, 64, 2, 5, 1), (500, 128, 0, 1, 0, 3, 1), (2, 16, 20000, 30000, 40000, 0, 9)])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables(cuda, seqs, page, lo, hi, c_hi, ended, pad, in_place):
    rng = np.random.default_rng(seqs * 1000 + page)
    lens, counts = rng.integers(lo, hi + 1, seqs), rng.integers(0, c_hi + 1, seqs)
    if c_hi == 1:
        counts[:] = 1
    if ended:
        counts[rng.integers(0, seqs, max(1, seqs // ended))] = -1
    rows = int(counts[counts > 0].sum()) + pad
    extra = int(sum(-(-(a + max(b, 0)) // page) for a, b in zip(lens, counts)))
    table, free, used = random_tables(rng, lens, page, extra, -(-int(max(lens + np.maximum(counts, 0))) // page) + 1)
    want = ref.tables(lens, counts, table, free, used, max(1, rows), len(free), page)
    assert want["status"] == 0
    same(run_tables(cuda, lens, counts, table, free, used, max(1, rows), len(free), page, in_place), want)


def test_tables_takes_the_last_free_page_and_no_more(cuda):
    rng = np.random.default_rng(4)
    lens, counts = [30, 64, 10], [3, 1, -1]
    table, free, used = random_tables(rng, lens, 16, 0, 6)           # nothing free: what sequence 2 gives back is all there is
    want = ref.tables(lens, counts, table, free, used, 8, len(free), 16)
    assert want["status"] == ref.NO_PAGES                            # two pages are needed (33 and 65 positions)
    same(run_tables(cuda, lens, counts, table, free, used, 8, len(free), 16), want)
    counts = [2, 1, -1]
    want = ref.tables(lens, counts, table, free, used, 8, len(free), 16)
    assert want["status"] == 0 and want["free_at"] == len(free)
    same(run_tables(cuda, lens, counts, table, free, used, 8, len(free), 16), want)


@pytest.mark.parametrize("what", ["rows", "long", "negative", "count", "stack", "beyond", "huge"])
@pytest.mark.parametrize("in_place", [False, True])
def test_a_step_that_does_not_fit_changes_nothing(cuda, what, in_place):
    rng = np.random.default_rng(5)
    lens, counts, rows, page = np.array([30, 64, 10, 0]), np.array([3, 1, -1, 20]), 24, 16
    table, free, used = random_tables(rng, lens, page, 9, 6)
    at = used
    if what == "rows": rows = 23
    if what == "long": counts[1], rows = 33, 100                     # 97 positions in six columns of 16
    if what == "negative": lens[2] = -1
    if what == "count": counts[0] = -2
    if what == "stack": at = 0                                       # a page comes back and there is no room below
    if what == "beyond": at = len(free) + 1
    if what == "huge": counts[:] = [2 ** 31 - 1] * 4
    want = ref.tables(lens, counts, table, free, at, rows, len(free), page)
    assert want["status"] == ref.BAD_STEP
    same(run_tables(cuda, lens, counts, table, free, at, rows, len(free), page, in_place), want)


def test_entries_that_name_no_page_give_no_slot(cuda):
    rng = np.random.default_rng(6)
    lens, counts = [30, 17, 40], [5, 40, -1]
    table, free, used = random_tables(rng, lens, 16, 5, 6)
    for bad in (-1, len(free), 2 ** 31 - 1, -2 ** 31):
        t, f = table.copy(), free.copy()
        t[0, 1], t[2, 0], f[used + 1] = bad, bad, bad                # a page held, one that comes back, a free one
        want = ref.tables(lens, counts, t, f, used, 50, len(free), 16)
        assert want["status"] == ref.BAD_PAGE and (want["slot"][:45] == -1).any()
        same(run_tables(cuda, lens, counts, t, f, used, 50, len(free), 16), want)


def test_tables_captured_and_replayed(cuda):
    """One captured step, replayed with other counts: lengths, table and stack live on the card and move on in place."""
    rng = np.random.default_rng(7)
    page, seqs, rows = 16, 6, 64
    lens = rng.integers(0, 40, seqs)
    table, free, used = random_tables(rng, lens, page, 60, 12)
    ext.device_status()
    L, C, T, F, at = dev(cuda, lens.astype(np.int32)), i32(cuda, seqs, fill=0), dev(cuda, table), dev(cuda, free), i32(cuda, 1, fill=used)
    start, seq, pos, slot = i32(cuda, seqs + 1), i32(cuda, rows), i32(cuda, rows), i32(cuda, rows)
    call = lambda: ext.paged_tables(L, T, start, seq, pos, slot, at, F, at, L, C, seqs, 12, rows, F.numel(), len(free), page, stream=cuda.cuda.current_stream().cuda_stream)
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.stream(side):
        call()                                                       # counts are 0: nothing moves
    cuda.cuda.current_stream().wait_stream(side)
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        call()
    lens, at_h = lens.tolist(), used
    for step in range(12):
        counts = rng.integers(0, 9, seqs)
        if step % 3 == 2:
            counts[step % seqs] = -1
        C.copy_(dev(cuda, counts.astype(np.int32)))
        graph.replay()
        cuda.cuda.synchronize()
        want = ref.tables(lens, counts, table, free, at_h, rows, len(free), page)
        n = lambda t: t.cpu().numpy()
        same(dict(new_lens=n(L), table=n(T), row_start=n(start), seq=n(seq), pos=n(pos), slot=n(slot), free_at=int(at), free=n(F), status=ext.device_status()), want)
        lens, table, free, at_h = want["new_lens"].tolist(), want["table"], want["free"], want["free_at"]
    assert want["status"] == 0


# ---------------------------------------------------------------------------------------------------------------------
# rows into the pool


def bits(rng, shape, dtype, scale=1.0):
    return to_bits((rng.standard_normal(shape) * scale).astype(np.float32), dtype)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("kvh,d,page,block,gap", [(2, 256, 256, 64, 0), (4, 128, 64, 16, 24), (1, 64, 128, 128, 8), (8, 128, 96, 32, 0), (1, 8, 16, 16, 0), (3, 72, 48, 16, 0), (2, 64, 64, 0, 0), (16, 256, 64, 64, 0)])
def test_write(cuda, dtype, kvh, d, page, block, gap):
    rng = np.random.default_rng(kvh * d + page)
    lens, counts = np.array([0, 1, 15, 63, 64, 200, 7, 31]), np.array([1, 300, 1, 1, 64, 56, 0, 97])
    table, order, _ = random_tables(rng, lens + counts, page, 2)
    pool, row = len(order), kvh * d
    k, v, means = bits(rng, (pool * page, row), dtype), bits(rng, (pool * page, row), dtype), bits(rng, (pool * page // max(block, 1), row), dtype)
    slots = [int(table[s, p // page]) * page + p % page for s in range(len(lens)) for p in range(lens[s], lens[s] + counts[s])] + [-1, -9, -2 ** 31]
    rows = len(slots)
    wide = bits(rng, (rows, 2 * row + gap), dtype)
    tk, tv, tm, tw = dev(cuda, k), dev(cuda, v), dev(cuda, means), dev(cuda, wide)
    ext.paged_write(tk, tv, tm if block else None, tw.data_ptr(), tw.data_ptr() + 2 * row, dev(cuda, np.array(slots, np.int32)), rows, kvh, d, pool, page, block, 2 * row + gap, 2 * row + gap, dtype)
    cuda.cuda.synchronize()
    assert ext.device_status() == 0
    done = []
    for r, s in enumerate(slots):
        if s >= 0:
            k[s], v[s] = wide[r, :row], wide[r, row:2 * row]
            if block and s % block == block - 1:
                done.append(s // block)
    assert np.array_equal(host_bits(tk), k) and np.array_equal(host_bits(tv), v)
    got = host_bits(tm)
    if not block:
        assert np.array_equal(got, means)
        return
    assert len(done) >= 3
    rest = np.ones(len(means), bool)
    rest[done] = False
    assert np.array_equal(got[rest], means[rest])
    vals = from_bits(k, dtype).astype(np.float64).reshape(-1, block, row)[done]
    want, size = vals.mean(1), np.abs(vals).mean(1)
    bound = np.maximum(np.abs(want) * STEP[dtype], FLOOR[dtype]) * 1.01 + (block + 1) * 2.0 ** -24 * size
    assert (np.abs(from_bits(got[done], dtype) - want) <= bound).all()


def test_write_a_position_at_a_time_leaves_the_same_means(cuda):
    """Rows that come one a step, all in one call or in ragged pieces: the same pool and the same means, bit for bit."""
    rng = np.random.default_rng(11)
    kvh, d, page, block, n = 2, 128, 64, 32, 150
    rows_k, rows_v = dev(cuda, bits(rng, (n, kvh * d), 1)), dev(cuda, bits(rng, (n, kvh * d), 1))
    slots = np.concatenate([np.array([2, 0, 1])[np.arange(n) // page] * page + np.arange(n) % page]).astype(np.int32)
    ts, outs = dev(cuda, slots), []
    for pieces in ([n], [1] * n, [40, 1, 7, 70, 32]):
        k, v, m = (cuda.zeros((x, kvh * d), dtype=cuda.int16, device="cuda") for x in (3 * page, 3 * page, 3 * page // block))
        at = 0
        for c in pieces:
            ext.paged_write(k, v, m, rows_k[at:], rows_v[at:], ts[at:].clone(), c, kvh, d, 3, page, block, dtype=1)
            at += c
        cuda.cuda.synchronize()
        outs.append([host_bits(x) for x in (k, v, m)])
    for o in outs[1:]:
        for a, b in zip(outs[0], o):
            assert np.array_equal(a, b)
    assert ext.device_status() == 0


def test_write_skips_a_slot_past_the_pool(cuda):
    rng = np.random.default_rng(12)
    k = cuda.zeros((4 * 16 + 16, 64), dtype=cuda.int16, device="cuda")
    v, m = cuda.zeros_like(k), cuda.zeros((5, 64), dtype=cuda.int16, device="cuda")
    rows = dev(cuda, bits(rng, (3, 64), 0))
    ext.paged_write(k, v, m, rows, rows, dev(cuda, np.array([4 * 16 + 15, 5, 2 ** 31 - 1], np.int32)), 3, 1, 64, 4, 16, 16)
    cuda.cuda.synchronize()
    assert ext.device_status() == ref.BAD_PAGE and ext.device_status() == 0
    assert cuda.equal(k[5], rows[1].view(cuda.int16)) and int((k != 0).any(1).sum()) == 1 and int((m != 0).sum()) == 0


# ---------------------------------------------------------------------------------------------------------------------
# attention over selected blocks


class Paged:
    """A pool with sequences in it: keys and values in 16 bits (NaN wherever no sequence has a position), means, a table."""

    def __init__(self, cuda, seed, lens, kvh, d, dtype, page, block, scale=1.0, stride=None):
        rng = np.random.default_rng(seed)
        self.rng, self.lens, self.kvh, self.d, self.dtype, self.page, self.block, self.cuda = rng, lens, kvh, d, dtype, page, block, cuda
        self.table, order, _ = random_tables(rng, lens, page, 2, stride)
        self.pool = len(order)
        nan = 0x7E01 if dtype == 0 else 0x7FC1
        self.k = np.full((self.pool * page, kvh, d), nan, np.uint16)
        self.v = self.k.copy()
        self.means = np.full((self.pool * page // block, kvh, d), nan, np.uint16)
        for s, n in enumerate(lens):
            p = np.arange(n)
            at = self.table[s, p // page] * page + p % page
            x = rng.standard_normal((n, kvh, d)) + 0.5 * np.repeat(rng.standard_normal((n // block + 1, kvh, d)), block, 0)[:n]
            self.k[at], self.v[at] = to_bits((x * scale).astype(np.float32), dtype), bits(rng, (n, kvh, d), dtype)
            whole = n // block
            if whole:
                m = from_bits(self.k[at[:whole * block]], dtype).reshape(whole, block, kvh, d).mean(1)
                self.means[at[:whole * block:block] // block] = to_bits(m.astype(np.float32), dtype)

    def run(self, seq, pos, q_heads, first, last, top, q=None, gap=0, want_o=True, want_res=True, table=None, stream=None, means=True):
        cuda, rows, d = self.cuda, len(seq), self.d
        self.last_q = wide = bits(self.rng, (rows, q_heads * d + gap), self.dtype) if q is None else q
        keep = first + last + top
        o = cuda.full((rows, q_heads, d), 0x1234, dtype=cuda.int16, device="cuda") if want_o else None
        res = cuda.full((rows, q_heads, d + 2), 77.0, device="cuda") if want_res else None
        chosen = i32(cuda, rows, self.kvh, keep)
        t = dev(cuda, self.table if table is None else table)
        hold = [dev(cuda, x) for x in (wide, self.k, self.v, self.means, np.array(seq, np.int32), np.array(pos, np.int32))]
        if stream is not None:
            stream.wait_stream(cuda.cuda.current_stream())
        ext.paged_sparse(o, res, chosen, hold[0], hold[1], hold[2], hold[3] if means else None, hold[4], hold[5], rows, t, t.shape[0], t.shape[1], self.pool, self.page, self.block,
                         q_heads, self.kvh, d, first, last, top, q_stride=wide.shape[1] if gap else 0, dtype=self.dtype, stream=stream.cuda_stream if stream is not None else None)
        cuda.cuda.synchronize()
        q = wide[:, :q_heads * d].reshape(rows, q_heads, d)
        return q, host_bits(o) if want_o else None, res.cpu().numpy() if want_res else None, chosen.cpu().numpy()

    def check(self, seq, pos, q_heads, first, last, top, got, table=None):
        q, o, res, chosen = got
        f = lambda x: from_bits(x, self.dtype).astype(np.float64)
        group = q_heads // self.kvh
        table = self.table if table is None else table
        k, v, means = f(self.k), f(self.v), f(self.means)
        for r, (s, p) in enumerate(zip(seq, pos)):
            if s < 0 or s >= len(table):
                assert o is None or (o[r] == 0x1234).all()
                assert res is None or (res[r] == 77.0).all()
                assert (chosen[r] == -77).all()
                continue
            if p < 0:
                assert o is None or (o[r] == 0).all()
                assert res is None or (np.isneginf(res[r, :, 0]).all() and (res[r, :, 1:] == 0).all())
                assert (chosen[r] == -1).all()
                continue
            row = np.where((table[s] >= 0) & (table[s] < self.pool), table[s], -1)
            row = np.concatenate([row, np.full(max(0, p // self.page + 1 - len(row)), -1, row.dtype)])
            for g in range(self.kvh):
                hs = slice(g * group, (g + 1) * group)
                ids, want, m, l, size, vmax = ref.sparse_row(f(q[r, hs]), k[:, g], v[:, g], means[:, g], row, p, self.page, self.block, first, last, top)
                assert chosen[r, g].tolist() == ids + [-1] * (first + last + top - len(ids)), (r, g)
                n = len(ids) * self.block
                fp = (2 * (2 * (self.d + 3) * 2.0 ** -24 * size + 2.0 ** -16 + 2.0 ** -20 + n * 2.0 ** -24) * vmax)[:, None]
                if o is not None:
                    err = np.abs(f(o[r, hs]) - want)
                    bound = fp + np.maximum(np.abs(want) + fp, 0) * STEP[self.dtype] + FLOOR[self.dtype]
                    assert (err <= bound).all(), (r, g, p, float((err - bound).max()))
                if res is not None:
                    assert (np.abs(res[r, hs, 2:] / res[r, hs, 1:2] - want) <= fp).all(), (r, g, p)
                    # (m, l) as a merge uses them: the logarithm of the whole sum
                    lse = res[r, hs, 0].astype(np.float64) + np.log(res[r, hs, 1].astype(np.float64))
                    assert (np.abs(lse - (m + np.log(l))) <= 2.0 ** -22 * (np.abs(m) + 1) + fp[:, 0] / max(vmax, 1e-9) + 1e-6).all(), (r, g, p)


LENS = [1, 15, 16, 17, 63, 64, 65, 700, 1500]


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("d,kvh,group,page,block,keep", [
    (64, 2, 1, 16, 16, (1, 2, 5)), (64, 1, 16, 64, 32, (0, 1, 3)), (128, 4, 4, 64, 64, (1, 2, 4)), (128, 2, 8, 256, 64, (0, 1, 0)), (128, 1, 12, 128, 128, (1, 1, 2)),
    (256, 2, 8, 256, 64, (2, 3, 6)), (256, 1, 16, 48, 16, (3, 1, 40)), (128, 1, 5, 96, 32, (1, 4, 200)), (64, 1, 64, 128, 64, (1, 1, 5)), (256, 1, 24, 64, 64, (0, 2, 3)),
    (128, 8, 1, 32, 32, (7, 1, 1))])
def test_sparse(cuda, dtype, d, kvh, group, page, block, keep):
    P = Paged(cuda, d + group + page, LENS, kvh, d, dtype, page, block)
    seq, pos = list(range(len(LENS))) + [8, 8, 7], [n - 1 for n in LENS] + [1499 - 600, 1040, 255]
    got = P.run(seq, pos, kvh * group, *keep, gap=8 if group == 5 else 0)
    assert ext.device_status() == 0
    P.check(seq, pos, kvh * group, *keep, got)


@pytest.mark.parametrize("d,block,lens,top", [(64, 16, [70000], 61), (64, 16, [40001, 33000], 900), (128, 64, [66000], 8), (256, 128, [20000, 1], 20)])
def test_sparse_over_long_sequences(cuda, d, block, lens, top):
    """More candidates than are looked at in one go, and choices of almost all and of few of them."""
    P = Paged(cuda, block, lens, 1, d, 1, 2 * block, block)
    seq, pos = list(range(len(lens))), [n - 1 for n in lens]
    got = P.run(seq, pos, 4, 1, 2, top)
    assert ext.device_status() == 0
    P.check(seq, pos, 4, 1, 2, top, got)


def test_sparse_drafted_positions_and_padding(cuda):
    """Several rows a sequence at their own positions, padded rows and rows before any position, in no order."""
    P = Paged(cuda, 21, [40, 333, 900], 2, 128, 1, 64, 16)
    seq = [2, 2, -1, 1, 2, 0, 1, -5, 1, 0, 3, 2 ** 31 - 1]
    pos = [899, 896, 3, 332, 0, 39, -1, -1, 331, -2 ** 31, 5, 5]
    got = P.run(seq, pos, 16, 1, 2, 6)
    assert ext.device_status() == ref.BAD_PAGE            # rows 10 and 11 name no sequence
    P.check(seq, pos, 16, 1, 2, 6, got)
    got = P.run(seq[:10], pos[:10], 16, 1, 2, 6, want_res=False)
    assert ext.device_status() == 0
    P.check(seq[:10], pos[:10], 16, 1, 2, 6, got)
    got = P.run(seq[:10], pos[:10], 16, 1, 2, 6, want_o=False)
    P.check(seq[:10], pos[:10], 16, 1, 2, 6, got)


def test_sparse_ties_nan_and_infinite_means(cuda):
    """Equal scores go to the lower block, NaN and minus infinity rank last together, +inf first; zeros of both signs are equal."""
    B = 16
    P = Paged(cuda, 22, [B * 300, B * 300, B * 300], 1, 64, 0, B, B)
    at = lambda s, b: int(P.table[s, b])                 # pages of one block: the mean's number is the page's
    one = to_bits(np.ones(64, np.float32), 0)
    for b in range(299):
        P.means[at(0, b), 0] = 0x8000 if b % 2 else 0    # every score is a zero
        P.means[at(1, b), 0] = to_bits(np.full(64, (b * 7919) % 5, np.float32), 0)      # five values, sixty blocks each
        P.means[at(2, b), 0] = one if b % 3 == 0 else 0x7E00 if b % 3 == 1 else to_bits(np.full(64, -np.inf, np.float32), 0)
    P.means[at(2, 200), 0] = to_bits(np.full(64, np.inf, np.float32), 0)
    q = to_bits(np.abs(np.random.default_rng(1).standard_normal((3, 4 * 64))).astype(np.float32) + 0.1, 0)
    for first, last, top in ((0, 1, 7), (1, 1, 100), (2, 3, 130), (0, 1, 298)):
        got = P.run([0, 1, 2], [B * 300 - 1] * 3, 4, first, last, top, q=q)
        P.check([0, 1, 2], [B * 300 - 1] * 3, 4, first, last, top, got)
    assert ext.device_status() == 0


def test_sparse_close_scores_are_told_apart(cuda):
    """Scores that agree to fp32's last digits, in every order: the choice is that of 64 bits."""
    B, n = 16, 257
    P = Paged(cuda, 23, [B * n], 1, 128, 1, B, B)
    rng = np.random.default_rng(3)
    base = (rng.standard_normal(128) * 30).astype(np.float32)
    for b in range(n - 1):
        x = base.copy()
        x[b % 128] = np.float32(x[b % 128] * (1 + 2.0 ** -7 * (b // 128 + 1)))          # one step of bf16 in one column
        P.means[P.table[0, b], 0] = to_bits(x, 1)
    q = to_bits((rng.standard_normal((1, 8 * 128)) * 2.0 ** rng.integers(-9, 3, 8 * 128)).astype(np.float32), 1)
    for top in (1, 17, 100, 200):
        got = P.run([0], [B * n - 1], 8, 0, 1, top, q=q)
        P.check([0], [B * n - 1], 8, 0, 1, top, got)


def test_sparse_bad_pages(cuda):
    """Entries that name no page: never an address, their blocks rank last, read as zeros where they are attended all the same, and are flagged."""
    P = Paged(cuda, 24, [700, 700, 100], 2, 128, 0, 64, 32)
    t = P.table.copy()
    t[0, 3], t[1, 10], t[2, 0] = -1, P.pool, 2 ** 31 - 1
    got = P.run([0], [699], 8, 1, 2, 4, table=t)
    assert ext.device_status() == ref.BAD_PAGE
    P.check([0], [699], 8, 1, 2, 4, got, t)
    for s, p in ((1, 699), (2, 99), (0, 200)):
        got = P.run([s], [p], 8, 1, 2, 4, table=t)
        assert ext.device_status() == ref.BAD_PAGE
        P.check([s], [p], 8, 1, 2, 4, got, t)
    short = np.ascontiguousarray(P.table[:, :2])          # rows of two columns for eleven pages
    got = P.run([1], [699], 8, 1, 2, 4, table=short)
    assert ext.device_status() == ref.BAD_PAGE
    P.check([1], [699], 8, 1, 2, 4, got, short)
    got = P.run([1], [120], 8, 1, 2, 4, table=short)
    assert ext.device_status() == 0
    P.check([1], [120], 8, 1, 2, 4, got, short)


@pytest.mark.parametrize("d,kvh,block,rows,keep", [(128, 1, 128, 20, (1, 1, 14)), (128, 2, 32, 10, (2, 2, 60)), (64, 4, 16, 5, (1, 2, 61)), (256, 1, 64, 20, (1, 2, 29))])
def test_sparse_many_rows_with_many_tiles_each(cuda, d, kvh, block, rows, keep):
    """Rows enough that each is one thread block's, which goes round its ring of tiles many times."""
    lens = [2900 - 37 * s for s in range(8)]
    P = Paged(cuda, 28, lens, kvh, d, 1, block, block)
    seq = [s for s in range(8) for _ in range(rows)]
    pos = [lens[s] - 1 - 11 * j for s in range(8) for j in range(rows)]
    got = P.run(seq, pos, 8 * kvh, *keep)
    again = P.run(seq, pos, 8 * kvh, *keep, q=got[0].reshape(len(seq), -1))
    assert ext.device_status() == 0
    for x, y in zip(got[1:], again[1:]):
        assert np.array_equal(x, y)
    P.check(seq, pos, 8 * kvh, *keep, got)


def test_sparse_at_a_position_far_past_the_table(cuda):
    """The last position there can be, over a row of a few columns: the blocks there are, then the lowest of those there are not."""
    B = 16
    P = Paged(cuda, 30, [B * 40, 5], 1, 64, 1, B, B)
    for top in (7, 60):
        _, o, _, chosen = P.run([0, 1], [2 ** 31 - 1, 2 ** 31 - 1], 4, 1, 2, top)
        assert ext.device_status() == ref.BAD_PAGE
        n, have = 2 ** 31 // B, -(-B * 40 // B)
        got = chosen[0, 0].tolist()
        assert got[0] == 0 and got[-2:] == [n - 2, n - 1]
        q = from_bits(P.last_q, 1).astype(np.float64).reshape(2, 4, 64)[0].sum(0)
        s = from_bits(P.means, 1).astype(np.float64)[P.table[0, :have], 0] @ q
        order = sorted(range(1, have), key=lambda b: (-s[b], b)) + list(range(have, have + top))
        assert got[1:-2] == sorted(order[:top]) and np.isfinite(from_bits(o[0], 1)).all()


def test_sparse_without_scores_needs_no_means(cuda):
    P = Paged(cuda, 25, [500, 20], 2, 64, 1, 64, 64)
    got = P.run([0, 1], [499, 19], 4, 2, 2, 0, means=False)
    P.check([0, 1], [499, 19], 4, 2, 2, 0, got)


def test_sparse_repeats_and_runs_on_a_stream_of_its_own(cuda):
    P = Paged(cuda, 26, [3000, 5000], 2, 128, 1, 128, 64)
    q = bits(P.rng, (2, 16 * 128), 1)
    a = P.run([0, 1], [2999, 4999], 16, 1, 2, 13, q=q)
    b = P.run([0, 1], [2999, 4999], 16, 1, 2, 13, q=q, stream=cuda.cuda.Stream())
    for x, y in zip(a[1:], b[1:]):
        assert np.array_equal(x, y)
    # and permuting which page holds what changes no bit
    perm = P.rng.permutation(P.pool)
    move = lambda x, n: np.concatenate([x.reshape(P.pool, n, *x.shape[1:])[[int(np.flatnonzero(perm == i)[0])]] for i in range(P.pool)]).reshape(x.shape)
    P.k, P.v, P.means = move(P.k, 128), move(P.v, 128), move(P.means, 2)
    c = P.run([0, 1], [2999, 4999], 16, 1, 2, 13, q=q, table=np.where(P.table >= 0, perm[np.maximum(P.table, 0)], -1).astype(np.int32))
    for x, y in zip(a[1:], c[1:]):
        assert np.array_equal(x, y)


def test_sparse_outputs_where_the_caller_wants_them(cuda):
    """No `chosen`; an output that starts on two bytes; either leaves the same bits, and nothing beside them."""
    P = Paged(cuda, 32, [900, 333], 2, 128, 0, 64, 32)
    q, o, _, _ = got = P.run([0, 1], [899, 332], 8, 1, 2, 6)
    P.check([0, 1], [899, 332], 8, 1, 2, 6, got)
    hold = [dev(cuda, x) for x in (q.reshape(2, -1), P.k, P.v, P.means, np.array([0, 1], np.int32), np.array([899, 332], np.int32), P.table)]
    wide = cuda.full((2 * 8 * 128 + 3,), 0x1234, dtype=cuda.int16, device="cuda")
    ext.paged_sparse(wide.data_ptr() + 2, None, None, hold[0], hold[1], hold[2], hold[3], hold[4], hold[5], 2, hold[6], 2, P.table.shape[1], P.pool, 64, 32, 8, 2, 128, 1, 2, 6)
    cuda.cuda.synchronize()
    b = host_bits(wide)
    assert np.array_equal(b[1:-2], o.reshape(-1)) and (b[[0, -2, -1]] == 0x1234).all() and ext.device_status() == 0


def test_two_captured_steps_beside_each_other(cuda):
    """Graphs of two pools replayed at the same time on two streams: the calls share nothing."""
    made = []
    for seed, dtype in ((40, 0), (41, 1)):
        P = Paged(cuda, seed, [4000, 2500, 777], 2, 64, dtype, 64, 16)
        seq, pos = [0, 1, 2], [3999, 2499, 776]
        q, o, res, chosen = got = P.run(seq, pos, 16, 1, 2, 20)
        P.check(seq, pos, 16, 1, 2, 20, got)
        hold = [dev(cuda, x) for x in (q.reshape(3, -1), P.k, P.v, P.means, np.array(seq, np.int32), np.array(pos, np.int32), P.table)]
        out, ids = cuda.zeros((3, 16, 64), dtype=cuda.int16, device="cuda"), i32(cuda, 3, 2, 23)
        graph, stream = cuda.cuda.CUDAGraph(), cuda.cuda.Stream()
        with cuda.cuda.graph(graph, stream=stream):
            for _ in range(20):
                ext.paged_sparse(out, None, ids, hold[0], hold[1], hold[2], hold[3], hold[4], hold[5], 3, hold[6], 3, P.table.shape[1], P.pool, 64, 16, 16, 2, 64, 1, 2, 20, dtype=dtype,
                                 stream=cuda.cuda.current_stream().cuda_stream)
        made.append((graph, stream, out, ids, o, chosen, hold))
    cuda.cuda.synchronize()
    for _ in range(5):
        for graph, stream, *_ in made:
            with cuda.cuda.stream(stream):
                graph.replay()
    cuda.cuda.synchronize()
    for _, _, out, ids, o, chosen, _ in made:
        assert np.array_equal(host_bits(out), o) and np.array_equal(ids.cpu().numpy(), chosen)
    assert ext.device_status() == 0


def test_sparse_with_every_block_kept_is_the_paged_decode(cuda):
    """Both are within the tolerance of the same 64-bit answer: within twice of it of each other."""
    P = Paged(cuda, 27, [1, 130, 777, 1500], 2, 128, 1, 128, 64)
    seq, pos = [0, 1, 2, 3], [n - 1 for n in P.lens]
    q, o, _, _ = got = P.run(seq, pos, 16, 1, 2, 30)
    P.check(seq, pos, 16, 1, 2, 30, got)
    plan = ext.Plan()
    plan.plan(P.lens, 16, 2, 128)
    o2 = cuda.zeros((4, 16, 128), dtype=cuda.int16, device="cuda")
    plan.decode(o2, None, dev(cuda, q.reshape(4, -1)), dev(cuda, P.k), dev(cuda, P.v), P.pool, 128, dev(cuda, P.table), P.table.shape[1], 1)
    cuda.cuda.synchronize()
    plan.close()
    a, b = from_bits(o, 1).astype(np.float64), from_bits(host_bits(o2), 1).astype(np.float64)
    # the decode rounds its weights to the type: half a step of each, at most max|v| < 5 away
    assert (np.abs(a - b) <= 2 * STEP[1] * (np.abs(a) + 5)).all()


# ---------------------------------------------------------------------------------------------------------------------
# the three together


def test_a_served_batch(cuda):
    """Prompts of ragged lengths enter, then steps of one position each with sequences that end and begin, all in one captured
    step: tables, rows into the pool, attention.  Every step against a cache kept on the host."""
    rng = np.random.default_rng(31)
    seqs, kvh, group, d, page, block, dtype, stride, pool, rows = 5, 2, 4, 128, 64, 32, 1, 8, 30, 420
    first, last, top = 1, 2, 3
    L, C, at = i32(cuda, seqs, fill=0), i32(cuda, seqs, fill=0), i32(cuda, 1, fill=0)
    T, F = i32(cuda, seqs, stride, fill=-1), dev(cuda, rng.permutation(pool).astype(np.int32))
    start, seq, pos, slot = i32(cuda, seqs + 1), i32(cuda, rows), i32(cuda, rows), i32(cuda, rows)
    kv = lambda n: cuda.full((n, kvh, d), 0x7FC1, dtype=cuda.int16, device="cuda")
    k, v, means = kv(pool * page), kv(pool * page), kv(pool * page // block)
    qkv = cuda.zeros((rows, (kvh * group + 2 * kvh) * d), dtype=cuda.int16, device="cuda")
    o, chosen = cuda.zeros((rows, kvh * group, d), dtype=cuda.int16, device="cuda"), i32(cuda, rows, kvh, first + last + top)
    wide, qw = qkv.shape[1], kvh * group * d

    def step():
        st = cuda.cuda.current_stream().cuda_stream
        ext.paged_tables(L, T, start, seq, pos, slot, at, F, at, L, C, seqs, stride, rows, pool, pool, page, stream=st)
        ext.paged_write(k, v, means, qkv.data_ptr() + 2 * qw, qkv.data_ptr() + 2 * (qw + kvh * d), slot, rows, kvh, d, pool, page, block, wide, wide, dtype, stream=st)
        ext.paged_sparse(o, None, chosen, qkv, k, v, means, seq, pos, rows, T, seqs, stride, pool, page, block, kvh * group, kvh, d, first, last, top, q_stride=wide, dtype=dtype, stream=st)

    ext.device_status()
    side = cuda.cuda.Stream()
    side.wait_stream(cuda.cuda.current_stream())
    with cuda.cuda.stream(side):
        step()                                            # no counts yet: nothing is written
    cuda.cuda.current_stream().wait_stream(side)
    cuda.cuda.synchronize()
    assert int((o != 0).sum()) == 0
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph):
        step()
    cache = [[np.zeros((0, kvh, d), np.uint16)] * 2 for _ in range(seqs)]
    plans = [[200, 1, 64, 0, 150]] + [[1, 1, 1, 0, 1]] * 4 + [[1, 1, -1, 33, 1], [1, 1, 100, 1, 1], [60, 0, 1, 1, -1], [1, 1, 1, 1, 65], [1, 1, 1, 1, 1]]
    f = lambda x: from_bits(x, dtype).astype(np.float64)
    for counts in plans:
        new = bits(rng, (rows, wide), dtype)
        qkv.copy_(dev(cuda, new))
        C.copy_(dev(cuda, np.array(counts, np.int32)))
        graph.replay()
        cuda.cuda.synchronize()
        assert ext.device_status() == 0
        r, got, ids = 0, host_bits(o), chosen.cpu().numpy()
        host_means = host_bits(means)
        table = T.cpu().numpy()
        for s, c in enumerate(counts):
            if c < 0:
                cache[s] = [np.zeros((0, kvh, d), np.uint16)] * 2
            for _ in range(max(c, 0)):
                rows_kv = new[r, qw:].reshape(2, kvh, d)
                cache[s] = [np.concatenate([cache[s][i], rows_kv[i:i + 1]]) for i in range(2)]
                r += 1
            if c <= 0:
                continue
            n = len(cache[s][0])
            # the cache as pages of its own, and the means that the card left
            own = np.arange(-(-n // page))
            pad = lambda x: np.concatenate([x, np.zeros((len(own) * page - n, kvh, d), np.uint16)])
            kk, vv = f(pad(cache[s][0])), f(pad(cache[s][1]))
            mm = f(host_means.reshape(pool, page // block, kvh, d)[table[s, own]].reshape(-1, kvh, d))
            whole = n // block
            true = kk[:whole * block].reshape(whole, block, kvh, d).mean(1) if whole else np.zeros((0, kvh, d))
            assert (np.abs(mm[:whole] - true) <= np.abs(true) * STEP[dtype] * 1.01 + (block + 1) * 2.0 ** -24 * 4).all()
            for g in range(kvh):
                q = f(new[r - 1, :qw].reshape(kvh, group, d)[g])
                want_ids, want, _, _, size, vmax = ref.sparse_row(q, kk[:, g], vv[:, g], mm[:, g], own, n - 1, page, block, first, last, top)
                assert ids[r - 1, g].tolist() == want_ids + [-1] * (first + last + top - len(want_ids))
                fp = (2 * (2 * (d + 3) * 2.0 ** -24 * size + 2.0 ** -16 + 2.0 ** -20 + n * 2.0 ** -24) * vmax)[:, None]
                err = np.abs(f(got[r - 1].reshape(kvh, group, d)[g]) - want)
                assert (err <= fp + (np.abs(want) + fp) * STEP[dtype]).all()
    lens = L.cpu().numpy()
    assert lens.tolist() == [len(c[0]) for c in cache]
