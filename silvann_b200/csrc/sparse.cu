/* sparse.cu — attention of new positions over the blocks of the paged pool that a cheap score selects
 * (silvann_b200_paged_sparse, include/silvann_b200.h): scores, choice and attention in one launch.
 *
 * A cluster of thread blocks (1 to 16) owns one row's query heads over one kv head (16 at most: more heads are more
 * clusters, which make the same choice).  Three phases:
 *
 *   scores  — every block's mean key is read once, from L2 or memory, and multiplied with the sum of the kv head's query
 *             heads in 64 bits; the cluster's thread blocks share the sequence's blocks and leave every score, as a float, in
 *             every thread block's shared memory.
 *   choice  — each thread block picks the same `top` blocks from the whole list, so nothing has to be sent round again: by the
 *             floats where their order tells, else by the 64 bits, which then follow.
 *   attend  — the blocks to attend are a short cache of their own: tiles of 32 KB of it are dealt to the thread blocks, arrive by TMA (128-byte swizzle) in a ring, and meet an online softmax with heads as the N dimension
 *             of the warp MMAs (S^T = K Q^T, O^T = V^T P^T).  Some warps share a tile by positions, and their sets share it by value
 *             columns (each set forms the scores, which is cheaper than more accumulators).  The partials
 *             meet through the cluster's shared memory, in a fixed order.  No scratch in global memory: calls share nothing.
 *
 * Why 64 bits for the scores: which block is chosen hangs on two scores next to each other, and a choice that went by the
 * order of a sum in fp32 would be one of the launch's shape.  The products of 16-bit values are exact there and the tree
 * over a mean's columns is the same wherever the mean lies.
 *
 * What bounds it.  Many rows of moderate length: memory (256 rows of 1,000 to 16,000 positions, 32 heads on 4 of 128, 16 blocks of 128
 * each: 172 us, 6.1 TB/s of means, keys and values).  Long rows: the phases' own chains of trips to memory and through shared
 * memory, during which little is in flight (32 rows of 1,024 to 100,000 positions, 16 heads on 2 of 256: 44 us, of which the tiles
 * are half; 24 us at memory's rate).  One row: that chain alone (8,192 positions 10.6 us, 262,144 positions 19.6 us in a graph).  Heads
 * of their own over 16-position blocks: the same and the issue of instructions (24 sequences of 5 drafted positions, 8 heads of 64: 64 us;
 * 0.48 instructions a cycle and scheduler, 24 % of DRAM).
 * Measured against, on the same cases: a choice that counts by barriers, or ranks every key against every other (among 4,096 blocks 12 to
 * 20 thousand cycles, now 7); scores written to the peers one by one (262,144 positions 22 us); 2 x 64 positions a tile at head_dim 256, one thread block an SM (49 us); means four lanes each instead of eight
 * (46 us); the tiles of the always attended blocks not asked for early (7 us more on the 256 rows). */
#include "../../include/silvann_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "paged_index.h"
#include "tensormap.cuh"
#include <atomic>
#include <math.h>
#include <stddef.h>
#include <string.h>

#define SV_EXPORT extern "C" __attribute__((visibility("default")))

int sv_ext_fail(int code, const char* fmt, ...);      /* ext.cu: records the message for silvann_b200_last_error */
namespace svf { extern std::atomic<uint64_t> g_counters[SILVANN_B200_COUNTERS]; }

namespace sv {

static constexpr int SPARSE_DEVICES = 64;
#define SP_WARPS 8
#define SP_THREADS (SP_WARPS * 32)
#define SP_CHUNK 4096u                        /* scores looked at in one go; the best of the chunks before them ride along */
#define SP_CAP (SP_CHUNK + SILVANN_B200_PAGED_KEEP_MAX + 8u)
#define SP_LIST 512u                          /* scores among which a warp looks for the border: sixteen a lane */

template <int D> struct SparseCfg {
    static constexpr int TP = D == 256 ? 32 : D == 128 ? 64 : 128;         /* positions a tile: 32 KB of K and V */
    static constexpr int PW = TP / 16;                    /* warps that share a tile by positions; SP_WARPS / PW share it by value columns */
    static constexpr int BOXES = D / 64;                  /* 64-column (128-byte) boxes a row */
    static constexpr int BOX_BYTES = TP * 128;
    static constexpr int K_BYTES = BOXES * BOX_BYTES;
    static constexpr int STAGE_BYTES = 2 * K_BYTES;       /* K then V */
    static constexpr int STAGES = D == 64 ? 2 : 3;        /* 96 KB, two thread blocks an SM; at 64 64 KB, three */
    static constexpr int OCC = D == 64 ? 3 : 2;           /* (at 64, on 120 rows of 8 kv heads: 64 us; two an SM 68, four with a ring of one stage 72) */
    /* scores: lanes a mean, 16-byte pieces of it a lane, means a warp takes in a round, rounds asked for at once */
    static constexpr int LPB = D == 256 ? 16 : 8;
    static constexpr int CPL = D / 8 / LPB;
    static constexpr int BPS = 32 / LPB;
    static constexpr int U = 8;
    static constexpr int WB = BPS * U;
};

struct SparseParams {
    void* o;
    float* res;
    int32_t* chosen;
    const uint16_t *q, *means;
    const int32_t *row_seq, *row_pos, *table;
    unsigned int *over, *status;
    uint64_t q_stride;
    PagedDiv per;                       /* blocks a page */
    uint32_t seqs, stride, pool_pages, page_pos, block, q_heads, kv_heads, group, head_blocks, first, last, top;
    uint32_t block_log, table_blocks;   /* blocks that a table row has columns for */
    uint32_t chunk, cap, choice_top;    /* scores looked at in one go, room for them, room for the chosen */
    uint32_t ring_bytes, choice_at, free_stages;      /* the ring, or what lies in its place before; where that begins; stages ahead of it */
    float scale_log2;
    bool o_wide;                        /* o starts on 8 bytes */
};

/* 16-bit values as doubles without a conversion (a shift and a mask run beside the multiply-adds, conversions take longer than them): the exponent and
 * mantissa bits moved to their place in a double's high word, which is the value times 2^-896 (bf16) or 2^-1008 (fp16),
 * subnormals included.  The query sum carries 2^800 or 2^900, so a score comes out times 2^-SHIFT.  An infinity
 * or a NaN would come out finite: `special` collects the magnitudes, and a mean that has one is summed again by conversion. */
template <int DT> struct Wide;
template <> struct Wide<SV_DTYPE_BF16> {
    static constexpr int SHIFT = 96;
    static constexpr uint32_t SPECIAL = 0x7F80u;
    static __device__ __forceinline__ double up() { return __hiloint2double((800 + 1023) << 20, 0); }
    static __device__ __forceinline__ double hi(uint32_t w) { return __hiloint2double(((int)w >> 3) & (int)0x8FFFE000, 0); }      /* (the sign stays, its copies go) */
    static __device__ __forceinline__ double lo(uint32_t w) { return hi(w << 16); }
};
template <> struct Wide<SV_DTYPE_FP16> {
    static constexpr int SHIFT = 108;
    static constexpr uint32_t SPECIAL = 0x7C00u;
    static __device__ __forceinline__ double up() { return __hiloint2double((900 + 1023) << 20, 0); }
    static __device__ __forceinline__ double hi(uint32_t w) { return __hiloint2double(((int)w >> 6) & (int)0x81FFFC00, 0); }      /* (the sign stays, its copies go) */
    static __device__ __forceinline__ double lo(uint32_t w) { return hi(w << 16); }
};

/* Orders as the score does, NaN with minus infinity. */
__device__ __forceinline__ unsigned long long score_key(double s) {
    if (!(s == s)) s = -INFINITY;
    const unsigned long long b = (unsigned long long)__double_as_longlong(s + 0.0);       /* -0 + 0 = +0: equal scores, equal keys */
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
/* The nearest float of a score (which carries 2^-SHIFT), NaN with minus infinity. */
template <int DT>
__device__ __forceinline__ float score_float(double s) { return s == s ? (float)(s * __hiloint2double((Wide<DT>::SHIFT + 1023) << 20, 0)) : -INFINITY; }

/* What the ring holds before the first tile: the choice's own tables, then, as long as the launch needs them, the scores of a chunk
 * of blocks behind the best of the chunks before. */
struct ChoiceTables {
    double qsum[256];
    float list_score[SP_LIST];
    uint32_t hist[256], n_list, pad[3];
    uint32_t warp_in[SP_WARPS], warp_tie[SP_WARPS];
    uint32_t bin, need, in_bin;
    float least;
};
struct Choice {
    ChoiceTables* t;
    uint32_t cap, top;                                                                            /* multiples of four */
    __device__ __forceinline__ float* score() const { return (float*)(t + 1); }                   /* [cap] to the nearest float: tells all but the closest apart; NaN where there is none */
    __device__ __forceinline__ int32_t* place() const { return (int32_t*)score() + cap; }         /* [cap] the block's number in the pool, -1: none */
    __device__ __forceinline__ uint32_t* key_hi() const { return (uint32_t*)score() + 2u * cap; } /* [cap] the score's 64-bit key (of the cluster's other thread blocks' */
    __device__ __forceinline__ uint32_t* key_lo() const { return (uint32_t*)score() + 3u * cap; } /* [cap] shares: only once it is asked for) */
    __device__ __forceinline__ uint32_t* ids() const { return (uint32_t*)score() + 4u * cap; }    /* [top] */
    __device__ __forceinline__ uint32_t* picked() const { return ids() + top; }                   /* [top] */
    __device__ __forceinline__ unsigned long long key(uint32_t i) const { return (unsigned long long)key_hi()[i] << 32 | key_lo()[i]; }
};

/* A histogram walked down from its top bin by one warp: the bin where the count reaches `need`, and what is still needed in it. */
__device__ __forceinline__ void hist_walk(const Choice S, uint32_t need, int lane) {
    uint32_t mine = 0u;
    for (int b = 0; b < 8; ++b) mine += S.t->hist[255 - 8 * lane - b];
    uint32_t upto = mine;
    for (int d = 1; d < 32; d <<= 1) { const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
    const unsigned reached = __ballot_sync(0xffffffffu, upto >= need);
    if (lane == __ffs(reached) - 1) {
        uint32_t covered = upto - mine, bin = 255u - 8u * (uint32_t)lane;
        for (int b = 0; b < 7 && covered + S.t->hist[bin] < need; ++b) covered += S.t->hist[bin--];
        S.t->bin = bin; S.t->need = need - covered; S.t->in_bin = S.t->hist[bin];
    }
}

/* Where the floats do not tell, as among many equal scores: the `take`-th greatest key found a byte at a time, then two passes
 * over all keys, one that counts and one that writes, in index order. */
__device__ __noinline__ void choose_by_bytes(const Choice S, uint32_t m, uint32_t take) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long known = 0ull, cut = 0ull;
    uint32_t ties = take;
    for (int shift = 56; shift >= 0; shift -= 8) {
        S.t->hist[tid] = 0u;
        __syncthreads();
        for (uint32_t i = tid; i < m; i += SP_THREADS)
            if ((S.key(i) & known) == cut) atomicAdd(&S.t->hist[(uint32_t)(S.key(i) >> shift) & 255u], 1u);
        __syncthreads();
        if (warp == 0) hist_walk(S, ties, lane);
        __syncthreads();
        cut |= (unsigned long long)S.t->bin << shift; ties = S.t->need; known |= 255ull << shift;
        __syncthreads();
    }
    /* every key above the cut and the first `ties` of those that equal it; each warp owns a run of indexes */
    const uint32_t run = ((m + SP_THREADS - 1) / SP_THREADS) * 32u, i0 = warp * run;
    uint32_t n_in = 0u, n_tie = 0u;
    for (uint32_t i = i0 + lane; i < i0 + run; i += 32) {
        n_in += __popc(__ballot_sync(0xffffffffu, i < m && S.key(i) > cut)); n_tie += __popc(__ballot_sync(0xffffffffu, i < m && S.key(i) == cut));
    }
    if (lane == 0) { S.t->warp_in[warp] = n_in; S.t->warp_tie[warp] = n_tie; }
    __syncthreads();
    uint32_t at = 0u, tied = 0u;
    for (int w = 0; w < warp; ++w) { at += S.t->warp_in[w]; tied += S.t->warp_tie[w]; }
    at += min(tied, ties);
    const unsigned below = (1u << lane) - 1u;
    for (uint32_t i = i0 + lane; i < i0 + run; i += 32) {
        const bool tie = i < m && S.key(i) == cut;
        const unsigned tb = __ballot_sync(0xffffffffu, tie);
        const bool in = (i < m && S.key(i) > cut) || (tie && tied + __popc(tb & below) < ties);
        const unsigned ib = __ballot_sync(0xffffffffu, in);
        if (in) S.picked()[at + __popc(ib & below)] = i;
        at += __popc(ib); tied += __popc(tb);
    }
    __syncthreads();
}

/* A number that exactly `take` of score[0..n) reach, n <= 32 K, or NaN when there is none: equal floats lie across the border,
 * or infinities do.  The interval between the least and the greatest finite score is halved by one warp that holds all scores, so that a
 * step is a compare, a vote and a population count, without a barrier. */
template <int K>
__device__ __forceinline__ float border(const float* score, uint32_t n, uint32_t take) {
    const uint32_t lane = threadIdx.x & 31u;
    float w[K];
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int x = 0; x < K; ++x) {
        w[x] = x * 32u + lane < n ? score[x * 32u + lane] : __int_as_float(0x7FFFFFFF);
        if (fabsf(w[x]) < INFINITY) { lo = fminf(lo, w[x]); hi = fmaxf(hi, w[x]); }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) { lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, x)); hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, x)); }
    auto reach = [&](float t) { uint32_t c = 0u;
#pragma unroll
        for (int x = 0; x < K; ++x) c += __popc(__ballot_sync(0xffffffffu, w[x] >= t));
        return c; };
    uint32_t c = reach(lo);
    if (c <= take) return c == take ? lo : __int_as_float(0x7FFFFFFF);
    for (int step = 0; step < 64; ++step) {       /* (a guess by the counts at both ends took fewer steps and more time) */
        const float mid = 0.5f * lo + 0.5f * hi;
        if (!(mid > lo && mid < hi)) break;
        c = reach(mid);
        if (c == take) return mid;
        if (c > take) lo = mid; else hi = mid;
    }
    return __int_as_float(0x7FFFFFFF);
}

/* The choice among few scores, one warp's work, four a lane. */
__device__ __noinline__ bool choose_few(const Choice S, uint32_t m, uint32_t take) {
    const uint32_t lane = threadIdx.x & 31u;
    if (threadIdx.x < 32u) {
        const float least = border<4>(S.score(), m, take);
        uint32_t at = 0u;
        if (least == least)
#pragma unroll
            for (uint32_t i = lane; i < 128u; i += 32u) {
                const bool is = i < m && S.score()[i] >= least;
                const unsigned in = __ballot_sync(0xffffffffu, is);
                if (is) S.picked()[at + __popc(in & ((1u << lane) - 1u))] = i;
                at += __popc(in);
            }
        if (lane == 0u) S.t->need = at;
    }
    __syncthreads();
    return S.t->need == take;
}

/* The choice among many: a histogram of 256 steps of equal width between the least and the greatest finite score finds the step that the
 * border lies in, which rarely holds more than a few (a tail of scores is thin); one warp finds the border among those. */
__device__ __noinline__ bool choose_many(const Choice S, uint32_t m, uint32_t take) {
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    float mn = INFINITY, mx = -INFINITY;
    for (uint32_t i = 4u * tid; i < m; i += 4u * SP_THREADS) {             /* (behind the last there are NaNs up to a multiple of four) */
        const float4 y = *reinterpret_cast<const float4*>(S.score() + i);
        const float f[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) if (fabsf(f[x]) < INFINITY) { mn = fminf(mn, f[x]); mx = fmaxf(mx, f[x]); }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) { mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, x)); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x)); }
    if (lane == 0u) { S.t->warp_in[warp] = __float_as_uint(mn); S.t->warp_tie[warp] = __float_as_uint(mx); }
    S.t->hist[tid] = 0u;
    if (tid == 0u) S.t->n_list = 0u;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SP_WARPS; ++w) { mn = fminf(mn, __uint_as_float(S.t->warp_in[w])); mx = fmaxf(mx, __uint_as_float(S.t->warp_tie[w])); }
    const float per = mx > mn ? __fdividef(255.99f, mx - mn) : 0.f, low = mx >= mn ? mn : 0.f;
    auto bin_of = [&](float f) { return (uint32_t)min(max((int)((f - low) * per), 0), 255); };     /* does not fall as f rises */
    for (uint32_t i = 4u * tid; i < m; i += 4u * SP_THREADS) {
        const float4 y = *reinterpret_cast<const float4*>(S.score() + i);
        const float f[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) if (f[x] == f[x]) atomicAdd(&S.t->hist[bin_of(f[x])], 1u);
    }
    __syncthreads();
    if (warp == 0u) hist_walk(S, take, lane);
    __syncthreads();
    const uint32_t bin = S.t->bin, need = S.t->need, in_bin = S.t->in_bin;
    if (in_bin > SP_LIST) return false;
    float least = -INFINITY;                      /* of the border's step, what reaches this is chosen */
    if (in_bin != need) {
        for (uint32_t i = 4u * tid; i < m; i += 4u * SP_THREADS) {
            const float4 y = *reinterpret_cast<const float4*>(S.score() + i);
            const float f[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) if (f[x] == f[x] && bin_of(f[x]) == bin) S.t->list_score[atomicAdd(&S.t->n_list, 1u)] = f[x];
        }
        __syncthreads();
        if (warp == 0u) {
            const float found = in_bin <= 32u ? border<1>(S.t->list_score, in_bin, need) : in_bin <= 128u ? border<4>(S.t->list_score, in_bin, need) : border<16>(S.t->list_score, in_bin, need);
            if (lane == 0u) S.t->least = found;
        }
        __syncthreads();
        least = S.t->least;
        if (!(least == least)) return false;
    }
    /* a thread's scores are neighbours now, so that its chosen ones are in order */
    const uint32_t run = (m + SP_THREADS * 4u - 1u) / (SP_THREADS * 4u) * 4u, i0 = tid * run, i1 = min(m, i0 + run);
    uint32_t hits = 0u;
    for (uint32_t i = i0, b = 0u; i < i1; i += 4u, b += 4u) {
        const float4 y = *reinterpret_cast<const float4*>(S.score() + i);
        const float f[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int x = 0; x < 4; ++x) { const uint32_t z = bin_of(f[x]); hits |= (f[x] == f[x] && (z > bin || (z == bin && f[x] >= least)) ? 1u : 0u) << (b + x); }
    }
    uint32_t upto = __popc(hits);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= d) upto += o; }
    __syncthreads();
    if (lane == 31u) S.t->warp_in[warp] = upto;
    __syncthreads();
    uint32_t at = upto - __popc(hits);
#pragma unroll
    for (uint32_t x = 0; x < SP_WARPS; ++x) if (x < warp) at += S.t->warp_in[x];
    for (; hits; hits &= hits - 1u, ++at) S.picked()[at] = i0 + __ffs(hits) - 1u;
    __syncthreads();
    return true;
}

/* The `take` greatest of the m scores (equal ones: the lower index), their indexes ascending into S.picked; m > take > 0; false when the
 * floats do not tell: the 64-bit keys have to (choose_by_bytes).  Called by SP_THREADS threads, with the same answer in all of them.
 * (125 scores: 2.3 thousand cycles the first way, 3.8 the second, with its barriers; 600 to 1,300: 5 the second way, 7 to 13 by a
 * warp that holds all of them.) */
__device__ __forceinline__ bool choose(const Choice S, uint32_t m, uint32_t take) { return m <= 128u ? choose_few(S, m, take) : choose_many(S, m, take); }

/* The score of a mean that holds an infinity or a NaN (any of a warp's `count`): summed by conversion.  Such a score is no finite number
 * whatever the order, so the order is the warp's own.  Answers the score of mean `want`, or `v` where that is an ordinary one. */
template <int D, int DT>
__device__ __noinline__ double special_score(const uint16_t* means, uint32_t row_elems, int32_t mine, int count, const double* qsum, int want, double v, int lpb) {
    using E = Elem<DT>;
    const int lane = threadIdx.x & 31;
    for (int b = 0; b < count; ++b) {
        const int32_t at = __shfl_sync(0xffffffffu, mine, b);
        if (at < 0) continue;
        bool is = false;
        double a = 0;
        for (int e = lane; e < D; e += 32) {
            const uint16_t h = means[(size_t)at * row_elems + e];
            is |= (h & 0x7FFFu) >= Wide<DT>::SPECIAL;
            const int ch = e / 8;
            a += (double)E::to_float(h) * qsum[(((ch / lpb) * 4 + (e % 8) / 2) * lpb + ch % lpb) * 2 + e % 2];
        }
        for (int x = 16; x > 0; x >>= 1) a += __shfl_xor_sync(0xffffffffu, a, x);
        if (__any_sync(0xffffffffu, is) && b == want) v = a;
    }
    return v;
}

__device__ __forceinline__ uint32_t peer_addr(const void* local, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
    return remote;
}

template <int D, int DT, int NHT>
__global__ void __launch_bounds__(SP_THREADS, SparseCfg<D>::OCC)
paged_sparse_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const SparseParams P) {
    using Cfg = SparseCfg<D>;
    using E = Elem<DT>;
    using W = Wide<DT>;
    constexpr int HPB = 8 * NHT, KS = D / 16, NW = SP_WARPS, PW = Cfg::PW, VS = KS / (NW / PW);      /* VS: 16-column steps of the value product a warp */
    constexpr int Q_BYTES = Cfg::BOXES * HPB * 128;
    constexpr bool QREG = NHT == 1;          /* 16 heads: the query's fragments are read from shared memory again for every tile */

    extern __shared__ uint8_t sp_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)sp_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t keep = P.first + P.last + P.top;
    uint8_t* ring = smem;
    const Choice S = {(ChoiceTables*)(ring + P.choice_at), P.cap, P.choice_top};
    uint8_t* q_base = ring + P.ring_bytes;
    float* meet = (float*)(q_base + Q_BYTES);                     /* [CL][HPB][D / CL] partials of this block's columns, from every peer */
    float* meet_ml = meet + HPB * D;                              /* [16][HPB][2] */
    uint64_t* full = (uint64_t*)(meet_ml + 16 * HPB * 2);
    uint64_t* empty = full + Cfg::STAGES;
    volatile uint32_t* abort_flag = (volatile uint32_t*)(empty + Cfg::STAGES);
    int32_t* slots = (int32_t*)(empty + Cfg::STAGES + 1);         /* [keep] the blocks' places in the pool: those always attended, then the chosen, then the row's own */

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t CL = cluster_nctarank(), crank = cluster_ctarank();
    const uint32_t unit = blockIdx.x / CL, hb = unit % P.head_blocks, kvh = (unit / P.head_blocks) % P.kv_heads, r = unit / P.head_blocks / P.kv_heads;
    const uint32_t head0 = kvh * P.group + hb * HPB, heads = min((uint32_t)HPB, P.group - hb * HPB);

    if (tid == 0) {
        for (int s = 0; s < Cfg::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], NW); }
        *abort_flag = 0u;
        mbar_fence_init();
        tma_prefetch_desc(&kmap); tma_prefetch_desc(&vmap);
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");      /* everything read below may be the work of the grid ahead */

    const int32_t seq = P.row_seq[r], pos = P.row_pos[r];
    /* the query does not hang on them: asked for at the same time */
    constexpr int QV = (HPB * (D / 8) + SP_THREADS - 1) / SP_THREADS;
    const uint16_t* qrow = P.q + (size_t)r * P.q_stride;
    uint4 qv[QV];
    double qs = 0;
#pragma unroll
    for (int x = 0; x < QV; ++x) {
        const uint32_t i = tid + x * SP_THREADS, h = i / (D / 8);
        qv[x] = h < heads ? *reinterpret_cast<const uint4*>(qrow + (size_t)(head0 + h) * D + (i % (D / 8)) * 8) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (P.top && tid < D) {
        const uint16_t* src = qrow + (size_t)kvh * P.group * D + tid;
#pragma unroll 8
        for (uint32_t h = 0; h < P.group; ++h) qs += (double)E::to_float(src[h * D]);
    }
    if (seq < 0 || (uint32_t)seq >= P.seqs) { if (seq >= 0 && tid == 0 && crank == 0 && P.status) atomicOr(P.status, SV_STATUS_BAD_PAGE); return; }
    const size_t out0 = (size_t)r * P.q_heads + head0;
    int32_t* chosen = P.chosen && hb == 0 && crank == 0 ? P.chosen + ((size_t)r * P.kv_heads + kvh) * keep : nullptr;
    if (pos < 0) {
        if (crank != 0) return;
        for (uint32_t i = tid; i < heads * D; i += blockDim.x) {
            if (P.o) ((uint16_t*)P.o)[out0 * D + i] = 0;
            if (P.res) { float* x = P.res + (out0 + i / D) * (D + 2); x[2 + i % D] = 0.f; if (i % D == 0) { x[0] = -INFINITY; x[1] = 0.f; } }
        }
        if (chosen) for (uint32_t i = tid; i < keep; i += blockDim.x) chosen[i] = -1;
        return;
    }
    const PagedChoice c = paged_choice((uint32_t)pos, P.block, P.first, P.last, P.top);
    /* blocks that the table row has no column for score minus infinity: of a position far past it, no more of them are looked at than
     * could be chosen */
    const uint32_t c_hi = min(c.hi, max(P.table_blocks, c.lo + c.take + 1u));
    const int32_t* row = P.table + (size_t)seq * P.stride;
    bool bad = false;
    /* a block whose page is none is asked for past the pool's last row, where TMA answers zeros */
    auto slot_of = [&](int32_t place) { return place < 0 ? (int32_t)(P.pool_pages * P.page_pos) : (int32_t)((uint32_t)place * P.block); };

    /* a peer's shared memory may be written only once the peer runs: arrive now, wait ahead of the first score */
    if (CL > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");

    /* A chunk's means are cut evenly over the cluster (in fours: its scores are sent round sixteen bytes at a time); a thread block's
     * `n` from `base` on are dealt to its warps BPS at a time, U times round: this lane's u-th is i0 + u * STRIDE + w_at + lane / LPB.
     * Lane l looks up the page of the (l / BPS)-th round's l % BPS-th. */
    constexpr uint32_t STRIDE = NW * Cfg::BPS;
    const uint32_t w_at = warp * Cfg::BPS;
    auto share = [&](uint32_t chunk) { return ((chunk + CL - 1u) / CL + 3u) & ~3u; };
    auto look_up = [&](uint32_t base, uint32_t n, uint32_t i0) {
        const uint32_t i = i0 + (lane / Cfg::BPS) * STRIDE + w_at + lane % Cfg::BPS;
        if (lane >= Cfg::WB || i >= n) return -1;
        const int32_t at = paged_block(row, P.stride, P.pool_pages, P.per, base + i);
        bad |= at < 0;
        return at;
    };
    uint4 x[Cfg::U][Cfg::CPL];
    auto load = [&](int32_t mine, int g) {                /* rounds g to g + 3; from L2: a mean is read once, and may be the grid ahead's work */
#pragma unroll
        for (int u = g; u < g + 4; ++u) {
            const int32_t at = __shfl_sync(0xffffffffu, mine, u * Cfg::BPS + lane / Cfg::LPB);
            const uint4* src = reinterpret_cast<const uint4*>(P.means + ((size_t)max(at, 0) * P.kv_heads + kvh) * D) + lane % Cfg::LPB;
#pragma unroll
            for (int y = 0; y < Cfg::CPL; ++y) x[u][y] = at >= 0 ? __ldcg(src + y * Cfg::LPB) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    int32_t mine = -1, next = -1;
    /* the blocks that are always attended: their pages are asked for first, and kept below while the means are on their way */
    auto always = [&](uint32_t i) { return i < c.lo ? i : c.hi + (i - c.lo - c.take); };
    const bool fixed = (uint32_t)tid < c.count && !((uint32_t)tid >= c.lo && (uint32_t)tid < c.lo + c.take);
    const int32_t fixed_at = fixed ? paged_block(row, P.stride, P.pool_pages, P.per, always(tid)) : 0;
    if (c.take) {
        const uint32_t chunk = min(P.chunk, c_hi - c.lo), per = share(chunk), from = min(chunk, crank * per);
        mine = look_up(c.lo + from, min(per, chunk - from), 0u);
        next = look_up(c.lo + from, min(per, chunk - from), STRIDE * Cfg::U);
        load(mine, 0);
        load(mine, 4);
    }
#pragma unroll
    for (int z = 0; z < QV; ++z) {
        const uint32_t i = tid + z * SP_THREADS, h = i / (D / 8), j = i % (D / 8);
        if (h < HPB) *reinterpret_cast<uint4*>(q_base + (j / 8) * (HPB * 128) + swz128(h, j % 8)) = qv[z];
    }
    /* the summed query in pairs, a round's pairs side by side for the lanes that share a mean */
    if (c.take && tid < D) S.t->qsum[((((tid / 8) / Cfg::LPB) * 4 + (tid % 8) / 2) * Cfg::LPB + (tid / 8) % Cfg::LPB) * 2 + tid % 2] = qs * W::up();
    for (uint32_t i = tid; i < keep; i += SP_THREADS) {
        if (i >= c.lo && i < c.lo + c.take) continue;
        if (i < c.count) {
            const int32_t at = i == (uint32_t)tid ? fixed_at : paged_block(row, P.stride, P.pool_pages, P.per, always(i));
            bad |= at < 0;
            slots[i < c.lo ? i : i + 1u == c.count ? i : i - c.take] = slot_of(at);
        }
        if (chosen) chosen[i] = i < c.count ? (int32_t)always(i) : -1;
    }
    /* Tile t of the positions to attend, in the order of `slots`, belongs to thread block t % CL. */
    const uint32_t live = (c.count - 1u) * P.block + ((uint32_t)pos & (P.block - 1u)) + 1u;      /* the row's own block comes last and may end early */
    const uint32_t tiles = (live + Cfg::TP - 1u) / Cfg::TP;
    const int nt = tiles > crank ? (int)((tiles - crank + CL - 1) / CL) : 0;

    /* the loads of tile `it`: one box of 64 columns by min(B, TP) positions a lane of one warp */
    constexpr uint32_t TP_LOG = Cfg::TP == 32 ? 5u : Cfg::TP == 64 ? 6u : 7u;
    const uint32_t br_log = min(P.block_log, TP_LOG), br = 1u << br_log;
    const uint64_t pol = l2_policy_evict_first();
    auto fetch = [&](int it) {
        const int s = it % Cfg::STAGES;
        const uint32_t p0 = (crank + it * CL) * Cfg::TP;
        const uint32_t boxes = min((uint32_t)Cfg::TP >> br_log, (live - p0 + br - 1u) >> br_log);
        uint8_t* st = ring + s * Cfg::STAGE_BYTES;
        if (lane == 0) mbar_expect_tx(&full[s], boxes * br * 128u * Cfg::BOXES * 2u);
        __syncwarp();
        for (uint32_t i = lane; i < boxes * Cfg::BOXES * 2u; i += 32) {
            const uint32_t b = i / (Cfg::BOXES * 2u), x = i % (Cfg::BOXES * 2u), col = x % Cfg::BOXES;
            const uint32_t at = p0 + b * br;
            const int32_t y = slots[at >> P.block_log] + (int32_t)(at & (P.block - 1u));
            tma_load_2d_hint(st + (x / Cfg::BOXES) * Cfg::K_BYTES + col * Cfg::BOX_BYTES + b * br * 128u, x < Cfg::BOXES ? (const void*)&kmap : (const void*)&vmap, &full[s],
                             (int32_t)(kvh * D + col * 64u), y, pol);
        }
        __syncwarp();
    };
    /* tiles of blocks that are always attended are asked for ahead of the scores, where the choice's tables leave their stage free */
    const uint32_t known = c.take ? (c.lo + P.last - 1u) * P.block : live;
    auto early = [&](int it) { return !c.take || (it < (int)P.free_stages && min((crank + it * CL + 1u) * Cfg::TP, live) <= known); };
    __syncthreads();
    if (warp < Cfg::STAGES && warp < nt && early(warp)) fetch(warp);
    if (CL > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

    /* ---- scores and choice, a chunk of blocks at a time ---- */
    const bool many = c_hi - c.lo > P.chunk;
    uint32_t have = 0;                                                    /* the best of the chunks so far: keys, place, ids [0..have) */
    for (uint32_t base = c.lo; c.take && base < c_hi; base += P.chunk) {
        const uint32_t chunk = min(P.chunk, c_hi - base), per = share(chunk), from = min(chunk, crank * per), n = min(per, chunk - from);
        const uint32_t front = (have + 3u) & ~3u;                         /* where the chunk's scores begin, on sixteen bytes */
        {
            if (base != c.lo) { mine = look_up(base + from, n, 0u); next = look_up(base + from, n, STRIDE * Cfg::U); load(mine, 0); load(mine, 4); }
            for (uint32_t i0 = 0; i0 < n; i0 += STRIDE * Cfg::U) {
                /* the places of the round after next, and, as soon as four of this one are multiplied, the next one's four */
                const int32_t later = look_up(base + from, n, i0 + 2u * STRIDE * Cfg::U);
                const bool on = i0 + STRIDE * Cfg::U < n;
                double s[Cfg::U];
                uint32_t special = 0u;
#pragma unroll
                for (int g = 0; g < Cfg::U; g += 4) {
                    s[g] = s[g + 1] = s[g + 2] = s[g + 3] = 0;
                    if (i0 + g * STRIDE + w_at < n)
#pragma unroll
                    for (int y = 0; y < Cfg::CPL; ++y) {
                        double a[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const double2 q2 = *reinterpret_cast<const double2*>(S.t->qsum + ((y * 4 + z) * Cfg::LPB + lane % Cfg::LPB) * 2);
#pragma unroll
                            for (int u = g; u < g + 4; ++u) {
                                const uint32_t w = z == 0 ? x[u][y].x : z == 1 ? x[u][y].y : z == 2 ? x[u][y].z : x[u][y].w;
                                a[u - g] = fma(W::lo(w), q2.x, a[u - g]); a[u - g] = fma(W::hi(w), q2.y, a[u - g]);
                                special = __vmaxu2(special, w & 0x7FFF7FFFu);
                            }
                        }
#pragma unroll
                        for (int u = 0; u < 4; ++u) s[g + u] += a[u];
                    }
                    if (on) load(next, g);
                }
                const int32_t old = mine;
                mine = next; next = later;
                /* the lanes' parts of eight means at once: each exchange halves what a lane still holds; whichever of two lanes
                 * adds, the sum is the same */
                constexpr int T0 = Cfg::LPB / 2, T1 = Cfg::LPB / 4, T2 = Cfg::LPB / 8;
                const bool up0 = (lane & T0) != 0, up1 = (lane & T1) != 0, up2 = (lane & T2) != 0;
                double a[4], b[2];
#pragma unroll
                for (int u = 0; u < 4; ++u) a[u] = (up0 ? s[4 + u] : s[u]) + __shfl_xor_sync(0xffffffffu, up0 ? s[u] : s[4 + u], T0);
#pragma unroll
                for (int u = 0; u < 2; ++u) b[u] = (up1 ? a[2 + u] : a[u]) + __shfl_xor_sync(0xffffffffu, up1 ? a[u] : a[2 + u], T1);
                double v = (up2 ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, up2 ? b[0] : b[1], T2);
                if (T2 == 2) v += __shfl_xor_sync(0xffffffffu, v, 1);
                const int u = (up0 ? 4 : 0) + (up1 ? 2 : 0) + (up2 ? 1 : 0);
                const int32_t at = __shfl_sync(0xffffffffu, old, u * Cfg::BPS + lane / Cfg::LPB);
                if (__any_sync(0xffffffffu, (special & 0xFFFFu) >= W::SPECIAL || (special >> 16) >= W::SPECIAL))
                    v = special_score<D, DT>(P.means + (size_t)kvh * D, P.kv_heads * D, old, Cfg::WB, S.t->qsum, u * Cfg::BPS + lane / Cfg::LPB, v, Cfg::LPB);
                const uint32_t i = i0 + u * STRIDE + w_at + lane / Cfg::LPB;
                if (i < n && lane % T2 == 0) {
                    const double score = at >= 0 ? v : -INFINITY;
                    const unsigned long long k = score_key(score);
                    const uint32_t z = front + from + i;
                    S.score()[z] = score_float<DT>(score); S.key_hi()[z] = (uint32_t)(k >> 32); S.key_lo()[z] = (uint32_t)k; S.place()[z] = at;
                }
            }
        }
        /* between the best of the chunks before and this chunk, and behind it: no scores, and keys that none has */
        if (tid < 4u) {
            if (have + tid < front) { S.score()[have + tid] = __int_as_float(0x7FFFFFFF); S.key_hi()[have + tid] = 0u; S.key_lo()[have + tid] = 0u; }
            S.score()[front + chunk + tid] = __int_as_float(0x7FFFFFFF); S.key_hi()[front + chunk + tid] = 0u; S.key_lo()[front + chunk + tid] = 0u;
        }
        /* this thread block's share of two arrays to every peer, four entries at a time (behind the chunk's last there is the same everywhere) */
        auto send = [&](const uint32_t* two) {
            for (uint32_t z = tid >> 1; z < (n + 3u) / 4u; z += SP_THREADS / 2u) {
                const uint32_t* src = two + (tid & 1u) * S.cap + front + from + z * 4u;
                const uint4 y = *reinterpret_cast<const uint4*>(src);
#pragma unroll 4
                for (uint32_t to = 0; to < CL; ++to)
                    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(peer_addr(src, to)), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w) : "memory");
            }
        };
        __syncthreads();
        if (CL > 1) {
            send((const uint32_t*)S.score());
            if (many) send(S.key_hi());                                     /* the best go on to the next chunk with their keys */
            cluster_sync_all();
        }
        const uint32_t m = front + chunk;
        const bool more = base + P.chunk < c_hi;
        /* (a chunk holds more blocks than can be chosen, or all there are: m > take) */
        if (!choose(S, m, c.take)) {                                      /* all of the cluster's thread blocks come by here, or none */
            __syncthreads();
            if (CL > 1 && !many) { send(S.key_hi()); cluster_sync_all(); }
            choose_by_bytes(S, m, c.take);
        }
        auto id_of = [&](uint32_t i) { return i < have ? S.ids()[i] : base + (i - front); };
        if (more) {
            /* the chosen move to the front, in order: read all, then write */
            constexpr int KP = SILVANN_B200_PAGED_KEEP_MAX / SP_THREADS;
            float ks[KP];
            uint32_t kh[KP], kl[KP], ii[KP];
            int32_t pp[KP];
#pragma unroll
            for (int z = 0; z < KP; ++z) {
                const uint32_t i = tid + z * SP_THREADS;
                if (i < c.take) { const uint32_t at = S.picked()[i]; ks[z] = S.score()[at]; kh[z] = S.key_hi()[at]; kl[z] = S.key_lo()[at]; ii[z] = id_of(at); pp[z] = S.place()[at]; }
            }
            __syncthreads();
#pragma unroll
            for (int z = 0; z < KP; ++z) {
                const uint32_t i = tid + z * SP_THREADS;
                if (i < c.take) { S.score()[i] = ks[z]; S.key_hi()[i] = kh[z]; S.key_lo()[i] = kl[z]; S.ids()[i] = ii[z]; S.place()[i] = pp[z]; }
            }
            have = c.take;
            /* no one writes the next scores over what a peer still reads */
            if (CL > 1) cluster_sync_all(); else __syncthreads();
        } else {
            for (uint32_t i = tid; i < c.take; i += SP_THREADS) {
                const uint32_t at = S.picked()[i];
                slots[c.lo + P.last - 1u + i] = slot_of(S.place()[at]);
                if (chosen) chosen[c.lo + i] = (int32_t)id_of(at);
            }
        }
    }
    fence_proxy_async_smem();            /* the scores' accesses to the ring come before the loads into it */
    __syncthreads();

    float m_run[NHT][2], l_run[NHT][2], oacc[NHT][VS][4];
#pragma unroll
    for (int n = 0; n < NHT; ++n) {
        m_run[n][0] = m_run[n][1] = -INFINITY; l_run[n][0] = l_run[n][1] = 0.f;
#pragma unroll
        for (int k = 0; k < VS; ++k) { oacc[n][k][0] = oacc[n][k][1] = oacc[n][k][2] = oacc[n][k][3] = 0.f; }
    }
    /* ---- attend ---- */
    if (warp < Cfg::STAGES && warp < nt && !early(warp)) fetch(warp);
    {
        const uint32_t q_u32 = smem_u32(q_base);
        auto load_qfrag = [&](int n, int kk, uint32_t& b0, uint32_t& b1) {
            /* B fragment of Q^T for heads n*8..n*8+7, columns kk*16..+15: two 8x8 blocks (chunks 2kk, 2kk+1) */
            const int chunk = 2 * kk + ((lane >> 3) & 1), hrow = n * 8 + (lane & 7);
            uint32_t r2, r3;
            ldsm_x4(q_u32 + (chunk / 8) * (HPB * 128) + swz128(hrow, chunk % 8), b0, b1, r2, r3);
        };
        uint32_t qf[QREG ? KS : 1][2];
        if (QREG) {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) load_qfrag(0, kk, qf[kk][0], qf[kk][1]);
        }
        const int r_lo = lane >> 2, wp = warp % PW, wc = warp / PW;      /* positions [16 wp, +16) of a tile, value columns [16 VS wc, +16 VS) */
        for (int it = 0; it < nt; ++it) {
            const int s = it % Cfg::STAGES;
            /* the warps take turns to ask for the tile that goes where the one before this lay, once all have left it */
            if (it > 0 && it - 1 + Cfg::STAGES < nt && warp == it % NW) {
                if (!mbar_wait(&empty[(it - 1) % Cfg::STAGES], ((it - 1) / Cfg::STAGES) & 1, abort_flag, P.status)) break;
                fetch(it - 1 + Cfg::STAGES);
            }
            if (!mbar_wait(&full[s], (it / Cfg::STAGES) & 1, abort_flag, P.status)) break;
            uint8_t* stage = ring + s * Cfg::STAGE_BYTES;
            const uint32_t kst = smem_u32(stage), vst = kst + Cfg::K_BYTES;
            const uint32_t p0 = (crank + it * CL) * Cfg::TP + wp * 16u;
            /* rows of V behind the row's own position may hold anything: zero, so that a zero weight times a NaN cannot reach the sum */
            if (p0 + 16u > live) {
                for (int i = lane; i < 16 * (VS * 2); i += 32) {
                    const int y = i / (VS * 2), j = wc * (VS * 2) + i % (VS * 2);
                    if (p0 + y >= live)
                        *reinterpret_cast<uint4*>(stage + Cfg::K_BYTES + (j / 8) * Cfg::BOX_BYTES + swz128(wp * 16 + y, j % 8)) = make_uint4(0u, 0u, 0u, 0u);
                }
                __syncwarp();
            }
            /* S^T[16 positions][heads] = K_tile Q^T, two interleaved accumulators per head tile */
            float sa[NHT][4], sb[NHT][4];
#pragma unroll
            for (int n = 0; n < NHT; ++n) { sa[n][0] = sa[n][1] = sa[n][2] = sa[n][3] = 0.f; sb[n][0] = sb[n][1] = sb[n][2] = sb[n][3] = 0.f; }
#pragma unroll
            for (int kk = 0; kk < KS; ++kk) {
                const int krow = wp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, chunk = 2 * kk + (lane >> 4);
                uint32_t a0, a1, a2, a3;
                ldsm_x4(kst + (chunk / 8) * Cfg::BOX_BYTES + swz128(krow, chunk % 8), a0, a1, a2, a3);
#pragma unroll
                for (int n = 0; n < NHT; ++n) {
                    uint32_t b0, b1;
                    if (QREG) { b0 = qf[kk][0]; b1 = qf[kk][1]; } else load_qfrag(n, kk, b0, b1);
                    if (kk & 1) mma16816<DT>(sb[n], a0, a1, a2, a3, b0, b1);
                    else        mma16816<DT>(sa[n], a0, a1, a2, a3, b0, b1);
                }
            }
            /* online softmax over positions (accumulator rows), per head (accumulator columns).  The weights go to the MMA as
             * two 16-bit parts, value and what its rounding left: the tensor pipe is a sixth busy, and one part alone would
             * double the answer's rounding error */
            uint32_t ph[NHT][2], pl[NHT][2];
            const bool v0 = p0 + r_lo < live, v1 = p0 + r_lo + 8 < live;
#pragma unroll
            for (int n = 0; n < NHT; ++n) {
                const float t0 = v0 ? (sa[n][0] + sb[n][0]) * P.scale_log2 : -INFINITY;   /* position r_lo,   head A */
                const float t1 = v0 ? (sa[n][1] + sb[n][1]) * P.scale_log2 : -INFINITY;   /* position r_lo,   head B */
                const float t2 = v1 ? (sa[n][2] + sb[n][2]) * P.scale_log2 : -INFINITY;   /* position r_lo+8, head A */
                const float t3 = v1 ? (sa[n][3] + sb[n][3]) * P.scale_log2 : -INFINITY;   /* position r_lo+8, head B */
                float ma = fmaxf(t0, t2), mb = fmaxf(t1, t3);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    ma = fmaxf(ma, __shfl_xor_sync(0xffffffffu, ma, x));
                    mb = fmaxf(mb, __shfl_xor_sync(0xffffffffu, mb, x));
                }
                const float na = fmaxf(m_run[n][0], ma), nb = fmaxf(m_run[n][1], mb);
                const float ua = (na == -INFINITY) ? 0.f : na, ub = (nb == -INFINITY) ? 0.f : nb;
                const float fa = fast_exp2(m_run[n][0] - ua), fb = fast_exp2(m_run[n][1] - ub);
                m_run[n][0] = na; m_run[n][1] = nb;
                const float e0 = fast_exp2(t0 - ua), e1 = fast_exp2(t1 - ub), e2 = fast_exp2(t2 - ua), e3 = fast_exp2(t3 - ub);
                const uint32_t w0 = E::pack2(e0, e1), w1 = E::pack2(e2, e3);
                const float2 f0 = E::unpack2(w0), f1 = E::unpack2(w1);
                ph[n][0] = movm_t(w0); ph[n][1] = movm_t(w1);
                pl[n][0] = movm_t(E::pack2(e0 - f0.x, e1 - f0.y)); pl[n][1] = movm_t(E::pack2(e2 - f1.x, e3 - f1.y));
                l_run[n][0] = l_run[n][0] * fa + (e0 + e2);
                l_run[n][1] = l_run[n][1] * fb + (e1 + e3);
                if (__any_sync(0xffffffffu, fa != 1.f || fb != 1.f)) {
#pragma unroll
                    for (int k = 0; k < VS; ++k) { oacc[n][k][0] *= fa; oacc[n][k][2] *= fa; oacc[n][k][1] *= fb; oacc[n][k][3] *= fb; }
                }
            }
            /* O^T[value column][head] += V_tile^T P^T */
#pragma unroll
            for (int mt = 0; mt < VS; ++mt) {
                const int j = lane >> 3, vrow = wp * 16 + (lane & 7) + (j >> 1) * 8, chunk = 2 * (wc * VS + mt) + (j & 1);
                uint32_t a0, a1, a2, a3;
                ldsm_x4_t(vst + (chunk / 8) * Cfg::BOX_BYTES + swz128(vrow, chunk % 8), a0, a1, a2, a3);
#pragma unroll
                for (int n = 0; n < NHT; ++n) {
                    mma16816<DT>(oacc[n][mt], a0, a1, a2, a3, ph[n][0], ph[n][1]);
                    mma16816<DT>(oacc[n][mt], a0, a1, a2, a3, pl[n][0], pl[n][1]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        /* the lanes that share a head column hold disjoint positions: fold their sums */
#pragma unroll
        for (int n = 0; n < NHT; ++n)
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                l_run[n][0] += __shfl_xor_sync(0xffffffffu, l_run[n][0], x);
                l_run[n][1] += __shfl_xor_sync(0xffffffffu, l_run[n][1], x);
            }
    }

    /* ---- the warps' partials meet in shared memory (the ring is free now), then the cluster's thread blocks ---- */
    __syncthreads();
    if (*abort_flag != 0u) {
        /* a wait gave up (the status word says so): copies asked for may still be on their way into the ring, so every stage gets
         * a bounded chance to land before the ring is written over */
        if (tid == 0)
            for (int s = 0; s < Cfg::STAGES && s < nt; ++s) {
                const int last = (nt - 1 - s) / Cfg::STAGES;
                for (uint32_t i = 0; i < (1u << 16) && !mbar_try_wait(&full[s], last & 1); ++i) {}
            }
        __syncthreads();
    }
    constexpr int WS = D + 4;                         /* a row of partials: the pad spreads the accumulators' columns over the banks */
    float* wm = (float*)ring;                         /* [PW][HPB] */
    float* wl = wm + PW * HPB;                        /* [PW][HPB] */
    float* wo = wl + PW * HPB;                        /* [PW][HPB][WS] */
    {
        const int r_lo = lane >> 2, c2 = (lane & 3) * 2, wp = warp % PW, wc = warp / PW;
#pragma unroll
        for (int n = 0; n < NHT; ++n) {
            const int ha = n * 8 + c2;
            if (r_lo == 0 && wc == 0) {
                wm[wp * HPB + ha] = m_run[n][0]; wm[wp * HPB + ha + 1] = m_run[n][1];
                wl[wp * HPB + ha] = l_run[n][0]; wl[wp * HPB + ha + 1] = l_run[n][1];
            }
#pragma unroll
            for (int k = 0; k < VS; ++k) {
                float* at = wo + (wp * HPB + ha) * WS + (wc * VS + k) * 16 + r_lo;
                at[0] = oacc[n][k][0];
                at[WS] = oacc[n][k][1];
                at[8] = oacc[n][k][2];
                at[WS + 8] = oacc[n][k][3];
            }
        }
    }
    __syncthreads();
    bool hit = false;
    /* four columns of a head's answer */
    auto answer = [&](uint32_t h, uint32_t e, float m, float l, const float (&acc)[4]) {
        const size_t hq = out0 + h;
        if (P.o) {
            const float inv = 1.0f / l;
            uint16_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = E::from_float(acc[x] * inv, hit);
            uint16_t* at = (uint16_t*)P.o + hq * D + e;
            if (P.o_wide) *reinterpret_cast<uint2*>(at) = make_uint2(w[0] | (uint32_t)w[1] << 16, w[2] | (uint32_t)w[3] << 16);
            else { at[0] = w[0]; at[1] = w[1]; at[2] = w[2]; at[3] = w[3]; }
        }
        if (P.res) {
            float* at = P.res + hq * (D + 2);
            at[2 + e] = acc[0]; at[3 + e] = acc[1]; at[4 + e] = acc[2]; at[5 + e] = acc[3];
            if (e == 0) { at[0] = m * SV_LN2; at[1] = l; }
        }
    };
    for (uint32_t i = tid; i < heads * (D / 4); i += SP_THREADS) {
        const uint32_t h = i / (D / 4), e = i % (D / 4) * 4u;
        float pm[PW], m = -INFINITY;
#pragma unroll
        for (int w = 0; w < PW; ++w) { pm[w] = wm[w * HPB + h]; m = fmaxf(m, pm[w]); }
        float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll
        for (int w = 0; w < PW; ++w) {
            const float f = pm[w] == -INFINITY ? 0.f : fast_exp2(pm[w] - m);
            const float4 x = *reinterpret_cast<const float4*>(wo + (w * HPB + h) * WS + e);
            acc[0] += x.x * f; acc[1] += x.y * f; acc[2] += x.z * f; acc[3] += x.w * f; l += wl[w * HPB + h] * f;
        }
        if (CL == 1) answer(h, e, m, l, acc);
        else {
            /* columns [c D/CL, (c+1) D/CL) of every head meet in thread block c */
            const uint32_t DS = D / CL, to = e / DS;
            const uint32_t at = peer_addr(meet + (crank * HPB + h) * DS + e % DS, to);
            asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(acc[0]), "f"(acc[1]), "f"(acc[2]), "f"(acc[3]) : "memory");
            if (e % DS == 0) asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(peer_addr(meet_ml + (crank * HPB + h) * 2, to)), "f"(m), "f"(l) : "memory");
        }
    }
    if (CL > 1) {
        cluster_sync_all();                           /* nothing is sent to a peer after this */
        const uint32_t DS = D / CL;
        /* four lanes share four columns of a head: each folds every fourth peer, then they fold each other's */
        for (uint32_t i0 = 0; i0 < heads * DS; i0 += SP_THREADS) {
            const uint32_t i = min(i0 + tid, heads * DS - 1u), part = i & 3u, h = i / DS, e = i % DS & ~3u;
            float2 ml[4];
            float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t x = 0; x < 4u; ++x) { ml[x] = part + 4u * x < CL ? *reinterpret_cast<const float2*>(meet_ml + ((part + 4u * x) * HPB + h) * 2) : make_float2(-INFINITY, 0.f); m = fmaxf(m, ml[x].x); }
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
#pragma unroll
            for (uint32_t x = 0; x < 4u; ++x)
                if (part + 4u * x < CL) {
                    const float f = ml[x].x == -INFINITY ? 0.f : fast_exp2(ml[x].x - m);
                    const float4 y = *reinterpret_cast<const float4*>(meet + ((part + 4u * x) * HPB + h) * DS + e);
                    acc[0] += y.x * f; acc[1] += y.y * f; acc[2] += y.z * f; acc[3] += y.w * f; l += ml[x].y * f;
                }
#pragma unroll
            for (int t = 1; t < 4; t <<= 1) {
#pragma unroll
                for (int y = 0; y < 4; ++y) acc[y] += __shfl_xor_sync(0xffffffffu, acc[y], t);
                l += __shfl_xor_sync(0xffffffffu, l, t);
            }
            if (part == 0 && i0 + tid < heads * DS) answer(h, crank * DS + e, m, l, acc);
        }
    }
    if (hit && P.over) atomicOr(P.over, SV_FAULT_OVERFLOW);
    if (bad && P.status) atomicOr(P.status, SV_STATUS_BAD_PAGE);
}

template <int D, int DT, int NHT>
static cudaError_t sparse_launch_one(const CUtensorMap& km, const CUtensorMap& vm, SparseParams& P, uint64_t units, cudaStream_t st) {
    using Cfg = SparseCfg<D>;
    const uint32_t keep = P.first + P.last + P.top;
    constexpr size_t rest = 1024 + Cfg::BOXES * 8 * NHT * 128 + 8 * NHT * (D + 32) * 4 + (2 * Cfg::STAGES + 1) * 8;
    constexpr size_t ring = (size_t)Cfg::STAGES * Cfg::STAGE_BYTES, choice_most = sizeof(ChoiceTables) + 16 * (SP_CAP + 4) + 8 * SILVANN_B200_PAGED_KEEP_MAX;
    static_assert(rest + (ring > choice_most ? ring : choice_most) + 127 + SILVANN_B200_PAGED_KEEP_MAX * 4 <= 227 * 1024, "a thread block's shared memory");
    static_assert(ring >= (size_t)Cfg::PW * 8 * NHT * (D + 6) * 4, "the partials fit the ring");
    static_assert(sizeof(ChoiceTables) % 16 == 0, "the scores begin on sixteen bytes");
    const size_t choice = sizeof(ChoiceTables) + 16 * (size_t)P.cap + 8 * (size_t)P.choice_top;
    P.ring_bytes = (uint32_t)((P.top && choice > ring ? choice : ring) + 127) & ~127u;
    P.choice_at = P.top && choice < P.ring_bytes ? (uint32_t)(P.ring_bytes - choice) & ~127u : 0u;
    P.free_stages = P.choice_at / Cfg::STAGE_BYTES;
    const size_t smem = rest + P.ring_bytes + (size_t)keep * 4;
    constexpr size_t most = rest + (ring > choice_most ? ring : choice_most) + 127 + SILVANN_B200_PAGED_KEEP_MAX * 4;
    /* As many thread blocks a row as fit the card at once, as far as a row's longest list of tiles goes round.  With 1, 2, 4, 8, 16 of them:
     * 32 long rows of 2 kv heads 115, 71, 44, 56, 94 us (the rule takes 4); one row of 262,144 positions 95, 56, 34, 24, 20 (16); 120 rows of
     * 8 kv heads 64, 85, 140, 274, 619 (1). */
    const uint32_t fit = (uint32_t)(228 * 1024 / (smem + 1024)), slots = device_sm_count() * (fit < (uint32_t)Cfg::OCC ? fit : (uint32_t)Cfg::OCC);
    const uint32_t tiles = (keep * P.block + Cfg::TP - 1u) / Cfg::TP;
    uint32_t cluster = 1u;
    while (cluster < 16u && units * cluster * 2u <= slots && cluster < tiles) cluster *= 2u;
    static std::atomic<bool> attr_set[SPARSE_DEVICES];
    int d = 0; cudaGetDevice(&d);
    if (d >= 0 && d < SPARSE_DEVICES && !attr_set[d].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(paged_sparse_kernel<D, DT, NHT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_sparse_kernel<D, DT, NHT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        attr_set[d].store(true, std::memory_order_release);
    }
    cudaError_t e = cudaErrorInvalidValue;
    for (; cluster > 0; cluster /= 2) {               /* a cluster that the card cannot place goes out again half as large */
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(units * cluster)); cfg.blockDim = dim3(SP_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
        cudaLaunchAttribute at[2];
        unsigned na = 0;
        if (cluster > 1u) { at[na].id = cudaLaunchAttributeClusterDimension; at[na].val.clusterDim.x = cluster; at[na].val.clusterDim.y = 1; at[na].val.clusterDim.z = 1; ++na; }
        if (pdl_allowed()) { at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[na].val.programmaticStreamSerializationAllowed = 1; ++na; }
        cfg.attrs = at; cfg.numAttrs = na;
        e = cudaLaunchKernelEx(&cfg, paged_sparse_kernel<D, DT, NHT>, km, vm, (const SparseParams)P);
        if (e == cudaSuccess) { note_launch(1); return cudaGetLastError(); }
        (void)cudaGetLastError();
    }
    return e;
}

static cudaError_t sparse_launch(SparseParams& P, const void* k, const void* v, uint32_t rows, uint32_t d, int dtype, cudaStream_t st) {
    const uint32_t nht = P.group <= 8u ? 1u : 2u;
    P.head_blocks = (P.group + 8u * nht - 1u) / (8u * nht);
    const uint64_t units = (uint64_t)rows * P.kv_heads * P.head_blocks, cols = (uint64_t)P.kv_heads * d;
    const uint32_t tp = d == 256 ? 32u : d == 128 ? 64u : 128u;
    /* a chunk holds all the blocks a table row can name, or more than can be chosen */
    const uint64_t most = (uint64_t)P.stride * P.per.d;
    P.choice_top = (P.top + 3u) & ~3u;
    P.block_log = P.block == 16u ? 4u : P.block == 32u ? 5u : P.block == 64u ? 6u : 7u;
    P.table_blocks = (uint32_t)(most < 0x7FFFFFFFull ? most : 0x7FFFFFFFull);
    P.chunk = (uint32_t)(most < SP_CHUNK ? most : SP_CHUNK);
    if (P.chunk < P.top + 4u) P.chunk = P.top + 4u;
    P.chunk = (P.chunk + 3u) & ~3u;
    P.cap = P.chunk + P.choice_top + 8u;
    CUtensorMap km, vm;
    const bool bf = dtype == SV_DTYPE_BF16;
    const uint32_t box = P.block < tp ? P.block : tp;
    if (!make_map_2d_sw128(&km, k, cols, (uint64_t)P.pool_pages * P.page_pos, cols * 2u, 64u, box, bf) || !make_map_2d_sw128(&vm, v, cols, (uint64_t)P.pool_pages * P.page_pos, cols * 2u, 64u, box, bf))
        return cudaErrorInvalidValue;
#define SV_SPARSE_CASE(DD, TT) return nht == 1u ? sparse_launch_one<DD, TT, 1>(km, vm, P, units, st) : sparse_launch_one<DD, TT, 2>(km, vm, P, units, st)
    if (!bf) { if (d == 64) SV_SPARSE_CASE(64, SV_DTYPE_FP16); else if (d == 128) SV_SPARSE_CASE(128, SV_DTYPE_FP16); else SV_SPARSE_CASE(256, SV_DTYPE_FP16); }
    else { if (d == 64) SV_SPARSE_CASE(64, SV_DTYPE_BF16); else if (d == 128) SV_SPARSE_CASE(128, SV_DTYPE_BF16); else SV_SPARSE_CASE(256, SV_DTYPE_BF16); }
#undef SV_SPARSE_CASE
}

}  // namespace sv

static inline bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

SV_EXPORT int silvann_b200_paged_sparse(void* o, float* res, int32_t* chosen, const void* q, uint64_t q_stride, const void* k_pool, const void* v_pool,
                                        const void* k_means, const int32_t* row_seq, const int32_t* row_pos, uint32_t rows, const int32_t* page_table,
                                        uint32_t seqs, uint32_t table_stride, uint64_t pool_pages, uint32_t page_positions, uint32_t block_positions,
                                        uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t first, uint32_t last, uint32_t top, int dtype,
                                        sv_fault* over, void* stream) {
    svf::g_counters[SILVANN_B200_COUNTER_EXT_CALLS].fetch_add(1, std::memory_order_relaxed);
    if ((!o && !res) || !q || !k_pool || !v_pool || (top && !k_means) || !row_seq || !row_pos || !page_table) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: a null operand");
    if (dtype != SILVANN_B200_DTYPE_FP16 && dtype != SILVANN_B200_DTYPE_BF16) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: dtype %d", dtype);
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: head_dim %u (64, 128 or 256)", head_dim);
    if (kv_heads == 0 || kv_heads > 4096u || q_heads == 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > 64u)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: %u query heads over %u kv heads (up to 64 each)", q_heads, kv_heads);
    if (rows == 0 || rows > (1u << 24) / kv_heads || seqs == 0 || table_stride == 0) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: %u rows, %u sequences of %u table columns", rows, seqs, table_stride);
    if (pool_pages == 0 || page_positions == 0 || pool_pages > 0x7FFFFFFFull / page_positions)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: pool of %llu pages of %u positions", (unsigned long long)pool_pages, page_positions);
    if ((block_positions != 16 && block_positions != 32 && block_positions != 64 && block_positions != 128) || page_positions % block_positions)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: blocks of %u positions (16, 32, 64 or 128) in pages of %u", block_positions, page_positions);
    if (last == 0 || (uint64_t)first + last + top > SILVANN_B200_PAGED_KEEP_MAX)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: first %u, last %u (at least 1), top %u: at most %u blocks a row", first, last, top, SILVANN_B200_PAGED_KEEP_MAX);
    const uint64_t q_row = (uint64_t)q_heads * head_dim;
    if (q_stride == 0) q_stride = q_row;
    if (q_stride < q_row || q_stride % 8u) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: rows of q %llu elements apart (a multiple of 8, at least %llu)", (unsigned long long)q_stride, (unsigned long long)q_row);
    if (!aligned(q, 16) || !aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(k_means, 16) || !aligned(o, 2) || !aligned(res, 4) || !aligned(chosen, 4) || !aligned(row_seq, 4) || !aligned(row_pos, 4) || !aligned(page_table, 4))
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: an operand's alignment is outside the kernel's fit");
    sv::SparseParams P;
    memset(&P, 0, sizeof P);
    P.o = o; P.res = res; P.chosen = chosen; P.q = (const uint16_t*)q; P.means = (const uint16_t*)k_means;
    P.row_seq = row_seq; P.row_pos = row_pos; P.table = page_table; P.over = over; P.status = sv::device_status_word(); P.q_stride = q_stride; P.seqs = seqs;
    P.stride = table_stride; P.pool_pages = (uint32_t)pool_pages; P.page_pos = page_positions; P.block = block_positions; P.per = sv::paged_div(page_positions / block_positions); P.q_heads = q_heads; P.kv_heads = kv_heads;
    P.group = q_heads / kv_heads; P.first = first; P.last = last; P.top = top; P.o_wide = aligned(o, 8); P.scale_log2 = (1.0f / sqrtf((float)head_dim)) * SV_LOG2E;
    cudaError_t e = sv::sparse_launch(P, k_pool, v_pool, rows, head_dim, dtype, (cudaStream_t)stream);
    if (e == cudaSuccess) return SILVANN_B200_OK;
    (void)cudaGetLastError();
    return sv_ext_fail(SILVANN_B200_E_CUDA, "paged_sparse: launch: %s", cudaGetErrorString(e));
}
