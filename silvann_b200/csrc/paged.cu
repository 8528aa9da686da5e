/* paged.cu — a serving step's tables built on the card, and the rows' way into the paged pool with the blocks' mean keys
 * (declared in include/silvann_b200.h). */
#include "../../include/silvann_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "paged_index.h"
#include <atomic>
#include <string.h>

#define SV_EXPORT extern "C" __attribute__((visibility("default")))

int sv_ext_fail(int code, const char* fmt, ...);      /* ext.cu: records the message for silvann_b200_last_error */
namespace svf { extern std::atomic<uint64_t> g_counters[SILVANN_B200_COUNTERS]; }
static inline void called() { svf::g_counters[SILVANN_B200_COUNTER_EXT_CALLS].fetch_add(1, std::memory_order_relaxed); }

namespace sv {

/* ---------------------------------------------------------------------------------------------------------- */
/* the step's tables                                                                                            */

#define SV_TABLES_THREADS 1024        /* of a thread block of a cluster; half of them where there is one block */
#define SV_TABLES_CLUSTER 8u
static constexpr int TABLES_DEVICES = 64;

struct TablesParams {
    int32_t *new_lens, *table, *row_start, *row_seq, *row_pos, *row_slot;
    uint32_t* free_out;
    int32_t* free_pages;
    const uint32_t* free_at;
    const int32_t *lens, *counts;
    unsigned int* status;
    PagedDiv page;                      /* positions a page */
    uint64_t most;                      /* positions a table row has pages for */
    uint32_t seqs, stride, rows, free_total, pool_pages;
};

/* What one sequence brings to the three sums: new positions, pages it takes, pages it gives back. */
struct TablesItem { uint32_t rows, need, back; bool bad; };
__device__ __forceinline__ uint32_t tables_pages(const TablesParams& P, uint32_t n) { return n ? paged_quot(n - 1u, P.page) + 1u : 0u; }
__device__ __forceinline__ TablesItem tables_item(const TablesParams& P, int32_t len, int32_t count) {
    TablesItem it = {0u, 0u, 0u, false};
    const uint32_t come = count > 0 ? (uint32_t)count : 0u;
    if (len < 0 || count < SILVANN_B200_PAGED_ENDED || (uint64_t)len + come > P.most || (uint64_t)len + come > 0x7FFFFFFFull) { it.bad = true; return it; }
    const uint32_t held = tables_pages(P, (uint32_t)len);
    if (count < 0) it.back = held;
    else { it.rows = come; it.need = tables_pages(P, (uint32_t)len + come) - held; }
    return it;
}
/* Sums stop at 2^32 - 1, beyond every size they are compared with. */
__device__ __forceinline__ uint32_t tables_add(uint32_t a, uint32_t b) { const uint32_t c = a + b; return c < a ? 0xFFFFFFFFu : c; }

/* The sequences that N items of a list belong to, each looked for among `n` from `lo` on: the last s with start[s] <= item among those
 * that have items.  The N searches go hand in hand. */
template <int N>
__device__ __forceinline__ void tables_owners(const uint32_t* start, uint32_t lo, uint32_t n, const uint32_t (&item)[N], uint32_t (&s)[N]) {
#pragma unroll
    for (int u = 0; u < N; ++u) s[u] = lo;
    while (n > 1u) {
        const uint32_t half = n >> 1;
#pragma unroll
        for (int u = 0; u < N; ++u) if (start[s[u] + half] <= item[u]) s[u] += half;
        n -= half;
    }
}
__device__ __forceinline__ uint32_t tables_owner(const uint32_t* start, uint32_t lo, uint32_t n, uint32_t item) {
    const uint32_t i[1] = {item};
    uint32_t s[1];
    tables_owners<1>(start, lo, n, i, s);
    return s[0];
}

/* New positions, U of them a lane: a warp takes 32 U neighbouring ones, whose sequences lie between those of its first and its last. */
template <int U>
__device__ __forceinline__ bool tables_rows(const TablesParams& P, const uint32_t* rows_s, const uint32_t* need_s, const int32_t* len_s, uint32_t n_rows, uint32_t bottom,
                                            uint32_t g_tid, uint32_t g_all) {
    const uint32_t lane = g_tid & 31u;
    bool strange = false;
    for (uint32_t r0 = (g_tid & ~31u) * U; r0 < P.rows; r0 += g_all * U) {
        uint32_t s_lo = 0u, span = 1u;
        if (r0 < n_rows) {
            const uint32_t ends[2] = {r0, min(r0 + 32u * U, n_rows) - 1u};
            uint32_t s[2];
            tables_owners<2>(rows_s, 0u, P.seqs, ends, s);
            s_lo = s[0]; span = s[1] - s[0] + 1u;
        }
        uint32_t row[U], s[U], off[U];
        int32_t pos[U], page[U];
#pragma unroll
        for (int u = 0; u < U; ++u) row[u] = r0 + u * 32u + lane;
        tables_owners<U>(rows_s, s_lo, span, row, s);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            page[u] = -1; off[u] = 0u; pos[u] = -1;
            if (row[u] < n_rows) {
                const uint32_t len = (uint32_t)len_s[s[u]], p = len + (row[u] - rows_s[s[u]]), col = paged_quot(p, P.page), held = tables_pages(P, len);
                pos[u] = (int32_t)p; off[u] = p - col * P.page.d;
                /* a page taken in this step is read from the stack, where it came from */
                page[u] = col < held ? P.table[(size_t)s[u] * P.stride + col] : __ldcg(P.free_pages + bottom + need_s[s[u]] + (col - held));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row[u] < P.rows) {
                const bool there = row[u] < n_rows, good = page[u] >= 0 && (uint32_t)page[u] < P.pool_pages;
                strange |= there && !good;
                P.row_seq[row[u]] = there ? (int32_t)s[u] : -1; P.row_pos[row[u]] = pos[u]; P.row_slot[row[u]] = good ? (int32_t)((uint32_t)page[u] * P.page.d + off[u]) : -1;
            }
    }
    return strange;
}

/* Every thread block of the one cluster makes the exclusive sums of (rows, need, back) over all sequences for itself, in its own shared
 * memory: the step is decided (it fits or is refused) before anything is written, without an exchange.  Then three flat lists — pages
 * that come back, pages handed out, new positions — are walked by all threads of the cluster.  One barrier of the cluster stands between
 * what reads the caller's arrays and what may write them in place, and between the pages that come back and those handed out.
 * What bounds it: latency.  A step is a handful of dependent reads and searches long (one new position each of 32 sequences: 2.8 us in a
 * graph; of 4,097, some ending: 9.4 us); the cluster is there for the steps that bring many positions (98 thousand from 61 prompts:
 * 11.2 us, 81 us on one thread block). */
__global__ void __launch_bounds__(SV_TABLES_THREADS, 1) paged_tables_kernel(const TablesParams P) {
    extern __shared__ uint32_t tsm[];
    uint32_t* rows_s = tsm;                       /* [seqs + 1] each */
    uint32_t* need_s = rows_s + P.seqs + 1;
    uint32_t* back_s = need_s + P.seqs + 1;
    int32_t* len_s = (int32_t*)(back_s + P.seqs + 1);
    __shared__ uint32_t warp_sum[3][SV_TABLES_THREADS / 32];
    const uint32_t threads = blockDim.x, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    const uint32_t CL = cluster_nctarank(), g_tid = cluster_ctarank() * threads + tid, g_all = CL * threads;
    const uint32_t per = (P.seqs + threads - 1u) / threads;
    const uint32_t i0 = min(P.seqs, tid * per), i1 = min(P.seqs, i0 + per);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t at = *P.free_at;

    uint32_t sum[3] = {0u, 0u, 0u};
    bool bad = false;
#pragma unroll 4
    for (uint32_t s = tid; s < P.seqs; s += threads) { len_s[s] = P.lens[s]; rows_s[s] = (uint32_t)P.counts[s]; }
    __syncthreads();
    for (uint32_t s = i0; s < i1; ++s) {
        const TablesItem it = tables_item(P, len_s[s], (int32_t)rows_s[s]);
        rows_s[s] = sum[0]; need_s[s] = sum[1]; back_s[s] = sum[2];                     /* up to here within this thread */
        sum[0] = tables_add(sum[0], it.rows); sum[1] = tables_add(sum[1], it.need); sum[2] = tables_add(sum[2], it.back); bad |= it.bad;
    }
    uint32_t before[3], all[3];
#pragma unroll
    for (int x = 0; x < 3; ++x) {
        uint32_t v = sum[x];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const uint32_t o = __shfl_up_sync(0xffffffffu, v, d); if (lane >= d) v = tables_add(v, o); }
        if (lane == 31u) warp_sum[x][warp] = v;
        before[x] = __shfl_up_sync(0xffffffffu, v, 1);
        if (lane == 0u) before[x] = 0u;
    }
    bad = __syncthreads_or(bad);
    /* every warp sums the warps' totals for itself */
#pragma unroll
    for (int x = 0; x < 3; ++x) {
        uint32_t v = lane < threads / 32u ? warp_sum[x][lane] : 0u;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const uint32_t o = __shfl_up_sync(0xffffffffu, v, d); if (lane >= d) v = tables_add(v, o); }
        const uint32_t ahead = __shfl_sync(0xffffffffu, v, (warp + 31u) & 31u);
        if (warp) before[x] = tables_add(before[x], ahead);
        all[x] = __shfl_sync(0xffffffffu, v, 31);
    }
    const bool bad_step = bad || all[0] > P.rows || at > P.free_total || all[2] > at;
    const bool no_pages = !bad_step && all[1] > P.free_total - (at - all[2]);

    if (bad_step || no_pages) {
        __syncthreads();
        if (CL > 1) cluster_sync_all();
        if (g_tid == 0) {
            if (P.status) atomicOr(P.status, bad_step ? SV_STATUS_BAD_STEP : SV_STATUS_NO_PAGES);
            *P.free_out = at;
        }
        for (uint32_t s = g_tid; s <= P.seqs; s += g_all) { if (s < P.seqs) P.new_lens[s] = len_s[s]; P.row_start[s] = 0; }
        for (uint32_t r = g_tid; r < P.rows; r += g_all) { P.row_seq[r] = -1; P.row_pos[r] = -1; P.row_slot[r] = -1; }
        return;
    }
    for (uint32_t s = i0; s < i1; ++s) { rows_s[s] += before[0]; need_s[s] += before[1]; back_s[s] += before[2]; }
    if (tid == 0) { rows_s[P.seqs] = all[0]; need_s[P.seqs] = all[1]; back_s[P.seqs] = all[2]; }
    __syncthreads();
    const uint32_t n_rows = all[0], n_need = all[1], n_back = all[2], bottom = at - n_back;
    bool strange = false;                          /* an entry that names no page of the pool */

    for (uint32_t j = g_tid; j < n_back; j += g_all) {
        const uint32_t s = tables_owner(back_s, 0u, P.seqs, j);
        const int32_t page = P.table[(size_t)s * P.stride + (j - back_s[s])];
        strange |= page < 0 || (uint32_t)page >= P.pool_pages;
        P.free_pages[bottom + j] = page;
    }
    if (CL > 1) cluster_sync_all(); else __syncthreads();
    for (uint32_t s = g_tid; s <= P.seqs; s += g_all) {
        P.row_start[s] = (int32_t)rows_s[s];
        if (s < P.seqs) P.new_lens[s] = back_s[s + 1] > back_s[s] ? 0 : len_s[s] + (int32_t)(rows_s[s + 1] - rows_s[s]);
    }
    if (g_tid == 0) *P.free_out = bottom + n_need;
    for (uint32_t j = g_tid; j < n_need; j += g_all) {
        const uint32_t s = tables_owner(need_s, 0u, P.seqs, j);
        const int32_t page = __ldcg(P.free_pages + bottom + j);
        strange |= page < 0 || (uint32_t)page >= P.pool_pages;
        P.table[(size_t)s * P.stride + tables_pages(P, (uint32_t)len_s[s]) + (j - need_s[s])] = page;
    }
    strange |= P.rows <= g_all ? tables_rows<1>(P, rows_s, need_s, len_s, n_rows, bottom, g_tid, g_all) : tables_rows<4>(P, rows_s, need_s, len_s, n_rows, bottom, g_tid, g_all);
    if (strange && P.status) atomicOr(P.status, SV_STATUS_BAD_PAGE);
}

static cudaError_t tables_launch(const TablesParams& P, cudaStream_t st) {
    const size_t smem = (size_t)4 * (P.seqs + 1) * sizeof(uint32_t);
    static std::atomic<bool> attr_set[TABLES_DEVICES];
    int d = 0; cudaGetDevice(&d);
    if (d >= 0 && d < TABLES_DEVICES && !attr_set[d].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(paged_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((size_t)4 * (SILVANN_B200_PAGED_SEQS_MAX + 1) * sizeof(uint32_t)));
        if (e != cudaSuccess) return e;
        attr_set[d].store(true, std::memory_order_release);
    }
    /* one thread block takes four rows a thread in a round; a cluster where there are more */
    const uint32_t cluster = P.rows <= 2u * SV_TABLES_THREADS ? 1u : SV_TABLES_CLUSTER;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster); cfg.blockDim = dim3(cluster > 1u ? SV_TABLES_THREADS : SV_TABLES_THREADS / 2); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    unsigned na = 0;
    if (cluster > 1u) { attr[na].id = cudaLaunchAttributeClusterDimension; attr[na].val.clusterDim.x = cluster; attr[na].val.clusterDim.y = 1; attr[na].val.clusterDim.z = 1; ++na; }
    if (pdl_allowed()) { attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[na].val.programmaticStreamSerializationAllowed = 1; ++na; }
    cfg.attrs = attr; cfg.numAttrs = na;
    cudaError_t e = cudaLaunchKernelEx(&cfg, paged_tables_kernel, P);
    if (e != cudaSuccess) return e;
    note_launch(1);
    return cudaGetLastError();
}

/* ---------------------------------------------------------------------------------------------------------- */
/* rows into the pool                                                                                           */

#define SV_WRITE_THREADS 256

struct WriteParams {
    uint4 *k_pool, *v_pool, *means;
    const uint4 *k_rows, *v_rows;
    const int32_t* slots;
    unsigned int* status;
    uint64_t k_stride, v_stride;        /* in uint4 */
    uint32_t rows, row_vec, pool_slots, block, block_log, run, runs_block;
};
#define SV_WRITE_RUN 8u             /* rows a thread copies, at most */
#define SV_WRITE_GROUP 16u          /* rows of a block that one thread sums */

template <int DT>
__device__ __forceinline__ void write_add(float (&sum)[8], const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) { const float2 f = Elem<DT>::unpack2(w[u]); sum[2 * u] += f.x; sum[2 * u + 1] += f.y; }
}

/* A thread copies 16 bytes of up to eight neighbouring rows, keys and values, all asked for at once.  Then the thread block takes the
 * blocks that its rows complete, one after the other: sixteen rows a thread, again all asked for at once (this call's rows, which the
 * caches still hold, or earlier ones in the pool), and the sixteens added up in order through shared memory — so a mean is the
 * same sum however its rows came, and no thread's way is longer than two such trips for each.
 * What bounds it: memory.  73,600 rows of 1 KB, keys and values: 58.5 us, 5.3 TB/s of rows read and written, 48.5 without means.
 * Measured against: a thread a column for runs of 64 rows that sums as it goes (98 us, the longest thread's way), and a block's
 * 64 rows summed again by the threads of its last row (119 us). */
template <int DT>
__global__ void __launch_bounds__(SV_WRITE_THREADS) paged_write_kernel(const WriteParams P) {
    using E = Elem<DT>;
    __shared__ uint32_t done[SV_WRITE_THREADS];
    __shared__ uint32_t n_done;
    __shared__ float4 part_sum[SV_WRITE_THREADS][2];
    const uint32_t tid = threadIdx.x, wide = min(P.row_vec, (uint32_t)SV_WRITE_THREADS), part = tid / wide;
    const uint32_t mask = P.block - 1u;
    if (tid == 0) n_done = 0u;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t per = P.runs_block * P.run, r0 = blockIdx.x * per, r1 = min(P.rows, r0 + per);      /* (the launch keeps their product in 32 bits) */
    bool bad = false;
    if (part < P.runs_block) {
        const uint32_t a0 = r0 + part * P.run, a1 = min(r1, a0 + P.run);
        for (uint32_t i = tid % wide; i < P.row_vec; i += SV_WRITE_THREADS) {
            int32_t slot[SV_WRITE_RUN];
            uint4 k[SV_WRITE_RUN], v[SV_WRITE_RUN];
#pragma unroll
            for (uint32_t u = 0; u < SV_WRITE_RUN; ++u) slot[u] = a0 + u < a1 ? P.slots[a0 + u] : -1;
#pragma unroll
            for (uint32_t u = 0; u < SV_WRITE_RUN; ++u) {
                if (slot[u] >= 0 && (uint32_t)slot[u] >= P.pool_slots) { bad = true; slot[u] = -1; }
                if (slot[u] >= 0) { k[u] = P.k_rows[(uint64_t)(a0 + u) * P.k_stride + i]; v[u] = P.v_rows[(uint64_t)(a0 + u) * P.v_stride + i]; }
            }
#pragma unroll
            for (uint32_t u = 0; u < SV_WRITE_RUN; ++u)
                if (slot[u] >= 0) { P.k_pool[(size_t)slot[u] * P.row_vec + i] = k[u]; P.v_pool[(size_t)slot[u] * P.row_vec + i] = v[u]; }
        }
    }
    if (bad && P.status) atomicOr(P.status, SV_STATUS_BAD_PAGE);
    if (!P.block) return;
    for (uint32_t base = r0; base < r1; base += SV_WRITE_THREADS) {
        __syncthreads();
        if (base + tid < r1) {
            const int32_t s = P.slots[base + tid];
            if (s >= 0 && (uint32_t)s < P.pool_slots && ((uint32_t)s & mask) == mask) done[atomicAdd(&n_done, 1u)] = base + tid;
        }
        __syncthreads();
        const uint32_t groups = P.block / SV_WRITE_GROUP, cols = SV_WRITE_THREADS / groups, g = tid / cols, c = tid - g * cols;
        const float inv = 1.0f / (float)P.block;
        const uint32_t n = n_done;
        for (uint32_t x = 0; x < n; ++x) {
            const uint32_t at = done[x];
            const int32_t s = P.slots[at];
            for (uint32_t i0 = 0; i0 < P.row_vec; i0 += cols) {
                const uint32_t i = i0 + c;
                float sum[8] = {};
                if (i < P.row_vec) {
                    uint4 k[SV_WRITE_GROUP];
#pragma unroll
                    for (uint32_t b = 0; b < SV_WRITE_GROUP; ++b) {
                        const uint32_t back = mask - (g * SV_WRITE_GROUP + b);
                        const bool here = back <= at && P.slots[at - min(back, at)] == s - (int32_t)back;
                        k[b] = here ? P.k_rows[(uint64_t)(at - back) * P.k_stride + i] : P.k_pool[(size_t)(s - (int32_t)back) * P.row_vec + i];
                    }
#pragma unroll
                    for (uint32_t b = 0; b < SV_WRITE_GROUP; ++b) write_add<DT>(sum, k[b]);
                }
                part_sum[tid][0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
                part_sum[tid][1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
                __syncthreads();
                if (g == 0u && i < P.row_vec) {
                    for (uint32_t y = 1; y < groups; ++y) {
                        const float4 lo = part_sum[y * cols + c][0], hi = part_sum[y * cols + c][1];
                        sum[0] += lo.x; sum[1] += lo.y; sum[2] += lo.z; sum[3] += lo.w; sum[4] += hi.x; sum[5] += hi.y; sum[6] += hi.z; sum[7] += hi.w;
                    }
                    P.means[(size_t)((uint32_t)s >> P.block_log) * P.row_vec + i] =
                        make_uint4(E::pack2(sum[0] * inv, sum[1] * inv), E::pack2(sum[2] * inv, sum[3] * inv), E::pack2(sum[4] * inv, sum[5] * inv), E::pack2(sum[6] * inv, sum[7] * inv));
                }
                __syncthreads();
            }
        }
        if (tid == 0) n_done = 0u;
    }
}

static cudaError_t write_launch(WriteParams& P, int dtype, cudaStream_t st) {
    const uint32_t wide = P.row_vec < SV_WRITE_THREADS ? P.row_vec : SV_WRITE_THREADS;
    P.runs_block = SV_WRITE_THREADS / wide;
    P.block_log = 0u;
    while (P.block_log < 7u && (1u << P.block_log) < P.block) ++P.block_log;
    /* eight rows a thread once that leaves every SM a thread block; fewer, down to one, below (8,033 rows of 1 KB: 11.4 us with eight
     * rows a thread, 12.7 with four, 17 with two; 73,600 rows: 59, 72, 109) */
    P.run = SV_WRITE_RUN;
    while (P.run > 1u && (uint64_t)P.rows * wide < (uint64_t)device_sm_count() * SV_WRITE_THREADS * P.run) P.run /= 2u;
    const uint64_t per = (uint64_t)P.runs_block * P.run, blocks = (P.rows + per - 1u) / per;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks); cfg.blockDim = dim3(SV_WRITE_THREADS); cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = pdl_allowed() ? 1u : 0u;
    cudaError_t e = dtype == SV_DTYPE_FP16 ? cudaLaunchKernelEx(&cfg, paged_write_kernel<SV_DTYPE_FP16>, (const WriteParams)P) : cudaLaunchKernelEx(&cfg, paged_write_kernel<SV_DTYPE_BF16>, (const WriteParams)P);
    if (e != cudaSuccess) return e;
    note_launch(1);
    return cudaGetLastError();
}

}  // namespace sv

static inline bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
static int cuda_fail(const char* what, cudaError_t e) {
    (void)cudaGetLastError();
    return sv_ext_fail(SILVANN_B200_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

SV_EXPORT int silvann_b200_paged_tables(int32_t* new_lens, int32_t* page_table, int32_t* row_start, int32_t* row_seq, int32_t* row_pos, int32_t* row_slot,
                                        uint32_t* free_out, int32_t* free_pages, const uint32_t* free_at, const int32_t* lens, const int32_t* counts,
                                        uint32_t seqs, uint32_t table_stride, uint32_t rows, uint32_t free_total, uint64_t pool_pages,
                                        uint32_t page_positions, void* stream) {
    called();
    const void* all[] = {new_lens, page_table, row_start, row_seq, row_pos, row_slot, free_out, free_pages, free_at, lens, counts};
    for (const void* p : all) if (!p || !aligned(p, 4)) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_tables: an operand is null or not 4-byte aligned");
    if (seqs == 0 || seqs > SILVANN_B200_PAGED_SEQS_MAX) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_tables: %u sequences (1 to %u)", seqs, SILVANN_B200_PAGED_SEQS_MAX);
    if (table_stride == 0 || rows == 0 || rows > 0x7FFFFFFFu || free_total == 0 || free_total > 0x7FFFFFFFu)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_tables: %u table columns, %u rows, a stack of %u pages", table_stride, rows, free_total);
    if (pool_pages == 0 || page_positions == 0 || pool_pages > 0x7FFFFFFFull / page_positions)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_tables: pool of %llu pages of %u positions", (unsigned long long)pool_pages, page_positions);
    sv::TablesParams P;
    P.new_lens = new_lens; P.table = page_table; P.row_start = row_start; P.row_seq = row_seq; P.row_pos = row_pos; P.row_slot = row_slot;
    P.free_out = free_out; P.free_pages = free_pages; P.free_at = free_at; P.lens = lens; P.counts = counts; P.status = sv::device_status_word();
    P.seqs = seqs; P.stride = table_stride; P.rows = rows; P.free_total = free_total; P.pool_pages = (uint32_t)pool_pages; P.page = sv::paged_div(page_positions);
    P.most = (uint64_t)table_stride * page_positions;
    cudaError_t e = sv::tables_launch(P, (cudaStream_t)stream);
    return e == cudaSuccess ? SILVANN_B200_OK : cuda_fail("paged_tables: launch", e);
}

SV_EXPORT int silvann_b200_paged_write(void* k_pool, void* v_pool, void* k_means, const void* k_rows, const void* v_rows, uint64_t k_stride,
                                       uint64_t v_stride, const int32_t* row_slot, uint32_t rows, uint32_t kv_heads, uint32_t head_dim,
                                       uint64_t pool_pages, uint32_t page_positions, uint32_t block_positions, int dtype, void* stream) {
    called();
    if (!k_pool || !v_pool || !k_rows || !v_rows || !row_slot || (block_positions && !k_means)) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_write: a null operand");
    if (dtype != SILVANN_B200_DTYPE_FP16 && dtype != SILVANN_B200_DTYPE_BF16) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_write: dtype %d", dtype);
    const uint64_t row = (uint64_t)kv_heads * head_dim;
    if (k_stride == 0) k_stride = row;
    if (v_stride == 0) v_stride = row;
    if (rows == 0 || rows > 0x7FFFFFFFu || row == 0 || row > (1ull << 20) || row % 8u || k_stride % 8u || v_stride % 8u || k_stride < row || v_stride < row)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_write: %u rows of %u x %u elements, %llu and %llu apart (multiples of 8)", rows, kv_heads, head_dim, (unsigned long long)k_stride, (unsigned long long)v_stride);
    if (pool_pages == 0 || page_positions == 0 || pool_pages > 0x7FFFFFFFull / page_positions)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_write: pool of %llu pages of %u positions", (unsigned long long)pool_pages, page_positions);
    if (block_positions && ((block_positions != 16 && block_positions != 32 && block_positions != 64 && block_positions != 128) || page_positions % block_positions))
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_write: blocks of %u positions (16, 32, 64 or 128) in pages of %u", block_positions, page_positions);
    if (!aligned(k_pool, 16) || !aligned(v_pool, 16) || !aligned(k_rows, 16) || !aligned(v_rows, 16) || !aligned(row_slot, 4) || (block_positions && !aligned(k_means, 16)))
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_write: rows, pools and means must be 16-byte aligned");
    sv::WriteParams P;
    P.k_pool = (uint4*)k_pool; P.v_pool = (uint4*)v_pool; P.means = (uint4*)k_means; P.k_rows = (const uint4*)k_rows; P.v_rows = (const uint4*)v_rows;
    P.slots = row_slot; P.status = sv::device_status_word(); P.k_stride = k_stride / 8u; P.v_stride = v_stride / 8u; P.rows = rows; P.row_vec = (uint32_t)(row / 8u);
    P.pool_slots = (uint32_t)(pool_pages * page_positions); P.block = block_positions;
    cudaError_t e = sv::write_launch(P, dtype, (cudaStream_t)stream);
    return e == cudaSuccess ? SILVANN_B200_OK : cuda_fail("paged_write: launch", e);
}
