/* sparse.cu — attention of new positions over the blocks of the paged pool that a cheap score selects
 * (silvann_b200_paged_sparse, include/silvann_b200.h). */
#include "../../include/silvann_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "paged_index.h"
#include <atomic>
#include <math.h>
#include <string.h>

#define SV_EXPORT extern "C" __attribute__((visibility("default")))

int sv_ext_fail(int code, const char* fmt, ...);      /* ext.cu: records the message for silvann_b200_last_error */
namespace svf { extern std::atomic<uint64_t> g_counters[SILVANN_B200_COUNTERS]; }

namespace sv {

static constexpr int SPARSE_DEVICES = 64;
#define SP_THREADS 256
#define SP_CHUNK 2048u      /* scores looked at in one go; the best of the chunks before them ride along */

struct SparseParams {
    void* o;
    float* res;
    int32_t* chosen;
    const uint16_t *q, *k, *v, *means;
    const int32_t *row_seq, *row_pos, *table;
    unsigned int *over, *status;
    uint64_t q_stride;
    uint32_t seqs, stride, pool_pages, page_pos, block, q_heads, kv_heads, group, first, last, top;
    float scale;
};

/* Orders as the score does, NaN with minus infinity. */
__device__ __forceinline__ unsigned long long score_key(double s) {
    if (!(s == s)) s = -INFINITY;
    const unsigned long long b = (unsigned long long)__double_as_longlong(s + 0.0);       /* -0 + 0 = +0: equal scores, equal keys */
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

/* The `take` greatest of keys[0..m) (equal keys: the lower index), their indexes ascending into out; m > take > 0. */
__device__ void select_keys(const unsigned long long* keys, uint32_t m, uint32_t take, uint32_t* out, uint32_t* hist /*[256 + 4]*/, uint32_t* warp_n /*[2][8]*/) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned long long known = 0, cut = 0;
    uint32_t need = take;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += SP_THREADS) hist[i] = 0u;
        __syncthreads();
        for (uint32_t i = tid; i < m; i += SP_THREADS)
            if ((keys[i] & known) == cut) atomicAdd(&hist[(uint32_t)(keys[i] >> shift) & 255u], 1u);
        __syncthreads();
        if (tid == 0) {
            uint32_t covered = 0u;
            int b = 255;
            for (; b > 0; --b) { if (covered + hist[b] >= need) break; covered += hist[b]; }
            hist[256] = (uint32_t)b; hist[257] = need - covered;
        }
        __syncthreads();
        cut |= (unsigned long long)hist[256] << shift; need = hist[257]; known |= 255ull << shift;
        __syncthreads();
    }
    /* every key above the cut and the first `need` that equal it, in index order */
    uint32_t done = 0u, ties = 0u;
    for (uint32_t base = 0; base < m; base += SP_THREADS) {
        const uint32_t i = base + tid;
        const bool above = i < m && keys[i] > cut, equal = i < m && keys[i] == cut;
        const unsigned eb = __ballot_sync(0xffffffffu, equal);
        if (lane == 0) warp_n[warp] = __popc(eb);
        __syncthreads();
        uint32_t e = ties + __popc(eb & ((1u << lane) - 1u)), e_all = 0u;
        for (int w = 0; w < SP_THREADS / 32; ++w) { if (w < warp) e += warp_n[w]; e_all += warp_n[w]; }
        const bool in = above || (equal && e < need);
        const unsigned ib = __ballot_sync(0xffffffffu, in);
        if (lane == 0) warp_n[8 + warp] = __popc(ib);
        __syncthreads();
        uint32_t at = done + __popc(ib & ((1u << lane) - 1u)), n_all = 0u;
        for (int w = 0; w < SP_THREADS / 32; ++w) { if (w < warp) at += warp_n[8 + w]; n_all += warp_n[8 + w]; }
        if (in) out[at] = i;
        done += n_all; ties += e_all;
        __syncthreads();
    }
}

template <int DT>
__global__ void __launch_bounds__(SP_THREADS) paged_sparse_kernel(const SparseParams P, const int D) {
    using E = Elem<DT>;
    extern __shared__ __align__(16) uint8_t sp_smem[];
    const uint32_t kvh = blockIdx.x, r = blockIdx.y, keep = P.first + P.last + P.top;
    double* qsum = (double*)sp_smem;                                             /* [D] */
    unsigned long long* keys = (unsigned long long*)(qsum + D);                  /* [SP_CHUNK + top] */
    uint32_t* key_id = (uint32_t*)(keys + SP_CHUNK + P.top);                      /* [SP_CHUNK + top] */
    uint32_t* picked = key_id + SP_CHUNK + P.top;                                 /* [top] */
    int32_t* ids = (int32_t*)(picked + P.top);                                    /* [keep] */
    float* acc = (float*)(ids + keep);                                           /* [group][D] */
    float* w = acc + P.group * D;                                                /* [group][16] */
    float* ml = w + P.group * 16;                                                /* [group][3]: m, l, factor */
    __shared__ uint32_t hist[260], warp_n[16];
    __shared__ double part[SP_THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t seq = P.row_seq[r];
    if (seq < 0 || (uint32_t)seq >= P.seqs) { if (seq >= 0 && tid == 0 && P.status) atomicOr(P.status, SV_STATUS_BAD_PAGE); return; }
    const int32_t p = P.row_pos[r];
    const int32_t* row = P.table + (size_t)seq * P.stride;
    const uint16_t* q = P.q + (size_t)r * P.q_stride + (size_t)kvh * P.group * D;
    const size_t head0 = (size_t)r * P.q_heads + kvh * P.group;
    int32_t* chosen = P.chosen ? P.chosen + ((size_t)r * P.kv_heads + kvh) * keep : nullptr;
    if (p < 0) {
        for (uint32_t i = tid; i < P.group * D; i += SP_THREADS) {
            if (P.o) ((uint16_t*)P.o)[head0 * D + i] = 0;
            if (P.res) { float* x = P.res + (head0 + i / D) * (D + 2); x[2 + i % D] = 0.f; if (i % D == 0) { x[0] = -INFINITY; x[1] = 0.f; } }
        }
        if (chosen) for (uint32_t i = tid; i < keep; i += SP_THREADS) chosen[i] = -1;
        return;
    }
    const PagedChoice c = paged_choice((uint32_t)p, P.block, P.first, P.last, P.top);
    bool bad = false;
    for (int e = tid; e < D; e += SP_THREADS) {
        double s = 0;
        for (uint32_t h = 0; h < P.group; ++h) s += (double)E::to_float(q[h * D + e]);
        qsum[e] = s;
    }
    __syncthreads();
    uint32_t have = 0;                                                    /* the best so far, at the front of keys */
    for (uint32_t base = c.lo; base < c.hi && c.take; base += SP_CHUNK) {
        const uint32_t n = min(SP_CHUNK, c.hi - base);
        for (uint32_t i = warp; i < n; i += SP_THREADS / 32) {
            const int32_t slot = paged_block_slot(row, P.stride, P.pool_pages, P.page_pos, P.block, base + i);
            double s = 0;
            if (slot >= 0) {
                const uint16_t* m = P.means + ((size_t)((uint32_t)slot / P.block) * P.kv_heads + kvh) * D;
                for (int e = lane; e < D; e += 32) s += qsum[e] * (double)E::to_float(m[e]);
                for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            } else { s = -INFINITY; bad = true; }
            if (lane == 0) { keys[have + i] = score_key(s); key_id[have + i] = base + i; }
        }
        __syncthreads();
        const uint32_t m = have + n;
        if (m <= c.take) { have = m; continue; }
        select_keys(keys, m, c.take, picked, hist, warp_n);
        __syncthreads();
        unsigned long long kk[4]; uint32_t ii[4];
        for (uint32_t i = tid, u = 0; i < c.take; i += SP_THREADS, ++u) { kk[u] = keys[picked[i]]; ii[u] = key_id[picked[i]]; }
        __syncthreads();
        for (uint32_t i = tid, u = 0; i < c.take; i += SP_THREADS, ++u) { keys[i] = kk[u]; key_id[i] = ii[u]; }
        __syncthreads();
        have = c.take;
    }
    for (uint32_t i = tid; i < keep; i += SP_THREADS) {
        int32_t id = -1;
        if (i < c.count) id = i < c.lo ? (int32_t)i : i < c.lo + c.take ? (int32_t)key_id[i - c.lo] : (int32_t)(c.hi + (i - c.lo - c.take));
        ids[i] = id;
        if (chosen) chosen[i] = id;
    }
    for (uint32_t i = tid; i < P.group * D; i += SP_THREADS) acc[i] = 0.f;
    for (uint32_t h = tid; h < P.group; h += SP_THREADS) { ml[3 * h] = -INFINITY; ml[3 * h + 1] = 0.f; }
    __syncthreads();
    const uint32_t live = (c.count - 1u) * P.block + (uint32_t)p % P.block + 1u;       /* the row's own block is the last and may end early */
    for (uint32_t t = 0; t < live; t += 16) {
        const uint32_t n = min(16u, live - t);
        const int32_t slot0 = paged_block_slot(row, P.stride, P.pool_pages, P.page_pos, P.block, (uint32_t)ids[t / P.block]);
        bad |= slot0 < 0;
        for (uint32_t i = tid; i < P.group * n; i += SP_THREADS) {
            const uint32_t h = i / n, j = i % n;
            float s = 0.f;
            if (slot0 >= 0) {
                const uint16_t* k = P.k + ((size_t)((uint32_t)slot0 + t % P.block + j) * P.kv_heads + kvh) * D;
                for (int e = 0; e < D; ++e) s += E::to_float(q[h * D + e]) * E::to_float(k[e]);
            }
            w[h * 16 + j] = s * P.scale;
        }
        __syncthreads();
        for (uint32_t h = tid; h < P.group; h += SP_THREADS) {
            float m = ml[3 * h];
            for (uint32_t j = 0; j < n; ++j) m = fmaxf(m, w[h * 16 + j]);
            const float u = m == -INFINITY ? 0.f : m, f = expf(ml[3 * h] - u);
            float l = ml[3 * h + 1] * f;
            for (uint32_t j = 0; j < n; ++j) { w[h * 16 + j] = expf(w[h * 16 + j] - u); l += w[h * 16 + j]; }
            ml[3 * h] = m; ml[3 * h + 1] = l; ml[3 * h + 2] = f;
        }
        __syncthreads();
        for (uint32_t i = tid; i < P.group * D; i += SP_THREADS) {
            const uint32_t h = i / D, e = i % D;
            float a = acc[i] * ml[3 * h + 2];
            if (slot0 >= 0)
                for (uint32_t j = 0; j < n; ++j) a += w[h * 16 + j] * E::to_float(P.v[((size_t)((uint32_t)slot0 + t % P.block + j) * P.kv_heads + kvh) * D + e]);
            acc[i] = a;
        }
        __syncthreads();
    }
    bool hit = false;
    for (uint32_t i = tid; i < P.group * D; i += SP_THREADS) {
        const uint32_t h = i / D, e = i % D;
        if (P.o) ((uint16_t*)P.o)[head0 * D + i] = E::from_float(acc[i] / ml[3 * h + 1], hit);
        if (P.res) { float* x = P.res + (head0 + h) * (D + 2); x[2 + e] = acc[i]; if (e == 0) { x[0] = ml[3 * h]; x[1] = ml[3 * h + 1]; } }
    }
    if (hit && P.over) atomicOr(P.over, SV_FAULT_OVERFLOW);
    if (bad && P.status) atomicOr(P.status, SV_STATUS_BAD_PAGE);
    (void)part;
}

static cudaError_t sparse_launch(const SparseParams& P, uint32_t rows, uint32_t d, int dtype, cudaStream_t st) {
    const size_t smem = 8 * d + 12 * (SP_CHUNK + (size_t)P.top) + 4 * (size_t)P.top + 4 * (size_t)(P.first + P.last + P.top) + 4 * (size_t)P.group * (d + 19);
    static std::atomic<bool> attr_set[SPARSE_DEVICES];
    int dev = 0; cudaGetDevice(&dev);
    if (dev >= 0 && dev < SPARSE_DEVICES && !attr_set[dev].load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(paged_sparse_kernel<SV_DTYPE_FP16>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_sparse_kernel<SV_DTYPE_BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
        if (e != cudaSuccess) return e;
        attr_set[dev].store(true, std::memory_order_release);
    }
    const dim3 grid(P.kv_heads, rows);
    if (dtype == SV_DTYPE_FP16) paged_sparse_kernel<SV_DTYPE_FP16><<<grid, SP_THREADS, smem, st>>>(P, (int)d);
    else paged_sparse_kernel<SV_DTYPE_BF16><<<grid, SP_THREADS, smem, st>>>(P, (int)d);
    note_launch(1);
    return cudaGetLastError();
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
    if (kv_heads == 0 || kv_heads > 65535u || q_heads == 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > 64u)
        return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: %u query heads over %u kv heads (up to 64 each)", q_heads, kv_heads);
    if (rows == 0 || rows > 65535u || seqs == 0 || table_stride == 0) return sv_ext_fail(SILVANN_B200_E_ARGUMENT, "paged_sparse: %u rows, %u sequences of %u table columns", rows, seqs, table_stride);
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
    P.o = o; P.res = res; P.chosen = chosen; P.q = (const uint16_t*)q; P.k = (const uint16_t*)k_pool; P.v = (const uint16_t*)v_pool; P.means = (const uint16_t*)k_means;
    P.row_seq = row_seq; P.row_pos = row_pos; P.table = page_table; P.over = over; P.status = sv::device_status_word(); P.q_stride = q_stride; P.seqs = seqs;
    P.stride = table_stride; P.pool_pages = (uint32_t)pool_pages; P.page_pos = page_positions; P.block = block_positions; P.q_heads = q_heads; P.kv_heads = kv_heads;
    P.group = q_heads / kv_heads; P.first = first; P.last = last; P.top = top; P.scale = 1.0f / sqrtf((float)head_dim);
    cudaError_t e = sv::sparse_launch(P, rows, head_dim, dtype, (cudaStream_t)stream);
    if (e == cudaSuccess) return SILVANN_B200_OK;
    (void)cudaGetLastError();
    return sv_ext_fail(SILVANN_B200_E_CUDA, "paged_sparse: launch: %s", cudaGetErrorString(e));
}
