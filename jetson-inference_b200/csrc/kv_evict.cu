// Cutting a K/V cache back to the rows that matter, and moving an accepted path's rows up
// (jinf_b200_kv_evict, jinf_b200_tree_commit), sm_100a.
//
// Both only move bytes. In place, a row moves to a lower place (the i-th kept row has number
// ids[i] >= i), so a thread block that reads a batch of rows in order before it writes their new
// places never overwrites a row that is still to be read; different byte columns of the rows are
// independent, which gives the parallelism.
#include "kv_ops.cuh"

namespace jinf {
namespace {

// Order of the masses as unsigned words: larger mass, larger word; NaN below everything; -0 as 0.
__device__ __forceinline__ uint32_t mass_rank(float x) {
    if (isnan(x)) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int SEL_THREADS = 1024;

// k_evict_select: the kept row numbers of one (sequence, kv head) per CTA. The n_pick rows of
// largest mass among rows n_sink .. n - n_recent - 1 by radix selection, 8 bits of the rank at
// a time (the count of ranks above a prefix), then the ids in order by a block scan.
__global__ void __launch_bounds__(SEL_THREADS)
    k_evict_select(const float* __restrict__ mass, const int32_t* __restrict__ n_rows, int32_t* __restrict__ ids,
                   int32_t* __restrict__ n_out, int n_kv_heads, int max_ctx, int n_keep, int n_sink, int n_recent) {
    __shared__ int hist[256];
    __shared__ int wsum[32];
    __shared__ int pick_digit, pick_left;
    const int seq = blockIdx.x / n_kv_heads, head = blockIdx.x % n_kv_heads, tid = threadIdx.x;
    const int n = min(max(n_rows[seq], 0), max_ctx);
    const float* mp = mass + (size_t)blockIdx.x * max_ctx;
    int32_t* op = ids + (size_t)blockIdx.x * n_keep;
    const int kept = min(n, n_keep);
    if (n_out && head == 0 && tid == 0) n_out[seq] = kept;
    for (int i = kept + tid; i < n_keep; i += SEL_THREADS) op[i] = -1;
    if (n <= n_keep) {
        for (int i = tid; i < n; i += SEL_THREADS) op[i] = i;
        return;
    }
    const int lo = n_sink, hi = n - n_recent;  // hi - lo > n_keep - n_sink - n_recent >= 0
    int left = n_keep - n_sink - n_recent;     // still to be picked among the ranks that match the prefix
    uint32_t prefix = 0, mask = 0;
    if (left > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += SEL_THREADS) {
                const uint32_t r = mass_rank(mp[i]);
                if ((r & mask) == prefix) atomicAdd(&hist[(r >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {  // the digit whose bin holds the left-th largest
                int d = 255, above = 0;
                while (d > 0 && above + hist[d] < left) above += hist[d--];
                pick_digit = d;
                pick_left = left - above;
            }
            __syncthreads();
            prefix |= (uint32_t)pick_digit << shift;
            mask |= 255u << shift;
            left = pick_left;
            __syncthreads();
        }
    }
    // ranks above `prefix` stay; of those equal to it the first `left`
    const bool none = n_keep == n_sink + n_recent;
    int kept_before = 0, equal_before = 0;
    for (int i0 = 0; i0 < n; i0 += SEL_THREADS) {
        const int i = i0 + tid;
        bool keep = false, equal = false;
        if (i < n) {
            if (i < lo || i >= hi) keep = true;
            else if (!none) {
                const uint32_t r = mass_rank(mp[i]);
                keep = r > prefix;
                equal = r == prefix;
            }
        }
        for (int pass = 0; pass < 2; ++pass) {  // the equal ones' places first, then the kept ones'
            const bool f = pass ? keep : equal;
            const uint32_t b = __ballot_sync(JINF_FULL_MASK, f);
            if ((tid & 31) == 0) wsum[tid >> 5] = __popc(b);
            __syncthreads();
            int before = __popc(b & ((1u << (tid & 31)) - 1u)), all = 0;
            for (int w = 0; w < 32; ++w) {
                if (w < (tid >> 5)) before += wsum[w];
                all += wsum[w];
            }
            __syncthreads();
            if (!pass) {
                if (equal && equal_before + before < left) keep = true;
                equal_before += all;
            } else {
                if (keep) op[kept_before + before] = i;
                kept_before += all;
            }
        }
    }
}

constexpr int MV_THREADS = 256, MV_CHUNKS = 4, MV_BATCH = 4;
constexpr int MV_ROWS = MV_THREADS / MV_CHUNKS * MV_BATCH;  // rows of a batch

// k_evict_move: row ids[i] -> row i. blockIdx.x = (sequence, kv head); blockIdx.y = K or V and a
// 64-byte column of the rows, and the mass (one more); blockIdx.z = batches (one block in place).
// Source and destination may be the same memory: no pointer to either is __restrict__.
__global__ void __launch_bounds__(MV_THREADS)
    k_evict_move(const KvPlanes src, const KvPlanes dst, const float* mass, float* mass_out,
                 const int32_t* __restrict__ ids, const int32_t* __restrict__ n_rows, int n_kv_heads, int row_bytes,
                 int n_keep) {
    const int seq = blockIdx.x / n_kv_heads, head = blockIdx.x % n_kv_heads, tid = threadIdx.x;
    const int n = min(min(max(n_rows[seq], 0), src.max_ctx), n_keep);
    const int32_t* ip = ids + (size_t)blockIdx.x * n_keep;
    const int cols = row_bytes / 64;
    if ((int)blockIdx.y == 2 * cols) {
        const float* from = mass + (size_t)blockIdx.x * src.max_ctx;
        float* to = mass_out + (size_t)blockIdx.x * dst.max_ctx;
        for (int i0 = blockIdx.z * MV_THREADS; i0 < n; i0 += gridDim.z * MV_THREADS) {
            const int i = i0 + tid;
            float x = 0.f;
            if (i < n) x = from[ip[i]];
            __syncthreads();
            if (i < n) to[i] = x;
            __syncthreads();
        }
        return;
    }
    const bool is_v = (int)blockIdx.y >= cols;
    const int64_t col = (blockIdx.y % cols) * 64 + (tid % MV_CHUNKS) * 16;
    const uint8_t* from = (is_v ? src.v : src.k) + seq * src.seq + head * src.head + col;
    uint8_t* to = (is_v ? dst.v : dst.k) + seq * dst.seq + head * dst.head + col;
    for (int b0 = blockIdx.z * MV_ROWS; b0 < n; b0 += gridDim.z * MV_ROWS) {
        uint4 x[MV_BATCH];
#pragma unroll
        for (int j = 0; j < MV_BATCH; ++j) {
            const int i = b0 + j * (MV_THREADS / MV_CHUNKS) + tid / MV_CHUNKS;
            if (i < n) x[j] = *reinterpret_cast<const uint4*>(from + (int64_t)ip[i] * src.row);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < MV_BATCH; ++j) {
            const int i = b0 + j * (MV_THREADS / MV_CHUNKS) + tid / MV_CHUNKS;
            if (i < n) *reinterpret_cast<uint4*>(to + (int64_t)i * dst.row) = x[j];
        }
        __syncthreads();
    }
}

constexpr int CM_WARPS = 4, CM_BATCH = 8;

// k_tree_commit: one warp per (sequence, kv head). A lane owns 16-byte columns of K and V (and
// lane 0 the mass) and moves them row by row, so no order between threads matters; the loads of
// CM_BATCH rows are in flight before their stores.
__global__ void __launch_bounds__(CM_WARPS * 32)
    k_tree_commit(const KvPlanes kv, float* mass, const int32_t* __restrict__ n_past, int max_past,
                  const int32_t* __restrict__ accepted, int accepted_stride, const int32_t* __restrict__ n_accepted,
                  int n_nodes, int32_t* __restrict__ n_out, int n_units, int n_kv_heads, int row_bytes) {
    const int unit = blockIdx.x * CM_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (unit >= n_units) return;
    const int seq = unit / n_kv_heads, head = unit % n_kv_heads;
    const int past = min(max(n_past[seq], 0), max_past);
    const int n = min(max(n_accepted[seq], 0), min(n_nodes, accepted_stride));
    const int32_t* acc = accepted + (size_t)seq * accepted_stride;
    const int chunks = row_bytes / 16;
    float* mp = mass ? mass + (size_t)unit * kv.max_ctx + past : nullptr;
    for (int i0 = 0; i0 < n; i0 += CM_BATCH) {
        int from[CM_BATCH];
#pragma unroll
        for (int j = 0; j < CM_BATCH; ++j) {
            from[j] = i0 + j < n ? acc[i0 + j] : -1;
            if (from[j] >= n_nodes || from[j] == i0 + j) from[j] = -1;
        }
        for (int c = lane; c < 2 * chunks; c += 32) {
            uint8_t* base = (c < chunks ? kv.k + c * 16 : kv.v + (c - chunks) * 16) + seq * kv.seq + head * kv.head +
                            past * kv.row;
            uint4 x[CM_BATCH];
#pragma unroll
            for (int j = 0; j < CM_BATCH; ++j)
                if (from[j] >= 0) x[j] = *reinterpret_cast<const uint4*>(base + from[j] * kv.row);
#pragma unroll
            for (int j = 0; j < CM_BATCH; ++j)
                if (from[j] >= 0) *reinterpret_cast<uint4*>(base + (i0 + j) * kv.row) = x[j];
        }
        if (mp && lane == 0) {
            float x[CM_BATCH];
#pragma unroll
            for (int j = 0; j < CM_BATCH; ++j)
                if (from[j] >= 0) x[j] = mp[from[j]];
#pragma unroll
            for (int j = 0; j < CM_BATCH; ++j)
                if (from[j] >= 0) mp[i0 + j] = x[j];
        }
    }
    if (n_out && head == 0 && lane == 0) n_out[seq] = past + n;
}

}  // namespace

cudaError_t kv_evict_launch(const KvPlanes& src, const KvPlanes& dst, bool in_place, const float* mass, float* mass_out,
                            const int32_t* n_rows, int32_t* ids, int32_t* n_out, int n_seqs, int n_kv_heads,
                            int row_bytes, int n_keep, int n_sink, int n_recent, cudaStream_t s) {
    const int units = n_seqs * n_kv_heads;
    k_evict_select<<<units, SEL_THREADS, 0, s>>>(mass, n_rows, ids, n_out, n_kv_heads, src.max_ctx, n_keep, n_sink,
                                                 n_recent);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const int batches = (n_keep + MV_ROWS - 1) / MV_ROWS;
    const dim3 grid((unsigned)units, (unsigned)(2 * (row_bytes / 64) + (mass_out ? 1 : 0)),
                    (unsigned)(in_place ? 1 : (batches < 64 ? batches : 64)));
    k_evict_move<<<grid, MV_THREADS, 0, s>>>(src, dst, mass, mass_out, ids, n_rows, n_kv_heads, row_bytes, n_keep);
    return cudaGetLastError();
}

cudaError_t tree_commit_launch(const KvPlanes& kv, float* mass, const int32_t* n_past, int max_past,
                               const int32_t* accepted, int accepted_stride, const int32_t* n_accepted, int n_nodes,
                               int32_t* n_out, int n_seqs, int n_kv_heads, int row_bytes, cudaStream_t s) {
    const int units = n_seqs * n_kv_heads;
    k_tree_commit<<<(units + CM_WARPS - 1) / CM_WARPS, CM_WARPS * 32, 0, s>>>(
        kv, mass, n_past, max_past, accepted, accepted_stride, n_accepted, n_nodes, n_out, units, n_kv_heads, row_bytes);
    return cudaGetLastError();
}

}  // namespace jinf
