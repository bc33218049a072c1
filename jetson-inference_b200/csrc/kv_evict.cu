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

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// *p of CTA `rank` of the cluster (p: this CTA's own)
__device__ __forceinline__ uint32_t remote_u32(const uint32_t* p, int rank) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// Order of the masses as unsigned words, 1 to 0xFF800000: larger mass, larger word; NaN below everything; -0 as 0.
__device__ __forceinline__ uint32_t mass_rank(float x) {
    if (isnan(x)) return 1u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int SEL_THREADS = 1024, SEL_WARPS = SEL_THREADS / 32, SEL_BINS = 2 * SEL_THREADS;
constexpr int SEL_BATCH = 8;  // rows of a thread read at a time
constexpr int SEL_KEYS = 40960;  // ranks of a CTA's slice kept in shared memory; a longer slice is read again each pass

// k_evict_select: the kept row numbers of one (sequence, kv head) per cluster of C CTAs, a contiguous
// slice of the rows each. The n_keep rows of largest rank by radix selection, 11, 11 and 10 bits: the slices'
// counts are added over distributed shared memory, one cluster barrier a round. Then every warp counts what
// it keeps of its own rows, a scan over warps and CTAs gives the places, and the warps write the numbers
// in order. The masses of 8192 rows are 32 KB: latency and the number of instructions a row bound it. Cycles
// at 8192 rows: masses 2900, a round 2000 to 2300 (half of it the scan of the bins), counting 900, writing
// 3000; with the ranks read again in every pass and the kept ends as conditions of each, 2000, 2800,
// 3800 and 5000.
template <int C>
__global__ void __launch_bounds__(SEL_THREADS)
    k_evict_select(const float* __restrict__ mass, const int32_t* __restrict__ n_rows, int32_t* __restrict__ ids,
                   int32_t* __restrict__ n_out, int n_kv_heads, int max_ctx, int n_keep, int n_sink, int n_recent, int n_keys) {
    extern __shared__ uint32_t keys[];  // n_keys of them
    __shared__ uint32_t hist[2][SEL_BINS];
    __shared__ uint32_t wsum[SEL_WARPS];
    __shared__ uint32_t pick[2];                 // digit, left
    __shared__ int wsure[SEL_WARPS], wequal[SEL_WARPS];
    __shared__ int total[2];                     // of this CTA: rows kept for sure, rows of the last rank
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int unit = blockIdx.x / C, part = blockIdx.x % C;
    const int seq = unit / n_kv_heads, head = unit % n_kv_heads;
    const int n = min(max(n_rows[seq], 0), max_ctx);
    const float* mp = mass + (size_t)unit * max_ctx;
    int32_t* op = ids + (size_t)unit * n_keep;
    pdl_trigger();  // the moves' CTAs may be set up; they wait for this kernel's end
    const int kept = min(n, n_keep);
    if (n_out && head == 0 && part == 0 && tid == 0) n_out[seq] = kept;
    for (int i = kept + part * SEL_THREADS + tid; i < n_keep; i += C * SEL_THREADS) op[i] = -1;
    if (n <= n_keep) {  // the same in the whole cluster
        for (int i = part * SEL_THREADS + tid; i < n; i += C * SEL_THREADS) op[i] = i;
        return;
    }
    // rows of this CTA: whole warps' spans, so that a warp's rows are consecutive
    const int span = (n + C * SEL_THREADS - 1) / (C * SEL_THREADS) * 32;  // rows of a warp
    const int base = part * SEL_WARPS * span, limit = min(n, base + SEL_WARPS * span);
    const int first = base + warp * span, steps = span / 32;
    // The same thread reads a row's rank in every pass: from registers where it has SEL_BATCH rows at most, else
    // from shared memory, or from the masses again. The first and the last rows rank above every mass and what
    // lies past the slice below, so that what stays is the n_keep rows of largest rank.
    const bool once = steps <= SEL_BATCH, stage = SEL_WARPS * span <= n_keys;
    uint32_t r[SEL_BATCH];
    auto ranks = [&](int s0) {  // of the masses
        float x[SEL_BATCH];
#pragma unroll
        for (int j = 0; j < SEL_BATCH; ++j) {
            const int i = first + 32 * (s0 + j) + lane;
            x[j] = s0 + j < steps && i < limit ? mp[i] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < SEL_BATCH; ++j) {
            const int i = first + 32 * (s0 + j) + lane;
            r[j] = s0 + j >= steps || i >= limit ? 0u : i < n_sink || i >= n - n_recent ? 0xFFFFFFFFu : mass_rank(x[j]);
        }
    };
    uint32_t* own = keys + warp * span + lane;
    auto read = [&](int s0) {
        if (once) return;
        if (!stage) return ranks(s0);
#pragma unroll
        for (int j = 0; j < SEL_BATCH; ++j) r[j] = s0 + j < steps ? own[32 * (s0 + j)] : 0u;
    };
    for (int s0 = 0; s0 < steps && (once || stage); s0 += SEL_BATCH) {
        ranks(s0);
        if (!once)
#pragma unroll
            for (int j = 0; j < SEL_BATCH; ++j)
                if (s0 + j < steps) own[32 * (s0 + j)] = r[j];
    }

    uint32_t left = n_keep;  // still to be picked among the ranks that match the prefix
    uint32_t prefix = 0, mask = 0;
    for (int round = 0; round < 3; ++round) {
        const int shift = round == 0 ? 21 : round == 1 ? 10 : 0;
        const uint32_t digit = round == 2 ? 1023u : 2047u;
        uint32_t* h = hist[round & 1];
        h[tid] = 0;
        h[tid + SEL_THREADS] = 0;
        __syncthreads();
        for (int s0 = 0; s0 < steps; s0 += SEL_BATCH) {
            read(s0);
#pragma unroll
            for (int j = 0; j < SEL_BATCH; ++j)
                if (r[j] && (r[j] & mask) == prefix) atomicAdd(&h[(r[j] >> shift) & digit], 1u);
        }
        if constexpr (C > 1) cluster_barrier(); else __syncthreads();
        // bins SEL_BINS - 1 - 2 tid and the one below: how many have a larger digit, and these
        const int bin = SEL_BINS - 1 - 2 * tid;
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            a += C > 1 ? remote_u32(&h[bin], c) : h[bin];
            b += C > 1 ? remote_u32(&h[bin - 1], c) : h[bin - 1];
        }
        uint32_t upto = a + b;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(JINF_FULL_MASK, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) wsum[warp] = upto;
        __syncthreads();
        upto += __reduce_add_sync(JINF_FULL_MASK, lane < warp ? wsum[lane] : 0u);
        const uint32_t above = upto - a - b;
        if (upto >= left && above < left) {  // one of the two bins holds the left-th largest
            const bool first = above + a >= left;
            pick[0] = first ? bin : bin - 1;
            pick[1] = first ? left - above : left - above - a;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        mask |= digit << shift;
        left = pick[1];
    }
    // ranks above `prefix` stay; of those equal to it the first `left`
    int n_sure = 0, n_equal = 0;
    for (int s0 = 0; s0 < steps; s0 += SEL_BATCH) {
        read(s0);
#pragma unroll
        for (int j = 0; j < SEL_BATCH; ++j) {
            n_sure += r[j] > prefix;
            n_equal += r[j] == prefix;
        }
    }
    n_sure = (int)__reduce_add_sync(JINF_FULL_MASK, (unsigned)n_sure);
    n_equal = (int)__reduce_add_sync(JINF_FULL_MASK, (unsigned)n_equal);
    if (lane == 0) {
        wsure[warp] = n_sure;
        wequal[warp] = n_equal;
    }
    __syncthreads();
    // this warp's place: what the CTAs and warps before it keep
    int place = 0, taken = 0;  // kept rows, and rows of the last rank, before
    auto add = [&](int s, int e) {
        place += s + min(max((int)left - taken, 0), e);
        taken += e;
    };
    if constexpr (C > 1) {
        if (warp == 0) {
            const int s = (int)__reduce_add_sync(JINF_FULL_MASK, (unsigned)wsure[lane]);
            const int e = (int)__reduce_add_sync(JINF_FULL_MASK, (unsigned)wequal[lane]);
            if (lane == 0) {
                total[0] = s;
                total[1] = e;
            }
        }
        cluster_barrier();
        for (int c = 0; c < part; ++c)
            add((int)remote_u32((uint32_t*)&total[0], c), (int)remote_u32((uint32_t*)&total[1], c));
    }
    {
        // the CTA's warps before this one: min(max(left - taken, 0), e) adds up to the same taken all at once
        const int s = (int)__reduce_add_sync(JINF_FULL_MASK, lane < warp ? (unsigned)wsure[lane] : 0u);
        const int e = (int)__reduce_add_sync(JINF_FULL_MASK, lane < warp ? (unsigned)wequal[lane] : 0u);
        add(s, e);
    }
    const uint32_t before = (1u << lane) - 1u;
    for (int s0 = 0; s0 < steps; s0 += SEL_BATCH) {
        read(s0);
#pragma unroll
        for (int j = 0; j < SEL_BATCH; ++j) {
            bool keep = r[j] > prefix;
            if (n_equal > 0) {  // few warps have such rows, and counting bits is slow
                const bool eq = r[j] == prefix;
                const uint32_t be = __ballot_sync(JINF_FULL_MASK, eq);
                keep |= eq && taken + __popc(be & before) < (int)left;
                taken += __popc(be);
            }
            const uint32_t bk = __ballot_sync(JINF_FULL_MASK, keep);
            if (keep) op[place + __popc(bk & before)] = first + 32 * (s0 + j) + lane;
            place += __popc(bk);
        }
    }
    if constexpr (C > 1) cluster_barrier();  // no CTA leaves while another may read its counts
}

constexpr int MV_THREADS = 256, MV_CHUNKS = 4, MV_BATCH = 8;
constexpr int MV_ROWS = MV_THREADS / MV_CHUNKS * MV_BATCH;  // rows of a batch

// k_evict_move, in place: row ids[i] -> row i. blockIdx.x = (sequence, kv head); blockIdx.y = K or V and
// a 64-byte column of the rows, and the mass (one more). A block takes the batches of rows in order.
// Source and destination are the same memory: no pointer to either is __restrict__.
__global__ void __launch_bounds__(MV_THREADS)
    k_evict_move(const KvPlanes src, const KvPlanes dst, const float* mass, float* mass_out,
                 const int32_t* __restrict__ ids, const int32_t* __restrict__ n_rows, int n_kv_heads, int row_bytes,
                 int n_keep) {
    pdl_wait();
    const int seq = blockIdx.x / n_kv_heads, head = blockIdx.x % n_kv_heads, tid = threadIdx.x;
    const int n = min(min(max(n_rows[seq], 0), src.max_ctx), n_keep);
    const int32_t* ip = ids + (size_t)blockIdx.x * n_keep;
    const int cols = row_bytes / 64;
    if ((int)blockIdx.y == 2 * cols) {
        const float* from = mass + (size_t)blockIdx.x * src.max_ctx;
        float* to = mass_out + (size_t)blockIdx.x * dst.max_ctx;
        for (int i0 = 0; i0 < n; i0 += MV_THREADS) {
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
    for (int b0 = 0; b0 < n; b0 += MV_ROWS) {
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

constexpr int CP_BATCH = 4;

// k_evict_copy, into another cache: whole rows (CH 16-byte chunks), CP_BATCH of them per thread in
// flight. blockIdx.x = batch of rows, so that neighbouring blocks read neighbouring rows; blockIdx.y =
// (sequence, kv head). HBM bounds it: 256 heads from 32768 rows to 8192 in 0.33 ms, 6.5 TB/s (8 rows a
// thread 0.43 ms, heads before batches in the grid 0.34); with the selection before it 0.38 ms.
template <int CH>
__global__ void __launch_bounds__(MV_THREADS)
    k_evict_copy(const KvPlanes src, const KvPlanes dst, const float* __restrict__ mass, float* __restrict__ mass_out,
                 const int32_t* __restrict__ ids, const int32_t* __restrict__ n_rows, int n_units, int n_kv_heads, int n_keep) {
    constexpr int LANES = MV_THREADS / CH;  // rows side by side
    pdl_wait();
    const int c = threadIdx.x % CH, i0 = blockIdx.x * LANES * CP_BATCH + threadIdx.x / CH;
    for (int unit = blockIdx.y; unit < n_units; unit += gridDim.y) {
        const int seq = unit / n_kv_heads, head = unit % n_kv_heads;
        const int n = min(min(max(n_rows[seq], 0), src.max_ctx), n_keep);
        const int32_t* ip = ids + (size_t)unit * n_keep;
        const int64_t so = seq * src.seq + head * src.head + c * 16, dof = seq * dst.seq + head * dst.head + c * 16;
        int from[CP_BATCH];
#pragma unroll
        for (int j = 0; j < CP_BATCH; ++j) from[j] = i0 + j * LANES < n ? __ldg(ip + i0 + j * LANES) : -1;
        uint4 x[2][CP_BATCH];
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int j = 0; j < CP_BATCH; ++j)
                if (from[j] >= 0) x[v][j] = __ldcs(reinterpret_cast<const uint4*>((v ? src.v : src.k) + so + from[j] * src.row));
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int j = 0; j < CP_BATCH; ++j)
                if (from[j] >= 0) __stcs(reinterpret_cast<uint4*>((v ? dst.v : dst.k) + dof + (i0 + j * LANES) * dst.row), x[v][j]);
        if (mass_out && c == 0) {
#pragma unroll
            for (int j = 0; j < CP_BATCH; ++j)
                if (from[j] >= 0)
                    mass_out[(size_t)unit * dst.max_ctx + i0 + j * LANES] = __ldg(mass + (size_t)unit * src.max_ctx + from[j]);
        }
    }
}

constexpr int CM_WARPS = 4, CM_BATCH = 8;

// k_tree_commit: one warp per (sequence, kv head). A lane owns 16-byte columns of K and V (and
// lane 0 the mass) and moves them row by row, so no order between threads matters; the loads of
// CM_BATCH rows are in flight before their stores.
// Latency bounds it: 32 layers of 8 heads, 5 of 26 rows, take 2.5 us back to back in a graph.
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

template <int C>
cudaError_t launch_select(int units, const float* mass, const int32_t* n_rows, int32_t* ids, int32_t* n_out, int n_kv_heads,
                          int max_ctx, int n_keep, int n_sink, int n_recent, cudaStream_t s) {
    const int slice = (max_ctx + C * SEL_THREADS - 1) / (C * SEL_THREADS) * SEL_THREADS;
    const int n_keys = slice <= SEL_KEYS ? slice : 0;
    const cudaError_t e = kv_allow_smem<k_evict_select<C>>(SEL_KEYS * (int)sizeof(uint32_t));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * C));
    cfg.blockDim = dim3(SEL_THREADS);
    cfg.dynamicSmemBytes = sizeof(uint32_t) * (size_t)n_keys;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_evict_select<C>, mass, n_rows, ids, n_out, n_kv_heads, max_ctx, n_keep, n_sink, n_recent, n_keys);
}

}  // namespace

cudaError_t kv_evict_launch(const KvPlanes& src, const KvPlanes& dst, bool in_place, const float* mass, float* mass_out,
                            const int32_t* n_rows, int32_t* ids, int32_t* n_out, int n_seqs, int n_kv_heads,
                            int row_bytes, int n_keep, int n_sink, int n_recent, cudaStream_t s) {
    const int units = n_seqs * n_kv_heads;
    // One CTA a head where its ranks fit shared memory, else clusters of 8, whose slices do up to 327680 rows.
    // Measured (us of the whole call, 8 heads to 2048 rows of 64 columns, one CTA / a cluster): 8192 rows 11.0 / 27.1,
    // 16384 17.2 / 27.5, 32768 27.0 / 28.1, 64 heads of 32768 35 / 111.
    cudaError_t e = src.max_ctx <= SEL_KEYS
                        ? launch_select<1>(units, mass, n_rows, ids, n_out, n_kv_heads, src.max_ctx, n_keep, n_sink, n_recent, s)
                        : launch_select<8>(units, mass, n_rows, ids, n_out, n_kv_heads, src.max_ctx, n_keep, n_sink, n_recent, s);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(MV_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (in_place) {
        cfg.gridDim = dim3((unsigned)units, (unsigned)(2 * (row_bytes / 64) + (mass_out ? 1 : 0)));
        return cudaLaunchKernelEx(&cfg, k_evict_move, src, dst, mass, mass_out, ids, n_rows, n_kv_heads, row_bytes, n_keep);
    }
    const int ch = row_bytes / 16, rows = MV_THREADS / ch * CP_BATCH, batches = (n_keep + rows - 1) / rows;
    cfg.gridDim = dim3((unsigned)batches, (unsigned)(units < 65535 ? units : 65535));
    return ch == 8 ? cudaLaunchKernelEx(&cfg, k_evict_copy<8>, src, dst, mass, mass_out, (const int32_t*)ids, n_rows, units, n_kv_heads, n_keep)
                   : cudaLaunchKernelEx(&cfg, k_evict_copy<16>, src, dst, mass, mass_out, (const int32_t*)ids, n_rows, units, n_kv_heads, n_keep);
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
