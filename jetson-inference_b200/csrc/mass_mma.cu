// Attention weight received by each cached row on the fifth-generation tensor cores
// (jinf_b200_attention_mass), sm_100a.
//
// S^T = K Q^T with keys as the MMA's 128 rows and up to 128 query rows as its columns: in tensor
// memory a lane is a key, so its sum over the query rows needs no exchange between threads. What
// bounds it: K from HBM while the query rows are few; the exponentials (16 a cycle and SM) when
// there are hundreds. A CTA takes a share of the key tiles (kv_ops.cuh); per up to 4 tiles of
// a kv head, kept in shared memory, it runs over the query rows 128 at a time:
//   warp 0      copies K tiles (TMA);
//   warps 1, 2  issue the MMAs into four score buffers of 128 columns, in turn: one issuer's turn (waits
//               and eight MMAs, 1200 cycles) is longer than the exponentials of a buffer (1024);
//   warp 3      brings 128 query rows into one of two stages, with -lse log2 e and the weight of each:
//               boxes of whole nodes by TMA when every node counts and nodes fill a stage evenly, else
//               the rows of weight != 0 one by one (16-byte asynchronous copies into the 128B-swizzled
//               layout; about 4000 cycles a stage where the boxes take 1500);
//   warps 4-11  two groups, one thread per key: take the score buffers in turn and add w e^(s - lse),
//               32 columns in registers ahead of the ones being added. With several stages a key's
//               two sums are added in the groups' order.
// Every wait is bounded; one that runs out sets the error word and ends the CTA.
#include "kv_ops.cuh"
#include "umma.cuh"

#include <math.h>

namespace jinf {
namespace {

constexpr int XT = 384;
constexpr int ATOM = 16384;  // 128 rows x 64 columns, 128B-swizzled
constexpr int KT = 4;        // key tiles kept while the query rows pass; also the ring of K tiles
constexpr int NB = 4;        // score buffers
constexpr int NR = 4;        // stages whose row factors are kept: the MMAs run ahead of the sums
constexpr int GROUPS = 2;

template <int HD>
struct MassMma {
    static constexpr int TILE = ATOM * (HD / 64);
    static constexpr int OFF_Q = KT * TILE;
    static constexpr int OFF_MISC = OFF_Q + 2 * TILE;
    struct Misc {
        uint64_t k_full[KT], k_free[KT], q_full[2], q_free[2], r_full[NR], r_free[NR], s_full[NB], s_free[NB], meet, drain[2];
        Share share;
        uint32_t tmem;
        int abort;
        alignas(16) float2 row[NR][128];    // of a stage's query rows: -lse log2 e, weight
        uint8_t row_node[NR][128];          // and their nodes
        uint8_t node[JINF_TREE_MAX_NODES];  // nodes of weight != 0, ascending (warp 3's)
        alignas(16) float sums[2][GROUPS][KT][128];
    };
    static constexpr int TOTAL = OFF_MISC + (int)sizeof(Misc) + 1024;
};
static_assert(MassMma<128>::TOTAL + 64 <= 232448, "shared memory");
static_assert(JINF_TREE_MAX_NODES <= 256, "node numbers are kept in bytes");
static_assert(GROUPS == 2 && NB % GROUPS == 0, "item parity picks the issuer, the group and so the buffer");

// Nodes of weight != 0, by a whole warp; their numbers, ascending, to `list` where it is not null.
__device__ __forceinline__ int active_nodes(const TreeParams& p, const float* weight, int seq, uint8_t* list) {
    if (!weight) {
        if (list)
            for (int t = threadIdx.x & 31; t < p.n_nodes; t += 32) list[t] = (uint8_t)t;
        return p.n_nodes;
    }
    const int lane = threadIdx.x & 31;
    int n = 0;
    for (int t0 = 0; t0 < p.n_nodes; t0 += 32) {
        const int t = t0 + lane;
        const bool on = t < p.n_nodes && weight[(size_t)seq * p.n_nodes + t] != 0.f;
        const uint32_t b = __ballot_sync(JINF_FULL_MASK, on);
        if (on && list) list[n + __popc(b & ((1u << lane) - 1u))] = (uint8_t)t;
        n += __popc(b);
    }
    return n;
}

template <bool BF, int HD>
__global__ void __launch_bounds__(XT, 1)
    k_mass_mma(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmq, const TreeParams p, const float* __restrict__ lse,
               const float* __restrict__ weight, float* __restrict__ mass) {
    using SM = MassMma<HD>;
    constexpr int TILE = SM::TILE, CH = HD / 8;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    typename SM::Misc& ms = *reinterpret_cast<typename SM::Misc*>(sm + SM::OFF_MISC);
    const uint32_t s_k = su32(sm), s_q = s_k + SM::OFF_Q;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < KT; ++i) {
            mb_init(su32(&ms.k_full[i]), 1);
            mb_init(su32(&ms.k_free[i]), 2);
        }
        for (int i = 0; i < 2; ++i) {
            mb_init(su32(&ms.q_full[i]), 1);
            mb_init(su32(&ms.q_free[i]), 2);
        }
        for (int i = 0; i < NR; ++i) {
            mb_init(su32(&ms.r_full[i]), 1);
            mb_init(su32(&ms.r_free[i]), 4 * GROUPS);
        }
        for (int i = 0; i < NB; ++i) {
            mb_init(su32(&ms.s_full[i]), 1);
            mb_init(su32(&ms.s_free[i]), 4);
        }
        mb_init(su32(&ms.meet), 4 * GROUPS);
        for (int i = 0; i < 2; ++i) mb_init(su32(&ms.drain[i]), 1);
        ms.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&ms.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 2) {
        Shares all;
        const Share sh = share_begin(p, blockIdx.x, gridDim.x, all);
        if (lane == 0) ms.share = sh;
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = ms.tmem;
    Share share = ms.share;
    Segment sg;

    // A wait by parity tells phase x only from x - 1, so each role waits for every phase of a barrier
    // in order (a score buffer belongs to one issuer and one group: NB is a multiple of GROUPS).
    // a bounded wait of a warp that also ends when another role gave up
    auto wait = [&](uint64_t& bar, uint32_t parity) -> bool {
        const uint32_t b = su32(&bar);
        bool done = false;
        for (unsigned long long it = 0; it < MB_SPIN && !done; ++it) {
            done = mb_try(b, parity);
            if ((it & 255) == 255 && *(volatile int*)&ms.abort) break;
        }
        if (!done && !atomicExch(&ms.abort, 1)) atomicExch(p.err, 1);
        return __all_sync(JINF_FULL_MASK, done);
    };
    auto arrive_warp = [&](uint64_t& bar) {
        __syncwarp();
        if (lane == 0) mb_arrive(su32(&bar));
    };
    // Every role walks the same loops: segments, then sets of key tiles, for each set stages of 128 query
    // rows, for each stage the set's tiles; a score buffer per (stage, tile), counted in `item`. With
    // several stages a set is up to KT tiles, which stay while the rows pass; with one the rows stay.
    auto set_of = [&](int stages) { return stages == 1 ? INT32_MAX : KT; };

    if (warp == 0) {
        uint32_t pos = 0;
        bool ok = true;
        while (ok && share.next(p, sg)) {
            if (active_nodes(p, weight, sg.seq, nullptr) == 0) continue;
            for (int t = sg.t0; t < sg.t1; ++t, ++pos) {
                const uint32_t slot = pos % KT;
                if (pos >= KT && !(ok = wait(ms.k_free[slot], (pos / KT - 1) & 1))) break;
                if (lane == 0) {
                    const uint32_t bar = su32(&ms.k_full[slot]);
                    mb_expect(bar, TILE);
#pragma unroll
                    for (int a = 0; a < HD / 64; ++a)
                        tma_load_4d(s_k + slot * TILE + a * ATOM, &tmk, 64 * a, t * KV_TILE, sg.head, sg.seq, bar);
                }
                __syncwarp();
            }
        }
        if (!ok && lane == 0)  // leave no copy in flight
            for (uint32_t s = 0; s < KT && s < pos; ++s) mb_wait(su32(&ms.k_full[s]), ((pos - 1 - s) / KT) & 1);
    } else if (warp < 3) {
        const uint32_t turn = warp - 1;
        const bool leader = elect_one();
        uint32_t pos = 0, fill = 0, item = 0;
        bool ok = true;
        while (ok && share.next(p, sg)) {
            const int rows = active_nodes(p, weight, sg.seq, nullptr) * p.group, stages = (rows + 127) / 128;
            if (rows == 0) continue;
            for (int t = sg.t0; ok && t < sg.t1;) {
                const int n = min(set_of(stages), sg.t1 - t);
                for (int st = 0; ok && st < stages; ++st, ++fill) {
                    if (!(ok = wait(ms.q_full[fill & 1], (fill >> 1) & 1))) break;
                    const int cols = min(128, (rows - 128 * st + 31) & ~31);
                    const uint32_t idesc = umma_idesc(BF, 128, 0, false) | ((uint32_t)(cols >> 3) << 17);
                    const uint64_t dq = umma_desc(s_q + (fill & 1) * TILE);
                    for (int j = 0; j < n; ++j, ++item) {
                        const uint32_t slot = (pos + j) % KT, b = item % NB;
                        if (st == 0 && !(ok = wait(ms.k_full[slot], ((pos + j) / KT) & 1))) break;
                        const bool mine = (item & 1) == turn;
                        if (mine && item >= NB && !(ok = wait(ms.s_free[b], (item / NB - 1) & 1))) break;
                        tc_after_sync();
                        if (leader) {
                            if (mine) {
                                const uint64_t dk = umma_desc(s_k + slot * TILE);
#pragma unroll
                                for (int kk = 0; kk < HD / 16; ++kk) {
                                    const uint32_t off = ((kk >> 2) * ATOM + (kk & 3) * 32) >> 4;
                                    umma_ss(tmem + 128 * b, dk + off, dq + off, idesc, kk > 0);
                                }
                                umma_commit(su32(&ms.s_full[b]));
                            }
                            if (st == stages - 1) umma_commit(su32(&ms.k_free[slot]));
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (leader) umma_commit(su32(&ms.q_free[fill & 1]));
                    __syncwarp();
                }
                pos += n;
                t += n;
            }
        }
        if (!ok && leader) {  // the MMAs already issued finish before the memory goes
            umma_commit(su32(&ms.drain[turn]));
            mb_wait(su32(&ms.drain[turn]), 0);
        }
    } else if (warp == 3) {
        uint8_t* list = ms.node;
        uint32_t fill = 0, boxed = 0;
        bool ok = true;
        while (ok && share.next(p, sg)) {
            const int rows = active_nodes(p, weight, sg.seq, list) * p.group, stages = (rows + 127) / 128;
            __syncwarp();
            if (rows == 0) continue;
            const bool boxes = rows == p.n_rows && 128 % p.group == 0;
            const int fills = stages > 1 ? (sg.t1 - sg.t0 + KT - 1) / KT * stages : 1;
            // lane l has rows l, l + 32, ..: where they are (-1: zeros), -lse log2 e, weight, node
            int64_t from[4];
            float2 bw[4];
            int node[4];
            auto rows_of = [&](int st) {
                float l[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int rr = 128 * st + 32 * k + lane;
                    from[k] = -1;
                    bw[k] = make_float2(-INFINITY, 0.f);
                    node[k] = 0;
                    l[k] = -INFINITY;
                    if (rr < rows) {
                        node[k] = list[rr / p.group];
                        const int h = sg.head * p.group + rr % p.group;
                        from[k] = (sg.seq * p.q_seq + node[k] * p.q_node + (int64_t)h * HD) * 2;
                        l[k] = lse[((size_t)sg.seq * p.n_nodes + node[k]) * p.n_heads + h];
                        bw[k].y = weight ? weight[(size_t)sg.seq * p.n_nodes + node[k]] : 1.f;
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (l[k] != -INFINITY) {
                        bw[k].x = -l[k] * LOG2E;
                    } else {  // a row that attended nothing adds nothing, whatever it holds
                        bw[k].y = 0.f;
                        from[k] = -1;
                    }
                }
            };
            rows_of(0);
            for (int x = 0; x < fills; ++x) {
                const uint32_t f = fill + x, s = f & 1;
                const int cols = min(128, (rows - 128 * (x % stages) + 31) & ~31), rs = f % NR;
                if (f >= NR && !(ok = wait(ms.r_free[rs], (f / NR - 1) & 1))) break;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    ms.row[rs][32 * k + lane] = bw[k];
                    ms.row_node[rs][32 * k + lane] = (uint8_t)node[k];
                }
                arrive_warp(ms.r_full[rs]);
                if (f >= 2 && !(ok = wait(ms.q_free[s], ((f >> 1) - 1) & 1))) break;
                const uint32_t dst = s_q + s * TILE;
                if (boxes) {
                    if (lane == 0) {
                        const uint32_t bar = su32(&ms.q_full[s]);
                        mb_expect(bar, TILE);
#pragma unroll
                        for (int a = 0; a < HD / 64; ++a)  // nodes past the last are zeros
                            tma_load_4d(dst + a * ATOM, &tmq, 64 * a, sg.head * p.group, x % stages * p.tile_nodes, sg.seq, bar);
                    }
                    __syncwarp();
                    boxed = f + 1;
                    if (x + 1 < fills) rows_of((x + 1) % stages);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 128 * CH / 32; ++i) {
                    const int r = (i * 32 + lane) / CH, c = lane % CH;  // 32 / CH rows at a time
                    const int64_t o = __shfl_sync(JINF_FULL_MASK, from[i * 32 / CH / 32], r & 31);
                    if (r < cols)
                        cp16_or_zero(dst + (c >> 3) * ATOM + r * 128 + (((c & 7) ^ (r & 7)) << 4), p.q + (o < 0 ? 0 : o) + c * 16,
                                     o >= 0);
                }
                cp_commit();
                if (x + 1 < fills) rows_of((x + 1) % stages);  // while the copies are under way
                cp_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                arrive_warp(ms.q_full[s]);
            }
            fill += fills;
        }
        if (!ok && lane == 0)  // leave no copy in flight
            for (uint32_t f = boxed > 2 ? boxed - 2 : 0; f < boxed; ++f) mb_wait(su32(&ms.q_full[f & 1]), (f >> 1) & 1);
    } else {
        const int w = (warp - 4) >> 2, key_in = 32 * (warp & 3) + lane;
        const uint32_t t_s = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const float c2 = p.scale * LOG2E;
        uint32_t fill = 0, item = 0, meets = 0;
        bool ok = true;
        while (ok && share.next(p, sg)) {
            const int rows = active_nodes(p, weight, sg.seq, nullptr) * p.group, stages = (rows + 127) / 128;
            const uint32_t* mask = p.mask ? p.mask + sg.seq * p.mask_seq : nullptr;
            float* mp = mass + ((size_t)sg.seq * p.n_kv_heads + sg.head) * p.max_ctx;
            for (int t = sg.t0; ok && t < sg.t1;) {
                const int n = min(set_of(stages), sg.t1 - t), items = n * stages;
                float acc[KT] = {0.f, 0.f, 0.f, 0.f};
                int seen = -1, released = 0;  // stages whose factors were waited for, and given back
                uint32_t va[32], vb[32];
                float old = 0.f, next_old = 0.f;
                // waits for item i and begins to read it
                auto open = [&](int i) {
                    const int st = i / n;
                    for (; ok && seen < st; ++seen) ok = wait(ms.r_full[(fill + seen + 1) % NR], ((fill + seen + 1) / NR) & 1);
                    if (!ok) return;
                    if (stages == 1) {
                        const int key = (t + i) * KV_TILE + key_in;
                        next_old = key < sg.past ? mp[key] : 0.f;
                    }
                    const uint32_t b = (item + i) % NB;
                    if (!(ok = wait(ms.s_full[b], ((item + i) / NB) & 1))) return;
                    tc_after_sync();
                    tmem_ld32(t_s + 128 * b, vb);
                };
                int i = (int)((w + GROUPS - item % GROUPS) % GROUPS);
                if (i < items) open(i);
                for (; ok && i < items; i += GROUPS) {
                    const int st = i / n, j = i - st * n, s = (fill + st) % NR;
                    const int cols = min(128, (rows - 128 * st + 31) & ~31);
                    const uint32_t b = (item + i) % NB;
                    const int key = (t + j) * KV_TILE + key_in;
                    const bool tail = (t + j + 1) * KV_TILE > sg.past;
                    old = next_old;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
                    for (int c = 0; ok && c < cols; c += 32) {
                        tmem_wait_ld();
                        tmem_pin32(vb);
#pragma unroll
                        for (int x = 0; x < 32; ++x) va[x] = vb[x];
                        if (c + 32 < cols) {
                            tmem_ld32(t_s + 128 * b + c + 32, vb);
                        } else {  // all read: the MMAs may use the buffer again; on to the next
                            tc_before_sync();
                            arrive_warp(ms.s_free[b]);
                            if (i + GROUPS < items) open(i + GROUPS);
                        }
                        if (tail) {  // a tree row counts where the query's node sees it
                            // this lane: the warp's 32 keys that query row c + lane sees
                            const uint32_t mine = seen_keys(p, mask, ms.row_node[s][c + lane], key - lane - sg.past);
#pragma unroll
                            for (int x = 0; x < 32; ++x) {
                                const float2 f = ms.row[s][c + x];
                                const uint32_t see = __shfl_sync(JINF_FULL_MASK, mine, x) >> lane;
                                const float e = fmaf(__uint_as_float(va[x]), c2, f.x);
                                sum[x & 3] = fmaf(f.y, (see & 1u) && f.y != 0.f ? ex2(e) : 0.f, sum[x & 3]);
                            }
                        } else {
                            const float4* f = reinterpret_cast<const float4*>(ms.row[s] + c);
#pragma unroll
                            for (int x = 0; x < 16; ++x) {
                                const float4 q = f[x];
                                const float e0 = ex2(fmaf(__uint_as_float(va[2 * x]), c2, q.x));
                                const float e1 = ex2(fmaf(__uint_as_float(va[2 * x + 1]), c2, q.z));
                                sum[x & 1] = fmaf(q.y, e0, sum[x & 1]);
                                sum[2 + (x & 1)] = fmaf(q.w, e1, sum[2 + (x & 1)]);
                            }
                        }
                    }
                    if (!ok) break;
                    const float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    if (stages == 1) {
                        if (key < sg.past + p.n_nodes) mp[key] = old + all;
                    } else {
#pragma unroll
                        for (int x = 0; x < KT; ++x) acc[x] += x == j ? all : 0.f;
                    }
                    // stages before that of the group's next item
                    const int upto = i + GROUPS < items ? (i + GROUPS) / n : st + 1;
                    for (; released < upto; ++released) arrive_warp(ms.r_free[(fill + released) % NR]);
                }
                if (!ok) break;
                for (; ok && released < stages; ++released) {  // stages without an item of this group, in order
                    for (; ok && seen < released; ++seen) ok = wait(ms.r_full[(fill + seen + 1) % NR], ((fill + seen + 1) / NR) & 1);
                    if (ok) arrive_warp(ms.r_free[(fill + released) % NR]);
                }
                if (!ok) break;
                if (stages != 1) {  // the groups' sums of each key, in order
                    float(*sums)[KT][128] = ms.sums[meets & 1];
#pragma unroll
                    for (int j = 0; j < KT; ++j) sums[w][j][key_in] = acc[j];
                    arrive_warp(ms.meet);
                    if (!(ok = wait(ms.meet, meets & 1))) break;
                    ++meets;
                    for (int j = w; j < min(n, KT); j += GROUPS) {
                        const int key = (t + j) * KV_TILE + key_in;
                        if (key < sg.past + p.n_nodes)
                            mp[key] = (key < sg.past ? mp[key] : 0.f) + (sums[0][j][key_in] + sums[1][j][key_in]);
                    }
                }
                item += items;
                fill += stages;
                t += n;
            }
        }
    }
    tc_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <bool BF, int HD>
cudaError_t launch_mass_mma(const TreeParams& p, const float* lse, const float* weight, float* mass, cudaStream_t s) {
    CUtensorMap mk, mq;
    if (!kv_tile_map(&mk, p.k, p, BF, HD) ||
        !rows_map(&mq, p.q, BF, HD, p.n_heads, HD, p.n_nodes, p.q_node, p.n_seqs, p.q_seq, p.group, p.tile_nodes))
        return cudaErrorInvalidValue;
    const cudaError_t e = cudaFuncSetAttribute(k_mass_mma<BF, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, MassMma<HD>::TOTAL);
    if (e != cudaSuccess) return e;
    const int64_t tiles = (int64_t)p.n_seqs * p.n_kv_heads * ((p.max_past + p.n_nodes + KV_TILE - 1) / KV_TILE);
    const int sms = kv_device_sms();
    k_mass_mma<BF, HD><<<(unsigned)(tiles < sms ? tiles : sms), XT, MassMma<HD>::TOTAL, s>>>(mk, mq, p, lse, weight, mass);
    return cudaGetLastError();
}

}  // namespace

cudaError_t mass_mma_launch(const TreeParams& p, bool bf, int head_dim, const float* lse, const float* weight, float* mass,
                            cudaStream_t s) {
    if (head_dim == 64) return bf ? launch_mass_mma<true, 64>(p, lse, weight, mass, s) : launch_mass_mma<false, 64>(p, lse, weight, mass, s);
    return bf ? launch_mass_mma<true, 128>(p, lse, weight, mass, s) : launch_mass_mma<false, 128>(p, lse, weight, mass, s);
}

}  // namespace jinf
