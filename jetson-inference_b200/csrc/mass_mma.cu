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
//   warp 3      brings 128 query rows into one of two stages, with the exponent's constant of each
//               (w e^(s - lse) = 2^(s log2 e + log2 w - lse log2 e)):
//               boxes of whole nodes by TMA when every node counts and nodes fill a stage evenly, else
//               the rows of weight > 0 one by one (16-byte asynchronous copies into the 128B-swizzled
//               layout; about 4000 cycles a stage where the boxes take 1500);
//   warps 4-11  two groups, one thread per key, one group per tile parity: 64 columns of two tiles into
//               registers, then w e^(s - lse) added up. A key's sum has one owner and one order.
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
constexpr int MASK_WORDS = JINF_TREE_MAX_NODES / 32, MASK_PITCH = MASK_WORDS + 1;  // odd: no bank conflicts down the rows

template <int HD>
struct MassMma {
    static constexpr int TILE = ATOM * (HD / 64);
    static constexpr int OFF_Q = KT * TILE;
    static constexpr int OFF_MISC = OFF_Q + 2 * TILE;
    struct Misc {
        uint64_t k_full[KT], k_free[KT], q_full[2], q_free[2], r_full[NR], r_free[NR], s_full[NB], s_free[NB], stagger, drain[2];
        Share share;
        uint32_t tmem;
        int abort;
        alignas(16) float bias[NR][128];    // of a stage's query rows: log2(weight) - lse log2 e
        uint32_t seen[NR][128][MASK_PITCH];  // where the stage meets tree rows: those that each row's node sees
        uint8_t node[JINF_TREE_MAX_NODES];  // nodes of weight > 0, ascending (warp 3's)
    };
    static constexpr int TOTAL = OFF_MISC + (int)sizeof(Misc) + 1024;
};
static_assert(MassMma<128>::TOTAL + 64 <= 232448, "shared memory");
static_assert(JINF_TREE_MAX_NODES <= 256, "node numbers are kept in bytes");
static_assert(GROUPS == 2 && NB == 4 && KT == 4, "two buffers, an issuer and a group per tile parity");

// Nodes of weight > 0, by a whole warp; their numbers, ascending, to `list` where it is not null.
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
        const bool on = t < p.n_nodes && weight[(size_t)seq * p.n_nodes + t] > 0.f;
        const uint32_t b = __ballot_sync(JINF_FULL_MASK, on);
        if (on && list) list[n + __popc(b & ((1u << lane) - 1u))] = (uint8_t)t;
        n += __popc(b);
    }
    return n;
}

// Keys whose first is tree row u0 (negative: -u0 cached rows come first), 32 of them, of the words of a row.
__device__ __forceinline__ uint32_t keys_seen(const uint32_t* words, int u0) {
    if (u0 <= -32) return 0xFFFFFFFFu;
    const int w = u0 >> 5;  // -1 where the first tree row is among the 32
    const uint32_t lo = w < 0 ? 0xFFFFFFFFu : w < MASK_WORDS ? words[w] : 0u;
    const uint32_t hi = w + 1 < MASK_WORDS ? words[w + 1] : 0u;
    return __funnelshift_r(lo, hi, u0 & 31);
}
// Bit j of lane i becomes bit i of lane j (five exchanges of halves).
__device__ __forceinline__ uint32_t transpose32(uint32_t x) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t m = 0x0000FFFFu;  // the low s bits of every 2 s
#pragma unroll
    for (uint32_t s = 16; s > 0; s >>= 1) {
        const uint32_t y = __shfl_xor_sync(JINF_FULL_MASK, x, s);
        x = lane & s ? (x & ~m) | ((y >> s) & m) : (x & m) | ((y & m) << s);
        m ^= m << (s >> 1);
    }
    return x;
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
        mb_init(su32(&ms.stagger), 4);
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
    // in order (a score buffer belongs to the issuer and the group of its tile's parity).
    auto wait = [&](uint64_t& bar, uint32_t parity) { return mb_wait_warp(su32(&bar), parity, &ms.abort, p.err); };
    auto arrive_warp = [&](uint64_t& bar) {
        __syncwarp();
        if (lane == 0) mb_arrive(su32(&bar));
    };
    // Every role walks the same loops: segments, then sets of key tiles, for each set stages of 128 query
    // rows, for each stage the set's tiles, a score buffer per (stage, tile). With
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
        const int turn = warp - 1;  // tiles of this parity
        const bool leader = elect_one();
        uint32_t pos = 0, fill = 0, mine = 0;
        bool ok = true;
        while (ok && share.next(p, sg)) {
            const int rows = active_nodes(p, weight, sg.seq, nullptr) * p.group, stages = (rows + 127) / 128;
            if (rows == 0) continue;
            // With several stages the exponentials bind: the second group starts half a stage after the first,
            // so that one's waits and reads fall into the other's sums instead of leaving both waiting.
            if (turn && mine == 0 && stages > 1 && !(ok = wait(ms.stagger, 0))) break;
            for (int t = sg.t0; ok && t < sg.t1;) {
                const int n = min(set_of(stages), sg.t1 - t);
                for (int st = 0; ok && st < stages; ++st, ++fill) {
                    if (!(ok = wait(ms.q_full[fill & 1], (fill >> 1) & 1))) break;
                    const int cols = min(128, (rows - 128 * st + 31) & ~31);
                    const uint32_t idesc = umma_idesc(BF, 128, 0, false) | ((uint32_t)(cols >> 3) << 17);
                    const uint64_t dq = umma_desc(s_q + (fill & 1) * TILE);
                    for (int j = 0; ok && j < n; ++j) {
                        const uint32_t slot = (pos + j) % KT;
                        if (st == 0 && !(ok = wait(ms.k_full[slot], ((pos + j) / KT) & 1))) break;
                        if ((j & 1) == turn) {
                            const uint32_t b = turn + 2 * (mine & 1);
                            if (mine >= 2 && !(ok = wait(ms.s_free[b], ((mine >> 1) - 1) & 1))) break;
                            ++mine;
                            tc_after_sync();
                            if (leader) {
                                const uint64_t dk = umma_desc(s_k + slot * TILE);
#pragma unroll
                                for (int kk = 0; kk < HD / 16; ++kk) {
                                    const uint32_t off = ((kk >> 2) * ATOM + (kk & 3) * 32) >> 4;
                                    umma_ss(tmem + 128 * b, dk + off, dq + off, idesc, kk > 0);
                                }
                                umma_commit(su32(&ms.s_full[b]));
                            }
                        }
                        if (st == stages - 1 && leader) umma_commit(su32(&ms.k_free[slot]));
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
            const uint32_t* mask = p.mask ? p.mask + sg.seq * p.mask_seq : nullptr;
            const bool boxes = rows == p.n_rows && 128 % p.group == 0;
            const int fills = stages > 1 ? (sg.t1 - sg.t0 + KT - 1) / KT * stages : 1;
            // lane l has rows l, l + 32, ..: where they are (-1: zeros), constant, node
            int64_t from[4];
            float bias[4];
            int node[4];
            auto rows_of = [&](int st) {
                float l[4], wt[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int rr = 128 * st + 32 * k + lane;
                    from[k] = -1;
                    bias[k] = -INFINITY;
                    node[k] = 0;
                    l[k] = -INFINITY;
                    wt[k] = 1.f;
                    if (rr < rows) {
                        node[k] = list[rr / p.group];
                        const int h = sg.head * p.group + rr % p.group;
                        from[k] = (sg.seq * p.q_seq + node[k] * p.q_node + (int64_t)h * HD) * 2;
                        l[k] = lse[((size_t)sg.seq * p.n_nodes + node[k]) * p.n_heads + h];
                        if (weight) wt[k] = weight[(size_t)sg.seq * p.n_nodes + node[k]];
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (l[k] != -INFINITY) bias[k] = fmaf(-l[k], LOG2E, log2f(wt[k]));
                    else from[k] = -1;  // a row that attended nothing adds nothing, whatever it holds
                }
            };
            rows_of(0);
            for (int x = 0; x < fills; ++x) {
                const uint32_t f = fill + x, s = f & 1;
                const int cols = min(128, (rows - 128 * (x % stages) + 31) & ~31), rs = f % NR;
                // the set's tiles, or with one stage all of the segment's, reach the tree's rows
                const bool meets = (stages > 1 ? min(sg.t1, sg.t0 + (x / stages + 1) * KT) : sg.t1) * KV_TILE > sg.past;
                if (f >= NR && !(ok = wait(ms.r_free[rs], (f / NR - 1) & 1))) break;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    ms.bias[rs][32 * k + lane] = bias[k];
                    if (meets) {
                        uint32_t words[MASK_WORDS];
#pragma unroll
                        for (int x = 0; x < MASK_WORDS; ++x) words[x] = seen_word(p, mask, node[k], x);
#pragma unroll
                        for (int x = 0; x < MASK_WORDS; ++x) ms.seen[rs][32 * k + lane][x] = words[x];
                    }
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
        const int w = (warp - 4) >> 2, key_in = 32 * (warp & 3) + lane;  // tiles of parity w
        const uint32_t t_s = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128 * w;
        const float c2 = p.scale * LOG2E;
        uint32_t fill = 0, mine = 0;
        bool ok = true;
        while (ok && share.next(p, sg)) {
            const int rows = active_nodes(p, weight, sg.seq, nullptr) * p.group, stages = (rows + 127) / 128;
            float* mp = mass + ((size_t)sg.seq * p.n_kv_heads + sg.head) * p.max_ctx + key_in;
            const int past = sg.past - key_in, end = past + p.n_nodes;  // of keys counted from key_in
            for (int t = sg.t0; ok && t < sg.t1;) {
                const int n = min(set_of(stages), sg.t1 - t);
                float acc[2] = {0.f, 0.f};  // several stages: of the set's tiles w and w + 2
                for (int st = 0; ok && st < stages; ++st, ++fill) {
                    const uint32_t rs = fill % NR;
                    if (!(ok = wait(ms.r_full[rs], (fill / NR) & 1))) break;
                    const int cols = rows - 128 * st;
                    // Two tiles at a time: a row's constant, a broadcast read of shared memory, serves both
                    // (one read a score would keep shared memory busier than the exponentials).
                    for (int j = w; ok && j < n; j += 4) {
                        const int key0 = (t + j) * KV_TILE, cnt = j + 2 < n ? 2 : 1;
                        const uint32_t b0 = mine & 1, b1 = b0 ^ 1;
                        float old0 = 0.f, old1 = 0.f;
                        if (stages == 1) {
                            if (key0 < past) old0 = mp[key0];
                            if (cnt == 2 && key0 + 2 * KV_TILE < past) old1 = mp[key0 + 2 * KV_TILE];
                        }
                        ok = wait(ms.s_full[w + 2 * b0], (mine >> 1) & 1);
                        if (ok && cnt == 2) ok = wait(ms.s_full[w + 2 * b1], ((mine + 1) >> 1) & 1);
                        if (!ok) break;
                        tc_after_sync();
                        const bool tail = key0 + (2 * cnt - 1) * KV_TILE > sg.past;
                        float s0[2] = {0.f, 0.f}, s1[2] = {0.f, 0.f};
#pragma unroll 1
                        for (int c = 0; c < 128; c += 64) {
                            // columns past the stage's rows hold scores of zeros, or of constant -inf
                            const bool on = c < cols, last = c + 64 >= min(cols, 128);
                            if (!on) break;
                            uint32_t va[2][32], vb[2][32];
                            tmem_ld32(t_s + 256 * b0 + c, va[0]);
                            tmem_ld32(t_s + 256 * b0 + c + 32, va[1]);
                            tmem_ld32(t_s + 256 * b1 + c, vb[0]);
                            tmem_ld32(t_s + 256 * b1 + c + 32, vb[1]);
                            tmem_wait_ld();
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                tmem_pin32(va[h]);
                                tmem_pin32(vb[h]);
                            }
                            if (last) {  // read: the MMAs may use the buffers again
                                tc_before_sync();
                                arrive_warp(ms.s_free[w + 2 * b0]);
                                if (cnt == 2) arrive_warp(ms.s_free[w + 2 * b1]);
                                if (w == 0 && mine == 0) arrive_warp(ms.stagger);
                            }
                            if (tail) {
                                // A tree row counts where the query's node sees it: the warp's 32 keys that query
                                // row c + 32 h + lane sees (none for a row that counts nothing), turned into the
                                // rows that see this lane's key.
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const int col = c + 32 * h + lane, u0 = key0 + key_in - lane - sg.past;
                                    const uint32_t* words = ms.seen[rs][col];
                                    const bool counts = ms.bias[rs][col] != -INFINITY;
                                    const uint32_t sa = transpose32(counts ? keys_seen(words, u0) : 0u);
                                    const uint32_t sb = transpose32(counts ? keys_seen(words, u0 + 2 * KV_TILE) : 0u);
#pragma unroll
                                    for (int x = 0; x < 32; ++x) {
                                        if (!(sa & (1u << x))) va[h][x] = 0xFF800000u;
                                        if (!(sb & (1u << x))) vb[h][x] = 0xFF800000u;
                                    }
                                }
                            }
                            const float4* f = reinterpret_cast<const float4*>(ms.bias[rs] + c);
                            if (cnt == 2) {
#pragma unroll
                                for (int x = 0; x < 16; ++x) {
                                    const float4 q = f[x];
                                    const uint32_t *a = va[x >> 3] + 4 * (x & 7), *b = vb[x >> 3] + 4 * (x & 7);
                                    s0[0] += ex2(fmaf(__uint_as_float(a[0]), c2, q.x));
                                    s1[0] += ex2(fmaf(__uint_as_float(b[0]), c2, q.x));
                                    s0[1] += ex2(fmaf(__uint_as_float(a[1]), c2, q.y));
                                    s1[1] += ex2(fmaf(__uint_as_float(b[1]), c2, q.y));
                                    s0[0] += ex2(fmaf(__uint_as_float(a[2]), c2, q.z));
                                    s1[0] += ex2(fmaf(__uint_as_float(b[2]), c2, q.z));
                                    s0[1] += ex2(fmaf(__uint_as_float(a[3]), c2, q.w));
                                    s1[1] += ex2(fmaf(__uint_as_float(b[3]), c2, q.w));
                                }
                            } else {
#pragma unroll
                                for (int x = 0; x < 16; ++x) {
                                    const float4 q = f[x];
                                    const uint32_t* a = va[x >> 3] + 4 * (x & 7);
                                    s0[0] += ex2(fmaf(__uint_as_float(a[0]), c2, q.x));
                                    s0[1] += ex2(fmaf(__uint_as_float(a[1]), c2, q.y));
                                    s0[0] += ex2(fmaf(__uint_as_float(a[2]), c2, q.z));
                                    s0[1] += ex2(fmaf(__uint_as_float(a[3]), c2, q.w));
                                }
                            }
                        }
                        mine += cnt;
                        const float all0 = s0[0] + s0[1], all1 = s1[0] + s1[1];
                        if (stages == 1) {
                            if (key0 < end) mp[key0] = old0 + all0;
                            if (cnt == 2 && key0 + 2 * KV_TILE < end) mp[key0 + 2 * KV_TILE] = old1 + all1;
                        } else {
                            acc[0] += all0;
                            acc[1] += all1;
                        }
                    }
                    if (ok) arrive_warp(ms.r_free[rs]);
                }
                if (!ok) break;
                if (stages != 1) {  // none or several
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int j = w + 2 * x, key0 = (t + j) * KV_TILE;
                        if (j < n && key0 < end) mp[key0] = (key0 < past ? mp[key0] : 0.f) + acc[x];
                    }
                }
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
    const cudaError_t e = kv_allow_smem<k_mass_mma<BF, HD>>(MassMma<HD>::TOTAL);
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
