// Draft-tree attention for many query rows (jinf_b200_tree_attention), sm_100a: the fifth-generation
// tensor cores, with the scores, the probabilities and the output accumulator in tensor memory.
//
// A CTA takes a block of up to 256 query rows (nodes x query heads of a kv head) over its share
// of key tiles (kv_ops.cuh), 128 keys a tile:
//   warp 0      copies K and V tiles (TMA boxes of 64 columns x 128 rows, 128B swizzle) into a ring;
//   warp 1      allocates tensor memory and issues the MMAs: S_w = Q_w K^T (both operands in shared
//               memory) and O_w += P_w V (P_w in tensor memory over S_w, V MN-major);
//   warps 2, 3  clean the V tiles that hold rows of the tree or reach past the last key: values
//               behind the end, and values that are not finite (a masked key's V would enter O as
//               0 * v), become 0, and the keys of the latter are noted;
//   warps 4-7, 8-11  two softmax groups, one thread per query row: read S_w, keep the running maximum
//               and sum, write P_w in the cache's type, and finish O_w.
// With more than 128 rows group w takes rows 128 w .. and both use every tile; with fewer the two
// groups take alternate tiles for the same rows and are joined at the end of a unit. Either way one
// group's softmax runs under the other's MMAs, and S, P and O never leave the SM.
//
// The accumulator is rescaled only when a row's maximum has grown by more than 2^8 since the last
// time: p is at most 2^8 then, which both 16-bit types and the fp32 sums hold with the precision
// that they have for p <= 1, and the rescaling (a read and a write of all of O) almost never runs.
// Every wait is bounded; one that runs out sets the workspace's error word and ends the CTA.
#include "kv_ops.cuh"
#include "tree_part.cuh"
#include "umma.cuh"

#include <math.h>

namespace jinf {
namespace {

constexpr int XT = 384;         // threads
constexpr int ATOM = 16384;     // 128 rows x 64 columns, 128B-swizzled
constexpr int BAD_SETS = 8;     // tail tiles whose notes may be alive at once (the ring holds fewer)
constexpr float GROW = 8.f;     // log2 of the growth of a maximum that is tolerated

template <int HD>
struct MmaSmem {
    static constexpr int TILE = ATOM * (HD / 64);
    static constexpr int ST = HD == 128 ? 5 : 10;  // ring stages (one K or V tile each)
    static constexpr int OFF_KV = 2 * TILE;
    static constexpr int OFF_MISC = OFF_KV + ST * TILE;
    struct Misc {
        uint64_t full[ST], empty[ST], vok[ST];
        uint64_t s_full[2], p_ready[2], pv_done[2], q_ready[2], flag_ok[2], join, drain;
        Share share;
        uint32_t tmem;
        int abort;
        uint32_t bad[BAD_SETS][2][4];  // one part per cleaning warp
        float jm[128], jl[128];
    };
    static constexpr int TOTAL = OFF_MISC + (int)sizeof(Misc) + 1024;
};
static_assert(MmaSmem<128>::TOTAL <= 232448 && MmaSmem<64>::TOTAL <= 232448, "shared memory");

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Tree rows 32 w .. 32 w + 31 that node t sees, as bits.
__device__ __forceinline__ uint32_t seen_word(const TreeParams& p, const uint32_t* mask, int t, int w) {
    if (w < 0 || w >= p.mask_words) return 0u;
    const int left = p.n_nodes - 32 * w;
    uint32_t x;
    if (mask) x = mask[t * p.mask_words + w];
    else x = t >= 32 * w + 31 ? 0xFFFFFFFFu : t < 32 * w ? 0u : (2u << (t - 32 * w)) - 1u;
    return left >= 32 ? x : x & ((1u << left) - 1u);
}
// Keys whose first is tree row u0 (negative: -u0 cached rows come first), 32 of them, as bits.
__device__ __forceinline__ uint32_t seen_keys(const TreeParams& p, const uint32_t* mask, int t, int u0) {
    if (u0 <= -32) return 0xFFFFFFFFu;
    if (u0 < 0) return (seen_word(p, mask, t, 0) << (-u0)) | ((1u << (-u0)) - 1u);
    return __funnelshift_r(seen_word(p, mask, t, u0 >> 5), seen_word(p, mask, t, (u0 >> 5) + 1), u0 & 31);
}

template <bool BF, int HD>
__global__ void __launch_bounds__(XT, 1)
    k_tree_mma(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const TreeParams p,
               uint16_t* __restrict__ out, float* __restrict__ lse, float* __restrict__ parts, int* __restrict__ err) {
    using SM = MmaSmem<HD>;
    constexpr int TILE = SM::TILE, ST = SM::ST;
    constexpr uint32_t ID_QK = umma_idesc(BF, 128, 128, false), ID_PV = umma_idesc(BF, 128, HD, true);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    typename SM::Misc& ms = *reinterpret_cast<typename SM::Misc*>(sm + SM::OFF_MISC);
    const uint32_t s_q = su32(sm), s_kv = s_q + SM::OFF_KV;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int block = blockIdx.x % p.row_blocks, group = blockIdx.x / p.row_blocks;
    const int row0 = block * p.block_rows, rows = min(p.block_rows, p.n_rows - row0);
    const bool two = rows > 128;  // two row tiles, one per softmax group; else alternate key tiles

    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            mb_init(su32(&ms.full[i]), 1);
            mb_init(su32(&ms.empty[i]), 1);
            mb_init(su32(&ms.vok[i]), 64);
        }
        for (int w = 0; w < 2; ++w) {
            mb_init(su32(&ms.s_full[w]), 1);
            mb_init(su32(&ms.p_ready[w]), 128);
            mb_init(su32(&ms.pv_done[w]), 1);
            mb_init(su32(&ms.q_ready[w]), 128);
            mb_init(su32(&ms.flag_ok[w]), 1);
        }
        mb_init(su32(&ms.join), 256);
        mb_init(su32(&ms.drain), 1);
        ms.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&ms.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 2) {
        const Share sh = share_begin(p, group, gridDim.x / p.row_blocks);
        if (lane == 0) ms.share = sh;
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t tmem = ms.tmem;
    Share share = ms.share;
    Segment sg;

    // a bounded wait that also ends when another role gave up
    auto wait = [&](uint64_t& bar, uint32_t parity) -> bool {
        const uint32_t b = su32(&bar);
        for (unsigned long long it = 0; it < MB_SPIN; ++it) {
            if (mb_try(b, parity)) return true;
            if ((it & 255) == 255 && *(volatile int*)&ms.abort) return false;
        }
        atomicExch(&ms.abort, 1);
        atomicExch(err, 1);
        return false;
    };
    // the same for a whole warp, which stays converged
    auto wait_all = [&](uint64_t& bar, uint32_t parity) -> bool {
        return __all_sync(JINF_FULL_MASK, wait(bar, parity));
    };
    // Ring positions of a segment of n tiles, from its base: K_0, then K_(i+1), V_i for every i (the
    // order in which the MMAs take them), the last V_i without a K.
    auto pos_k = [](int i) { return i ? 2 * i - 1 : 0; };
    auto pos_v = [](int i, int n) { return i + 1 < n ? 2 * i + 2 : 2 * n - 1; };

    if (warp == 0) {
        if (lane == 0) {  // ---- copies
            uint32_t pos = 0;
            bool ok = true;
            while (ok && share.next(p, sg)) {
                const int n = sg.t1 - sg.t0;
                for (int x = 0; ok && x < 2 * n; ++x, ++pos) {
                    // x-th of the order above
                    const bool is_k = x == 0 || ((x & 1) && x < 2 * n - 1);
                    const int i = x == 0 ? 0 : is_k ? (x + 1) / 2 : x == 2 * n - 1 ? n - 1 : x / 2 - 1;
                    const uint32_t slot = pos % ST, fill = pos / ST;
                    if (fill && !(ok = wait(ms.empty[slot], (fill - 1) & 1))) break;
                    const uint32_t bar = su32(&ms.full[slot]);
                    mb_expect(bar, TILE);
#pragma unroll
                    for (int a = 0; a < HD / 64; ++a)
                        tma_load_4d(s_kv + slot * TILE + a * ATOM, is_k ? &tmk : &tmv, 64 * a, (sg.t0 + i) * KV_TILE,
                                    sg.head, sg.seq, bar);
                }
            }
            if (!ok)  // leave no copy in flight
                for (uint32_t s = 0; s < ST && s < pos; ++s) mb_wait(su32(&ms.full[s]), ((pos - 1 - s) / ST) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {  // ---- MMAs
            uint32_t base = 0, np[2] = {0, 0}, nq[2] = {0, 0}, vok_ph = 0;
            bool ok = true;
            auto full = [&](uint32_t pos) { return wait(ms.full[pos % ST], (pos / ST) & 1); };
            auto qk = [&](int w, uint32_t pos) {
                tc_after_sync();
                const uint32_t a = s_q + w * TILE, b = s_kv + (pos % ST) * TILE;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * ATOM + (kk & 3) * 32;
                    umma_ss(tmem + 128 * w, umma_desc(a + off), umma_desc(b + off), ID_QK, kk > 0);
                }
                umma_commit(su32(&ms.s_full[w]));
            };
            auto pv = [&](int w, uint32_t pos, bool accumulate) {
                tc_after_sync();
                const uint32_t b = s_kv + (pos % ST) * TILE;
#pragma unroll
                for (int kk = 0; kk < KV_TILE / 16; ++kk)
                    umma_ts(tmem + 256 + 128 * w, tmem + 128 * w + 8 * kk, umma_desc(b + kk * 2048, ATOM), ID_PV,
                            accumulate || kk > 0);
                umma_commit(su32(&ms.pv_done[w]));
            };
            while (ok && share.next(p, sg)) {
                const int n = sg.t1 - sg.t0;
                if (!(ok = full(base))) break;
                for (int w = 0; w < (two ? 2 : 1); ++w) {
                    if (!(ok = wait(ms.q_ready[w], nq[w]++ & 1))) break;
                    qk(w, base);
                }
                if (!ok) break;
                umma_commit(su32(&ms.empty[base % ST]));
                if (!two && n > 1) {
                    const uint32_t k1 = base + pos_k(1);
                    if (!(ok = full(k1) && wait(ms.q_ready[1], nq[1]++ & 1))) break;
                    qk(1, k1);
                    umma_commit(su32(&ms.empty[k1 % ST]));
                }
                for (int i = 0; ok && i < n; ++i) {
                    const uint32_t v = base + pos_v(i, n);
                    const bool tail = (sg.t0 + i + 1) * KV_TILE > sg.past;
                    if (!(ok = full(v))) break;
                    if (tail) {
                        const uint32_t s = v % ST;
                        if (!(ok = wait(ms.vok[s], (vok_ph >> s) & 1))) break;
                        vok_ph ^= 1u << s;
                    }
                    // the tile whose scores come next in the group's turn
                    const int step = two ? 1 : 2;
                    const bool more = i + step < n;
                    const uint32_t k = base + pos_k(i + step);
                    for (int x = 0; x < (two ? 2 : 1); ++x) {
                        const int w = two ? x : i & 1;
                        if (!(ok = wait(ms.p_ready[w], np[w]++ & 1))) break;
                        pv(w, v, two ? i > 0 : i > 1);
                        if (tail) mb_arrive(su32(&ms.flag_ok[w]));
                        if (more) {
                            if (x == 0 && !(ok = full(k))) break;
                            qk(w, k);
                        }
                    }
                    if (!ok) break;
                    umma_commit(su32(&ms.empty[v % ST]));
                    if (more) umma_commit(su32(&ms.empty[k % ST]));
                }
                base += 2 * n;
            }
            if (!ok) {  // the MMAs already issued finish before the memory goes
                umma_commit(su32(&ms.drain));
                mb_wait(su32(&ms.drain), 0);
            }
        }
    } else if (warp < 4) {
        // ---- clean the tail tiles' V
        uint32_t base = 0, ord = 0;
        bool ok = true;
        while (ok && share.next(p, sg)) {
            const int n = sg.t1 - sg.t0, n_keys = sg.past + p.n_nodes;
            for (int i = max(0, sg.past / KV_TILE - sg.t0); i < n; ++i, ++ord) {
                const uint32_t pos = base + pos_v(i, n);
                if (!(ok = wait_all(ms.full[pos % ST], (pos / ST) & 1))) break;
                uint32_t* bad = ms.bad[ord % BAD_SETS][warp - 2];
                if (lane < 4) bad[lane] = 0;
                __syncwarp();
                uint8_t* v = sm + SM::OFF_KV + (pos % ST) * TILE;
                const int key0 = (sg.t0 + i) * KV_TILE;
                for (int x = tid - 64; x < TILE / 16; x += 64) {
                    const int kk = (x >> 3) & 127, key = key0 + kk;
                    if (key < sg.past) continue;
                    uint4* at = reinterpret_cast<uint4*>(v) + x;
                    uint4 y = *at;
                    bool change = false;
                    if (key >= n_keys) {
                        y = make_uint4(0u, 0u, 0u, 0u);
                        change = true;
                    } else {
                        uint32_t* w = reinterpret_cast<uint32_t*>(&y);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (nonfinite2<BF>(w[e])) {
                                if (nonfinite2<BF>(w[e] & 0xFFFFu)) w[e] &= 0xFFFF0000u;
                                if (nonfinite2<BF>(w[e] & 0xFFFF0000u)) w[e] &= 0xFFFFu;
                                change = true;
                            }
                        if (change) atomicOr(&bad[kk >> 5], 1u << (kk & 31));
                    }
                    if (change) *at = y;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mb_arrive(su32(&ms.vok[pos % ST]));
            }
            base += 2 * n;
        }
    } else {
        // ---- softmax groups
        const int w = (warp - 4) >> 2, r = tid - 128 - 128 * w;  // row of the group's tile
        const int br = two ? 128 * w + r : r;                     // row of the block
        const bool valid = br < rows, warp_on = (two ? 128 * w : 0) + 32 * (warp & 3) < rows;
        const int rr = valid ? row0 + br : row0, node = rr / p.group, head_in = rr % p.group;
        const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t t_s = tmem + lane_off + 128 * w, t_o = tmem + lane_off + 256 + 128 * w;
        const float c2 = p.scale * LOG2E, grow = GROW / c2;
        const int step = two ? 1 : 2;
        uint32_t done = 0, tails = 0, ord = 0;  // tiles of this group; its tail tiles; the CTA's tail tiles
        uint32_t joins = 0;
        bool ok = true;
        auto meet = [&]() {  // both groups
            mb_arrive(su32(&ms.join));
            return wait_all(ms.join, joins++ & 1);
        };
        while (ok && share.next(p, sg)) {
            const int n = sg.t1 - sg.t0;
            const uint32_t* mask = p.mask ? p.mask + sg.seq * p.mask_seq : nullptr;
            const int first_tail = max(0, sg.past / KV_TILE - sg.t0);  // of the segment
            const bool mine = two || w < n;                            // the group has a tile
            float m = -INFINITY, l = 0.f;
            if (mine) {
                if (valid) {
                    const uint4* src = reinterpret_cast<const uint4*>(
                        p.q + (sg.seq * p.q_seq + node * p.q_node + (int64_t)(sg.head * p.group + head_in) * HD) * 2);
                    uint8_t* dst = sm + w * TILE + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
                    for (int c = 0; c < HD / 8; ++c)
                        *reinterpret_cast<uint4*>(dst + (c >> 3) * ATOM + (((c & 7) ^ (r & 7)) << 4)) = __ldg(src + c);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mb_arrive(su32(&ms.q_ready[w]));
            }
            for (int i = two ? 0 : w; i < n; i += step) {
                const bool tail = i >= first_tail;
                if (!(ok = wait_all(ms.s_full[w], done & 1))) break;
                tc_after_sync();
                if (warp_on) {
                    const int u0 = (sg.t0 + i) * KV_TILE - sg.past;
                    // two columns blocks of 32 scores at a time; read again below rather than kept, which
                    // would take 128 registers
                    auto scores = [&](int c, uint32_t (&a)[32], uint32_t (&b)[32]) {
                        tmem_ld32(t_s + 32 * c, a);
                        tmem_ld32(t_s + 32 * c + 32, b);
                        tmem_wait_ld();
                        tmem_pin32(a);
                        tmem_pin32(b);
                        if (tail) {
                            const uint32_t sa = seen_keys(p, mask, node, u0 + 32 * c);
                            const uint32_t sb = seen_keys(p, mask, node, u0 + 32 * c + 32);
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                if (!((sa >> j) & 1u)) a[j] = 0xFF800000u;
                                if (!((sb >> j) & 1u)) b[j] = 0xFF800000u;
                            }
                        }
                    };
                    uint32_t va[32], vb[32];
                    float mx = -INFINITY;
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        scores(c, va, vb);
#pragma unroll
                        for (int j = 0; j < 32; ++j) mx = fmaxf(mx, fmaxf(__uint_as_float(va[j]), __uint_as_float(vb[j])));
                    }
                    if (i < step) {
                        m = mx;
                    } else {
                        const bool need = mx > m + grow;  // also when nothing was seen yet (m = -inf)
                        if (__any_sync(JINF_FULL_MASK, need)) {
                            const float f = need ? ex2((m - mx) * c2) : 1.f;
                            if (need) m = mx;
                            l *= f;
                            ok = wait_all(ms.pv_done[w], (done - 1) & 1);
                            tc_after_sync();
                            for (int c = 0; c < HD / 32; ++c) {
                                uint32_t o[32];
                                tmem_ld32(t_o + 32 * c, o);
                                tmem_wait_ld();
                                tmem_pin32(o);
#pragma unroll
                                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                                tmem_st32(t_o + 32 * c, o);
                            }
                            tmem_wait_st();
                        }
                    }
                    const float mb = m == -INFINITY ? 0.f : m * c2;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        scores(c, va, vb);
                        uint32_t pk[32];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const float a = ex2(fmaf(__uint_as_float(va[2 * j]), c2, -mb));
                            const float b = ex2(fmaf(__uint_as_float(va[2 * j + 1]), c2, -mb));
                            const float e = ex2(fmaf(__uint_as_float(vb[2 * j]), c2, -mb));
                            const float f = ex2(fmaf(__uint_as_float(vb[2 * j + 1]), c2, -mb));
                            sum[0] += a;
                            sum[1] += b;
                            sum[2] += e;
                            sum[3] += f;
                            pk[j] = pack2<BF>(a, b);
                            pk[16 + j] = pack2<BF>(e, f);
                        }
                        // over scores of column 32 c / 2 and on, which have been read
                        tmem_st32(t_s + 16 * c, pk);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_wait_st();
                }
                tc_before_sync();
                mb_arrive(su32(&ms.p_ready[w]));
                ++done;
                if (tail) {
                    const uint32_t(*notes)[4] = ms.bad[(ord + i - first_tail) % BAD_SETS];
                    if (!(ok = wait_all(ms.flag_ok[w], tails++ & 1))) break;
                    uint32_t any = 0;
#pragma unroll
                    for (int x = 0; x < 4; ++x) any |= notes[0][x] | notes[1][x];
                    if (any && warp_on) {  // values that are not finite, to the rows that see their key
                        ok = wait_all(ms.pv_done[w], (done - 1) & 1);
                        tc_after_sync();
                        for (int kk = 0; kk < KV_TILE; ++kk) {
                            if (!(((notes[0][kk >> 5] | notes[1][kk >> 5]) >> (kk & 31)) & 1u)) continue;
                            const int key = (sg.t0 + i) * KV_TILE + kk;
                            const bool see = valid && tree_sees(p, mask, node, key - sg.past);
                            const uint16_t* vr = reinterpret_cast<const uint16_t*>(
                                p.v + (sg.seq * p.kv_seq + sg.head * p.kv_head + key * p.kv_row) * 2);
                            for (int c = 0; c < HD / 32; ++c) {
                                uint32_t o[32];
                                tmem_ld32(t_o + 32 * c, o);
                                tmem_wait_ld();
                                tmem_pin32(o);
#pragma unroll
                                for (int j = 0; j < 32; ++j) {
                                    const float x = to_f32<BF>(vr[32 * c + j]);
                                    if (see && !(fabsf(x) <= 3.4028235e38f)) o[j] = __float_as_uint(__uint_as_float(o[j]) + x);
                                }
                                tmem_st32(t_o + 32 * c, o);
                                tmem_wait_st();
                            }
                        }
                    }
                }
                if (!ok) break;
            }
            if (!ok) break;
            ord += n - min(n, first_tail);
            // ---- the unit's rows, or this group's part of them
            if (mine) {
                if (!(ok = wait_all(ms.pv_done[w], (done - 1) & 1))) break;
                tc_after_sync();
            }
            const bool whole = sg.t0 == 0 && sg.t1 == sg.tiles;
            const size_t orow = ((size_t)sg.seq * p.n_nodes + node) * p.n_heads + sg.head * p.group + head_in;
            float* part = parts + ((size_t)blockIdx.x * 2 + (sg.t0 == 0 ? 1 : 0)) * part_floats(p.block_rows, HD);
            const bool join = !two && n > 1;
            float* js = reinterpret_cast<float*>(sm);  // [128][HD], 16-byte chunk c of row r at c ^ (r & 7), over Q
            float f0 = 1.f, f1 = 0.f;
            if (join) {
                if (!(ok = meet())) break;  // both groups' MMAs over Q are done
                if (w == 1) {
                    if (warp_on) {
                        for (int c = 0; c < HD / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld32(t_o + 32 * c, o);
                            tmem_wait_ld();
                            tmem_pin32(o);
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                *reinterpret_cast<uint4*>(js + r * HD + (((8 * c + j) ^ (r & 7)) << 2)) =
                                    make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                        }
                        ms.jm[r] = m;
                        ms.jl[r] = l;
                    }
                }
                if (!(ok = meet())) break;
                if (w == 0 && warp_on) {
                    const float m1 = ms.jm[r], mj = fmaxf(m, m1), bj = mj == -INFINITY ? 0.f : mj;
                    f0 = ex2((m - bj) * c2);
                    f1 = ex2((m1 - bj) * c2);
                    l = l * f0 + ms.jl[r] * f1;
                    m = mj;
                }
            }
            if (warp_on && (two || w == 0)) {
                const float inv = whole ? (l > 0.f ? 1.f / l : l == 0.f ? 1.f : l) : 1.f;  // an empty row stays 0
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(t_o + 32 * c, o);
                    tmem_wait_ld();
                    tmem_pin32(o);
                    float x[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(o[j]);
                    if (join) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float4 y = *reinterpret_cast<const float4*>(js + r * HD + (((8 * c + j) ^ (r & 7)) << 2));
                            x[4 * j] = x[4 * j] * f0 + y.x * f1;
                            x[4 * j + 1] = x[4 * j + 1] * f0 + y.y * f1;
                            x[4 * j + 2] = x[4 * j + 2] * f0 + y.z * f1;
                            x[4 * j + 3] = x[4 * j + 3] * f0 + y.w * f1;
                        }
                    }
                    if (!valid) continue;
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<uint4*>(out + orow * HD + 32 * c + 8 * j) =
                                make_uint4(pack2<BF>(x[8 * j] * inv, x[8 * j + 1] * inv),
                                           pack2<BF>(x[8 * j + 2] * inv, x[8 * j + 3] * inv),
                                           pack2<BF>(x[8 * j + 4] * inv, x[8 * j + 5] * inv),
                                           pack2<BF>(x[8 * j + 6] * inv, x[8 * j + 7] * inv));
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<float4*>(part + ((size_t)(8 * c + j) * p.block_rows + br) * 4) =
                                make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
                    }
                }
                if (valid) {
                    if (whole) {
                        if (lse) lse[orow] = l == 0.f ? -INFINITY : m * p.scale + logf(l);
                    } else {
                        part[(size_t)p.block_rows * HD + br] = m;
                        part[(size_t)p.block_rows * (HD + 1) + br] = l;
                    }
                }
            }
            if (join && !(ok = meet())) break;  // Q's memory is free again
            tc_before_sync();
        }
    }
    tc_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    pdl_trigger();
}

bool make_map(CUtensorMap* map, const void* base, const TreeParams& p, int hd, bool bf) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)p.max_ctx, (cuuint64_t)p.n_kv_heads, (cuuint64_t)p.n_seqs};
    // the stride of an axis of one element is never used
    const cuuint64_t strides[3] = {(cuuint64_t)(p.max_ctx > 1 ? p.kv_row * 2 : 256),
                                   (cuuint64_t)(p.n_kv_heads > 1 ? p.kv_head * 2 : 256),
                                   (cuuint64_t)(p.n_seqs > 1 ? p.kv_seq * 2 : 256)};
    const cuuint32_t box[4] = {64, (cuuint32_t)KV_TILE, 1, 1}, estr[4] = {1, 1, 1, 1};
    return enc(map, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims,
               strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF, int HD>
cudaError_t launch_mma(const TreeParams& p, const TreePlan& plan, uint16_t* out, float* lse, float* parts, int* err,
                       cudaStream_t s) {
    CUtensorMap mk, mv;
    if (!make_map(&mk, p.k, p, HD, BF) || !make_map(&mv, p.v, p, HD, BF)) return cudaErrorInvalidValue;
    const cudaError_t e =
        cudaFuncSetAttribute(k_tree_mma<BF, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, MmaSmem<HD>::TOTAL);
    if (e != cudaSuccess) return e;
    k_tree_mma<BF, HD><<<plan.n_groups * plan.row_blocks, XT, MmaSmem<HD>::TOTAL, s>>>(mk, mv, p, out, lse, parts, err);
    return cudaGetLastError();
}

}  // namespace

bool tree_mma_fits(const jinf_b200_kv* kv) {
    auto ok = [](int n, int64_t stride) { return n == 1 || (stride > 0 && stride * 2 < ((int64_t)1 << 40)); };
    return ok(kv->max_ctx, kv->row_stride) && ok(kv->n_kv_heads, kv->head_stride) && ok(kv->n_seqs, kv->seq_stride);
}

cudaError_t tree_mma_launch(const TreeParams& p, const TreePlan& plan, bool bf, int head_dim, uint16_t* out, float* lse,
                            float* parts, int* err, cudaStream_t s) {
    if (head_dim == 64)
        return bf ? launch_mma<true, 64>(p, plan, out, lse, parts, err, s) : launch_mma<false, 64>(p, plan, out, lse, parts, err, s);
    return bf ? launch_mma<true, 128>(p, plan, out, lse, parts, err, s) : launch_mma<false, 128>(p, plan, out, lse, parts, err, s);
}

}  // namespace jinf
