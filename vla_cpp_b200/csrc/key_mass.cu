// The attention weight that every cached row got from a call's query tokens, accumulated over calls:
//
//   m'[b][h][j] = decay m[b][h][j] + sum over the g heads of kv head h and the S tokens of  exp(scale q . k_j - lse)
//
// with the log-sum-exp of each query row given, so a row's weights need neither its maximum nor its sum.  The transposed product
// K Q^T puts keys on the lanes of TMEM and query rows on its columns: a thread owns one key and adds up its columns in
// registers -- nothing is reduced across threads but the parts of the columns, no atomics, the same bits every time.
//
// Work unit = (observation, kv head, 256 keys) for a pair of CTAs (tcgen05 cta_group::2, M = 256): each holds 128 keys and stages half
// of every chunk of query rows, so that an SM fetches half of what 128 keys of its own would need -- with a CTA per 128 keys the
// fetching of query rows took 2,000 cycles per 128 of them, twice the exponentials.  Persistent pairs walk the units:
//   loader warp      TMA: the unit's K tile and its query rows, chunks of at most NQ, through rings whose depths share 192 KB
//   MMA warp         even CTA: D[256 keys][n rows] = K Q_chunk^T, n = the chunk's rows rounded up to 32 (one token: 32 columns), NB
//                    accumulators; odd CTA: tells the even one what has landed
//   16 sum warps     four per lane quarter, 128 columns of every second (heads of 256: fourth) chunk each: p = 2^(s c - lse')
//
// One query token: K streams once, HBM bounds it.  Many: the exponentials (16 per clock and SM) at heads of 64 and 128, at 256 their sum
// with the product's chain.  Measured (graph replay, cold L2): 4 x 816 tokens, 20 / 5 heads of 128, over 4,097 to 8,190 keys 151 us (142 with
// the pages in L2), 90 of them the exponential unit's; a polynomial on the FMA pipe for every fourth or eighth of them was slower, though
// 38 % of the issue slots are in use: what held it up was not found.
// 64 x 51 tokens, 8 / 1 heads of 256, over 304 to 816 keys 26.6 us (20.5); one token over 16,001 keys 14 to 16 us (10.3).
#include <cuda_bf16.h>

#include "f32x2.cuh"
#include "host_common.h"
#include "ragged.cuh"
#include "tc5.cuh"

namespace vb {

constexpr int KM_PARTS = 4;  // sum warps per lane quarter
constexpr int KM_SUMS = 4 * KM_PARTS, KM_LOADER = KM_SUMS, KM_MMA = KM_SUMS + 1, KM_THREADS = 32 * (KM_SUMS + 2);

struct KeyMassParams {
    const float *lse;      // [n_obs][n_q][S]: an item's g * S rows in one piece
    const float *mass_in;  // [n_obs][n_kv][cap] or nullptr
    float *mass_out;
    const int32_t *lens, *pad;
    int R, n_obs, n_kv, cap, max_len, n_chunks, page0, box_rows, k_stages, q_stages;
    float scale_log2, decay;
    int *status;
};

template <int HD, int NQ_>
struct KeyMassSmem {
    static constexpr int CB = HD / 64;                // 64-element column blocks
    static constexpr int NQ = NQ_;                    // query rows per chunk
    static constexpr int NB = 512 / NQ;               // accumulators
    static constexpr int MAX_STAGES = 6;
    static constexpr int K_BYTES = CB * 128 * 128;    // [CB][128 keys][128 B]
    static constexpr int Q_BYTES = CB * (NQ / 2) * 128;  // [CB][box_rows][128 B]: this CTA's half of a chunk
    static constexpr int RING = 192 * 1024;
    static constexpr int BAR_OFF = RING;
    static constexpr int PPC = NQ / 128, G = KM_PARTS / PPC;  // parts that share a chunk, 128 columns each; groups of them
    static constexpr int LSE_OFF = BAR_OFF + 512;     // float [KM_SUMS][128]
    static constexpr int SUM_OFF = LSE_OFF + KM_SUMS * 128 * 4;  // float [2][KM_PARTS - 1][128]
    static constexpr int TOTAL = SUM_OFF + 2 * (KM_PARTS - 1) * 128 * 4 + 1024;
    static_assert(NB == G, "a group of sum warps has an accumulator of its own");
    static_assert(2 * K_BYTES + 2 * Q_BYTES <= RING && TOTAL <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ float km_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A stage of a ring and the parity its barriers are at.
struct KmStage {
    uint32_t i = 0, ph = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++i == n) {
            i = 0;
            ph ^= 1u;
        }
    }
};

template <int HD, int NQ>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(KM_THREADS, 1)
key_mass_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const KeyMassParams p) {
    using L = KeyMassSmem<HD, NQ>;
    extern __shared__ uint8_t km_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(km_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    constexpr int MS = L::MAX_STAGES;
    uint64_t *k_full = bars, *k_free = k_full + MS, *q_full = k_free + MS, *q_free = q_full + MS, *a_full = q_free + MS, *a_free = a_full + 4;
    uint64_t *meet = a_free + 4;  // [4] the warps of a lane quarter
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(meet + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;
    const WaitCtx wc{abort_flag, p.status};
    const uint32_t KS = p.k_stages, QS = p.q_stages;
    const uint32_t both = rank == 0 ? 2u : 1u;  // even CTA: its own TMA and the odd CTA's word

    if (threadIdx.x == 0) {
        for (int i = 0; i < MS; ++i) {
            mbar_init(&k_full[i], both);
            mbar_init(&k_free[i], 1);
            mbar_init(&q_full[i], both);
            mbar_init(&q_free[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&a_full[i], 1);
            mbar_init(&a_free[i], 2 * 4 * L::PPC);  // a chunk's sum warps in both CTAs (used in the even one)
            mbar_init(&meet[i], 32 * KM_PARTS);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    __syncthreads();
    cluster_sync_all();
    if (warp == KM_MMA) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&q_map);
        tma_prefetch_desc(&k_map);
    }
    pdl_launch_dependents();
    pdl_wait();

    // the keys of an observation that are there; the same for every role
    auto len_of = [&](int obs) { return p.lens ? min(max(p.lens[obs], 0), p.max_len) : p.max_len; };
    RaggedCursor cursor(len_of, p.n_obs, p.n_kv, 256);
    RaggedUnit unit;
    auto columns_of = [&](int c) { return (min(p.R - c * L::NQ, L::NQ) + 31) & ~31; };

    if (warp == KM_LOADER) {
        KmStage k, q;
        bool ok = true;
        const uint32_t q_stage = (uint32_t)(L::CB * p.box_rows * 128);
        uint8_t *const q_smem = smem + KS * L::K_BYTES;
        for (int ui = cid; ok && cursor.find(ui, unit); ui += ncl) {
            const int item = unit.obs * p.n_kv + unit.kvh, key0 = unit.block * 256 + (int)rank * 128;
            ok = warp_wait(&k_free[k.i], k.ph ^ 1u, wc, DEV_TIMEOUT_EMPTY);
            if (!ok) break;
            if (elect_one()) {
                mbar_expect_tx(&k_full[k.i], L::K_BYTES);
                for (int cb = 0; cb < L::CB; ++cb)
                    tma_load_3d(smem + k.i * L::K_BYTES + cb * 16384, &k_map, &k_full[k.i], cb * 64, key0, p.page0 + item);
            }
            k.next(KS);
            for (int c = 0; c < p.n_chunks; ++c) {
                ok = warp_wait(&q_free[q.i], q.ph ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                if (elect_one()) {
                    mbar_expect_tx(&q_full[q.i], q_stage);
                    const int row = c * L::NQ + (int)rank * (columns_of(c) >> 1);
                    for (int cb = 0; cb < L::CB; ++cb)
                        tma_load_3d(q_smem + q.i * q_stage + cb * p.box_rows * 128, &q_map, &q_full[q.i], cb * 64, row, item);
                }
                q.next(QS);
            }
        }
    } else if (warp == KM_MMA) {
        KmStage k, q, acc;
        bool ok = true;
        if (rank == 0) {  // the whole warp walks the units, one elected lane issues
            const uint32_t k_base = smem_u32(smem), q_base = k_base + KS * L::K_BYTES;
            const uint32_t q_cb = (uint32_t)p.box_rows * 128, q_stage = L::CB * q_cb;
            for (int ui = cid; ok && cursor.find(ui, unit); ui += ncl) {
                ok = warp_wait(&k_full[k.i], k.ph, wc, DEV_TIMEOUT_FULL);
                if (!ok) break;
                const uint32_t k_addr = k_base + k.i * L::K_BYTES;
                for (int c = 0; c < p.n_chunks; ++c) {
                    ok = warp_wait(&q_full[q.i], q.ph, wc, DEV_TIMEOUT_FULL);
                    if (ok) ok = warp_wait(&a_free[acc.i], acc.ph ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t idesc = make_idesc(1, 1, 1, 0, 0, 256, columns_of(c));
                    const uint32_t q_addr = q_base + q.i * q_stage, d = tmem_base + acc.i * L::NQ;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk)
                            mma_f16_pair(d, smem_desc_sw128(k_addr + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                                         smem_desc_sw128(q_addr + (kk >> 2) * q_cb + (kk & 3) * 32, 16, 1024), idesc, kk != 0 ? 1u : 0u);
                        tc_commit_pair(&a_full[acc.i], 3);
                        tc_commit_pair(&q_free[q.i], 3);
                        if (c + 1 == p.n_chunks) tc_commit_pair(&k_free[k.i], 3);
                    }
                    q.next(QS);
                    acc.next(L::NB);
                }
                k.next(KS);
            }
        } else {
            for (int ui = cid; ok && cursor.find(ui, unit); ui += ncl) {
                ok = warp_wait(&k_full[k.i], k.ph, wc, DEV_TIMEOUT_FULL);
                if (!ok) break;
                if (lane == 0) mbar_arrive_cluster(&k_full[k.i], 0);
                k.next(KS);
                for (int c = 0; c < p.n_chunks; ++c) {
                    ok = warp_wait(&q_full[q.i], q.ph, wc, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_cluster(&q_full[q.i], 0);
                    q.next(QS);
                }
            }
        }
    } else {
        // Parts in groups: a chunk is one group's, the next chunk the next group's, so that the groups are at different points of their work
        // (all of them on every chunk, a quarter of its columns each, they waited and computed in step).  Which group begins a
        // unit turns from unit to unit; `rel`, the group's place in that turn, says which chunks it adds up, and where its sum goes, so a
        // unit's sums do not depend on what the pair did before.  The groups meet at a unit's end: going on to the next one, with the sums handed to
        // the group that ends last, was slower (4 x 816 tokens, heads of 128, 141 us instead of 136 with the pages in L2), since the
        // accumulators are filled in order and either group's delay is the other's.  A unit that is one part's alone needs no
        // meeting and its group takes every G-th (one token over 16,001 rows 14 us, 16 with one unit at a time).
        constexpr int PPC = L::PPC, G = L::G, NBLK = 4;
        const int qtr = warp & 3, part = warp >> 2, sub = part % PPC, group = part / PPC;
        float *ls = reinterpret_cast<float *>(smem + L::LSE_OFF) + warp * 128;
        float *sum_s = reinterpret_cast<float *>(smem + L::SUM_OFF);
        const uint32_t lane_sel = (uint32_t)(qtr * 32) << 16;
        const F2 scale2 = f2(p.scale_log2, p.scale_log2);
        float lv[NBLK];  // the next chunk's lse, requested while this one is worked on
        auto fetch_lse = [&](bool there, const RaggedUnit &u, int c) {
#pragma unroll
            for (int i = 0; i < NBLK; ++i) {
                const int r = c * L::NQ + sub * 128 + i * 32 + lane;
                lv[i] = there && c < p.n_chunks && r < p.R ? p.lse[(long long)(u.obs * p.n_kv + u.kvh) * p.R + r] : -INFINITY;
            }
        };
        const bool alone = PPC == 1 && p.n_chunks == 1;
        uint32_t un = alone ? (uint32_t)group : 0u;  // units of the pair
        auto rel_of = [&](uint32_t u) { return alone ? 0 : (int)(((uint32_t)group + G - u % G) % G); };
        bool ok = true;
        bool there = cursor.find(cid + (int)un * ncl, unit);
        fetch_lse(there, unit, rel_of(un));
        while (ok && there) {
            const RaggedUnit now = unit;
            const uint32_t qu = un * (uint32_t)p.n_chunks, turn = un & 1u;  // chunks in front of this unit
            const int rel = rel_of(un);
            un += alone ? (uint32_t)G : 1u;
            const int rel_next = rel_of(un);
            there = cursor.find(cid + (int)un * ncl, unit);
            const int item = now.obs * p.n_kv + now.kvh, key0 = now.block * 256 + (int)rank * 128, obs = now.obs;
            F2 acc[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = f2(0.0f, 0.0f);
            if (rel >= p.n_chunks) fetch_lse(there, unit, rel_next);
            for (int c = rel; c < p.n_chunks; c += G) {
                const uint32_t q = qu + (uint32_t)c, ab = q % L::NB;
                // Rows past the last, and rows that saw nothing (-inf), weigh nothing: 2^(0 - inf).  Their scores may be anything (a column that
                // no row stands behind, a query that nobody wrote), so they are taken as 0: lane i keeps which ones of 32-column block i.
                unsigned unseen = 0;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < NBLK; ++i) {
                    const unsigned of_block = __ballot_sync(0xffffffffu, lv[i] == -INFINITY);
                    unseen = lane == i ? of_block : unseen;
                    ls[i * 32 + lane] = lv[i] == -INFINITY ? -INFINITY : -1.4426950408889634f * lv[i];
                }
                __syncwarp();
                if (c + G < p.n_chunks) fetch_lse(true, now, c + G);
                else fetch_lse(there, unit, rel_next);
                ok = warp_wait(&a_full[ab], q / L::NB & 1u, wc, DEV_TIMEOUT_ACCUM);
                if (!ok) break;
                tc_fence_after();
                const int n = min(p.R - c * L::NQ - sub * 128, 128);  // of this warp's columns; may be 0 or less
                const uint32_t d = tmem_base + lane_sel + ab * L::NQ + (uint32_t)(sub * 128);
#pragma unroll
                for (int b = 0; b < NBLK; ++b) {
                    uint32_t s[32];
                    if (b * 32 < n) {
                        tmem_ld32(d + (uint32_t)(b * 32), s);
                        tmem_ld_wait();
                    }
                    if (b + 1 == NBLK) {  // the accumulator is out of TMEM
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (rank == 0) mbar_arrive(&a_free[ab]);
                            else mbar_arrive_cluster(&a_free[ab], 0);
                        }
                    }
                    if (b * 32 >= n) continue;
                    const unsigned none = __shfl_sync(0xffffffffu, unseen, b);
                    if (none) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[e] = none & (1u << e) ? 0u : s[e];
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        const ulonglong2 la = *reinterpret_cast<const ulonglong2 *>(ls + b * 32 + e);
                        const ulonglong2 lb = *reinterpret_cast<const ulonglong2 *>(ls + b * 32 + e + 4);
                        const unsigned long long l[4] = {la.x, la.y, lb.x, lb.y};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const F2 t = f2_fma(f2(__uint_as_float(s[e + 2 * i]), __uint_as_float(s[e + 2 * i + 1])), scale2, F2{l[i]});
                            float t0, t1;
                            f2_get(t, t0, t1);
                            acc[i] = f2_add(acc[i], f2(km_ex2(t0), km_ex2(t1)));
                        }
                    }
                }
            }
            if (!ok) break;
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) f2_get(acc[i], x[2 * i], x[2 * i + 1]);
            float sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
            // the parts of the columns meet; the slots are used in turn, so one meeting per unit is enough
            float *slot = sum_s + turn * ((KM_PARTS - 1) * 128) + qtr * 32 + lane;
            const int place = rel * PPC + sub;
            if (!alone) {
                if (place) slot[(place - 1) * 128] = sum;
                mbar_arrive(&meet[qtr]);
                ok = warp_wait(&meet[qtr], turn, wc, DEV_TIMEOUT_MISC);
                if (!ok) break;
            }
            const int key = key0 + qtr * 32 + lane;
            if (!place && key < now.len) {
                if (!alone) {
#pragma unroll
                    for (int i = 0; i < KM_PARTS - 1; ++i) sum += slot[i * 128];
                }
                if (p.pad && key >= p.pad[2 * obs] && key < p.pad[2 * obs + 1]) sum = 0.0f;
                const long long at = (long long)item * p.cap + key;
                p.mass_out[at] = p.mass_in ? fmaf(p.decay, p.mass_in[at], sum) : sum;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA may exit while the other can still signal its barriers
    if (warp == KM_MMA) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <int HD, int NQ>
static int launch_key_mass(const vlab200_kv_store *st, const void *q, KeyMassParams &p, int max_units, cudaStream_t stream) {
    using L = KeyMassSmem<HD, NQ>;
    p.n_chunks = (p.R + L::NQ - 1) / L::NQ;
    p.box_rows = p.R >= L::NQ ? L::NQ / 2 : ((p.R + 31) & ~31) / 2;  // a multiple of 8: whole swizzle groups
    // A unit that takes its query rows in one chunk streams keys: the ring goes to K.  More chunks: K stays, query rows stream.
    const int q_stage = L::CB * p.box_rows * 128;
    p.q_stages = p.n_chunks > 1 ? (L::RING - 2 * L::K_BYTES) / q_stage : (L::RING - 4 * q_stage) / L::K_BYTES == (L::RING - 2 * q_stage) / L::K_BYTES ? 4 : 2;
    if (p.q_stages > L::MAX_STAGES) p.q_stages = L::MAX_STAGES;
    p.k_stages = (L::RING - p.q_stages * q_stage) / L::K_BYTES;
    if (p.k_stages > L::MAX_STAGES) p.k_stages = L::MAX_STAGES;
    CUtensorMap qmap, kmap;
    {
        const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)p.R, (uint64_t)st->n_obs * st->n_kv};
        const uint64_t strides[2] = {(uint64_t)HD * 2, (uint64_t)p.R * HD * 2};
        const uint32_t box[3] = {64, (uint32_t)p.box_rows, 1};
        if (int rc = make_tensor_map(&qmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    }
    {
        const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)st->cap, (uint64_t)st->n_layers * st->n_obs * st->n_kv};
        const uint64_t strides[2] = {(uint64_t)HD * 2, (uint64_t)st->cap * HD * 2};
        const uint32_t box[3] = {64, 128, 1};
        if (int rc = make_tensor_map(&kmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, st->k_pages, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
            return rc;
    }
    if (int rc = ensure_dyn_smem(key_mass_kernel<HD, NQ>, L::TOTAL)) return rc;
    const int pairs = sm_count() / 2;
    return launch_pdl(key_mass_kernel<HD, NQ>, dim3(2 * (max_units < pairs ? max_units : pairs)), dim3(KM_THREADS), L::TOTAL, stream, qmap, kmap, p);
}

}  // namespace vb

extern "C" int32_t vlab200_key_mass(const vlab200_kv_store *st, int32_t layer, const void *q, const float *lse, const float *mass_in,
                                    float *mass_out, int32_t S, int32_t n_q, const int32_t *lens, int32_t max_len,
                                    const int32_t *pad_ranges, float scale, float decay, void *stream) {
    if (!st || !st->k_pages || !q || !lse || !mass_out) return VLAB200_ERR_ARG;
    if (layer < 0 || layer >= st->n_layers || S <= 0 || n_q <= 0 || st->n_obs <= 0 || st->n_kv <= 0 || n_q % st->n_kv) return VLAB200_ERR_ARG;
    if (max_len < 0 || max_len > st->cap || !(scale >= 0.0f) || !(decay >= 0.0f)) return VLAB200_ERR_ARG;
    if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(st->k_pages) & 15)) return VLAB200_ERR_ARG;
    const int hd = st->head_dim;
    if (hd != 64 && hd != 128 && hd != 256) return VLAB200_ERR_UNSUPPORTED;
    const long long R = (long long)(n_q / st->n_kv) * S, tiles = (max_len + 255LL) / 256, units = vb::size_product({st->n_obs, st->n_kv, tiles});
    if (R > 0x7fffff00LL || units > 0x7fffff00LL || vb::size_product({st->n_layers, st->n_obs, st->n_kv}) > 0x7fffff00LL) {
        vb::set_last_error("key_mass: more than 2^31 query rows per kv head, pages or key tiles");
        return VLAB200_ERR_UNSUPPORTED;
    }
    if (max_len == 0) return VLAB200_OK;
    const long long items = (long long)st->n_obs * st->n_kv, q_b = vb::size_product({items, R, hd, 2}), mass_b = vb::size_product({items, st->cap, 4});
    const vb::MemRange out[] = {{mass_out, mass_b}};
    const vb::MemRange in[] = {{q, q_b}, {lse, vb::size_product({items, R, 4})}, {st->k_pages, vb::size_product({st->n_layers, items, st->cap, hd, 2})},
                               {lens, st->n_obs * 4LL}, {pad_ranges, st->n_obs * 8LL}, {mass_in == mass_out ? nullptr : mass_in, mass_b}};
    if (vb::writes_overlap(out, 1, in, 6)) return VLAB200_ERR_ARG;
    vb::KeyMassParams p;
    p.lse = lse;
    p.mass_in = decay == 0.0f ? nullptr : mass_in;
    p.mass_out = mass_out;
    p.lens = lens;
    p.pad = pad_ranges;
    p.R = (int)R;
    p.n_kv = st->n_kv;
    p.cap = st->cap;
    p.max_len = max_len;
    p.n_obs = st->n_obs;
    p.page0 = layer * st->n_obs * st->n_kv;
    p.scale_log2 = 1.4426950408889634f * (scale > 0.0f ? scale : 1.0f / sqrtf((float)hd));
    p.decay = decay;
    p.status = vb::device_status_ptr();
    if (!p.status) return vb::cuda_fail(cudaGetLastError(), "device_status_ptr");
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    // Rows that fill one chunk of 128 are one group's alone: four units at a time in four accumulators, instead of two in two.
    if (hd == 64) return R <= 128 ? vb::launch_key_mass<64, 128>(st, q, p, (int)units, cs) : vb::launch_key_mass<64, 256>(st, q, p, (int)units, cs);
    if (hd == 128) return R <= 128 ? vb::launch_key_mass<128, 128>(st, q, p, (int)units, cs) : vb::launch_key_mass<128, 256>(st, q, p, (int)units, cs);
    return vb::launch_key_mass<256, 128>(st, q, p, (int)units, cs);
}
