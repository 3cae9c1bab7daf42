// The attention weight that every cached row got from a call's query tokens, accumulated over calls:
//
//   m'[b][h][j] = decay m[b][h][j] + sum over the g heads of kv head h and the S tokens of  exp(scale q . k_j - lse)
//
// with the log-sum-exp of each query row given, so a row's weights need neither its maximum nor its sum.  The transposed product
// K Q^T puts keys on the lanes of TMEM and query rows on its columns: a thread owns one key and adds up its columns in
// registers -- nothing is reduced across threads but the two halves of the columns, no atomics, the same bits every time.
//
// Work unit = (observation, kv head, 128 keys).  Persistent CTAs walk the units:
//   loader warp      TMA: the unit's K tile through a ring of KS, its query rows in chunks of at most NQ through a ring of QS
//   MMA warp         D[128 keys][n rows] = K_tile Q_chunk^T, n = the chunk's rows rounded up to 16 (one token: 16 columns), NB accumulators
//   8 sum warps      lane quarter = warp & 3, column half = warp >> 2: p = 2^(s c - lse'), two columns per FMA instruction
//
// One query token: K streams once, HBM bounds it.  Many: 16 exponentials per clock and SM (heads of 64 and 128) or the product (256).
#include <cuda_bf16.h>

#include "host_common.h"
#include "tc5.cuh"

namespace vb {

constexpr int KM_THREADS = 320;  // warps 0-7 sums, 8 loader, 9 MMA
constexpr int KM_LOADER = 8, KM_MMA = 9;

struct KeyMassParams {
    const float *lse;      // [n_obs][n_q][S]: an item's g * S rows in one piece
    const float *mass_in;  // [n_obs][n_kv][cap] or nullptr
    float *mass_out;
    const int32_t *lens, *pad;
    int R, n_kv, cap, max_len, n_tiles, n_units, n_chunks, page0, box_rows;
    float scale_log2, decay;
    int *status;
};

template <int HD>
struct KeyMassSmem {
    static constexpr int CB = HD / 64;                // 64-element column blocks
    static constexpr int NQ = HD == 256 ? 64 : 128;   // query rows per chunk
    static constexpr int KS = HD == 128 ? 3 : 2, QS = 2;
    static constexpr int NB = HD == 64 ? 2 : 4;       // accumulators
    static constexpr int K_BYTES = CB * 128 * 128;    // [CB][128 keys][128 B]
    static constexpr int Q_BYTES = CB * NQ * 128;     // [CB][box_rows][128 B]
    static constexpr int Q_OFF = KS * K_BYTES, BAR_OFF = Q_OFF + QS * Q_BYTES;
    static constexpr int LSE_OFF = BAR_OFF + 256;     // float [2][8 warps][NQ / 2]
    static constexpr int SUM_OFF = LSE_OFF + 2 * 8 * (NQ / 2) * 4;  // float [2][128]
    static constexpr int TOTAL = SUM_OFF + 2 * 128 * 4 + 1024;
    static constexpr int TMEM_COLS = NB * NQ;
    static_assert(TMEM_COLS == 256 || TMEM_COLS == 512, "TMEM");
    static_assert(TOTAL <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ float km_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int HD>
__global__ void __launch_bounds__(KM_THREADS, HD == 64 ? 2 : 1)
key_mass_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const KeyMassParams p) {
    using L = KeyMassSmem<HD>;
    extern __shared__ uint8_t km_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(km_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    uint64_t *k_full = bars, *k_free = bars + 3, *q_full = bars + 6, *q_free = bars + 8, *a_full = bars + 10, *a_free = bars + 14;
    uint64_t *meet = bars + 18;  // [4] the two warps of a lane quarter
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 22);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wc{abort_flag, p.status};

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::KS; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_free[i], 1);
        }
        for (int i = 0; i < L::QS; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_free[i], 1);
        }
        for (int i = 0; i < L::NB; ++i) {
            mbar_init(&a_full[i], 1);
            mbar_init(&a_free[i], 8);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&meet[i], 64);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == KM_MMA) {
        tmem_alloc(tmem_slot, L::TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
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

    if (warp == KM_LOADER) {
        if (lane == 0) {
            uint32_t ku = 0, qu = 0;
            bool ok = true;
            const uint32_t q_tx = (uint32_t)(L::CB * p.box_rows * 128);
            for (int unit = blockIdx.x; ok && unit < p.n_units; unit += gridDim.x) {
                const int item = unit / p.n_tiles, key0 = unit % p.n_tiles * 128;
                if (key0 >= len_of(item / p.n_kv)) continue;
                const int ks = ku % L::KS;
                ok = mbar_wait(&k_free[ks], (ku / L::KS & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                mbar_expect_tx(&k_full[ks], L::K_BYTES);
                for (int cb = 0; cb < L::CB; ++cb)
                    tma_load_3d(smem + ks * L::K_BYTES + cb * 16384, &k_map, &k_full[ks], cb * 64, key0, p.page0 + item);
                ++ku;
                for (int c = 0; c < p.n_chunks; ++c, ++qu) {
                    const int qs = qu % L::QS;
                    ok = mbar_wait(&q_free[qs], (qu / L::QS & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                    if (!ok) break;
                    mbar_expect_tx(&q_full[qs], q_tx);
                    for (int cb = 0; cb < L::CB; ++cb)
                        tma_load_3d(smem + L::Q_OFF + qs * L::Q_BYTES + cb * p.box_rows * 128, &q_map, &q_full[qs], cb * 64, c * L::NQ, item);
                }
            }
        }
    } else if (warp == KM_MMA) {
        const uint32_t k_base = smem_u32(smem), q_base = k_base + L::Q_OFF;
        const uint32_t q_cb = (uint32_t)p.box_rows * 128;
        uint32_t ku = 0, qu = 0;
        bool ok = true;
        for (int unit = blockIdx.x; ok && unit < p.n_units; unit += gridDim.x) {
            const int item = unit / p.n_tiles, key0 = unit % p.n_tiles * 128;
            if (key0 >= len_of(item / p.n_kv)) continue;
            const uint32_t ks = ku % L::KS;
            ok = warp_wait(&k_full[ks], ku / L::KS & 1u, wc, DEV_TIMEOUT_FULL);
            if (!ok) break;
            const uint32_t k_addr = k_base + ks * L::K_BYTES;
            for (int c = 0; c < p.n_chunks; ++c, ++qu) {
                const uint32_t qs = qu % L::QS, ab = qu % L::NB;
                ok = warp_wait(&q_full[qs], qu / L::QS & 1u, wc, DEV_TIMEOUT_FULL);
                if (ok) ok = warp_wait(&a_free[ab], (qu / L::NB & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                tc_fence_after();
                const int n = (min(p.R - c * L::NQ, L::NQ) + 15) & ~15;
                const uint32_t idesc = make_idesc(1, 1, 1, 0, 0, 128, n);
                const uint32_t q_addr = q_base + qs * L::Q_BYTES, d = tmem_base + ab * L::NQ;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk)
                        mma_f16(d, smem_desc_sw128(k_addr + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024),
                                smem_desc_sw128(q_addr + (kk >> 2) * q_cb + (kk & 3) * 32, 16, 1024), idesc, kk != 0 ? 1u : 0u);
                    tc_commit(&a_full[ab]);
                    tc_commit(&q_free[qs]);
                    if (c + 1 == p.n_chunks) tc_commit(&k_free[ks]);
                }
            }
            ++ku;
        }
    } else {
        const int qtr = warp & 3, half = warp >> 2;
        constexpr int HALF = L::NQ / 2;  // columns of a chunk that this warp adds up
        float *lse_s = reinterpret_cast<float *>(smem + L::LSE_OFF) + warp * HALF;
        float *sum_s = reinterpret_cast<float *>(smem + L::SUM_OFF);
        const uint32_t lane_sel = (uint32_t)(qtr * 32) << 16;
        uint32_t qu = 0, un = 0;
        bool ok = true;
        for (int unit = blockIdx.x; ok && unit < p.n_units; unit += gridDim.x) {
            const int item = unit / p.n_tiles, key0 = unit % p.n_tiles * 128, obs = item / p.n_kv;
            const int len = len_of(obs);
            if (key0 >= len) continue;
            const float *lse = p.lse + (long long)item * p.R;
            float sum = 0.0f;
            for (int c = 0; c < p.n_chunks; ++c, ++qu) {
                const uint32_t ab = qu % L::NB;
                // rows past the last, and rows that saw nothing (-inf), weigh nothing: 2^(s - inf)
                float *ls = lse_s + (qu & 1u) * (8 * HALF);
#pragma unroll
                for (int i = 0; i < HALF / 32; ++i) {
                    const int r = c * L::NQ + half * HALF + i * 32 + lane;
                    const float v = r < p.R ? lse[r] : INFINITY;
                    ls[i * 32 + lane] = v == -INFINITY ? -INFINITY : -1.4426950408889634f * v;
                }
                __syncwarp();
                ok = mbar_wait(&a_full[ab], qu / L::NB & 1u, wc, DEV_TIMEOUT_ACCUM);
                if (!ok) break;
                tc_fence_after();
                const int n = min(p.R - c * L::NQ - half * HALF, HALF);  // of this warp's columns; may be 0 or less
                float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
                for (int b = 0; b < HALF / 32; ++b) {
                    if (b * 32 >= n) break;
                    uint32_t s[32];
                    tmem_ld32(tmem_base + lane_sel + ab * L::NQ + (uint32_t)(half * HALF + b * 32), s);
                    tmem_ld_wait();
                    if (n < b * 32 + 32) {  // columns that no row stands behind hold anything
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[e] = b * 32 + e < n ? s[e] : 0u;
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 l4 = *reinterpret_cast<const float4 *>(ls + b * 32 + e);
                        a0 += km_ex2(fmaf(__uint_as_float(s[e]), p.scale_log2, l4.x));
                        a1 += km_ex2(fmaf(__uint_as_float(s[e + 1]), p.scale_log2, l4.y));
                        a0 += km_ex2(fmaf(__uint_as_float(s[e + 2]), p.scale_log2, l4.z));
                        a1 += km_ex2(fmaf(__uint_as_float(s[e + 3]), p.scale_log2, l4.w));
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_free[ab]);
                sum += a0 + a1;
            }
            if (!ok) break;
            // the two halves of the columns meet; the slots are used in turn, so one meeting per unit is enough
            float *slot = sum_s + (un & 1u) * 128;
            if (half) slot[qtr * 32 + lane] = sum;
            mbar_arrive(&meet[qtr]);
            ok = mbar_wait(&meet[qtr], un & 1u, wc, DEV_TIMEOUT_MISC);
            if (!ok) break;
            ++un;
            const int key = key0 + qtr * 32 + lane;
            if (!half && key < len) {
                sum += slot[qtr * 32 + lane];
                if (p.pad && key >= p.pad[2 * obs] && key < p.pad[2 * obs + 1]) sum = 0.0f;
                const long long at = (long long)item * p.cap + key;
                p.mass_out[at] = p.mass_in ? fmaf(p.decay, p.mass_in[at], sum) : sum;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == KM_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem_base, L::TMEM_COLS);
    }
}

template <int HD>
static int launch_key_mass(const vlab200_kv_store *st, const void *q, KeyMassParams &p, cudaStream_t stream) {
    using L = KeyMassSmem<HD>;
    p.n_chunks = (p.R + L::NQ - 1) / L::NQ;
    p.box_rows = p.R >= L::NQ ? L::NQ : (p.R + 15) & ~15;
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
    if (int rc = ensure_dyn_smem(key_mass_kernel<HD>, L::TOTAL)) return rc;
    const int slots = (HD == 64 ? 2 : 1) * sm_count();
    return launch_pdl(key_mass_kernel<HD>, dim3(p.n_units < slots ? p.n_units : slots), dim3(KM_THREADS), L::TOTAL, stream, qmap, kmap, p);
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
    const long long R = (long long)(n_q / st->n_kv) * S, tiles = (max_len + 127LL) / 128, units = (long long)st->n_obs * st->n_kv * tiles;
    if (R > 0x7fffff00LL || units > 0x7fffff00LL || (long long)st->n_layers * st->n_obs * st->n_kv > 0x7fffff00LL) {
        vb::set_last_error("key_mass: more than 2^31 query rows per kv head, pages or key tiles");
        return VLAB200_ERR_UNSUPPORTED;
    }
    if (max_len == 0) return VLAB200_OK;
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
    p.n_tiles = (int)tiles;
    p.n_units = (int)units;
    p.page0 = layer * st->n_obs * st->n_kv;
    p.scale_log2 = 1.4426950408889634f * (scale > 0.0f ? scale : 1.0f / sqrtf((float)hd));
    p.decay = decay;
    p.status = vb::device_status_ptr();
    if (!p.status) return vb::cuda_fail(cudaGetLastError(), "device_status_ptr");
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (hd == 64) return vb::launch_key_mass<64>(st, q, p, cs);
    if (hd == 128) return vb::launch_key_mass<128>(st, q, p, cs);
    return vb::launch_key_mass<256>(st, q, p, cs);
}
