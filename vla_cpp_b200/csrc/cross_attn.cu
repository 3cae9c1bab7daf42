// Attention of a call's query tokens to cached rows whose number differs from observation to observation:
//
//   out = softmax(scale q K^T over the visible rows) V,     lse = log sum exp(scale q K^T)
//
// visible: row < len[b], not in the observation's hidden range [lo, hi).  A row that sees nothing gives 0 and -inf, whatever the pages hold.
//
// Up to 16 query rows per kv head: cross_few_kernel, below.
// Heads of 64 and 128, a unit = (observation, kv head, 256 of the g S stacked query rows), one CTA:
//   loader warp       TMA: the two 128-row Q tiles of a unit, K and V in blocks of 128 rows through rings
//   MMA warp          O_t += P_t V_j with P_t read from TMEM, XA_EARLY of the block's rows while the softmax is at the others, then
//                     S_t = Q_t K_(j+1)^T, for the tiles t = 0, 1 in turn: the tensor pipe works on one tile while the other is in its
//                     softmax.  (A warp per tile: the tiles fell into step, both at the exponentials and then both at the pipe.)
//   V cleaner         zeroes hidden rows
//   2 x 4 warps       one per tile and lane quarter, a row per thread: maximum, 2^(s c - m), row sum, P over S in TMEM
// TMEM: O_0, O_1 and one S per tile (512 columns at heads of 128).  Both the exponentials (16 per clock and SM) and the products need
// 1,024 clocks per tile and block at heads of 128; at 64 the exponentials bound it.  Blocks of 64 rows with two S buffers per tile were
// slower: a product whose A comes from shared memory takes 64 clocks a step of 16 whether N is 64 or 128.
//
// Work is dealt out in one of two ways (cross_plan says which).  Whole: a CTA takes whole units, the longest observations first.  Cut: the
// units' blocks form one list and every CTA takes an equal piece of it, so few units leave no SM idle; a unit cut by a piece's border
// leaves un-normalised rows with their maximum and sum in the workspace, at most two pieces per CTA, and cross_combine_kernel merges them
// in order.
//
// Measured (graph replay, cold L2): 4 prompts of 816 tokens, 20 / 5 heads of 128, over 4,097 to 8,190 rows 201 us = 1,020 TFLOP/s (in a stream
// of calls on changing inputs 214 = 955); there the chain of a
// tile's block -- S, softmax, P V, some 3,400 clocks -- bounds it, of which the pipe computes 2,048 for the two tiles.  64 x 50 tokens, 15 / 5
// heads of 64, over 113 to 241 rows 22 us, and 64 x 51 tokens, 8 / 1 heads of 256, over 304 to 816 rows 35 us: the chain of a unit's blocks
// (2,400 to 3,000 clocks each), of the first loads (5,000 to 8,000 with the launch) and of the store bounds those.
#include <cuda_bf16.h>

#include "f32x2.cuh"
#include "host_common.h"
#include "ragged.cuh"
#include "tc5.cuh"

namespace vb {

constexpr int XA_BKV = 128;      // rows of K / V per block
constexpr int XA_THREADS = 384;  // warps 0-3 tile 0, 4-7 tile 1, 8 loader, 9 MMA, 10 V cleaner, 11 fills the warpgroup that gives up registers
constexpr int XA_LOADER = 8, XA_MMA = 9, XA_CLEANER = 10;
constexpr int XA_EARLY = 96;     // of a block's rows: their P V runs beside the softmax of the others (64: 205 us instead of 197 in the longest case)
// Registers of a thread: 384 x 168 at launch = 64,512; 2 x 128 x 192 + 128 x 120 = 64,512 after the split.  With 208 + 88 the issuing warp kept its
// descriptors and the next unit in local memory: 64 x 50 tokens over 113 to 241 rows 24.6 us instead of 22.6, the longest case 203 instead of 199.
constexpr int XA_REGS_SOFTMAX = 192, XA_REGS_REST = 120;
constexpr float XA_RAISE = 8.0f; // the running maximum is raised, and O rescaled, only by blocks that exceed it by more than 2^8

struct CrossParams {
    __nv_bfloat16 *out;  // [n_obs][S][n_q * HD]
    float *lse;          // [n_obs][n_q][S] or nullptr
    const int32_t *lens, *pad;
    int S, n_q, n_kv, g, R, n_obs, max_len, page0;
    int n_mt, unit_rows; // units per item and their rows
    int n_work;          // CTAs (CTA pairs) the blocks are dealt to
    int round_r, round_u, bin_shift;  // n_work in observations and units; see XaOrder
    int by_unit;         // cross_combine_kernel: a block per unit (and rows), not per CTA
    int out_al32;
    float scale_log2;
    int *status;
    float *ws_o;         // [2 n_work][ws_rows][HD], nullptr: whole units
    float *ws_ml;        // [2 n_work][ws_rows][2]: maximum (log2 units), row sum
    int ws_rows;
};

__device__ __forceinline__ int xa_len(const CrossParams &p, int obs) {
    return p.lens ? min(max(p.lens[obs], 0), p.max_len) : p.max_len;
}
__device__ __forceinline__ float xa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// log2 of a row sum, off by 2^-22: the fast logarithm's error is that of a whole number plus it, once its argument lies in [0.75, 1.5).
__device__ __forceinline__ float xa_log2(float x) {
    const int bits = __float_as_int(x), k = (bits - 0x3f400000) >> 23;
    const float r = (float)k + __log2f(__int_as_float(bits - (k << 23)));
    return x < INFINITY ? r : x;  // infinite or no number: as it is
}
__device__ __forceinline__ float xa_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A row of an item (g heads of S tokens): token * n_q + head.
__device__ __forceinline__ int xa_place(const CrossParams &p, int row) {
    const int head = row / p.S;
    return (row - head * p.S) * p.n_q + head;
}
// The hidden range of an observation; (none, none) if it has none.
__device__ __forceinline__ void xa_pad(const CrossParams &p, int obs, int &lo, int &hi) {
    lo = p.pad ? max(p.pad[2 * obs], 0) : 0;
    hi = p.pad ? p.pad[2 * obs + 1] : 0;
    if (hi <= lo) lo = hi = 0x7fffffff;
}
// The blocks of all units, and the piece of CTA `c` of `n`.
__device__ __forceinline__ int xa_total_blocks(const CrossParams &p) {  // whole warp
    int sum = 0;
    for (int b = threadIdx.x & 31; b < p.n_obs; b += 32) sum += (xa_len(p, b) + XA_BKV - 1) / XA_BKV;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum * p.n_kv * p.n_mt;
}
__device__ __forceinline__ int xa_div(unsigned long long a, unsigned b) {  // a 64-bit division takes 500 clocks
    return a >> 32 ? (int)(a / b) : (int)((unsigned)a / b);
}
__device__ __forceinline__ int xa_border(int c, int n, int total) { return xa_div((unsigned long long)c * (unsigned)total, (unsigned)n); }
__device__ __forceinline__ int xa_cta_of(int block, int n, int total) {  // whose piece a block is in
    return xa_div((unsigned long long)(block + 1u) * (unsigned)n - 1u, (unsigned)total);
}

struct XaSegment {  // a run of blocks [j0, j1) of one unit
    int obs, kvh, mt, j0, j1, len, slot;  // slot: of the workspace; -1: the unit is whole
    int pad_lo, pad_hi;                   // hidden rows
};

// Whole units of up to XA_SORT observations: those with most blocks first, dealt to the CTAs there and back, so that who has a long one first
// has a short one next (64 observations of 3 to 7 blocks, two units each, on 74 pairs: 14 blocks for some pairs in the order of the
// observations, 9 so; 8.5 on average).  Every CTA sorts for itself (a counting sort, the same in all of them): a bin per number of blocks, or
// per 2^bin_shift of them, and the last for observations without rows.
constexpr int XA_SORT = 256, XA_BINS = 64;
struct XaOrder {
    int4 item[XA_SORT];                // observation, length, hidden range
    int count[XA_SORT / 32][XA_BINS];  // by groups of 32 observations
    int n_live;                        // observations that have rows
};
__device__ __forceinline__ void xa_sort_clear(XaOrder &o, int n_threads) {  // a barrier of the block later: xa_sort
    for (int i = threadIdx.x; i < XA_SORT / 32 * XA_BINS; i += n_threads) (&o.count[0][0])[i] = 0;
}
template <int THREADS>
__device__ __forceinline__ void xa_sort(const CrossParams &p, XaOrder &o) {  // the whole block
    constexpr int N = (XA_SORT + THREADS - 1) / THREADS, W = THREADS / 32;  // observations per thread
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (p.n_obs + 31) >> 5;
    int4 mine[N];
    int bin[N], rank[N];  // (lanes without an observation share a bin that is not counted)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int g = warp + i * W;  // of the groups of 32 observations
        mine[i] = make_int4(g * 32 + lane, 0, 0, 0);
        bin[i] = XA_BINS;
        if (g >= warps) continue;
        if (mine[i].x < p.n_obs) {
            mine[i].y = xa_len(p, mine[i].x);
            xa_pad(p, mine[i].x, mine[i].z, mine[i].w);
            const int most = (p.max_len + XA_BKV - 1) / XA_BKV >> p.bin_shift;
            bin[i] = mine[i].y > 0 ? most - ((mine[i].y + XA_BKV - 1) / XA_BKV >> p.bin_shift) : XA_BINS - 1;
        }
        const unsigned same = __match_any_sync(0xffffffffu, bin[i]);
        rank[i] = __popc(same & ((1u << lane) - 1u));
        if (bin[i] < XA_BINS && rank[i] == 0) o.count[g][bin[i]] = __popc(same);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int g = warp + i * W;
        if (g >= warps) continue;
        int sum[2] = {0, 0}, before[2] = {0, 0};  // of this lane's two bins: all of them, those of the groups in front
        for (int w = 0; w < warps; ++w) {
            const int2 c = *reinterpret_cast<const int2 *>(&o.count[w][2 * lane]);
            if (w == g) {
                before[0] = sum[0];
                before[1] = sum[1];
            }
            sum[0] += c.x;
            sum[1] += c.y;
        }
        int incl = sum[0] + sum[1];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += up;
        }
        const int at0 = incl - sum[0] - sum[1] + before[0], at1 = incl - sum[1] + before[1];
        const int even = __shfl_sync(0xffffffffu, at0, bin[i] >> 1), odd = __shfl_sync(0xffffffffu, at1, bin[i] >> 1);
        if (bin[i] < XA_BINS) o.item[(bin[i] & 1 ? odd : even) + rank[i]] = mine[i];
        if (g == 0 && lane == 31) o.n_live = p.n_obs - sum[1];
    }
    __syncthreads();
}

// The segments of a CTA (pair): whole units in the order above, or (LIST) a piece of the list of all blocks.
template <bool LIST, typename LenOf>
struct XaWork;
template <typename LenOf>
struct XaWork<false, LenOf> {
    const XaOrder &order;
    const CrossParams &p;
    int upo, live;           // units of an observation, observations
    int my_r, my_u;          // place of this CTA in a round, counted in observations and units
    int base_r, base_u;      // of the round
    bool back;
    __device__ __forceinline__ XaWork(LenOf, const CrossParams &p, const XaOrder &o, int cta) : order(o), p(p) {
        upo = p.n_kv * p.n_mt;
        live = o.n_live;
        my_r = cta / upo;
        my_u = cta - my_r * upo;
        base_r = base_u = 0;
        back = false;
    }
    __device__ __forceinline__ bool next(XaSegment &s) {
        int r = base_r + my_r, u = base_u + my_u;
        base_r += p.round_r;
        base_u += p.round_u;
        if (base_u >= upo) {
            base_u -= upo;
            ++base_r;
        }
        if (back) {  // from the end of the round
            r = base_r - my_r;
            u = base_u - 1 - my_u;
            if (u < 0) {
                u += upo;
                --r;
            }
        } else if (u >= upo) {
            u -= upo;
            ++r;
        }
        back = !back;
        if (r >= live) return false;
        const int4 it = order.item[r];
        s.obs = it.x;
        s.len = it.y;
        s.pad_lo = it.z;
        s.pad_hi = it.w;
        s.kvh = p.n_mt == 1 ? u : u / p.n_mt;
        s.mt = p.n_mt == 1 ? 0 : u - s.kvh * p.n_mt;
        s.j0 = 0;
        s.j1 = (it.y + XA_BKV - 1) / XA_BKV;
        s.slot = -1;
        return true;
    }
};
template <typename LenOf>
struct XaWork<true, LenOf> {
    RaggedCursor<LenOf> cur;
    const CrossParams &p;
    int w, w1, c, n_mt;
    bool whole_units;
    __device__ __forceinline__ XaWork(LenOf f, const CrossParams &p, const XaOrder &, int cta) : cur(f, p.n_obs, p.n_kv * p.n_mt, XA_BKV), p(p) {
        c = cta;
        n_mt = p.n_mt;
        whole_units = p.ws_o == nullptr;
        const int total = xa_total_blocks(p), n = min(p.n_work, total);
        w = cta < n ? xa_border(cta, n, total) : total;
        w1 = cta < n ? xa_border(cta + 1, n, total) : total;
    }
    __device__ __forceinline__ bool next(XaSegment &s) {  // whole warp
        RaggedUnit u;
        while (w < w1 && cur.find(w, u)) {
            const int nb = (u.len + XA_BKV - 1) / XA_BKV;
            if (whole_units && u.block > 0) {  // begun by the CTA before, which finishes it
                w += nb - u.block;
                continue;
            }
            s.obs = u.obs;
            s.len = u.len;
            xa_pad(p, s.obs, s.pad_lo, s.pad_hi);
            s.kvh = u.kvh / n_mt;
            s.mt = u.kvh - s.kvh * n_mt;
            s.j0 = u.block;
            s.j1 = whole_units ? nb : min(nb, u.block + (w1 - w));
            s.slot = s.j0 == 0 && s.j1 == nb ? -1 : 2 * c + (s.j0 > 0 ? 0 : 1);
            w += s.j1 - s.j0;
            return true;
        }
        return false;
    }
};

template <int HD>
struct CrossSmem {
    static constexpr int CB = HD / 64, BKV = XA_BKV;  // 64-element column blocks
    static constexpr int Q_BYTES = CB * 128 * 128;          // a tile: [CB][128 rows][128 B]
    static constexpr int KV_BYTES = CB * BKV * 128;
    static constexpr int STAGES = HD == 64 ? 4 : 2, QS = HD == 64 ? 2 : 1;  // K and V blocks; units' Q tiles
    static constexpr int K_OFF = QS * 2 * Q_BYTES, V_OFF = K_OFF + STAGES * KV_BYTES, BAR_OFF = V_OFF + STAGES * KV_BYTES;
    static constexpr int ORDER_OFF = BAR_OFF + 512, TOTAL = ORDER_OFF + (int)sizeof(XaOrder) + 1024;
    static constexpr int S_COL = 2 * HD;  // O_0, O_1, S_0, S_1
    static_assert(S_COL + 2 * BKV <= 512 && TOTAL <= 227 * 1024, "TMEM, shared memory");
};

// Rows of empty observations: 0 and -inf.  CTA (pair) c looks after every n_work-th of them (LIST: of all observations).
template <int HD, bool LIST>
__device__ __forceinline__ void xa_fill_empty(const CrossParams &p, const XaOrder &order, int c, int tid, int n_threads) {
    for (int i = (LIST ? 0 : order.n_live) + c; i < p.n_obs; i += p.n_work) {
        if (LIST && xa_len(p, i) > 0) continue;
        const int obs = LIST ? i : order.item[i].x;
        const long long n = (long long)p.n_q * p.S;
        uint4 *out = reinterpret_cast<uint4 *>(p.out + obs * n * HD);
        for (long long i = tid; i < n * (HD / 8); i += n_threads) out[i] = make_uint4(0, 0, 0, 0);
        if (p.lse)
            for (long long i = tid; i < n; i += n_threads) p.lse[obs * n + i] = -INFINITY;
    }
}

// Does the mask hide rows of the block that begins at row c0?
__device__ __forceinline__ bool xa_dirty(int c0, int len, int pad_lo, int pad_hi) {
    return c0 + XA_BKV > len || (c0 < pad_hi && c0 + XA_BKV > pad_lo);
}

// Hidden rows of a V block meet weights of 0, and 0 times what stands there need not be 0.  So a dirty block's TMA completes on v_raw, and
// this warp zeroes those rows in shared memory and then says v_full in its place.
template <int CB>
__device__ __forceinline__ void xa_clean_blocks(XaSegment &s, bool &ok, uint32_t &jb, uint8_t *v_smem, int stages, int stage_bytes,
                                                uint64_t *v_raw, uint64_t *v_full, uint32_t &raw_phase, const WaitCtx &wc) {
    const int lane = threadIdx.x & 31;
    const int pad_lo = s.pad_lo, pad_hi = s.pad_hi;
    for (int j = s.j0; ok && j < s.j1; ++j, ++jb) {
        const int c0 = j * XA_BKV;
        if (!xa_dirty(c0, s.len, pad_lo, pad_hi)) continue;
        const uint32_t st = jb % (uint32_t)stages;
        ok = warp_wait(&v_raw[st], raw_phase >> st & 1u, wc, DEV_TIMEOUT_FULL);
        if (!ok) break;
        raw_phase ^= 1u << st;  // a stage's raw barrier turns with its dirty blocks only
        uint4 *v = reinterpret_cast<uint4 *>(v_smem + st * (uint32_t)stage_bytes);
        for (int r = lane >> 3; r < XA_BKV; r += 4) {  // [CB][XA_BKV rows][128 B]
            const int row = c0 + r;
            if (row >= s.len || (row >= pad_lo && row < pad_hi)) {
#pragma unroll
                for (int cb = 0; cb < CB; ++cb) v[(cb * XA_BKV + r) * 8 + (lane & 7)] = make_uint4(0, 0, 0, 0);
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
    }
}

// -inf over the hidden ones of 32 columns that begin at row c0.  Which those are is the same for all rows: one word of bits, and groups that hide
// nothing cost nothing (every column of a block tested for length and range took 2,000 clocks, of the groups concerned 1,000).
__device__ __forceinline__ uint32_t xa_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ void xa_mask32(uint32_t (&x)[32], int c0, int len, int pad_lo, int pad_hi) {
    const uint32_t seen = xa_below(len - c0) & ~(xa_below(pad_hi - c0) & ~xa_below(pad_lo - c0));
    if (seen != 0xffffffffu) {
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = seen & (1u << e) ? x[e] : 0xff800000u;
    }
}

// COLS columns of O of one row per thread, out of TMEM: divided and rounded to dst, or (ws) as they are.  The loads of 32 N columns are in flight
// at once (N = 2 at heads of 256; 64 and 128 have no registers for it: 64 x 50 tokens 20.7 us instead of 18.7).  `out_of_tmem` runs when all have
// been read.
template <int COLS, int N, typename F>
__device__ __forceinline__ void xa_drain(uint32_t o_addr, bool row_ok, __nv_bfloat16 *dst, float inv, int al32, float *ws, F out_of_tmem) {
    const F2 inv2 = f2(inv, inv);
#pragma unroll
    for (int c0 = 0; c0 < COLS; c0 += 32 * N) {
        uint32_t o[N][32];
#pragma unroll
        for (int i = 0; i < N; ++i) tmem_ld32(o_addr + (uint32_t)(c0 + 32 * i), o[i]);
        tmem_ld_wait();
        if (c0 + 32 * N == COLS) out_of_tmem();
        if (!row_ok) continue;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) {
            const uint32_t(&v)[32] = o[i / 2];
            const int h = 16 * (i & 1), at = c0 + 16 * i;
            uint32_t w[8];
            if (ws) {
#pragma unroll
                for (int q = 0; q < 16; q += 8) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = v[h + q + e];
                    st_global_v8(ws + at + q, w);
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = f2_bf16(f2_mul(f2(__uint_as_float(v[h + 2 * e]), __uint_as_float(v[h + 2 * e + 1])), inv2));
            if (al32) {
                st_global_v8(dst + at, w);
            } else {
                uint4 *d4 = reinterpret_cast<uint4 *>(dst + at);
                d4[0] = make_uint4(w[0], w[1], w[2], w[3]);
                d4[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
    }
}

template <int HD, bool LIST>
__global__ void __launch_bounds__(XA_THREADS, 1)
cross_attn_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                  const __grid_constant__ CUtensorMap v_map, const CrossParams p) {
    using L = CrossSmem<HD>;
    constexpr int BKV = L::BKV;
    constexpr uint32_t NS = L::STAGES, QS = L::QS;
    extern __shared__ uint8_t xa_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(xa_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    uint64_t *k_full = bars + 2, *k_free = bars + 6, *v_full = bars + 10, *v_free = bars + 14;
    uint64_t *s_full = bars + 18, *pv_done = bars + 20, *o_free = bars + 22;  // [2 tiles]
    uint64_t *p_full = bars + 24;                                             // [2 tiles][early rows of a block, the others]
    uint64_t *v_raw = bars + 28, *q_full = bars + 32, *q_free = bars + 34;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 36);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wc{abort_flag, p.status};
    XaOrder &order = *reinterpret_cast<XaOrder *>(smem + L::ORDER_OFF);
    if (!LIST) xa_sort_clear(order, XA_THREADS);

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < QS; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_free[i], 1);
        }
        for (uint32_t i = 0; i < NS; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_raw[i], 1);
            mbar_init(&v_free[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&pv_done[i], 1);
            mbar_init(&o_free[i], 4);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&p_full[i], 4);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == XA_MMA) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&q_map);
        tma_prefetch_desc(&k_map);
        tma_prefetch_desc(&v_map);
    }
    pdl_wait();
    pdl_launch_dependents();  // after the wait: cross_combine_kernel reads the lengths before its own

    auto len_of = [&](int obs) { return xa_len(p, obs); };
    if (!LIST) xa_sort<XA_THREADS>(p, order);
    if (warp < XA_LOADER) xa_fill_empty<HD, LIST>(p, order, blockIdx.x, threadIdx.x, 32 * XA_LOADER);
    XaWork<LIST, decltype(len_of)> work(len_of, p, order, blockIdx.x);
    XaSegment s;
    bool ok = true;

    if (warp == XA_LOADER) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XA_REGS_REST));
        uint32_t si = 0, jb = 0;
        for (; ok && work.next(s); ++si) {
            const int item = s.obs * p.n_kv + s.kvh, row0 = s.mt * 256;
            const int tiles = p.R > row0 + 128 ? 2 : 1;
            const int pad_lo = s.pad_lo, pad_hi = s.pad_hi;
            const uint32_t qs = si % QS;
            ok = warp_wait(&q_free[qs], (si / QS & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
            if (!ok) break;
            if (elect_one()) {
                mbar_expect_tx(&q_full[qs], tiles * L::Q_BYTES);
                for (int t = 0; t < tiles; ++t)
                    for (int cb = 0; cb < L::CB; ++cb)
                        tma_load_3d(smem + (qs * 2 + t) * L::Q_BYTES + cb * 16384, &q_map, &q_full[qs], cb * 64, row0 + t * 128, item);
            }
            for (int j = s.j0; j < s.j1; ++j, ++jb) {
                const uint32_t st = jb % NS, ph = (jb / NS) & 1u;
                ok = warp_wait(&k_free[st], ph ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                if (elect_one()) {
                    mbar_expect_tx(&k_full[st], L::KV_BYTES);
                    for (int cb = 0; cb < L::CB; ++cb)
                        tma_load_3d(smem + L::K_OFF + st * L::KV_BYTES + cb * (BKV * 128), &k_map, &k_full[st], cb * 64, j * BKV, p.page0 + item);
                }
                ok = warp_wait(&v_free[st], ph ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                if (elect_one()) {
                    uint64_t *landed = xa_dirty(j * BKV, s.len, pad_lo, pad_hi) ? &v_raw[st] : &v_full[st];
                    mbar_expect_tx(landed, L::KV_BYTES);
                    for (int cb = 0; cb < L::CB; ++cb)
                        tma_load_3d(smem + L::V_OFF + st * L::KV_BYTES + cb * (BKV * 128), &v_map, landed, cb * 64, j * BKV, p.page0 + item);
                }
            }
        }
    } else if (warp == XA_CLEANER) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XA_REGS_REST));
        uint32_t jb = 0, raw_phase = 0;
        while (ok && work.next(s)) xa_clean_blocks<L::CB>(s, ok, jb, smem + L::V_OFF, NS, L::KV_BYTES, v_raw, v_full, raw_phase, wc);
    } else if (warp == XA_MMA) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XA_REGS_REST));
        constexpr uint32_t idesc_s = make_idesc(1, 1, 1, 0, 0, 128, BKV), idesc_o = make_idesc(1, 1, 1, 0, 1, 128, HD);
        const uint64_t q_desc0 = smem_desc_sw128(smem_u32(smem), 16, 1024), k_desc0 = smem_desc_sw128(smem_u32(smem) + L::K_OFF, 16, 1024);
        const uint64_t v_desc0 = smem_desc_sw128(smem_u32(smem) + L::V_OFF, BKV * 128, 1024);
        auto issue_s = [&](uint32_t qs, int t, uint32_t st) {
            const uint64_t q = q_desc0 + (uint64_t)((qs * 2 + t) * (L::Q_BYTES >> 4)), k = k_desc0 + (uint64_t)(st * (L::KV_BYTES >> 4));
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    mma_f16(tmem_base + L::S_COL + t * BKV, q + (uint64_t)((kk >> 2) * 1024 + (kk & 3) * 2),
                            k + (uint64_t)((kk >> 2) * (BKV * 8) + (kk & 3) * 2), idesc_s, kk != 0 ? 1u : 0u);
                tc_commit(&s_full[t]);
            }
        };
        uint32_t si = 0, jb = 0;
        uint32_t blk[2] = {0, 0}, seg[2] = {0, 0};  // blocks and segments of each tile so far
        // S of a segment's first block follows the P V of the segment before: by tile where its Q has its own stage, behind both otherwise.
        // A tile's S buffer held the P of its last block: that P V was issued before, and the pipe keeps the order of one warp's products.
        auto tiles_of = [&](const XaSegment &g) { return p.R > g.mt * 256 + 128 ? 2 : 1; };
        XaSegment after;
        bool here = work.next(s);
        if (here) {
            ok = warp_wait(&q_full[0], 0, wc, DEV_TIMEOUT_FULL);
            if (ok) ok = warp_wait(&k_full[0], 0, wc, DEV_TIMEOUT_FULL);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < tiles_of(s); ++t) issue_s(0, t, 0);
                if (elect_one()) {
                    tc_commit(&k_free[0]);
                    if (s.j1 - s.j0 == 1) tc_commit(&q_free[0]);
                }
            }
        }
        for (; ok && here; ++si) {
            const int tiles = tiles_of(s);
            const uint32_t qs = si % QS, qn = (si + 1) % QS;
            const bool next = work.next(after);
            const int tiles_n = next ? tiles_of(after) : 0;
            for (int j = s.j0; ok && j < s.j1; ++j, ++jb) {
                const uint32_t st = jb % NS, sn = (jb + 1) % NS;
                const uint64_t v = v_desc0 + (uint64_t)(st * (L::KV_BYTES >> 4));
                const bool more = j + 1 < s.j1, early = QS > 1 && !more && next;
                // what comes early is waited for before the softmax is
                ok = warp_wait(&v_full[st], (jb / NS) & 1u, wc, DEV_TIMEOUT_FULL);
                if (ok && (more || early)) ok = warp_wait(&k_full[sn], ((jb + 1) / NS) & 1u, wc, DEV_TIMEOUT_FULL);
                if (ok && early) ok = warp_wait(&q_full[qn], (si + 1) / QS & 1u, wc, DEV_TIMEOUT_FULL);
                for (int t = 0; ok && t < tiles; ++t) {
                    if (j == s.j0) ok = warp_wait(&o_free[t], (seg[t] & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                    if (ok) ok = warp_wait(&p_full[2 * t], blk[t] & 1u, wc, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t pt = tmem_base + L::S_COL + t * BKV, o = tmem_base + t * HD;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < XA_EARLY / 16; ++kk)
                            mma_f16_tmem_a(o, pt + (uint32_t)(kk * 8), v + (uint64_t)(kk * 128), idesc_o, j == s.j0 && kk == 0 ? 0u : 1u);
                    }
                    ok = warp_wait(&p_full[2 * t + 1], blk[t] & 1u, wc, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int kk = XA_EARLY / 16; kk < BKV / 16; ++kk)
                            mma_f16_tmem_a(o, pt + (uint32_t)(kk * 8), v + (uint64_t)(kk * 128), idesc_o, 1u);
                        tc_commit(&pv_done[t]);
                    }
                    if (more) issue_s(qs, t, sn);
                    else if (early && t < tiles_n) issue_s(qn, t, sn);
                    ++blk[t];
                }
                if (!ok) break;
                if (elect_one()) tc_commit(&v_free[st]);
                if (!more && next) {  // the S blocks of the next segment that are not issued yet
                    if (!early) {
                        ok = warp_wait(&k_full[sn], ((jb + 1) / NS) & 1u, wc, DEV_TIMEOUT_FULL);
                        if (ok) ok = warp_wait(&q_full[qn], (si + 1) / QS & 1u, wc, DEV_TIMEOUT_FULL);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    for (int t = early ? tiles : 0; t < tiles_n; ++t) issue_s(qn, t, sn);
                }
                if (elect_one()) {
                    if (more || next) tc_commit(&k_free[sn]);
                    if (j + 2 == s.j1) tc_commit(&q_free[qs]);  // a segment's last S blocks have been issued
                    if (!more && next && after.j1 - after.j0 == 1) tc_commit(&q_free[qn]);
                }
            }
            for (int t = 0; t < tiles; ++t) ++seg[t];
            s = after;
            here = next;
        }
    } else if (warp > XA_CLEANER) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XA_REGS_REST));
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(XA_REGS_SOFTMAX));
        const int t = warp >> 2, qtr = warp & 3;
        const uint32_t lane_sel = (uint32_t)(qtr * 32) << 16;
        const uint32_t s_addr = tmem_base + L::S_COL + t * BKV + lane_sel, o_addr = tmem_base + t * HD + lane_sel;
        const F2 scale2 = f2(p.scale_log2, p.scale_log2);
        uint32_t blk = 0;  // blocks of this tile so far
        auto next = [&](XaSegment &g) {  // with rows in this tile
            do {
                if (!work.next(g)) return false;
            } while (t == 1 && g.mt * 256 + 128 >= p.R);
            return true;
        };
        XaSegment after;
        int mt_of_place = -1, place = 0;  // of this thread's row: token * n_q + head of the kv head's group
        for (bool here = next(s); ok && here; s = after) {
            const int row0 = s.mt * 256 + t * 128;
            const int lr = t * 128 + qtr * 32 + lane, row = s.mt * 256 + lr;  // in the unit, in the item
            const bool live = row0 + qtr * 32 < p.R;                          // of the warp
            const int pad_lo = s.pad_lo, pad_hi = s.pad_hi;
            float m_used = -INFINITY, l_sum = 0.0f;  // running maximum in log2 units, row sum
            for (int j = s.j0; j < s.j1; ++j, ++blk) {
                ok = warp_wait(&s_full[t], blk & 1u, wc, DEV_TIMEOUT_FULL);
                if (!ok) break;
                tc_fence_after();
                const int c0 = j * BKV;
                const bool dirty = xa_dirty(c0, s.len, pad_lo, pad_hi);
                uint32_t x[4][32];
                float mref = 0.0f;
                if (live) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) tmem_ld32(s_addr + (uint32_t)(i * 32), x[i]);
                    tmem_ld_wait();
                    if (dirty) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) xa_mask32(x[i], c0 + i * 32, s.len, pad_lo, pad_hi);
                    }
                    float mx[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mx[i] = fmaxf(__uint_as_float(x[i][0]), __uint_as_float(x[i][1]));
#pragma unroll
                        for (int e = 2; e < 32; e += 2) mx[i] = xa_max3(mx[i], __uint_as_float(x[i][e]), __uint_as_float(x[i][e + 1]));
                    }
                    const float bm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
                    const bool raise = bm > m_used + XA_RAISE;
                    if (__any_sync(0xffffffffu, raise)) {
                        float factor = 1.0f;
                        if (raise) {
                            factor = m_used == -INFINITY ? 0.0f : xa_ex2(m_used - bm);
                            m_used = bm;
                            l_sum *= factor;
                        }
                        if (j > s.j0) {  // O was summed under the old maximum
                        ok = warp_wait(&pv_done[t], (blk - 1) & 1u, wc, DEV_TIMEOUT_ACCUM);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            uint32_t ov[16];
                            tmem_ld16(o_addr + (uint32_t)c, ov);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 16; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * factor);
                            tmem_st16(o_addr + (uint32_t)c, ov);
                        }
                        }
                    }
                    mref = m_used == -INFINITY ? 0.0f : m_used;
                }
                const F2 neg = f2(-mref, -mref);
                F2 sum[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
                // quarter q's exponentials are asked for before quarter q - 1's are summed and packed
#pragma unroll
                for (int q = 0; q <= BKV / 32; ++q) {
                    if (live && q < BKV / 32) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const F2 a = f2_fma(f2(__uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1])), scale2, neg);
                            float a0, a1;
                            f2_get(a, a0, a1);
                            x[q][e] = __float_as_uint(xa_ex2(a0));
                            x[q][e + 1] = __float_as_uint(xa_ex2(a1));
                        }
                    }
                    if (q == 0) continue;
                    if (live) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const F2 pr = f2(__uint_as_float(x[q - 1][e]), __uint_as_float(x[q - 1][e + 1]));
                            sum[(e >> 1) & 1] = f2_add(sum[(e >> 1) & 1], pr);
                            pk[e >> 1] = f2_bf16(pr);  // weights are rounded to 8 bits for the product, their sum is not
                        }
                        tmem_st16(s_addr + (uint32_t)((q - 1) * 16), pk);
                    }
                    if (q == XA_EARLY / 32 || q == BKV / 32) {
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[2 * t + (q == BKV / 32 ? 1 : 0)]);
                    }
                }
                float u0, u1, u2, u3;
                f2_get(sum[0], u0, u1);
                f2_get(sum[1], u2, u3);
                l_sum += (u0 + u1) + (u2 + u3);
            }
            if (!ok) break;
            // ---- O / l -> bf16 -> out, or the piece into the workspace; what comes next and the rows' places are worked out meanwhile ----
            here = next(after);
            const bool row_ok = row < p.R;
            if (s.mt != mt_of_place) {
                mt_of_place = s.mt;
                place = xa_place(p, row);
            }
            const float inv = l_sum == 0.0f ? 0.0f : __fdividef(1.0f, l_sum);
            __nv_bfloat16 *dst = p.out + ((long long)s.obs * p.S * p.n_q + s.kvh * p.g + place) * HD;
            float *wo = LIST && s.slot >= 0 ? p.ws_o + ((long long)s.slot * p.ws_rows + lr) * HD : nullptr;
            if (row_ok) {
                if (wo)
                    *reinterpret_cast<float2 *>(p.ws_ml + ((long long)s.slot * p.ws_rows + lr) * 2) = make_float2(m_used, l_sum);
                else if (p.lse)
                    p.lse[((long long)s.obs * p.n_kv + s.kvh) * p.R + row] = l_sum == 0.0f ? -INFINITY : (m_used + xa_log2(l_sum)) * 0.6931471805599453f;
            }
            ok = warp_wait(&pv_done[t], (blk - 1) & 1u, wc, DEV_TIMEOUT_ACCUM);
            if (!ok) break;
            tc_fence_after();
            auto out_of_tmem = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_free[t]);
            };
            if (live) xa_drain<HD, 1>(o_addr, row_ok, dst, inv, p.out_al32, wo, out_of_tmem);
            else out_of_tmem();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == XA_MMA) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// ------------------------------------------------------------------ heads of 256: CTA pairs --
// O alone takes 256 columns of TMEM and K, V of 128 rows 64 KB each, so one CTA has room for one tile and no second block.  A pair of CTAs
// (tcgen05 cta_group::2, M = 256) shares every block: each stages half of K's rows and half of V's columns, and holds one of the
// unit's two tiles.  Two S buffers lie behind O; two warps of the even CTA issue the products, Q K^T up to a block ahead of P V; the odd CTA
// tells the even one what has landed.  P lies over its S, so the S of the block two further on waits for the P V to be complete: the pipe does
// not keep the order of two warps' products.  With a counter of the blocks issued instead, S overtook the last steps of P V in one call of a thousand
// behind another kernel with cold caches, and the counter gave nothing: 64 x 51 tokens over 304 to 816 rows 28.9 us, 29.0 so.
//   8 softmax warps   lane quarter = warp & 3, column half = warp >> 2: the two warps of a row exchange maxima and sums through shared memory
// A unit's O is drained after the next unit's first block, so the pipe does not wait for it.
constexpr int XP_THREADS = 384, XP_LOADER = 8, XP_S = 9, XP_PV = 10, XP_CLEANER = 11;

struct CrossPairSmem {
    static constexpr int HD = 256, CB = 4, CBH = 2;  // 64-element column blocks of the head, and of the half of V that a CTA stages
    static constexpr int STAGES = 2, NS = 2;
    static constexpr int Q_BYTES = CB * 128 * 128, K_BYTES = CB * 64 * 128, V_BYTES = CBH * 128 * 128;
    static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + STAGES * K_BYTES, BAR_OFF = V_OFF + STAGES * V_BYTES;
    static constexpr int SUM_SETS = 2;             // of row-sum slots
    static constexpr int XCH_OFF = BAR_OFF + 256;  // float [2][2 halves][128]: block maxima, used in turn; then [SUM_SETS][2 halves][128]: row sums
    static constexpr int ORDER_OFF = XCH_OFF + (2 + SUM_SETS) * 2 * 128 * 4, TOTAL = ORDER_OFF + (int)sizeof(XaOrder) + 1024;
    static_assert(TOTAL <= 227 * 1024, "shared memory");
};

template <bool LIST>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(XP_THREADS, 1)
cross_attn_pair_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map, const CrossParams p) {
    using L = CrossPairSmem;
    constexpr int HD = L::HD, BKV = XA_BKV;
    constexpr uint32_t ST = L::STAGES, NS = L::NS;
    extern __shared__ uint8_t xp_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(xp_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    uint64_t *q_full = bars, *q_free = bars + 1, *o_done = bars + 2, *o_free = bars + 3;
    uint64_t *k_full = bars + 4, *k_free = bars + 6, *v_full = bars + 8, *v_free = bars + 10;  // [ST]
    uint64_t *s_full = bars + 12, *p_full = bars + 14, *pv_done = bars + 16;                   // [NS]
    uint64_t *meet = bars + 18;                                                                // [4] the two warps of a lane quarter
    uint64_t *v_raw = bars + 22;                                                               // [ST]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 24);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const WaitCtx wc{abort_flag, p.status};
    const uint32_t both = rank == 0 ? 2u : 1u;  // even CTA: its own TMA and the odd CTA's word
    XaOrder &order = *reinterpret_cast<XaOrder *>(smem + L::ORDER_OFF);
    if (!LIST) xa_sort_clear(order, XP_THREADS);

    if (threadIdx.x == 0) {
        mbar_init(q_full, both);
        mbar_init(q_free, 1);
        mbar_init(o_done, 1);
        mbar_init(o_free, 16);  // the softmax warps of both CTAs (used in the even one)
        for (uint32_t i = 0; i < ST; ++i) {
            mbar_init(&k_full[i], both);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_full[i], both);
            mbar_init(&v_free[i], 1);
            mbar_init(&v_raw[i], 1);
        }
        for (uint32_t i = 0; i < NS; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 16);
            mbar_init(&pv_done[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&meet[i], 64);
        *abort_flag = 0;
        fence_barrier_init();
    }
    __syncthreads();
    cluster_sync_all();
    if (warp == XP_S) {
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
        tma_prefetch_desc(&v_map);
    }
    pdl_wait();
    pdl_launch_dependents();  // after the wait: cross_combine_kernel reads the lengths before its own

    auto len_of = [&](int obs) { return xa_len(p, obs); };
    if (!LIST) xa_sort<XP_THREADS>(p, order);
    if (warp < XP_LOADER) xa_fill_empty<HD, LIST>(p, order, blockIdx.x >> 1, rank * 32 * XP_LOADER + threadIdx.x, 64 * XP_LOADER);
    XaWork<LIST, decltype(len_of)> work(len_of, p, order, blockIdx.x >> 1);
    XaSegment s;
    bool ok = true;
    uint32_t si = 0, jb = 0;  // segments and blocks so far

    if (warp == XP_LOADER) {
        for (; ok && work.next(s); ++si) {
            const int item = s.obs * p.n_kv + s.kvh;
            const int pad_lo = s.pad_lo, pad_hi = s.pad_hi;
            ok = warp_wait(q_free, (si & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
            if (!ok) break;
            if (elect_one()) {
                mbar_expect_tx(q_full, L::Q_BYTES);
                for (int cb = 0; cb < L::CB; ++cb)
                    tma_load_3d(smem + cb * 16384, &q_map, q_full, cb * 64, s.mt * 256 + (int)rank * 128, item);
            }
            for (int j = s.j0; j < s.j1; ++j, ++jb) {
                const uint32_t st = jb % ST, ph = (jb / ST) & 1u;
                ok = warp_wait(&k_free[st], ph ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                if (elect_one()) {
                    mbar_expect_tx(&k_full[st], L::K_BYTES);
                    for (int cb = 0; cb < L::CB; ++cb)
                        tma_load_3d(smem + L::K_OFF + st * L::K_BYTES + cb * 8192, &k_map, &k_full[st], cb * 64, j * BKV + (int)rank * 64,
                                    p.page0 + item);
                }
                ok = warp_wait(&v_free[st], ph ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                if (elect_one()) {
                    uint64_t *landed = xa_dirty(j * BKV, s.len, pad_lo, pad_hi) ? &v_raw[st] : &v_full[st];
                    mbar_expect_tx(landed, L::V_BYTES);
                    for (int cb = 0; cb < L::CBH; ++cb)
                        tma_load_3d(smem + L::V_OFF + st * L::V_BYTES + cb * 16384, &v_map, landed, ((int)rank * L::CBH + cb) * 64,
                                    j * BKV, p.page0 + item);
                }
            }
        }
    } else if (warp == XP_CLEANER) {  // of this CTA's half of V's columns
        uint32_t raw_phase = 0;
        while (ok && work.next(s)) xa_clean_blocks<L::CBH>(s, ok, jb, smem + L::V_OFF, ST, L::V_BYTES, v_raw, v_full, raw_phase, wc);
    } else if (warp == XP_S) {
        if (rank == 0) {
            constexpr uint32_t idesc_s = make_idesc(1, 1, 1, 0, 0, 256, BKV);
            const uint64_t q_desc0 = smem_desc_sw128(smem_u32(smem), 16, 1024), k_desc0 = smem_desc_sw128(smem_u32(smem) + L::K_OFF, 16, 1024);
            for (; ok && work.next(s); ++si) {
                ok = warp_wait(q_full, si & 1u, wc, DEV_TIMEOUT_FULL);
                for (int j = s.j0; ok && j < s.j1; ++j, ++jb) {
                    ok = warp_wait(&k_full[jb % ST], (jb / ST) & 1u, wc, DEV_TIMEOUT_FULL);
                    // the P V of the block that used this S buffer has read its weights
                    if (ok && jb >= NS) ok = warp_wait(&pv_done[jb % NS], (jb / NS & 1u) ^ 1u, wc, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t st = jb % ST, d = tmem_base + HD + (jb % NS) * BKV;
                    const uint64_t k_desc = k_desc0 + (uint64_t)(st * (L::K_BYTES >> 4));
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk)
                            mma_f16_pair(d, q_desc0 + (uint64_t)((kk >> 2) * 1024 + (kk & 3) * 2), k_desc + (uint64_t)((kk >> 2) * 512 + (kk & 3) * 2),
                                         idesc_s, kk != 0 ? 1u : 0u);
                        tc_commit_pair(&s_full[jb % NS], 3);
                        tc_commit_pair(&k_free[st], 3);
                        if (j + 1 == s.j1) tc_commit_pair(q_free, 3);
                    }
                }
            }
        } else {
            for (; ok && work.next(s); ++si) {
                ok = warp_wait(q_full, si & 1u, wc, DEV_TIMEOUT_FULL);
                if (!ok) break;
                if (lane == 0) mbar_arrive_cluster(q_full, 0);
                for (int j = s.j0; j < s.j1; ++j, ++jb) {
                    const uint32_t st = jb % ST, ph = (jb / ST) & 1u;
                    ok = warp_wait(&k_full[st], ph, wc, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_cluster(&k_full[st], 0);
                    ok = warp_wait(&v_full[st], ph, wc, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_cluster(&v_full[st], 0);
                }
            }
        }
    } else if (warp == XP_PV) {
        if (rank == 0) {
            constexpr uint32_t idesc_o = make_idesc(1, 1, 1, 0, 1, 256, HD);
            const uint64_t v_desc0 = smem_desc_sw128(smem_u32(smem) + L::V_OFF, 16384, 1024);
            for (; ok && work.next(s); ++si) {
                for (int j = s.j0; j < s.j1; ++j, ++jb) {
                    const uint32_t sb = jb % NS, st = jb % ST;
                    ok = warp_wait(&p_full[sb], (jb / NS) & 1u, wc, DEV_TIMEOUT_FULL);
                    if (ok) ok = warp_wait(&v_full[st], (jb / ST) & 1u, wc, DEV_TIMEOUT_FULL);
                    if (ok && j == s.j0) ok = warp_wait(o_free, (si & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t v_desc = v_desc0 + (uint64_t)(st * (L::V_BYTES >> 4));
                    const uint32_t p_tmem = tmem_base + HD + sb * BKV;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < BKV / 16; ++kk)
                            mma_f16_tmem_a_pair(tmem_base, p_tmem + (uint32_t)(kk * 8), v_desc + (uint64_t)(kk * 128), idesc_o,
                                                j != s.j0 || kk != 0 ? 1u : 0u);
                        tc_commit_pair(&pv_done[sb], 3);
                        tc_commit_pair(&v_free[st], 3);
                        if (j + 1 == s.j1) tc_commit_pair(o_done, 3);
                    }
                }
            }
        }
    } else {
        const int qtr = warp & 3, half = warp >> 2;
        const uint32_t lane_sel = (uint32_t)(qtr * 32) << 16;
        float *xch = reinterpret_cast<float *>(smem + L::XCH_OFF);
        const int my_slot = qtr * 32 + lane, lr = (int)rank * 128 + my_slot;  // row of the unit
        const F2 scale2 = f2(p.scale_log2, p.scale_log2);
        uint32_t met = 0;
        auto pair_sync = [&]() -> bool {
            mbar_arrive(&meet[qtr]);
            return warp_wait(&meet[qtr], (met++) & 1u, wc, DEV_TIMEOUT_MISC);
        };
        auto arrive_even = [&](uint64_t *bar) {  // one arrival per warp on the even CTA's barrier
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(bar);
                else mbar_arrive_cluster(bar, 0);
            }
        };
        int mt_of_place = -1, place = 0;  // of this thread's row: token * n_q + head of the kv head's group
        auto is_live = [&](const XaSegment &sg) { return sg.mt * 256 + (int)rank * 128 + qtr * 32 < p.R; };  // has the warp rows
        // segment `u` is complete: O / l -> bf16 -> out, or the piece into the workspace
        auto drain = [&](uint32_t u, const XaSegment &sg, float m, float l_mine) -> bool {
            const bool live = is_live(sg);
            const int row = sg.mt * 256 + lr;
            const bool row_ok = row < p.R;
            float inv = 0.0f, *wo = nullptr;
            __nv_bfloat16 *dst = nullptr;
            if (live) {  // while the last P V runs
                // Two sets of slots, used in turn.  One was not enough: a last segment of one block is drained right behind the drain before
                // it, and a warp could write its sum while the other, late out of their meeting, had yet to read the one that stood there.
                float *sums = xch + 512 + (u % L::SUM_SETS) * 256;
                sums[half * 128 + my_slot] = l_mine;
                if (!pair_sync()) return false;
                const float l = l_mine + sums[(half ^ 1) * 128 + my_slot];
                if (sg.mt != mt_of_place) {
                    mt_of_place = sg.mt;
                    place = xa_place(p, row);
                }
                inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
                dst = p.out + ((long long)sg.obs * p.S * p.n_q + sg.kvh * p.g + place) * HD + half * (HD / 2);
                if (LIST && sg.slot >= 0) wo = p.ws_o + ((long long)sg.slot * p.ws_rows + lr) * HD + half * (HD / 2);
                if (row_ok && half == 0) {
                    if (wo)
                        *reinterpret_cast<float2 *>(p.ws_ml + ((long long)sg.slot * p.ws_rows + lr) * 2) = make_float2(m, l);
                    else if (p.lse)
                        p.lse[((long long)sg.obs * p.n_kv + sg.kvh) * p.R + row] = l == 0.0f ? -INFINITY : (m + xa_log2(l)) * 0.6931471805599453f;
                }
            }
            if (!warp_wait(o_done, u & 1u, wc, DEV_TIMEOUT_ACCUM)) return false;
            tc_fence_after();
            auto out_of_tmem = [&]() {
                tc_fence_before();
                arrive_even(o_free);
            };
            if (live) xa_drain<HD / 2, 2>(tmem_base + lane_sel + (uint32_t)(half * (HD / 2)), row_ok, dst, inv, p.out_al32, wo, out_of_tmem);
            else out_of_tmem();
            return true;  // (this set is next written behind segment u + 1's meeting, or that of segment u + 2's first block)
        };
        XaSegment prev;
        float prev_m = 0.0f, prev_l = 0.0f;
        for (bool here = true; ok && here; ++si) {
            here = work.next(s);
            if (!here) s.j0 = s.mt = 0, s.j1 = 1;  // behind the last segment: its drain alone, by the same instructions (a copy of them would not be cached)
            const int pad_lo = s.pad_lo, pad_hi = s.pad_hi;
            const bool live = here && is_live(s);
            float m_used = -INFINITY, l_sum = 0.0f;  // running maximum in log2 units (the same in both halves), this half's part of the row sum
            for (int j = s.j0; j < s.j1; ++j, ++jb) {
                const uint32_t sb = jb % NS;
                const uint32_t s_addr = tmem_base + HD + sb * BKV + lane_sel;
                if (here) {
                    ok = warp_wait(&s_full[sb], (jb / NS) & 1u, wc, DEV_TIMEOUT_FULL);
                    if (!ok) break;
                    tc_fence_after();
                }
                if (live) {
                uint32_t x[2][32];
                tmem_ld32(s_addr + (uint32_t)(half * 64), x[0]);
                tmem_ld32(s_addr + (uint32_t)(half * 64 + 32), x[1]);
                tmem_ld_wait();
                const int b0 = j * BKV, c0 = b0 + half * 64;
                const bool dirty = xa_dirty(b0, s.len, pad_lo, pad_hi);
                if (dirty) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) xa_mask32(x[i], c0 + i * 32, s.len, pad_lo, pad_hi);
                }
                float mx[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mx[i] = fmaxf(__uint_as_float(x[i][0]), __uint_as_float(x[i][1]));
#pragma unroll
                    for (int e = 2; e < 32; e += 2) mx[i] = xa_max3(mx[i], __uint_as_float(x[i][e]), __uint_as_float(x[i][e + 1]));
                }
                float bm = fmaxf(mx[0], mx[1]);
                float *xm = xch + (jb & 1u) * 256;  // two sets of slots, used in turn: one meeting per block is enough
                xm[half * 128 + my_slot] = bm;
                ok = pair_sync();
                if (!ok) break;
                bm = fmaxf(bm, xm[(half ^ 1) * 128 + my_slot]) * p.scale_log2;
                float factor = 1.0f;
                const bool raise = bm > m_used + XA_RAISE;
                if (raise) {
                    factor = m_used == -INFINITY ? 0.0f : xa_ex2(m_used - bm);
                    m_used = bm;
                    l_sum *= factor;
                }
                if (j > s.j0 && __any_sync(0xffffffffu, raise)) {  // O was summed under the old maximum
                    ok = warp_wait(&pv_done[(jb - 1) % NS], ((jb - 1) / NS) & 1u, wc, DEV_TIMEOUT_ACCUM);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 32) {
                        uint32_t ov[32];
                        tmem_ld32(tmem_base + lane_sel + (uint32_t)c, ov);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * factor);
                        tmem_st32(tmem_base + lane_sel + (uint32_t)c, ov);
                    }
                    tmem_st_wait();
                }
                const float mref = m_used == -INFINITY ? 0.0f : m_used;
                const F2 neg = f2(-mref, -mref);
                F2 sum[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
                uint32_t pk[32];
#pragma unroll
                for (int e = 0; e < 64; e += 2) {
                    const F2 a = f2_fma(f2(__uint_as_float(x[e >> 5][e & 31]), __uint_as_float(x[e >> 5][(e & 31) + 1])), scale2, neg);
                    float a0, a1;
                    f2_get(a, a0, a1);
                    const F2 pr = f2(xa_ex2(a0), xa_ex2(a1));
                    sum[(e >> 1) & 1] = f2_add(sum[(e >> 1) & 1], pr);
                    pk[e >> 1] = f2_bf16(pr);  // weights are rounded to 8 bits for the product, their sum is not
                }
                float u0, u1, u2, u3;
                f2_get(sum[0], u0, u1);
                f2_get(sum[1], u2, u3);
                l_sum += (u0 + u1) + (u2 + u3);
                // P (128 rows of V, bf16) over the first 64 columns of S; both halves have read theirs: they met
                tmem_st32(s_addr + (uint32_t)(half * 32), pk);
                tmem_st_wait();
                }
                if (here) {
                    tc_fence_before();
                    arrive_even(&p_full[sb]);
                }
                if (j == s.j0 && si > 0) {
                    ok = drain(si - 1, prev, prev_m, prev_l);
                    if (!ok) break;
                }
            }
            if (!ok) break;
            prev = s;
            prev_m = m_used;
            prev_l = l_sum;
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // neither CTA may exit while the other can still signal its barriers
    if (warp == XP_S) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ------------------------------------------------------------------ few query rows --
// Units of up to 16 rows (a token, of every head of a group): K and V are read once and next to nothing is computed, so what counts is bytes in
// flight and a short chain behind them.  Tiles of 128 or 256 rows would be empty for the most part, and TMEM, its allocation and the pair's
// launch cost more than the products; 16 rows are what mma.sync (16 x 8 x 16) takes.  Measured: see cross_plan.
//   loader warp   TMA: Q (16 rows), K and V in blocks of 64 rows, one barrier for both, running ahead over the segments
//   4 warps       16 of a block's rows each, with a maximum, a sum and an O of their own; a warp zeroes its hidden rows of V itself.
//                 A segment's end: their O meet in shared memory and are added by all
constexpr int XF_ROWS = 16, XF_WARPS = 4, XF_THREADS = 32 * (XF_WARPS + 1), XF_BKV = 16 * XF_WARPS;

template <int HD>
struct CrossFewSmem {
    static constexpr int CB = HD / 64, PER_SM = HD == 256 ? 1 : 2;                        // CTAs
    static constexpr int STAGES = HD == 64 ? 4 : 2, QS = HD == 128 ? 1 : 2;               // blocks of K and V; segments' Q
    static constexpr int Q_BYTES = CB * XF_ROWS * 128, KV_BYTES = CB * XF_BKV * 128;      // [CB][rows][128 B]
    static constexpr int Q_OFF = STAGES * 2 * KV_BYTES, O_OFF = Q_OFF + QS * Q_BYTES, O_STRIDE = HD + 8;
    static constexpr int ML_OFF = O_OFF + XF_WARPS * XF_ROWS * O_STRIDE * 4;              // float O [warp][row][O_STRIDE], float2 [warp][row]
    static constexpr int BAR_OFF = ML_OFF + XF_WARPS * XF_ROWS * 8, ORDER_OFF = BAR_OFF + 128, TOTAL = ORDER_OFF + (int)sizeof(XaOrder) + 1024;
    static_assert(ORDER_OFF % 16 == 0 && TOTAL <= 227 * 1024 && PER_SM * (TOTAL + 1024) <= 228 * 1024, "shared memory");
};
__device__ __forceinline__ void xf_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void xf_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void xf_ldmatrix_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <int HD, bool LIST>
__global__ void __launch_bounds__(XF_THREADS, CrossFewSmem<HD>::PER_SM)
cross_few_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                 const CrossParams p) {
    using L = CrossFewSmem<HD>;
    constexpr uint32_t NS = L::STAGES, QS = L::QS;
    extern __shared__ uint8_t xf_smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(xf_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::BAR_OFF);
    uint64_t *full = bars, *free_ = bars + 4, *q_full = bars + 8, *q_free = bars + 10, *o_full = bars + 12, *o_free = bars + 13;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(bars + 14);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wc{abort_flag, p.status};
    XaOrder &order = *reinterpret_cast<XaOrder *>(smem + L::ORDER_OFF);
    if (!LIST) xa_sort_clear(order, XF_THREADS);
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&free_[i], XF_WARPS);
        }
        for (uint32_t i = 0; i < QS; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_free[i], XF_WARPS);
        }
        mbar_init(o_full, XF_WARPS);
        mbar_init(o_free, XF_WARPS);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&q_map);
        tma_prefetch_desc(&k_map);
        tma_prefetch_desc(&v_map);
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();  // after the wait: cross_combine_kernel reads the lengths before its own
    auto len_of = [&](int obs) { return xa_len(p, obs); };
    if (!LIST) xa_sort<XF_THREADS>(p, order);
    XaWork<LIST, decltype(len_of)> work(len_of, p, order, blockIdx.x);
    XaSegment s;
    bool ok = true;
    uint32_t it = 0, si = 0;  // blocks of 64 rows and segments so far
    auto begin_of = [&]() { return s.j0 * (XA_BKV / XF_BKV); };
    auto end_of = [&]() { return min(s.j1 * (XA_BKV / XF_BKV), (s.len + XF_BKV - 1) / XF_BKV); };
    if (warp == XF_WARPS) {
        for (; ok && work.next(s); ++si) {
            const int item = s.obs * p.n_kv + s.kvh;
            const uint32_t qs = si % QS;
            ok = warp_wait(&q_free[qs], (si / QS & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
            if (!ok) break;
            if (elect_one()) {
                mbar_expect_tx(&q_full[qs], L::Q_BYTES);
                for (int cb = 0; cb < L::CB; ++cb)
                    tma_load_3d(smem + L::Q_OFF + qs * L::Q_BYTES + cb * (XF_ROWS * 128), &q_map, &q_full[qs], cb * 64, 0, item);
            }
            const int end = end_of();
            for (int i = begin_of(); i < end; ++i, ++it) {
                const uint32_t st = it % NS;
                ok = warp_wait(&free_[st], (it / NS & 1u) ^ 1u, wc, DEV_TIMEOUT_EMPTY);
                if (!ok) break;
                if (elect_one()) {
                    uint8_t *stage = smem + st * (2 * L::KV_BYTES);
                    mbar_expect_tx(&full[st], 2 * L::KV_BYTES);
                    for (int cb = 0; cb < L::CB; ++cb) tma_load_3d(stage + cb * (XF_BKV * 128), &k_map, &full[st], cb * 64, i * XF_BKV, p.page0 + item);
                    for (int cb = 0; cb < L::CB; ++cb)
                        tma_load_3d(stage + L::KV_BYTES + cb * (XF_BKV * 128), &v_map, &full[st], cb * 64, i * XF_BKV, p.page0 + item);
                }
            }
        }
    } else {
        const int r = lane >> 2, t = lane & 3;
        float *const s_o = reinterpret_cast<float *>(smem + L::O_OFF);
        float2 *const s_ml = reinterpret_cast<float2 *>(smem + L::ML_OFF);
        // rows of the 8 x 8 matrices that this lane gives ldmatrix the addresses of, and which 16-byte chunk (swizzled by the row)
        const int row_a = (lane & 7) + (lane >> 3 & 1) * 8, chunk_a = lane >> 4;  // A, and V transposed
        const int row_b = (lane & 7) + (lane >> 4) * 8, chunk_b = lane >> 3 & 1;  // K
        const int swz = lane & 7;
        const uint32_t base = smem_u32(smem);
        for (; ok && work.next(s); ++si) {
            const uint32_t qs = si % QS;
            ok = warp_wait(&q_full[qs], si / QS & 1u, wc, DEV_TIMEOUT_FULL);
            if (!ok) break;
            const uint32_t q_at = base + L::Q_OFF + qs * L::Q_BYTES + (uint32_t)(row_a * 128);
            float acc[HD / 8][4];
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // of query rows r and r + 8; l: of this lane's columns
            const int end = end_of();
            for (int i = begin_of(); i < end; ++i, ++it) {
                const uint32_t st = it % NS, k_at = base + st * (2 * L::KV_BYTES) + (uint32_t)(warp * 16 * 128), v_at = k_at + L::KV_BYTES;
                ok = warp_wait(&full[st], it / NS & 1u, wc, DEV_TIMEOUT_FULL);
                if (!ok) break;
                const int first = i * XF_BKV + warp * 16;
                auto seen = [&](int row) { return row < s.len && (row < s.pad_lo || row >= s.pad_hi); };
                const bool dirty = first + 16 > s.len || (first < s.pad_hi && first + 16 > s.pad_lo);
                if (dirty) {  // hidden rows of V meet weights of 0, and 0 times what stands there need not be 0
                    uint4 *v = reinterpret_cast<uint4 *>(smem + st * (2 * L::KV_BYTES) + L::KV_BYTES) + warp * 16 * 8;
                    for (int n = lane; n < 16 * 8; n += 32)
                        if (!seen(first + n / 8))
                            for (int cb = 0; cb < L::CB; ++cb) v[cb * (XF_BKV * 8) + n] = make_uint4(0, 0, 0, 0);
                    __syncwarp();
                }
                float c[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    uint32_t a[4], b[4];
                    xf_ldmatrix(a, q_at + (uint32_t)((kk >> 2) * (XF_ROWS * 128) + (((kk & 3) * 2 + chunk_a) ^ swz) * 16));
                    xf_ldmatrix(b, k_at + (uint32_t)((kk >> 2) * (XF_BKV * 128) + row_b * 128 + (((kk & 3) * 2 + chunk_b) ^ swz) * 16));
                    xf_mma(c[0], a, b[0], b[1]);
                    xf_mma(c[1], a, b[2], b[3]);
                }
                // c[n][e]: query row r + 8 (e / 2), cached row first + 8 n + 2 t + e % 2
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) c[n][e] = !dirty || seen(first + 8 * n + 2 * t + (e & 1)) ? c[n][e] * p.scale_log2 : -INFINITY;
                float f[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float top = fmaxf(fmaxf(c[0][2 * h], c[0][2 * h + 1]), fmaxf(c[1][2 * h], c[1][2 * h + 1]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    top = fmaxf(top, m[h]);
                    const float ref = top == -INFINITY ? 0.0f : top;
                    f[h] = m[h] == -INFINITY ? 0.0f : xa_ex2(m[h] - ref);
                    m[h] = top;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        c[n][2 * h] = xa_ex2(c[n][2 * h] - ref);
                        c[n][2 * h + 1] = xa_ex2(c[n][2 * h + 1] - ref);
                    }
                    l[h] = l[h] * f[h] + ((c[0][2 * h] + c[0][2 * h + 1]) + (c[1][2 * h] + c[1][2 * h + 1]));
                }
                if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) {
                        acc[n][0] *= f[0];
                        acc[n][1] *= f[0];
                        acc[n][2] *= f[1];
                        acc[n][3] *= f[1];
                    }
                }
                // weights are rounded to 8 bits for the product, their sum is not
                const uint32_t w[4] = {f2_bf16(f2(c[0][0], c[0][1])), f2_bf16(f2(c[0][2], c[0][3])), f2_bf16(f2(c[1][0], c[1][1])),
                                       f2_bf16(f2(c[1][2], c[1][3]))};
#pragma unroll
                for (int n = 0; n < HD / 16; ++n) {
                    uint32_t b[4];
                    xf_ldmatrix_t(b, v_at + (uint32_t)((n >> 2) * (XF_BKV * 128) + row_a * 128 + (((n & 3) * 2 + chunk_a) ^ swz) * 16));
                    xf_mma(acc[2 * n], w, b[0], b[1]);
                    xf_mma(acc[2 * n + 1], w, b[2], b[3]);
                }
                // What this lane read of the stage (and of Q), and the zeros it wrote, come before the fill that follows the arrival; the reads have
                // arrived, the products in front of the fence take them.
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&free_[st]);
            }
            if (!ok) break;
            if (lane == 0) mbar_arrive(&q_free[qs]);  // (fenced with the segment's last block; a segment has at least one)
            ok = warp_wait(o_free, (si & 1u) ^ 1u, wc, DEV_TIMEOUT_MISC);  // the segment before has been read
            if (!ok) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                if (t == 0) s_ml[warp * XF_ROWS + r + 8 * h] = make_float2(m[h], l[h]);
                if (r + 8 * h < p.R) {
                    float2 *o = reinterpret_cast<float2 *>(s_o + (warp * XF_ROWS + r + 8 * h) * L::O_STRIDE + 2 * t);
#pragma unroll
                    for (int n = 0; n < HD / 8; ++n) o[4 * n] = make_float2(acc[n][2 * h], acc[n][2 * h + 1]);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(o_full);
            ok = warp_wait(o_full, si & 1u, wc, DEV_TIMEOUT_MISC);
            if (!ok) break;
            for (int row = warp; row < p.R; row += XF_WARPS) {
                float f[XF_WARPS], top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < XF_WARPS; ++w) {
                    f[w] = s_ml[w * XF_ROWS + row].x;
                    top = fmaxf(top, f[w]);
                }
                F2 o[HD / 64];  // two columns in 64
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) o[c] = f2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < XF_WARPS; ++w) {
                    f[w] = f[w] == -INFINITY ? 0.0f : xa_ex2(f[w] - top);
                    sum = fmaf(s_ml[w * XF_ROWS + row].y, f[w], sum);
                    const float2 *x = reinterpret_cast<const float2 *>(s_o + (w * XF_ROWS + row) * L::O_STRIDE) + lane;
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) o[c] = f2_fma(f2(x[32 * c].x, x[32 * c].y), f2(f[w], f[w]), o[c]);
                }
                if (LIST && s.slot >= 0) {
                    const long long piece = (long long)s.slot * p.ws_rows + row;
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) {
                        float x, y;
                        f2_get(o[c], x, y);
                        reinterpret_cast<float2 *>(p.ws_o + piece * HD)[32 * c + lane] = make_float2(x, y);
                    }
                    if (lane == 0) *reinterpret_cast<float2 *>(p.ws_ml + piece * 2) = make_float2(top, sum);
                    continue;
                }
                const float inv = sum == 0.0f ? 0.0f : __fdividef(1.0f, sum);
                uint32_t *dst = reinterpret_cast<uint32_t *>(p.out + ((long long)s.obs * p.S * p.n_q + s.kvh * p.g + xa_place(p, row)) * HD) + lane;
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) dst[32 * c] = f2_bf16(f2_mul(o[c], f2(inv, inv)));
                if (p.lse && lane == 0)
                    p.lse[((long long)s.obs * p.n_kv + s.kvh) * p.R + row] = sum == 0.0f ? -INFINITY : (top + xa_log2(sum)) * 0.6931471805599453f;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
        }
        xa_fill_empty<HD, LIST>(p, order, blockIdx.x, threadIdx.x, 32 * XF_WARPS);
    }
    __syncthreads();
}

// Rows of units that were cut: M = max m_i, O = sum O_i 2^(m_i - M), l = sum l_i 2^(m_i - M), pieces in order.  Block x looks after unit x,
// or, where there are more units than CTAs, after the one that CTA x began and did not finish.  TEAM warps share a row: 1 where a unit's rows
// are many (two pieces or three of each), 32 where they are few and the pieces as many as there are CTAs (one token, 8 / 1 heads of 256,
// over 16,001 rows, the whole call with tiles of 256 rows: 43 us with a warp per row, 24 so).
template <int HD, int TEAM>
__global__ void __launch_bounds__(TEAM > 1 ? 32 * TEAM : 256) cross_combine_kernel(const CrossParams p) {
    constexpr int WARPS = TEAM > 1 ? TEAM : 8;
    __shared__ __align__(8) float s_o[WARPS][TEAM > 1 ? HD : 1], s_l[WARPS], s_m[WARPS];
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int total = xa_total_blocks(p), n = min(p.n_work, total), upo = p.n_kv * p.n_mt;  // units of an observation
    int obs = 0, u = 0, nb = 0, first = 0, c0 = 0, c1 = 0;  // the unit's observation, place in it and blocks; its first block in the list, the
    if (total > 0) {                                        // CTAs that have that one and the last (the same one: whole, nothing to merge)
        if (p.by_unit) {
            obs = blockIdx.x / upo;
            u = blockIdx.x - obs * upo;
            nb = (xa_len(p, obs) + XA_BKV - 1) / XA_BKV;
            int before = 0;
            for (int i = lane; i < obs; i += 32) before += (xa_len(p, i) + XA_BKV - 1) / XA_BKV;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
            first = before * upo + u * nb;
            if (nb > 0) c0 = xa_cta_of(first, n, total);
        } else if ((int)blockIdx.x < n) {
            c0 = blockIdx.x;
            const int begin = xa_border(c0, n, total), end = xa_border(c0 + 1, n, total);
            auto len_of = [&](int i) { return xa_len(p, i); };
            RaggedCursor cur(len_of, p.n_obs, upo, XA_BKV);
            RaggedUnit at;
            if (cur.find(end - 1, at) && end - 1 - at.block >= begin) {  // (begun before this CTA: the one that began it merges it)
                obs = at.obs;
                u = at.kvh;
                nb = (at.len + XA_BKV - 1) / XA_BKV;
                first = end - 1 - at.block;
            }
        }
        c1 = nb > 0 ? xa_cta_of(first + nb - 1, n, total) : c0;
    }
    // For the pieces; the lengths were complete before the kernel in front let this one begin.  Every block waits, those without work too: who
    // follows this kernel takes its end for the end of the one in front.
    pdl_wait();
    if (c0 == c1) return;
    const int kvh = u / p.n_mt, row0 = (u - kvh * p.n_mt) * p.unit_rows, rows = min(p.R - row0, p.unit_rows);
    constexpr int NV = HD / 64;  // pairs of columns per lane
    for (int r0 = blockIdx.y * (WARPS / TEAM); r0 < rows; r0 += gridDim.y * (WARPS / TEAM)) {
        const int lr = r0 + warp / TEAM, member = warp % TEAM;
        if (TEAM == 1 && lr >= rows) return;
        auto slot_of = [&](int c) { return (long long)(2 * c + (c == c0 ? 1 : 0)) * p.ws_rows + lr; };
        float2 acc[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] = make_float2(0.0f, 0.0f);
        float l = 0.0f, M = -INFINITY;
        for (int c = c0 + member; c <= c1; c += 4 * TEAM) {  // four pieces asked for at once, under the maximum so far
            float2 v[4][NV], ml[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long at = slot_of(min(c + i * TEAM, c1));
                ml[i] = *reinterpret_cast<const float2 *>(p.ws_ml + at * 2);
#pragma unroll
                for (int k = 0; k < NV; ++k) v[i][k] = reinterpret_cast<const float2 *>(p.ws_o + at * HD)[k * 32 + lane];
            }
            // (a piece that was asked for twice has its weight once)
            const float top = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M);
            const float old = M == -INFINITY ? 0.0f : xa_ex2(M - top);
            M = top;
            l *= old;
#pragma unroll
            for (int k = 0; k < NV; ++k) acc[k] = make_float2(acc[k].x * old, acc[k].y * old);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = c + i * TEAM > c1 || ml[i].x == -INFINITY ? 0.0f : xa_ex2(ml[i].x - M);
                l = fmaf(ml[i].y, w, l);
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    acc[k].x = fmaf(v[i][k].x, w, acc[k].x);
                    acc[k].y = fmaf(v[i][k].y, w, acc[k].y);
                }
            }
        }
        const int row = row0 + lr, head = kvh * p.g + row / p.S, tok = row % p.S;
        __nv_bfloat16 *dst = p.out + (((long long)obs * p.S + tok) * p.n_q + head) * HD;
        if (TEAM > 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k) reinterpret_cast<float2 *>(s_o[warp])[k * 32 + lane] = acc[k];
            if (lane == 0) {
                s_l[warp] = l;
                s_m[warp] = M;
            }
            __syncthreads();
            l = 0.0f;
#pragma unroll
            for (int w = 0; w < TEAM; ++w) M = fmaxf(M, s_m[w]);
            float o = 0.0f;
            const int col = threadIdx.x < HD ? threadIdx.x : 0;
#pragma unroll
            for (int w = 0; w < TEAM; ++w) {
                const float scale = s_m[w] == -INFINITY ? 0.0f : xa_ex2(s_m[w] - M);
                l = fmaf(s_l[w], scale, l);
                o = fmaf(s_o[w][col], scale, o);
            }
            const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
            if (threadIdx.x < HD) {
                const int i = col;
                dst[i] = __float2bfloat16_rn(o * inv);
            }
            __syncthreads();
        } else {
            const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
#pragma unroll
            for (int k = 0; k < NV; ++k)
                reinterpret_cast<__nv_bfloat162 *>(dst)[k * 32 + lane] = __floats2bfloat162_rn(acc[k].x * inv, acc[k].y * inv);
        }
        if (p.lse && lane == 0 && member == 0)
            p.lse[((long long)obs * p.n_q + head) * p.S + tok] = l == 0.0f ? -INFINITY : (M + xa_log2(l)) * 0.6931471805599453f;
    }
}

template <int HD>
static int launch_combine(CrossParams p, cudaStream_t stream) {
    const int units = p.n_obs * p.n_kv * p.n_mt;
    p.by_unit = units <= p.n_work ? 1 : 0;
    const unsigned gx = (unsigned)(p.by_unit ? units : p.n_work);
    if (p.ws_rows <= 64)  // a row per block
        return launch_pdl(cross_combine_kernel<HD, 32>, dim3(gx, (unsigned)p.ws_rows), dim3(1024), 0, stream, p);
    return launch_pdl(cross_combine_kernel<HD, 1>, dim3(gx, 8), dim3(256), 0, stream, p);  // 32 rows per block
}

// Units, workers and workspace of a call; the same for the size query and the launch.
struct CrossPlan {
    int unit_rows, n_mt, n_work, ws_rows;
    bool few;            // up to 16 query rows: cross_few_kernel
    long long ws_bytes;  // 0: no unit is cut
};
static CrossPlan cross_plan(int hd, long long items, int R, int max_len, int n_sm) {
    CrossPlan c;
    c.unit_rows = 256;
    c.n_mt = (R + 255) / 256;
    c.few = R <= XF_ROWS;
    c.n_work = c.few ? (hd == 256 ? CrossFewSmem<256>::PER_SM : hd == 128 ? CrossFewSmem<128>::PER_SM : CrossFewSmem<64>::PER_SM) * n_sm : hd == 256 ? n_sm / 2 : n_sm;
    c.ws_rows = R < 256 ? R : 256;
    // Whole units take rounds of n_work; cut ones fill the last round, for the pieces' way through the workspace and a second kernel: the
    // time of some 6 blocks, and of 10 more where the pieces are full tiles.  Cut / whole, us: one token of 8 / 1 heads of 256 over 16,001
    // rows 21 / 233; 4 x 816 tokens of 20 / 5 heads of 128 over 4,097 to 8,190 rows 219 / 199; 64 x 51 tokens of 8 / 1 heads of 256 over
    // 304 to 816 rows 55 / 37; 64 x 50 tokens of 15 / 5 heads of 64 over 113 to 241 rows 45 / 31.  Few rows: only where there are fewer units
    // than CTAs (320 units of one token, heads of 128, 304 to 816 rows: 70 / 35).
    // Few rows against tiles of 256 (cold / pages in L2): one token over 16,001 rows, heads of 256 20.5 / 14.6 against 24.6 / 20.4, of 128 24.6 /
    // 16.6 against 30.7 / 23.8, of 64 20.5 / 13.6 against 26.7 / 20.8; 256 observations of 200 to 400 rows, heads of 256 30.8 / 19.1 against
    // 36.9 / 28.9, of 128 55 / 44 against 68 / 60, of 64 36.9 / 28.9 against 57 / 55; 64 observations of 408 to 816 rows, heads of 256, the
    // same (24.6 / 18.6 against 24.6 / 18.7).
    const long long units = items * c.n_mt, nb = (max_len + XA_BKV - 1) / XA_BKV, rounds = (units + c.n_work - 1) / c.n_work;
    const bool cut = (!c.few || units < c.n_work) && (rounds * c.n_work - units) * nb > (6LL + 10LL * c.ws_rows / 256) * c.n_work;
    c.ws_bytes = cut ? 2LL * c.n_work * c.ws_rows * (hd + 2) * 4 : 0;
    return c;
}

template <int HD>
static int launch_cross(const vlab200_kv_store *st, const void *q, CrossParams &p, const CrossPlan &plan, cudaStream_t stream) {
    const bool list = p.ws_o || p.n_obs > XA_SORT;
    const uint64_t pages = (uint64_t)st->n_layers * st->n_obs * st->n_kv;
    CUtensorMap qmap, kmap, vmap;
    const uint64_t qdims[3] = {(uint64_t)HD, (uint64_t)p.R, (uint64_t)st->n_obs * st->n_kv}, qstr[2] = {(uint64_t)HD * 2, (uint64_t)p.R * HD * 2};
    const uint64_t dims[3] = {(uint64_t)HD, (uint64_t)(p.max_len > 0 ? p.max_len : 1), pages}, str[2] = {(uint64_t)HD * 2, (uint64_t)st->cap * HD * 2};
    const uint32_t few = XF_BKV, qbox[3] = {64, plan.few ? (uint32_t)XF_ROWS : 128u, 1}, vbox[3] = {64, plan.few ? few : 128u, 1};
    const uint32_t kbox[3] = {64, plan.few ? few : HD == 256 ? 64u : 128u, 1};  // a CTA of a pair stages half of a block's K rows
    int rc = make_tensor_map(&qmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q, qdims, qstr, qbox, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = make_tensor_map(&kmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, st->k_pages, dims, str, kbox, CU_TENSOR_MAP_SWIZZLE_128B);
    if (!rc) rc = make_tensor_map(&vmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, st->v_pages, dims, str, vbox, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc) return rc;
    if (plan.few) {
        const auto kernel = list ? cross_few_kernel<HD, true> : cross_few_kernel<HD, false>;
        if ((rc = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), CrossFewSmem<HD>::TOTAL))) return rc;
        rc = launch_pdl(kernel, dim3((unsigned)plan.n_work), dim3(XF_THREADS), CrossFewSmem<HD>::TOTAL, stream, qmap, kmap, vmap, p);
    } else if constexpr (HD == 256) {
        const auto kernel = list ? cross_attn_pair_kernel<true> : cross_attn_pair_kernel<false>;
        if ((rc = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), CrossPairSmem::TOTAL))) return rc;
        rc = launch_pdl(kernel, dim3(2 * (unsigned)plan.n_work), dim3(XP_THREADS), CrossPairSmem::TOTAL, stream, qmap, kmap, vmap, p);
    } else {
        const auto kernel = list ? cross_attn_kernel<HD, true> : cross_attn_kernel<HD, false>;
        if ((rc = ensure_dyn_smem(reinterpret_cast<const void *>(kernel), CrossSmem<HD>::TOTAL))) return rc;
        rc = launch_pdl(kernel, dim3((unsigned)plan.n_work), dim3(XA_THREADS), CrossSmem<HD>::TOTAL, stream, qmap, kmap, vmap, p);
    }
    if (rc || !p.ws_o) return rc;
    return launch_combine<HD>(p, stream);
}

// More query rows per kv head, pages or blocks of 256 x 128 scores than are counted in 32 bits?
static bool cross_too_large(const vlab200_kv_store *st, int S, int n_q, int max_len) {
    const long long R = (long long)(n_q / st->n_kv) * S;
    return R > 0x7fffff00LL || size_product({st->n_obs, st->n_kv, st->n_layers}) > 0x7fffff00LL ||
           size_product({st->n_obs, st->n_kv, (R + 255) / 256, (max_len + 127LL) / 128}) > 0x7fffff00LL;
}
static bool cross_shape_ok(const vlab200_kv_store *st, int S, int n_q) {
    return st && st->n_layers > 0 && st->n_obs > 0 && st->n_kv > 0 && st->cap > 0 && S > 0 && n_q > 0 && n_q % st->n_kv == 0;
}

}  // namespace vb

extern "C" {

int64_t vlab200_cross_attention_ws_bytes(const vlab200_kv_store *st, int32_t S, int32_t n_q, int32_t max_len) {
    if (!vb::cross_shape_ok(st, S, n_q) || max_len < 0 || max_len > st->cap || vb::cross_too_large(st, S, n_q, max_len)) return -1;
    const int n_sm = vb::sm_count();
    return n_sm ? vb::cross_plan(st->head_dim, (long long)st->n_obs * st->n_kv, (n_q / st->n_kv) * S, max_len, n_sm).ws_bytes : -1;
}

int32_t vlab200_cross_attention(const vlab200_kv_store *st, int32_t layer, const void *q, void *out, float *lse, int32_t S, int32_t n_q,
                                const int32_t *lens, int32_t max_len, const int32_t *pad_ranges, float scale, void *ws,
                                int64_t ws_bytes, void *stream) {
    if (!vb::cross_shape_ok(st, S, n_q) || !st->k_pages || !st->v_pages || !q || !out) return VLAB200_ERR_ARG;
    if (layer < 0 || layer >= st->n_layers || max_len < 0 || max_len > st->cap || !(scale >= 0.0f) || ws_bytes < 0) return VLAB200_ERR_ARG;
    const uintptr_t al = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(st->k_pages) |
                         reinterpret_cast<uintptr_t>(st->v_pages);
    if ((al & 15) || (reinterpret_cast<uintptr_t>(ws) & 31)) return VLAB200_ERR_ARG;
    const int hd = st->head_dim;
    if (hd != 64 && hd != 128 && hd != 256) return VLAB200_ERR_UNSUPPORTED;
    if (vb::cross_too_large(st, S, n_q, max_len)) {
        vb::set_last_error("cross_attention: more than 2^31 query rows per kv head, pages or blocks of 256 x 128 scores");
        return VLAB200_ERR_UNSUPPORTED;
    }
    const long long R = (long long)(n_q / st->n_kv) * S, items = (long long)st->n_obs * st->n_kv;
    const long long q_b = vb::size_product({items, R, hd, 2}), pages_b = vb::size_product({st->n_layers, items, st->cap, hd, 2});
    const vb::MemRange written[] = {{out, q_b}, {lse, items * R * 4}, {ws, ws_bytes}};
    const vb::MemRange read[] = {{q, q_b}, {st->k_pages, pages_b}, {st->v_pages, pages_b}, {lens, st->n_obs * 4LL}, {pad_ranges, st->n_obs * 8LL}};
    if (vb::writes_overlap(written, 3, read, 5)) return VLAB200_ERR_ARG;
    const int n_sm = vb::sm_count();
    if (!n_sm) return vb::cuda_fail(cudaGetLastError(), "sm_count");
    const vb::CrossPlan plan = vb::cross_plan(hd, items, (int)R, max_len, n_sm);
    if (ws && ws_bytes < plan.ws_bytes) return VLAB200_ERR_ARG;
    vb::CrossParams p;
    p.out = static_cast<__nv_bfloat16 *>(out);
    p.lse = lse;
    p.lens = lens;
    p.pad = pad_ranges;
    p.S = S;
    p.n_q = n_q;
    p.n_kv = st->n_kv;
    p.g = n_q / st->n_kv;
    p.R = (int)R;
    p.n_obs = st->n_obs;
    p.max_len = max_len;
    p.page0 = layer * st->n_obs * st->n_kv;
    p.n_mt = plan.n_mt;
    p.unit_rows = plan.unit_rows;
    p.n_work = plan.n_work;
    const long long upo = (long long)p.n_kv * p.n_mt;
    p.round_r = (int)(p.n_work / upo);
    p.round_u = (int)(p.n_work % upo);
    p.bin_shift = 0;
    while (((max_len + 127LL) / 128 >> p.bin_shift) > vb::XA_BINS - 2) ++p.bin_shift;
    p.out_al32 = (reinterpret_cast<uintptr_t>(out) & 31) == 0 ? 1 : 0;
    p.scale_log2 = 1.4426950408889634f * (scale > 0.0f ? scale : 1.0f / sqrtf((float)hd));
    p.status = vb::device_status_ptr();
    if (!p.status) return vb::cuda_fail(cudaGetLastError(), "device_status_ptr");
    p.ws_rows = plan.ws_rows;
    p.ws_o = plan.ws_bytes ? static_cast<float *>(ws) : nullptr;
    p.ws_ml = p.ws_o ? p.ws_o + 2LL * plan.n_work * plan.ws_rows * hd : nullptr;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (hd == 64) return vb::launch_cross<64>(st, q, p, plan, cs);
    if (hd == 128) return vb::launch_cross<128>(st, q, p, plan, cs);
    return vb::launch_cross<256>(st, q, p, plan, cs);
}

}  // extern "C"
