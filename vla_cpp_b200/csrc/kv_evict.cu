// Eviction from a prefix cache: of every page (layer, observation, kv head) the `keep` rows that matter most move to another store, in
// their order.  The first `sink` and the last `recent` rows of an observation stay in any case, then the rows of largest accumulated
// attention weight (vlab200_key_mass), ties to the lower row.
//
// The keep-th largest key of a page decides -- the weight's bits mapped so that they compare as whole numbers, protected rows on top,
// no-numbers at the bottom.  Pages of up to 1,024 rows: one kernel, a warp of every block finds it bit by bit with the keys in registers, then
// the block copies its rows.  Longer pages: a block each finds it 8 bits at a time from histograms, a second kernel copies.  K and V rows go
// 16 bytes per thread: all there is to move, HBM bounds it.  Measured (graph replay, cold L2): 1,152 pages of 304 to 816 rows of 256, 387 of
// them kept, 158 us = 5.7 TB/s of the 6.45 of a copy (151 in a stream of calls), 144 of them the copy's; with histograms and a second kernel
// 184.  16 pages of 241 rows of 64, 120 kept, 10.2 us (14.3).
// Above 1,024 rows the selection bounds it, a chain of barriers per 256 rows, five times over a page's weights: 80 pages of 16,384 rows of 64,
// 4,096 kept, 170 us = 1.0 TB/s; 144 pages of 8,192 rows of 256, 2,048 kept, 193 us = 3.2; 1,152 pages of 1,600 rows of 256, 800 kept, 387 us =
// 4.9.  Call after call without a graph the first two take 351 and 322; why was not looked into.
#include "host_common.h"
#include "tc5.cuh"

namespace vb {

constexpr int KE_THREADS = 256;

struct EvictParams {
    const float *mass;  // [n_layers][n_obs][n_kv][src_cap]
    float *mass_out;    // [n_layers][n_obs][n_kv][dst_cap] or nullptr
    const int32_t *lens;
    int32_t *kept, *lens_out;  // [n_layers][n_obs][n_kv][keep], [n_obs] or nullptr
    const uint4 *k, *v;
    uint4 *k_out, *v_out;
    int n_obs, n_kv, src_cap, dst_cap, max_len, keep, sink, recent;
    long long n_pages;
    int row_chunks;  // 16-byte pieces of a row
};

__device__ __forceinline__ int ev_len(const EvictParams &p, int obs) {
    return p.lens ? min(max(p.lens[obs], 0), p.max_len) : p.max_len;
}

// larger key = kept earlier: 0 for a weight that is no number, 0xffffffff for a protected row
__device__ __forceinline__ uint32_t ev_key(const EvictParams &p, float mass, int row, int len) {
    if (row < p.sink || row >= len - p.recent) return 0xffffffffu;
    const float m = mass + 0.0f;  // -0 and 0 are the same weight
    if (m != m) return 0u;
    const uint32_t b = __float_as_uint(m);
    return b & 0x80000000u ? ~b : b | 0x80000000u;  // in [2^23 - 1, 2^32 - 2^23]
}

// Rows [t0, n) of a page, every `stride`-th round of KE_THREADS / row_chunks rows, by the whole block; four rows of K and of V per thread in
// flight.
__device__ __forceinline__ void ev_move(const EvictParams &p, long long page, const int32_t *rows, int n, int slice, int slices) {
    constexpr int U = 4;
    const int per = KE_THREADS / p.row_chunks, step = slices * per, col = threadIdx.x % p.row_chunks;
    const long long from = page * p.src_cap * p.row_chunks + col, to = page * p.dst_cap * p.row_chunks + col;
    for (int t = slice * per + threadIdx.x / p.row_chunks; t < n; t += U * step) {
        int row[U];
        uint4 a[U], b[U];
#pragma unroll
        for (int i = 0; i < U; ++i) row[i] = t + i * step < n ? rows[t + i * step] : -1;
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (row[i] >= 0) {
                const long long src = from + (long long)row[i] * p.row_chunks;
                a[i] = p.k[src];
                b[i] = p.v[src];
            }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (row[i] >= 0) {
                const long long dst = to + (long long)(t + i * step) * p.row_chunks;
                p.k_out[dst] = a[i];
                p.v_out[dst] = b[i];
            }
    }
}

// KPL keys per lane: pages of up to 32 KPL rows.  Block (page, slice): its first warp selects, all of it moves its slice of the rows; what
// other blocks move covers the selection.
template <int KPL>
__global__ void __launch_bounds__(KE_THREADS) kv_evict_page_kernel(const EvictParams p) {
    __shared__ int32_t s_rows[32 * KPL];
    pdl_launch_dependents();
    pdl_wait();
    const long long page = blockIdx.x;
    const int obs = (int)((unsigned)page / (unsigned)p.n_kv % (unsigned)p.n_obs);
    const int len = ev_len(p, obs), n = min(len, p.keep);
    const float *mass = p.mass + page * p.src_cap;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        uint32_t key[KPL];
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const int r = i * 32 + lane;
            key[i] = r < len ? __float_as_uint(mass[r]) : 0u;
        }
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const int r = i * 32 + lane;
            key[i] = r < len ? ev_key(p, __uint_as_float(key[i]), r, len) : 0u;
        }
        // the largest threshold that at least n keys reach; n keys that reach it exactly will do
        uint32_t limit = 0;
        int left = n;  // rows at the threshold that are kept: the first ones
        if (len > n && n > 0) {
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t cand = limit | 1u << bit;
                int part[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < KPL; ++i) part[i & 3] += key[i] >= cand ? 1 : 0;
                const int c = __reduce_add_sync(0xffffffffu, (part[0] + part[1]) + (part[2] + part[3]));
                if (c >= n) limit = cand;
                if (c == n) break;
            }
            int above = 0;
#pragma unroll
            for (int i = 0; i < KPL; ++i) above += key[i] > limit ? 1 : 0;
            left = n - __reduce_add_sync(0xffffffffu, above);
        }
        const unsigned before = (1u << lane) - 1u;
        int done = 0, equals = 0;
#pragma unroll
        for (int i = 0; i < KPL; ++i) {
            const int r = i * 32 + lane;
            const bool above = r < len && (len <= n || key[i] > limit), equal = r < len && len > n && key[i] == limit;
            const unsigned eq = __ballot_sync(0xffffffffu, equal);
            const bool take = above || (equal && equals + __popc(eq & before) < left);
            const unsigned tk = __ballot_sync(0xffffffffu, take);
            if (take) s_rows[done + __popc(tk & before)] = r;
            done += __popc(tk);
            equals += __popc(eq);
        }
    }
    __syncthreads();
    if (blockIdx.y == 0) {
        if (p.lens_out && page < (long long)p.n_obs * p.n_kv && page % p.n_kv == 0 && threadIdx.x == 0) p.lens_out[obs] = n;
        for (int i = threadIdx.x; i < p.keep; i += KE_THREADS) p.kept[page * p.keep + i] = i < n ? s_rows[i] : -1;
        if (p.mass_out)
            for (int i = threadIdx.x; i < p.dst_cap; i += KE_THREADS) p.mass_out[page * p.dst_cap + i] = i < n ? mass[s_rows[i]] : 0.0f;
    }
    ev_move(p, page, s_rows, n, blockIdx.y, gridDim.y);
}

__global__ void __launch_bounds__(KE_THREADS) kv_evict_select_kernel(const EvictParams p) {
    __shared__ int hist[256];
    __shared__ int s_bin, s_left;
    __shared__ int s_warp[2][KE_THREADS / 32];
    pdl_launch_dependents();
    pdl_wait();
    const long long page = blockIdx.x;
    const int obs = (int)((unsigned)page / (unsigned)p.n_kv % (unsigned)p.n_obs);
    const int len = ev_len(p, obs), n = min(len, p.keep);
    const float *mass = p.mass + page * p.src_cap;
    int32_t *kept = p.kept + page * p.keep;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (p.lens_out && page < (long long)p.n_obs * p.n_kv && page % p.n_kv == 0 && tid == 0) p.lens_out[obs] = n;
    // the keep-th largest key, and how many rows of exactly that key are kept
    uint32_t prefix = 0;
    int left = n;
    if (len > n) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            hist[tid] = 0;
            __syncthreads();
            for (int r0 = 0; r0 < len; r0 += KE_THREADS) {
                const int r = r0 + tid;
                const uint32_t key = r < len ? ev_key(p, mass[r], r, len) : 0u;
                const bool in = r < len && (shift == 24 || (key ^ prefix) >> (shift + 8) == 0);
                // rows of a warp that fall into one bin are counted by one of them
                const int bin = in ? (int)(key >> shift & 255u) : 256 + lane;
                const unsigned same = __match_any_sync(0xffffffffu, bin);
                if (in && (same & ((1u << lane) - 1u)) == 0) atomicAdd(&hist[bin], __popc(same));
            }
            __syncthreads();
            if (warp == 0) {  // bins from the top: the first whose count reaches `left`
                int c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += c[i] = hist[255 - (lane * 8 + i)];
                int incl = sum;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, incl, d);
                    if (lane >= d) incl += up;
                }
                const unsigned reach = __ballot_sync(0xffffffffu, incl >= left);
                if (lane == __ffs(reach) - 1) {
                    int above = incl - sum, i = 0;
                    while (above + c[i] < left) above += c[i++];
                    s_bin = 255 - (lane * 8 + i);
                    s_left = left - above;
                }
            }
            __syncthreads();
            prefix |= (uint32_t)s_bin << shift;
            left = s_left;
            __syncthreads();
        }
    }
    // kept rows in order: those above the keep-th key, and the first `left` of its equals
    int done = 0, equals = 0;  // kept rows and rows equal to it in front of these
    for (int r0 = 0; r0 < len; r0 += KE_THREADS) {
        const int r = r0 + tid;
        bool above = false, equal = false;
        if (r < len) {
            if (len <= n) {
                above = true;
            } else {
                const uint32_t key = ev_key(p, mass[r], r, len);
                above = key > prefix;
                equal = key == prefix;
            }
        }
        const unsigned eq = __ballot_sync(0xffffffffu, equal), before = (1u << lane) - 1u;
        if (lane == 0) s_warp[0][warp] = __popc(eq);
        __syncthreads();
        int eq_before = equals, eq_all = 0;
#pragma unroll
        for (int w = 0; w < KE_THREADS / 32; ++w) {
            eq_before += w < warp ? s_warp[0][w] : 0;
            eq_all += s_warp[0][w];
        }
        const bool take = above || (equal && eq_before + __popc(eq & before) < left);
        const unsigned tk = __ballot_sync(0xffffffffu, take);
        if (lane == 0) s_warp[1][warp] = __popc(tk);
        __syncthreads();
        int at = done, all = 0;
#pragma unroll
        for (int w = 0; w < KE_THREADS / 32; ++w) {
            at += w < warp ? s_warp[1][w] : 0;
            all += s_warp[1][w];
        }
        if (take) {
            at += __popc(tk & before);
            kept[at] = r;
            if (p.mass_out) p.mass_out[page * p.dst_cap + at] = mass[r];
        }
        done += all;
        equals += eq_all;
        // s_warp[0] is written again only after every thread has passed the second barrier, s_warp[1] after the next round's first
    }
    for (int i = n + tid; i < p.keep; i += KE_THREADS) kept[i] = -1;
    if (p.mass_out)
        for (int i = n + tid; i < p.dst_cap; i += KE_THREADS) p.mass_out[page * p.dst_cap + i] = 0.0f;
}

__global__ void __launch_bounds__(KE_THREADS) kv_evict_move_kernel(const EvictParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const long long page = blockIdx.x;
    const int obs = (int)((unsigned)page / (unsigned)p.n_kv % (unsigned)p.n_obs);
    ev_move(p, page, p.kept + page * p.keep, min(ev_len(p, obs), p.keep), blockIdx.y, gridDim.y);
}

}  // namespace vb

extern "C" int32_t vlab200_kv_evict(const vlab200_kv_store *src, const vlab200_kv_store *dst, const float *mass, const int32_t *lens,
                                    int32_t max_len, int32_t keep, int32_t sink, int32_t recent, int32_t *kept, float *mass_out,
                                    int32_t *lens_out, void *stream) {
    if (!src || !dst || !src->k_pages || !src->v_pages || !dst->k_pages || !dst->v_pages || !mass || !kept) return VLAB200_ERR_ARG;
    if (src->n_layers <= 0 || src->n_obs <= 0 || src->n_kv <= 0 || src->cap <= 0 || dst->cap <= 0) return VLAB200_ERR_ARG;
    if (src->n_layers != dst->n_layers || src->n_obs != dst->n_obs || src->n_kv != dst->n_kv || src->head_dim != dst->head_dim) return VLAB200_ERR_ARG;
    if (max_len < 0 || max_len > src->cap || keep <= 0 || keep > dst->cap || sink < 0 || recent < 0 || sink > keep - recent) return VLAB200_ERR_ARG;
    const int hd = src->head_dim;
    if (hd != 64 && hd != 128 && hd != 256) return VLAB200_ERR_UNSUPPORTED;
    const uintptr_t al = reinterpret_cast<uintptr_t>(src->k_pages) | reinterpret_cast<uintptr_t>(src->v_pages) |
                         reinterpret_cast<uintptr_t>(dst->k_pages) | reinterpret_cast<uintptr_t>(dst->v_pages);
    if (al & 15) return VLAB200_ERR_ARG;
    const long long pages = vb::size_product({src->n_layers, src->n_obs, src->n_kv});
    if (pages > 0x7fffffffLL) {
        vb::set_last_error("kv_evict: more than 2^31 - 1 pages");
        return VLAB200_ERR_UNSUPPORTED;
    }
    // rows are read while others are written: nothing that is written may overlap anything that is read, or one another
    const long long src_b = vb::size_product({pages, src->cap, hd, 2}), dst_b = vb::size_product({pages, dst->cap, hd, 2});
    const vb::MemRange in[] = {{src->k_pages, src_b}, {src->v_pages, src_b}, {mass, pages * src->cap * 4}, {lens, src->n_obs * 4LL}};
    const vb::MemRange out[] = {{dst->k_pages, dst_b}, {dst->v_pages, dst_b}, {kept, pages * keep * 4}, {mass_out, pages * dst->cap * 4},
                                {lens_out, src->n_obs * 4LL}};
    if (vb::writes_overlap(out, 5, in, 4)) return VLAB200_ERR_ARG;
    vb::EvictParams p;
    p.mass = mass;
    p.mass_out = mass_out;
    p.lens = lens;
    p.kept = kept;
    p.lens_out = lens_out;
    p.k = static_cast<const uint4 *>(src->k_pages);
    p.v = static_cast<const uint4 *>(src->v_pages);
    p.k_out = static_cast<uint4 *>(dst->k_pages);
    p.v_out = static_cast<uint4 *>(dst->v_pages);
    p.n_obs = src->n_obs;
    p.n_kv = src->n_kv;
    p.src_cap = src->cap;
    p.dst_cap = dst->cap;
    p.max_len = max_len;
    p.keep = keep;
    p.sink = sink;
    p.recent = recent;
    p.n_pages = pages;
    p.row_chunks = hd / 8;
    const int n_sm = vb::sm_count();
    if (!n_sm) return vb::cuda_fail(cudaGetLastError(), "sm_count");
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    // enough blocks for four on every SM, none with less than a round of rows
    const int rounds = (keep + vb::KE_THREADS / p.row_chunks - 1) / (vb::KE_THREADS / p.row_chunks);
    long long slices = (4LL * n_sm + pages - 1) / pages;
    if (slices > rounds) slices = rounds;
    const dim3 grid((unsigned)pages, (unsigned)slices), block(vb::KE_THREADS);
    if (max_len <= 256) return vb::launch_pdl(vb::kv_evict_page_kernel<8>, grid, block, 0, cs, p);
    if (max_len <= 512) return vb::launch_pdl(vb::kv_evict_page_kernel<16>, grid, block, 0, cs, p);
    if (max_len <= 1024) return vb::launch_pdl(vb::kv_evict_page_kernel<32>, grid, block, 0, cs, p);
    if (int rc = vb::launch_pdl(vb::kv_evict_select_kernel, dim3((unsigned)pages), block, 0, cs, p)) return rc;
    return vb::launch_pdl(vb::kv_evict_move_kernel, grid, block, 0, cs, p);
}
