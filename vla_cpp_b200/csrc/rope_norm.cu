// Per-head RMSNorm of q and k, rotary positions and the append of K / V to the pages, in one pass over a projection's rows:
//
//   y = x / sqrt(mean(x^2) + eps) * w            (a head's columns; 32 bits; left out where there is no w)
//   a_i = pos * f_i                              (64 bits, brought into half a turn before it is rounded to 32)
//   (y_u, y_v) -> (y_u c - y_v s, y_v c + y_u s) with c = m cos a_i, s = m sin a_i;  half layout: u, v = i, i + r / 2;
//                                                 interleaved: u, v = 2 i, 2 i + 1;  columns from r on stay
//   one rounding to bf16; V is rounded only.
//
// The op reads and writes every element once and does some ten operations on it: HBM bounds it.  A warp takes a token and walks its
// heads, 8 columns (16 bytes of bf16) per lane, so the token's cosines and sines stay in registers (every lane computes
// r / 64 of them, they are exchanged through shared memory once per token) and a head's partner columns come by
// shuffle.  Loads of two steps are in flight per warp.  Few tokens: a token's heads are dealt over several warps.
#include <cuda_bf16.h>

#include <cmath>

#include "host_common.h"
#include "tc5.cuh"

namespace vb {

constexpr int RN_WARPS = 8;

struct RopeNormParams {
    const void *x;
    long long x_stride;  // elements between rows
    const float *q_norm, *k_norm;
    const double *freqs;
    const int32_t *pos, *row0, *n_tok;
    __nv_bfloat16 *q_out, *k, *v;  // k, v: pages of the layer
    long long M;                   // n_obs * S rows
    int S, n_q, n_kv, n_heads, cap, prefix_len, rot, parts;  // n_heads: heads of a row; parts: warps that share a token
    float eps, mscale;
};

enum : int { ROPE_PAIRS = 0, ROPE_HALF_LANES = 1, ROPE_HALF_ANY = 2 };

// 8 columns of a lane as float32
template <bool F32>
struct RnChunk;
template <>
struct RnChunk<false> {
    uint4 r;
    __device__ __forceinline__ void load(const void *x, long long i) { r = *reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(x) + i); }
    __device__ __forceinline__ void get(float (&f)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[2 * e] = __uint_as_float(w[e] << 16);
            f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
};
template <>
struct RnChunk<true> {
    float4 a, b;
    __device__ __forceinline__ void load(const void *x, long long i) {
        const float4 *s = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i);
        a = s[0];
        b = s[1];
    }
    __device__ __forceinline__ void get(float (&f)[8]) {
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
};

template <int HD, int MODE, bool F32>
__global__ void __launch_bounds__(RN_WARPS * 32) qk_norm_rope_kernel(const RopeNormParams p) {
    constexpr int LH = HD / 8;         // lanes per head
    constexpr int HPW = 32 / LH;       // heads per warp and step
    constexpr int DEPTH = F32 ? 2 : 4; // steps whose loads are in flight
    __shared__ __align__(16) float s_cos[RN_WARPS][HD / 2], s_sin[RN_WARPS][HD / 2], s_w[2][HD];
    __shared__ float s_y[MODE == ROPE_HALF_ANY ? RN_WARPS : 1][MODE == ROPE_HALF_ANY ? 256 : 1];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long task = (long long)blockIdx.x * RN_WARPS + warp;
    const long long m = task / p.parts;
    const int part = (int)(task % p.parts);
    const int obs = (int)(m / p.S), t = (int)(m % p.S);
    const bool exists = m < p.M;
    const bool live = exists && (p.n_tok == nullptr || t < p.n_tok[obs]);
    const int jl = lane % LH, c0 = jl * 8;
    const int n_steps = (p.n_heads + HPW - 1) / HPW, hstep = p.parts * HPW;
    const int head0 = part * HPW + lane / LH;
    const long long x_row = m * p.x_stride + c0;
    RnChunk<F32> ring[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (live && head0 + d * hstep < p.n_heads) ring[d].load(p.x, x_row + (long long)(head0 + d * hstep) * HD);
    for (int i = threadIdx.x; i < 2 * HD; i += RN_WARPS * 32) {
        const float *w = i < HD ? p.q_norm : p.k_norm;
        s_w[0][i] = w ? w[i < HD ? i : i - HD] : 1.0f;
    }
    __syncthreads();
    if (!exists) return;
    if (!live) {  // a padding token: q is zero, its row of the pages stays as it is
        for (int head = head0; head < p.n_q; head += hstep)
            *reinterpret_cast<uint4 *>(p.q_out + (((long long)obs * p.n_q + head) * p.S + t) * HD + c0) = make_uint4(0, 0, 0, 0);
        return;
    }
    const long long row = (p.row0 ? (long long)p.row0[obs] : (long long)p.prefix_len) + t;
    const double pos = p.pos ? (double)p.pos[m] : (double)row;
    const int half = p.rot >> 1;
    for (int i = lane; i < half; i += 32) {
        // whole turns go before the rounding to 32 bits: a position of 10^6 would otherwise lose 0.06 of a radian
        double turns = pos * p.freqs[i] * 0.15915494309189533577;
        turns -= rint(turns);
        float sn, cs;
        sincospif(2.0f * (float)turns, &sn, &cs);
        s_cos[warp][i] = cs * p.mscale;
        s_sin[warp][i] = sn * p.mscale;
    }
    __syncwarp();
    constexpr int NCS = MODE == ROPE_PAIRS ? 4 : 8;
    float cs[NCS], sn[NCS];  // of this lane's columns: 1 and 0 where they are not rotated
    int partner = lane;      // ROPE_HALF_LANES: the lane with the other column of every pair
#pragma unroll
    for (int e = 0; e < NCS; ++e) {
        cs[e] = 1.0f;
        sn[e] = 0.0f;
        if (MODE == ROPE_PAIRS) {
            const int i = c0 / 2 + e;
            if (i < half) {
                cs[e] = s_cos[warp][i];
                sn[e] = s_sin[warp][i];
            }
        } else {
            const int c = c0 + e;
            if (c < p.rot) {
                const int i = c < half ? c : c - half;
                cs[e] = s_cos[warp][i];
                sn[e] = c < half ? -s_sin[warp][i] : s_sin[warp][i];  // y_u c - y_v s, y_v c + y_u s
            }
        }
    }
    const bool turned = c0 < p.rot;
    if (MODE == ROPE_HALF_LANES && turned) partner = c0 < half ? lane + half / 8 : lane - half / 8;
    const bool row_ok = row >= 0 && row < p.cap;
    float w[8];
    int w_of = -1;  // whose norm weights w holds: 0 q, 1 k
    int head = head0;
    for (int step = part; step < n_steps; step += p.parts * DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d, head += hstep) {
            if (step + d * p.parts >= n_steps) break;  // the same for every lane
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = 0.0f;
            if (head < p.n_heads) ring[d].get(y);
            if (head + DEPTH * hstep < p.n_heads) ring[d].load(p.x, x_row + (long long)(head + DEPTH * hstep) * HD);
            const bool is_q = head < p.n_q, is_v = head >= p.n_q + p.n_kv;
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
#pragma unroll
            for (int off = LH / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
            const bool normed = !is_v && (is_q ? p.q_norm != nullptr : p.k_norm != nullptr);
            const float inv = normed ? 1.0f / sqrtf(ss * (1.0f / HD) + p.eps) : 1.0f;
            if (!is_v && w_of != (is_q ? 0 : 1)) {
                w_of = is_q ? 0 : 1;
                *reinterpret_cast<float4 *>(w) = *reinterpret_cast<const float4 *>(&s_w[w_of][c0]);
                *reinterpret_cast<float4 *>(w + 4) = *reinterpret_cast<const float4 *>(&s_w[w_of][c0 + 4]);
            }
            float o[8];
            if (MODE == ROPE_PAIRS) {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = y[e] * inv * w[e];
                if (turned) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a = o[2 * e], b = o[2 * e + 1];
                        o[2 * e] = a * cs[e] - b * sn[e];
                        o[2 * e + 1] = b * cs[e] + a * sn[e];
                    }
                }
            } else if (MODE == ROPE_HALF_LANES) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float a = y[e] * inv * w[e];
                    const float b = __shfl_sync(0xffffffffu, a, partner);
                    o[e] = turned ? a * cs[e] + b * sn[e] : a;
                }
            } else {
                float *sy = s_y[warp] + (lane / LH) * HD;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e] = y[e] * inv * w[e];
                    sy[c0 + e] = o[e];
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int c = c0 + e;
                    if (c < p.rot) o[e] = o[e] * cs[e] + sy[c < half ? c + half : c - half] * sn[e];
                }
                __syncwarp();
            }
            uint32_t r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 h = is_v ? __floats2bfloat162_rn(y[2 * e], y[2 * e + 1]) : __floats2bfloat162_rn(o[2 * e], o[2 * e + 1]);
                r[e] = *reinterpret_cast<const uint32_t *>(&h);
            }
            __nv_bfloat16 *dst = nullptr;
            if (is_q)
                dst = p.q_out + (((long long)obs * p.n_q + head) * p.S + t) * HD + c0;
            else if (head < p.n_heads && row_ok)
                dst = (is_v ? p.v : p.k) + (((long long)obs * p.n_kv + head - p.n_q - (is_v ? p.n_kv : 0)) * p.cap + row) * HD + c0;
            if (dst) *reinterpret_cast<uint4 *>(dst) = make_uint4(r[0], r[1], r[2], r[3]);
        }
    }
}

template <int HD, int MODE, bool F32>
static int launch_rope_norm(RopeNormParams &p, cudaStream_t stream) {
    constexpr int HPW = 32 / (HD / 8);
    const int n_steps = (p.n_heads + HPW - 1) / HPW;
    // a warp per token once the tokens alone fill the machine (16 warps on every SM); fewer tokens: their heads over as many warps
    const long long fill = 16LL * sm_count();
    long long parts = p.M >= fill ? 1 : (fill + p.M - 1) / p.M;
    p.parts = (int)(parts < n_steps ? parts : n_steps);
    const long long blocks = (p.M * p.parts + RN_WARPS - 1) / RN_WARPS;
    if (blocks > 0x7fffffffLL) return VLAB200_ERR_UNSUPPORTED;
    return launch_pdl(qk_norm_rope_kernel<HD, MODE, F32>, dim3((unsigned)blocks), dim3(RN_WARPS * 32), 0, stream, p);
}

template <int HD, bool F32>
static int dispatch_rope_norm(RopeNormParams &p, int interleaved, cudaStream_t stream) {
    if (interleaved) return launch_rope_norm<HD, ROPE_PAIRS, F32>(p, stream);
    // partner columns 8 r' apart sit in the same place of another lane's 8
    if (p.rot % 16 == 0) return launch_rope_norm<HD, ROPE_HALF_LANES, F32>(p, stream);
    return launch_rope_norm<HD, ROPE_HALF_ANY, F32>(p, stream);
}

}  // namespace vb

extern "C" {

int32_t vlab200_rope_freqs(double *freqs_host, float *mscale_host, int32_t rot_dim, double base, int32_t scaling, double factor,
                           int32_t original_len) {
    if (!freqs_host || !mscale_host || rot_dim <= 0 || rot_dim % 2 || !(base > 1.0) || scaling < 0 || scaling > 3) return VLAB200_ERR_ARG;
    if (scaling != 0 && !(factor >= 1.0 && std::isfinite(factor))) return VLAB200_ERR_ARG;
    if (scaling == 3 && original_len <= 0) return VLAB200_ERR_ARG;
    const double two_pi = 6.283185307179586477;
    if (scaling == 2 && rot_dim > 2) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    double lo = 0.0, hi = 0.0;
    if (scaling == 3) {
        // the pairs that turn 32 times and once within the original length: faster ones keep their angles, slower ones are stretched
        const double per_pair = 2.0 * std::log(base);
        lo = std::fmax(std::floor(rot_dim * std::log(original_len / (32.0 * two_pi)) / per_pair), 0.0);
        hi = std::fmin(std::ceil(rot_dim * std::log(original_len / two_pi) / per_pair), rot_dim - 1.0);
    }
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double ramp = std::fmin(std::fmax((i - lo) / std::fmax(hi - lo, 1e-3), 0.0), 1.0);
            f = f / factor * ramp + f * (1.0 - ramp);
        }
        freqs_host[i] = f;
    }
    *mscale_host = scaling == 3 ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return VLAB200_OK;
}

int32_t vlab200_qk_norm_rope_append(const vlab200_kv_store *st, int32_t layer, const vlab200_qk_norm_rope_args *a, void *stream) {
    if (!st || !a || !a->x || !a->q_out || (a->rot_dim > 0 && !a->freqs)) return VLAB200_ERR_ARG;
    if (a->with_kv && (!st->k_pages || !st->v_pages)) return VLAB200_ERR_ARG;
    if (layer < 0 || layer >= st->n_layers || st->n_obs < 0 || a->S < 0 || a->n_q <= 0 || st->n_kv <= 0 || st->cap <= 0) return VLAB200_ERR_ARG;
    const int hd = st->head_dim;
    if (hd != 64 && hd != 128 && hd != 256) return VLAB200_ERR_UNSUPPORTED;
    if (a->rot_dim < 0 || a->rot_dim % 2 || a->rot_dim > hd || !(a->eps >= 0.0f)) return VLAB200_ERR_ARG;
    const int n_heads = a->n_q + (a->with_kv ? 2 * st->n_kv : 0);
    const int es = a->x_is_f32 ? 4 : 2;
    if (a->x_stride < (int64_t)n_heads * hd || a->x_stride * es % 16) return VLAB200_ERR_ARG;
    const uintptr_t al = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->q_out) |
                         (a->with_kv ? reinterpret_cast<uintptr_t>(st->k_pages) | reinterpret_cast<uintptr_t>(st->v_pages) : 0);
    if (al & 15) return VLAB200_ERR_ARG;
    vb::RopeNormParams p;
    p.M = (long long)st->n_obs * a->S;
    if (p.M == 0) return VLAB200_OK;
    const long long page0 = (long long)layer * st->n_obs * st->n_kv * st->cap * hd;
    p.x = a->x;
    p.x_stride = a->x_stride;
    p.q_norm = a->q_norm;
    p.k_norm = a->k_norm;
    p.freqs = a->freqs;
    p.pos = a->pos;
    p.row0 = a->row0;
    p.n_tok = a->n_tok;
    p.q_out = static_cast<__nv_bfloat16 *>(a->q_out);
    p.k = a->with_kv ? static_cast<__nv_bfloat16 *>(st->k_pages) + page0 : nullptr;
    p.v = a->with_kv ? static_cast<__nv_bfloat16 *>(st->v_pages) + page0 : nullptr;
    p.S = a->S;
    p.n_q = a->n_q;
    p.n_kv = st->n_kv;
    p.n_heads = n_heads;
    p.cap = st->cap;
    p.prefix_len = st->prefix_len;
    p.rot = a->rot_dim;
    p.eps = a->eps;
    p.mscale = a->mscale;
    cudaStream_t cs = static_cast<cudaStream_t>(stream);
    if (hd == 64) return a->x_is_f32 ? vb::dispatch_rope_norm<64, true>(p, a->interleaved, cs) : vb::dispatch_rope_norm<64, false>(p, a->interleaved, cs);
    if (hd == 128) return a->x_is_f32 ? vb::dispatch_rope_norm<128, true>(p, a->interleaved, cs) : vb::dispatch_rope_norm<128, false>(p, a->interleaved, cs);
    return a->x_is_f32 ? vb::dispatch_rope_norm<256, true>(p, a->interleaved, cs) : vb::dispatch_rope_norm<256, false>(p, a->interleaved, cs);
}

}  // extern "C"
