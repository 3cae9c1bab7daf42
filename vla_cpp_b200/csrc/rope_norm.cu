// Per-head RMSNorm of q and k, rotary positions and the append of K / V to the pages, in one pass over a projection's rows:
//
//   y = x / sqrt(mean(x^2) + eps) * w            (a head's columns; 32 bits; left out where there is no w)
//   a_i = pos * f_i                              (64 bits, whole turns taken out before it is rounded to 32)
//   (y_u, y_v) -> (y_u c - y_v s, y_v c + y_u s) with c = m cos a_i, s = m sin a_i;  half layout: u, v = i, i + r / 2;
//                                                 interleaved: u, v = 2 i, 2 i + 1;  columns from r on stay
//   one rounding to bf16; V is rounded only.
//
// The op reads and writes every element once and does some ten operations on it.  A warp takes a token and walks its heads, 16 columns
// per lane, so the products of norm weights with the token's cosines and sines stay in registers from head to head (the warp computes
// the token's r / 2 of each once and exchanges them through shared memory).  In the half layout a lane holds columns 8 j .. 8 j + 7 and
// their partners r / 2 further on, so the rotation needs no exchange.  Few tokens: a token's heads are dealt over several warps.
//
// Measured (graph replay, cold L2): 33 prefixes of 306 to 816 tokens, 8 + 2 heads of 256 in bf16, 55 us = 4.1 TB/s of the 6.45 of a copy (49 in a
// stream of calls; an elementwise kernel of torch moves as many bytes in 41).  Loads and stores alone take 47 us, arithmetic alone 40: 16 warps of 128 registers issue half
// of the time and hide neither wholly.  A table of the heads' places instead of arithmetic per step 59 -> 53; no change from rows straight to
// shared memory instead of through registers, nor from equal numbers of live tokens per warp; slower: 24 warps of 80 registers (57), two steps
// at a time (56); whole rows by bulk copies of a loader warp 51, but 64 x 51 tokens of 15 + 10 heads of 64 in float32 22 instead of 17.
#include <cuda_bf16.h>

#include <cmath>

#include "f32x2.cuh"
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
    unsigned M;                    // n_obs * S rows
    int S, n_q, n_kv, n_heads, nsq, nsk, cap, prefix_len, rot, parts;  // n_heads: heads of a row; parts: warps that share a token
    float eps, mscale;
};

enum : int { ROPE_PAIRS = 0, ROPE_HALF_LANES = 1, ROPE_HALF_ANY = 2 };

// 8 columns of a lane
template <bool F32>
struct RnChunk;
template <>
struct RnChunk<false> {
    uint4 r;
    __device__ __forceinline__ void load(const uint8_t *s) { r = *reinterpret_cast<const uint4 *>(s); }
    __device__ __forceinline__ void get(F2 (&f)[4]) {
        f[0] = f2(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u));
        f[1] = f2(__uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u));
        f[2] = f2(__uint_as_float(r.z << 16), __uint_as_float(r.z & 0xffff0000u));
        f[3] = f2(__uint_as_float(r.w << 16), __uint_as_float(r.w & 0xffff0000u));
    }
    __device__ __forceinline__ uint4 as_bf16() { return r; }
};
template <>
struct RnChunk<true> {
    float4 a, b;
    __device__ __forceinline__ void load(const uint8_t *s) {
        a = reinterpret_cast<const float4 *>(s)[0];
        b = reinterpret_cast<const float4 *>(s)[1];
    }
    __device__ __forceinline__ void get(F2 (&f)[4]) {
        f[0] = f2(a.x, a.y);
        f[1] = f2(a.z, a.w);
        f[2] = f2(b.x, b.y);
        f[3] = f2(b.z, b.w);
    }
    __device__ __forceinline__ uint4 as_bf16() {
        F2 f[4];
        get(f);
        return make_uint4(f2_bf16(f[0]), f2_bf16(f[1]), f2_bf16(f[2]), f2_bf16(f[3]));
    }
};

// A token of a warp, and what the warp has to know of it before it works on it (fetched while it works on the one before).
struct RnToken {
    long long row, pos;
    unsigned m;
    int obs, t;
    bool exists, live;
};
__device__ __forceinline__ bool rn_live(const RnToken &k, const RopeNormParams &p) {
    return k.exists && (p.n_tok == nullptr || k.t < p.n_tok[k.obs]);
}
__device__ __forceinline__ void lds_f2x4(F2 (&f)[4], const float *s) {  // 8 floats, 16-byte aligned
    const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(s), b = *reinterpret_cast<const ulonglong2 *>(s + 4);
    f[0].v = a.x;
    f[1].v = a.y;
    f[2].v = b.x;
    f[3].v = b.y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int HD, bool F32>
struct RnSmem {
    static constexpr int STAGE = 512 * (F32 ? 4 : 2);  // a step: 512 columns of 32 / (HD / 16) heads
    static constexpr int DEPTH = 4;                    // steps in flight per warp
    static constexpr int TRIG = RN_WARPS * DEPTH * STAGE, WEIGHT = TRIG + RN_WARPS * HD * 4, TURN = WEIGHT + 2 * HD * 4;
    static constexpr int STEPS = TURN + HD / 2 * 8;    // RnStep [steps of a token][heads of a step]
};
// Where the columns of a head come from and go to, but for the token: the same for all tokens, worked out once per block.
struct __align__(16) RnStep {
    __nv_bfloat16 *dst;  // of the q rows or the page at token / row 0 of observation 0
    int src;             // byte offset in a row of x; negative: no such head
    int pad;
};

template <int HD, int MODE, bool F32>
__global__ void __launch_bounds__(RN_WARPS * 32, 2) qk_norm_rope_kernel(const RopeNormParams p) {
    using L = RnSmem<HD, F32>;
    constexpr int LH = HD / 16;   // lanes per head: two chunks of 8 columns each
    constexpr int HPW = 32 / LH;  // heads per warp and step
    constexpr int ES = F32 ? 4 : 2;
    constexpr unsigned DEPTH = L::DEPTH;
    extern __shared__ __align__(16) uint8_t rn_smem[];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    uint8_t *const ring = rn_smem + warp * (int)DEPTH * L::STAGE;
    float *const s_cos = reinterpret_cast<float *>(rn_smem + L::TRIG) + warp * HD, *const s_sin = s_cos + HD / 2;
    float *const s_w = reinterpret_cast<float *>(rn_smem + L::WEIGHT);                  // [2][HD]
    long long *const s_turn = reinterpret_cast<long long *>(rn_smem + L::TURN);         // turns per position in units of 2^-64
    const int half = p.rot >> 1;
    // This lane's two chunks start at columns cu and cv.  Half layout with rot % 16 == 0: the two columns of every pair are in one lane
    // (columns from rot on: two chunks side by side); otherwise half a head apart, so that neighbouring lanes read neighbouring chunks.
    const int jl = lane % LH, lh = lane / LH;
    const bool across = MODE == ROPE_HALF_LANES && jl < (p.rot >> 4);
    const int cu = MODE != ROPE_HALF_LANES || across ? jl * 8 : jl * 16;
    const int cv = MODE != ROPE_HALF_LANES ? HD / 2 + jl * 8 : across ? half + jl * 8 : jl * 16 + 8;
    const bool turned = MODE == ROPE_HALF_LANES ? across : cu < p.rot;
    // a token's steps: those of its q heads, then of its k heads, then of its v heads, HPW heads each; this warp takes every parts-th
    const int nsq = p.nsq, nsqk = p.nsq + p.nsk, n_steps = p.nsq + 2 * p.nsk;
    const int q_head = p.S * HD, kv_head = p.cap * HD;
    RnStep *const steps = reinterpret_cast<RnStep *>(rn_smem + L::STEPS);
    for (int i = threadIdx.x; i < n_steps * HPW; i += RN_WARPS * 32) {
        const int s = i / HPW, kind = s < nsq ? 0 : s < nsqk ? 1 : 2;
        const int h = (s - (kind == 0 ? 0 : kind == 1 ? nsq : nsqk)) * HPW + i % HPW;  // among its kind
        RnStep e;
        e.src = h < (kind == 0 ? p.n_q : p.n_kv) ? (h + (kind == 0 ? 0 : kind == 1 ? p.n_q : p.n_q + p.n_kv)) * HD * ES : -1;
        e.dst = (kind == 0 ? p.q_out : kind == 1 ? p.k : p.v) + (long long)h * (kind == 0 ? q_head : kv_head);
        e.pad = 0;
        steps[i] = e;
    }
    for (int i = threadIdx.x; i < 2 * HD; i += RN_WARPS * 32) {
        const float *w = i < HD ? p.q_norm : p.k_norm;
        s_w[i] = w ? w[i < HD ? i : i - HD] : 1.0f;
    }
    if (threadIdx.x < half) {
        const double turns = p.freqs[threadIdx.x] * 0.15915494309189533577;
        s_turn[threadIdx.x] = __double2ll_rn((turns - rint(turns)) * 18446744073709551616.0);
    }
    // warps are dealt to (token, part): a warp keeps its part from token to token, n_warps is a multiple of parts wherever it has several
    const unsigned n_tok_warps = gridDim.x * RN_WARPS / (unsigned)p.parts, task = blockIdx.x * RN_WARPS + warp;
    const int part = (int)(task % (unsigned)p.parts);
    const int d_obs = (int)(n_tok_warps / (unsigned)p.S), d_t = (int)(n_tok_warps - (unsigned)d_obs * (unsigned)p.S);
    auto step_on = [&](RnToken &k) {  // to the warp's next token
        k.m += n_tok_warps;
        k.obs += d_obs;
        k.t += d_t;
        if (k.t >= p.S) {
            k.t -= p.S;
            ++k.obs;
        }
        k.exists = k.m < p.M;
    };
    auto fetch = [&](RnToken &k) {
        k.live = rn_live(k, p);
        k.row = (k.live && p.row0 ? (long long)p.row0[k.obs] : (long long)p.prefix_len) + k.t;
        k.pos = k.live && p.pos ? (long long)p.pos[k.m] : k.row;
    };
    RnToken tok;
    tok.m = task / (unsigned)p.parts;
    tok.obs = (int)(tok.m / (unsigned)p.S);
    tok.t = (int)(tok.m - (unsigned)tok.obs * (unsigned)p.S);
    tok.exists = tok.m < p.M;
    fetch(tok);
    // The loads run DEPTH steps ahead through all of the warp's live tokens, each lane's own 2 x 8 columns straight to shared memory, so that
    // no step waits for them at a token's border either.
    RnToken ld = tok;
    const int my_steps = (n_steps - part + p.parts - 1) / p.parts;
    const RnStep *const my_step0 = steps + part * HPW + lh;
    const int step_stride = p.parts * HPW;
    const long long row_bytes = p.x_stride * ES, row_jump = row_bytes * n_tok_warps;
    const uint8_t *ld_row = static_cast<const uint8_t *>(p.x) + (long long)tok.m * row_bytes + cu * ES;
    const RnStep *ld_step = my_step0;
    int ld_left = my_steps;
    const int v_off = (cv - cu) * ES;
    const uint32_t my_ring = smem_u32(ring) + (uint32_t)((lh * HD + cu) * ES);
    uint32_t issue_at = 0, use_at = 0;  // byte offsets of stages in the ring
    static_assert(((DEPTH * L::STAGE) & (DEPTH * L::STAGE - 1)) == 0, "a ring's size is a power of two");
    auto next_live = [&]() {
        do {
            step_on(ld);
            ld_row += row_jump;
            ld.live = rn_live(ld, p);
        } while (ld.exists && !ld.live);
    };
    if (ld.exists && !ld.live) next_live();
    __syncthreads();
    auto issue = [&]() {
        if (ld.exists) {
            const int src_off = ld_step->src;
            if (src_off >= 0) {
                const uint8_t *src = ld_row + src_off;
                const uint32_t dst = my_ring + issue_at;
#pragma unroll
                for (int i = 0; i < ES / 2; ++i) {
                    cp_async16(dst + 16 * i, src + 16 * i);
                    cp_async16(dst + (uint32_t)v_off + 16 * i, src + v_off + 16 * i);
                }
            }
            ld_step += step_stride;
            if (--ld_left == 0) {
                ld_left = my_steps;
                ld_step = my_step0;
                next_live();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        issue_at = (issue_at + L::STAGE) & (DEPTH * L::STAGE - 1);
    };
#pragma unroll
    for (unsigned d = 0; d < DEPTH; ++d) issue();
    RnToken nxt;
    for (; tok.exists; tok = nxt) {
        nxt = tok;
        step_on(nxt);
        fetch(nxt);
        const long long q_at = ((long long)tok.obs * p.n_q * p.S + tok.t) * HD;
        if (!tok.live) {  // a padding token: q is zero, its row of the pages stays as it is
            for (int s = part; s < nsq; s += p.parts) {
                const RnStep e = steps[s * HPW + lh];
                if (e.src < 0) break;
                *reinterpret_cast<uint4 *>(e.dst + q_at + cu) = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4 *>(e.dst + q_at + cv) = make_uint4(0, 0, 0, 0);
            }
            continue;
        }
        const bool row_ok = tok.row >= 0 && tok.row < p.cap;
        const long long kv_at = (long long)tok.obs * p.n_kv * kv_head + tok.row * HD;
        __syncwarp();
        for (int i = lane; i < half; i += 32) {
            // The angle in units of 2^-64 turns: whole turns drop out of the product, which would otherwise cost a float32 angle 0.06 of
            // a radian at position 10^6.  What is left lies within half a turn, where the fast sine and cosine are off by 2^-21 at
            // most: 2^-13 of the rounding to bf16 that follows.
            const unsigned long long a = (unsigned long long)tok.pos * (unsigned long long)s_turn[i];
            const float rad = (float)(int)(a >> 32) * 1.4629180792671596e-9f;  // 2 pi 2^-32
            s_cos[i] = __cosf(rad) * p.mscale;
            s_sin[i] = __sinf(rad) * p.mscale;
        }
        __syncwarp();
        // half layout:  out_u = scale (y_u au - y_v bv),  out_v = scale (y_v av + y_u bu): norm weights times cosine (a) and sine (b)
        // interleaved:  the same within a chunk, with the pair's two products side by side
        F2 au[4], av[4], bu[4], bv[4];
        int kind = -1;  // whose norm weights they hold: 0 q, 1 k
        const RnStep *at_step = my_step0;
        for (int s = part; s < n_steps; s += p.parts, at_step += step_stride) {
            {
                const RnStep to = *at_step;
                const uint8_t *const stage = ring + use_at + lh * HD * ES;
                use_at = (use_at + L::STAGE) & (DEPTH * L::STAGE - 1);
                asm volatile("cp.async.wait_group %0;" ::"n"((int)DEPTH - 1) : "memory");
                if (MODE == ROPE_HALF_ANY) __syncwarp();
                RnChunk<F32> xu, xv;
                xu.load(stage + cu * ES);
                xv.load(stage + cv * ES);
                F2 zu[4], zv[4];  // ROPE_HALF_ANY: partners in the middle of other lanes' chunks
                if (MODE == ROPE_HALF_ANY) {
                    auto z_of = [&](int c) {
                        if (c >= p.rot) return 0.0f;
                        const int at = c < half ? c + half : c - half;
                        return F32 ? reinterpret_cast<const float *>(stage)[at]
                                   : __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(stage)[at]);
                    };
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        zu[e] = f2(z_of(cu + 2 * e), z_of(cu + 2 * e + 1));
                        zv[e] = f2(z_of(cv + 2 * e), z_of(cv + 2 * e + 1));
                    }
                    __syncwarp();
                }
                issue();
                const int now = s < nsq ? 0 : s < nsqk ? 1 : 2;
                uint4 du, dv;
                if (now == 2) {
                    du = xu.as_bf16();
                    dv = xv.as_bf16();
                } else {
                    if (kind != now) {
                        kind = now;
                        const float *w = s_w + kind * HD, *ct = s_cos, *st = s_sin;
                        if (MODE == ROPE_HALF_LANES) {
                            lds_f2x4(au, w + cu);
                            lds_f2x4(av, w + cv);
                            if (across) {
                                F2 c[4], sn[4];
                                lds_f2x4(c, ct + cu);
                                lds_f2x4(sn, st + cu);
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    bu[e] = f2_mul(au[e], sn[e]);
                                    bv[e] = f2_mul(f2_mul(av[e], sn[e]), f2(-1.0f, -1.0f));
                                    au[e] = f2_mul(au[e], c[e]);
                                    av[e] = f2_mul(av[e], c[e]);
                                }
                            }
                        } else if (MODE == ROPE_PAIRS) {
                            lds_f2x4(au, w + cu);
                            lds_f2x4(av, w + cv);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int iu = (cu >> 1) + e, iv = (cv >> 1) + e;
                                const float cc = iu < half ? ct[iu] : 1.0f, ss = iu < half ? st[iu] : 0.0f;
                                const float dc = iv < half ? ct[iv] : 1.0f, ds = iv < half ? st[iv] : 0.0f;
                                float lo, hi;
                                f2_get(au[e], lo, hi);
                                bu[e] = f2(-(hi * ss), lo * ss);
                                f2_get(av[e], lo, hi);
                                bv[e] = f2(-(hi * ds), lo * ds);
                                au[e] = f2_mul(au[e], f2(cc, cc));
                                av[e] = f2_mul(av[e], f2(dc, dc));
                            }
                        } else {
                            auto a_of = [&](int x) { return x < p.rot ? w[x] * ct[x < half ? x : x - half] : w[x]; };
                            auto b_of = [&](int x) { return x >= p.rot ? 0.0f : x < half ? -(w[x + half] * st[x]) : w[x - half] * st[x - half]; };
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int c = 2 * e;
                                au[e] = f2(a_of(cu + c), a_of(cu + c + 1));
                                av[e] = f2(a_of(cv + c), a_of(cv + c + 1));
                                bu[e] = f2(b_of(cu + c), b_of(cu + c + 1));
                                bv[e] = f2(b_of(cv + c), b_of(cv + c + 1));
                            }
                        }
                    }
                    F2 yu[4], yv[4], ou[4], ov[4];
                    xu.get(yu);
                    xv.get(yv);
                    F2 s2 = f2_mul(yu[0], yu[0]), s3 = f2_mul(yv[0], yv[0]);
#pragma unroll
                    for (int e = 1; e < 4; ++e) {
                        s2 = f2_fma(yu[e], yu[e], s2);
                        s3 = f2_fma(yv[e], yv[e], s3);
                    }
                    float sa, sb, sc, sd;
                    f2_get(s2, sa, sb);
                    f2_get(s3, sc, sd);
                    float ss = (sa + sb) + (sc + sd);
#pragma unroll
                    for (int off = LH / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ou[e] = f2_mul(yu[e], au[e]);
                        ov[e] = f2_mul(yv[e], av[e]);
                    }
                    if (MODE == ROPE_HALF_LANES) {
                        if (turned) {  // columns that are not rotated stay clear of the others' infinities
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                ou[e] = f2_fma(yv[e], bv[e], ou[e]);
                                ov[e] = f2_fma(yu[e], bu[e], ov[e]);
                            }
                        }
                    } else if (MODE == ROPE_PAIRS) {
                        if (turned) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float lo, hi;
                                f2_get(yu[e], lo, hi);
                                if (cu + 2 * e < p.rot) ou[e] = f2_fma(f2(hi, lo), bu[e], ou[e]);
                                f2_get(yv[e], lo, hi);
                                if (cv + 2 * e < p.rot) ov[e] = f2_fma(f2(hi, lo), bv[e], ov[e]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ou[e] = f2_fma(zu[e], bu[e], ou[e]);
                            ov[e] = f2_fma(zv[e], bv[e], ov[e]);
                        }
                    }
                    const bool normed = (now == 0 ? p.q_norm : p.k_norm) != nullptr;
                    const float inv = normed ? rsqrtf(ss * (1.0f / HD) + p.eps) : 1.0f;
                    const F2 inv2 = f2(inv, inv);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        ou[e] = f2_mul(ou[e], inv2);
                        ov[e] = f2_mul(ov[e], inv2);
                    }
                    du = make_uint4(f2_bf16(ou[0]), f2_bf16(ou[1]), f2_bf16(ou[2]), f2_bf16(ou[3]));
                    dv = make_uint4(f2_bf16(ov[0]), f2_bf16(ov[1]), f2_bf16(ov[2]), f2_bf16(ov[3]));
                }
                if (to.src >= 0 && (now == 0 || row_ok)) {
                    __nv_bfloat16 *dst = to.dst + (now == 0 ? q_at : kv_at);
                    *reinterpret_cast<uint4 *>(dst + cu) = du;
                    *reinterpret_cast<uint4 *>(dst + cv) = dv;
                }
            }
        }
    }
}

template <int HD, int MODE, bool F32>
static int launch_rope_norm(RopeNormParams &p, cudaStream_t stream) {
    constexpr int HPW = 32 / (HD / 16);
    p.nsq = (p.n_q + HPW - 1) / HPW;
    p.nsk = p.n_heads > p.n_q ? (p.n_kv + HPW - 1) / HPW : 0;
    const int n_steps = p.nsq + 2 * p.nsk, smem = RnSmem<HD, F32>::STEPS + n_steps * HPW * (int)sizeof(RnStep);
    if (int rc = ensure_dyn_smem(qk_norm_rope_kernel<HD, MODE, F32>, smem)) return rc;
    // Persistent: two blocks on every SM.  A warp takes whole tokens once every warp has four of them; fewer tokens: their heads over
    // 2, 4 or 8 warps (a power of two divides the number of warps), and over as many as there are steps where one round does it.
    const unsigned max_blocks = 2u * (unsigned)sm_count(), n_warps = max_blocks * RN_WARPS;
    unsigned parts = 1;
    while (parts < 8 && (long long)parts * p.M < 4LL * n_warps && (int)parts * 2 <= n_steps) parts *= 2;
    if ((long long)p.M * n_steps <= (long long)n_warps) parts = (unsigned)n_steps;
    p.parts = (int)parts;
    unsigned blocks = (unsigned)(((long long)p.M * parts + RN_WARPS - 1) / RN_WARPS < max_blocks ? ((long long)p.M * parts + RN_WARPS - 1) / RN_WARPS : max_blocks);
    return launch_pdl(qk_norm_rope_kernel<HD, MODE, F32>, dim3(blocks), dim3(RN_WARPS * 32), smem, stream, p);
}

template <int HD, bool F32>
static int dispatch_rope_norm(RopeNormParams &p, int interleaved, cudaStream_t stream) {
    if (interleaved) return launch_rope_norm<HD, ROPE_PAIRS, F32>(p, stream);
    // Chunks of 8 columns and the chunks of their partners, in one lane; at other widths the partners lie in the middle of other lanes' chunks and
    // are read one by one.  33 x 816 tokens, 8 + 2 heads of 256, bf16, 276 MB (graph replay, cold L2): 256 columns rotated 55 us, 250 133, 100 96;
    // 64 x 51 tokens, 15 + 10 heads of 64, float32: 32 columns 18.4, 20 24.6.
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
    const long long heads = a->n_q + (a->with_kv ? 2LL * st->n_kv : 0), rows = (long long)st->n_obs * a->S;
    const int es = a->x_is_f32 ? 4 : 2;
    if (a->x_stride < heads * hd || a->x_stride % (16 / es)) return VLAB200_ERR_ARG;
    const uintptr_t al = reinterpret_cast<uintptr_t>(a->x) | reinterpret_cast<uintptr_t>(a->q_out) |
                         (a->with_kv ? reinterpret_cast<uintptr_t>(st->k_pages) | reinterpret_cast<uintptr_t>(st->v_pages) : 0);
    if (al & 15) return VLAB200_ERR_ARG;
    vb::RopeNormParams p;
    if (rows == 0) return VLAB200_OK;
    if (rows > 0x7fffffffLL || (long long)a->S * hd > 0x7fffffffLL || heads > 2048 || (long long)st->cap * hd > 0x7fffffffLL ||
        (a->with_kv && vb::size_product({st->n_layers, st->n_obs, st->n_kv}) > 0x7fffffffLL) ||
        vb::size_product({rows, a->x_stride, es}) == LLONG_MAX) {
        vb::set_last_error("qk_norm_rope_append: more than 2^31 - 1 rows, pages or elements of a page, 2,048 heads of a row, or 2^63 bytes of x");
        return VLAB200_ERR_UNSUPPORTED;
    }
    const int n_heads = (int)heads;
    const long long pages_b = a->with_kv ? vb::size_product({st->n_layers, st->n_obs, st->n_kv, st->cap, hd, 2}) : 0;
    const vb::MemRange out[] = {{a->q_out, rows * a->n_q * hd * 2}, {st->k_pages, pages_b}, {st->v_pages, pages_b}};
    const vb::MemRange in[] = {{a->x, ((rows - 1) * a->x_stride + n_heads * hd) * es}, {a->q_norm, hd * 4}, {a->k_norm, hd * 4},
                               {a->freqs, a->rot_dim * 4LL}, {a->pos, rows * 4}, {a->row0, st->n_obs * 4LL}, {a->n_tok, st->n_obs * 4LL}};
    if (vb::writes_overlap(out, 3, in, 7)) return VLAB200_ERR_ARG;
    p.M = (unsigned)rows;
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
