// Work units of a call whose observations differ in length: observation b has units_of(b) = blocks(len[b]) * n_kv of them, none if it is
// empty.  A persistent grid that took every n-th unit of a rectangle (longest length x observations) left some CTAs half the work of
// others; here unit k is the k-th that exists.  A whole warp walks the list together: 32 observations' unit counts are scanned with
// shuffles, and k only grows, so a block of 32 is loaded once.
#pragma once
#include <cstdint>

namespace vb {

struct RaggedUnit {
    int obs, kvh, block;  // block: of the unit's observation and kv head, counted from 0
    int len;              // rows of the observation
};

template <typename LenOf>
struct RaggedCursor {
    LenOf len_of;  // rows of an observation
    int n_obs, n_kv, per_block;
    int obs0, base;      // first observation of the loaded 32, units in front of it
    int len, nblk, cnt, incl;  // of this lane's observation: rows, blocks, units, units up to and with it
    int total;           // units of the loaded 32

    __device__ __forceinline__ RaggedCursor(LenOf f, int n_obs_, int n_kv_, int per_block_, bool used = true)
        : len_of(f), n_obs(n_obs_), n_kv(n_kv_), per_block(per_block_) {
        obs0 = base = len = nblk = cnt = incl = total = 0;
        if (used) load();
    }
    __device__ __forceinline__ void load() {
        const int lane = threadIdx.x & 31;
        len = obs0 + lane < n_obs ? len_of(obs0 + lane) : 0;
        nblk = (len + per_block - 1) / per_block;
        cnt = nblk * n_kv;
        incl = cnt;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += up;
        }
        total = __shfl_sync(0xffffffffu, incl, 31);
    }
    // the k-th unit; false if there are not that many.  k must not fall from call to call.
    __device__ __forceinline__ bool find(int k, RaggedUnit &u) {
        while (k - base >= total) {
            if (obs0 + 32 >= n_obs) return false;
            base += total;
            obs0 += 32;
            load();
        }
        const int l = __ffs(__ballot_sync(0xffffffffu, incl > k - base)) - 1;
        const int n = __shfl_sync(0xffffffffu, nblk, l), at = k - base - __shfl_sync(0xffffffffu, incl - cnt, l);
        u.obs = obs0 + l;
        u.len = __shfl_sync(0xffffffffu, len, l);
        // at / n by the fast reciprocal, put right: a whole division is a third of the walk's time
        u.kvh = n_kv == 1 ? 0 : (int)__fdividef((float)at, (float)n);
        u.block = at - u.kvh * n;
        while (u.block < 0) {
            --u.kvh;
            u.block += n;
        }
        while (u.block >= n) {
            ++u.kvh;
            u.block -= n;
        }
        return true;
    }
};

}  // namespace vb
