// Token-by-token recurrences on a pool of states (include/cgdr_recurrence.h).
#pragma once

#include <cstdint>

#include "vec_io.cuh"

namespace cgdr {

// A row's state in the pool: -1 for a padded row.  Every thread of the block
// calls it; `bad` is set where the index is past the pool or was named by an
// earlier row.  Rows of one call must not share a state, since their blocks
// run at the same time; the scan over the earlier rows costs one load a
// thread per 256 rows and is hidden behind the state's own loads.
struct PoolRow {
    int64_t slot;
    bool bad;
};

struct PoolIndex {
    const void* idx;  // nullptr: row b owns state b
    int32_t is64;
    int64_t slots;
    __device__ __forceinline__ int64_t at(int64_t b) const
    {
        if (!idx) return b;
        return is64 ? static_cast<const int64_t*>(idx)[b] : static_cast<const int32_t*>(idx)[b];
    }
    // whether an earlier row names `slot`, as far as this thread's share goes
    __device__ __forceinline__ bool seen_before(int64_t b, int64_t slot) const
    {
        bool seen = false;
        if (idx && slot >= 0)
            for (int64_t i = threadIdx.x; i < b; i += blockDim.x) seen |= at(i) == slot;
        return seen;
    }
};

// ---- the gated delta rule -------------------------------------------------------------

struct DeltaStepParams {
    const void *q, *k, *v, *beta;
    const float* g;         // nullptr: no gate
    const int32_t* lens;    // nullptr: one token a row
    void *state, *out;
    int32_t* status;        // nullptr: not reported
    PoolIndex pool;
    int64_t B, T, Nv, rep, Dk, Dv, v_tiles;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh, b_st, b_sh, g_st, g_sh;
    int64_t s_sn, s_sh, s_sv;
    float scale;
    int32_t beta_f32;
};

constexpr int kDeltaThreads = 256;
constexpr int kDeltaLanes = 8;                             // lanes that share one state row
constexpr int kDeltaRows = kDeltaThreads / kDeltaLanes;    // state rows of a CTA per R

// One CTA: 32 R rows of one head's state [Dv, Dk] of one sequence.  Row v of
// the state meets k and q along Dk only, so rows are independent: eight lanes
// hold a row (four neighbouring elements a lane and step, 16-byte accesses
// for fp32) in registers from the first token to the last.  With S the old
// row, S k and S q are reduced together and
//     o = scale (a S q + d (k q)),   d = beta (v - a S k)
// needs no second pass over the updated row.  All loads of the state are
// issued before the row's place in the pool is checked against the earlier
// rows.  The kernel is bound by the states' traffic (read once, written
// once); k, q and v are re-read by the CTAs of a head from L2.
template <typename TX, typename TS, int NV, int R, bool ALIGNED>
__global__ void __launch_bounds__(kDeltaThreads) delta_step_kernel(const DeltaStepParams p)
{
    __shared__ int64_t warp_sum[kDeltaThreads / 32];
    const int64_t vt = blockIdx.x % p.v_tiles;
    const int64_t h = (blockIdx.x / p.v_tiles) % p.Nv;
    const int64_t b = blockIdx.x / p.v_tiles / p.Nv;
    const int lane = threadIdx.x % kDeltaLanes;
    const int64_t v0 = vt * (kDeltaRows * R) + threadIdx.x / kDeltaLanes;

    const int64_t slot = p.pool.at(b);
    bool live = slot >= 0 && slot < p.pool.slots;
    const bool past = slot >= p.pool.slots;

    float s[R][NV * 4];
    const int64_t head = slot * p.s_sn + h * p.s_sh;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t v = v0 + r * kDeltaRows;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = (j * kDeltaLanes + lane) * 4;
            if (live && v < p.Dv && e < p.Dk) {
                const auto pk = load_pack<TS, 4, ALIGNED>(static_cast<const TS*>(p.state) + head + v * p.s_sv + e,
                                                          static_cast<int>(p.Dk) - e);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[r][j * 4 + i] = to_f32(pk.e[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[r][j * 4 + i] = 0.0f;
            }
        }
    }

    // the row's first token, and whether an earlier row owns its state
    int64_t begin = b, len = 1;
    bool cut = false;
    if (p.lens) {
        int64_t sum = 0;
        for (int64_t i = threadIdx.x; i < b; i += kDeltaThreads) {
            const int32_t n = p.lens[i];
            sum += n > 0 ? n : 0;
        }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(~0u, sum, m);
        if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = sum;
        len = p.lens[b];
        cut = len < 0;
        if (cut) len = 0;
    }
    const bool dup = __syncthreads_or(p.pool.seen_before(b, slot));
    if (p.lens) {
        begin = 0;
#pragma unroll
        for (int i = 0; i < kDeltaThreads / 32; ++i) begin += warp_sum[i];
        if (begin + len > p.T) {
            cut = true;
            begin = begin < p.T ? begin : p.T;
            len = p.T - begin;
        }
    }
    live = live && !dup;
    const int64_t end = begin + len;
    if (p.status && vt == 0 && h == 0 && threadIdx.x == 0) {
        const int bits = ((past || dup) ? 0x4 : 0) | ((cut || (p.lens && b == p.B - 1 && end != p.T)) ? 0x2 : 0);
        if (bits) atomicOr(p.status, bits);
    }

    const int64_t hk = h / p.rep;
    TX* const out = static_cast<TX*>(p.out) + h * p.o_sh;
    if (live) {
        for (int64_t t = begin; t < end; ++t) {
            const TX* const kt = static_cast<const TX*>(p.k) + t * p.k_st + hk * p.k_sh;
            const TX* const qt = static_cast<const TX*>(p.q) + t * p.q_st + hk * p.q_sh;
            float k[NV * 4], q[NV * 4], vv[R];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = (j * kDeltaLanes + lane) * 4;
                if (e < p.Dk) {
                    const int valid = static_cast<int>(p.Dk) - e;
                    const auto pk = load_pack<TX, 4, ALIGNED>(kt + e, valid);
                    const auto pq = load_pack<TX, 4, ALIGNED>(qt + e, valid);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        k[j * 4 + i] = to_f32(pk.e[i]);
                        q[j * 4 + i] = to_f32(pq.e[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) k[j * 4 + i] = q[j * 4 + i] = 0.0f;
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t v = v0 + r * kDeltaRows;
                vv[r] = v < p.Dv ? to_f32(static_cast<const TX*>(p.v)[t * p.v_st + h * p.v_sh + v]) : 0.0f;
            }
            const int64_t bi = t * p.b_st + h * p.b_sh;
            const float beta = p.beta_f32 ? static_cast<const float*>(p.beta)[bi]
                                          : to_f32(static_cast<const TX*>(p.beta)[bi]);
            const float a = p.g ? expf(p.g[t * p.g_st + h * p.g_sh]) : 1.0f;

            float kq = 0.0f, sk[R], sq[R];
#pragma unroll
            for (int i = 0; i < NV * 4; ++i) kq = fmaf(k[i], q[i], kq);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                sk[r] = sq[r] = 0.0f;
#pragma unroll
                for (int i = 0; i < NV * 4; ++i) {
                    sk[r] = fmaf(s[r][i], k[i], sk[r]);
                    sq[r] = fmaf(s[r][i], q[i], sq[r]);
                }
            }
#pragma unroll
            for (int m = kDeltaLanes / 2; m > 0; m >>= 1) {
                kq += __shfl_xor_sync(~0u, kq, m);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    sk[r] += __shfl_xor_sync(~0u, sk[r], m);
                    sq[r] += __shfl_xor_sync(~0u, sq[r], m);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t v = v0 + r * kDeltaRows;
                const float d = beta * (vv[r] - a * sk[r]);
#pragma unroll
                for (int i = 0; i < NV * 4; ++i) s[r][i] = fmaf(a, s[r][i], d * k[i]);
                if (lane == 0 && v < p.Dv) out[t * p.o_st + v] = from_f32<TX>(p.scale * fmaf(a, sq[r], d * kq));
            }
        }
        if (len > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t v = v0 + r * kDeltaRows;
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int e = (j * kDeltaLanes + lane) * 4;
                    if (v < p.Dv && e < p.Dk)
                        store_pack<TS, 4, ALIGNED>(static_cast<TS*>(p.state) + head + v * p.s_sv + e, &s[r][j * 4],
                                                   static_cast<int>(p.Dk) - e);
                }
            }
        }
    }
    // padded rows, and rows behind the last sequence
    const int64_t zero_from = live ? end : begin;
    const int64_t zero_to = b == p.B - 1 ? p.T : end;
    if (lane == 0)
        for (int64_t t = zero_from; t < zero_to; ++t)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int64_t v = v0 + r * kDeltaRows;
                if (v < p.Dv) out[t * p.o_st + v] = from_f32<TX>(0.0f);
            }
}

// ---- the diagonal recurrence --------------------------------------------------------------

struct LinearStepParams {
    const void *x, *g;
    float* state;
    void* out;
    int32_t* status;
    PoolIndex pool;
    int64_t B, D, tiles;
    int64_t x_sb, g_sb, o_sb, s_sn;
};

constexpr int kLinearStepThreads = 256;

// One thread: V channels of one row (16 bytes of fp32 state with V = 4).
// Bound by the traffic of the states and by launch latency.
template <typename TX, typename TG, int V>
__global__ void __launch_bounds__(kLinearStepThreads) linear_step_kernel(const LinearStepParams p)
{
    const int64_t b = blockIdx.x / p.tiles;
    const int64_t c = ((blockIdx.x % p.tiles) * kLinearStepThreads + threadIdx.x) * V;
    const int64_t slot = p.pool.at(b);
    const bool in_pool = slot >= 0 && slot < p.pool.slots;
    const bool mine = c < p.D;
    Pack<float, V> s;
    Pack<TX, V> x;
    Pack<TG, V> g;
    float* const at = p.state + slot * p.s_sn + c;
    if (in_pool && mine) {
        s = load_pack<float, V, true>(at);
        x = load_pack<TX, V, true>(static_cast<const TX*>(p.x) + b * p.x_sb + c);
        g = load_pack<TG, V, true>(static_cast<const TG*>(p.g) + b * p.g_sb + c);
    }
    const bool dup = __syncthreads_or(p.pool.seen_before(b, slot));
    if (p.status && blockIdx.x % p.tiles == 0 && threadIdx.x == 0 && (dup || slot >= p.pool.slots))
        atomicOr(p.status, 0x4);
    if (!mine) return;
    float h[V];
    if (in_pool && !dup) {
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = fmaf(expf(to_f32(g.e[i])), s.e[i], to_f32(x.e[i]));
        store_pack<float, V, true>(at, h);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = 0.0f;
    }
    store_pack<TX, V, true>(static_cast<TX*>(p.out) + b * p.o_sb + c, h);
}

}  // namespace cgdr
