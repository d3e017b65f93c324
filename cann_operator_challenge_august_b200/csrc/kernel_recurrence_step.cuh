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
    __device__ __forceinline__ int64_t at(unsigned b) const
    {
        if (!idx) return b;
        return is64 ? static_cast<const int64_t*>(idx)[b] : static_cast<const int32_t*>(idx)[b];
    }
    // whether an earlier row names `slot`, as far as this thread's share goes
    __device__ __forceinline__ bool seen_before(unsigned b, int64_t slot) const
    {
        bool seen = false;
        if (idx && slot >= 0)
            for (unsigned i = threadIdx.x; i < b; i += blockDim.x) seen |= at(i) == slot;
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
    int64_t T;
    uint32_t B, Nv, rep, Dk, Dv, v_tiles;
    int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, o_st, o_sh, b_st, b_sh, g_st, g_sh;
    int64_t s_sn, s_sh, s_sv;
    float scale;
    int32_t beta_f32;
};

constexpr int kDeltaThreads = 256;
constexpr int kDeltaLanes = 8;                             // lanes that share one state row
constexpr int kDeltaRows = kDeltaThreads / kDeltaLanes;    // state rows of a CTA per R

// CTAs an SM that the registers are held to, so that nothing spills: a lane keeps
// NV R pieces of four.
constexpr int kDeltaBlocks(int nv, int r) { return nv * r <= 4 ? 3 : 2; }

// What a token brings to a lane: its pieces of k and q, the rows' v, beta and g.
template <typename TX, int NV, int R>
struct DeltaToken {
    Pack<TX, 4> k[NV], q[NV];
    TX v[R];
    float beta, g;
};

// One CTA: 32 R rows of one head's state [Dv, Dk] of one sequence.  Row v of
// the state meets k and q along Dk only, so rows are independent: eight lanes
// hold a row (four neighbouring elements a lane and step, 16-byte accesses
// for fp32) in registers from the first token to the last.  With S the old
// row, S k and S q are reduced together and
//     o = scale (a S q + d (k q)),   d = beta (v - a S k)
// needs no second pass over the updated row.  The loads of the state, and of
// the token where its place is known, are issued before the row's place in the
// pool is checked against the earlier rows; indexes are 32-bit and each row has
// one pointer (64-bit divisions and products were half the instructions).  The
// kernel is bound by the states' traffic (read once, written once): 204 us for
// 256 rows of 32 heads of 128 x 128 in fp32, 5.3 TB/s, from 242 us; k, q and v
// are re-read by the CTAs of a head from L2.  What is left is the latency of a
// CTA's single pass (load, reduce, store) with two CTAs an SM; with bf16 states,
// half the bytes a lane, it bounds the kernel.
template <typename TX, typename TS, int NV, int R, bool ALIGNED>
__global__ void __launch_bounds__(kDeltaThreads, kDeltaBlocks(NV, R)) delta_step_kernel(const DeltaStepParams p)
{
    __shared__ int64_t warp_sum[kDeltaThreads / 32];
    // 32-bit indexes (the grid is below 2^31); offsets into tensors are 64-bit
    const unsigned vt = blockIdx.x % p.v_tiles, bh = blockIdx.x / p.v_tiles;
    const unsigned h = bh % p.Nv, b = bh / p.Nv;
    const int lane = threadIdx.x % kDeltaLanes;
    const int v0 = static_cast<int>(vt) * (kDeltaRows * R) + threadIdx.x / kDeltaLanes;
    const int Dk = p.Dk, Dv = p.Dv;

    const unsigned hk = h / p.rep;
    DeltaToken<TX, NV, R> token;
    auto load_token = [&](int64_t t) {
        const TX* const kt = static_cast<const TX*>(p.k) + t * p.k_st + hk * p.k_sh + lane * 4;
        const TX* const qt = static_cast<const TX*>(p.q) + t * p.q_st + hk * p.q_sh + lane * 4;
        const TX* const vt_ = static_cast<const TX*>(p.v) + t * p.v_st + h * p.v_sh + v0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = Dk - (j * kDeltaLanes + lane) * 4;
            token.k[j] = token.q[j] = pack_zero<TX, 4>();
            if (left > 0) {
                token.k[j] = load_pack<TX, 4, ALIGNED>(kt + j * kDeltaLanes * 4, left);
                token.q[j] = load_pack<TX, 4, ALIGNED>(qt + j * kDeltaLanes * 4, left);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) token.v[r] = v0 + r * kDeltaRows < Dv ? vt_[r * kDeltaRows] : from_f32<TX>(0.0f);
        const int64_t bi = t * p.b_st + h * p.b_sh;
        token.beta = p.beta_f32 ? static_cast<const float*>(p.beta)[bi] : to_f32(static_cast<const TX*>(p.beta)[bi]);
        token.g = p.g ? p.g[t * p.g_st + h * p.g_sh] : 0.0f;
    };
    if (!p.lens) load_token(b);

    const int64_t slot = p.pool.at(b);
    bool live = slot >= 0 && slot < p.pool.slots;
    const bool past = slot >= p.pool.slots;

    // this lane's elements of row v0 + 32 r: places j * 32 + lane * 4 and the next three
    TS* row[R];
#pragma unroll
    for (int r = 0; r < R; ++r)
        row[r] = static_cast<TS*>(p.state) + slot * p.s_sn + h * p.s_sh + (v0 + r * kDeltaRows) * p.s_sv + lane * 4;
    Pack<TS, 4> raw[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int left = Dk - (j * kDeltaLanes + lane) * 4;
            raw[r][j] = pack_zero<TS, 4>();
            if (live && v0 + r * kDeltaRows < Dv && left > 0)
                raw[r][j] = load_pack<TS, 4, ALIGNED>(row[r] + j * kDeltaLanes * 4, left);
        }

    // the row's first token, and whether an earlier row owns its state
    int64_t begin = b, len = 1;
    bool cut = false;
    if (p.lens) {
        int64_t sum = 0;
        for (unsigned i = threadIdx.x; i < b; i += kDeltaThreads) {
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
    const bool last = b == p.B - 1;
    if (p.status && vt == 0 && h == 0 && threadIdx.x == 0) {
        const int bits = ((past || dup) ? 0x4 : 0) | ((cut || (p.lens && last && end != p.T)) ? 0x2 : 0);
        if (bits) atomicOr(p.status, bits);
    }

    TX* out = static_cast<TX*>(p.out) + begin * p.o_st + h * p.o_sh + v0;
    if (live && len > 0) {
        float s[R][NV * 4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < NV * 4; ++i) s[r][i] = to_f32(raw[r][i / 4].e[i % 4]);
        for (int64_t t = begin; t < end; ++t) {
            if (p.lens) load_token(t);
            float k[NV * 4], q[NV * 4], vv[R];
#pragma unroll
            for (int i = 0; i < NV * 4; ++i) {
                k[i] = to_f32(token.k[i / 4].e[i % 4]);
                q[i] = to_f32(token.q[i / 4].e[i % 4]);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) vv[r] = to_f32(token.v[r]);
            const float beta = token.beta, a = p.g ? expf(token.g) : 1.0f;

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
                const float d = beta * (vv[r] - a * sk[r]);
#pragma unroll
                for (int i = 0; i < NV * 4; ++i) s[r][i] = fmaf(a, s[r][i], d * k[i]);
                if (lane == 0 && v0 + r * kDeltaRows < Dv)
                    out[r * kDeltaRows] = from_f32<TX>(p.scale * fmaf(a, sq[r], d * kq));
            }
            out += p.o_st;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int left = Dk - (j * kDeltaLanes + lane) * 4;
                if (v0 + r * kDeltaRows < Dv && left > 0)
                    store_pack<TS, 4, ALIGNED>(row[r] + j * kDeltaLanes * 4, &s[r][j * 4], left);
            }
    }
    // padded rows, and rows behind the last sequence
    const int64_t zero_from = live ? end : begin, zero_to = last ? p.T : end;
    if (lane == 0)
        for (int64_t t = zero_from; t < zero_to; ++t, out += p.o_st)
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (v0 + r * kDeltaRows < Dv) out[r * kDeltaRows] = from_f32<TX>(0.0f);
}

// ---- the diagonal recurrence --------------------------------------------------------------

struct LinearStepParams {
    const void *x, *g;
    float* state;
    void* out;
    int32_t* status;
    PoolIndex pool;
    int64_t D;
    uint32_t tiles;
    int64_t x_sb, g_sb, o_sb, s_sn;
};

constexpr int kLinearStepThreads = 256;

// One thread: V channels of one row (16 bytes of fp32 state with V = 4).  Bound
// by the states' traffic in large batches (1000 rows of 4100 channels in 16 us a
// call) and by the launch in small ones (12 us a call for 64 rows of 4096).
template <typename TX, typename TG, int V>
__global__ void __launch_bounds__(kLinearStepThreads) linear_step_kernel(const LinearStepParams p)
{
    const unsigned b = blockIdx.x / p.tiles;
    const int64_t c = (static_cast<int64_t>(blockIdx.x % p.tiles) * kLinearStepThreads + threadIdx.x) * V;
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
