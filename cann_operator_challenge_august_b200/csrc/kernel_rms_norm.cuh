// Root-mean-square norm with the residual's addition or a silu gate, forwards
// (16- or 8-bit output) and backwards (include/cgdr_rms_norm.h).
#pragma once

#include <cuda_fp8.h>

#include <cstdint>

#include "vec_io.cuh"

namespace cgdr {

struct NormParams {
    const void *x, *w, *residual, *gate;  // residual, gate: may be nullptr
    void *y, *z;
    float* scale;  // 8-bit output: one per group
    int64_t R, D, x_s, r_s, a_s, y_s, z_s;
    int32_t group_lanes;  // lanes that share a scale; 0: the whole row
    int32_t w_f32, aligned;
    float eps;
};

struct NormBackwardParams {
    const void *z, *w, *gate, *dy, *dz;  // gate, dz: may be nullptr
    void *dx, *dgate;                    // may be nullptr
    float* dw;                           // partial sums [gridDim.x, D]; nullptr: not wanted
    int64_t R, D, z_s, a_s, dy_s, dz_s, dx_s, da_s;
    int32_t w_f32, aligned;
    float eps;
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> norm_load(const T* p, int32_t aligned, int valid)
{
    return aligned ? load_pack<T, V, true>(p) : load_pack<T, V, false>(p, valid);
}

template <typename T, int V>
__device__ __forceinline__ void norm_store(T* p, const float* v, int32_t aligned, int valid)
{
    if (aligned) store_pack<T, V, true>(p, v);
    else store_pack<T, V, false>(p, v, valid);
}

// weight[c .. c + V) as fp32 (the address of `w` is checked with the rows')
template <typename T, int V>
__device__ __forceinline__ void norm_weight(const void* w, int32_t w_f32, int32_t aligned, int64_t c, int valid,
                                            float* out)
{
    if (w_f32) {
        const float* const f = static_cast<const float*>(w) + c;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const auto pk = norm_load<float, 4>(f + i, aligned, valid - i);
#pragma unroll
            for (int k = 0; k < 4; ++k) out[i + k] = pk.e[k];
        }
    } else {
        const auto pk = norm_load<T, V>(static_cast<const T*>(w) + c, aligned, valid);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = to_f32(pk.e[i]);
    }
}

// 1 / (1 + e^-x): 0 and 1 in the limits, by the hardware's exponential and
// reciprocal (each within 2 ulp)
__device__ __forceinline__ float sigmoid_fast(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Sums (or NaN-keeping maxima) over the LPR lanes of a row: shuffles inside a
// warp, then shared memory where a row spans the block.  `slot` tells two
// reductions of one row apart.
template <int LPR, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float (*shared)[32], int slot)
{
#pragma unroll
    for (int m = (LPR < 32 ? LPR : 32) / 2; m > 0; m >>= 1) {
        const float o = __shfl_xor_sync(~0u, v, m);
        v = MAX ? max_nan(v, o) : v + o;
    }
    if constexpr (LPR > 32) {
        constexpr int W = LPR / 32;
        if (threadIdx.x % 32 == 0) shared[slot][threadIdx.x / 32] = v;
        __syncthreads();
        v = shared[slot][0];
#pragma unroll
        for (int i = 1; i < W; ++i) v = MAX ? max_nan(v, shared[slot][i]) : v + shared[slot][i];
    }
    return v;
}

constexpr int norm_threads(int lpr) { return lpr <= 32 ? 256 : lpr; }
constexpr int norm_rows(int lpr) { return lpr <= 32 ? 256 / lpr : 1; }

// LPR lanes share a row and hold it in registers, NV pieces of 16 bytes each,
// so every input is read once and every output written once: the kernel is
// bound by DRAM.  Piece j of lane l holds columns (j LPR + l) V .. + V.
template <typename TX, int LPR, int NV, bool FP8>
__global__ void __launch_bounds__(norm_threads(LPR)) norm_forward_kernel(const NormParams p)
{
    constexpr int V = 16 / sizeof(TX);
    __shared__ float shared[2][32];
    const int lane = threadIdx.x % LPR;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * norm_rows(LPR) + threadIdx.x / LPR;
    const bool in = row < p.R;
    float z[NV][V];
    Pack<TX, V> gate[NV];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = static_cast<int64_t>(j * LPR + lane) * V;
        const int valid = static_cast<int>(p.D - c);
        if (in && valid > 0) {
            const auto x = norm_load<TX, V>(static_cast<const TX*>(p.x) + row * p.x_s + c, p.aligned, valid);
            if (p.gate)
                gate[j] = norm_load<TX, V>(static_cast<const TX*>(p.gate) + row * p.a_s + c, p.aligned, valid);
            if (p.residual) {
                const auto r = norm_load<TX, V>(static_cast<const TX*>(p.residual) + row * p.r_s + c, p.aligned, valid);
#pragma unroll
                for (int i = 0; i < V; ++i) z[j][i] = to_f32(from_f32<TX>(to_f32(x.e[i]) + to_f32(r.e[i])));
                norm_store<TX, V>(static_cast<TX*>(p.z) + row * p.z_s + c, z[j], p.aligned, valid);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) z[j][i] = to_f32(x.e[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                z[j][i] = 0.0f;
                gate[j].e[i] = from_f32<TX>(0.0f);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) ss = fmaf(z[j][i], z[j][i], ss);
    }
    ss = row_reduce<LPR, false>(ss, shared, 0);
    const float r = rsqrtf(ss / static_cast<float>(p.D) + p.eps);
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int64_t c = static_cast<int64_t>(j * LPR + lane) * V;
        const int valid = static_cast<int>(p.D - c);
        if (in && valid > 0) {
            float w[V];
            norm_weight<TX, V>(p.w, p.w_f32, p.aligned, c, valid, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                z[j][i] *= r * w[i];
                if (p.gate) {
                    const float a = to_f32(gate[j].e[i]);
                    z[j][i] *= a * sigmoid_fast(a);
                }
                if constexpr (FP8) amax = max_nan(amax, fabsf(z[j][i]));
            }
            if constexpr (!FP8) norm_store<TX, V>(static_cast<TX*>(p.y) + row * p.y_s + c, z[j], p.aligned, valid);
        }
        if constexpr (FP8) {
            if (p.group_lanes) {  // uniform: a scale for each group of lanes of this piece
                for (int m = p.group_lanes / 2; m > 0; m >>= 1) amax = max_nan(amax, __shfl_xor_sync(~0u, amax, m));
                // the clamp keeps a NaN
                const float scale = (amax < 1e-12f ? 1e-12f : amax) * (1.0f / 448.0f);
                if (in && valid > 0) {
                    const float inv = 1.0f / scale;
#pragma unroll
                    for (int i = 0; i < V; ++i) z[j][i] *= inv;
                    if (lane % p.group_lanes == 0) p.scale[(row * p.D + c) / (p.group_lanes * V)] = scale;
                }
                amax = 0.0f;
            }
        }
    }
    if constexpr (FP8) {
        float inv = 1.0f;
        if (!p.group_lanes) {
            amax = row_reduce<LPR, true>(amax, shared, 1);
            const float scale = (amax < 1e-12f ? 1e-12f : amax) * (1.0f / 448.0f);
            inv = 1.0f / scale;
            if (in && lane == 0) p.scale[row] = scale;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = static_cast<int64_t>(j * LPR + lane) * V;
            const int valid = static_cast<int>(p.D - c);
            if (!in || valid <= 0) continue;
            uint8_t* const to = static_cast<uint8_t*>(p.y) + row * p.y_s + c;
            alignas(8) uint8_t q[V];
#pragma unroll
            for (int i = 0; i < V; i += 2)
                *reinterpret_cast<__nv_fp8x2_storage_t*>(q + i) =
                    __nv_cvt_float2_to_fp8x2(make_float2(z[j][i] * inv, z[j][i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            if (p.aligned) {
                using Raw = typename RawOf<V>::type;
                *reinterpret_cast<Raw*>(to) = *reinterpret_cast<const Raw*>(q);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i < valid) to[i] = q[i];
            }
        }
    }
}

// The same split of a row.  With u = dy w silu(gate), both sums of a row are
// taken in one reduction,
//     dx = r u - z r^3 mean(u z) + dz,   r = (mean(z^2) + eps)^(-1/2)
// so r is recomputed from z rather than kept.  Blocks walk over the rows and
// keep their share of dweight in registers; it leaves the block once, summed
// over its rows in a fixed order, and a second kernel adds the blocks.
template <typename TX, int LPR, int NV>
__global__ void __launch_bounds__(norm_threads(LPR)) norm_backward_kernel(const NormBackwardParams p)
{
    constexpr int V = 16 / sizeof(TX);
    constexpr int G = norm_rows(LPR);
    __shared__ float shared[4][32];
    __shared__ float part[G > 1 ? G : 1][G > 1 ? LPR * NV * V : 1];
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    float dw[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] = 0.0f;
    const int64_t blocks = (p.R + G - 1) / G;
    int turn = 0;
    for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x, turn ^= 2) {
        const int64_t row = blk * G + group;
        const bool in = row < p.R;
        Pack<TX, V> z[NV], dy[NV], gate[NV], dz[NV];
        float ss = 0.0f, su = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = static_cast<int64_t>(j * LPR + lane) * V;
            const int valid = static_cast<int>(p.D - c);
            if (in && valid > 0) {
                z[j] = norm_load<TX, V>(static_cast<const TX*>(p.z) + row * p.z_s + c, p.aligned, valid);
                dy[j] = norm_load<TX, V>(static_cast<const TX*>(p.dy) + row * p.dy_s + c, p.aligned, valid);
                if (p.gate)
                    gate[j] = norm_load<TX, V>(static_cast<const TX*>(p.gate) + row * p.a_s + c, p.aligned, valid);
                if (p.dz) dz[j] = norm_load<TX, V>(static_cast<const TX*>(p.dz) + row * p.dz_s + c, p.aligned, valid);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = static_cast<int64_t>(j * LPR + lane) * V;
            const int valid = static_cast<int>(p.D - c);
            if (in && valid > 0) {
                float w[V];
                norm_weight<TX, V>(p.w, p.w_f32, p.aligned, c, valid, w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float f = to_f32(z[j].e[i]);
                    float u = to_f32(dy[j].e[i]) * w[i];
                    if (p.gate) {
                        const float a = to_f32(gate[j].e[i]);
                        u *= a * sigmoid_fast(a);
                    }
                    ss = fmaf(f, f, ss);
                    su = fmaf(u, f, su);
                }
            }
        }
        ss = row_reduce<LPR, false>(ss, shared, turn);
        su = row_reduce<LPR, false>(su, shared, turn + 1);
        const float inv_d = 1.0f / static_cast<float>(p.D);
        const float r = rsqrtf(ss * inv_d + p.eps);
        const float m = r * r * (su * inv_d);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int64_t c = static_cast<int64_t>(j * LPR + lane) * V;
            const int valid = static_cast<int>(p.D - c);
            if (!in || valid <= 0) continue;
            float w[V], dx[V], da[V];
            norm_weight<TX, V>(p.w, p.w_f32, p.aligned, c, valid, w);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float f = to_f32(z[j].e[i]), n = f * r;
                float d = to_f32(dy[j].e[i]), u = d * w[i];
                if (p.gate) {
                    const float a = to_f32(gate[j].e[i]), s = sigmoid_fast(a), act = a * s;
                    da[i] = u * n * (s + act * (1.0f - s));
                    u *= act;
                    d *= act;
                }
                dw[j][i] = fmaf(d, n, dw[j][i]);
                dx[i] = r * (u - f * m);
                if (p.dz) dx[i] += to_f32(dz[j].e[i]);
            }
            if (p.dx) norm_store<TX, V>(static_cast<TX*>(p.dx) + row * p.dx_s + c, dx, p.aligned, valid);
            if (p.dgate) norm_store<TX, V>(static_cast<TX*>(p.dgate) + row * p.da_s + c, da, p.aligned, valid);
        }
    }
    if (!p.dw) return;
    float* const to = p.dw + static_cast<int64_t>(blockIdx.x) * p.D;
    if constexpr (G > 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) part[group][(j * LPR + lane) * V + i] = dw[j][i];
        __syncthreads();
        for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < G; ++k) s += part[k][c];
            to[c] = s;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int64_t c = static_cast<int64_t>(j * LPR + lane) * V + i;
                if (c < p.D) to[c] = dw[j][i];
            }
    }
}

// dweight[c] = sum over blocks of their partial sums: 32 columns a block, 32
// threads a column, joined in a fixed order.
template <typename TW>
__global__ void __launch_bounds__(1024) norm_weight_kernel(const float* part, int64_t blocks, int64_t D, TW* dw)
{
    __shared__ float sum[32][33];
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
    float s = 0.0f;
    if (c < D)
        for (int64_t i = threadIdx.y; i < blocks; i += 32) s += part[i * D + c];
    sum[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    float t = sum[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) t += __shfl_xor_sync(~0u, t, m);
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.y;
    if (threadIdx.x == 0 && at < D) dw[at] = from_f32<TW>(t);
}

}  // namespace cgdr
