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
    int32_t R, D;
    uint32_t x_s, r_s, a_s, y_s, z_s;  // bytes from row to row
    int32_t group;                     // columns that share a scale
    int32_t w_f32;
    float eps, inv_d;
};

struct NormBackwardParams {
    const void *z, *w, *gate, *dy, *dz;  // gate, dz: may be nullptr
    void *dx, *dgate;                    // may be nullptr
    float* dw;                           // partial sums [gridDim.x, D]; nullptr: not wanted
    int32_t R, D;
    uint32_t z_s, a_s, dy_s, dz_s, dx_s, da_s;  // bytes from row to row
    int32_t w_f32;
    float eps, inv_d;
};

// Column c of row `row`; rows are `stride` bytes apart (one multiply-add).
template <typename T>
__device__ __forceinline__ T* norm_at(const void* base, uint32_t row, uint32_t stride, int c)
{
    return reinterpret_cast<T*>(reinterpret_cast<uint64_t>(base) + static_cast<uint64_t>(row) * stride) + c;
}

// weight[c .. c + V) as fp32
template <typename T, int V>
__device__ __forceinline__ void norm_weight(const void* w, int32_t w_f32, int c, float* out)
{
    if (w_f32) {
        constexpr int F = V < 4 ? V : 4;
#pragma unroll
        for (int i = 0; i < V; i += F) {
            const auto pk = load_pack<float, F, true>(static_cast<const float*>(w) + c + i);
#pragma unroll
            for (int k = 0; k < F; ++k) out[i + k] = pk.e[k];
        }
    } else {
        const auto pk = load_pack<T, V, true>(static_cast<const T*>(w) + c);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = to_f32(pk.e[i]);
    }
}

// 1 / (1 + e^-x): 0 and 1 in the limits, by the hardware's exponential and
// reciprocal (within 2 and 1 ulp; a result below 2^-126 is 0)
__device__ __forceinline__ float sigmoid_fast(float x)
{
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
}

__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr int norm_threads(int lpr) { return lpr <= 32 ? 256 : lpr; }
constexpr int norm_rows(int lpr) { return lpr <= 32 ? 256 / lpr : 1; }
// Blocks an SM that the registers are held to: 1536 threads forwards (1024 with
// two pieces a lane), 512 to 1024 backwards.
constexpr int norm_forward_blocks(int lpr, int nv)
{
    return nv == 1 ? 1536 / norm_threads(lpr) : nv == 2 ? 1024 / norm_threads(lpr) : 1;
}
constexpr int norm_backward_blocks(int lpr) { return lpr <= 128 ? 4 : lpr <= 256 ? 3 : lpr <= 512 ? 2 : 1; }

// Sums of N values (or NaN-keeping maxima) over the LPR lanes of a row:
// shuffles inside a warp, then `shared` where a row spans the block.  Two
// reductions that follow one another use different parts of it.
template <int LPR, bool MAX, int N>
__device__ __forceinline__ void row_reduce(float (&v)[N], float (*shared)[32])
{
#pragma unroll
    for (int m = (LPR < 32 ? LPR : 32) / 2; m > 0; m >>= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float o = __shfl_xor_sync(~0u, v[k], m);
            v[k] = MAX ? max_nan(v[k], o) : v[k] + o;
        }
    if constexpr (LPR > 32) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (threadIdx.x % 32 == 0) shared[k][threadIdx.x / 32] = v[k];
        __syncthreads();
        // every warp joins the warps' values by shuffles (reading all of them
        // would be the longer half of a lane's instructions)
        constexpr int W = LPR / 32;
        const int lane = threadIdx.x % 32;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = shared[k][lane % W];
#pragma unroll
            for (int m = W / 2; m > 0; m >>= 1) {
                const float o = __shfl_xor_sync(~0u, v[k], m);
                v[k] = MAX ? max_nan(v[k], o) : v[k] + o;
            }
        }
    }
}

// scale of a group whose largest |y| is `amax`; the clamp keeps a NaN
__device__ __forceinline__ float norm_scale(float amax) { return (amax < 1e-12f ? 1e-12f : amax) * (1.0f / 448.0f); }

// 1 / scale, within 1 ulp
__device__ __forceinline__ float norm_inverse(float scale)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
    return r;
}

// V values of a row as e4m3, to the nearest, saturating.
template <int V>
__device__ __forceinline__ void norm_store_fp8(uint8_t* to, const float* v)
{
    alignas(8) uint8_t q[V];
    if constexpr (V == 1) {
        q[0] = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
        *to = q[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2)
            *reinterpret_cast<__nv_fp8x2_storage_t*>(q + i) =
                __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE, __NV_E4M3);
        using Raw = typename RawOf<V>::type;
        *reinterpret_cast<Raw*>(to) = *reinterpret_cast<const Raw*>(q);
    }
}

// LPR lanes share a row and hold it in registers, NV pieces of V columns each
// (16 bytes; one column where rows are not made of 16-byte pieces), so every
// input is read once and every output written once: the kernel is bound by
// DRAM.  Piece j of lane l holds columns (j LPR + l) V .. + V.  z is kept as it
// is stored, in its own type, and the weight is read after the row's sum (from
// L1), so that few registers leave many rows in flight: 183 us on 32768 x 4096
// bf16 with a residual (5.9 TB/s), 144 us on 1048576 x 128 gated (5.6), 152 us
// of it in e4m3 (4.4, bound by instructions).  Blocks that walk over the rows
// with the weight in registers and the next row prefetched were slower when
// they were tried (244 against 226 us on 32768 x 4096), and so were two or four
// rows a lane (204 and 264 against 165 us on 1048576 x 128) and twice the
// pieces in half the lanes (163 against 144 us there).
template <typename TX, int V, int LPR, int NV, bool FP8>
__global__ void __launch_bounds__(norm_threads(LPR), norm_forward_blocks(LPR, NV)) norm_forward_kernel(const NormParams p)
{
    constexpr int G = norm_rows(LPR);
    __shared__ float shared[2][1][32];
    // with one column a lane a group spans warps: its maximum, as the ordered
    // bits of a value that is not negative
    constexpr int kGroups = FP8 && V == 1 ? (LPR * NV + 31) / 32 : 1;
    __shared__ unsigned group_max[G][kGroups];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const int row = static_cast<int>(blockIdx.x * G + sub);
    const bool whole = p.group == p.D;  // one scale a row
    const int D = p.D;
    Pack<TX, V> x[NV], r[NV], gate[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
        if (row < p.R && c < D) {
            x[j] = load_pack<TX, V, true>(norm_at<const TX>(p.x, row, p.x_s, c));
            if (p.residual) r[j] = load_pack<TX, V, true>(norm_at<const TX>(p.residual, row, p.r_s, c));
            if (p.gate) gate[j] = load_pack<TX, V, true>(norm_at<const TX>(p.gate, row, p.a_s, c));
        }
    }
    float sum[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
        if (row >= p.R || c >= D) continue;
        if (p.residual) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = to_f32(x[j].e[i]) + to_f32(r[j].e[i]);
            x[j] = to_pack<TX, V>(f);
            *reinterpret_cast<Pack<TX, V>*>(norm_at<TX>(p.z, row, p.z_s, c)) = x[j];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sum[0] = fmaf(to_f32(x[j].e[i]), to_f32(x[j].e[i]), sum[0]);
    }
    if constexpr (FP8 && V == 1) {
        for (int i = threadIdx.x; i < G * kGroups; i += blockDim.x) (&group_max[0][0])[i] = 0;
        __syncthreads();
    }
    row_reduce<LPR, false>(sum, shared[0]);

    const float inv_rms = rsqrtf(fmaf(sum[0], p.inv_d, p.eps));

    float y[FP8 ? NV : 1][V], amax[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
        const bool in = row < p.R && c < D;
        float* const v = y[FP8 ? j : 0];
        if (in) {
            norm_weight<TX, V>(p.w, p.w_f32, c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] *= to_f32(x[j].e[i]) * inv_rms;
            if (p.gate) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float a = to_f32(gate[j].e[i]);
                    v[i] *= a * sigmoid_fast(a);
                }
            }
            if constexpr (!FP8) store_pack<TX, V, true>(norm_at<TX>(p.y, row, p.y_s, c), v);
        }
        if constexpr (FP8) {
            float most = 0.0f;
            if (in) {
#pragma unroll
                for (int i = 0; i < V; ++i) most = max_nan(most, fabsf(v[i]));
            }
            if (whole) {
                amax[0] = max_nan(amax[0], most);
            } else if constexpr (V == 1) {
                if (in) atomicMax(&group_max[sub][c / p.group], __float_as_uint(most));
            } else {  // a group lies in neighbouring lanes of one piece
                const int lanes = p.group / V;
                for (int m = lanes / 2; m > 0; m >>= 1) most = max_nan(most, __shfl_xor_sync(~0u, most, m));
                if (in) {
                    const float scale = norm_scale(most), inv = norm_inverse(scale);
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] *= inv;
                    norm_store_fp8<V>(norm_at<uint8_t>(p.y, row, p.y_s, c), v);
                    if (lane % lanes == 0) p.scale[static_cast<int64_t>(row) * (D / p.group) + c / p.group] = scale;
                }
            }
        }
    }
    if constexpr (FP8) {
        if (!whole && V > 1) return;
        if (whole) row_reduce<LPR, true>(amax, shared[1]);
        else __syncthreads();
        float scale = norm_scale(amax[0]);
        if (whole && lane == 0 && row < p.R) p.scale[row] = scale;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + lane) * V;
            if (row >= p.R || c >= D) continue;
            if (!whole) {
                scale = norm_scale(__uint_as_float(group_max[sub][c / p.group]));
                if (c % p.group == 0) p.scale[static_cast<int64_t>(row) * (D / p.group) + c / p.group] = scale;
            }
            const float inv = norm_inverse(scale);
#pragma unroll
            for (int i = 0; i < V; ++i) y[j][i] *= inv;
            norm_store_fp8<V>(norm_at<uint8_t>(p.y, row, p.y_s, c), y[j]);
        }
    }
}

// The same split of a row.  With u = dy w silu(gate), both sums of a row are
// taken in one reduction,
//     dx = r u - z r^3 mean(u z) + dz,   r = (mean(z^2) + eps)^(-1/2)
// so r is recomputed from z rather than kept.  Blocks walk over the rows; a
// lane's columns stay the same, so the weight and dweight's share live in
// registers: 219 us on 32768 x 4096 bf16 with a residual (4.9 TB/s), 240 us on
// 1048576 x 128 gated (5.6).  Prefetching the next row took the registers of
// half the warps (310 against 234 us on 32768 x 4096 when it was tried).  dweight leaves a block once, summed
// over its rows in a fixed order, and a second kernel adds the blocks.
template <typename TX, int V, int LPR, int NV, bool GATE>
__global__ void __launch_bounds__(norm_threads(LPR), norm_backward_blocks(LPR))
    norm_backward_kernel(const NormBackwardParams p)
{
    constexpr int G = norm_rows(LPR);
    __shared__ float shared[2][2][32];
    __shared__ float part[G][G > 1 ? LPR * NV * V : 1];
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    float w[NV][V], dw[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LPR + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) w[j][i] = dw[j][i] = 0.0f;
        if (c < p.D) norm_weight<TX, V>(p.w, p.w_f32, c, w[j]);
    }
    struct Row {
        Pack<TX, V> z[NV], dy[NV], gate[GATE ? NV : 1], dz[NV];
    };
    auto load = [&](int blk, Row& r) {
        const int row = blk * G + group;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + lane) * V;
            r.z[j] = r.dy[j] = r.gate[GATE ? j : 0] = pack_zero<TX, V>();
            if (row < p.R && c < p.D) {
                r.z[j] = load_pack<TX, V, true>(norm_at<const TX>(p.z, row, p.z_s, c));
                r.dy[j] = load_pack<TX, V, true>(norm_at<const TX>(p.dy, row, p.dy_s, c));
                if (GATE) r.gate[GATE ? j : 0] = load_pack<TX, V, true>(norm_at<const TX>(p.gate, row, p.a_s, c));
                if (p.dz) r.dz[j] = load_pack<TX, V, true>(norm_at<const TX>(p.dz, row, p.dz_s, c));
            }
        }
    };
    const int blocks = (p.R + G - 1) / G;
    int turn = 0;
    for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x, turn ^= 1) {
        const int row = blk * G + group;
        const bool in = row < p.R;
        Row now;
        load(blk, now);
        float sums[2] = {0.0f, 0.0f}, sig[GATE ? NV : 1][V];
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float f = to_f32(now.z[j].e[i]);
                float u = to_f32(now.dy[j].e[i]) * w[j][i];
                if (GATE) {
                    const float a = to_f32(now.gate[GATE ? j : 0].e[i]);
                    sig[GATE ? j : 0][i] = sigmoid_fast(a);
                    u *= a * sig[GATE ? j : 0][i];
                }
                sums[0] = fmaf(f, f, sums[0]);
                sums[1] = fmaf(u, f, sums[1]);
            }
        row_reduce<LPR, false>(sums, shared[turn]);
        const float r = rsqrtf(fmaf(sums[0], p.inv_d, p.eps));
        const float m = sums[1] * p.inv_d * r * r * r;  // in an order that does not underflow
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LPR + lane) * V;
            float dx[V], da[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float f = to_f32(now.z[j].e[i]), n = f * r;
                float d = to_f32(now.dy[j].e[i]);
                if (GATE) {
                    const float a = to_f32(now.gate[GATE ? j : 0].e[i]), s = sig[GATE ? j : 0][i], act = a * s;
                    da[i] = d * w[j][i] * n * fmaf(act, 1.0f - s, s);
                    d *= act;
                }
                dw[j][i] = fmaf(d, n, dw[j][i]);
                dx[i] = r * (d * w[j][i]) - f * m;
            }
            if (in && c < p.D) {
                if (p.dz) {
#pragma unroll
                    for (int i = 0; i < V; ++i) dx[i] += to_f32(now.dz[j].e[i]);
                }
                if (p.dx) store_pack<TX, V, true>(norm_at<TX>(p.dx, row, p.dx_s, c), dx);
                if (GATE && p.dgate) store_pack<TX, V, true>(norm_at<TX>(p.dgate, row, p.da_s, c), da);
            }
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
                const int c = (j * LPR + lane) * V + i;
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
