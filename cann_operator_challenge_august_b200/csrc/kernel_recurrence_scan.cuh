// The diagonal recurrence over whole sequences, forwards and backwards
// (include/cgdr_recurrence.h).
#pragma once

#include <cstdint>

#include "vec_io.cuh"

namespace cgdr {

constexpr int kScanChunk = 64;  // CGDR_RECURRENCE_CHUNK

struct ScanParams {
    const void *x, *g, *d_out;
    const float *h0, *d_ht;
    const int64_t* cu;       // nullptr: every batch row is one sequence
    void *out, *dx, *dg;
    float *ht, *d_h0, *chunk;
    int64_t B, T, D, N;
    int64_t x_sb, x_st, g_sb, g_st, o_sb, o_st, do_sb, do_st, dx_sb, dx_st, dg_sb, dg_st;
    int64_t h0_sn, ht_sn, dht_sn, dh0_sn;
};

struct ScanSeq {
    int64_t b, begin, end, tail;  // tail: rows [end, tail) belong to no sequence
};

__device__ __forceinline__ int64_t scan_bound(const ScanParams& p, int64_t n)
{
    const int64_t c = p.cu[n];
    return c < 0 ? 0 : c > p.T ? p.T : c;
}

__device__ __forceinline__ ScanSeq scan_seq(const ScanParams& p, int64_t n)
{
    ScanSeq s;
    s.b = p.cu ? 0 : n;
    s.begin = p.cu ? scan_bound(p, n) : 0;
    s.end = p.cu ? scan_bound(p, n + 1) : p.T;
    s.tail = n == p.N - 1 ? p.T : s.end;
    return s;
}

// One thread: one channel of one sequence, token by token.
template <typename TX, typename TG>
__global__ void __launch_bounds__(128) scan_forward_kernel(const ScanParams p)
{
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x, n = blockIdx.y;
    if (c >= p.D) return;
    const ScanSeq s = scan_seq(p, n);
    const TX* const x = static_cast<const TX*>(p.x) + s.b * p.x_sb + c;
    const TG* const g = static_cast<const TG*>(p.g) + s.b * p.g_sb + c;
    TX* const o = static_cast<TX*>(p.out) + s.b * p.o_sb + c;
    const int64_t nc = (p.T + kScanChunk - 1) / kScanChunk;
    float h = p.h0 ? p.h0[n * p.h0_sn + c] : 0.0f;
    for (int64_t t = s.begin; t < s.end; ++t) {
        if (p.chunk && t % kScanChunk == 0) p.chunk[(s.b * nc + t / kScanChunk) * p.D + c] = h;
        h = fmaf(expf(to_f32(g[t * p.g_st])), h, to_f32(x[t * p.x_st]));
        o[t * p.o_st] = from_f32<TX>(h);
    }
    if (p.ht) p.ht[n * p.ht_sn + c] = h;
    for (int64_t t = s.end; t < s.tail; ++t) o[t * p.o_st] = from_f32<TX>(0.0f);
}

template <typename TX, typename TG>
__global__ void __launch_bounds__(128) scan_backward_kernel(const ScanParams p)
{
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x, n = blockIdx.y;
    if (c >= p.D) return;
    const ScanSeq s = scan_seq(p, n);
    const TX* const x = static_cast<const TX*>(p.x) + s.b * p.x_sb + c;
    const TG* const g = static_cast<const TG*>(p.g) + s.b * p.g_sb + c;
    const TX* const d_out = p.d_out ? static_cast<const TX*>(p.d_out) + s.b * p.do_sb + c : nullptr;
    TX* const dx = p.dx ? static_cast<TX*>(p.dx) + s.b * p.dx_sb + c : nullptr;
    TG* const dg = p.dg ? static_cast<TG*>(p.dg) + s.b * p.dg_sb + c : nullptr;
    const int64_t nc = (p.T + kScanChunk - 1) / kScanChunk;
    for (int64_t t = s.end; t < s.tail; ++t) {
        if (dx) dx[t * p.dx_st] = from_f32<TX>(0.0f);
        if (dg) dg[t * p.dg_st] = from_f32<TG>(0.0f);
    }
    float u = p.d_ht ? p.d_ht[n * p.dht_sn + c] : 0.0f;  // exp(g_{t+1}) dh_{t+1}
    float before[kScanChunk];                            // h_{t-1}
    for (int64_t stop = s.end; stop > s.begin;) {
        const int64_t floor = (stop - 1) / kScanChunk * kScanChunk;
        const int64_t first = floor > s.begin ? floor : s.begin;
        float h = first > s.begin ? p.chunk[(s.b * nc + first / kScanChunk) * p.D + c]
                  : p.h0          ? p.h0[n * p.h0_sn + c]
                                  : 0.0f;
        for (int64_t t = first; t < stop; ++t) {
            before[t - first] = h;
            h = fmaf(expf(to_f32(g[t * p.g_st])), h, to_f32(x[t * p.x_st]));
        }
        for (int64_t t = stop - 1; t >= first; --t) {
            const float dh = u + (d_out ? to_f32(d_out[t * p.do_st]) : 0.0f);
            u = dh * expf(to_f32(g[t * p.g_st]));
            if (dx) dx[t * p.dx_st] = from_f32<TX>(dh);
            if (dg) dg[t * p.dg_st] = from_f32<TG>(u * before[t - first]);
        }
        stop = first;
    }
    if (p.d_h0) p.d_h0[n * p.dh0_sn + c] = u;
}

}  // namespace cgdr
