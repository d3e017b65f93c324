// Host side of include/cgdr_recurrence.h: argument checks and launches.  No
// device memory is allocated here.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <initializer_list>

#include "../../include/cgdr_recurrence.h"
#include "host_util.cuh"
#include "kernel_recurrence_scan.cuh"
#include "kernel_recurrence_step.cuh"

using namespace cgdr;
using namespace cgdr::host;

static_assert(kScanChunk == CGDR_RECURRENCE_CHUNK, "the saved states' spacing is part of the interface");

namespace {

bool float_type(int32_t dt) { return dt == CGDR_DT_BF16 || dt == CGDR_DT_FLOAT16 || dt == CGDR_DT_FLOAT32; }

int64_t bytes_of(int32_t dt) { return dt == CGDR_DT_FLOAT32 ? 4 : 2; }

// Whether pieces of `v` neighbouring elements of every row start on a
// multiple of their size and no row ends inside one.
bool pieces_aligned(const cgdrTensor* t, int v)
{
    if (!present(t)) return true;
    if ((reinterpret_cast<uintptr_t>(t->data) % (bytes_of(t->dtype) * v)) != 0) return false;
    if (t->shape[t->ndim - 1] % v != 0) return false;
    for (int i = 0; i < t->ndim - 1; ++i)
        if (t->shape[i] > 1 && t->strides[i] % v != 0) return false;
    return true;
}

cgdrStatus check_contiguous(const cgdrTensor* t, const char* name)
{
    int64_t want = 1;
    for (int i = t->ndim - 1; i >= 0; --i) {
        if (t->shape[i] > 1 && t->strides[i] != want) return fail(CGDR_STATUS_BAD_STRIDE, "%s must be contiguous", name);
        want *= t->shape[i];
    }
    return CGDR_STATUS_SUCCESS;
}

cgdrStatus check_pool(const cgdrTensor* state, const cgdrTensor* idx, int64_t B, PoolIndex* pool)
{
    memset(pool, 0, sizeof(*pool));
    const int64_t slots = state->shape[0];
    pool->slots = slots;
    for (int i = 0; i < state->ndim; ++i)
        if (state->shape[i] > 1 && state->strides[i] == 0)
            return fail(CGDR_STATUS_BAD_STRIDE, "state is updated in place and must not be an expanded view");
    if (!present(idx)) {
        if (B > slots)
            return fail(CGDR_STATUS_BAD_SHAPE, "%lld rows need as many states, the pool has %lld",
                        static_cast<long long>(B), static_cast<long long>(slots));
        return CGDR_STATUS_SUCCESS;
    }
    cgdrStatus st;
    if ((st = check_rank(idx, 1, "state_indices"))) return st;
    if (idx->dtype != CGDR_DT_INT32 && idx->dtype != CGDR_DT_INT64)
        return fail(CGDR_STATUS_BAD_DTYPE, "state_indices must be int32 or int64");
    if (!shape_is(idx, {B})) return fail(CGDR_STATUS_BAD_SHAPE, "state_indices must have shape [B]");
    if ((st = check_contiguous(idx, "state_indices"))) return st;
    pool->idx = idx->data;
    pool->is64 = idx->dtype == CGDR_DT_INT64;
    return CGDR_STATUS_SUCCESS;
}

cgdrStatus cuda_failed(const char* what, cudaError_t e)
{
    cudaGetLastError();
    return fail(CGDR_STATUS_CUDA_ERROR, "%s: %s", what, cudaGetErrorString(e));
}

cgdrStatus launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_failed(what, e);
    g_err[0] = '\0';
    return CGDR_STATUS_SUCCESS;
}

cgdrStatus clear_status(int32_t* status, cudaStream_t stream)
{
    if (!status) return CGDR_STATUS_SUCCESS;
    const cudaError_t e = cudaMemsetAsync(status, 0, sizeof(int32_t), stream);
    if (e != cudaSuccess) return fail(CGDR_STATUS_CUDA_ERROR, "cudaMemsetAsync: %s", cudaGetErrorString(e));
    return CGDR_STATUS_SUCCESS;
}

// ---- the gated delta rule ---------------------------------------------------------------

template <typename TX, typename TS, int NV, int R, bool ALIGNED>
void run_delta(DeltaStepParams& p, cudaStream_t stream)
{
    p.v_tiles = (p.Dv + kDeltaRows * R - 1) / (kDeltaRows * R);
    delta_step_kernel<TX, TS, NV, R, ALIGNED>
        <<<p.B * p.Nv * p.v_tiles, kDeltaThreads, 0, stream>>>(p);
}

template <typename TX, typename TS>
void dispatch_delta(DeltaStepParams& p, bool aligned, cudaStream_t stream)
{
    // Two state rows a lane group where that still gives every SM a CTA: 52
    // against 61 us for 64 rows of 32 heads of 128 x 128, 4.1 against 5.5 us for
    // 4, 3.0 against 2.8 us for one (32 heads, 64 CTAs).  Rows of more than 128
    // take a lane's registers alone: 28 against 32 us for 16 rows of 16 heads of
    // 256 x 256 with one.
    const bool wide = static_cast<int64_t>(p.B) * p.Nv * ((p.Dv + 2 * kDeltaRows - 1) / (2 * kDeltaRows)) >= 148;
    const int nv = p.Dk <= 64 ? 2 : p.Dk <= 128 ? 4 : 8;
    if (!aligned) {
        if (nv == 2) run_delta<TX, TS, 2, 1, false>(p, stream);
        else if (nv == 4) run_delta<TX, TS, 4, 1, false>(p, stream);
        else run_delta<TX, TS, 8, 1, false>(p, stream);
    } else if (nv == 8) {
        run_delta<TX, TS, 8, 1, true>(p, stream);
    } else if (wide) {
        if (nv == 2) run_delta<TX, TS, 2, 2, true>(p, stream);
        else run_delta<TX, TS, 4, 2, true>(p, stream);
    } else {
        if (nv == 2) run_delta<TX, TS, 2, 1, true>(p, stream);
        else run_delta<TX, TS, 4, 1, true>(p, stream);
    }
}

template <typename TX>
void dispatch_delta_state(DeltaStepParams& p, bool state_f32, bool aligned, cudaStream_t stream)
{
    if (state_f32) dispatch_delta<TX, float>(p, aligned, stream);
    else dispatch_delta<TX, __nv_bfloat16>(p, aligned, stream);
}

// ---- the diagonal recurrence --------------------------------------------------------------

// Calls f.template operator()<TX, TG>() for x's and g's types.
template <typename F>
void with_types(int32_t dx, int32_t dg, F&& f)
{
    if (dx == CGDR_DT_FLOAT32) f.template operator()<float, float>();
    else if (dx == CGDR_DT_BF16 && dg == CGDR_DT_BF16) f.template operator()<__nv_bfloat16, __nv_bfloat16>();
    else if (dx == CGDR_DT_BF16) f.template operator()<__nv_bfloat16, float>();
    else if (dg == CGDR_DT_FLOAT16) f.template operator()<__half, __half>();
    else f.template operator()<__half, float>();
}

cgdrStatus check_gate_types(const cgdrTensor* x, const cgdrTensor* g)
{
    if (!float_type(x->dtype)) return fail(CGDR_STATUS_BAD_DTYPE, "x must be bfloat16, float16 or float32");
    if (g->dtype != x->dtype && g->dtype != CGDR_DT_FLOAT32)
        return fail(CGDR_STATUS_BAD_DTYPE, "g must have x's type or be float32");
    return CGDR_STATUS_SUCCESS;
}

// The kernels step over 16 rows with 32-bit offsets.
cgdrStatus check_row_stride(const cgdrTensor* t, const char* name)
{
    if (t->shape[1] > 1 && t->strides[1] >= (int64_t(1) << 25))
        return fail(CGDR_STATUS_UNSUPPORTED, "%s's rows must be less than 2^25 elements apart", name);
    return CGDR_STATUS_SUCCESS;
}

// Arguments that the forward and the backward pass share.
cgdrStatus check_scan(const cgdrTensor* x, const cgdrTensor* g, const cgdrTensor* h0, const cgdrTensor* cu,
                      ScanParams* p)
{
    memset(p, 0, sizeof(*p));
    if (!present(x) || !present(g)) return fail(CGDR_STATUS_NULL_ARGUMENT, "x and g are required");
    cgdrStatus st;
    if ((st = check_rank(x, 3, "x")) || (st = check_rank(g, 3, "g"))) return st;
    if (present(h0) && (st = check_rank(h0, 2, "initial_state"))) return st;
    if (present(cu) && (st = check_rank(cu, 1, "cu_seqlens"))) return st;
    if ((st = check_gate_types(x, g))) return st;
    if (present(cu) && cu->dtype != CGDR_DT_INT64) return fail(CGDR_STATUS_BAD_DTYPE, "cu_seqlens must be int64");
    const int64_t B = x->shape[0], T = x->shape[1], D = x->shape[2];
    if (B <= 0 || T <= 0 || D <= 0) return fail(CGDR_STATUS_BAD_SHAPE, "dimensions must be positive");
    if (!shape_is(g, {B, T, D})) return fail(CGDR_STATUS_BAD_SHAPE, "g must have shape [B, T, D]");
    int64_t N = B;
    if (present(cu)) {
        if (B != 1) return fail(CGDR_STATUS_BAD_VARLEN, "variable-length input needs B == 1");
        if (cu->shape[0] < 2) return fail(CGDR_STATUS_BAD_VARLEN, "cu_seqlens needs at least two entries");
        if ((st = check_contiguous(cu, "cu_seqlens"))) return st;
        N = cu->shape[0] - 1;
        p->cu = static_cast<const int64_t*>(cu->data);
    }
    if (T >= (int64_t(1) << 30) || D >= (int64_t(1) << 30) || N >= (int64_t(1) << 16))
        return fail(CGDR_STATUS_UNSUPPORTED, "T and D must fit in 30 bits and the sequences in 16");
    if ((st = check_inner_contiguous(x, "x")) || (st = check_inner_contiguous(g, "g"))) return st;
    if ((st = check_row_stride(x, "x")) || (st = check_row_stride(g, "g"))) return st;
    p->B = B; p->T = T; p->D = D; p->N = N;
    p->x = x->data; p->x_sb = x->strides[0]; p->x_st = x->strides[1];
    p->g = g->data; p->g_sb = g->strides[0]; p->g_st = g->strides[1];
    if (present(h0)) {
        if (h0->dtype != CGDR_DT_FLOAT32) return fail(CGDR_STATUS_BAD_DTYPE, "initial_state must be float32");
        if (!shape_is(h0, {N, D})) return fail(CGDR_STATUS_BAD_SHAPE, "initial_state must have shape [N, D]");
        if ((st = check_inner_contiguous(h0, "initial_state"))) return st;
        p->h0 = static_cast<const float*>(h0->data);
        p->h0_sn = h0->strides[0];
    }
    return CGDR_STATUS_SUCCESS;
}

// An optional [B, T, D] tensor of a given type, or an optional [N, D] fp32 one.
cgdrStatus check_like(const cgdrTensor* t, int32_t dtype, const ScanParams& p, const char* name)
{
    if (!present(t)) return CGDR_STATUS_SUCCESS;
    cgdrStatus st;
    if ((st = check_rank(t, 3, name))) return st;
    if (t->dtype != dtype) return fail(CGDR_STATUS_BAD_DTYPE, "%s has the wrong type", name);
    if (!shape_is(t, {p.B, p.T, p.D})) return fail(CGDR_STATUS_BAD_SHAPE, "%s must have shape [B, T, D]", name);
    if ((st = check_inner_contiguous(t, name))) return st;
    return check_row_stride(t, name);
}

cgdrStatus check_state(const cgdrTensor* t, const ScanParams& p, const char* name)
{
    if (!present(t)) return CGDR_STATUS_SUCCESS;
    cgdrStatus st;
    if ((st = check_rank(t, 2, name))) return st;
    if (t->dtype != CGDR_DT_FLOAT32) return fail(CGDR_STATUS_BAD_DTYPE, "%s must be float32", name);
    if (!shape_is(t, {p.N, p.D})) return fail(CGDR_STATUS_BAD_SHAPE, "%s must have shape [N, D]", name);
    return check_inner_contiguous(t, name);
}

cgdrStatus check_chunks(const cgdrTensor* t, ScanParams* p)
{
    cgdrStatus st;
    if ((st = check_rank(t, 3, "chunk_states"))) return st;
    if (t->dtype != CGDR_DT_FLOAT32) return fail(CGDR_STATUS_BAD_DTYPE, "chunk_states must be float32");
    if (!shape_is(t, {p->B, (p->T + kScanChunk - 1) / kScanChunk, p->D}))
        return fail(CGDR_STATUS_BAD_SHAPE, "chunk_states must have shape [B, ceil(T/128), D]");
    if ((st = check_contiguous(t, "chunk_states"))) return st;
    p->chunk = static_cast<float*>(t->data);
    return CGDR_STATUS_SUCCESS;
}

// CTAs of a cluster, which share a slab's tokens: doubled while all CTAs still
// fit on the GPU at once (`resident` CTAs an SM) and have a tile each.
int32_t scan_cluster(const ScanParams& p, int64_t slabs, int tile, int most, int64_t resident)
{
    int32_t c = 1;
    while (c < most && c * tile < p.T && 2 * c * slabs <= 148 * resident) c *= 2;
    return c;
}

// Whether TMA can read the rows: base and strides are multiples of 16 bytes.
bool tma_rows(const cgdrTensor* t)
{
    if (!present(t)) return true;
    const int64_t v = 16 / bytes_of(t->dtype);
    if (reinterpret_cast<uintptr_t>(t->data) % 16 != 0) return false;
    for (int i = 0; i < 2; ++i)
        if (t->shape[i] > 1 && (t->strides[i] % v != 0 || t->strides[i] <= 0)) return false;
    return true;
}

cgdrStatus scan_map(const cgdrTensor* t, int V, CUtensorMap* map, const char* name)
{
    if (!present(t)) return CGDR_STATUS_SUCCESS;
    const int64_t B = t->shape[0], T = t->shape[1], D = t->shape[2], v = 16 / bytes_of(t->dtype);
    // a dimension of one element has no stride of its own; any multiple of 16 bytes serves
    const int64_t row = T > 1 ? t->strides[1] : (D + v - 1) / v * v;
    const int64_t batch = B > 1 ? t->strides[0] : T * row;
    return make_rows_map(map, t->data, static_cast<int>(bytes_of(t->dtype)), D, T, row, B, batch, 32 * V, kScanSteps, name);
}

template <typename K>
cudaError_t launch_scan(K kernel, ScanParams& p, const ScanMapsTma& maps, int V, int W, int smem, int cluster,
                        cudaStream_t stream)
{
    // 16 warps an SM by registers, fewer where shared memory does not hold them:
    // the ring, the maps of warps and CTAs, and 1 KB of the system's
    int64_t resident = 16 / W;
    const int64_t fit = 227 * 1024 / (smem + V * 512 * (W + W / 2 + cluster) + 256 + 1024);
    if (resident > fit) resident = fit;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int64_t slabs = (p.D + 32 * V - 1) / (32 * V);
    p.cluster = scan_cluster(p, slabs * p.B, W * kScanSteps, cluster, resident);
    // Neighbouring slabs keep pace where every CTA has a slab of its own and all
    // are resident at once, two an SM.  (With clusters along the tokens it
    // brought nothing, 318 against 327 us forwards on 65536 x 4096; one CTA an
    // SM leaves too few places for clusters of eight, 120 against 162 us on
    // 32768 x 2048 with fp32 gates.)
    p.pace = 1;
    if (p.cluster == 1 && resident >= 2 && slabs * p.B <= 148 * resident)
        while (p.pace < 4 && slabs % (2 * p.pace) == 0) p.pace *= 2;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(p.cluster * p.pace);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(slabs * p.cluster), static_cast<unsigned>(p.B));
    cfg.blockDim = dim3(static_cast<unsigned>(32 * W));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<const ScanParams>(p), maps);
}

// How the rows are read: by TMA with two channels a lane (or one, below), by
// cp.async with two where rows are no multiple of 16 bytes, else one channel a
// lane.  (Four channels a lane, 256-byte rows of 16-bit types, leave one CTA an
// SM and were slower: 382 against 302 us forwards on 65536 x 4096.)
enum class ScanPath { kTma, kPairs, kSingle };

// Channels a lane by TMA: two, but one of 16-bit x with fp32 gates, whose ring
// would leave one CTA an SM (146 against 184 us forwards and 318 against 376 us
// backwards on 65536 x 1024 with 8 sequences, 160 and 255 against 164 and 262 us
// on 32768 x 2048 with 16).
constexpr int scan_channels(int64_t x_bytes, int64_t g_bytes) { return x_bytes == 2 && g_bytes == 4 ? 1 : 2; }

struct ScanLaunch {
    ScanParams& p;
    const ScanMapsTma& maps;
    ScanPath path;
    bool backward;
    cudaStream_t stream;
    cudaError_t error = cudaSuccess;
    template <typename TX, typename TG, int V, bool TMA>
    void go()
    {
        // Eight warps a CTA.  Forwards four, where there are too few slabs for a
        // CTA each (clusters share the tokens) but enough for clusters of eight
        // to fill the GPU: 300 against 328 us on 65536 x 4096 (64 slabs), but
        // 225 against 182 us on 65536 x 2048 (32 slabs).  With cu_seqlens eight:
        // a border holds up a longer segment less often (130 against 159 us for
        // 16 sequences in 32768 x 2048).
        const int64_t slabs = (p.D + 32 * V - 1) / (32 * V) * p.B;
        const bool four = !p.cu && slabs <= 148 && slabs * kScanForwardCluster >= 148 * 3;
        if (backward)
            error = launch_scan(scan_backward_kernel<TX, TG, V, 8, TMA>, p, maps, V, 8, scan_backward_smem<TX, TG, V, 8>(),
                                kScanBackwardCluster, stream);
        else if (four)
            error = launch_scan(scan_forward_kernel<TX, TG, V, 4, TMA>, p, maps, V, 4, scan_forward_smem<TX, TG, V, 4>(),
                                kScanForwardCluster, stream);
        else
            error = launch_scan(scan_forward_kernel<TX, TG, V, 8, TMA>, p, maps, V, 8, scan_forward_smem<TX, TG, V, 8>(),
                                kScanForwardCluster, stream);
    }
    template <typename TX, typename TG>
    void operator()()
    {
        if (path == ScanPath::kTma) go<TX, TG, scan_channels(sizeof(TX), sizeof(TG)), true>();
        else if (path == ScanPath::kPairs) go<TX, TG, 2, false>();
        else go<TX, TG, 1, false>();
    }
};

cgdrStatus run_scan(ScanParams& p, const cgdrTensor* x, const cgdrTensor* g, const cgdrTensor* d_out,
                    std::initializer_list<const cgdrTensor*> outs, bool backward, const char* what, void* stream)
{
    bool pairs = pieces_aligned(x, 2) && pieces_aligned(g, 2) && pieces_aligned(d_out, 2);
    for (const cgdrTensor* t : outs) pairs = pairs && pieces_aligned(t, 2);
    const bool tma = pairs && tma_rows(x) && tma_rows(g) && tma_rows(d_out);
    const int V = scan_channels(bytes_of(x->dtype), bytes_of(g->dtype));
    ScanMapsTma maps;
    memset(&maps, 0, sizeof(maps));
    cgdrStatus st;
    if (tma && ((st = scan_map(x, V, &maps.x, "x")) || (st = scan_map(g, V, &maps.g, "g")) ||
                (st = scan_map(d_out, V, &maps.d_out, "d_out"))))
        return st;
    ScanLaunch launch{p, maps, tma ? ScanPath::kTma : pairs ? ScanPath::kPairs : ScanPath::kSingle, backward,
                      static_cast<cudaStream_t>(stream)};
    with_types(x->dtype, g->dtype, launch);
    if (launch.error != cudaSuccess) return cuda_failed(what, launch.error);
    return launched(what);
}

struct LaunchStep {
    LinearStepParams& p;
    unsigned rows;
    bool aligned;
    cudaStream_t stream;
    template <typename TX, typename TG, int V>
    void go()
    {
        p.tiles = static_cast<uint32_t>((p.D + kLinearStepThreads * V - 1) / (kLinearStepThreads * V));
        linear_step_kernel<TX, TG, V>
            <<<rows * p.tiles, kLinearStepThreads, 0, stream>>>(p);
    }
    template <typename TX, typename TG>
    void operator()()
    {
        if (aligned) go<TX, TG, 4>();
        else go<TX, TG, 1>();
    }
};

}  // namespace

extern "C" {

cgdrStatus cgdrRecurrentGatedDeltaRule(const cgdrTensor* query, const cgdrTensor* key, const cgdrTensor* value,
                                       const cgdrTensor* beta, const cgdrTensor* state,
                                       const cgdrTensor* actual_seq_lengths, const cgdrTensor* g,
                                       const cgdrTensor* state_indices, float scale, const cgdrTensor* out,
                                       int32_t* device_status, void* stream_ptr)
{
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    for (const cgdrTensor* t : {query, key, value, beta, state, out})
        if (!t) return fail(CGDR_STATUS_NULL_ARGUMENT, "query, key, value, beta, state and out are required");
    cgdrStatus st;
    if ((st = check_rank(query, 3, "query")) || (st = check_rank(key, 3, "key")) ||
        (st = check_rank(value, 3, "value")) || (st = check_rank(beta, 2, "beta")) ||
        (st = check_rank(state, 4, "state")) || (st = check_rank(out, 3, "out")))
        return st;
    const bool has_len = present(actual_seq_lengths), has_g = present(g);
    if (has_len && (st = check_rank(actual_seq_lengths, 1, "actual_seq_lengths"))) return st;
    if (has_g && (st = check_rank(g, 2, "g"))) return st;
    if (!float_type(query->dtype)) return fail(CGDR_STATUS_BAD_DTYPE, "query must be bfloat16, float16 or float32");
    for (const cgdrTensor* t : {key, value, out})
        if (t->dtype != query->dtype) return fail(CGDR_STATUS_BAD_DTYPE, "query, key, value and out must have one type");
    if (beta->dtype != query->dtype && beta->dtype != CGDR_DT_FLOAT32)
        return fail(CGDR_STATUS_BAD_DTYPE, "beta must have query's type or be float32");
    if (state->dtype != CGDR_DT_FLOAT32 && state->dtype != CGDR_DT_BF16)
        return fail(CGDR_STATUS_BAD_DTYPE, "state must be float32 or bfloat16");
    if (has_g && g->dtype != CGDR_DT_FLOAT32) return fail(CGDR_STATUS_BAD_DTYPE, "g must be float32");
    if (has_len && actual_seq_lengths->dtype != CGDR_DT_INT32)
        return fail(CGDR_STATUS_BAD_DTYPE, "actual_seq_lengths must be int32");

    const int64_t T = query->shape[0], Nk = query->shape[1], Dk = query->shape[2];
    const int64_t Nv = value->shape[1], Dv = value->shape[2], S = state->shape[0];
    if (T < 0 || Nk <= 0 || Nv <= 0 || Dk <= 0 || Dv <= 0)
        return fail(CGDR_STATUS_BAD_SHAPE, "head counts and widths must be positive");
    if (!shape_is(key, {T, Nk, Dk})) return fail(CGDR_STATUS_BAD_SHAPE, "key must have query's shape");
    if (value->shape[0] != T) return fail(CGDR_STATUS_BAD_SHAPE, "value must have shape [T, Nv, Dv]");
    if (Nv % Nk != 0) return fail(CGDR_STATUS_BAD_SHAPE, "Nv must be a multiple of Nk");
    if (!shape_is(beta, {T, Nv})) return fail(CGDR_STATUS_BAD_SHAPE, "beta must have shape [T, Nv]");
    if (has_g && !shape_is(g, {T, Nv})) return fail(CGDR_STATUS_BAD_SHAPE, "g must have shape [T, Nv]");
    if (!shape_is(state, {S, Nv, Dv, Dk})) return fail(CGDR_STATUS_BAD_SHAPE, "state must have shape [S, Nv, Dv, Dk]");
    if (!shape_is(out, {T, Nv, Dv})) return fail(CGDR_STATUS_BAD_SHAPE, "out must have shape [T, Nv, Dv]");
    if (Dk > 256) return fail(CGDR_STATUS_UNSUPPORTED, "Dk must be at most 256");
    const int64_t B = has_len ? actual_seq_lengths->shape[0] : T;
    DeltaStepParams p;
    memset(&p, 0, sizeof(p));
    if ((st = check_pool(state, state_indices, B, &p.pool))) return st;
    for (const cgdrTensor* t : {query, key, value, state, out})
        if ((st = check_inner_contiguous(t, "query/key/value/state/out"))) return st;
    if (has_len && (st = check_contiguous(actual_seq_lengths, "actual_seq_lengths"))) return st;
    for (const cgdrTensor* t : {beta, g})
        if (present(t) && (t->strides[0] < 0 || t->strides[1] < 0))
            return fail(CGDR_STATUS_BAD_STRIDE, "negative stride");
    if (B == 0 || T == 0) return clear_status(device_status, stream);
    for (const cgdrTensor* t : {query, key, value, beta, state, out})
        if (!t->data) return fail(CGDR_STATUS_NULL_ARGUMENT, "query, key, value, beta, state and out are required");
    // grid of the narrowest tiles (32 rows)
    const int64_t tiles = (Dv + kDeltaRows - 1) / kDeltaRows;
    if (Nv >= (int64_t(1) << 31) || B > (int64_t(1) << 31) / Nv || B * Nv >= (int64_t(1) << 31) / tiles)
        return fail(CGDR_STATUS_UNSUPPORTED, "B * Nv * ceil(Dv / 32) must fit in 31 bits");

    p.q = query->data; p.k = key->data; p.v = value->data; p.beta = beta->data;
    p.g = has_g ? static_cast<const float*>(g->data) : nullptr;
    p.lens = has_len ? static_cast<const int32_t*>(actual_seq_lengths->data) : nullptr;
    p.state = state->data; p.out = out->data; p.status = device_status;
    p.T = T;
    p.B = static_cast<uint32_t>(B); p.Nv = static_cast<uint32_t>(Nv); p.rep = static_cast<uint32_t>(Nv / Nk);
    p.Dk = static_cast<uint32_t>(Dk); p.Dv = static_cast<uint32_t>(Dv);
    p.q_st = query->strides[0]; p.q_sh = query->strides[1];
    p.k_st = key->strides[0]; p.k_sh = key->strides[1];
    p.v_st = value->strides[0]; p.v_sh = value->strides[1];
    p.o_st = out->strides[0]; p.o_sh = out->strides[1];
    p.b_st = beta->strides[0]; p.b_sh = beta->strides[1];
    if (has_g) { p.g_st = g->strides[0]; p.g_sh = g->strides[1]; }
    p.s_sn = state->strides[0]; p.s_sh = state->strides[1]; p.s_sv = state->strides[2];
    p.scale = scale > 0.0f ? scale : 1.0f / sqrtf(static_cast<float>(Dk));
    p.beta_f32 = beta->dtype == CGDR_DT_FLOAT32;
    const bool aligned = pieces_aligned(query, 4) && pieces_aligned(key, 4) && pieces_aligned(state, 4);
    if ((st = clear_status(device_status, stream))) return st;
    const bool f32 = state->dtype == CGDR_DT_FLOAT32;
    if (query->dtype == CGDR_DT_BF16) dispatch_delta_state<__nv_bfloat16>(p, f32, aligned, stream);
    else if (query->dtype == CGDR_DT_FLOAT16) dispatch_delta_state<__half>(p, f32, aligned, stream);
    else dispatch_delta_state<float>(p, f32, aligned, stream);
    return launched("recurrent gated delta rule");
}

cgdrStatus cgdrGatedLinearRecurrence(const cgdrTensor* x, const cgdrTensor* g, const cgdrTensor* initial_state,
                                     const cgdrTensor* cu_seqlens, const cgdrTensor* out,
                                     const cgdrTensor* final_state, const cgdrTensor* chunk_states, void* stream)
{
    ScanParams p;
    cgdrStatus st;
    if ((st = check_scan(x, g, initial_state, cu_seqlens, &p))) return st;
    if (!present(out)) return fail(CGDR_STATUS_NULL_ARGUMENT, "out is required");
    if ((st = check_like(out, x->dtype, p, "out")) || (st = check_state(final_state, p, "final_state"))) return st;
    if (present(chunk_states) && (st = check_chunks(chunk_states, &p))) return st;
    p.out = out->data; p.o_sb = out->strides[0]; p.o_st = out->strides[1];
    if (present(final_state)) {
        p.ht = static_cast<float*>(final_state->data);
        p.ht_sn = final_state->strides[0];
    }
    return run_scan(p, x, g, nullptr, {out}, false, "gated linear recurrence", stream);
}

cgdrStatus cgdrGatedLinearRecurrenceBackward(const cgdrTensor* x, const cgdrTensor* g,
                                             const cgdrTensor* initial_state, const cgdrTensor* cu_seqlens,
                                             const cgdrTensor* chunk_states, const cgdrTensor* d_out,
                                             const cgdrTensor* d_final_state, const cgdrTensor* dx,
                                             const cgdrTensor* dg, const cgdrTensor* d_initial_state, void* stream)
{
    ScanParams p;
    cgdrStatus st;
    if ((st = check_scan(x, g, initial_state, cu_seqlens, &p))) return st;
    if (!present(chunk_states)) return fail(CGDR_STATUS_NULL_ARGUMENT, "chunk_states is required");
    if (!present(d_out) && !present(d_final_state))
        return fail(CGDR_STATUS_NULL_ARGUMENT, "d_out or d_final_state is required");
    if (!present(dx) && !present(dg) && !present(d_initial_state))
        return fail(CGDR_STATUS_NULL_ARGUMENT, "dx, dg or d_initial_state is required");
    if ((st = check_chunks(chunk_states, &p)) || (st = check_like(d_out, x->dtype, p, "d_out")) ||
        (st = check_like(dx, x->dtype, p, "dx")) || (st = check_like(dg, g->dtype, p, "dg")) ||
        (st = check_state(d_final_state, p, "d_final_state")) ||
        (st = check_state(d_initial_state, p, "d_initial_state")))
        return st;
    if (present(d_out)) { p.d_out = d_out->data; p.do_sb = d_out->strides[0]; p.do_st = d_out->strides[1]; }
    if (present(dx)) { p.dx = dx->data; p.dx_sb = dx->strides[0]; p.dx_st = dx->strides[1]; }
    if (present(dg)) { p.dg = dg->data; p.dg_sb = dg->strides[0]; p.dg_st = dg->strides[1]; }
    if (present(d_final_state)) {
        p.d_ht = static_cast<const float*>(d_final_state->data);
        p.dht_sn = d_final_state->strides[0];
    }
    if (present(d_initial_state)) {
        p.d_h0 = static_cast<float*>(d_initial_state->data);
        p.dh0_sn = d_initial_state->strides[0];
    }
    return run_scan(p, x, g, d_out, {dx, dg}, true, "gated linear recurrence, backward", stream);
}

cgdrStatus cgdrGatedLinearRecurrenceStep(const cgdrTensor* x, const cgdrTensor* g, const cgdrTensor* state,
                                         const cgdrTensor* state_indices, const cgdrTensor* out,
                                         int32_t* device_status, void* stream_ptr)
{
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    for (const cgdrTensor* t : {x, g, state, out})
        if (!t) return fail(CGDR_STATUS_NULL_ARGUMENT, "x, g, state and out are required");
    cgdrStatus st;
    if ((st = check_rank(x, 2, "x")) || (st = check_rank(g, 2, "g")) || (st = check_rank(state, 2, "state")) ||
        (st = check_rank(out, 2, "out")) || (st = check_gate_types(x, g)))
        return st;
    if (state->dtype != CGDR_DT_FLOAT32) return fail(CGDR_STATUS_BAD_DTYPE, "state must be float32");
    if (out->dtype != x->dtype) return fail(CGDR_STATUS_BAD_DTYPE, "out must have x's type");
    const int64_t B = x->shape[0], D = x->shape[1], S = state->shape[0];
    if (B < 0 || D <= 0) return fail(CGDR_STATUS_BAD_SHAPE, "D must be positive");
    if (!shape_is(g, {B, D}) || !shape_is(out, {B, D}))
        return fail(CGDR_STATUS_BAD_SHAPE, "x, g and out must have one shape");
    if (!shape_is(state, {S, D})) return fail(CGDR_STATUS_BAD_SHAPE, "state must have shape [S, D]");
    LinearStepParams p;
    memset(&p, 0, sizeof(p));
    if ((st = check_pool(state, state_indices, B, &p.pool))) return st;
    for (const cgdrTensor* t : {x, g, state, out})
        if ((st = check_inner_contiguous(t, "x/g/state/out"))) return st;
    if (B == 0) return clear_status(device_status, stream);
    for (const cgdrTensor* t : {x, g, state, out})
        if (!t->data) return fail(CGDR_STATUS_NULL_ARGUMENT, "x, g, state and out are required");
    const int64_t tiles = (D + kLinearStepThreads - 1) / kLinearStepThreads;
    if (B >= (int64_t(1) << 31) / tiles) return fail(CGDR_STATUS_UNSUPPORTED, "B * ceil(D / 256) must fit in 31 bits");
    p.x = x->data; p.g = g->data; p.state = static_cast<float*>(state->data); p.out = out->data;
    p.status = device_status;
    p.D = D;
    p.x_sb = x->strides[0]; p.g_sb = g->strides[0]; p.o_sb = out->strides[0]; p.s_sn = state->strides[0];
    const bool aligned =
        pieces_aligned(x, 4) && pieces_aligned(g, 4) && pieces_aligned(state, 4) && pieces_aligned(out, 4);
    if ((st = clear_status(device_status, stream))) return st;
    with_types(x->dtype, g->dtype, LaunchStep{p, static_cast<unsigned>(B), aligned, stream});
    return launched("gated linear recurrence step");
}

}  // extern "C"
