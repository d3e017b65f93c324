// Host side of include/cgdr_rms_norm.h: argument checks and launches.  No
// device memory is allocated here.
#include <cuda_runtime.h>

#include <cstring>

#include "../../include/cgdr_rms_norm.h"
#include "host_util.cuh"
#include "kernel_rms_norm.cuh"

using namespace cgdr;
using namespace cgdr::host;

namespace {

constexpr int64_t kMaxColumns = 16384;
// Blocks of the backward pass at most: four for each of the B200's 148 SMs.  A
// constant, so that the workspace's size and the order of dweight's sum do
// not depend on the device that is current.
constexpr int64_t kBackwardBlocks = 592;

int64_t bytes_of(int32_t dt) { return dt == CGDR_DT_FLOAT32 ? 4 : dt == CGDR_DT_FP8_E4M3 ? 1 : 2; }

// Pieces of `v` elements start on a multiple of their size (16 at most).
bool pieces_aligned(const cgdrTensor* t, int64_t v)
{
    if (!present(t)) return true;
    const int64_t bytes = bytes_of(t->dtype) * v < 16 ? bytes_of(t->dtype) * v : 16;
    return reinterpret_cast<uintptr_t>(t->data) % bytes == 0 && t->shape[t->ndim - 1] % v == 0 &&
           (t->ndim < 2 || t->shape[0] <= 1 || t->strides[0] % v == 0);
}

uint32_t row_bytes(const cgdrTensor* t) { return static_cast<uint32_t>(t->shape[0] > 1 ? t->strides[0] * bytes_of(t->dtype) : 0); }

// The kernels take rows less than 4 GiB apart.
cgdrStatus check_row_stride(const cgdrTensor* t, const char* name)
{
    if (t->shape[0] > 1 && t->strides[0] >= (int64_t(1) << 30))
        return fail(CGDR_STATUS_UNSUPPORTED, "%s's rows must be less than 2^30 elements apart", name);
    return CGDR_STATUS_SUCCESS;
}

// An optional [R, D] tensor of type dt.
cgdrStatus check_rows(const cgdrTensor* t, int32_t dt, int64_t R, int64_t D, const char* name)
{
    if (!present(t)) return CGDR_STATUS_SUCCESS;
    cgdrStatus st;
    if ((st = check_rank(t, 2, name))) return st;
    if (t->dtype != dt) return fail(CGDR_STATUS_BAD_DTYPE, "%s has the wrong type", name);
    if (!shape_is(t, {R, D})) return fail(CGDR_STATUS_BAD_SHAPE, "%s must have shape [R, D]", name);
    if ((st = check_inner_contiguous(t, name))) return st;
    return check_row_stride(t, name);
}

cgdrStatus check_x(const cgdrTensor* x, const cgdrTensor* weight, const char* name)
{
    if (!present(x) || !present(weight)) return fail(CGDR_STATUS_NULL_ARGUMENT, "%s and weight are required", name);
    cgdrStatus st;
    if ((st = check_rank(x, 2, name)) || (st = check_rank(weight, 1, "weight"))) return st;
    if (x->dtype != CGDR_DT_BF16 && x->dtype != CGDR_DT_FLOAT16 && x->dtype != CGDR_DT_FLOAT32)
        return fail(CGDR_STATUS_BAD_DTYPE, "%s must be bfloat16, float16 or float32", name);
    if (weight->dtype != x->dtype && weight->dtype != CGDR_DT_FLOAT32)
        return fail(CGDR_STATUS_BAD_DTYPE, "weight must have %s's type or be float32", name);
    const int64_t R = x->shape[0], D = x->shape[1];
    if (R <= 0 || D <= 0) return fail(CGDR_STATUS_BAD_SHAPE, "dimensions must be positive");
    if (!shape_is(weight, {D})) return fail(CGDR_STATUS_BAD_SHAPE, "weight must have shape [D]");
    if (D > kMaxColumns)
        return fail(CGDR_STATUS_UNSUPPORTED, "D must be at most %lld", static_cast<long long>(kMaxColumns));
    if (R >= (int64_t(1) << 31) - 4096) return fail(CGDR_STATUS_UNSUPPORTED, "R must be less than 2^31 - 4096");
    if ((st = check_inner_contiguous(x, name)) || (st = check_row_stride(x, name))) return st;
    return check_inner_contiguous(weight, "weight");
}

// Calls f.template operator()<TX, V, LPR, NV>() for x's type and row length.
// Pieces of 16 bytes, one a lane up to 512 lanes: few registers a lane and many
// rows in flight (two pieces in half the lanes: 193 against 188 us forwards on
// 32768 x 4096, 332 against 234 backwards; with 1024 lanes a row's barrier
// costs more: 270 against 197 us on 16384 x 8192).  Single columns where rows
// are not made of such pieces.
template <typename TX, typename F>
void with_shape(int64_t D, bool pieces, F& f)
{
    constexpr int V = 16 / sizeof(TX);
    if (!pieces) {
        if (D <= 128) f.template operator()<TX, 1, 32, 4>();
        else if (D <= 1024) f.template operator()<TX, 1, 256, 4>();
        else if (D <= 4096) f.template operator()<TX, 1, 512, 8>();
        else f.template operator()<TX, 1, 1024, 16>();
        return;
    }
    const int64_t n = (D + V - 1) / V;
    if (n <= 8) f.template operator()<TX, V, 8, 1>();
    else if (n <= 16) f.template operator()<TX, V, 16, 1>();
    else if (n <= 32) f.template operator()<TX, V, 32, 1>();
    else if (n <= 64) f.template operator()<TX, V, 64, 1>();
    else if (n <= 128) f.template operator()<TX, V, 128, 1>();
    else if (n <= 256) f.template operator()<TX, V, 256, 1>();
    else if (n <= 512) f.template operator()<TX, V, 512, 1>();
    else if (n <= 1024) f.template operator()<TX, V, 512, 2>();
    else if (n <= 2048) f.template operator()<TX, V, 1024, 2>();
    else if constexpr (V == 4) f.template operator()<TX, V, 1024, 4>();
}

template <typename F>
void with_type(int32_t dt, int64_t D, bool pieces, F&& f)
{
    if (dt == CGDR_DT_BF16) with_shape<__nv_bfloat16>(D, pieces, f);
    else if (dt == CGDR_DT_FLOAT16) with_shape<__half>(D, pieces, f);
    else with_shape<float>(D, pieces, f);
}

struct LaunchForward {
    const NormParams& p;
    bool fp8;
    cudaStream_t stream;
    template <typename TX, int V, int LPR, int NV>
    void operator()()
    {
        const unsigned grid = static_cast<unsigned>((p.R + norm_rows(LPR) - 1) / norm_rows(LPR));
        if (fp8) norm_forward_kernel<TX, V, LPR, NV, true><<<grid, norm_threads(LPR), 0, stream>>>(p);
        else norm_forward_kernel<TX, V, LPR, NV, false><<<grid, norm_threads(LPR), 0, stream>>>(p);
    }
};

struct LaunchBackward {
    const NormBackwardParams& p;
    cudaStream_t stream;
    int64_t grid = 0;
    template <typename TX, int V, int LPR, int NV>
    void operator()()
    {
        // as many blocks as are resident together
        constexpr int64_t kMost = 148 * norm_backward_blocks(LPR);
        static_assert(kMost <= kBackwardBlocks, "the workspace holds a row of partial sums a block");
        grid = (p.R + norm_rows(LPR) - 1) / norm_rows(LPR);
        if (grid > kMost) grid = kMost;
        const unsigned n = static_cast<unsigned>(grid);
        if (p.gate) norm_backward_kernel<TX, V, LPR, NV, true><<<n, norm_threads(LPR), 0, stream>>>(p);
        else norm_backward_kernel<TX, V, LPR, NV, false><<<n, norm_threads(LPR), 0, stream>>>(p);
    }
};

uint64_t backward_bytes(int64_t R, int64_t D)
{
    return static_cast<uint64_t>(R < kBackwardBlocks ? R : kBackwardBlocks) * D * sizeof(float);
}

template <typename TW>
void sum_weight(const NormBackwardParams& p, int64_t blocks, const cgdrTensor* dw, cudaStream_t stream)
{
    norm_weight_kernel<TW><<<static_cast<unsigned>((p.D + 31) / 32), dim3(32, 32), 0, stream>>>(
        p.dw, blocks, p.D, static_cast<TW*>(dw->data));
}

cgdrStatus launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(CGDR_STATUS_CUDA_ERROR, "%s: %s", what, cudaGetErrorString(e));
    g_err[0] = '\0';
    return CGDR_STATUS_SUCCESS;
}

}  // namespace

extern "C" {

cgdrStatus cgdrRmsNorm(const cgdrTensor* x, const cgdrTensor* weight, const cgdrTensor* residual,
                       const cgdrTensor* gate, double eps, int64_t group, const cgdrTensor* y,
                       const cgdrTensor* y_scale, const cgdrTensor* z, void* stream)
{
    cgdrStatus st;
    if ((st = check_x(x, weight, "x"))) return st;
    if (!present(y)) return fail(CGDR_STATUS_NULL_ARGUMENT, "y is required");
    if (present(residual) != present(z))
        return fail(CGDR_STATUS_NULL_ARGUMENT, "residual and z must be both present or both absent");
    const int64_t R = x->shape[0], D = x->shape[1];
    const bool fp8 = present(y_scale);
    if ((st = check_rows(residual, x->dtype, R, D, "residual")) || (st = check_rows(gate, x->dtype, R, D, "gate")) ||
        (st = check_rows(z, x->dtype, R, D, "z")) ||
        (st = check_rows(y, fp8 ? int32_t(CGDR_DT_FP8_E4M3) : x->dtype, R, D, "y")))
        return st;
    if (!(eps >= 0.0)) return fail(CGDR_STATUS_BAD_SHAPE, "eps must not be negative");
    NormParams p;
    memset(&p, 0, sizeof(p));
    const int64_t V = 16 / bytes_of(x->dtype);
    if (fp8) {
        if (group != D && group != 32 && group != 64 && group != 128)
            return fail(CGDR_STATUS_UNSUPPORTED, "group must be D, 32, 64 or 128");
        if (D % group != 0) return fail(CGDR_STATUS_BAD_SHAPE, "group must divide D");
        if ((st = check_rank(y_scale, 2, "y_scale"))) return st;
        if (y_scale->dtype != CGDR_DT_FLOAT32) return fail(CGDR_STATUS_BAD_DTYPE, "y_scale must be float32");
        if (!shape_is(y_scale, {R, D / group}))
            return fail(CGDR_STATUS_BAD_SHAPE, "y_scale must have shape [R, D / group]");
        if ((y_scale->shape[1] > 1 && y_scale->strides[1] != 1) || (R > 1 && y_scale->strides[0] != D / group))
            return fail(CGDR_STATUS_BAD_STRIDE, "y_scale must be contiguous");
        p.scale = static_cast<float*>(y_scale->data);
        p.group = static_cast<int32_t>(group);
    }
    p.x = x->data; p.x_s = row_bytes(x);
    p.w = weight->data; p.w_f32 = weight->dtype == CGDR_DT_FLOAT32;
    p.y = y->data; p.y_s = row_bytes(y);
    if (present(residual)) {
        p.residual = residual->data; p.r_s = row_bytes(residual);
        p.z = z->data; p.z_s = row_bytes(z);
    }
    if (present(gate)) { p.gate = gate->data; p.a_s = row_bytes(gate); }
    p.R = static_cast<int32_t>(R);
    p.D = static_cast<int32_t>(D);
    p.eps = static_cast<float>(eps);
    p.inv_d = static_cast<float>(1.0 / static_cast<double>(D));
    const bool pieces = pieces_aligned(x, V) && pieces_aligned(weight, V) && pieces_aligned(residual, V) &&
                        pieces_aligned(gate, V) && pieces_aligned(y, V) && pieces_aligned(z, V);
    with_type(x->dtype, D, pieces, LaunchForward{p, fp8, static_cast<cudaStream_t>(stream)});
    return launched("rms norm");
}

cgdrStatus cgdrRmsNormBackwardGetWorkspaceSize(const cgdrTensor* z, const cgdrTensor* dweight,
                                               uint64_t* workspace_size)
{
    if (!z || !workspace_size) return fail(CGDR_STATUS_NULL_ARGUMENT, "z and workspace_size are required");
    cgdrStatus st;
    if ((st = check_rank(z, 2, "z"))) return st;
    *workspace_size = present(dweight) ? backward_bytes(z->shape[0], z->shape[1]) : 0;
    return CGDR_STATUS_SUCCESS;
}

cgdrStatus cgdrRmsNormBackward(const cgdrTensor* z, const cgdrTensor* weight, const cgdrTensor* gate, double eps,
                               const cgdrTensor* dy, const cgdrTensor* dz, const cgdrTensor* dx,
                               const cgdrTensor* dweight, const cgdrTensor* dgate, void* workspace,
                               uint64_t workspace_size, void* stream_ptr)
{
    cudaStream_t stream = static_cast<cudaStream_t>(stream_ptr);
    cgdrStatus st;
    if ((st = check_x(z, weight, "z"))) return st;
    if (!present(dy)) return fail(CGDR_STATUS_NULL_ARGUMENT, "dy is required");
    if (!present(dx) && !present(dweight) && !present(dgate))
        return fail(CGDR_STATUS_NULL_ARGUMENT, "dx, dweight or dgate is required");
    if (present(dgate) && !present(gate)) return fail(CGDR_STATUS_NULL_ARGUMENT, "dgate needs gate");
    const int64_t R = z->shape[0], D = z->shape[1];
    for (const cgdrTensor* t : {gate, dy, dz, dx, dgate})
        if ((st = check_rows(t, z->dtype, R, D, "gate/dy/dz/dx/dgate"))) return st;
    if (!(eps >= 0.0)) return fail(CGDR_STATUS_BAD_SHAPE, "eps must not be negative");
    NormBackwardParams p;
    memset(&p, 0, sizeof(p));
    if (present(dweight)) {
        if ((st = check_rank(dweight, 1, "dweight"))) return st;
        if (dweight->dtype != weight->dtype) return fail(CGDR_STATUS_BAD_DTYPE, "dweight must have weight's type");
        if (!shape_is(dweight, {D})) return fail(CGDR_STATUS_BAD_SHAPE, "dweight must have shape [D]");
        if ((st = check_inner_contiguous(dweight, "dweight"))) return st;
        if (!workspace) return fail(CGDR_STATUS_NULL_ARGUMENT, "workspace must not be NULL");
        if (workspace_size < backward_bytes(R, D))
            return fail(CGDR_STATUS_WORKSPACE_TOO_SMALL, "workspace must hold %llu bytes",
                        static_cast<unsigned long long>(backward_bytes(R, D)));
        if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return fail(CGDR_STATUS_WORKSPACE_TOO_SMALL, "workspace must be 16-byte aligned");
        p.dw = static_cast<float*>(workspace);
    }
    p.z = z->data; p.z_s = row_bytes(z);
    p.w = weight->data; p.w_f32 = weight->dtype == CGDR_DT_FLOAT32;
    p.dy = dy->data; p.dy_s = row_bytes(dy);
    if (present(gate)) { p.gate = gate->data; p.a_s = row_bytes(gate); }
    if (present(dz)) { p.dz = dz->data; p.dz_s = row_bytes(dz); }
    if (present(dx)) { p.dx = dx->data; p.dx_s = row_bytes(dx); }
    if (present(dgate)) { p.dgate = dgate->data; p.da_s = row_bytes(dgate); }
    p.R = static_cast<int32_t>(R);
    p.D = static_cast<int32_t>(D);
    p.eps = static_cast<float>(eps);
    p.inv_d = static_cast<float>(1.0 / static_cast<double>(D));
    const int64_t V = 16 / bytes_of(z->dtype);
    bool pieces = pieces_aligned(weight, V);
    for (const cgdrTensor* t : {z, gate, dy, dz, dx, dgate}) pieces = pieces && pieces_aligned(t, V);
    LaunchBackward launch{p, stream};
    with_type(z->dtype, D, pieces, launch);
    if ((st = launched("rms norm, backward"))) return st;
    if (p.dw) {
        if (dweight->dtype == CGDR_DT_FLOAT32) sum_weight<float>(p, launch.grid, dweight, stream);
        else if (dweight->dtype == CGDR_DT_BF16) sum_weight<__nv_bfloat16>(p, launch.grid, dweight, stream);
        else sum_weight<__half>(p, launch.grid, dweight, stream);
        return launched("rms norm, backward");
    }
    return CGDR_STATUS_SUCCESS;
}

}  // extern "C"
