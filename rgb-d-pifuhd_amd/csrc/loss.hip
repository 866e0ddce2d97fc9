// Supervised-forward loss of the reference (`CustomBCELoss.forward`, net_util.py:45-66) as a device reduction, alone
// (pifu_bce_loss) or with its gradient in the same pass (pifu_bce_loss_grad).  Deterministic: per-block partial sums in a fixed order
// (double), then a single-block fixed-order sum.
#include "linear_common.h"

namespace {

constexpr int LOSS_BLOCKS = 1024, BCE_ONE_BLOCK = 1024;

struct BceArgs {
    const float *pred, *gt;      // [B][n]
    const float *gamma;          // [B] or null (fixed_gamma)
    const float *w;              // null, [B] (w_full = 0) or [B][n] (w_full = 1)
    int64_t n;                   // elements per batch entry
    int64_t total;               // B * n
    float fixed_gamma;
    int brock, w_full;
    double *partial;             // [LOSS_BLOCKS]
    float *out;
};

// clamp(pred, 1e-5, 1 - 1e-5); a NaN stays one, as in the reference's clamp: the loss of a forward pass that went wrong says so
__device__ __forceinline__ float bce_clamp(float pred)
{
    return pred < 1e-5f ? 1e-5f : pred > 1.0f - 1e-5f ? 1.0f - 1e-5f : pred;
}

// one term of the weighted cross entropy, in fp32 like the reference's tensor expression:
//   p = clamp(pred, 1e-5, 1 - 1e-5);  t = gt (brock: 3 gt - 1)
//   -(g t log p + (1 - g)(1 - t) log(1 - p)) * w
__device__ __forceinline__ float bce_term(float pred, float gt, float g, float w, int brock)
{
    const float p = bce_clamp(pred);
    const float t = brock ? 3.0f * gt - 1.0f : gt;
    const float pos = g * t * logf(p);
    const float neg = (1.0f - g) * (1.0f - t) * logf(1.0f - p);
    return -(pos + neg) * w;
}

__global__ void k_bce_partial(const BceArgs a)
{
    __shared__ double red[256];
    double acc = 0.0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.total; i += (int64_t)gridDim.x * 256) {
        const int64_t b = i / a.n;
        const float g = a.gamma ? a.gamma[b] : a.fixed_gamma;
        const float w = a.w ? (a.w_full ? a.w[i] : a.w[b]) : 1.0f;
        acc += (double)bce_term(a.pred[i], a.gt[i], g, w, a.brock);
    }
    red[threadIdx.x] = acc;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) a.partial[blockIdx.x] = red[0];
}

// value and gradient in one pass.  Elementwise: bound by its bytes (2 x sizeof(T) + 4, + 4 with a weight per element)
template <class T> struct BceGradArgs {
    BceArgs l;                   // l.pred is unused
    const T *pred;
    T *grad;
    float scale, out_scale;      // scale / total, scale
};

// d term / d pred: the clamp passes a gradient only between its bounds (and none for a NaN)
__device__ __forceinline__ float bce_slope(float pred, float gt, float g, float w, int brock)
{
    const float t = brock ? 3.0f * gt - 1.0f : gt;
    const float s = (1.0f - g) * (1.0f - t) / (1.0f - pred) - g * t / pred;
    return pred >= 1e-5f && pred <= 1.0f - 1e-5f ? s * w : 0.0f;
}

// bce_term with one logarithm where the target is 0 or 1: the other one's factor is 0
__device__ __forceinline__ float bce_value(float pred, float gt, float g, float w, int brock)
{
    if (brock || !(gt == 0.f || gt == 1.f)) return bce_term(pred, gt, g, w, brock);
    const float p = bce_clamp(pred);
    return -((gt == 0.f ? 1.0f - g : g) * logf(gt == 0.f ? 1.0f - p : p)) * w;
}

// A lane takes 8 consecutive elements of a batch entry.  A grid of one block finishes the value itself: 5000 points in 5.9 us.
// 4 x 2000001 bf16 with a weight per point: 28 us, 3.4 TB/s (the logarithms' instructions take about 14 us of it; two per element
// instead of one: 31 us).
template <class T> __global__ void __launch_bounds__(BCE_ONE_BLOCK) k_bce_grad(const BceGradArgs<T> a)
{
    __shared__ double red[BCE_ONE_BLOCK];
    double acc = 0.0;
    const int64_t chunks = (a.l.n + 7) / 8, all = a.l.total / a.l.n * chunks;
    for (int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; c < all; c += (int64_t)gridDim.x * blockDim.x) {
        const int64_t b = c / chunks, col = (c - b * chunks) * 8, at = b * a.l.n + col, left = a.l.n - col;
        const int valid = left >= 8 ? 8 : (int)left;
        const float g = a.l.gamma ? a.l.gamma[b] : a.l.fixed_gamma, w = a.l.w && !a.l.w_full ? a.l.w[b] : 1.0f;
        float p[8], gt[8], ws[8];
        load8(a.pred + at, valid, p);
        load8(a.l.gt + at, valid, gt);
        if (a.l.w_full) load8(a.l.w + at, valid, ws);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) ws[i] = w;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i < valid) acc += (double)bce_value(p[i], gt[i], g, ws[i], a.l.brock);
            p[i] = bce_slope(p[i], gt[i], g, ws[i], a.l.brock) * a.scale;
        }
        store8(a.grad + at, valid, p);
    }
    if (!a.l.partial) return;
    red[threadIdx.x] = acc;
    __syncthreads();
    for (int o = blockDim.x / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) *a.l.out = (float)(red[0] / (double)a.l.total) * a.out_scale;
        else a.l.partial[blockIdx.x] = red[0];
    }
}

__global__ void k_bce_final(const double *partial, int nblocks, int64_t total, float scale, float *out)
{
    __shared__ double red[256];
    double acc = 0.0;
    for (int i = threadIdx.x; i < nblocks; i += 256) acc += partial[i];
    red[threadIdx.x] = acc;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) *out = (float)(red[0] / (double)total) * scale;
}

}  // namespace

extern "C" int pifu_bce_loss(pifu_ctx *ctx, const float *pred, const float *gt, int batch, int64_t n, const float *gamma,
                             float fixed_gamma, const float *w, int w_per_element, int brock, float *out, pifu_stream stream)
{
    PIFU_REQUIRE(ctx && pred && gt && out, PIFU_ERR_INVALID, "pifu_bce_loss: null argument");
    PIFU_REQUIRE(batch > 0 && n > 0, PIFU_ERR_INVALID, "pifu_bce_loss: empty input (the reference's mean() would be nan)");
    PIFU_USE(ctx, stream);
    PIFU_HIP(hipSetDevice(ctx->device));
    int rc = pifu_ensure(ctx->misc, LOSS_BLOCKS * sizeof(double));
    if (rc) return rc;
    BceArgs a{};
    a.pred = pred; a.gt = gt; a.gamma = gamma; a.w = w; a.n = n; a.total = (int64_t)batch * n;
    a.fixed_gamma = fixed_gamma; a.brock = brock != 0; a.w_full = w_per_element != 0;
    a.partial = reinterpret_cast<double *>(ctx->misc.p);      // stream-ordered scratch
    a.out = out;
    const int nblocks = (int)((a.total + 1023) / 1024 < LOSS_BLOCKS ? (a.total + 1023) / 1024 : LOSS_BLOCKS);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(k_bce_partial, dim3(nblocks), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_bce_final, dim3(1), dim3(256), 0, st, (const double *)a.partial, nblocks, a.total, 1.0f, out);
    PIFU_HIP(hipGetLastError());
    return PIFU_OK;
}

template <class T> static int bce_grad(const BceArgs &l, const void *pred, void *grad, float scale, hipStream_t st)
{
    BceGradArgs<T> a{};
    a.l = l; a.pred = (const T *)pred; a.grad = (T *)grad;
    a.scale = (float)((double)scale / (double)l.total);
    a.out_scale = scale;
    // up to 8192 elements: one block of 1024 lanes, one launch; else 256 lanes a block and a second kernel for the blocks' sums
    const int64_t chunks = l.total / l.n * ((l.n + 7) / 8);
    const bool one = chunks <= BCE_ONE_BLOCK;
    int nblocks = one ? 1 : (int)(chunks < (int64_t)LOSS_BLOCKS * 256 ? (chunks + 255) / 256 : LOSS_BLOCKS);
    PIFU_LAUNCH(k_bce_grad<T>, dim3(nblocks), dim3(one ? BCE_ONE_BLOCK : 256), 0, st, &a);
    if (one || !l.partial) return PIFU_OK;
    const double *partial = l.partial;
    int64_t total = l.total;
    float *out = l.out;
    PIFU_LAUNCH(k_bce_final, dim3(1), dim3(256), 0, st, &partial, &nblocks, &total, &scale, &out);
    return PIFU_OK;
}

extern "C" int pifu_bce_loss_grad(pifu_ctx *ctx, int dtype, const void *pred, const float *gt, int batch, int64_t n,
                                  const float *gamma, float fixed_gamma, const float *w, int w_per_element, int brock, float scale,
                                  float *out, void *grad, void *workspace, int64_t workspace_bytes, pifu_stream stream)
{
    static_assert(PIFU_BCE_WORKSPACE >= LOSS_BLOCKS * sizeof(double), "one partial sum per block");
    PIFU_REQUIRE(ctx && pred && gt && grad, PIFU_ERR_INVALID, "pifu_bce_loss_grad: null argument");
    PIFU_REQUIRE(pifu_dtype_ok(dtype), PIFU_ERR_INVALID, "pifu_bce_loss_grad: dtype %d is not PIFU_F32, PIFU_BF16 or PIFU_F16", dtype);
    PIFU_REQUIRE(batch > 0 && n > 0, PIFU_ERR_INVALID, "pifu_bce_loss_grad: empty input (the reference's mean() would be nan)");
    PIFU_REQUIRE(!out || (workspace && workspace_bytes >= PIFU_BCE_WORKSPACE), PIFU_ERR_NOMEM,
                 "pifu_bce_loss_grad: the value needs a workspace of %d bytes", PIFU_BCE_WORKSPACE);
    PIFU_REQUIRE((uintptr_t)workspace % 8 == 0, PIFU_ERR_INVALID, "pifu_bce_loss_grad: the workspace is not 8-byte aligned");
    PifuDeviceGuard guard(ctx->device);
    PIFU_HIP(guard.err);
    BceArgs l{};
    l.gt = gt; l.gamma = gamma; l.w = w; l.n = n; l.total = (int64_t)batch * n;
    l.fixed_gamma = fixed_gamma; l.brock = brock != 0; l.w_full = w_per_element != 0;
    l.partial = out ? (double *)workspace : nullptr;
    l.out = out;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == PIFU_F32) return bce_grad<float>(l, pred, grad, scale, st);
    if (dtype == PIFU_BF16) return bce_grad<bf16_t>(l, pred, grad, scale, st);
    return bce_grad<f16_t>(l, pred, grad, scale, st);
}
