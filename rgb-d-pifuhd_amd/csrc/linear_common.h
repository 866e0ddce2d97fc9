// Element types, 8-element chunks, activations and the 8-bit checkpoint codec of the training operators (linear.hip, pack8.hip,
// loss.hip).  gfx950 only.
#pragma once
#include <type_traits>

#include "linear_plan.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// Makes `ctx`'s device the current one for the duration of an entry point and puts the caller's back afterwards.
struct PifuDeviceGuard {
    int before = -1;
    hipError_t err = hipSuccess;
    explicit PifuDeviceGuard(int device)
    {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else if (err == hipSuccess) before = -1;
    }
    ~PifuDeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
};

// A kernel launch's own error, so that one left behind by somebody else's call is not reported here.
#define PIFU_LAUNCH(kernel, grid, block, lds, st, ...)                                                       \
    do {                                                                                                     \
        void *launch_args_[] = {__VA_ARGS__};                                                                \
        PIFU_HIP(hipLaunchKernel((const void *)(kernel), (grid), (block), launch_args_, (lds), (st)));       \
    } while (0)

static inline bool pifu_dtype_ok(int dtype) { return dtype == PIFU_F32 || dtype == PIFU_BF16 || dtype == PIFU_F16; }

// ---- chunks: 8 consecutive elements of a row.  Rows start at any address the element type allows (an odd pitch of 257 bf16
// elements is a case of the classifier's own): the packed struct lets the compiler use the widest loads, which gfx950 executes
// at any byte address.
template <int BYTES, int ALIGN> struct alignas(ALIGN) __attribute__((packed)) Bytes { uint32_t v[BYTES / 4]; };

// f(first row, how many of the lane's rows, 256 / tx apart, whether its chunk is whole) for the rows of a lane in block `block` of a
// cut.  Whole chunks have code of their own: a test at each load would hold back the loads behind it (200000 x 1024 bf16 unpacked in
// 175 us instead of 107).
template <class F> __device__ __forceinline__ void each_row(int tx, int64_t rows, int64_t block, int64_t m, int valid, F f)
{
    const int step = 256 / tx;
    const int64_t first = block * rows, last = first + rows < m ? first + rows : m;
    int64_t row = first + threadIdx.x / tx;
    auto run = [&](auto whole) {
        for (; row + 3 * step < last; row += 4 * step) f(row, std::integral_constant<int, 4>(), whole);
        for (; row < last; row += step) f(row, std::integral_constant<int, 1>(), whole);
    };
    if (valid >= 8) run(std::true_type());
    else if (valid > 0) run(std::false_type());
}

template <class T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

template <class T> __device__ __forceinline__ void load8(const T *p, int valid, float v[8])
{
    if (valid >= 8) {
        typedef Bytes<8 * sizeof(T), sizeof(T)> B;
        union { B b; T t[8]; } u;
        u.b = *reinterpret_cast<const B *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f(u.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < valid ? to_f(p[i]) : 0.f;
    }
}

template <class T> __device__ __forceinline__ void store8(T *p, int valid, const float v[8])
{
    if (valid >= 8) {
        typedef Bytes<8 * sizeof(T), sizeof(T)> B;
        union { B b; T t[8]; } u;
#pragma unroll
        for (int i = 0; i < 8; i++) u.t[i] = (T)v[i];
        *reinterpret_cast<B *>(p) = u.b;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) if (i < valid) p[i] = (T)v[i];
    }
}

// ---- activations, fp32, on the hardware's exponential and reciprocal.  The comparisons let a NaN through.  exp_f's argument is
// rounded to fp32 in base 2, so its value is off by up to |x| 2^-23 of itself: 2^-17 at the far end of sigmoid and silu, where the
// result is under 2^-80 (a second product and sum to correct it would be paid by every element of every epilogue).
__device__ __forceinline__ float exp_f(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + exp_f(-z)); }

// The normal distribution below -|z|, given e = exp(-z^2 / 2): erfc(x) = t q(t) exp(-x^2) with t = 1 / (1 + 0.335 x), x = |z| / sqrt 2,
// and q a polynomial fitted (minimax, relative) to 1.6e-7 over x in [0, 14].  No cancellation in the tail, one exponential for
// gelu and its derivative together; gelu is off by at most 2.4e-7, the rounding of fp32 itself at |z| ~ 4 (the library's erff costs
// three times the instructions, and its 1 + erf cancels there).
__device__ __forceinline__ float normal_tail(float z, float e)
{
    const float t = __builtin_amdgcn_rcpf(1.f + 0.23688077f * fabsf(z));
    float q = -0.1201652793f;
    q = q * t + 0.3765159764f;
    q = q * t - 0.2283688949f;
    q = q * t + 0.3096832858f;
    q = q * t + 0.09449353218f;
    q = q * t + 0.1911898964f;
    q = q * t + 0.1875818349f;
    q = q * t + 0.1890694859f;
    return 0.5f * t * q * e;
}

__device__ __forceinline__ float gelu_f(float z)
{
    const float tail = normal_tail(z, exp_f(-0.5f * z * z));
    return z * (z < 0.f ? tail : 1.f - tail);
}

template <int N, class F> __device__ __forceinline__ void each(float *v, F f)
{
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = f(v[i]);
}

// the activation of N values: chosen once for all of them
template <int N> __device__ __forceinline__ void act_all(float *v, int act)
{
    switch (act) {
        case PIFU_ACT_RELU: each<N>(v, [](float z) { return z < 0.f ? 0.f : z; }); break;
        case PIFU_ACT_LEAKY_RELU: each<N>(v, [](float z) { return z < 0.f ? z * 0.01f : z; }); break;
        case PIFU_ACT_SIGMOID: each<N>(v, [](float z) { return sigmoid_f(z); }); break;
        case PIFU_ACT_TANH:
#pragma unroll 1
            for (int i = 0; i < N; i++) v[i] = tanhf(v[i]);
            break;
        case PIFU_ACT_GELU: each<N>(v, [](float z) { return gelu_f(z); }); break;
        case PIFU_ACT_SILU: each<N>(v, [](float z) { return z * sigmoid_f(z); }); break;
        default: break;
    }
}

// sigmoid(z) sigmoid(-z), the derivative of the sigmoid at +-z: in this form nothing cancels on the saturated side (s (1 - s) of a
// rounded s is off by a fifth at z = 15 and 0 from 17 on)
__device__ __forceinline__ float sigmoid_slope(float z)
{
    const float e = exp_f(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.f + e);
    return e * r * r;
}

// g[i] *= derivative of the activation, from the pre-activations v or (from_output) from v = act(z)
template <int N, class F> __device__ __forceinline__ void each_times(float *g, const float *v, F f)
{
#pragma unroll
    for (int i = 0; i < N; i++) g[i] *= f(v[i]);
}

template <int N> __device__ __forceinline__ void slope_all(float *g, const float *v, int act, int from_output)
{
    switch (act) {
        case PIFU_ACT_RELU: each_times<N>(g, v, [](float z) { return z <= 0.f ? 0.f : 1.f; }); break;
        case PIFU_ACT_LEAKY_RELU: each_times<N>(g, v, [](float z) { return z <= 0.f ? 0.01f : 1.f; }); break;
        case PIFU_ACT_SIGMOID:
            if (from_output) each_times<N>(g, v, [](float s) { return s * (1.f - s); });
            else each_times<N>(g, v, [](float z) { return sigmoid_slope(z); });
            break;
        case PIFU_ACT_TANH:
            if (from_output) each_times<N>(g, v, [](float t) { return (1.f - t) * (1.f + t); });
            else each_times<N>(g, v, [](float z) { return 4.f * sigmoid_slope(2.f * z); });      // tanh z = 2 sigmoid(2 z) - 1
            break;
        case PIFU_ACT_GELU:
            each_times<N>(g, v, [](float z) {
                const float e = exp_f(-0.5f * z * z), tail = normal_tail(z, e);
                return (z < 0.f ? tail : 1.f - tail) + z * 0.39894228040143268f * e;
            });
            break;
        case PIFU_ACT_SILU: each_times<N>(g, v, [](float z) { const float s = sigmoid_f(z); return s * (1.f + z * (1.f - s)); }); break;
        default: break;
    }
}

// ---- 8-bit checkpoints.  A block is 4 chunks; four neighbouring lanes (lane & ~3) hold its chunks.
// scale byte of a block whose largest finite magnitude is a
__device__ __forceinline__ uint32_t pack8_scale(float a)
{
    const uint32_t bits = __float_as_uint(a);
    const int b = (int)(bits >> 23) + ((bits & 0x7fffffu) > 0x600000u) - 8;
    return (uint32_t)(b < 1 ? 1 : b);
}
__device__ __forceinline__ float pack8_unit(uint32_t scale) { return __uint_as_float(scale << 23); }                // 2^(scale - 127)
__device__ __forceinline__ float pack8_inverse(uint32_t scale) { return __uint_as_float((254u - scale) << 23); }    // 2^(127 - scale)

__device__ __forceinline__ float pack8_finite(float v) { const float a = fabsf(v); return a <= 3.402823466e38f ? a : 0.f; }

// the codes of one chunk, lowest element in the lowest byte
__device__ __forceinline__ uint2 pack8_codes(const float v[8], float inverse)
{
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = fabsf(v[i]) <= 3.402823466e38f ? v[i] * inverse : __uint_as_float(0x7fc00000u);
    uint2 r;
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    r.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    r.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], lo, true);
    return r;
}

// the largest of four neighbouring lanes' values
__device__ __forceinline__ float quad_max(float a)
{
    a = fmaxf(a, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(a), 0xb1, 0xf, 0xf, true)));       // lanes 1 0 3 2
    return fmaxf(a, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(a), 0x4e, 0xf, 0xf, true)));    // lanes 2 3 0 1
}

// Packs the chunk v (columns col .. col + 7 of row `codes` / `scales`) together with the three neighbouring lanes that hold the
// rest of its block; every lane of the four calls it, `valid` (<= 0: none) columns of the chunk exist.
__device__ __forceinline__ void pack8_chunk(uint8_t *codes, uint8_t *scales, int64_t col, int valid, const float v[8])
{
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) a = i < valid ? fmaxf(a, pack8_finite(v[i])) : a;
    a = quad_max(a);
    if (valid <= 0) return;
    const uint32_t s = pack8_scale(a);
    const uint2 q = pack8_codes(v, pack8_inverse(s));
    if (valid >= 8) {
        typedef Bytes<8, 1> B;
        B b;
        b.v[0] = q.x; b.v[1] = q.y;
        *reinterpret_cast<B *>(codes + col) = b;
    } else {
        for (int i = 0; i < valid; i++) codes[col + i] = (uint8_t)((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xffu);
    }
    if ((col & 31) == 0) scales[col >> 5] = (uint8_t)s;
}

typedef float f32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void unpack8_codes(uint2 q, float unit, float v[8])
{
    const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.x, true);
    const f32x2_t c = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)q.y, true);
    v[0] = a.x * unit; v[1] = a.y * unit; v[2] = b.x * unit; v[3] = b.y * unit;
    v[4] = c.x * unit; v[5] = c.y * unit; v[6] = d.x * unit; v[7] = d.y * unit;
}

// raw codes of columns col .. col + 7 (valid >= 1 of them exist; the rest read as code 0)
__device__ __forceinline__ uint2 load_codes(const uint8_t *codes, int64_t col, int valid)
{
    if (valid >= 8) {
        typedef Bytes<8, 1> B;
        const B b = *reinterpret_cast<const B *>(codes + col);
        return make_uint2(b.v[0], b.v[1]);
    }
    uint2 q = make_uint2(0, 0);
    for (int i = 0; i < valid; i++) {
        const uint32_t c = codes[col + i];
        if (i < 4) q.x |= c << (8 * i); else q.y |= c << (8 * (i - 4));
    }
    return q;
}

// A matrix that is either dense or a checkpoint.
template <class T> struct Source {
    const T *x = nullptr;
    int64_t ldx = 0;
    const uint8_t *codes = nullptr, *scales = nullptr;
    int64_t ldc = 0, lds = 0;
    __host__ __device__ bool any() const { return x || codes; }
    __device__ __forceinline__ float value(int64_t row, int64_t col) const
    {
        if (x) return to_f(x[row * ldx + col]);
        return __builtin_amdgcn_cvt_f32_fp8((int)codes[row * ldc + col], 0) * pack8_unit(scales[row * lds + (col >> 5)]);
    }
};
