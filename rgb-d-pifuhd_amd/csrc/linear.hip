// Linear layers with their epilogue and their backward pass (pifu_linear, pifu_linear_backward).
//
// Every product is out[i][j] = sum_p A(i, p) B(j, p):
//   forward  y  = x w^T     A = x  [m][k]  rows along p     B = w [n][k]  rows along p
//   input    gx = dz w      A = dz [m][n]  rows along p     B = w [n][k]  rows along j
//   weights  gw = dz^T h    A = dz [m][n]  rows along i     B = h [m][k]  rows along j (dense or decoded from a checkpoint)
// One kernel, k_product, takes the operands in either order; what differs is the layout of their tiles in LDS.
#include "linear_common.h"

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// ---- the epilogue of one output chunk (8 columns of a row)
template <class T> struct Epilogue {
    int act;
    const T *bias, *residual;
    T *y, *z;
    int64_t ldr, ldy, ldz;
    uint8_t *codes, *scales;
    int64_t ldc, lds;
};

// v: the product's chunk at (row, col), `valid` columns of which exist (<= 0: none).  The four lanes of a block call it together.
template <class T> __device__ __forceinline__ void finish_chunk(const Epilogue<T> &e, int64_t row, int64_t col, int valid, float v[8])
{
    if (e.bias && valid > 0) {
        float b[8];
        load8(e.bias + col, valid, b);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += b[i];
    }
    if (e.codes) pack8_chunk(e.codes + row * e.ldc, e.scales + row * e.lds, col, valid, v);
    if (valid <= 0) return;
    if (e.z) store8(e.z + row * e.ldz + col, valid, v);
    if (e.act != PIFU_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_f(v[i], e.act);
    }
    if (e.residual) {
        float r[8];
        load8(e.residual + row * e.ldr + col, valid, r);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] += r[i];
    }
    store8(e.y + row * e.ldy + col, valid, v);
}

// ---- one operand of a product
template <class T> struct Operand {
    Source<T> m;
    int act;                 // applied to what is decoded (x_act)
};

template <class T> struct ProductArgs {
    Operand<T> a, b;
    int64_t I, J, P;
    int64_t tiles_j;
    Epilogue<T> e;
};

// geometry per element type: a tile is 128 bytes deep along p whatever the type, so both types stage 8 16-byte chunks per row
template <class T> struct Geom { static constexpr int VEC = 16 / sizeof(T), BK = 8 * VEC; };

union Chunk16 { uint4 u; uint32_t w[4]; float f[4]; bf16_t b[8]; f16_t h[8]; };
__device__ __forceinline__ float *elems(Chunk16 &c, float) { return c.f; }
__device__ __forceinline__ bf16_t *elems(Chunk16 &c, bf16_t) { return c.b; }
__device__ __forceinline__ f16_t *elems(Chunk16 &c, f16_t) { return c.h; }

// 16 bytes of row `row` from column `col` on, zero outside [0, cols)
template <class T, bool ACT> __device__ __forceinline__ uint4 stage(const Operand<T> &o, int64_t row, int64_t col, int64_t cols)
{
    constexpr int VEC = Geom<T>::VEC;
    Chunk16 c;
    c.u = make_uint4(0, 0, 0, 0);
    const int64_t left = cols - col;
    if (left <= 0) return c.u;
    T *t = elems(c, T());
    if (o.m.x) {
        const T *p = o.m.x + row * o.m.ldx + col;
        if (left >= VEC) {
            typedef Bytes<16, sizeof(T)> B;
            const B b = *reinterpret_cast<const B *>(p);
            c.u = make_uint4(b.v[0], b.v[1], b.v[2], b.v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) if (i < left) t[i] = p[i];
        }
        if (!ACT) return c.u;
        float v[8];
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = act_f((float)t[i], o.act);
#pragma unroll
        for (int i = 0; i < VEC; i++) t[i] = i < left ? (T)v[i] : (T)0.f;
        return c.u;
    }
    // a block is 32 columns and a chunk 4 or 8 at a multiple of its width: one scale per chunk
    float v[8];
    const uint8_t *q = o.m.codes + row * o.m.ldc;
    const float unit = pack8_unit(o.m.scales[row * o.m.lds + (col >> 5)]);
    const int valid = left >= 8 ? 8 : (int)left;
    unpack8_codes(load_codes(q, col, VEC == 8 ? valid : (valid > 4 ? 4 : valid)), unit, v);
#pragma unroll
    for (int i = 0; i < VEC; i++) t[i] = i < left ? (T)(ACT ? act_f(v[i], o.act) : v[i]) : (T)0.f;
    return c.u;
}

// LDS position (in elements) of a tile's chunk.  Rows along p: [row][8 chunks], the chunk index XORed with the row so that the 32
// lanes of a fragment read 32 rows' chunks from all banks.  Rows along the output: [p][R], 32-element groups XORed so that the
// four p rows of a transposed read (16-bit types) or the two halves of a wave (fp32) lie in different banks.
template <class T, int R, bool ALONG_P> __device__ __forceinline__ int lds_at(int row, int col)
{
    constexpr int VEC = Geom<T>::VEC, BK = Geom<T>::BK;
    if (ALONG_P) return row * BK + ((((col / VEC) ^ row) & 7) * VEC) + col % VEC;
    constexpr int GROUPS = R / 32;
    const int key = sizeof(T) == 2 ? row & (GROUPS < 4 ? GROUPS - 1 : 3) : (row >> 2) & (GROUPS < 2 ? 0 : 1);
    return row * R + (col ^ (key * 32));
}

template <class T> struct Frag;
template <> struct Frag<bf16_t> { typedef bf16_t V __attribute__((ext_vector_type(8))); };
template <> struct Frag<f16_t> { typedef f16_t V __attribute__((ext_vector_type(8))); };
template <> struct Frag<float> { typedef float V __attribute__((ext_vector_type(4))); };

// Fragment `step` of the 32 output indexes from r0 on: lane l holds index r0 + l % 32.  16-bit types: the 8 p from 16 step + 8 (l / 32);
// fp32: the 4 p from 8 step + 4 (l / 32), one per matrix instruction.
template <class T, int R, bool ALONG_P> __device__ __forceinline__ typename Frag<T>::V fragment(const T *lds, int r0, int step, int lane)
{
    typedef typename Frag<T>::V V;
    constexpr int VEC = Geom<T>::VEC;
    const int half = lane >> 5;
    if (ALONG_P) return *reinterpret_cast<const V *>(lds + lds_at<T, R, true>(r0 + (lane & 31), (2 * step + half) * VEC));
    if constexpr (sizeof(T) == 2) {
        // a transposed read hands 16 lanes 4 p of 16 output indexes: lane i of the 16 points at p row i / 4, columns 4 (i % 4) ..
        const int i = lane & 15, g = lane >> 4;
        const int p = 16 * step + 8 * (g >> 1) + (i >> 2), r = r0 + 16 * (g & 1) + 4 * (i & 3);
        typedef __attribute__((address_space(3))) s16x4_t L;
        union { s16x4_t s[2]; V v; } u;
        u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)(lds + lds_at<T, R, false>(p, r)));
        u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L *)(lds + lds_at<T, R, false>(p + 4, r)));
        return u.v;
    } else {
        V v;
#pragma unroll
        for (int s = 0; s < 4; s++) v[s] = lds[lds_at<T, R, false>(8 * step + 4 * half + s, r0 + (lane & 31))];
        return v;
    }
}

__device__ __forceinline__ f32x16_t mfma(Frag<bf16_t>::V a, Frag<bf16_t>::V b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16_t mfma(Frag<f16_t>::V a, Frag<f16_t>::V b, f32x16_t c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16_t mfma(Frag<float>::V a, Frag<float>::V b, f32x16_t c)
{
#pragma unroll
    for (int s = 0; s < 4; s++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], c, 0, 0, 0);
    return c;
}

// ---- the product: tiles of BM x BN outputs, one block of (BM / 64) x (BN / 64) waves each, a wave holding 64 x 64 outputs as 2 x 2
// matrix accumulators.  The next tile's chunks are fetched into registers while the present one is multiplied from LDS.
template <class T, int BM, int BN, bool A_P, bool B_P, bool ACT>
__global__ void __launch_bounds__(BM * BN / 64) k_product(const ProductArgs<T> a)
{
    constexpr int VEC = Geom<T>::VEC, BK = Geom<T>::BK, NT = BM * BN / 64;
    constexpr int AN = BM * 8 / NT, BN_ = BN * 8 / NT;
    constexpr int PITCH = 72;                                   // floats per row of a wave's epilogue slab (64 + 8: no bank conflicts)
    constexpr int LDS_A = BM * 128, LDS_B = BN * 128, LDS_E = NT / 64 * 32 * PITCH * 4;
    __shared__ __attribute__((aligned(16))) char lds[LDS_A + LDS_B > LDS_E ? LDS_A + LDS_B : LDS_E];
    T *la = reinterpret_cast<T *>(lds), *lb = reinterpret_cast<T *>(lds + LDS_A);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = wave / (BN / 64) * 64, wj = wave % (BN / 64) * 64;
    const int64_t ti = blockIdx.x / a.tiles_j, tj = blockIdx.x - ti * a.tiles_j;
    const int64_t i0 = ti * BM, j0 = tj * BN;

    f32x16_t acc[2][2];
#pragma unroll
    for (int x = 0; x < 2; x++)
#pragma unroll
        for (int y = 0; y < 2; y++) acc[x][y] = f32x16_t{};

    uint4 ra[AN], rb[BN_];
    auto fetch = [&](int64_t p0) {
#pragma unroll
        for (int it = 0; it < AN; it++) {
            const int q = it * NT + tid;
            if (A_P) {
                const int64_t row = i0 + q / 8;                 // rows past the end repeat the last one: their outputs are not stored
                ra[it] = stage<T, false>(a.a, row < a.I ? row : a.I - 1, p0 + q % 8 * VEC, a.P);
            } else {
                const int64_t p = p0 + q / (BM / VEC);
                ra[it] = p < a.P ? stage<T, false>(a.a, p, i0 + q % (BM / VEC) * VEC, a.I) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int it = 0; it < BN_; it++) {
            const int q = it * NT + tid;
            if (B_P) {
                const int64_t row = j0 + q / 8;
                rb[it] = stage<T, ACT>(a.b, row < a.J ? row : a.J - 1, p0 + q % 8 * VEC, a.P);
            } else {
                const int64_t p = p0 + q / (BN / VEC);
                rb[it] = p < a.P ? stage<T, ACT>(a.b, p, j0 + q % (BN / VEC) * VEC, a.J) : make_uint4(0, 0, 0, 0);
            }
        }
    };
    if (a.P > 0) fetch(0);
    for (int64_t p0 = 0; p0 < a.P; p0 += BK) {
        __syncthreads();
#pragma unroll
        for (int it = 0; it < AN; it++) {
            const int q = it * NT + tid;
            const int at = A_P ? lds_at<T, BM, true>(q / 8, q % 8 * VEC) : lds_at<T, BM, false>(q / (BM / VEC), q % (BM / VEC) * VEC);
            *reinterpret_cast<uint4 *>(la + at) = ra[it];
        }
#pragma unroll
        for (int it = 0; it < BN_; it++) {
            const int q = it * NT + tid;
            const int at = B_P ? lds_at<T, BN, true>(q / 8, q % 8 * VEC) : lds_at<T, BN, false>(q / (BN / VEC), q % (BN / VEC) * VEC);
            *reinterpret_cast<uint4 *>(lb + at) = rb[it];
        }
        __syncthreads();
        if (p0 + BK < a.P) fetch(p0 + BK);
#pragma unroll
        for (int step = 0; step < 4; step++) {
            typename Frag<T>::V fa[2], fb[2];
#pragma unroll
            for (int x = 0; x < 2; x++) {
                fa[x] = fragment<T, BM, A_P>(la, wi + 32 * x, step, lane);
                fb[x] = fragment<T, BN, B_P>(lb, wj + 32 * x, step, lane);
            }
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int y = 0; y < 2; y++) acc[x][y] = mfma(fa[x], fb[y], acc[x][y]);
        }
    }
    __syncthreads();

    // epilogue: 32 rows of the wave's 64 columns at a time go through its own LDS slab, so that a lane gets 8 columns of a row
    // (matrix accumulators hold one column and 16 rows per lane)
    float *slab = reinterpret_cast<float *>(lds) + wave * 32 * PITCH;
    const int64_t col = j0 + wj + (lane & 7) * 8;
    const int64_t left = a.J - col;
    const int valid = left >= 8 ? 8 : (int)left;
#pragma unroll
    for (int x = 0; x < 2; x++) {
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                slab[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * PITCH + 32 * y + (lane & 31)] = acc[x][y][r];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int it = 0; it < 4; it++) {
            const int r = it * 8 + (lane >> 3);
            const int64_t row = i0 + wi + 32 * x + r;
            float v[8];
            const f32x4_t lo = *reinterpret_cast<const f32x4_t *>(slab + r * PITCH + (lane & 7) * 8);
            const f32x4_t hi = *reinterpret_cast<const f32x4_t *>(slab + r * PITCH + (lane & 7) * 8 + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = lo[i]; v[4 + i] = hi[i]; }
            if (row < a.I) finish_chunk(a.e, row, col, valid, v);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// ---- dz = grad * act'(kept) and its column sums.  A block takes `rows` rows and TX * 8 columns: TX lanes along a row, 256 / TX rows
// at a time.  Sums run in fp32 over a block's rows and in double over the blocks, in a fixed order.
template <class T> struct SlopeArgs {
    const T *grad; int64_t ldg;
    Source<T> kept;
    T *dz;                   // [m][n] or null
    float *sums;             // [blocks][n] or null
    int64_t m, n, rows;
    int act, from_output, tx;
};

template <class T> __global__ void __launch_bounds__(256) k_slope(const SlopeArgs<T> a)
{
    __shared__ float red[256 * 8];
    const int tx = a.tx, lane = threadIdx.x & (tx - 1), ty = threadIdx.x / tx, step = 256 / tx;
    const int64_t col = ((int64_t)blockIdx.y * tx + lane) * 8, first = (int64_t)blockIdx.x * a.rows;
    const int64_t last = first + a.rows < a.m ? first + a.rows : a.m;
    const int64_t left = a.n - col;
    const int valid = left >= 8 ? 8 : (int)left;
    float sum[8] = {0.f};
    if (valid > 0) {
        for (int64_t row = first + ty; row < last; row += step) {
            float g[8];
            load8(a.grad + row * a.ldg + col, valid, g);
            if (a.act != PIFU_ACT_NONE) {
                float v[8];
                a.kept.chunk(row, col, valid, v);
#pragma unroll
                for (int i = 0; i < 8; i++) g[i] *= act_slope(v[i], a.act, a.from_output);
                if (a.dz) store8(a.dz + row * a.n + col, valid, g);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] += g[i];
        }
    }
    if (!a.sums) return;
#pragma unroll
    for (int i = 0; i < 8; i++) red[threadIdx.x * 8 + i] = sum[i];
    __syncthreads();
    for (int o = step / 2; o > 0; o >>= 1) {
        if (ty < o) {
#pragma unroll
            for (int i = 0; i < 8; i++) red[threadIdx.x * 8 + i] += red[(threadIdx.x + o * tx) * 8 + i];
        }
        __syncthreads();
    }
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < 8; i++) if (i < valid) a.sums[(int64_t)blockIdx.x * a.n + col + i] = red[threadIdx.x * 8 + i];
    }
}

template <class T> __global__ void __launch_bounds__(256) k_column_sums(const float *sums, int64_t blocks, int64_t n, T *out)
{
    __shared__ double red[256];
    const int lane = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + lane;
    double s = 0.0;
    if (col < n) for (int64_t b = ty; b < blocks; b += 8) s += (double)sums[b * n + col];
    red[threadIdx.x] = s;
    __syncthreads();
    if (ty == 0 && col < n) {
        for (int i = 1; i < 8; i++) s += red[i * 32 + lane];
        out[col] = (T)(float)s;
    }
}

// ---- host side
constexpr int64_t MAX_BLOCKS = 0x7fffffff;
constexpr int64_t MAX_WIDTH = 65535 * 256;         // n and k: 256 columns per block of a grid whose y extent is 65535 at most

struct Plan {
    int64_t dz = 0, sums = 0, total = 0;       // workspace: offsets, bytes
    int64_t sum_blocks = 0, sum_rows = 0;
    int tx = 1;
};

Plan plan_backward(const pifu_linear_grad_args &g)
{
    Plan p;
    int64_t at = 0;
    if (g.act != PIFU_ACT_NONE && (g.gx || g.gw)) { p.dz = at; at += round_up(g.m * g.n * pifu_elem_bytes(g.dtype), 256); }
    while (p.tx < 32 && p.tx * 8 < g.n) p.tx *= 2;
    const int64_t step = 256 / p.tx;
    p.sum_blocks = g.m < step * 256 ? (g.m + step - 1) / step : 256;
    if (p.sum_blocks < 1) p.sum_blocks = 1;
    p.sum_rows = round_up((g.m + p.sum_blocks - 1) / p.sum_blocks, step);
    if (p.sum_rows < 1) p.sum_rows = 1;
    p.sum_blocks = (g.m + p.sum_rows - 1) / p.sum_rows;
    if (p.sum_blocks < 1) p.sum_blocks = 1;
    if (g.gb) { p.sums = at; at += round_up(p.sum_blocks * g.n * 4, 256); }
    p.total = at;
    return p;
}

template <class T, bool A_P, bool B_P, bool ACT> int product(const ProductArgs<T> &args, hipStream_t st)
{
    ProductArgs<T> a = args;
    a.tiles_j = (a.J + 127) / 128;
    const int64_t blocks = (a.I + 127) / 128 * a.tiles_j;
    PIFU_REQUIRE(blocks <= MAX_BLOCKS, PIFU_ERR_INVALID, "a product of %lld x %lld outputs is more than one launch can hold",
                 (long long)a.I, (long long)a.J);
    PIFU_LAUNCH((k_product<T, 128, 128, A_P, B_P, ACT>), dim3((unsigned)blocks), dim3(256), 0, st, &a);
    return PIFU_OK;
}

template <class T> int forward(const pifu_linear_args &g, hipStream_t st)
{
    ProductArgs<T> a{};
    a.a.m.x = (const T *)g.x; a.a.m.ldx = g.ldx;
    a.b.m.x = (const T *)g.w; a.b.m.ldx = g.ldw;
    a.I = g.m; a.J = g.n; a.P = g.k;
    a.e.act = g.act;
    a.e.bias = (const T *)g.bias;
    a.e.residual = (const T *)g.residual; a.e.ldr = g.ldr;
    a.e.y = (T *)g.y; a.e.ldy = g.ldy;
    a.e.z = (T *)g.z; a.e.ldz = g.ldz;
    a.e.codes = g.z8.codes; a.e.ldc = g.z8.ld; a.e.scales = g.z8.scales; a.e.lds = g.z8.ld_scales;
    return product<T, true, true, false>(a, st);
}

template <class T> Source<T> source(const void *x, int64_t ldx, const pifu_packed8 &p)
{
    Source<T> s;
    s.x = (const T *)x; s.ldx = ldx;
    if (!x) { s.codes = p.codes; s.ldc = p.ld; s.scales = p.scales; s.lds = p.ld_scales; }
    return s;
}

template <class T> int backward(const pifu_linear_grad_args &g, char *ws, hipStream_t st)
{
    const Plan p = plan_backward(g);
    const bool slope = g.act != PIFU_ACT_NONE;
    T *dz = slope && (g.gx || g.gw) ? (T *)(ws + p.dz) : nullptr;
    if (dz || g.gb) {
        SlopeArgs<T> s{};
        s.grad = (const T *)g.grad; s.ldg = g.ldg;
        if (slope) s.kept = source<T>(g.z, g.ldz, g.z8);
        s.dz = dz;
        s.sums = g.gb ? (float *)(ws + p.sums) : nullptr;
        s.m = g.m; s.n = g.n; s.rows = p.sum_rows; s.act = g.act; s.from_output = g.from_output; s.tx = p.tx;
        const int64_t wide = (g.n + p.tx * 8 - 1) / (p.tx * 8);
        PIFU_LAUNCH(k_slope<T>, dim3((unsigned)p.sum_blocks, (unsigned)wide), dim3(256), 0, st, &s);
        if (g.gb) {
            const float *sums = s.sums;
            int64_t blocks = p.sum_blocks, n = g.n;
            T *out = (T *)g.gb;
            PIFU_LAUNCH(k_column_sums<T>, dim3((unsigned)((n + 31) / 32)), dim3(256), 0, st, &sums, &blocks, &n, &out);
        }
    }
    ProductArgs<T> a{};
    a.a.m.x = dz ? dz : (const T *)g.grad;
    a.a.m.ldx = dz ? g.n : g.ldg;
    if (g.gx && g.m > 0) {
        a.b.m.x = (const T *)g.w; a.b.m.ldx = g.ldw;
        a.I = g.m; a.J = g.k; a.P = g.n;
        a.e.y = (T *)g.gx; a.e.ldy = g.ldgx;
        const int rc = product<T, true, false, false>(a, st);
        if (rc) return rc;
    }
    if (g.gw) {
        a.b.m = source<T>(g.x, g.ldx, g.x8);
        a.b.act = g.x_act;
        a.I = g.n; a.J = g.k; a.P = g.m;
        a.e.y = (T *)g.gw; a.e.ldy = g.ldgw;
        const int rc = g.x_act == PIFU_ACT_NONE ? product<T, false, false, false>(a, st) : product<T, false, false, true>(a, st);
        if (rc) return rc;
    }
    return PIFU_OK;
}

bool act_ok(int act) { return act >= PIFU_ACT_NONE && act <= PIFU_ACT_SILU; }

int check_matrix(const char *name, const char *what, int dtype, const void *p, int64_t ld, int64_t cols)
{
    PIFU_REQUIRE(ld >= cols, PIFU_ERR_INVALID, "%s: the row pitch of %s (%lld) is smaller than its row (%lld)", name, what, (long long)ld,
                 (long long)cols);
    PIFU_REQUIRE((uintptr_t)p % pifu_elem_bytes(dtype) == 0, PIFU_ERR_INVALID, "%s: %s is not aligned to its element type", name, what);
    return PIFU_OK;
}

int check_packed(const char *name, const char *what, const pifu_packed8 &p, int64_t cols)
{
    PIFU_REQUIRE(p.scales && p.ld >= cols && p.ld_scales >= (cols + 31) / 32, PIFU_ERR_INVALID,
                 "%s: %s has no scales or a row pitch smaller than its row", name, what);
    return PIFU_OK;
}

#define PIFU_CHECKED(call) do { const int rc_ = (call); if (rc_) return rc_; } while (0)

int check_forward(pifu_ctx *ctx, const pifu_linear_args *g)
{
    const char *name = "pifu_linear";
    PIFU_REQUIRE(ctx && g, PIFU_ERR_INVALID, "%s: null argument", name);
    PIFU_REQUIRE(pifu_dtype_ok(g->dtype), PIFU_ERR_INVALID, "%s: dtype %d is not PIFU_F32, PIFU_BF16 or PIFU_F16", name, g->dtype);
    PIFU_REQUIRE(act_ok(g->act), PIFU_ERR_INVALID, "%s: unknown activation %d", name, g->act);
    PIFU_REQUIRE(g->m >= 0 && g->n >= 1 && g->k >= 1 && g->n <= MAX_WIDTH && g->k <= MAX_WIDTH, PIFU_ERR_INVALID, "%s: bad shape m %lld, n %lld, k %lld", name, (long long)g->m,
                 (long long)g->n, (long long)g->k);
    if (g->m == 0) return PIFU_OK;
    PIFU_REQUIRE(g->x && g->w && g->y, PIFU_ERR_INVALID, "%s: null matrix", name);
    PIFU_CHECKED(check_matrix(name, "x", g->dtype, g->x, g->ldx, g->k));
    PIFU_CHECKED(check_matrix(name, "w", g->dtype, g->w, g->ldw, g->k));
    PIFU_CHECKED(check_matrix(name, "y", g->dtype, g->y, g->ldy, g->n));
    if (g->bias) PIFU_CHECKED(check_matrix(name, "bias", g->dtype, g->bias, g->n, g->n));
    if (g->residual) PIFU_CHECKED(check_matrix(name, "residual", g->dtype, g->residual, g->ldr, g->n));
    if (g->z) PIFU_CHECKED(check_matrix(name, "z", g->dtype, g->z, g->ldz, g->n));
    if (g->z8.codes) PIFU_CHECKED(check_packed(name, "z8", g->z8, g->n));
    return PIFU_OK;
}

int check_backward(pifu_ctx *ctx, const pifu_linear_grad_args *g)
{
    const char *name = "pifu_linear_backward";
    PIFU_REQUIRE(ctx && g, PIFU_ERR_INVALID, "%s: null argument", name);
    PIFU_REQUIRE(pifu_dtype_ok(g->dtype), PIFU_ERR_INVALID, "%s: dtype %d is not PIFU_F32, PIFU_BF16 or PIFU_F16", name, g->dtype);
    PIFU_REQUIRE(act_ok(g->act) && act_ok(g->x_act), PIFU_ERR_INVALID, "%s: unknown activation %d / %d", name, g->act, g->x_act);
    PIFU_REQUIRE(!g->from_output || g->act <= PIFU_ACT_TANH, PIFU_ERR_INVALID,
                 "%s: the derivative of this activation does not follow from its output: keep the pre-activation", name);
    PIFU_REQUIRE(g->m >= 0 && g->n >= 1 && g->k >= 1 && g->n <= MAX_WIDTH && g->k <= MAX_WIDTH, PIFU_ERR_INVALID, "%s: bad shape m %lld, n %lld, k %lld", name, (long long)g->m,
                 (long long)g->n, (long long)g->k);
    if (g->gx) PIFU_CHECKED(check_matrix(name, "gx", g->dtype, g->gx, g->ldgx, g->k));
    if (g->gw) PIFU_CHECKED(check_matrix(name, "gw", g->dtype, g->gw, g->ldgw, g->k));
    if (g->gb) PIFU_CHECKED(check_matrix(name, "gb", g->dtype, g->gb, g->n, g->n));
    if (g->m == 0) return PIFU_OK;
    PIFU_REQUIRE(g->grad, PIFU_ERR_INVALID, "%s: null gradient", name);
    PIFU_CHECKED(check_matrix(name, "grad", g->dtype, g->grad, g->ldg, g->n));
    if (g->act != PIFU_ACT_NONE) {
        PIFU_REQUIRE(g->z || g->z8.codes, PIFU_ERR_INVALID, "%s: an activation's derivative needs what the forward pass kept", name);
        if (g->z) PIFU_CHECKED(check_matrix(name, "z", g->dtype, g->z, g->ldz, g->n));
        else PIFU_CHECKED(check_packed(name, "z8", g->z8, g->n));
    }
    if (g->gw) {
        PIFU_REQUIRE(g->x || g->x8.codes, PIFU_ERR_INVALID, "%s: the gradient of w needs the input", name);
        if (g->x) PIFU_CHECKED(check_matrix(name, "x", g->dtype, g->x, g->ldx, g->k));
        else PIFU_CHECKED(check_packed(name, "x8", g->x8, g->k));
    }
    if (g->gx) {
        PIFU_REQUIRE(g->w, PIFU_ERR_INVALID, "%s: the gradient of x needs w", name);
        PIFU_CHECKED(check_matrix(name, "w", g->dtype, g->w, g->ldw, g->k));
    }
    return PIFU_OK;
}

int check_workspace(const char *name, void *workspace, int64_t bytes, int64_t needed)
{
    PIFU_REQUIRE(bytes >= needed && (!needed || workspace), PIFU_ERR_NOMEM, "%s: the workspace has %lld bytes, %lld are needed", name,
                 (long long)bytes, (long long)needed);
    PIFU_REQUIRE((uintptr_t)workspace % 16 == 0, PIFU_ERR_INVALID, "%s: the workspace is not 16-byte aligned", name);
    return PIFU_OK;
}

}  // namespace

extern "C" int64_t pifu_linear_workspace(pifu_ctx *ctx, const pifu_linear_args *args)
{
    const int rc = check_forward(ctx, args);
    return rc ? rc : 0;
}

extern "C" int pifu_linear(pifu_ctx *ctx, const pifu_linear_args *args, void *workspace, int64_t workspace_bytes, pifu_stream stream)
{
    PIFU_CHECKED(check_forward(ctx, args));
    if (args->m == 0) return PIFU_OK;
    PIFU_CHECKED(check_workspace("pifu_linear", workspace, workspace_bytes, 0));
    PifuDeviceGuard guard(ctx->device);
    PIFU_HIP(guard.err);
    hipStream_t st = (hipStream_t)stream;
    if (args->dtype == PIFU_F32) return forward<float>(*args, st);
    if (args->dtype == PIFU_BF16) return forward<bf16_t>(*args, st);
    return forward<f16_t>(*args, st);
}

extern "C" int64_t pifu_linear_backward_workspace(pifu_ctx *ctx, const pifu_linear_grad_args *args)
{
    const int rc = check_backward(ctx, args);
    return rc ? rc : plan_backward(*args).total;
}

extern "C" int pifu_linear_backward(pifu_ctx *ctx, const pifu_linear_grad_args *args, void *workspace, int64_t workspace_bytes,
                                    pifu_stream stream)
{
    PIFU_CHECKED(check_backward(ctx, args));
    PIFU_CHECKED(check_workspace("pifu_linear_backward", workspace, workspace_bytes, plan_backward(*args).total));
    PifuDeviceGuard guard(ctx->device);
    PIFU_HIP(guard.err);
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
    if (args->dtype == PIFU_F32) return backward<float>(*args, ws, st);
    if (args->dtype == PIFU_BF16) return backward<bf16_t>(*args, ws, st);
    return backward<f16_t>(*args, ws, st);
}
