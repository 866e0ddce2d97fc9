// 8-bit checkpoints of activations as operators of their own: pifu_pack8 / pifu_unpack8.  (linear.hip packs in the epilogue of a
// product and decodes inside the backward pass; both use the codec of linear_common.h.)
// Elementwise: bound by the bytes moved, sizeof(T) + 1 + 1/32 per element.  A lane holds 8 consecutive columns, four lanes a block
// that shares a scale: the block's maximum is two lane exchanges, no shared memory.
#include "linear_common.h"

namespace {

template <class T> struct Pack8Args {
    const T *x; T *y;
    int64_t ldx, rows, cols, chunks;      // chunks: lanes per row, a multiple of 4 (whole blocks)
    uint8_t *codes, *scales;
    int64_t ldc, lds;
    RowCut cut;
};

// A lane takes a chunk at a time, blocks take them in turn: 200000 x 1024 bf16 in 149 us, 4.2 TB/s.  (Four rows of a lane at once, as
// below: 3 % more, and 5000 x 385 fp32 in 6.9 us instead of 4.0.)
template <class T> __global__ void __launch_bounds__(256) k_pack8(const Pack8Args<T> a)
{
    const int64_t total = a.rows * a.chunks;
    // chunks is a multiple of 4 and the stride of 256: the four lanes of a block stay together in every pass of the loop
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / a.chunks, col = (i - row * a.chunks) * 8;
        const int64_t left = a.cols - col;
        const int valid = left >= 8 ? 8 : (int)left;
        float v[8] = {0.f};
        if (valid > 0) load8(a.x + row * a.ldx + col, valid, v);
        pack8_chunk(a.codes + row * a.ldc, a.scales + row * a.lds, col, valid, v);
    }
}

// Four rows of a lane at a time, their loads in flight together: 200000 x 1024 bf16 in 107 us, 5.8 TB/s (a chunk at a time: 178 us).
template <class T> __global__ void __launch_bounds__(256) k_unpack8(const Pack8Args<T> a)
{
    const int lane = threadIdx.x & (a.cut.tx - 1), step = 256 / a.cut.tx;
    const int64_t col = ((int64_t)blockIdx.x * a.cut.tx + lane) * 8, left = a.cols - col;
    const int valid = left >= 8 ? 8 : (int)left;
    if (valid <= 0) return;
    auto rows = [&](int64_t row, auto count, auto whole) {
        constexpr int N = decltype(count)::value;
        const int n = decltype(whole)::value ? 8 : valid;
        uint2 q[N];
        uint32_t scale[N];
#pragma unroll
        for (int u = 0; u < N; u++) {
            q[u] = load_codes(a.codes + (row + u * step) * a.ldc, col, n);
            scale[u] = a.scales[(row + u * step) * a.lds + (col >> 5)];
        }
#pragma unroll
        for (int u = 0; u < N; u++) {
            float v[8];
            unpack8_codes(q[u], pack8_unit(scale[u]), v);
            store8(a.y + (row + u * step) * a.ldx + col, n, v);
        }
    };
    each_row(a.cut.tx, a.cut.rows, blockIdx.y, a.rows, valid, rows);
}

constexpr int64_t PACK8_BLOCKS = 256 * 32;       // enough to fill the chip several times over; k_pack8 loops

template <class T> int run(bool pack, void *x, int64_t ldx, int64_t rows, int64_t cols, const pifu_packed8 &p, hipStream_t st)
{
    Pack8Args<T> a{(const T *)x, (T *)x, ldx, rows, cols, (cols + 31) / 32 * 4, p.codes, p.scales, p.ld, p.ld_scales,
                   RowCut(rows, cols, 65535)};
    const int64_t blocks = (rows * a.chunks + 255) / 256;
    if (pack) PIFU_LAUNCH(k_pack8<T>, dim3((unsigned)(blocks < PACK8_BLOCKS ? blocks : PACK8_BLOCKS)), dim3(256), 0, st, &a);
    else PIFU_LAUNCH(k_unpack8<T>, dim3((unsigned)a.cut.wide, (unsigned)a.cut.blocks), dim3(256), 0, st, &a);
    return PIFU_OK;
}

int checked(const char *name, pifu_ctx *ctx, int dtype, const void *x, int64_t ldx, int64_t rows, int64_t cols, const pifu_packed8 *p,
            bool pack, hipStream_t st)
{
    PIFU_REQUIRE(ctx && p, PIFU_ERR_INVALID, "%s: null argument", name);
    PIFU_REQUIRE(pifu_dtype_ok(dtype), PIFU_ERR_INVALID, "%s: dtype %d is not PIFU_F32, PIFU_BF16 or PIFU_F16", name, dtype);
    PIFU_REQUIRE(rows >= 0 && cols >= 1, PIFU_ERR_INVALID, "%s: bad shape %lld x %lld", name, (long long)rows, (long long)cols);
    if (rows == 0) return PIFU_OK;
    PIFU_REQUIRE(x && p->codes && p->scales, PIFU_ERR_INVALID, "%s: null matrix", name);
    PIFU_REQUIRE(ldx >= cols && p->ld >= cols && p->ld_scales >= (cols + 31) / 32, PIFU_ERR_INVALID,
                 "%s: a row pitch is smaller than its row (%lld columns: ldx %lld, ld %lld, ld_scales %lld)", name, (long long)cols,
                 (long long)ldx, (long long)p->ld, (long long)p->ld_scales);
    // k_unpack8 has its blocks of columns along x, at least 512 columns each in rows this long; k_pack8 loops
    PIFU_REQUIRE(cols <= (pack ? (int64_t)0x7fffffff * 256 : MAX_BLOCKS * 512), PIFU_ERR_INVALID,
                 "%s: rows of %lld columns are more than one launch can hold", name, (long long)cols);
    PIFU_REQUIRE((uintptr_t)x % pifu_elem_bytes(dtype) == 0, PIFU_ERR_INVALID, "%s: x is not aligned to its element type", name);
    PifuDeviceGuard guard(ctx->device);
    PIFU_HIP(guard.err);
    void *v = const_cast<void *>(x);
    if (dtype == PIFU_F32) return run<float>(pack, v, ldx, rows, cols, *p, st);
    if (dtype == PIFU_BF16) return run<bf16_t>(pack, v, ldx, rows, cols, *p, st);
    return run<f16_t>(pack, v, ldx, rows, cols, *p, st);
}

}  // namespace

extern "C" int pifu_pack8(pifu_ctx *ctx, int dtype, const void *x, int64_t ldx, int64_t rows, int64_t cols, const pifu_packed8 *out,
                          pifu_stream stream)
{
    return checked("pifu_pack8", ctx, dtype, x, ldx, rows, cols, out, true, (hipStream_t)stream);
}

extern "C" int pifu_unpack8(pifu_ctx *ctx, int dtype, const pifu_packed8 *in, int64_t rows, int64_t cols, void *x, int64_t ldx,
                            pifu_stream stream)
{
    return checked("pifu_unpack8", ctx, dtype, x, ldx, rows, cols, in, false, (hipStream_t)stream);
}
