// Linear layers with their epilogue and their backward pass (pifu_linear, pifu_linear_backward).
//
// Every product is out[i][j] = sum_p A(i, p) B(j, p):
//   forward  y  = x w^T     A = x  [m][k]  rows along p     B = w [n][k]  rows along p
//   input    gx = dz w      A = dz [m][n]  rows along p     B = w [n][k]  rows along j
//   weights  gw = dz^T h    A = dz [m][n]  rows along i     B = h [m][k]  rows along j (decoded first where x is a checkpoint)
// One kernel, k_product, takes the operands in either order; what differs is the layout of their tiles in LDS.  16-bit types: dz and h
// may be held as two halves each (HALVES_MOST), or gw be taken from scaled fp16 (k_column_max).  Up to 8 rows of a
// forward pass (k_few_rows) and up to 4 outputs of a backward pass (k_narrow) are bound by bytes and have kernels without matrix
// instructions.
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

// v: the product's chunks at rows row, row + step, .. and columns col .. col + 7, `valid` of which exist (<= 0: none).  The four lanes
// of a block of columns call it together.  N rows at a time: each stage runs over all of them, so that their memory accesses and
// chains of arithmetic overlap.
template <class T, int N>
__device__ __forceinline__ void finish_chunks(const Epilogue<T> &e, const float bias[8], int64_t row, int step, int64_t rows,
                                              int64_t col, int valid, float v[N][8])
{
    float r[N][8];
    if (e.residual) {
#pragma unroll
        for (int u = 0; u < N; u++)
            if (row + u * step < rows && valid > 0) load8(e.residual + (row + u * step) * e.ldr + col, valid, r[u]);
    }
#pragma unroll
    for (int u = 0; u < N; u++)
#pragma unroll
        for (int i = 0; i < 8; i++) v[u][i] += bias[i];
    if (e.codes) {
#pragma unroll
        for (int u = 0; u < N; u++)
            if (row + u * step < rows)
                pack8_chunk(e.codes + (row + u * step) * e.ldc, e.scales + (row + u * step) * e.lds, col, valid, v[u]);
    }
    if (valid <= 0) return;
    if (e.z) {
#pragma unroll
        for (int u = 0; u < N; u++)
            if (row + u * step < rows) store8(e.z + (row + u * step) * e.ldz + col, valid, v[u]);
    }
    act_all<8 * N>(v[0], e.act);
    if (e.residual) {
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < 8; i++) v[u][i] += r[u][i];
    }
#pragma unroll
    for (int u = 0; u < N; u++)
        if (row + u * step < rows) store8(e.y + (row + u * step) * e.ldy + col, valid, v[u]);
}

template <class T> __device__ __forceinline__ void load_bias(const Epilogue<T> &e, int64_t col, int valid, float b[8])
{
#pragma unroll
    for (int i = 0; i < 8; i++) b[i] = 0.f;
    if (e.bias && valid > 0) load8(e.bias + col, valid, b);
}

// ---- one operand of a product: a dense matrix
template <class T> struct Operand {
    const T *x;
    int64_t ld;
    int64_t cols;            // elements of a row that may be read (at least its extent)
};

// T: type of the operands, O: of the outputs
template <class T, class O = T> struct ProductArgs {
    Operand<T> a, b;
    int64_t I, J, P;
    // The sum over p is run through `runs` times.  In the second run A's elements lie half_a further, in the last one B's half_b
    // further (0: an operand that is whole): a b = a1 b1 + a2 b1 + a1 b2; a2 b2 is as small as what a2 and b2 were rounded by.
    int runs, half_a, half_b;
    int64_t tiles_i, tiles_j;
    // Tiles 0 .. whole - 1 (in the order of tile_at) belong to one block each.  The others, which would leave most of the chip idle, are
    // split along p: part s of one of them multiplies p tiles s * per .. (s + 1) * per - 1 and leaves its sums in part[(tile - whole) *
    // splits + s][BM][BN]; k_join adds them up in order and finishes.
    int64_t whole, splits, per;
    float *part;
    Epilogue<O> e;
    const int *exp_i, *exp_j;          // T != O: rows of A and B were multiplied by 2^exp[index]
};

// the sums of scaled operands, N rows of a chunk of columns: scaled back
template <class T, class O, int N> __device__ __forceinline__ void unscale(const ProductArgs<T, O> &a, int64_t row, int step, int64_t col,
                                                                           int valid, float v[N][8])
{
    if constexpr (!std::is_same<T, O>::value) {
        int ej[8];
#pragma unroll
        for (int i = 0; i < 8; i++) ej[i] = i < valid ? a.exp_j[col + i] : 0;
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int ei = row + u * step < a.I ? a.exp_i[row + u * step] : 0;
#pragma unroll
            for (int i = 0; i < 8; i++) v[u][i] = __builtin_amdgcn_ldexpf(v[u][i], -(ei + ej[i]));
        }
    }
}

// geometry per element type: a tile is 128 bytes deep along p whatever the type, so both types stage 8 16-byte chunks per row
template <class T> struct Geom { static constexpr int VEC = 16 / sizeof(T), BK = 8 * VEC; };

union Chunk16 { uint4 u; float f[4]; bf16_t b[8]; f16_t h[8]; };
__device__ __forceinline__ float *elems(Chunk16 &c, float) { return c.f; }
__device__ __forceinline__ bf16_t *elems(Chunk16 &c, bf16_t) { return c.b; }
__device__ __forceinline__ f16_t *elems(Chunk16 &c, f16_t) { return c.h; }

// 16 bytes of a row from p on, `left` elements of which exist (the rest is zero)
template <class T> __device__ __forceinline__ uint4 load16(const T *p)
{
    typedef Bytes<16, sizeof(T)> B;
    const B b = *reinterpret_cast<const B *>(p);
    return make_uint4(b.v[0], b.v[1], b.v[2], b.v[3]);
}
template <class T> __device__ __forceinline__ uint4 load16(const T *p, int64_t left)
{
    constexpr int VEC = Geom<T>::VEC;
    if (left >= VEC) return load16(p);
    Chunk16 c;
    c.u = make_uint4(0, 0, 0, 0);
    T *t = elems(c, T());
#pragma unroll
    for (int i = 0; i < VEC; i++) if (i < left) t[i] = p[i];
    return c.u;
}

// LDS position (in elements) of a tile's chunk.  Rows along p: [row][8 chunks], the chunk index XORed with the row so that the 32
// lanes of a fragment read 32 rows' chunks from all banks.  Rows along the output: [p][R], 32-element groups XORed so that the
// four p rows of a transposed read (16-bit types) or the two halves of a wave (fp32) lie in different banks.
template <class T, int R> __device__ __forceinline__ int group_key(int p)
{
    constexpr int GROUPS = R / 32;
    return sizeof(T) == 2 ? p & (GROUPS < 4 ? GROUPS - 1 : 3) : (p >> 2) & (GROUPS < 2 ? 0 : 1);
}
template <class T, int R, bool ALONG_P> __device__ __forceinline__ int lds_at(int row, int col)
{
    constexpr int VEC = Geom<T>::VEC, BK = Geom<T>::BK;
    if (ALONG_P) return row * BK + ((((col / VEC) ^ row) & 7) * VEC) + col % VEC;
    return row * R + (col ^ (group_key<T, R>(row) * 32));
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

__device__ __forceinline__ f32x16_t mfma(Frag<bf16_t>::V a, Frag<bf16_t>::V b, f32x16_t c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma(Frag<f16_t>::V a, Frag<f16_t>::V b, f32x16_t c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma(Frag<float>::V a, Frag<float>::V b, f32x16_t c)
{
#pragma unroll
    for (int s = 0; s < 4; s++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], b[s], c, 0, 0, 0);
    return c;
}

typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_ptr_t;

// One LDS-DMA piece: lane i's 16 bytes from `base` + voff land at LDS address lds_addr + 16 i.  voff >= `records` reads as zeros.
// In asm because the compiler orders every later LDS read behind a transfer that it knows about; the kernel waits for them
// itself (dma_wait, before the barrier that publishes the tile).  s_nop: the scalar operands may come fresh from a vector
// instruction (5 wait states before a memory instruction reads them), M0 from the line above (1).  The compiler owns M0.
__device__ __forceinline__ void lds_dma(unsigned lds_addr, unsigned voff, u32x4_t rsrc)
{
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\t"
                 "s_mov_b32 m0, %1\n\t"
                 "s_nop 2\n\t"
                 "buffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
                 "s_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds_addr), "v"(voff), "s"(rsrc)
                 : "memory");
}
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One operand's way into LDS.  R output indexes per tile, NT threads; ALONG_P: which axis of memory is contiguous.  DMA: whole aligned
// chunks by LDS-DMA; otherwise through registers, any alignment and extent.
template <class T, int R, int NT, bool ALONG_P, bool DMA> struct Loader {
    static constexpr int VEC = Geom<T>::VEC, BK = Geom<T>::BK, N = R * 8 / NT, PER = R / VEC;      // PER: chunks per p row
    const T *x;
    int64_t ld, r0, extent, P;         // first output index of the tile, number of output indexes, depth
    uint4 reg[DMA ? 1 : N];
    unsigned voff[DMA ? N : 1];
    unsigned lds_base, to;
    u32x4_t rsrc;
    bool zero;
    int chunk;                         // DMA along p: this lane's first column of the tile

    __device__ __forceinline__ void init(const Operand<T> &o, int64_t first, int64_t ext, int64_t p, const T *lds, int tid)
    {
        x = o.x; ld = o.ld; r0 = first; extent = ext; P = p;
        if constexpr (DMA) {
            const int lane = tid & 63, wave = tid >> 6;
            lds_base = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(lds_ptr_t)(lds) + wave * 1024u);
            chunk = ((lane & 7) ^ ((lane >> 3) & 7)) * VEC;
#pragma unroll
            for (int it = 0; it < N; it++) {
                const int q = it * NT + tid;
                if (ALONG_P) {
                    const int64_t row = r0 + q / 8;             // rows past the end repeat the last one: their outputs are not stored
                    voff[it] = (unsigned)(((row < extent ? row : extent - 1) - r0) * ld + chunk) * (unsigned)sizeof(T);
                } else {
                    const int k = q / PER;
                    int64_t col = q % PER * VEC ^ (group_key<T, R>(k) * 32);
                    if (r0 + col >= o.cols) col = o.cols - VEC - r0;     // (repeats the last chunk, likewise not stored)
                    voff[it] = (unsigned)(k * ld + col) * (unsigned)sizeof(T);
                }
            }
        }
    }
    // Starts the tile at p0 (if `there` is one) of the operand's half at `half` on its way: into registers here, or, DMA, piece by piece
    // (dma()) into LDS at `offset`.
    __device__ __forceinline__ void fetch(int64_t p0, int64_t half, bool there, unsigned offset, int tid)
    {
        const T *const x = this->x + half;
        if constexpr (DMA) {
            const uint64_t at = (uint64_t)(ALONG_P ? x + r0 * ld + p0 : x + p0 * ld + r0);
            unsigned records = DMA_SPAN;
            if (!ALONG_P) {
                // p rows from P on lie past the end of the matrix: they read as zeros
                const int64_t rest = ((P - p0) * ld - r0) * (int64_t)sizeof(T);
                if (rest < (int64_t)DMA_SPAN) records = (unsigned)rest;
            }
            if (!there) records = 0;
            rsrc = u32x4_t{(unsigned)at, (unsigned)(at >> 32) & 0xffffu, records, 0x00020000u};
            to = lds_base + offset;
            zero = ALONG_P && p0 + chunk >= P;
        } else if (there) {
            const bool whole = p0 + BK <= P && (ALONG_P || r0 + R <= extent);
#pragma unroll
            for (int it = 0; it < N; it++) {
                const int q = it * NT + tid;
                if (ALONG_P) {
                    const int64_t row = r0 + q / 8;
                    const T *at = x + (row < extent ? row : extent - 1) * ld + p0 + q % 8 * VEC;
                    reg[it] = whole ? load16(at) : load16(at, P - p0 - q % 8 * VEC);
                } else {
                    const int64_t k = p0 + q / PER;
                    const T *at = x + k * ld + r0 + q % PER * VEC;
                    reg[it] = whole ? load16(at) : load16(at, k < P ? extent - r0 - q % PER * VEC : 0);
                }
            }
        }
    }
    __device__ __forceinline__ void dma(int it) const
    {
        if constexpr (DMA) lds_dma(to + it * (NT * 16u), zero ? DMA_SPAN + 1u : voff[it], rsrc);
    }
    // puts what fetch() brought into registers into the tile at `lds`
    __device__ __forceinline__ void store(T *lds, int tid) const
    {
        if constexpr (!DMA) {
#pragma unroll
            for (int it = 0; it < N; it++) {
                const int q = it * NT + tid;
                const int at = ALONG_P ? lds_at<T, R, true>(q / 8, q % 8 * VEC) : lds_at<T, R, false>(q / PER, q % PER * VEC);
                *reinterpret_cast<uint4 *>(lds + at) = reg[it];
            }
        }
    }
};

// Tile t in the order in which blocks take them: groups of 8 row tiles walked column by column, so that the tiles in flight at one
// time share rows and columns in the L2s.
__device__ __forceinline__ void tile_at(int64_t t, int64_t tiles_i, int64_t tiles_j, int64_t *ti, int64_t *tj)
{
    const int64_t group = t / (8 * tiles_j), in = t - group * 8 * tiles_j;
    const int64_t height = tiles_i - group * 8 < 8 ? tiles_i - group * 8 : 8;
    *tj = in / height;
    *ti = group * 8 + in - *tj * height;
}

// Blocks go to the 8 XCDs in turn (block b to XCD b % 8), each with an L2 of its own: every XCD gets a contiguous run of [0, total).
__device__ __forceinline__ int64_t xcd_run(int64_t b, int64_t total)
{
    const int64_t xcd = b & 7, each = total >> 3, more = total & 7;
    return xcd * each + (xcd < more ? xcd : more) + (b >> 3);
}

// ---- the product: tiles of BM x BN outputs, a wave holding WM x WN of them.  Bound by the matrix instructions in large products:
// 16384 x 4096 x 4096 bf16 forward with gelu and checkpoint 572 us (962 TFLOP/s), gx 493 us (1116), gw from scaled fp16 485 us (1133),
// 4 % less or more from box to box; a library product of the same size in bf16 alone reaches 1231, 1100 and 954 TFLOP/s.  Small ones
// wait for their transfers: with its join, 5000 x 1024 x 512 fp32 runs at 85 (gx) and 89 (gw) of 154 TFLOP/s, 5000 x 769 x 256 fp32 at
// 54 (64 without).
// Tiles are double-buffered in LDS with one barrier per tile: while tile t is multiplied, tile t + 1 lands in the other buffer.
// Fragments are fetched one step ahead of the matrix instructions that use them, across the barrier too, which stands before the last
// step's instructions.
// HALVES (runs > 1) is a variant of its own: the offsets of the halves would cost the others 4 to 10 %.
template <class T, class O, int BM, int BN, int WM, int WN, bool A_P, bool B_P, bool A_DMA, bool B_DMA, bool HALVES>
__global__ void __launch_bounds__(BM / WM * (BN / WN) * 64) k_product(const ProductArgs<T, O> a)
{
    constexpr int BK = Geom<T>::BK, NT = BM / WM * (BN / WN) * 64, MI = WM / 32, NJ = WN / 32;
    constexpr int PITCH = WN + 8;                               // floats per row of a wave's epilogue slab: no bank conflicts
    constexpr int TILE_A = BM * 128, TILE = TILE_A + BN * 128, SLABS = NT / 64 * 32 * PITCH * 4;
    __shared__ __attribute__((aligned(1024))) char lds[2 * TILE > SLABS ? 2 * TILE : SLABS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;
    const int64_t depth = (a.P + BK - 1) / BK;
    int64_t ti, tj, first = 0, last = HALVES ? depth * a.runs : depth;      // p tiles of this block
    float *part = nullptr;
    if (blockIdx.x < a.whole) {
        tile_at(xcd_run(blockIdx.x, a.whole), a.tiles_i, a.tiles_j, &ti, &tj);
    } else {
        const int64_t rest = a.tiles_i * a.tiles_j - a.whole;
        const int64_t b = xcd_run(blockIdx.x - a.whole, rest * a.splits);
        const int64_t s = b / rest, t = b - s * rest;           // (neighbours share their p range)
        tile_at(a.whole + t, a.tiles_i, a.tiles_j, &ti, &tj);
        if (a.splits > 1) {
            first = s * a.per;
            last = first + a.per < last ? first + a.per : last;
            part = a.part + (t * a.splits + s) * (BM * BN);
        }
    }
    const int64_t i0 = ti * BM, j0 = tj * BN;

    f32x16_t acc[MI][NJ];
#pragma unroll
    for (int x = 0; x < MI; x++)
#pragma unroll
        for (int y = 0; y < NJ; y++) acc[x][y] = f32x16_t{};

    Loader<T, BM, NT, A_P, A_DMA> la;
    Loader<T, BN, NT, B_P, B_DMA> lb;
    la.init(a.a, i0, a.I, a.P, reinterpret_cast<T *>(lds), tid);
    lb.init(a.b, j0, a.J, a.P, reinterpret_cast<T *>(lds + TILE_A), tid);
    auto tile_a = [&](int64_t t) { return reinterpret_cast<T *>(lds + (t & 1) * TILE); };
    auto tile_b = [&](int64_t t) { return reinterpret_cast<T *>(lds + (t & 1) * TILE + TILE_A); };
    auto fetch = [&](int64_t t, bool there) {
        int64_t p = t, half_a = 0, half_b = 0;
        if constexpr (HALVES) {
            const int run = __builtin_amdgcn_readfirstlane((t >= depth) + (t >= 2 * depth));
            p -= run * depth;
            half_a = __builtin_amdgcn_readfirstlane(run == 1 ? a.half_a : 0);
            half_b = __builtin_amdgcn_readfirstlane(run && run == a.runs - 1 ? a.half_b : 0);
        }
        la.fetch(p * BK, half_a, there, (unsigned)(t & 1) * TILE, tid);
        lb.fetch(p * BK, half_b, there, (unsigned)(t & 1) * TILE, tid);
    };
    constexpr int PIECES_A = A_DMA ? la.N : 0, PIECES = PIECES_A + (B_DMA ? lb.N : 0);
    auto piece = [&](int i) {
        if (i < PIECES_A) la.dma(i);
        else lb.dma(i - PIECES_A);
    };
    auto pieces = [&]() {
#pragma unroll
        for (int i = 0; i < PIECES; i++) piece(i);
    };
    auto store = [&](int64_t t) {
        la.store(tile_a(t), tid);
        lb.store(tile_b(t), tid);
    };
    typename Frag<T>::V fa[2][MI], fb[2][NJ];
    auto read = [&](int64_t t, int step, int into) {
#pragma unroll
        for (int x = 0; x < MI; x++) fa[into][x] = fragment<T, BM, A_P>(tile_a(t), wi + 32 * x, step, lane);
#pragma unroll
        for (int y = 0; y < NJ; y++) fb[into][y] = fragment<T, BN, B_P>(tile_b(t), wj + 32 * y, step, lane);
    };
    auto multiply = [&](int from, int i) {
        const int x = i / NJ, y = i % NJ;
        acc[x][y] = mfma(fa[from][x], fb[from][y], acc[x][y]);
    };
    if (first < last) {
        fetch(first, true);
        pieces();
        store(first);
        if (A_DMA || B_DMA) dma_wait();
        tile_barrier();
        fetch(first + 1, first + 1 < last);
        pieces();
        read(first, 0, 0);
    }
    for (int64_t t = first; t < last; t++) {
#pragma unroll
        for (int step = 0; step < 3; step++) {
            read(t, step + 1, (step + 1) & 1);
            if (step == 2 && t + 1 < last) store(t + 1);
#pragma unroll
            for (int x = 0; x < MI * NJ; x++) multiply(step & 1, x);
        }
        if (A_DMA || B_DMA) dma_wait();
        tile_barrier();                                         // tile t + 1 is whole, and nobody reads tile t any more
        read(t + 1, 0, 0);                                      // (after the last tile: what the buffer holds, never used)
        // The transfers of tile t + 2 go out between the matrix instructions, whose time hides their issue.  Past the last tile they
        // bring zeros into the free buffer without reading memory: a branch here would make every wait behind it a full one.
        fetch(t + 2, t + 2 < last);
#pragma unroll
        for (int x = 0; x < MI * NJ; x++) {
            multiply(1, x);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = PIECES * x / (MI * NJ); i < PIECES * (x + 1) / (MI * NJ); i++) piece(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (A_DMA || B_DMA) dma_wait();
    tile_barrier();

    // epilogue: 32 rows of the wave's columns at a time go through its own LDS slab, so that a lane gets 8 columns of a row
    // (matrix accumulators hold one column and 16 rows per lane)
    constexpr int CHUNKS = WN / 8, ROWS = 64 / CHUNKS;
    float *slab = reinterpret_cast<float *>(lds) + wave * 32 * PITCH;
    const int64_t col = j0 + wj + lane % CHUNKS * 8;
    const int64_t left = a.J - col;
    const int valid = left >= 8 ? 8 : (int)left;
    float bias[8];
    load_bias(a.e, col, part ? 0 : valid, bias);
#pragma unroll
    for (int x = 0; x < MI; x++) {
#pragma unroll
        for (int y = 0; y < NJ; y++)
#pragma unroll
            for (int r = 0; r < 16; r++)
                slab[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * PITCH + 32 * y + (lane & 31)] = acc[x][y][r];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        constexpr int PASSES = 32 / ROWS, U = PASSES < 4 ? PASSES : 4;
#pragma unroll 1
        for (int it = 0; it < PASSES; it += U) {
            const int r = it * ROWS + lane / CHUNKS;
            float v[U][8];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const f32x4_t *from = reinterpret_cast<const f32x4_t *>(slab + (r + u * ROWS) * PITCH + lane % CHUNKS * 8);
                const f32x4_t lo = from[0], hi = from[1];
                if (part) {
                    f32x4_t *to = reinterpret_cast<f32x4_t *>(part + (wi + 32 * x + r + u * ROWS) * BN + wj + lane % CHUNKS * 8);
                    to[0] = lo;
                    to[1] = hi;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) { v[u][i] = lo[i]; v[u][4 + i] = hi[i]; }
            }
            if (!part) {
                unscale<T, O, U>(a, i0 + wi + 32 * x + r, ROWS, col, valid, v);
                finish_chunks<O, U>(a.e, bias, i0 + wi + 32 * x + r, ROWS, a.I, col, valid, v);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

// the parts of the split tiles, added up in order; a lane per chunk of 8 columns
template <class T, class O, int BM, int BN> __global__ void __launch_bounds__(256) k_join(const ProductArgs<T, O> a)
{
    constexpr int CHUNKS = BN / 8, PER_TILE = BM * CHUNKS / 256;
    const int64_t t = blockIdx.x / PER_TILE;
    const int q = (int)(blockIdx.x - t * PER_TILE) * 256 + threadIdx.x, r = q / CHUNKS, c = q % CHUNKS * 8;
    int64_t ti, tj;
    tile_at(a.whole + t, a.tiles_i, a.tiles_j, &ti, &tj);
    const int64_t row = ti * BM + r, col = tj * BN + c, left = a.J - col;
    if (row >= a.I) return;                                    // (a row's chunks leave together)
    const int valid = left >= 8 ? 8 : (int)left;
    f32x4_t lo = {}, hi = {};
    if (valid > 0) {
        const float *p = a.part + t * a.splits * (BM * BN) + r * BN + c;
#pragma unroll 4
        for (int64_t s = 0; s < a.splits; s++, p += BM * BN) {
            lo += reinterpret_cast<const f32x4_t *>(p)[0];
            hi += reinterpret_cast<const f32x4_t *>(p)[1];
        }
    }
    float v[1][8], bias[8];
#pragma unroll
    for (int i = 0; i < 4; i++) { v[0][i] = lo[i]; v[0][4 + i] = hi[i]; }
    unscale<T, O, 1>(a, row, 0, col, valid, v);
    load_bias(a.e, col, valid, bias);
    finish_chunks<O, 1>(a.e, bias, row, 0, a.I, col, valid, v);
}

// ---- a handful of rows: the weight's bytes are all there is to move, so every wave reads whole rows of it straight into registers and
// keeps the sums of M rows of x; lanes split the depth.  CB columns per block: 8, or with a checkpoint the 32 that share a scale.
// 1 x 4096 x 4096 bf16: 6.9 us, 4.9 TB/s (64 x 64 tiles split along p and joined: 15.8 us); 1 x 257 x 1024 fp32: 3.7 us (9.0).
template <class T> struct FewArgs {
    const T *x, *w;
    int64_t ldx, ldw, m, n, k;
    Epilogue<T> e;
};

template <class T, int M, int CB> __global__ void __launch_bounds__(512) k_few_rows(const FewArgs<T> a)
{
    constexpr int WAVES = 8, NC = CB / WAVES;
    __shared__ __attribute__((aligned(16))) float sums[M][CB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c0 = (int64_t)blockIdx.x * CB;
    float acc[M][NC];
#pragma unroll
    for (int r = 0; r < M; r++)
#pragma unroll
        for (int c = 0; c < NC; c++) acc[r][c] = 0.f;
    const T *wrow[NC], *xrow[M];
#pragma unroll
    for (int c = 0; c < NC; c++) {
        const int64_t col = c0 + wave * NC + c;                  // columns and rows past the end repeat the last one and are not stored
        wrow[c] = a.w + (col < a.n ? col : a.n - 1) * a.ldw;
    }
#pragma unroll
    for (int r = 0; r < M; r++) xrow[r] = a.x + (r < a.m ? r : a.m - 1) * a.ldx;
    auto step = [&](int64_t p, int valid) {
        float w[NC][8];
#pragma unroll
        for (int c = 0; c < NC; c++) load8(wrow[c] + p, valid, w[c]);
#pragma unroll
        for (int r = 0; r < M; r++) {
            float x[8];
            load8(xrow[r] + p, valid, x);
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int i = 0; i < 8; i++) acc[r][c] += x[i] * w[c][i];
        }
    };
    int64_t p = lane * 8;
#pragma unroll 4
    for (; p + 8 <= a.k; p += 512) step(p, 8);
    if (p < a.k) step(p, (int)(a.k - p));
#pragma unroll
    for (int r = 0; r < M; r++)
#pragma unroll
        for (int c = 0; c < NC; c++) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) acc[r][c] += __shfl_xor(acc[r][c], o);
            if (lane == 0) sums[r][wave * NC + c] = acc[r][c];
        }
    __syncthreads();
    constexpr int CHUNKS = CB / 8;
    if (threadIdx.x >= M * CHUNKS) return;
    const int r = threadIdx.x / CHUNKS, c = threadIdx.x % CHUNKS * 8;
    if (r >= a.m) return;                                        // (a row's chunks leave together)
    const int64_t col = c0 + c, left = a.n - col;
    const int valid = left >= 8 ? 8 : (int)left;
    float v[1][8], bias[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[0][i] = sums[r][c + i];
    load_bias(a.e, col, valid, bias);
    finish_chunks<T, 1>(a.e, bias, r, 0, a.m, col, valid, v);
}

enum Kept { NOTHING, DENSE, PACKED };

// one chunk of what was kept, as it was loaded
template <class T, int KEPT> struct Piece {
    float dense[KEPT == DENSE ? 8 : 1];
    uint2 codes;
    uint32_t scale;
    __device__ __forceinline__ void load(const Source<T> &s, int64_t row, int64_t col, int valid)
    {
        if constexpr (KEPT == DENSE) load8(s.x + row * s.ldx + col, valid, dense);
        if constexpr (KEPT == PACKED) {
            codes = load_codes(s.codes + row * s.ldc, col, valid);
            scale = s.scales[row * s.lds + (col >> 5)];
        }
    }
    __device__ __forceinline__ void values(float v[8]) const
    {
        if constexpr (KEPT == DENSE)
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = dense[i];
        if constexpr (KEPT == PACKED) unpack8_codes(codes, pack8_unit(scale), v);
    }
};

// A value that 16 bits round as two that they hold: to twice the bits (bf16: 2^-18 of it, fp16: 2^-22 or 2^-25), and up to twice the
// type's largest value.  An infinity or a NaN is whole.
template <class T> __device__ __forceinline__ void halves(const float v[8], float first[8], float second[8])
{
    const float most = std::is_same<T, f16_t>::value ? 65504.f : 3.38953139e38f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float r = to_f((T)v[i]);
        first[i] = fabsf(r) <= most || !(fabsf(v[i]) <= 3.402823466e38f) ? r : copysignf(most, v[i]);
        second[i] = fabsf(first[i]) <= most ? v[i] - first[i] : 0.f;
    }
}

// stores v as T, HALVES: as two, the second one `half` elements further
template <class T, bool HALVES> __device__ __forceinline__ void store_halves(T *p, int64_t half, const float v[8])
{
    if constexpr (HALVES) {
        float first[8], second[8];
        halves<T>(v, first, second);
        store8(p, 8, first);
        store8(p + half, 8, second);
    } else {
        store8(p, 8, v);
    }
}

// ---- the values of a checkpoint (or a dense matrix), with an activation, as a dense matrix whose rows the product can fetch by LDS-DMA
template <class T, class O> struct DecodeArgs {
    Source<T> from;
    int64_t rows, cols, ldx, half;      // half: where a row's second halves start, or 0
    O *x;
    int act;
    RowCut cut;
    const int *exps;         // O != T: columns are multiplied by 2^exps[column]
};

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }      // -126 <= e <= 127

__device__ __forceinline__ void column_scales(const int *exps, int64_t col, int valid, float scale[8])
{
#pragma unroll
    for (int i = 0; i < 8; i++) scale[i] = i < valid ? power_of_two(exps[col + i]) : 0.f;
}

template <class T, class O, int FROM, bool HALVES> __global__ void __launch_bounds__(256) k_decode(const DecodeArgs<T, O> a)
{
    const int lane = threadIdx.x & (a.cut.tx - 1), step = 256 / a.cut.tx;
    const int64_t col = ((int64_t)blockIdx.y * a.cut.tx + lane) * 8, left = a.cols - col;
    const int valid = left >= 8 ? 8 : (int)left;
    if (valid <= 0) return;
    float scale[8];
    if constexpr (!std::is_same<T, O>::value) column_scales(a.exps, col, valid, scale);
    auto rows = [&](int64_t row, auto count, auto whole) {
        constexpr int N = decltype(count)::value;
        const int n = decltype(whole)::value ? 8 : valid;
        Piece<T, FROM> x[N];
        float v[N][8];
#pragma unroll
        for (int u = 0; u < N; u++) x[u].load(a.from, row + u * step, col, n);
#pragma unroll
        for (int u = 0; u < N; u++) x[u].values(v[u]);
        act_all<8 * N>(v[0], a.act);
#pragma unroll
        for (int u = 0; u < N; u++) {
            if constexpr (!std::is_same<T, O>::value)
#pragma unroll
                for (int i = 0; i < 8; i++) v[u][i] *= scale[i];
            // Whole chunks: the pitch is a multiple of 8.  What lies past the row enters sums where rows run along p (the copies of x
            // and w that no activation changes): the other operand's is zero there too, and both must be finite, which zeros are.
            store_halves<O, HALVES>(a.x + (row + u * step) * a.ldx + col, a.half, v[u]);
        }
    };
    each_row(a.cut.tx, a.cut.rows, blockIdx.x, a.rows, valid, rows);
}

// ---- Exponents for operands that are computed on the way into a product.  A bf16 operand that is itself a rounded result (dz, or an
// activation of what was kept) costs the product half a step of 8 bits; where both are, their gradient gw is taken in fp16 (11 bits)
// instead: every column of dz and of h is multiplied by the power of two that puts a bound of its magnitudes into [2^13, 2^14), and
// gw's rows and columns by the inverse ones.  The bound is the largest over the column of what bound_act and bound_slope give for each
// element, so a column far into an activation's flat side keeps its 11 bits as well.  Values down to 2^-29 of the bound keep at least
// the precision bf16 has; what lies under 2^-38 of it counts as zero.
constexpr int TARGET = 13;

// Upper bounds of |act(x)| for the smooth activations, at most 17 times as large (gelu at x = -13: Phi(-a) < exp(-a^2 / 2) / 2).  The
// activations' own instructions would bound the passes: 16384 x 4096, gelu, 8 bits: 45 us for dz and 28 for h instead of 57 and 58.
template <int N> __device__ __forceinline__ void bound_act(float *v, int act)
{
    switch (act) {
        case PIFU_ACT_SIGMOID: each<N>(v, [](float x) { return exp_f(x < 0.f ? x : 0.f); }); break;
        case PIFU_ACT_TANH: each<N>(v, [](float x) { const float a = fabsf(x); return a > 1.f ? 1.f : a; }); break;
        case PIFU_ACT_GELU: each<N>(v, [](float x) { return x < 0.f ? -0.5f * x * exp_f(-0.5f * x * x) : x; }); break;
        case PIFU_ACT_SILU: each<N>(v, [](float x) { return x < 0.f ? -x * exp_f(x) : x; }); break;
        default: break;
    }
}

// g[i] times an upper bound of |act'(z)|, or of half of it, so that no finite g gives an infinity (a magnitude is then under 2^15, still
// in fp16's range).  As tight, but where the derivative of gelu or silu changes its sign.  gelu', z < 0: |Phi(z) + z phi(z)| <
// (1 / 2 + 0.4 |z|) exp(-z^2 / 2); silu': |s (1 + z (1 - s))| < (1 + |z|) exp(z); their largest values are 1.129 and 1.0999.
template <int N> __device__ __forceinline__ void bound_slope(float *g, const float *v, int act, int from_output)
{
    if (from_output) { slope_all<N>(g, v, act, from_output); return; }
    switch (act) {
        case PIFU_ACT_SIGMOID: each_times<N>(g, v, [](float z) { return exp_f(-fabsf(z)); }); break;
        case PIFU_ACT_TANH: each_times<N>(g, v, [](float z) { return fminf(4.f * exp_f(-2.f * fabsf(z)), 1.f); }); break;
        case PIFU_ACT_GELU:
            each_times<N>(g, v, [](float z) { return z < 0.f ? (0.25f - 0.2f * z) * exp_f(-0.5f * z * z) : 0.565f; });
            break;
        case PIFU_ACT_SILU: each_times<N>(g, v, [](float z) { return z < 0.f ? (0.5f - 0.5f * z) * exp_f(z) : 0.55f; }); break;
        default: break;
    }
}

struct MaxArgs {
    const bf16_t *grad; int64_t ldg;                  // SLOPE: of dz = grad * act'(from), else of h = act(from)
    Source<bf16_t> from;
    float *part;                                      // [cut.blocks][cols]
    int64_t rows, cols;
    int act, from_output;
    RowCut cut;
};

// the largest finite bound in each column of dz or h over a block's rows
template <int FROM, bool SLOPE> __global__ void __launch_bounds__(256) k_column_max(const MaxArgs a)
{
    __shared__ float red[256 * 8];
    const int tx = a.cut.tx, lane = threadIdx.x & (tx - 1), ty = threadIdx.x / tx, step = 256 / tx;
    const int64_t col = ((int64_t)blockIdx.y * tx + lane) * 8, left = a.cols - col;
    const int valid = left >= 8 ? 8 : (int)left;
    float most[8] = {0.f};
    auto rows = [&](int64_t row, auto count, auto whole) {
        constexpr int N = decltype(count)::value;
        const int n = decltype(whole)::value ? 8 : valid;
        float g[N][8], v[N][8];
        Piece<bf16_t, FROM> from[N];
#pragma unroll
        for (int u = 0; u < N; u++) from[u].load(a.from, row + u * step, col, n);
        if constexpr (SLOPE) {
#pragma unroll
            for (int u = 0; u < N; u++) load8(a.grad + (row + u * step) * a.ldg + col, n, g[u]);
        }
#pragma unroll
        for (int u = 0; u < N; u++) from[u].values(v[u]);
        if constexpr (SLOPE) bound_slope<8 * N>(g[0], v[0], a.act, a.from_output);
        else bound_act<8 * N>(v[0], a.act);
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < 8; i++) most[i] = fmaxf(most[i], pack8_finite(SLOPE ? g[u][i] : v[u][i]));
    };
    each_row(tx, a.cut.rows, blockIdx.x, a.rows, valid, rows);
#pragma unroll
    for (int i = 0; i < 8; i++) red[threadIdx.x * 8 + i] = most[i];
    __syncthreads();
    for (int o = step / 2; o > 0; o >>= 1) {
        if (ty < o) {
#pragma unroll
            for (int i = 0; i < 8; i++) red[threadIdx.x * 8 + i] = fmaxf(red[threadIdx.x * 8 + i], red[(threadIdx.x + o * tx) * 8 + i]);
        }
        __syncthreads();
    }
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < 8; i++) if (i < valid) a.part[(int64_t)blockIdx.x * a.cols + col + i] = red[threadIdx.x * 8 + i];
    }
}

// exps[c] from the blocks' maxima of column c
struct ExpArgs {
    const float *part; int *exps;
    int64_t blocks, cols;
};
__global__ void __launch_bounds__(256) k_exponents(const ExpArgs a, const ExpArgs b)
{
    const ExpArgs &e = blockIdx.y ? b : a;
    const int lane = threadIdx.x & 15;
    const int64_t c = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (c >= e.cols) return;                          // (the 16 lanes of a column leave together)
    float most = 0.f;
    for (int64_t i = lane; i < e.blocks; i += 16) most = fmaxf(most, e.part[i * e.cols + c]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    int x = TARGET + 127 - (int)(__float_as_uint(most) >> 23);
    x = most == 0.f ? 0 : x > 126 ? 126 : x;
    if (lane == 0) e.exps[c] = x;
}

// ---- dz = grad * act'(kept) and its column sums.  Bound by its bytes: 50000 x 1024 bf16 with an 8-bit leaky ReLU in 46 us, 5.6 TB/s;
// 16384 x 4096 bf16 with an 8-bit gelu and dz in both 16-bit types 86 us, 5.5 TB/s.  Sums run in fp32 over a block's rows and in double
// over the blocks, in a fixed order.
template <class T> struct SlopeArgs {
    const T *grad; int64_t ldg;
    Source<T> kept;
    T *dz; int64_t lddz, half;           // [m][n] or null; half: where a row's second halves start, or 0
    f16_t *scaled; const int *exps;      // [m][lddz]: dz, its columns times 2^exps[column]; or null
    float *sums;             // [blocks][n] or null
    int64_t m, n;
    int act, from_output;
    RowCut cut;
};

template <class T, int KEPT, bool HALVES> __global__ void __launch_bounds__(256) k_slope(const SlopeArgs<T> a)
{
    __shared__ float red[256 * 8];
    const int tx = a.cut.tx, lane = threadIdx.x & (tx - 1), ty = threadIdx.x / tx, step = 256 / tx;
    const int64_t col = ((int64_t)blockIdx.y * tx + lane) * 8;
    const int64_t left = a.n - col;
    const int valid = left >= 8 ? 8 : (int)left;
    float sum[8] = {0.f}, scale[8];
    if (a.scaled) column_scales(a.exps, col, valid, scale);
    auto rows = [&](int64_t row, auto count, auto whole) {      // `count` rows at a time: all their loads go out before the first use
        constexpr int N = decltype(count)::value;
        const int n = decltype(whole)::value ? 8 : valid;
        float g[N][8], v[N][8];
        Piece<T, KEPT> kept[N];
#pragma unroll
        for (int u = 0; u < N; u++) kept[u].load(a.kept, row + u * step, col, n);
#pragma unroll
        for (int u = 0; u < N; u++) load8(a.grad + (row + u * step) * a.ldg + col, n, g[u]);
        if constexpr (KEPT != NOTHING) {
#pragma unroll
            for (int u = 0; u < N; u++) kept[u].values(v[u]);
            slope_all<8 * N>(g[0], v[0], a.act, a.from_output);
            if (a.dz) {
#pragma unroll
                for (int u = 0; u < N; u++) store_halves<T, HALVES>(a.dz + (row + u * step) * a.lddz + col, a.half, g[u]);
            }
            if (a.scaled) {
#pragma unroll
                for (int u = 0; u < N; u++) {
                    float s[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) s[i] = g[u][i] * scale[i];
                    store8(a.scaled + (row + u * step) * a.lddz + col, 8, s);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] += g[u][i];
    };
    each_row(a.cut.tx, a.cut.rows, blockIdx.x, a.m, valid, rows);
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
    const int lane = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const int64_t col = (int64_t)blockIdx.x * 8 + lane;
    double s = 0.0;
    if (col < n) {
#pragma unroll 4
        for (int64_t b = ty; b < blocks; b += 32) s += (double)sums[b * n + col];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (ty == 0 && col < n) {
        for (int i = 1; i < 32; i++) s += red[i * 8 + lane];
        out[col] = (T)(float)s;
    }
}

// ---- the backward pass of a layer with up to NARROW outputs (the classifier's head has one): matrix instructions would multiply tiles
// of zeros.  Cut as k_slope is; a lane keeps its columns of w and of gw in registers,
// so x is read once and gx written once, and dz and h never leave fp32.  Bound by those bytes; 5000 x 385 x 1 fp16 takes 10.2 us and
// 3.9 us for the sums over the blocks, the depth of its chains of loads (through the products: 27 us in five launches).
template <class T> struct NarrowArgs {
    const T *grad; int64_t ldg;
    Source<T> kept, x;
    const T *w; int64_t ldw;
    T *gx; int64_t ldgx;     // or null
    float *part;             // [blocks][(gw: n k) + n], or null
    int64_t m, k;
    int n, act, from_output, x_act;
    RowCut cut;
};

template <class T, int N, int X> __global__ void __launch_bounds__(256) k_narrow(const NarrowArgs<T> a)
{
    __shared__ float red[256 * 8];
    const int tx = a.cut.tx, lane = threadIdx.x & (tx - 1), ty = threadIdx.x / tx, step = 256 / tx;
    const int64_t col = ((int64_t)blockIdx.y * tx + lane) * 8;
    const int64_t left = a.k - col;
    const int valid = left >= 8 ? 8 : (int)left;
    float w[N][8], gw[N][8], gb[N];
#pragma unroll
    for (int c = 0; c < N; c++) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[c][i] = gw[c][i] = 0.f;
        gb[c] = 0.f;
        if (a.gx && c < a.n && valid > 0) load8(a.w + c * a.ldw + col, valid, w[c]);
    }
    auto rows = [&](int64_t row, auto count, auto whole) {
        constexpr int U = decltype(count)::value;
        const int n = decltype(whole)::value ? 8 : valid;
        Piece<T, X> x[U];
        float g[U][N], v[U][N];
#pragma unroll
        for (int u = 0; u < U; u++) x[u].load(a.x, row + u * step, col, n);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t r = row + u * step;
#pragma unroll
            for (int c = 0; c < N; c++) {
                g[u][c] = c < a.n ? to_f(a.grad[r * a.ldg + c]) : 0.f;
                v[u][c] = c < a.n && a.kept.any() ? a.kept.value(r, c) : 0.f;
            }
        }
        slope_all<U * N>(g[0], v[0], a.act, a.from_output);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (a.gx) {
                float o[8] = {0.f};
#pragma unroll
                for (int c = 0; c < N; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) o[i] += g[u][c] * w[c][i];
                store8(a.gx + (row + u * step) * a.ldgx + col, n, o);
            }
            if constexpr (X != NOTHING) {
                float h[8];
                x[u].values(h);
                act_all<8>(h, a.x_act);
#pragma unroll
                for (int c = 0; c < N; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) gw[c][i] += g[u][c] * h[i];
            }
#pragma unroll
            for (int c = 0; c < N; c++) gb[c] += g[u][c];
        }
    };
    each_row(a.cut.tx, a.cut.rows, blockIdx.x, a.m, valid, rows);
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.x * ((X != NOTHING ? a.n * a.k : 0) + a.n);
    if constexpr (X != NOTHING) {
#pragma unroll
        for (int c = 0; c < N; c++) {
            if (c >= a.n) break;
#pragma unroll
            for (int i = 0; i < 8; i++) red[threadIdx.x * 8 + i] = gw[c][i];
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
                for (int i = 0; i < 8; i++) if (i < valid) part[c * a.k + col + i] = red[threadIdx.x * 8 + i];
            }
            __syncthreads();
        }
        part += a.n * a.k;
    }
    if (blockIdx.y) return;
    if (lane == 0) {
#pragma unroll
        for (int c = 0; c < N; c++) red[c * 256 + ty] = gb[c];
    }
    __syncthreads();
    if ((int)threadIdx.x < a.n) {
        float sum = 0.f;
        for (int y = 0; y < step; y++) sum += red[threadIdx.x * 256 + y];
        part[threadIdx.x] = sum;
    }
}

template <class T> struct NarrowJoin {
    const float *part;
    int64_t blocks, weights, k, n;           // weights: n k, or 0 without gw
    T *gw; int64_t ldgw;
    T *gb;
};

template <class T> __global__ void __launch_bounds__(256) k_narrow_join(const NarrowJoin<T> a)
{
    __shared__ double red[256];
    const int lane = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const int64_t at = (int64_t)blockIdx.x * 8 + lane, cols = a.weights + a.n;
    double s = 0.0;
    if (at < cols) {
#pragma unroll 4
        for (int64_t b = ty; b < a.blocks; b += 32) s += (double)a.part[b * cols + at];
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (ty || at >= cols) return;
    for (int i = 1; i < 32; i++) s += red[i * 8 + lane];
    if (at < a.weights) a.gw[at / a.k * a.ldgw + at % a.k] = (T)(float)s;
    else if (a.gb) a.gb[at - a.weights] = (T)(float)s;
}

// ---- host side
template <class T> bool dma_ok(const Operand<T> &o) { return ::dma_ok(sizeof(T), o.x, o.ld, o.cols); }

template <class T, class O, int B, bool A_P, bool B_P, bool A_DMA, bool B_DMA, bool HALVES = false>
int launch(ProductArgs<T, O> &a, hipStream_t st)
{
    PIFU_LAUNCH((k_product<T, O, B, B, B / 2, B / 2, A_P, B_P, A_DMA, B_DMA, HALVES>),
                dim3((unsigned)(a.whole + (a.tiles_i * a.tiles_j - a.whole) * a.splits)), dim3(256), 0, st, &a);
    return PIFU_OK;
}

template <class T, class O, int TILE, bool A_P, bool B_P> int launch_tile(ProductArgs<T, O> &a, const Cut &c, hipStream_t st)
{
    constexpr int B = 64 << TILE;
    constexpr bool ONLY_DMA = TILE == 2 || !std::is_same<T, O>::value, HALVES = !ONLY_DMA && sizeof(T) == 2 && !B_P;
    PIFU_REQUIRE((!c.a_dma || dma_ok(a.a)) && (!c.b_dma || dma_ok(a.b)) && (!ONLY_DMA || (c.a_dma && c.b_dma)) &&
                 (a.runs == 1 || (HALVES && (c.a_dma || !a.half_a) && (c.b_dma || !a.half_b))), PIFU_ERR_INVALID, "a product of %lld x %lld outputs was planned for other operands", (long long)a.I, (long long)a.J);
    int rc = PIFU_ERR_INVALID;
    if (a.runs > 1) {
        if constexpr (HALVES) {
            if (c.a_dma && c.b_dma) rc = launch<T, O, B, A_P, B_P, true, true, true>(a, st);
            else if (c.a_dma) rc = launch<T, O, B, A_P, B_P, true, false, true>(a, st);
            else if constexpr (!A_P) rc = launch<T, O, B, A_P, B_P, false, true, true>(a, st);      // (grad as it lies and h in halves)
        }
    } else if constexpr (ONLY_DMA) {
        rc = launch<T, O, B, A_P, B_P, true, true>(a, st);
    } else {
        if (c.a_dma && c.b_dma) rc = launch<T, O, B, A_P, B_P, true, true>(a, st);
        else if (c.a_dma) rc = launch<T, O, B, A_P, B_P, true, false>(a, st);
        else if (c.b_dma) rc = launch<T, O, B, A_P, B_P, false, true>(a, st);
        else rc = launch<T, O, B, A_P, B_P, false, false>(a, st);
    }
    if (rc || a.splits == 1) return rc;
    PIFU_LAUNCH((k_join<T, O, B, B>), dim3((unsigned)((a.tiles_i * a.tiles_j - a.whole) * (B * B / 2048))), dim3(256), 0, st, &a);
    return PIFU_OK;
}

template <bool A_P, bool B_P, class T, class O> int product(const ProductArgs<T, O> &args, const Cut &c, float *part, hipStream_t st)
{
    ProductArgs<T, O> a = args;
    a.tiles_i = c.tiles_i; a.tiles_j = c.tiles_j; a.whole = c.whole; a.splits = c.splits; a.per = c.per; a.part = part;
    if (c.tile == 0) return launch_tile<T, O, 0, A_P, B_P>(a, c, st);
    if (c.tile == 1) return launch_tile<T, O, 1, A_P, B_P>(a, c, st);
    if constexpr (sizeof(T) == 2) return launch_tile<T, O, 2, A_P, B_P>(a, c, st);
    return PIFU_ERR_INVALID;
}

template <class T> Source<T> source(const void *x, int64_t ldx, const pifu_packed8 &p)
{
    Source<T> s;
    s.x = (const T *)x; s.ldx = ldx;
    if (!x) { s.codes = p.codes; s.ldc = p.ld; s.scales = p.scales; s.lds = p.ld_scales; }
    return s;
}

template <class T, class O>
int decode(const Source<T> &from, int64_t rows, int64_t cols, O *x, int64_t ldx, int act, const int *exps, hipStream_t st, int64_t half = 0)
{
    const DecodeArgs<T, O> d{from, rows, cols, ldx, half, x, act, RowCut(rows, cols, MAX_BLOCKS), exps};
    const dim3 grid((unsigned)d.cut.blocks, (unsigned)d.cut.wide);
    if constexpr (std::is_same<T, O>::value && sizeof(T) == 2)
        if (half) {
            if (from.x) PIFU_LAUNCH((k_decode<T, O, DENSE, true>), grid, dim3(256), 0, st, (void *)&d);
            else PIFU_LAUNCH((k_decode<T, O, PACKED, true>), grid, dim3(256), 0, st, (void *)&d);
            return PIFU_OK;
        }
    if (from.x) PIFU_LAUNCH((k_decode<T, O, DENSE, false>), grid, dim3(256), 0, st, (void *)&d);
    else PIFU_LAUNCH((k_decode<T, O, PACKED, false>), grid, dim3(256), 0, st, (void *)&d);
    return PIFU_OK;
}

template <class T, int M> int few_rows(const FewArgs<T> &a, hipStream_t st)
{
    if (a.e.codes) PIFU_LAUNCH((k_few_rows<T, M, 32>), dim3((unsigned)((a.n + 31) / 32)), dim3(512), 0, st, (void *)&a);
    else PIFU_LAUNCH((k_few_rows<T, M, 8>), dim3((unsigned)((a.n + 7) / 8)), dim3(512), 0, st, (void *)&a);
    return PIFU_OK;
}

template <class T> int forward(const pifu_linear_args &g, const Forward &f, char *ws, hipStream_t st)
{
    Epilogue<T> e{};
    e.act = g.act;
    e.bias = (const T *)g.bias;
    e.residual = (const T *)g.residual; e.ldr = g.ldr;
    e.y = (T *)g.y; e.ldy = g.ldy;
    e.z = (T *)g.z; e.ldz = g.ldz;
    e.codes = g.z8.codes; e.ldc = g.z8.ld; e.scales = g.z8.scales; e.lds = g.z8.ld_scales;
    if (g.m <= FEW_ROWS) {
        const FewArgs<T> a{(const T *)g.x, (const T *)g.w, g.ldx, g.ldw, g.m, g.n, g.k, e};
        if (g.m <= 2) return g.m == 1 ? few_rows<T, 1>(a, st) : few_rows<T, 2>(a, st);
        return g.m <= 4 ? few_rows<T, 4>(a, st) : few_rows<T, FEW_ROWS>(a, st);
    }
    ProductArgs<T> a{};
    a.a = {(const T *)g.x, g.ldx, g.k};
    a.b = {(const T *)g.w, g.ldw, g.k};
    if (f.ldx) {
        T *x = (T *)(ws + f.x);
        const int rc = decode<T, T>(source<T>(g.x, g.ldx, {}), g.m, g.k, x, f.ldx, PIFU_ACT_NONE, nullptr, st);
        if (rc) return rc;
        a.a = {x, f.ldx, f.ldx};
    }
    if (f.ldw) {
        T *w = (T *)(ws + f.w);
        const int rc = decode<T, T>(source<T>(g.w, g.ldw, {}), g.n, g.k, w, f.ldw, PIFU_ACT_NONE, nullptr, st);
        if (rc) return rc;
        a.b = {w, f.ldw, f.ldw};
    }
    a.I = g.m; a.J = g.n; a.P = g.k;
    a.runs = 1;
    a.e = e;
    return product<true, true>(a, f.cut, (float *)(ws + f.total - f.cut.bytes()), st);
}

template <class T, int N> int narrow(const NarrowArgs<T> &a, dim3 grid, bool gw, hipStream_t st)
{
    if (!gw) PIFU_LAUNCH((k_narrow<T, N, NOTHING>), grid, dim3(256), 0, st, (void *)&a);
    else if (a.x.x) PIFU_LAUNCH((k_narrow<T, N, DENSE>), grid, dim3(256), 0, st, (void *)&a);
    else PIFU_LAUNCH((k_narrow<T, N, PACKED>), grid, dim3(256), 0, st, (void *)&a);
    return PIFU_OK;
}

template <class T> int backward_narrow(const pifu_linear_grad_args &g, const Plan &p, char *ws, hipStream_t st)
{
    NarrowArgs<T> a{};
    a.grad = (const T *)g.grad; a.ldg = g.ldg;
    if (g.act != PIFU_ACT_NONE) a.kept = source<T>(g.z, g.ldz, g.z8);
    if (g.gw) a.x = source<T>(g.x, g.ldx, g.x8);
    a.w = (const T *)g.w; a.ldw = g.ldw;
    a.gx = (T *)g.gx; a.ldgx = g.ldgx;
    a.part = g.gw || g.gb ? (float *)ws : nullptr;
    a.m = g.m; a.k = g.k;
    a.n = (int)g.n; a.act = g.act; a.from_output = g.from_output; a.x_act = g.x_act; a.cut = p.cut;
    const dim3 grid((unsigned)p.cut.blocks, (unsigned)p.cut.wide);
    const int rc = g.n == 1 ? narrow<T, 1>(a, grid, g.gw, st) : narrow<T, NARROW>(a, grid, g.gw, st);
    if (rc || !a.part) return rc;
    NarrowJoin<T> j{a.part, p.cut.blocks, g.gw ? g.n * g.k : 0, g.k, g.n, (T *)g.gw, g.ldgw, (T *)g.gb};
    PIFU_LAUNCH(k_narrow_join<T>, dim3((unsigned)((j.weights + j.n + 7) / 8)), dim3(256), 0, st, &j);
    return PIFU_OK;
}

// gw = dz^T h; I: the type the operands enter the product in
template <class T, class I>
int weight_gradient(const pifu_linear_grad_args &g, const Plan &p, const Operand<I> &dz, char *ws, hipStream_t st)
{
    ProductArgs<I, T> a{};
    a.a = dz;
    a.exp_i = (const int *)(ws + p.exp_i); a.exp_j = (const int *)(ws + p.exp_j);
    if (decodes(g)) {
        I *h = (I *)(ws + p.h);
        if (g.m > 0) {
            const int rc = decode<T, I>(source<T>(g.x, g.ldx, g.x8), g.m, g.k, h, p.pitch_h(), g.x_act, a.exp_j, st, p.halves_h ? p.ldh : 0);
            if (rc) return rc;
        }
        a.b = {h, p.pitch_h(), p.ldh};
    } else {
        a.b = {(const I *)g.x, g.ldx, g.k};
    }
    a.I = g.n; a.J = g.k; a.P = g.m;
    a.runs = 1 + p.halves_dz + p.halves_h;
    a.half_a = p.halves_dz ? (int)p.lddz : 0;
    a.half_b = p.halves_h ? (int)p.ldh : 0;
    a.e.y = (T *)g.gw; a.e.ldy = g.ldgw;
    return product<false, false>(a, p.gw, (float *)(ws + p.part), st);
}

template <class T> int backward(const pifu_linear_grad_args &g, const Plan &p, char *ws, hipStream_t st)
{
    if (p.narrow) return backward_narrow<T>(g, p, ws, st);
    const bool slope = g.act != PIFU_ACT_NONE;
    T *dz = slope && (g.gx || (g.gw && !p.scaled)) ? (T *)(ws + p.dz) : nullptr;
    int *exp_i = (int *)(ws + p.exp_i), *exp_j = (int *)(ws + p.exp_j);
    if constexpr (std::is_same<T, bf16_t>::value)
        if (p.scaled) {
            MaxArgs i{(const bf16_t *)g.grad, g.ldg, source<bf16_t>(g.z, g.ldz, g.z8), (float *)(ws + p.max_i),
                      g.m, g.n, g.act, g.from_output, p.max_cut_i};
            MaxArgs j{nullptr, 0, source<bf16_t>(g.x, g.ldx, g.x8), (float *)(ws + p.max_j), g.m, g.k, g.x_act, 0, p.max_cut_j};
            const dim3 grid_i((unsigned)i.cut.blocks, (unsigned)i.cut.wide), grid_j((unsigned)j.cut.blocks, (unsigned)j.cut.wide);
            if (g.z) PIFU_LAUNCH((k_column_max<DENSE, true>), grid_i, dim3(256), 0, st, &i);
            else PIFU_LAUNCH((k_column_max<PACKED, true>), grid_i, dim3(256), 0, st, &i);
            if (g.x) PIFU_LAUNCH((k_column_max<DENSE, false>), grid_j, dim3(256), 0, st, &j);
            else PIFU_LAUNCH((k_column_max<PACKED, false>), grid_j, dim3(256), 0, st, &j);
            ExpArgs ei{i.part, exp_i, i.cut.blocks, g.n}, ej{j.part, exp_j, j.cut.blocks, g.k};
            PIFU_LAUNCH(k_exponents, dim3((unsigned)(((g.n > g.k ? g.n : g.k) + 15) / 16), 2), dim3(256), 0, st, &ei, &ej);
        }
    if (dz || p.scaled || g.gb) {
        SlopeArgs<T> s{};
        s.grad = (const T *)g.grad; s.ldg = g.ldg;
        if (slope) s.kept = source<T>(g.z, g.ldz, g.z8);
        s.dz = dz; s.lddz = p.pitch_dz(); s.half = p.halves_dz ? p.lddz : 0;
        if (p.scaled) { s.scaled = (f16_t *)(ws + p.dz16); s.exps = exp_i; }
        s.sums = g.gb ? (float *)(ws + p.sums) : nullptr;
        s.m = g.m; s.n = g.n; s.act = g.act; s.from_output = g.from_output; s.cut = p.cut;
        const dim3 grid((unsigned)p.cut.blocks, (unsigned)p.cut.wide);
        if (!slope) PIFU_LAUNCH((k_slope<T, NOTHING, false>), grid, dim3(256), 0, st, &s);
        else if (!s.half) {
            if (g.z) PIFU_LAUNCH((k_slope<T, DENSE, false>), grid, dim3(256), 0, st, &s);
            else PIFU_LAUNCH((k_slope<T, PACKED, false>), grid, dim3(256), 0, st, &s);
        } else if constexpr (sizeof(T) == 2) {
            if (g.z) PIFU_LAUNCH((k_slope<T, DENSE, true>), grid, dim3(256), 0, st, &s);
            else PIFU_LAUNCH((k_slope<T, PACKED, true>), grid, dim3(256), 0, st, &s);
        }
        if (g.gb) {
            const float *sums = s.sums;
            int64_t blocks = p.cut.blocks, n = g.n;
            T *out = (T *)g.gb;
            PIFU_LAUNCH(k_column_sums<T>, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, &sums, &blocks, &n, &out);
        }
    }
    ProductArgs<T> a{};
    a.a = dz ? Operand<T>{dz, p.pitch_dz(), p.lddz} : Operand<T>{(const T *)g.grad, g.ldg, g.n};
    if (g.gx && g.m > 0) {
        a.b = {(const T *)g.w, g.ldw, g.k};
        if (p.ldw) {
            T *w = (T *)(ws + p.w);
            const int rc = decode<T, T>(source<T>(g.w, g.ldw, {}), g.n, g.k, w, p.ldw, PIFU_ACT_NONE, nullptr, st);
            if (rc) return rc;
            a.b = {w, p.ldw, p.ldw};
        }
        a.I = g.m; a.J = g.k; a.P = g.n;
        a.runs = 1 + p.halves_dz;
        a.half_a = p.halves_dz ? (int)p.lddz : 0;
        a.e.y = (T *)g.gx; a.e.ldy = g.ldgx;
        const int rc = product<true, false>(a, p.gx, (float *)(ws + p.part), st);
        if (rc) return rc;
    }
    if (g.gw) {
        if constexpr (std::is_same<T, bf16_t>::value)
            if (p.scaled) return weight_gradient<T, f16_t>(g, p, {(const f16_t *)(ws + p.dz16), p.lddz, p.lddz}, ws, st);
        return weight_gradient<T, T>(g, p, a.a, ws, st);
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
    PIFU_REQUIRE(g->m >= 0 && g->n >= 1 && g->k >= 1 && g->n <= MAX_WIDTH && g->k <= MAX_WIDTH, PIFU_ERR_INVALID,
                 "%s: bad shape m %lld, n %lld, k %lld", name, (long long)g->m, (long long)g->n, (long long)g->k);
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
    PIFU_REQUIRE(g->m >= 0 && g->n >= 1 && g->k >= 1 && g->n <= MAX_WIDTH && g->k <= MAX_WIDTH, PIFU_ERR_INVALID,
                 "%s: bad shape m %lld, n %lld, k %lld", name, (long long)g->m, (long long)g->n, (long long)g->k);
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

template <class G> int check_fits(const char *name, const G &g, bool fits)
{
    PIFU_REQUIRE(fits, PIFU_ERR_INVALID, "%s: m %lld, n %lld, k %lld has more outputs than one launch can hold", name, (long long)g.m,
                 (long long)g.n, (long long)g.k);
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
    PIFU_CHECKED(check_forward(ctx, args));
    if (args->m == 0) return 0;
    const Forward plan = plan_forward(*args);
    PIFU_CHECKED(check_fits("pifu_linear", *args, plan.fits));
    return plan.total;
}

extern "C" int pifu_linear(pifu_ctx *ctx, const pifu_linear_args *args, void *workspace, int64_t workspace_bytes, pifu_stream stream)
{
    PIFU_CHECKED(check_forward(ctx, args));
    if (args->m == 0) return PIFU_OK;
    const Forward plan = plan_forward(*args);
    PIFU_CHECKED(check_fits("pifu_linear", *args, plan.fits));
    PIFU_CHECKED(check_workspace("pifu_linear", workspace, workspace_bytes, plan.total));
    PifuDeviceGuard guard(ctx->device);
    PIFU_HIP(guard.err);
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
    if (args->dtype == PIFU_F32) return forward<float>(*args, plan, ws, st);
    if (args->dtype == PIFU_BF16) return forward<bf16_t>(*args, plan, ws, st);
    return forward<f16_t>(*args, plan, ws, st);
}

extern "C" int64_t pifu_linear_backward_workspace(pifu_ctx *ctx, const pifu_linear_grad_args *args)
{
    PIFU_CHECKED(check_backward(ctx, args));
    const Plan plan = plan_backward(*args);
    PIFU_CHECKED(check_fits("pifu_linear_backward", *args, plan.fits));
    return plan.total;
}

extern "C" int pifu_linear_backward(pifu_ctx *ctx, const pifu_linear_grad_args *args, void *workspace, int64_t workspace_bytes,
                                    pifu_stream stream)
{
    PIFU_CHECKED(check_backward(ctx, args));
    const Plan plan = plan_backward(*args);
    PIFU_CHECKED(check_fits("pifu_linear_backward", *args, plan.fits));
    PIFU_CHECKED(check_workspace("pifu_linear_backward", workspace, workspace_bytes, plan.total));
    PifuDeviceGuard guard(ctx->device);
    PIFU_HIP(guard.err);
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
    if (args->dtype == PIFU_F32) return backward<float>(*args, plan, ws, st);
    if (args->dtype == PIFU_BF16) return backward<bf16_t>(*args, plan, ws, st);
    return backward<f16_t>(*args, plan, ws, st);
}
