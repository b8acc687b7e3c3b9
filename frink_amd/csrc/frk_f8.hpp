// Weights in 8-bit floating point with a scale for each block (FRK_KIND_FP8_BLOCK): what its kernels and the runtime share.
//
//   y[t][r] = sum over the 128-wide blocks b of  S[r / 128][b] * 2^e[t][b] * sum_i W[r][128 b + i] * q[t][128 b + i]
//
// W: OCP E4M3 codes, S: an f32 scale for every 128 rows x 128 columns of a matrix, q and e: the activations, quantized here
// block by block.  e is the least exponent, -100 or more, with amax <= 448 * 2^e, so x * 2^-e is exact and q is x rounded
// ONCE, to the nearest E4M3 (halves to even): an f32 scale amax / 448 would round the quotient first, and the two roundings
// together miss the nearest value now and then.  A power of two costs no accuracy where E4M3 is normal.  (Below 448 * 2^-100 =
// 3.5e-28 a block's values go towards zero.)
// Infinities and NaN take no part in amax and become E4M3's NaN.
//
// The products run on the bf16 matrix cores: a code and q * 2^(e - 16) are bf16 numbers (normal ones: q * 2^e is 2^-109 or more), and their
// sums come out as f32 sums do.  With the 16 no block's sum overflows before it meets its scale: 128 * 448 times the largest
// activation, 240 * 2^120, is 2^143.7.  All sums are of 2^-16 of their value; the last one is multiplied back, exactly from 2^-126 on.
// The 8-bit cores, twice as fast, add every eight products within 14 bits of the largest (measured on v_mfma_f32_16x16x32_fp8_fp8 and
// v_mfma_scale_f32_16x16x128_f8f6f4 alike: a product 2^-14 of its neighbour is lost, from the ninth on 2^-23 counts):
// against 64-bit sums of 128 products of normal values 1.5e-5 in the 2-norm, of codes drawn evenly 5.1e-5; bf16 9e-9, 8e-8.
#pragma once

#include "frk_device.hpp"

namespace frk {

constexpr int F8_BLOCK = 128;
constexpr int F8_STRIP = 16;              // weight rows that lie together
constexpr int F8_PIECE = F8_STRIP * F8_BLOCK;  // bytes of a strip's block: what a wavefront's two loads bring

// A resident stack of `matrices` matrices of rows x cols: every 16 rows a strip, a strip's blocks one after the other, and a
// block as [2 halves][64 lanes][16 bytes] -- lane l row l % 16, half h columns 32 (l / 16) + 16 h .. + 15 -- so that a wavefront's
// load is 1 KB in one piece and brings the operands of 16x16x32 products, eight codes each.  (A product's k runs over a lane
// group's own columns, in any order, as long as the activations have the same.)  Rows past a matrix's last and columns past the
// last are zeros.  Behind the strips the scales, [matrices][row blocks][blocks].
struct F8Mat {
    const uint8_t *q;
    const float *s;
    int rows, strips, blocks, row_blocks;  // of one matrix
};
static inline size_t f8_blocks(size_t n) { return (n + F8_BLOCK - 1) / F8_BLOCK; }
static inline size_t f8_strips(size_t rows) { return (rows + F8_STRIP - 1) / F8_STRIP; }
static inline F8Mat f8_mat(const frk_weights *w) {
    const size_t rows = w->rows / w->matrices;
    F8Mat m;
    m.q = w->dev;
    m.s = reinterpret_cast<const float *>(w->dev + w->layout.off_a);
    m.rows = (int)rows;
    m.strips = (int)f8_strips(rows);
    m.blocks = (int)f8_blocks(w->cols);
    m.row_blocks = (int)f8_blocks(rows);
    return m;
}

// Activations: q * 2^(e - F8_DOWN) as bf16, zeros past cols; [rows][blocks][128], or (`strips`) every sixteen rows a strip, a strip's blocks one after
// the other, a block as [4 products][64 lanes][8], lane l row l % 16, product k columns 32 (l / 16) + 8 k .. + 7: a wavefront's
// load of a product's operand is then 1 KB in one piece (rows past the last hold whatever the memory did).
constexpr int F8_DOWN = 16;
constexpr float F8_UP = 65536.0f;  // what a result is multiplied by
struct F8Acts {
    uint16_t *v;
    int rows;
    bool strips;
};
static inline size_t f8_acts_bytes(size_t rows, size_t cols) { return round_up((rows + 15) / 16 * 16 * f8_blocks(cols) * F8_BLOCK * 2, 256); }
static inline F8Acts f8_acts_carve(void *base, size_t rows, bool strips = false) {
    F8Acts a;
    a.strips = strips;
    a.v = (uint16_t *)base;
    a.rows = (int)rows;
    return a;
}

// where column `in` of block b of a row lies in strips
__device__ __forceinline__ size_t f8_strip_at(size_t row, int b, int in, int blocks) {
    return ((row >> 4) * blocks + b) * (F8_STRIP * F8_BLOCK) + (size_t)((in >> 3 & 3) * 512 + ((in >> 5) * 16 + (row & 15)) * 8 + (in & 7));
}

// ---- quantization: 32 lanes a block, four neighbouring values each (whole lines a load, and a store of eight bytes a lane) ----
__device__ __forceinline__ uint32_t f8_half_max(uint32_t v) {  // over 32 lanes
    v = max(v, (uint32_t)dpp_i<DPP_QUAD_XOR1>((int)v));
    v = max(v, (uint32_t)dpp_i<DPP_QUAD_XOR2>((int)v));
    v = max(v, (uint32_t)dpp_i<DPP_HALF_MIRROR>((int)v));
    v = max(v, (uint32_t)dpp_i<DPP_ROW_MIRROR>((int)v));
#if defined(__HIP_DEVICE_COMPILE__)
    const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // rows 0, 0, 2, 2 and 1, 1, 3, 3
    v = max((uint32_t)rows[0], (uint32_t)rows[1]);
#endif
    return v;
}
// the four values' codes; `scale` = 2^(e - F8_DOWN) of the block
__device__ __forceinline__ uint32_t f8_quantize4(const float (&v)[4], float &scale) {
    // magnitudes compare as their bits
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    top = f8_half_max(top);
    // hardly ever: infinities and NaN, which take no part, or a largest magnitude above 240 * 2^120, from which on the next code's
    // value is no float
    constexpr uint32_t PLAIN = 0x7f700000u;
    const bool special = __any(top > PLAIN);  // (uniform)
    if (special) {
        top = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t m = __float_as_uint(v[i]) & 0x7fffffffu;
            top = max(top, m < 0x7f800000u ? min(m, PLAIN) : 0u);
        }
        top = f8_half_max(top);
    }
    // 448 = 1.75 * 2^8: e is the exponent less 8, one more where the mantissa is above 1.75
    const int b = (int)((top + 0x1fffffu) >> 23) - 8;
    const uint32_t biased = (uint32_t)max(b, 127 - 100);
    scale = __uint_as_float((biased - F8_DOWN) << 23);
    const float up = __uint_as_float((254u - biased) << 23);  // 2^-e
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; i++) z[i] = v[i] * up;
    if (special) {
        const float most = biased == 127 + 120 ? 240.0f : 448.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) z[i] = fminf(fmaxf(z[i], -most), most);
    }
    uint32_t codes = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    codes = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], p, true);
#endif
    if (special) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if ((__float_as_uint(v[j]) & 0x7f800000u) == 0x7f800000u) codes = (codes & ~(0xffu << (8 * j))) | (0x7fu << (8 * j));
    }
    return codes;
}

// four values of a row from column k on, zeros past `cols`; WIDE: rows whose 16-byte pieces are aligned and whole
template <bool WIDE>
__device__ __forceinline__ void f8_load4(const float *__restrict__ row, int k, int cols, float (&v)[4]) {
    if (WIDE) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k < cols) a = *reinterpret_cast<const float4 *>(row + k);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = k + i < cols ? row[k + i] : 0.0f;
    }
}
static inline bool f8_wide_rows(const float *x, size_t cols) { return cols % 4 == 0 && (uintptr_t)x % 16 == 0; }

typedef __bf16 f8_v2bf __attribute__((ext_vector_type(2)));
// four codes as bf16 times `scale` (a power of two)
__device__ __forceinline__ uint2 f8_to_bf16(uint32_t codes, float scale) {
    uint2 out = make_uint2(0, 0);
#if defined(__HIP_DEVICE_COMPILE__)
    const f8_v2bf lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true);
    __builtin_memcpy(&out.x, &lo, 4);
    __builtin_memcpy(&out.y, &hi, 4);
#endif
    return out;
}

// eight blocks of a row by a wavefront, all their loads ahead; with `up` of silu(x) * up, element by element
constexpr int F8_QUANTIZE_BLOCKS = 8;
template <bool WIDE>
__device__ __forceinline__ void f8_quantize_blocks(const float *__restrict__ x, const float *__restrict__ up, size_t row, int first, int cols, int blocks,
                                                   int lane, const F8Acts &out) {
    constexpr int N = F8_QUANTIZE_BLOCKS / 2;
    const int k = first * F8_BLOCK + lane * 4;
    float v[N][4], u[N][4];
#pragma unroll
    for (int i = 0; i < N; i++) f8_load4<WIDE>(x + row * (size_t)cols, k + i * 2 * F8_BLOCK, cols, v[i]);
    if (up) {
#pragma unroll
        for (int i = 0; i < N; i++) f8_load4<WIDE>(up + row * (size_t)cols, k + i * 2 * F8_BLOCK, cols, u[i]);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) v[i][j] = silu_as_host(v[i][j]) * u[i][j];
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (first + 2 * i >= blocks) break;  // (uniform)
        float scale;
        const uint32_t codes = f8_quantize4(v[i], scale);
        const int b = first + 2 * i + (lane >> 5), in = (lane & 31) * 4;
        const size_t at = out.strips ? f8_strip_at(row, b, in, blocks)
                                     : (row * blocks + b) * F8_BLOCK + in;
        if (b < blocks) *reinterpret_cast<uint2 *>(out.v + at) = f8_to_bf16(codes, scale);
    }
}

// A product: of dense batches, or of tiles {matrix, first row of the order, rows in use, first row of y}, where row i of the order
// reads activation row src[i] (i itself without a list).
struct F8Gemm {
    F8Mat w;
    F8Acts a;
    const int *src;
    const int4 *tiles;  // null: dense, matrix blockIdx.y
    const int *n_tiles;
    int M;  // dense: rows of x
    size_t ldy;
    float *y;
};
// over tiles of a shape (weight rows x tokens); parts > 1 (dense): shares of the columns, each its own copy of y, part_stride floats apart
enum { F8_TILE_256x128, F8_TILE_256x64, F8_TILE_128x32, F8_TILE_SHAPES };
struct F8TileSize {
    int rows, tokens, threads;
};
constexpr F8TileSize F8_TILE_SIZE[F8_TILE_SHAPES] = {{256, 128, 512}, {256, 64, 256}, {128, 32, 128}};
// A status: whether tok_tiles tiles of tokens fit a grid, in `sheets` (matrices times parts), and gathered rows of activations (0: a list's are in
// order) their 32-bit offsets.  Asked before a call takes memory or launches anything.
int f8_tiles_fit(const frk_weights *w, int shape, size_t tok_tiles, size_t sheets, size_t gathered);
int launch_f8_tile(const F8Gemm &g, int shape, size_t tok_tiles, size_t matrices, int parts, size_t part_stride, hipStream_t s);
// How a dense batch is multiplied: by the rows kernel (shape -1; `fused`: its own quantization), or over tiles in `parts` shares
struct F8Plan {
    int shape, parts;
    bool fused;
    size_t acts_bytes, parts_bytes;  // of scratch memory
};
constexpr size_t F8_ROWS_TOKENS = 64;  // most of the rows kernel
F8Plan f8_plan(const frk_weights *w, size_t batch, bool quantized = false);  // quantized: never `fused`

// ---- entry points for the runtime and the expert layers ----
int f8_on_current_device(const frk_weights *w);  // a status: what every entry point refuses before it launches anything
Layout f8_layout(size_t rows, size_t cols, size_t matrices, size_t *bytes);
int launch_f8_repack(const uint8_t *src, const float *scales, const frk_weights *w, hipStream_t s);
// `quantized`: ws holds the batch from a call before, of a plan with the same layout (both of the rows kernel or both over tiles)
int launch_f8_gemm(const frk_weights *w, const F8Plan &plan, const float *x, size_t batch, float *y, void *ws, bool quantized, void *parts, hipStream_t s);
int f8_grouped_fits(const frk_weights *w, size_t x_rows, size_t pairs, bool gathered);  // a status, as f8_tiles_fit's
size_t f8_grouped_workspace_bytes(const frk_weights *w, size_t x_rows, size_t pairs);
int launch_f8_grouped(const frk_weights *w, const int32_t *group_off, const int32_t *gather, const float *x, size_t x_rows, size_t pairs,
                      float *y, void *ws, hipStream_t s);
// an expert layer's few slots: y[slot] = product of expert ids[slot] and row slot / slots_a_row of x; with `up` silu(w x) * (up x).  A slot
// whose id is no expert is left as it was; without ids every slot is matrix 0's
bool f8_slots_fit(size_t cols);
bool f8_few_slots(size_t slots, size_t experts, size_t hidden, size_t ffn);
int launch_f8_slots(const frk_weights *w, const frk_weights *up, const int32_t *ids, size_t slots, int slots_a_row, const float *x, float *y, hipStream_t s);
int f8_grouped_shape(size_t pairs, size_t groups);  // the tiles' shape
// rows of x (of silu(x) * up) quantized; `used`: a row whose entry is negative is left as it is
int launch_f8_quantize(const float *x, const float *up, size_t rows, size_t cols, const int *used, const F8Acts &out, hipStream_t s);
// the products of the tiles {matrix, first row of the order, rows in use (up to the shape's tokens), first row of y}; row i of the order
// is activation row src[i], or i
int launch_f8_tiles(const frk_weights *w, const F8Acts &acts, int shape, const int *src, const int4 *tiles, const int *n_tiles, size_t max_tiles, float *y,
                    hipStream_t s);

}  // namespace frk
