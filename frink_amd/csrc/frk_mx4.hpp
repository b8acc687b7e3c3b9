// Microscaled 4-bit floating point (MXFP4) on both sides of a product: what its kernels, the norm's and the runtime share.
//
//   y[t][r] = sum over the 32-wide blocks b of  2^(ew[r][b] + ex[t][b] - 254) * sum_i cw[r][32 b + i] * cx[t][32 b + i]
//
// c: E2M1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), e: E8M0 bytes.  A block of floats is quantized under
// 2^(floor(log2(amax)) - 2), which leaves its largest magnitude between 4 and 8; each value becomes the nearest E2M1 number, halves
// the even code, magnitudes above 6 the number 6.  A block with an infinity or a NaN gets the byte 255, E8M0's NaN, and zero codes.
// Blocks of magnitudes below 2^-124 have the byte 0, whose scale is 2^-127.
#pragma once

#include "frk_device.hpp"

namespace frk {

constexpr int MX4_BLOCK = 32;

// Quantized rows: codes [rows][blocks][16] with byte i of a block its elements i (low half) and i + 16, scales [rows][blocks].  A row is
// padded with zero blocks to a multiple of sixteen, so that whole lines are read.  (The order of a GGUF block: a product's k may run in any
// order that both operands have.)
struct Mx4Acts {
    uint8_t *codes, *scales;
    int rows, blocks;
};
static inline size_t mx4_padded_blocks(size_t cols) { return (cols / MX4_BLOCK + 15) / 16 * 16; }
static inline size_t mx4_acts_bytes(size_t rows, size_t cols) {
    const size_t n = rows * mx4_padded_blocks(cols);
    return n * 16 + round_up(n, 256);
}
static inline Mx4Acts mx4_acts_carve(void *base, size_t rows, size_t cols) {
    Mx4Acts a;
    a.rows = (int)rows;
    a.blocks = (int)mx4_padded_blocks(cols);
    a.codes = (uint8_t *)base;
    a.scales = a.codes + rows * (size_t)a.blocks * 16;
    return a;
}

// over the eight lanes of a block, four neighbouring values each
__device__ __forceinline__ uint32_t mx4_block_max(uint32_t v) {
    v = max(v, (uint32_t)dpp_i<DPP_QUAD_XOR1>((int)v));
    v = max(v, (uint32_t)dpp_i<DPP_QUAD_XOR2>((int)v));
    return max(v, (uint32_t)dpp_i<DPP_HALF_MIRROR>((int)v));
}
// the scale byte of a block whose largest magnitude has these bits
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t top) { return top >= 0x7f800000u ? 255u : (uint32_t)max((int)(top >> 23) - 2, 0); }
// the codes of four values, in the low halves of four bytes; `by` is the block's scale byte
__device__ __forceinline__ uint32_t mx4_codes4(const float (&v)[4], uint32_t by) {
    uint32_t codes = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    const float up = __uint_as_float((254u - min(by, 252u)) << 23);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0] * up, 0.0f, 1.0f, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[1] * up, 0.0f, 1.0f, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2] * up, 0.0f, 1.0f, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[3] * up, 0.0f, 1.0f, 3);
#endif
    return by == 255u ? 0u : codes;
}
__device__ __forceinline__ uint32_t mx4_top4(const float (&v)[4]) {  // magnitudes compare as their bits
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    return top;
}
// Eight lanes a block, four neighbouring values each: lanes 0 .. 3 of the eight end with a dword of codes each, all with the scale byte.
__device__ __forceinline__ uint32_t mx4_quantize4(const float (&v)[4], uint32_t &by) {
    by = mx4_scale_byte(mx4_block_max(mx4_top4(v)));
    const uint32_t codes = mx4_codes4(v, by);
    constexpr int DPP_ROW_SHL4 = 0x104;  // lane i <- lane i + 4
    return codes | ((uint32_t)dpp_i<DPP_ROW_SHL4>((int)codes) << 4);
}
// 256 values of a row, chunk `c`, a wavefront's (lane 4 l .. 4 l + 3); past the row's columns zeros
__device__ __forceinline__ void mx4_store_chunk(const Mx4Acts &out, size_t row, int c, int lane, const float (&v)[4]) {
    uint32_t by;
    const uint32_t codes = mx4_quantize4(v, by);
    const size_t block = row * out.blocks + (size_t)c * 8 + (lane >> 3);
    if ((lane & 4) == 0) *reinterpret_cast<uint32_t *>(out.codes + block * 16 + (lane & 3) * 4) = codes;
    if ((lane & 7) == 0) out.scales[block] = (uint8_t)by;
}

__device__ __forceinline__ float mx4_scale(uint32_t by) {
    return by == 255u ? __uint_as_float(0x7fc00000u) : by == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(by << 23);
}

// ---- numbers of the types that norms and quantizations take ----
enum { FLOATS_F32 = FRK_TYPE_F32, FLOATS_BF16 = FRK_TYPE_BF16, FLOATS_F16 = FRK_TYPE_F16 };
template <int TYPE>
struct Floats;
template <>
struct Floats<FLOATS_F32> {
    typedef float type;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Floats<FLOATS_BF16> {
    typedef uint16_t type;
    static __device__ __forceinline__ float get(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t put(float v) {  // to the nearest, halves to even
        const __bf16 b = (__bf16)v;
        uint16_t o;
        __builtin_memcpy(&o, &b, 2);
        return o;
    }
};
template <>
struct Floats<FLOATS_F16> {
    typedef uint16_t type;
    static __device__ __forceinline__ float get(uint16_t v) { return h2f(v); }
    static __device__ __forceinline__ uint16_t put(float v) { return f2h_bits(v); }
};
inline size_t floats_size(int type) { return type == FLOATS_F32 ? 4 : 2; }
// four values from column k on, zeros past `cols`; WIDE: rows whose pieces of four are whole and aligned to their size
template <int TYPE, bool WIDE>
__device__ __forceinline__ void floats_load4(const typename Floats<TYPE>::type *row, int k, int cols, float (&v)[4]) {
    typedef typename Floats<TYPE>::type T;
    struct alignas(4 * sizeof(T)) Four {
        T t[4];
    };
    if (WIDE) {
        Four f = {};
        if (k < cols) f = *reinterpret_cast<const Four *>(row + k);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = Floats<TYPE>::get(f.t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = k + i < cols ? Floats<TYPE>::get(row[k + i]) : 0.0f;
    }
}
template <int TYPE, bool WIDE>
__device__ __forceinline__ void floats_store4(typename Floats<TYPE>::type *row, int k, int cols, const float (&v)[4]) {
    typedef typename Floats<TYPE>::type T;
    struct alignas(4 * sizeof(T)) Four {
        T t[4];
    };
    if (WIDE) {
        Four f;
#pragma unroll
        for (int i = 0; i < 4; i++) f.t[i] = Floats<TYPE>::put(v[i]);
        if (k < cols) *reinterpret_cast<Four *>(row + k) = f;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (k + i < cols) row[k + i] = Floats<TYPE>::put(v[i]);
    }
}
inline bool floats_wide(const void *p, size_t cols, int type) { return cols % 4 == 0 && (uintptr_t)p % (4 * floats_size(type)) == 0; }

// ---- products ----
struct Mx4Gemm {
    const uint8_t *W;  // resident MXFP4 rows: codes [blocks][16], then scale bytes [blocks]
    size_t row_stride;
    int rows, blocks;
    Mx4Acts a;
    int M;
    float *y;
    size_t ldy;
};
// over tiles: weight rows x tokens, `parts` shares of the columns, each its own copy of y, part_stride floats apart
enum { MX4_TILE_256x256, MX4_TILE_256x128, MX4_TILE_128x128, MX4_TILE_64x128, MX4_TILE_64x64, MX4_TILE_SHAPES };
struct Mx4TileSize {
    int rows, tokens, threads;
};
constexpr Mx4TileSize MX4_TILE_SIZE[MX4_TILE_SHAPES] = {{256, 256, 256}, {256, 128, 512}, {128, 128, 256}, {64, 128, 256}, {64, 64, 256}};
bool mx4_tiles_fit(const frk_weights *w, int shape, size_t batch);  // whether a grid holds them
int launch_mx4_tile(const Mx4Gemm &g, int shape, int parts, size_t part_stride, hipStream_t s);
// How a batch is multiplied: by the rows kernel (shape -1; `fused`: its own quantization), or over tiles in `parts` shares
struct Mx4Plan {
    int shape, parts;
    bool fused;
    size_t acts_bytes, parts_bytes;  // of scratch memory
};
Mx4Plan mx4_plan(const frk_weights *w, size_t batch, bool quantized);
int mx4_gemm_fits(const frk_weights *w, const Mx4Plan &plan, size_t batch);  // a status
// x, or (where not null) the batch that `acts` holds
int launch_mx4_gemm(const frk_weights *w, const Mx4Plan &plan, const float *x, const Mx4Acts *acts, size_t batch, float *y, void *ws, void *parts,
                    hipStream_t s);
int launch_mx4_quantize(const float *x, size_t rows, size_t cols, const Mx4Acts &out, hipStream_t s);
int launch_mx4_values(const Mx4Acts &a, size_t cols, float *out, hipStream_t s);
int launch_quantize_mxfp4(int type, const void *x, size_t n, uint8_t *blocks, hipStream_t s);
int launch_dequantize_mxfp4(const uint8_t *blocks, size_t n, float *out, hipStream_t s);

}  // namespace frk
