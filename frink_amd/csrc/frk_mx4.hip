// MXFP4 (frk_mx4.hpp has the mathematics): quantization to rows and to GGUF blocks, the values back, and the products of a few tokens
// over MXFP4 matrices as they are stored.
#include "frk_mx4.hpp"

#include <algorithm>
#include <atomic>

namespace frk {

typedef int mx4_v4i __attribute__((ext_vector_type(4)));
typedef int mx4_v8i __attribute__((ext_vector_type(8)));
typedef float mx4_v4f __attribute__((ext_vector_type(4)));

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

// ---- a batch's rows: a wavefront four chunks of 256 columns at a time ----
constexpr int MX4_CHUNKS = 4;
template <bool WIDE>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const float *__restrict__ x, size_t jobs, int jobs_a_row, int cols, Mx4Acts out) {
    const int lane = threadIdx.x & 63, chunks = out.blocks / 8;
    for (size_t j = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); j < jobs; j += (size_t)gridDim.x * 4) {
        const size_t row = j / jobs_a_row;
        const int first = (int)(j % jobs_a_row) * MX4_CHUNKS;
        float v[MX4_CHUNKS][4];
#pragma unroll
        for (int i = 0; i < MX4_CHUNKS; i++) floats_load4<FLOATS_F32, WIDE>(x + row * (size_t)cols, (first + i) * 256 + lane * 4, cols, v[i]);
#pragma unroll
        for (int i = 0; i < MX4_CHUNKS; i++)
            if (first + i < chunks) mx4_store_chunk(out, row, first + i, lane, v[i]);  // (uniform)
    }
}
int launch_mx4_quantize(const float *x, size_t rows, size_t cols, const Mx4Acts &out, hipStream_t s) {
    const int jobs_a_row = (out.blocks / 8 + MX4_CHUNKS - 1) / MX4_CHUNKS;
    const size_t jobs = rows * jobs_a_row;
    if (jobs == 0) return FRK_OK;
    const dim3 grid((unsigned)std::min<size_t>((jobs + 3) / 4, 1 << 16));
    if (floats_wide(x, cols, FLOATS_F32)) hipLaunchKernelGGL(mx4_quantize_kernel<true>, grid, dim3(256), 0, s, x, jobs, jobs_a_row, (int)cols, out);
    else hipLaunchKernelGGL(mx4_quantize_kernel<false>, grid, dim3(256), 0, s, x, jobs, jobs_a_row, (int)cols, out);
    FRK_LAUNCH_CHECK("mx4_quantize");
    return FRK_OK;
}

// two values of a byte of codes, low half first, without their scale
__device__ __forceinline__ float2 mx4_two(uint32_t four, int which) {
    float2 o = make_float2(0.0f, 0.0f);
#if defined(__HIP_DEVICE_COMPILE__)
    typedef float two_t __attribute__((ext_vector_type(2)));
    const two_t v = which == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, 1.0f, 0)
                    : which == 1 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, 1.0f, 1)
                    : which == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, 1.0f, 2)
                                 : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(four, 1.0f, 3);
    o = make_float2(v.x, v.y);
#endif
    return o;
}
// what the quantized rows stand for: a wavefront 256 values at a time
template <bool WIDE>
__global__ __launch_bounds__(256) void mx4_values_kernel(Mx4Acts a, size_t jobs, int jobs_a_row, int cols, float *__restrict__ out) {
    const int lane = threadIdx.x & 63;
    for (size_t j = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); j < jobs; j += (size_t)gridDim.x * 4) {
        const size_t row = j / jobs_a_row;
        const int c = (int)(j % jobs_a_row);
        const size_t block = row * a.blocks + (size_t)c * 8 + (lane >> 3);
        const uint32_t codes = *reinterpret_cast<const uint32_t *>(a.codes + block * 16 + (lane & 3) * 4) >> (lane & 4);
        const float scale = mx4_scale(a.scales[block]);
        const float v[4] = {mx4_two(codes, 0).x * scale, mx4_two(codes, 1).x * scale, mx4_two(codes, 2).x * scale, mx4_two(codes, 3).x * scale};
        floats_store4<FLOATS_F32, WIDE>(out + row * (size_t)cols, c * 256 + lane * 4, cols, v);
    }
}
int launch_mx4_values(const Mx4Acts &a, size_t cols, float *out, hipStream_t s) {
    const size_t jobs_a_row = (cols + 255) / 256, jobs = (size_t)a.rows * jobs_a_row;
    const dim3 grid((unsigned)std::min<size_t>((jobs + 3) / 4, 1 << 16));
    if (floats_wide(out, cols, FLOATS_F32)) hipLaunchKernelGGL(mx4_values_kernel<true>, grid, dim3(256), 0, s, a, jobs, (int)jobs_a_row, (int)cols, out);
    else hipLaunchKernelGGL(mx4_values_kernel<false>, grid, dim3(256), 0, s, a, jobs, (int)jobs_a_row, (int)cols, out);
    FRK_LAUNCH_CHECK("mx4_values");
    return FRK_OK;
}

// ---- GGUF blocks: the scale byte, then sixteen bytes of codes.  256 of them are 4352 bytes, 272 pieces of sixteen: a workgroup puts them
// together in LDS.  Four lanes a block: of floats, a lane elements 4 l .. and 16 + 4 l .., whose codes share bytes; of two-byte numbers, eight
// neighbours (sixteen bytes a load), whose codes meet those of the lane two further on.  14336 x 4096 of bf16 27.6 us, of f32 48, back 44, one matrix
// after another: 5.4, 5.5 and 6.0 TB/s, what memory gives.  Behind a kernel that has just written 235 MB (the way back, a fill) the first takes 41 to 43: what that one
// left in the caches goes out to memory beside it. ----
constexpr int GGUF_BLOCKS = 256;
__device__ __forceinline__ void lds_put32(uint8_t *to, uint32_t v) { __builtin_memcpy(to, &v, 4); }  // (of any alignment)
template <int TYPE, bool WIDE>
__global__ __launch_bounds__(256) void quantize_mxfp4_kernel(const typename Floats<TYPE>::type *__restrict__ x, size_t blocks, uint8_t *__restrict__ out, bool whole) {
    typedef typename Floats<TYPE>::type T;
    constexpr bool TWO_BYTES = sizeof(T) == 2;
    constexpr int N = GGUF_BLOCKS / 64;
    __shared__ __align__(16) uint8_t lds[GGUF_BLOCKS * MXFP4_BYTES];
    const int part = threadIdx.x & 3, low = TWO_BYTES ? 8 * part : 4 * part, high = TWO_BYTES ? 8 * part + 4 : 16 + 4 * part;
    for (size_t first = (size_t)blockIdx.x * GGUF_BLOCKS; first < blocks; first += (size_t)gridDim.x * GGUF_BLOCKS) {
        float a[N][4], b[N][4];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const size_t block = first + i * 64 + (threadIdx.x >> 2);
            const int left = block < blocks ? MX4_BLOCK : 0;
            const T *const from = x + block * MX4_BLOCK;
            if (TWO_BYTES && WIDE) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (left) v = *reinterpret_cast<const uint4 *>(from + low);
                const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    a[i][j] = Floats<TYPE>::get((T)(d[j >> 1] >> (16 * (j & 1))));
                    b[i][j] = Floats<TYPE>::get((T)(d[2 + (j >> 1)] >> (16 * (j & 1))));
                }
            } else {
                floats_load4<TYPE, WIDE>(from, low, left, a[i]);
                floats_load4<TYPE, WIDE>(from, high, left, b[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            uint32_t top = max(mx4_top4(a[i]), mx4_top4(b[i]));
            top = max(top, (uint32_t)dpp_i<DPP_QUAD_XOR1>((int)top));
            top = max(top, (uint32_t)dpp_i<DPP_QUAD_XOR2>((int)top));
            const uint32_t by = mx4_scale_byte(top), ca = mx4_codes4(a[i], by), cb = mx4_codes4(b[i], by);
            uint8_t *const to = lds + (i * 64 + (threadIdx.x >> 2)) * MXFP4_BYTES;
            if (part == 0) to[0] = (uint8_t)by;
            if (TWO_BYTES) {
                const uint32_t fa = (uint32_t)dpp_i<DPP_QUAD_XOR2>((int)ca), fb = (uint32_t)dpp_i<DPP_QUAD_XOR2>((int)cb);
                if (part < 2) lds_put32(to + 1 + low, ca | fa << 4), lds_put32(to + 5 + low, cb | fb << 4);
            } else {
                lds_put32(to + 1 + low, ca | cb << 4);
            }
        }
        __syncthreads();
        const size_t bytes = (blocks - first < GGUF_BLOCKS ? blocks - first : GGUF_BLOCKS) * MXFP4_BYTES;
        uint8_t *const to = out + first * MXFP4_BYTES;
        if (whole && bytes == sizeof lds) {
            for (int i = threadIdx.x; i < (int)sizeof lds / 16; i += 256) reinterpret_cast<uint4 *>(to)[i] = reinterpret_cast<const uint4 *>(lds)[i];
        } else {
            for (size_t i = threadIdx.x; i < bytes; i += 256) to[i] = lds[i];
        }
        __syncthreads();
    }
}
template <int TYPE>
static int go_quantize_mxfp4(const void *x, size_t blocks, uint8_t *out, hipStream_t s) {
    typedef typename Floats<TYPE>::type T;
    const dim3 grid((unsigned)std::min<size_t>((blocks + GGUF_BLOCKS - 1) / GGUF_BLOCKS, 1 << 16));
    const bool whole = (uintptr_t)out % 16 == 0;
    if ((uintptr_t)x % 16 == 0) hipLaunchKernelGGL((quantize_mxfp4_kernel<TYPE, true>), grid, dim3(256), 0, s, (const T *)x, blocks, out, whole);
    else hipLaunchKernelGGL((quantize_mxfp4_kernel<TYPE, false>), grid, dim3(256), 0, s, (const T *)x, blocks, out, whole);
    FRK_LAUNCH_CHECK("quantize_mxfp4");
    return FRK_OK;
}
int launch_quantize_mxfp4(int type, const void *x, size_t n, uint8_t *blocks, hipStream_t s) {
    switch (type) {
    case FLOATS_F32: return go_quantize_mxfp4<FLOATS_F32>(x, n / MX4_BLOCK, blocks, s);
    case FLOATS_BF16: return go_quantize_mxfp4<FLOATS_BF16>(x, n / MX4_BLOCK, blocks, s);
    default: return go_quantize_mxfp4<FLOATS_F16>(x, n / MX4_BLOCK, blocks, s);
    }
}
// (WIDE: a kernel of its own.  As a branch in front of the stores the compiler made both sides single dwords: 14336 x 4096 77 us.)
template <bool WIDE>
__global__ __launch_bounds__(256) void dequantize_mxfp4_kernel(const uint8_t *__restrict__ in, size_t blocks, float *__restrict__ out, bool whole) {
    __shared__ __align__(16) uint8_t lds[GGUF_BLOCKS * MXFP4_BYTES];
    for (size_t first = (size_t)blockIdx.x * GGUF_BLOCKS; first < blocks; first += (size_t)gridDim.x * GGUF_BLOCKS) {
        const int n = (int)(blocks - first < GGUF_BLOCKS ? blocks - first : GGUF_BLOCKS);
        const uint8_t *const from = in + first * MXFP4_BYTES;
        if (whole && n == GGUF_BLOCKS) {
            for (int i = threadIdx.x; i < (int)sizeof lds / 16; i += 256) reinterpret_cast<uint4 *>(lds)[i] = reinterpret_cast<const uint4 *>(from)[i];
        } else {
            for (int i = threadIdx.x; i < n * MXFP4_BYTES; i += 256) lds[i] = from[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < GGUF_BLOCKS * 8 / 256; i++) {
            const int four = i * 256 + (int)threadIdx.x, b = min(four >> 3, n - 1);  // four elements: 4 (four % 4) .., of the upper half if (four & 4)
            const uint8_t *const block = lds + b * MXFP4_BYTES;
            uint32_t codes;
            __builtin_memcpy(&codes, block + 1 + 4 * (four & 3), 4);
            codes = codes >> (four & 4);  // (the low halves of the bytes are this thread's)
            const float scale = mx4_scale(block[0]);
            const float v[4] = {mx4_two(codes, 0).x * scale, mx4_two(codes, 1).x * scale, mx4_two(codes, 2).x * scale, mx4_two(codes, 3).x * scale};
            floats_store4<FLOATS_F32, WIDE>(out + first * MX4_BLOCK, four * 4, n * MX4_BLOCK, v);
        }
        __syncthreads();
    }
}
int launch_dequantize_mxfp4(const uint8_t *blocks, size_t n, float *out, hipStream_t s) {
    const size_t nb = n / MX4_BLOCK;
    const dim3 grid((unsigned)std::min<size_t>((nb + GGUF_BLOCKS - 1) / GGUF_BLOCKS, 1 << 16));
    const bool whole = (uintptr_t)blocks % 16 == 0;
    if ((uintptr_t)out % 16 == 0) hipLaunchKernelGGL(dequantize_mxfp4_kernel<true>, grid, dim3(256), 0, s, blocks, nb, out, whole);
    else hipLaunchKernelGGL(dequantize_mxfp4_kernel<false>, grid, dim3(256), 0, s, blocks, nb, out, whole);
    FRK_LAUNCH_CHECK("dequantize_mxfp4");
    return FRK_OK;
}

// ---- A few tokens: the weights' bytes bound it.  A workgroup of NW wavefronts has sixteen weight rows and up to 16 TT tokens; its
// wavefronts share the columns, 512 at a time (a unit: sixteen blocks of a row), and their sums meet in LDS.  Lane l has weight row l % 16 and,
// in product k of a unit's four (v_mfma_scale_f32_16x16x128_f8f6f4), block 4 k + l / 16.  The weights come through LDS, 256 bytes of a row in one
// piece: loaded as operands, sixteen bytes of sixteen rows side by side, one token of 14336 x 4096 took 10.3 us, not 8.3 (31 MB, 3.8 TB/s from launch to
// end; 32000 x 4096 14.7 us, 4.7 TB/s).
// FUSED: up to four tokens are quantized by the workgroup itself, a wavefront its own columns'. ----
struct Mx4Rows {
    Mx4Gemm g;
    const float *x;  // FUSED
    int cols;
};
constexpr int MX4_UNIT = 16, MX4_FUSED = 4;           // blocks; tokens
constexpr int MX4_FUSED_UNIT = MX4_UNIT * 16 + MX4_UNIT;  // bytes of LDS a token and unit
constexpr int MX4_STRIP_UNIT = 16 * 256;  // bytes of codes of sixteen rows' unit
constexpr size_t MX4_FUSED_LDS = 32 * 1024;

template <int NW, int SR, int TT, bool FUSED, bool WIDE>
__global__ __launch_bounds__(64 * NW) void mx4_rows_kernel(Mx4Rows r) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int E2M1 = 4;
    extern __shared__ __align__(16) uint8_t mx4_rows_lds[];  // [wavefronts][strips][MX4_STRIP_UNIT], then (FUSED) [units][tokens][MX4_FUSED_UNIT]
    static_assert(TT * 1024 <= MX4_STRIP_UNIT, "a wavefront's sums lie where its weights did");
    const Mx4Gemm &g = r.g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const int units = (g.blocks + MX4_UNIT - 1) / MX4_UNIT, strip = blockIdx.x * SR;
    const int u0 = units * wave / NW, u1 = units * (wave + 1) / NW;
    const uint8_t *row[SR];
#pragma unroll
    for (int r = 0; r < SR; r++) row[r] = g.W + (size_t)min((strip + r) * 16 + li, g.rows - 1) * g.row_stride;
    // A request brings a unit of four rows, sixteen lanes a row in one piece; place p of row r holds block p ^ r % 16, so that the sixteen rows' reads
    // touch all banks.
    uint8_t *const staged = mx4_rows_lds + wave * SR * MX4_STRIP_UNIT;
    const uint32_t staged_at = lds_address(staged);
    const uint8_t *const first = g.W + (size_t)strip * 16 * g.row_stride;
    uint32_t row_off[SR][4];
#pragma unroll
    for (int r = 0; r < SR; r++)
#pragma unroll
        for (int q = 0; q < 4; q++) row_off[r][q] = (uint32_t)min(r * 16 + 4 * q + lg, g.rows - 1 - strip * 16) * (uint32_t)g.row_stride;
    mx4_v4f acc[SR][TT];
#pragma unroll
    for (int r = 0; r < SR; r++)
#pragma unroll
        for (int t = 0; t < TT; t++) acc[r][t] = mx4_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (u0 < u1) {
        // the scales: a row's sixteen bytes, of which product k takes byte l / 16 of dword k
        uint4 w[SR][4], ws[SR], next_ws[SR], x[TT][4], xs[TT];
        auto w_off = [&](int u, int r, int q) { return row_off[r][q] + (uint32_t)min(u * MX4_UNIT + (li ^ (4 * q + lg)), g.blocks - 1) * 16; };
        auto fetch_w = [&](int u) {
            // (blocks past the row's last: the last one's codes, which meet zeros)
#pragma unroll
            for (int r = 0; r < SR; r++) {
#pragma unroll
                for (int q = 0; q < 4; q++) dma16_nt(staged_at + r * MX4_STRIP_UNIT + q * 1024, first, w_off(u, r, q));
                next_ws[r] = stream_load16(row[r] + (size_t)g.blocks * 16 + u * MX4_UNIT);
            }
        };
        auto take_w = [&]() {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int r = 0; r < SR; r++) {
#pragma unroll
                for (int k = 0; k < 4; k++) w[r][k] = *reinterpret_cast<const uint4 *>(staged + r * MX4_STRIP_UNIT + li * 256 + ((4 * k + lg) ^ li) * 16);
                ws[r] = next_ws[r];
            }
        };
        auto fetch_x = [&](int u) {
#pragma unroll
            for (int t = 0; t < TT; t++) {
                const size_t at = (size_t)min(16 * t + li, g.M - 1) * g.a.blocks + u * MX4_UNIT;
#pragma unroll
                for (int k = 0; k < 4; k++) x[t][k] = reinterpret_cast<const uint4 *>(g.a.codes)[at + 4 * k + lg];
                xs[t] = *reinterpret_cast<const uint4 *>(g.a.scales + at);
            }
        };
        uint8_t *const own = mx4_rows_lds + NW * SR * MX4_STRIP_UNIT + (size_t)u0 * g.M * MX4_FUSED_UNIT;  // FUSED: this wavefront's units
        if (FUSED) {
            float v[MX4_FUSED][2][4];
            for (int u = u0; u < u1; u++) {  // (all tokens' values asked for at once, the first unit's in front of the weights)
#pragma unroll
                for (int t = 0; t < MX4_FUSED; t++)
                    if (t < g.M) {
#pragma unroll
                        for (int i = 0; i < 2; i++) floats_load4<FLOATS_F32, WIDE>(r.x + (size_t)t * r.cols, u * 512 + i * 256 + lane * 4, r.cols, v[t][i]);
                    }
                if (u == u0) fetch_w(u0);
#pragma unroll
                for (int t = 0; t < MX4_FUSED; t++)
                    if (t < g.M) {
                        uint8_t *const to = own + ((size_t)(u - u0) * g.M + t) * MX4_FUSED_UNIT;
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            uint32_t by;
                            const uint32_t codes = mx4_quantize4(v[t][i], by);
                            const int b = 8 * i + (lane >> 3);
                            if ((lane & 4) == 0) *reinterpret_cast<uint32_t *>(to + b * 16 + (lane & 3) * 4) = codes;
                            if ((lane & 7) == 0) to[MX4_UNIT * 16 + b] = (uint8_t)by;
                        }
                    }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wavefront reads its own stores only)
        } else {
            fetch_w(u0);
        }
        auto consume = [&](int u) {
            if (FUSED) {
                const uint8_t *const from = own + ((size_t)(u - u0) * g.M + min(li, g.M - 1)) * MX4_FUSED_UNIT;
#pragma unroll
                for (int k = 0; k < 4; k++) x[0][k] = *reinterpret_cast<const uint4 *>(from + (4 * k + lg) * 16);
                xs[0] = *reinterpret_cast<const uint4 *>(from + MX4_UNIT * 16);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                mx4_v8i a[SR];
                int ew[SR];
#pragma unroll
                for (int r = 0; r < SR; r++) {
                    const uint4 &v = w[r][k];
                    const uint32_t wb[4] = {ws[r].x, ws[r].y, ws[r].z, ws[r].w};
                    a[r] = mx4_v8i{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
                    // (past the row's last block whatever lies there: no byte of it may be a NaN)
                    ew[r] = u * MX4_UNIT + 4 * k + lg < g.blocks ? (int)(wb[k] >> (8 * lg)) : 0;
                }
#pragma unroll
                for (int t = 0; t < TT; t++) {
                    const uint32_t xb[4] = {xs[t].x, xs[t].y, xs[t].z, xs[t].w};
                    const mx4_v8i b = {(int)x[t][k].x, (int)x[t][k].y, (int)x[t][k].z, (int)x[t][k].w, 0, 0, 0, 0};
#pragma unroll
                    for (int r = 0; r < SR; r++)
                        acc[r][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[r], b, acc[r][t], E2M1, E2M1, 0, ew[r], 0, (int)(xb[k] >> (8 * lg)));
                }
            }
        };
        for (int u = u0; u < u1; u++) {
            if (!FUSED) fetch_x(u);
            take_w();
            if (u + 1 < u1) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the place is read)
                fetch_w(u + 1);
            }
            consume(u);
        }
    }
    // (the compiler does not count a product's wait states, eighteen at most, across the branches between it and the reads of its sum)
#pragma unroll
    for (int r = 0; r < SR; r++)
#pragma unroll
        for (int t = 0; t < TT; t++) asm volatile("s_nop 15\n\ts_nop 3" : "+v"(acc[r][t]));
#pragma unroll
    for (int r = 0; r < SR; r++)
#pragma unroll
        for (int t = 0; t < TT; t++)
            reinterpret_cast<float4 *>(staged)[(r * TT + t) * 64 + lane] = make_float4(acc[r][t][0], acc[r][t][1], acc[r][t][2], acc[r][t][3]);
    __syncthreads();
    static_assert(SR * TT <= NW, "a wavefront a strip and tile of tokens");
    if (wave >= SR * TT) return;
    const int tok = 16 * (wave % TT) + li, r0 = (strip + wave / TT) * 16 + 4 * lg;
    const float4 *const sums = reinterpret_cast<const float4 *>(mx4_rows_lds) + wave * 64 + lane;
    float4 v = sums[0];
#pragma unroll
    for (int k = 1; k < NW; k++) {
        const float4 o = sums[k * (SR * MX4_STRIP_UNIT / 16)];
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
    }
    if (tok >= g.M) return;
    float *const dst = g.y + (size_t)tok * g.ldy + r0;
    const float out[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (r0 + i < g.rows) dst[i] = out[i];
#endif
}
template <int NW, int SR, int TT, bool FUSED>
static int go_mx4_rows(const Mx4Rows &r, size_t fused_lds, hipStream_t s) {
    const dim3 grid((unsigned)((r.g.rows + 16 * SR - 1) / (16 * SR)));
    const bool wide = FUSED && floats_wide(r.x, (size_t)r.cols, FLOATS_F32);
    const size_t lds = NW * SR * MX4_STRIP_UNIT + fused_lds;
    static std::atomic<uint64_t> sized{0};  // a bit a device (two threads may set the same attributes)
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && (dev >= 64 || !(sized.load(std::memory_order_relaxed) >> dev & 1))) {
        const int most = (int)(NW * SR * MX4_STRIP_UNIT + (FUSED ? MX4_FUSED_LDS : 0));
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(&mx4_rows_kernel<NW, SR, TT, FUSED, FUSED>), hipFuncAttributeMaxDynamicSharedMemorySize, most);
        if (FUSED && e == hipSuccess)
            e = hipFuncSetAttribute(reinterpret_cast<const void *>(&mx4_rows_kernel<NW, SR, TT, FUSED, false>), hipFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == hipSuccess && dev < 64) sized.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
    }
    if (e != hipSuccess) return set_error(FRK_ERR_HIP, "hipFuncSetAttribute(mx4_rows): %s", hipGetErrorString(e));
    if (wide) hipLaunchKernelGGL((mx4_rows_kernel<NW, SR, TT, FUSED, FUSED>), grid, dim3(64 * NW), lds, s, r);
    else hipLaunchKernelGGL((mx4_rows_kernel<NW, SR, TT, FUSED, false>), grid, dim3(64 * NW), lds, s, r);
    FRK_LAUNCH_CHECK("mx4_rows");
    return FRK_OK;
}

constexpr size_t MX4_ROWS_TOKENS = 32;  // most of the rows kernel
// By estimated time, in us: the rows kernel by what it reads (a strip's unit 0.95 ns with one tile of tokens, 1.4 with two); a stage of 256 columns takes a
// tile's workgroups `alone` while each has a CU to itself, `shared` times the workgroups a CU from there on (up to what a CU holds; more are another
// round), a round besides `ends` + `ends_shared` times those.  Shares of the columns cost a second launch and the traffic of the parts.  Every tile
// and number of shares timed at 104 sizes (17 to 4096 tokens, 1024 x 4096 to 32000 x 4096, 4096 x 14336): the choice is within 1 % of the fastest on
// average, 13 % off at 4096 tokens of 8192 x 1024.
Mx4Plan mx4_plan(const frk_weights *w, size_t batch, bool quantized) {
    const size_t units = (w->cols / MX4_BLOCK + MX4_UNIT - 1) / MX4_UNIT, stages = (w->cols + 255) / 256, n = batch * w->rows;
    Mx4Plan p{-1, 1, !quantized && batch <= MX4_FUSED && batch * units * MX4_FUSED_UNIT <= MX4_FUSED_LDS, 0, 0};
    if (p.fused) return p;
    if (!quantized) p.acts_bytes = mx4_acts_bytes(batch, w->cols);
    double least = 1e300;
    if (batch <= MX4_ROWS_TOKENS) {
        const double read = (double)((w->rows + 15) / 16) * (double)units;
        least = 2.0 + (batch <= 16 ? 0.8 + 0.95e-3 * read : 1.0 + 1.4e-3 * read);
    }
    static constexpr struct {
        double alone, shared, ends, ends_shared, held;  // workgroups that a CU holds
    } COST[MX4_TILE_SHAPES] = {{1.36, 1.81, 6.6, 8.0, 1}, {0.86, 1.12, 1.0, 7.4, 1}, {0.49, 0.73, 1.35, 2.0, 1}, {0.34, 0.45, 1.0, 0.7, 2}, {0.28, 0.35, 1.0, 0.0, 2}};
    for (int shape = 0; shape < MX4_TILE_SHAPES; shape++) {
        if (!mx4_tiles_fit(w, shape, batch)) continue;
        for (int parts = 1; parts <= 8; parts *= 2) {
            if (parts > 1 && (2 * (size_t)parts > stages || parts * n * 4 > SPLIT_PARTS_BYTES)) break;
            const Mx4TileSize t = MX4_TILE_SIZE[shape];
            const auto &c = COST[shape];
            const double fill = (double)((w->rows + t.rows - 1) / t.rows) * (double)((batch + t.tokens - 1) / t.tokens) * parts / 256.0;
            const double rounds = std::floor(fill / c.held + 1e-9), rest = fill - rounds * c.held, chain = (double)((stages + parts - 1) / parts);
            auto round = [&](double f) { return chain * std::max(c.alone, c.shared * f) + c.ends + c.ends_shared * f; };
            double us = 2.0 + rounds * round(c.held) + (rest > 1e-9 ? round(rest) : 0.0);
            if (parts > 1) {
                const double mb = 4e-6 * (double)n * parts;
                us += 1.7 + 0.43 * std::min(mb, 10.0) + 0.08 * std::max(mb - 10.0, 0.0);
            }
            if (us < least) least = us, p.shape = shape, p.parts = parts;
        }
    }
    if (p.parts > 1) p.parts_bytes = p.parts * n * 4;
    return p;
}
int mx4_gemm_fits(const frk_weights *w, const Mx4Plan &plan, size_t batch) {
    if (w->kind != FRK_KIND_MXFP4) return set_error(FRK_ERR_UNSUPPORTED, "MXFP4 activations feed MXFP4 weights only (kind %d)", w->kind);
    int dev = -1;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return set_error(FRK_ERR_HIP, "hipGetDevice: %s", hipGetErrorString(e));
    if (dev != w->device) return set_error(FRK_ERR_ARG, "the matrix is on device %d, the current device is %d", w->device, dev);
    // (lane offsets within a tile are 32 bits wide, columns of a fused row an int)
    if (w->cols > (1u << 23)) return set_error(FRK_ERR_SHAPE, "shape too large: %zu columns (at most 2^23)", w->cols);
    if (batch > (size_t)1 << 30) return set_error(FRK_ERR_SHAPE, "a batch of %zu rows is too large", batch);
    if ((w->rows + 15) / 16 * 512 > 0xffffffffu) return set_error(FRK_ERR_SHAPE, "shape too large: %zu rows", w->rows);
    if (plan.shape < 0 && batch > MX4_ROWS_TOKENS) return set_error(FRK_ERR_SHAPE, "%zu rows times %zu: more tiles than a grid holds", w->rows, batch);
    return FRK_OK;
}
int launch_mx4_gemm(const frk_weights *w, const Mx4Plan &plan, const float *x, const Mx4Acts *acts, size_t batch, float *y, void *ws, void *parts,
                    hipStream_t s) {
    Mx4Rows r{};
    Mx4Gemm &g = r.g;
    g.W = w->dev;
    g.row_stride = w->layout.row_stride;
    g.rows = (int)w->rows;
    g.blocks = (int)(w->cols / MX4_BLOCK);
    g.M = (int)batch;
    g.ldy = w->rows;
    if (acts) {
        g.a = *acts;
    } else if (!plan.fused) {
        g.a = mx4_acts_carve(ws, batch, w->cols);
        int rc = launch_mx4_quantize(x, batch, w->cols, g.a, s);
        if (rc) return rc;
    }
    if (plan.shape >= 0) {
        const size_t n = batch * w->rows;
        g.y = plan.parts > 1 ? (float *)parts : y;
        int rc = launch_mx4_tile(g, plan.shape, plan.parts, n, s);
        if (rc || plan.parts == 1) return rc;
        return launch_sum_parts((const float *)parts, plan.parts, n, y, s);
    }
    g.y = y;
    r.x = x;
    r.cols = (int)w->cols;
    // Strips a workgroup, and its wavefronts.  us, the quantization included, eight wavefronts of one strip / two / four: 4096 x 4096 1 token 4.2 / 5.3 /
    // 7.4, 16 tokens 7.4 / 8.5 / 10.8; 14336 x 4096 1 token 8.5 / 8.6 / 8.5, 4 11.1 / 10.0 / 9.3, 16 13.6 / 12.6 / 12.0; 32000 x 4096 1 token 15.3 / 14.8 /
    // 16.2, 16 23.6 / 19.9 / 20.5 (four strips: one workgroup a CU, so 1024 strips at a time).  Sixteen wavefronts a strip for long rows of up to four
    // tokens: 4096 x 14336 1 token 9.0 against 10.2, 4 12.9 against 15.8.
    const size_t units = (g.blocks + MX4_UNIT - 1) / MX4_UNIT, lds = batch * units * MX4_FUSED_UNIT, strips = (w->rows + 15) / 16;
    if (plan.fused) {
        if (strips < 448) return units >= 16 ? go_mx4_rows<16, 1, 1, true>(r, lds, s) : go_mx4_rows<8, 1, 1, true>(r, lds, s);
        return strips < 512 || strips > 1024 || batch == 1 ? go_mx4_rows<8, 2, 1, true>(r, lds, s) : go_mx4_rows<8, 4, 1, true>(r, lds, s);
    }
    // (more tokens of so many rows that more strips would pay are the tiles' but for a few sizes)
    if (batch > 16) return go_mx4_rows<8, 1, 2, false>(r, 0, s);
    return strips < 448 ? go_mx4_rows<8, 1, 1, false>(r, 0, s) : go_mx4_rows<8, 2, 1, false>(r, 0, s);
}

}  // namespace frk
