// Products with weights in 8-bit floating point, a scale for each block of 128 x 128 (frk_f8.hpp has the mathematics and the
// layouts): registration, the dequantizer, the activations' quantization and the GEMM, dense and grouped.  The reference has no
// such kind; its entry points' shapes are those of the others (include/frink_hip.h).
#include "frk_f8.hpp"

#include <algorithm>

namespace frk {

typedef __bf16 f8_v8bf __attribute__((ext_vector_type(8)));
typedef float f8_v4f __attribute__((ext_vector_type(4)));

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

Layout f8_layout(size_t rows, size_t cols, size_t matrices, size_t *bytes) {
    const size_t m_rows = rows / matrices;
    Layout l;
    l.row_stride = f8_blocks(cols) * F8_BLOCK;
    l.off_a = matrices * f8_strips(m_rows) * F8_STRIP * l.row_stride;
    *bytes = l.off_a + round_up(matrices * f8_blocks(m_rows) * f8_blocks(cols) * 4, 256);
    return l;
}

// where column k of row r (of matrix m) lies
__device__ __forceinline__ size_t f8_at(const F8Mat &w, size_t m, int r, int k) {
    const size_t piece = (m * w.strips + r / F8_STRIP) * w.blocks + k / F8_BLOCK;
    const int in = k % F8_BLOCK;
    return piece * F8_PIECE + (size_t)((in >> 4 & 1) * 1024 + ((in >> 5) * 16 + r % F8_STRIP) * 16 + (in & 15));
}

// a thread per sixteen bytes of the resident copy
__global__ __launch_bounds__(256) void f8_repack_kernel(const uint8_t *__restrict__ src, uint8_t *__restrict__ dst, F8Mat w, size_t cols,
                                                        size_t words, bool whole) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (size_t)gridDim.x * 256) {
        const size_t piece = i / 128, strip = piece / w.blocks;
        const int half = (int)(i >> 6 & 1), lane = (int)(i & 63);
        const size_t m = strip / w.strips;
        const int r = (int)(strip % w.strips) * F8_STRIP + (lane & 15);
        const size_t k = (piece % w.blocks) * F8_BLOCK + (lane >> 4) * 32 + half * 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < w.rows && k < cols) {
            const uint8_t *from = src + (m * w.rows + r) * cols + k;
            if (whole) {
                v = *reinterpret_cast<const uint4 *>(from);
            } else {
                uint32_t d[4] = {0, 0, 0, 0};
                for (int j = 0; j < 16; j++)
                    if (k + j < cols) d[j >> 2] |= (uint32_t)from[j] << (8 * (j & 3));
                v = make_uint4(d[0], d[1], d[2], d[3]);
            }
        }
        reinterpret_cast<uint4 *>(dst)[i] = v;
    }
}
// (the scales by a kernel too: a copy of any alignment, and nothing that a captured graph could not replay)
__global__ __launch_bounds__(256) void f8_scales_kernel(const float *__restrict__ src, float *__restrict__ dst, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) dst[i] = src[i];
}
int launch_f8_repack(const uint8_t *src, const float *scales, const frk_weights *w, hipStream_t s) {
    const F8Mat m = f8_mat(w);
    const size_t words = w->matrices * m.strips * (size_t)m.blocks * (F8_PIECE / 16);
    const bool whole = w->cols % 16 == 0 && (uintptr_t)src % 16 == 0;
    hipLaunchKernelGGL(f8_repack_kernel, dim3((unsigned)std::min<size_t>((words + 255) / 256, 1 << 20)), dim3(256), 0, s, src, w->dev, m, w->cols,
                       words, whole);
    FRK_LAUNCH_CHECK("f8_repack");
    const size_t n = w->matrices * m.row_blocks * (size_t)m.blocks;
    hipLaunchKernelGGL(f8_scales_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, 4096)), dim3(256), 0, s, scales,
                       reinterpret_cast<float *>(w->dev + w->layout.off_a), n);
    FRK_LAUNCH_CHECK("f8_scales");
    return FRK_OK;
}

// out[i] = row (ids ? ids[i] : i) of the stack; a code times its scale, one rounding
__global__ __launch_bounds__(256) void f8_dequant_kernel(F8Mat w, size_t all_rows, const int32_t *__restrict__ ids, size_t n_out, int cols,
                                                         float *__restrict__ out) {
    const size_t total = n_out * (size_t)cols;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const size_t o = i / cols;
        const int k = (int)(i % cols);
        const size_t row = ids ? (size_t)min(max((long long)ids[o], 0ll), (long long)all_rows - 1) : o;
        const size_t m = row / w.rows;
        const int r = (int)(row % w.rows);
#if defined(__HIP_DEVICE_COMPILE__)
        const float code = __builtin_amdgcn_cvt_f32_fp8((int)w.q[f8_at(w, m, r, k)], 0);
#else
        const float code = 0.0f;
#endif
        out[i] = code * w.s[(m * w.row_blocks + r / F8_BLOCK) * w.blocks + k / F8_BLOCK];
    }
}
int launch_f8_dequant_rows(const frk_weights *w, const int32_t *ids, size_t n_out, float *out, hipStream_t s) {
    if (n_out == 0) return FRK_OK;
    const size_t n = n_out * w->cols;
    hipLaunchKernelGGL(f8_dequant_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1 << 20)), dim3(256), 0, s, f8_mat(w), w->rows, ids,
                       n_out, (int)w->cols, out);
    FRK_LAUNCH_CHECK("f8_dequant");
    return FRK_OK;
}

// ---- quantization of a batch: a wavefront eight blocks of a row ----
template <bool WIDE>
__global__ __launch_bounds__(256) void f8_quantize_kernel(const float *__restrict__ x, const float *__restrict__ up, size_t jobs, int parts, int cols,
                                                          int blocks, const int *__restrict__ used, F8Acts out) {
    const int lane = threadIdx.x & 63;
    for (size_t j = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); j < jobs; j += (size_t)gridDim.x * 4) {
        const size_t row = j / parts;
        if (used && used[row] < 0) continue;
        f8_quantize_blocks<WIDE>(x, up, row, (int)(j % parts) * F8_QUANTIZE_BLOCKS, cols, blocks, lane, out);
    }
}
int launch_f8_quantize(const float *x, const float *up, size_t rows, size_t cols, const int *used, const F8Acts &out, hipStream_t s) {
    const int blocks = (int)f8_blocks(cols), parts = (blocks + F8_QUANTIZE_BLOCKS - 1) / F8_QUANTIZE_BLOCKS;
    const size_t jobs = rows * parts;
    if (jobs == 0) return FRK_OK;
    const dim3 grid((unsigned)std::min<size_t>((jobs + 3) / 4, 1 << 16));
    const bool wide = f8_wide_rows(x, cols) && (!up || f8_wide_rows(up, cols));
    if (wide) hipLaunchKernelGGL(f8_quantize_kernel<true>, grid, dim3(256), 0, s, x, up, jobs, parts, (int)cols, blocks, used, out);
    else hipLaunchKernelGGL(f8_quantize_kernel<false>, grid, dim3(256), 0, s, x, up, jobs, parts, (int)cols, blocks, used, out);
    FRK_LAUNCH_CHECK("f8_quantize");
    return FRK_OK;
}

// ---- the GEMM.  A workgroup of eight wavefronts has one strip of sixteen weight rows and up to 16 TT tokens; its wavefronts
// share the columns, in order, and their sums meet in LDS. ----
constexpr int F8_WAVES = 8;
constexpr int F8_MAX_TOKENS = 64;  // of a workgroup
template <int TT>
__global__ __launch_bounds__(64 * F8_WAVES) void f8_gemm_kernel(F8Gemm g) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ float4 sums[F8_WAVES][TT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int strip = (int)(blockIdx.x % (unsigned)g.w.strips), t_index = (int)(blockIdx.x / (unsigned)g.w.strips);
    int4 tile;
    size_t y_col;  // of the matrix's first row
    if (g.tiles) {
        if (t_index >= *g.n_tiles) return;
        tile = g.tiles[t_index];
        y_col = 0;
    } else {
        const int first = t_index * 16 * TT;
        tile = make_int4((int)blockIdx.y, first, min(16 * TT, g.M - first), first);
        y_col = (size_t)blockIdx.y * g.w.rows;
    }
    const int b0 = g.w.blocks * wave / F8_WAVES, b1 = g.w.blocks * (wave + 1) / F8_WAVES;
    const uint8_t *wq = g.w.q + (((size_t)tile.x * g.w.strips + strip) * g.w.blocks) * F8_PIECE + lane * 16;
    const float *ws = g.w.s + ((size_t)tile.x * g.w.row_blocks + strip * F8_STRIP / F8_BLOCK) * g.w.blocks;
    int row[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
        const int i = tile.y + min(16 * t + (lane & 15), tile.z - 1);
        row[t] = min(max(g.src ? g.src[i] : i, 0), g.a.rows - 1);
    }
    f8_v4f acc[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) acc[t] = f8_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    auto operand = [](uint32_t lo, uint32_t hi) {
        const uint2 a = f8_to_bf16(lo, 1.0f), b = f8_to_bf16(hi, 1.0f);
        const uint4 v = make_uint4(a.x, a.y, b.x, b.y);
        f8_v8bf o;
        __builtin_memcpy(&o, &v, 16);
        return o;
    };
    for (int b = b0; b < b1; b++) {
        const uint4 w0 = *reinterpret_cast<const uint4 *>(wq + (size_t)b * F8_PIECE), w1 = *reinterpret_cast<const uint4 *>(wq + (size_t)b * F8_PIECE + 1024);
        const f8_v8bf w[4] = {operand(w0.x, w0.y), operand(w0.z, w0.w), operand(w1.x, w1.y), operand(w1.z, w1.w)};
        const float s = ws[b];
#pragma unroll
        for (int t = 0; t < TT; t++) {
            const f8_v8bf *x = reinterpret_cast<const f8_v8bf *>(g.a.v + ((size_t)row[t] * g.w.blocks + b) * F8_BLOCK + (lane >> 4) * 32);
            f8_v4f p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 4; k++) p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[k], x[k], p, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) acc[t][r] = __builtin_fmaf(p[r], s, acc[t][r]);
        }
    }
#pragma unroll
    for (int t = 0; t < TT; t++) sums[wave][t][lane] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
    __syncthreads();
    for (int i = threadIdx.x; i < TT * 64; i += 64 * F8_WAVES) {
        const int t = i >> 6, l = i & 63, tok = 16 * t + (l & 15);
        float4 v = sums[0][t][l];
#pragma unroll
        for (int k = 1; k < F8_WAVES; k++) {
            const float4 o = sums[k][t][l];
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
        if (tok >= tile.z) continue;
        const int r0 = strip * F8_STRIP + 4 * (l >> 4);
        float *dst = g.y + (size_t)(tile.w + tok) * g.ldy + y_col;
        const float out[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (r0 + r < g.w.rows) dst[r0 + r] = out[r];
    }
#endif
}

size_t f8_gemm_workspace_bytes(const frk_weights *w, size_t batch) { return f8_acts_bytes(batch, w->cols); }
int launch_f8_gemm(const frk_weights *w, const float *x, size_t batch, float *y, void *ws, hipStream_t s) {
    F8Gemm g{};
    g.w = f8_mat(w);
    g.a = f8_acts_carve(ws, batch);
    g.M = (int)batch;
    g.ldy = w->rows;
    g.y = y;
    int rc = launch_f8_quantize(x, nullptr, batch, w->cols, nullptr, g.a, s);
    if (rc) return rc;
    const size_t tok_tiles = (batch + F8_MAX_TOKENS - 1) / F8_MAX_TOKENS;
    const size_t jobs = g.w.strips * tok_tiles;
    if (jobs > 0x7fffffffu || w->matrices > 65535) return set_error(FRK_ERR_SHAPE, "%zu rows over %zu matrices of %d: too many", batch, w->matrices, g.w.rows);
    const dim3 grid((unsigned)jobs, (unsigned)w->matrices);
    if (batch > 64) return launch_f8_tile(g, 128, (batch + 127) / 128, w->matrices, 1, 0, s);
    if (batch <= 16) hipLaunchKernelGGL(f8_gemm_kernel<1>, grid, dim3(64 * F8_WAVES), 0, s, g);
    else if (batch <= 32) hipLaunchKernelGGL(f8_gemm_kernel<2>, grid, dim3(64 * F8_WAVES), 0, s, g);
    else hipLaunchKernelGGL(f8_gemm_kernel<4>, grid, dim3(64 * F8_WAVES), 0, s, g);
    FRK_LAUNCH_CHECK("f8_gemm");
    return FRK_OK;
}

// ---- grouped: the tile list of the groups given.  Offsets are clamped to 0 .. pairs and made non-decreasing (each the largest
// so far), so the tiles are at most pairs / tokens + groups whatever the list holds.  One workgroup of 1024 threads, a group each. ----
__global__ __launch_bounds__(1024) void f8_tiles_kernel(const int32_t *__restrict__ group_off, int n_groups, int pairs, int tokens, int4 *__restrict__ tiles,
                                                        int *__restrict__ n_tiles) {
    __shared__ int off[1025], at[1025];
    const int tid = threadIdx.x;
    for (int g = tid; g <= n_groups; g += 1024) off[g] = min(max(group_off[g], 0), pairs);
    __syncthreads();
    if (tid == 0) {
        int top = 0, n = 0;
        for (int g = 0; g <= n_groups; g++) {
            const int from = top;
            top = max(top, off[g]);
            if (g) {
                at[g - 1] = n;
                n += (top - from + tokens - 1) / tokens;
            }
            off[g] = top;
        }
        *n_tiles = n;
    }
    __syncthreads();
    if (tid < n_groups) {
        const int n = off[tid + 1] - off[tid];
        for (int i = 0; i * tokens < n; i++)
            tiles[at[tid] + i] = make_int4(tid, off[tid] + i * tokens, min(tokens, n - i * tokens), off[tid] + i * tokens);
    }
}
static size_t f8_max_tiles(size_t pairs, size_t groups, int tokens) { return pairs / (size_t)tokens + std::min(groups, pairs); }
static int f8_tile_tokens(size_t pairs, size_t groups) {
    const size_t mean = pairs / groups;
    return mean >= 96 ? 128 : mean >= 16 ? 64 : 32;
}
size_t f8_grouped_workspace_bytes(const frk_weights *w, size_t x_rows, size_t pairs) {
    return f8_acts_bytes(x_rows, w->cols) + 256 + f8_max_tiles(pairs, w->matrices, 32) * 16;
}
int launch_f8_tiles(const frk_weights *w, const F8Acts &acts, int tokens, const int *src, const int4 *tiles, const int *n_tiles, size_t max_tiles, float *y,
                    hipStream_t s) {
    F8Gemm g{};
    g.w = f8_mat(w);
    g.a = acts;
    g.src = src;
    g.tiles = tiles;
    g.n_tiles = n_tiles;
    g.ldy = g.w.rows;
    g.y = y;
    return launch_f8_tile(g, tokens, max_tiles, 1, 1, 0, s);
}
int launch_f8_grouped(const frk_weights *w, const int32_t *group_off, const int32_t *gather, const float *x, size_t x_rows, size_t pairs,
                      float *y, void *ws, hipStream_t s) {
    const F8Acts acts = f8_acts_carve(ws, x_rows);
    const int tokens = f8_tile_tokens(pairs, w->matrices);
    int *n_tiles = (int *)((char *)ws + f8_acts_bytes(x_rows, w->cols));
    int4 *tiles = (int4 *)(n_tiles + 64);
    int rc = launch_f8_quantize(x, nullptr, x_rows, w->cols, nullptr, acts, s);
    if (rc) return rc;
    hipLaunchKernelGGL(f8_tiles_kernel, dim3(1), dim3(1024), 0, s, group_off, (int)w->matrices, (int)pairs, tokens, tiles, n_tiles);
    FRK_LAUNCH_CHECK("f8_tile_list");
    return launch_f8_tiles(w, acts, tokens, gather, tiles, n_tiles, f8_max_tiles(pairs, w->matrices, tokens), y, s);
}

}  // namespace frk
