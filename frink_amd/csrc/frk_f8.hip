// Products with weights in 8-bit floating point, a scale for each block of 128 x 128 (frk_f8.hpp has the mathematics and the
// layouts): registration, the dequantizer, the activations' quantization and the GEMM, dense and grouped.  The reference has no
// such kind; its entry points' shapes are those of the others (include/frink_hip.h).
#include "frk_f8.hpp"

#include <algorithm>
#include <cmath>

namespace frk {

typedef __bf16 f8_v8bf __attribute__((ext_vector_type(8)));
typedef float f8_v4f __attribute__((ext_vector_type(4)));

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

int f8_on_current_device(const frk_weights *w) {
    int dev = -1;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return set_error(FRK_ERR_HIP, "hipGetDevice: %s", hipGetErrorString(e));
    if (dev != w->device) return set_error(FRK_ERR_ARG, "the matrix is on device %d, the current device is %d", w->device, dev);
    return FRK_OK;
}

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
    int rc = f8_on_current_device(w);
    if (rc) return rc;
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

// ---- A few tokens: the weights' bytes and the launch's own chain of steps bound it.  A workgroup of NW wavefronts has one strip of sixteen
// weight rows and up to 16 TT tokens; its wavefronts share the columns, in order, straight from memory into registers, D blocks
// ahead, and their sums meet in LDS.
//   DENSE  strip blockIdx.x, matrix blockIdx.y, all tokens
//   PAIRS  strip blockIdx.x, pair blockIdx.y of a grouped product: every sixteenth (FUSED: fourth) pair of its group takes the
//          group's next sixteen (four), the others end at once.  No list is made in front of it: each wavefront looks the group up itself
//   SLOTS  strip blockIdx.x, (token, slot) blockIdx.y of an expert layer: the matrix is the slot's expert (FUSED only).  With `up` the strip of
//          both stacks, and y = silu(gate) * up
// FUSED: a few tokens (PAIRS: F8_FUSED) are quantized by the workgroup itself (a wavefront its own columns', while its first codes
// are on their way), not by a launch in front. ----
enum { F8_DENSE = 0, F8_PAIRS = 1, F8_SLOTS = 2, F8_SLOTS_GLU = 3 };
struct F8Rows {
    F8Mat w, up;        // up: SLOTS_GLU
    F8Acts a;           // not FUSED
    const float *x;     // FUSED
    int cols, x_rows;
    int M;                          // DENSE
    const int *group_off, *gather;  // PAIRS
    int n_groups, pairs;
    const int *ids;                 // SLOTS: experts, of n_groups; a slot's activation row is slot / slots_a_row
    int slots_a_row;
    size_t ldy;
    float *y;
};
constexpr size_t F8_FUSED = 4;
constexpr size_t F8_FUSED_LDS = 56 * 1024;  // beside the 8 KB of sums: what a launch may have without more ado

// the range of up to `most` pairs that pair `p` leads, by the offsets clamped and made non-decreasing (each the largest so far): {group, first, number};
// a number of 0: it leads none
__device__ __forceinline__ int4 f8_lead(const int *__restrict__ off, int n_groups, int pairs, int p, int most, int lane) {
    int begin = 0;  // a lane's part of the largest before
    for (int i0 = 0; i0 <= n_groups; i0 += 256) {
        // 256 at once: one trip to memory for most lists (eight pairs of 128 groups of 768 x 2048: the kernel 6.9 -> 6.6 us, sixteen 9.7 -> 8.0)
        int v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = i0 + 64 * j + lane <= n_groups ? off[i0 + 64 * j + lane] : 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[j] = min(max(v[j], 0), pairs);
            const uint64_t above = __ballot(v[j] > p);
            if (above) {  // (uniform) the first offset above p ends the pair's group
                const int first = __builtin_ctzll(above), after = i0 + 64 * j + first, end = __builtin_amdgcn_readlane(v[j], first);
                const int half = (int)f8_half_max((uint32_t)max(begin, lane < first ? v[j] : 0));
                begin = max(__builtin_amdgcn_readlane(half, 0), __builtin_amdgcn_readlane(half, 32));
                if (after == 0 || (p - begin) % most) return make_int4(0, 0, 0, 0);
                return make_int4(after - 1, p, min(most, end - p), 0);
            }
            begin = max(begin, v[j]);
        }
    }
    return make_int4(0, 0, 0, 0);
}

template <int NW, int TT, int D, bool FUSED, int MODE, bool WIDE>
__global__ __launch_bounds__(64 * NW) void f8_rows_kernel(F8Rows g) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool PAIRS = MODE == F8_PAIRS, SLOTS = MODE == F8_SLOTS || MODE == F8_SLOTS_GLU;
    constexpr int NM = MODE == F8_SLOTS_GLU ? 2 : 1;  // stacks
    static_assert(MODE == F8_DENSE || TT == 1, "sixteen pairs");
    static_assert(!SLOTS || FUSED, "a slot's row");
    extern __shared__ __align__(16) uint8_t f8_rows_lds[];  // FUSED: [blocks][tokens][128] bf16
    __shared__ float4 sums[NW][NM * TT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int strip = blockIdx.x, blocks = g.w.blocks;
    int matrix, first, used;
    size_t y_col = 0;
    if (PAIRS) {
        const int4 lead = f8_lead(g.group_off, g.n_groups, g.pairs, (int)blockIdx.y, FUSED ? (int)F8_FUSED : 16, lane);
        matrix = __builtin_amdgcn_readfirstlane(lead.x), first = __builtin_amdgcn_readfirstlane(lead.y), used = __builtin_amdgcn_readfirstlane(lead.z);
        if (used == 0) return;
    } else if (SLOTS) {
        matrix = g.ids ? g.ids[blockIdx.y] : 0, first = blockIdx.y, used = 1;
        if (matrix < 0 || matrix >= g.n_groups) return;  // (adds nothing to its token)
    } else {
        matrix = blockIdx.y, first = 0, used = min(16 * TT, g.M);
        y_col = (size_t)matrix * g.w.rows;
    }
    const int b0 = (int)((long long)blocks * wave / NW), b1 = (int)((long long)blocks * (wave + 1) / NW);
    const uint8_t *wq[NM];
    const float *ws[NM];
#pragma unroll
    for (int m = 0; m < NM; m++) {
        const F8Mat &w = m ? g.up : g.w;
        wq[m] = w.q + (((size_t)matrix * w.strips + strip) * blocks) * F8_PIECE + lane * 16;
        ws[m] = w.s + ((size_t)matrix * w.row_blocks + strip * F8_STRIP / F8_BLOCK) * blocks;
    }
    // this lane's activation rows; lanes past the last token read its (eight tokens of 14336 x 4096: 15.8 us, with sixteen's traffic 19.2)
    int row[TT], token[TT];
#pragma unroll
    for (int t = 0; t < TT; t++) {
        token[t] = (lane & 48) + min(lane & 15, max(used - 1 - 16 * t, 0));
        const int i = first + min(16 * t + (lane & 15), used - 1);
        row[t] = SLOTS ? i / g.slots_a_row : min(max(PAIRS && g.gather ? g.gather[i] : i, 0), g.x_rows - 1);
    }
    f8_v4f acc[NM * TT];
#pragma unroll
    for (int t = 0; t < NM * TT; t++) acc[t] = f8_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (b0 < b1) {
        // the next 64 blocks' scales, one a lane (a scalar load a block is waited for with the one just asked for)
        float scales[NM];
#pragma unroll
        for (int m = 0; m < NM; m++) scales[m] = ws[m][min(b0 + lane, b1 - 1)];
        __builtin_amdgcn_sched_barrier(0);  // (first, so that its wait is not one for the codes)
        auto next_scales = [&](int b) {
            if (b == b0 || ((b - b0) & 63)) return;
#pragma unroll
            for (int m = 0; m < NM; m++)
                asm volatile("global_load_dword %0, %1, %2\n\ts_waitcnt vmcnt(0)" : "=v"(scales[m]) : "v"((uint32_t)min(b + lane, b1 - 1) * 4u), "s"(ws[m]) : "memory");
        };
        static_assert(64 % D == 0, "whole rounds");
        uint4 w[D][NM][2], x[FUSED ? 1 : D][TT][4];
        auto fetch_w = [&](int u, int b) {
            // (past the last-level cache, as weights met once a step are: 3 to 7 % faster than plain loads on matrices that aren't in it)
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const uint8_t *const at = wq[m] + (size_t)min(b, b1 - 1) * F8_PIECE;
                w[u][m][0] = stream_load16(at);
                w[u][m][1] = stream_load16(at + 1024);
            }
        };
        auto fetch_x = [&](int u, int b) {
#pragma unroll
            for (int t = 0; t < TT; t++) {
                const size_t piece = PAIRS ? (size_t)row[t] * blocks + min(b, b1 - 1) : ((size_t)min(t, (g.x_rows - 1) >> 4) * blocks + min(b, b1 - 1)) * F8_STRIP;
                const uint4 *const at = reinterpret_cast<const uint4 *>(g.a.v + piece * F8_BLOCK) + (PAIRS ? (lane >> 4) * 4 : token[t]);
#pragma unroll
                for (int k = 0; k < 4; k++) x[u][t][k] = at[PAIRS ? k : k * 64];
            }
        };
        uint16_t *const own = reinterpret_cast<uint16_t *>(f8_rows_lds) + (size_t)b0 * used * F8_BLOCK;  // FUSED: [block - b0][token][128]
        if (FUSED) {
            constexpr int N = 4;  // pairs of blocks a pass
            float v[N][4];
            auto load = [&](int t, int at) {
                const float *const xr = g.x + (size_t)__builtin_amdgcn_readlane(row[0], t) * g.cols;
#pragma unroll
                for (int i = 0; i < N; i++) f8_load4<WIDE>(xr, (at + 2 * i) * F8_BLOCK + lane * 4, min(g.cols, b1 * F8_BLOCK), v[i]);
            };
            auto store = [&](int t, int at) {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (at + 2 * i >= b1) break;  // (uniform)
                    float scale;
                    const uint32_t codes = f8_quantize4(v[i], scale);
                    const int b = at + 2 * i + (lane >> 5);
                    if (b < b1) *reinterpret_cast<uint2 *>(own + ((size_t)(b - b0) * used + t) * F8_BLOCK + (lane & 31) * 4) = f8_to_bf16(codes, scale);
                }
            };
            load(0, b0);
#pragma unroll
            for (int u = 0; u < D; u++) fetch_w(u, b0 + u);
            store(0, b0);
            for (int t = 0, at = b0 + 2 * N; t < used; t++, at = b0)
                for (; at < b1; at += 2 * N) {
                    load(t, at);
                    store(t, at);
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wavefront reads its own stores only)
        } else {
#pragma unroll
            for (int u = 0; u < D; u++) fetch_w(u, b0 + u), fetch_x(u, b0 + u);
        }
        const uint16_t *const own_lane = own + min(lane & 15, used - 1) * F8_BLOCK + (lane >> 4) * 32;
        auto consume = [&](int u, int b) {
#pragma unroll
            for (int m = 0; m < NM; m++) {
                const float by = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scales[m]), (b - b0) & 63));
                f8_v8bf wv[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint4 &raw = w[u][m][k >> 1];
                    const uint2 lo = f8_to_bf16(k & 1 ? raw.z : raw.x, 1.0f), hi = f8_to_bf16(k & 1 ? raw.w : raw.y, 1.0f);
                    const uint4 both = make_uint4(lo.x, lo.y, hi.x, hi.y);
                    __builtin_memcpy(&wv[k], &both, 16);
                }
#pragma unroll
                for (int t = 0; t < TT; t++) {
                    f8_v4f p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        f8_v8bf xv;
                        if (FUSED) xv = *reinterpret_cast<const f8_v8bf *>(own_lane + (size_t)(b - b0) * used * F8_BLOCK + k * 8);
                        else __builtin_memcpy(&xv, &x[u][t][k], 16);
                        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[k], xv, p, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[m * TT + t][r] = __builtin_fmaf(p[r], by, acc[m * TT + t][r]);
                }
            }
        };
        // Requests without a branch around them, so that the wait for a block counts those behind it; and no branch between a product
        // and the reads of its sum: the compiler does not count its wait states across one that splits and joins.
        int b = b0;
        for (; b + 2 * D <= b1; b += D) {
            next_scales(b);
#pragma unroll
            for (int u = 0; u < D; u++) {
                consume(u, b + u);
                fetch_w(u, b + u + D);
                if (!FUSED) fetch_x(u, b + u + D);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        for (; b < b1; b += D) {
            next_scales(b);
#pragma unroll
            for (int u = 0; u < D; u++) {
                if (b + u >= b1) break;  // (uniform)
                consume(u, b + u);
#pragma unroll
                for (int t = 0; t < NM * TT; t++) asm volatile("" : "+v"(acc[t]));
                if (b + u + D < b1) {
                    fetch_w(u, b + u + D);
                    if (!FUSED) fetch_x(u, b + u + D);
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NM * TT; t++) sums[wave][t][lane] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
    __syncthreads();
    const int last_wave = min(NW, TT);  // a wavefront a tile of tokens
    if (wave >= last_wave) return;
    const int t = wave, tok = 16 * t + (lane & 15);
    auto total = [&](int i) {
        float4 v = sums[0][i][lane];
#pragma unroll
        for (int k = 1; k < NW; k++) {
            const float4 o = sums[k][i][lane];
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
        }
        return make_float4(v.x * F8_UP, v.y * F8_UP, v.z * F8_UP, v.w * F8_UP);
    };
    float4 v = total(t);
    if (NM == 2) {
        const float4 u = total(TT);  // (TT is 1)
        v = make_float4(silu_as_host(v.x) * u.x, silu_as_host(v.y) * u.y, silu_as_host(v.z) * u.z, silu_as_host(v.w) * u.w);
    }
    if (tok >= used) return;
    const int r0 = strip * F8_STRIP + 4 * (lane >> 4);
    float *const dst = g.y + (size_t)(first + tok) * g.ldy + y_col;
    const float out[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int r = 0; r < 4; r++)
        if (r0 + r < g.w.rows) dst[r0 + r] = out[r];
#endif
}

template <int NW, int TT, int D, bool FUSED, int MODE>
static int go_f8_rows(const F8Rows &g, const dim3 &grid, size_t lds, hipStream_t s) {
    // (WIDE: how a FUSED one reads x)
    if (FUSED && f8_wide_rows(g.x, (size_t)g.cols)) hipLaunchKernelGGL((f8_rows_kernel<NW, TT, D, FUSED, MODE, FUSED>), grid, dim3(64 * NW), lds, s, g);
    else hipLaunchKernelGGL((f8_rows_kernel<NW, TT, D, FUSED, MODE, false>), grid, dim3(64 * NW), lds, s, g);
    FRK_LAUNCH_CHECK("f8_rows");
    return FRK_OK;
}

constexpr size_t F8_ROWS_TOKENS = 64;  // most of the rows kernel
static bool f8_fused_fits(size_t tokens, size_t cols) { return tokens * f8_blocks(cols) * F8_BLOCK * 2 <= F8_FUSED_LDS; }
// Of a dense batch: up to four tokens; up to eight where the strips are one round of the chip and a token's quantization, which every workgroup
// does, is short.  In us, so / with a launch for it (rows x columns): 4096 x 4096 one token 5.6 / 8.7, four 7.6 / 9.1, six 9.0 / 9.2; 2880 x 2880 four 6.6 / 8.4, six
// 8.0 / 8.6, eight 9.2 / 8.8; 768 x 2048 eight 6.8 / 7.9, twelve 8.5 / 8.2; 14336 x 4096 (3.5 rounds) one 11.5 / 15.9, four 15.8 / 16.2, six 20.8 / 16.3.
static bool f8_fused(size_t tokens, const frk_weights *w, const F8Mat &m) {
    if (!f8_fused_fits(tokens, w->cols)) return false;
    return tokens <= F8_FUSED || (tokens <= 2 * F8_FUSED && (size_t)m.strips * w->matrices <= 256 && tokens * w->cols <= 20480);
}

// By estimated time.  Both kernels are a chain of steps a wavefront until the chip is full: a block of 128 columns takes a tile's wavefronts
// as long alone on a CU as beside the CU's other workgroups, up to how many fit; a strip of the rows kernel likewise.  Shares of the
// columns cost a second launch, 3.3 us, and the traffic of the parts.  Every kernel, tile and number of shares timed at 35 sizes (24 to 4096
// tokens, 576 x 7168 to 14336 x 4096): the choice is within 4 % of the fastest but for 512 tokens of 4096 x 14336 (74 against 71 us), 1500 of 2048 x 2048 (27.7
// against 26.1) and 384 of 4096 x 4096 (32.2 against 28.8).
F8Plan f8_plan(const frk_weights *w, size_t batch) {
    const F8Mat m = f8_mat(w);
    F8Plan best{-1, 1, f8_fused(batch, w, m), 0, 0};
    if (best.fused) return best;
    best.acts_bytes = f8_acts_bytes(batch, w->cols);
    if (batch <= 16) return best;  // (the tiles hold 32 tokens and more)
    double least = 1e30;
    if (batch <= F8_ROWS_TOKENS) {
        const double rounds = std::max(1.0, (double)(m.strips * w->matrices) / 256.0);
        least = 5.0 + rounds * std::max(0.5, m.blocks / 32.0) * (batch <= 32 ? 5.5 : 9.0);
    }
    static constexpr struct {
        double slots, alone, full;  // workgroups of the chip; us a block
    } COST[F8_TILE_SHAPES] = {{256, 1.36, 1.60}, {512, 0.87, 1.72}, {1024, 0.68, 1.30}};
    static constexpr int SHARES[] = {1, 2, 3, 4, 6, 8, 12, 16};
    const size_t n = batch * w->rows;
    for (int shape = 0; shape < F8_TILE_SHAPES; shape++)
        for (int parts : SHARES) {
            if (parts > 1 && (parts > m.blocks / 2 || parts * n * 4 > SPLIT_PARTS_BYTES)) break;
            const F8TileSize t = F8_TILE_SIZE[shape];
            const double groups = (double)((m.rows + t.rows - 1) / t.rows) * (double)((batch + t.tokens - 1) / t.tokens) * (double)w->matrices * parts;
            const double fill = groups / COST[shape].slots, whole = std::floor(fill + 0.02), rest = fill - whole;
            // a round that isn't full: as long as the workgroups are (nearly) alone on their CUs, then the fullest CU counts
            static constexpr double HALF[F8_TILE_SHAPES] = {0.0, 0.5, 0.35}, JUMP[F8_TILE_SHAPES] = {0.0, 0.6, 0.0};
            const double alone = COST[shape].alone, full = COST[shape].full, half = HALF[shape], jump = JUMP[shape];
            const double partly = rest <= half ? alone : alone + (full - alone) * (jump + (1.0 - jump) * (rest - half) / (1.0 - half));
            const double chain = (double)((m.blocks + parts - 1) / parts);
            double us = 7.0 + whole * (chain * full + 1.0) + (rest > 0.0 ? chain * partly + 1.0 : 0.0);
            if (parts > 1) us += 3.3 + 0.45e-6 * 4.0 * (double)n * parts;
            if (us < least) {
                least = us;
                best.shape = shape;
                best.parts = parts;
            }
        }
    if (best.parts > 1) best.parts_bytes = best.parts * n * 4;
    return best;
}
int launch_f8_gemm(const frk_weights *w, const F8Plan &plan, const float *x, size_t batch, float *y, void *ws, bool quantized, void *parts, hipStream_t s) {
    const F8Mat m = f8_mat(w);
    const F8Acts acts = f8_acts_carve(ws, batch, plan.shape < 0);
    if (!plan.fused && !quantized) {
        int rc = launch_f8_quantize(x, nullptr, batch, w->cols, nullptr, acts, s);
        if (rc) return rc;
    }
    if (plan.shape >= 0) {
        F8Gemm g{};
        g.w = m;
        g.a = acts;
        g.M = (int)batch;
        g.ldy = w->rows;
        const size_t n = batch * w->rows, tokens = (size_t)F8_TILE_SIZE[plan.shape].tokens;
        g.y = plan.parts > 1 ? (float *)parts : y;
        int rc = launch_f8_tile(g, plan.shape, (batch + tokens - 1) / tokens, w->matrices, plan.parts, n, s);
        if (rc || plan.parts == 1) return rc;
        return launch_sum_parts((const float *)parts, plan.parts, n, y, s);
    }
    F8Rows g{};
    g.w = m;
    g.a = acts;
    g.x = x;
    g.cols = (int)w->cols;
    g.x_rows = g.M = (int)batch;
    g.ldy = w->rows;
    g.y = y;
    const dim3 grid((unsigned)m.strips, (unsigned)w->matrices);
    if (plan.fused) return go_f8_rows<8, 1, 4, true, F8_DENSE>(g, grid, batch * m.blocks * F8_BLOCK * 2, s);
    if (batch <= 16) return go_f8_rows<8, 1, 4, false, F8_DENSE>(g, grid, 0, s);
    if (batch <= 32) return go_f8_rows<8, 2, 2, false, F8_DENSE>(g, grid, 0, s);
    return go_f8_rows<8, 4, 1, false, F8_DENSE>(g, grid, 0, s);
}

// ---- grouped: the tile list of the groups given.  Offsets are clamped to 0 .. pairs and made non-decreasing (each the largest
// so far), so the tiles are at most pairs / tokens + groups whatever the list holds.  1024 threads, a group each. ----
struct F8TilesArgs {
    const int32_t *group_off;
    int n_groups, pairs, tokens;
    int4 *tiles;
    int *n_tiles;
};
__device__ __forceinline__ void f8_tile_list(const F8TilesArgs &a) {
    __shared__ int wave_top[16], wave_sum[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the largest offset up to and with this group's first, and with its end
    const int mine = tid < a.n_groups ? min(max(a.group_off[tid], 0), a.pairs) : 0;
    const int end = tid < a.n_groups ? min(max(a.group_off[tid + 1], 0), a.pairs) : 0;
    int top = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(top, m);
        if (lane >= m) top = max(top, o);
    }
    if (lane == 63) wave_top[wave] = top;
    __syncthreads();
    for (int w = 0; w < wave; w++) top = max(top, wave_top[w]);
    const int n = tid < a.n_groups ? max(end - top, 0) : 0, tiles = (n + a.tokens - 1) / a.tokens;
    int sum = tiles;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(sum, m);
        if (lane >= m) sum += o;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int at = sum - tiles, total = 0;
    for (int w = 0; w < 16; w++) {
        if (w < wave) at += wave_sum[w];
        total += wave_sum[w];
    }
    for (int i = 0; i < tiles; i++) a.tiles[at + i] = make_int4(tid, top + i * a.tokens, min(a.tokens, n - i * a.tokens), top + i * a.tokens);
    if (tid == 0) *a.n_tiles = total;
}
// beside the quantization, which does not depend on it: workgroup 0 makes the list
template <bool WIDE>
__global__ __launch_bounds__(1024) void f8_tiles_quantize_kernel(F8TilesArgs a, const float *__restrict__ x, size_t jobs, int parts, int cols, int blocks,
                                                                 F8Acts out) {
    if (blockIdx.x == 0) {
        f8_tile_list(a);
        return;
    }
    const int lane = threadIdx.x & 63;
    for (size_t j = (size_t)(blockIdx.x - 1) * 16 + (threadIdx.x >> 6); j < jobs; j += (size_t)(gridDim.x - 1) * 16)
        f8_quantize_blocks<WIDE>(x, nullptr, j / parts, (int)(j % parts) * F8_QUANTIZE_BLOCKS, cols, blocks, lane, out);
}
static size_t f8_max_tiles(size_t pairs, size_t groups, int tokens) { return pairs / (size_t)tokens + std::min(groups, pairs); }
// Measured in us with tiles of 256x128 / 256x64 / 128x32 (weight rows x pairs): 32 groups of 2880 x 2880 and 256 pairs each on average 188 / 180 / 243, 64
// 95 / 98 / 96, 32 88 / 68 / 75, 16 85 / 64 / 60; 128 of 768 x 2048 and 128 pairs 108 / 85 / 105, 32 68 / 54 / 59, 16 64 / 50 / 46, 4 63 / 47 / 42.
// Large groups, 256x128 / 256x64: 32 of 2880 x 2880 and 1024 pairs 612 / 590, 8 of 1792 x 4096 and 512 105 / 68, 1024 123 / 121, 8 of 14336 x 4096 and 512 483 / 475,
// 1024 889 / 896, 4 of 4096 x 4096 and 2048 269 / 247.
int f8_grouped_shape(size_t pairs, size_t groups) { return pairs >= 24 * groups ? F8_TILE_256x64 : F8_TILE_128x32; }
// A few pairs: a launch that looks the groups up itself.  In us, so / by tiles, a token's pairs over different groups: 128 groups of 768 x 2048, 16 pairs 8.0 /
// 16.5, 32 14.5 / 16.9, 48 19.6 / 20.3, 64 24.2 / 23.0; 32 of 2880 x 2880, 16 pairs 25.0 / 33.2, 32 40.1 / 39.8, 48 53.4 / 49.8; 8 of 1792 x 4096, 16 15.0 / 26.0.
static bool f8_few_pairs(size_t pairs, size_t groups) { return pairs <= 32 && groups >= pairs / 2; }
// Of an expert layer: each slot by itself, its row quantized by the workgroups that read it.  The layer in us, so / bucketed: 32 experts of 2880 x 2880, 4
// slots 25 / 65, 16 77 / 95, 24 108 / 99, 32 140 / 106; 128 of 768 x 2048, 8 slots 20 / 45, 24 39 / 49, 32 48 / 51, 48 66 / 58; 8 of 1792 x 4096, 8 slots 37 / 70.
bool f8_slots_fit(size_t cols) { return f8_blocks(cols) * F8_BLOCK * 2 <= F8_FUSED_LDS - 8 * 1024; }  // (8 KB more of sums)
bool f8_few_slots(size_t slots, size_t experts, size_t hidden, size_t ffn) { return slots <= 24 && f8_few_pairs(slots, experts) && f8_slots_fit(std::max(hidden, ffn)); }
int launch_f8_slots(const frk_weights *w, const frk_weights *up, const int32_t *ids, size_t slots, int slots_a_row, const float *x, float *y, hipStream_t s) {
    F8Rows g{};
    g.w = f8_mat(w);
    if (up) g.up = f8_mat(up);
    g.x = x;
    g.cols = (int)w->cols;
    g.ids = ids;
    g.n_groups = (int)w->matrices;
    g.slots_a_row = slots_a_row;
    g.ldy = g.w.rows;
    g.y = y;
    const dim3 grid((unsigned)g.w.strips, (unsigned)slots);
    const size_t lds = (size_t)g.w.blocks * F8_BLOCK * 2;
    return up ? go_f8_rows<8, 1, 4, true, F8_SLOTS_GLU>(g, grid, lds, s) : go_f8_rows<8, 1, 4, true, F8_SLOTS>(g, grid, lds, s);
}
int f8_grouped_fits(const frk_weights *w, size_t x_rows, size_t pairs, bool gathered) {
    if (f8_few_pairs(pairs, w->matrices)) return FRK_OK;
    const int shape = f8_grouped_shape(pairs, w->matrices);
    return f8_tiles_fit(w, shape, f8_max_tiles(pairs, w->matrices, F8_TILE_SIZE[shape].tokens), 1, gathered ? x_rows : 0);
}
size_t f8_grouped_workspace_bytes(const frk_weights *w, size_t x_rows, size_t pairs) {
    return f8_acts_bytes(x_rows, w->cols) + 256 + f8_max_tiles(pairs, w->matrices, 32) * 16;
}
int launch_f8_tiles(const frk_weights *w, const F8Acts &acts, int shape, const int *src, const int4 *tiles, const int *n_tiles, size_t max_tiles, float *y,
                    hipStream_t s) {
    F8Gemm g{};
    g.w = f8_mat(w);
    g.a = acts;
    g.src = src;
    g.tiles = tiles;
    g.n_tiles = n_tiles;
    g.ldy = g.w.rows;
    g.y = y;
    return launch_f8_tile(g, shape, max_tiles, 1, 1, 0, s);
}
int launch_f8_grouped(const frk_weights *w, const int32_t *group_off, const int32_t *gather, const float *x, size_t x_rows, size_t pairs,
                      float *y, void *ws, hipStream_t s) {
    const F8Acts acts = f8_acts_carve(ws, x_rows);
    const bool few = f8_few_pairs(pairs, w->matrices), fused = few && f8_fused_fits(F8_FUSED, w->cols);
    if (few && !fused) {
        int rc = launch_f8_quantize(x, nullptr, x_rows, w->cols, nullptr, acts, s);
        if (rc) return rc;
    }
    if (few) {
        F8Rows g{};
        g.w = f8_mat(w);
        g.a = acts;
        g.x = x;
        g.cols = (int)w->cols;
        g.x_rows = (int)x_rows;
        g.group_off = group_off;
        g.gather = gather;
        g.n_groups = (int)w->matrices;
        g.pairs = (int)pairs;
        g.ldy = g.w.rows;
        g.y = y;
        const dim3 grid((unsigned)g.w.strips, (unsigned)pairs);
        return fused ? go_f8_rows<8, 1, 4, true, F8_PAIRS>(g, grid, F8_FUSED * g.w.blocks * F8_BLOCK * 2, s) : go_f8_rows<8, 1, 4, false, F8_PAIRS>(g, grid, 0, s);
    }
    const int shape = f8_grouped_shape(pairs, w->matrices), tokens = F8_TILE_SIZE[shape].tokens;
    int *n_tiles = (int *)((char *)ws + f8_acts_bytes(x_rows, w->cols));
    int4 *tiles = (int4 *)(n_tiles + 64);
    const F8TilesArgs list{group_off, (int)w->matrices, (int)pairs, tokens, tiles, n_tiles};
    const int blocks = (int)f8_blocks(w->cols), parts = (blocks + F8_QUANTIZE_BLOCKS - 1) / F8_QUANTIZE_BLOCKS;
    const size_t jobs = x_rows * parts;
    const dim3 grid((unsigned)std::min<size_t>(1 + (jobs + 15) / 16, 1 << 14));
    if (f8_wide_rows(x, w->cols)) hipLaunchKernelGGL(f8_tiles_quantize_kernel<true>, grid, dim3(1024), 0, s, list, x, jobs, parts, (int)w->cols, blocks, acts);
    else hipLaunchKernelGGL(f8_tiles_quantize_kernel<false>, grid, dim3(1024), 0, s, list, x, jobs, parts, (int)w->cols, blocks, acts);
    FRK_LAUNCH_CHECK("f8_tiles_quantize");
    return launch_f8_tiles(w, acts, shape, gather, tiles, n_tiles, f8_max_tiles(pairs, w->matrices, tokens), y, s);
}

}  // namespace frk
