// Root-mean-square norm of rows, with the residual's addition in front and a quantization of the result behind:
//   h = x + residual, rounded to their type;  r = 1 / sqrt(mean(h^2) + eps), in 64 bits, rounded to f32 once;  y = (h r) w, two products
// rounded to f32 each; y in the input's type, or as the products of this library read activations (Q8_K; FP8: frk_f8.hpp; MXFP4: frk_mx4.hpp).
// With the sum of squares in 64 bits (each square exact) r does not depend on the order of the additions but for a value in 2^28, so neither do
// the quantized values on how a row is split between lanes.
//
// Memory bounds it: x and the residual are read once, h and the result written once.  A row is up to sixteen wavefronts', a lane four
// neighbouring values of every 256 -- what the quantizations' blocks are dealt by, too -- in registers between the sum and the products.
#include "frk_norm.hpp"

#include <algorithm>

namespace frk {

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// 256 values of a row (four a lane) in the form that the products read
template <int FORM>
__device__ __forceinline__ void store_quantized(const NormOut &out, size_t row, bool live, int c, int lane, const float (&v)[4]) {
    if (FORM == ACTS_FP8) {
        float scale;
        const uint32_t codes = f8_quantize4(v, scale);
        const uint2 two = f8_to_bf16(codes, scale);
        const int b = 2 * c + (lane >> 5), in = (lane & 31) * 4;
        if (b < out.f8_blocks) {
            if (out.f8.v) *reinterpret_cast<uint2 *>(out.f8.v + (row * out.f8_blocks + b) * F8_BLOCK + in) = two;
            if (out.f8_strips.v)
                *reinterpret_cast<uint2 *>(out.f8_strips.v + f8_strip_at(row, b, in, out.f8_blocks)) = two;
        }
    } else if (FORM == ACTS_Q8_K) {
        float d;
        int sum;
        const uint32_t quants = quantize_q8_k_lane(make_float4(v[0], v[1], v[2], v[3]), d, sum);
        const int nb = out.q8k_blocks;
        if (out.plain.q && live) {
            reinterpret_cast<uint32_t *>(out.plain.q + (row * nb + c) * QK_K)[lane] = quants;
            if ((lane & 3) == 0) out.plain.bsums[(row * nb + c) * 16 + (lane >> 2)] = (int16_t)sum;
            if (lane == 0) out.plain.d[row * nb + c] = d;
        }
        if (out.tiled.q) {
            const size_t rec = (row >> 5) * nb + c;
            const int r = (int)(row & 31), g = lane >> 2;
            *reinterpret_cast<uint32_t *>(out.tiled.q + rec * 8192 + ((lane >> 3) * 64 + (g & 1) * 32 + r) * 16 + (lane & 3) * 4) = quants;
            if ((lane & 3) == 0) out.tiled.bs[rec * 512 + ((g >> 3) * 32 + r) * 8 + (g & 7)] = (_Float16)sum;
            if (lane == 0) out.tiled.d[rec * 32 + r] = d;
        }
    } else if (FORM == ACTS_MXFP4) {
        mx4_store_chunk(out.mx4, row, c, lane, v);
    }
}

// `waves` wavefronts a row, the workgroup's others another row.  CHUNKS: of 256 values of a row that a wavefront holds; 0: any number, which
// are read a second time behind the sum.
template <int TYPE, int CHUNKS, int FORM, bool WIDE>
__global__ __launch_bounds__(1024) void rms_norm_kernel(NormArgs a, NormOut out) {
    typedef typename Floats<TYPE>::type T;
    __shared__ double sums[2][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int rows_wg = (int)(blockDim.x >> 6) / a.waves, mine = wave % a.waves, slot = wave - mine;
    const int cols = a.cols, chunks = a.chunks;
    int parity = 0;
    for (size_t row0 = (size_t)blockIdx.x * rows_wg; row0 < a.rows; row0 += (size_t)gridDim.x * rows_wg, parity ^= 1) {
        const size_t row = row0 + wave / a.waves;
        const bool live = row < a.batch, there = row < a.rows;  // (rows past the batch, of a last tile: zeros)
        const T *const x = (const T *)a.x + (live ? row * (size_t)cols : 0);
        const T *const res = (const T *)a.residual + (live ? row * (size_t)cols : 0);
        T *const h_out = (T *)a.sum + row * (size_t)cols;
        constexpr int N = CHUNKS ? CHUNKS : 1;
        float h[N][4];
        double sum = 0.0;
        auto load = [&](int c, float (&v)[4], bool store) {
            const int k = c * 256 + lane * 4;
            floats_load4<TYPE, WIDE>(x, k, live ? cols : 0, v);
            if (a.residual) {
                float u[4];
                floats_load4<TYPE, WIDE>(res, k, live ? cols : 0, u);
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = Floats<TYPE>::get(Floats<TYPE>::put(v[i] + u[i]));
            }
            if (store && live) floats_store4<TYPE, WIDE>(h_out, k, cols, v);
        };
        auto add = [&](const float (&v)[4]) {
#pragma unroll
            for (int i = 0; i < 4; i++) sum = fma((double)v[i], (double)v[i], sum);
        };
        if (CHUNKS) {
#pragma unroll
            for (int i = 0; i < N; i++) load(mine + i * a.waves, h[i], a.sum != nullptr);
#pragma unroll
            for (int i = 0; i < N; i++) add(h[i]);
        } else {
            for (int c = mine; c < chunks; c += a.waves) {
                load(c, h[0], a.sum != nullptr);
                add(h[0]);
            }
        }
        sum = wave_sum64(sum);
        if (a.waves > 1) {  // (uniform over the launch)
            if (lane == 0) sums[parity][wave] = sum;
            __syncthreads();
            sum = sums[parity][slot];
            for (int w = 1; w < a.waves; w++) sum += sums[parity][slot + w];
        }
        const float r = (float)(1.0 / sqrt(sum / (double)cols + a.eps));
        auto finish = [&](int c, const float (&v)[4]) {
            const int k = c * 256 + lane * 4;
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = v[i] * r;
            if (a.weight) {
                float w[4];
                if (a.weight_type == FLOATS_F32) floats_load4<FLOATS_F32, WIDE>((const float *)a.weight, k, cols, w);
                else if (a.weight_type == FLOATS_BF16) floats_load4<FLOATS_BF16, WIDE>((const uint16_t *)a.weight, k, cols, w);
                else floats_load4<FLOATS_F16, WIDE>((const uint16_t *)a.weight, k, cols, w);
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] *= w[i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!live || k + i >= cols) y[i] = 0.0f;  // (0 times an infinite r is none)
            if (a.y && live) floats_store4<TYPE, WIDE>((T *)a.y + row * (size_t)cols, k, cols, y);
            if (FORM != ACTS_NONE && there) store_quantized<FORM>(out, row, live, c, lane, y);
        };
        if (CHUNKS) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (mine + i * a.waves < chunks) finish(mine + i * a.waves, h[i]);
        } else {
            // (the residual, where the sum may have taken its place or x's, is in the sum)
            for (int c = mine; c < chunks; c += a.waves) {
                if (a.sum) floats_load4<TYPE, WIDE>(h_out, c * 256 + lane * 4, live ? cols : 0, h[0]);
                else load(c, h[0], false);
                finish(c, h[0]);
            }
        }
    }
}

template <int TYPE, int FORM, bool WIDE>
static int go_rms_norm(NormArgs a, const NormOut &out, hipStream_t s) {
    // Few rows: as many wavefronts a row as it has chunks, up to sixteen.  Many rows: four chunks a wavefront.
    const int chunks = a.chunks;
    const bool few = a.rows <= 512;
    int waves = 1;
    while (waves < 16 && waves * (few ? 1 : 4) < chunks) waves *= 2;
    a.waves = waves;
    const int waves_wg = std::max(waves, few ? 1 : 4);
    const size_t rows_wg = (size_t)(waves_wg / waves);
    const dim3 grid((unsigned)std::min<size_t>((a.rows + rows_wg - 1) / rows_wg, 1 << 16)), block(64 * waves_wg);
    if (chunks <= waves) hipLaunchKernelGGL((rms_norm_kernel<TYPE, 1, FORM, WIDE>), grid, block, 0, s, a, out);
    else if (chunks <= 4 * waves) hipLaunchKernelGGL((rms_norm_kernel<TYPE, 4, FORM, WIDE>), grid, block, 0, s, a, out);
    else hipLaunchKernelGGL((rms_norm_kernel<TYPE, 0, FORM, WIDE>), grid, block, 0, s, a, out);
    FRK_LAUNCH_CHECK("rms_norm");
    return FRK_OK;
}
template <int TYPE, int FORM>
static int go_rms_norm_wide(const NormArgs &a, const NormOut &out, hipStream_t s) {
    const size_t n = (size_t)a.cols;
    auto wide = [&](const void *p, int type) { return !p || floats_wide(p, n, type); };
    if (wide(a.x, TYPE) && wide(a.residual, TYPE) && wide(a.sum, TYPE) && wide(a.y, TYPE) && wide(a.weight, a.weight_type)) return go_rms_norm<TYPE, FORM, true>(a, out, s);
    return go_rms_norm<TYPE, FORM, false>(a, out, s);
}
template <int TYPE>
static int go_rms_norm_type(const NormArgs &a, int form, const NormOut &out, hipStream_t s) {
    switch (form) {
    case ACTS_FP8: return go_rms_norm_wide<TYPE, ACTS_FP8>(a, out, s);
    case ACTS_Q8_K: return go_rms_norm_wide<TYPE, ACTS_Q8_K>(a, out, s);
    case ACTS_MXFP4: return go_rms_norm_wide<TYPE, ACTS_MXFP4>(a, out, s);
    default: return go_rms_norm_wide<TYPE, ACTS_NONE>(a, out, s);
    }
}
int launch_rms_norm(int type, NormArgs a, int form, const NormOut &out, hipStream_t s) {
    // a form's rows are padded with zeros to whole blocks, MXFP4's to sixteen
    a.chunks = form == ACTS_MXFP4 ? out.mx4.blocks / 8 : (a.cols + 255) / 256;
    switch (type) {
    case FLOATS_F32: return go_rms_norm_type<FLOATS_F32>(a, form, out, s);
    case FLOATS_BF16: return go_rms_norm_type<FLOATS_BF16>(a, form, out, s);
    default: return go_rms_norm_type<FLOATS_F16>(a, form, out, s);
    }
}

// ---- what quantized rows stand for ----
__global__ __launch_bounds__(256) void q8_k_values_kernel(Q8KActs plain, Q8KTiled tiled, int nb, size_t n, float *__restrict__ out) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t block = i / QK_K;
        if (plain.q) {
            out[i] = (float)plain.q[i] * plain.d[block];
        } else {
            const int row = (int)(block / nb), kb = (int)(block % nb);
            out[i] = (float)tiled.q[q8k_tiled_index(nb, row, kb, (int)(i % QK_K))] * tiled.d[((size_t)(row >> 5) * nb + kb) * 32 + (row & 31)];
        }
    }
}
int launch_q8_k_values(const Q8KActs &plain, const Q8KTiled &tiled, size_t rows, size_t cols, float *out, hipStream_t s) {
    const size_t n = rows * cols;
    hipLaunchKernelGGL(q8_k_values_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1 << 16)), dim3(256), 0, s, plain, tiled, (int)(cols / QK_K), n, out);
    FRK_LAUNCH_CHECK("q8_k_values");
    return FRK_OK;
}
__global__ __launch_bounds__(256) void acts_values_fp8_kernel(F8Acts a, int cols, int blocks, size_t n, float *__restrict__ out) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t row = i / cols;
        const int k = (int)(i % cols), b = k / F8_BLOCK, in = k % F8_BLOCK;
        const size_t at = a.strips ? f8_strip_at(row, b, in, blocks) : (row * blocks + b) * F8_BLOCK + in;
        out[i] = __uint_as_float((uint32_t)a.v[at] << 16) * F8_UP;
    }
}
int launch_f8_values(const F8Acts &a, size_t cols, float *out, hipStream_t s) {
    const size_t n = (size_t)a.rows * cols;
    hipLaunchKernelGGL(acts_values_fp8_kernel, dim3((unsigned)std::min<size_t>((n + 255) / 256, 1 << 16)), dim3(256), 0, s, a, (int)cols, (int)f8_blocks(cols), n, out);
    FRK_LAUNCH_CHECK("f8_values");
    return FRK_OK;
}

}  // namespace frk
