// Root-mean-square norm of rows, with the residual's addition in front and a quantization of the result behind:
//   h = x + residual, rounded to their type;  r = 1 / sqrt(mean(h^2) + eps), in 64 bits, rounded to f32 once;  y = (h r) w, two products
// rounded to f32 each; y in the input's type, or as the products of this library read activations (Q8_K; FP8: frk_f8.hpp; MXFP4: frk_mx4.hpp).
// With the sum of squares in 64 bits (each square exact) r does not depend on the order of the additions but for a value in 2^28, so neither do
// the quantized values on how a row is split between lanes.
//
// Memory bounds it: x and the residual are read once, h and the result written once.  A row is up to sixteen wavefronts', a lane four
// neighbouring values of every 256 -- what the quantizations' blocks are dealt by, too -- in registers between the sum and the products.
// 16384 x 4096 of f32 with a residual 191 us, 1.07 GB (5.6 TB/s, part of it from the caches); 1 x 4096 to FP8 4.4, of which a launch that does
// nothing is 2.
#include "frk_norm.hpp"

#include <algorithm>

namespace frk {

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

// v (op) lane-permuted v, the permutation given by a DPP control word
template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)dpp_i<CTRL>((int)b) | (uint64_t)(uint32_t)dpp_i<CTRL>((int)(b >> 32)) << 32));
}
__device__ __forceinline__ double row_sum64(double v) {  // over sixteen lanes
    v += dpp_d<DPP_QUAD_XOR1>(v);
    v += dpp_d<DPP_QUAD_XOR2>(v);
    v += dpp_d<DPP_HALF_MIRROR>(v);
    v += dpp_d<DPP_ROW_MIRROR>(v);
    return v;
}
__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)b, lane) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32));
}
__device__ __forceinline__ double wave_sum64(double v) {
    v = row_sum64(v);
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
// 1 / sqrt(a) to a few units in the last place of 64 bits: the instruction's value and two of Newton's steps (a root and a quotient correct to the
// last bit are 60 instructions more, and the f32 that it is rounded to differs once in 2^27)
__device__ __forceinline__ double inverse_root(double a) {
    double y = __builtin_amdgcn_rsq(a);
    if (a > 0.0 && a < 1.0e300) {  // (zero and infinity: the instruction's)
        y = fma(y, fma(-0.5 * a * y, y, 0.5), y);
        y = fma(y, fma(-0.5 * a * y, y, 0.5), y);
    }
    return y;
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

// A workgroup's place where an XCD (workgroup id mod 8) is to have eight neighbours at a time, in a grid of whole 64s: Q8_K's tiles have pieces of
// eight rows in a line, which are then put together in one L2 (a norm after the other, 512 x 4096 8.8 -> 8.0 to 8.3 us, 16384 x 4096
// 202 -> 172 to 180).
__device__ __forceinline__ unsigned in_eights(unsigned b) { return gridDim.x % 64 ? b : (b & ~63u) + (b & 7) * 8 + (b >> 3 & 7); }

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
    for (size_t row0 = (size_t)(FORM == ACTS_Q8_K ? in_eights(blockIdx.x) : blockIdx.x) * rows_wg; row0 < a.rows; row0 += (size_t)gridDim.x * rows_wg, parity ^= 1) {
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
        auto load_weight = [&](int c, float (&w)[4]) {
            const int k = c * 256 + lane * 4;
            if (!a.weight) return;
            if (a.weight_type == FLOATS_F32) floats_load4<FLOATS_F32, WIDE>((const float *)a.weight, k, cols, w);
            else if (a.weight_type == FLOATS_BF16) floats_load4<FLOATS_BF16, WIDE>((const uint16_t *)a.weight, k, cols, w);
            else floats_load4<FLOATS_F16, WIDE>((const uint16_t *)a.weight, k, cols, w);
        };
        float w[N][4];
        if (CHUNKS) {
#pragma unroll
            for (int i = 0; i < N; i++) load(mine + i * a.waves, h[i], a.sum != nullptr);
#pragma unroll
            for (int i = 0; i < N; i++) load_weight(mine + i * a.waves, w[i]);  // (here: not another trip to memory behind the sum)
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
            const double part = sums[parity][slot + (lane & 15 & (a.waves - 1))];
            sum = row_sum64((lane & 15) < a.waves ? part : 0.0);
        }
        const float r = (float)inverse_root(fma(sum, a.inverse_cols, a.eps));
        auto finish = [&](int c, const float (&v)[4], const float (&w)[4]) {
            int k = c * 256 + lane * 4;
            if (!WIDE) asm("" : "+v"(k));  // (the addresses made anew: kept from the loads they spilled)
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = v[i] * r;
            if (a.weight) {
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
                if (mine + i * a.waves < chunks) finish(mine + i * a.waves, h[i], w[i]);
        } else {
            // (the residual, where the sum may have taken its place or x's, is in the sum)
            for (int c = mine; c < chunks; c += a.waves) {
                if (a.sum) floats_load4<TYPE, WIDE>(h_out, c * 256 + lane * 4, live ? cols : 0, h[0]);
                else load(c, h[0], false);
                load_weight(c, w[0]);
                finish(c, h[0], w[0]);
            }
        }
    }
}

template <int TYPE, int FORM, bool WIDE>
static int go_rms_norm(NormArgs a, const NormOut &out, hipStream_t s) {
    // Two chunks a wavefront, four where the rows fill the chip.  us (a launch after the other, x and the residual of 4 batches in turn, f32 to FP8),
    // chunks a wavefront 1 / 2 / 4 / 8: 4096 columns, 1 row 3.9 / 3.9 / 5.0 / 9.0, 512 rows 8.7 / 7.7 / 8.5 / 13.4, 2048 rows 30.4 / 27.7 / 29.0 /
    // 31.0; of 8192 columns (sixteen wavefronts hold two) 2 / 4 / 8: 1 row 4.7 / 5.5 / 9.5, 128 rows 6.3 / 7.3 / 12.8, 512 rows 13.9 / 12.8 / 15.9.
    const int chunks = a.chunks, most = a.rows > 256 ? 8 : 16;
    int waves = 1;
    while ((waves < most && 2 * waves < chunks) || (waves < 16 && 4 * waves < chunks)) waves *= 2;
    a.waves = waves;
    const int waves_wg = std::max(waves, a.rows > 512 ? 4 : 1);
    const size_t rows_wg = (size_t)(waves_wg / waves);
    size_t groups = std::min<size_t>((a.rows + rows_wg - 1) / rows_wg, 1 << 16);
    if (FORM == ACTS_Q8_K && groups > 32) groups = (groups + 63) / 64 * 64;
    const dim3 grid((unsigned)groups), block(64 * waves_wg);
    if (chunks <= 2 * waves) hipLaunchKernelGGL((rms_norm_kernel<TYPE, 2, FORM, WIDE>), grid, block, 0, s, a, out);
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
    a.inverse_cols = 1.0 / a.cols;
    a.chunks = form == ACTS_MXFP4 ? out.mx4.blocks / 8 : (a.cols + 255) / 256;
    switch (type) {
    case FLOATS_F32: return go_rms_norm_type<FLOATS_F32>(a, form, out, s);
    case FLOATS_BF16: return go_rms_norm_type<FLOATS_BF16>(a, form, out, s);
    default: return go_rms_norm_type<FLOATS_F16>(a, form, out, s);
    }
}

// ---- what quantized rows stand for: a wavefront 256 values at a time, a workgroup the same columns of eight rows (a line of Q8_K's tiles: in
// rows' order 16384 x 4096 took 81.7 us, not 72.6) ----
template <int FORM, bool WIDE>
__global__ __launch_bounds__(512) void acts_values_kernel(NormOut in, size_t rows, int chunks, int cols, float *__restrict__ out) {
    const int lane = threadIdx.x & 63;
    const size_t jobs = (rows + 7) / 8 * chunks;
    for (size_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const size_t row = j / chunks * 8 + (threadIdx.x >> 6);
        const int c = (int)(j % chunks);
        if (row >= rows) continue;
        float v[4];
        if (FORM == ACTS_FP8) {
            const F8Acts &a = in.f8.v ? in.f8 : in.f8_strips;
            const int b = min(2 * c + (lane >> 5), in.f8_blocks - 1), at = (lane & 31) * 4;
            const uint2 two = *reinterpret_cast<const uint2 *>(a.v + (a.strips ? f8_strip_at(row, b, at, in.f8_blocks) : (row * in.f8_blocks + b) * F8_BLOCK + at));
            const uint32_t d[2] = {two.x, two.y};
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = __uint_as_float(i & 1 ? d[i >> 1] & 0xffff0000u : d[i >> 1] << 16) * F8_UP;
        } else {
            const int nb = in.q8k_blocks;
            const size_t rec = (row >> 5) * nb + c;
            const uint32_t q = in.plain.q ? reinterpret_cast<const uint32_t *>(in.plain.q + (row * nb + c) * QK_K)[lane]
                                          : *reinterpret_cast<const uint32_t *>(in.tiled.q + q8k_tiled_index(nb, (int)row, c, lane * 4));
            const float d = in.plain.q ? in.plain.d[row * nb + c] : in.tiled.d[rec * 32 + (row & 31)];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (float)(int8_t)(q >> (8 * i)) * d;
        }
        floats_store4<FLOATS_F32, WIDE>(out + row * (size_t)cols, c * 256 + lane * 4, cols, v);
    }
}
template <int FORM>
static int go_acts_values(const NormOut &in, size_t rows, size_t cols, float *out, hipStream_t s) {
    const size_t chunks = (cols + 255) / 256;
    const dim3 grid((unsigned)std::min<size_t>((rows + 7) / 8 * chunks, 1 << 16));
    if (floats_wide(out, cols, FLOATS_F32)) hipLaunchKernelGGL((acts_values_kernel<FORM, true>), grid, dim3(512), 0, s, in, rows, (int)chunks, (int)cols, out);
    else hipLaunchKernelGGL((acts_values_kernel<FORM, false>), grid, dim3(512), 0, s, in, rows, (int)chunks, (int)cols, out);
    FRK_LAUNCH_CHECK("acts_values");
    return FRK_OK;
}
int launch_acts_values(int form, const NormOut &in, size_t rows, size_t cols, float *out, hipStream_t s) {
    if (form == ACTS_MXFP4) return launch_mx4_values(in.mx4, cols, out, s);
    return form == ACTS_FP8 ? go_acts_values<ACTS_FP8>(in, rows, cols, out, s) : go_acts_values<ACTS_Q8_K>(in, rows, cols, out, s);
}

}  // namespace frk
