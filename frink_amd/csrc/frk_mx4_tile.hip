// Products of MXFP4 matrices and MXFP4 activations (frk_mx4.hpp) over large tiles on the block-scaled matrix cores
// (v_mfma_scale_f32_32x32x64_f8f6f4): sixteen bytes of E2M1 codes are a lane's operand, its block's E8M0 byte the scale.
//   y[t][r] = sum over blocks b of 2^(sw[r][b] + sx[t][b] - 254) * sum over the 32 of b of w x
// Products of codes and a block's sum are exact, blocks add up in f32.
// What bounds it: a full chip of 256 x 256 tiles (4096 tokens of 4096 x 14336) its 239 thousand cycles, of which the matrix cores are busy 48 %, and the
// clock that its power leaves: 116 us behind the quantization in front of it (4.1 PFLOP/s, 2.1 GHz), 130 to 140 one product after the other (3.4 to
// 3.7; 1.7 to 1.85 GHz; the products without anything else 86, with the operands' reads 110); fewer workgroups the time from a request to its bytes, which is why smaller tiles have three or four
// stages (64 tokens of 14336 x 4096, two stages / three / four of 64 x 64: 13.7 / 9.4 / 8.8 us; 512 of 4096 x 14336, two / three of 64 x 128:
// 43.2 / 28.6).
#include "frk_mx4.hpp"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace frk {

typedef int mx4_v4i __attribute__((ext_vector_type(4)));
typedef int mx4_v8i __attribute__((ext_vector_type(8)));
typedef float mx4_v16f __attribute__((ext_vector_type(16)));

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

// RW x TW wavefronts of MR groups of 32 weight rows x MT groups of 32 tokens each.  A stage is eight blocks (256 columns) of every row:
// 128 bytes of codes, eight lanes a row in one piece.  STAGES of them are in LDS or on their way there.
template <int RW, int TW, int MR, int MT, int DEPTH>
struct Mx4TileShape {
    static constexpr int WAVES = RW * TW, ROWS = RW * MR * 32, TOKENS = TW * MT * 32, ALL = ROWS + TOKENS;
    static constexpr int STAGES = DEPTH, STAGE = ALL * 128, SCALES = ALL * 16;  // scales: sixteen blocks, of two stages
    static constexpr int W_REQUESTS = ROWS / 8 / WAVES, X_REQUESTS = TOKENS / 8 / WAVES, REQUESTS = W_REQUESTS + X_REQUESTS;
    static constexpr int S_REQUESTS = (ALL / 64 + WAVES - 1) / WAVES;
    static_assert(W_REQUESTS * 8 * WAVES == ROWS && X_REQUESTS * 8 * WAVES == TOKENS && ROWS % 64 == 0 && TOKENS % 64 == 0, "whole requests");
    static constexpr int PITCH = MR * 32 + 4;  // floats a token in the results' place in LDS: sixteen lanes' pieces in different banks
    static constexpr int SCALE_PLACES = STAGES > 3 ? 4 : 2;  // (a power of two: STAGES / 2 + 1 pairs of stages are on their way)
    static constexpr size_t LDS = STAGES * STAGE + SCALE_PLACES * SCALES;
    static_assert((size_t)WAVES * 32 * PITCH * 4 <= LDS, "a group of tokens of every wavefront");
    static_assert(LDS <= 160 * 1024, "LDS of a CU");
};

template <int RW, int TW, int MR, int MT, int DEPTH>
__global__ __launch_bounds__(64 * RW * TW, 1) void mx4_tile_kernel(Mx4Gemm g, int row_tiles, int tok_tiles, int parts, size_t part_stride) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = Mx4TileShape<RW, TW, MR, MT, DEPTH>;
    constexpr int E2M1 = 4;
    extern __shared__ __align__(16) uint8_t mx4_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int rw = wave % RW, tw = wave / RW;
    // An XCD (workgroup id mod 8) takes a run of the list, which goes through panels of eight token tiles row tile by row tile: its CUs
    // then work on tiles that share their blocks in its L2.
    const int total = row_tiles * tok_tiles, per_xcd = (total + 7) / 8;
    const int index = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per_xcd || index >= total) return;
    const int panel = index / (8 * row_tiles), wide_panel = min(8, tok_tiles - 8 * panel), in_panel = index - panel * 8 * row_tiles;
    const int row0 = in_panel / wide_panel * T::ROWS, tok0 = (8 * panel + in_panel % wide_panel) * T::TOKENS;
    // this part's stages
    const int part = (int)blockIdx.y, stages = (g.blocks + 7) / 8;
    const int from = (int)((long long)stages * part / parts), until = (int)((long long)stages * (part + 1) / parts);
    const uint32_t lds0 = lds_address(mx4_lds);

    // ---- requests: place p of row r of a stage holds piece p ^ (r / 2) % 8, so that the sixteen rows that LDS serves together touch all banks
    uint32_t w_off[T::W_REQUESTS], x_off[T::X_REQUESTS], s_off[T::S_REQUESTS];
    const uint8_t *const w_base = g.W + (size_t)row0 * g.row_stride;
    const uint8_t *const x_base = g.a.codes + (size_t)tok0 * g.a.blocks * 16;
    const uint8_t *const xs_base = g.a.scales + (size_t)tok0 * g.a.blocks;
    const uint8_t *const ws_base = w_base + (size_t)g.blocks * 16;
    const int last_row = g.rows - 1 - row0, last_token = g.M - 1 - tok0;
#pragma unroll
    for (int c = 0; c < T::W_REQUESTS; c++) {
        const int r = (c * T::WAVES + wave) * 8 + (lane >> 3);
        w_off[c] = (uint32_t)min(r, last_row) * (uint32_t)g.row_stride + (uint32_t)((lane & 7) ^ ((r >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int c = 0; c < T::X_REQUESTS; c++) {
        const int r = (c * T::WAVES + wave) * 8 + (lane >> 3);
        x_off[c] = (uint32_t)min(r, last_token) * (uint32_t)(g.a.blocks * 16) + (uint32_t)((lane & 7) ^ ((r >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int c = 0; c < T::S_REQUESTS; c++) {  // 64 rows a request, weight rows first
        const int q = min(c * T::WAVES + wave, T::ALL / 64 - 1), r = q * 64 + lane;
        s_off[c] = q * 64 < T::ROWS ? (uint32_t)min(r, last_row) * (uint32_t)g.row_stride : (uint32_t)min(r - T::ROWS, last_token) * (uint32_t)g.a.blocks;
    }
    // the places of the stages in front of the present one (which STAGES - 1 behind it takes), of the present one and of the next
    uint32_t before = (T::STAGES - 1) * T::STAGE, here = 0, next = T::STAGE;
    auto request_codes = [&](int i, uint32_t place, int c) {  // request c of stage i
        const uint32_t to = lds0 + place;
        if (c < T::W_REQUESTS) dma16(to + (uint32_t)(c * T::WAVES + wave) * 1024, w_base + (size_t)i * 128, w_off[c]);
        else dma16(to + T::ROWS * 128 + (uint32_t)((c - T::W_REQUESTS) * T::WAVES + wave) * 1024, x_base + (size_t)i * 128, x_off[c - T::W_REQUESTS]);
    };
    auto request_scales = [&](int i) {  // of the two stages that i is one of
        const uint32_t to = lds0 + T::STAGES * T::STAGE + (uint32_t)((i >> 1) & (T::SCALE_PLACES - 1)) * T::SCALES;
#pragma unroll
        for (int c = 0; c < T::S_REQUESTS; c++) {
            const int q = min(c * T::WAVES + wave, T::ALL / 64 - 1);
            dma16(to + (uint32_t)q * 1024, (q * 64 < T::ROWS ? ws_base : xs_base) + (size_t)(i >> 1) * 16, s_off[c]);
        }
    };
    mx4_v16f acc[MT][MR];
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int r = 0; r < MR; r++) acc[t][r] = mx4_v16f{0.0f};
    // where this lane's blocks 4 lh + k of its row lie in a group of 32 rows: 16 k flipped
    const uint32_t piece_at = (uint32_t)(li * 128 + ((4 * lh) ^ ((li >> 1) & 7)) * 16);
    const uint32_t w_lane = (uint32_t)(rw * MR * 32) * 128, x_lane = (uint32_t)(T::ROWS + tw * MT * 32) * 128;

    // A stage is four steps of MR x MT products, a step one block of every lane.  Beside a step's products the wavefront reads the next step's
    // operands.  In front of a stage's last step it waits for the next stage and for everybody to have read the present one, whose place
    // is then asked for again, STAGES stages on: a third of the requests beside each of the next three steps.
    mx4_v4i w[2][MR], x[2][MT];
    int ws[MR], xs[MT], next_ws[MR], next_xs[MT];
    auto read_scales = [&](int i) {
        const uint8_t *const sc = mx4_lds + T::STAGES * T::STAGE + (size_t)((i >> 1) & (T::SCALE_PLACES - 1)) * T::SCALES + (i & 1) * 8 + lh * 4 + li * 16;
#pragma unroll
        for (int r = 0; r < MR; r++) next_ws[r] = *reinterpret_cast<const int *>(sc + (rw * MR + r) * 512);
#pragma unroll
        for (int t = 0; t < MT; t++) next_xs[t] = *reinterpret_cast<const int *>(sc + T::ROWS * 16 + (tw * MT + t) * 512);
    };
    auto read = [&](uint32_t place, int k, int n) {  // operand n of step k of the stage there
        const uint8_t *const st = mx4_lds + place + (piece_at ^ (uint32_t)(k * 16));
        if (n < MR) w[k & 1][n] = *reinterpret_cast<const mx4_v4i *>(st + w_lane + n * 4096);
        else x[k & 1][n - MR] = *reinterpret_cast<const mx4_v4i *>(st + x_lane + (n - MR) * 4096);
    };
    // (the reads beside the first half of the products, so that they have come when the others are done)
    constexpr int PRODUCTS = MR * MT, READS = MR + MT, READS_EACH = (2 * READS + PRODUCTS - 1) / PRODUCTS, FIRST = (T::REQUESTS + 2) / 3, SECOND = (2 * T::REQUESTS + 1) / 3;
    // step K's products and what goes beside them: operands of the next step (stage I), requests BEGIN .. END - 1 of stage A
#define FRK_MX4_STEP(K, FROM, ASK, A, TO, BEGIN, END)                                                                                           \
    _Pragma("unroll") for (int t = 0; t < MT; t++) _Pragma("unroll") for (int r = 0; r < MR; r++) {                                            \
        const mx4_v4i &xv = x[K & 1][t], &wv = w[K & 1][r];                                                                                    \
        const int at = t * MR + r;                                                                                                             \
        acc[t][r] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_v8i{wv[0], wv[1], wv[2], wv[3], 0, 0, 0, 0},                           \
                                                                    mx4_v8i{xv[0], xv[1], xv[2], xv[3], 0, 0, 0, 0}, acc[t][r], E2M1, E2M1, K, \
                                                                    ws[r], K, xs[t]);                                                          \
        if (K == 3 && at == 0) read_scales(i + 1);                                                                                               \
        _Pragma("unroll") for (int n = at * READS_EACH; n < min((at + 1) * READS_EACH, READS); n++) read(FROM, (K + 1) & 3, n);                \
        if (ASK) {                                                                                                                             \
            constexpr int COUNT = (END) - (BEGIN);                                                                                            \
            _Pragma("unroll") for (int c = (BEGIN) + at * COUNT / PRODUCTS; c < (BEGIN) + (at + 1) * COUNT / PRODUCTS; c++) request_codes(A, TO, c); \
        }                                                                                                                                      \
        __builtin_amdgcn_sched_barrier(0);                                                                                                     \
    }
    // LEFT: how many stages behind the present one there are (STAGES: or more)
    auto stage = [&](int i, auto left) {
        constexpr int LEFT = decltype(left)::value;
        // (a row's last stage may reach past its blocks: the codes there meet zeros, but a byte 255 would make them NaN.  Only there, and only here:
        // behind the reads themselves it is a wait for them)
        int mask = -1;
        if (LEFT == 0) {
            const int live = g.blocks - (i * 8 + 4 * lh);
            mask = live >= 4 ? -1 : live > 0 ? (int)(0xffffffffu >> (32 - 8 * live)) : 0;
        }
#pragma unroll
        for (int r = 0; r < MR; r++) ws[r] = next_ws[r] & mask;
#pragma unroll
        for (int t = 0; t < MT; t++) xs[t] = next_xs[t];
        FRK_MX4_STEP(0, here, LEFT >= T::STAGES - 1, i + T::STAGES - 1, before, FIRST, SECOND)
        if (LEFT >= T::STAGES - 1 && !((i + T::STAGES - 1) & 1)) request_scales(i + T::STAGES - 1);
        FRK_MX4_STEP(1, here, LEFT >= T::STAGES - 1, i + T::STAGES - 1, before, SECOND, T::REQUESTS)
        FRK_MX4_STEP(2, here, false, 0, 0, 0, 0)
        // (all but the requests of the stages behind the next one)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((LEFT < 2 ? 0 : LEFT < T::STAGES ? LEFT - 1 : T::STAGES - 2) * T::REQUESTS) : "memory");
        lds_barrier();
        // (behind the last stage whatever lies there, which nobody multiplies)
        FRK_MX4_STEP(3, next, LEFT >= T::STAGES, i + T::STAGES, here, 0, FIRST)
        before = here, here = next, next = next == (T::STAGES - 1) * T::STAGE ? 0 : next + T::STAGE;
    };
    if (from < until) {
        request_scales(from);
#pragma unroll
        for (int n = 1; n < T::STAGES - 1; n++)
            if (!((from + n) & 1) && from + n < until) request_scales(from + n);
#pragma unroll
        for (int n = 0; n < T::STAGES - 1; n++)
            if (from + n < until) {
#pragma unroll
                for (int c = 0; c < T::REQUESTS; c++) request_codes(from + n, n * T::STAGE, c);
            }
        if (from + T::STAGES - 1 < until) {
#pragma unroll
            for (int c = 0; c < FIRST; c++) request_codes(from + T::STAGES - 1, (T::STAGES - 1) * T::STAGE, c);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((T::STAGES - 2) * T::REQUESTS + FIRST) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        lds_barrier();
        read_scales(from);
#pragma unroll
        for (int n = 0; n < READS; n++) read(0, 0, n);
    }
    int i = from;
    for (; i + T::STAGES < until; i++) stage(i, std::integral_constant<int, T::STAGES>());
    if (T::STAGES > 3 && i + 3 < until) stage(i++, std::integral_constant<int, 3>());
    if (T::STAGES > 2 && i + 2 < until) stage(i++, std::integral_constant<int, 2>());
    if (i + 1 < until) stage(i++, std::integral_constant<int, 1>());
    if (i < until) stage(i, std::integral_constant<int, 0>());
#undef FRK_MX4_STEP
    // (the compiler does not count a product's wait states, eighteen at most, across the branches between it and the reads of its sum)
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    // ---- register i of a lane: weight row 8 (i / 4) + 4 (lane / 32) + i % 4 of a group, token lane % 32.  Through LDS, a group of tokens at a time and
    // each wavefront in a place of its own, so that a store writes whole lines, sixteen bytes a lane (a dword a lane, whichever way round: 17000
    // of the 76000 cycles of a tile of 4096 columns).
    lds_barrier();  // (the last reads)
    constexpr int LANES = MR * 8, TOKENS_EACH = 64 / LANES;  // of a token, tokens a store
    float *const own = reinterpret_cast<float *>(mx4_lds) + wave * 32 * T::PITCH;
    const int row_first = row0 + rw * MR * 32 + (lane % LANES) * 4;
    float *const y = g.y + part * part_stride + row_first;
    const bool wide = g.ldy % 4 == 0 && part_stride % 4 == 0 && (g.rows & 3) == 0 && (reinterpret_cast<uintptr_t>(g.y) & 15) == 0;
#pragma unroll
    for (int t = 0; t < MT; t++) {
#pragma unroll
        for (int r = 0; r < MR; r++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *reinterpret_cast<float4 *>(own + li * T::PITCH + r * 32 + q * 8 + lh * 4) =
                    make_float4(acc[t][r][4 * q], acc[t][r][4 * q + 1], acc[t][r][4 * q + 2], acc[t][r][4 * q + 3]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wavefront reads its own stores only)
#pragma unroll
        for (int j = 0; j < 32 / TOKENS_EACH; j++) {
            const int in = j * TOKENS_EACH + lane / LANES, tok = tok0 + (tw * MT + t) * 32 + in;
            const float4 v = *reinterpret_cast<const float4 *>(own + in * T::PITCH + (lane % LANES) * 4);
            if (tok >= g.M) continue;
            float *const dst = y + (size_t)tok * g.ldy;
            if (wide) {
                if (row_first < g.rows) *reinterpret_cast<float4 *>(dst) = v;
            } else {
                const float out[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int n = 0; n < 4; n++)
                    if (row_first + n < g.rows) dst[n] = out[n];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
#endif
}

template <int RW, int TW, int MR, int MT, int DEPTH>
static int go_mx4_tile(const Mx4Gemm &g, int parts, size_t part_stride, hipStream_t s) {
    using T = Mx4TileShape<RW, TW, MR, MT, DEPTH>;
    const size_t row_tiles = ((size_t)g.rows + T::ROWS - 1) / T::ROWS, tok_tiles = ((size_t)g.M + T::TOKENS - 1) / T::TOKENS, total = row_tiles * tok_tiles;
    static std::atomic<uint64_t> sized{0};  // a bit a device (two threads may set the same attribute)
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && (dev >= 64 || !(sized.load(std::memory_order_relaxed) >> dev & 1))) {
        e = hipFuncSetAttribute(reinterpret_cast<const void *>(&mx4_tile_kernel<RW, TW, MR, MT, DEPTH>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)T::LDS);
        if (e == hipSuccess && dev < 64) sized.fetch_or((uint64_t)1 << dev, std::memory_order_relaxed);
    }
    if (e != hipSuccess) return set_error(FRK_ERR_HIP, "hipFuncSetAttribute(mx4_tile): %s", hipGetErrorString(e));
    hipLaunchKernelGGL((mx4_tile_kernel<RW, TW, MR, MT, DEPTH>), dim3((unsigned)((total + 7) / 8 * 8), (unsigned)parts), dim3(64 * T::WAVES), T::LDS, s, g,
                       (int)row_tiles, (int)tok_tiles, parts, part_stride);
    FRK_LAUNCH_CHECK("mx4_tile");
    return FRK_OK;
}
bool mx4_tiles_fit(const frk_weights *w, int shape, size_t batch) {
    const Mx4TileSize t = MX4_TILE_SIZE[shape];
    const size_t row_tiles = (w->rows + t.rows - 1) / t.rows, tok_tiles = (batch + t.tokens - 1) / t.tokens;
    return (row_tiles * tok_tiles + 7) / 8 * 8 * t.threads <= 0xffffffffu;
}
int launch_mx4_tile(const Mx4Gemm &g, int shape, int parts, size_t part_stride, hipStream_t s) {
    switch (shape) {
    case MX4_TILE_256x256: return go_mx4_tile<2, 2, 4, 4, 2>(g, parts, part_stride, s);
    case MX4_TILE_256x128: return go_mx4_tile<4, 2, 2, 2, 3>(g, parts, part_stride, s);
    case MX4_TILE_128x128: return go_mx4_tile<2, 2, 2, 2, 3>(g, parts, part_stride, s);
    case MX4_TILE_64x128: return go_mx4_tile<1, 4, 2, 1, 3>(g, parts, part_stride, s);
    default: return go_mx4_tile<2, 2, 1, 1, 4>(g, parts, part_stride, s);
    }
}

}  // namespace frk
