// Products with weights in 8-bit floating point, a scale for each block of 128 x 128 (frk_f8.hpp), over large tiles: batches of
// more than a few dozen rows, dense and grouped.
#include "frk_f8.hpp"

#include <algorithm>

namespace frk {

typedef __bf16 f8_v8bf __attribute__((ext_vector_type(8)));
typedef float f8_v16f __attribute__((ext_vector_type(16)));

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

// RW x TW wavefronts of MR tiles of 32 weight rows x MT tiles of 32 tokens each
template <int RW, int TW, int MR, int MT, int STAGES>
struct F8TileShape {
    static constexpr int WAVES = RW * TW, ROWS = RW * MR * 32, TOKENS = TW * MT * 32;
    static constexpr int W_BYTES = ROWS * F8_BLOCK, X_BYTES = TOKENS * F8_BLOCK * 2, STAGE = W_BYTES + X_BYTES;
    static constexpr int W_REQ = W_BYTES / 1024 / WAVES, X_REQ = X_BYTES / 1024 / WAVES;
    static_assert(W_REQ * WAVES * 1024 == W_BYTES && X_REQ * WAVES * 1024 == X_BYTES, "whole requests");
    static constexpr int REQUESTS = W_REQ + X_REQ;  // of a wavefront and block
    static_assert(STAGES >= 2 && REQUESTS * (STAGES - 1) < 64, "requests that a wait can count");
    static constexpr size_t LDS = STAGES * STAGE;
    static_assert(LDS <= 160 * 1024 && F8_BLOCK % (MR * 32) == 0, "LDS of a CU; a wavefront's rows in one block of scales");
};

template <int RW, int TW, int MR, int MT, int STAGES>
__global__ __launch_bounds__(64 * RW * TW, 2) void f8_tile_kernel(F8Gemm g, int row_tiles, int tok_tiles, int matrices, int parts, size_t part_stride) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = F8TileShape<RW, TW, MR, MT, STAGES>;
    extern __shared__ __align__(16) uint8_t f8_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int rw = wave % RW, tw = wave / RW;
    // An XCD (workgroup id mod 8) takes a run of the list, which goes through panels of eight token tiles row tile by row tile: its 32
    // CUs then work on 4 row tiles x 8 token tiles, whose blocks its L2 holds once.
    if (g.tiles) tok_tiles = min(*g.n_tiles, tok_tiles);
    const int total = row_tiles * tok_tiles, per_xcd = (total + 7) / 8;
    const int index = ((int)blockIdx.x & 7) * per_xcd + ((int)blockIdx.x >> 3);
    if (((int)blockIdx.x >> 3) >= per_xcd || index >= total) return;
    const int panel = index / (8 * row_tiles), wide_panel = min(8, tok_tiles - 8 * panel), in_panel = index - panel * 8 * row_tiles;
    const int row_tile = in_panel / wide_panel, tok_tile = 8 * panel + in_panel % wide_panel;
    int4 tile;
    size_t y_col = 0;
    if (g.tiles) {
        tile = g.tiles[tok_tile];
    } else {
        const int first = tok_tile * T::TOKENS;
        tile = make_int4((int)blockIdx.y % matrices, first, min(T::TOKENS, g.M - first), first);
        y_col = (size_t)tile.x * g.w.rows;
    }
    // this part's columns
    const int part = (int)blockIdx.y / matrices, blocks = g.w.blocks;
    const int from = (int)((long long)blocks * part / parts), until = (int)((long long)blocks * (part + 1) / parts);
    const uint32_t lds0 = lds_address(f8_lds);
    const int strip0 = row_tile * (T::ROWS / F8_STRIP);

    // ---- requests: a stage holds the rows' strips as they lie in memory, then the tokens, 256 bytes each, piece p of token t in
    // place p ^ t % 16
    uint32_t x_off[T::X_REQ];
    const uint8_t *x_base = reinterpret_cast<const uint8_t *>(g.a.v);
    const int first_row = g.src ? 0 : min(tile.y, g.a.rows - 1);
    x_base += (size_t)first_row * blocks * (F8_BLOCK * 2);
#pragma unroll
    for (int c = 0; c < T::X_REQ; c++) {
        const int t = (wave * T::X_REQ + c) * 4 + (lane >> 4), i = min(t, tile.z - 1);
        const uint32_t row = (uint32_t)(min(max(g.src ? g.src[tile.y + i] : tile.y + i, 0), g.a.rows - 1) - first_row);
        x_off[c] = row * (uint32_t)blocks * (F8_BLOCK * 2) + (uint32_t)((lane & 15) ^ (t & 15)) * 16;
    }
    uint32_t w_off[T::W_REQ];
#pragma unroll
    for (int c = 0; c < T::W_REQ; c++) {
        const int n = wave * T::W_REQ + c, strip = min(strip0 + (n >> 1), g.w.strips - 1) - strip0;
        w_off[c] = (uint32_t)strip * (uint32_t)blocks * F8_PIECE + (uint32_t)((n & 1) * 1024 + lane * 16);
    }
    const uint8_t *const w_base = g.w.q + ((size_t)tile.x * g.w.strips + strip0) * blocks * F8_PIECE;
    auto request = [&](int slot, int b, int c) {
        const uint32_t to = lds0 + (uint32_t)slot * T::STAGE;
        if (c < T::W_REQ) dma16(to + (wave * T::W_REQ + c) * 1024, w_base + (size_t)b * F8_PIECE, w_off[c]);
        else dma16(to + T::W_BYTES + (wave * T::X_REQ + c - T::W_REQ) * 1024, x_base + (size_t)b * (F8_BLOCK * 2), x_off[c - T::W_REQ]);
    };
    // (scalar loads: a vector load's wait would be one for the requests in flight too)
    typedef const __attribute__((address_space(4))) float *scalar_floats;
    const scalar_floats scales =
        (scalar_floats)(uintptr_t)(g.w.s + ((size_t)tile.x * g.w.row_blocks + min((strip0 * F8_STRIP + rw * MR * 32) / F8_BLOCK, g.w.row_blocks - 1)) * blocks);

    f8_v16f acc[MR][MT];
#pragma unroll
    for (int i = 0; i < MR; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f8_v16f{0.0f};
    // this lane's places in a stage: its row's and its tokens'
    const uint32_t w_lane = (uint32_t)(rw * MR * 2 * F8_PIECE + (li >> 4) * F8_PIECE + lh * 1024 + (li & 15) * 16);
    uint32_t x_lane[4];
#pragma unroll
    for (int q = 0; q < 4; q++) x_lane[q] = (uint32_t)(T::W_BYTES + (tw * MT * 32 + li) * 256 + (((4 * q + 2 * lh) ^ (li & 15)) * 16));
    // product k: piece 2 (2 (k / 2) + lane / 32) + k % 2 of a token
    auto read_x = [&](const uint8_t *st, int j, int k) {
        return *reinterpret_cast<const f8_v8bf *>(st + j * 32 * 256 + (x_lane[k >> 1] ^ (uint32_t)((k & 1) * 16)));
    };
    auto read_w = [&](const uint8_t *st, int i, int k) { return *reinterpret_cast<const uint4 *>(st + i * 2 * F8_PIECE + w_lane + k * 256); };
    auto convert = [&](const uint4 (&raw)[4], int k) {  // product k's codes
        const uint4 &v = raw[k >> 1];
        const uint2 a = f8_to_bf16(k & 1 ? v.z : v.x, 1.0f), b = f8_to_bf16(k & 1 ? v.w : v.y, 1.0f);
        const uint4 both = make_uint4(a.x, a.y, b.x, b.y);
        f8_v8bf o;
        __builtin_memcpy(&o, &both, 16);
        return o;
    };

    // ---- A block is MR * MT steps of one tile's eight products.  Beside a step's products the wavefront adds the step before's sums, scaled,
    // converts the next row tile's codes (in a row tile's last step), and in a block's last row tile reads the next block's
    // tokens and first codes: that block is waited for in front of it, behind which nobody reads the present one any more.
    for (int a = 0; a < STAGES; a++)
        for (int c = 0; c < T::REQUESTS; c++) request(a, min(from + a, until - 1), c);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::REQUESTS * (STAGES - 1)) : "memory");
    lds_barrier();
    f8_v8bf x[MT][8], w[8];
    uint4 raw[4];
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
        for (int k = 0; k < 8; k++) x[j][k] = read_x(f8_lds, j, k);
#pragma unroll
    for (int k = 0; k < 4; k++) raw[k] = read_w(f8_lds, 0, k);
#pragma unroll
    for (int k = 0; k < 8; k++) w[k] = convert(raw, k);
    f8_v16f p[2] = {f8_v16f{0.0f}, f8_v16f{0.0f}};
    float s_before = 0.0f, s = scales[from];
    int slot = 0, next_slot = 1;
    constexpr int STEPS = MR * MT;
    static_assert(STEPS % 2 == 0, "the two sums");
    for (int b = from; b < until; b++) {
        const uint8_t *const st = f8_lds + (size_t)slot * T::STAGE, *const next = f8_lds + (size_t)next_slot * T::STAGE;
        const float s_next = scales[min(b + 1, until - 1)];
#pragma unroll
        for (int n = 0; n < STEPS; n++) {
            const int i = n / MT, j = n % MT;
            const bool last = i == MR - 1;  // the block's last row tile
            if (last && j == 0) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::REQUESTS * (STAGES - 2)) : "memory");
                lds_barrier();
                __builtin_amdgcn_s_setprio(1);
            }
            if (n == 0) __builtin_amdgcn_s_setprio(0);
            f8_v16f &sum = p[n & 1], &before = p[(n + 1) & 1];
            f8_v16f &to = n == 0 ? acc[MR - 1][MT - 1] : acc[(n - 1) / MT][(n - 1) % MT];
            const float by = n == 0 ? s_before : s;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (k == 0) sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[k], x[j][k], (f8_v16f{0.0f}), 0, 0, 0);
                else sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[k], x[j][k], sum, 0, 0, 0);
                if (j == 0 && k < 4) raw[k] = last ? read_w(next, 0, k) : read_w(st, i + 1, k);
                if (last) x[j][k] = read_x(next, j, k);
                to[2 * k] = __builtin_fmaf(before[2 * k], by, to[2 * k]);
                to[2 * k + 1] = __builtin_fmaf(before[2 * k + 1], by, to[2 * k + 1]);
                if (j == MT - 1) w[k] = convert(raw, k);
                if (last && j == 0) {  // (past the end the last block again, which nobody reads)
#pragma unroll
                    for (int c = k * T::REQUESTS / 8; c < (k + 1) * T::REQUESTS / 8; c++) request(slot, min(b + STAGES, until - 1), c);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" : "+v"(to));  // (the sums stay here: sunk further down, every product's are alive at once)
        }
        s_before = s;
        s = s_next;
        slot = next_slot;
        next_slot = next_slot == STAGES - 1 ? 0 : next_slot + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (nothing comes into LDS that is no longer this workgroup's)
#pragma unroll
    for (int r = 0; r < 16; r++) acc[MR - 1][MT - 1][r] = __builtin_fmaf(p[1][r], s_before, acc[MR - 1][MT - 1][r]);
    // register r of a lane: row 8 (r / 4) + 4 (lane / 32) + r % 4 of a tile, token lane % 32
    const bool wide = g.ldy % 4 == 0 && (g.w.rows & 3) == 0 && part_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(g.y) & 15) == 0;
#pragma unroll
    for (int j = 0; j < MT; j++) {
        const int t = (tw * MT + j) * 32 + li;
        if (t >= tile.z) continue;
        float *const dst = g.y + part * part_stride + (size_t)(tile.w + t) * g.ldy + y_col;
#pragma unroll
        for (int i = 0; i < MR; i++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int r0 = strip0 * F8_STRIP + (rw * MR + i) * 32 + 8 * q + 4 * lh;
                if (wide) {
                    if (r0 < g.w.rows) *reinterpret_cast<float4 *>(dst + r0) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (r0 + r < g.w.rows) dst[r0 + r] = acc[i][j][4 * q + r];
                }
            }
    }
#endif
}

template <int RW, int TW, int MR, int MT, int STAGES>
static int go_f8_tile(const F8Gemm &g, size_t tok_tiles, size_t matrices, int parts, size_t part_stride, hipStream_t s) {
    using T = F8TileShape<RW, TW, MR, MT, STAGES>;
    const size_t row_tiles = ((size_t)g.w.rows + T::ROWS - 1) / T::ROWS, total = row_tiles * tok_tiles;
    if (total > 0x7ffffff8u || matrices * parts > 65535) return set_error(FRK_ERR_SHAPE, "%zu x %zu tiles of %zu matrices: too many", row_tiles, tok_tiles, matrices);
    if (total == 0) return FRK_OK;
    // (a request's offset of a lane is 32 bits wide: a gathered row's from the first, others' from their tile's)
    if (g.src && (size_t)g.a.rows * g.w.blocks * (F8_BLOCK * 2) > 0xffffffffu)
        return set_error(FRK_ERR_SHAPE, "%d gathered rows of %d blocks: more than 4 GiB of quantized activations", g.a.rows, g.w.blocks);
    static bool sized = false;  // a benign race: every thread sets the same attribute
    if (!sized) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&f8_tile_kernel<RW, TW, MR, MT, STAGES>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)T::LDS);
        if (e != hipSuccess) return set_error(FRK_ERR_HIP, "hipFuncSetAttribute(f8_tile): %s", hipGetErrorString(e));
        sized = true;
    }
    hipLaunchKernelGGL((f8_tile_kernel<RW, TW, MR, MT, STAGES>), dim3((unsigned)((total + 7) / 8 * 8), (unsigned)(matrices * parts)), dim3(64 * T::WAVES), T::LDS, s,
                       g, (int)row_tiles, (int)tok_tiles, (int)matrices, parts, part_stride);
    FRK_LAUNCH_CHECK("f8_tile");
    return FRK_OK;
}
int launch_f8_tile(const F8Gemm &g, int tokens, size_t tok_tiles, size_t matrices, int parts, size_t part_stride, hipStream_t s) {
    if (tokens == 128) return go_f8_tile<4, 2, 2, 2, 2>(g, tok_tiles, matrices, parts, part_stride, s);
    if (tokens == 64) return go_f8_tile<2, 2, 2, 1, 2>(g, tok_tiles, matrices, parts, part_stride, s);
    return go_f8_tile<4, 1, 2, 1, 2>(g, tok_tiles, matrices, parts, part_stride, s);
}

}  // namespace frk
