// Products with weights in 8-bit floating point, a scale for each block of 128 x 128 (frk_f8.hpp), over large tiles: batches of
// more than a few dozen rows, dense and grouped.
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

// RW x TW wavefronts of four strips of 16 weight rows x MT strips of 16 tokens each
constexpr int F8_MR = 4;
template <int RW, int TW, int MT>
struct F8TileShape {
    static constexpr int SHAPE = TW == 2 ? F8_TILE_256x128 : RW == 4 ? F8_TILE_256x64 : F8_TILE_128x32;
    static constexpr int WAVES = RW * TW, ROWS = RW * F8_MR * F8_STRIP, TOKENS = TW * MT * 16, STAGES = 3;
    static constexpr int STAGE = TOKENS * F8_BLOCK * 2, REQUESTS = STAGE / 1024 / WAVES;  // of tokens; requests of a wavefront
    static_assert(REQUESTS * WAVES * 1024 == STAGE, "whole requests");
    static constexpr size_t LDS = STAGES * STAGE;
    static_assert(LDS <= 160 * 1024 && F8_BLOCK % (F8_MR * F8_STRIP) == 0, "LDS of a CU; a wavefront's rows in one block of scales");
    // a step is G row strips by all token strips: four chains of products that do not depend on each other
    static constexpr int G = MT >= 4 ? 1 : 4 / MT, STEPS = F8_MR / G;
    static_assert(F8_MR % G == 0 && STEPS % 2 == 0, "whole steps, the two sums");
};

template <int RW, int TW, int MT>
__global__ __launch_bounds__(64 * RW * TW, 2) void f8_tile_kernel(F8Gemm g, int row_tiles, int tok_tiles, int matrices, int parts, size_t part_stride) {
#if defined(__HIP_DEVICE_COMPILE__)
    using T = F8TileShape<RW, TW, MT>;
    static_assert(T::ROWS == F8_TILE_SIZE[T::SHAPE].rows && T::TOKENS == F8_TILE_SIZE[T::SHAPE].tokens && 64 * T::WAVES == F8_TILE_SIZE[T::SHAPE].threads, "the table");
    constexpr int MR = F8_MR, G = T::G, STEPS = T::STEPS, STAGES = T::STAGES;
    extern __shared__ __align__(16) uint8_t f8_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4;
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
    const int strip0 = row_tile * (T::ROWS / F8_STRIP) + rw * MR;  // of this wavefront

    // ---- tokens: a stage holds them 256 bytes each, piece p of token t in place (p / 4 + 4 (p % 4)) ^ t % 16.  (LDS serves lanes 0-3, 12-15 and
    // 20-27 of a 16-byte read together, 4-11 with 16-19 and 28-31: in place p ^ t % 16 every two of those share their banks.)
    uint32_t x_off[T::REQUESTS];
    const uint8_t *x_base = reinterpret_cast<const uint8_t *>(g.a.v);
    const int first_row = g.src ? 0 : min(tile.y, g.a.rows - 1);
    x_base += (size_t)first_row * blocks * (F8_BLOCK * 2);
#pragma unroll
    for (int c = 0; c < T::REQUESTS; c++) {
        const int t = (wave * T::REQUESTS + c) * 4 + (lane >> 4), i = min(t, tile.z - 1);
        const uint32_t row = (uint32_t)(min(max(g.src ? g.src[tile.y + i] : tile.y + i, 0), g.a.rows - 1) - first_row);
        const int place = (lane & 15) ^ (t & 15);
        x_off[c] = row * (uint32_t)blocks * (F8_BLOCK * 2) + (uint32_t)(place >> 2 | (place & 3) << 2) * 16;
    }
    auto request = [&](int slot, int b, int c) {
        dma16(lds0 + (uint32_t)slot * T::STAGE + (wave * T::REQUESTS + c) * 1024, x_base + (size_t)b * (F8_BLOCK * 2), x_off[c]);
    };
    const uint32_t x_lane = (uint32_t)((tw * MT * 16 + li) * 256 + ((lg ^ li) * 16));  // this lane's token's four pieces
    auto read_x = [&](const uint8_t *st, int j, int k) { return *reinterpret_cast<const f8_v8bf *>(st + j * 16 * 256 + (x_lane ^ (uint32_t)(k * 64))); };
    // ---- codes: straight into registers, a block ahead (LDS, at 128 bytes a cycle and CU, has enough to do with the tokens)
    const uint8_t *w_base[MR];
#pragma unroll
    for (int i = 0; i < MR; i++)
        w_base[i] = g.w.q + ((size_t)tile.x * g.w.strips + min(strip0 + i, g.w.strips - 1)) * blocks * F8_PIECE;
    uint4 raw[MR][2];
    auto load_w = [&](int i, int b) {
        const uint32_t off = (uint32_t)b * F8_PIECE + (uint32_t)lane * 16;
        raw[i][0] = *reinterpret_cast<const uint4 *>(w_base[i] + off);
        raw[i][1] = *reinterpret_cast<const uint4 *>(w_base[i] + off + 1024);
    };
    auto convert = [&](const uint4 (&r)[2], int k) {  // product k's codes
        const uint4 &v = r[k >> 1];
        const uint2 a = f8_to_bf16(k & 1 ? v.z : v.x, 1.0f), b = f8_to_bf16(k & 1 ? v.w : v.y, 1.0f);
        const uint4 both = make_uint4(a.x, a.y, b.x, b.y);
        f8_v8bf o;
        __builtin_memcpy(&o, &both, 16);
        return o;
    };
    // The scales of the next 64 blocks, one a lane: a scalar load in every block is waited for together with the reads of LDS, and a
    // vector load's wait would be one for the requests in flight too.
    const float *const scales = g.w.s + ((size_t)tile.x * g.w.row_blocks + min(strip0 * F8_STRIP / F8_BLOCK, g.w.row_blocks - 1)) * blocks;
    auto load_scales = [&](int first) {
        float v;
        asm volatile("global_load_dword %0, %1, %2\n\ts_waitcnt vmcnt(0)" : "=v"(v) : "v"((uint32_t)min(first + lane, blocks - 1) * 4u), "s"(scalar_pointer(scales)) : "memory");
        return v;
    };
    float lane_scales = load_scales(from);
    auto scale_of = [&](int b) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lane_scales), (b - from) & 63)); };

    f8_v4f acc[MR][MT];
#pragma unroll
    for (int i = 0; i < MR; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = f8_v4f{0.0f, 0.0f, 0.0f, 0.0f};

    // ---- A block is STEPS steps of four chains of four products.  Beside a step's products the wavefront adds the step before's sums, scaled,
    // converts the next step's codes and asks for those of the next block in their place; in a block's last step it reads the
    // next block's tokens, waited for in front of it.  By then everybody has the present block's in registers.
#pragma unroll
    for (int c = 0; c < T::REQUESTS; c++) request(0, from, c);
#pragma unroll
    for (int i = 0; i < MR; i++) load_w(i, from);
#pragma unroll
    for (int a = 1; a < STAGES; a++)
#pragma unroll
        for (int c = 0; c < T::REQUESTS; c++) request(a, min(from + a, until - 1), c);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(T::REQUESTS * (STAGES - 1)) : "memory");
    lds_barrier();
    f8_v8bf x[MT][4], w[G][4];
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) x[j][k] = read_x(f8_lds, j, k);
#pragma unroll
    for (int i = 0; i < G; i++) {
#pragma unroll
        for (int k = 0; k < 4; k++) w[i][k] = convert(raw[i], k);
        load_w(i, min(from + 1, until - 1));
    }
    f8_v4f p[2][G][MT];
#pragma unroll
    for (int i = 0; i < G; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) p[1][i][j] = f8_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float s_before = 0.0f, s = scale_of(from);
    int slot = 0, next_slot = 1;
    for (int b = from; b < until; b++) {
        const uint8_t *const next = f8_lds + (size_t)next_slot * T::STAGE;
        if (((b + 1 - from) & 63) == 0) lane_scales = load_scales(b + 1);
        const float s_next = scale_of(b + 1);
#pragma unroll
        for (int n = 0; n < STEPS; n++) {
            const bool last = n == STEPS - 1;
            if (last) {
                // the next block's tokens have landed: behind their requests there are at least a stage's and 6 loads of codes,
                // eight and more, of which at most eight may be on their way
                asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                lds_barrier();
                __builtin_amdgcn_s_setprio(1);
            }
            if (n == 0) __builtin_amdgcn_s_setprio(0);
            const int before = n == 0 ? STEPS - 1 : n - 1, after = last ? 0 : n + 1;  // steps
            const float by = n == 0 ? s_before : s;
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int i = 0; i < G; i++)
#pragma unroll
                    for (int j = 0; j < MT; j++) {
                        constexpr int CHAINS = G * MT, SLOTS = 4 * CHAINS;
                        const int at = (k * G + i) * MT + j;  // of SLOTS
                        f8_v4f &sum = p[n & 1][i][j];
                        if (k == 0) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i][k], x[j][k], (f8_v4f{0.0f, 0.0f, 0.0f, 0.0f}), 0, 0, 0);
                        else sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i][k], x[j][k], sum, 0, 0, 0);
                        if (last && i == G - 1) x[j][k] = read_x(next, j, k);
                        // one of the step before's sums: register at / CHAINS of chain at % CHAINS
                        f8_v4f &to = acc[before * G + at % CHAINS / MT][at % MT];
                        to[at / CHAINS] = __builtin_fmaf(p[(n + 1) & 1][at % CHAINS / MT][at % MT][at / CHAINS], by, to[at / CHAINS]);
                        if (j == MT - 1) w[i][k] = convert(raw[after * G + i], k);
                        if (at == SLOTS - 1) {
#pragma unroll
                            for (int c = 0; c < G; c++) load_w(after * G + c, min(b + (last ? 2 : 1), until - 1));
                        }
                        if (last) {  // (past the end the last block again, which nobody reads)
#pragma unroll
                            for (int c = at * T::REQUESTS / SLOTS; c < (at + 1) * T::REQUESTS / SLOTS; c++) request(slot, min(b + STAGES, until - 1), c);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
            for (int i = 0; i < G; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) asm volatile("" : "+v"(acc[before * G + i][j]));  // (sunk further down, every step's sums are alive at once)
        }
        s_before = s;
        s = s_next;
        slot = next_slot;
        next_slot = next_slot == STAGES - 1 ? 0 : next_slot + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (nothing comes into LDS that is no longer this workgroup's)
#pragma unroll
    for (int i = 0; i < G; i++)
#pragma unroll
        for (int j = 0; j < MT; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[(STEPS - 1) * G + i][j][r] = __builtin_fmaf(p[1][i][j][r], s_before, acc[(STEPS - 1) * G + i][j][r]);
    // register r of a lane: row 4 (lane / 16) + r of a strip, token lane % 16
    const bool wide = g.ldy % 4 == 0 && (g.w.rows & 3) == 0 && part_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(g.y) & 15) == 0;
#pragma unroll
    for (int j = 0; j < MT; j++) {
        const int t = (tw * MT + j) * 16 + li;
        if (t >= tile.z) continue;
        float *const dst = g.y + part * part_stride + (size_t)(tile.w + t) * g.ldy + y_col;
#pragma unroll
        for (int i = 0; i < MR; i++) {
            const int r0 = (strip0 + i) * F8_STRIP + 4 * lg;
            const float4 v = make_float4(acc[i][j][0] * F8_UP, acc[i][j][1] * F8_UP, acc[i][j][2] * F8_UP, acc[i][j][3] * F8_UP);
            if (wide) {
                if (r0 < g.w.rows) *reinterpret_cast<float4 *>(dst + r0) = v;
            } else {
                const float out[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (r0 + r < g.w.rows) dst[r0 + r] = out[r];
            }
        }
    }
#endif
}

template <int RW, int TW, int MT>
static int go_f8_tile(const F8Gemm &g, size_t tok_tiles, size_t matrices, int parts, size_t part_stride, hipStream_t s) {
    using T = F8TileShape<RW, TW, MT>;
    const size_t row_tiles = ((size_t)g.w.rows + T::ROWS - 1) / T::ROWS, total = row_tiles * tok_tiles;
    static bool sized = false;  // a benign race: every thread sets the same attribute
    if (!sized) {
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&f8_tile_kernel<RW, TW, MT>), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)T::LDS);
        if (e != hipSuccess) return set_error(FRK_ERR_HIP, "hipFuncSetAttribute(f8_tile): %s", hipGetErrorString(e));
        sized = true;
    }
    hipLaunchKernelGGL((f8_tile_kernel<RW, TW, MT>), dim3((unsigned)((total + 7) / 8 * 8), (unsigned)(matrices * parts)), dim3(64 * T::WAVES), T::LDS, s,
                       g, (int)row_tiles, (int)tok_tiles, (int)matrices, parts, part_stride);
    FRK_LAUNCH_CHECK("f8_tile");
    return FRK_OK;
}
int f8_tiles_fit(const frk_weights *w, int shape, size_t tok_tiles, size_t sheets, size_t gathered) {
    const F8Mat m = f8_mat(w);
    const F8TileSize t = F8_TILE_SIZE[shape];
    const size_t row_tiles = ((size_t)m.rows + t.rows - 1) / t.rows;
    if ((row_tiles * tok_tiles + 7) / 8 * 8 * t.threads > 0xffffffffu || sheets > 65535)
        return set_error(FRK_ERR_SHAPE, "%zu x %zu tiles %zu times: more than a grid holds", row_tiles, tok_tiles, sheets);
    // (a request's offset of a lane is 32 bits wide: a gathered row's from the first, others' from their tile's)
    if (gathered * m.blocks * (F8_BLOCK * 2) > 0xffffffffu)
        return set_error(FRK_ERR_SHAPE, "%zu gathered rows of %d blocks: more than 4 GiB of quantized activations", gathered, m.blocks);
    return FRK_OK;
}
int launch_f8_tile(const F8Gemm &g, int shape, size_t tok_tiles, size_t matrices, int parts, size_t part_stride, hipStream_t s) {
    switch (shape) {
    case F8_TILE_256x128: return go_f8_tile<4, 2, 4>(g, tok_tiles, matrices, parts, part_stride, s);
    case F8_TILE_256x64: return go_f8_tile<4, 1, 4>(g, tok_tiles, matrices, parts, part_stride, s);
    default: return go_f8_tile<2, 1, 2>(g, tok_tiles, matrices, parts, part_stride, s);
    }
}

}  // namespace frk
