// Routing by a rule (frk_hip_route_dev): scores softmax or sigmoid, a bias that takes part in the choice only, groups of
// experts, the top k, their weights.  The reference's counterparts live in crates/frink-moe; its plain softmax router with
// its f32 arithmetic is route_top_k_softmax_kernel (frk_moe.hip).
//
// Scores are doubles, so that experts whose scores differ by less than an f32 step are told apart; scores that are the same double go by
// index (sigmoids of logits above 37 are all one).
#include "frk_device.hpp"

#include <algorithm>

namespace frk {

#define FRK_LAUNCH_CHECK(what)                                                                          \
    do {                                                                                                \
        hipError_t e_ = hipGetLastError();                                                              \
        if (e_ != hipSuccess) return set_error(FRK_ERR_HIP, what " launch: %s", hipGetErrorString(e_)); \
    } while (0)

struct RouteArgs {
    const float *logits, *bias;
    size_t batch;
    int n_experts, k, sigmoid, norm, groups, top_groups, group_best;
    bool wide;          // a lane's experts in one load, of logits and bias
    int group_lanes;    // a group is that many whole lanes' experts (a power of two up to 16); 0: it isn't
    uint32_t group_of;  // expert i of group size s: i * group_of >> 20 = i / s, group_of = ceil(2^20 / s), for i and s up to 1024
    float scale;
    int32_t *ids;
    float *weights;
};

__device__ __forceinline__ double wave_max_f64(double v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = fmax(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {  // uniform
    v = max(v, (uint32_t)dpp_i<DPP_QUAD_XOR1>((int)v));
    v = max(v, (uint32_t)dpp_i<DPP_QUAD_XOR2>((int)v));
    v = max(v, (uint32_t)dpp_i<DPP_HALF_MIRROR>((int)v));
    v = max(v, (uint32_t)dpp_i<DPP_ROW_MIRROR>((int)v));
#if defined(__HIP_DEVICE_COMPILE__)
    const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)rows[0], (uint32_t)rows[1]);
    return max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 32));
#else
    return v;
#endif
}
__device__ __forceinline__ double read_lane_f64(double v, int lane) {  // lane: uniform
    const int lo = __builtin_amdgcn_readlane(__double2loint(v), lane), hi = __builtin_amdgcn_readlane(__double2hiint(v), lane);
    return __hiloint2double(hi, lo);
}
// Numbers in the order of their f32 roundings (which keep the order of doubles, but for making some equal); 0: none
__device__ __forceinline__ uint32_t route_key(double c) {
    const uint32_t bits = __float_as_uint((float)c);
    return c > -__builtin_inf() ? (bits & 0x80000000u ? ~bits : bits | 0x80000000u) : 0u;
}

// exp(y) for y <= 0: y = n ln 2 + r, |r| <= ln 2 / 2, the exponential's series to r^13 (the next term is below 2^-57) and 2^n, within a
// unit or so in the last place; gradual below 2^-1022, 0 from -746 on.  Half the instructions of the library's, which has no such bounds
// to rely on: 16384 tokens of 256 experts 33 -> 30 us.
__device__ __forceinline__ double route_exp(double y) {
    y = fmax(y, -746.0);
    const double n = __builtin_rint(y * 1.4426950408889634);
    // ln 2 as two numbers, the first with zeros behind its upper 32 bits so that n times it is exact
    double r = __builtin_fma(-n, 0x1.62e42feep-1, y);
    r = __builtin_fma(-n, 0x1.a39ef35793c76p-33, r);
    double s = 1.0 / 6227020800.0;
    s = __builtin_fma(s, r, 1.0 / 479001600.0);
    s = __builtin_fma(s, r, 1.0 / 39916800.0);
    s = __builtin_fma(s, r, 1.0 / 3628800.0);
    s = __builtin_fma(s, r, 1.0 / 362880.0);
    s = __builtin_fma(s, r, 1.0 / 40320.0);
    s = __builtin_fma(s, r, 1.0 / 5040.0);
    s = __builtin_fma(s, r, 1.0 / 720.0);
    s = __builtin_fma(s, r, 1.0 / 120.0);
    s = __builtin_fma(s, r, 1.0 / 24.0);
    s = __builtin_fma(s, r, 1.0 / 6.0);
    s = __builtin_fma(s, r, 0.5);
    s = __builtin_fma(s, r, 1.0);
    s = __builtin_fma(s, r, 1.0);
    return ldexp(s, (int)n);
}
// 1 / d for d in [1, 1024 * 2^10]: the reciprocal instruction's and two steps of Newton's
__device__ __forceinline__ double route_reciprocal(double d) {
#if defined(__HIP_DEVICE_COMPILE__)
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
#else
    return 1.0 / d;
#endif
}

// the lane that holds the other half of a run of 2^(step + 1) lanes, each half of which agrees already; step < 4
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    return __hiloint2double(dpp_i<CTRL>(__double2hiint(v)), dpp_i<CTRL>(__double2loint(v)));
}
struct Best2 {
    double first, second;
};
__device__ __forceinline__ Best2 best2(const Best2 &a, const Best2 &b) {
    return {fmax(a.first, b.first), fmax(fmin(a.first, b.first), fmax(a.second, b.second))};
}
template <int CTRL>
__device__ __forceinline__ Best2 best2_dpp(const Best2 &a) {
    return best2(a, Best2{dpp_f64<CTRL>(a.first), dpp_f64<CTRL>(a.second)});
}
template <int NR>
__device__ __forceinline__ void route_load(const float *__restrict__ from, int n, bool wide, int lane, float missing, float (&v)[NR]) {
    if (wide && NR > 1) {
        if (lane * NR < n) {
            constexpr int W = NR < 4 ? NR : 4;
            typedef float vec __attribute__((ext_vector_type(W)));
#pragma unroll
            for (int q = 0; q < NR / W; q++) {
                const vec t = reinterpret_cast<const vec *>(from + lane * NR)[q];
#pragma unroll
                for (int j = 0; j < W; j++) v[W * q + j] = t[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < NR; j++) v[j] = missing;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < NR; j++) v[j] = lane * NR + j < n ? from[lane * NR + j] : missing;
}

// A wavefront a token, four to a workgroup; lane l holds experts NR l .. NR l + NR - 1, n_experts <= 64 NR.
// Bound by issue: the scores' exponentials and divisions, the groups' best, then the k maxima, which are looked for among the scores' f32 roundings --
// a chain of DPP steps instead of trips through LDS for doubles -- and settled among the doubles where two share one.
constexpr int ROUTE_WAVES = 4;
template <int NR>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_kernel(RouteArgs a) {
    __shared__ __align__(16) double choices[ROUTE_WAVES][64 * NR];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = a.n_experts;
    const size_t token = (size_t)blockIdx.x * ROUTE_WAVES + wave;
    if (token >= a.batch) return;
    const double out = -__builtin_inf();
    double p[NR], c[NR];
    float x[NR], bias[NR], top = -__builtin_inff();
    route_load<NR>(a.logits + token * n, n, a.wide, lane, -__builtin_inff(), x);
#pragma unroll
    for (int j = 0; j < NR; j++) bias[j] = 0.0f;
    if (a.bias) route_load<NR>(a.bias, n, a.wide, lane, 0.0f, bias);
#pragma unroll
    for (int j = 0; j < NR; j++) {
        if (!(x[j] > -__builtin_inff())) x[j] = -__builtin_inff();  // (NaN: masked like -inf)
        top = fmaxf(top, x[j]);
    }
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < NR; j++) {  // 1 / (1 + e) or e / (1 + e) with e = exp(-|x|): no overflow
            const double e = route_exp(-fabs((double)x[j]));
            const double r = route_reciprocal(1.0 + e);
            p[j] = x[j] >= 0.0f ? r : e * r;
        }
    } else {
        top = wave_max(top);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NR; j++) {
            // (+inf less +inf: those experts share)
            p[j] = x[j] > -__builtin_inff() ? (x[j] == top ? 1.0 : route_exp((double)x[j] - (double)top)) : 0.0;
            sum += p[j];
        }
        sum = wave_sum_f64(sum);
        const double by = sum > 0.0 ? route_reciprocal(sum) : 0.0;
#pragma unroll
        for (int j = 0; j < NR; j++) p[j] *= by;
    }
#pragma unroll
    for (int j = 0; j < NR; j++) {
        c[j] = x[j] > -__builtin_inff() ? p[j] + (double)bias[j] : out;
        if (!(c[j] > out)) c[j] = out;  // (a bias that is NaN)
    }
    double *const shared = choices[wave];
    if (a.groups > 1) {
        Best2 best{out, out};
        int lanes, group;
        if (a.group_lanes) {
            lanes = a.group_lanes;
            group = lane / lanes;  // (a power of two)
#pragma unroll
            for (int j = 0; j < NR; j++) best = best2(best, Best2{c[j], out});
            if (lanes > 1) best = best2_dpp<DPP_QUAD_XOR1>(best);
            if (lanes > 2) best = best2_dpp<DPP_QUAD_XOR2>(best);
            if (lanes > 4) best = best2_dpp<DPP_HALF_MIRROR>(best);
            if (lanes > 8) best = best2_dpp<DPP_ROW_MIRROR>(best);
        } else {
            const int size = n / a.groups;
#pragma unroll
            for (int j = 0; j < NR; j++) shared[lane * NR + j] = c[j];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wavefront reads its own stores only)
            // a group by `lanes` lanes, a power of two
            lanes = 1 << (31 - __builtin_clz(64 / a.groups));
            group = lane / lanes;
            if (group < a.groups)
                for (int i = lane & (lanes - 1); i < size; i += lanes) best = best2(best, Best2{shared[group * size + i], out});
            for (int m = 1; m < lanes; m <<= 1) best = best2(best, Best2{__shfl_xor(best.first, m), __shfl_xor(best.second, m)});
        }
        const double value = a.group_best == 2 && best.second > out ? best.first + best.second : best.first;
        // a group is used if fewer than top_groups stand before it
        int before = 0;
        for (int g = 0; g < a.groups; g++) {
            const double v = read_lane_f64(value, g * lanes);
            before += v > value || (v == value && g < group);
        }
        const bool mine_used = group < a.groups && before < a.top_groups;
        if (a.group_lanes) {
#pragma unroll
            for (int j = 0; j < NR; j++) c[j] = mine_used ? c[j] : out;
        } else {
            const uint64_t used = __ballot(mine_used);
#pragma unroll
            for (int j = 0; j < NR; j++)
                if (lane * NR + j < n && !(used >> ((uint32_t)(lane * NR + j) * a.group_of >> 20) * lanes & 1)) c[j] = out;
        }
    }
    uint32_t key[NR];
#pragma unroll
    for (int j = 0; j < NR; j++) key[j] = route_key(c[j]);
    int mine = -1;  // lane s keeps the s-th slot's expert
    bool settled = false;
    if (NR <= 4) {
        // a lane's keys in falling order, so that only the first of each lane stand for election
        uint32_t sorted[NR], order[NR];
#pragma unroll
        for (int j = 0; j < NR; j++) sorted[j] = key[j], order[j] = (uint32_t)j;
        auto exchange = [&](int i, int j) {
            const bool turn = sorted[i] < sorted[j];
            const uint32_t big = turn ? sorted[j] : sorted[i], small = turn ? sorted[i] : sorted[j];
            const uint32_t of_big = turn ? order[j] : order[i], of_small = turn ? order[i] : order[j];
            sorted[i] = big, sorted[j] = small, order[i] = of_big, order[j] = of_small;
        };
        if (NR == 2) exchange(0, NR - 1);
        if (NR == 4) exchange(0, NR / 4), exchange(NR / 2, NR - 1), exchange(0, NR / 2), exchange(NR / 4, NR - 1), exchange(NR / 4, NR / 2);
        bool shared_key = false;
        uint32_t rest = 0;  // the order, the first in the lowest bits
#pragma unroll
        for (int j = 0; j < NR; j++) {
            if (j > 0) shared_key |= sorted[j] == sorted[j - 1] && sorted[j] != 0;
            rest |= order[j] << (2 * j);
        }
        settled = __ballot(shared_key) == 0;
        for (int s = 0; settled && s < a.k; s++) {
            const uint32_t best = wave_max_u32(sorted[0]);
            if (best == 0) break;  // (uniform: no expert left)
            const uint64_t holders = __ballot(sorted[0] == best);
            settled = (holders & (holders - 1)) == 0;
            const int winner = __builtin_ctzll(holders);
            const int at = winner * NR + (int)((uint32_t)__builtin_amdgcn_readlane((int)rest, winner) & 3u);
            mine = lane == s ? at : mine;
            const bool won = lane == winner;
#pragma unroll
            for (int j = 0; j < NR; j++) sorted[j] = won ? (j + 1 < NR ? sorted[j + 1 < NR ? j + 1 : j] : 0u) : sorted[j];
            rest = won ? rest >> 2 : rest;
        }
    }
    if (!settled) {  // (uniform)
        mine = -1;
        for (int s = 0; s < a.k; s++) {
            uint32_t best = key[0];
#pragma unroll
            for (int j = 1; j < NR; j++) best = max(best, key[j]);
            best = wave_max_u32(best);
            if (best == 0) break;  // (uniform: no expert left)
            uint64_t holders[NR], any = 0;
            int number = 0;
#pragma unroll
            for (int j = 0; j < NR; j++) {
                holders[j] = __ballot(key[j] == best);
                any |= holders[j];
                number += __builtin_popcountll(holders[j]);
            }
            if (number > 1) {  // (uniform) the largest of them, then the first that holds it
                double most = out;
#pragma unroll
                for (int j = 0; j < NR; j++) most = fmax(most, key[j] == best ? c[j] : out);
                most = wave_max_f64(most);
                any = 0;
#pragma unroll
                for (int j = 0; j < NR; j++) {
                    holders[j] = __ballot(key[j] == best && c[j] == most);
                    any |= holders[j];
                }
            }
            const int winner = __builtin_ctzll(any);
            int place = 0;
#pragma unroll
            for (int j = NR - 1; j >= 0; j--) place = holders[j] >> winner & 1 ? j : place;
#pragma unroll
            for (int j = 0; j < NR; j++) key[j] = lane == winner && j == place ? 0u : key[j];
            mine = lane == s ? winner * NR + place : mine;
        }
    }
#pragma unroll
    for (int j = 0; j < NR; j++) shared[lane * NR + j] = p[j];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    double w = mine >= 0 ? shared[mine] : 0.0;
    if (a.norm) {
        const double total = wave_sum_f64(w);
        w = total > 0.0 ? w / total : 0.0;
    }
    if (lane < a.k) {
        a.ids[token * a.k + lane] = mine;
        a.weights[token * a.k + lane] = (float)(w * (double)a.scale);
    }
}

int launch_route(const float *logits, size_t batch, int n_experts, int k, const frk_route_rule &rule, int32_t *ids, float *weights, hipStream_t s) {
    RouteArgs a;
    a.logits = logits;
    a.bias = rule.bias_dev;
    a.n_experts = n_experts;
    a.k = k;
    a.sigmoid = rule.score == FRK_SCORE_SIGMOID;
    a.norm = rule.norm;
    a.groups = rule.groups;
    a.top_groups = rule.top_groups;
    a.group_best = rule.group_best;
    const uint32_t size = (uint32_t)(n_experts / rule.groups);
    a.group_of = ((1u << 20) + size - 1) / size;
    int nr = 1;
    while (64 * nr < n_experts) nr *= 2;
    a.wide = n_experts % nr == 0 && ((uintptr_t)logits | (uintptr_t)(rule.bias_dev ? rule.bias_dev : logits)) % (4 * std::min(nr, 4)) == 0;
    const uint32_t lanes = size % nr == 0 ? size / nr : 0;
    a.group_lanes = lanes && (lanes & (lanes - 1)) == 0 && lanes <= 16 ? (int)lanes : 0;
    a.scale = rule.scale;
    a.ids = ids;
    a.weights = weights;
    // (a grid holds fewer than 2^32 threads, 64 a token)
    constexpr size_t TOKENS = (size_t)1 << 25;
    for (size_t first = 0; first < batch; first += TOKENS) {
        a.batch = std::min(TOKENS, batch - first);
#define FRK_GO(NR) hipLaunchKernelGGL(route_kernel<NR>, dim3((unsigned)((a.batch + ROUTE_WAVES - 1) / ROUTE_WAVES)), dim3(64 * ROUTE_WAVES), 0, s, a)
        switch (nr) {
        case 1: FRK_GO(1); break;
        case 2: FRK_GO(2); break;
        case 4: FRK_GO(4); break;
        case 8: FRK_GO(8); break;
        default: FRK_GO(16); break;
        }
#undef FRK_GO
        FRK_LAUNCH_CHECK("route");
        a.logits += TOKENS * (size_t)n_experts;
        a.ids += TOKENS * (size_t)k;
        a.weights += TOKENS * (size_t)k;
    }
    return FRK_OK;
}

}  // namespace frk
