// Routing by a rule (frk_hip_route_dev): scores softmax or sigmoid, a bias that takes part in the choice only, groups of
// experts, the top k, their weights.  The reference's counterparts live in crates/frink-moe; its plain softmax router with
// its f32 arithmetic is route_top_k_softmax_kernel (frk_moe.hip).
//
// Scores are doubles: two experts whose scores differ by less than an f32 step are chosen as their logits say, and the same
// whatever order a sum was added in.
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

// A wavefront a token, four to a workgroup; expert i lives in lane i % 64, register i / 64, n_experts <= 64 NR.
// Bound by the vector ALU: the scores' exponentials and divisions, then the k maxima, which are looked for among the scores' f32 roundings --
// a chain of DPP steps instead of trips through LDS for doubles -- and settled among the doubles where two share the largest.
constexpr int ROUTE_WAVES = 4;
template <int NR>
__global__ __launch_bounds__(64 * ROUTE_WAVES) void route_kernel(RouteArgs a) {
    __shared__ double choices[ROUTE_WAVES][64 * NR];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), n = a.n_experts;
    const size_t token = (size_t)blockIdx.x * ROUTE_WAVES + wave;
    if (token >= a.batch) return;
    const float *l = a.logits + token * n;
    const double out = -__builtin_inf();
    double p[NR], c[NR];
    float x[NR], bias[NR], top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NR; j++) x[j] = lane + 64 * j < n ? l[lane + 64 * j] : -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NR; j++) bias[j] = a.bias && lane + 64 * j < n ? a.bias[lane + 64 * j] : 0.0f;
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
    if (a.groups > 1) {
        double *const choice = choices[wave];
#pragma unroll
        for (int j = 0; j < NR; j++) choice[lane + 64 * j] = c[j];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (a wavefront reads its own stores only)
        const int size = n / a.groups;
        // a group by `lanes` lanes, a power of two
        const int lanes = 1 << (31 - __builtin_clz(64 / a.groups)), group = lane / lanes;
        double first = out, second = out;
        if (group < a.groups)
            for (int i = lane & (lanes - 1); i < size; i += lanes) {
                const double v = choice[group * size + i];
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
        for (int m = 1; m < lanes; m <<= 1) {
            const double f = __shfl_xor(first, m), s = __shfl_xor(second, m);
            second = fmax(fmin(first, f), fmax(second, s));
            first = fmax(first, f);
        }
        const double value = a.group_best == 2 && second > out ? first + second : first;
        // a group is used if fewer than top_groups stand before it
        int before = 0;
        for (int g = 0; g < a.groups; g++) {
            const double v = read_lane_f64(value, g * lanes);
            before += v > value || (v == value && g < group);
        }
        const uint64_t used = __ballot(group < a.groups && before < a.top_groups);
#pragma unroll
        for (int j = 0; j < NR; j++)
            if (lane + 64 * j < n && !(used >> ((uint32_t)(lane + 64 * j) * a.group_of >> 20) * lanes & 1)) c[j] = out;
    }
    uint32_t key[NR];
#pragma unroll
    for (int j = 0; j < NR; j++) key[j] = route_key(c[j]);
    int mine = -1;  // lane s keeps the s-th slot's expert
    for (int s = 0; s < a.k; s++) {
        uint32_t best = key[0];
#pragma unroll
        for (int j = 1; j < NR; j++) best = max(best, key[j]);
        best = wave_max_u32(best);
        if (best == 0) break;  // (uniform: no expert left)
        int at = 0, number = 0;
#pragma unroll
        for (int j = NR - 1; j >= 0; j--) {
            const uint64_t holders = __ballot(key[j] == best);
            if (holders) at = 64 * j + __builtin_ctzll(holders);
            number += __builtin_popcountll(holders);
        }
        if (number > 1) {  // (uniform) the largest of them, then the first that holds it
            double most = out;
#pragma unroll
            for (int j = 0; j < NR; j++) most = fmax(most, key[j] == best ? c[j] : out);
            most = wave_max_f64(most);
#pragma unroll
            for (int j = NR - 1; j >= 0; j--) {
                const uint64_t holders = __ballot(key[j] == best && c[j] == most);
                if (holders) at = 64 * j + __builtin_ctzll(holders);
            }
        }
#pragma unroll
        for (int j = 0; j < NR; j++)
            if (at >> 6 == j) key[j] = lane == (at & 63) ? 0u : key[j];  // (uniform condition)
        mine = lane == s ? at : mine;
    }
    double *const scores = choices[wave];
#pragma unroll
    for (int j = 0; j < NR; j++) scores[lane + 64 * j] = p[j];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    double w = mine >= 0 ? scores[mine] : 0.0;
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
    a.batch = batch;
    a.n_experts = n_experts;
    a.k = k;
    a.sigmoid = rule.score == FRK_SCORE_SIGMOID;
    a.norm = rule.norm;
    a.groups = rule.groups;
    a.top_groups = rule.top_groups;
    a.group_best = rule.group_best;
    const uint32_t size = (uint32_t)(n_experts / rule.groups);
    a.group_of = ((1u << 20) + size - 1) / size;
    a.scale = rule.scale;
    a.ids = ids;
    a.weights = weights;
#define FRK_GO(NR) hipLaunchKernelGGL(route_kernel<NR>, dim3((unsigned)((batch + ROUTE_WAVES - 1) / ROUTE_WAVES)), dim3(64 * ROUTE_WAVES), 0, s, a)
    if (n_experts <= 64) FRK_GO(1);
    else if (n_experts <= 128) FRK_GO(2);
    else if (n_experts <= 256) FRK_GO(4);
    else if (n_experts <= 512) FRK_GO(8);
    else FRK_GO(16);
#undef FRK_GO
    FRK_LAUNCH_CHECK("route");
    return FRK_OK;
}

}  // namespace frk
