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

// A wavefront a token; expert i lives in lane i % 64, register i / 64, n_experts <= 64 NR.
template <int NR>
__global__ __launch_bounds__(64) void route_kernel(RouteArgs a) {
    __shared__ double choice[64 * NR];
    const int lane = threadIdx.x, n = a.n_experts;
    const size_t token = blockIdx.x;
    const float *l = a.logits + token * n;
    const double out = -__builtin_inf();
    double p[NR], c[NR];
    float x[NR], top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NR; j++) {
        x[j] = lane + 64 * j < n ? l[lane + 64 * j] : -__builtin_inff();
        if (!(x[j] > -__builtin_inff())) x[j] = -__builtin_inff();  // (NaN: masked like -inf)
        top = fmaxf(top, x[j]);
    }
    if (a.sigmoid) {
#pragma unroll
        for (int j = 0; j < NR; j++) p[j] = x[j] > -__builtin_inff() ? 1.0 / (1.0 + exp(-(double)x[j])) : 0.0;
    } else {
        top = wave_max(top);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NR; j++) {
            // (+inf less +inf: those experts share)
            p[j] = x[j] > -__builtin_inff() ? (x[j] == top ? 1.0 : exp((double)x[j] - (double)top)) : 0.0;
            sum += p[j];
        }
        sum = wave_sum_f64(sum);
#pragma unroll
        for (int j = 0; j < NR; j++) p[j] = sum > 0.0 ? p[j] / sum : 0.0;
    }
#pragma unroll
    for (int j = 0; j < NR; j++) {
        const int i = lane + 64 * j;
        c[j] = x[j] > -__builtin_inff() ? (a.bias ? p[j] + (double)a.bias[i] : p[j]) : out;
        if (!(c[j] > out)) c[j] = out;  // (a bias that is NaN)
    }
    if (a.groups > 1) {
#pragma unroll
        for (int j = 0; j < NR; j++) choice[lane + 64 * j] = c[j];
        __syncthreads();
        const int size = n / a.groups;
        double value = out;
        if (lane < a.groups) {  // a group a lane
            double first = out, second = out;
            for (int i = 0; i < size; i++) {
                const double v = choice[lane * size + i];
                second = fmax(second, fmin(first, v));
                first = fmax(first, v);
            }
            value = a.group_best == 2 && second > out ? first + second : first;
        }
        // a group is used if fewer than top_groups stand before it
        int before = 0;
        for (int g = 0; g < a.groups; g++) {
            const double v = __shfl(value, g);
            before += v > value || (v == value && g < lane);
        }
        const uint64_t used = __ballot(lane < a.groups && before < a.top_groups);
#pragma unroll
        for (int j = 0; j < NR; j++)
            if (!(used >> ((lane + 64 * j) / size & 63) & 1)) c[j] = out;
    }
    double total = 0.0, mine = 0.0;  // lane s keeps the s-th slot
    int mine_i = -1;
    for (int s = 0; s < a.k; s++) {
        double best = out;
#pragma unroll
        for (int j = 0; j < NR; j++) best = fmax(best, c[j]);
        best = wave_max_f64(best);
        if (!(best > out)) break;  // (uniform: no expert left)
        int at = 0;
#pragma unroll
        for (int j = NR - 1; j >= 0; j--) {
            const uint64_t holders = __ballot(c[j] == best);
            if (holders) at = 64 * j + __builtin_ctzll(holders);
        }
        double w = 0.0;
#pragma unroll
        for (int j = 0; j < NR; j++)
            if (at == lane + 64 * j) w = p[j], c[j] = out;
        w = __shfl(w, at & 63);
        if (lane == s) mine = w, mine_i = at;
        total += w;
    }
    if (lane < a.k) {
        a.ids[token * a.k + lane] = mine_i;
        const double w = !a.norm ? mine : total > 0.0 ? mine / total : 0.0;
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
    a.scale = rule.scale;
    a.ids = ids;
    a.weights = weights;
#define FRK_GO(NR) hipLaunchKernelGGL(route_kernel<NR>, dim3((unsigned)batch), dim3(64), 0, s, a)
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
