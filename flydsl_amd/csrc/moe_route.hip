// Routing to experts with a bias for balance and groups of experts, in front of the expert sorter or a product grouped by expert (gfx950).
//
//   s = sigmoid(x) or softmax(x)     the experts' scores, x the router's logits
//   c = s + bias                     what is compared (c = s without a bias)
//   the experts lie in `groups` runs of equal length; a run is worth the sum of its two best c, or its best; the topk_groups best runs are kept
//   ids = the topk best c of these, weights = s[ids] (times 1 / max(their sum, 1e-20) if renormalised) times `scale`
// Of equal ones the lower index is taken.  Scores and comparisons are in 64 bits: of 256 experts' scores in 32 bits one token in 5,000 has two at the border that differ by less than their
// rounding, and which expert runs would hang on the order of a sum.  A logit of -Inf or NaN, and a c that is NaN, count as -Inf: such an expert is taken when nothing else
// is left, with weight 0.
//
// A token belongs to L lanes of a wavefront, a power of two, VPT experts to a lane; a lane's experts are of one run, so the runs' worth is one butterfly over the LG lanes of a run and
// their order a count of better ones.  A round of the selection is a tree over the lane's values, a butterfly over the token's lanes with v_max_f64 alone, and a ballot that finds the first
// lane that holds the maximum: no index travels with the values.  A taken value becomes NaN, which a maximum ignores.
// Bound: launch latency for decode; for prefill the rounds' dependent instructions.
#include "moe_gating.h"
#include "moe_route.h"

namespace {

template <int S>
__device__ __forceinline__ double route_xchg(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)gate_xchg<S>((int)(uint32_t)u), hi = (uint32_t)gate_xchg<S>((int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

template <int LO, int N, int VPT>
__device__ __forceinline__ double route_max(const double (&c)[VPT]) {
    if constexpr (N == 1) return c[LO];
    else return __builtin_fmax(route_max<LO, N / 2>(c), route_max<LO + N / 2, N / 2>(c));
}

template <typename T, int VPT>
__global__ void __launch_bounds__(256) k_route(RouteParams p) {
    const int L = p.lanes, sh = __builtin_ctz(L), gsh = __builtin_ctz(p.lanes_group);
    const int gl = (int)threadIdx.x & (L - 1), slot = (int)threadIdx.x >> sh;
    const int t = (int)blockIdx.x * (256 >> sh) + slot;
    const bool live = t < p.tokens;
    const int run = gl >> gsh, part = (gl & (p.lanes_group - 1)) * VPT;  // the lane's run of experts and its first one there
    const int size = p.experts / p.groups;
    const int have = run < p.groups ? (size - part < VPT ? size - part : VPT) : 0;  // experts of this lane (0 and less: none)
    const int c0 = run * size + part;
    const T* row = static_cast<const T*>(p.gating) + (size_t)(live ? t : 0) * p.experts;
    __shared__ float won[256 * GATE_KEEP];  // weights of a token's winners (topk <= experts <= 32 lanes, topk <= 32)
    float* mine = won + slot * p.topk;

    constexpr double NO = -__builtin_inf();
    double c[VPT];
    float w[VPT];
    float x[VPT], mx = -INFINITY;
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        x[v] = v < have ? gate_to_f32<T>(row[c0 + v]) : -INFINITY;
        if (!(x[v] >= -INFINITY)) x[v] = -INFINITY;  // NaN
        mx = fmaxf(mx, x[v]);
    }
    if (p.softmax) {
        gate_steps(sh, [&](auto S) { mx = fmaxf(mx, gate_xchg<decltype(S)::value>(mx)); });
        double sum = 0;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            c[v] = x[v] == mx ? 1.0 : exp((double)x[v] - (double)mx);  // (infinities share what there is; a row of -Inf is masked below)
            sum += x[v] == -INFINITY ? 0.0 : c[v];
        }
        gate_steps(sh, [&](auto S) { sum += route_xchg<decltype(S)::value>(sum); });
        const double inv = 1.0 / sum;
#pragma unroll
        for (int v = 0; v < VPT; v++) c[v] *= inv;
    } else {
#pragma unroll
        for (int v = 0; v < VPT; v++) c[v] = 1.0 / (1.0 + exp(-(double)x[v]));
    }
#pragma unroll
    for (int v = 0; v < VPT; v++) {
        w[v] = (float)c[v];
        if (p.bias && v < have) c[v] += (double)p.bias[c0 + v];
        if (x[v] == -INFINITY || c[v] != c[v]) c[v] = NO, w[v] = 0.0f;
    }

    if (p.topk_groups < p.groups) {
        double m1 = NO, m2 = NO;  // the lane's two best
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            m2 = __builtin_fmax(m2, __builtin_fmin(m1, c[v]));
            m1 = __builtin_fmax(m1, c[v]);
        }
        gate_steps(gsh, [&](auto S) {
            const double o1 = route_xchg<decltype(S)::value>(m1), o2 = route_xchg<decltype(S)::value>(m2);
            m2 = __builtin_fmax(__builtin_fmin(m1, o1), __builtin_fmax(m2, o2));
            m1 = __builtin_fmax(m1, o1);
        });
        const double worth = !p.top2 ? m1 : m2 == NO ? NO : m1 + m2;
        int better = 0;
        for (int r = 0; r < p.groups; r++) {
            const double o = __shfl(worth, ((int)threadIdx.x & 63 & ~(L - 1)) + (r << gsh), 64);
            better += (o > worth) | ((o == worth) & (r < run));
        }
        if (better >= p.topk_groups) {
#pragma unroll
            for (int v = 0; v < VPT; v++) c[v] = NO, w[v] = 0.0f;
        }
    }
#pragma unroll
    for (int v = 0; v < VPT; v++) c[v] = v < have ? c[v] : __builtin_nan("");

    const int shift = (int)threadIdx.x & 63 & ~(L - 1);
    const uint64_t token_lanes = (L == 64 ? ~0ull : (1ull << L) - 1);
    for (int k = 0; k < p.topk; k++) {
        const double local = route_max<0, VPT>(c);
        double best = local;
        gate_steps(sh, [&](auto S) { best = __builtin_fmax(best, route_xchg<decltype(S)::value>(best)); });
        const uint64_t holders = (__ballot(local == best) >> shift) & token_lanes;
        if (gl == __builtin_ctzll(holders | (1ull << 63))) {
            bool open = true;
            int at = 0;
            float weight = 0.0f;
#pragma unroll
            for (int v = 0; v < VPT; v++) {
                const bool take = open & (c[v] == best);
                at = take ? v : at;
                weight = take ? w[v] : weight;
                c[v] = take ? __builtin_nan("") : c[v];
                open = open & !take;
            }
            mine[k] = weight;
            if (live) p.indices[(size_t)t * p.topk + k] = c0 + at;
        }
    }
    wave_lds_order();  // (a token's lanes are neighbours in one wavefront)
    float sum = 0.0f;
    if (p.renorm)
        for (int k = 0; k < p.topk; k++) sum += mine[k];
    const float over = p.renorm ? fmaxf(sum, 1e-20f) : 1.0f;
    if (live)
        for (int k = gl; k < p.topk; k += L) p.weights[(size_t)t * p.topk + k] = mine[k] / over * p.scale;
}

template <typename T>
hipError_t launch_t(const RouteParams& p, int vpt, hipStream_t stream) {
    const int per = 256 / p.lanes;
    const dim3 grid((unsigned)((p.tokens + per - 1) / per)), block(256);
    switch (vpt) {
        case 4: hipLaunchKernelGGL((k_route<T, 4>), grid, block, 0, stream, p); break;
        case 8: hipLaunchKernelGGL((k_route<T, 8>), grid, block, 0, stream, p); break;
        case 16: hipLaunchKernelGGL((k_route<T, 16>), grid, block, 0, stream, p); break;
        default: hipLaunchKernelGGL((k_route<T, 32>), grid, block, 0, stream, p); break;
    }
    return hipGetLastError();
}

inline int up2(int v) {
    int p = 1;
    while (p < v) p <<= 1;
    return p;
}

}  // namespace

// dtype: 0 fp32, 1 bf16, 2 fp16
hipError_t psg_launch_moe_route(RouteParams p, int dtype, hipStream_t stream) {
    if (p.topk_groups >= p.groups) p.groups = p.topk_groups = 1;  // every run is kept: one run
    const int size = p.experts / p.groups;
    // the fewest values a lane that 64 lanes allow: with up to 64 runs of a power of two of lanes each, 32 hold 1024 experts in any division
    int vpt = 4;
    while (up2(p.groups) * up2((size + vpt - 1) / vpt) > 64) vpt <<= 1;
    p.lanes_group = up2((size + vpt - 1) / vpt);
    p.lanes = up2(p.groups) * p.lanes_group;
    switch (dtype) {
        case 0: return launch_t<float>(p, vpt, stream);
        case 1: return launch_t<uint16_t>(p, vpt, stream);
        case 2: return launch_t<_Float16>(p, vpt, stream);
    }
    return hipErrorInvalidValue;
}
