// Routing to experts with a bias for balance and groups of experts, in front of the expert sorter or a product grouped by expert (gfx950).
//
//   s = sigmoid(x) or softmax(x)     the experts' scores, x the router's logits
//   c = s + bias                     what is compared (without a bias x itself, which orders like s)
//   the experts lie in `groups` runs of equal length; a run is worth the sum of its two best c, or its best; the topk_groups best runs are kept
//   ids = the topk best c of these, weights = s[ids] (times 1 / max(their sum, 1e-20) if renormalised) times `scale`
// Of equal ones the lower index is taken.  Scores and comparisons are in 64 bits: of 256 experts' scores in 32 bits one token in 5,000 has two at the border that differ by less than their
// rounding, and which expert runs would hang on the order of a sum.  A logit of -Inf or NaN, and a c that is NaN, count as -Inf: such an expert is taken when nothing else
// is left, with weight 0.
//
// 64 bits for all experts are ten times the instructions, so the experts are selected in 32 bits first, and looked at in 64 afterwards: the topk taken, one a lane, must lie in their order, and the last of
// them above the best that was not taken by more than the 32 bits may be off.  Where that does not hold for a token (one in some hundreds), its wavefront selects again in 64 bits.
// A token belongs to L lanes of a wavefront, a power of two, VPT experts to a lane; a lane's experts are of one run, so the runs' worth is one butterfly over the LG lanes of a run and their order a
// count of better ones.  In 32 bits a value is an unsigned number that orders like the float, its last bits replaced by the expert's place in the lane; a lane sorts its own once
// (a network of minimum and maximum), and a round is a butterfly of v_max_u32 over the token's lanes' first ones, a ballot for the first lane that holds the maximum, and a step forward in that lane.
// Weights stay in 64 bits until they are stored.
// Bound: launch latency for decode (1 x 256 of 8 groups: 6.1 us); for prefill the instructions, 16384 x 256 in 25.5 us, 934 vector instructions a wavefront of two tokens (with all of it in 64 bits the best split
// took 26.4, by softmax 22.4 against 19.1, and a token alone 6.8).
#include "moe_gating.h"
#include "moe_route.h"
#include <type_traits>

namespace {

// lane ^ 16 and ^ 32 as vector instructions (the crossbar takes a hundred cycles): both halves of the pair, in an order that does not matter to what is done with them
template <int S, class F>
__device__ __forceinline__ uint32_t route_join(uint32_t v, F&& f) {
    if constexpr (S < 4) {
        return f(v, (uint32_t)gate_xchg<S>((int)v));
    } else {
        const auto r = S == 4 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return f((uint32_t)r[0], (uint32_t)r[1]);
    }
}
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

// 1 / d for d in [1, infinity], to a unit in the last place (infinity as 2^1022)
__device__ __forceinline__ double route_rcp(double d) {
    d = __builtin_fmin(d, 0x1p1022);
    double r = __builtin_amdgcn_rcp(d);
    r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
}

// an unsigned number that orders like the float (no NaN), and back
__device__ __forceinline__ uint32_t route_key(float f) {
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float route_value(uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// s[0] >= s[1] >= ...: K. Batcher's odd-even merges ("Sorting networks and their applications", 1968)
template <int LO, int N, int R, int VPT>
__device__ __forceinline__ void route_merge(uint32_t (&s)[VPT]) {
    auto order = [&](int a, int b) __attribute__((always_inline)) {
        const uint32_t hi = s[a] > s[b] ? s[a] : s[b], lo = s[a] > s[b] ? s[b] : s[a];
        s[a] = hi, s[b] = lo;
    };
    if constexpr (2 * R < N) {
        route_merge<LO, N, 2 * R>(s);
        route_merge<LO + R, N, 2 * R>(s);
#pragma unroll
        for (int i = LO + R; i + R < LO + N; i += 2 * R) order(i, i + R);
    } else {
        order(LO, LO + R);
    }
}
template <int LO, int N, int VPT>
__device__ __forceinline__ void route_sort(uint32_t (&s)[VPT]) {
    if constexpr (N > 1) {
        route_sort<LO, N / 2>(s);
        route_sort<LO + N / 2, N / 2>(s);
        route_merge<LO, N, 1>(s);
    }
}

// How far a score + bias in 32 bits may be from the same in 64: the exponential is off by a unit, 2^-23, and by the rounding of its argument, |a| 2^-22.8 of which at most a |a| exp(-|a|) <= 0.37th part, or
// a quarter for a sigmoid, is left in the score; the sum or 1 + e, its reciprocal and their product by 2^-23 each, so a score, 1 at most, by 2^-20.8 altogether; and half a unit of the sum with the bias
__device__ __forceinline__ float route_slack(float f) { return __builtin_fmaf(fabsf(f), 0x1p-24f, 0x1p-20f); }

struct Winner {
    double c;       // what was compared
    double weight;  // score
    int index;      // negative: not to be taken, but nothing else was left
};

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
    const bool bias = p.bias != nullptr, some = p.topk_groups < p.groups;
    extern __shared__ Winner winners[];  // topk + 1 a token
    Winner* const mine = winners + slot * (p.topk + 1);

    constexpr uint32_t PLACE = VPT - 1;
    constexpr double NO = -__builtin_inf();
    double mx = 0, inv = 1.0;
    // the lane's logits and bias; what is not there is read from the front (a load behind a branch waits by itself, sixteen of them took 12 us)
    float x[VPT], b[VPT];
    auto fetch = [&](auto* from, auto to_f32, float (&out)[VPT]) __attribute__((always_inline)) {
        using E = std::remove_cv_t<std::remove_pointer_t<decltype(from)>>;
        if (p.vec) {  // every lane's are there or none, on as many bytes
            struct alignas(sizeof(E) * VPT < 16 ? sizeof(E) * VPT : 16) Vec { E v[VPT]; };
            const Vec raw = *reinterpret_cast<const Vec*>(from + (have > 0 ? c0 : 0));
#pragma unroll
            for (int v = 0; v < VPT; v++) out[v] = to_f32(raw.v[v]);
        } else {
            E raw[VPT];
#pragma unroll
            for (int v = 0; v < VPT; v++) raw[v] = from[v < have ? c0 + v : 0];
#pragma unroll
            for (int v = 0; v < VPT; v++) out[v] = to_f32(raw[v]);
        }
    };
    fetch(row, [](T l) { return gate_to_f32<T>(l); }, x);
    if (bias) fetch(p.bias, [](float f) { return f; }, b);
#pragma unroll
    for (int v = 0; v < VPT; v++) x[v] = v < have && x[v] > -INFINITY ? x[v] + 0.0f : -INFINITY;  // (NaN too; and -0 to +0, which it equals but whose number below would be lower)
    // the score but for the softmax's sum; infinities share what there is
    auto score = [&](float l) __attribute__((always_inline)) {
        if (p.softmax) return l == (float)mx ? 1.0 : exp((double)l - mx);
        return route_rcp(1.0 + exp(-(double)l));
    };
    auto score32 = [&](float l) __attribute__((always_inline)) {
        if (p.softmax) return l == (float)mx ? (float)inv : __builtin_amdgcn_exp2f((l - (float)mx) * 1.44269504f) * (float)inv;
        return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(l * -1.44269504f));
    };
    if (p.softmax) {
        float m = -INFINITY;
#pragma unroll
        for (int v = 0; v < VPT; v++) m = fmaxf(m, x[v]);
        gate_steps(sh, [&](auto S) { m = fmaxf(m, gate_xchg<decltype(S)::value>(m)); });
        mx = m;
        double sum = 0;
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            sum += x[v] > -INFINITY ? score(x[v]) : 0.0;
            asm volatile("" : "+v"(sum));  // (one after the other: sixteen exponentials at once take 300 registers)
        }
        gate_steps(sh, [&](auto S) { sum += route_xchg<decltype(S)::value>(sum); });
        inv = 1.0 / sum;
    }
    // what the winner of expert e is compared by, and its score
    auto look = [&](int e, double& c, double& weight) __attribute__((always_inline)) {
        const float l = gate_to_f32<T>(row[e]);
        const double s = score(l) * inv;
        c = bias ? s + (double)p.bias[e] : (double)l;
        weight = s;
    };

    const int shift = (int)threadIdx.x & 63 & ~(L - 1);
    const uint64_t token_lanes = L == 64 ? ~0ull : (1ull << L) - 1;
    bool again = false;  // this token needs 64 bits
    {
        float f[VPT];
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            f[v] = x[v];
            if (bias) f[v] = score32(x[v]) + b[v];
            if (!(x[v] > -INFINITY) || f[v] != f[v]) f[v] = -INFINITY;
        }
        if (some) {
            float m1 = -INFINITY, m2 = -INFINITY;  // the lane's two best
#pragma unroll
            for (int v = 0; v < VPT; v++) {
                m2 = fmaxf(m2, fminf(m1, f[v]));
                m1 = fmaxf(m1, f[v]);
            }
            gate_steps(gsh, [&](auto S) {
                const float o1 = gate_xchg<decltype(S)::value>(m1), o2 = gate_xchg<decltype(S)::value>(m2);
                m2 = fmaxf(fminf(m1, o1), fmaxf(m2, o2));
                m1 = fmaxf(m1, o1);
            });
            const float worth = !p.top2 ? m1 : m2 == -INFINITY ? -INFINITY : bias ? m1 + m2 : score32(m1) + score32(m2);
            const bool exact = !bias && !p.top2;  // (logits: no slack, and of equal ones the lower)
            // A worth is off by what its two values are, half a unit of each and 2^-19.8 together, and by the rounding of their sum, half a unit of it.  The values' magnitudes together are the sum's and, where
            // their signs differ, twice the smaller one (h), which may be far above the sum.  For two runs with |o| <= 2 |worth| that is (8 |worth| + 4 h) 2^-24 + 2^-18.8 at most, the rounding of the
            // bound in it; where |o| is larger, the two are half of it apart.  h is the token's largest: a run that a bias of -10^9 masks has
            // none, and keeps the others' bounds as they are (16384 x 256 with one such run 26.1 us; with the largest sum of magnitudes as everyone's bound 41, all tokens in 64 bits).
            float slack = 0.0f;
            if (!exact) {
                const float both = p.top2 && bias ? fmaxf(fminf(m1, -m2), 0.0f) : 0.0f;
                uint32_t h = __builtin_bit_cast(uint32_t, both);
                if (__ballot(both > 0.0f) != 0) gate_steps(sh, [&](auto S) { h = route_join<decltype(S)::value>(h, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); });
                const float most = __builtin_bit_cast(float, h);
                slack = __builtin_fmaf(fabsf(worth), 0x1p-20f, __builtin_fmaf(most, 0x1p-21f, 0x1p-18f));
                again = (run < p.groups && !(fabsf(worth) < 0x1p100f)) || !(most < 0x1p100f);  // (infinite ones too, whose bounds are no numbers)
            }
            int better = 0, rivals = 0;
            for (int r = 0; r < p.groups; r++) {
                const float o = __shfl(worth, shift + (r << gsh), 64);
                better += exact ? (o > worth) | ((o == worth) & (r < run)) : o > worth + slack;
                rivals += (r != run) & (o >= worth - slack);
            }
            const bool out = better >= p.topk_groups;
            again |= !exact && run < p.groups && !out && rivals >= p.topk_groups;
            if (out) {
#pragma unroll
                for (int v = 0; v < VPT; v++) f[v] = -INFINITY;
            }
        }
        uint32_t s[VPT];
#pragma unroll
        for (int v = 0; v < VPT; v++) s[v] = v < have ? (route_key(f[v]) & ~PLACE) | (PLACE - (uint32_t)v) : 0u;
        route_sort<0, VPT>(s);
        const uint32_t none = route_key(-INFINITY) & ~PLACE;
        uint32_t last = 0, next = 0;  // the values of the last one taken and of the best that is not
        for (int k = 0; k <= p.topk; k++) {
            const uint32_t first = s[0] & ~PLACE;
            uint32_t best = first;
            gate_steps(sh, [&](auto S) { best = route_join<decltype(S)::value>(best, [](uint32_t a, uint32_t b) { return a > b ? a : b; }); });
            last = next, next = best;
            const uint64_t holders = (__ballot(first == best) >> shift) & token_lanes;
            if (gl == __builtin_ctzll(holders | (1ull << 63)) && k < p.topk) {
                mine[k].index = (c0 + (int)(PLACE - (s[0] & PLACE))) | (best == none ? (int)0x80000000 : 0);
#pragma unroll
                for (int v = 0; v + 1 < VPT; v++) s[v] = s[v + 1];
                s[VPT - 1] = 0;
            }
        }
        wave_lds_order();  // (a token's lanes are neighbours in one wavefront)
        for (int k = gl; k < p.topk; k += L) {
            Winner& w = mine[k];
            double c, weight;
            look(w.index & 0x7FFFFFFF, c, weight);
            w.c = w.index < 0 ? NO : c;
            w.weight = w.index < 0 ? 0.0 : weight;
        }
        wave_lds_order();
        for (int k = gl; k < p.topk; k += L) {
            const Winner w = mine[k];
            if (k + 1 < p.topk) {
                const Winner o = mine[k + 1];
                again |= !(w.c > o.c || (w.c == o.c && (w.index & 0x7FFFFFFF) < (o.index & 0x7FFFFFFF)));
            } else if (next != 0) {  // (0: nothing is left)
                const float rest = route_value(next);
                if (!bias) again |= sizeof(T) == 4 && last == next && next != none;  // (a 16-bit logit has nothing in its last bits: equal values are equal logits, in the order of their indices)
                // (the place took up to PLACE units of the number's last bits)
                else again |= next == none ? last == none : !(w.c > (double)route_value(next | PLACE) + (double)route_slack(rest));
            }
        }
    }
    const bool redo = __ballot(again) != 0;
    if (redo) {
        double c[VPT];
#pragma unroll
        for (int v = 0; v < VPT; v++) {
            c[v] = bias ? score(x[v]) * inv + (double)b[v] : (double)x[v];
            if (!(x[v] > -INFINITY) || c[v] != c[v]) c[v] = NO;
            asm volatile("" : "+v"(c[v]));
        }
        if (some) {
            double m1 = NO, m2 = NO;
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
            const double worth = !p.top2 ? m1 : m2 == NO ? NO : bias ? m1 + m2 : (score((float)m1) + score((float)m2)) * inv;
            int better = 0;
            for (int r = 0; r < p.groups; r++) {
                const double o = __shfl(worth, shift + (r << gsh), 64);
                better += (o > worth) | ((o == worth) & (r < run));
            }
            if (better >= p.topk_groups) {
#pragma unroll
                for (int v = 0; v < VPT; v++) c[v] = NO;
            }
        }
#pragma unroll
        for (int v = 0; v < VPT; v++) c[v] = v < have ? c[v] : __builtin_nan("");  // (a maximum passes over NaN: what is not there, and what has been taken)
        for (int k = 0; k < p.topk; k++) {
            const double local = route_max<0, VPT>(c);
            double best = local;
            gate_steps(sh, [&](auto S) { best = __builtin_fmax(best, route_xchg<decltype(S)::value>(best)); });
            const uint64_t holders = (__ballot(local == best) >> shift) & token_lanes;
            if (gl == __builtin_ctzll(holders | (1ull << 63))) {
                int at = 0;
#pragma unroll
                for (int v = VPT - 1; v >= 0; v--) at = c[v] == best ? v : at;  // the first of equal ones
#pragma unroll
                for (int v = 0; v < VPT; v++) c[v] = v == at ? __builtin_nan("") : c[v];
                mine[k].index = (c0 + at) | (best == NO ? (int)0x80000000 : 0);
            }
        }
        wave_lds_order();
        for (int k = gl; k < p.topk; k += L) {
            Winner& w = mine[k];
            double unused, weight;
            look(w.index & 0x7FFFFFFF, unused, weight);
            w.weight = w.index < 0 ? 0.0 : weight;
        }
        wave_lds_order();
    }
    double factor = p.scale;  // (weights in 64 bits until they are stored, one rounding)
    if (p.renorm) {
        double all = 0.0;
        for (int k = 0; k < p.topk; k++) all += mine[k].weight;
        factor /= __builtin_fmax(all, 1e-20);
    }
    if (live) {
        for (int k = gl; k < p.topk; k += L) {
            const Winner w = mine[k];
            p.indices[(size_t)t * p.topk + k] = w.index & 0x7FFFFFFF;
            p.weights[(size_t)t * p.topk + k] = (float)(w.weight * factor);
        }
    }
}

template <typename T>
hipError_t launch_t(const RouteParams& p, int vpt, hipStream_t stream) {
    const int per = 256 / p.lanes;
    const dim3 grid((unsigned)((p.tokens + per - 1) / per)), block(256);
    const size_t lds = (size_t)per * (p.topk + 1) * sizeof(Winner);
    switch (vpt) {
        case 4: hipLaunchKernelGGL((k_route<T, 4>), grid, block, lds, stream, p); break;
        case 8: hipLaunchKernelGGL((k_route<T, 8>), grid, block, lds, stream, p); break;
        case 16: hipLaunchKernelGGL((k_route<T, 16>), grid, block, lds, stream, p); break;
        default: hipLaunchKernelGGL((k_route<T, 32>), grid, block, lds, stream, p); break;
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
    // Four values a lane (the shortest way through one token) while the chip holds all the wavefronts at once, 8192 of them: 1 x 256 in 6.7 us against 8.4 with eight and 11.5 with sixteen,
    // 1024 x 256 7.7 / 10.6 / 14.7, 4096 x 256 11.7 / 12.9 / 16.0.  Beyond, the instructions count, and two tokens a wavefront share them: 16384 x 256 26.7 / 26.1 / 28.6 with groups and
    // 24.2 / 19.1 / 19.1 by softmax.  And more where 64 lanes would not hold a token: with up to 64 runs of a power of two of lanes each, 32 hold 1024 experts in any division.  Sixteen (five
    // wavefronts a SIMD) take 9.4 us for 1 x 1024, 26.6 for 4096 x 1024 and 68.6 for 16384 x 1024, thirty-two (three, and 128 of the scalars kept in vector registers) 15.7 / 36.0 / 81.2 there and 14.8 / 42.3 / 107
    // for 33 groups of 31, which need them.
    auto lanes = [&](int vpt) { return up2(p.groups) * up2((size + vpt - 1) / vpt); };
    int vpt = (int64_t)p.tokens * lanes(4) > 8192 * 64 ? 8 : 4;
    while (lanes(vpt) > 64) vpt <<= 1;
    p.lanes_group = up2((size + vpt - 1) / vpt);
    p.lanes = lanes(vpt);
    const int esz = dtype == 0 ? 4 : 2, chunk = vpt * esz < 16 ? vpt * esz : 16, bias_chunk = vpt * 4 < 16 ? vpt * 4 : 16;
    p.vec = size % vpt == 0 && reinterpret_cast<uintptr_t>(p.gating) % chunk == 0 && ((size_t)p.experts * esz) % chunk == 0 && reinterpret_cast<uintptr_t>(p.bias) % bias_chunk == 0;
    switch (dtype) {
        case 0: return launch_t<float>(p, vpt, stream);
        case 1: return launch_t<uint16_t>(p, vpt, stream);
        case 2: return launch_t<_Float16>(p, vpt, stream);
    }
    return hipErrorInvalidValue;
}
