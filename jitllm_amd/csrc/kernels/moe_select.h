// A mixture's router in its general form (jl_moe_select_dev): softmax or sigmoid scores, a bias that moves the selection and
// not the weights, groups of experts of which the best stay, the k_used best, weights renormalised and scaled.  moe.h's
// moe_route_body is the form without bias and groups.
//
//   score  s = f32(exp(l - max) / sum)  or  f32(1 / (1 + exp(-l)))     f64, narrowed once: neighbouring scores decide the order
//   choice c = s + bias                                                 f32
//   an expert can be taken where l > -inf and c is a number > -inf; with groups, where its group is kept
//   group's value = its best c, or the sum of its two best (a missing second adds nothing); the k_group best groups stay
//   k_used rounds of "largest c, lowest index on a tie"; a place without an expert gets the id n_expert and the weight 0
//   weight = s / (sum of the taken s in their order + 1e-20), or s; times scale
#pragma once
#include "args.h"
#include "common.h"
#include "moe.h"

// Order of f32 values as signed integers; INT_MIN: cannot be taken (+ 0.0f: -0 and 0 are one value).
__device__ __forceinline__ i32 select_key(float c) {
    const i32 b = __builtin_bit_cast(i32, c + 0.0f);
    return c > -__builtin_inff() ? (b >= 0 ? b : b ^ 0x7fffffff) : (i32)0x80000000;
}
__device__ __forceinline__ float select_value(i32 key) { return __builtin_bit_cast(float, key >= 0 ? key : key ^ 0x7fffffff); }

// The largest key of the wavefront.
__device__ __forceinline__ i32 select_wave_max(i32 key) {
    const i32 none = (i32)0x80000000;
#define STEP(C, M) key = max(key, dpp_i32<C, M>(none, key));
    JL_ROUTE_STEPS(STEP)
#undef STEP
    return __builtin_amdgcn_readlane(key, 63);
}

// One wavefront a row, NG experts a lane at most (expert = lane + 64 i).  keys: n_expert words of LDS, read where there are groups.
template <int NG>
__device__ __forceinline__ void moe_select_body(const MoeSelectArgs& p, i32* keys) {
    const int lane = threadIdx.x & 63, n = p.n_expert;
    const i32 none = (i32)0x80000000;
    const float ninf = -__builtin_inff();
    const size_t row = blockIdx.x;
    const float* lg = p.logits + row * (size_t)n;
    float v[NG], sc[NG];
    i32 key[NG];
    float mx = ninf;
#pragma unroll
    for (int i = 0; i < NG; i++) {
        const int e = lane + 64 * i;
        v[i] = e < n ? lg[min(e, n - 1)] : ninf;
        if (v[i] > mx) mx = v[i];
    }
    if (p.sigmoid) {
#pragma unroll
        for (int i = 0; i < NG; i++) {
            sc[i] = 0.f;
            if (64 * i < n) sc[i] = (float)(1.0 / (1.0 + exp(-(double)v[i])));
        }
    } else {
        mx = route_wave_max(mx);
        double sum = 0.0, ex[NG];
#pragma unroll
        for (int i = 0; i < NG; i++) {
            ex[i] = 0.0;
            if (64 * i < n) ex[i] = v[i] == ninf ? 0.0 : exp((double)v[i] - (double)mx);
            sum += ex[i];
        }
        sum = route_wave_sum(sum);
#pragma unroll
        for (int i = 0; i < NG; i++) sc[i] = (float)(ex[i] / sum);
    }
#pragma unroll
    for (int i = 0; i < NG; i++) {
        const int e = lane + 64 * i;
        float c = sc[i];
        if (p.bias && e < n) c += p.bias[e];
        key[i] = e < n && v[i] != ninf ? select_key(c) : none;
    }
    if (p.n_group > 1) {
        const int size = n / p.n_group;
#pragma unroll
        for (int i = 0; i < NG; i++)
            if (lane + 64 * i < n) keys[lane + 64 * i] = key[i];
        __syncthreads();
        i32 a = none, b = none;   // a group's best two, lane = group
        if (lane < p.n_group)
            for (int j = 0; j < size; j++) {
                const i32 t = keys[lane * size + j];
                b = max(b, min(a, t));
                a = max(a, t);
            }
        i32 g = a;
        if (p.group_top > 1 && b != none) g = select_key(select_value(a) + select_value(b));
        uint64_t kept = 0;
        for (int r = 0; r < p.k_group; r++) {
            const i32 best = select_wave_max(g);
            if (best == none) break;   // uniform
            const int at = __builtin_ctzll(__ballot(g == best));
            kept |= 1ull << at;
            if (lane == at) g = none;
        }
#pragma unroll
        for (int i = 0; i < NG; i++) {
            const int e = min(lane + 64 * i, n - 1);
            if (!((kept >> (e / size)) & 1)) key[i] = none;
        }
    }
    float total = 0.f, chosen = 0.f;   // lane r keeps the r-th taken score and its expert
    i32 expert = n;
    for (int r = 0; r < p.k_used; r++) {
        i32 best = key[0];
#pragma unroll
        for (int i = 1; i < NG; i++) best = max(best, key[i]);
        best = select_wave_max(best);
        if (best == none) break;   // uniform
        bool open = true;
#pragma unroll
        for (int i = 0; i < NG; i++) {
            if (!open || 64 * i >= n) continue;   // uniform
            const uint64_t holds = __ballot(key[i] == best);
            if (!holds) continue;
            const int at = __builtin_ctzll(holds);
            const float s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(i32, sc[i]), at));
            if (lane == at) key[i] = none;
            if (lane == r) {
                expert = 64 * i + at;
                chosen = s;
            }
            total += s;
            open = false;
        }
    }
    if (lane < p.k_used) {
        p.sel[row * p.sel_stride + lane] = (u32)expert;
        p.wt[row * p.k_used + lane] = (p.renorm ? chosen / (total + 1e-20f) : chosen) * p.scale;
    }
}
