// A mixture's router in its general form (jl_moe_select_dev): softmax or sigmoid scores, a bias that moves the selection and
// not the weights, groups of experts of which the best stay, the k_used best, weights renormalised and scaled.  moe.h's
// moe_route_body is the form without bias and groups.
//
//   score  s = f32(exp(l - max) / sum)  or  f32(1 / (1 + exp(-l)))     f64, narrowed once: neighbouring scores decide the order
//   choice c = s + bias                                                 f32
//   an expert can be taken where l is a number > -inf and c is a number > -inf; with groups, where its group is kept
//   group's value = its best c, or the sum of its two best (a missing second adds nothing); the k_group best groups stay
//   k_used rounds of "largest c, lowest index on a tie"; a place without an expert gets the id n_expert and the weight 0
//   weight = s / (sum of the taken s in their order + 1e-20), or s; times scale
//
// One wavefront a row, NG experts a lane side by side.  With many rows the kernel is bound by its vector instructions, not by
// its bytes (16384 rows of 384 experts: 18.6 us, 22.4 in the first form, a chain of wave maxima over 32-bit keys and the library's f64
// exponential and division; 25 MB would take 5.5), with one row by their latency.  So:
//   * the f64 exponential is eighteen instructions (an f64 multiply-add costs what an f32 one does here) and the quotient a
//     reciprocal refined in three multiply-adds: either is off by under 2^-50, where the narrowing to f32 keeps 2^-24;
//   * the selection goes by packed keys, the 22 high bits of c's order over the expert's index, which a lane sorts once and then only
//     shifts: a round is a wave maximum of the lanes' heads.  Packed keys that differ in their high bits are in c's order; where two
//     of them do not -- one row in ten of sigmoid scores, one in three hundred of softmax ones -- what was taken is put in order by its
//     whole keys, and where more than 64 experts are that near to one another (scores that are all one value) the row takes whole keys
//     from the start.
#pragma once
#include "args.h"
#include "common.h"
#include "moe.h"

// e^x for |x| <= 800 (0 and infinity past f64's range), to 2^-51 or so: x = n ln2 + r with |r| <= ln2 / 2, the exponential's series in r
// up to r^12 / 12! (the next term is under 2^-52), times 2^n.
__device__ __forceinline__ double select_exp(double x) {
    const double n = __builtin_rint(x * 1.4426950408889634074);
    double r = __builtin_fma(-n, 0x1.62e42fefa39efp-1, x);   // ln2 in two parts
    r = __builtin_fma(-n, 0x1.abc9e3b39803fp-56, r);
    double p = 1.0 / 479001600.0;
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// 1 / d for a positive normal d below 2^1020: the hardware's estimate y (22 bits or more) times 1 + e + e^2, e = 1 - d y.
__device__ __forceinline__ double select_rcp(double d) {
    const double y = __builtin_amdgcn_rcp(d), e = __builtin_fma(-d, y, 1.0);
    return __builtin_fma(y, __builtin_fma(e, e, e), y);
}
// Order of f32 values other than -0 (a choice is none: scores are not negative) as unsigned integers; no finite value and no +inf is 0, which
// marks "cannot be taken".
__device__ __forceinline__ u32 select_key(float c) {
    const u32 b = __float_as_uint(c);
    return c > -__builtin_inff() ? b ^ ((u32)((i32)b >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float select_value(u32 k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ u32 select_wave_max(u32 key) {
#define STEP(C, M) key = max(key, (u32)dpp_i32<C, M>(0, (i32)key));
    JL_ROUTE_STEPS(STEP)
#undef STEP
    return (u32)__builtin_amdgcn_readlane((i32)key, 63);
}
// The best two of `lanes` consecutive lanes' pairs (a >= b), a power of two; every lane has them.
__device__ __forceinline__ void select_best_two(u32& a, u32& b, int lanes) {
    auto meet = [&](u32 oa, u32 ob) {
        b = max(min(a, oa), max(b, ob));
        a = max(a, oa);
    };
#define MEET(CTRL) meet((u32)dpp_i32<CTRL, 0xf>(0, (i32)a), (u32)dpp_i32<CTRL, 0xf>(0, (i32)b))
    if (lanes >= 2) MEET(JL_DPP_QUAD_XOR1);
    if (lanes >= 4) MEET(JL_DPP_QUAD_XOR2);
    if (lanes >= 8) MEET(JL_DPP_ROW_HALF_MIRROR);
    if (lanes >= 16) MEET(JL_DPP_ROW_MIRROR);
#undef MEET
    if (lanes >= 32) meet(__shfl_xor(a, 16, 64), __shfl_xor(b, 16, 64));
}

// keys, scores: 64 NG words of LDS each, the wavefront's own.  PACKED: by packed keys; else a round looks for the largest whole key and
// its first place.
template <int NG, bool PACKED>
__device__ __forceinline__ void moe_select_body(const MoeSelectArgs& p, size_t row, u32* keys, float* scores) {
    constexpr int VW = NG % 4 == 0 ? 4 : NG % 2 == 0 ? 2 : 1;   // elements a load, where rows keep their alignment
    const int lane = threadIdx.x & 63, n = p.n_expert, e0 = lane * NG, k = p.k_used;
    const float inf = __builtin_inff();
    float v[NG], s[NG];
    auto load = [&](const float* at, float (&to)[NG], float none) {
        if (VW > 1 && p.wide) {   // uniform
            typedef float vec __attribute__((ext_vector_type(VW)));
#pragma unroll
            for (int i = 0; i < NG; i += VW) {
                vec q;
#pragma unroll
                for (int j = 0; j < VW; j++) q[j] = none;
                if (e0 + i < n) q = *(const vec*)(at + e0 + i);
#pragma unroll
                for (int j = 0; j < VW; j++) to[i + j] = q[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < NG; i++) to[i] = e0 + i < n ? at[e0 + i] : none;
        }
    };
    load(p.logits + row * (size_t)n, v, -inf);
    float bias[NG];
    if (p.bias) load(p.bias, bias, 0.f);
    bool fine = true;   // the row has scores
    if (p.sigmoid) {
#pragma unroll
        for (int i = 0; i < NG; i++) s[i] = (float)select_rcp(1.0 + select_exp((double)fminf(fmaxf(-v[i], -700.f), 700.f)));   // (f32 has no e^-700)
    } else {
        float mx = -inf;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < NG; i++) {
            mx = fmaxf(mx, v[i]);
            odd = odd || !(v[i] < inf);
        }
        mx = route_wave_max(mx);
        fine = mx > -inf && !__ballot(odd);
        double sum = 0.0, ex[NG];
#pragma unroll
        for (int i = 0; i < NG; i++) {
            ex[i] = select_exp(fmax((double)v[i] - (double)mx, -800.0));   // (e^-800 is 0 here; in f32 mx - 800 is mx from 2^34 on)
            sum += ex[i];
        }
        const double inv = select_rcp(fine ? route_wave_sum(sum) : 1.0);
#pragma unroll
        for (int i = 0; i < NG; i++) s[i] = (float)(ex[i] * inv);
    }
    u32 key[NG];
#pragma unroll
    for (int i = 0; i < NG; i++) key[i] = fine && v[i] > -inf ? select_key(p.bias ? s[i] + bias[i] : s[i]) : 0u;

    if (p.n_group > 1) {
        const int size = n / p.n_group, lpg = size / NG;   // lanes a group, where groups are whole lanes
        const bool whole = lpg * NG == size && lpg > 0 && (lpg & (lpg - 1)) == 0 && lpg <= 32;
        u32 a = 0, b = 0;
        uint64_t kept = 0;   // of groups
        if (whole) {
#pragma unroll
            for (int i = 0; i < NG; i++) {
                b = max(b, min(a, key[i]));
                a = max(a, key[i]);
            }
            select_best_two(a, b, lpg);
        } else {   // lane = group, through LDS
#pragma unroll
            for (int i = 0; i < NG; i++) keys[e0 + i] = key[i];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (a wavefront's own LDS)
            if (lane < p.n_group)
                for (int j = 0; j < size; j++) {
                    const u32 t = keys[lane * size + j];
                    b = max(b, min(a, t));
                    a = max(a, t);
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        u32 g = a;
        if (p.group_top > 1 && b) g = max(select_key(select_value(a) + select_value(b) + 0.0f), 1u);   // (a sum of -inf is the last, not no group)
        const int per = whole ? lpg : 1;
        for (int r = 0; r < p.k_group; r++) {
            const u32 best = select_wave_max(g);
            if (best == 0) break;   // uniform
            const int at = __builtin_ctzll(__ballot(g == best)) / per;   // the lowest group
            kept |= 1ull << at;
            if (lane / per == at) g = 0;
        }
        if (whole) {
            const bool stays = (kept >> (lane / per)) & 1;   // (lanes behind the last expert have no keys)
#pragma unroll
            for (int i = 0; i < NG; i++) key[i] = stays ? key[i] : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < NG; i++) key[i] = (kept >> ((u32)min(e0 + i, n - 1) * (u32)p.inv_size >> 20)) & 1 ? key[i] : 0u;
        }
    }
    int expert = 0, c = 0;   // lane r keeps the r-th taken expert and its score; c of them
    float mys = 0.f, total = 0.f;   // (added in selection order)
    auto rounds = [&]() {
        int r = 0;
        for (; r < k; r++) {
            u32 m = key[0];
#pragma unroll
            for (int i = 1; i < NG; i++) m = max(m, key[i]);
            const u32 best = select_wave_max(m);
            if (best == 0) break;   // uniform
            const int from = __builtin_ctzll(__ballot(m == best));
            // (choices between places of an array as bits, or the compiler makes an index, and memory, of them)
            int at = NG - 1;
            u32 sc = __float_as_uint(s[NG - 1]);
#pragma unroll
            for (int i = NG - 2; i >= 0; i--) {
                const u32 hit = key[i] == best ? ~0u : 0u;
                at = hit ? i : at;
                sc = (__float_as_uint(s[i]) & hit) | (sc & ~hit);
            }
            const u32 mine = lane == from ? ~0u : 0u;
#pragma unroll
            for (int i = 0; i < NG; i++) key[i] &= ~(at == i ? mine : 0u);
            const int e = from * NG + __builtin_amdgcn_readlane(at, from);
            const float taken = __uint_as_float((u32)__builtin_amdgcn_readlane((i32)sc, from));
            if (lane == r) {
                expert = e;
                mys = taken;
            }
            total += taken;
        }
        return r;
    };
    if constexpr (PACKED) {
#pragma unroll
        for (int i = 0; i < NG; i++) {
            keys[e0 + i] = key[i];
            scores[e0 + i] = s[i];
        }
        u32 pk[NG];
#pragma unroll
        for (int i = 0; i < NG; i++) pk[i] = key[i] ? (key[i] & ~1023u) | (u32)(1023 - e0 - i) : 0u;
#pragma unroll
        for (int a = 0; a + 1 < NG; a++)   // descending
#pragma unroll
            for (int b = NG - 1; b > a; b--) {
                const u32 x = max(pk[b - 1], pk[b]), y = min(pk[b - 1], pk[b]);
                pk[b - 1] = x;
                pk[b] = y;
            }
        u32 mine = 0, last = 0;   // lane r keeps the r-th taken
        bool near = false;        // two of them have the same high bits
        for (; c < 64; c++) {
            const u32 best = select_wave_max(pk[0]);
            if (best == 0 || (c >= k && best >> 10 != last >> 10)) break;   // uniform
            near = near || (c && best >> 10 == last >> 10);
            last = best;
            mine = lane == c ? best : mine;
            const u32 own = pk[0] == best ? ~0u : 0u;   // (bits, as in rounds())
#pragma unroll
            for (int i = 0; i + 1 < NG; i++) pk[i] = (pk[i + 1] & own) | (pk[i] & ~own);
            pk[NG - 1] &= ~own;
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        expert = 1023 - (int)(mine & 1023);   // lanes below c
        if (near && c < 64) {
            const u32 whole = lane < c ? keys[expert] : 0u;
            int rank = 0;
            for (int j = 0; j < c; j++) {
                const u32 kj = (u32)__builtin_amdgcn_readlane((i32)whole, j);
                const int ej = __builtin_amdgcn_readlane(expert, j);
                rank += kj > whole || (kj == whole && ej < expert);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (lane < c) keys[rank] = (u32)expert;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (lane < c) expert = (int)keys[lane];
        } else if (c == 64) {
            c = rounds();
        }
        if (total == 0.f) {   // (not by rounds(), or by it with scores that add up to nothing)
            c = min(c, k);
            mys = lane < c ? scores[expert] : 0.f;
            for (int r = 0; r < c; r++) total += __uint_as_float((u32)__builtin_amdgcn_readlane((i32)__float_as_uint(mys), r));
        }
    } else {
        c = rounds();
    }
    if (lane < k) {
        p.sel[row * p.sel_stride + lane] = (u32)(lane < c ? expert : n);
        p.wt[row * k + lane] = (p.renorm ? mys / (total + 1e-20f) : mys) * p.scale;
    }
}
