// Rows normed between two projections: residual added, RMSNorm, and the normed row in f32 / f16 / bf16 or in the activation
// quantizer's int8 form (jl_norm_rows_dev).  The reference's RMSNormQuantRows (jit/gpu/kernels/elem.go:252-267) in the f64
// of its host form (internal/oracle/oracle.go:230-240), with the block's residual add in front:
//
//   h = resid + alpha * x                       f32, product and sum each rounded (as a matvec's riding residual add)
//   inv = 1 / sqrt(mean(h^2) + eps)             f64: squares of f32 values are exact in it, and a row's sum keeps 29 bits more
//   y = f32(f64(h) * f64(w) * inv)              than the f32 it is narrowed to, so y does not depend on the order of the sum
//   q, as, sum16 = the quantizer of y           (quantize.h: bit for bit jl_quantize_act_dev over y)
//
// A row is read once, kept in registers across the sum, and written once: the kernel is bound by its bytes.  With the residual and int8 4096 rows of 7168 take
// 82 us (393 MB, 4.8 TB/s), of 14336 161 (785 MB, 4.9), 512 of 4096 7.8 (28 MB; one round of workgroups, its ramp and tail); one row of 4096 2.7 in f32, near the launch.
#pragma once
#include "args.h"
#include "common.h"
#include "quantize.h"

#pragma clang fp contract(off)

// Four elements of a row, element 4g on, as f32.  VEC: the row is 16-byte (8-byte) aligned and a multiple of four long.
template <bool VEC>
__device__ __forceinline__ f32x4 norm_load(const void* p, size_t at, int type, int left) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (type == JL_F32) {
        const float* f = (const float*)p + at;
        if (VEC) return *(const f32x4*)f;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) v[i] = f[i];
        return v;
    }
    const uint16_t* h = (const uint16_t*)p + at;
    uint16_t b[4] = {0, 0, 0, 0};
    if (VEC) {
        const u32x2 w = *(const u32x2*)h;
        b[0] = (uint16_t)w.x; b[1] = (uint16_t)(w.x >> 16); b[2] = (uint16_t)w.y; b[3] = (uint16_t)(w.y >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) b[i] = h[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = type == JL_F16 ? half_bits_to_f32(b[i]) : __uint_as_float((u32)b[i] << 16);
    return v;
}

template <bool VEC>
__device__ __forceinline__ void norm_store(void* p, size_t at, int type, int left, f32x4 v) {
    if (type == JL_F32) {
        float* f = (float*)p + at;
        if (VEC) {
            *(f32x4*)f = v;
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < left) f[i] = v[i];
        return;
    }
    uint16_t b[4];
#pragma unroll
    for (int i = 0; i < 4; i++)   // round to nearest even, by the hardware's conversions
        b[i] = type == JL_F16 ? __builtin_bit_cast(uint16_t, (_Float16)v[i]) : __builtin_bit_cast(uint16_t, (__bf16)v[i]);
    uint16_t* h = (uint16_t*)p + at;
    if (VEC) {
        *(u32x2*)h = u32x2{(u32)b[0] | (u32)b[1] << 16, (u32)b[2] | (u32)b[3] << 16};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < left) h[i] = b[i];
}

template <int CTRL> __device__ __forceinline__ double dpp_add_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const u32 lo = (u32)dpp_i32<CTRL, 0xf>(0, (i32)(u32)b), hi = (u32)dpp_i32<CTRL, 0xf>(0, (i32)(u32)(b >> 32));
    return v + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// Sum over the LPR consecutive lanes of a row; every lane has it.
template <int LPR> __device__ __forceinline__ double norm_lane_sum(double v) {
    v = dpp_add_f64<JL_DPP_QUAD_XOR1>(v);
    v = dpp_add_f64<JL_DPP_QUAD_XOR2>(v);
    v = dpp_add_f64<JL_DPP_ROW_HALF_MIRROR>(v);
    v = dpp_add_f64<JL_DPP_ROW_MIRROR>(v);
    if (LPR >= 32) v += __shfl_xor(v, 16, JL_WAVE);
    if (LPR >= 64) v += __shfl_xor(v, 32, JL_WAVE);
    return v;
}

// LPR lanes of a wavefront a row (WG false), or a whole workgroup a row (WG, LPR = 64), NI groups of four elements a thread.
template <int LPR, int NI, bool WG, bool VEC>
__device__ __forceinline__ void norm_rows_body(const NormRowsArgs& p, double* part) {
    const int tid = threadIdx.x;
    const int lane = WG ? tid : tid % LPR;                       // of the row's threads
    const int nthr = WG ? p.threads : LPR;
    const size_t row = WG ? blockIdx.x : (size_t)blockIdx.x * (256 / LPR) + tid / LPR;
    const bool here = WG || row < (size_t)p.rows;
    const int n = p.n;
    // w after the sum: beside h it does not fit the registers of 1024 threads (with it one row of 14336 took 20 us in this form, now one of 65536 does)
    constexpr bool LATE = NI > 8;
    f32x4 h[NI], w[LATE ? 1 : NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = 4 * (lane + nthr * i);
        const bool live = here && e < n;
        h[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (!LATE) w[LATE ? 0 : i] = h[i];
        if (live) {
            h[i] = norm_load<VEC>(p.x, row * p.x_stride + e, p.x_type, n - e);
            if (!LATE) w[LATE ? 0 : i] = p.w ? norm_load<VEC>(p.w, e, JL_F32, n - e) : f32x4{1.f, 1.f, 1.f, 1.f};
            if (p.resid) {
                const f32x4 r = norm_load<VEC>(p.resid, row * p.resid_stride + e, JL_F32, n - e);
                h[i] = r + p.alpha * h[i];
            }
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) sum = __builtin_fma((double)h[i][j], (double)h[i][j], sum);
    sum = norm_lane_sum<LPR>(sum);
    if (WG) {
        const int nw = p.threads / 64;
        if (nw > 1) {
            if ((tid & 63) == 0) part[tid >> 6] = sum;
            __syncthreads();
            sum = 0.0;
            for (int i = 0; i < nw; i++) sum += part[i];
        }
    }
    const double inv = 1.0 / sqrt(sum / (double)n + (double)p.eps);
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int e = 4 * (lane + nthr * i);
        const bool live = here && e < n;
        f32x4 y, g = w[LATE ? 0 : i];
        if (LATE) g = live && p.w ? norm_load<VEC>(p.w, e, JL_F32, n - e) : f32x4{1.f, 1.f, 1.f, 1.f};
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = (float)((double)h[i][j] * (double)g[j] * inv);
        if (live && p.resid_out) norm_store<VEC>(p.resid_out, row * p.resid_stride + e, JL_F32, n - e, h[i]);
        if (live && p.y) norm_store<VEC>(p.y, row * p.y_stride + e, p.y_type, n - e, y);
        if (p.q) {
            u32 m = max(max(abs_bits(y.x), abs_bits(y.y)), max(abs_bits(y.z), abs_bits(y.w)));
            m = window_amax(live ? m : 0u, min(p.per, LPR / 8));
            float d;
            i32 s;
            const u32 q = quantize4(y, m, d, s);
            if (live) {
                ((u32*)(p.q + row * (size_t)n))[e / 4] = q;
                if ((e & 15) == 0) p.s16[row * (size_t)(n / 16) + e / 16] = (float)s;
                if ((e & 31) == 0) p.as[row * (size_t)(n / 32) + e / 32] = d;
            }
        }
    }
}
