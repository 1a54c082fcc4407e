// Low-rank adapters of many requests beside the projections they share (jl_adapter_group_dev): token t of adapter a = ids[t] gets
//   out_i[t] = base_i[t] + scale[a] * B_i[a] (A_i[a] x[t]),     A_i [n_adapter][rank][k], B_i [n_adapter][rows_i][rank]
// for up to four projections that read one x.  Products and sums in f32 whatever the types; a token whose id no adapter has, or
// whose adapter has rank 0, gets base alone.
//
// Two kernels: adapter_down writes u = scale * A x to a workspace of [ntok][n][rank] floats, adapter_up adds B u to base.
#pragma once
#include "args.h"
#include "common.h"

typedef __bf16 ad_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 ad_f16x8 __attribute__((ext_vector_type(8)));
struct AdF8 { float v[8]; };

// Eight consecutive elements from 16-byte aligned p + at, as f32.
template <int T> __device__ __forceinline__ AdF8 adapter_load8(const void* p, size_t at) {
    AdF8 r;
    if (T == JL_F32) {
        const f32x4 a = *(const f32x4*)((const float*)p + at), b = *(const f32x4*)((const float*)p + at + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) { r.v[i] = a[i]; r.v[4 + i] = b[i]; }
    } else {
        const u32x4 w = *(const u32x4*)((const uint16_t*)p + at);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
            r.v[i] = T == JL_F16 ? half_bits_to_f32(h) : __uint_as_float((u32)h << 16);
        }
    }
    return r;
}
template <int T> __device__ __forceinline__ float adapter_load1(const void* p, size_t at) {
    if (T == JL_F32) return ((const float*)p)[at];
    const uint16_t h = ((const uint16_t*)p)[at];
    return T == JL_F16 ? half_bits_to_f32(h) : __uint_as_float((u32)h << 16);
}

// The adapter of a token and its rank; -1: none.
__device__ __forceinline__ int adapter_of(const AdapterArgs& p, int tok, int& rank) {
    const u32 id = p.ids[tok];
    rank = 0;
    if (id >= (u32)p.n_adapter) return -1;
    rank = p.ranks ? (int)min(p.ranks[id], (u32)p.rank) : p.rank;
    return rank > 0 ? (int)id : -1;
}

// grid = (tokens, ceil(rank / 4), projections), block = 256: a wavefront a row of A.
template <int T, int XT>
__device__ __forceinline__ void adapter_down_body(const AdapterArgs& p) {
    const int tok = blockIdx.x, i = blockIdx.z, lane = threadIdx.x & 63;
    const int r = blockIdx.y * 4 + (threadIdx.x >> 6);
    int rank;
    const int a = adapter_of(p, tok, rank);
    if (a < 0 || r >= rank) return;
    const size_t arow = ((size_t)a * p.rank + r) * p.k, xrow = (size_t)tok * p.k;
    float s = 0.f;
    for (int e = 8 * lane; e < p.k; e += 512) {
        const AdF8 w = adapter_load8<T>(p.a[i], arow + e), x = adapter_load8<XT>(p.x, xrow + e);
#pragma unroll
        for (int j = 0; j < 8; j++) s = __builtin_fmaf(w.v[j], x.v[j], s);
    }
    s = wave_sum_to_lane63(s);
    if (lane == 63) p.u[((size_t)tok * p.n + i) * p.rank + r] = (p.scale ? p.scale[a] : 1.f) * s;
}

// grid = (tokens, ceil(rows / 256), projections), block = 256: a thread a row of B, LDS = rank floats.
template <int T>
__device__ __forceinline__ void adapter_up_body(const AdapterArgs& p, float* u) {
    const int tok = blockIdx.x, i = blockIdx.z, rows = p.rows[i];
    const int row = blockIdx.y * 256 + threadIdx.x;
    if (blockIdx.y * 256 >= (u32)rows) return;
    int rank;
    const int a = adapter_of(p, tok, rank);
    for (int r = threadIdx.x; r < rank; r += 256) u[r] = p.u[((size_t)tok * p.n + i) * p.rank + r];
    __syncthreads();
    if (row >= rows) return;
    const size_t at = (size_t)tok * rows + row;
    float s = 0.f;
    if (a >= 0) {
        const size_t brow = ((size_t)a * rows + row) * p.rank;
        int r = 0;
        if (p.rank % 8 == 0)
            for (; r + 8 <= rank; r += 8) {
                const AdF8 w = adapter_load8<T>(p.b[i], brow + r);
#pragma unroll
                for (int j = 0; j < 8; j++) s = __builtin_fmaf(w.v[j], u[r + j], s);
            }
        for (; r < rank; r++) s = __builtin_fmaf(adapter_load1<T>(p.b[i], brow + r), u[r], s);
    }
    p.out[i][at] = p.base[i] ? (a >= 0 ? p.base[i][at] + s : p.base[i][at]) : s;
}
