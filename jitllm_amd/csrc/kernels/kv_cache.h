// Rows of keys and values into the pages of a cache and back (jl_kv_write_dev, jl_kv_read_dev).
//
//   16-bit rows: the value rounded to nearest even.  8-bit rows, one f32 scale a position and head: the activation quantizer's
//   arithmetic (quantize.h) with the row as its window, d = amax / 127, q = round-half-away(f32(x * f32(1 / d))); read back as f32(q * d).
//
// A row takes `lanes` lanes of a wavefront, eight elements each: one or two 16-byte loads, one 16- or 8-byte store, and the amax
// by lane moves.  Bytes bind, in whole lines of rows that lie where the pages do: 8191 tokens of 8 heads of 128, f32 to 8 bits, 19.8 us (4.2 TB/s), back to bf16 12.0 (4.2);
// 50001 tokens in any order of 4 heads of 96, bf16 to f32, 59 (3.9; rows of 192 bytes meet two lines of 128; a large copy has 5.0).  Two rows a thread side by side
// change nothing (19.9, 12.0, 59.1), four elements a lane with stores of whole lines take 93.5 for 59.  A token whose sequence, position or page is none of the cache's is written nowhere and read back as zeros.
#pragma once
#include "args.h"
#include "common.h"
#include "norm_rows.h"
#include "quantize.h"

#pragma clang fp contract(off)

#define JL_I8 24

// Element index of a row's first element, or ~0: no such place.
__device__ __forceinline__ bool kv_place(const KvArgs& c, u32 seq, u32 pos, u32& page, u32& slot) {
    slot = pos & ((1u << c.shift) - 1);
    const u32 at = pos >> c.shift;
    if (seq >= c.n_seq || at >= c.table_pages) return false;
    page = c.table[(size_t)seq * c.table_stride + at];
    return page < c.n_page;
}

__device__ __forceinline__ void kv_load8(const void* p, size_t at, int type, bool vec, f32x4& a, f32x4& b) {
    if (vec && type != JL_F32) {
        const u32x4 w = *(const u32x4*)((const uint16_t*)p + at);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint16_t lo = (uint16_t)w[i], hi = (uint16_t)(w[i] >> 16), lo2 = (uint16_t)w[i + 2], hi2 = (uint16_t)(w[i + 2] >> 16);
            a[2 * i] = type == JL_F16 ? half_bits_to_f32(lo) : __uint_as_float((u32)lo << 16);
            a[2 * i + 1] = type == JL_F16 ? half_bits_to_f32(hi) : __uint_as_float((u32)hi << 16);
            b[2 * i] = type == JL_F16 ? half_bits_to_f32(lo2) : __uint_as_float((u32)lo2 << 16);
            b[2 * i + 1] = type == JL_F16 ? half_bits_to_f32(hi2) : __uint_as_float((u32)hi2 << 16);
        }
    } else if (vec) {
        a = norm_load<true>(p, at, type, 4);
        b = norm_load<true>(p, at + 4, type, 4);
    } else {
        a = norm_load<false>(p, at, type, 4);
        b = norm_load<false>(p, at + 4, type, 4);
    }
}
__device__ __forceinline__ u32x4 kv_bits8(int type, f32x4 a, f32x4 b) {   // eight 16-bit values, to nearest even
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = i < 2 ? a[2 * i] : b[2 * i - 4], y = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
        const uint16_t lo = type == JL_F16 ? __builtin_bit_cast(uint16_t, (_Float16)x) : __builtin_bit_cast(uint16_t, (__bf16)x);
        const uint16_t hi = type == JL_F16 ? __builtin_bit_cast(uint16_t, (_Float16)y) : __builtin_bit_cast(uint16_t, (__bf16)y);
        w[i] = (u32)lo | (u32)hi << 16;
    }
    return w;
}
__device__ __forceinline__ void kv_store8(void* p, size_t at, int type, bool vec, f32x4 a, f32x4 b) {
    if (vec && type != JL_F32) {
        *(u32x4*)((uint16_t*)p + at) = kv_bits8(type, a, b);
    } else if (vec) {
        norm_store<true>(p, at, type, 4, a);
        norm_store<true>(p, at + 4, type, 4, b);
    } else {
        norm_store<false>(p, at, type, 4, a);
        norm_store<false>(p, at + 4, type, 4, b);
    }
}

// Four values by the window's step (quantize4 without the half-block's sum).
__device__ __forceinline__ u32 kv_quantize4(f32x4 v, float inv) {
    const i32 a = round_half_away(v.x * inv), b = round_half_away(v.y * inv), c = round_half_away(v.z * inv), e = round_half_away(v.w * inv);
    return (u32)(a & 0xFF) | ((u32)(b & 0xFF) << 8) | ((u32)(c & 0xFF) << 16) | ((u32)e << 24);
}

// grid = (rows / (256 / lanes), 2): y 0 the keys, 1 the values.
template <bool WRITE> __device__ __forceinline__ void kv_rows_body(const KvRowsArgs& p) {
    const KvArgs& c = p.c;
    const bool keys = blockIdx.y == 0;
    void* const x = keys ? p.k : p.v;
    if (!x) return;
    const size_t stride = keys ? p.k_stride : p.v_stride;
    const int lane = threadIdx.x & (p.lanes - 1), e = 8 * lane;
    const size_t row = (size_t)blockIdx.x * (256 / p.lanes) + threadIdx.x / p.lanes;   // (a launch has fewer threads than 2^32)
    const u32 t = (u32)row / (u32)c.n_kv, head = (u32)row - t * (u32)c.n_kv;
    const bool here = t < (u32)p.ntok, live = here && e < c.d;
    const size_t at = t * stride + (size_t)head * c.d + e;
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    if (WRITE && live) kv_load8(x, at, p.type, p.vec, a, b);
    u32 page = 0, slot = 0;
    const bool ok = here && kv_place(c, p.seq ? p.seq[t] : t, p.pos[t], page, slot);
    const size_t to = page * c.page_stride + head * c.head_stride + slot * c.row_stride + e;
    const size_t scale_at = ((size_t)page * c.n_kv + head) << c.shift | slot;
    void* const pool = keys ? c.k : c.v;
    float* const scales = keys ? c.k_scale : c.v_scale;
    if (WRITE) {
        if (c.type == JL_I8) {
            u32 m = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) m = max(m, max(abs_bits(a[i]), abs_bits(b[i])));
            m = window_amax(m, p.lanes / 8);
            const float d = __uint_as_float(m) / 127.0f;
            float inv = 1.0f / d;
            if (!(inv < __builtin_inff())) inv = 0.0f;   // (a row of zeros, or of nothing above 2^-121: zeros)
            if (live && ok) {
                *(u32x2*)((int8_t*)pool + to) = u32x2{kv_quantize4(a, inv), kv_quantize4(b, inv)};
                if (lane == 0) scales[scale_at] = d;
            }
        } else if (live && ok) {
            *(u32x4*)((uint16_t*)pool + to) = kv_bits8(c.type, a, b);
        }
    } else if (live) {
        if (ok && c.type == JL_I8) {
            const u32x2 w = *(const u32x2*)((const int8_t*)pool + to);
            const float d = scales[scale_at];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                a[i] = (float)(i32)(int8_t)(w.x >> 8 * i) * d;
                b[i] = (float)(i32)(int8_t)(w.y >> 8 * i) * d;
            }
        } else if (ok) {
            kv_load8(pool, to, c.type, true, a, b);
        }
        kv_store8(x, at, p.type, p.vec, a, b);
    }
}
