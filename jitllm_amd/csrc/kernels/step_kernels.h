// The kernels of a decode step that stand between a block's projections and behind the last one.
#pragma once
#include "attend_many.h"
#include "attend_one.h"
#include "kv_cache.h"
#include "sample.h"

// grid = (rows / (256 / lanes), 2), block = 256
extern "C" __global__ __launch_bounds__(256) void jl_kv_write(KvRowsArgs p) { kv_rows_body<true>(p); }
extern "C" __global__ __launch_bounds__(256) void jl_kv_read(KvRowsArgs p) { kv_rows_body<false>(p); }

// _q<pieces of q>; over a bf16 cache one piece of q goes with two of the weights (a 16-bit result), three with three
// grid = p.wgs, or p.units * planes where p.whole; block = 256; _m: units of several tokens
#define JL_ATTEND_ONE_M(T, TYPE, DP, QP, PP, NAME, MANY)                                                                            \
    extern "C" __global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void jl_attend_one_##T##_d##DP##_q##QP##NAME(AttendArgs p) {    \
        __shared__ __attribute__((aligned(16))) float lds[4 * 16 * (DP + 4) + 128];                                                 \
        __shared__ uint64_t find[6];                                                                                                \
        attend_one_body<TYPE, DP, QP, PP, MANY>(p, lds, find);                                                                      \
    }
#define JL_ATTEND_ONE(T, TYPE, DP, QP, PP) JL_ATTEND_ONE_M(T, TYPE, DP, QP, PP, , false) JL_ATTEND_ONE_M(T, TYPE, DP, QP, PP, _m, true)
// grid = p.wgs, or p.units * planes where p.whole; block = 64 WAVES
#define JL_ATTEND_MANY(T, TYPE, DP, QP, PP, WAVES, OCC)                                                                             \
    extern "C" __global__ __launch_bounds__(64 * WAVES, OCC) void jl_attend_many_##T##_d##DP##_q##QP##_w##WAVES(AttendArgs p) {     \
        __shared__ u32x4 lds[2 * at_stage_words<DP>() / 4 + 2 * 32 + 3];                                                            \
        __shared__ uint64_t find[WAVES + 2];                                                                                        \
        attend_many_body<TYPE, DP, QP, PP, WAVES>(p, lds, find);                                                                    \
    }
#define JL_ATTEND_Q(T, TYPE, QP, PP)                                                                                                \
    JL_ATTEND_ONE(T, TYPE, 64, QP, PP) JL_ATTEND_ONE(T, TYPE, 128, QP, PP) JL_ATTEND_ONE(T, TYPE, 256, QP, PP)                      \
    JL_ATTEND_MANY(T, TYPE, 64, QP, PP, 4, 4) JL_ATTEND_MANY(T, TYPE, 128, QP, PP, 4, 2) JL_ATTEND_MANY(T, TYPE, 256, QP, PP, 4, 1) \
    JL_ATTEND_MANY(T, TYPE, 64, QP, PP, 8, 4) JL_ATTEND_MANY(T, TYPE, 128, QP, PP, 8, QP == 1 ? 4 : 2) JL_ATTEND_MANY(T, TYPE, 256, QP, PP, 8, 2)
JL_ATTEND_Q(f16, JL_F16, 1, 2) JL_ATTEND_Q(f16, JL_F16, 2, 2) JL_ATTEND_Q(i8, JL_I8, 1, 2) JL_ATTEND_Q(i8, JL_I8, 2, 2)
JL_ATTEND_Q(bf16, JL_BF16, 1, 2) JL_ATTEND_Q(bf16, JL_BF16, 3, 3)
// grid = (p.wgs, columns), block = 256; _wide: sixteen columns a workgroup
#define JL_ATTEND_JOIN(DP)                                                                                                          \
    extern "C" __global__ __launch_bounds__(256) void jl_attend_join_d##DP(AttendArgs p) {                                          \
        __shared__ __attribute__((aligned(16))) float lds[4 * DP + 4];                                                              \
        attend_join_body<DP>(p, lds);                                                                                               \
    }
#define JL_ATTEND_JOIN_WIDE(DP)                                                                                                     \
    extern "C" __global__ __launch_bounds__(256) void jl_attend_join_wide_d##DP(AttendArgs p) { attend_join_wide_body<DP>(p); }
JL_ATTEND_JOIN_WIDE(64) JL_ATTEND_JOIN_WIDE(128) JL_ATTEND_JOIN_WIDE(256)
JL_ATTEND_JOIN(64) JL_ATTEND_JOIN(128) JL_ATTEND_JOIN(256)

// grid = (slices, rows), block = 512
extern "C" __global__ __launch_bounds__(512) void jl_sample_max(SampleArgs p) {
    __shared__ u32 lds[3];
    sample_max_body(p, lds);
}
extern "C" __global__ __launch_bounds__(512) void jl_sample_bins(SampleArgs p) {
    __shared__ uint64_t sums[JL_SA_BINS];
    __shared__ u32 counts[JL_SA_BINS];
    sample_bins_body(p, counts, sums);
}
extern "C" __global__ __launch_bounds__(512) void jl_sample_gather(SampleArgs p) {
    __shared__ uint64_t scan[8];
    __shared__ u32 told[10], keys[JL_SA_LIST], places[JL_SA_LIST];
    sample_gather_body(p, scan, told, keys, places);
}
// grid = rows, block = 256
extern "C" __global__ __launch_bounds__(256) void jl_sample_take(SampleArgs p) {
    __shared__ SampleLds s;
    sample_take_body(p, s);
}
