// The kernels of a decode step that stand between a block's projections and behind the last one.
#pragma once
#include "attend.h"
#include "kv_cache.h"
#include "sample.h"

// grid = (rows / (256 / lanes), 2), block = 256
extern "C" __global__ __launch_bounds__(256) void jl_kv_write(KvRowsArgs p) { kv_rows_body<true>(p); }
extern "C" __global__ __launch_bounds__(256) void jl_kv_read(KvRowsArgs p) { kv_rows_body<false>(p); }

// grid = p.wgs, block = 256
#define JL_ATTEND(T, TYPE, DP, QP, NT)                                                                                              \
    extern "C" __global__ __launch_bounds__(256, DP == 256 ? 1 : 2) void jl_attend_##T##_d##DP##_q##QP##_n##NT(AttendArgs p) {      \
        __shared__ __attribute__((aligned(16))) float lds[4 * 16 * (DP + 4) + 128];                                                 \
        __shared__ uint64_t find[8];                                                                                                \
        attend_body<TYPE, DP, QP, NT>(p, lds, find);                                                                                \
    }
#define JL_ATTEND_Q(T, TYPE, QP)                                                                                                    \
    JL_ATTEND(T, TYPE, 64, QP, 1) JL_ATTEND(T, TYPE, 64, QP, 2) JL_ATTEND(T, TYPE, 128, QP, 1) JL_ATTEND(T, TYPE, 128, QP, 2)       \
    JL_ATTEND(T, TYPE, 256, QP, 1)
JL_ATTEND_Q(f16, JL_F16, 1) JL_ATTEND_Q(f16, JL_F16, 2) JL_ATTEND_Q(i8, JL_I8, 1) JL_ATTEND_Q(i8, JL_I8, 2)
JL_ATTEND_Q(bf16, JL_BF16, 1) JL_ATTEND_Q(bf16, JL_BF16, 3)
#define JL_ATTEND_JOIN(DP, NT)                                                                                                      \
    extern "C" __global__ __launch_bounds__(256) void jl_attend_join_d##DP##_n##NT(AttendArgs p) {                                  \
        __shared__ uint64_t find[8];                                                                                                \
        attend_join_body<DP, NT>(p, find);                                                                                          \
    }
JL_ATTEND_JOIN(64, 1) JL_ATTEND_JOIN(64, 2) JL_ATTEND_JOIN(128, 1) JL_ATTEND_JOIN(128, 2) JL_ATTEND_JOIN(256, 1)

// grid = rows, block = 1024
extern "C" __global__ __launch_bounds__(1024) void jl_sample(SampleArgs p) {
    __shared__ SampleLds s;
    sample_body(p, s);
}
