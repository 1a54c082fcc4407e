// Many new tokens over a cache -- prompts, long drafts: more than sixteen columns a unit (attend.h).
//
// Each of a workgroup's four or eight wavefronts has a tile of sixteen columns; the rows of 64 positions at a time go through LDS, as the fragments the matrix
// instruction takes (a fragment a kilobyte, a lane's sixteen bytes behind the next lane's: no bank is met twice), so rows are read once for 64 or 128 columns, and 8-bit
// values turned into f16 once.  Half of the wavefronts bring the values, half the keys, of the next 64 positions while all of them multiply: one barrier a step.  A
// wavefront keeps its columns' sums to the end, so nothing is exchanged; they leave through LDS as whole rows (64 tokens of a prompt 27.6 -> 22.9 us: the code that runs
// once is fetched once, and is most of a short call).
//
// A step of 128 columns x 64 positions x 128 has 384 matrix instructions over four SIMDs (0.64 us at the peak rate), 256 vector instructions a wavefront, 290 KB through LDS, and
// takes 1.65: each unit is busy a fifth to a third of the time, and the rest is the wavefronts' waits at the same places (bringing the rows is a quarter of a call: 8192 tokens 850 us,
// 600 with rows that stand in LDS already).  Measured (32 heads over 8 of 128, bf16): a prompt of 8192 856 us, 642 TFLOP/s of the product's operations, 960 of the
// instructions' (P in two pieces; a library's product of 8192^3 reaches 1400); of 2048 87, of 512 23; 3 x 683 over 2048 120 (f16 124, 8-bit rows with f32 q and out 172).
// Tried and not kept: every other span of a unit in a workgroup of its own (3 x 683: 141 for 133), a raised priority around the products (134 to 139 for 133), keys by
// loads that write LDS directly (150 for 133).
#pragma once
#include "attend.h"

template <int DP> constexpr int at_stage_words() { return (4 * (DP / 32) + 2 * (DP / 16)) * 256; }   // 64 positions' fragments

// lds: words [2][at_stage_words], then [2] of scales: keys' [64], values' [64]; then [2] of marks [4], and one mark of the span.
template <int TYPE, int DP, int QP, int PP, int WAVES>
__device__ __forceinline__ void attend_many_body(const AttendArgs& p, u32x4* lds, uint64_t* find) {
    constexpr bool BF = TYPE == JL_BF16, I8 = TYPE == JL_I8;
    static_assert(WAVES * 16 * DP <= 2 * at_stage_words<DP>(), "the columns' rows in the stages' LDS");
    constexpr int C = DP / 16, KC = DP / 32, B = I8 ? 1 : 2, VB = C * B;   // elements of the values a lane, fragments of a key, bytes
    constexpr int KL = I8 ? KC / 2 : KC, VW = (C * B * 4 / WAVES + 3) / 4;   // loads of a tile of keys; words of values a position and lane
    constexpr int STAGE = at_stage_words<DP>() / 4;       // in 16-byte pieces
    constexpr float OFF = BF ? 0.f : JL_AT_OFF;
    const float inf = __builtin_inff();
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    float* const scales = (float*)(lds + 2 * STAGE);      // [2][128]
    u32* const marks = (u32*)(scales + 2 * 128);          // [2][4]: tiles on no page, values that are no number, of each half

    AtWork job;
    u32 unit_end = 0, w = 0;
    AtJoin join = {0, 0, 0, 0, 0, {0, 0, 0}};
    if (p.whole) {   // (the last units, which see most of a prompt, first; a key head's on one L2)
        const u32 planes = (u32)p.c.n_kv * (u32)p.blocks, b = blockIdx.x, i = b / planes, unit = (u32)p.units - 1 - i;
        job.plane = b - i * planes;
        job.off = 0;
        job.first = 0;
        job.end = ~0ull;
        unit_end = min((unit + 1) * (u32)p.per, (u32)p.ntok);
        job.tok = unit * (u32)p.per;
    } else {
        w = at_group_of(blockIdx.x, (u32)p.wgs);
        if (!at_work<true, WAVES>(p, w, find, job)) {
            if (threadIdx.x == 0) at_join_of<DP>(p)[w] = join;
            return;
        }
    }
    const u32 row_bytes = (u32)p.c.row_stride * B;
    const size_t head_bytes = p.c.head_stride * B, page_bytes = p.c.page_stride * B;
    const u32 in_page = (1u << p.c.shift) - 1;
    // What a wavefront brings of 64 positions: of four, two bring the values of 32 positions each and two the keys; of eight, four bring the values of 32 positions and
    // half of the elements, four the keys of 16.
    constexpr int VS = WAVES / 4, TILES = 2 / VS, CV = C / VS;      // shares of the values' elements; tiles of keys; elements a lane
    const bool brings_keys = wave >= WAVES / 2;
    const int half = brings_keys ? (wave - WAVES / 2) * TILES / 2 : wave & 1, share = wave >> 1;      // (share: of the values)
    const int tile0 = brings_keys ? (wave - WAVES / 2) * TILES % 2 : 0;
    // a lane's bytes of a tile's rows, for what its wavefront brings
    u32 ko[KL];
#pragma unroll
    for (int c = 0; c < KL; c++) {
        const int d = I8 ? 64 * c + 16 * g : 32 * c + 8 * g;
        ko[c] = d < p.c.d ? n * row_bytes + (u32)d * B : JL_AT_NOWHERE;
    }
    const u32 vo = C * n < p.c.d ? 4 * g * row_bytes + (u32)n * VB + (u32)(share & (VS - 1)) * CV * B : JL_AT_NOWHERE;

    for (uint64_t at = job.first; at < job.end;) {
        const AtSpan span = at_span<true>(p, job.tok);
        const u32 lo = span.lo, hi = span.hi, plane = job.plane, c0 = job.off, n_chunks = at_chunks(lo, hi);
        job.tok = span.t1;
        if (!p.whole && job.tok == (u32)p.ntok) {
            job.tok = 0;
            job.plane++;
        }
        if (c0 >= n_chunks) {      // (a span of the first unit that others have)
            job.off -= n_chunks;
            continue;
        }
        job.off = 0;
        const u32 left = (u32)min((uint64_t)(n_chunks - c0), job.end - at);
        const u32 kv = p.blocks > 1 ? plane / (u32)p.blocks : plane;
        // steps of 64 positions, from the chunk's first on, up to the last that any token sees
        const u32 s0 = max(2 * (lo / JL_AT_CHUNK + c0), lo / 64), s1 = min(2 * (lo / JL_AT_CHUNK + c0 + left), (hi + 63) / 64);
        const u32* const pages = p.c.table + (size_t)span.seq * p.c.table_stride;
        const char* const from = (const char*)(brings_keys ? p.c.k : p.c.v) + kv * head_bytes;
        const float* const from_scales = brings_keys ? p.c.k_scale : p.c.v_scale;

        // A value that is no number, in a place that only some of the tokens see, would reach the others as 0 * NaN: such a span is passed over
        // again, a token at a time, with zeros for what that token does not see.
        u32 only = ~0u, zlo = lo, zhi = hi;       // the token; what is not zeros

        u32 pg = 0, page[2];
        auto look = [&](u32 s) {
            const u32 at0 = (s + (lane >> 1)) * 64 + half * 32 + 16 * (lane & 1);
            pg = s + (lane >> 1) < s1 && at0 < hi && at0 + 16 > lo ? pages[at0 >> p.c.shift] : ~0u;
        };
        u32 st[8 * VW > 4 * TILES * KL ? 8 * VW : 4 * TILES * KL];
        float sc = 0.f;
        auto ask = [&](u32 s) {
            if (((s - s0) & 31) == 0) look(s);
            const u32 p0 = s * 64 + half * 32;
            at_rsrc rs[2];
            size_t sa[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                page[i] = (u32)__builtin_amdgcn_readlane((i32)pg, (int)(2 * ((s - s0) & 31) + i));
                const u32 slot = (p0 + 16 * i) & in_page, held = page[i] < p.c.n_page ? page[i] : 0u;
                rs[i] = at_buffer(from + held * page_bytes + (size_t)slot * row_bytes);
                sa[i] = ((((size_t)held * p.c.n_kv + kv) << p.c.shift) + slot) + n;
            }
            if (brings_keys) {
#pragma unroll
                for (int i = 0; i < TILES; i++) {
                    const at_rsrc r = TILES == 1 && tile0 ? rs[1] : rs[i];
#pragma unroll
                    for (int c = 0; c < KL; c++) {
                        const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(r, ko[c], 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) st[(i * KL + c) * 4 + e] = y[e];
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if constexpr (VW == 1 && CV * B == 2) st[4 * i + r] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs[i], vo, r * row_bytes, 0);
                        else if constexpr (VW == 1) st[4 * i + r] = __builtin_amdgcn_raw_buffer_load_b32(rs[i], vo, r * row_bytes, 0);
                        else if constexpr (VW == 2) {
                            const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(rs[i], vo, r * row_bytes, 0);
                            st[(4 * i + r) * 2] = y.x; st[(4 * i + r) * 2 + 1] = y.y;
                        } else {
#pragma unroll
                            for (int e = 0; e < VW; e += 4) {
                                const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(rs[i], vo + 4 * e, r * row_bytes, 0);
#pragma unroll
                                for (int f = 0; f < 4; f++) st[(4 * i + r) * VW + e + f] = y[f];
                            }
                        }
                    }
            }
            if constexpr (I8) sc = from_scales[(lane >> 4) & 1 ? sa[1] : sa[0]];
        };
        auto put = [&](u32 s) {
            u32x4* const to = lds + (s & 1) * STAGE;
            const u32 p0 = s * 64 + half * 32;
            const bool none = max(page[0], page[1]) >= p.c.n_page;
            if (brings_keys) {
#pragma unroll
                for (int i = 0; i < TILES; i++)
#pragma unroll
                    for (int c = 0; c < KC; c++) {
                        u32x4 y;
                        if constexpr (I8) {   // bytes b to f16: 0x6400 | (b + 128) is 1152 + b
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const u32 t2 = __builtin_amdgcn_perm(0u, st[(i * KL + c / 2) * 4 + 2 * (c % 2) + j / 2], j % 2 ? 0x0c030c02u : 0x0c010c00u) ^ 0x64806480u;
                                y[j] = __builtin_bit_cast(u32, __builtin_bit_cast(f16x2, t2) - f16x2{(_Float16)1152, (_Float16)1152});
                            }
                        } else {
                            y = u32x4{st[(i * KL + c) * 4], st[(i * KL + c) * 4 + 1], st[(i * KL + c) * 4 + 2], st[(i * KL + c) * 4 + 3]};
                        }
                        to[((2 * half + tile0 + i) * KC + c) * 64 + lane] = y;
                    }
                if (lane == 0 && tile0 == 0) marks[(s & 1) * 4 + half] = (page[0] >= p.c.n_page ? 1u : 0u) | (page[1] >= p.c.n_page ? 2u : 0u);
                if constexpr (I8)
                    if (lane < 32 && tile0 == 0) scales[(s & 1) * 128 + half * 32 + lane] = sc;
            } else {
                if (none || p0 < zlo || p0 + 32 > zhi) {   // zeros for what no token sees: what lies there may be no number
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const u32 at0 = p0 + 16 * (j / 4) + 4 * g + j % 4;
                        const bool seen = page[j / 4] < p.c.n_page && at0 >= zlo && at0 < zhi;
#pragma unroll
                        for (int e = 0; e < VW; e++) st[j * VW + e] = seen ? st[j * VW + e] : 0u;
                    }
                    const u32 at0 = p0 + (lane & 31);
                    if (!(page[(lane >> 4) & 1] < p.c.n_page && at0 >= zlo && at0 < zhi)) sc = 0.f;
                }
                if (!I8 && only == ~0u && span.t1 - span.t0 > 1 && (p0 < span.lo_all || p0 + 32 > span.hi_all)) {
                    u16x2 big = {0, 0};
#pragma unroll
                    for (int j = 0; j < 8 * VW; j++) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, st[j] & 0x7fff7fffu));
                    if (max(big.x, big.y) >= (BF ? 0x7f80 : 0x7c00)) marks[8] = 1;
                }
#pragma unroll
                for (int j = 0; j < CV; j++) {
                    u32x4 vt;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if constexpr (I8) {
                            const u32 b = j % 4;
                            const u32 t2 = __builtin_amdgcn_perm(st[(2 * r + 1) * VW + j / 4], st[2 * r * VW + j / 4], 0x0c000c00u | b | (4 + b) << 16) ^ 0x64806480u;
                            vt[r] = __builtin_bit_cast(u32, __builtin_bit_cast(f16x2, t2) - f16x2{(_Float16)1152, (_Float16)1152});
                        } else {
                            vt[r] = __builtin_amdgcn_perm(st[(2 * r + 1) * VW + j / 2], st[2 * r * VW + j / 2], j % 2 ? 0x07060302u : 0x05040100u);
                        }
                    }
                    to[(4 * KC + half * C + share * CV + j) * 64 + lane] = vt;
                }
                if constexpr (I8)
                    if (lane < 32 && share == 0) scales[(s & 1) * 128 + 64 + half * 32 + lane] = sc;
            }
        };
        // the column
        u32 tok, head, clo, chi;
        const bool live = at_column(p, span.t0, span.t1, plane, (u32)wave * 16 + n, tok, head);
        {
            u32 q0;
            at_sees(p, tok, q0, clo, chi);
        }
        if (!live) clo = chi = 0;
        u32 wlo = live ? clo : ~0u, whi = chi, wlo_all = clo, whi_all = live ? chi : ~0u;      // of the wavefront's columns
#pragma unroll
        for (int d = 1; d < 16; d *= 2) {
            wlo = min(wlo, (u32)__shfl_xor((int)wlo, d, 64)); whi = max(whi, (u32)__shfl_xor((int)whi, d, 64));
            wlo_all = max(wlo_all, (u32)__shfl_xor((int)wlo_all, d, 64)); whi_all = min(whi_all, (u32)__shfl_xor((int)whi_all, d, 64));
        }
        wlo = at_uni(wlo); whi = at_uni(whi); wlo_all = at_uni(wlo_all); whi_all = at_uni(whi_all);
        u32x4 qf[QP][KC];
        float qs;
        {
            float x[KC][8];
            at_load_query<I8, KC>(p, live, tok, head, x);
            at_query<BF, QP, KC>(p, x, qf, qs);
        }

        for (;;) {
        f32x4 acc[C];
        float m = -inf, l = 0.f;
        int ve = -200;          // 8-bit rows: the column's acc is times 2^-ve
#pragma unroll
        for (int j = 0; j < C; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

        if (s0 < s1) ask(s0);
        __syncthreads();        // (the pass before has read its last stage)
        if (threadIdx.x == 0) marks[8] = 0;
        __syncthreads();
        if (s0 < s1) put(s0);
        __syncthreads();
        for (u32 s = s0; s < s1; s++) {
            if (s + 1 < s1) ask(s + 1);
            const u32x4* const in = lds + (s & 1) * STAGE;
            const u32* const mark = marks + (s & 1) * 4;
            const u32 p0 = s * 64;
            if (p0 < whi && p0 + 64 > wlo) {
                const u32 none = at_uni(mark[0] | mark[1] << 2);
                const bool edge = p0 < wlo_all || p0 + 64 > whi_all || none;
                const u32x4* const kin = in + lane;
                const u32x4* const vin = in + 4 * KC * 64 + lane;
                // (fragments two ahead of the products that take them)
                f32x4 sco[4];
                u32x4 kt[3] = {kin[0], kin[KC * 64], {0, 0, 0, 0}};
#pragma unroll
                for (int i = 0; i < 4 * KC; i++) {      // tile i % 4, piece i / 4 of the row
                    if (i + 2 < 4 * KC) kt[(i + 2) % 3] = kin[((i + 2) % 4 * KC + (i + 2) / 4) * 64];
#pragma unroll
                    for (int q = 0; q < QP; q++)
                        sco[i % 4] = at_mfma<BF>(kt[i % 3], qf[q][i / 4], i / 4 || q ? sco[i % 4] : f32x4{0.f, 0.f, 0.f, 0.f});
                }
                f32x4 vs[4];
                if constexpr (I8) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        sco[i] *= *(const f32x4*)(scales + (s & 1) * 128 + 16 * i + 4 * g);
                        vs[i] = *(const f32x4*)(scales + (s & 1) * 128 + 64 + 16 * i + 4 * g);
                    }
                }
                u32x4 vt[3] = {vin[0], vin[C * 64], {0, 0, 0, 0}}, pf[2][PP];
                float y[16], by = qs;       // scores are y by
#pragma unroll
                for (int j = 0; j < 16; j++) y[j] = sco[j / 4][j % 4];
                if (edge || p.cap != 0.f) {
                    by = 1.f;
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        y[j] *= qs;
                        if (p.cap != 0.f) {
                            y[j] = p.cap * JL_AT_LOG2E * at_tanh(y[j]);
                            asm volatile("" : "+v"(y[j]));     // (one after the other: side by side they take the loop's registers)
                        }
                        const u32 at0 = p0 + 16 * (j / 4) + 4 * g + j % 4;
                        const bool sees = !(none >> (j / 4) & 1) && at0 >= clo && at0 < chi;
                        y[j] = sees ? y[j] : -inf;
                        if constexpr (I8) vs[j / 4][j % 4] = sees ? vs[j / 4][j % 4] : 0.f;      // (this column's: others may see it)
                    }
                }
                if constexpr (I8) {   // the running power of two over the scales of the values that the column sees
                    float big = 0.f;      // (a scale may be of either sign)
#pragma unroll
                    for (int j = 0; j < 16; j++) big = fmaxf(big, fabsf(vs[j / 4][j % 4]));
                    big = at_max4(big);
                    const int to = max(ve, big > 0.f ? __builtin_amdgcn_frexp_expf(big) : -200);
                    if (__ballot(to > ve)) {
#pragma unroll
                        for (int j = 0; j < C; j++)
#pragma unroll
                            for (int r = 0; r < 4; r++) acc[j][r] = __builtin_amdgcn_ldexpf(acc[j][r], ve - to);
                        ve = to;
                    }
                }
                float top = y[0];
#pragma unroll
                for (int j = 1; j < 16; j++) top = fmaxf(top, y[j]);
                top = fmaxf(at_max4(top) * by, m);
                if (__ballot(top > m + JL_AT_SLACK(BF))) {
                    const float turn = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);   // (from -inf: 0)
                    l *= turn;
#pragma unroll
                    for (int j = 0; j < C; j++) acc[j] *= turn;
                    m = top;
                }
                const float from = OFF - (m > -inf ? m : 0.f);
                float sums[4];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    y[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j], by, from));
                    sums[j / 4] = j % 4 ? sums[j / 4] + y[j] : y[j];
                    if constexpr (I8) y[j] *= __builtin_amdgcn_ldexpf(vs[j / 4][j % 4], -ve);
                }
                l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int q = 0; q < PP; q++)
#pragma unroll
                        for (int j = 0; j < 4; j++) pf[h][q][j] = at_piece<BF>(y[8 * h + 2 * j], y[8 * h + 2 * j + 1]);
#pragma unroll
                for (int i = 0; i < 2 * C; i++) {      // element i / 2, half i % 2
                    if (i + 2 < 2 * C) vt[(i + 2) % 3] = vin[((i + 2) % 2 * C + (i + 2) / 2) * 64];
#pragma unroll
                    for (int q = 0; q < PP; q++) acc[i / 2] = at_mfma<BF>(vt[i % 3], pf[i % 2][q], acc[i / 2]);
                }
            }
            if (s + 1 < s1) put(s + 1);
            __syncthreads();
        }

        if (!I8 && only == ~0u && at_uni(marks[8])) {
            u32 q0;
            only = span.t0;
            at_sees(p, only, q0, zlo, zhi);
            zlo = at_uni(zlo); zhi = at_uni(zhi);
            continue;
        }
        const u32 slot = 2 * w + (at == job.first ? 0u : 1u);
        const bool whole = left == n_chunks;
        if (c0 == 0 && !whole) join = AtJoin{span.t0, span.t1, plane, job.share.holder(at + n_chunks - 1) + 1, slot, {0, 0, 0}};
        // through LDS, where each wavefront has its columns, so that rows leave whole
        const float sum = at_sum4(l);
        float by = I8 ? __builtin_amdgcn_ldexpf(1.f, ve) : 1.f;
        const bool gives = live && (only == ~0u || tok == only);
        const u32 col0 = (u32)wave * 16;
        if (whole && gives) by *= at_finish(p, tok, head, m, sum, OFF, g == 0);
        if (!whole && gives && g == 0) *at_part_ml<DP>(p, slot, col0 + n) = f32x2{m, sum};
        float* const mine = (float*)lds + wave * 16 * DP;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < C; j += 4) *(f32x4*)(mine + n * DP + C * (4 * g + i) + j) = f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]} * by;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // (a wavefront's own LDS)
        const u32 out_tok = gives ? tok : ~0u, quad = (lane & (DP / 4 - 1)) * 4;
#pragma unroll 1
        for (int c = lane / (DP / 4); c < 16; c += 256 / DP) {       // a column's row of four-element pieces
            const u32 t = (u32)__shfl((int)out_tok, c, 64), h = (u32)__shfl((int)head, c, 64);
            const f32x4 y = *(const f32x4*)(mine + c * DP + quad);
            const float v[4] = {y.x, y.y, y.z, y.w};
            if (t == ~0u) continue;
            if (!whole) *(f32x4*)(at_part<DP>(p, slot, col0 + c) + quad) = y;
            else if (quad < (u32)p.c.d) at_store<4>(p, t, h, (int)quad, v);
        }
        if (only == ~0u || ++only == span.t1) break;
        u32 q0;
        at_sees(p, only, q0, zlo, zhi);
        zlo = at_uni(zlo); zhi = at_uni(zhi);
        }
        at += left;
        if (p.whole && span.t1 == unit_end) break;
    }
    if (!p.whole && threadIdx.x == 0) at_join_of<DP>(p)[w] = join;
}
