// A new token a sequence, or a few, over their cache: up to sixteen columns a unit (attend.h).
//
// MANY: units of several tokens.  A workgroup's wavefronts take 32 positions each of a chunk, with sums of their own that meet in LDS at a span's end.  What bounds it is
// how many loads are on their way: a step's keys are asked for as soon as the ones before them have been multiplied, its values likewise, so a wavefront always has
// a step of each in flight; the page numbers of 32 steps lie in its lanes.  q is asked for ahead of the rows (behind them its wait is theirs: 7.7 -> 9.4 us over 777).
// Measured (8 key heads of 128; this kernel, then the join): 64 sequences to 8192 of 8-bit rows 119 + 5 us (4.7 TB/s), one of 131071 bf16 97 + 7.4 (5.5 TB/s), one
// of 777 f16 7.7 + 3.3: launches and four trips to memory one after the other.
// Rows are read through buffer descriptors, whose bound gives zeros to the lanes behind a row that is no power of two wide.
#pragma once
#include "attend.h"

// LDS: floats [4][16][DP + 4], [4][16][2]; find: 16 words of 8 bytes.
template <int TYPE, int DP, int QP, int PP, bool MANY>
__device__ __forceinline__ void attend_one_body(const AttendArgs& p, float* lds, uint64_t* find) {
    constexpr bool BF = TYPE == JL_BF16, I8 = TYPE == JL_I8;
    constexpr int C = DP / 16, KC = DP / 32, B = I8 ? 1 : 2, VB = C * B;   // bytes of V a position and lane
    constexpr int KL = I8 ? KC / 2 : KC, VW = (VB + 3) / 4;
    constexpr int ROW = DP + 4;
    constexpr float OFF = BF ? 0.f : JL_AT_OFF;
    const float inf = __builtin_inff();
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    AtWork job;
    u32 unit_end = 0, w = 0;
    AtJoin join = {0, 0, 0, 0, 0, {0, 0, 0}};
    if (p.whole) {
        const u32 planes = (u32)p.c.n_kv * (u32)p.blocks, unit = blockIdx.x / planes;
        job.plane = blockIdx.x - unit * planes;
        job.off = 0;
        job.first = 0;
        job.end = ~0ull;
        job.tok = unit * (u32)p.per;
        unit_end = min(job.tok + (u32)p.per, (u32)p.ntok);
    } else {
        w = at_group_of(blockIdx.x, (u32)p.wgs);
        if (!at_work<MANY, 4>(p, w, find, job)) {
            if (threadIdx.x == 0) at_join_of<DP>(p)[w] = join;
            return;
        }
    }

    const u32 row_bytes = (u32)p.c.row_stride * B;      // (16 rows are less than 2^31 bytes)
    const size_t head_bytes = p.c.head_stride * B, page_bytes = p.c.page_stride * B;
    const u32 in_page = (1u << p.c.shift) - 1;
    float* const ml = lds + 4 * 16 * ROW;
    // a lane's bytes of a tile's keys (position n) and values (positions 4g..4g+3)
    u32 ko[KL];
#pragma unroll
    for (int c = 0; c < KL; c++) {
        const int d = I8 ? 64 * c + 16 * g : 32 * c + 8 * g;
        ko[c] = d < p.c.d ? n * row_bytes + (u32)d * B : JL_AT_NOWHERE;
    }
    const u32 vo = C * n < p.c.d ? 4 * g * row_bytes + (u32)n * VB : JL_AT_NOWHERE;

    for (uint64_t at = job.first; at < job.end;) {
        const AtSpan span = at_span<MANY>(p, job.tok);
        const u32 lo = span.lo, hi = span.hi, plane = job.plane, c0 = job.off, n_chunks = at_chunks(lo, hi);
        job.tok = span.t1;
        if (!p.whole && job.tok == (u32)p.ntok) {
            job.tok = 0;
            job.plane++;
        }
        if (MANY && c0 >= n_chunks) {      // (a span of the first unit that others have)
            job.off -= n_chunks;
            continue;
        }
        job.off = 0;
        const u32 left = (u32)min((uint64_t)(n_chunks - c0), job.end - at);
        const u32 kv = p.blocks > 1 ? plane / (u32)p.blocks : plane;
        u32 tok, head, clo = lo, chi = hi;      // of this lane's column
        const bool col_live = at_column(p, span.t0, span.t1, plane, n, tok, head);
        if (MANY) {
            u32 s0;
            at_sees(p, tok, s0, clo, chi);
        }
        const u32 base = lo / JL_AT_CHUNK + c0;         // this workgroup's first chunk
        const u32* const pages = p.c.table + (size_t)span.seq * p.c.table_stride;
        const char* const k0 = (const char*)p.c.k + kv * head_bytes;
        const char* const v0 = (const char*)p.c.v + kv * head_bytes;

        // page of this lane's tile among those of 32 steps
        u32 pg = 0;
        auto look = [&](u32 k) {
            const u32 at0 = (base + k + (lane >> 1)) * JL_AT_CHUNK + wave * 32 + 16 * (lane & 1);
            pg = k + (lane >> 1) < left && at0 < hi && at0 + 16 > lo ? pages[at0 >> p.c.shift] : ~0u;
        };
        // A value that is no number, in a place that only some of the tokens see, would reach the others as 0 * NaN: such a span is passed over
        // again, a token at a time, with zeros for what that token does not see.
        u32 only = ~0u, zlo = lo, zhi = hi;       // the token; what is not zeros
        bool odd = false;
        for (;;) {
        look(0);

        float x[KC][8];
        at_load_query<I8, KC>(p, col_live, tok, head, x);
        u32x4 kf[2][KL];
        u32 vw[8][VW];
        f32x4 ks[2], vs[2];
        u32 page[2], vpage[2];      // of the keys and of the values on their way
        auto tile = [&](u32 id, const char* from, u32 at0) {
            return at_buffer(from + (id < p.c.n_page ? id : 0u) * page_bytes + (size_t)(at0 & in_page) * row_bytes);
        };
        auto scales = [&](u32 id, const float* from, u32 at0) {
            return *(const f32x4*)(from + ((((size_t)(id < p.c.n_page ? id : 0u) * p.c.n_kv + kv) << p.c.shift) + (at0 & in_page) + 4 * g));
        };
        auto ask_k = [&](u32 k) {
            const u32 p0 = (base + k) * JL_AT_CHUNK + wave * 32;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                page[i] = (u32)__builtin_amdgcn_readlane((i32)pg, (int)(2 * (k & 31) + i));
                const at_rsrc r = tile(page[i], k0, p0 + 16 * i);
#pragma unroll
                for (int c = 0; c < KL; c++) kf[i][c] = __builtin_amdgcn_raw_buffer_load_b128(r, ko[c], 0, 0);
                if constexpr (I8) ks[i] = scales(page[i], p.c.k_scale, p0 + 16 * i);
            }
        };
        auto ask_v = [&](u32 k) {
            const u32 p0 = (base + k) * JL_AT_CHUNK + wave * 32;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const at_rsrc rs = tile(vpage[i], v0, p0 + 16 * i);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (VW == 1) vw[4 * i + r][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, vo, r * row_bytes, 0);
                    else if constexpr (VW == 2) {
                        const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(rs, vo, r * row_bytes, 0);
                        vw[4 * i + r][0] = y.x; vw[4 * i + r][1] = y.y;
                    } else {
#pragma unroll
                        for (int e = 0; e < VW; e += 4) {
                            const u32x4 y = __builtin_amdgcn_raw_buffer_load_b128(rs, vo + 4 * e, r * row_bytes, 0);
                            vw[4 * i + r][e] = y.x; vw[4 * i + r][e + 1] = y.y; vw[4 * i + r][e + 2] = y.z; vw[4 * i + r][e + 3] = y.w;
                        }
                    }
                }
                if constexpr (I8) vs[i] = scales(vpage[i], p.c.v_scale, p0 + 16 * i);
            }
        };
        ask_k(0);
        vpage[0] = page[0]; vpage[1] = page[1];
        ask_v(0);

        u32x4 qf[QP][KC];
        float qs;
        at_query<BF, QP, KC>(p, x, qf, qs);

        f32x4 acc[C];
        float m = -inf, l = 0.f;
        int ve = -200;          // 8-bit rows: the column's acc is times 2^-ve
#pragma unroll
        for (int j = 0; j < C; j++) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

        for (u32 k = 0; k < left; k++) {
            const u32 p0 = (base + k) * JL_AT_CHUNK + wave * 32;
            const bool edge = p0 < (MANY ? span.lo_all : lo) || p0 + 32 > (MANY ? span.hi_all : hi) || max(page[0], page[1]) >= p.c.n_page;
            f32x4 s[2];
            f32x4 kx[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (I8) kx[i] = ks[i];
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    u32x4 y;
                    if constexpr (I8) {   // bytes b to f16: 0x6400 | (b + 128) is 1152 + b
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const u32 t2 = __builtin_amdgcn_perm(0u, kf[i][c / 2][2 * (c % 2) + j / 2], j % 2 ? 0x0c030c02u : 0x0c010c00u) ^ 0x64806480u;
                            y[j] = __builtin_bit_cast(u32, __builtin_bit_cast(f16x2, t2) - f16x2{(_Float16)1152, (_Float16)1152});
                        }
                    } else {
                        y = kf[i][c];
                    }
#pragma unroll
                    for (int q = 0; q < QP; q++) s[i] = at_mfma<BF>(y, qf[q][c], s[i]);
                }
            }
            // the next keys
            u32 seen[2] = {page[0], page[1]};
            if (k + 1 < left) {
                if (((k + 1) & 31) == 0) look(k + 1);
                ask_k(k + 1);
            }

            float y[8], by = qs;       // scores are y by
#pragma unroll
            for (int j = 0; j < 8; j++) {
                y[j] = s[j / 4][j % 4];
                if constexpr (I8) y[j] *= kx[j / 4][j % 4];
            }
            const bool masks = edge || (MANY && only != ~0u);
            if (masks || p.cap != 0.f) {
                by = 1.f;
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] *= qs;
                if (p.cap != 0.f) {
#pragma unroll
                    for (int j = 0; j < 8; j++) y[j] = p.cap * JL_AT_LOG2E * at_tanh(y[j]);
                }
                if (masks) {   // what is hidden: no score, and zeros for values (what lies there may be no number)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const u32 at0 = p0 + 16 * (j / 4) + 4 * g + j % 4;
                        const bool held = seen[j / 4] < p.c.n_page, sees = held && at0 >= clo && at0 < chi, one = MANY ? held && at0 >= zlo && at0 < zhi : sees;
                        y[j] = sees ? y[j] : -inf;
#pragma unroll
                        for (int e2 = 0; e2 < VW; e2++) vw[j][e2] = one ? vw[j][e2] : 0u;
                        if constexpr (I8) vs[j / 4][j % 4] = sees ? vs[j / 4][j % 4] : 0.f;      // (this column's: others may see it)
                    }
                }
            }
            if (MANY && !I8 && edge && only == ~0u) {
                u16x2 big = {0, 0};
#pragma unroll
                for (int r = 0; r < 8; r++)
#pragma unroll
                    for (int e2 = 0; e2 < VW; e2++) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, vw[r][e2] & 0x7fff7fffu));
                odd = odd || max(big.x, big.y) >= (BF ? 0x7f80 : 0x7c00);
            }
            float top = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
            top = fmaxf(at_max4(top) * by, m);
            if (__ballot(top > m + JL_AT_SLACK(BF))) {
                const float turn = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);   // (from -inf: 0)
                l *= turn;
#pragma unroll
                for (int j = 0; j < C; j++) acc[j] *= turn;
                m = top;
            }
            if constexpr (I8) {   // the running power of two over the scales of the values that the column sees
                float big = 0.f;      // (a scale may be of either sign)
#pragma unroll
                for (int j = 0; j < 8; j++) big = fmaxf(big, fabsf(vs[j / 4][j % 4]));
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
            const float from = OFF - (m > -inf ? m : 0.f);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                y[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j], by, from));
                l += y[j];
                if constexpr (I8) y[j] *= __builtin_amdgcn_ldexpf(vs[j / 4][j % 4], -ve);
            }
            u32x4 pf[PP];
#pragma unroll
            for (int q = 0; q < PP; q++)
#pragma unroll
                for (int j = 0; j < 4; j++) pf[q][j] = at_piece<BF>(y[2 * j], y[2 * j + 1]);
            auto turned = [&](int j) {   // the values' fragment j
                u32x4 vt;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (I8) {
                        const u32 b = j % 4;
                        const u32 t2 = __builtin_amdgcn_perm(vw[2 * r + 1][j / 4], vw[2 * r][j / 4], 0x0c000c00u | b | (4 + b) << 16) ^ 0x64806480u;
                        vt[r] = __builtin_bit_cast(u32, __builtin_bit_cast(f16x2, t2) - f16x2{(_Float16)1152, (_Float16)1152});
                    } else {
                        vt[r] = __builtin_amdgcn_perm(vw[2 * r + 1][j / 2], vw[2 * r][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
                    }
                }
                return vt;
            };
#pragma unroll
            for (int j = 0; j < C; j++) {
                const u32x4 vt = turned(j);
#pragma unroll
                for (int q = 0; q < PP; q++) acc[j] = at_mfma<BF>(vt, pf[q], acc[j]);
            }
            if (k + 1 < left) {   // the next values
                vpage[0] = page[0]; vpage[1] = page[1];
                ask_v(k + 1);
            }
        }

        // the four wavefronts' sums to one
        const float sum = at_sum4(l);
        __syncthreads();
        if (g == 0) {
            ml[(wave * 16 + n) * 2] = m;
            ml[(wave * 16 + n) * 2 + 1] = sum;
        }
        if (MANY && !I8 && only == ~0u) {
            if (__syncthreads_or(odd && span.t1 - span.t0 > 1)) {
                u32 s0;
                only = span.t0;
                at_sees(p, only, s0, zlo, zhi);
                zlo = at_uni(zlo); zhi = at_uni(zhi);
                continue;
            }
        }
        const u32 slot = 2 * w + (at == job.first ? 0u : 1u);
        const bool whole = left == n_chunks;
        __syncthreads();
        float all = -inf;
#pragma unroll
        for (int k = 0; k < 4; k++) all = fmaxf(all, ml[(k * 16 + n) * 2]);
        float turn = m == all ? 1.f : __builtin_amdgcn_exp2f(m - all);   // (a wavefront that saw nothing: 0 times its zeros)
        if constexpr (I8) turn = __builtin_amdgcn_ldexpf(turn, ve);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < C; j += 4)
                *(f32x4*)(lds + (wave * 16 + n) * ROW + C * (4 * g + i) + j) = f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]} * turn;
        __syncthreads();
        // thread: column tid / 16, C elements
        const u32 col = threadIdx.x >> 4, d0 = C * (threadIdx.x & 15);
        u32 its, of;
        if (at_column(p, span.t0, span.t1, plane, col, its, of) && (!MANY || only == ~0u || its == only)) {
            float mm = -inf, lsum = 0.f, y[C];
#pragma unroll
            for (int k = 0; k < 4; k++) mm = fmaxf(mm, ml[(k * 16 + col) * 2]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float mk = ml[(k * 16 + col) * 2];
                lsum += ml[(k * 16 + col) * 2 + 1] * (mk == mm ? 1.f : __builtin_amdgcn_exp2f(mk - mm));
            }
#pragma unroll
            for (int i = 0; i < C; i += 4) {
                f32x4 z = *(const f32x4*)(lds + col * ROW + d0 + i);
#pragma unroll
                for (int k = 1; k < 4; k++) z += *(const f32x4*)(lds + (k * 16 + col) * ROW + d0 + i);
#pragma unroll
                for (int r = 0; r < 4; r++) y[i + r] = z[r];
            }
            if (whole) {
                const float inv = at_finish(p, its, of, mm, lsum, OFF, d0 == 0);
#pragma unroll
                for (int i = 0; i < C; i++) y[i] *= inv;
                if (d0 < (u32)p.c.d) at_store<C>(p, its, of, d0, y);
            } else {
                if (d0 == 0) *at_part_ml<DP>(p, slot, col) = f32x2{mm, lsum};
#pragma unroll
                for (int i = 0; i < C; i += 4) *(f32x4*)(at_part<DP>(p, slot, col) + d0 + i) = f32x4{y[i], y[i + 1], y[i + 2], y[i + 3]};
            }
        }
        if (!MANY || only == ~0u || ++only == span.t1) break;
        u32 s0;
        at_sees(p, only, s0, zlo, zhi);
        zlo = at_uni(zlo); zhi = at_uni(zhi);
        }
        if (c0 == 0 && left < n_chunks) join = AtJoin{span.t0, span.t1, plane, job.share.holder(at + n_chunks - 1) + 1, 2 * w + (at == job.first ? 0u : 1u), {0, 0, 0}};
        at += left;
        if (p.whole && span.t1 == unit_end) break;
    }
    if (!p.whole && threadIdx.x == 0) at_join_of<DP>(p)[w] = join;
}
