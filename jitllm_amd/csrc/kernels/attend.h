// Attention of new tokens over a paged cache (jl_attend_dev).  Token t of sequence s sees the positions lo = max(0, len - window) to
// hi = len of s; for each of its heads
//
//   s_p = scale * (q . k_p), or cap * tanh(scale * (q . k_p) / cap);   w_p = e^(s_p - m);   out = sum w_p v_p / (sum w_p + e^(sink - m))
//
// in one pass with a running maximum m.  A token and a head are a COLUMN of sixteen: `group` heads share a key head, and where tokens of one
// sequence follow each other `per` of them share the pass (a UNIT: `per` tokens, one key head).  On the matrix cores, 16x16x32:
//
//   S^T = K Q^T: a lane (n = lane & 15, g = lane >> 4) holds of column n the scores of positions 4g..4g+3 of each tile of sixteen.
//   O^T = V^T P^T: k runs over 32 positions, slot (g, j) being position 4g + j of the first tile for j < 4 and of the second behind it,
//     which is where S^T left them: P goes from one product to the next without leaving its lane.
//   V lies [position][d]; a lane loads its eight positions' rows, c = DP / 16 elements each from d = c n on (a row of 16 lanes is whole), and
//     turns them into the c fragments of eight positions each by byte permutes: fragment j holds d = c n + j.
//   A column's m, sum and O stay in the four lanes of its n: the running maximum is two lane swaps, rescaling is in-lane.
//
// Precision: K and V are exact in the instruction's type (8-bit rows as f16 integers, their scale applied to S, and to P relative to a running power of two); q and
// P are split into pieces that hold 22 (f16) or 24 and 16 or 24 (bf16) bits, so what rounds is the f32 sums, as in a plain product in f32.
//
// Work: a unit's positions in chunks of 128 (a workgroup's four wavefronts, 32 each).  The workgroups share the chunks of all units and key heads
// evenly, whatever their lengths, each a contiguous run of them; a unit that ends up with more than one workgroup leaves partial sums that attend_join adds up.
#pragma once
#include "args.h"
#include "common.h"
#include "kv_cache.h"

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 at_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

#define JL_AT_CHUNK 128      // positions a workgroup's step
#define JL_AT_LOG2E 1.4426950408889634f
#define JL_AT_LN2 0.6931471805599453f

template <bool BF> __device__ __forceinline__ f32x4 at_mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(at_bf16x8, a), __builtin_bit_cast(at_bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(at_f16x8, a), __builtin_bit_cast(at_f16x8, b), c, 0, 0, 0);
}
// Two values in the type's bits, to nearest even, and what that leaves of them.
template <bool BF> __device__ __forceinline__ u32 at_piece(float& x, float& y) {
    if constexpr (BF) {
        const at_bf16x2 h = {(__bf16)x, (__bf16)y};
        x -= (float)h.x;
        y -= (float)h.y;
        return __builtin_bit_cast(u32, h);
    } else {
        const f16x2 h = {(_Float16)x, (_Float16)y};
        x -= (float)h.x;
        y -= (float)h.y;
        return __builtin_bit_cast(u32, h);
    }
}
// Largest of the four lanes of a column; every one of them has it.
__device__ __forceinline__ float at_max4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float at_sum4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// tanh: the series up to 0.3 (the next term is under 2^-24 of the sum there, where 1 - 2 / (e^2y + 1) cancels), the exponential's form beyond.
__device__ __forceinline__ float at_tanh(float y) {
    const float z = y * y;
    const float small = y + y * z * (-1.f / 3.f + z * (2.f / 15.f + z * (-17.f / 315.f + z * (62.f / 2835.f))));
    const float large = 1.f - 2.f / (__builtin_amdgcn_exp2f(2.f * JL_AT_LOG2E * y) + 1.f);
    return z < 0.09f ? small : large;
}

// ---- which positions, units and chunks -----------------------------------------

__device__ __forceinline__ void at_sees(const AttendArgs& p, u32 t, u32& seq, u32& lo, u32& hi) {
    seq = p.seq ? p.seq[t] : t;
    hi = seq < p.c.n_seq ? p.len[t] : 0u;
    hi = min((uint64_t)hi, (uint64_t)p.c.table_pages << p.c.shift);
    lo = p.window && hi > (u32)p.window ? hi - (u32)p.window : 0u;
}
__device__ __forceinline__ u32 at_chunks(u32 lo, u32 hi) { return hi > lo ? ((hi - 1) / JL_AT_CHUNK) - lo / JL_AT_CHUNK + 1 : 0u; }

// Tokens t to `end` of a unit that follow each other in one sequence, and what they see together.
struct AtRun {
    u32 t, end, seq, lo, hi;            // [lo, hi): seen by one of them
    u32 lo_all, hi_all;                 // [lo_all, hi_all): by all
};
__device__ __forceinline__ AtRun at_run(const AttendArgs& p, u32 t, u32 last) {
    AtRun r;
    r.t = t;
    at_sees(p, t, r.seq, r.lo, r.hi);
    r.lo_all = r.lo;
    r.hi_all = r.hi;
    for (r.end = t + 1; r.end < last; r.end++) {
        u32 seq, lo, hi;
        at_sees(p, r.end, seq, lo, hi);
        if (seq != r.seq) break;
        r.lo = min(r.lo, lo);
        r.hi = max(r.hi, hi);
        r.lo_all = max(r.lo_all, lo);
        r.hi_all = min(r.hi_all, hi);
    }
    return r;
}
// A unit's chunks, one at least: a unit that sees nothing has its zeros written.
__device__ __forceinline__ u32 at_unit_chunks(const AttendArgs& p, u32 unit) {
    const u32 last = min((unit + 1) * (u32)p.per, (u32)p.ntok);
    u32 n = 0;
    for (u32 t = unit * p.per; t < last;) {
        const AtRun r = at_run(p, t, last);
        n += at_chunks(r.lo, r.hi);
        t = r.end;
    }
    return max(n, 1u);
}

// The chunks of all units of one key head, and where chunk `at` of them lies.  LDS: 260 words.  at >= total: only the total.
struct AtFound { u32 unit, off; };
__device__ __forceinline__ uint64_t at_total(const AttendArgs& p, uint64_t* lds, u32& mine0, uint64_t& before) {
    const u32 tid = threadIdx.x, q = ((u32)p.units + 255) / 256;
    mine0 = tid * q;
    uint64_t mine = 0;
    for (u32 i = 0; i < q; i++)
        if (mine0 + i < (u32)p.units) mine += at_unit_chunks(p, mine0 + i);
    // inclusive sums over the wavefront, then over the four
    uint64_t s = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)s, d, 64);
        if ((int)(tid & 63) >= d) s += o;
    }
    if ((tid & 63) == 63) lds[tid >> 6] = s;
    __syncthreads();
    uint64_t total = 0;
    before = s - mine;
    for (u32 w = 0; w < 4; w++) {
        if (w < tid >> 6) before += lds[w];
        total += lds[w];
    }
    __syncthreads();
    return total;
}
// Unit and chunk of place `at` (below the total), by the thread whose units hold it; every thread has them.
__device__ __forceinline__ AtFound at_find(const AttendArgs& p, uint64_t at, u32 mine0, uint64_t before, uint64_t total, uint64_t* lds) {
    const u32 q = ((u32)p.units + 255) / 256;
    u32* const out = (u32*)(lds + 4);
    if (at >= before && mine0 < (u32)p.units) {
        uint64_t b = before;
        for (u32 i = 0; i < q && mine0 + i < (u32)p.units; i++) {
            const u32 n = at_unit_chunks(p, mine0 + i);
            if (at < b + n) {
                out[0] = mine0 + i;
                out[1] = (u32)(at - b);
                break;
            }
            b += n;
        }
    }
    __syncthreads();
    AtFound f = {(u32)__builtin_amdgcn_readfirstlane((i32)out[0]), (u32)__builtin_amdgcn_readfirstlane((i32)out[1])};
    __syncthreads();
    return f;
}
__device__ __forceinline__ uint64_t at_first(const AttendArgs& p, uint64_t all, u32 w) { return all * w / (u32)p.wgs; }
// Workgroups that follow each other share an L2 (eight of them, blockIdx modulo 8): neighbours' units often read the same rows.
__device__ __forceinline__ u32 at_group_of(const AttendArgs& p) {
    const u32 b = blockIdx.x;
    return (p.wgs & 7) == 0 ? (b & 7) * ((u32)p.wgs >> 3) + (b >> 3) : b;
}

// ---- the pass --------------------------------------------------------------------

// A column's value written: c elements from d0 on.
template <int C> __device__ __forceinline__ void at_store(const AttendArgs& p, u32 t, u32 head, int d0, const float (&v)[C]) {
    const size_t at = t * p.out_stride + (size_t)head * p.c.d + d0;
#pragma unroll
    for (int i = 0; i < C; i += 4) {
        const f32x4 x = {v[i], v[i + 1], v[i + 2], v[i + 3]};
        if (p.out_vec) norm_store<true>(p.out, at + i, p.out_type, 4, x);
        else norm_store<false>(p.out, at + i, p.out_type, 4, x);
    }
}
// What a column's sums come to: 1 / (sum + sink), and lse.  m in units of log2, l times 2^OFF.
__device__ __forceinline__ float at_finish(const AttendArgs& p, u32 t, u32 head, float m, float l, float off, bool writes) {
    float scale = 1.f;
    if (l == 0.f) {   // nothing seen
        if (p.lse && writes) p.lse[(size_t)t * p.n_head + head] = p.sink ? p.sink[head] : -__builtin_inff();
        return 0.f;
    }
    if (p.sink) {
        const float s = p.sink[head] * JL_AT_LOG2E, top = fmaxf(m, s);
        if (top > -__builtin_inff()) {
            scale = __builtin_amdgcn_exp2f(m - top);          // (m of nothing: 0)
            l = l * scale + __builtin_amdgcn_exp2f(s - top + off);
            m = top;
        }
    }
    if (p.lse && writes) p.lse[(size_t)t * p.n_head + head] = (m + __builtin_amdgcn_logf(l) - off) * JL_AT_LN2;
    return scale / l;
}

// TYPE of the cache, DP the row's elements rounded up to 64, 128 or 256, QP pieces of q, NT column tiles of sixteen.
// LDS: floats [4][16][DP + 4], [4][16][2] and the search's words.
template <int TYPE, int DP, int QP, int NT>
__device__ __forceinline__ void attend_body(const AttendArgs& p, float* lds, uint64_t* find) {
    constexpr bool BF = TYPE == JL_BF16, I8 = TYPE == JL_I8;
    constexpr int C = DP / 16, KC = DP / 32, VW = I8 ? (C + 3) / 4 : C / 2;   // words of V a position and lane
    constexpr int ROW = DP + 4;
    constexpr float OFF = BF ? 0.f : 14.f;           // P times 2^14 in f16, whose smallest are 2^-24
    const float inf = __builtin_inff();
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const u32 w = at_group_of(p);

    u32 mine0;
    uint64_t before;
    const uint64_t total = at_total(p, find, mine0, before);
    const u32 planes = (u32)p.c.n_kv * (u32)p.blocks;
    const uint64_t all = total * planes, first = at_first(p, all, w), end = at_first(p, all, w + 1);
    if (first >= end) return;
    u32 plane = (u32)(first / total);
    AtFound f = at_find(p, first - plane * total, mine0, before, total, find);

    const size_t row_bytes = p.c.row_stride * (I8 ? 1 : 2);
    float* const ml = lds + 4 * 16 * ROW;

    for (uint64_t at = first; at < end;) {
        const u32 unit = f.unit, u_first = unit * (u32)p.per, u_last = min(u_first + (u32)p.per, (u32)p.ntok);
        const u32 n_chunks = at_unit_chunks(p, unit), c0 = f.off, c1 = (u32)min((uint64_t)n_chunks, c0 + (end - at));
        const u32 kv = plane / (u32)p.blocks, block = plane - kv * (u32)p.blocks;

        // the columns: token, head, what it sees
        u32 tok[NT], head[NT], clo[NT], chi[NT];
        bool col_live[NT];
        u32x4 qf[NT][QP][KC];
        float qs[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const u32 col = block * (16 * NT) + nt * 16 + n;
            const u32 r = p.per > 1 ? col / (u32)p.group : 0u, h = col - r * (u32)p.group;
            col_live[nt] = h < (u32)p.group && r < (u32)p.per && u_first + r < u_last;
            tok[nt] = u_first + (col_live[nt] ? r : 0u);
            head[nt] = kv * (u32)p.group + (col_live[nt] ? h : 0u);
            u32 seq;
            at_sees(p, tok[nt], seq, clo[nt], chi[nt]);
            const size_t q0 = tok[nt] * p.q_stride + (size_t)head[nt] * p.c.d;
            float x[KC][8];
            float most = 0.f;
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const int d = I8 ? 64 * (c / 2) + 16 * g + 8 * (c % 2) : 32 * c + 8 * g;
                f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
                if (col_live[nt] && d < p.c.d) kv_load8(p.q, q0 + d, p.q_type, true, a, b);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    x[c][j] = a[j];
                    x[c][j + 4] = b[j];
                    most = fmaxf(most, fmaxf(fabsf(a[j]), fabsf(b[j])));
                }
            }
            int e = 0;
            if (!BF) {   // into f16's range: the column's largest to [2^14, 2^15)
                most = at_max4(most);
                e = most > 0.f && most < inf ? 14 - __builtin_amdgcn_frexp_expf(most) + 1 : 0;
            }
            qs[nt] = __builtin_amdgcn_ldexpf(p.scale, -e);
            if (p.cap == 0.f) qs[nt] *= JL_AT_LOG2E;
            else qs[nt] /= p.cap;
#pragma unroll
            for (int c = 0; c < KC; c++) {
#pragma unroll
                for (int j = 0; j < 8; j++) x[c][j] = __builtin_amdgcn_ldexpf(x[c][j], e);
#pragma unroll
                for (int k = 0; k < QP; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++) qf[nt][k][c][j] = at_piece<BF>(x[c][2 * j], x[c][2 * j + 1]);
            }
        }

        f32x4 acc[NT][C];
        float m[NT], l[NT];
        int ve = -200;          // 8-bit rows: acc is times 2^-ve
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt] = -inf;
            l[nt] = 0.f;
#pragma unroll
            for (int j = 0; j < C; j++) acc[nt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        u32 skip = c0, left = c1 - c0;
        for (u32 t = u_first; t < u_last && left;) {
            const AtRun run = at_run(p, t, u_last);
            t = run.end;
            u32 nc = at_chunks(run.lo, run.hi);
            if (skip >= nc) {
                skip -= nc;
                continue;
            }
            const u32 k0 = run.lo / JL_AT_CHUNK + skip;
            nc = min(nc - skip, left);
            skip = 0;
            left -= nc;
            const u32* const pages = p.c.table + (size_t)run.seq * p.c.table_stride;
            for (u32 k = k0; k < k0 + nc; k++) {
                const u32 p0 = k * JL_AT_CHUNK + wave * 32;
                if (p0 >= run.hi || p0 + 32 <= run.lo) continue;
                // pages of the two tiles; a tile on no page is hidden
                bool there[2];
                const char *kb[2], *vb[2];
                size_t sb[2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const u32 at0 = p0 + 16 * i;
                    u32 page = at0 < run.hi ? pages[at0 >> p.c.shift] : p.c.n_page;
                    there[i] = page < p.c.n_page;
                    page = there[i] ? page : 0u;
                    const u32 slot = at0 & ((1u << p.c.shift) - 1);
                    const size_t o = (page * p.c.page_stride + kv * p.c.head_stride) * (I8 ? 1 : 2) + slot * row_bytes;
                    kb[i] = (const char*)p.c.k + o;
                    vb[i] = (const char*)p.c.v + o;
                    sb[i] = (((size_t)page * p.c.n_kv + kv) << p.c.shift) + slot;
                }
                const bool edge = !(p0 >= run.lo_all && p0 + 32 <= run.hi_all && there[0] && there[1]) || run.t != u_first || run.end != u_last;
                u32x4 kf[2][I8 ? KC / 2 : KC];
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int c = 0; c < (I8 ? KC / 2 : KC); c++) {
                        const int d = I8 ? 64 * c + 16 * g : 32 * c + 8 * g;
                        kf[i][c] = u32x4{0, 0, 0, 0};
                        if (d < p.c.d) kf[i][c] = *(const u32x4*)(kb[i] + n * row_bytes + (I8 ? d : 2 * d));
                    }
                u32 vw[8][VW];
#pragma unroll
                for (int r = 0; r < 8; r++) {
                    const int i = r / 4;
#pragma unroll
                    for (int x = 0; x < VW; x++) vw[r][x] = 0;
                    const u32 at0 = p0 + 16 * i + 4 * g + r % 4;
                    if (C * n < p.c.d && (!edge || (there[i] && at0 >= run.lo && at0 < run.hi))) {
                        const char* const src = vb[i] + (4 * g + r % 4) * row_bytes + C * n * (I8 ? 1 : 2);
                        if constexpr (VW == 1) vw[r][0] = *(const u32*)src;
                        else if constexpr (VW == 2) {
                            const u32x2 y = *(const u32x2*)src;
                            vw[r][0] = y.x; vw[r][1] = y.y;
                        } else {
#pragma unroll
                            for (int x = 0; x < VW; x += 4) {
                                const u32x4 y = *(const u32x4*)(src + 4 * x);
                                vw[r][x] = y.x; vw[r][x + 1] = y.y; vw[r][x + 2] = y.z; vw[r][x + 3] = y.w;
                            }
                        }
                    }
                }
                f32x4 ks[2], vs[2];
                if constexpr (I8) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        ks[i] = *(const f32x4*)(p.c.k_scale + sb[i] + 4 * g);
                        vs[i] = *(const f32x4*)(p.c.v_scale + sb[i] + 4 * g);
                        if (edge) {
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const u32 at0 = p0 + 16 * i + 4 * g + r;
                                if (!(there[i] && at0 >= run.lo && at0 < run.hi)) vs[i][r] = 0.f;
                            }
                        }
                    }
                    // the running power of two over the values' scales
                    float most = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) most = fmaxf(most, vs[i][r]);
                    most = at_max4(most);
                    const int e = most > 0.f ? __builtin_amdgcn_frexp_expf(most) : -200;
                    if (__builtin_amdgcn_readfirstlane(e) > ve) {
                        const int to = __builtin_amdgcn_readfirstlane(e);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int j = 0; j < C; j++)
#pragma unroll
                                for (int r = 0; r < 4; r++) acc[nt][j][r] = __builtin_amdgcn_ldexpf(acc[nt][j][r], ve - to);
                        ve = to;
                    }
                }

                f32x4 s[NT][2];
#pragma unroll
                for (int i = 0; i < 2; i++) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) s[nt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < KC; c++) {
                        u32x4 kx;
                        if constexpr (I8) {   // bytes b to f16: 0x6400 | (b + 128) is 1152 + b
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const u32 src = kf[i][c / 2][2 * (c % 2) + j / 2];
                                const u32 t2 = __builtin_amdgcn_perm(0u, src, j % 2 ? 0x0c030c02u : 0x0c010c00u) ^ 0x64806480u;
                                const f16x2 y = __builtin_bit_cast(f16x2, t2) - f16x2{(_Float16)1152, (_Float16)1152};
                                kx[j] = __builtin_bit_cast(u32, y);
                            }
                        } else {
                            kx = kf[i][c];
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int k = 0; k < QP; k++) s[nt][i] = at_mfma<BF>(kx, qf[nt][k][c], s[nt][i]);
                    }
                }

                u32x4 pf[NT][3];
                const int pieces = BF && p.out_type == JL_F32 ? 3 : 2;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float x[8];
                    u32 hidden = 0;
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            float y = s[nt][i][r] * qs[nt];
                            if constexpr (I8) y *= ks[i][r];
                            if (p.cap != 0.f) y = p.cap * JL_AT_LOG2E * at_tanh(y);
                            if (edge) {
                                const u32 at0 = p0 + 16 * i + 4 * g + r;
                                const bool sees = there[i] && tok[nt] >= run.t && tok[nt] < run.end && at0 >= clo[nt] && at0 < chi[nt];
                                y = sees ? y : -inf;
                                hidden |= sees ? 0u : 1u << (4 * i + r);
                            }
                            x[4 * i + r] = y;
                        }
                    float top = x[0];
#pragma unroll
                    for (int j = 1; j < 8; j++) top = fmaxf(top, x[j]);
                    top = fmaxf(at_max4(top), m[nt]);
                    if (__ballot(top > m[nt])) {
                        const float turn = m[nt] == top ? 1.f : __builtin_amdgcn_exp2f(m[nt] - top);   // (from -inf: 0)
                        l[nt] *= turn;
#pragma unroll
                        for (int j = 0; j < C; j++) acc[nt][j] *= turn;
                        m[nt] = top;
                    }
                    const float base = (m[nt] > -inf ? m[nt] : 0.f) - OFF;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        x[j] = __builtin_amdgcn_exp2f(x[j] - base);
                        l[nt] += x[j];
                    }
                    if constexpr (I8) {
#pragma unroll
                        for (int j = 0; j < 8; j++) x[j] = hidden >> j & 1 ? 0.f : x[j] * __builtin_amdgcn_ldexpf(vs[j / 4][j % 4], -ve);   // (a hidden scale may be no number)
                    }
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        if (k < pieces)
#pragma unroll
                            for (int j = 0; j < 4; j++) pf[nt][k][j] = at_piece<BF>(x[2 * j], x[2 * j + 1]);
                }

                // positions that only some tokens of the run see, and a value among them that is no number: 0 * NaN would reach the others
                bool apart = false;
                if (!I8 && edge && run.end - run.t > 1 && (p0 < run.lo_all || p0 + 32 > run.hi_all)) {
                    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                    u16x2 big = {0, 0};
#pragma unroll
                    for (int r = 0; r < 8; r++)
#pragma unroll
                        for (int x = 0; x < VW; x++) big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2, vw[r][x] & 0x7fff7fffu));
                    const bool odd = max(big.x, big.y) >= (BF ? 0x7f80 : 0x7c00);
                    apart = __ballot(odd) != 0;
                }
                auto turned = [&](int j, u32 rows) {   // values' fragment j of the lane's positions that are in `rows`
                    u32x4 vt;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if constexpr (I8) {
                            const u32 b = j % 4;
                            const u32 t2 = __builtin_amdgcn_perm(vw[2 * r + 1][j / 4], vw[2 * r][j / 4], 0x0c000c00u | b | (4 + b) << 16) ^ 0x64806480u;
                            const f16x2 y = __builtin_bit_cast(f16x2, t2) - f16x2{(_Float16)1152, (_Float16)1152};
                            vt[r] = __builtin_bit_cast(u32, y);
                        } else {
                            vt[r] = __builtin_amdgcn_perm(vw[2 * r + 1][j / 2], vw[2 * r][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
                        }
                        if (rows != 0xffu) vt[r] &= (rows >> 2 * r & 1 ? 0xffffu : 0u) | (rows >> 2 * r & 2 ? 0xffff0000u : 0u);
                    }
                    return vt;
                };
                auto product = [&](u32x4 vt, int nt, f32x4 to) {
                    to = at_mfma<BF>(vt, pf[nt][0], to);
                    to = at_mfma<BF>(vt, pf[nt][1], to);
                    if constexpr (BF)
                        if (pieces == 3) to = at_mfma<BF>(vt, pf[nt][2], to);
                    return to;
                };
                if (!apart) {
#pragma unroll
                    for (int j = 0; j < C; j++) {
                        const u32x4 vt = turned(j, 0xffu);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) acc[nt][j] = product(vt, nt, acc[nt][j]);
                    }
                } else {
                    for (u32 tt = run.t; tt < run.end; tt++) {
                        u32 seq, lo, hi, rows = 0;
                        at_sees(p, tt, seq, lo, hi);
#pragma unroll
                        for (int r = 0; r < 8; r++) {
                            const u32 at0 = p0 + 16 * (r / 4) + 4 * g + r % 4;
                            if (at0 >= lo && at0 < hi) rows |= 1u << r;
                        }
#pragma unroll
                        for (int j = 0; j < C; j++) {
                            const u32x4 vt = turned(j, rows | 0x100u);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const f32x4 y = product(vt, nt, f32x4{0.f, 0.f, 0.f, 0.f});
                                if (tok[nt] == tt) acc[nt][j] += y;
                            }
                        }
                    }
                }
            }
        }

        // the four wavefronts' sums to one
        const bool whole = c0 == 0 && c1 == n_chunks;
        const u32 slot = 2 * w + (at == first ? 0u : 1u);
        float* const part = p.part + (size_t)slot * (16 * NT) * (DP + 2);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const float sum = at_sum4(l[nt]);
            __syncthreads();
            if (g == 0) {
                ml[(wave * 16 + n) * 2] = m[nt];
                ml[(wave * 16 + n) * 2 + 1] = sum;
            }
            __syncthreads();
            float top = -inf, lsum = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) top = fmaxf(top, ml[(k * 16 + n) * 2]);
            float turn = m[nt] == top ? 1.f : __builtin_amdgcn_exp2f(m[nt] - top);   // (a wavefront that saw nothing: exp2(-inf), its sums are 0)
            if constexpr (I8) turn = __builtin_amdgcn_ldexpf(turn, ve);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < C; j += 4) {
                    const f32x4 y = {acc[nt][j][i] * turn, acc[nt][j + 1][i] * turn, acc[nt][j + 2][i] * turn, acc[nt][j + 3][i] * turn};
                    *(f32x4*)(lds + (wave * 16 + n) * ROW + C * (4 * g + i) + j) = y;
                }
            __syncthreads();
            // thread: column tid / 16, C elements
            const int col = threadIdx.x >> 4, d0 = C * (threadIdx.x & 15);
            float mm = -inf;
#pragma unroll
            for (int k = 0; k < 4; k++) mm = fmaxf(mm, ml[(k * 16 + col) * 2]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float mk = ml[(k * 16 + col) * 2];
                lsum += ml[(k * 16 + col) * 2 + 1] * (mk == mm ? 1.f : __builtin_amdgcn_exp2f(mk - mm));
            }
            float y[C];
#pragma unroll
            for (int i = 0; i < C; i++) {
                y[i] = 0.f;
#pragma unroll
                for (int k = 0; k < 4; k++) y[i] += lds[(k * 16 + col) * ROW + d0 + i];
            }
            if (whole) {
                const u32 cc = block * (16 * NT) + nt * 16 + col;
                const u32 r = p.per > 1 ? cc / (u32)p.group : 0u, h = cc - r * (u32)p.group;
                if (h < (u32)p.group && r < (u32)p.per && u_first + r < u_last) {
                    const float inv = at_finish(p, u_first + r, kv * (u32)p.group + h, mm, lsum, OFF, d0 == 0);
#pragma unroll
                    for (int i = 0; i < C; i++) y[i] *= inv;
                    if (d0 < p.c.d) at_store<C>(p, u_first + r, kv * (u32)p.group + h, d0, y);
                }
            } else {
                float* const to = part + (nt * 16 + col) * (DP + 2);
                if (d0 == 0) {
                    to[DP] = mm;
                    to[DP + 1] = lsum;
                }
#pragma unroll
                for (int i = 0; i < C; i++) to[d0 + i] = y[i];
            }
        }
        at += c1 - c0;
        f.off = 0;
        f.unit = unit + 1;
        if (f.unit == (u32)p.units) {
            f.unit = 0;
            plane++;
        }
    }
}

// The partial sums of a unit that several workgroups had, added up by one: that of the first of them.  grid = wgs, block = 256.
template <int DP, int NT> __device__ __forceinline__ void attend_join_body(const AttendArgs& p, uint64_t* find) {
    constexpr int C = DP / 16;
    const float inf = __builtin_inff(), off = p.c.type == JL_BF16 ? 0.f : 14.f;
    const u32 w = blockIdx.x;
    u32 mine0;
    uint64_t before;
    const uint64_t total = at_total(p, find, mine0, before);
    const u32 planes = (u32)p.c.n_kv * (u32)p.blocks;
    const uint64_t all = total * planes, first = at_first(p, all, w), end = at_first(p, all, w + 1);
    if (first >= end) return;
    const u32 plane = (u32)((end - 1) / total);
    const AtFound f = at_find(p, end - 1 - plane * total, mine0, before, total, find);
    const uint64_t u0 = end - 1 - f.off, u1 = u0 + at_unit_chunks(p, f.unit);
    if (u1 <= end || u0 < first) return;   // ends here, or began earlier
    const u32 kv = plane / (u32)p.blocks, block = plane - kv * (u32)p.blocks, u_first = f.unit * (u32)p.per, u_last = min(u_first + (u32)p.per, (u32)p.ntok);
    u32 last = w + 1;
    while (at_first(p, all, last) < u1) last++;   // [w, last)
    const size_t stride = (size_t)2 * (16 * NT) * (DP + 2);
    const int d0 = C * (threadIdx.x & 15);
    for (int nt = 0; nt < NT; nt++) {
        const int col = threadIdx.x >> 4;
        const u32 cc = block * (16 * NT) + nt * 16 + col;
        const u32 r = p.per > 1 ? cc / (u32)p.group : 0u, h = cc - r * (u32)p.group;
        if (!(h < (u32)p.group && r < (u32)p.per && u_first + r < u_last)) continue;
        const float* const mine = p.part + (nt * 16 + col) * (DP + 2);
        auto of = [&](u32 k) { return mine + k * stride + (k == w && u0 != first ? stride / 2 : 0); };
        float mm = -inf, l = 0.f, y[C];
        for (u32 k = w; k < last; k++)
            if (at_first(p, all, k) < at_first(p, all, k + 1)) mm = fmaxf(mm, of(k)[DP]);
#pragma unroll
        for (int i = 0; i < C; i++) y[i] = 0.f;
        for (u32 k = w; k < last; k++) {
            if (at_first(p, all, k) == at_first(p, all, k + 1)) continue;
            const float* const a = of(k);
            const float turn = a[DP] == mm ? 1.f : __builtin_amdgcn_exp2f(a[DP] - mm);
            l += a[DP + 1] * turn;
#pragma unroll
            for (int i = 0; i < C; i++) y[i] += a[d0 + i] * turn;
        }
        const float inv = at_finish(p, u_first + r, kv * (u32)p.group + h, mm, l, off, d0 == 0);
#pragma unroll
        for (int i = 0; i < C; i++) y[i] *= inv;
        if (d0 < p.c.d) at_store<C>(p, u_first + r, kv * (u32)p.group + h, d0, y);
    }
}
