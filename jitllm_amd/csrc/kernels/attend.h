// Attention of new tokens over a paged cache (jl_attend_dev).  Token t of sequence s sees the positions lo = max(0, len - window) to
// hi = len of s; for each of its heads
//
//   s_p = scale * (q . k_p), or cap * tanh(scale * (q . k_p) / cap);   w_p = e^(s_p - m);   out = sum w_p v_p / (sum w_p + e^(sink - m))
//
// in one pass with a running maximum m.  A token and a head are a COLUMN: the `group` heads that share a key head, and of several tokens of one sequence
// `per` (a UNIT), meet the same rows.  On the matrix cores, 16x16x32, sixteen columns a tile:
//
//   S^T = K Q^T: a lane (n = lane & 15, g = lane >> 4) holds of column n the scores of positions 4g..4g+3 of each tile of sixteen.
//   O^T = V^T P^T: k runs over 32 positions, slot (g, j) being position 4g + j of the first tile for j < 4 and of the second behind it,
//     which is where S^T left them: P goes from one product to the next without leaving its lane.
//   V lies [position][d]; a lane takes its eight positions' rows, c = DP / 16 elements each from d = c n on (a row of 16 lanes is whole), and
//     turns them into the c fragments of eight positions each by byte permutes: fragment j holds d = c n + j.
//   A column's m, sum and O stay in the four lanes of its n: the running maximum is two lane swaps, rescaling is in-lane.
//
// Precision: K and V are exact in the instruction's type (8-bit rows as f16 integers, their scale applied to S, and to P relative to a running power of two over the scales that the column sees); q and
// P are split into pieces that hold 22 (f16) or 24 and 16 or 24 (bf16) bits, so what rounds is the f32 sums, as in a plain product in f32.
//
// Two forms.  attend_one.h: up to sixteen columns, a workgroup's wavefronts take 32 positions each, bound by bytes.  attend_many.h: the wavefronts take columns each and
// share the rows through LDS, bound by the matrix and vector units.  Work is cut in chunks of 128 positions, and the workgroups share the chunks of all
// units and key heads evenly whatever their lengths, each a contiguous run of them; what ends up with more than one leaves partial sums that attend_join adds up.  Where
// units are many or short each is a workgroup's as it is, and nothing is joined.
#pragma once
#include "args.h"
#include "common.h"
#include "kv_cache.h"

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 at_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The running maximum stays until a score is more than SLACK (of log2) over it: most steps then rescale nothing.  P is times 2^OFF in f16, whose smallest
// are 2^-24 and whose largest 2^16.
#define JL_AT_OFF 13.f
#define JL_AT_SLACK(BF) ((BF) ? 8.f : 2.875f)
#define JL_AT_CHUNK 128      // positions a workgroup's step
#define JL_AT_LOG2E 1.4426950408889634f
#define JL_AT_LN2 0.6931471805599453f

template <bool BF> __device__ __forceinline__ f32x4 at_mfma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(at_bf16x8, a), __builtin_bit_cast(at_bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(at_f16x8, a), __builtin_bit_cast(at_f16x8, b), c, 0, 0, 0);
}
// Two values in the type's bits, to nearest even, and what that leaves of them: of those very bits.  (Left to itself the compiler converts the values again for the
// difference; where a value is a product, once from the product as it was rounded and once by an instruction that multiplies and converts: now and then the two are a
// step apart, and a weight over 8-bit rows was off by 2^-11 of itself.)
template <bool BF> __device__ __forceinline__ u32 at_piece(float& x, float& y) {
    if constexpr (BF) {
        const at_bf16x2 h = {(__bf16)x, (__bf16)y};
        u32 b = __builtin_bit_cast(u32, h);
        asm("" : "+v"(b));
        x -= __uint_as_float(b << 16);
        y -= __uint_as_float(b & 0xffff0000u);
        return b;
    } else {
        u32 b = __builtin_bit_cast(u32, f16x2{(_Float16)x, (_Float16)y});
        asm("" : "+v"(b));
        const f16x2 h = __builtin_bit_cast(f16x2, b);
        x -= (float)h.x;
        y -= (float)h.y;
        return b;
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

template <int CTRL> __device__ __forceinline__ float dpp_f32_max(float v) { return __builtin_bit_cast(float, dpp_i32<CTRL, 0xf>(0, __builtin_bit_cast(i32, v))); }
// tanh: the series up to 0.3 (the next term is under 2^-24 of the sum there, where 1 - 2 / (e^2y + 1) cancels), the exponential's form beyond.
__device__ __forceinline__ float at_tanh(float y) {
    const float z = y * y;
    const float small = y + y * z * (-1.f / 3.f + z * (2.f / 15.f + z * (-17.f / 315.f + z * (62.f / 2835.f))));
    const float large = 1.f - 2.f / (__builtin_amdgcn_exp2f(2.f * JL_AT_LOG2E * y) + 1.f);
    return z < 0.09f ? small : large;
}

// ---- which positions, units and chunks -----------------------------------------

__device__ __forceinline__ void at_sees(const AttendArgs& p, u32 t, u32& seq, u32& lo, u32& hi) {
    const u32 n = p.len[t];      // (both loads on their way together)
    seq = p.seq ? p.seq[t] : t;
    hi = seq < p.c.n_seq ? min(n, p.c.table_pages << p.c.shift) : 0u;      // (2^31 positions at most)
    lo = p.window && hi > (u32)p.window ? hi - (u32)p.window : 0u;
}
// Chunks of what is seen, one at least: a token that sees nothing has its zeros written.
__device__ __forceinline__ u32 at_chunks(u32 lo, u32 hi) { return hi > lo ? ((hi - 1) / JL_AT_CHUNK) - lo / JL_AT_CHUNK + 1 : 1u; }

// Tokens t0 to t1 of one sequence that share a pass: those of a unit that follow each other.
struct AtSpan {
    u32 t0, t1, seq, lo, hi;     // [lo, hi): seen by one of them
    u32 lo_all, hi_all;          // [lo_all, hi_all): by all
};
__device__ __forceinline__ u32 at_uni(u32 v) { return (u32)__builtin_amdgcn_readfirstlane((i32)v); }
// The span that begins at t, by a whole wavefront.
template <bool MANY> __device__ __forceinline__ AtSpan at_span(const AttendArgs& p, u32 t) {
    AtSpan s;
    s.t0 = t;
    s.t1 = t + 1;
    if (!MANY) {
        at_sees(p, t, s.seq, s.lo, s.hi);
        s.seq = at_uni(s.seq); s.lo = at_uni(s.lo); s.hi = at_uni(s.hi);
        s.lo_all = s.lo; s.hi_all = s.hi;
        return s;
    }
    const u32 end = min((t / (u32)p.per + 1) * (u32)p.per, (u32)p.ntok), lane = threadIdx.x & 63;
    s.lo = s.hi_all = ~0u;
    s.hi = s.lo_all = 0;
    for (u32 at = t; at < end; at += 64) {     // (uniform)
        u32 seq, lo, hi;
        at_sees(p, min(at + lane, end - 1), seq, lo, hi);
        if (at == t) s.seq = at_uni(seq);
        const uint64_t others = __ballot(seq != s.seq || at + lane >= end);
        const u32 n = others ? (u32)__builtin_ctzll(others) : 64u;
        if (lane < n) {
            s.lo = min(s.lo, lo); s.hi = max(s.hi, hi); s.lo_all = max(s.lo_all, lo); s.hi_all = min(s.hi_all, hi);
        }
        s.t1 = at + n;
        if (n < 64) break;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        s.lo = min(s.lo, (u32)__shfl_xor((int)s.lo, d, 64)); s.hi = max(s.hi, (u32)__shfl_xor((int)s.hi, d, 64));
        s.lo_all = max(s.lo_all, (u32)__shfl_xor((int)s.lo_all, d, 64)); s.hi_all = min(s.hi_all, (u32)__shfl_xor((int)s.hi_all, d, 64));
    }
    s.t1 = at_uni(s.t1);
    s.lo = at_uni(s.lo); s.hi = at_uni(s.hi); s.lo_all = at_uni(s.lo_all); s.hi_all = at_uni(s.hi_all);
    return s;
}
// The chunks of a unit's spans, by one thread.
template <bool MANY> __device__ __forceinline__ u32 at_unit_chunks(const AttendArgs& p, u32 unit) {
    u32 seq0, lo, hi;
    const u32 t0 = unit * (u32)p.per, end = min(t0 + (u32)p.per, (u32)p.ntok);
    at_sees(p, t0, seq0, lo, hi);
    u32 sum = 0;
    if (MANY) {
#pragma unroll 1
        for (u32 t = t0 + 1; t < end; t += 4) {
            u32 seq[4], l[4], h[4];
#pragma unroll
            for (u32 i = 0; i < 4; i++) at_sees(p, min(t + i, end - 1), seq[i], l[i], h[i]);     // (the last again changes nothing)
#pragma unroll
            for (u32 i = 0; i < 4; i++) {
                const bool more = seq[i] == seq0;
                sum += more ? 0u : at_chunks(lo, hi);
                lo = more ? min(lo, l[i]) : l[i];
                hi = more ? max(hi, h[i]) : h[i];
                seq0 = seq[i];
            }
        }
    }
    return sum + at_chunks(lo, hi);
}

// The workgroups' shares of all chunks: q each, one more for the first r.
struct AtShare {
    uint64_t q;
    u32 r, n;      // of n workgroups that have any
    __device__ uint64_t first(u32 w) const { return q * w + min(w, r); }
    __device__ u32 holder(uint64_t at) const {   // of chunk `at`
        const uint64_t big = (q + 1) * r;
        if ((q >> 31) == 0 && (at >> 32) == 0) return at < big ? (u32)at / ((u32)q + 1) : r + (u32)(at - big) / max((u32)q, 1u);
        return (u32)(at < big ? at / (q + 1) : r + (at - big) / q);
    }
};
__device__ __forceinline__ AtShare at_share(uint64_t all, u32 wgs) {
    AtShare s;
    s.n = (u32)min((uint64_t)wgs, all);
    s.q = (all >> 32) == 0 ? (u32)all / s.n : all / s.n;
    s.r = (u32)(all - s.q * s.n);
    return s;
}
// Workgroups that follow each other share an L2 (eight of them, blockIdx modulo 8): neighbours' units often read the same rows.
__device__ __forceinline__ u32 at_group_of(u32 b, u32 wgs) { return (wgs & 7) == 0 ? (b & 7) * (wgs >> 3) + (b >> 3) : b; }

// Sums over the workgroup's WAVES wavefronts: before this thread, and all.  LDS: WAVES words of 8 bytes.
template <int WAVES> __device__ __forceinline__ uint64_t at_before(uint64_t mine, uint64_t* lds, uint64_t& total) {
    const u32 tid = threadIdx.x;
    uint64_t s = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)s, d, 64);
        if ((int)(tid & 63) >= d) s += o;
    }
    if ((tid & 63) == 63) lds[tid >> 6] = s;
    __syncthreads();
    uint64_t before = s - mine;
    total = 0;
#pragma unroll
    for (u32 w = 0; w < WAVES; w++) {
        before += w < tid >> 6 ? lds[w] : 0;
        total += lds[w];
    }
    return before;
}

// A workgroup's share: chunks first to end of all, and where the first lies.  LDS: WAVES + 1 words of 8 bytes.  False: none (the whole workgroup alike).
struct AtWork {
    uint64_t first, end;
    AtShare share;
    u32 plane, tok, off;      // its unit's first token (later: the next span's), and the unit's chunks that are before it
};
template <bool MANY, int WAVES> __device__ __forceinline__ bool at_work(const AttendArgs& p, u32 w, uint64_t* lds, AtWork& k) {
    u32* const told = (u32*)(lds + WAVES);
    const u32 q = ((u32)p.units + 255) / 256, mine0 = threadIdx.x * q;
    uint64_t mine = 0, total, before = 0, at = 0;
    // twice: the sums, and the unit that has the first chunk, by the thread whose units have it
#pragma unroll 1
    for (int pass = 0; pass < 2; pass++) {
        if (pass == 0 || (at >= before && at < before + mine)) {
            uint64_t b = before;
#pragma unroll 1
            for (u32 i = 0; i < q; i++) {
                if (mine0 + i >= (u32)p.units) break;
                const u32 c = at_unit_chunks<MANY>(p, mine0 + i);
                if (pass && at >= b && at < b + c) {
                    told[0] = mine0 + i;
                    told[1] = (u32)(at - b);
                }
                b += c;
            }
            if (pass == 0) mine = b;
        }
        if (pass) break;
        before = at_before<WAVES>(mine, lds, total);
        const u32 planes = (u32)p.c.n_kv * (u32)p.blocks;
        k.share = at_share(total * planes, (u32)p.wgs);
        if (w >= k.share.n) return false;
        k.first = k.share.first(w);
        k.end = k.share.first(w + 1);
        k.plane = at_uni(planes == 1 ? 0u : (k.first >> 32) == 0 && (total >> 32) == 0 ? (u32)k.first / (u32)total : (u32)(k.first / total));
        at = k.first - k.plane * total;
        if (q == 1) {
            if (at >= before && at < before + mine) {
                told[0] = mine0;
                told[1] = (u32)(at - before);
            }
            break;
        }
    }
    __syncthreads();
    k.off = at_uni(told[1]);
    k.tok = at_uni(told[0]) * (u32)p.per;
    return true;
}

// Partial sums: [2 wgs][columns][DP], then [2 wgs][columns][2] of m and l, then a workgroup's word: what it is the first to have a part of.
struct AtJoin { u32 t0, t1, plane, last, slot, pad[3]; };   // last 0: none; else one more than the last workgroup that has a part of it
template <int DP> __device__ __forceinline__ float* at_part(const AttendArgs& p, u32 slot, u32 col) { return p.part + ((size_t)slot * p.part_cols + col) * DP; }
template <int DP> __device__ __forceinline__ f32x2* at_part_ml(const AttendArgs& p, u32 slot, u32 col) {
    return (f32x2*)(p.part + (size_t)2 * p.wgs * p.part_cols * DP) + (size_t)slot * p.part_cols + col;
}
template <int DP> __device__ __forceinline__ AtJoin* at_join_of(const AttendArgs& p) { return (AtJoin*)(p.part + (size_t)2 * p.wgs * p.part_cols * (DP + 2)); }

// Column `col` of a span and block: its token and head.  Heads of a token follow each other.
__device__ __forceinline__ bool at_column(const AttendArgs& p, u32 t0, u32 t1, u32 plane, u32 col, u32& tok, u32& head) {
    u32 kv = plane, h = col, r = 0;
    if (p.blocks > 1) {          // (a token a unit)
        kv = plane / (u32)p.blocks;
        h += (plane - kv * (u32)p.blocks) * (u32)p.part_cols;
    } else if (p.per > 1) {
        r = (u32)(((uint64_t)col * (u32)p.inv_group) >> 16);     // col / group, for columns below 256
        h = col - r * (u32)p.group;
    }
    const bool live = h < (u32)p.group && t0 + r < t1;
    tok = t0 + (live ? r : 0u);
    head = kv * (u32)p.group + (live ? h : 0u);
    return live;
}

typedef __amdgpu_buffer_rsrc_t at_rsrc;
__device__ __forceinline__ at_rsrc at_buffer(const void* p) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000); }
#define JL_AT_NOWHERE 0x7fffffff      // an offset behind every buffer: reads zeros

// C elements of a column written.
template <int C> __device__ __forceinline__ void at_store(const AttendArgs& p, u32 t, u32 head, int d0, const float (&v)[C]) {
    const size_t at = t * p.out_stride + (size_t)head * p.c.d + d0;
    if (p.out_type == JL_F32) {
        float* const out = (float*)p.out + at;
        if (p.out_vec) {
#pragma unroll
            for (int i = 0; i < C; i += 4) *(f32x4*)(out + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < C; i++) out[i] = v[i];
        }
        return;
    }
    uint16_t* const out = (uint16_t*)p.out + at;
    u32 b[C / 2];
    if (p.out_type == JL_F16) {
#pragma unroll
        for (int i = 0; i < C / 2; i++) b[i] = __builtin_bit_cast(u32, f16x2{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
    } else {
#pragma unroll
        for (int i = 0; i < C / 2; i++) b[i] = __builtin_bit_cast(u32, at_bf16x2{(__bf16)v[2 * i], (__bf16)v[2 * i + 1]});
    }
    if (p.out_vec) {
#pragma unroll
        for (int i = 0; i < C / 2; i += 2) *(u32x2*)(out + 2 * i) = u32x2{b[i], b[i + 1]};
    } else {
#pragma unroll
        for (int i = 0; i < C; i++) out[i] = (uint16_t)(b[i / 2] >> 16 * (i % 2));
    }
}
// A column's q, a lane's eight elements of each piece of 32 (asked for ahead of the rows, which come behind it); then in QP pieces, as the matrix instruction takes
// them, and what its scores are times.
template <bool I8, int KC> __device__ __forceinline__ void at_load_query(const AttendArgs& p, bool live, u32 tok, u32 head, float (&x)[KC][8]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int c = 0; c < KC; c++) {
        const int d = I8 ? 64 * (c / 2) + 16 * g + 8 * (c % 2) : 32 * c + 8 * g;
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (live && d < p.c.d) kv_load8(p.q, tok * p.q_stride + (size_t)head * p.c.d + d, p.q_type, true, a, b);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[c][j] = a[j];
            x[c][j + 4] = b[j];
        }
    }
}
template <bool BF, int QP, int KC>
__device__ __forceinline__ void at_query(const AttendArgs& p, float (&x)[KC][8], u32x4 (&qf)[QP][KC], float& qs) {
    float most = 0.f;
    int e = 0;
    if (!BF) {   // into f16's range: the column's largest to [2^14, 2^15)
#pragma unroll
        for (int c = 0; c < KC; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(x[c][j]));
        most = at_max4(most);
        e = most > 0.f && most < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(most) : 0;
    }
    qs = __builtin_amdgcn_ldexpf(fabsf(p.scale), -e);    // (a negative scale's sign goes to q: the largest score is the largest product)
    qs = p.cap == 0.f ? qs * JL_AT_LOG2E : qs / p.cap;
    const u32 sign = __float_as_uint(p.scale) & 0x80000000u;
#pragma unroll
    for (int c = 0; c < KC; c++) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[c][j] = __uint_as_float(__float_as_uint(BF ? x[c][j] : __builtin_amdgcn_ldexpf(x[c][j], e)) ^ sign);
#pragma unroll
        for (int k = 0; k < QP; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) qf[k][c][j] = at_piece<BF>(x[c][2 * j], x[c][2 * j + 1]);
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

// ---- partial sums joined ------------------------------------------------------------

// grid = (wgs, columns), block = 256: a column's parts by sixteen groups of lanes.  (Four columns a workgroup, a wavefront every fourth part: 12.5 us for 7.4 where 64
// parts a key head are joined, 7.7 for 5.6 with 8 parts of rows of 256.)  LDS: floats [4][DP], [4].
template <int DP> __device__ __forceinline__ void attend_join_body(const AttendArgs& p, float* lds) {
    constexpr int C = DP / 16;
    const u32 w = blockIdx.x;
    const AtJoin j = at_join_of<DP>(p)[w];
    if (j.last == 0) return;
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane >> 4, x = lane & 15, d0 = C * x, col = blockIdx.y;
    u32 tok, head;
    if (!at_column(p, j.t0, j.t1, j.plane, col, tok, head)) return;      // (the whole workgroup)
    const float off = p.c.type == JL_BF16 ? 0.f : JL_AT_OFF;
    auto slot = [&](u32 k) { return k == w ? j.slot : 2 * k; };
    float mm = -__builtin_inff(), l = 0.f;
    f32x4 y[C / 4];
#pragma unroll
    for (int i = 0; i < C / 4; i++) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (u32 k = w + lane; k < j.last; k += 64) mm = fmaxf(mm, (*at_part_ml<DP>(p, slot(k), col)).x);
    mm = fmaxf(mm, dpp_f32_max<JL_DPP_QUAD_XOR1>(mm));
    mm = fmaxf(mm, dpp_f32_max<JL_DPP_QUAD_XOR2>(mm));
    mm = fmaxf(mm, dpp_f32_max<JL_DPP_ROW_HALF_MIRROR>(mm));
    mm = fmaxf(mm, dpp_f32_max<JL_DPP_ROW_MIRROR>(mm));
    mm = at_max4(mm);
#pragma unroll 4
    for (u32 k = w + 4 * wave + c; k < j.last; k += 16) {
        const f32x2 ml = *at_part_ml<DP>(p, slot(k), col);
        const float turn = ml.x == mm ? 1.f : __builtin_amdgcn_exp2f(ml.x - mm);
        l += ml.y * turn;
#pragma unroll
        for (int i = 0; i < C / 4; i++) y[i] += *(const f32x4*)(at_part<DP>(p, slot(k), col) + d0 + 4 * i) * turn;
    }
    l = at_sum4(l);
#pragma unroll
    for (int i = 0; i < C / 4; i++) {
#pragma unroll
        for (int r = 0; r < 4; r++) y[i][r] = at_sum4(y[i][r]);
        if (c == 0) *(f32x4*)(lds + wave * DP + d0 + 4 * i) = y[i];
    }
    if (lane == 0) lds[4 * DP + wave] = l;
    __syncthreads();
    if (threadIdx.x >= 16) return;
    float out[C];
    l = lds[4 * DP] + lds[4 * DP + 1] + lds[4 * DP + 2] + lds[4 * DP + 3];
#pragma unroll
    for (int i = 0; i < C; i++) {
        out[i] = lds[d0 + i];
#pragma unroll
        for (int k = 1; k < 4; k++) out[i] += lds[k * DP + d0 + i];
    }
    const float inv = at_finish(p, tok, head, mm, l, off, d0 == 0);
#pragma unroll
    for (int i = 0; i < C; i++) out[i] *= inv;
    if (d0 < (u32)p.c.d) at_store<C>(p, tok, head, d0, out);
}

// The same where a span has many columns: a wavefront four of them, over all parts.  grid = (wgs, columns / 16), block = 256.
template <int DP> __device__ __forceinline__ void attend_join_wide_body(const AttendArgs& p) {
    constexpr int C = DP / 16;
    const u32 w = blockIdx.x;
    const AtJoin j = at_join_of<DP>(p)[w];
    if (j.last == 0) return;
    const u32 lane = threadIdx.x & 63, x = lane & 15, d0 = C * x, col = blockIdx.y * 16 + (threadIdx.x >> 6) * 4 + (lane >> 4);
    u32 tok, head;
    if (!at_column(p, j.t0, j.t1, j.plane, col, tok, head)) return;
    auto slot = [&](u32 k) { return k == w ? j.slot : 2 * k; };
    float mm = -__builtin_inff(), l = 0.f, out[C];
    f32x4 y[C / 4];
#pragma unroll 4
    for (u32 k = w; k < j.last; k++) mm = fmaxf(mm, (*at_part_ml<DP>(p, slot(k), col)).x);
#pragma unroll
    for (int i = 0; i < C / 4; i++) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (u32 k = w; k < j.last; k++) {
        const f32x2 ml = *at_part_ml<DP>(p, slot(k), col);
        const float turn = ml.x == mm ? 1.f : __builtin_amdgcn_exp2f(ml.x - mm);
        l += ml.y * turn;
#pragma unroll
        for (int i = 0; i < C / 4; i++) y[i] += *(const f32x4*)(at_part<DP>(p, slot(k), col) + d0 + 4 * i) * turn;
    }
    const float inv = at_finish(p, tok, head, mm, l, p.c.type == JL_BF16 ? 0.f : JL_AT_OFF, d0 == 0);
#pragma unroll
    for (int i = 0; i < C; i++) out[i] = y[i / 4][i % 4] * inv;
    if (d0 < (u32)p.c.d) at_store<C>(p, tok, head, d0, out);
}
