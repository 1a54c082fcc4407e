// Low-rank adapters of many requests beside the projections they share (jl_adapter_group_dev): token t of adapter a = ids[t] gets
//   out_i[t] = base_i[t] + scale[a] * B_i[a] (A_i[a] x[t]),     A_i [n_adapter][rank][k], B_i [n_adapter][rows_i][rank]
// for up to four projections that read one x.  A token whose id no adapter has, or whose adapter has rank 0, gets base alone.
//
// Two kernels on the bf16 matrix cores: adapter_down makes u = scale * A x for tiles of sixteen tokens of one adapter, adapter_up adds
// B u to base.  Both take 64 (16) consecutive tokens and find for themselves which of them share an adapter (a ballot per adapter met), so
// nothing is sorted beforehand; a token meets its own adapter only, so no number of another's can reach it.
//
// Products are exact: an f32 value is three bf16 values (8 mantissa bits each, cut off, not rounded), an f16 value two, and every
// piece of one operand meets every piece of the other in the f32 accumulator -- one matrix instruction for bf16 x bf16, three for f32 x
// against bf16 adapters, nine for f32 x f32.  What rounds is the f32 sum, as in a dot product in f32.  (An infinity cut into pieces
// leaves a NaN: it was going to be no finite number.)
//
// adapter_up is bound by base and out, adapter_down by x (many tokens) or the adapters (few).
#pragma once
#include "args.h"
#include "common.h"

typedef __bf16 ad_bf16x8 __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(2))) ad_u32x4_a2 { u32x4 v; };
struct __attribute__((packed, aligned(4))) ad_f32x4_a4 { f32x4 v; };

template <int T> struct AdType {   // 16-bit: a fragment's eight values as they lie
    static constexpr int pieces = T == JL_F16 ? 2 : 1;
    u32x4 w;
    __device__ __forceinline__ void load(const void* p, size_t at) { w = ((const ad_u32x4_a2*)((const uint16_t*)p + at))->v; }
    // the first `left` of the eight (the others are not touched and read 0)
    __device__ __forceinline__ void load_some(const void* p, size_t at, int left) {
        if (left >= 8) return load(p, at);
        w = u32x4{0, 0, 0, 0};
        for (int i = 0; i < left; i++) {
            const u32 h = ((const uint16_t*)p)[at + i];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i / 2 == j) w[j] |= h << (16 * (i & 1));
        }
    }
    __device__ __forceinline__ float value(int i) const {
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        return T == JL_F16 ? half_bits_to_f32(h) : __uint_as_float((u32)h << 16);
    }
};
template <> struct AdType<JL_F32> {
    static constexpr int pieces = 3;
    f32x4 w[2];
    __device__ __forceinline__ void load(const void* p, size_t at) {
        w[0] = ((const ad_f32x4_a4*)((const float*)p + at))->v;
        w[1] = ((const ad_f32x4_a4*)((const float*)p + at + 4))->v;
    }
    __device__ __forceinline__ void load_some(const void* p, size_t at, int left) {
        if (left >= 8) return load(p, at);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i / 4][i & 3] = i < left ? ((const float*)p)[at + i] : 0.f;
    }
    __device__ __forceinline__ float value(int i) const { return w[i / 4][i & 3]; }
};

// Eight f32 values as N bf16 fragments: the high half of the bits, the high half of what that leaves, ...  Exact where the value has at most
// 8 N mantissa bits.
template <int N> __device__ __forceinline__ void ad_split(float (&v)[8], u32x4 (&out)[N]) {
#pragma unroll
    for (int n = 0; n < N; n++) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const u32 a = __float_as_uint(v[2 * j]), b = __float_as_uint(v[2 * j + 1]);
            out[n][j] = __builtin_amdgcn_perm(b, a, 0x07060302);
            if (n + 1 < N) {
                v[2 * j] -= __uint_as_float(a & 0xFFFF0000u);
                v[2 * j + 1] -= __uint_as_float(b & 0xFFFF0000u);
            }
        }
    }
}
template <int T> __device__ __forceinline__ void ad_pieces(const AdType<T>& r, u32x4 (&out)[AdType<T>::pieces]) {
    if constexpr (T == JL_BF16) {
        out[0] = r.w;
    } else {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r.value(i);
        ad_split<AdType<T>::pieces>(v, out);
    }
}
// acc[row][token] += sum over 32 k of a[row][k] b[token][k]; lane = (k / 8) * 16 + row (token), result lane = (row / 4) * 16 + token.
// The smallest products first.
template <int PA, int PB> __device__ __forceinline__ f32x4 ad_mfma(const u32x4 (&a)[PA], const u32x4 (&b)[PB], f32x4 acc) {
#pragma unroll
    for (int s = PA + PB - 2; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < PA; i++)
            if (s - i >= 0 && s - i < PB)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8, a[i]), __builtin_bit_cast(ad_bf16x8, b[s - i]), acc, 0, 0, 0);
    return acc;
}

// A lane's token of the chunk [first, first + size): its adapter, n_adapter where it has none; 0xFFFFFFFF: no token.
__device__ __forceinline__ u32 ad_id(const AdapterArgs& p, int first, int size) {
    const int lane = threadIdx.x & 63, tok = first + lane;
    if (lane >= size || tok >= p.ntok) return 0xFFFFFFFFu;
    u32 id = min(p.ids[tok], (u32)p.n_adapter);
    if (p.ranks && id < (u32)p.n_adapter && p.ranks[id] == 0) id = (u32)p.n_adapter;
    return id;
}
__device__ __forceinline__ int ad_rank(const AdapterArgs& p, u32 id) { return p.ranks ? (int)min(p.ranks[id], (u32)p.rank) : p.rank; }

// ---------------------------------------------------------------- u = scale * A x
// grid = (tile slots of a chunk of 64 tokens, chunks, column passes * K slices), block = 256, LDS = 4 NT KB.
// A tile is up to sixteen tokens of one adapter; workgroup (slot, chunk) takes the chunk's tiles slot, slot + gridDim.x, ...  The four
// wavefronts cut the workgroup's slice of K in four and add their sums through LDS; NT tiles of sixteen columns (rows of A, all
// projections' side by side, each rounded up to sixteen) a pass.  u is [K slices][ntok][n * rank_pad].
template <int T, int XT, int NT>
__device__ __forceinline__ void adapter_down_body(const AdapterArgs& p, f32x4* red) {
    constexpr int PW = AdType<T>::pieces, PX = AdType<XT>::pieces;
    constexpr int UN = NT * sizeof(AdType<T>) <= 16 ? 8 : NT * sizeof(AdType<T>) <= 64 ? 2 : 1;   // K steps asked for at a time
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunk = blockIdx.y * 64, pass = blockIdx.z % p.passes, slice = blockIdx.z / p.passes;
    const int rp = p.rank_pad, ncol = p.n * rp, tiles = ncol / 16;
    const u32 id = ad_id(p, chunk, 64);
    const int steps = p.k / 32, part = slice * 4 + wave, parts = p.slices * 4;
    const int lo = (int)((long)steps * part / parts), hi = (int)((long)steps * (part + 1) / parts);

    int seen = 0, want = blockIdx.x;
    uint64_t rest = __ballot(id < (u32)p.n_adapter);
    while (rest) {   // uniform, and the same in every wavefront
        const int lead = __builtin_ctzll(rest);
        const u32 a = (u32)__builtin_amdgcn_readlane((i32)id, lead);
        uint64_t of = __ballot(id == a);
        const int all = __builtin_popcountll(of), nt = (all + 15) / 16;
        if (want >= seen + nt) {
            seen += nt;
            rest &= ~of;
            continue;
        }
        const int sub = want - seen, count = min(16, all - 16 * sub);
        for (int i = 0; i < 16 * sub; i++) of &= of - 1;
        int tok = chunk + __builtin_ctzll(of);   // the lane's token, lane % 16 of the tile; the first where there are fewer
        for (int i = 0; i < count; i++) {
            if ((lane & 15) == i) tok = chunk + __builtin_ctzll(of);
            of &= of - 1;
        }
        const int rank = ad_rank(p, a);
        const size_t xat = (size_t)tok * p.k + 8 * (lane >> 4);
        const void* wp[NT];
        size_t wat[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int c = min(pass * NT + t, tiles - 1), i = c * 16 / rp, r = min(c * 16 % rp + (lane & 15), rank - 1);
            wp[t] = p.a[i];
            wat[t] = ((size_t)a * p.rank + r) * p.k + 8 * (lane >> 4);
        }
        f32x4 acc[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        auto group = [&](int s, auto un) {
            constexpr int U = decltype(un)::value;
            AdType<XT> x[U];
            AdType<T> w[U][NT];
#pragma unroll
            for (int u = 0; u < U; u++) {
                x[u].load(p.x, xat + 32 * (size_t)(s + u));
#pragma unroll
                for (int t = 0; t < NT; t++) w[u][t].load(wp[t], wat[t] + 32 * (size_t)(s + u));
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                u32x4 xp[PX];
                ad_pieces<XT>(x[u], xp);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    u32x4 wq[PW];
                    ad_pieces<T>(w[u][t], wq);
                    acc[t] = ad_mfma<PW, PX>(wq, xp, acc[t]);
                }
            }
        };
        int s = lo;
        for (; s + UN <= hi; s += UN) group(s, GemmIntC<UN>{});
        if constexpr (UN > 1)
            for (; s < hi; s++) group(s, GemmIntC<1>{});
#pragma unroll
        for (int t = 0; t < NT; t++) red[(wave * NT + t) * 64 + lane] = acc[t];
        __syncthreads();
        const float g = p.scale ? p.scale[a] : 1.f;
        for (int t = wave; t < NT; t += 4) {
            const int c = pass * NT + t;
            if (c >= tiles) break;
            f32x4 v = red[t * 64 + lane];
#pragma unroll
            for (int w = 1; w < 4; w++) v += red[(w * NT + t) * 64 + lane];
            const int r = c * 16 % rp + 4 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = r + i < rank ? g * v[i] : 0.f;
            if ((lane & 15) < count) *(f32x4*)(p.u + ((size_t)slice * p.ntok + tok) * ncol + c * 16 + 4 * (lane >> 4)) = v;
        }
        __syncthreads();
        want += gridDim.x;
    }
}

// ---------------------------------------------------------------- out = base + B u
// grid = (column blocks of all projections, group slots of a chunk of 16 TT tokens, chunks), block = 64 p.up_waves, a wavefront 64 columns
// (rows of B).  A group is the chunk's tokens of one adapter (or of none), up to TT tiles of sixteen; B's fragments meet all of them.
// u's fragments, its K slices added, lie in LDS as bf16 pieces, a rank of 128 at a time.
// VEC: rows of out and base on 16-byte boundaries.
#define JL_AD_UP_LDS(TT) ((TT) * 4 * 3 * 1024 + (TT) * 16 * 4)
template <int T, int TT, bool VEC>
__device__ __forceinline__ void adapter_up_body(const AdapterArgs& p, uint8_t* smem) {
    constexpr int PW = AdType<T>::pieces;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = 64 * p.up_waves;
    const int chunk = blockIdx.z * 16 * TT;
    int pi = 0, cb = blockIdx.x;   // projection, column block in it
    while (pi + 1 < p.n && cb >= (p.rows[pi] + threads - 1) / threads) {
        cb -= (p.rows[pi] + threads - 1) / threads;
        pi++;
    }
    const int rows = p.rows[pi], col0 = cb * threads + wave * 64;
    const float* base = p.base[pi];
    float* out = p.out[pi];
    const int rp = p.rank_pad, ncol = p.n * rp;
    u32x4* frag = (u32x4*)smem;                                   // [ks][tile][piece][lane]
    int* toks = (int*)(smem + TT * 4 * 3 * 1024);
    const u32 id = ad_id(p, chunk, 16 * TT);

    int at = 0;
    uint64_t rest = __ballot(id != 0xFFFFFFFFu);
    while (rest) {   // uniform, and the same in every wavefront
        const int lead = __builtin_ctzll(rest);
        const u32 a = (u32)__builtin_amdgcn_readlane((i32)id, lead);
        const uint64_t of = __ballot(id == a);
        rest &= ~of;
        if (at++ % (int)gridDim.y != (int)blockIdx.y) continue;
        const int count = __builtin_popcountll(of), nt = (count + 15) / 16;
        const bool none = a >= (u32)p.n_adapter;
        if (none && base == out) continue;
        if (wave == 0 && id == a) toks[__builtin_popcountll(of & ((1ull << lane) - 1))] = chunk + lane;
        __syncthreads();
        // base, asked for ahead of everything
        f32x4 bs[TT][4], acc[TT][4];
        size_t oat[TT];
        bool live[TT];
#pragma unroll
        for (int tt = 0; tt < TT; tt++) {
            const int m = 16 * tt + (lane & 15);
            live[tt] = m < count;
            oat[tt] = (size_t)toks[min(m, count - 1)] * rows;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int col = col0 + 16 * c + 4 * (lane >> 4);
                bs[tt][c] = acc[tt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (tt < nt && base) {
                    if (VEC) {
                        if (col < rows) bs[tt][c] = *(const f32x4*)(base + oat[tt] + col);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (col + i < rows) bs[tt][c][i] = base[oat[tt] + col + i];
                    }
                }
            }
        }
        const int rank = none ? 0 : ad_rank(p, a);
        for (int r0 = 0; r0 < rank; r0 += 128) {
            const int nk = min(4, (rank - r0 + 31) / 32);
            for (int f = wave; f < nk * nt; f += p.up_waves) {
                const int ks = f / nt, tt = f % nt, m = 16 * tt + (lane & 15), r = r0 + 32 * ks + 8 * (lane >> 4);
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = 0.f;
                if (m < count && r < rp) {
                    const float* u = p.u + (size_t)toks[m] * ncol + pi * rp + r;
                    for (int s = 0; s < p.slices; s++, u += (size_t)p.ntok * ncol) {
                        const f32x4 lo = *(const f32x4*)u, hi = *(const f32x4*)(u + 4);
#pragma unroll
                        for (int i = 0; i < 4; i++) { v[i] += lo[i]; v[4 + i] += hi[i]; }
                    }
                }
                u32x4 o[3];
                ad_split<3>(v, o);
#pragma unroll
                for (int n = 0; n < 3; n++) frag[((ks * TT + tt) * 3 + n) * 64 + lane] = o[n];
            }
            __syncthreads();
            for (int ks = 0; ks < nk; ks++) {
                const int r = r0 + 32 * ks + 8 * (lane >> 4);
                u32x4 wq[4][PW];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const int col = min(col0 + 16 * c + (lane & 15), rows - 1);
                    AdType<T> w;
                    w.load_some(p.b[pi], ((size_t)a * rows + col) * p.rank + min(r, rank), min(max(rank - r, 0), 8));
                    ad_pieces<T>(w, wq[c]);
                }
#pragma unroll
                for (int tt = 0; tt < TT; tt++) {
                    if (tt >= nt) continue;
                    u32x4 uq[3];
#pragma unroll
                    for (int n = 0; n < 3; n++) uq[n] = frag[((ks * TT + tt) * 3 + n) * 64 + lane];
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[tt][c] = ad_mfma<PW, 3>(wq[c], uq, acc[tt][c]);
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int tt = 0; tt < TT; tt++) {
            if (tt >= nt || !live[tt]) continue;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int col = col0 + 16 * c + 4 * (lane >> 4);
                const f32x4 v = none ? bs[tt][c] : base ? bs[tt][c] + acc[tt][c] : acc[tt][c];
                if (VEC) {
                    if (col < rows) *(f32x4*)(out + oat[tt] + col) = v;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (col + i < rows) out[oat[tt] + col + i] = v[i];
                }
            }
        }
        __syncthreads();   // (toks is the next group's)
    }
}
