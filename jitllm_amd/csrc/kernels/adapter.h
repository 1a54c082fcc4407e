// Low-rank adapters of many requests beside the projections they share (jl_adapter_group_dev): token t of adapter a = ids[t] gets
//   out_i[t] = base_i[t] + scale[a] * B_i[a] (A_i[a] x[t]),     A_i [n_adapter][rank][k], B_i [n_adapter][rows_i][rank]
// for up to four projections that read one x.  A token whose id no adapter has, or whose adapter has rank 0, gets base alone.
//
// Many tokens: adapter_group puts the tokens of an adapter side by side; then on the bf16 matrix cores, for tiles of up to 64 of them, adapter_down
// makes sums of u = A x over slices of K and adapter_up adds B u to base (where many column blocks would each add the slices up, adapter_sum does
// it first).  Few tokens, or few of each adapter: dot products in f32, in two launches or one (the end of this file).  A token meets its own adapter
// only, so no number of another's can reach it.
//
// Products are exact: an f32 value is three bf16 values (8 mantissa bits each, cut off, not rounded), an f16 value two, and every
// piece of one operand meets every piece of the other in the f32 accumulator -- one matrix instruction for bf16 x bf16, three for f32 x
// against bf16 adapters, nine for f32 x f32.  What rounds is the f32 sum, as in a dot product in f32.  (An infinity cut into pieces
// leaves a NaN, as does one that meets a zero piece: it was going to be no finite number.  A bf16 value ends at 2^-133: what an f32 value has below that is lost,
// from 2^-110 on nothing.)
//
// What decides the layout of the work (measured on MI355X): sixteen rows of 64 bytes a load, as the matrix instruction's operands and results lie, run
// at two thirds of the rate of rows of 256 bytes, so x, base and out are moved by rows and change places in LDS; and with few tokens a call is
// trips to memory one after the other, so everything whose address is known is asked for at once.
#pragma once
#include "args.h"
#include "common.h"

typedef __bf16 ad_bf16x8 __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(2))) ad_u32x4_a2 { u32x4 v; };
struct __attribute__((packed, aligned(2))) ad_u32x2_a2 { u32x2 v; };
struct __attribute__((packed, aligned(2))) ad_u32_a2 { u32 v; };
struct __attribute__((packed, aligned(4))) ad_f32x4_a4 { f32x4 v; };
struct __attribute__((packed, aligned(4))) ad_u32x2_a4 { u32x2 v; };

template <int T> struct AdType {   // 16-bit: a fragment's eight values as they lie
    static constexpr int pieces = T == JL_F16 ? 2 : 1;
    u32x4 w;
    __device__ __forceinline__ void load(const void* p, size_t at) { w = ((const ad_u32x4_a2*)((const uint16_t*)p + at))->v; }
    // The first `left` of the eight: a four, a two and a one of them, as far as they are there.  place() puts them where they belong, zeros behind them;
    // it is apart from the loads so that nothing waits for one of them before all are on their way.
    __device__ __forceinline__ void load_some(const void* p, size_t at, int left) {
        if (left >= 8) return load(p, at);
        const uint16_t* h = (const uint16_t*)p + at;
        w = u32x4{0, 0, 0, 0};
        if (left & 4) {
            const u32x2 four = ((const ad_u32x2_a2*)h)->v;
            w[0] = four.x;
            w[1] = four.y;
        }
        if (left & 2) w[2] = ((const ad_u32_a2*)(h + (left & 4)))->v;
        if (left & 1) w[3] = h[left & 6];
    }
    __device__ __forceinline__ void place(int left) {
        if (left >= 8) return;
        const u32 hi = left & 4 ? ~0u : 0u, next = left & 2 ? ~0u : 0u, a = w[2] | (w[3] & ~next), b = w[3] & next;   // (bits: no index into registers)
        w = u32x4{w[0] | (a & ~hi), w[1] | (b & ~hi), a & hi, b & hi};
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
        const float* f = (const float*)p + at;
        w[0] = w[1] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (left & 4) w[0] = ((const ad_f32x4_a4*)f)->v;
        if (left & 2) {
            const u32x2 two = ((const ad_u32x2_a4*)(f + (left & 4)))->v;
            w[1][0] = __uint_as_float(two.x);
            w[1][1] = __uint_as_float(two.y);
        }
        if (left & 1) w[1][2] = f[left & 6];
    }
    __device__ __forceinline__ void place(int left) {
        if (left >= 8) return;
        const u32 hi = left & 4 ? ~0u : 0u, next = left & 2 ? ~0u : 0u, one = __float_as_uint(w[1][2]);
        const u32 r[3] = {__float_as_uint(w[1][0]) | (one & ~next), __float_as_uint(w[1][1]), one & next};
#pragma unroll
        for (int i = 0; i < 3; i++) {
            w[0][i] = __uint_as_float(__float_as_uint(w[0][i]) | (r[i] & ~hi));
            w[1][i] = __uint_as_float(r[i] & hi);
        }
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

__device__ __forceinline__ int ad_rank(const AdapterArgs& p, u32 id) { return p.ranks ? (int)min(p.ranks[id], (u32)p.rank) : p.rank; }

// Four consecutive elements as f32.
template <int T> struct AdQuad {
    u32x2 w;
    __device__ __forceinline__ void load(const void* p, size_t at) { w = *(const u32x2*)((const uint16_t*)p + at); }
    __device__ __forceinline__ float value(int i) const {
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        return T == JL_F16 ? half_bits_to_f32(h) : __uint_as_float((u32)h << 16);
    }
};
template <> struct AdQuad<JL_F32> {
    f32x4 w;
    __device__ __forceinline__ void load(const void* p, size_t at) { w = *(const f32x4*)((const float*)p + at); }
    __device__ __forceinline__ float value(int i) const { return w[i]; }
};

// ---------------------------------------------------------------- tokens by adapter
// perm: the tokens, those of an adapter side by side (those without one last); tiles: {adapter, first place in perm, tokens} of pieces of up to
// 64 of them, n_adapter for those without one, 0 tokens behind the last.  The order inside an adapter is whatever the LDS additions make
// it: no result depends on what else is in a token's tile.  One workgroup of 1024; LDS: n_adapter + 1 counters, 32 totals.
__device__ __forceinline__ void adapter_group_body(const AdapterArgs& p, u32* count) {
    const int tid = threadIdx.x, kinds = p.n_adapter + 1, lane = tid & 63, wave = tid >> 6;
    u32* tot = count + kinds;
    auto kind = [&](int t) {
        const u32 id = min(p.ids[t], (u32)p.n_adapter);
        return p.ranks && id < (u32)p.n_adapter && p.ranks[id] == 0 ? (u32)p.n_adapter : id;
    };
    u32 mine[4];   // of the first 4096 tokens; later ones are read again
#pragma unroll
    for (int i = 0; i < 4; i++) mine[i] = tid + 1024 * i < p.ntok ? kind(tid + 1024 * i) : 0;
    for (int i = tid; i < kinds; i += 1024) count[i] = 0;
    __syncthreads();
    // a token's place among its kind's so far; one addition for a wavefront whose tokens are all of a kind (a prompt's), which LDS would take one by one
    auto take = [&](u32 k, bool live) {
        const uint64_t on = __ballot(live);
        const u32 first = (u32)__builtin_amdgcn_readfirstlane((i32)k);
        if (on == ~0ull && __ballot(k == first) == ~0ull) {
            u32 at = 0;
            if (lane == 0) at = atomicAdd(&count[first], 64u);
            return (u32)__builtin_amdgcn_readfirstlane((i32)at) + lane;
        }
        return live ? atomicAdd(&count[k], 1u) : 0u;
    };
#pragma unroll
    for (int i = 0; i < 4; i++) (void)take(mine[i], tid + 1024 * i < p.ntok);
    for (int t0 = 4096; t0 < p.ntok; t0 += 1024) (void)take(t0 + tid < p.ntok ? kind(t0 + tid) : 0, t0 + tid < p.ntok);
    __syncthreads();
    // places and tiles before a thread's run of kinds
    const int per = (kinds + 1023) / 1024, lo = min(tid * per, kinds), hi = min(lo + per, kinds);
    u32 np = 0, nt = 0;
    for (int i = lo; i < hi; i++) {
        np += count[i];
        nt += (count[i] + 63) / 64;
    }
    u32 sp = np, st = nt;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u32 a = __shfl_up(sp, off, 64), b = __shfl_up(st, off, 64);
        if (lane >= off) {
            sp += a;
            st += b;
        }
    }
    if (lane == 63) {
        tot[wave] = sp;
        tot[16 + wave] = st;
    }
    __syncthreads();
    for (int w = 0; w < wave; w++) {
        sp += tot[w];
        st += tot[16 + w];
    }
    u32 all = 0;
    for (int w = 0; w < 16; w++) all += tot[16 + w];
    u32 place = sp - np, tile = st - nt;
    for (int i = lo; i < hi; i++) {
        const u32 n = count[i];
        for (u32 t = 0; t < n; t += 64) ((u32x4*)p.tiles)[tile++] = u32x4{(u32)i, place + t, min(64u, n - t), 0};
        count[i] = place;
        place += n;
    }
    for (u32 t = all + tid; t < (u32)p.max_tiles; t += 1024) ((u32x4*)p.tiles)[t] = u32x4{(u32)p.n_adapter, 0, 0, 0};
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool live = tid + 1024 * i < p.ntok;
        const u32 at = take(mine[i], live);
        if (live) p.perm[at] = tid + 1024 * i;
    }
    for (int t0 = 4096; t0 < p.ntok; t0 += 1024) {
        const bool live = t0 + tid < p.ntok;
        const u32 at = take(live ? kind(t0 + tid) : 0, live);
        if (live) p.perm[at] = t0 + tid;
    }
}
struct AdTile {
    u32 a;
    int count, nt, rank;
    bool none;
    // toks: the tile's tokens, in LDS behind the next barrier.  False: no such tile.
    __device__ __forceinline__ bool of(const AdapterArgs& p, int tile, int* toks) {
        const u32x4 t = ((const u32x4*)p.tiles)[tile];
        count = (int)t.z;
        if (count == 0) return false;
        a = t.x;
        none = a >= (u32)p.n_adapter;
        nt = (count + 15) / 16;
        rank = none ? 0 : ad_rank(p, a);
        if (threadIdx.x < 64 && (int)threadIdx.x < count) toks[threadIdx.x] = p.perm[t.y + threadIdx.x];
        return true;
    }
};

// ---------------------------------------------------------------- sums of A x
// grid = (tiles, 1, passes * slices), block = 256.  A workgroup takes a tile's up to 64 tokens (four of sixteen), NT column
// tiles a wavefront (sixteen rows of A each; all projections' side by side, a rank rounded up to sixteen) and a slice of K, 128 at a time: x by
// rows of 512 bytes through registers, cut into pieces on the way to LDS, where all four wavefronts read it; A's fragments straight from
// memory, each once a workgroup.  Writes part [slices][ntok][n * rank_pad].
// LDS: [pieces][64 tokens][136] bf16 (a row's 272 bytes put sixteen rows' reads on different banks).
#define JL_AD_DOWN_K 128
#define JL_AD_DOWN_ROW 136
template <int T, int XT, int NT>
__device__ __forceinline__ void adapter_down_body(const AdapterArgs& p, uint16_t* sx, int* toks) {
    constexpr int PW = AdType<T>::pieces, PX = AdType<XT>::pieces, ROW = JL_AD_DOWN_ROW;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int pass = blockIdx.z % p.passes, slice = blockIdx.z / p.passes;
    const int ctiles = p.rank_pad / 16, all = p.n * ctiles, c0 = (pass * 4 + wave) * NT;
    const int steps = (p.k + JL_AD_DOWN_K - 1) / JL_AD_DOWN_K;
    const int lo = steps * slice / p.slices, hi = steps * (slice + 1) / p.slices;   // (slices <= steps)
    AdTile tile;
    if (!tile.of(p, blockIdx.x, toks) || tile.none) return;
    const u32 a = tile.a;
    const int count = tile.count, rank = tile.rank;
    __syncthreads();
    {
        const void* wp[NT];
        size_t wat[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int c = min(c0 + t, all - 1), i = c / ctiles, r = min((c - i * ctiles) * 16 + (lane & 15), rank - 1);
            wp[t] = p.a[i];
            wat[t] = ((size_t)a * p.rank + r) * p.k + 8 * (lane >> 4);
        }
        auto run = [&](auto tiles) {   // (of the group, rounded up to one or four: no branch between the matrix instructions)
            constexpr int MT = decltype(tiles)::value;
            // a thread's rows of x: token 8 i + tid / 32 of the group, four elements from 4 (tid % 32) on
            size_t xat[2 * MT];
#pragma unroll
            for (int i = 0; i < 2 * MT; i++) xat[i] = (size_t)toks[min(8 * i + tid / 32, count - 1)] * p.k;
            AdQuad<XT> x[2 * MT];
            AdType<T> w[4][NT];
            // (past the end of K: its last elements, which meet nothing)
            auto load_x = [&](int s) {
                const int e = min(s * JL_AD_DOWN_K + 4 * (tid & 31), p.k - 4);
#pragma unroll
                for (int i = 0; i < 2 * MT; i++) x[i].load(p.x, xat[i] + e);
            };
            auto load_w = [&](int s, int q) {
                const int e = min(s * JL_AD_DOWN_K + 32 * q, p.k - 32);
#pragma unroll
                for (int t = 0; t < NT; t++) w[q][t].load(wp[t], wat[t] + e);
            };
            f32x4 acc[MT][NT];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int t = 0; t < NT; t++) acc[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            load_x(lo);
#pragma unroll
            for (int q = 0; q < 4; q++) load_w(lo, q);
            for (int s = lo; s < hi; s++) {
#pragma unroll
                for (int i = 0; i < 2 * MT; i++) {
                    float v[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] = x[i].value(j);
#pragma unroll
                    for (int n = 0; n < PX; n++) {
                        u32 b[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            b[j] = __float_as_uint(v[j]);
                            if (n + 1 < PX) v[j] -= __uint_as_float(b[j] & 0xFFFF0000u);
                        }
                        *(u32x2*)(sx + (n * 64 + 8 * i + tid / 32) * ROW + 4 * (tid & 31)) =
                            u32x2{__builtin_amdgcn_perm(b[1], b[0], 0x07060302), __builtin_amdgcn_perm(b[3], b[2], 0x07060302)};
                    }
                }
                lds_barrier();
                const int next = min(s + 1, hi - 1), nq = min(4, (p.k - s * JL_AD_DOWN_K) / 32);
                load_x(next);
                if (c0 < all) {
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        if (q < nq) {
                            u32x4 xq[MT][PX], wq[NT][PW];
#pragma unroll
                            for (int m = 0; m < MT; m++)
#pragma unroll
                                for (int n = 0; n < PX; n++) xq[m][n] = *(const u32x4*)(sx + (n * 64 + 16 * m + (lane & 15)) * ROW + 32 * q + 8 * (lane >> 4));
#pragma unroll
                            for (int t = 0; t < NT; t++) ad_pieces<T>(w[q][t], wq[t]);
                            load_w(next, q);
                            // the smallest products first; a piece's products of all tiles side by side
#pragma unroll
                            for (int o = PW + PX - 2; o >= 0; o--)
#pragma unroll
                                for (int i = 0; i < PW; i++)
                                    if (o - i >= 0 && o - i < PX) {
#pragma unroll
                                        for (int m = 0; m < MT; m++)
#pragma unroll
                                            for (int t = 0; t < NT; t++)
                                                acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ad_bf16x8, wq[t][i]),
                                                                                                    __builtin_bit_cast(ad_bf16x8, xq[m][o - i]), acc[m][t], 0, 0, 0);
                                    }
                        }
                    }
                }
                lds_barrier();
            }
#pragma unroll
            for (int m = 0; m < MT; m++) {
                if (16 * m + (lane & 15) >= count) continue;
                float* u = p.part + ((size_t)slice * p.ntok + toks[16 * m + (lane & 15)]) * all * 16 + 4 * (lane >> 4);
#pragma unroll
                for (int t = 0; t < NT; t++)
                    if (c0 + t < all) *(f32x4*)(u + (c0 + t) * 16) = acc[m][t];
            }
        };
        if (tile.nt > 1) run(GemmIntC<4>{});
        else run(GemmIntC<1>{});
    }
}

// Eight of a token's u, of projection pi from r on: the slices added up, times the adapter's scale, 0 from its rank on, as bf16 pieces.
__device__ __forceinline__ void ad_sum_u(const AdapterArgs& p, int tok, int pi, int r, float scale, int rank, u32x4 (&o)[3]) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = 0.f;
    if (r < p.rank_pad) {
        const int ncol = p.n * p.rank_pad;
        const float* u = p.part + (size_t)tok * ncol + pi * p.rank_pad + r;
        const size_t step = (size_t)p.ntok * ncol;
        for (int s = 0; s < p.slices; s += 4) {   // four slices on their way at a time
            f32x4 lo[4], hi[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const float* at = u + step * min(s + q, p.slices - 1);
                lo[q] = *(const f32x4*)at;
                hi[q] = *(const f32x4*)(at + 4);
            }
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (s + q < p.slices) {
#pragma unroll
                    for (int i = 0; i < 4; i++) { v[i] += lo[q][i]; v[4 + i] += hi[q][i]; }
                }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r + i < rank ? scale * v[i] : 0.f;
    }
    ad_split<3>(v, o);
}
// part -> u [ntok][n][K steps of 32][3 pieces][32] bf16.  grid = ceil(ntok * n * K steps * 8 / 256), block = 256: a thread four of a row, all slices on
// their way at a time.
__device__ __forceinline__ void adapter_sum_body(const AdapterArgs& p) {
    const int ks = (p.rank_pad + 31) / 32, ncol = p.n * p.rank_pad;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int quad = (int)(i % (ks * 8)), pi = (int)(i / (ks * 8) % p.n), r = 4 * quad;
    const size_t tok = i / ((size_t)ks * 8 * p.n);
    if (tok >= (size_t)p.ntok) return;
    const float* at = p.part + tok * ncol + pi * p.rank_pad + min(r, p.rank_pad - 4);
    f32x4 v[16];
#pragma unroll
    for (int s = 0; s < 16; s++) v[s] = s < p.slices ? *(const f32x4*)(at + (size_t)s * p.ntok * ncol) : f32x4{0.f, 0.f, 0.f, 0.f};
    const u32 id = p.ids[tok];
    if (id >= (u32)p.n_adapter) return;   // (nobody reads u of a token without an adapter)
    const int rank = ad_rank(p, id);
    const float scale = p.scale ? p.scale[id] : 1.f;
#pragma unroll
    for (int s = 1; s < 16; s++) v[0] += v[s];
#pragma unroll
    for (int e = 0; e < 4; e++) v[0][e] = r + e < rank ? scale * v[0][e] : 0.f;
    uint16_t* u = p.u + ((tok * p.n + pi) * ks + quad / 8) * 96 + quad % 8 * 4;
#pragma unroll
    for (int n = 0; n < 3; n++) {
        u32 b[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            b[e] = __float_as_uint(v[0][e]);
            v[0][e] -= __uint_as_float(b[e] & 0xFFFF0000u);
        }
        *(u32x2*)(u + 32 * n) = u32x2{__builtin_amdgcn_perm(b[1], b[0], 0x07060302), __builtin_amdgcn_perm(b[3], b[2], 0x07060302)};
    }
}

// ---------------------------------------------------------------- out = base + B u
// A fragment of B: eight columns of row `col` of the adapter's sheet from r on, zeros from its rank on.
template <int T>
__device__ __forceinline__ void ad_load_b(AdType<T>& w, const AdapterArgs& p, int pi, u32 a, int col, int r, int rank) {
    w.load_some(p.b[pi], ((size_t)a * p.rows[pi] + col) * p.rank + min(r, rank), min(max(rank - r, 0), 8));   // (place() it)
}
// The projection of a column block and the block's number in it; width: columns a block.
__device__ __forceinline__ int ad_projection(const AdapterArgs& p, int& block, int width) {
    int i = 0;
    while (i + 1 < p.n && block >= (p.rows[i] + width - 1) / width) {
        block -= (p.rows[i] + width - 1) / width;
        i++;
    }
    return i;
}

// grid = (blocks of 256 columns of all projections, tiles), block = 256, a wavefront 64 columns (rows of B; two such sets a workgroup
// were slower everywhere: 2048 tokens rank 64 beside 2 x 14336 149.8 against 143.8 us, beside 4096 57 against 50).  u's fragments of the tile's (up to four) sixteens lie in LDS, KS K steps of 32 at a time; B's stay in registers and meet
// one after the other.  A tile's sums change places in LDS and meet base by rows of 256 bytes, asked for a tile ahead.
// KS = 1: ranks up to 32, 2: up to 64.  MANY: any rank, KS steps at a time; the four tiles' sums stay in registers and base is read at the end.
// VEC: rows of out and base on 16-byte boundaries.
// LDS: frag [4 tiles][KS][3][64] x 16 bytes, move [4 wavefronts][16][68] floats, toks [64].
#define JL_AD_MOVE 68
template <int T, int KS, bool MANY, bool VEC>
__device__ __forceinline__ void adapter_up_body(const AdapterArgs& p, u32x4* frag, float* move, int* toks) {
    constexpr int PW = AdType<T>::pieces;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int block = blockIdx.x;
    const int pi = ad_projection(p, block, 256);
    const int rows = p.rows[pi], ksteps = (p.rank_pad + 31) / 32;
    const float* base = p.base[pi];
    float* out = p.out[pi];
    move += wave * 16 * JL_AD_MOVE;
    AdTile tile;
    if (!tile.of(p, blockIdx.y, toks) || (tile.none && base == out)) return;
    {
        const bool none = tile.none;
        const u32 a = tile.a;
        const int count = tile.count, nt = tile.nt, rank = tile.rank;
        const float scale = none || !p.scale ? 1.f : p.scale[a];
        __syncthreads();
        // by rows: token 4 i + lane / 16 of a tile, four columns from 4 (lane % 16) on
        f32x4 bs[4];
        size_t oat[4];
        auto load_base = [&](int tt, int col) {
            const int c = col + 4 * (lane & 15);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                oat[i] = (size_t)toks[min(16 * tt + 4 * i + (lane >> 4), count - 1)] * rows + c;
                bs[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (base) {
                    if (VEC) {
                        if (c < rows) bs[i] = *(const f32x4*)(base + oat[i]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (c + e < rows) bs[i][e] = base[oat[i] + e];
                    }
                }
            }
        };
        auto finish = [&](int tt, int col, f32x4 (&acc)[4], const f32x4 (&b0)[4], const size_t (&o0)[4]) {
            f32x4 v[4];
            if (none) {
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = b0[i];
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++) *(f32x4*)(move + (lane & 15) * JL_AD_MOVE + 16 * c + 4 * (lane >> 4)) = acc[c];
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (a wavefront's own LDS)
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = *(const f32x4*)(move + (4 * i + (lane >> 4)) * JL_AD_MOVE + 4 * (lane & 15));
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (base)
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = b0[i] + v[i];
            }
            const int c = col + 4 * (lane & 15);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (16 * tt + 4 * i + (lane >> 4) >= count) continue;
                if (VEC) {
                    if (c < rows) *(f32x4*)(out + o0[i]) = v[i];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (c + e < rows) out[o0[i] + e] = v[i][e];
                }
            }
        };
        auto stage = [&](int s0) {   // u's fragments of K steps [s0, s0 + KS)
            for (int f = wave; f < nt * KS; f += 4) {
                const int tt = f / KS, s = s0 + f % KS, m = 16 * tt + (lane & 15);
                u32x4 o[3];
                const int tok = toks[min(m, count - 1)];
                if (p.slices) {
                    ad_sum_u(p, tok, pi, 32 * s + 8 * (lane >> 4), scale, rank, o);
                } else {
                    const uint16_t* u = p.u + (((size_t)tok * p.n + pi) * ksteps + min(s, ksteps - 1)) * 96 + 8 * (lane >> 4);
#pragma unroll
                    for (int n = 0; n < 3; n++) o[n] = *(const u32x4*)(u + 32 * n);
                }
#pragma unroll
                for (int n = 0; n < 3; n++) frag[((tt * KS + f % KS) * 3 + n) * 64 + lane] = o[n];
            }
        };
        auto load_b = [&](int s0, int col, u32x4 (&wq)[KS][4][PW]) {
            AdType<T> w[KS][4];
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int c = 0; c < 4; c++) ad_load_b<T>(w[s][c], p, pi, a, min(col + 16 * c + (lane & 15), rows - 1), 32 * (s0 + s) + 8 * (lane >> 4), rank);
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    w[s][c].place(max(rank - 32 * (s0 + s) - 8 * (lane >> 4), 0));
                    ad_pieces<T>(w[s][c], wq[s][c]);
                }
        };
        auto multiply = [&](int tt, const u32x4 (&wq)[KS][4][PW], f32x4 (&acc)[4]) {
#pragma unroll
            for (int s = 0; s < KS; s++) {
                u32x4 uq[3];
#pragma unroll
                for (int n = 0; n < 3; n++) uq[n] = frag[((tt * KS + s) * 3 + n) * 64 + lane];
#pragma unroll
                for (int c = 0; c < 4; c++) acc[c] = ad_mfma<PW, 3>(wq[s][c], uq, acc[c]);
            }
        };
        const int col = block * 256 + wave * 64;
        if constexpr (!MANY) {
            if (col < rows) load_base(0, col);
            if (!none) stage(0);
            __syncthreads();
            if (col >= rows) return;
            u32x4 wq[KS][4][PW];
            if (!none) load_b(0, col, wq);
            for (int tt = 0; tt < nt; tt++) {
                f32x4 acc[4], b0[4];
                size_t o0[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
                    b0[c] = bs[c];
                    o0[c] = oat[c];
                }
                if (tt + 1 < nt) load_base(tt + 1, col);
                if (!none) multiply(tt, wq, acc);
                finish(tt, col, acc, b0, o0);
            }
        } else {   // (every wavefront takes part in the staging)
            f32x4 acc[4][4];
#pragma unroll
            for (int tt = 0; tt < 4; tt++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[tt][c] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (!none)
                for (int s0 = 0; 32 * s0 < rank; s0 += KS) {
                    stage(s0);
                    __syncthreads();
                    if (col < rows) {
                        u32x4 wq[KS][4][PW];
                        load_b(s0, col, wq);
#pragma unroll
                        for (int tt = 0; tt < 4; tt++)
                            if (tt < nt) multiply(tt, wq, acc[tt]);
                    }
                    __syncthreads();
                }
            if (col < rows) {
#pragma unroll
                for (int tt = 0; tt < 4; tt++)
                    if (tt < nt) {
                        load_base(tt, col);
                        finish(tt, col, acc[tt], bs, oat);
                    }
            }
        }
    }
}

// ---------------------------------------------------------------- few tokens: dot products in f32
// Sums over the wavefront of RB values a lane; lane l has those of rows 4 i + l % 4 in s[i].  Half of the values leave a lane with each of the
// first two steps: 52 instructions for sixteen rows, where a sum at a time would take 96 (and those were a third of the kernels' time).
template <int RB> __device__ __forceinline__ void ad_wave_rows(float (&s)[RB]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < RB / 2; i++) {
        const float keep = lane & 1 ? s[2 * i + 1] : s[2 * i], give = lane & 1 ? s[2 * i] : s[2 * i + 1];
        s[i] = keep + dpp_f32<JL_DPP_QUAD_XOR1, 0xf>(give);
    }
#pragma unroll
    for (int i = 0; i < RB / 4; i++) {
        const float keep = lane & 2 ? s[2 * i + 1] : s[2 * i], give = lane & 2 ? s[2 * i] : s[2 * i + 1];
        float v = keep + dpp_f32<JL_DPP_QUAD_XOR2, 0xf>(give);
        v += dpp_f32<0x124, 0xf>(v);   // rotations by four and eight lanes of sixteen
        v += dpp_f32<0x128, 0xf>(v);
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        s[i] = __uint_as_float(h[0]) + __uint_as_float(h[1]);
    }
}
// Dot products of RB rows of A (row, row + step, ..., the last again past `rank`) with a token's x over the pieces q, q + pieces, ... of 256
// elements of K, four a lane.
template <int T, int RB> __device__ __forceinline__ void ad_rows(const AdapterArgs& p, int pi, u32 id, int rank, size_t xrow, int row, int step, int q, int pieces, float (&sum)[RB]) {
    const int lane = threadIdx.x & 63, k = p.k;
#pragma unroll
    for (int j = 0; j < RB; j++) sum[j] = 0.f;
    for (; q * 256 < k; q += pieces) {
        const int e = q * 256 + 4 * lane, at = min(e, k - 4);
        AdQuad<T> w[RB];
#pragma unroll
        for (int j = 0; j < RB; j++) w[j].load(p.a[pi], ((size_t)id * p.rank + min(row + j * step, rank - 1)) * k + at);
        float x[4];
        if (p.x_type == JL_F32) {
            AdQuad<JL_F32> v;
            v.load(p.x, xrow + at);
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = v.value(i);
        } else {
            AdQuad<JL_BF16> v;
            v.load(p.x, xrow + at);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint16_t h = (uint16_t)(v.w[i / 2] >> (16 * (i & 1)));
                x[i] = p.x_type == JL_F16 ? half_bits_to_f32(h) : __uint_as_float((u32)h << 16);
            }
        }
        if (e < k) {
#pragma unroll
            for (int j = 0; j < RB; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) sum[j] = __builtin_fmaf(w[j].value(i), x[i], sum[j]);
        }
    }
}
// Columns of out.  L lanes a column: eight elements of a row of B each (rank <= 8 L); a wavefront's 64 columns are L loads of 64 / L rows, whole
// lines, and lane l ends up with column l % L * (64 / L) + l / L.  A row's last eight elements start where they end with the row, also where the
// lane before has the first of them: those meet zeros (ad_first says how many).
template <int L> __device__ __forceinline__ int ad_first(int r0, int bank_rank) { return L == 1 ? 0 : max(r0 - (bank_rank - 8), 0); }   // (L > 1: rank > 8)
template <int N> __device__ __forceinline__ float ad_lane_sum(float v) {   // over N consecutive lanes; each has it
    if (N >= 2) v += dpp_f32<JL_DPP_QUAD_XOR1, 0xf>(v);
    if (N >= 4) v += dpp_f32<JL_DPP_QUAD_XOR2, 0xf>(v);
    if (N >= 8) v += dpp_f32<JL_DPP_ROW_HALF_MIRROR, 0xf>(v);
    return v;
}
// A lane's eight of u, which lie in LDS.
template <int L> __device__ __forceinline__ void ad_take_u(const AdapterArgs& p, const float* us, float (&u)[8]) {
    const int r0 = 8 * ((threadIdx.x & 63) % L);
    if (L == 1 || p.rank % 8 == 0) {   // uniform; 16-byte reads
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = us[r0 + i];
    } else {
        const int first = ad_first<L>(r0, p.rank);
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] = i < first ? 0.f : us[r0 - first + i];
    }
}
template <int T, int L> struct AdColumns {
    AdType<T> b[L];
    float base;
    // (B by the bank's rank: the adapter's own is known later)
    __device__ __forceinline__ void load(const AdapterArgs& p, int pi, u32 id, size_t orow, int col) {
        const int lane = threadIdx.x & 63, rows = p.rows[pi], r0 = 8 * (lane % L), r = r0 - ad_first<L>(r0, p.rank), mine = col + lane % L * (64 / L) + lane / L;
        base = p.base[pi] && mine < rows ? p.base[pi][orow + mine] : 0.f;
#pragma unroll
        for (int j = 0; j < L; j++) {
            const size_t at = ((size_t)id * rows + min(col + j * (64 / L) + lane / L, rows - 1)) * p.rank + r;
            if (L > 1) b[j].load(p.b[pi], at);
            else b[j].load_some(p.b[pi], at, p.rank);   // (uniform)
        }
    }
    __device__ __forceinline__ void finish(const AdapterArgs& p, int pi, size_t orow, int col, int rank, const float (&u)[8]) {
        const int lane = threadIdx.x & 63, r0 = 8 * (lane % L), first = ad_first<L>(r0, p.rank), mine = col + lane % L * (64 / L) + lane / L, left = rank - r0 + first;
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < L; j++) {
            float v = 0.f;
            if (L == 1) b[j].place(p.rank);
            if (p.ranks || (L > 1 && p.rank != 8 * L)) {   // columns of B from the adapter's rank on may hold anything
#pragma unroll
                for (int i = 0; i < 8; i++) v = __builtin_fmaf(i >= first && i < left ? b[j].value(i) : 0.f, u[i], v);
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) v = __builtin_fmaf(b[j].value(i), u[i], v);
            }
            v = ad_lane_sum<L>(v);
            if (lane % L == j) d = v;
        }
        if (mine < p.rows[pi]) p.out[pi][orow + mine] = !p.base[pi] ? d : rank ? base + d : base;
    }
};
// base (zeros without one) to the columns of a token without an adapter: those of a workgroup of `threads` from col on, `sets` times.
__device__ __forceinline__ void ad_copy(const AdapterArgs& p, int pi, size_t orow, int col, int threads, int sets) {
    const float* base = p.base[pi];
    if (base == p.out[pi]) return;
    for (int s = 0; s < sets; s++, col += threads)
        if (col < p.rows[pi]) p.out[pi][orow + col] = base ? base[orow + col] : 0.f;
}

// One launch: a workgroup makes u of one token for one projection -- its sixteen wavefronts cut K (and the rows of A where K is short) among
// them -- and then a block of 1024 columns of out.  Every column block makes u anew: A and x come from L2 then, which costs less than a second
// launch while the rank is small (4096 x 4096, one token: rank 8 4.6 us, 16 6.1; the two launches below 6.5 and 6.8).  What counts here is the
// number of trips to memory one after the other: the adapter's id, then base, B, A and x together, then out.
// grid = (column blocks of all projections, ntok), block = 1024.  LDS: part [16][8 L] and u [8 L] floats.
#define JL_AD_ONE_LDS(L) (17 * 8 * (L))
template <int T, int L>
__device__ __forceinline__ void adapter_one_body(const AdapterArgs& p, float* lds) {
    constexpr int R = 8 * L, RB = R < 16 || T == JL_F32 ? 8 : 16;   // rows of A asked for at a time, as many as the registers hold beside B
    float* part = lds;
    float* us = lds + 16 * R;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tok = blockIdx.y;
    int block = blockIdx.x;
    const int pi = ad_projection(p, block, 1024);
    const u32 id = p.ids[tok];
    const size_t orow = (size_t)tok * p.rows[pi];
    if (id >= (u32)p.n_adapter) return ad_copy(p, pi, orow, block * 1024 + (int)threadIdx.x, 1024, 1);   // uniform
    const int rank = ad_rank(p, id);
    const int col = block * 1024 + wave * 64;
    const bool here = col < p.rows[pi];
    AdColumns<T, L> c;
    if (here) c.load(p, pi, id, orow, col);
    // wavefront = (piece of K modulo pieces, rows modulo 16 / pieces)
    const int np = (p.k + 255) / 256, pieces = np > 8 ? 16 : np > 4 ? 8 : np > 2 ? 4 : np;   // a power of two
    const int piece = wave & (pieces - 1), step = 16 / pieces;
    for (int r = wave / pieces; r < p.rank; r += RB * step) {
        float sum[RB];
        ad_rows<T, RB>(p, pi, id, p.rank, (size_t)tok * p.k, r, step, piece, pieces, sum);
        ad_wave_rows<RB>(sum);
#pragma unroll
        for (int i = 0; i < RB / 4; i++) {
            const int row = r + (4 * i + lane) * step;
            if (lane < 4 && row < p.rank) part[piece * R + row] = sum[i];
        }
    }
    __syncthreads();
    if (threadIdx.x < R) {
        float v = 0.f;
        if ((int)threadIdx.x < rank) {
            for (int q = 0; q < pieces; q++) v += part[q * R + threadIdx.x];
            v *= p.scale ? p.scale[id] : 1.f;
        }
        us[threadIdx.x] = v;
    }
    __syncthreads();
    if (!here) return;
    float u[8];
    ad_take_u<L>(p, us, u);
    c.finish(p, pi, orow, col, rank, u);
}

// Two launches.  Sums of A x of a token: grid = (slices of 1024 elements of K modulo p.slices, ntok, projections * ceil(rank / 16)), block = 256, a
// wavefront sixteen rows of A over 256 elements; part as adapter_down's.
template <int T> __device__ __forceinline__ void adapter_dots_body(const AdapterArgs& p, float* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tok = blockIdx.y, ctiles = p.rank_pad / 16;
    const int pi = blockIdx.z / ctiles, r = blockIdx.z % ctiles * 16;
    const u32 id = p.ids[tok];
    if (id >= (u32)p.n_adapter) return;
    // (the first tile does not wait for the adapter's own rank: adapter_cols uses no u from there on)
    if (r && r >= ad_rank(p, id)) return;   // uniform
    float sum[16];
    ad_rows<T, 16>(p, pi, id, p.rank, (size_t)tok * p.k, r, 1, (int)blockIdx.x * 4 + wave, p.slices * 4, sum);
    ad_wave_rows<16>(sum);
    if (lane < 4)
#pragma unroll
        for (int i = 0; i < 4; i++) lds[wave * 16 + 4 * i + lane] = sum[i];
    __syncthreads();
    if (threadIdx.x < 16)
        p.part[((size_t)blockIdx.x * p.ntok + tok) * p.n * p.rank_pad + pi * p.rank_pad + r + threadIdx.x] =
            lds[threadIdx.x] + lds[16 + threadIdx.x] + (lds[32 + threadIdx.x] + lds[48 + threadIdx.x]);
}
// Columns of out from it: grid = (blocks of 256 p.up_sets columns of all projections, ntok), block = 256, LDS = 8 L floats.
template <int T, int L> __device__ __forceinline__ void adapter_cols_body(const AdapterArgs& p, float* us) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tok = blockIdx.y;
    int block = blockIdx.x;
    const int pi = ad_projection(p, block, 256 * p.up_sets);
    const int ncol = p.n * p.rank_pad;
    float v[16];
    if (threadIdx.x < 8 * L) {   // (asked for before the id is known; past the rank's padding, and past what adapter_dots wrote: not used)
        const float* at = p.part + (size_t)tok * ncol + pi * p.rank_pad + min((int)threadIdx.x, p.rank_pad - 1);
#pragma unroll
        for (int s = 0; s < 16; s++) v[s] = s < p.slices ? at[(size_t)s * p.ntok * ncol] : 0.f;
    }
    const u32 id = p.ids[tok];
    const size_t orow = (size_t)tok * p.rows[pi];
    if (id >= (u32)p.n_adapter) return ad_copy(p, pi, orow, block * 256 * p.up_sets + (int)threadIdx.x, 256, p.up_sets);   // uniform
    const int rank = ad_rank(p, id);
    int col = block * 256 * p.up_sets + wave * 64;
    AdColumns<T, L> c;
    if (col < p.rows[pi]) c.load(p, pi, id, orow, col);
    if (threadIdx.x < 8 * L) {
        float t = 0.f;
        if ((int)threadIdx.x < rank) {
#pragma unroll
            for (int s = 0; s < 16; s++) t += v[s];
            t *= p.scale ? p.scale[id] : 1.f;
        }
        us[threadIdx.x] = t;
    }
    __syncthreads();
    float u[8];
    ad_take_u<L>(p, us, u);
    for (int s = 0; s < p.up_sets && col < p.rows[pi]; s++, col += 256) {
        if (s) c.load(p, pi, id, orow, col);
        c.finish(p, pi, orow, col, rank, u);
    }
}
