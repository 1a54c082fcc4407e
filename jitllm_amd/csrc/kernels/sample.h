// A token a row of logits (jl_sample_dev): temperature, the k largest, the nucleus, those near the largest, and one of them by a given number.
//
//   w_i = e^((x_i - max) / T)            order: x descending, index ascending
//   kept = the shortest of: the first k; the shortest beginning whose sum reaches top_p of the first k's sum; those with w_i >= min_p; one at least
//   token = the first kept i, by index, whose sum of the kept w up to i exceeds u W
//
// Whole numbers: w is kept as round(w 2^44) in 64 bits, so sums do not depend on their order and a border falls the same way whatever threads met it
// (in f32 one row in a few thousand of a flat distribution would take a neighbour's token).  w itself is f64's, to 2^-44.
//
// The order is made only where it decides.  Four launches, rows cut into slices so that a few rows fill the chip:
//   sample_max     a slice's largest, its first place, and how many candidates
//   sample_bins    counts (and sums, where only the nucleus cuts) over 2048 bins of the distance from the largest, 64 of them a temperature
//   sample_gather  from the bins: how far the kept can reach.  Up to 1024 candidates there: all of them into a list (LIST).  More: each slice's sum of what is kept
//                  for sure, and the candidates of the bin in which the cut falls into the list (LARGE); a cut in a bin of more, or a nucleus of more than 1024 of
//                  the k largest: SLOW.  (A bin has about n / 64 of the density of x / T: 262144 distinct values of spread 2 at T = 1.5, a nucleus of 0.95, are there,
//                  64 such rows 793 us for 81 at T = 1)
//   sample_take    a workgroup a row: the list sorted, the cuts, and the token, from the list or from the slice in which u falls.  SLOW rows are done here from
//                  the start: the cut's bin divided again by keys and, where one key is left, by index.
//
// One row: four launches, each a few trips to memory (131072 values, the 40 largest and their nucleus: 19 us, 3.5 + 4.4 + 6.4 + 5.1).  Many: three reads of the row, the weights
// behind the largest, the cut behind the weights' sums, and f64 beside them (256 x 200003, a nucleus of 0.95: 180 us back to back, by trace 44 + 66 + 75 + 19; a read alone is 43).
#pragma once
#include "args.h"
#include "common.h"
#include "norm_rows.h"

#pragma clang fp contract(off)

#define JL_SA_FEW 64
#define JL_SA_DONE 0
#define JL_SA_LISTED 1
#define JL_SA_LARGE 2
#define JL_SA_SLOW 3

// The row's values as ordered whole numbers; 0: no candidate.
__device__ __forceinline__ u32 sample_key(float x) {
    const u32 b = __float_as_uint(x + 0.0f);   // (-0 is 0)
    return x > -__builtin_inff() ? b ^ ((u32)((i32)b >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float sample_value(u32 k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// a b + c, c in scalar registers (the compiler makes the two-address form of it, with a copy of c each).
__device__ __forceinline__ double sample_fma(double a, double b, double c) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
    return d;
}

struct SampleRow {
    float max;        // of the row
    double a;         // log2 e / temperature
    float fine;       // bins a unit of x
    // e^((x - max) / T) = 2^y, y = n + f with |f| <= 1/2: 2^f as 1 + f q(f), q of the eighth degree through (2^f - 1) / f at the nine Chebyshev points: off by
    // under 2^-44.  x is a candidate.  (Largest infinities: their difference is no number, and counts as 0.)
    __device__ double weight(float x) const {
        const double y = fmax(fmin(((double)x - (double)max) * a, 0.0), -1000.0);
        const double z = y + 0x1.8p52, f = y - (z - 0x1.8p52);     // (n in z's low bits)
        double p = sample_fma(f, 0x1.b638718fee5a8p-24, 0x1.63d136366db24p-20);
        p = sample_fma(p, f, 0x1.ffcb95269d85ap-17);
        p = sample_fma(p, f, 0x1.4308ac85aa947p-13);
        p = sample_fma(p, f, 0x1.5d87fe86f82cdp-10);
        p = sample_fma(p, f, 0x1.3b2ab7181b755p-7);
        p = sample_fma(p, f, 0x1.c6b08d7047e8bp-5);
        p = sample_fma(p, f, 0x1.ebfbdff823cedp-3);
        p = sample_fma(p, f, 0x1.62e42fefa39efp-1);
        return __builtin_ldexp(__builtin_fma(p, f, 1.0), (int)(u32)__builtin_bit_cast(uint64_t, z));
    }
    static __device__ uint64_t rounded(double w) { return __builtin_bit_cast(uint64_t, __builtin_fma(w, 0x1p44, 0x1p52)) & ((1ull << 52) - 1); }   // the low bits of w 2^44 + 2^52
    __device__ uint64_t whole(float x) const { return rounded(weight(x)); }
    __device__ uint64_t kept(float x, float low) const {   // 0 where min_p takes it out
        const double w = weight(x);
        return low > 0.f && !(w >= (double)low) ? 0 : rounded(w);
    }
    __device__ u32 bin(float x) const {          // falls as x rises
        const float d = __builtin_fmaf(x, -0.5f, 0.5f * max) * (2.f * fine);        // (by halves: max - x may be beyond f32; infinities apart: NaN or infinite)
        return x == max ? 0u : d < (float)(JL_SA_BINS - 1) ? (u32)d : (u32)JL_SA_BINS - 1u;
    }
};

// Four values from element `at` on, `left` of them there: a wide load wherever the row starts.
__device__ __forceinline__ f32x4 sample_load(const SampleArgs& p, size_t at, int left) {
    f32x4 v;
    if (left < 4) return norm_load<false>(p.logits, at, p.type, left);
    if (p.type == JL_F32) {
        const u32x4 w = ((const u32x4_a4*)((const float*)p.logits + at))->v;
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __uint_as_float(w[i]);
    } else {
        const u32x2 w = ((const u32x2_a2*)((const uint16_t*)p.logits + at))->v;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const u32 h = i % 2 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu;
            v[i] = p.type == JL_F16 ? half_bits_to_f32((uint16_t)h) : __uint_as_float(h << 16);
        }
    }
    return v;
}
// f(value, index) for the elements from to end of a row, four in a row a lane, 4 * LANES together; four such loads are on their way.
template <int LANES, class F> __device__ __forceinline__ void sample_range(const SampleArgs& p, size_t row, int from, int end, int lane, F f) {
    const size_t at = row * p.stride;
    int i = from + 4 * lane;
    for (; i + 3 * 4 * LANES + 4 <= end; i += 4 * 4 * LANES) {
        f32x4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = sample_load(p, at + i + k * 4 * LANES, 4);
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) f(v[k][j], (u32)(i + k * 4 * LANES + j));
    }
    for (; i < end; i += 4 * LANES) {
        const f32x4 v = sample_load(p, at + i, end - i);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < end) f(v[j], (u32)(i + j));
    }
}
// A slice (a workgroup's) and the part of it that a wavefront has.
__device__ __forceinline__ void sample_slice(const SampleArgs& p, int slice, int& from, int& end) {
    from = min(slice * p.slice_len, p.n);
    end = min(from + p.slice_len, p.n);
}
__device__ __forceinline__ void sample_part(const SampleArgs& p, int part, int& from, int& end) {
    int s0, s1;
    sample_slice(p, part / JL_SA_PARTS, s0, s1);
    from = min(s0 + part % JL_SA_PARTS * p.part_len, s1);
    end = min(from + p.part_len, s1);
}

__device__ __forceinline__ uint64_t sample_scan64(uint64_t v) {      // inclusive sums over a wavefront
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}
// ... over WAVES of them; total to every thread.  LDS: WAVES words.
template <int WAVES> __device__ __forceinline__ uint64_t sample_scan(uint64_t* lds, uint64_t v, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = sample_scan64(v);
    __syncthreads();
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    total = 0;
    uint64_t before = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        before += w < wave ? lds[w] : 0;
        total += lds[w];
    }
    return v + before;
}
__device__ __forceinline__ u32 sample_wave_max(u32 v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = max(v, (u32)__shfl_xor((int)v, d, 64));
    return v;
}

// Settings of a row, and what sample_max found.
struct SampleSet {
    SampleRow r;
    u32 best, first, valid;   // key of the largest, its first place; candidates
    u32 k;                    // 0: not a cut
    float p, low;
    bool greedy, nucleus;
};
__device__ __forceinline__ SampleSet sample_set(const SampleArgs& p, size_t row) {
    SampleSet s;
    const SampleRowWs& ws = ((const SampleRowWs*)p.ws)[row];
    const int lane = threadIdx.x & 63;     // a slice a lane
    const u32 top = lane < p.slices ? ws.top[lane] : 0u, at = lane < p.slices ? ws.at[lane] : 0u;
    const float t = p.temperature ? p.temperature[row] : 1.f;
    const u32 k = p.top_k ? p.top_k[row] : 0u;
    s.p = p.top_p ? p.top_p[row] : 1.f;
    s.low = p.min_p ? p.min_p[row] : 0.f;
    s.valid = lane < p.slices ? ws.many[lane] : 0u;
    s.best = sample_wave_max(top);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) s.valid += (u32)__shfl_xor((int)s.valid, d, 64);
    s.best = (u32)__builtin_amdgcn_readfirstlane((i32)s.best);
    s.valid = (u32)__builtin_amdgcn_readfirstlane((i32)s.valid);
    s.first = (u32)__builtin_amdgcn_readlane((i32)at, (int)__builtin_ctzll(__ballot(top == s.best)));   // the first slice that has it
    s.greedy = s.best == 0 || !(t > 0.f) || s.low > 1.f;      // (nothing reaches a min_p above one: the first is left)
    s.r.max = sample_value(s.best);
    s.r.a = fmax(1.4426950408889634074 / (double)t, 0x1p-200);      // (not 0: at an infinite temperature an infinite distance still weighs nothing, finite ones 1)
    s.r.fine = fminf(64.f / t, 1e30f);
    s.k = k < s.valid ? k : 0u;
    s.nucleus = s.p < 1.f;
    return s;
}
// The smallest value that `holds` is true of, where it is true of all values from there on, or NaN: of none, not of an infinity either.  64 keys at a time.
template <class F> __device__ __forceinline__ float sample_edge(F holds) {
    u32 lo = 0x007fffffu;      // (the key of -infinity: false)
    const u32 lane = threadIdx.x & 63;
#pragma unroll
    for (int shift = 26; ; shift = max(shift - 6, 0)) {
        const uint64_t key = (uint64_t)lo + ((uint64_t)(lane + 1) << shift);
        const uint64_t yes = __ballot(key > 0xff800000u || holds(sample_value((u32)key)));   // (the key of +infinity)
        const u32 n = yes ? (u32)__builtin_ctzll(yes) : 64u;
        if (shift == 0) return sample_value(lo + n + 1);      // (0xff800001 is a NaN)
        lo += n << shift;
    }
}

// grid = (slices, rows), block = 512.  LDS: 3 words.
__device__ __forceinline__ void sample_max_body(const SampleArgs& p, u32* lds) {
    const size_t row = blockIdx.y;
    SampleRowWs& ws = ((SampleRowWs*)p.ws)[row];
    const int slice = blockIdx.x;
    for (int i = slice * 512 + threadIdx.x; i < JL_SA_BINS; i += p.slices * 512) {
        ws.counts[i] = 0;
        ws.sums[i] = 0;
    }
    if (slice == 0 && threadIdx.x == 0) ws.fill = 0;
    if (threadIdx.x < 3) lds[threadIdx.x] = threadIdx.x == 1 ? ~0u : 0u;
    __syncthreads();
    int from, end;
    sample_slice(p, slice, from, end);
    u32 top = 0, many = 0, at = ~0u;
    sample_range<512>(p, row, from, end, threadIdx.x, [&](float x, u32 i) {
        const u32 k = sample_key(x);
        many += k != 0;
        at = k > top ? i : at;
        top = max(top, k);
    });
    const u32 best = sample_wave_max(top);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) many += (u32)__shfl_xor((int)many, d, 64);
    if ((threadIdx.x & 63) == 0) {
        atomicMax(&lds[0], best);
        atomicAdd(&lds[2], many);
    }
    __syncthreads();
    if (top && top == lds[0]) atomicMin(&lds[1], at);
    __syncthreads();
    if (threadIdx.x == 0) {
        ws.top[slice] = lds[0];
        ws.at[slice] = lds[1];
        ws.many[slice] = lds[2];
    }
}

// grid = (slices, rows), block = 512.  LDS: counts [BINS], sums [BINS].
__device__ __forceinline__ void sample_bins_body(const SampleArgs& p, u32* counts, uint64_t* sums) {
    const size_t row = blockIdx.y;
    const SampleSet s = sample_set(p, row);
    if (s.greedy || !(s.k || s.nucleus || s.low > 0.f)) return;
    SampleRowWs& ws = ((SampleRowWs*)p.ws)[row];
    const bool weighs = s.nucleus && !s.k;
    for (int i = threadIdx.x; i < JL_SA_BINS; i += 512) {
        counts[i] = 0;
        if (weighs) sums[i] = 0;
    }
    __syncthreads();
    int from, end;
    sample_slice(p, blockIdx.x, from, end);
    // (the last bin's count is what is left over, its sum nothing)
    if (weighs)
        sample_range<512>(p, row, from, end, threadIdx.x, [&](float x, u32) {
            const u32 b = x > -__builtin_inff() ? s.r.bin(x) : (u32)JL_SA_BINS;
            if (b < JL_SA_BINS - 1) {
                atomicAdd(&counts[b], 1u);
                atomicAdd((unsigned long long*)&sums[b], (unsigned long long)s.r.whole(x));
            }
        });
    else
        sample_range<512>(p, row, from, end, threadIdx.x, [&](float x, u32) {
            const u32 b = x > -__builtin_inff() ? s.r.bin(x) : (u32)JL_SA_BINS;
            if (b < JL_SA_BINS - 1) atomicAdd(&counts[b], 1u);
        });
    __syncthreads();
    for (int i = threadIdx.x; i < JL_SA_BINS - 1; i += 512) {
        const u32 c = counts[i];
        if (c) {
            atomicAdd(&ws.counts[i], c);
            if (weighs && sums[i]) atomicAdd((unsigned long long*)&ws.sums[i], (unsigned long long)sums[i]);
        }
    }
}

// grid = (slices, rows), block = 512.  LDS: 8 words of 8 bytes, then 10 of 4, and a list of keys and of places.
__device__ __forceinline__ void sample_gather_body(const SampleArgs& p, uint64_t* scan, u32* told, u32* keys, u32* places) {
    const size_t row = blockIdx.y;
    const SampleSet s = sample_set(p, row);
    SampleRowWs& ws = ((SampleRowWs*)p.ws)[row];
    const bool writes = blockIdx.x == 0 && threadIdx.x == 0;
    if (s.greedy) {
        if (writes) ws.mode = JL_SA_DONE;
        return;
    }
    // The bin that min_p ends in, or one behind it: -ln(min_p) temperatures, 64 bins each.
    const u32 low_bin = s.low > 0.f ? (u32)fminf((float)(JL_SA_BINS - 1), -__logf(s.low) * 64.f * 1.0001f + 2.f) : (u32)JL_SA_BINS - 1;
    u32 mode = JL_SA_LARGE, cut = JL_SA_BINS, before = 0;    // the bin of the cut (LARGE) or the last bin (LISTED); candidates before it
    uint64_t mass = 0;
    if (s.k || s.nucleus || s.low > 0.f) {
        constexpr int PER = JL_SA_BINS / 512;
        const bool weighs = s.nucleus && !s.k;      // (the bins have sums)
        const int b0 = PER * threadIdx.x;
        u32 c[PER];
        uint64_t m[PER], cs = 0, ms = 0, all, mass_all = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            c[j] = ws.counts[b0 + j];
            m[j] = weighs ? ws.sums[b0 + j] : 0;
            cs += c[j];
            ms += m[j];
        }
        if (threadIdx.x < 8) told[threadIdx.x] = threadIdx.x == 0 ? (u32)JL_SA_BINS : 0u;
        uint64_t cb = sample_scan<8>(scan, cs, all) - cs, mb = 0;
        if (weighs) mb = sample_scan<8>(scan, ms, mass_all) - ms;
        const double reach = (double)s.p * (double)mass_all;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const u32 b = b0 + j, n = b == JL_SA_BINS - 1 ? s.valid - (u32)cb : c[j];      // (the last bin has what is left over)
            const uint64_t ce = cb + n, me = mb + m[j];
            const bool crossed = s.k ? ce >= s.k && cb < s.k : s.nucleus && n && (double)me >= reach && !(cb && (double)mb >= reach);
            if (crossed) {
                told[0] = b;
                told[1] = (u32)cb;
                told[2] = (u32)ce;
                told[3] = (u32)mb;
                told[4] = (u32)(mb >> 32);
            }
            if (b == low_bin) told[5] = (u32)ce;
            cb = ce;
            mb = me;
        }
        __syncthreads();
        cut = told[0];
        before = told[1];
        mass = (uint64_t)told[4] << 32 | told[3];
        const u32 through = told[2], low_through = told[5];
        // (a list is sorted twice: from JL_SA_FEW on, or so, its cut and the parts' sums are faster; 200 of 131072 13.4 us against 10.5)
        const u32 few = s.k && s.nucleus ? JL_SA_LIST : JL_SA_FEW;
        if (s.low > 0.f && low_bin < cut && !(s.k && s.nucleus)) {   // min_p ends first
            mode = low_through <= few ? JL_SA_LISTED : JL_SA_LARGE;
            cut = mode == JL_SA_LISTED ? low_bin : (u32)JL_SA_BINS;
        } else if (cut < JL_SA_BINS) {
            mode = through <= few ? JL_SA_LISTED : s.k && s.nucleus ? JL_SA_SLOW : through - before <= JL_SA_LIST ? JL_SA_LARGE : JL_SA_SLOW;
        }
        if (writes) ws.all = mass_all;
    }
    if (writes) {
        ws.mode = mode;
        ws.bin = cut;
        ws.before = before;
        ws.mass = mass;
    }
    if (mode == JL_SA_SLOW) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, part = blockIdx.x * JL_SA_PARTS + wave;
    int from, end;
    sample_part(p, part, from, end);
    // by value: what goes into the list, from `list` on and not from `below` on; what is kept for sure, from `sure` on (min_p's border in it; NaN: nothing, where the
    // cut is in the largest's bin, which may hold infinities)
    const bool cuts = cut < JL_SA_BINS;
    auto append = [&](float x, u32 i) {
        const u32 at = atomicAdd(&told[8], 1u);
        if (at < JL_SA_LIST) {
            keys[at] = sample_key(x);
            places[at] = i;
        }
    };
    // the workgroup's list behind those of the others (a word's atomic add an element, from all workgroups, took half of the launch)
    auto flush = [&]() {
        __syncthreads();
        const u32 n = min(told[8], (u32)JL_SA_LIST);
        if (threadIdx.x == 0) told[9] = n ? atomicAdd(&ws.fill, n) : 0u;
        __syncthreads();
        for (u32 i = threadIdx.x; i < n; i += 512) {
            const u32 at = told[9] + i;
            if (at < JL_SA_LIST) {
                ws.key[at] = keys[i];
                ws.idx[at] = places[i];
            }
        }
    };
    if (threadIdx.x == 0) told[8] = 0;
    __syncthreads();
    uint64_t sum = 0;
    float list = sample_edge([&](float x) { return s.r.bin(x) <= cut; });
    if (mode == JL_SA_LISTED) {
        sample_range<64>(p, row, from, end, lane, [&](float x, u32 i) {
            if (x >= list) append(x, i);
        });
        flush();
        return;
    }
    const float below = cuts ? sample_edge([&](float x) { return s.r.bin(x) < cut; }) : list;
    float sure = below;
    if (s.low > 0.f) {
        const float edge = sample_edge([&](float x) { return s.r.weight(x) >= (double)s.low; });
        if (edge > below) sure = edge;
    }
    if (!cuts) list = sure;
    sample_range<64>(p, row, from, end, lane, [&](float x, u32 i) {
        if (x >= list) {
            if (x >= sure) sum += s.r.whole(x);
            else if (!(x >= below)) append(x, i);
        }
    });
    if (cuts) flush();
    if (mode == JL_SA_LARGE) {
        sum = sample_scan64(sum);
        if (lane == 63) ws.part[part] = sum;
    }
}

// ---- a workgroup a row ------------------------------------------------------------------

#define JL_SA_WAVES 4
#define JL_SA_THREADS 256
struct SampleLds {
    uint64_t mass[JL_SA_BINS];
    u32 count[JL_SA_BINS];
    u32 key[JL_SA_LIST], idx[JL_SA_LIST];
    uint64_t tile[512];              // sums of tiles of a range, or of the row's parts
    uint64_t scan[JL_SA_WAVES];
    uint64_t at_mass;
    u32 at, at_count, at_n, fill, lo, hi, res_key, res_idx;
};
#define JL_SA_TILE 1024      // elements of a workgroup's step in index order

template <class F> __device__ __forceinline__ void sample_each(const SampleArgs& p, size_t row, F f) { sample_range<JL_SA_THREADS>(p, row, 0, p.n, threadIdx.x, f); }

// The first element by index, of those from to end, with crosses(sum of weight(x, i) up to and with it); ~0: none.  weight is 0 for elements that are not in the sum.
template <class W, class X> __device__ __forceinline__ u32 sample_cross(const SampleArgs& p, SampleLds& s, size_t row, int from, int end, W weight, X crosses, uint64_t& total) {
    const int tiles = (end - from + JL_SA_TILE - 1) / JL_SA_TILE, lane = threadIdx.x & 63;   // (512 at most)
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += JL_SA_THREADS) s.tile[i] = 0;
    if (threadIdx.x == 0) s.at = ~0u;
    __syncthreads();
    const size_t at = row * p.stride;
    auto load = [&](int i) { return sample_load(p, at + i, end - i); };
    for (int i = from + 4 * (int)threadIdx.x, k = 0; k < tiles; k++, i += JL_SA_TILE) {
        uint64_t sum = 0;
        if (i < end) {
            const f32x4 v = load(i);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < end) sum += weight(v[j], (u32)(i + j));
        }
        sum = sample_scan64(sum);
        if (lane == 63 && sum) atomicAdd((unsigned long long*)&s.tile[k], (unsigned long long)sum);
    }
    __syncthreads();
    // two tiles a thread
    const uint64_t t0 = s.tile[2 * threadIdx.x], t1 = s.tile[2 * threadIdx.x + 1];
    uint64_t c = sample_scan<JL_SA_WAVES>(s.scan, t0 + t1, total) - t0 - t1;
    bool had = c != 0 && crosses(c);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint64_t t = j ? t1 : t0;
        if (t && !had && crosses(c + t)) {
            s.at = 2 * threadIdx.x + j;
            s.at_mass = c;
            had = true;
        }
        c += t;
    }
    __syncthreads();
    const u32 tile = s.at;
    const uint64_t before = s.at_mass;
    __syncthreads();
    if (tile == ~0u) return ~0u;   // uniform
    if (threadIdx.x == 0) s.at = ~0u;
    const int i = from + (int)tile * JL_SA_TILE + 4 * (int)threadIdx.x;
    uint64_t part[4] = {0, 0, 0, 0}, mine = 0, all;
    if (i < end) {
        const f32x4 v = load(i);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (i + j < end) part[j] = weight(v[j], (u32)(i + j));
            mine += part[j];
        }
    }
    c = before + sample_scan<JL_SA_WAVES>(s.scan, mine, all) - mine;
    had = c != 0 && crosses(c);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (part[j] && !had && crosses(c + part[j])) {
            s.at = (u32)(i + j);
            had = true;
        }
        c += part[j];
    }
    __syncthreads();
    const u32 found = s.at;
    __syncthreads();
    return found;
}

// What is kept: elements not behind (key, idx) in the order.
struct SampleCut {
    u32 key, idx;
    uint64_t mass;     // of those
    __device__ bool keeps(u32 k, u32 i) const { return k > key || (k == key && i <= idx); }
};

// Counts and sums of the bins (bin(x, key) < BINS, or ~0: not in it).
template <class B> __device__ __forceinline__ void sample_count(const SampleArgs& p, SampleLds& s, size_t row, const SampleRow& r, B bin) {
    __syncthreads();
    for (int i = threadIdx.x; i < JL_SA_BINS; i += JL_SA_THREADS) {
        s.mass[i] = 0;
        s.count[i] = 0;
    }
    __syncthreads();
    sample_each(p, row, [&](float x, u32) {
        const u32 k = sample_key(x), b = k ? bin(x, k) : ~0u;
        if (b < JL_SA_BINS) {
            atomicAdd(&s.count[b], 1u);
            atomicAdd((unsigned long long*)&s.mass[b], (unsigned long long)r.whole(x));
        }
    });
    __syncthreads();
}

// The bin in which crosses(count, mass) with the bins up to it is first true, and what lies before it: s.at, s.at_count, s.at_mass, s.at_n.
// None: s.at stays ~0.
template <class X> __device__ __forceinline__ void sample_find(SampleLds& s, u32 count0, uint64_t mass0, X crosses) {
    if (threadIdx.x == 0) s.at = ~0u;
    constexpr int PER = JL_SA_BINS / JL_SA_THREADS;
    const int b0 = PER * threadIdx.x;
    uint64_t c = 0, m = 0, all;
    for (int j = 0; j < PER; j++) {
        c += s.count[b0 + j];
        m += s.mass[b0 + j];
    }
    uint64_t cb = sample_scan<JL_SA_WAVES>(s.scan, c, all) - c + count0, mb = sample_scan<JL_SA_WAVES>(s.scan, m, all) - m + mass0;
    for (int j = 0; j < PER; j++) {
        const u32 cj = s.count[b0 + j];
        const uint64_t mj = s.mass[b0 + j];
        if (cj && crosses((u32)(cb + cj), mb + mj) && !(cb && crosses((u32)cb, mb))) {
            s.at = b0 + j;
            s.at_count = (u32)cb;
            s.at_mass = mb;
            s.at_n = cj;
        }
        cb += cj;
        mb += mj;
    }
    __syncthreads();
}

// A SLOW row's cut: the last element kept, in the order, such that crosses(count, mass) up to it is first true.  False: nothing crosses.
template <class X> __device__ __forceinline__ bool sample_cut(const SampleArgs& p, SampleLds& s, size_t row, const SampleRow& r, X crosses, SampleCut& cut) {
    sample_count(p, s, row, r, [&](float x, u32) { return r.bin(x); });
    sample_find(s, 0, 0, crosses);
    if (s.at == ~0u) return false;   // uniform
    const u32 bin0 = s.at;
    u32 n = s.at_n, count = s.at_count, klo = 1, khi = ~0u;
    uint64_t mass = s.at_mass;
    __syncthreads();
    if (n > JL_SA_LIST) {
        if (threadIdx.x == 0) {
            s.lo = ~0u;
            s.hi = 0;
        }
        __syncthreads();
        u32 lo = ~0u, hi = 0;
        sample_each(p, row, [&](float x, u32) {
            const u32 k = sample_key(x);
            if (k && r.bin(x) == bin0) {
                lo = min(lo, k);
                hi = max(hi, k);
            }
        });
        atomicMin(&s.lo, lo);
        atomicMax(&s.hi, hi);
        __syncthreads();
        klo = s.lo;
        khi = s.hi;
        while (n > JL_SA_LIST && klo < khi) {
            int shift = 0;
            while ((khi - klo) >> shift >= JL_SA_BINS) shift++;
            sample_count(p, s, row, r, [&](float x, u32 k) { return r.bin(x) == bin0 && k >= klo && k <= khi ? (khi - k) >> shift : ~0u; });
            sample_find(s, count, mass, crosses);
            n = s.at_n;
            count = s.at_count;
            mass = s.at_mass;
            const u32 top = khi - (s.at << shift), width = (1u << shift) - 1;
            __syncthreads();
            klo = top - klo > width ? top - width : klo;
            khi = top;
        }
    }
    if (n > JL_SA_LIST) {   // one key, many times: by index
        const uint64_t w0 = r.whole(sample_value(klo));
        uint64_t total;
        // counted: sums of 1, the crossing by count and mass
        cut.idx = sample_cross(p, s, row, 0, p.n, [&](float x, u32) { return (uint64_t)(sample_key(x) == klo); },
                               [&](uint64_t c) { return crosses(count + (u32)c, mass + c * w0); }, total);
        cut.key = klo;
        // how many that are: again over those up to it
        const u32 last = cut.idx;
        sample_cross(p, s, row, 0, p.n, [&](float x, u32 i) { return (uint64_t)(sample_key(x) == klo && i <= last); }, [&](uint64_t) { return false; }, total);
        cut.mass = mass + total * w0;
        return true;
    }
    __syncthreads();
    if (threadIdx.x == 0) s.fill = 0;
    __syncthreads();
    sample_each(p, row, [&](float x, u32 i) {
        const u32 k = sample_key(x);
        if (k && k >= klo && k <= khi && r.bin(x) == bin0) {
            const u32 at = atomicAdd(&s.fill, 1u);
            if (at < JL_SA_LIST) {
                s.key[at] = k;
                s.idx[at] = i;
            }
        }
    });
    __syncthreads();
    // an element at a time: those ahead of it, and their weights
    uint64_t* const w = s.mass;   // (the bins have been read)
    for (u32 i = threadIdx.x; i < n; i += JL_SA_THREADS) w[i] = r.whole(sample_value(s.key[i]));
    __syncthreads();
    for (u32 e = threadIdx.x; e < n; e += JL_SA_THREADS) {
        const u32 k = s.key[e], i = s.idx[e];
        u32 ahead = 0;
        uint64_t m = 0;
        for (u32 j = 0; j < n; j++) {
            const bool is = s.key[j] > k || (s.key[j] == k && s.idx[j] < i);
            ahead += is;
            m += is ? w[j] : 0;
        }
        const u32 cb = count + ahead;
        if (crosses(cb + 1, mass + m + w[e]) && !(cb && crosses(cb, mass + m))) {
            s.res_key = k;
            s.res_idx = i;
            s.at_mass = mass + m + w[e];
        }
    }
    __syncthreads();
    cut.key = s.res_key;
    cut.idx = s.res_idx;
    cut.mass = s.at_mass;
    __syncthreads();
    return true;
}

// 64 NQ elements of a workgroup's (Q = 4), or a wavefront's (Q = 1) list, ascending; element e + THREADS q is thread e's q-th.  The network needs as many
// as n rounded up to a power of two.
template <int NQ, bool WG> __device__ __forceinline__ void sample_sort(uint64_t* lds, uint64_t (&v)[NQ], u32 n) {
    constexpr u32 T = WG ? JL_SA_THREADS : 64;
    const u32 tid = WG ? threadIdx.x : threadIdx.x & 63;
    u32 size = 64;
    while (WG && size < n) size *= 2;
    for (u32 k = 2; k <= size; k *= 2)
        for (u32 j = k / 2; j; j /= 2) {
            if (j >= T) {      // between the thread's own
#pragma unroll
                for (u32 q = 0; q < NQ; q++) {
                    const u32 o = q ^ (j / T);
                    if (o > q && o < NQ) {
                        const bool up = ((tid + T * q) & k) == 0;
                        const uint64_t a = v[q], b = v[o];
                        const bool turn = up ? a > b : a < b;
                        v[q] = turn ? b : a;
                        v[o] = turn ? a : b;
                    }
                }
                continue;
            }
            if (WG && j >= 64) {
                __syncthreads();
#pragma unroll
                for (int q = 0; q < NQ; q++) lds[tid + T * q] = v[q];
                __syncthreads();
            }
#pragma unroll
            for (int q = 0; q < NQ; q++) {
                const uint64_t o = WG && j >= 64 ? lds[(tid ^ j) + T * q] : (uint64_t)__shfl_xor((unsigned long long)v[q], (int)j, 64);
                const bool up = ((tid + T * q) & k) == 0, lower = (tid & j) == 0;
                v[q] = (up == lower) == (v[q] < o) ? v[q] : o;
            }
        }
    if (WG) __syncthreads();
}

// The token of a LISTED row, or (LARGE) the cut's element and the kept of the list into their parts' sums.  NQ elements a thread; WG false: by one wavefront.
template <int NQ, bool WG, class G>
__device__ __forceinline__ void sample_list(const SampleArgs& p, SampleLds& s, const SampleRowWs& ws, const SampleSet& set, float u, u32 n, SampleCut& cut, G give) {
    constexpr u32 T = WG ? JL_SA_THREADS : 64;
    const u32 tid = WG ? threadIdx.x : threadIdx.x & 63;
    const SampleRow& r = set.r;
    const bool large = ws.mode == JL_SA_LARGE;
    const uint64_t base = large ? ws.mass : 0, row_all = ws.all;
    const u32 before = large ? ws.before : 0;
    uint64_t v[NQ], w[NQ], through[NQ];
    // descending by key, ascending by index: ascending by the key's complement
#pragma unroll
    for (int q = 0; q < NQ; q++) v[q] = tid + T * q < n ? (uint64_t)~ws.key[tid + T * q] << 32 | ws.idx[tid + T * q] : ~0ull;
    sample_sort<NQ, WG>(s.mass, v, n);
    // sums up to and with each, and the number of kept
    uint64_t sum = base;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        w[q] = tid + T * q < n ? r.whole(sample_value(~(u32)(v[q] >> 32))) : 0;
        uint64_t all;
        if (WG) through[q] = sum + sample_scan<JL_SA_WAVES>(s.scan, w[q], all);
        else {
            through[q] = sum + sample_scan64(w[q]);
            all = 0;
        }
        sum += all;
    }
    u32 kept = set.k ? min(n, set.k - before) : n;
    if (set.nucleus) {
        uint64_t all = row_all;
        if (set.k) {
            if (WG) {
                __syncthreads();
#pragma unroll
                for (int q = 0; q < NQ; q++)
                    if (tid + T * q == kept - 1) s.at_mass = through[q];
                __syncthreads();
                all = s.at_mass;
            } else {
                all = __shfl((unsigned long long)through[0], (int)kept - 1, 64);
            }
        }
        const double reach = (double)set.p * (double)all;
        if (WG) {
            __syncthreads();
            if (tid == 0) s.at = kept;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < NQ; q++)
            {
                const uint64_t over = __ballot(tid + T * q < kept && (double)through[q] >= reach);
                if (over && (tid & 63) == (u32)__builtin_ctzll(over)) atomicMin(&s.at, tid + T * q + 1);
            }
            __syncthreads();
            kept = s.at;
        } else {
            const uint64_t over = __ballot(tid < kept && (double)through[0] >= reach);
            if (over) kept = (u32)__builtin_ctzll(over) + 1;
        }
    }
    if (WG && large) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const u32 e = tid + T * q, idx = (u32)v[q];
            if (e == kept - 1) {
                s.res_key = ~(u32)(v[q] >> 32);
                s.res_idx = idx;
            }
            if (e < kept && w[q] && (!(set.low > 0.f) || r.weight(sample_value(~(u32)(v[q] >> 32))) >= (double)set.low)) {
                const u32 slice = idx / (u32)p.slice_len, part = slice * JL_SA_PARTS + (idx - slice * (u32)p.slice_len) / (u32)p.part_len;
                atomicAdd((unsigned long long*)&s.tile[part], (unsigned long long)w[q]);
            }
        }
        __syncthreads();
        cut.key = s.res_key;
        cut.idx = s.res_idx;
        return;
    }
    // those that min_p keeps, by index; the place in the list goes along
    uint64_t by[NQ], mine[NQ], c[NQ], total = 0;
    if (WG) __syncthreads();
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const u32 e = tid + T * q;
        const bool in = e < kept && w[q] && (!(set.low > 0.f) || r.weight(sample_value(~(u32)(v[q] >> 32))) >= (double)set.low);
        if (WG) s.mass[1024 + e] = w[q];
        by[q] = in ? (v[q] & 0xffffffffu) << 32 | e : ~0ull;
    }
    if (WG) __syncthreads();
    sample_sort<NQ, WG>(s.mass, by, n);
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const uint64_t there = WG ? s.mass[1024 + ((u32)by[q] & 1023)] : (uint64_t)__shfl((unsigned long long)w[0], (int)(by[0] & 63), 64);
        mine[q] = by[q] == ~0ull ? 0 : there;
        uint64_t all;
        if (WG) c[q] = total + sample_scan<JL_SA_WAVES>(s.scan, mine[q], all);
        else {
            c[q] = sample_scan64(mine[q]);
            all = __shfl((unsigned long long)c[q], 63, 64);
        }
        total += all;
    }
    const double over = (double)u * (double)total;
    u32 at;      // the first over it, or the last
    if (WG) {
        __syncthreads();
        if (tid == 0) {
            s.at = ~0u;
            s.hi = 0;
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const uint64_t yes = __ballot(mine[q] && (double)c[q] > over), any = __ballot(mine[q] != 0);
            if (yes && (tid & 63) == (u32)__builtin_ctzll(yes)) atomicMin(&s.at, tid + T * q);
            if (any && (tid & 63) == 63u - (u32)__builtin_clzll(any)) atomicMax(&s.hi, tid + T * q);
        }
        __syncthreads();
        at = s.at != ~0u ? s.at : s.hi;
    } else {
        const uint64_t yes = __ballot(mine[0] && (double)c[0] > over), any = __ballot(mine[0] != 0);
        at = (u32)(yes ? __builtin_ctzll(yes) : 63 - __builtin_clzll(any));
    }
#pragma unroll
    for (int q = 0; q < NQ; q++)
        if (tid + T * q == at) give((u32)(by[q] >> 32), (double)mine[q] / (double)total);
}

// A LARGE row's cut among the list, without sorting it: its keys' range in 256, and the few elements of the one in which the cut falls in order, by one
// wavefront.  What is kept goes into the parts' sums.  False: that one has more than 64 (ties).
__device__ __forceinline__ bool sample_near(const SampleArgs& p, SampleLds& s, const SampleRowWs& ws, const SampleSet& set, u32 n, SampleCut& cut) {
    const u32 tid = threadIdx.x;
    const SampleRow& r = set.r;
    if (tid == 0) {
        s.lo = ~0u;
        s.hi = 0;
        s.at = ~0u;
        s.fill = 0;
    }
    s.mass[tid] = 0;
    s.count[tid] = 0;
    u32 key[4], idx[4], lo = ~0u, hi = 0;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const u32 e = tid + JL_SA_THREADS * q;
        key[q] = e < n ? ws.key[e] : 0u;
        idx[q] = e < n ? ws.idx[e] : 0u;
        lo = min(lo, key[q] - 1u);       // (0: none)
        hi = max(hi, key[q]);
    }
    lo = ~sample_wave_max(~lo);
    hi = sample_wave_max(hi);
    __syncthreads();
    if ((tid & 63) == 0) {
        atomicMin(&s.lo, lo);
        atomicMax(&s.hi, hi);
    }
    __syncthreads();
    hi = s.hi;
    const u32 range = hi - (s.lo + 1u);
    const int shift = max(0, 32 - (int)__builtin_clz(range | 1u) - 8);
    uint64_t w[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        if (!key[q]) continue;
        w[q] = r.whole(sample_value(key[q]));
        const u32 b = (hi - key[q]) >> shift;
        atomicAdd(&s.count[b], 1u);
        atomicAdd((unsigned long long*)&s.mass[b], (unsigned long long)w[q]);
    }
    __syncthreads();
    const u32 c = s.count[tid];
    const uint64_t m = s.mass[tid];
    uint64_t all;
    const uint64_t ce = ws.before + sample_scan<JL_SA_WAVES>(s.scan, c, all), me = ws.mass + sample_scan<JL_SA_WAVES>(s.scan, m, all);
    const double reach = (double)set.p * (double)ws.all;
    const uint64_t cb = ce - c, mb = me - m;
    const bool crossed = c && (set.k ? ce >= set.k && cb < set.k : (double)me >= reach && !(cb && (double)mb >= reach));
    if (crossed) {
        s.at = tid;
        s.at_count = (u32)cb;
        s.at_mass = mb;
        s.at_n = c;
    }
    __syncthreads();
    const u32 at = s.at, many = s.at_n, before = s.at_count;
    const uint64_t mass = s.at_mass;
    if (at == ~0u || many > 64) {
        __syncthreads();
        return false;
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
        if (key[q] && (hi - key[q]) >> shift == at) {
            const u32 to = atomicAdd(&s.fill, 1u);
            s.key[to] = key[q];
            s.idx[to] = idx[q];
        }
    __syncthreads();
    if (tid < 64) {
        uint64_t v[1] = {tid < many ? (uint64_t)~s.key[tid] << 32 | s.idx[tid] : ~0ull};
        sample_sort<1, false>(s.mass, v, many);
        const uint64_t mine = tid < many ? r.whole(sample_value(~(u32)(v[0] >> 32))) : 0, through = mass + sample_scan64(mine);
        u32 last = many - 1;
        if (set.k) last = min(last, set.k - before - 1);
        else {
            const uint64_t over = __ballot(tid < many && (double)through >= reach);
            if (over) last = (u32)__builtin_ctzll(over);
        }
        if (tid == last) {
            s.res_key = ~(u32)(v[0] >> 32);
            s.res_idx = (u32)v[0];
        }
    }
    __syncthreads();
    cut.key = s.res_key;
    cut.idx = s.res_idx;
#pragma unroll
    for (int q = 0; q < 4; q++)
        if (key[q] && cut.keeps(key[q], idx[q]) && w[q] && (!(set.low > 0.f) || r.weight(sample_value(key[q])) >= (double)set.low)) {
            const u32 slice = idx[q] / (u32)p.slice_len, part = slice * JL_SA_PARTS + (idx[q] - slice * (u32)p.slice_len) / (u32)p.part_len;
            atomicAdd((unsigned long long*)&s.tile[part], (unsigned long long)w[q]);
        }
    __syncthreads();
    return true;
}

// grid = rows, block = 256.
__device__ __forceinline__ void sample_take_body(const SampleArgs& p, SampleLds& s) {
    const size_t row = blockIdx.x;
    const SampleRowWs& ws = ((const SampleRowWs*)p.ws)[row];
    const u32 tid = threadIdx.x, mode = ws.mode, fill = min(ws.fill, (u32)JL_SA_LIST), bin = ws.bin;
    const float u = p.u[row];
    const SampleSet set = sample_set(p, row);
    const SampleRow& r = set.r;
    auto give = [&](u32 token, double prob) {
        p.token[row] = token;
        if (p.prob) p.prob[row] = (float)prob;
    };
    if (set.greedy) {
        if (tid == 0) give(set.best ? set.first : (u32)p.n, set.best ? 1.0 : 0.0);
        return;
    }
    SampleCut cut = {1u, ~0u, 0};
    if (mode == JL_SA_LISTED) {
        if (fill <= 64) {
            if (tid < 64) sample_list<1, false>(p, s, ws, set, u, fill, cut, give);
        } else if (fill <= JL_SA_THREADS) {
            sample_list<1, true>(p, s, ws, set, u, fill, cut, give);
        } else {
            sample_list<4, true>(p, s, ws, set, u, fill, cut, give);
        }
        return;
    }
    const int parts = p.slices * JL_SA_PARTS;
    if (mode == JL_SA_LARGE) {
        for (int i = tid; i < 512; i += JL_SA_THREADS) s.tile[i] = i < parts ? ws.part[i] : 0;
        __syncthreads();
        if (bin < JL_SA_BINS && !sample_near(p, s, ws, set, fill, cut)) {
            if (fill <= JL_SA_THREADS) sample_list<1, true>(p, s, ws, set, u, fill, cut, give);
            else sample_list<4, true>(p, s, ws, set, u, fill, cut, give);
        }
    } else {
        if (set.k) sample_cut(p, s, row, r, [&](u32 c, uint64_t) { return c >= set.k; }, cut);
        if (set.nucleus) {
            uint64_t all = cut.mass;
            if (!set.k) {
                uint64_t sum = 0;
                sample_each(p, row, [&](float x, u32) { sum += sample_key(x) ? r.whole(x) : 0; });
                sample_scan<JL_SA_WAVES>(s.scan, sum, all);
            }
            const double reach = (double)set.p * (double)all;
            sample_cut(p, s, row, r, [&](u32, uint64_t m) { return (double)m >= reach; }, cut);
        }
        __syncthreads();
        for (int i = tid; i < 512; i += JL_SA_THREADS) s.tile[i] = 0;
        __syncthreads();
        for (int i = (int)tid >> 6; i < parts; i += JL_SA_WAVES) {
            int from, end;
            sample_part(p, i, from, end);
            uint64_t sum = 0;
            sample_range<64>(p, row, from, end, tid & 63, [&](float x, u32 e) {
                const u32 key = sample_key(x);
                if (key && cut.keeps(key, e)) sum += r.kept(x, set.low);
            });
            sum = sample_scan64(sum);
            if ((tid & 63) == 63) s.tile[i] = sum;
        }
        __syncthreads();
    }
    // the part in which the sum exceeds u of it, two parts a thread; and the token there
    const uint64_t t0 = s.tile[2 * tid], t1 = s.tile[2 * tid + 1];
    uint64_t total, c = sample_scan<JL_SA_WAVES>(s.scan, t0 + t1, total) - t0 - t1;
    const double over = (double)u * (double)total;
    if (tid == 0) {
        s.at = ~0u;
        s.hi = 0;
    }
    __syncthreads();
    bool had = c && (double)c > over;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint64_t t = j ? t1 : t0;
        const uint64_t any = __ballot(t != 0);
        if (any && (tid & 63) == 63u - (u32)__builtin_clzll(any)) atomicMax(&s.hi, 2 * tid + j);
        if (t && !had && (double)(c + t) > over) {
            s.at = 2 * tid + j;
            s.at_mass = c;
            had = true;
        }
        c += t;
    }
    __syncthreads();
    const bool found = s.at != ~0u;
    const uint64_t before = s.at_mass;
    int from, end;
    sample_part(p, (int)(found ? s.at : s.hi), from, end);
    __syncthreads();
    auto weight = [&](float x, u32 i) -> uint64_t {
        const u32 key = sample_key(x);
        return key && cut.keeps(key, i) ? r.kept(x, set.low) : 0;
    };
    u32 token = ~0u;
    uint64_t in;
    if (found) token = sample_cross(p, s, row, from, end, weight, [&](uint64_t m) { return (double)(before + m) > over; }, in);
    if (token == ~0u) {   // u is 1 or more, or no number: the last that is kept
        if (tid == 0) s.hi = 0;
        __syncthreads();
        u32 at = 0;
        sample_range<JL_SA_THREADS>(p, row, from, end, tid, [&](float x, u32 i) { at = weight(x, i) ? max(at, i) : at; });
        atomicMax(&s.hi, at);
        __syncthreads();
        token = s.hi;
    }
    if (tid == 0) {
        const float x = norm_load<false>(p.logits, row * p.stride + token, p.type, 1)[0];
        give(token, (double)weight(x, token) / (double)total);
    }
}
