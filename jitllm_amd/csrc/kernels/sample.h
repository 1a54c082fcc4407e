// A token a row of logits (jl_sample_dev): temperature, the k largest, the nucleus, those near the largest, and one of them by a given number.
//
//   w_i = e^((x_i - max) / T)            order: x descending, index ascending
//   kept = the shortest of: the first k; the shortest beginning whose sum reaches top_p of the first k's sum; those with w_i >= min_p; one at least
//   token = the first kept i, by index, whose sum of the kept w up to i exceeds u W
//
// Whole numbers: w is kept as round(w 2^44) in 64 bits, so sums do not depend on their order and a border falls the same way whatever threads met it
// (in f32 one row in a few thousand of a flat distribution would take a neighbour's token).  w itself is f64's, to 2^-50.
//
// The order is made only where it decides.  Four launches, rows cut into slices so that a few rows fill the chip:
//   sample_max     a slice's largest, its first place, and how many candidates
//   sample_bins    counts (and sums, where only the nucleus cuts) over 2048 bins of the distance from the largest, 64 of them a temperature
//   sample_gather  from the bins: how far the kept can reach.  Up to 1024 candidates there: all of them into a list (LIST).  More: each slice's sum of what is kept
//                  for sure, and the candidates of the bin in which the cut falls into the list (LARGE); a cut in a bin of more, or a nucleus of more than 1024 of
//                  the k largest: SLOW
//   sample_take    a workgroup a row: the list sorted, the cuts, and the token, from the list or from the slice in which u falls.  SLOW rows are done here from
//                  the start: the cut's bin divided again by keys and, where one key is left, by index.
#pragma once
#include "args.h"
#include "common.h"
#include "moe_select.h"
#include "norm_rows.h"

#pragma clang fp contract(off)

#define JL_SA_TILE 4096      // elements of a workgroup's pass in index order

#define JL_SA_DONE 0
#define JL_SA_LISTED 1
#define JL_SA_LARGE 2
#define JL_SA_SLOW 3

struct SampleLds {
    uint64_t mass[JL_SA_BINS];
    u32 count[JL_SA_BINS];
    u32 key[JL_SA_LIST], idx[JL_SA_LIST];
    uint64_t tile[256];
    uint64_t slices[JL_SA_SLICES];
    uint64_t wsum[16];
    uint64_t at_mass;
    u32 wcnt[16];
    u32 at, at_count, at_n, fill, lo, hi, res_key, res_idx;
};

// The row's values as ordered whole numbers; 0: no candidate.
__device__ __forceinline__ u32 sample_key(float x) {
    const u32 b = __float_as_uint(x + 0.0f);   // (-0 is 0)
    return x > -__builtin_inff() ? b ^ ((u32)((i32)b >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float sample_value(u32 k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

struct SampleRow {
    float max;        // of the row
    double inv_t;     // 1 / temperature
    float fine;       // bins a unit of x
    __device__ double weight(float x) const { return x == max ? 1.0 : select_exp(fmax(((double)x - (double)max) * inv_t, -800.0)); }
    __device__ uint64_t whole(float x) const {   // round(w 2^44): the low bits of w 2^44 + 2^52
        return __builtin_bit_cast(uint64_t, __builtin_fma(weight(x), 0x1p44, 0x1p52)) & ((1ull << 52) - 1);
    }
    __device__ uint64_t kept(float x, u32 i, float low, u32 first) const {   // 0 where min_p takes it out
        const double w = weight(x);
        return low > 0.f && !(w >= (double)low) && i != first ? 0 : __builtin_bit_cast(uint64_t, __builtin_fma(w, 0x1p44, 0x1p52)) & ((1ull << 52) - 1);
    }
    __device__ u32 bin(float x) const {          // falls as x rises
        const float d = (max - x) * fine;        // (infinities apart: NaN or infinite)
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
// f(value, index) for the elements from to end of a row, four in a row a thread; four such loads are on their way.
template <int THREADS, class F> __device__ __forceinline__ void sample_range(const SampleArgs& p, size_t row, int from, int end, F f) {
    const size_t at = row * p.stride;
    int i = from + 4 * (int)threadIdx.x;
    for (; i + 3 * 4 * THREADS + 4 <= end; i += 4 * 4 * THREADS) {
        f32x4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = sample_load(p, at + i + k * 4 * THREADS, 4);
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) f(v[k][j], (u32)(i + k * 4 * THREADS + j));
    }
    for (; i < end; i += 4 * THREADS) {
        const f32x4 v = sample_load(p, at + i, end - i);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < end) f(v[j], (u32)(i + j));
    }
}
template <class F> __device__ __forceinline__ void sample_each(const SampleArgs& p, size_t row, F f) { sample_range<1024>(p, row, 0, p.n, f); }

// Inclusive sum over the workgroup's threads; total to every one.
__device__ __forceinline__ uint64_t sample_scan(SampleLds& s, uint64_t v, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)v, d, 64);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) s.wsum[wave] = v;
    __syncthreads();
    total = 0;
    uint64_t before = 0;
    for (int w = 0; w < 16; w++) {
        before += w < wave ? s.wsum[w] : 0;
        total += s.wsum[w];
    }
    return v + before;
}

// The first element by index with crosses(sum of weight(x, i) up to and with it); ~0: none.  weight is 0 for elements that are not in the sum.
// Of the elements from to end (from a multiple of four).
template <class W, class X> __device__ __forceinline__ u32 sample_cross(const SampleArgs& p, SampleLds& s, size_t row, int from, int end, W weight, X crosses, uint64_t& total) {
    const int tiles = (end - from + JL_SA_TILE - 1) / JL_SA_TILE;   // (256 at most)
    __syncthreads();
    if (threadIdx.x < 256) s.tile[threadIdx.x] = 0;
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
        if (sum) atomicAdd((unsigned long long*)&s.tile[k], (unsigned long long)sum);
    }
    __syncthreads();
    uint64_t before = 0;
    total = 0;
    int tile = -1;
    for (int k = 0; k < tiles; k++) {
        const uint64_t t = s.tile[k];
        if (tile < 0 && t && crosses(total + t)) {
            tile = k;
            before = total;
        }
        total += t;
    }
    if (tile >= 0) {   // uniform
        const int i = from + tile * JL_SA_TILE + 4 * (int)threadIdx.x;
        uint64_t part[4] = {0, 0, 0, 0}, mine = 0, all;
        if (i < end) {
            const f32x4 v = load(i);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (i + j < end) part[j] = weight(v[j], (u32)(i + j));
                mine += part[j];
            }
        }
        uint64_t c = before + sample_scan(s, mine, all) - mine;
        const bool had = c != 0 && crosses(c);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool is = part[j] && crosses(c + part[j]);
            if (is && !had) atomicMin(&s.at, (u32)(i + j));
            c += part[j];
        }
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

// Counts and sums of the bins (bin(x, key) < BINS, or ~0: not in it), then over the bins before each.
template <class B> __device__ __forceinline__ void sample_bins(const SampleArgs& p, SampleLds& s, size_t row, const SampleRow& r, B bin) {
    __syncthreads();
    for (int i = threadIdx.x; i < JL_SA_BINS; i += 1024) {
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
    constexpr int PER = JL_SA_BINS / 1024;
    const int b0 = PER * threadIdx.x;
    uint64_t c = 0, m = 0, all;
#pragma unroll
    for (int j = 0; j < PER; j++) {
        c += s.count[b0 + j];
        m += s.mass[b0 + j];
    }
    uint64_t cb = sample_scan(s, c, all) - c + count0, mb = sample_scan(s, m, all) - m + mass0;
    if (c && crosses((u32)(cb + c), mb + m) && !(cb && crosses((u32)cb, mb))) {
#pragma unroll
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
    }
    __syncthreads();
}

// The last element kept, in the order, such that crosses(count, mass) up to it is first true.  False: nothing crosses.
template <class X> __device__ __forceinline__ bool sample_cut(const SampleArgs& p, SampleLds& s, size_t row, const SampleRow& r, X crosses, SampleCut& cut) {
    sample_bins(p, s, row, r, [&](float x, u32) { return r.bin(x); });
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
            sample_bins(p, s, row, r, [&](float x, u32 k) { return r.bin(x) == bin0 && k >= klo && k <= khi ? (khi - k) >> shift : ~0u; });
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
        const float x0 = sample_value(klo);
        const uint64_t w0 = r.whole(x0);
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
    // a thread an element: those ahead of it, and their weights
    const u32 tid = threadIdx.x;
    uint64_t* const w = s.mass;   // (the bins have been read)
    if (tid < n) w[tid] = r.whole(sample_value(s.key[tid]));
    __syncthreads();
    if (tid < n) {
        const u32 k = s.key[tid], i = s.idx[tid];
        u32 ahead = 0;
        uint64_t m = 0;
        for (u32 j = 0; j < n; j++) {
            const bool is = s.key[j] > k || (s.key[j] == k && s.idx[j] < i);
            ahead += is;
            m += is ? w[j] : 0;
        }
        const u32 cb = count + ahead;
        if (crosses(cb + 1, mass + m + w[tid]) && !(cb && crosses(cb, mass + m))) {
            s.res_key = k;
            s.res_idx = i;
            s.at_mass = mass + m + w[tid];
        }
    }
    __syncthreads();
    cut.key = s.res_key;
    cut.idx = s.res_idx;
    cut.mass = s.at_mass;
    __syncthreads();
    return true;
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
    s.best = top;
    s.valid = lane < p.slices ? ws.many[lane] : 0u;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        s.best = max(s.best, (u32)__shfl_xor((int)s.best, d, 64));
        s.valid += (u32)__shfl_xor((int)s.valid, d, 64);
    }
    s.best = (u32)__builtin_amdgcn_readfirstlane((i32)s.best);
    s.valid = (u32)__builtin_amdgcn_readfirstlane((i32)s.valid);
    s.first = (u32)__builtin_amdgcn_readlane((i32)at, (int)__builtin_ctzll(__ballot(top == s.best)));   // the first slice that has it
    const float t = p.temperature ? p.temperature[row] : 1.f;
    s.greedy = s.best == 0 || !(t > 0.f);
    s.r.max = sample_value(s.best);
    s.r.inv_t = 1.0 / (double)t;
    s.r.fine = fminf(64.f / t, 1e30f);
    const u32 k = p.top_k ? p.top_k[row] : 0u;
    s.k = k < s.valid ? k : 0u;
    s.p = p.top_p ? p.top_p[row] : 1.f;
    s.low = p.min_p ? p.min_p[row] : 0.f;
    s.nucleus = s.p < 1.f;
    return s;
}
__device__ __forceinline__ void sample_slice(const SampleArgs& p, int slice, int& from, int& end) {
    from = slice * p.slice_len;
    end = min(from + p.slice_len, p.n);
}

// grid = (slices, rows), block = 512.  LDS: 4 words.
__device__ __forceinline__ void sample_max_body(const SampleArgs& p, u32* lds) {
    const size_t row = blockIdx.y;
    SampleRowWs& ws = ((SampleRowWs*)p.ws)[row];
    const int slice = blockIdx.x;
    for (int i = slice * 512 + threadIdx.x; i < JL_SA_BINS; i += p.slices * 512) {
        ws.counts[i] = 0;
        ws.sums[i] = 0;
    }
    if (slice == 0 && threadIdx.x == 0) ws.fill = 0;
    if (threadIdx.x < 4) lds[threadIdx.x] = threadIdx.x == 1 ? ~0u : 0u;
    __syncthreads();
    int from, end;
    sample_slice(p, slice, from, end);
    u32 top = 0, many = 0, at = ~0u;
    sample_range<512>(p, row, from, end, [&](float x, u32 i) {
        const u32 k = sample_key(x);
        many += k != 0;
        at = k > top ? i : at;
        top = max(top, k);
    });
    u32 best = top;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        best = max(best, (u32)__shfl_xor((int)best, d, 64));
        many += (u32)__shfl_xor((int)many, d, 64);
    }
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
    sample_range<512>(p, row, from, end, [&](float x, u32) {
        const u32 b = x > -__builtin_inff() ? s.r.bin(x) : (u32)JL_SA_BINS;
        if (b < JL_SA_BINS - 1) {   // (the last bin's count is what is left over, its sum nothing)
            atomicAdd(&counts[b], 1u);
            if (weighs) atomicAdd((unsigned long long*)&sums[b], (unsigned long long)s.r.whole(x));
        }
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

// Inclusive sums over 512 threads.  LDS: 8 words.
__device__ __forceinline__ uint64_t sample_scan512(uint64_t* lds, uint64_t v, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)v, d, 64);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    total = 0;
    uint64_t before = 0;
#pragma unroll
    for (int w = 0; w < 8; w++) {
        before += w < wave ? lds[w] : 0;
        total += lds[w];
    }
    return v + before;
}

// grid = (slices, rows), block = 512.  LDS: 8 words of 8 bytes, then 8 of 4.
__device__ __forceinline__ void sample_gather_body(const SampleArgs& p, uint64_t* scan, u32* told) {
    const size_t row = blockIdx.y;
    const SampleSet s = sample_set(p, row);
    SampleRowWs& ws = ((SampleRowWs*)p.ws)[row];
    const bool writes = blockIdx.x == 0 && threadIdx.x == 0;
    if (s.greedy) {
        if (writes) ws.mode = JL_SA_DONE;
        return;
    }
    // The bin that min_p ends in, or one behind it: -ln(min_p) temperatures, 64 bins each.
    const u32 low_bin = s.low > 0.f ? (u32)fminf((float)(JL_SA_BINS - 1), fmaxf(-__logf(fminf(s.low, 1.f)) * 64.f * 1.0001f + 2.f, 0.f)) : (u32)JL_SA_BINS - 1;
    u32 mode = JL_SA_LARGE, cut = JL_SA_BINS, before = 0;    // the bin of the cut (LARGE) or the last bin (LIST); candidates before it
    uint64_t mass = 0;
    if (s.k || s.nucleus || s.low > 0.f) {
        constexpr int PER = JL_SA_BINS / 512;
        const bool weighs = s.nucleus && !s.k;      // (the bins have sums)
        const int b0 = PER * threadIdx.x;
        u32 c[PER];
        uint64_t m[PER], cs = 0, ms = 0, all, mass_all;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            c[j] = ws.counts[b0 + j];
            m[j] = weighs ? ws.sums[b0 + j] : 0;
            cs += c[j];
            ms += m[j];
        }
        if (threadIdx.x < 8) told[threadIdx.x] = threadIdx.x < 2 ? (u32)JL_SA_BINS : 0u;
        uint64_t cb = sample_scan512(scan, cs, all) - cs, mb = 0;
        mass_all = 0;
        if (weighs) mb = sample_scan512(scan, ms, mass_all) - ms;
        const double reach = (double)s.p * (double)mass_all;
        // told: 0 the cut's bin, 1 low_bin's count through it, ... ; the last bin has what is left over
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const u32 b = b0 + j, n = b == JL_SA_BINS - 1 ? s.valid - (u32)cb : c[j];
            const uint64_t ce = cb + n, me = mb + m[j];
            const bool crossed = s.k ? ce >= s.k && cb < s.k : s.nucleus && n && (double)me >= reach && !(cb && (double)mb >= reach);
            if (crossed) {
                told[0] = b;
                told[2] = (u32)cb;
                told[3] = (u32)mb;
                told[4] = (u32)(mb >> 32);
                told[5] = (u32)ce;
            }
            if (b == low_bin) told[6] = (u32)ce;
            cb = ce;
            mb = me;
        }
        __syncthreads();
        cut = told[0];
        before = told[2];
        mass = (uint64_t)told[4] << 32 | told[3];
        const u32 through = told[5], low_through = told[6];
        if (s.low > 0.f && low_bin < cut && !(s.k && s.nucleus)) {   // min_p ends first
            if (low_through <= JL_SA_LIST) {
                mode = JL_SA_LISTED;
                cut = low_bin;
            } else {
                cut = JL_SA_BINS;
            }
        } else if (cut < JL_SA_BINS) {
            mode = through <= JL_SA_LIST ? JL_SA_LISTED : s.k && s.nucleus ? JL_SA_SLOW : through - before <= JL_SA_LIST ? JL_SA_LARGE : JL_SA_SLOW;
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
    int from, end;
    sample_slice(p, blockIdx.x, from, end);
    uint64_t sum = 0, total;
    sample_range<512>(p, row, from, end, [&](float x, u32 i) {
        const u32 key = sample_key(x);
        if (!key) return;
        const u32 b = s.r.bin(x);
        if (mode == JL_SA_LISTED ? b <= cut : b == cut) {
            const u32 at = atomicAdd(&ws.fill, 1u);
            if (at < JL_SA_LIST) {
                ws.key[at] = key;
                ws.idx[at] = i;
            }
        } else if (mode == JL_SA_LARGE && b < cut) {
            sum += s.r.kept(x, i, s.low, s.first);
        }
    });
    if (mode == JL_SA_LARGE) {
        sample_scan512(scan, sum, total);
        if (threadIdx.x == 0) ws.slice[blockIdx.x] = total;
    }
}

// The workgroup's list of up to 1024 (a thread an element), ascending.
__device__ __forceinline__ uint64_t sample_sort(uint64_t* lds, uint64_t v, u32 n) {
    const u32 tid = threadIdx.x;
    u32 size = 64;
    while (size < n) size *= 2;
    for (u32 k = 2; k <= size; k *= 2)
        for (u32 j = k / 2; j; j /= 2) {
            uint64_t o;
            if (j < 64) {
                o = __shfl_xor((unsigned long long)v, (int)j, 64);
            } else {
                __syncthreads();
                lds[tid] = v;
                __syncthreads();
                o = lds[tid ^ j];
            }
            const bool up = (tid & k) == 0, lower = (tid & j) == 0;
            v = (up == lower) == (v < o) ? v : o;
        }
    __syncthreads();
    return v;
}

// The same within a wavefront, and its inclusive sums.
__device__ __forceinline__ uint64_t sample_sort64(uint64_t v) {
    const u32 lane = threadIdx.x & 63;
#pragma unroll
    for (u32 k = 2; k <= 64; k *= 2)
#pragma unroll
        for (u32 j = k / 2; j; j /= 2) {
            const uint64_t o = __shfl_xor((unsigned long long)v, (int)j, 64);
            v = (((lane & k) == 0) == ((lane & j) == 0)) == (v < o) ? v : o;
        }
    return v;
}
__device__ __forceinline__ uint64_t sample_scan64(uint64_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// grid = rows, block = 1024.
__device__ __forceinline__ void sample_take_body(const SampleArgs& p, SampleLds& s) {
    const size_t row = blockIdx.x;
    const SampleRowWs& ws = ((const SampleRowWs*)p.ws)[row];
    const SampleSet set = sample_set(p, row);
    const u32 tid = threadIdx.x, mode = ws.mode;
    const SampleRow& r = set.r;
    auto give = [&](u32 token, double prob) {
        p.token[row] = token;
        if (p.prob) p.prob[row] = (float)prob;
    };
    if (set.greedy) {
        if (tid == 0) give(set.best ? set.first : (u32)p.n, set.best ? 1.0 : 0.0);
        return;
    }
    const float u = p.u[row];
    SampleCut cut = {1u, ~0u, 0};
    if (mode == JL_SA_LISTED && ws.fill <= 64) {   // by one wavefront
        if (tid >= 64) return;
        const u32 n = ws.fill;
        uint64_t v = sample_sort64(tid < n ? (uint64_t)~ws.key[tid] << 32 | ws.idx[tid] : ~0ull);
        const float x = sample_value(~(u32)(v >> 32));
        const uint64_t w = tid < n ? r.whole(x) : 0, through = sample_scan64(w);
        u32 kept = set.k ? min(n, set.k) : n;
        if (set.nucleus) {
            const uint64_t all = set.k ? (uint64_t)__shfl((unsigned long long)through, (int)kept - 1, 64) : ws.all;
            const uint64_t over = __ballot(tid < kept && (double)through >= (double)set.p * (double)all);
            if (over) kept = (u32)__builtin_ctzll(over) + 1;
        }
        const bool in = tid < kept && (!(set.low > 0.f) || r.weight(x) >= (double)set.low || tid == 0);
        // by index; the place in the list goes along
        const uint64_t by = sample_sort64(in ? (v & 0xffffffffu) << 32 | tid : ~0ull);
        const uint64_t there = __shfl((unsigned long long)w, (int)(by & 63), 64), mine = by == ~0ull ? 0 : there;
        const uint64_t c = sample_scan64(mine), total = __shfl((unsigned long long)c, 63, 64);
        const uint64_t over = __ballot(mine && (double)c > (double)u * (double)total), any = __ballot(mine != 0);
        if (tid == (u32)(over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any))) give((u32)(by >> 32), (double)mine / (double)total);
        return;
    }
    if (mode == JL_SA_LISTED || (mode == JL_SA_LARGE && ws.bin < JL_SA_BINS)) {
        const u32 n = min(ws.fill, (u32)JL_SA_LIST);
        // descending by key, ascending by index: ascending by the key's complement
        uint64_t v = tid < n ? (uint64_t)~ws.key[tid] << 32 | ws.idx[tid] : ~0ull;
        v = sample_sort(s.mass, v, n);
        const u32 key = ~(u32)(v >> 32), idx = (u32)v;
        const bool live = tid < n;
        const uint64_t w = live ? r.whole(sample_value(key)) : 0;
        uint64_t all;
        const uint64_t base = mode == JL_SA_LARGE ? ws.mass : 0;
        const u32 before = mode == JL_SA_LARGE ? ws.before : 0;
        const uint64_t through = base + sample_scan(s, w, all);      // sums up to and with this one
        u32 kept = n;
        if (set.k) kept = min(kept, set.k - before);
        __syncthreads();
        if (tid == 0) s.at = kept;
        if (tid == kept - 1) s.at_mass = through;
        __syncthreads();
        if (set.nucleus) {
            const double reach = (double)set.p * (double)(set.k ? s.at_mass : ws.all);
            if (tid < kept && (double)through >= reach) atomicMin(&s.at, tid + 1);
            __syncthreads();
        }
        kept = s.at;
        __syncthreads();
        if (mode == JL_SA_LARGE) {
            if (tid == kept - 1) {
                s.res_key = key;
                s.res_idx = idx;
            }
            __syncthreads();
            cut.key = s.res_key;
            cut.idx = s.res_idx;
        } else {
            // those of them that min_p keeps, by index
            const bool in = tid < kept && (!(set.low > 0.f) || r.weight(sample_value(key)) >= (double)set.low || tid == 0);
            __syncthreads();
            if (tid < n) s.mass[1024 + tid] = in ? w : 0;
            uint64_t by = in ? (uint64_t)idx << 32 | tid : ~0ull;
            __syncthreads();
            by = sample_sort(s.mass, by, n);
            const bool has = by != ~0ull;
            const uint64_t mine = has ? s.mass[1024 + (u32)by] : 0;
            uint64_t total;
            const uint64_t c = sample_scan(s, mine, total);
            const double over = (double)u * (double)total;
            __syncthreads();
            if (tid == 0) {
                s.at = ~0u;
                s.hi = 0;
            }
            __syncthreads();
            if (mine && (double)c > over) atomicMin(&s.at, tid);
            if (mine) atomicMax(&s.hi, tid);
            __syncthreads();
            if (tid == (s.at != ~0u ? s.at : s.hi)) give((u32)(by >> 32), (double)mine / (double)total);
            return;
        }
        // the list's kept into their slices' sums
        if (tid < (u32)p.slices) s.tile[tid] = ws.slice[tid];
        __syncthreads();
        if (tid < kept) {
            const uint64_t k = r.kept(sample_value(key), idx, set.low, set.first);
            if (k) atomicAdd((unsigned long long*)&s.tile[idx / (u32)p.slice_len], (unsigned long long)k);
        }
        __syncthreads();
    } else if (mode == JL_SA_LARGE) {
        if (tid < (u32)p.slices) s.tile[tid] = ws.slice[tid];
        __syncthreads();
    } else {
        if (set.k) sample_cut(p, s, row, r, [&](u32 c, uint64_t) { return c >= set.k; }, cut);
        if (set.nucleus) {
            uint64_t all = cut.mass;
            if (!set.k) {
                uint64_t sum = 0;
                sample_each(p, row, [&](float x, u32) { sum += sample_key(x) ? r.whole(x) : 0; });
                sample_scan(s, sum, all);
            }
            const double reach = (double)set.p * (double)all;
            sample_cut(p, s, row, r, [&](u32, uint64_t m) { return (double)m >= reach; }, cut);
        }
        for (int i = 0; i < p.slices; i++) {
            int from, end;
            sample_slice(p, i, from, end);
            uint64_t sum = 0, all;
            sample_range<1024>(p, row, from, end, [&](float x, u32 e) {
                const u32 key = sample_key(x);
                if (key && cut.keeps(key, e)) sum += r.kept(x, e, set.low, set.first);
            });
            sample_scan(s, sum, all);
            if (tid == 0) s.slices[i] = all;
        }
        __syncthreads();
        if (tid < (u32)p.slices) s.tile[tid] = s.slices[tid];
        __syncthreads();
    }
    // the slice in which the sum exceeds u of it, a slice a lane; and the token there
    const int lane = tid & 63;
    const uint64_t mine = lane < p.slices ? s.tile[lane] : 0;
    uint64_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint64_t o = __shfl_up((unsigned long long)sum, d, 64);
        if (lane >= d) sum += o;
    }
    const uint64_t total = __shfl((unsigned long long)sum, 63, 64);
    const double over = (double)u * (double)total;
    const uint64_t over_at = __ballot(mine && (double)sum > over), any = __ballot(mine != 0);
    const int slice = over_at ? __builtin_ctzll(over_at) : -1, last = any ? 63 - __builtin_clzll(any) : 0;
    const uint64_t before = __shfl((unsigned long long)(sum - mine), slice < 0 ? 0 : slice, 64);
    __syncthreads();
    auto weight = [&](float x, u32 i) -> uint64_t {
        const u32 key = sample_key(x);
        return key && cut.keeps(key, i) ? r.kept(x, i, set.low, set.first) : 0;
    };
    int from, end;
    sample_slice(p, slice < 0 ? last : slice, from, end);
    u32 token = ~0u;
    uint64_t in;
    if (slice >= 0) token = sample_cross(p, s, row, from, end, weight, [&](uint64_t c) { return (double)(before + c) > over; }, in);
    if (token == ~0u) {   // u is 1 or more, or no number: the last that is kept
        if (tid == 0) s.hi = 0;
        __syncthreads();
        u32 at = 0;
        sample_range<1024>(p, row, from, end, [&](float x, u32 i) { at = weight(x, i) ? max(at, i) : at; });
        atomicMax(&s.hi, at);
        __syncthreads();
        token = s.hi;
    }
    if (tid == 0) {
        const float x = norm_load<false>(p.logits, row * p.stride + token, p.type, 1)[0];
        give(token, (double)weight(x, token) / (double)total);
    }
}
