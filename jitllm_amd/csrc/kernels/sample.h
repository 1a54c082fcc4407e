// A token a row of logits (jl_sample_dev): temperature, the k largest, the nucleus, those near the largest, and one of them by a given number.
//
//   w_i = e^((x_i - max) / T)            order: x descending, index ascending
//   kept = the shortest of: the first k; the shortest beginning whose sum reaches top_p of the first k's sum; those with w_i >= min_p; one at least
//   token = the first kept i, by index, whose sum of the kept w up to i exceeds u W
//
// Whole numbers: w is kept as round(w 2^44) in 64 bits, so sums do not depend on their order and a border falls the same way whatever threads met it
// (in f32 one row in a few thousand of a flat distribution would take a neighbour's token).  w itself is f64's, to 2^-50.
//
// A workgroup a row.  The order is never made: counts and sums over 4096 bins of the distance from the largest find the bin in which k or top_p falls, and
// that bin's few elements are ranked among themselves; where it holds more than fit (a flat row), its keys' range is cut into 4096 again, and where one
// key is left, ties are counted by index.  So a row is read five times, once from memory.
#pragma once
#include "args.h"
#include "common.h"
#include "moe_select.h"
#include "norm_rows.h"

#pragma clang fp contract(off)

#define JL_SA_BINS 4096
#define JL_SA_LIST 1024
#define JL_SA_TILE 4096      // elements of a workgroup's pass in index order

struct SampleLds {
    uint64_t mass[JL_SA_BINS];
    u32 count[JL_SA_BINS];
    u32 key[JL_SA_LIST], idx[JL_SA_LIST];
    uint64_t tile[256];
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
    __device__ u32 bin(float x) const {          // falls as x rises
        const float d = (max - x) * fine;        // (infinities apart: NaN or infinite)
        return x == max ? 0u : d < (float)(JL_SA_BINS - 1) ? (u32)d : (u32)JL_SA_BINS - 1u;
    }
};

// f(value, index) for every element of the row, four in a row a thread.
template <class F> __device__ __forceinline__ void sample_each(const SampleArgs& p, size_t row, F f) {
    const size_t at = row * p.stride;
    for (int i = 4 * threadIdx.x; i < p.n; i += 4096) {
        const f32x4 v = p.vec && i + 4 <= p.n ? norm_load<true>(p.logits, at + i, p.type, 4) : norm_load<false>(p.logits, at + i, p.type, p.n - i);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < p.n) f(v[j], (u32)(i + j));
    }
}

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
template <class W, class X> __device__ __forceinline__ u32 sample_cross(const SampleArgs& p, SampleLds& s, size_t row, W weight, X crosses, uint64_t& total) {
    const int tiles = (p.n + JL_SA_TILE - 1) / JL_SA_TILE;   // (256 at most)
    __syncthreads();
    if (threadIdx.x < 256) s.tile[threadIdx.x] = 0;
    if (threadIdx.x == 0) s.at = ~0u;
    __syncthreads();
    const size_t at = row * p.stride;
    auto load = [&](int i) { return p.vec && i + 4 <= p.n ? norm_load<true>(p.logits, at + i, p.type, 4) : norm_load<false>(p.logits, at + i, p.type, p.n - i); };
    for (int i = 4 * threadIdx.x, k = 0; k < tiles; k++, i += JL_SA_TILE) {
        uint64_t sum = 0;
        if (i < p.n) {
            const f32x4 v = load(i);
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < p.n) sum += weight(v[j], (u32)(i + j));
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
        const int i = tile * JL_SA_TILE + 4 * threadIdx.x;
        uint64_t part[4] = {0, 0, 0, 0}, mine = 0, all;
        if (i < p.n) {
            const f32x4 v = load(i);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (i + j < p.n) part[j] = weight(v[j], (u32)(i + j));
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
    const int b0 = 4 * threadIdx.x;
    uint64_t c = 0, m = 0, all;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        c += s.count[b0 + j];
        m += s.mass[b0 + j];
    }
    uint64_t cb = sample_scan(s, c, all) - c + count0, mb = sample_scan(s, m, all) - m + mass0;
    if (c && crosses((u32)(cb + c), mb + m) && !(cb && crosses((u32)cb, mb))) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
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
        cut.idx = sample_cross(p, s, row, [&](float x, u32) { return (uint64_t)(sample_key(x) == klo); },
                               [&](uint64_t c) { return crosses(count + (u32)c, mass + c * w0); }, total);
        cut.key = klo;
        // how many that are: again over those up to it
        const u32 last = cut.idx;
        sample_cross(p, s, row, [&](float x, u32 i) { return (uint64_t)(sample_key(x) == klo && i <= last); }, [&](uint64_t) { return false; }, total);
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

__device__ __forceinline__ void sample_body(const SampleArgs& p, SampleLds& s) {
    const size_t row = blockIdx.x;
    const float inf = __builtin_inff();
    // the largest, its first place, and how many candidates there are
    if (threadIdx.x == 0) {
        s.hi = 0;
        s.fill = 0;
        s.lo = ~0u;
    }
    __syncthreads();
    u32 top = 0, many = 0, at = ~0u;
    sample_each(p, row, [&](float x, u32 i) {
        const u32 k = sample_key(x);
        many += k != 0;
        if (k > top) {
            top = k;
            at = i;
        }
    });
    atomicMax(&s.hi, top);
    atomicAdd(&s.fill, many);
    __syncthreads();
    const u32 best = s.hi, valid = s.fill;
    if (best && top == best) atomicMin(&s.lo, at);
    __syncthreads();
    const u32 first = s.lo;
    __syncthreads();
    const float t = p.temperature ? p.temperature[row] : 1.f;
    if (best == 0 || !(t > 0.f)) {
        if (threadIdx.x == 0) {
            p.token[row] = best ? first : (u32)p.n;
            if (p.prob) p.prob[row] = best ? 1.f : 0.f;
        }
        return;
    }
    SampleRow r;
    r.max = sample_value(best);
    r.inv_t = 1.0 / (double)t;
    r.fine = fminf(128.f / t, 1e30f);
    SampleCut cut = {1u, ~0u, 0};
    const u32 k = p.top_k ? p.top_k[row] : 0u;
    const float top_p = p.top_p ? p.top_p[row] : 1.f, min_p = p.min_p ? p.min_p[row] : 0.f;
    bool cut_k = false;
    if (k && k < valid) cut_k = sample_cut(p, s, row, r, [&](u32 c, uint64_t) { return c >= k; }, cut);
    if (top_p < 1.f) {
        uint64_t all = cut.mass;
        if (!cut_k) {
            uint64_t sum = 0;
            sample_each(p, row, [&](float x, u32) { sum += sample_key(x) ? r.whole(x) : 0; });
            sample_scan(s, sum, all);
        }
        const double reach = (double)top_p * (double)all;
        sample_cut(p, s, row, r, [&](u32, uint64_t m) { return (double)m >= reach; }, cut);
    }
    auto weight = [&](float x, u32 i) -> uint64_t {
        const u32 key = sample_key(x);
        if (!key || !cut.keeps(key, i)) return 0;
        const double w = r.weight(x);
        return (min_p > 0.f && !(w >= (double)min_p) && i != first) ? 0 : __builtin_bit_cast(uint64_t, __builtin_fma(w, 0x1p44, 0x1p52)) & ((1ull << 52) - 1);
    };
    // the sum first: u times it is what a sum has to exceed
    uint64_t sum = 0, all;
    sample_each(p, row, [&](float x, u32 i) { sum += weight(x, i); });
    sample_scan(s, sum, all);
    const double over = (double)p.u[row] * (double)all;
    uint64_t total;
    u32 token = sample_cross(p, s, row, weight, [&](uint64_t c) { return (double)c > over; }, total);
    if (token == ~0u) {   // u is 1 or more, or no number: the last that is kept
        if (threadIdx.x == 0) s.hi = 0;
        __syncthreads();
        u32 last = 0;
        sample_each(p, row, [&](float x, u32 i) { last = weight(x, i) ? max(last, i) : last; });
        atomicMax(&s.hi, last);
        __syncthreads();
        token = s.hi;
    }
    if (threadIdx.x == 0) {
        p.token[row] = token;
        if (p.prob) {
            const float x = norm_load<false>(p.logits, row * p.stride + token, p.type, 1)[0];
            p.prob[row] = (float)((double)weight(x, token) / (double)all);
        }
    }
    (void)inf;
}
