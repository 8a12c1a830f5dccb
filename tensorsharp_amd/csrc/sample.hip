// The next token of each row of logits: temperature, top-k, top-p, min-p and a draw from a given random number.
//
// Candidates are ranked by (logit, lower index first); what top-k and top-p keep is a prefix of that order, so each is a logit and how
// many of its equals stay.  Weights e^((l - l_max) / T) are formed in 64-bit floating point and held as whole multiples of 2^-43:
// sums of them are exact and the same in every order, so that neither a tile nor an atomic can move the border of a prefix or the
// place of a draw.  (What is rounded away is below 2^-44 of the likeliest candidate's weight.)
//
// A row is cut into chunks, a workgroup each, and those into 16 segments, a wavefront each.
//   sample_top_kernel    the largest logit of each chunk, and of each of 64 groups of it
//   sample_sums_kernel   by what the row asks for:
//                        top-k with k at most the number of groups: as many groups reach the k-th largest of their maxima, so the k
//                        candidates are among those that do - these are listed, in order, per segment
//                        another cut: a histogram of the chunk over the distance to the largest logit, of counts (a larger k) or weights (top-p)
//                        nothing but min-p: the weights of each segment
//   sample_draw_kernel   one workgroup per row: from a histogram the bin in which the cut falls and the list up to it; the exact cut
//                        among the listed; the draw
// Each row's settings are device data, so every launch finds out for itself what its row needs.
#include "tship_internal.h"

#include <algorithm>

namespace tship {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 1024;
constexpr int kGroups = 64;                                          // of a chunk: what 16 lanes of a segment's wavefront read
constexpr int kMinChunk = 4096, kMaxChunks = 32;
constexpr int kListed = 4096;                                        // candidates that the last kernel keeps in LDS
constexpr int kRanked = 256;                                         // up to so many are ranked by comparing each with each
constexpr double kOne = 8796093022208.0;                             // 2^43: 2^20 of them stay below 2^63
constexpr uint32_t kLowestKey = 0x007fffffu;                         // of -infinity; NaN has 0

// larger logit, larger key; both zeros the same
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __float_as_uint(l + 0.0f);
    return l != l ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

struct SampleArgs {
    const float* logits;
    int64_t ld;
    int vocab, chunks, seg_len;                                      // a chunk has 16 segments of seg_len logits
    const float* uniforms;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* tokens;
    float* probabilities;
    uint64_t* tops;                                                  // [row][chunk]: key of the largest logit, complement of its index
    uint32_t* groups;                                                // [row][chunk][group]: key of the largest logit
    uint64_t* hist;                                                  // [row][chunk][bin]
    uint64_t* sums;                                                  // [row][segment]: weights
    uint32_t* counts;                                                // [row][segment]: listed
    uint64_t* list;                                                  // [row][segment][seg_len]: key and index
};

enum { kDone, kWhole, kTopK, kManyK, kTopP };                        // nothing to draw; no cut but min-p; cut by count (of few, of many); by weight only

struct Row {
    double by, p, least;         // by: log2 e / temperature
    float top;
    uint32_t top_key;
    int top_index, k, kind;
};
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) { return (uint64_t)__shfl_xor((unsigned long long)v, o); }
__device__ __forceinline__ uint64_t wave_max(uint64_t v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, shfl_xor64(v, o));
    return v;
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += shfl_xor64(v, o);
    return v;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v)             // inclusive
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t below = (uint64_t)__shfl_up((unsigned long long)v, o);
        if (lane >= o) v += below;
    }
    return v;
}

// every wavefront works it out for itself
__device__ __forceinline__ Row row_of(const SampleArgs& A, int row)
{
    const int lane = threadIdx.x & 63;
    Row r;
    const uint64_t best = wave_max(lane < A.chunks ? A.tops[row * A.chunks + lane] : 0);
    const float t = A.temperature[row];
    r.top_key = (uint32_t)(best >> 32);
    r.top_index = (int)~(uint32_t)best;
    r.top = logit_of(r.top_key);
    r.by = 1.44269504088896340736 / (double)t;
    r.k = A.top_k ? A.top_k[row] : 0;
    r.p = A.top_p ? (double)A.top_p[row] : 1.0;
    r.least = A.min_p ? (double)A.min_p[row] : 0.0;
    r.kind = r.top_key <= kLowestKey || !(t > 0.f) ? kDone : r.k > 0 && r.k < A.vocab ? (r.k <= A.chunks * kGroups ? kTopK : kManyK) : r.p < 1.0 ? kTopP : kWhole;
    return r;
}
// 2^y, -60 <= y <= 0 (what is below counts as 2^-60, which no sum holds): the whole part of y goes to the exponent; the rest, at most a
// half, through the Taylor series of e^(y ln 2) up to the 11th power (what is left out: (ln 2 / 2)^12 / 12! = 6e-15).
__device__ __forceinline__ double power_of_two(double y)
{
    constexpr double L = 0.693147180559945309417, kRound = 6755399441055744.0;       // 1.5 x 2^52: an addition rounds to whole numbers
    const double t = fmax(y, -60.0) + kRound, z = fmax(y, -60.0) - (t - kRound);
    constexpr double L2 = L * L, L3 = L2 * L, L4 = L3 * L, L5 = L4 * L, L6 = L5 * L, L7 = L6 * L, L8 = L7 * L, L9 = L8 * L, L10 = L9 * L, L11 = L10 * L;
    double s = L11 / 39916800.0;
    s = __builtin_fma(s, z, L10 / 3628800.0);
    s = __builtin_fma(s, z, L9 / 362880.0);
    s = __builtin_fma(s, z, L8 / 40320.0);
    s = __builtin_fma(s, z, L7 / 5040.0);
    s = __builtin_fma(s, z, L6 / 720.0);
    s = __builtin_fma(s, z, L5 / 120.0);
    s = __builtin_fma(s, z, L4 / 24.0);
    s = __builtin_fma(s, z, L3 / 6.0);
    s = __builtin_fma(s, z, L2 / 2.0);
    s = __builtin_fma(s, z, L);
    s = __builtin_fma(s, z, 1.0);
    return __hiloint2double(__double2hiint(s) + (__double2loint(t) << 20), __double2loint(s));
}
__device__ __forceinline__ double weight_of(uint32_t key, const Row& r)
{
    // (the largest is 1 where it is infinite too, and its distance to the others no number)
    const double w = power_of_two(((double)logit_of(key) - (double)r.top) * r.by);
    return key <= kLowestKey ? 0.0 : key == r.top_key ? 1.0 : w;
}
// w 2^43 to the nearest whole number: what an addition of 2^52 leaves in the fraction
__device__ __forceinline__ uint64_t whole(double w) { return (uint64_t)__double_as_longlong(__builtin_fma(w, kOne, 4503599627370496.0)) & 0xfffffffffffffull; }

// Bins of the distance to the largest logit, 64 to an octave from 1/16 to 4096; a larger logit never has the higher bin.
__device__ __forceinline__ int bin_of(uint32_t key, const Row& r)
{
    const float d = r.top_key == key ? 0.f : r.top - logit_of(key);
    return min(kBins - 1, max(0, (int)(__float_as_uint(d) >> 17) - (123 << 6) + 1));
}

// inclusive sum over the threads of the workgroup; *total: over all
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* red, uint64_t* total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) red[wave] = v;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const uint64_t s = red[w];
        before += w < wave ? s : 0;
        all += s;
    }
    *total = all;
    return v + before;
}
// what a share of a total is, as the least sum that has it: 1 at least
__device__ __forceinline__ uint64_t share_of(double p, uint64_t total)
{
    return min((uint64_t)fmin((double)total, fmax(1.0, ceil(p * (double)total))), total);
}
// the first sum in index order that exceeds u of the total is the first that reaches this
__device__ __forceinline__ uint64_t drawn(const SampleArgs& A, int row, uint64_t total)
{
    const double u = fmin(fmax((double)A.uniforms[row], 0.0), 1.0);
    return min((uint64_t)(u * (double)total) + 1, total);
}
__device__ __forceinline__ void chosen(const SampleArgs& A, int row, int index, uint32_t key, uint64_t total, const Row& r)
{
    A.tokens[row] = index;
    if (A.probabilities) A.probabilities[row] = (float)(weight_of(key, r) * kOne / (double)total);
}

// grid (chunks, rows)
__global__ void __launch_bounds__(kThreads) sample_top_kernel(const SampleArgs A)
{
    __shared__ uint64_t red[kWaves];
    const int row = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int begin = (blockIdx.x * kWaves + wave) * A.seg_len, end = min(A.vocab, begin + A.seg_len);
    const float* x = A.logits + row * A.ld;
    uint64_t best = 0;
#pragma unroll 4
    for (int i = begin + lane; i < end; i += 64) best = max(best, (uint64_t)key_of(x[i]) << 32 | (uint32_t)~i);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) best = max(best, shfl_xor64(best, o));
    if ((lane & 15) == 0) A.groups[(row * A.chunks + blockIdx.x) * kGroups + threadIdx.x / 16] = (uint32_t)(best >> 32);
    best = max(best, shfl_xor64(best, 16));
    best = max(best, shfl_xor64(best, 32));
    if (lane == 0) red[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 0; w < kWaves; ++w) best = max(best, red[w]);
        A.tops[row * A.chunks + blockIdx.x] = best;
    }
}

// Candidates in bins up to `last` among the segments seg0 .. seg0 + segs - 1 (at most 64), in order, from list on; returns how many.
// Of the candidates most segments have none, which their groups tell.
__device__ __forceinline__ uint32_t list_segments(const SampleArgs& A, const Row& r, int row, int seg0, int segs, int last, uint64_t* list)
{
    const int lane = threadIdx.x & 63, begin = seg0 * A.seg_len, end = min(A.vocab, begin + segs * A.seg_len);
    const float* x = A.logits + row * A.ld;
    uint32_t top = 0;
    if (lane < segs) {
        const uint4 g = *reinterpret_cast<const uint4*>(A.groups + (row * A.chunks * kWaves + seg0 + lane) * 4);
        top = max(max(g.x, g.y), max(g.z, g.w));
    }
    const uint64_t some = __ballot(top > kLowestKey && bin_of(top, r) <= last);
    // bin_of(l) <= last in one subtraction, where no infinity is in the way
    const bool plain = last < kBins - 1 && r.top < INFINITY;
    const float border = __uint_as_float((uint32_t)(last + (123 << 6)) << 17);
    uint32_t n = 0;
    constexpr int W = 16;
    for (int i0 = begin; i0 < end; i0 += 64 * W) {
        const int s0 = (i0 - begin) / A.seg_len, s1 = min(63, (i0 - begin + 64 * W - 1) / A.seg_len);
        if (((some >> s0) & (~0ull >> (63 - (s1 - s0)))) == 0) continue;
        float l[W];
#pragma unroll
        for (int j = 0; j < W; ++j) l[j] = i0 + 64 * j + lane < end ? x[i0 + 64 * j + lane] : -INFINITY;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const bool in = plain ? r.top - l[j] < border : key_of(l[j]) > kLowestKey && bin_of(key_of(l[j]), r) <= last;
            const uint64_t lanes = __ballot(in);
            if (lanes == 0) continue;
            if (in) list[n + __popcll(lanes & ((1ull << lane) - 1))] = (uint64_t)key_of(l[j]) << 32 | (uint32_t)(i0 + 64 * j + lane);
            n += __popcll(lanes);
        }
    }
    return n;
}

__global__ void __launch_bounds__(kThreads) sample_sums_kernel(const SampleArgs A)
{
    __shared__ uint64_t hist[kBins], red[kWaves];
    __shared__ int cut;
    const int row = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // (asked for beside what the row's settings come from)
    const int groups = A.chunks * kGroups;
    uint32_t tops[kMaxChunks * kGroups / kThreads];
#pragma unroll
    for (int i = 0; i < kMaxChunks * kGroups / kThreads; ++i) {
        const int g = threadIdx.x + i * kThreads;
        tops[i] = g < groups ? A.groups[row * groups + g] : 0;
    }
    const Row r = row_of(A, row);
    if (r.kind == kDone) return;
    const float* x = A.logits + row * A.ld;
    const int seg = chunk * kWaves + wave, begin = seg * A.seg_len, end = min(A.vocab, begin + A.seg_len);
    if (r.kind == kWhole) {
        uint64_t sum = 0;
#pragma unroll 4
        for (int i = begin + lane; i < end; i += 64) {
            const double w = weight_of(key_of(x[i]), r);
            sum += w >= r.least || i == r.top_index ? whole(w) : 0;
        }
        sum = wave_sum(sum);
        if (lane == 0) A.sums[(int64_t)row * A.chunks * kWaves + seg] = sum;
        return;
    }
    hist[threadIdx.x] = 0;
    __syncthreads();
    if (r.kind == kTopK) {
#pragma unroll
        for (int i = 0; i < kMaxChunks * kGroups / kThreads; ++i)
            if (tops[i] > kLowestKey) atomicAdd((unsigned long long*)&hist[bin_of(tops[i], r)], 1ull);
        if (threadIdx.x == 0) cut = kBins - 1;                       // (fewer groups with a candidate than k)
        __syncthreads();
        uint64_t all;
        const uint64_t mine = hist[threadIdx.x], cum = block_scan(mine, red, &all);
        if (cum >= (uint64_t)r.k && cum - mine < (uint64_t)r.k) cut = threadIdx.x;
        __syncthreads();
        const uint32_t n = list_segments(A, r, row, seg, 1, cut, A.list + ((int64_t)row * A.chunks * kWaves + seg) * A.seg_len);
        if (lane == 0) A.counts[(int64_t)row * A.chunks * kWaves + seg] = n;
        return;
    }
#pragma unroll 4
    for (int i = begin + lane; i < end; i += 64) {
        const uint32_t key = key_of(x[i]);
        const uint64_t v = key <= kLowestKey ? 0 : r.kind == kManyK ? 1 : whole(weight_of(key, r));
        if (v) atomicAdd((unsigned long long*)&hist[bin_of(key, r)], (unsigned long long)v);
    }
    __syncthreads();
    A.hist[((int64_t)row * A.chunks + chunk) * kBins + threadIdx.x] = hist[threadIdx.x];
}

struct Prefix {
    uint32_t key;                // logits above stay, and `ties` of the equal ones
    uint32_t ties;
};

__global__ void __launch_bounds__(kThreads) sample_draw_kernel(const SampleArgs A)
{
    __shared__ uint64_t red[kWaves], hist[256], rest;
    __shared__ int place;
    __shared__ uint32_t offset[kMaxChunks * kWaves + 1], keys[kListed], indices[kListed];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, segs = A.chunks * kWaves;
    const float* x = A.logits + row * A.ld;
    // (both asked for beside what the row's settings come from; which of them was written depends on these)
    const uint32_t count = tid < segs ? A.counts[(int64_t)row * segs + tid] : 0;
    const uint64_t sum_here = tid < segs ? A.sums[(int64_t)row * segs + tid] : 0;
    const Row r = row_of(A, row);
    if (r.kind == kDone) {
        if (tid == 0) {
            A.tokens[row] = r.top_key <= kLowestKey ? -1 : r.top_index;
            if (A.probabilities) A.probabilities[row] = r.top_key <= kLowestKey ? 0.f : 1.f;
        }
        return;
    }
    if (r.kind == kWhole) {
        // the segment that the draw falls in, then the place in it
        uint64_t total;
        const uint64_t mine = sum_here, cum = block_scan(mine, red, &total), want = drawn(A, row, total);
        if (cum >= want && cum - mine < want) {
            rest = want - (cum - mine);
            place = tid;
        }
        __syncthreads();
        uint64_t left = rest;
        const int begin = place * A.seg_len, end = min(A.vocab, begin + A.seg_len);
        for (int i0 = begin; i0 < end; i0 += kThreads) {
            const int i = i0 + tid;
            const uint32_t key = i < end ? key_of(x[i]) : 0;
            const double w = weight_of(key, r);
            const uint64_t v = w >= r.least || i == r.top_index ? whole(w) : 0;
            uint64_t all;
            const uint64_t c = block_scan(v, red, &all);
            if (c >= left && c - v < left) chosen(A, row, i, key, total, r);
            if (all >= left) return;                                 // uniform
            left -= all;
        }
        return;
    }

    // all weights, where a share of them is wanted; the lists are of segments, or of the run of segments of each wavefront here
    uint64_t weights_of_all = 0;
    int lists = segs, list_len = A.seg_len;
    uint32_t listed_here;
    if (r.kind != kTopK) {
        uint64_t mine = 0, total;
#pragma unroll 8
        for (int c = 0; c < A.chunks; ++c) mine += A.hist[((int64_t)row * A.chunks + c) * kBins + tid];
        const uint64_t cum = block_scan(mine, red, &total), need = r.kind == kManyK ? (uint64_t)r.k : share_of(r.p, total);
        if (tid == 0) place = kBins - 1;                             // (fewer candidates than k)
        __syncthreads();
        if (cum >= need && cum - mine < need) place = tid;
        __syncthreads();
        const int last = place;
        lists = kWaves;
        list_len = A.chunks * A.seg_len;
        listed_here = list_segments(A, r, row, wave * A.chunks, A.chunks, last, A.list + (int64_t)row * segs * A.seg_len + (int64_t)wave * list_len);
        weights_of_all = total;
        if (lane == 0) offset[wave + 1] = listed_here;
        __syncthreads();
    }

    // the listed candidates by their position in index order
    uint64_t listed;
    {
        const uint64_t mine = tid >= lists ? 0 : r.kind == kTopK ? count : offset[tid + 1], cum = block_scan(mine, red, &listed);
        if (tid < lists) offset[tid + 1] = (uint32_t)cum;
        if (tid == 0) offset[0] = 0;
        __syncthreads();
    }
    const int n = (int)listed;
    const uint64_t* list = A.list + (int64_t)row * segs * A.seg_len;
    const bool near = n <= kListed;
    // list of position i: the last one that begins at or before it
    auto entry_at = [&](int i) {
        int lo = 0, hi = lists - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if ((int)offset[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        return list[(int64_t)lo * list_len + (i - (int)offset[lo])];
    };
    if (near) {
        for (int i = tid; i < n; i += kThreads) {
            const uint64_t e = entry_at(i);
            indices[i] = (uint32_t)e;
            keys[i] = (uint32_t)(e >> 32);
        }
        __syncthreads();
    }
    auto at = [&](int i, uint32_t* key) {
        if (near) {
            *key = keys[i];
            return (int)indices[i];
        }
        const uint64_t e = entry_at(i);
        *key = (uint32_t)(e >> 32);
        return (int)(uint32_t)e;
    };

    if (n <= kRanked) {
        // Everyone counts who is ahead and what they weigh; the others are shared by as many threads as there are for each.
        struct Entry { uint64_t order, weight; };
        __shared__ Entry entries[kRanked];
        __shared__ uint64_t aheads[kRanked];
        __shared__ int ranks[kRanked];
        const bool in = tid < n;
        const uint32_t key = in ? keys[tid] : 0;
        const double w = in ? weight_of(key, r) : 0.0;
        const uint64_t mine = in ? whole(w) : 0;
        if (tid < kRanked) {
            entries[tid] = {(uint64_t)key << 32 | (uint32_t)~tid, mine};
            aheads[tid] = 0;
            ranks[tid] = 0;
        }
        __syncthreads();
        {
            const int wide = n <= 64 ? 64 : n <= 128 ? 128 : 256, e = tid & (wide - 1), share = (n + kThreads / wide - 1) / (kThreads / wide);
            const int j0 = min(n, tid / wide * share), j1 = min(n, j0 + share);
            const uint64_t order = entries[e].order;
            int rank = 0;
            uint64_t ahead = 0;
#pragma unroll 4
            for (int j = j0; j < j1; ++j) {
                const Entry o = entries[j];
                const bool before = o.order > order;
                rank += before;
                ahead += before ? o.weight : 0;
            }
            if (rank > 0) {
                atomicAdd(&ranks[e], rank);
                atomicAdd((unsigned long long*)&aheads[e], (unsigned long long)ahead);
            }
        }
        __syncthreads();
        const int rank = in ? ranks[tid] : 0;
        const uint64_t ahead = in ? aheads[tid] : 0;
        bool stays = in && (r.kind == kTopP || rank < r.k);
        if (r.p < 1.0) {
            uint64_t total = weights_of_all;
            if (r.kind != kTopP) block_scan(stays ? mine : 0, red, &total);
            stays = stays && (rank == 0 || ahead < share_of(r.p, total));
        }
        stays = stays && (w >= r.least || rank == 0);
        uint64_t total;
        const uint64_t v = stays ? mine : 0, cum = block_scan(v, red, &total), want = drawn(A, row, total);
        if (cum >= want && cum - v < want) chosen(A, row, (int)indices[tid], key, total, r);
        return;
    }

    // A key eight bits at a time: the digit in whose bin `left` falls, counted from the top; left becomes what is needed of that bin.
    // False where all bins together hold less.
    auto each = [&](auto&& f) {
        for (int i = tid; i < n; i += kThreads) {
            uint32_t key;
            at(i, &key);
            f(key);
        }
    };
    auto select = [&](uint64_t& left, uint32_t& prefix, auto&& values) {
        prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            if (tid == 0) place = -1;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            values([&](uint32_t key, uint64_t v) {
                if ((key & mask) == prefix) atomicAdd((unsigned long long*)&hist[(key >> shift) & 255], (unsigned long long)v);
            });
            __syncthreads();
            if (wave == 0) {
                uint64_t b[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    b[i] = hist[255 - 4 * lane - i];
                    sum += b[i];
                }
                const uint64_t cum = wave_scan(sum), lanes = __ballot(cum >= left);
                if (lanes != 0 && lane == __ffsll((unsigned long long)lanes) - 1) {
                    uint64_t needed = left - (cum - sum);
                    int i = 0;
                    while (i < 3 && b[i] < needed) needed -= b[i++];
                    place = 255 - 4 * lane - i;
                    rest = needed;
                }
            }
            __syncthreads();
            if (place < 0) return false;                             // uniform
            prefix |= (uint32_t)place << shift;
            left = rest;
            __syncthreads();
        }
        return true;
    };
    Prefix P{kLowestKey, 0};
    if (r.kind != kTopP) {
        uint64_t left = (uint64_t)r.k;
        uint32_t key;
        if (select(left, key, [&](auto&& add) { each([&](uint32_t k) { add(k, 1); }); })) P = {key, (uint32_t)left};
    }
    if (r.p < 1.0) {
        const uint64_t tied = P.ties ? whole(weight_of(P.key, r)) * P.ties : 0;
        uint64_t total = weights_of_all;
        if (r.kind != kTopP) {
            uint64_t sum = 0;
            each([&](uint32_t key) { sum += key > P.key ? whole(weight_of(key, r)) : 0; });
            block_scan(sum, red, &total);
            total += tied;
        }
        uint64_t left = share_of(r.p, total);
        uint32_t key;
        select(left, key, [&](auto&& add) {
            each([&](uint32_t k) {
                if (k > P.key) add(k, whole(weight_of(k, r)));
            });
            if (tid == 0 && tied) add(P.key, tied);
        });
        const uint64_t w = max(whole(weight_of(key, r)), (uint64_t)1);
        const uint32_t ties = (uint32_t)min((left + w - 1) / w, (uint64_t)0xffffffffu);
        if (key > P.key) P = {key, ties};
        else P.ties = min(P.ties, ties);
    }
    // Every thread has a run of positions.  First the one that holds the last of the equal ones that stay.
    const int per = (n + kThreads - 1) / kThreads, first = min(n, tid * per), end = min(n, first + per);
    int tie_end = 0;
    if (P.ties) {
        uint64_t seen = 0, all;
        uint32_t key;
        for (int i = first; i < end; ++i) {
            at(i, &key);
            seen += key == P.key;
        }
        const uint64_t before = block_scan(seen, red, &all) - seen;
        if (tid == 0) place = n;
        __syncthreads();
        if (before < P.ties && before + seen >= P.ties) {
            uint64_t c = before;
            int i = first;
            for (; c < P.ties; ++i) {
                at(i, &key);
                c += key == P.key;
            }
            place = i;
        }
        __syncthreads();
        tie_end = place;
    }
    auto kept = [&](int i, uint32_t* key, int* index) -> uint64_t {
        *index = at(i, key);
        if (*key < P.key || (*key == P.key && i >= tie_end)) return 0;
        const double w = weight_of(*key, r);
        return w >= r.least || *index == r.top_index ? whole(w) : 0;
    };
    uint64_t sum = 0, total;
    uint32_t key = 0;
    int index = 0;
    for (int i = first; i < end; ++i) sum += kept(i, &key, &index);
    const uint64_t cum = block_scan(sum, red, &total), want = drawn(A, row, total);
    if (cum >= want && cum - sum < want) {
        uint64_t c = cum - sum;
        for (int i = first; c < want; ++i) c += kept(i, &key, &index);
        chosen(A, row, index, key, total, r);
    }
}

struct SampleLayout {
    int chunks, seg_len;
    size_t tops, groups, hist, sums, counts, list, total;            // byte offsets; for `rows` rows
};
SampleLayout layout_of(int rows, int vocab)
{
    SampleLayout L{};
    // chunks that are worth a workgroup, two workgroups per CU at most
    L.chunks = std::max(1, std::min({kMaxChunks, 2 * device_info().num_cus / rows, (vocab + kMinChunk - 1) / kMinChunk}));
    L.seg_len = ((vocab + L.chunks * kWaves - 1) / (L.chunks * kWaves) + 63) / 64 * 64;
    size_t off = 0;
    auto take = [&](size_t b) {
        const size_t o = off;
        off += (b + 255) & ~(size_t)255;
        return o;
    };
    const size_t n = rows, segs = (size_t)L.chunks * kWaves;
    L.tops = take(n * L.chunks * 8);
    L.groups = take(n * L.chunks * kGroups * 4);
    L.hist = take(n * L.chunks * kBins * 8);
    L.sums = take(n * segs * 8);
    L.counts = take(n * segs * 4);
    L.list = take(n * segs * L.seg_len * 8);
    L.total = off;
    return L;
}
// Rows of a launch.  Their lists take twice the memory of their logits, and a row takes 17 KiB for its histogram and list at least; a stream keeps what a call
// took.
int rows_at_once(int rows, int vocab)
{
    constexpr size_t kMost = (size_t)5 << 26;
    int n = std::min(rows, 65535);
    for (;;) {
        const size_t bytes = layout_of(n, vocab).total;
        if (n == 1 || bytes <= kMost) return n;
        n = std::max(1, std::min(n - 1, (int)((double)n * (double)kMost / (double)bytes)));
    }
}

}  // namespace

size_t sample_ws_bytes(int rows, int vocab) { return layout_of(rows_at_once(rows, vocab), vocab).total; }

bool launch_sample(const float* logits, int64_t ld, int rows, int vocab, const float* uniforms, const float* temperature, const int32_t* top_k,
                   const float* top_p, const float* min_p, int32_t* tokens, float* probabilities, void* ws, hipStream_t stream)
{
    const int most = rows_at_once(rows, vocab);
    const SampleLayout L = layout_of(most, vocab);
    char* base = static_cast<char*>(ws);
    for (int r0 = 0; r0 < rows; r0 += most) {
        const int n = std::min(most, rows - r0);
        SampleArgs a{};
        a.logits = logits + r0 * ld;
        a.ld = ld;
        a.vocab = vocab;
        a.chunks = L.chunks;
        a.seg_len = L.seg_len;
        a.uniforms = uniforms + r0;
        a.temperature = temperature + r0;
        a.top_k = top_k ? top_k + r0 : nullptr;
        a.top_p = top_p ? top_p + r0 : nullptr;
        a.min_p = min_p ? min_p + r0 : nullptr;
        a.tokens = tokens + r0;
        a.probabilities = probabilities ? probabilities + r0 : nullptr;
        a.tops = reinterpret_cast<uint64_t*>(base + L.tops);
        a.hist = reinterpret_cast<uint64_t*>(base + L.hist);
        a.groups = reinterpret_cast<uint32_t*>(base + L.groups);
        a.sums = reinterpret_cast<uint64_t*>(base + L.sums);
        a.counts = reinterpret_cast<uint32_t*>(base + L.counts);
        a.list = reinterpret_cast<uint64_t*>(base + L.list);
        const dim3 grid(L.chunks, n), block(kThreads);
        hipLaunchKernelGGL(sample_top_kernel, grid, block, 0, stream, a);
        if (!hip_ok(hipGetLastError(), "sample launch")) return false;
        hipLaunchKernelGGL(sample_sums_kernel, grid, block, 0, stream, a);
        if (!hip_ok(hipGetLastError(), "sample launch")) return false;
        hipLaunchKernelGGL(sample_draw_kernel, dim3(n), block, 0, stream, a);
        if (!hip_ok(hipGetLastError(), "sample launch")) return false;
    }
    return true;
}

}  // namespace tship
