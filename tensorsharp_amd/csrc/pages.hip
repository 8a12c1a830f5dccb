// The life of a cache's pages: who has which (tables, reference counts, lengths, all on the device), and copies of pages between caches.
//
//   page_drop_kernel, page_plan_kernel, page_fill_kernel (page_few_kernel)          sequences get other lengths
//   fork_plan_kernel (fork_tables_kernel or fork_rows_kernel, fork_store_kernel)    sequences go on from what others have
//   compact_plan_kernel (compact_tables_kernel)              used pages move to the front
//   copy_pages_kernel                                        pages of one cache or two, of one type or two
//
// The lists are short next to the caches (a reference count for each page, an entry for each page of a sequence), so what counts is the number of dependent steps.  What
// has to know all sequences in order - sums up to a sequence - is one workgroup, and so are the pages of a fork's few copies and of a compaction, thousands in a
// step; where many pages are given out every wavefront has 64 of them, and their sums come between two launches.  What walks over the tables has a workgroup for
// 1024 entries.  One to three launches a call, nothing that one workgroup waits for another for.  Counts change by atomic additions of whole numbers, whose
// order changes nothing.
#include "tship_internal.h"
#include "mx4.h"
#include "paged_tiles.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

namespace tship {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kRowThreads = 256, kRowEntries = 4 * kRowThreads;     // of a table that a workgroup walks over

constexpr int kLocal = 4096;         // sequences of which a workgroup keeps what it knows in LDS

// what the calls keep in scratch: a few numbers, some for each sequence, one for each page, and a table's rows
struct Scratch {
    int* head;            // [16]
    int *a, *b, *c, *d;   // [sequences]
    int* pages;           // [pages]
    int* rows;            // [sequences x entries]
};
__host__ __device__ __forceinline__ Scratch scratch_of(const PagePoolArgs& P)
{
    int* at = P.scratch;
    const int64_t n = P.seqs;
    return {at, at + 16, at + 16 + n, at + 16 + 2 * n, at + 16 + 3 * n, at + 16 + 4 * n, at + 16 + 4 * n + P.num_pages};
}

__device__ __forceinline__ int pages_of(const PagePoolArgs& P, int64_t tokens)
{
    if (tokens <= 0) return 0;
    return (int)min((int64_t)P.max_pages, ((int64_t)tokens + P.page_size - 1) / P.page_size);
}
__device__ __forceinline__ bool is_page(const PagePoolArgs& P, int e) { return (uint32_t)e < (uint32_t)P.num_pages; }

// Sum of v over the workgroup's threads before this one, and over all of them.
__device__ __forceinline__ int64_t before_me(int64_t v, int64_t* all)
{
    __shared__ int64_t waves[kPlanWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t sum = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t below = __shfl_up((long long)sum, o);
        if (lane >= o) sum += below;
    }
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    int64_t first = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        if (w < wave) first += waves[w];
        total += waves[w];
    }
    __syncthreads();
    *all = total;
    return first + sum - v;
}

// the same of numbers whose sum has 32 bits, in registers
__device__ __forceinline__ int before_me(int v, int* all)
{
    __shared__ int waves[kPlanWaves];
    const int scan = lane_scan(v), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((threadIdx.x & 63) == 63) waves[wave] = scan;
    __syncthreads();
    int first = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        if (w < wave) first += waves[w];
        total += waves[w];
    }
    __syncthreads();
    *all = total;
    return first + scan - v;
}

// The lowest free pages.  A thread takes 16 pages that follow one another.
constexpr int kScan = 16 * kPlanThreads;
__device__ __forceinline__ uint32_t free_here(const int32_t* references, int p, int end)
{
    uint32_t bits = 0;
    if (p < end - 15) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int4 r = *reinterpret_cast<const int4*>(references + p + 4 * i);
            bits |= (uint32_t)((r.x <= 0) | (r.y <= 0) << 1 | (r.z <= 0) << 2 | (r.w <= 0) << 3) << (4 * i);
        }
    } else {
        for (int i = 0; i < 16 && p < end - i; ++i) bits |= (uint32_t)(references[p + i] <= 0) << i;
    }
    return bits;
}
// Calls each(number, page) for the lowest `want` free pages or as many as there are; returns how many it found (perhaps some more).
template <typename F>
__device__ __forceinline__ int find_free(const int32_t* references, int pages, int want, F&& each)
{
    int found = 0;
    for (int64_t p = 0; p < pages && found < want; p += kScan) {
        const int64_t mine = p + 16 * (int)threadIdx.x;
        uint32_t free = mine < pages ? free_here(references, (int)mine, pages) : 0;
        int all;
        int number = found + before_me((int)__popc(free), &all);
        for (; free != 0 && number < want; free &= free - 1) each(number++, (int)mine + __ffs(free) - 1);
        found += all;
    }
    return found;
}

// Pages in steps of up to 32768: wavefront w has 256 L of them that follow one another, lane i four of each 256, so that L loads of 16 bytes a lane are under way at once and lie
// side by side.
constexpr int kLoads = 8;
struct Step {
    int4 r[kLoads];              // references; -1 where there is no page
    int loads;                   // L
    int first;                   // this wavefront's
};
__device__ __forceinline__ int pages_in(int loads) { return loads * 256 * kPlanWaves; }
__device__ __forceinline__ Step step_at(const int32_t* references, int begin, int end)
{
    Step t;
    t.loads = max(0, min(kLoads, (end - begin + pages_in(1) - 1) / pages_in(1)));
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    t.first = begin + wave * 256 * t.loads;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int p = t.first + 256 * i + 4 * lane;
        t.r[i] = int4{-1, -1, -1, -1};
        if (i < t.loads && p < end) {
            if (p + 4 <= end) t.r[i] = *reinterpret_cast<const int4*>(references + p);
            else {
                t.r[i].x = references[p];
                if (p + 1 < end) t.r[i].y = references[p + 1];
                if (p + 2 < end) t.r[i].z = references[p + 2];
            }
        }
    }
    return t;
}
// four bits of each load: which pages are in use
__device__ __forceinline__ uint32_t used_of(const Step& t)
{
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) bits |= (uint32_t)((t.r[i].x > 0) | (t.r[i].y > 0) << 1 | (t.r[i].z > 0) << 2 | (t.r[i].w > 0) << 3) << (4 * i);
    return bits;
}
// of one number a wavefront: the sum of those before this one's, and of all
__device__ __forceinline__ int waves_before(int mine, int* all)
{
    __shared__ int sums[kPlanWaves];
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = mine;
    __syncthreads();
    int first = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        if (w < (int)(threadIdx.x >> 6)) first += sums[w];
        total += sums[w];
    }
    __syncthreads();
    *all = total;
    return first;
}
// Calls each(page, used, number of used pages before it) for every page of the step that exists; before: of the wavefronts before
template <typename F>
__device__ __forceinline__ void pages_of_step(const Step& t, uint32_t used, int before, int end, F&& each)
{
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        if (i >= t.loads) break;
        const uint32_t mine = (used >> (4 * i)) & 15;
        int n = before;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t b = __ballot((mine >> j) & 1);
            n = __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, n));
            before += __popcll(b);
        }
        const int p = t.first + 256 * i + 4 * (threadIdx.x & 63);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (p + j < end) each(p + j, (mine >> j) & 1, n);
            n += (mine >> j) & 1;
        }
    }
}

// Atomic operations on memory are done in the second-level cache: what they leave is read there too, once every wavefront's have arrived.
template <bool LOCAL>
__device__ __forceinline__ int seen(const int* at)
{
    return LOCAL ? *at : __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <bool LOCAL>
__device__ __forceinline__ void put(int* at, int v)
{
    if constexpr (LOCAL) *at = v;
    else __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void settled()
{
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
}

// ---- other lengths -------------------------------------------------------------------------------

// bits of the free pages, in a pool's scratch, and how many of each part of `part` pages are free
constexpr int kPart = 64, kMostParts = 4096;
struct FreePages {
    uint32_t* bits;
    int* counts;
    int parts;
};
__device__ __forceinline__ FreePages free_of(const PagePoolArgs& P, int part)
{
    const int words = (P.num_pages + 63) / 64 * 2;
    int* at = scratch_of(P).pages;
    return {reinterpret_cast<uint32_t*>(at), at + words, (P.num_pages + part - 1) / part};
}

__device__ __forceinline__ int64_t goal_of(const PagePoolArgs& P, const int32_t* lengths, int s)
{
    const int n = lengths[s];
    return n < 0 ? P.context_lens[s] : min((int64_t)n, (int64_t)P.max_pages * P.page_size);
}

// grid (chunks of entries, sequences): entries behind the ends of shorter sequences
__global__ void __launch_bounds__(kRowThreads) page_drop_kernel(const PagePoolArgs P, const int32_t* lengths)
{
    const int s = blockIdx.y;
    const int held = pages_of(P, P.context_lens[s]), goal = pages_of(P, goal_of(P, lengths, s));
    const int first = max(goal, (int)blockIdx.x * kRowEntries), last = min(held, ((int)blockIdx.x + 1) * kRowEntries);
    for (int j = first + threadIdx.x; j < last; j += kRowThreads) {
        int32_t* entry = P.table + s * P.table_stride + j;
        const int e = *entry;
        if (is_page(P, e)) atomicAdd(P.references + e, -1);
        *entry = -1;
    }
}

// Which pages are free, as bits, and how many of every part of them, a wavefront's each; the last workgroup: how many pages each longer sequence needs, and where its
// pages begin in the list of the lowest free ones.  (One workgroup for all of it: 13.6 us for 110000 pages and 24000 wanted; in parts of 64
// pages 4.5, and what follows 4.0 instead of 3.0.  Parts of 256: 3.8 and 6.2.)
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PagePoolArgs P, const int32_t* lengths, int part)
{
    const Scratch W = scratch_of(P);
    const FreePages F = free_of(P, part);
    if (blockIdx.x + 1 < gridDim.x) {
        const int lane = threadIdx.x & 63, number = blockIdx.x * kPlanWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int64_t begin = (int64_t)number * part;
        if (begin >= P.num_pages) return;
        int count = 0;
        for (int64_t p0 = begin; p0 < min(begin + part, (int64_t)P.num_pages); p0 += kPart) {
            int r[kPart / 64];
#pragma unroll
            for (int i = 0; i < kPart / 64; ++i) r[i] = p0 + 64 * i + lane < P.num_pages ? P.references[p0 + 64 * i + lane] : 1;
#pragma unroll
            for (int i = 0; i < kPart / 64; ++i) {
                const uint64_t bits = __ballot(r[i] <= 0);
                count += __popcll(bits);
                if (lane < 2 && p0 + 64 * i < P.num_pages) F.bits[(p0 >> 5) + 2 * i + lane] = (uint32_t)(bits >> (32 * lane));
            }
        }
        if (lane == 0) F.counts[number] = count;
        return;
    }
    int64_t need = 0, copies = 0;
    for (int s0 = 0; s0 < P.seqs; s0 += kPlanThreads) {
        const int s = s0 + threadIdx.x;
        int wants = 0, copied = 0, held = 0;
        if (s < P.seqs) {
            const int64_t tokens = P.context_lens[s], goal = goal_of(P, lengths, s);
            held = pages_of(P, tokens);
            if (goal > tokens) {
                wants = pages_of(P, goal) - held;
                // (the last page is begun, and not this sequence's alone)
                if (held > 0 && tokens % P.page_size != 0) {
                    const int e = P.table[s * P.table_stride + held - 1];
                    copied = is_page(P, e) && P.references[e] > 1;
                }
            }
        }
        int64_t all, copies_here;
        const int64_t at = need + before_me(wants + copied, &all), number = copies + before_me(copied, &copies_here);
        if (s < P.seqs) {
            W.a[s] = held;
            W.b[s] = (int)min(at, (int64_t)INT32_MAX);
            W.c[s] = copied ? (int)number : -1;
        }
        need += all;
        copies += copies_here;
    }
    if (threadIdx.x == 0) {
        W.head[0] = (int)(need & UINT32_MAX);
        W.head[1] = (int)(need >> 32);
        W.head[2] = (int)copies;
    }
}

// the last of the numbers (which do not fall) that is at most i; of(s): the s-th, the first is at most i
template <typename F>
__device__ __forceinline__ int last_at_most(int count, int i, F&& of)
{
    int s = 0;
    for (int above = count; above - s > 1;) {
        const int half = (s + above) >> 1;
        if (of(half) <= i) s = half;
        else above = half;
    }
    return s;
}
// Page number i of those that are given out goes to sequence s, whose first is number `at`: behind the `held` that it has, or, first of all, in the place of the begun page that
// others have (copy: its number among the copies, -1: none).
__device__ __forceinline__ void give_page(const PagePoolArgs& P, int i, int page, int s, int at, int held, int copy, int32_t* moves)
{
    int32_t* row = P.table + s * P.table_stride;
    P.references[page] = 1;
    if (copy < 0 || i > at) {
        row[held + i - at - (copy >= 0)] = page;
    } else {
        const int begun = row[held - 1];
        row[held - 1] = page;
        atomicAdd(P.references + begun, -1);
        moves[2 * copy] = begun;
        moves[2 * copy + 1] = page;
    }
}

// Each free page among the lowest finds the entry that it goes into, if there are enough; the last workgroup: lengths, and what else is to be said.  LOCAL: what is
// known of the sequences fits LDS, where the page's sequence is looked for by halves.
template <bool LOCAL>
__global__ void __launch_bounds__(kPlanThreads) page_fill_kernel(const PagePoolArgs P, const int32_t* lengths, int32_t* moves, int32_t* missing, int part)
{
    __shared__ int local[LOCAL ? 3 * kLocal : 1], sums[kPlanWaves][2];
    const Scratch W = scratch_of(P);
    const FreePages F = free_of(P, part);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, first = blockIdx.x * kPlanWaves;
    const bool last = blockIdx.x + 1 == gridDim.x;
    const int64_t begin = (int64_t)(first + wave) * part, end = last ? 0 : min(begin + part, (int64_t)P.num_pages);
    // (what there is to read is asked for at once: need and copies, bits, sequences and counts)
    const int low = W.head[0], high = W.head[1], copies = W.head[2];
    auto word = [&](int64_t p0) { return p0 < end ? F.bits[(p0 >> 5) + (lane >> 5)] : 0u; };
    uint32_t next = word(begin);
    const int count = lane < wave && first + lane < F.parts ? F.counts[first + lane] : 0;
    int before = 0, found = 0;                                       // free pages of the workgroups before this one, of all
    for (int i = threadIdx.x; i < F.parts; i += kPlanThreads) {
        const int n = F.counts[i];
        found += n;
        if (i < first) before += n;
    }
    if constexpr (LOCAL) {
        if (!last)
            for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) local[s] = W.b[s], local[kLocal + s] = W.a[s], local[2 * kLocal + s] = W.c[s];
    }
    const int64_t need = (int64_t)high << 32 | (uint32_t)low;
    if (need == 0 && !last) return;
    found = lane_sum(found);
    before = lane_sum(before);
    if (lane == 0) sums[wave][0] = found, sums[wave][1] = before;
    int number = lane_sum(count);
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) all += sums[w][0], number += sums[w][1];
    const bool fits = all >= need;
    if (last) {
        for (int i = threadIdx.x; i < P.seqs; i += kPlanThreads) {
            if (!fits || i >= copies) moves[2 * i] = moves[2 * i + 1] = -1;
            const int64_t tokens = P.context_lens[i], goal = goal_of(P, lengths, i);
            if (goal < tokens || (fits && goal > tokens)) P.context_lens[i] = (int)goal;
        }
        if (threadIdx.x == 0) missing[0] = fits ? 0 : (int)min(need - all, (int64_t)INT32_MAX);
        return;
    }
    if (!fits) return;
    for (int64_t p0 = begin; p0 < end && number < need; p0 += 64) {
        const uint64_t bits = __ballot((next >> (lane & 31)) & 1);
        next = word(p0 + 64);
        const int i = number + __popcll(bits & ((1ull << lane) - 1)), page = (int)p0 + lane;
        number += __popcll(bits);
        if (!((bits >> lane) & 1) || i >= need) continue;
        // (a sequence that wants none begins where the next does)
        const int s = last_at_most(P.seqs, i, [&](int k) { return LOCAL ? local[k] : W.b[k]; });
        give_page(P, i, page, s, LOCAL ? local[s] : W.b[s], LOCAL ? local[kLocal + s] : W.a[s], LOCAL ? local[2 * kLocal + s] : W.c[s], moves);
    }
}

// All of it in one launch, where one workgroup is enough: a thread for each sequence, 16 pages for each thread, 32 entries at most (48 sequences of 2400 tokens, 32 a page: 7 us for
// 11 in three launches, 6 for 10 on the host).
constexpr int kFewEntries = 32 * kPlanThreads;
__host__ __device__ __forceinline__ bool one_workgroup(const PagePoolArgs& P)
{
    return P.seqs <= kPlanThreads && P.num_pages <= kScan && (int64_t)P.seqs * P.max_pages <= kFewEntries;
}
// two sums over the threads before this one and over all of them, one barrier (sums: of this call alone)
struct Two {
    int a, b;
};
__device__ __forceinline__ Two before_me(Two v, Two* all, Two (&sums)[kPlanWaves])
{
    const Two scan{lane_scan(v.a), lane_scan(v.b)};
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((threadIdx.x & 63) == 63) sums[wave] = scan;
    __syncthreads();
    Two first{0, 0}, total{0, 0};
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const Two x = sums[w];
        if (w < wave) first.a += x.a, first.b += x.b;
        total.a += x.a, total.b += x.b;
    }
    *all = total;
    return {first.a + scan.a - v.a, first.b + scan.b - v.b};
}
__global__ void __launch_bounds__(kPlanThreads) page_few_kernel(const PagePoolArgs P, const int32_t* lengths, int32_t* moves, int32_t* missing)
{
    __shared__ int begins[kPlanThreads], held_of[kPlanThreads], copy_of[kPlanThreads];
    __shared__ Two sums[3][kPlanWaves];
    __shared__ uint16_t list[kScan];                                 // the lowest free pages
    const int s = threadIdx.x;
    const bool mine = s < P.seqs;
    const int64_t tokens = mine ? P.context_lens[s] : 0, goal = mine ? goal_of(P, lengths, s) : 0;
    const int held = pages_of(P, tokens), to = pages_of(P, goal);
    const bool grows = goal > tokens;
    const bool into_begun = grows && held > 0 && tokens % P.page_size != 0;
    const int last = into_begun ? P.table[s * P.table_stride + held - 1] : -1;
    auto begin_of = [&](int k) { return begins[k]; };
    // entries behind the ends of shorter sequences, one after the other
    Two drops;
    begins[s] = before_me(Two{max(0, held - to), 0}, &drops, sums[0]).a;
    held_of[s] = to;
    __syncthreads();
    constexpr int kAtOnce = 4;
    for (int i0 = s; i0 < drops.a; i0 += kAtOnce * kPlanThreads) {
        int32_t* entry[kAtOnce];
        int e[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const int i = i0 + k * kPlanThreads;
            e[k] = -1;
            entry[k] = nullptr;
            if (i >= drops.a) continue;
            const int of = last_at_most(P.seqs, i, begin_of);
            entry[k] = P.table + of * P.table_stride + held_of[of] + (i - begins[of]);
            e[k] = *entry[k];
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (is_page(P, e[k])) atomicAdd(P.references + e[k], -1);
            if (entry[k]) *entry[k] = -1;
        }
    }
    settled();
    // what longer ones need, and free pages
    uint32_t free = 16 * s < P.num_pages ? free_here(P.references, 16 * s, P.num_pages) : 0;
    // (the last page is begun, and not this sequence's alone)
    const int copied = is_page(P, last) && seen<false>(P.references + last) > 1;
    Two need, found;
    const Two at = before_me(Two{(grows ? to - held : 0) + copied, copied}, &need, sums[1]);
    int i = before_me(Two{(int)__popc(free), 0}, &found, sums[2]).a;
    const bool fits = found.a >= need.a;
    begins[s] = at.a;
    held_of[s] = held;
    copy_of[s] = copied ? at.b : -1;
    for (; fits && free != 0 && i < need.a; free &= free - 1) list[i++] = (uint16_t)(16 * s + __ffs(free) - 1);
    __syncthreads();
    for (int n = s; fits && n < need.a; n += kPlanThreads) {
        const int of = last_at_most(P.seqs, n, begin_of);
        give_page(P, n, list[n], of, begins[of], held_of[of], copy_of[of], moves);
    }
    if (mine) {
        if (!fits || s >= need.b) moves[2 * s] = moves[2 * s + 1] = -1;
        if (goal < tokens || (fits && grows)) P.context_lens[s] = (int)goal;
    }
    if (s == 0) missing[0] = fits ? 0 : need.a - found.a;
}

// ---- forks ---------------------------------------------------------------------------------------

// One workgroup; LOCAL: what it works out of sequences fits LDS (4096 of them; through memory each of its steps is a trip there and back, 9.4 us for 32 sequences).  For the kernels behind
// it a: the sequence that each becomes, c: the fresh page in place of the begun one, -1: none, d: tokens before
// TABLES: and the tables, where their entries are 16 a thread at most (32 beams of 2000 tokens: 2 us less than in two launches)
constexpr int kForkEach = 16;
template <bool LOCAL, bool TABLES>
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const PagePoolArgs P, const int32_t* children, const int32_t* parents, int count,
                                                                 int32_t* moves, int32_t* missing)
{
    extern __shared__ __attribute__((aligned(16))) int local[];
    const Scratch W = scratch_of(P);
    // of: that each becomes; low: the lowest that becomes it; tokens and begun page before; in LDS also the number of each one's copy and their pages, and before
    // these the last pair of each, with its number above
    int *of_all = LOCAL ? local : W.a, *low = LOCAL ? local + kLocal : W.b, *tokens = LOCAL ? local + 2 * kLocal : W.d, *begun = LOCAL ? local + 3 * kLocal : W.c;
    int *number_of = LOCAL ? local + 4 * kLocal : W.rows, *fresh_of = local + 5 * kLocal;           // (rows of the table come there later)
    unsigned long long* pairs = reinterpret_cast<unsigned long long*>(local + 4 * kLocal);
    auto there = [] {
        if constexpr (LOCAL) __syncthreads();
        else settled();
    };
    for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) {
        if constexpr (LOCAL) pairs[s] = 0;
        else put<LOCAL>(of_all + s, -1);
        put<LOCAL>(low + s, P.seqs);
        const int n = P.context_lens[s], held = pages_of(P, n);
        int page = -1;
        if (held > 0 && n % P.page_size != 0 && n <= (int64_t)P.max_pages * P.page_size) page = P.table[s * P.table_stride + held - 1];
        tokens[s] = n;
        begun[s] = is_page(P, page) ? page : -1;
    }
    there();
    // (lists may have as many pairs as 32 bits count: what walks over them counts in 64)
    for (int64_t i = threadIdx.x; i < count; i += kPlanThreads) {
        const int child = children[i], parent = parents[i];
        if ((uint32_t)child >= (uint32_t)P.seqs || (uint32_t)parent >= (uint32_t)P.seqs) continue;
        if constexpr (LOCAL) atomicMax(pairs + child, (unsigned long long)(i + 1) << 32 | (uint32_t)parent);
        else atomicMax(of_all + child, (int)i);
    }
    there();
    for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) {
        int of = s;
        if constexpr (LOCAL) {
            if (const unsigned long long pair = pairs[s]) of = (int)(uint32_t)pair;
        } else {
            if (const int pair = seen<LOCAL>(of_all + s); pair >= 0) of = parents[pair];
        }
        put<LOCAL>(of_all + s, of);
        atomicMin(low + of, s);
    }
    there();
    // (a parent that stays what it is keeps its begun page)
    int need = 0;
    for (int s0 = 0; s0 < P.seqs; s0 += kPlanThreads) {
        const int s = s0 + threadIdx.x;
        int copied = 0, of = 0;
        if (s < P.seqs) {
            of = seen<LOCAL>(of_all + s);
            const int keeper = seen<LOCAL>(of_all + of) == of ? of : seen<LOCAL>(low + of);
            copied = keeper != s && begun[of] >= 0;
        }
        int all;
        const int number = need + before_me(copied, &all);
        if (copied) moves[2 * number] = begun[of];                   // (as many as there are children at most)
        if (s < P.seqs) number_of[s] = copied ? number : -1;
        need += all;
    }
    const int found = need == 0 ? 0 : find_free(P.references, P.num_pages, need, [&](int i, int page) {
        moves[2 * i + 1] = page;
        if constexpr (LOCAL) fresh_of[i] = page;
    });
    const bool fits = found >= need;
    if (threadIdx.x == 0) {
        W.head[0] = fits;
        missing[0] = fits ? 0 : need - found;
    }
    there();
    for (int64_t i = threadIdx.x; i < count; i += kPlanThreads)
        if (!fits || i >= need) moves[2 * i] = moves[2 * i + 1] = -1;
    for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) {
        const int number = number_of[s], fresh = fits && number >= 0 ? LOCAL ? fresh_of[number] : moves[2 * number + 1] : -1;
        if constexpr (TABLES) {
            low[s] = fresh;
            if (fits && of_all[s] != s) P.context_lens[s] = tokens[of_all[s]];
        } else {
            if constexpr (LOCAL) W.a[s] = of_all[s], W.d[s] = tokens[s];
            W.c[s] = fresh;
        }
    }
    if constexpr (TABLES) {
        if (!fits) return;
        __syncthreads();
        const uint32_t entries = P.seqs * P.max_pages, room = P.max_pages;
        int entry[kForkEach], was[kForkEach];
        int32_t* at[kForkEach];
#pragma unroll
        for (int n = 0; n < kForkEach; ++n) {
            const uint32_t i = threadIdx.x + n * kPlanThreads, row = i / room, j = i - row * room;
            entry[n] = was[n] = -1;
            at[n] = nullptr;
            if (i >= entries) continue;
            const int s = row, of = of_all[s];
            if (of == s) continue;
            const int held = pages_of(P, tokens[of]);
            at[n] = P.table + s * P.table_stride + j;
            if ((int)j < pages_of(P, tokens[s])) was[n] = *at[n];
            if ((int)j < held) entry[n] = (int)j == held - 1 && low[s] >= 0 ? low[s] : P.table[of * P.table_stride + j];
        }
        __syncthreads();                                             // (what rows become has been read)
#pragma unroll
        for (int n = 0; n < kForkEach; ++n) {
            if (!at[n]) continue;
            *at[n] = entry[n];
            if (entry[n] == was[n]) continue;
            if (is_page(P, entry[n])) atomicAdd(P.references + entry[n], 1);
            if (is_page(P, was[n])) atomicAdd(P.references + was[n], -1);
        }
    }
}

// Rows of up to 1024 sequences, a workgroup for 16 entries of all of them: what they become is read before any of it is written.  What a sequence becomes comes
// first, through LDS, then all that is read of the table at once (sequence after sequence 8.6 us for 192 of them).
constexpr int kForkEntries = 16, kForkRows = kPlanThreads / kForkEntries, kForkMost = kPlanThreads;
__global__ void __launch_bounds__(kPlanThreads) fork_tables_kernel(const PagePoolArgs P)
{
    __shared__ int4 becomes[kForkMost];                              // of, entries before, entries, fresh page
    const Scratch W = scratch_of(P);
    const bool fits = W.head[0] != 0;
    const int s_mine = threadIdx.x, j = blockIdx.x * kForkEntries + threadIdx.x % kForkEntries, s0 = threadIdx.x / kForkEntries;
    if (s_mine < P.seqs) {
        const int of = W.a[s_mine], fresh = W.c[s_mine], before = W.d[s_mine], tokens = W.d[of];
        becomes[s_mine] = {of, pages_of(P, before), pages_of(P, tokens), fresh};
        if (fits && blockIdx.x == 0 && of != s_mine) P.context_lens[s_mine] = tokens;
    }
    if (!fits) return;
    __syncthreads();
    int entry[kForkMost / kForkRows], old[kForkMost / kForkRows];
    uint32_t changes = 0;
#pragma unroll
    for (int n = 0; n < kForkMost / kForkRows; ++n) {
        const int s = s0 + n * kForkRows;
        entry[n] = old[n] = -1;
        if (s >= P.seqs || j >= P.max_pages) continue;
        const int4 b = becomes[s];
        if (b.x == s) continue;
        changes |= 1u << n;
        if (j < b.z) entry[n] = P.table[b.x * P.table_stride + j];
        if (j < b.y) old[n] = P.table[s * P.table_stride + j];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kForkMost / kForkRows; ++n) {
        const int s = s0 + n * kForkRows;
        if (!((changes >> n) & 1)) continue;
        const int4 b = becomes[s];
        const int e = b.w >= 0 && j == b.z - 1 ? b.w : entry[n];
        P.table[s * P.table_stride + j] = e;
        if (e == old[n]) continue;
        if (is_page(P, e)) atomicAdd(P.references + e, 1);
        if (is_page(P, old[n])) atomicAdd(P.references + old[n], -1);
    }
}
// grid (chunks of entries, sequences): the rows of those that change, and the counts; the table stays as it is until all rows are read
__global__ void __launch_bounds__(kRowThreads) fork_rows_kernel(const PagePoolArgs P)
{
    const Scratch W = scratch_of(P);
    const int s = blockIdx.y, of = W.a[s];
    if (of == s || W.head[0] == 0) return;
    const int before = pages_of(P, W.d[s]), held = pages_of(P, W.d[of]), fresh = W.c[s];
    const int last = min(P.max_pages, ((int)blockIdx.x + 1) * kRowEntries);
    for (int j = blockIdx.x * kRowEntries + threadIdx.x; j < last; j += kRowThreads) {
        int e = j < held ? P.table[of * P.table_stride + j] : -1;
        if (fresh >= 0 && j == held - 1) e = fresh;
        W.rows[(int64_t)s * P.max_pages + j] = e;
        if (is_page(P, e) && j < held) atomicAdd(P.references + e, 1);
        if (j < before) {
            const int old = P.table[s * P.table_stride + j];
            if (is_page(P, old)) atomicAdd(P.references + old, -1);
        }
    }
}
__global__ void __launch_bounds__(kRowThreads) fork_store_kernel(const PagePoolArgs P)
{
    const Scratch W = scratch_of(P);
    const int s = blockIdx.y, of = W.a[s];
    if (of == s || W.head[0] == 0) return;
    const int last = min(P.max_pages, ((int)blockIdx.x + 1) * kRowEntries);
    for (int j = blockIdx.x * kRowEntries + threadIdx.x; j < last; j += kRowThreads) P.table[s * P.table_stride + j] = W.rows[(int64_t)s * P.max_pages + j];
    if (blockIdx.x == 0 && threadIdx.x == 0) P.context_lens[s] = W.d[of];
}

// ---- compaction ----------------------------------------------------------------------------------

// One workgroup.  With U pages in use and n of them before page p, a free page p < U is hole number p - n, and a page p >= U in use goes into hole number U - 1 - n (the last
// one into the first hole), so that each finds its place in the list by itself.  pages[p]: where page p is afterwards (from U on)
// TABLES: with the tables, where one workgroup is enough for these too (48 sequences, 5000 pages: 8 us, in two launches 6 and 3)
template <bool TABLES>
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PagePoolArgs P, int32_t* moves, int max_moves)
{
    const Scratch W = scratch_of(P);
    const Step first = step_at(P.references, 0, P.num_pages);
    int used = 0, all;
    waves_before(lane_sum(__popc(used_of(first))), &used);
    for (int p = pages_in(first.loads); p < P.num_pages;) {
        const Step t = step_at(P.references, p, P.num_pages);
        waves_before(lane_sum(__popc(used_of(t))), &all);
        used += all;
        p += pages_in(t.loads);
    }
    int n = 0, above = 0;                                            // above: of this lane's pages, those in use from U on
    for (int p = 0; p < P.num_pages;) {
        const Step t = p == 0 ? first : step_at(P.references, p, P.num_pages);
        const uint32_t bits = used_of(t);
        const int before = waves_before(lane_sum(__popc(bits)), &all);
        pages_of_step(t, bits, n + before, P.num_pages, [&](int page, bool is_used, int k) {
            if (page < used && !is_used && page - k < max_moves) moves[2 * (page - k) + 1] = page;
            if (page >= used && is_used && used - 1 - k < max_moves) moves[2 * (used - 1 - k)] = page;
            if (page >= used) W.pages[page] = page;
            above += page >= used && is_used;
        });
        n += all;
        p += pages_in(t.loads);
    }
    int count;
    waves_before(lane_sum(above), &count);                           // (and what has been written is there)
    settled();
    for (int64_t i = threadIdx.x; i < max_moves; i += kPlanThreads) {        // (of a list of 2^31 - 1 moves 32 bits would pass the end)
        if (i >= count) {
            moves[2 * i] = moves[2 * i + 1] = -1;
            continue;
        }
        const int from = moves[2 * i], to = moves[2 * i + 1];
        W.pages[from] = to;
        P.references[to] = P.references[from];
        P.references[from] = 0;
    }
    if constexpr (!TABLES) {
        if (threadIdx.x == 0) W.head[1] = used;
        return;
    }
    settled();
    constexpr int kAtOnce = 4;
    const uint32_t entries = P.seqs * P.max_pages, room = P.max_pages;
    for (uint32_t i0 = threadIdx.x; i0 < entries; i0 += kAtOnce * kPlanThreads) {
        int32_t* entry[kAtOnce];
        int e[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            const uint32_t i = i0 + k * kPlanThreads, s = i / room, j = i - s * room;
            e[k] = -1;
            if (i >= entries || (int)j >= pages_of(P, P.context_lens[s])) continue;
            entry[k] = P.table + s * P.table_stride + j;
            e[k] = *entry[k];
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k)
            if (is_page(P, e[k]) && e[k] >= used) *entry[k] = seen<false>(W.pages + e[k]);
    }
}

// grid (chunks of entries, sequences)
__global__ void __launch_bounds__(kRowThreads) compact_tables_kernel(const PagePoolArgs P)
{
    const Scratch W = scratch_of(P);
    const int s = blockIdx.y, used = W.head[1], held = pages_of(P, P.context_lens[s]);
    const int last = min(held, ((int)blockIdx.x + 1) * kRowEntries);
    for (int j = blockIdx.x * kRowEntries + threadIdx.x; j < last; j += kRowThreads) {
        int32_t* entry = P.table + s * P.table_stride + j;
        const int e = *entry;
        if (is_page(P, e) && e >= used) *entry = W.pages[e];
    }
}

// ---- copies --------------------------------------------------------------------------------------

struct F32 {
    typedef float type;
};
struct F16 {
    typedef __half type;
};
struct BF16 {
    typedef __hip_bfloat16 type;
};
struct MX4 {};

template <typename T>
__device__ __forceinline__ void load8(const char* at, float (&x)[8])
{
    alignas(16) typename T::type v[8];
#pragma unroll
    for (unsigned i = 0; i < sizeof(v) / 16; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(at)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(v[0]) == 4) x[i] = v[i];
        else if constexpr (std::is_same<typename T::type, __half>::value) x[i] = __half2float(v[i]);
        else x[i] = __bfloat162float(v[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(char* at, const float (&x)[8])
{
    alignas(16) typename T::type v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(v[0]) == 4) v[i] = x[i];
        else if constexpr (std::is_same<typename T::type, __half>::value) v[i] = __float2half(x[i]);
        else v[i] = __float2bfloat16(x[i]);
    }
#pragma unroll
    for (unsigned i = 0; i < sizeof(v) / 16; ++i) reinterpret_cast<uint4*>(at)[i] = reinterpret_cast<const uint4*>(v)[i];
}

constexpr int kCopyThreads = 256, kCopyUnits = 4;

// A lane takes eight values of a row, 16 bytes of a 16-bit cache, so that lanes side by side take what lies side by side; four lanes have a block of a cache in four bits.
// Four of them at once, so that their loads are under way together.  Workgroups go through the items (pair, chunk of a page, keys or values) in turn: lists have room for more
// pairs than there mostly are, and a workgroup for each of those that are not there took 7 of 25 us (350 of 1543 pairs).  Bound: memory (400 pages of 64 x 8 x 128 from bf16 into
// four bits or back, 133 MB: 21 us, 6.2 TB/s).
template <typename S, typename D>
__device__ __forceinline__ void copy_chunk(const PageCopyArgs& A, int from, int to, uint32_t chunk, bool values)
{
    const PageRows &s = A.src[values], &d = A.dst[values];
    constexpr bool from4 = std::is_same<S, MX4>::value, to4 = std::is_same<D, MX4>::value;
    const char* src = s.at + from * s.page;
    char* dst = d.at + to * d.page;
#pragma unroll
    for (int n = 0; n < kCopyUnits; ++n) {
        const uint32_t unit = (chunk * kCopyUnits + n) * kCopyThreads + threadIdx.x;
        if (unit >= A.units) break;
        const uint32_t row = A.by_row.quot(unit), u = unit - row * A.by_row.d;
        const uint32_t outer = A.by_inner.quot(row), inner = row - outer * A.by_inner.d;
        const int64_t s_row = outer * s.outer + inner * s.inner, d_row = outer * d.outer + inner * d.inner;
        if constexpr (from4 && to4) {
            *reinterpret_cast<uint32_t*>(dst + d_row + 4 * u) = *reinterpret_cast<const uint32_t*>(src + s_row + 4 * u);
            if (u % 4 == 0)
                d.scales[to * d.scale_page + outer * d.scale_outer + inner * d.scale_inner + u / 4] =
                    s.scales[from * s.scale_page + outer * s.scale_outer + inner * s.scale_inner + u / 4];
        } else if constexpr (std::is_same<S, D>::value) {
            constexpr int kBytes = 8 * sizeof(typename S::type);
            uint4 v[kBytes / 16];
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) v[i] = *reinterpret_cast<const uint4*>(src + s_row + kBytes * u + 16 * i);
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) *reinterpret_cast<uint4*>(dst + d_row + kBytes * u + 16 * i) = v[i];
        } else {
            float x[8];
            if constexpr (from4)
                mx4_values(*reinterpret_cast<const uint32_t*>(src + s_row + 4 * u), s.scales[from * s.scale_page + outer * s.scale_outer + inner * s.scale_inner + u / 4], x);
            else
                load8<S>(src + s_row + 8 * sizeof(typename S::type) * u, x);
            if constexpr (to4) {
                const uint32_t e = mx4_scale(mx4_top(x));
                *reinterpret_cast<uint32_t*>(dst + d_row + 4 * u) = mx4_codes(x, e);
                if (u % 4 == 0) d.scales[to * d.scale_page + outer * d.scale_outer + inner * d.scale_inner + u / 4] = (uint8_t)e;
            } else {
                store8<D>(dst + d_row + 8 * sizeof(typename D::type) * u, x);
            }
        }
    }
}

template <typename S, typename D>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const int32_t* moves, const PageCopyArgs A)
{
    for (uint32_t item = blockIdx.x; item < A.items; item += gridDim.x) {
        const uint32_t pair = A.by_chunks.quot(item), rest = item - pair * A.by_chunks.d;
        const int from = moves[2 * (int64_t)pair], to = moves[2 * (int64_t)pair + 1];
        if ((uint32_t)from >= (uint32_t)A.src_pages || (uint32_t)to >= (uint32_t)A.dst_pages || (A.same && from == to)) continue;
        copy_chunk<S, D>(A, from, to, rest >> 1, rest & 1);
    }
}

dim3 row_grid(const PagePoolArgs& P) { return dim3((P.max_pages + kRowEntries - 1) / kRowEntries, P.seqs); }

}  // namespace

// (4 more than the parts: bits and counts of a pool of a few pages)
int64_t page_pool_scratch(int64_t seqs, int64_t max_pages, int64_t num_pages) { return 16 + 4 * seqs + num_pages + seqs * max_pages + 4; }

bool launch_resize_sequences(const PagePoolArgs& P, const int32_t* lengths, int32_t* moves, int32_t* missing, hipStream_t stream)
{
    if (one_workgroup(P)) {
        hipLaunchKernelGGL(page_few_kernel, dim3(1), dim3(kPlanThreads), 0, stream, P, lengths, moves, missing);
        return hip_ok(hipGetLastError(), "resize_sequences launch");
    }
    hipLaunchKernelGGL(page_drop_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P, lengths);
    if (!hip_ok(hipGetLastError(), "resize_sequences launch")) return false;
    const int part = kPart * (int)((P.num_pages + (int64_t)kPart * kMostParts - 1) / ((int64_t)kPart * kMostParts));
    const dim3 grid((unsigned)((P.num_pages + (int64_t)part * kPlanWaves - 1) / ((int64_t)part * kPlanWaves) + 1));
    hipLaunchKernelGGL(page_plan_kernel, grid, dim3(kPlanThreads), 0, stream, P, lengths, part);
    if (!hip_ok(hipGetLastError(), "resize_sequences launch")) return false;
    const auto fill = P.seqs <= kLocal ? page_fill_kernel<true> : page_fill_kernel<false>;
    hipLaunchKernelGGL(fill, grid, dim3(kPlanThreads), 0, stream, P, lengths, moves, missing, part);
    return hip_ok(hipGetLastError(), "resize_sequences launch");
}

bool launch_fork_sequences(const PagePoolArgs& P, const int32_t* children, const int32_t* parents, int count, int32_t* moves, int32_t* missing,
                           hipStream_t stream)
{
    constexpr size_t lds = 6 * kLocal * sizeof(int);
    const bool local = P.seqs <= kLocal, tables = local && (int64_t)P.seqs * P.max_pages <= kForkEach * kPlanThreads;
    const auto plan = tables ? fork_plan_kernel<true, true> : local ? fork_plan_kernel<true, false> : fork_plan_kernel<false, false>;
    if (local && !raise_lds_limit(reinterpret_cast<const void*>(plan), lds)) return false;
    hipLaunchKernelGGL(plan, dim3(1), dim3(kPlanThreads), local ? lds : 0, stream, P, children, parents, count, moves, missing);
    if (tables) return hip_ok(hipGetLastError(), "fork_sequences launch");
    if (!hip_ok(hipGetLastError(), "fork_sequences launch")) return false;
    // (a launch has fewer than 2^32 threads: of rows of more entries each takes two kernels, as those of many sequences)
    const int64_t columns = ((int64_t)P.max_pages + kForkEntries - 1) / kForkEntries;
    if (P.seqs <= kForkMost && columns * kPlanThreads <= UINT32_MAX) {
        hipLaunchKernelGGL(fork_tables_kernel, dim3((unsigned)columns), dim3(kPlanThreads), 0, stream, P);
        return hip_ok(hipGetLastError(), "fork_sequences launch");
    }
    hipLaunchKernelGGL(fork_rows_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P);
    if (!hip_ok(hipGetLastError(), "fork_sequences launch")) return false;
    hipLaunchKernelGGL(fork_store_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P);
    return hip_ok(hipGetLastError(), "fork_sequences launch");
}

bool launch_compact_pages(const PagePoolArgs& P, int32_t* moves, int max_moves, hipStream_t stream)
{
    const bool one = one_workgroup(P);
    hipLaunchKernelGGL(one ? compact_plan_kernel<true> : compact_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0, stream, P, moves, max_moves);
    if (one) return hip_ok(hipGetLastError(), "compact_pages launch");
    if (!hip_ok(hipGetLastError(), "compact_pages launch")) return false;
    hipLaunchKernelGGL(compact_tables_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P);
    return hip_ok(hipGetLastError(), "compact_pages launch");
}

template <typename S>
static auto copy_kernel_to(int type)
{
    switch (type) {
    case kTypeF32: return copy_pages_kernel<S, F32>;
    case kTypeF16: return copy_pages_kernel<S, F16>;
    case kTypeBF16: return copy_pages_kernel<S, BF16>;
    default: return copy_pages_kernel<S, MX4>;
    }
}

bool launch_copy_pages(const int32_t* moves, int count, PageCopyArgs args, int src_type, int dst_type, hipStream_t stream)
{
    const int64_t chunks = 2 * (((int64_t)args.units + kCopyThreads * kCopyUnits - 1) / (kCopyThreads * kCopyUnits)), items = chunks * count;
    if (items > INT32_MAX) {
        set_last_error("copy_pages: too many pages for one call.");
        return false;
    }
    args.items = (uint32_t)items;
    args.by_chunks = FastDiv((uint32_t)chunks);
    const dim3 grid((unsigned)std::min<int64_t>(items, 16 * device_info().num_cus));
    const auto kern = src_type == kTypeF32 ? copy_kernel_to<F32>(dst_type)
        : src_type == kTypeF16             ? copy_kernel_to<F16>(dst_type)
        : src_type == kTypeBF16            ? copy_kernel_to<BF16>(dst_type)
                                           : copy_kernel_to<MX4>(dst_type);
    hipLaunchKernelGGL(kern, grid, dim3(kCopyThreads), 0, stream, moves, args);
    return hip_ok(hipGetLastError(), "copy_pages launch");
}

}  // namespace tship
