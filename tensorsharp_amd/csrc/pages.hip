// The life of a cache's pages: who has which (tables, reference counts, lengths, all on the device), and copies of pages between caches.
//
//   page_drop_kernel, page_plan_kernel, page_fill_kernel     sequences get other lengths
//   fork_plan_kernel, fork_rows_kernel, fork_store_kernel    sequences go on from what others have
//   compact_plan_kernel, compact_tables_kernel               used pages move to the front
//   copy_pages_kernel                                        pages of one cache or two, of one type or two
//
// The lists are short next to the caches (a reference count for each page, an entry for each page of a sequence), so what counts is the number of dependent steps.  What
// has to know all sequences or all pages in order - sums up to a sequence, the lowest free pages - is one workgroup that takes 16384 pages in a step; what
// walks over the tables has a workgroup for 1024 entries.  Two or three launches a call, nothing that one workgroup waits for another for.  Counts change by
// atomic additions of whole numbers, whose order changes nothing.
#include "tship_internal.h"
#include "mx4.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>
#include <type_traits>

namespace tship {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kRowThreads = 256, kRowEntries = 4 * kRowThreads;     // of a table that a workgroup walks over

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

// 16 pages of a thread: which of them are as wanted, as bits
constexpr int kScan = 16 * kPlanThreads;
template <bool FREE>
__device__ __forceinline__ uint32_t pages_here(const int32_t* references, int64_t p0, int64_t end)
{
    uint32_t bits = 0;
    if (p0 + 16 <= end) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int4 r = *reinterpret_cast<const int4*>(references + p0 + 4 * i);
            bits |= ((r.x <= 0) == FREE ? 1u : 0u) << (4 * i) | ((r.y <= 0) == FREE ? 2u : 0u) << (4 * i) | ((r.z <= 0) == FREE ? 4u : 0u) << (4 * i) |
                ((r.w <= 0) == FREE ? 8u : 0u) << (4 * i);
        }
    } else {
        for (int i = 0; i < 16 && p0 + i < end; ++i) bits |= ((references[p0 + i] <= 0) == FREE ? 1u : 0u) << i;
    }
    return bits;
}
// Calls each(number, page) for every page of [begin, end) (begin a multiple of 16) that is free (used), numbered from below, until `want` are found; returns how
// many there are up to where it stopped.
template <bool FREE, typename F>
__device__ __forceinline__ int64_t find_pages(const int32_t* references, int64_t begin, int64_t end, int64_t want, F&& each)
{
    int64_t found = 0;
    for (int64_t p = begin; p < end && found < want; p += kScan) {
        const int64_t mine = p + 16 * (int64_t)threadIdx.x;
        uint32_t bits = pages_here<FREE>(references, mine, end);
        int64_t all;
        int64_t number = found + before_me(__popc(bits), &all);
        for (; bits != 0; bits &= bits - 1) each(number++, mine + __ffs(bits) - 1);
        found += all;
    }
    return found;
}

// ---- other lengths -------------------------------------------------------------------------------

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

// one workgroup: how many pages each longer sequence needs, where its pages begin in the list of the lowest free ones, and that list
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const PagePoolArgs P, const int32_t* lengths, int32_t* moves, int32_t* missing)
{
    const Scratch W = scratch_of(P);
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
    const int64_t found = need == 0 ? 0 : find_pages<true>(P.references, 0, P.num_pages, need, [&](int64_t i, int64_t page) {
        if (i < need) W.pages[i] = (int)page;
    });
    const bool fits = found >= need;
    for (int i = threadIdx.x; i < P.seqs; i += kPlanThreads)
        if (!fits || i >= copies) moves[2 * i] = moves[2 * i + 1] = -1;
    if (threadIdx.x == 0) {
        W.head[0] = fits;
        missing[0] = fits ? 0 : (int)min(need - found, (int64_t)INT32_MAX);
    }
    for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) {
        const int64_t tokens = P.context_lens[s], goal = goal_of(P, lengths, s);
        W.d[s] = fits && goal > tokens ? pages_of(P, goal) : 0;
        if (goal < tokens || (fits && goal > tokens)) P.context_lens[s] = (int)goal;
    }
}

// grid (chunks of entries, sequences): the pages of longer sequences
__global__ void __launch_bounds__(kRowThreads) page_fill_kernel(const PagePoolArgs P, int32_t* moves)
{
    const Scratch W = scratch_of(P);
    const int s = blockIdx.y, goal = W.d[s];
    if (goal == 0) return;
    const int held = W.a[s], at = W.b[s], number = W.c[s], own = number >= 0 ? 1 : 0;
    int32_t* row = P.table + s * P.table_stride;
    const int first = max(held, (int)blockIdx.x * kRowEntries), last = min(goal, ((int)blockIdx.x + 1) * kRowEntries);
    for (int j = first + threadIdx.x; j < last; j += kRowThreads) {
        const int page = W.pages[at + own + j - held];
        row[j] = page;
        P.references[page] = 1;
    }
    if (own && blockIdx.x == 0 && threadIdx.x == 0) {
        const int page = W.pages[at], begun = row[held - 1];
        row[held - 1] = page;
        P.references[page] = 1;
        atomicAdd(P.references + begun, -1);
        moves[2 * number] = begun;
        moves[2 * number + 1] = page;
    }
}

// ---- forks ---------------------------------------------------------------------------------------

// Maxima and minima are formed in the second-level cache: what they leave is read there too, once every wavefront's have arrived.
__device__ __forceinline__ int seen(const int* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void settled()
{
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
}

// One workgroup.  a: the sequence that each becomes; b: the lowest that becomes it; c: the fresh page in place of the begun one, -1: none; d: tokens before
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(const PagePoolArgs P, const int32_t* children, const int32_t* parents, int count,
                                                                 int32_t* moves, int32_t* missing)
{
    const Scratch W = scratch_of(P);
    for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) {
        __hip_atomic_store(W.a + s, -1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(W.b + s, P.seqs, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        W.d[s] = P.context_lens[s];
    }
    settled();
    for (int i = threadIdx.x; i < count; i += kPlanThreads)
        if ((uint32_t)children[i] < (uint32_t)P.seqs && (uint32_t)parents[i] < (uint32_t)P.seqs) atomicMax(W.a + children[i], i);
    settled();
    for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) {
        const int pair = seen(W.a + s), of = pair >= 0 ? parents[pair] : s;
        __hip_atomic_store(W.a + s, of, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        atomicMin(W.b + of, s);
    }
    settled();
    // (a parent that stays what it is keeps its begun page)
    auto begun_page = [&](int of) -> int {
        const int tokens = W.d[of], held = pages_of(P, tokens);
        if (held == 0 || tokens % P.page_size == 0 || tokens > (int64_t)P.max_pages * P.page_size) return -1;
        const int e = P.table[of * P.table_stride + held - 1];
        return is_page(P, e) ? e : -1;
    };
    int64_t need = 0;
    for (int s0 = 0; s0 < P.seqs; s0 += kPlanThreads) {
        const int s = s0 + threadIdx.x;
        int copied = 0;
        if (s < P.seqs) {
            const int of = seen(W.a + s), keeper = seen(W.a + of) == of ? of : seen(W.b + of);
            copied = keeper != s && begun_page(of) >= 0;
        }
        int64_t all;
        const int64_t number = need + before_me(copied, &all);
        if (s < P.seqs) W.c[s] = copied ? (int)number : -1;
        need += all;
    }
    const int64_t found = need == 0 ? 0 : find_pages<true>(P.references, 0, P.num_pages, need, [&](int64_t i, int64_t page) {
        if (i < need) W.pages[i] = (int)page;
    });
    const bool fits = found >= need;
    if (threadIdx.x == 0) {
        W.head[0] = fits;
        missing[0] = fits ? 0 : (int)(need - found);
    }
    for (int i = threadIdx.x; i < count; i += kPlanThreads)
        if (!fits || i >= need) moves[2 * i] = moves[2 * i + 1] = -1;
    __syncthreads();                                                 // (the list)
    if (!fits) return;
    for (int s = threadIdx.x; s < P.seqs; s += kPlanThreads) {
        const int number = W.c[s];
        if (number < 0) continue;
        const int page = W.pages[number];
        W.c[s] = page;
        moves[2 * number] = begun_page(seen(W.a + s));
        moves[2 * number + 1] = page;
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

// One workgroup: the holes below the number of used pages, then the used pages from there on, of which the last goes into the first hole.  pages[p]: where page p
// is afterwards (from that number on)
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PagePoolArgs P, int32_t* moves, int max_moves)
{
    const Scratch W = scratch_of(P);
    for (int i = threadIdx.x; i < max_moves; i += kPlanThreads) moves[2 * i] = moves[2 * i + 1] = -1;
    int64_t mine = 0, used;
    for (int64_t p = 16 * (int64_t)threadIdx.x; p < P.num_pages; p += kScan) mine += __popc(pages_here<false>(P.references, p, P.num_pages));
    before_me(mine, &used);                                          // (and the list is cleared)
    if (threadIdx.x == 0) W.head[1] = (int)used;
    const int64_t holes = find_pages<true>(P.references, 0, used, INT64_MAX, [&](int64_t i, int64_t page) {
        if (i < max_moves) moves[2 * i + 1] = (int)page;
    });
    __syncthreads();
    // (the scan begins at a multiple of 16: pages below the number that are used are passed over)
    const int64_t begin = used & ~(int64_t)15;
    int64_t skipped;
    before_me(threadIdx.x < 16 && begin + threadIdx.x < used ? P.references[begin + threadIdx.x] > 0 : 0, &skipped);
    for (int64_t p = begin; p < P.num_pages; p += kScan) {           // (all pages keep their place but for those that follow)
        const int64_t at = p + 16 * (int64_t)threadIdx.x;
        for (int i = 0; i < 16; ++i)
            if (at + i < P.num_pages) W.pages[at + i] = (int)(at + i);
    }
    __syncthreads();
    find_pages<false>(P.references, begin, P.num_pages, INT64_MAX, [&](int64_t i, int64_t page) {
        const int64_t k = holes - 1 - (i - skipped);
        if (page < used || k < 0 || k >= max_moves) return;
        const int to = moves[2 * k + 1];
        moves[2 * k] = (int)page;
        W.pages[page] = to;
        P.references[to] = P.references[page];
        P.references[page] = 0;
    });
    // (pages that stay, as there is no room in the list: their holes are taken out of it already, by number)
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

// grid (pairs, chunks of a page, keys and values): a lane takes eight values of a row, 16 bytes of a 16-bit cache, so that lanes side by side take what lies side by
// side; four lanes have a block of a cache in four bits.  Four of them at once, so that their loads are under way together.  Bound: memory.
template <typename S, typename D>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const int32_t* moves, const PageCopyArgs A)
{
    const int from = moves[2 * (int64_t)blockIdx.x], to = moves[2 * (int64_t)blockIdx.x + 1];
    if ((uint32_t)from >= (uint32_t)A.src_pages || (uint32_t)to >= (uint32_t)A.dst_pages || (A.same && from == to)) return;
    const PageRows &s = A.src[blockIdx.z], &d = A.dst[blockIdx.z];
    constexpr bool from4 = std::is_same<S, MX4>::value, to4 = std::is_same<D, MX4>::value;
    const char* src = s.at + from * s.page;
    char* dst = d.at + to * d.page;
#pragma unroll
    for (int n = 0; n < kCopyUnits; ++n) {
        const uint32_t unit = (blockIdx.y * kCopyUnits + n) * kCopyThreads + threadIdx.x;
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

dim3 row_grid(const PagePoolArgs& P) { return dim3((P.max_pages + kRowEntries - 1) / kRowEntries, P.seqs); }

}  // namespace

int64_t page_pool_scratch(int64_t seqs, int64_t max_pages, int64_t num_pages) { return 16 + 4 * seqs + num_pages + seqs * max_pages; }

bool launch_resize_sequences(const PagePoolArgs& P, const int32_t* lengths, int32_t* moves, int32_t* missing, hipStream_t stream)
{
    hipLaunchKernelGGL(page_drop_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P, lengths);
    if (!hip_ok(hipGetLastError(), "resize_sequences launch")) return false;
    hipLaunchKernelGGL(page_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, P, lengths, moves, missing);
    if (!hip_ok(hipGetLastError(), "resize_sequences launch")) return false;
    hipLaunchKernelGGL(page_fill_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P, moves);
    return hip_ok(hipGetLastError(), "resize_sequences launch");
}

bool launch_fork_sequences(const PagePoolArgs& P, const int32_t* children, const int32_t* parents, int count, int32_t* moves, int32_t* missing,
                           hipStream_t stream)
{
    hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, P, children, parents, count, moves, missing);
    if (!hip_ok(hipGetLastError(), "fork_sequences launch")) return false;
    hipLaunchKernelGGL(fork_rows_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P);
    if (!hip_ok(hipGetLastError(), "fork_sequences launch")) return false;
    hipLaunchKernelGGL(fork_store_kernel, row_grid(P), dim3(kRowThreads), 0, stream, P);
    return hip_ok(hipGetLastError(), "fork_sequences launch");
}

bool launch_compact_pages(const PagePoolArgs& P, int32_t* moves, int max_moves, hipStream_t stream)
{
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, P, moves, max_moves);
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

bool launch_copy_pages(const int32_t* moves, int count, const PageCopyArgs& args, int src_type, int dst_type, hipStream_t stream)
{
    const dim3 grid(count, (args.units + kCopyThreads * kCopyUnits - 1) / (kCopyThreads * kCopyUnits), 2);
    if (grid.y > 65535) {
        set_last_error("copy_pages: pages are too large.");
        return false;
    }
    const auto kern = src_type == kTypeF32 ? copy_kernel_to<F32>(dst_type)
        : src_type == kTypeF16             ? copy_kernel_to<F16>(dst_type)
        : src_type == kTypeBF16            ? copy_kernel_to<BF16>(dst_type)
                                           : copy_kernel_to<MX4>(dst_type);
    hipLaunchKernelGGL(kern, grid, dim3(kCopyThreads), 0, stream, moves, args);
    return hip_ok(hipGetLastError(), "copy_pages launch");
}

}  // namespace tship
