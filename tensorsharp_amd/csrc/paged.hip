// What a step over many sequences needs between the fused QKV projection and the output projection: rotary positions, the store of new
// keys and values into the pages of a cache, and attention over the pages.
//
//   rope_kernel              head-wise rotation of a [tokens x heads x head_dim] tensor
//   rope_store_kernel        norm and rotation of q and k heads of QKV rows, k and v into the cache
//   paged_attention_kernel   softmax(scale q K^T) V of a sequence's new tokens over its pages
#include "tship_internal.h"

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <algorithm>

namespace tship {
namespace {

constexpr int kMaxDim = 256;

typedef float f2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// ---- rotary positions ----------------------------------------------------------------------------

// cosine and sine of pair i at a position.  The angle is formed in 64 bits and brought to revolutions in -1/2 .. 1/2 there: at position
// 10^6 an angle of 32 bits is 0.03 radians off.  What is left loses nothing in 32 bits.
__device__ __forceinline__ f2_t turn_of(const RopeSpec& R, int pair, int position)
{
    double f = exp2(R.step * pair);
    if (R.factors) f /= (double)R.factors[pair];
    const double kept = R.ext == 0.0 ? 0.0 : R.ext * (1.0 - fmin(1.0, fmax(0.0, (pair - R.low) / R.range)));
    f *= R.freq_scale * (1.0 - kept) + kept;
    double turns = (double)position * (f * 0.15915494309189533577);
    turns -= rint(turns);
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    return f2_t{c * R.size, s * R.size};
}

// Four dimensions of a head that one lane holds: lane u < dims / 4 the pairs 2u and 2u + 1, the lanes behind them four dimensions
// that are not turned.
struct Quad {
    f2_t a, b;           // pair 2u is (a.x, b.x); of what is not turned, dimensions 0, 1 and 2, 3
};
__device__ __forceinline__ Quad load_quad(const float* head, const RopeSpec& R, int u)
{
    if (R.mode == 2 && 4 * u < R.dims)
        return {*reinterpret_cast<const f2_t*>(head + 2 * u), *reinterpret_cast<const f2_t*>(head + R.dims / 2 + 2 * u)};
    const f4_t v = *reinterpret_cast<const f4_t*>(head + 4 * u);
    if (4 * u < R.dims) return {f2_t{v.x, v.z}, f2_t{v.y, v.w}};
    return {f2_t{v.x, v.y}, f2_t{v.z, v.w}};
}
__device__ __forceinline__ Quad turned(const Quad& q, const RopeSpec& R, int u, const f2_t* turns)
{
    if (4 * u >= R.dims) return q;
    const f2_t t0 = turns[2 * u], t1 = turns[2 * u + 1];
    return {f2_t{q.a.x * t0.x - q.b.x * t0.y, q.a.y * t1.x - q.b.y * t1.y}, f2_t{q.a.x * t0.y + q.b.x * t0.x, q.a.y * t1.y + q.b.y * t1.x}};
}
// T: float, __half or __hip_bfloat16
template <typename T>
__device__ __forceinline__ T rounded(float v)
{
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __float2half(v);
    else return __float2bfloat16(v);
}
template <typename T>
__device__ __forceinline__ void put2(T* at, float x, float y)
{
    struct alignas(2 * sizeof(T)) Two { T x, y; };
    *reinterpret_cast<Two*>(at) = Two{rounded<T>(x), rounded<T>(y)};
}
template <typename T>
__device__ __forceinline__ void put4(T* at, float x, float y, float z, float w)
{
    struct alignas(4 * sizeof(T)) Four { T x, y, z, w; };
    *reinterpret_cast<Four*>(at) = Four{rounded<T>(x), rounded<T>(y), rounded<T>(z), rounded<T>(w)};
}
template <typename T>
__device__ __forceinline__ void store_quad(T* head, const Quad& q, const RopeSpec& R, int u)
{
    if (4 * u >= R.dims) {
        put4(head + 4 * u, q.a.x, q.a.y, q.b.x, q.b.y);
    } else if (R.mode == 2) {
        put2(head + 2 * u, q.a.x, q.a.y);
        put2(head + R.dims / 2 + 2 * u, q.b.x, q.b.y);
    } else {
        put4(head + 4 * u, q.a.x, q.b.x, q.a.y, q.b.y);
    }
}

constexpr int kRopeThreads = 256;

// grid (tokens, head chunks): LANES lanes hold a head, a workgroup takes 256 / LANES heads at a time.  The angles of a token are worked
// out once per workgroup, one pair per thread.
// Bound: memory, and for few tokens the latency of the angles and one trip to memory.
template <int LANES>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const float* x, float* out, const int32_t* positions, int heads, int head_dim,
                                                            int64_t x_token, int64_t x_head, int64_t o_token, int64_t o_head, const RopeSpec R)
{
    __shared__ f2_t turns[kMaxDim / 2];
    constexpr int kHeads = kRopeThreads / LANES;
    const int64_t t = blockIdx.x;
    const int u = threadIdx.x % LANES;
    const bool live = 4 * u < head_dim;
    const int position = positions[t];
    if ((int)threadIdx.x < R.dims / 2) turns[threadIdx.x] = turn_of(R, threadIdx.x, position);
    __syncthreads();
    for (int h = blockIdx.y * kHeads + threadIdx.x / LANES; h < heads; h += gridDim.y * kHeads)
        if (live) store_quad(out + t * o_token + h * o_head, turned(load_quad(x + t * x_token + h * x_head, R, u), R, u, turns), R, u);
}

// Which sequence's new token a row is: the number of sequences that end at or before it (row_starts does not fall, and is cut to the
// rows there are).  Every wavefront looks for itself, 64 sequences at a time.
struct Place {
    int seq, first, count;       // seq -1: of none
};
__device__ __forceinline__ Place place_of_row(const PagedKv& C, int row)
{
    const int lane = threadIdx.x & 63;
    int seq = 0;
    for (int s0 = 0; s0 < C.seqs; s0 += 64) {
        const bool before = s0 + lane < C.seqs && C.row_starts[s0 + lane + 1] <= row;
        const uint64_t ends = __ballot(before);
        seq += __popcll(ends);
        if (~ends != 0 ) break;
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    if (seq >= C.seqs) return {-1, 0, 0};
    const int first = C.row_starts[seq], end = C.row_starts[seq + 1];
    if (row < first) return {-1, 0, 0};
    return {seq, first, end - first};
}
// page of a sequence's position, -1: none
__device__ __forceinline__ int page_of(const PagedKv& C, int seq, int position, int* within)
{
    const int p = (int)C.page.quot((uint32_t)position);
    *within = position - p * (int)C.page.d;
    if (p >= C.max_pages) return -1;
    const int id = C.table[seq * C.table_stride + p];
    return (uint32_t)id < (uint32_t)C.num_pages ? id : -1;
}

template <int LANES, typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_store_kernel(const float* qkv, int64_t ld_qkv, float* query, int64_t ld_query, int heads,
                                                                  const int32_t* positions, const float* q_norm, const float* k_norm,
                                                                  float eps, const PagedKv C, const RopeSpec R)
{
    __shared__ f2_t turns[kMaxDim / 2];
    constexpr int kHeads = kRopeThreads / LANES;
    const int t = blockIdx.x;
    const Place at = place_of_row(C, t);
    if (at.seq < 0) return;                                          // uniform
    const int u = threadIdx.x % LANES, dim = C.head_dim, all = heads + 2 * C.kv_heads;
    const bool live = 4 * u < dim;
    const int where = C.context_lens[at.seq] - at.count + (t - at.first);
    const int position = positions ? positions[t] : where;
    int within = 0;
    const int page = where >= 0 ? page_of(C, at.seq, where, &within) : -1;
    if ((int)threadIdx.x < R.dims / 2) turns[threadIdx.x] = turn_of(R, threadIdx.x, position);
    __syncthreads();
    // (the loop's length is that of the first lane's head, so that the lanes of a wavefront stay together for the sums of the norm)
    for (int h0 = blockIdx.y * kHeads; h0 < all; h0 += gridDim.y * kHeads) {
        const int h = h0 + threadIdx.x / LANES;
        const bool here = live && h < all;
        const float* src = qkv + t * ld_qkv + (int64_t)min(h, all - 1) * dim;
        const bool is_v = h >= heads + C.kv_heads;
        Quad q{};
        if (here) {
            if (is_v) {
                const f4_t v = *reinterpret_cast<const f4_t*>(src + 4 * u);
                q = {f2_t{v.x, v.y}, f2_t{v.z, v.w}};
            } else {
                q = load_quad(src, R, u);
            }
        }
        const float* norm = h < heads ? q_norm : k_norm;
        if (q_norm || k_norm) {                                      // uniform
            float ss = q.a.x * q.a.x + q.a.y * q.a.y + q.b.x * q.b.x + q.b.y * q.b.y;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
            if (here && !is_v && norm) {
                const float by = 1.0f / sqrtf(ss / (float)dim + eps);
                const Quad w = load_quad(norm, R, u);
                q = {q.a * by * w.a, q.b * by * w.b};
            }
        }
        if (!here) continue;
        if (h < heads) {
            store_quad(query + t * ld_query + (int64_t)h * dim, turned(q, R, u, turns), R, u);
        } else if (page >= 0) {
            if (is_v) {
                T* dst = reinterpret_cast<T*>(C.v) + page * C.v_page + within * C.v_token + (h - heads - C.kv_heads) * C.v_head;
                put4(dst + 4 * u, q.a.x, q.a.y, q.b.x, q.b.y);
            } else {
                T* dst = reinterpret_cast<T*>(C.k) + page * C.k_page + within * C.k_token + (h - heads) * C.k_head;
                store_quad(dst, turned(q, R, u, turns), R, u);
            }
        }
    }
}

int lanes_of(int head_dim) { return head_dim <= 32 ? 8 : head_dim <= 64 ? 16 : head_dim <= 128 ? 32 : 64; }

// ---- attention -----------------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ float widened(T v)
{
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else return __bfloat162float(v);
}

constexpr int kAttnThreads = 256;

// One workgroup per (row, head): a pass over the keys with a running maximum and sum, 256 keys at a time - a thread per key for the
// scores, a thread per dimension for the weighted values.
template <typename T>
__global__ void __launch_bounds__(kAttnThreads) paged_attention_kernel(const float* query, int64_t ld_query, float* out, int64_t ld_out, int group,
                                                                       float scale, int window, const float* sinks, const PagedKv C)
{
    __shared__ float sq[kMaxDim], sw[kAttnThreads], sred[4];
    __shared__ int64_t sv[kAttnThreads];
    const int t = blockIdx.x, h = blockIdx.y, g = h / group, dim = C.head_dim, tid = threadIdx.x;
    const Place at = place_of_row(C, t);
    if (at.seq < 0) return;
    const int p = C.context_lens[at.seq] - at.count + (t - at.first);
    if (tid < dim) sq[tid] = query[t * ld_query + (int64_t)h * dim + tid] * scale;
    __syncthreads();
    const int lo = window > 0 ? max(0, p - window + 1) : 0;
    const int hi = (int)min((int64_t)p + 1, (int64_t)C.max_pages * C.page.d);
    auto all = [&](float x, auto op) {
        for (int o = 32; o > 0; o >>= 1) x = op(x, __shfl_xor(x, o));
        __syncthreads();
        if ((tid & 63) == 0) sred[tid >> 6] = x;
        __syncthreads();
        return op(op(sred[0], sred[1]), op(sred[2], sred[3]));
    };
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int j0 = lo; j0 < hi; j0 += kAttnThreads) {
        const int j = j0 + tid;
        int within = 0;
        const int page = j < hi ? page_of(C, at.seq, j, &within) : -1;
        float s = -INFINITY;
        if (page >= 0) {
            const T* k = reinterpret_cast<const T*>(C.k) + page * C.k_page + within * C.k_token + g * C.k_head;
            s = 0.f;
            for (int d = 0; d < dim; ++d) s += sq[d] * widened(k[d]);
        }
        sv[tid] = page >= 0 ? page * C.v_page + within * C.v_token + g * C.v_head : -1;
        const float mn = fmaxf(m, all(s, [](float a, float b) { return fmaxf(a, b); }));
        if (mn == -INFINITY) continue;                               // uniform
        const float w = expf(s - mn), f = expf(m - mn);
        sw[tid] = w;
        l = l * f + all(w, [](float a, float b) { return a + b; });
        acc *= f;
        m = mn;
        if (tid < dim)
            for (int i = 0; i < min(kAttnThreads, hi - j0); ++i)
                if (sv[i] >= 0) acc += sw[i] * widened(reinterpret_cast<const T*>(C.v)[sv[i] + tid]);
        __syncthreads();
    }
    if (sinks && l > 0.f) {
        const float mn = fmaxf(m, sinks[h]), f = expf(m - mn);
        l = l * f + expf(sinks[h] - mn);
        acc *= f;
    }
    if (tid < dim) out[t * ld_out + (int64_t)h * dim + tid] = l > 0.f ? acc / l : 0.f;
}

}  // namespace

bool launch_rope(const float* x, int64_t x_token, int64_t x_head, float* out, int64_t o_token, int64_t o_head, int tokens, int heads,
                 int head_dim, const int32_t* positions, const RopeSpec& rope, hipStream_t stream)
{
    const int lanes = lanes_of(head_dim), at_once = kRopeThreads / lanes;
    const int chunks = std::max(1, std::min((heads + at_once - 1) / at_once, 2048 / tokens));
    const dim3 grid(tokens, chunks);
#define TSHIP_ROPE(L)                                                                                                              \
    hipLaunchKernelGGL((rope_kernel<L>), grid, dim3(kRopeThreads), 0, stream, x, out, positions, heads, head_dim, x_token, x_head, o_token, o_head, rope)
    switch (lanes) {
    case 8: TSHIP_ROPE(8); break;
    case 16: TSHIP_ROPE(16); break;
    case 32: TSHIP_ROPE(32); break;
    default: TSHIP_ROPE(64); break;
    }
#undef TSHIP_ROPE
    return hip_ok(hipGetLastError(), "rope launch");
}

bool launch_rope_store(const float* qkv, int64_t ld_qkv, float* query, int64_t ld_query, int rows, int heads, const PagedKv& cache,
                       const int32_t* positions, const float* q_norm, const float* k_norm, float eps, const RopeSpec& rope, hipStream_t stream)
{
    const int lanes = lanes_of(cache.head_dim), at_once = kRopeThreads / lanes, all = heads + 2 * cache.kv_heads;
    const int chunks = std::max(1, std::min((all + at_once - 1) / at_once, 2048 / rows));
    const dim3 grid(rows, chunks);
#define TSHIP_STORE(L, T)                                                                                                              \
    hipLaunchKernelGGL((rope_store_kernel<L, T>), grid, dim3(kRopeThreads), 0, stream, qkv, ld_qkv, query, ld_query, heads, positions, q_norm, \
                       k_norm, eps, cache, rope)
#define TSHIP_STORE_T(L)                                           \
    switch (cache.element_type) {                                  \
    case kTypeF32: TSHIP_STORE(L, float); break;                   \
    case kTypeF16: TSHIP_STORE(L, __half); break;                  \
    default: TSHIP_STORE(L, __hip_bfloat16); break;                \
    }
    switch (lanes) {
    case 8: TSHIP_STORE_T(8) break;
    case 16: TSHIP_STORE_T(16) break;
    case 32: TSHIP_STORE_T(32) break;
    default: TSHIP_STORE_T(64) break;
    }
#undef TSHIP_STORE_T
#undef TSHIP_STORE
    return hip_ok(hipGetLastError(), "rope store launch");
}

PagedAttnPlan plan_paged_attention(int, int, const PagedKv&, int) { return {1, 1, 1, 0}; }

bool launch_paged_attention(const PagedAttnPlan&, const float* query, int64_t ld_query, float* out, int64_t ld_out, int rows, int heads,
                            const PagedKv& cache, float scale, int window, const float* sinks, void*, hipStream_t stream)
{
    const dim3 grid(rows, heads);
#define TSHIP_ATTEND(T)                                                                                                                    \
    hipLaunchKernelGGL((paged_attention_kernel<T>), grid, dim3(kAttnThreads), 0, stream, query, ld_query, out, ld_out, heads / cache.kv_heads, \
                       scale, window, sinks, cache)
    switch (cache.element_type) {
    case kTypeF32: TSHIP_ATTEND(float); break;
    case kTypeF16: TSHIP_ATTEND(__half); break;
    default: TSHIP_ATTEND(__hip_bfloat16); break;
    }
#undef TSHIP_ATTEND
    return hip_ok(hipGetLastError(), "paged attention launch");
}

}  // namespace tship
