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
#include <cmath>
#include <type_traits>

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
//
// The rows that share a KV head - (new token, head of the group), token after token - are cut into tiles.  A tile walks over its keys
// with a running maximum and sum:
//   S^T = K Q^T        keys x rows, so that a lane holds one row and its maximum, sum and scale need no other lanes but the one that has
//                      the row's other keys
//   P = 2^(c S - m)    in the registers that the next product takes as its operand: its keys are counted in the order in which S^T
//                      leaves them, and V is read from LDS transposed in that order
//   O^T += V^T P^T
// on v_mfma_f32_32x32x16.  The result is fp32 and so are queries; rounding q or P to 16 bits would leave 1e-4 of the result.  Both are
// cut into parts instead that the matrix instruction takes exactly: two of fp16 (22 bits; the row of q under a power of two of its
// own), or three of bf16 (24 bits), and an fp32 cache likewise when it is read from LDS.  Products per element of a score: 2 for an fp16 cache,
// 3 for bf16, 6 for fp32 (those above 2^-24).
//
// Sequences with at most 32 rows (answers): all wavefronts have the same rows and walk over different keys, each through LDS of its
// own, and meet at the end.  Others (prompts): tiles of 128 rows, each wavefront has 32 of them and all share the keys in LDS.
// With few tiles the keys are cut further over workgroups (splits), whose states paged_combine_kernel joins.

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t* lds_t;

constexpr int kAttnWaves = 4, kAttnThreads = 64 * kAttnWaves;
constexpr int kKeyRows = 32;         // rows of a sequence up to which its wavefronts share rows and not keys
constexpr int kTileRows = 32 * kAttnWaves;
constexpr float kLog2e = 1.44269504088896340736f;
// Weights are kept as 2^7 times what they are against the running maximum, which follows the true one only when that is 2^8 larger:
// they stay below 2^15, which fp16 holds, the accumulators are rescaled a few times a row instead of at every step, and weights down to
// 2^-21 of the largest have all their 22 bits.
constexpr float kBias = 7.f, kSlack = 8.f;

// rows that a lane's page has not (past the end, or no page at all) are read from here
__device__ __attribute__((aligned(16))) uint8_t g_zero_row[kMaxDim * 4];

struct AttnArgs {
    const float* query;
    float* out;
    const float* sinks;
    float* partial;              // [row][head][split][head_dim] weighted values, then [row][head][split] (maximum, sum)
    int64_t ld_query, ld_out;
    float c;                     // |scale| log2 e
    float sign;                  // of scale, 0 where it is 0
    int rows, heads, group, window, splits, min_keys;
    FastDiv by_group;
    PagedKv cache;
};

// A tile: rows row0 .. row0 + count - 1 of the rows of a sequence, whose new tokens are rows first .. of the batch and begin at
// position p0; and its keys.
struct AttnTile {
    int first, tokens, p0, row0, count;
    int seq;
    int lo, hi;
};
__device__ __forceinline__ int tiles_of(int rows) { return rows <= kKeyRows ? (rows > 0 ? 1 : 0) : (rows + kTileRows - 1) / kTileRows; }
__device__ __forceinline__ void keys_of(const AttnArgs& A, AttnTile& t)
{
    const int p_first = t.p0 + (int)A.by_group.quot(t.row0), p_last = t.p0 + (int)A.by_group.quot(t.row0 + t.count - 1);
    t.lo = A.window > 0 ? max(0, p_first - A.window + 1) : 0;
    t.hi = (int)min((int64_t)p_last + 1, (int64_t)A.cache.max_pages * A.cache.page.d);
}
// keys of a split, a multiple of 128 (a step of four wavefronts), and from it how many splits there are
__device__ __forceinline__ int split_keys(const AttnArgs& A, const AttnTile& t)
{
    const int span = t.hi - t.lo;
    const int wanted = max(1, min(A.splits, (span + A.min_keys - 1) / A.min_keys));
    return ((span + wanted - 1) / wanted + 127) / 128 * 128;
}
__device__ __forceinline__ int clamped(int v, int hi) { return max(0, min(v, hi)); }
// The idx-th tile from the end (the last tiles of a prompt have the most keys and go first); every wavefront looks for itself.
__device__ __forceinline__ bool find_tile(const AttnArgs& A, int idx, AttnTile& t)
{
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int s0 = 0; s0 < A.cache.seqs; s0 += 64) {
        const int s = s0 + lane;
        int n = 0;
        if (s < A.cache.seqs) n = max(0, clamped(A.cache.row_starts[s + 1], A.rows) - clamped(A.cache.row_starts[s], A.rows));
        int sum = tiles_of(n * A.group);
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        total += sum;
    }
    int want = total - 1 - idx;
    if (want < 0) return false;
    for (int s0 = 0;; s0 += 64) {
        const int s = s0 + lane;
        int start = 0, n = 0;
        if (s < A.cache.seqs) {
            start = clamped(A.cache.row_starts[s], A.rows);
            n = max(0, clamped(A.cache.row_starts[s + 1], A.rows) - start);
        }
        const int mine = tiles_of(n * A.group);
        int cum = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const int below = __shfl_up(cum, o);
            if (lane >= o) cum += below;
        }
        const uint64_t here = __ballot(want < cum);
        if (here == 0) {
            want -= __shfl(cum, 63);
            continue;
        }
        const int at = __ffsll((unsigned long long)here) - 1;
        t.seq = s0 + at;
        t.first = __builtin_amdgcn_readlane(start, at);
        t.tokens = __builtin_amdgcn_readlane(n, at);
        want -= __builtin_amdgcn_readlane(cum - mine, at);
        break;
    }
    want = __builtin_amdgcn_readfirstlane(want);
    const int rows = t.tokens * A.group;
    t.row0 = want * kTileRows;
    t.count = min(rows - t.row0, rows <= kKeyRows ? kKeyRows : kTileRows);
    t.p0 = __builtin_amdgcn_readfirstlane(A.cache.context_lens[t.seq]) - t.tokens;
    keys_of(A, t);
    return true;
}

__device__ __forceinline__ uint32_t high_halves(float x, float y) { return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u); }
__device__ __forceinline__ float below_bf16(float x) { return x - __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
// eight floats as three times eight bf16 that sum up to them
__device__ __forceinline__ void cut3(const float (&x)[8], u4_t (&part)[3])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = below_bf16(x0), y1 = below_bf16(x1);
        part[0][i] = high_halves(x0, x1);
        part[1][i] = high_halves(y0, y1);
        part[2][i] = high_halves(below_bf16(y0), below_bf16(y1));
    }
}
// eight floats in fp16's range as twice eight fp16: what two roundings towards zero leave is below 2^-20 of each
__device__ __forceinline__ void cut2(const float (&x)[8], u4_t (&part)[2])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto hi = __builtin_amdgcn_cvt_pkrtz(x[2 * i], x[2 * i + 1]);
        const auto lo = __builtin_amdgcn_cvt_pkrtz(x[2 * i] - (float)hi[0], x[2 * i + 1] - (float)hi[1]);
        part[0][i] = __builtin_bit_cast(uint32_t, hi);
        part[1][i] = __builtin_bit_cast(uint32_t, lo);
    }
}
__device__ __forceinline__ float both_halves(float x, float (*op)(float, float))
{
    const u2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float added(float a, float b) { return a + b; }

// TYPE: 0 fp32, 1 fp16, 2 bf16 cache; HD: head_dim rounded up to what the tiles are made for
template <int TYPE, int HD>
struct Attn {
    static constexpr int kElem = TYPE == 0 ? 4 : 2;
    static constexpr int kRow = HD * kElem, kPieces = kRow / 16;     // a key (value) in LDS, 16 bytes at a time
    static constexpr int kParts = TYPE == 1 ? 2 : 3;                 // of q and of the weights
    static constexpr int kCacheParts = TYPE == 0 ? 3 : 1;
    static constexpr int kSteps = HD / 16, kDims = HD / 32;
    static constexpr int NT = TYPE == 1 ? 2 : 1;                     // 32-key blocks of a step where wavefronts share the keys
    static constexpr int kKeyWaves = TYPE == 0 ? 2 : 4;              // wavefronts that have keys of their own
    static constexpr int kBlock = 32 * kRow;                         // bytes of 32 keys
    static constexpr int kCopies = kPieces / 2;                      // wavefront-wide copies of 32 keys
    static constexpr int kLds = kBlock * 2 * (2 * NT > kKeyWaves ? 2 * NT : kKeyWaves);

    // Where piece p of a row lies: rows are a multiple of 128 bytes apart (192: of 64), so eight neighbouring keys read at one piece, and the
    // four keys of a transposed read, are spread over the banks.
    __device__ static __forceinline__ int k_swizzle(int key) { return kPieces % 8 == 0 ? key & 7 : (key >> 1) & 3; }
    __device__ static __forceinline__ int v_swizzle(int key)
    {
        return TYPE == 0 ? key & 7 : kPieces % 8 == 0 ? (key & 3) << 1 : ((key >> 1) & 1) << 1;
    }

    typedef typename std::conditional<TYPE == 1, h8_t, b8_t>::type operand_t;
    __device__ static __forceinline__ f16_t mfma(const u4_t& a, const u4_t& b, const f16_t& c)
    {
        if constexpr (TYPE == 1) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
    }

    const AttnArgs& A;
    const AttnTile t;
    const int kvh, lane, col, half;
    lds_t lds;
    u4_t q[kParts][kSteps];
    f16_t o[kDims];
    float c, m, l;                   // score to exponent, running maximum (as an exponent), this lane's part of the sum
    int p, lo;                       // position of this lane's row, first key it sees

    __device__ __forceinline__ Attn(const AttnArgs& args, const AttnTile& tile, int kv_head, lds_t smem)
        : A(args), t(tile), kvh(kv_head), lane(threadIdx.x & 63), col(lane & 31), half(lane >> 5), lds(smem)
    {
    }

    // row of the tile -> token and head
    __device__ __forceinline__ void place(int row, int* token, int* head) const
    {
        const int r = t.row0 + row, i = (int)A.by_group.quot(r);
        *token = i;
        *head = kvh * A.group + (r - i * A.group);
    }

    __device__ __forceinline__ void load_rows(int row)
    {
        const bool live = row < t.count;
        int token, head;
        place(live ? row : 0, &token, &head);
        const float* src = A.query + (int64_t)(t.first + token) * A.ld_query + (int64_t)head * A.cache.head_dim;
        p = t.p0 + token;
        lo = A.window > 0 ? p - A.window + 1 : 0;
        auto eight = [&](int s, float (&x)[8]) {
            const int d = 16 * s + 8 * half;
            f4_t a = {0.f, 0.f, 0.f, 0.f}, b = a;
            if (live && d < A.cache.head_dim) {
                a = *reinterpret_cast<const f4_t*>(src + d);
                b = *reinterpret_cast<const f4_t*>(src + d + 4);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i] * A.sign;
                x[4 + i] = b[i] * A.sign;
            }
        };
        c = A.c;
        int e = 0;
        if constexpr (TYPE == 1) {
            // the row's largest at 2^13 .. 2^14 (its own pass: kept in between, the row would not fit beside its parts)
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                float x[8];
                eight(s, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
            }
            top = both_halves(top, larger);
            if (top > 0.f && top < INFINITY) e = 14 - __builtin_amdgcn_frexp_expf(top);
            c = ldexpf(A.c, -e);
            asm volatile("" ::: "memory");
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            float x[8];
            eight(s, x);
            u4_t part[kParts];
            if constexpr (TYPE == 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = ldexpf(x[i], e);
                cut2(x, part);
            } else {
                cut3(x, part);
            }
#pragma unroll
            for (int i = 0; i < kParts; ++i) q[i][s] = part[i];
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
        m = -INFINITY;
        l = 0.f;
    }

    // ---- keys and values into LDS ----
    // Lane i has the id of page id_base + i; read again when a step passes the last of them.  (Held like this they cost a load
    // every 64 pages and no load beside the copies, whose waits count loads.)
    int ids, id_base = -64;
    template <int KEYS>
    __device__ __forceinline__ int page_id(int key0, int mine, int end)
    {
        const int first = (int)A.cache.page.quot((uint32_t)key0);   // uniform
        if ((int)A.cache.page.quot((uint32_t)(key0 + KEYS - 1)) - id_base >= 64) {
            id_base = first;
            ids = A.cache.table[t.seq * A.cache.table_stride + min(first + lane, A.cache.max_pages - 1)];
        }
        const int id = __shfl(ids, (int)A.cache.page.quot((uint32_t)mine) - id_base);
        return mine < end ? id : -1;
    }
    struct Rows {
        uint64_t k, v;               // addresses of this lane's key and value
        uint64_t there;              // which lanes' are in the cache
    };
    __device__ __forceinline__ Rows rows_of(int key, int id) const
    {
        const bool ok = (uint32_t)id < (uint32_t)A.cache.num_pages;
        const int within = key - (int)A.cache.page.quot((uint32_t)key) * (int)A.cache.page.d;
        const int64_t zero = (int64_t)(uintptr_t)g_zero_row;
        const int64_t k = (int64_t)(uintptr_t)A.cache.k + (id * A.cache.k_page + within * A.cache.k_token + kvh * A.cache.k_head) * kElem;
        const int64_t v = (int64_t)(uintptr_t)A.cache.v + (id * A.cache.v_page + within * A.cache.v_token + kvh * A.cache.v_head) * kElem;
        return {(uint64_t)(ok ? k : zero), (uint64_t)(ok ? v : zero), __ballot(ok)};
    }
    // copy n of a block: 64 pieces that follow one another in LDS
    template <bool V>
    __device__ __forceinline__ void copy(uint64_t rows, int n, lds_t block) const
    {
        const int slot = n * 64 + lane, row = slot / kPieces, piece = (slot - row * kPieces) ^ (V ? v_swizzle(row) : k_swizzle(row));
        uint64_t at = (uint64_t)__shfl((unsigned long long)rows, row);
        if (piece * 16 >= A.cache.head_dim * kElem) at = (uint64_t)(uintptr_t)g_zero_row;
        at += piece * 16;
        // (In assembly, because the compiler would wait for every copy under way in front of each transposed read.  It writes no register
        // but m0, which nothing else here uses.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(block + n * 1024))),
                     "v"(at)
                     : "memory", "m0");
#pragma clang diagnostic pop
    }

    // ---- one product step ----
    __device__ __forceinline__ u4_t read16(lds_t at) const { return *reinterpret_cast<const __attribute__((address_space(3))) u4_t*>(at); }
    __device__ __forceinline__ float read4(lds_t at) const { return *reinterpret_cast<const __attribute__((address_space(3))) float*>(at); }

    // S^T of 32 keys
    __device__ __forceinline__ f16_t scores(lds_t block) const
    {
        f16_t s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
        const lds_t row = block + col * kRow;
        const int x = k_swizzle(col);
        // (the swizzle changes the lower bits of a piece's number only, so that one address serves every kAgain-th step)
        constexpr int kAgain = (kPieces % 8 == 0 ? 8 : 4) / (TYPE == 0 ? 4 : 2);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int j = i % kAgain, further = (i - j) * (TYPE == 0 ? 64 : 32);
            if constexpr (TYPE != 0) {
                const u4_t a = read16(row + (((2 * j + half) ^ x) << 4) + further);
#pragma unroll
                for (int n = 0; n < kParts; ++n) s = mfma(a, q[n][i], s);
            } else {
                const u4_t a0 = read16(row + (((4 * j + 2 * half) ^ x) << 4) + further), a1 = read16(row + (((4 * j + 2 * half + 1) ^ x) << 4) + further);
                float v[8];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    v[n] = __uint_as_float(a0[n]);
                    v[4 + n] = __uint_as_float(a1[n]);
                }
                u4_t part[3];
                cut3(v, part);
                s = products(part, i, s);
            }
        }
        return s;
    }
    __device__ __forceinline__ f16_t products(const u4_t (&a)[3], int i, f16_t s) const
    {
        s = mfma(a[2], q[0][i], s);
        s = mfma(a[1], q[1][i], s);
        s = mfma(a[0], q[2][i], s);
        s = mfma(a[1], q[0][i], s);
        s = mfma(a[0], q[1][i], s);
        return mfma(a[0], q[0][i], s);
    }
    // Of the 16 scores of a lane number i belongs to key 8 (i / 4) + 4 half + i % 4 of the block.
    __device__ __forceinline__ void mask(f16_t& s, int key0, uint64_t there) const
    {
        const uint32_t bits = (uint32_t)(there >> (4 * half));
        const int last = p - key0 - 4 * half, first = lo - key0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int k = 8 * (i / 4) + i % 4;
            if (k > last || k < first || !((bits >> k) & 1)) s[i] = -INFINITY;
        }
    }
    __device__ __forceinline__ void follow_maximum(const f16_t* s, int blocks)
    {
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < blocks; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        top = both_halves(top, larger) * c;
        if (__any(top > m + kSlack)) {                               // (m starts at -infinity)
            const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            l *= f;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            m = mn;
        }
    }
    // weights of a block's scores, their sum, and O^T += V^T P^T
    __device__ __forceinline__ void weigh(const f16_t& s, lds_t block)
    {
        const float bias = kBias - (m == -INFINITY ? 0.f : m);
        const int x = v_swizzle((lane & 15) >> 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                                // 16 keys
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * h + i], c, bias));
                l += w[i];
            }
            u4_t part[kParts];
            if constexpr (TYPE == 1) cut2(w, part);
            else cut3(w, part);
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                if constexpr (TYPE != 0) {
                    // a lane gives the place of four dimensions of one key and gets one dimension of four keys, within 16 lanes
                    const int piece = (4 * (d & 1) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ x;
                    const lds_t at = block + (4 * half + ((lane & 15) >> 2)) * kRow + (piece << 4) + (lane & 1) * 8 + 16 * h * kRow + (d & ~1) * 64;
                    const s4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)at);
                    const s4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)(at + 8 * kRow));
                    const u2_t a0 = __builtin_bit_cast(u2_t, v0), a1 = __builtin_bit_cast(u2_t, v1);
                    const u4_t a = {a0.x, a0.y, a1.x, a1.y};
#pragma unroll
                    for (int n = 0; n < kParts; ++n) o[d] = mfma(a, part[n], o[d]);
                } else {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int key = 4 * half + i % 4;
                        v[i] = read4(block + key * kRow + (((col >> 2) ^ v_swizzle(key)) << 4) + (col & 3) * 4 + (16 * h + 8 * (i / 4)) * kRow + 128 * d);
                    }
                    u4_t a[3];
                    cut3(v, a);
                    f16_t acc = o[d];
                    acc = mfma(a[2], part[0], acc);
                    acc = mfma(a[1], part[1], acc);
                    acc = mfma(a[0], part[2], acc);
                    acc = mfma(a[1], part[0], acc);
                    acc = mfma(a[0], part[1], acc);
                    o[d] = mfma(a[0], part[0], acc);
                }
            }
        }
    }

    // ---- where a row's state goes ----
    __device__ __forceinline__ float* values_of(int token, int head, int split) const
    {
        return A.partial + (((int64_t)(t.first + token) * A.heads + head) * A.splits + split) * A.cache.head_dim;
    }
    __device__ __forceinline__ f2_t* state_of(int token, int head, int split) const
    {
        return reinterpret_cast<f2_t*>(A.partial + (int64_t)A.rows * A.heads * A.splits * A.cache.head_dim) +
               (((int64_t)(t.first + token) * A.heads + head) * A.splits + split);
    }
    // what a row's sum is divided by: with the sink, 1 / 0 never
    __device__ __forceinline__ float over_sum(float sum, float top, int head) const
    {
        if (!(sum > 0.f)) return 0.f;
        if (A.sinks) sum += __builtin_amdgcn_exp2f(A.sinks[head] * kLog2e - top + kBias);
        return 1.0f / sum;
    }

    // all wavefronts over the same keys, 32 rows each
    __device__ __forceinline__ void shared_keys(int begin, int end, int split)
    {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        load_rows(32 * wave + col);
        const int p_first = t.p0 + (int)A.by_group.quot(t.row0 + min(32 * wave, t.count - 1));
        const int p_last = t.p0 + (int)A.by_group.quot(t.row0 + min(32 * wave + 31, t.count - 1));
        const int lo_last = A.window > 0 ? p_last - A.window + 1 : 0;
        constexpr int kKeys = 32 * NT;
        const int mine = lane & (kKeys - 1);
        auto stage = [&](const Rows& r, lds_t buffer) {
#pragma unroll
            for (int n = 0; n < (NT * kCopies + kAttnWaves - 1) / kAttnWaves; ++n)
                if (NT * kCopies % kAttnWaves == 0 || wave + kAttnWaves * n < NT * kCopies) {
                    copy<false>(r.k, wave + kAttnWaves * n, buffer);
                    copy<true>(r.v, wave + kAttnWaves * n, buffer + NT * kBlock);
                }
        };
        int buffer = 0;
        if (begin < end) {
            // copies go a step ahead; those behind the last key bring zeros that nothing reads
            Rows rows = rows_of(begin + mine, page_id<kKeys>(begin, begin + mine, end));
            stage(rows, lds);
            for (int key0 = begin; key0 < end; key0 += kKeys) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                const lds_t here = lds + buffer * (2 * NT * kBlock);
                const uint64_t there = rows.there;
                buffer ^= 1;
                rows = rows_of(key0 + kKeys + mine, page_id<kKeys>(key0 + kKeys, key0 + kKeys + mine, end));
                stage(rows, lds + buffer * (2 * NT * kBlock));
                // (a wavefront without rows copies only, as does one whose rows see none of the keys)
                if (32 * wave < t.count && key0 <= p_last) {
                    f16_t s[NT];
#pragma unroll
                    for (int b = 0; b < NT; ++b) s[b] = scores(here + b * kBlock);
                    if (~there != 0 || key0 + kKeys - 1 > p_first || key0 < lo_last) {
#pragma unroll
                        for (int b = 0; b < NT; ++b) mask(s[b], key0 + 32 * b, there >> (32 * b));
                    }
                    follow_maximum(s, NT);
#pragma unroll
                    for (int b = 0; b < NT; ++b) weigh(s[b], here + (NT + b) * kBlock);
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the last copies, before this LDS may be another workgroup's
        }
        const int row = 32 * wave + col;
        l = both_halves(l, added);
        if (row >= t.count) return;
        int token, head;
        place(row, &token, &head);
        float* dst;
        float by = 1.f;
        if (A.splits == 1) {
            dst = A.out + (int64_t)(t.first + token) * A.ld_out + (int64_t)head * A.cache.head_dim;
            by = over_sum(l, m, head);
        } else {
            dst = values_of(token, head, split);
            if (half == 0) *state_of(token, head, split) = f2_t{m, l};
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 32 * d + 8 * i + 4 * half;
                if (at < A.cache.head_dim)
                    *reinterpret_cast<f4_t*>(dst + at) = f4_t{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * by;
            }
    }

    // every wavefront over keys of its own, the same (up to 32) rows
    __device__ __forceinline__ void own_keys(int begin, int end, int split)
    {
        __shared__ f2_t states[kAttnWaves][32];
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        load_rows(col);
        const int p_last = t.p0 + t.tokens - 1;
        const int lo_last = A.window > 0 ? p_last - A.window + 1 : 0;
        const lds_t kb = lds + wave * 2 * kBlock, vb = kb + kBlock;
        int key0 = begin + 32 * wave;
        constexpr int kStride = 32 * kKeyWaves;
        if (wave < kKeyWaves && key0 < end) {
            auto stage = [&](auto is_v, uint64_t rows, lds_t block) {
#pragma unroll
                for (int n = 0; n < kCopies; ++n) copy<decltype(is_v)::value>(rows, n, block);
            };
            Rows rows = rows_of(key0 + col, page_id<32>(key0, key0 + col, end));
            stage(std::false_type(), rows.k, kb);
            stage(std::true_type(), rows.v, vb);
            for (; key0 < end; key0 += kStride) {
                // loads answer in order: with kCopies of them left, the values behind the keys, the keys have arrived
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCopies) : "memory");
                f16_t s[1] = {scores(kb)};
                const uint64_t there = rows.there;
                rows = rows_of(key0 + kStride + col, page_id<32>(key0 + kStride, key0 + kStride + col, end));
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                stage(std::false_type(), rows.k, kb);
                if (~there != 0 || key0 + 31 > t.p0 || key0 < lo_last) mask(s[0], key0, there);
                follow_maximum(s, 1);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCopies) : "memory");                 // the values too: the next keys are left
                weigh(s[0], vb);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                stage(std::true_type(), rows.v, vb);
            }
        }
        l = both_halves(l, added);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (wave < kKeyWaves) {
            if (half == 0) states[wave][col] = f2_t{m, l};
            const lds_t row = lds + (wave * 32 + col) * HD * 4;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<__attribute__((address_space(3))) f4_t*>(row + (((8 * d + 2 * i + half) ^ (col & 7)) << 4)) =
                        f4_t{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        }
        __syncthreads();
        const int pieces = A.cache.head_dim / 4;
        for (int i = threadIdx.x; i < t.count * pieces; i += kAttnThreads) {
            const int row = i / pieces, piece = i - row * pieces;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kKeyWaves; ++w) top = fmaxf(top, states[w][row].x);
            const float base = top == -INFINITY ? 0.f : top;
            float sum = 0.f;
            f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kKeyWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(states[w][row].x - base);
                sum += states[w][row].y * f;
                v += *reinterpret_cast<const __attribute__((address_space(3))) f4_t*>(lds + (w * 32 + row) * HD * 4 + ((piece ^ (row & 7)) << 4)) * f;
            }
            int token, head;
            place(row, &token, &head);
            if (A.splits == 1) {
                *reinterpret_cast<f4_t*>(A.out + (int64_t)(t.first + token) * A.ld_out + (int64_t)head * A.cache.head_dim + 4 * piece) =
                    v * over_sum(sum, top, head);
            } else {
                *reinterpret_cast<f4_t*>(values_of(token, head, split) + 4 * piece) = v;
                if (piece == 0) *state_of(token, head, split) = f2_t{top, sum};
            }
        }
    }
};

// grid (KV heads x tiles, splits)
template <int TYPE, int HD>
__global__ void __launch_bounds__(kAttnThreads, HD <= 128 ? 2 : 1) paged_attention_kernel(const AttnArgs A)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int kvh = blockIdx.x % A.cache.kv_heads, idx = blockIdx.x / A.cache.kv_heads, split = blockIdx.y;
    AttnTile t;
    if (!find_tile(A, idx, t)) return;
    const int len = split_keys(A, t), begin = t.lo + split * len, end = min(begin + len, t.hi);
    if (begin >= end && (split > 0 || A.splits > 1)) return;         // (rows that see nothing are set to zero by the first split, or when splits are joined)
    Attn<TYPE, HD> a(A, t, kvh, (lds_t)smem);
    if (t.tokens * A.group <= kKeyRows) a.own_keys(begin, end, split);
    else a.shared_keys(begin, end, split);
}

// one wavefront per (row, head): the splits of its tile
__global__ void __launch_bounds__(kAttnThreads) paged_combine_kernel(const AttnArgs A)
{
    const int lane = threadIdx.x & 63, row = blockIdx.x, head = blockIdx.y * kAttnWaves + (threadIdx.x >> 6), dim = A.cache.head_dim;
    const Place at = place_of_row(A.cache, row);
    if (at.seq < 0 || head >= A.heads) return;
    AttnTile t;
    const int start = clamped(at.first, A.rows);
    t.first = start;
    t.tokens = clamped(at.first + at.count, A.rows) - start;
    t.seq = at.seq;
    t.p0 = A.cache.context_lens[at.seq] - t.tokens;
    const int r = (row - start) * A.group + head % A.group, rows = t.tokens * A.group;
    t.row0 = rows <= kKeyRows ? 0 : r / kTileRows * kTileRows;
    t.count = min(rows - t.row0, rows <= kKeyRows ? kKeyRows : kTileRows);
    keys_of(A, t);
    const int span = t.hi - t.lo, len = split_keys(A, t), splits = span > 0 ? (span + len - 1) / len : 0;
    const int64_t first = ((int64_t)row * A.heads + head) * A.splits;
    const float* values = A.partial + first * dim;
    const f2_t* states = reinterpret_cast<const f2_t*>(A.partial + (int64_t)A.rows * A.heads * A.splits * dim) + first;
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 64) top = fmaxf(top, states[s].x);
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f4_t acc = {0.f, 0.f, 0.f, 0.f};
    const bool mine = 4 * lane < dim;
    for (int s = 0; s < splits; ++s) {
        const f2_t st = states[s];
        const float f = __builtin_amdgcn_exp2f(st.x - base);
        sum += st.y * f;
        if (mine) acc += *reinterpret_cast<const f4_t*>(values + (int64_t)s * dim + 4 * lane) * f;
    }
    float by = 0.f;
    if (sum > 0.f) {
        if (A.sinks) sum += __builtin_amdgcn_exp2f(A.sinks[head] * kLog2e - base + kBias);
        by = 1.0f / sum;
    }
    if (mine) *reinterpret_cast<f4_t*>(A.out + (int64_t)row * A.ld_out + (int64_t)head * dim + 4 * lane) = acc * by;
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

PagedAttnPlan plan_paged_attention(int rows, int heads, const PagedKv& cache, int window)
{
    const int group = heads / cache.kv_heads;
    const int64_t all = (int64_t)rows * group;
    PagedAttnPlan plan{};
    // (a sequence of at most 32 rows has one tile, others a tile per 128 rows begun: no more than this, whatever the lengths)
    plan.tiles = (int)(all / kTileRows + std::min<int64_t>(cache.seqs, rows));
    const int64_t items = (int64_t)plan.tiles * cache.kv_heads, keys = (int64_t)cache.max_pages * cache.page.d;
    const bool few = all <= (int64_t)kKeyRows * cache.seqs;          // mostly answers
    plan.min_keys = few ? 256 : 512;
    const int64_t span = window > 0 ? std::min<int64_t>(keys, (int64_t)window + (few ? kKeyRows : kTileRows)) : keys;
    const int64_t wanted = few ? 2048 / items : items >= 384 ? 1 : 768 / items;
    plan.splits = (int)std::max<int64_t>(1, std::min<int64_t>({wanted, (span + plan.min_keys - 1) / plan.min_keys, 1024}));
    if (plan.splits > 1) plan.ws_bytes = (size_t)rows * heads * plan.splits * (cache.head_dim + 2) * sizeof(float);
    return plan;
}

template <int TYPE, int HD>
static bool launch_attention(const AttnArgs& args, const dim3& grid, hipStream_t stream)
{
    const auto kern = paged_attention_kernel<TYPE, HD>;
    constexpr size_t lds = Attn<TYPE, HD>::kLds;
    if (!raise_lds_limit(reinterpret_cast<const void*>(kern), lds)) return false;
    hipLaunchKernelGGL(kern, grid, dim3(kAttnThreads), lds, stream, args);
    return hip_ok(hipGetLastError(), "paged attention launch");
}
template <int TYPE>
static bool launch_attention(const AttnArgs& args, const dim3& grid, hipStream_t stream)
{
    const int dim = args.cache.head_dim;
    if (dim <= 64) return launch_attention<TYPE, 64>(args, grid, stream);
    if (dim <= 96) return launch_attention<TYPE, 96>(args, grid, stream);
    if (dim <= 128) return launch_attention<TYPE, 128>(args, grid, stream);
    if (dim <= 192) return launch_attention<TYPE, 192>(args, grid, stream);
    return launch_attention<TYPE, 256>(args, grid, stream);
}

bool launch_paged_attention(const PagedAttnPlan& plan, const float* query, int64_t ld_query, float* out, int64_t ld_out, int rows, int heads,
                            const PagedKv& cache, float scale, int window, const float* sinks, void* ws, hipStream_t stream)
{
    AttnArgs args{};
    args.query = query;
    args.out = out;
    args.sinks = sinks;
    args.partial = static_cast<float*>(ws);
    args.ld_query = ld_query;
    args.ld_out = ld_out;
    args.c = scale == 0.f ? 1.f : (float)(std::fabs((double)scale) * 1.44269504088896340736);
    args.sign = scale == 0.f ? 0.f : scale < 0.f ? -1.f : 1.f;
    args.rows = rows;
    args.heads = heads;
    args.group = heads / cache.kv_heads;
    args.window = window;
    args.splits = plan.splits;
    args.min_keys = plan.min_keys;
    args.by_group = FastDiv((uint32_t)args.group);
    args.cache = cache;
    if ((int64_t)plan.tiles * cache.kv_heads > INT32_MAX || (int64_t)rows * args.group > INT32_MAX) {
        set_last_error("paged_attention: too many rows for one call.");
        return false;
    }
    const dim3 grid((unsigned)(plan.tiles * cache.kv_heads), plan.splits);
    bool ok;
    switch (cache.element_type) {
    case kTypeF32: ok = launch_attention<0>(args, grid, stream); break;
    case kTypeF16: ok = launch_attention<1>(args, grid, stream); break;
    default: ok = launch_attention<2>(args, grid, stream); break;
    }
    if (!ok || plan.splits == 1) return ok;
    hipLaunchKernelGGL(paged_combine_kernel, dim3(rows, (heads + kAttnWaves - 1) / kAttnWaves), dim3(kAttnThreads), 0, stream, args);
    return hip_ok(hipGetLastError(), "paged attention combine launch");
}

}  // namespace tship
