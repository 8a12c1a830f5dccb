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
#include <utility>

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
// Bound: memory (2048 tokens of 32 heads of 128: 11.9 us, 67 MB in and out at 5.7 TB/s, a large copy 5.2), and for few tokens the latency of
// the angles and one trip to memory (24 tokens: 3.1 us).
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

// Which sequence's new token a row of `rows` is: the number of sequences that end at or before it (row_starts does not fall, and is cut to
// the rows there are).  Every wavefront looks for itself, 64 sequences at a time.
struct Place {
    int seq, first, count;       // seq -1: of none
};
__device__ __forceinline__ Place place_of_row(const PagedKv& C, int row, int rows)
{
    const int lane = threadIdx.x & 63;
    int seq = 0;
    for (int s0 = 0; s0 < C.seqs; s0 += 64) {
        const bool before = s0 + lane < C.seqs && C.row_starts[s0 + lane + 1] <= row;
        const uint64_t ends = __ballot(before);
        seq += __popcll(ends);
        if (~ends != 0) break;
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    if (seq >= C.seqs) return {-1, 0, 0};
    const int first = max(0, C.row_starts[seq]), end = min(rows, C.row_starts[seq + 1]);
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

// grid (rows, head chunks), lanes and angles as above; the lanes of a head add the squares of its norm.  One pass: a row is read once, and what
// a query, key and value head become is written where the attention reads it.  Bound: memory (3515 rows of 32 + 2 x 8 heads of 128 into bf16 pages: 32 us
// on the device, 158 MB at 4.9 TB/s), and for few rows the way from lengths to page to address (24 rows: 4 us).
template <int LANES, typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_store_kernel(const float* qkv, int64_t ld_qkv, float* query, int64_t ld_query, int heads,
                                                                  const int32_t* positions, const float* q_norm, const float* k_norm,
                                                                  float eps, const PagedKv C, const RopeSpec R)
{
    __shared__ f2_t turns[kMaxDim / 2];
    constexpr int kHeads = kRopeThreads / LANES;
    const int t = blockIdx.x;
    const Place at = place_of_row(C, t, gridDim.x);
    if (at.seq < 0) return;                                          // uniform
    const int u = threadIdx.x % LANES, dim = C.head_dim, all = heads + 2 * C.kv_heads;
    const bool live = 4 * u < dim;
    const int where = max(C.context_lens[at.seq], -(1 << 30)) - at.count + (t - at.first);
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
// m need not be the maximum: weights are 2^kUnit times what they are against m, a whole number that follows when a step's largest score is more
// than kRise above it, so that the accumulators are rescaled (exactly) a few times a row and not at every step.  In two parts of fp16 a weight's last
// bit is 2^-24, so that one below 2^-2 has less than 22 bits: nothing beside what larger ones have summed up to, unless their values are next to
// nothing, as those of a first token that takes what no other key asks for are.  So for an fp16 cache m comes down too, where a step's largest score is
// kFall below it, once in kWait steps at most (peaked scores would have it at every step: prompts took 1.4 to 2 times as long).  It is set kAhead above
// the largest score, whose weight is 2^8 then, or right at a score that stands kApart above the step's others, which have 2^-39 of its weight left to
// them.  For other caches weights begin at 2^7, so that the parts of small values and weights stay normal numbers; where large values add up to
// infinity then, the rows are done again by plainly().
//
// Sequences with at most 32 rows (answers): all wavefronts have the same rows and walk over different keys, each through LDS of its
// own, and meet at the end.  Others (prompts): tiles of 128 rows, each wavefront has 32 of them and all share the keys in LDS.
// With few tiles the keys are cut further over workgroups, whose states paged_combine_kernel joins.

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef float f16_t __attribute__((ext_vector_type(16)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint8_t* lds_t;

constexpr int kAttnWaves = 4, kAttnThreads = 64 * kAttnWaves;
constexpr int kKeyRows = 32;         // rows of a sequence up to which its wavefronts share rows and not keys
constexpr int kTileRows = 32 * kAttnWaves;
constexpr int kMaxPieces = 1024;      // that a tile's keys are cut into
constexpr float kLog2e = 1.44269504088896340736f;
// rows that a lane's page has not (past the end, or no page at all) are read from here
__device__ __attribute__((aligned(16))) uint8_t g_zero_row[kMaxDim * 4];

struct AttnArgs {
    const float* query;
    float* out;
    const float* sinks;
    float* partial;              // [piece][KV head][row of the tile][head_dim] weighted values, then [piece][KV head][row] (unit, sum)
    int64_t ld_query, ld_out;
    float c;                     // |scale| log2 e
    float sign;                  // of scale, 0 where it is 0
    int rows, group, window, capacity;
    int slots, slot_rows;        // of partial
    FastDiv by_group;
    PagedKv cache;
};

// A tile: rows row0 .. row0 + count - 1 of the rows of a sequence, whose new tokens are rows first .. of the batch and begin at
// position p0; and the keys that it has, or the piece of them that a workgroup takes.
struct AttnTile {
    int first, tokens, p0, row0, count;
    int seq;
    int lo, hi;
    int cuts, slot;              // pieces of its keys; where the first one's (this one's) state goes
};
__device__ __forceinline__ int tiles_of(int rows) { return rows <= kKeyRows ? (rows > 0 ? 1 : 0) : (rows + kTileRows - 1) / kTileRows; }
__device__ __forceinline__ int clamped(int v, int hi) { return max(0, min(v, hi)); }
// inclusive sum over the lanes of a wavefront, in registers
__device__ __forceinline__ int lane_scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);          // from the lane 1, 2, 4, 8 below, within 16 lanes
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);         // the last lane of 16 to the next 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);         // of 32 to the upper 32
    return v;
}
__device__ __forceinline__ int lane_sum(int v) { return __builtin_amdgcn_readlane(lane_scan(v), 63); }

// What the kernels need to find their piece.  It stands in front of the other arguments: the hardware delivers the first 14 dwords in
// registers at wave launch (a structure is read from the argument block instead), so that the lengths are asked for at once.
struct Lens {
    const int32_t* row_starts;
    const int32_t* context_lens;
    int seqs, rows, group, window;
    int pieces;                  // per KV head that the chip takes at once; 0: keys are not cut
    int capacity;                // positions that the page table has room for
};
#define TSHIP_LENS_ARGS const int32_t *row_starts, const int32_t *context_lens, int seqs, int rows, int group, int window, int pieces, int capacity
#define TSHIP_LENS Lens{row_starts, context_lens, seqs, rows, group, window, pieces, capacity}

// 64 sequences, one per lane
struct Lanes {
    int start, n, context;
    int tiles, steps;            // steps of 128 keys that a tile has at most
    __device__ __forceinline__ void load(const Lens& H, int s0)
    {
        const int s = s0 + (threadIdx.x & 63);
        start = n = context = 0;
        if (s < H.seqs) {
            const int a = H.row_starts[s], b = H.row_starts[s + 1];
            context = max(H.context_lens[s], -(1 << 30));
            start = clamped(a, H.rows);
            n = max(0, clamped(b, H.rows) - start);
        }
        tiles = tiles_of(n * H.group);
        // (a tile's rows are of at most 128 tokens)
        int span = min(max(0, context), H.capacity);
        if (H.window > 0) span = (int)min((int64_t)span, (int64_t)H.window + min(n, kTileRows));
        steps = (span + 127) >> 7;
    }
    __device__ __forceinline__ int cuts(int len) const { return max(1, (steps + len - 1) / len); }
};

// Steps of 128 keys that pieces have to save a tile to be worth it.  Joining them takes 5 us where they are few, 8.5 for many short tiles, 7.5
// for long ones (3 of it the second launch, which comes wherever the page table has room for as many positions).  A step takes a short tile of
// 64, 128, 256 dimensions 1.0, 1.4, 2.9 us in fp16 (bf16 0.9, 1.6, 3.5; fp32, by fewer wavefronts, 2.1, 8.4, 19.3) and a long one 2.6, 4.4,
// 8.7 (bf16 4.1, 5.6, 12.2; fp32 7.4, 12.5, 29.5): by the dimensions, near enough.  One sequence of 512 keys, 256 dimensions and 8 KV heads: cut
// 37 us, uncut 90 in fp32, 18 and 22 in fp16; 16 of 128 dimensions in fp16: 17 and 13.
struct Worth {
    int few, many, tall;
};
__host__ __device__ constexpr Worth worth_of(int type, int hd, int key_waves)
{
    const int step = hd * (type == kTypeF32 ? 14 : 5) / (10 * key_waves);                  // 0.1 us
    const int tall = hd * (type == kTypeF32 ? 110 : type == kTypeF16 ? 40 : 55) / 100;
    return {(50 + step - 1) / step, (85 + step - 1) / step, (75 + tall - 1) / tall};
}
__host__ __device__ constexpr int key_waves_of(int type, int hd) { return type != kTypeF32 || hd == 64 ? 4 : hd == 96 || hd == 192 ? 3 : 2; }
__host__ __device__ constexpr int dims_of(int dim) { return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }

// How many steps of 128 keys a piece has, so that the pieces of all tiles are about as many as the chip takes at once and as long as one
// another (more would wait for a second round, fewer or unequal ones leave compute units without work).  At least their mean, in
// a few tries up to what is certain to be enough.  32 sequences of 4096 keys and 8 KV heads: 104 us in 512 pieces, 107 in 1024, 136 in 4096.
__device__ __forceinline__ int piece_steps(const Lens& H, int kv_heads, Worth least, Lanes& L)
{
    constexpr int kUncut = 1 << 24;
    L.load(H, 0);
    if (H.pieces == 0) return kUncut;
    int tiles = 0;
    float steps = 0.f;
    for (int s0 = 0;;) {
        tiles += lane_sum(L.tiles);
        steps += (float)lane_sum(min(L.tiles * min(L.steps, 1 << 16), 1 << 24));
        s0 += 64;
        if (s0 >= H.seqs) break;
        L.load(H, s0);
    }
    if (tiles >= H.pieces) {
        if (H.seqs > 64) L.load(H, 0);
        return kUncut;
    }
    const float mean = steps / (float)H.pieces, enough = fmaxf(steps / (float)(H.pieces - tiles), mean);
    int len = 0;
    bool worth = false;
    float f = 1.f;
    for (int i = 0;; ++i, f *= 1.15f) {
        // (a length that no tile exceeds ends it in any case)
        len = i < 5 ? max(1, (int)ceilf(fminf(mean * f, enough))) : i == 5 ? max(1, (int)ceilf(enough)) : len + len / 8 + 1;
        int all = 0;
        worth = false;
        for (int s0 = 0; s0 < H.seqs; s0 += 64) {
            if (H.seqs > 64) L.load(H, s0);
            all += lane_sum(L.tiles * L.cuts(len));
            worth |= __any(L.steps - len >= (L.n * H.group > kKeyRows ? least.tall : tiles * kv_heads >= 64 ? least.many : least.few));
        }
        if (all <= H.pieces) break;
    }
    if (!worth) len = kUncut;
    if (H.seqs > 64) L.load(H, 0);
    return len;
}

// rows and keys of tile number `tile` of the sequence of lane `at`
__device__ __forceinline__ void set_tile(const AttnArgs& A, const Lanes& L, int s0, int at, int tile, int len, AttnTile& t)
{
    t.seq = s0 + at;
    t.first = __builtin_amdgcn_readlane(L.start, at);
    t.tokens = __builtin_amdgcn_readlane(L.n, at);
    t.p0 = __builtin_amdgcn_readlane(L.context, at) - t.tokens;
    t.cuts = __builtin_amdgcn_readlane(L.cuts(len), at);
    const int rows = t.tokens * A.group;
    t.row0 = tile * kTileRows;
    t.count = min(rows - t.row0, rows <= kKeyRows ? kKeyRows : kTileRows);
    const int p_first = t.p0 + (int)A.by_group.quot(t.row0), p_last = t.p0 + (int)A.by_group.quot(t.row0 + t.count - 1);
    t.hi = min(p_last + 1, A.capacity);
    t.lo = min(first_key(p_first, A.window), max(0, t.hi));          // (a window may lie behind what the table has room for)
}
// keys of each piece of a tile, whole steps of 128
__device__ __forceinline__ int piece_keys(const AttnTile& t) { return ((max(0, t.hi - t.lo) + 127) / 128 + t.cuts - 1) / t.cuts * 128; }

__device__ __forceinline__ int64_t slot_row(const AttnArgs& A, int slot, int kvh, int row) { return ((int64_t)slot * A.cache.kv_heads + kvh) * A.slot_rows + row; }
__device__ __forceinline__ f2_t* states_of(const AttnArgs& A)
{
    return reinterpret_cast<f2_t*>(A.partial + (int64_t)A.slots * A.cache.kv_heads * A.slot_rows * A.cache.head_dim);
}
// behind the states: piece_steps, from the attention for the kernel that joins
__device__ __forceinline__ int* steps_of(const AttnArgs& A) { return reinterpret_cast<int*>(states_of(A) + (int64_t)A.slots * A.cache.kv_heads * A.slot_rows); }

// The idx-th piece from the end (the last tiles of a prompt have the most keys and go first); every wavefront looks for itself.
__device__ __forceinline__ bool find_piece(const Lens& H, const AttnArgs& A, int kv_heads, Worth least, int idx, AttnTile& t)
{
    Lanes L;
    const int len = piece_steps(H, kv_heads, least, L);
    if (H.pieces > 0 && blockIdx.x == 0 && idx == 0 && threadIdx.x == 0) *steps_of(A) = len;
    int cum = lane_scan(L.tiles * L.cuts(len)), total = __builtin_amdgcn_readlane(cum, 63);
    for (int s0 = 64; s0 < H.seqs; s0 += 64) {
        L.load(H, s0);
        total += lane_sum(L.tiles * L.cuts(len));
    }
    int want = total - 1 - idx, s0 = 0;
    if (want < 0) return false;
    t.slot = want;
    if (H.seqs > 64) L.load(H, 0);
    while (want >= __builtin_amdgcn_readlane(cum, 63)) {             // (fewer than the total)
        want -= __builtin_amdgcn_readlane(cum, 63);
        s0 += 64;
        L.load(H, s0);
        cum = lane_scan(L.tiles * L.cuts(len));
    }
    const int at = __ffsll((unsigned long long)__ballot(want < cum)) - 1;
    const int cuts = __builtin_amdgcn_readlane(L.cuts(len), at);
    want -= __builtin_amdgcn_readlane(cum, at) - __builtin_amdgcn_readlane(L.tiles, at) * cuts;
    set_tile(A, L, s0, at, want / cuts, len, t);
    const int keys = piece_keys(t), begin = t.lo + want % cuts * keys;
    t.hi = min(begin + keys, t.hi);
    t.lo = begin;
    return true;
}
// What a row's weighted values are multiplied by: 1 / (sum + the sink's weight), sum being counted in units of 2^unit; 1 / 0 never.  (The sink may be far
// above the units that m came down to.)
__device__ __forceinline__ float over_sum(const AttnArgs& A, float sum, float unit, int head)
{
    if (!(sum > 0.f)) return 0.f;
    if (!A.sinks) return 1.0f / sum;
    const float e = A.sinks[head] * kLog2e - unit, h = fmaxf(e, 0.f), by = __builtin_amdgcn_exp2f(-h);
    return by / (sum * by + (e > 0.f ? 1.f : __builtin_amdgcn_exp2f(e)));
}
// the tile of a row and head and its first piece; false: of no sequence
__device__ __forceinline__ bool find_row(const Lens& H, const AttnArgs& A, int row, int head, AttnTile& t, int* in_tile)
{
    const int len = *steps_of(A);
    Lanes L;
    int before = 0;
    for (int s0 = 0; s0 < H.seqs; s0 += 64) {
        L.load(H, s0);
        const int cum = lane_scan(L.tiles * L.cuts(len));
        const uint64_t has = __ballot(row >= L.start && row < L.start + L.n);
        if (has) {
            const int at = __ffsll((unsigned long long)has) - 1;
            const int cuts = __builtin_amdgcn_readlane(L.cuts(len), at);
            const int r = (row - __builtin_amdgcn_readlane(L.start, at)) * H.group + head % H.group;
            const int tile = __builtin_amdgcn_readlane(L.n, at) * H.group <= kKeyRows ? 0 : r / kTileRows;
            set_tile(A, L, s0, at, tile, len, t);
            t.slot = before + __builtin_amdgcn_readlane(cum, at) + (tile - __builtin_amdgcn_readlane(L.tiles, at)) * cuts;
            *in_tile = r - t.row0;
            return true;
        }
        before += __builtin_amdgcn_readlane(cum, 63);
    }
    return false;
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
// eight floats in fp16's range as twice eight fp16, both to nearest: what is left is below 2^-24 of each, or 2^-25 where that is more
__device__ __forceinline__ void cut2(const float (&x)[8], u4_t (&part)[2])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2_t hi = __builtin_convertvector((f2_t{x[2 * i], x[2 * i + 1]}), h2_t);
        const h2_t lo = __builtin_convertvector((f2_t{x[2 * i] - (float)hi[0], x[2 * i + 1] - (float)hi[1]}), h2_t);
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

template <int... I, typename F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f)
{
    (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each_of(F&& f)
{
    each_of(std::make_integer_sequence<int, N>(), f);
}

// TYPE: 0 fp32, 1 fp16, 2 bf16 cache; HD: head_dim rounded up to what the tiles are made for
template <int TYPE, int HD>
struct Attn {
    static constexpr int kElem = TYPE == 0 ? 4 : 2;
    static constexpr int kRow = HD * kElem, kPieces = kRow / 16;     // a key (value) in LDS, 16 bytes at a time
    static constexpr int kParts = TYPE == 1 ? 2 : 3;                 // of q and of the weights
    static constexpr int kCacheParts = TYPE == 0 ? 3 : 1;
    static constexpr int kSteps = HD / 16, kDims = HD / 32;
    // of the weights, as exponents (see above)
    static constexpr float kUnit = TYPE == 1 ? 15.f : 7.f, kRise = TYPE == 1 ? 0.f : 8.f, kAhead = TYPE == 1 ? 7.f : 0.f, kFall = 20.f, kApart = 20.f, kMost = 64.f;
    static constexpr int kWait = 16;
    static constexpr int NT = TYPE == 1 ? 2 : 1;                     // 32-key blocks of a step where wavefronts share the keys
    static constexpr bool kOneWave = HD > 128;     // registers for one workgroup per CU
    static constexpr bool kTight = HD == 256 || (TYPE == 0 && HD >= 128);
    static constexpr int kKeyWaves = key_waves_of(TYPE, HD);   // wavefronts that have keys of their own
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
    float c, m, l, l_rest;           // score to exponent, what weights are counted against, this lane's part of their sum and what its roundings left
    float low;                       // fp16: a step's largest score below this takes m with it
    int wait;                        // steps until it may
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
        lo = first_key(p, A.window);
        if (!live) src = reinterpret_cast<const float*>(g_zero_row);
        auto eight = [&](int s, float (&x)[8]) {
            const float* at = (16 * s < A.cache.head_dim ? src : reinterpret_cast<const float*>(g_zero_row)) + 16 * s + 8 * half;
            const f4_t a = *reinterpret_cast<const f4_t*>(at), b = *reinterpret_cast<const f4_t*>(at + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = a[i] * A.sign;
                x[4 + i] = b[i] * A.sign;
            }
        };
        c = A.c;
        int e = 0;
        // fp16: the row's largest is brought to 2^13 .. 2^14, so it is needed first; where the row does not fit beside its parts, it is read twice
        constexpr bool kTwice = TYPE == 1 && HD > 128;
        float all[kSteps][8];
        if constexpr (TYPE == 1) {
            float top = 0.f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                eight(s, all[s]);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(all[s][i]));
            }
            top = both_halves(top, larger);
            if (top > 0.f && top < INFINITY) e = 14 - __builtin_amdgcn_frexp_expf(top);
            c = ldexpf(A.c, -e);
            if constexpr (kTwice) asm volatile("" ::: "memory");
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            u4_t part[kParts];
            if constexpr (TYPE != 1 || kTwice) eight(s, all[s]);
            if constexpr (TYPE == 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) all[s][i] = ldexpf(all[s][i], e);
                cut2(all[s], part);
            } else {
                cut3(all[s], part);
            }
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                q[i][s] = part[i];
                // (large heads: what the accumulators of the result and of the scores leave of the accumulation registers holds rows, which the matrix
                // instruction reads there as well; left to itself the compiler spills to memory)
                if (kOneWave && kDims * 16 + 16 + (i + 1) * kSteps * 4 <= 256) asm volatile("" : "+a"(q[i][s]));
            }
        }
        no_rows();
    }
    // nothing seen yet
    __device__ __forceinline__ void no_rows()
    {
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
        m = low = -INFINITY;
        l = l_rest = 0.f;
        wait = 0;
        stay();
    }

    // ---- keys and values into LDS ----
    // Lane i has the id of page id_base + i; read again when a step passes the last of them.  (Held like this they cost a load
    // every 64 pages and no load beside the copies, whose waits count loads.)
    int ids, id_base = -64;
    __device__ __forceinline__ int page_id(int key, int end) const
    {
        const int id = __shfl(ids, (int)A.cache.page.quot((uint32_t)key) - id_base);
        return key < end && (uint32_t)id < (uint32_t)A.cache.num_pages ? id : -1;
    }
    // Where a row takes 8, 16 or 32 lanes of a copy, its address reaches them from a lane of the same 16 in a register permutation: a lane
    // finds the address of the row that its 16 lanes copy by number lane % 16 of the copies that its wavefront makes (copies wave,
    // wave + 4, .. where wavefronts share the keys).  In other cases lane i finds that of row i, and it goes through a shuffle.
    static constexpr bool kNear = kPieces == 8 || kPieces == 16 || kPieces == 32;
    template <bool SHARED>
    __device__ __forceinline__ int held_row(int wave) const
    {
        if constexpr (!kNear) return lane & (SHARED ? 32 * NT - 1 : 31);
        constexpr int kMine = SHARED ? NT * kCopies / kAttnWaves : kCopies;
        static_assert(!kNear || kMine <= (kPieces == 8 ? 8 : 16));
        const int j = lane & (kPieces == 8 ? 7 : 15) & (kMine - 1), n = SHARED ? wave + kAttnWaves * j : j, group = lane >> 4;
        return kPieces == 8 ? 8 * n + 2 * group + ((lane >> 3) & 1) : kPieces == 16 ? 4 * n + group : 2 * n + (group >> 1);
    }
    struct Rows {
        uint64_t k, v;               // addresses of a key and its value
        uint64_t there;              // which keys of the step are in the cache
    };
    // of the step from key0 on; keys from `end` on are not there
    template <bool SHARED>
    __device__ __forceinline__ Rows rows_of(int key0, int end, int wave)
    {
        constexpr int kKeys = SHARED ? 32 * NT : 32;
        const int first = (int)A.cache.page.quot((uint32_t)key0);   // uniform
        if ((int)A.cache.page.quot((uint32_t)(key0 + kKeys - 1)) - id_base >= 64) {
            id_base = first;
            ids = A.cache.table[t.seq * A.cache.table_stride + min(first + lane, A.cache.max_pages - 1)];
        }
        const int key = key0 + held_row<SHARED>(wave), id = page_id(key, end);
        const uint64_t there = __ballot((kNear ? page_id(key0 + (lane & (kKeys - 1)), end) : id) >= 0);
        const int within = key - (int)A.cache.page.quot((uint32_t)key) * (int)A.cache.page.d;
        const int64_t zero = (int64_t)(uintptr_t)g_zero_row;
        const int64_t k = (int64_t)(uintptr_t)A.cache.k + (id * A.cache.k_page + within * A.cache.k_token + kvh * A.cache.k_head) * kElem;
        const int64_t v = (int64_t)(uintptr_t)A.cache.v + (id * A.cache.v_page + within * A.cache.v_token + kvh * A.cache.v_head) * kElem;
        return {(uint64_t)(id >= 0 ? k : zero), (uint64_t)(id >= 0 ? v : zero), there};
    }
    // x of lane J of the 16 (rows of 8 lanes: of lane J for the lower eight, 8 + J for the upper)
    template <int J>
    __device__ __forceinline__ static uint32_t from_near(uint32_t x)
    {
        int r = __builtin_amdgcn_update_dpp(0, (int)x, 0x150 + J, 0xf, 0xf, true);
        if constexpr (kPieces == 8) r = __builtin_amdgcn_update_dpp(r, (int)x, 0x150 + 8 + J, 0xf, 0xc, false);
        return (uint32_t)r;
    }
    // the lane's number: where registers are short, what follows from it is worked out at every step
    __device__ __forceinline__ int lane_here() const
    {
        int ln = lane;
        if constexpr (kTight) asm volatile("" : "+v"(ln));
        return ln;
    }
    // copy n of a block, the wavefront's J-th: 64 pieces that follow one another in LDS
    template <bool V, int J>
    __device__ __forceinline__ void copy(uint64_t rows, int n, lds_t block, int ln) const
    {
        const int slot = n * 64 + ln, row = slot / kPieces, piece = (slot - row * kPieces) ^ (V ? v_swizzle(row) : k_swizzle(row));
        uint64_t at;
        if constexpr (kNear) at = (uint64_t)from_near<J>((uint32_t)(rows >> 32)) << 32 | from_near<J>((uint32_t)rows);
        else at = (uint64_t)__shfl((unsigned long long)rows, row);
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

    // S^T of 32 keys.  The products of an fp32 cache's parts below the first are summed apart from the large ones, which leaves a sixth of the roundings
    // at the size of the score: 2 rows at 7345 positions of 192 dimensions 5.1e-7 off, 1.0e-6 in one sum.  Up to 192 dimensions they have an accumulator
    // of their own; there are no registers for one beyond, and they go first, the keys being read a second time for the large ones (32 x 4096 positions of
    // 256 dimensions 675 us, a prompt of 1024 1005; with an accumulator of their own 60 to 90 registers are spilled, 777 and 950).
    __device__ __forceinline__ f16_t scores(lds_t block) const
    {
        constexpr bool kTwoSums = TYPE == 0 && HD <= 192, kTwoPasses = TYPE == 0 && HD > 192;
        f16_t s, below;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = below[i] = 0.f;
        const lds_t row = block + col * kRow;
        const int x = k_swizzle(col);
        // (the swizzle changes the lower bits of a piece's number only, so that one address serves every kAgain-th step)
        constexpr int kAgain = (kPieces % 8 == 0 ? 8 : 4) / (TYPE == 0 ? 4 : 2);
        auto eight = [&](int i, float (&v)[8]) {
            const int j = i % kAgain, further = (i - j) * 64;
            const u4_t a0 = read16(row + (((4 * j + 2 * half) ^ x) << 4) + further), a1 = read16(row + (((4 * j + 2 * half + 1) ^ x) << 4) + further);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                v[n] = __uint_as_float(a0[n]);
                v[4 + n] = __uint_as_float(a1[n]);
            }
        };
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            if constexpr (TYPE != 0) {
                const int j = i % kAgain, further = (i - j) * 32;
                const u4_t a = read16(row + (((2 * j + half) ^ x) << 4) + further);
#pragma unroll
                for (int n = 0; n < kParts; ++n) s = mfma(a, q[n][i], s);
            } else {
                step_here();
                float v[8];
                eight(i, v);
                u4_t a[3];
                cut3(v, a);
                f16_t& small = kTwoSums ? below : s;
                small = mfma(a[2], q[0][i], small);
                small = mfma(a[1], q[1][i], small);
                small = mfma(a[0], q[2][i], small);
                small = mfma(a[1], q[0][i], small);
                small = mfma(a[0], q[1][i], small);
                if constexpr (kTwoSums) s = mfma(a[0], q[0][i], s);
            }
        }
        if constexpr (kTwoSums) s += below;
        if constexpr (kTwoPasses) {
            asm volatile("" ::: "memory");                           // (the parts of all steps do not fit)
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                step_here();
                float v[8];
                eight(i, v);
                const u4_t a = {high_halves(v[0], v[1]), high_halves(v[2], v[3]), high_halves(v[4], v[5]), high_halves(v[6], v[7])};
                s = mfma(a, q[0][i], s);
            }
        }
        return s;
    }
    // Where registers are short, a step's reads stay behind the step before.  No instantiation may spill vector registers: of a spilled operand the
    // compiler has brought back three of the four registers (of a second part of q, results 2e-3 off).
    __device__ __forceinline__ static void step_here()
    {
        if constexpr (TYPE == 0 && HD == 128) __builtin_amdgcn_sched_barrier(0);
    }
    // Of the 16 scores of a lane number i belongs to key 8 (i / 4) + 4 half + i % 4 of the block.
    __device__ __forceinline__ void mask(f16_t& s, int key0, uint64_t there) const
    {
        const int below = 4 * (lane_here() >> 5);
        const uint32_t bits = (uint32_t)(there >> below);
        const int last = p - key0 - below, first = lo - key0 - below;
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
        const bool above = top > m + kRise, below = TYPE == 1 && wait <= 0 && top < low && top > -INFINITY;
        --wait;
        if (__any(above || below)) {                                 // (m starts at -infinity)
            float mn = m;
            if (above) mn = __builtin_ceilf(top) + kAhead;
            if constexpr (TYPE == 1) {
                // (all but one or two of the step's scores are below `others` if that is below them: the lower of the maxima of eight and of eight others)
                const f16_t& x = s[0];
                const float some = fmaxf(fmaxf(x[1], x[6]), fmaxf(x[11], x[12])), more = fmaxf(fmaxf(x[3], x[4]), fmaxf(x[9], x[14]));
                const float others = fminf(both_halves(some, larger), both_halves(more, larger)) * c;
                if (above && top - others > kApart) mn = __builtin_ceilf(top);
                if (above) low = mn - kFall;
                if (__any(below)) {
                    // (not so far down that the sum passes 2^kMost: with values up to 2^16 the accumulators stay finite)
                    const float least = m - fmaxf(0.f, kMost - (float)__builtin_amdgcn_frexp_expf(both_halves(l, larger)));
                    wait = kWait;
                    if (below) {
                        mn = __builtin_ceilf(top) + kAhead;
                        low = mn < least ? -INFINITY : mn - kFall;
                        mn = fmaxf(mn, least);
                    }
                }
            }
            const float f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            l *= f;
            l_rest *= f;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= f;
            m = mn;
        }
        stay();
    }
    // large heads: the accumulators stay in accumulation registers from one step to the next
    __device__ __forceinline__ void stay()
    {
        if constexpr (kOneWave) {
#pragma unroll
            for (int d = 0; d < kDims; ++d) asm volatile("" : "+a"(o[d]));
        }
    }
    // Whether one of the wavefront's rows has an infinity or NaN in its result.  The matrix instruction brings those of values to rows that do
    // not see them, and an infinity meets the zero parts of what is cut; either leaves NaN (0 x infinity) that stays, so it is looked for at
    // the end, and such rows are done again by plainly().
    __device__ __forceinline__ bool odd_result(int row) const
    {
        float z = 0.f;                                               // (a chain: a tree of comparisons takes registers from the loop)
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) z = __builtin_fmaf(o[d][i], 0.f, z);
        return __any(row < t.count && z != z);
    }
    // The sum of the weights goes over all keys of a row, one step after the other.  Small weights beside a large sum lose the same bits at every step
    // (4096 keys 16 e-folds below the first one: 4e-4 of the sum), so what each addition rounds away is kept and added at the end.
    __device__ __forceinline__ void add_weights(float sum)
    {
        const float large = fmaxf(l, sum), small = fminf(l, sum);
        l = large + small;
        l_rest += small - (l - large);
    }
    // weights of a block's scores, and O^T += V^T P^T; returns their sum
    __device__ __forceinline__ float weigh(const f16_t& s, lds_t block)
    {
        float sum = 0.f;
        const float bias = kUnit - (m == -INFINITY ? 0.f : m);
        const int x = v_swizzle((lane & 15) >> 2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                                // 16 keys
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * h + i], c, bias));
                sum += w[i];
            }
            u4_t part[kParts];
            if constexpr (TYPE == 1) cut2(w, part);
            else cut3(w, part);
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                step_here();
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
        return sum;
    }

    // ---- where a row's state goes ----
    __device__ __forceinline__ float* values_of(int row) const { return A.partial + slot_row(A, t.slot, kvh, row) * A.cache.head_dim; }
    __device__ __forceinline__ f2_t* state_of(int row) const { return states_of(A) + slot_row(A, t.slot, kvh, row); }
    // Rows of the tile (piece) again, each over the keys that it sees and no others: a lane per key for the scores, a lane per dimension (of
    // 64) for the values, whose mean is carried along, so that finite values never add up to infinity.  Slow, for rows with infinities or NaN in their results.
    __device__ __forceinline__ void plainly(int row, int step)
    {
        const int dim = A.cache.head_dim;
        for (int n = 0; n < 32 && row < t.count; ++n, row += step) {
            int token, head;
            place(row, &token, &head);
            const float* src = A.query + (int64_t)(t.first + token) * A.ld_query + (int64_t)head * dim;
            const int last = t.p0 + token, first = first_key(last, A.window);
            float top = -INFINITY, sum = 0.f, mean[HD / 64 + 1] = {};
            for (int j0 = t.lo; j0 < t.hi; j0 += 64) {
                const int j = j0 + lane;
                int id = -1;
                if (j < t.hi && j >= first && j <= last) id = A.cache.table[t.seq * A.cache.table_stride + (int)A.cache.page.quot((uint32_t)j)];
                const bool seen = (uint32_t)id < (uint32_t)A.cache.num_pages;
                const uint64_t lanes = __ballot(seen);
                if (lanes == 0) continue;
                const int within = j - (int)A.cache.page.quot((uint32_t)j) * (int)A.cache.page.d;
                const int64_t v_at = seen ? id * A.cache.v_page + within * A.cache.v_token + kvh * A.cache.v_head : 0;
                float score = -INFINITY;
                if (seen) {
                    const int64_t k_at = id * A.cache.k_page + within * A.cache.k_token + kvh * A.cache.k_head;
                    float dot = 0.f;
                    for (int d = 0; d < dim; ++d) dot += src[d] * A.sign * element(A.cache.k, k_at + d);
                    score = dot * A.c;
                }
                float most = score;
                for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
                const float mn = fmaxf(top, __builtin_ceilf(most)), base = mn == -INFINITY ? 0.f : mn, f = __builtin_amdgcn_exp2f(top - base);
                const float w = seen ? __builtin_amdgcn_exp2f(score - base) : 0.f;
                float all = w;
                for (int o = 32; o > 0; o >>= 1) all += __shfl_xor(all, o);
                const float before = sum * f;
                sum = before + all;
                top = mn;
                const float by = sum == 0.f ? 0.f : 1.0f / sum;      // (weights of 0 alone: nothing; NaN stays)
#pragma unroll
                for (int i = 0; i <= HD / 64; ++i) mean[i] *= before * by;
                for (uint64_t rest = lanes; rest != 0; rest &= rest - 1) {
                    const int at = __ffsll((unsigned long long)rest) - 1;
                    const float wk = __shfl(w, at) * by;
                    const int64_t vk = (int64_t)__shfl((long long)v_at, at);
#pragma unroll
                    for (int i = 0; i <= HD / 64; ++i)
                        if (64 * i + lane < dim) mean[i] += wk * element(A.cache.v, vk + 64 * i + lane);
                }
            }
            // a piece's state in units in which its sum is at most 1
            const int e = sum > 0.f ? __builtin_amdgcn_frexp_expf(sum) : 0;
            const float part = ldexpf(sum, -e);
            float* dst = t.cuts == 1 ? A.out + (int64_t)(t.first + token) * A.ld_out + (int64_t)head * dim : values_of(row);
            const float by = t.cuts == 1 ? sum * over_sum(A, sum, top, head) : part;
#pragma unroll
            for (int i = 0; i <= HD / 64; ++i)
                if (64 * i + lane < dim) dst[64 * i + lane] = mean[i] * by;
            if (t.cuts > 1 && lane == 0) *state_of(row) = f2_t{top + (float)e, part};
        }
    }
    __device__ __forceinline__ float element(const char* base, int64_t at) const
    {
        if constexpr (TYPE == 0) return reinterpret_cast<const float*>(base)[at];
        else if constexpr (TYPE == 1) return __half2float(reinterpret_cast<const __half*>(base)[at]);
        else return __bfloat162float(reinterpret_cast<const __hip_bfloat16*>(base)[at]);
    }

    // all wavefronts over the same keys, 32 rows each (the return of both: whether these, of own_keys() all, have to be done by plainly())
    __device__ __forceinline__ bool shared_keys()
    {
        const int begin = t.lo, end = t.hi;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int p_first = t.p0 + (int)A.by_group.quot(t.row0 + min(32 * wave, t.count - 1));
        const int p_last = t.p0 + (int)A.by_group.quot(t.row0 + min(32 * wave + 31, t.count - 1));
        const int lo_last = first_key(p_last, A.window);
        constexpr int kKeys = 32 * NT, kMine = (NT * kCopies + kAttnWaves - 1) / kAttnWaves;
        auto stage = [&](const Rows& r, lds_t buffer) {
            const int ln = lane_here();
            each_of<kMine>([&](auto j) {
                constexpr int J = decltype(j)::value;
                const int n = wave + kAttnWaves * J;
                if (NT * kCopies % kAttnWaves == 0 || n < NT * kCopies) {
                    copy<false, J>(r.k, n, buffer, ln);
                    copy<true, J>(r.v, n, buffer + NT * kBlock, ln);
                }
            });
        };
        int buffer = 0;
        if (begin < end) {
            // copies go a step ahead; those behind the last key bring zeros that nothing reads
            Rows rows = rows_of<true>(begin, end, wave);
            stage(rows, lds);
            load_rows(32 * wave + col);                              // (while the first keys are on their way)
            for (int key0 = begin; key0 < end; key0 += kKeys) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                const lds_t here = lds + buffer * (2 * NT * kBlock);
                const uint64_t there = rows.there;
                buffer ^= 1;
                rows = rows_of<true>(key0 + kKeys, end, wave);
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
                    float sum = 0.f;
#pragma unroll
                    for (int b = 0; b < NT; ++b) sum += weigh(s[b], here + (NT + b) * kBlock);
                    add_weights(sum);
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the last copies, before this LDS may be another workgroup's
        } else {
            no_rows();
        }
        const int row = 32 * wave + (lane_here() & 31);
        if (odd_result(row)) return true;
        l = both_halves(l + l_rest, added);
        if (row >= t.count) return false;
        int token, head;
        place(row, &token, &head);
        float* dst;
        float by = 1.f;
        if (t.cuts == 1) {
            dst = A.out + (int64_t)(t.first + token) * A.ld_out + (int64_t)head * A.cache.head_dim;
            by = over_sum(A, l, m - kUnit, head);
        } else {
            dst = values_of(row);
            if (half == 0) *state_of(row) = f2_t{m - kUnit, l};
        }
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 32 * d + 8 * i + 4 * half;
                if (at < A.cache.head_dim)
                    *reinterpret_cast<f4_t*>(dst + at) = f4_t{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * by;
            }
        return false;
    }

    // every wavefront over keys of its own, the same (up to 32) rows
    __device__ __forceinline__ bool own_keys()
    {
        const int begin = t.lo, end = t.hi;
        __shared__ f2_t states[kAttnWaves][32];
        __shared__ int odd[kAttnWaves];
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int p_last = t.p0 + t.tokens - 1;
        const int lo_last = first_key(p_last, A.window);
        const lds_t kb = lds + wave * 2 * kBlock, vb = kb + kBlock;
        int key0 = begin + 32 * wave;
        constexpr int kStride = 32 * kKeyWaves;
        if (wave < kKeyWaves && key0 < end) {
            auto stage = [&](auto is_v, uint64_t rows, lds_t block) {
                const int ln = lane_here();
                each_of<kCopies>([&](auto n) { copy<decltype(is_v)::value, decltype(n)::value>(rows, decltype(n)::value, block, ln); });
            };
            Rows rows = rows_of<false>(key0, end, wave);
            stage(std::false_type(), rows.k, kb);
            stage(std::true_type(), rows.v, vb);
            load_rows(col);                                          // (while the first keys are on their way)
            for (; key0 < end; key0 += kStride) {
                // loads answer in order: with kCopies of them left, the values behind the keys, the keys have arrived
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCopies) : "memory");
                f16_t s[1] = {scores(kb)};
                const uint64_t there = rows.there;
                rows = rows_of<false>(key0 + kStride, end, wave);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                stage(std::false_type(), rows.k, kb);
                if (~there != 0 || key0 + 31 > t.p0 || key0 < lo_last) mask(s[0], key0, there);
                follow_maximum(s, 1);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCopies) : "memory");                 // the values too: the next keys are left
                add_weights(weigh(s[0], vb));
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                stage(std::true_type(), rows.v, vb);
            }
        }
        else {
            no_rows();
        }
        l = both_halves(l + l_rest, added);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (wave < kKeyWaves) {
            if (const bool found = odd_result(col); lane == 0) odd[wave] = found;
            if (half == 0) states[wave][col] = f2_t{m - kUnit, l};
            const lds_t row = lds + (wave * 32 + col) * HD * 4;
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<__attribute__((address_space(3))) f4_t*>(row + (((8 * d + 2 * i + half) ^ (col & 7)) << 4)) =
                        f4_t{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
        }
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int w = 0; w < kKeyWaves; ++w) any |= odd[w];
        if (__builtin_amdgcn_readfirstlane(any)) return true;
        const int pieces = A.cache.head_dim / 4;
        for (int i = threadIdx.x; i < t.count * pieces; i += kAttnThreads) {
            const int row = i / pieces, piece = i - row * pieces;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kKeyWaves; ++w) top = fmaxf(top, states[w][row].x);
            // (two powers more, so that what up to four of them have adds up to no infinity)
            const float unit = top + 2.f, base = top == -INFINITY ? 0.f : unit;
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
            if (t.cuts == 1) {
                *reinterpret_cast<f4_t*>(A.out + (int64_t)(t.first + token) * A.ld_out + (int64_t)head * A.cache.head_dim + 4 * piece) =
                    v * over_sum(A, sum, unit, head);
            } else {
                *reinterpret_cast<f4_t*>(values_of(row) + 4 * piece) = v;
                if (piece == 0) *state_of(row) = f2_t{unit, sum};
            }
        }
        return false;
    }
};

// grid (KV heads, pieces)
template <int TYPE, int HD>
__global__ void __launch_bounds__(kAttnThreads, (Attn<TYPE, HD>::kOneWave ? 1 : 2)) paged_attention_kernel(TSHIP_LENS_ARGS, const AttnArgs A)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int kvh = blockIdx.x, idx = blockIdx.z * gridDim.y + blockIdx.y;
    AttnTile t;
    if (!find_piece(TSHIP_LENS, A, gridDim.x, worth_of(TYPE, HD, key_waves_of(TYPE, HD)), idx, t)) return;
    Attn<TYPE, HD> a(A, t, kvh, (lds_t)smem);
    const bool own = t.tokens * A.group <= kKeyRows;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (own ? a.own_keys() : a.shared_keys()) a.plainly(own ? wave : 32 * wave, own ? kAttnWaves : 1);
}

__host__ __device__ constexpr int wide_of(int dim) { return dim <= 64 ? 16 : dim <= 128 ? 32 : 64; }

// The pieces of a row's tile, for one head.  A head takes 16, 32 or 64 lanes.  WAVES 1, where there are many rows: grid (KV heads, wavefronts / 4),
// a wavefront has a row's heads of one KV head, the lanes side by side different ones, and goes through all pieces.  (KV heads lead in both kernels'
// grids: with 8 of them a piece is read on the die whose cache it was written through.)  WAVES 4: grid (rows, heads), the lanes side by side and the
// wavefronts have different pieces.  Bound: the way from the lengths to the states, then memory (512 rows of 32 heads of 128 in 4 pieces, 34 MB: 9.7
// us; 11.0 with rows leading).
template <int WAVES>
__global__ void __launch_bounds__(kAttnThreads) paged_combine_kernel(TSHIP_LENS_ARGS, const AttnArgs A)
{
    __shared__ f2_t sums[kAttnWaves];
    __shared__ f4_t values_in[kAttnWaves][kMaxDim / 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), dim = A.cache.head_dim;
    const int wide = wide_of(dim), d = 4 * (lane & (wide - 1)), parts = 64 / wide, part = lane / wide;
    int row, head;
    bool mine = d < dim;
    if constexpr (WAVES == 1) {
        const int chunks = (A.group + parts - 1) / parts, at = blockIdx.y * kAttnWaves + wave;
        row = at / chunks;
        const int in_group = at % chunks * parts + part;
        if (row >= A.rows) return;
        mine = mine && in_group < A.group;
        head = blockIdx.x * A.group + min(in_group, A.group - 1);
    } else {
        row = blockIdx.x;
        head = blockIdx.y;
    }
    AttnTile t;
    int in_tile;
    if (!find_row(TSHIP_LENS, A, row, head, t, &in_tile) || t.cuts == 1) return;      // (the same for all heads of a row)
    const int cuts = t.cuts, step = WAVES == 1 ? 1 : WAVES * parts;
    const int64_t first = slot_row(A, t.slot, head / A.group, in_tile), next = (int64_t)A.cache.kv_heads * A.slot_rows;
    const float* values = A.partial + first * dim;
    const f2_t* states = states_of(A) + first;
    constexpr int U = WAVES == 1 ? 8 : 4;
    // (a piece's values may be as large as fp32 is: what is joined counts in units of 2^(top + kSpare), which leave room for kMaxPieces of them)
    constexpr float kSpare = 10.f;
    static_assert(kMaxPieces <= 1 << (int)kSpare);
    f4_t acc = {0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, sum = 0.f;
    auto join = [&](float t, float w, const f4_t& v, float spare) {
        const float m = fmaxf(top, t), base = m == -INFINITY ? 0.f : m;
        const float f = __builtin_amdgcn_exp2f(top - base), g = __builtin_amdgcn_exp2f(t - base - spare);
        sum = sum * f + w * g;
        acc = acc * f + v * g;
        top = m;
    };
    for (int s0 = WAVES == 1 ? 0 : wave * parts + part; s0 < cuts; s0 += U * step) {
        f2_t st[U];
        f4_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(s0 + u * step, cuts - 1);
            st[u] = states[s * next];
            v[u] = mine ? *reinterpret_cast<const f4_t*>(values + s * next * dim + d) : f4_t{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u * step < cuts) join(st[u].x, st[u].y, v[u], kSpare);
    }
    if constexpr (WAVES > 1) {
        for (int o = wide; o < 64; o <<= 1) {
            const float t = __shfl_xor(top, o), w = __shfl_xor(sum, o);
            f4_t v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __shfl_xor(acc[i], o);
            join(t, w, v, 0.f);
        }
        if (lane == 0) sums[wave] = f2_t{top, sum};
        if (lane < wide) values_in[wave][lane] = acc;
        __syncthreads();
        if (wave > 0 || lane >= wide) return;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) join(sums[w].x, sums[w].y, values_in[w][lane], 0.f);
    }
    if (!mine) return;
    *reinterpret_cast<f4_t*>(A.out + (int64_t)row * A.ld_out + (int64_t)head * dim + d) = acc * over_sum(A, sum, top + kSpare, head);
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
    const int group = heads / cache.kv_heads, dim = cache.head_dim;
    const int64_t all = (int64_t)rows * group;
    PagedAttnPlan plan{};
    // (a sequence of at most 32 rows has one tile, others a tile per 128 rows begun: no more than this, whatever the lengths)
    const int64_t tiles = all / kTileRows + std::min<int64_t>(cache.seqs, rows);
    // workgroups that are resident at once
    const int at_once = device_info().num_cus * (dim <= 64 && cache.element_type != kTypeF32 ? 3 : dim <= 128 ? 2 : 1);
    const int64_t pieces = std::min(kMaxPieces, std::max(1, at_once / cache.kv_heads)), keys = (int64_t)cache.max_pages * cache.page.d;
    const int64_t most = std::min<int64_t>(keys, window > 0 ? window : keys);
    const int hd = dims_of(dim);
    const Worth least = worth_of(cache.element_type, hd, key_waves_of(cache.element_type, hd));
    const bool cut = (all + kTileRows - 1) / kTileRows < pieces &&
        most > 128 * (all > (int64_t)kKeyRows * cache.seqs                                 ? std::min(least.few, least.tall)
                      : std::min<int64_t>(cache.seqs, rows) * cache.kv_heads >= 64 ? least.many
                                                                                   : least.few);
    plan.pieces = cut ? (int)pieces : 0;
    plan.slots = (int)std::min<int64_t>(INT32_MAX, cut ? std::max(tiles, pieces) : tiles);
    plan.slot_rows = all <= kKeyRows ? kKeyRows : kTileRows;
    // (a tile that is cut is one of at most `pieces` pieces)
    if (cut) plan.ws_bytes = (size_t)pieces * cache.kv_heads * plan.slot_rows * (dim + 2) * sizeof(float) + sizeof(int);
    return plan;
}

template <int TYPE, int HD>
static bool launch_attention(const Lens& H, const AttnArgs& args, const dim3& grid, hipStream_t stream)
{
    const auto kern = paged_attention_kernel<TYPE, HD>;
    constexpr size_t lds = Attn<TYPE, HD>::kLds;
    if (!raise_lds_limit(reinterpret_cast<const void*>(kern), lds)) return false;
    hipLaunchKernelGGL(kern, grid, dim3(kAttnThreads), lds, stream, H.row_starts, H.context_lens, H.seqs, H.rows, H.group, H.window, H.pieces, H.capacity, args);
    return hip_ok(hipGetLastError(), "paged attention launch");
}
template <int TYPE>
static bool launch_attention(const Lens& H, const AttnArgs& args, const dim3& grid, hipStream_t stream)
{
    switch (dims_of(args.cache.head_dim)) {
    case 64: return launch_attention<TYPE, 64>(H, args, grid, stream);
    case 96: return launch_attention<TYPE, 96>(H, args, grid, stream);
    case 128: return launch_attention<TYPE, 128>(H, args, grid, stream);
    case 192: return launch_attention<TYPE, 192>(H, args, grid, stream);
    default: return launch_attention<TYPE, 256>(H, args, grid, stream);
    }
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
    args.group = heads / cache.kv_heads;
    args.window = window;
    args.capacity = cache.max_pages * (int)cache.page.d;
    args.slots = plan.pieces;
    args.slot_rows = plan.slot_rows;
    args.by_group = FastDiv((uint32_t)args.group);
    args.cache = cache;
    if ((int64_t)plan.slots * cache.kv_heads > INT32_MAX || (int64_t)rows * args.group > INT32_MAX) {
        set_last_error("paged_attention: too many rows for one call.");
        return false;
    }
    const Lens H{cache.row_starts, cache.context_lens, cache.seqs, rows, args.group, window, plan.pieces, args.capacity};
    const unsigned layers = (plan.slots + 65534u) / 65535u;
    const dim3 grid(cache.kv_heads, (plan.slots + layers - 1) / layers, layers);
    bool ok;
    switch (cache.element_type) {
    case kTypeF32: ok = launch_attention<0>(H, args, grid, stream); break;
    case kTypeF16: ok = launch_attention<1>(H, args, grid, stream); break;
    default: ok = launch_attention<2>(H, args, grid, stream); break;
    }
    if (!ok || plan.pieces == 0) return ok;
    if ((int64_t)rows * heads <= 8 * device_info().num_cus) {
        hipLaunchKernelGGL(paged_combine_kernel<kAttnWaves>, dim3(rows, heads), dim3(kAttnThreads), 0, stream, H.row_starts, H.context_lens, H.seqs, H.rows, H.group, H.window,
                           H.pieces, H.capacity, args);
    } else {
        const int parts = 64 / wide_of(cache.head_dim), waves = rows * ((args.group + parts - 1) / parts);
        hipLaunchKernelGGL(paged_combine_kernel<1>, dim3(cache.kv_heads, (waves + kAttnWaves - 1) / kAttnWaves), dim3(kAttnThreads), 0, stream, H.row_starts, H.context_lens,
                           H.seqs, H.rows, H.group, H.window, H.pieces, H.capacity, args);
    }
    return hip_ok(hipGetLastError(), "paged attention combine launch");
}

}  // namespace tship
