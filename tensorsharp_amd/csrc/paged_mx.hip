// Attention over a paged cache in four bits (MXFP4: blocks of 32 along a head).
//
// The tiles, pieces and states are those of the attention over caches of 16 and 32 bits (paged_tiles.h), and so are the products' order, S^T = K Q^T and
// O^T += V^T P^T, and what weights are counted against.  What differs follows from the block format:
//
// * K goes into the block-scaled matrix instruction as it is: a lane's operand is one block, 16 bytes of codes and the power as the operand's scale, loaded
//   from memory into the registers that the instruction reads.  Nothing is unpacked.  A row of Q is cut into kParts terms of fp6 (E2M3, four significant bits) in
//   blocks of 32 with a power of its own each, the next one from what rounding left, so that five of them hold 22 bits and more of the block's largest.  A
//   term takes a quarter of the time of one in 16 bits: 5 / 4 of a product in 16 bits, where the exact values in bf16 would take three, and their unpacking.
// * V's blocks lie along its dimensions, but O^T adds over keys, along which the powers differ: there is no such operand.  A lane turns one block into bf16 (exact:
//   two significant bits and the power) with the instruction that converts two codes at a time, through LDS, from which the operand is read transposed.
//   Weights go in as three parts of bf16, 24 bits.
//
// Bound: answers by memory (32 sequences of 4096 to 16384 positions, 8 KV heads of 128: 305 MB in 70 us, 4.4 TB/s, of which 7 are a workgroup's start - lengths, pages, first
// keys, one trip after the other - and 5 more the join; one answer of 4001 positions 11 us and 4).  Prompts by vector instructions - weights, their cutting, values to
// bf16 - beside the matrix instructions, which are busy half of the time (509 tokens of 32 heads over 4096 positions: 80 us and 10 for the join; the products alone take 58).
#include "tship_internal.h"
#include "mx4.h"
#include "paged_tiles.h"

namespace tship {
namespace {

typedef int i8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u6_t __attribute__((ext_vector_type(6)));
typedef float v32_t __attribute__((ext_vector_type(32)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));

constexpr int kParts = 5;

// 32 floats of a row as fp6 terms with a power each (biased; byte i of scale[i / 4])
struct Terms {
    u6_t t[kParts];
    uint32_t scale[2];
};
// The least power of which the largest magnitude is at most 7.5, the last fp6 value; at least 2^-126, 255 for infinities and NaN.
__device__ __forceinline__ uint32_t fp6_power(uint32_t top)
{
    if (top >= 0x7f800000u) return 255;
    const int e = (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x700000u ? 1 : 0);
    return e < 1 ? 1u : (uint32_t)e;
}
__device__ __forceinline__ void cut_terms(f16_t a, f16_t b, Terms& out)      // a: the even ones, b: the odd ones
{
    out.scale[0] = out.scale[1] = 0;
#pragma unroll
    for (int n = 0; n < kParts; ++n) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max(top, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
        const uint32_t e = fp6_power(top);
        const float by = __uint_as_float(e == 255 ? 127u << 23 : e << 23);
        out.t[n] = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(a, b, by);
        // (The conversion writes its first results before it has read its last values, so that these may not share registers, which the compiler would have them do where
        // a and b are of no further use: now and then the last term of 96 dimensions came out another.)
        asm volatile("" ::"v"(out.t[n]), "v"(a), "v"(b), "v"(by));
        out.scale[n / 4] |= e << (8 * (n % 4));
        if (n + 1 < kParts) {
            const v32_t back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(out.t[n], by);
            asm volatile("" ::"v"(back), "v"(out.t[n]), "v"(by));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                a[i] -= back[2 * i];
                b[i] -= back[2 * i + 1];
            }
        }
    }
}
__device__ __forceinline__ i8_t operand(const u4_t& x) { return i8_t{(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0}; }
__device__ __forceinline__ i8_t operand(const u6_t& x) { return i8_t{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)x[4], (int)x[5], 0, 0}; }

// a block of codes with its power as 32 bf16 values, 16 bytes at a time
__device__ __forceinline__ u4_t as_bf16(uint32_t codes, float scale)
{
    u4_t r;
    r[0] = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, (b2_t)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    return r;
}

typedef __attribute__((address_space(3))) u4_t* lds4_t;
typedef const __attribute__((address_space(1))) uint8_t* mem_t;      // (a generic pointer's loads would be counted with LDS)
typedef const __attribute__((address_space(1))) u4_t* mem4_t;

// HD: head_dim rounded up to what the tiles are made for
template <int HD>
struct AttnMx {
    static constexpr int kBlocks = HD / 32;                          // of a key (value)
    static constexpr float kUnit = 7.f, kRise = 8.f;                 // weights begin at 2^7, m follows a score 2^8 above it
    // A value in LDS has 32 bytes behind it: what a transposed read takes at a time is 32 bytes of each of eight keys, which then lie in different banks.
    static constexpr int kRow = HD * 2 + 32;
    static constexpr int kOwnLds = kAttnWaves * 32 * kRow;           // of wavefronts that have keys of their own
    static_assert(32 * kRow >= 16 * HD * 4, "the states take the place of the values");
    static constexpr int NB = HD > 192 ? 1 : 2, kKeys = 32 * NB;     // 32-key blocks of a step where wavefronts share the keys: as many as registers hold
    static constexpr int kSharedLds = 2 * kKeys * kRow;
    static constexpr int kLds = kOwnLds > kSharedLds ? kOwnLds : kSharedLds;

    const AttnArgs& A;
    const MxScales& X;
    const AttnTile t;
    const int kvh, thread, lane, wave;
    lds_t lds;

    __device__ __forceinline__ AttnMx(const AttnArgs& args, const MxScales& scales, const AttnTile& tile, int kv_head, int thread_id, lds_t smem)
        : A(args), X(scales), t(tile), kvh(kv_head), thread(thread_id), lane(thread_id & 63), wave(__builtin_amdgcn_readfirstlane(thread_id >> 6)), lds(smem)
    {
    }

    __device__ __forceinline__ void place(int row, int* token, int* head) const
    {
        const int r = t.row0 + row, i = (int)A.by_group.quot(r);
        *token = i;
        *head = kvh * A.group + (r - i * A.group);
    }
    __device__ __forceinline__ float* values_of(int row) const { return A.partial + slot_row(A, t.slot, kvh, row) * A.cache.head_dim; }
    __device__ __forceinline__ f2_t* state_of(int row) const { return states_of(A) + slot_row(A, t.slot, kvh, row); }
    __device__ __forceinline__ int blocks() const { return A.cache.head_dim / 32; }

    // Block `block` of a row of the tile, even and odd dimensions apart as the conversion takes them; rows and blocks that are not there are zero.  (Loaded ahead of
    // keys and values and cut behind them, while they are on their way: loads answer in order.)
    struct RowBlock {
        f16_t a, b;
    };
    __device__ __forceinline__ void load_row(int row, int block, RowBlock& x) const
    {
        const bool live = row < t.count && block < blocks();
        int token, head;
        place(row < t.count ? row : 0, &token, &head);
        const float* src = live ? A.query + (int64_t)(t.first + token) * A.ld_query + (int64_t)head * A.cache.head_dim + 32 * block : reinterpret_cast<const float*>(g_zero_row);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const f4_t v = *(const __attribute__((address_space(1))) f4_t*)(uint64_t)(uintptr_t)(src + 4 * i);
            x.a[2 * i] = v[0], x.b[2 * i] = v[1], x.a[2 * i + 1] = v[2], x.b[2 * i + 1] = v[3];
        }
    }
    __device__ __forceinline__ void cut_row(const RowBlock& x, Terms& out) const { cut_terms(x.a * A.sign, x.b * A.sign, out); }

    // ---- where keys lie ----
    // Lane i has the id of page id_base + i of the sequence: read again when a step passes the last of them, so that no step's loads wait for a
    // table's (loads are waited for in order, with everything before them).
    int ids, id_base = -64;
    __device__ __forceinline__ void bring_pages(int p0, int keys)
    {
        const int page = (int)A.cache.page.quot((uint32_t)p0);       // uniform
        // (what follows the first positions may begin before the end of their last step)
        if (page < id_base || (int)A.cache.page.quot((uint32_t)(p0 + keys - 1)) - id_base >= 64) {
            id_base = page;
            ids = A.cache.table[t.seq * A.cache.table_stride + min(page + lane, A.cache.max_pages - 1)];
            asm volatile("" : "+v"(ids));                            // (it is waited for here, and nowhere else)
        }
    }
    // The row at a position that is among those pages.  One that is not there is a row of page 0: its codes may be any, so what is loaded of it counts
    // with a power that makes it nothing.
    struct Row {
        uint32_t page, within;
        bool there;
    };
    __device__ __forceinline__ Row row_at(int p, int end) const
    {
        const int q = (int)A.cache.page.quot((uint32_t)p), id = __shfl(ids, q - id_base);
        const bool there = p < end && (uint32_t)id < (uint32_t)A.cache.num_pages;
        return {there ? (uint32_t)id : 0u, (uint32_t)(p - q * (int)A.cache.page.d), there};
    }
    // Where rows lie: pages and tokens are below 2^32 bytes apart, so that each is one multiplication, and mostly one serves codes and scales of keys and values
    // (X.alike: a row has 16 bytes of codes for one of scales, so their strides are 16 times those of scales where both are dense).
    struct Place {
        uint64_t k, v, ks, vs;                                       // bytes from a head's first row
    };
    template <bool ALIKE>
    __device__ __forceinline__ Place place_of(const Row& r) const
    {
        auto at = [&](int64_t page, int64_t token) { return (uint64_t)r.page * (uint32_t)page + (uint64_t)r.within * (uint32_t)token; };
        const uint64_t k = at(A.cache.k_page, A.cache.k_token);
        if constexpr (ALIKE) return {k, k, k >> 4, k >> 4};
        return {k, at(A.cache.v_page, A.cache.v_token), at(X.k_page, X.k_token), at(X.v_page, X.v_token)};
    }
    __device__ __forceinline__ uint32_t block_of(int block) const { return min(block, blocks() - 1); }
    __device__ __forceinline__ uint64_t keys() const { return (uint64_t)(uintptr_t)A.cache.k + kvh * A.cache.k_head; }
    __device__ __forceinline__ uint64_t values() const { return (uint64_t)(uintptr_t)A.cache.v + kvh * A.cache.v_head; }
    __device__ __forceinline__ uint64_t key_scales() const { return (uint64_t)(uintptr_t)X.k + kvh * X.k_head; }
    __device__ __forceinline__ uint64_t value_scales() const { return (uint64_t)(uintptr_t)X.v + kvh * X.v_head; }

    // ---- infinities and NaN ----
    // an eighth of an element: fp32 holds that of all, whose powers go up to 2^127 (and down to 2^-127: means below 2^-123 lose up to three bits)
    __device__ __forceinline__ float eighth(mem_t codes, mem_t scales, int d) const
    {
        const uint32_t c = codes[d >> 1] >> (4 * (d & 1)), m = c & 7;
        const float size = m < 2 ? 0.0625f * m : __uint_as_float(((m >> 1) + 123u) << 23 | (m & 1) << 22);
        return (c & 8 ? -size : size) * mx4_power(scales[d >> 5]);
    }
    // Rows of the tile (piece) again, each over the keys that it sees and no others: a lane per key for the scores, a lane per dimension (of
    // 64) for the values, of eighths of which the mean is carried along, so that finite values never add up to infinity, nor do those that codes of the greatest powers have
    // beyond fp32.  Slow, for rows with infinities or NaN in their results; only for rows that have not been written yet, whose places may be those of the query.
    __device__ __forceinline__ void plainly(int row, int step, int end)
    {
        const int dim = A.cache.head_dim;
        for (end = min(end, t.count); row < end; row += step) {
            int token, head;
            place(row, &token, &head);
            const float* src = A.query + (int64_t)(t.first + token) * A.ld_query + (int64_t)head * dim;
            const int last = t.p0 + token, first = first_key(last, A.window);
            float top = -INFINITY, sum = 0.f, mean[HD / 64 + 1] = {};
            for (int j0 = t.lo; j0 < t.hi; j0 += 64) {
                const int j = t.position(j0) + lane;
                int id = -1;
                if ((j0 < t.head || j >= first) && j <= last && j < t.end_at(j0)) id = A.cache.table[t.seq * A.cache.table_stride + (int)A.cache.page.quot((uint32_t)j)];
                const bool seen = (uint32_t)id < (uint32_t)A.cache.num_pages;
                const uint64_t lanes = __ballot(seen);
                if (lanes == 0) continue;
                const Row at{seen ? (uint32_t)id : 0u, (uint32_t)(j - (int)A.cache.page.quot((uint32_t)j) * (int)A.cache.page.d), seen};
                const Place place_here = place_of<false>(at);
                const mem_t v_at = (mem_t)(values() + place_here.v), vs_at = (mem_t)(value_scales() + place_here.vs);
                float score = -INFINITY;
                if (seen) {
                    const mem_t k = (mem_t)(keys() + place_here.k), ks = (mem_t)(key_scales() + place_here.ks);
                    float dot = 0.f;
                    for (int d = 0; d < dim; ++d) dot += src[d] * A.sign * eighth(k, ks, d);
                    score = dot * A.c * 8.f;
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
                    const int lane_of = __ffsll((unsigned long long)rest) - 1;
                    const float wk = __shfl(w, lane_of) * by;
                    const mem_t v = (mem_t)__shfl((unsigned long long)v_at, lane_of);
                    const mem_t vs = (mem_t)__shfl((unsigned long long)vs_at, lane_of);
#pragma unroll
                    for (int i = 0; i <= HD / 64; ++i)
                        if (64 * i + lane < dim) mean[i] += wk * eighth(v, vs, 64 * i + lane);
                }
            }
            // a piece's state in units in which its sum is at most an eighth
            const int e = (sum > 0.f ? __builtin_amdgcn_frexp_expf(sum) : 0) + 3;
            const float part = ldexpf(sum, -e);
            float* dst = t.cuts == 1 ? A.out + (int64_t)(t.first + token) * A.ld_out + (int64_t)head * dim : values_of(row);
            const float by = 8.f * (t.cuts == 1 ? sum * over_sum(A, sum, top, head) : part);
#pragma unroll
            for (int i = 0; i <= HD / 64; ++i)
                if (64 * i + lane < dim) dst[64 * i + lane] = mean[i] * by;
            if (t.cuts > 1 && lane == 0) *state_of(row) = f2_t{top + (float)e, part};
        }
    }

    __device__ __forceinline__ static void add_weights(float sum, float& l, float& rest)
    {
        const float large = fmaxf(l, sum), small = fminf(l, sum);
        l = large + small;
        rest += small - (l - large);
    }
    __device__ __forceinline__ static u4_t transposed(lds_t at, lds_t further)
    {
        const s4_t v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)at);
        const s4_t v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)further);
        const u2_t a0 = __builtin_bit_cast(u2_t, v0), a1 = __builtin_bit_cast(u2_t, v1);
        return u4_t{a0.x, a0.y, a1.x, a1.y};
    }
    // a block's values into LDS
    __device__ __forceinline__ static void put_values(const u4_t& codes, uint32_t e, lds_t at)
    {
        const float scale = __uint_as_float(e << 23);                // (0 is 2^-127 to the instruction and 255 NaN)
#pragma unroll
        for (int i = 0; i < 4; ++i) *(lds4_t)(at + 16 * i) = as_bf16(codes[i], scale);
    }

    // ---- few rows: every wavefront over keys of its own, 16 rows at a time ----
    static constexpr int kChunks = (HD + 127) / 128, kTiles = HD / 16;

    // A step of 16 KB keys (64 in place of 32: 86 us for 80 of 32 answers, fewer of them under way): key idx of each 16, block 4 c + g of it
    static constexpr int KB = 2;
    struct Step {
        u4_t k[KB][kChunks], v[KB][kChunks];
        uint8_t ks[KB][kChunks], vs[KB][kChunks];                    // (as loaded: widened ahead of their use they would be waited for)
        uint64_t there;                                              // a bit for each key
    };
    // blocks of a lane in a head's first row
    struct Blocks {
        uint64_t k[kChunks], v[kChunks], ks[kChunks], vs[kChunks];
    };
    __device__ __forceinline__ void load_step(int key, int idx, const Blocks& of, Step& s)
    {
        const int p0 = t.position(key);
        bring_pages(p0, 16 * KB);
        if (X.alike) load_rows<true>(p0, t.end_at(key), idx, of, s);
        else load_rows<false>(p0, t.end_at(key), idx, of, s);
    }
    template <bool ALIKE>
    __device__ __forceinline__ void load_rows(int p0, int end, int idx, const Blocks& of, Step& s) const
    {
        s.there = 0;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const Row at = row_at(p0 + 16 * b + idx, end);
            s.there |= (uint64_t)(__ballot(at.there) & 0xffff) << (16 * b);
            const Place here = place_of<ALIKE>(at);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                s.k[b][c] = *(mem4_t)(of.k[c] + here.k);
                s.ks[b][c] = *(mem_t)(of.ks[c] + here.ks);
                s.v[b][c] = *(mem4_t)(of.v[c] + here.v);
                s.vs[b][c] = *(mem_t)(of.vs[c] + here.vs);
            }
        }
    }
    __device__ __forceinline__ static float of_rows(float x, float (*op)(float, float))
    {
        const u2_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return both_halves(op(__uint_as_float(r.x), __uint_as_float(r.y)), op);
    }

    // rows r0 .. r0 + 15 of the tile; whether these have to be done by plainly()
    __device__ __forceinline__ bool own_keys(int r0)
    {
        __shared__ f2_t states[kAttnWaves][16];
        __shared__ int odd[kAttnWaves];
        const int idx = lane & 15, g = lane >> 4, row = r0 + idx;
        const int rows = min(16, t.count - r0);
        f4_t o[kTiles];
#pragma unroll
        for (int d = 0; d < kTiles; ++d) o[d] = f4_t{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f, l_rest = 0.f;
        const lds_t mine_values = lds + wave * (16 * KB * kRow);
        int key = t.lo + 16 * KB * wave;
        id_base = -64;                                               // (the keys of the rows before are begun again)
        constexpr int kStride = 16 * KB * kAttnWaves;
        constexpr uint64_t kWhole = (1ull << (16 * KB)) - 1;
        if (key < t.hi) {
            Blocks of;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const uint32_t block = block_of(4 * c + g);
                of.k[c] = keys() + 16 * block, of.v[c] = values() + 16 * block, of.ks[c] = key_scales() + block, of.vs[c] = value_scales() + block;
            }
            RowBlock x[kChunks];
#pragma unroll
            for (int c = 0; c < kChunks; ++c) load_row(row, 4 * c + g, x[c]);
            asm volatile("" ::: "memory");
            Step even, odd_one;
            load_step(key, idx, of, even);
            asm volatile("" ::: "memory");
            load_step(key + kStride, idx, of, odd_one);
            asm volatile("" ::: "memory");
            Terms q[kChunks];
#pragma unroll
            for (int c = 0; c < kChunks; ++c) cut_row(x[c], q[c]);
            int token, head;
            place(min(row, t.count - 1), &token, &head);
            const int p = t.p0 + token, lo = first_key(p, A.window), lo_last = first_key(t.p0 + t.tokens - 1, A.window);
            auto step = [&](Step& now) {
                const int p0 = t.position(key);
                const bool whole = now.there == kWhole, in_head = key < t.head;
                if constexpr (HD != 128) {                           // (lanes without a block have another's, for which rows have zeros: NaN would stay one)
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
#pragma unroll
                        for (int b = 0; b < KB; ++b) now.ks[b][c] = 4 * c + g < blocks() ? now.ks[b][c] : 0;
                }
                if (!whole) {                                        // (a value of the least power under a weight of 0)
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
#pragma unroll
                        for (int b = 0; b < KB; ++b) now.vs[b][c] = (now.there >> (16 * b + idx)) & 1 ? now.vs[b][c] : 0;
                }
                f4_t s[KB];
#pragma unroll
                for (int b = 0; b < KB; ++b) s[b] = f4_t{0.f, 0.f, 0.f, 0.f};
                // (small terms first, the blocks in turn)
                auto product = [&](auto part) {
                    constexpr int n = decltype(part)::value;
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
#pragma unroll
                        for (int b = 0; b < KB; ++b)
                            s[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(now.k[b][c]), operand(q[c].t[n]), s[b], 4, 2, 0, (int)now.ks[b][c], n % 4,
                                                                                    (int)q[c].scale[n / 4]);
                };
                each_of<kParts>([&](auto i) { product(std::integral_constant<int, kParts - 1 - decltype(i)::value>()); });
                // the values of the step, for the transposed reads below
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int c = 0; c < kChunks; ++c)
                        if (4 * c + g < kBlocks) put_values(now.v[b][c], now.vs[b][c], mine_values + (16 * b + idx) * kRow + 64 * (4 * c + g));
                // score i of block b belongs to key 16 b + 4 g + i
                if (!whole || p0 + 16 * KB - 1 > t.p0 || (!in_head && p0 < lo_last)) {
                    const int last = p - p0 - 4 * g, first = in_head ? 0 : lo - p0 - 4 * g;
                    const uint64_t there = now.there >> (4 * g);
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int k = 16 * b + i;
                            if (k > last || k < first || !((there >> k) & 1)) s[b][i] = -INFINITY;
                        }
                }
                float top = s[0][0];
#pragma unroll
                for (int i = 1; i < 4 * KB; ++i) top = fmaxf(top, s[i / 4][i % 4]);
                top = of_rows(top, larger) * A.c;
                if (__any(top > m + kRise)) {                        // (m starts at -infinity)
                    float mn = m;
                    if (top > m + kRise) mn = __builtin_ceilf(top);
                    const float f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
                    l *= f;
                    l_rest *= f;
#pragma unroll
                    for (int d = 0; d < kTiles; ++d) o[d] *= f;
                    m = mn;
                }
                const float bias = kUnit - (m == -INFINITY ? 0.f : m);
                float sum = 0.f;
                // a lane gives the place of four dimensions of one key and gets one dimension of four keys, within 16 lanes
                const lds_t at = mine_values + (4 * g + (idx >> 2)) * kRow + 8 * (idx & 3);
#pragma unroll
                for (int h = 0; h < KB / 2; ++h) {                   // 32 keys
                    float w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * h + i / 4][i % 4], A.c, bias));
                        sum += w[i];
                    }
                    u4_t part[3];
                    cut3(w, part);
#pragma unroll
                    for (int d = 0; d < kTiles; ++d) {
                        const u4_t a = transposed(at + 32 * d + 32 * h * kRow, at + 32 * d + (32 * h + 16) * kRow);
#pragma unroll
                        for (int n = 2; n >= 0; --n)
                            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, part[n]), o[d], 0, 0, 0);
                    }
                }
                add_weights(sum, l, l_rest);
            };
            // Two steps are under way: what a step has is loaded anew behind it, in this order and whether there is one or not, so that each waits for its own
            // loads alone (they are counted).
            for (; key < t.hi; key += kStride) {
                step(even);
                load_step(key + 2 * kStride, idx, of, even);
                asm volatile("" ::: "memory");
                key += kStride;
                if (key < t.hi) step(odd_one);
                load_step(key + 2 * kStride, idx, of, odd_one);
                asm volatile("" ::: "memory");
            }
        }
        l = of_rows(l + l_rest, added);
        float z = 0.f;
#pragma unroll
        for (int d = 0; d < kTiles; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) z = __builtin_fmaf(o[d][i], 0.f, z);
        __syncthreads();                                             // (the states take the place of the values)
        if (const bool found = __any(idx < rows && z != z); lane == 0) odd[wave] = found;
        if (g == 0) states[wave][idx] = f2_t{m - kUnit, l};
        const lds_t mine = lds + (wave * 16 + idx) * HD * 4;
#pragma unroll
        for (int d = 0; d < kTiles; ++d)
            *reinterpret_cast<__attribute__((address_space(3))) f4_t*>(mine + (((4 * d + g) ^ (idx & 7)) << 4)) = o[d];
        __syncthreads();
        int any = 0;
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) any |= odd[w];
        const bool again = __builtin_amdgcn_readfirstlane(any);
        const int pieces = A.cache.head_dim / 4;
        for (int i = thread; !again && i < rows * pieces; i += kAttnThreads) {
            const int r = i / pieces, piece = i - r * pieces;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, states[w][r].x);
            // (two powers more, so that what up to four of them have adds up to no infinity)
            const float unit = top + 2.f, base = top == -INFINITY ? 0.f : unit;
            float sum = 0.f;
            f4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(states[w][r].x - base);
                sum += states[w][r].y * f;
                v += *reinterpret_cast<const __attribute__((address_space(3))) f4_t*>(lds + (w * 16 + r) * HD * 4 + ((piece ^ (r & 7)) << 4)) * f;
            }
            int token, head;
            place(r0 + r, &token, &head);
            if (t.cuts == 1) {
                *reinterpret_cast<f4_t*>(A.out + (int64_t)(t.first + token) * A.ld_out + (int64_t)head * A.cache.head_dim + 4 * piece) =
                    v * over_sum(A, sum, unit, head);
            } else {
                *reinterpret_cast<f4_t*>(values_of(r0 + r) + 4 * piece) = v;
                if (piece == 0) *state_of(r0 + r) = f2_t{unit, sum};
            }
        }
        __syncthreads();                                             // (before the next rows)
        return again;
    }

    // ---- many rows: all wavefronts over the same keys, 32 rows each ----
    static constexpr int kHalves = (HD + 63) / 64, kDims = HD / 32, kMine = (kKeys * kBlocks + kAttnThreads - 1) / kAttnThreads;

    // keys of a step: key col of each 32, block 2 c + half of it
    struct Keys {
        u4_t k[NB][kHalves];
        uint8_t ks[NB][kHalves];
        uint64_t there;              // (bits of keys that a step has not are set)
    };
    struct KeyBlocks {
        uint64_t k[kHalves], ks[kHalves];
    };
    __device__ __forceinline__ void load_keys(int key, int col, const KeyBlocks& of, Keys& s)
    {
        const int p0 = t.position(key);
        bring_pages(p0, kKeys);
        if (X.alike) load_keys<true>(p0, t.end_at(key), col, of, s);
        else load_keys<false>(p0, t.end_at(key), col, of, s);
    }
    template <bool ALIKE>
    __device__ __forceinline__ void load_keys(int p0, int end, int col, const KeyBlocks& of, Keys& s) const
    {
        s.there = NB == 2 ? 0 : ~0xffffffffull;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const Row at = row_at(p0 + 32 * b + col, end);
            s.there |= (__ballot(at.there) & 0xffffffffull) << (32 * b);
            const Place here = place_of<ALIKE>(at);
#pragma unroll
            for (int c = 0; c < kHalves; ++c) {
                s.k[b][c] = *(mem4_t)(of.k[c] + here.k);
                s.ks[b][c] = *(mem_t)(of.ks[c] + here.ks);
            }
        }
    }
    // and the blocks of values that a thread turns
    struct Values {
        u4_t v[kMine];
        uint8_t vs[kMine];
        bool there[kMine];
    };
    struct ValueBlocks {
        uint64_t v[kMine], vs[kMine];
    };
    __device__ __forceinline__ void load_values(int key, const ValueBlocks& of, Values& s)
    {
        const int p0 = t.position(key);
        bring_pages(p0, kKeys);
        if (X.alike) load_values<true>(p0, t.end_at(key), of, s);
        else load_values<false>(p0, t.end_at(key), of, s);
    }
    template <bool ALIKE>
    __device__ __forceinline__ void load_values(int p0, int end, const ValueBlocks& of, Values& s) const
    {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            const Row at = row_at(p0 + min((n * kAttnThreads + thread) / kBlocks, kKeys - 1), end);
            const Place here = place_of<ALIKE>(at);
            s.there[n] = at.there;
            s.v[n] = *(mem4_t)(of.v[n] + here.v);
            s.vs[n] = *(mem_t)(of.vs[n] + here.vs);
        }
    }
    __device__ __forceinline__ void turn_values(const Values& s, lds_t buffer) const
    {
#pragma unroll
        for (int n = 0; n < kMine; ++n) {
            const int unit = n * kAttnThreads + thread, row = unit / kBlocks, block = unit - row * kBlocks;
            if (kKeys * kBlocks % kAttnThreads == 0 || row < kKeys) put_values(s.v[n], s.there[n] ? s.vs[n] : 0, buffer + row * kRow + 64 * block);
        }
    }

    __device__ __forceinline__ bool shared_keys()
    {
        const int col = lane & 31, half = lane >> 5, row = 32 * wave + col;
        const int p_first = t.p0 + (int)A.by_group.quot(t.row0 + min(32 * wave, t.count - 1));
        const int p_last = t.p0 + (int)A.by_group.quot(t.row0 + min(32 * wave + 31, t.count - 1));
        const int lo_last = first_key(p_last, A.window);
        f16_t o[kDims];
        auto nothing_yet = [&]() {
#pragma unroll
            for (int d = 0; d < kDims; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
        };
        float m = -INFINITY, l = 0.f, l_rest = 0.f;
        if (t.lo >= t.hi) {
            nothing_yet();
        } else {
            Keys step;
            Values turned;
            KeyBlocks keys_at;
            ValueBlocks values_at;
#pragma unroll
            for (int c = 0; c < kHalves; ++c) keys_at.k[c] = keys() + 16 * block_of(2 * c + half), keys_at.ks[c] = key_scales() + block_of(2 * c + half);
#pragma unroll
            for (int n = 0; n < kMine; ++n) {
                const uint32_t block = block_of((n * kAttnThreads + thread) % kBlocks);
                values_at.v[n] = values() + 16 * block, values_at.vs[n] = value_scales() + block;
            }
            load_keys(t.lo, col, keys_at, step);
            load_values(t.lo, values_at, turned);
            asm volatile("" ::: "memory");
            // (rows behind them here: held ahead of their cutting they would take registers that are not there)
            Terms q[kHalves];
#pragma unroll
            for (int c = 0; c < kHalves; ++c) {
                RowBlock x;
                load_row(row, 2 * c + half, x);
                cut_row(x, q[c]);
            }
            asm volatile("" ::: "memory");                           // (the accumulators come after the cutting of rows, which takes registers too)
            nothing_yet();
            int token, head;
            place(min(row, t.count - 1), &token, &head);
            const int p = t.p0 + token, lo = first_key(p, A.window);
            int buffer = 0;
            for (int key = t.lo; key < t.hi; key += kKeys) {
                const lds_t here = lds + buffer * (kKeys * kRow);
                buffer ^= 1;
                turn_values(turned, here);
                __syncthreads();                                     // (what the other buffer held has been read by all)
                load_values(key + kKeys, values_at, turned);
                const int p0 = t.position(key);
                const bool in_head = key < t.head, mine = 32 * wave < t.count && p0 <= p_last;
                f16_t s[NB];
                if (mine) {
                    if constexpr (HD % 64 != 0 || HD == 64 || HD > 128) {                // (see own_keys)
#pragma unroll
                        for (int c = 0; c < kHalves; ++c)
#pragma unroll
                            for (int b = 0; b < NB; ++b) step.ks[b][c] = 2 * c + half < blocks() ? step.ks[b][c] : 0;
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[b][i] = 0.f;
                    auto product = [&](auto part) {
                        constexpr int n = decltype(part)::value;
#pragma unroll
                        for (int c = 0; c < kHalves; ++c)
#pragma unroll
                            for (int b = 0; b < NB; ++b)
                                s[b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(step.k[b][c]), operand(q[c].t[n]), s[b], 4, 2, 0, (int)step.ks[b][c], n % 4,
                                                                                       (int)q[c].scale[n / 4]);
                    };
                    each_of<kParts>([&](auto i) { product(std::integral_constant<int, kParts - 1 - decltype(i)::value>()); });
                }
                const uint64_t there = step.there;
                load_keys(key + kKeys, col, keys_at, step);
                if (!mine) continue;
                // score i of block b belongs to key 32 b + 8 (i / 4) + 4 half + i % 4
                if (~there != 0 || p0 + kKeys - 1 > p_first || (!in_head && p0 < lo_last)) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int below = 32 * b + 4 * half, last = p - p0 - below, first = in_head ? 0 : lo - p0 - below;
                        const uint32_t bits = (uint32_t)(there >> below);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int k = 8 * (i / 4) + i % 4;
                            if (k > last || k < first || !((bits >> k) & 1)) s[b][i] = -INFINITY;
                        }
                    }
                }
                float top = s[0][0];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
                top = both_halves(top, larger) * A.c;
                if (__any(top > m + kRise)) {
                    float mn = m;
                    if (top > m + kRise) mn = __builtin_ceilf(top);
                    const float f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
                    l *= f;
                    l_rest *= f;
#pragma unroll
                    for (int d = 0; d < kDims; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] *= f;
                    m = mn;
                }
                const float bias = kUnit - (m == -INFINITY ? 0.f : m);
                float sum = 0.f;
                const lds_t at = here + (4 * half + ((lane & 15) >> 2)) * kRow + 32 * ((lane >> 4) & 1) + 8 * (lane & 3);
#pragma unroll
                for (int h = 0; h < 2 * NB; ++h) {                   // 16 keys
                    float w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h / 2][8 * (h % 2) + i], A.c, bias));
                        sum += w[i];
                    }
                    u4_t part[3];
                    cut3(w, part);
#pragma unroll
                    for (int d = 0; d < kDims; ++d) {
                        const u4_t a = transposed(at + 64 * d + 16 * h * kRow, at + 64 * d + (16 * h + 8) * kRow);
#pragma unroll
                        for (int n = 2; n >= 0; --n)
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, part[n]), o[d], 0, 0, 0);
                    }
                }
                add_weights(sum, l, l_rest);
            }
        }
        float z = 0.f;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) z = __builtin_fmaf(o[d][i], 0.f, z);
        if (__any(row < t.count && z != z)) return true;
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
};

// What a step of a long tile takes, a short one's being 1.  (A prompt's chunk beside two dozen answers: 1.5 to 4.5 are within 3 % of each other but for 256
// dimensions, 257 us at 1.5 and 147 from 2.2 on.)
constexpr float kTall = 3.f;

// grid (KV heads, workgroups)
template <int HD>
__global__ void __launch_bounds__(kAttnThreads, HD > 128 ? 1 : 2) paged_mx_attention_kernel(TSHIP_LENS_ARGS, const AttnArgs A, const MxScales X)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int kvh = blockIdx.x, idx = blockIdx.z * gridDim.y + blockIdx.y;
    const Lens H = TSHIP_LENS;
    // (every line of the arguments is asked for at once: read where they are needed they cost one trip to memory after the other, 3 us)
    asm volatile("" ::"s"(A.query), "s"(A.ld_out), "s"(A.by_group.m), "s"(A.cache.k), "s"(A.cache.v_head), "s"(A.cache.table_stride), "s"(A.cache.max_pages), "s"(X.k), "s"(X.v_head));
    const Deal deal = deal_out(H, gridDim.x, worth_of(kTypeMXFP4, HD, kAttnWaves), kTall);
    if (H.pieces > 0 && blockIdx.x == 0 && idx == 0 && threadIdx.x == 0) *deal_of(A) = deal;
    AttnTile t;
    const bool whole = deal.tall < 0;
    if (whole || idx < deal.tall) {
        if (!(whole ? find_whole(H, A, idx, t) : find_tall(H, A, deal, idx, t))) return;
        if (t.tokens * A.group > kKeyRows) {
            AttnMx<HD> a(A, X, t, kvh, threadIdx.x, (lds_t)smem);
            if (__builtin_expect(a.shared_keys(), 0)) a.plainly(32 * a.wave, 1, 32 * a.wave + 32);
            return;
        }
    } else if (idx >= H.pieces) {
        return;
    }
    const int run = idx - deal.tall;
    for (int at = whole ? 0 : run * deal.run_steps, end = whole ? 1 : at + deal.run_steps; at < end;) {
        const int steps = whole ? 1 : find_run(H, A, deal, run, at, t);
        if (steps == 0) return;
        at += steps;
        if (!whole && !t.mine) continue;
        int thread = threadIdx.x;
        asm volatile("" : "+v"(thread));                             // (what follows from it is worked out for each tile: kept from one to the next it would be spilled)
        AttnMx<HD> a(A, X, t, kvh, thread, (lds_t)smem);
        int again = 0;                                               // a bit for every 16 rows, which have not been written then
        for (int r0 = 0; r0 < t.count; r0 += 16) again |= (int)a.own_keys(r0) << (r0 / 16);
        if (__builtin_expect(again, 0)) a.plainly((again & 1 ? 0 : 16) + a.wave, kAttnWaves, again & 2 ? 32 : 16);
    }
}

template <int HD>
bool launch_mx(const Lens& H, const AttnArgs& args, const MxScales& scales, const dim3& grid, hipStream_t stream)
{
    const auto kern = paged_mx_attention_kernel<HD>;
    constexpr size_t lds = AttnMx<HD>::kLds;
    if (!raise_lds_limit(reinterpret_cast<const void*>(kern), lds)) return false;
    hipLaunchKernelGGL(kern, grid, dim3(kAttnThreads), lds, stream, TSHIP_LENS_OF(H), args, scales);
    return hip_ok(hipGetLastError(), "paged attention launch");
}

}  // namespace

bool launch_mx_attention(const Lens& H, const AttnArgs& args, const MxScales& scales, const dim3& grid, hipStream_t stream)
{
    switch (dims_of(args.cache.head_dim)) {
    case 64: return launch_mx<64>(H, args, scales, grid, stream);
    case 96: return launch_mx<96>(H, args, scales, grid, stream);
    case 128: return launch_mx<128>(H, args, scales, grid, stream);
    case 192: return launch_mx<192>(H, args, scales, grid, stream);
    default: return launch_mx<256>(H, args, scales, grid, stream);
    }
}

}  // namespace tship
