// What the attention over pages has in common whatever the cache's type: the rows that share a KV head, token after token, cut into tiles, the keys of a tile
// and the pieces that they are cut into, where the states of pieces go, and arithmetic on registers.
#pragma once
#include "tship_internal.h"

#include <utility>

namespace tship {

constexpr int kMaxDim = 256;

typedef float f2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));

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
static __device__ __attribute__((aligned(16))) uint8_t g_zero_row[kMaxDim * 4];

struct AttnArgs {
    const float* query;
    float* out;
    const float* sinks;
    float* partial;              // [piece][KV head][row of the tile][head_dim] weighted values, then [piece][KV head][row] (unit, sum)
    int64_t ld_query, ld_out;
    float c;                     // |scale| log2 e
    float sign;                  // of scale, 0 where it is 0
    int rows, group, window, first, capacity;
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
    bool mine;                   // of a run: it has a part of the tile's keys, not only of what the tile costs besides
    // With first positions that stay visible the keys are numbered on: positions 0 .. head_end - 1 as 0 .. head - 1 (whole steps of the kernel's, so that none
    // has keys of both), then the window's, `jump` further on.  All rows see of the former what lies before them, of the latter what is in their window.
    int head, head_end, jump;
    __device__ __forceinline__ int position(int key) const { return key < head ? key : key + jump; }
    __device__ __forceinline__ int end_at(int key) const { return key < head ? min(head_end, hi) : hi + jump; }      // of the positions from that key's on
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
// the largest of numbers that are not negative (lanes that have none below them get 0)
__device__ __forceinline__ int lane_max(int v)
{
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(v, 63);
}

// What the kernels need to find their piece.  It stands in front of the other arguments: the hardware delivers the first 14 dwords in
// registers at wave launch (a structure is read from the argument block instead), so that the lengths are asked for at once.
struct Lens {
    const int32_t* row_starts;
    const int32_t* context_lens;
    int seqs, rows, group, window, first;
    int pieces;                  // per KV head that the chip takes at once; 0: keys are not cut
    int capacity;                // positions that the page table has room for
};
#define TSHIP_LENS_ARGS const int32_t *row_starts, const int32_t *context_lens, int seqs, int rows, int group, int window, int first, int pieces, int capacity
#define TSHIP_LENS_OF(H) H.row_starts, H.context_lens, H.seqs, H.rows, H.group, H.window, H.first, H.pieces, H.capacity
#define TSHIP_LENS Lens{row_starts, context_lens, seqs, rows, group, window, first, pieces, capacity}

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
        if (H.window > 0) span = (int)min((int64_t)span, (int64_t)H.window + min(n, kTileRows) + ((int64_t)H.first + 63) / 64 * 64);
        steps = (span + 127) >> 7;
    }
    __device__ __forceinline__ int cuts(int len) const { return max(1, (steps + len - 1) / len); }
};

// Steps of 128 keys that pieces have to save a tile to be worth it.  Joining them takes 5 us where they are few, 8.5 for many short tiles, 7.5
// for long ones (3 of it the second launch, which comes wherever the page table has room for as many positions).  A step takes a short tile of
// 64, 128, 256 dimensions 1.0, 1.4, 2.9 us in fp16 (bf16 0.9, 1.6, 3.5; fp32, by fewer wavefronts, 2.1, 8.4, 19.3) and a long one 2.6, 4.4,
// 8.7 (bf16 4.1, 5.6, 12.2; fp32 7.4, 12.5, 29.5; four bits nearly as fp16): by the dimensions, near enough.  One sequence of 512 keys, 256 dimensions and 8 KV heads: cut
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
    t.head = t.head_end = t.jump = 0;
    if (A.first > 0) {                                               // (with a window)
        const int hi = max(0, t.hi), begin = max(t.lo, A.first);
        t.lo = 0;
        t.head_end = min(hi, A.first);
        // (steps of 64 for fp16 and four bits, else of 32: of five first positions and a window of 128 over bf16 a tile has 6 steps in place of 7)
        const int step = A.cache.element_type == kTypeF16 || A.cache.element_type == kTypeMXFP4 ? 64 : 32;
        t.head = (t.head_end + step - 1) & ~(step - 1);
        if (hi > A.first) {
            t.jump = begin - t.head;
            t.hi = hi - t.jump;
        }
    }
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
// ---- another way to deal out the same work ----
// Pieces of sequences whose lengths have nothing to do with each other are between half as long and as long as the longest.  Here the steps of all short tiles (of
// sequences with at most 32 rows), one after the other, are cut into runs of equal length: a run may have the end of one tile, whole ones and the beginning of another, to
// which its workgroup turns one after the other.  Long tiles are cut into pieces by themselves, with their share of the workgroups, one piece each.  Parts of tiles
// have slots as pieces have: a long tile's piece its number, a run's part the number of its workgroup plus that of its tile.
// A tile costs its workgroup more than its steps: its rows, page ids and first keys come one trip to memory after the other, and the states of the wavefronts meet at its end (9 us, a step
// 1.6), so in a run it counts as so many steps more.
constexpr int kTurn = 5;
struct Deal {
    int tall;                    // workgroups for pieces of long tiles; -1: every tile is one workgroup's
    int tall_steps, run_steps;   // 128 keys each: of a piece, of a run
};
__device__ __forceinline__ bool is_tall(const Lens& H, const Lanes& L) { return L.n * H.group > kKeyRows; }
__device__ __forceinline__ int tall_tiles(const Lens& H, const Lanes& L) { return is_tall(H, L) ? L.tiles : 0; }
__device__ __forceinline__ int short_steps(const Lens& H, const Lanes& L) { return L.tiles > 0 && !is_tall(H, L) ? kTurn + max(1, min(L.steps, 1 << 16)) : 0; }
// tall: what a step of a long tile takes, a short one's being 1
__device__ __forceinline__ Deal deal_out(const Lens& H, int kv_heads, Worth least, float tall)
{
    constexpr Deal kWhole{-1, 0, 0};
    if (H.pieces == 0) return kWhole;
    Lanes L;
    int tiles = 0, long_tiles = 0, most = 0, long_most = 0;
    uint32_t steps = 0;                                              // (exactly: the runs have to have all of them; up to 1024 tiles of 65541, more are not dealt out)
    float long_steps = 0.f;
    for (int s0 = 0; s0 < H.seqs; s0 += 64) {
        L.load(H, s0);
        const int n = short_steps(H, L), m = tall_tiles(H, L);
        tiles += lane_sum(L.tiles);
        long_tiles += lane_sum(m);
        steps += (uint32_t)lane_sum(n);
        long_steps += (float)lane_sum(min(m * min(L.steps, 1 << 16), 1 << 24));
        most = max(most, lane_max(n));
        long_most = max(long_most, lane_max(m > 0 ? L.steps : 0));
    }
    if (tiles >= H.pieces) return kWhole;
    const bool runs = tiles > long_tiles;
    Deal d{0, 1, 1};
    if (long_tiles > 0) {
        const float share = tall * long_steps / (tall * long_steps + (float)steps);
        d.tall = runs ? min(max((int)(share * H.pieces + 0.5f), long_tiles), H.pieces - 1) : H.pieces;
        // (a length that no tile exceeds ends it in any case: there are no more tiles than pieces)
        for (d.tall_steps = max(1, (int)ceilf(long_steps / (float)d.tall));; d.tall_steps += 1 + d.tall_steps / 16) {
            int all = 0;
            for (int s0 = 0; s0 < H.seqs; s0 += 64) {
                L.load(H, s0);
                all += lane_sum(min(tall_tiles(H, L) * L.cuts(d.tall_steps), 1 << 24));
            }
            if (all <= d.tall) break;
        }
    }
    if (runs) d.run_steps = max(1, (int)((steps + (H.pieces - d.tall) - 1) / (uint32_t)(H.pieces - d.tall)));
    const bool worth = (long_tiles > 0 && long_most - d.tall_steps >= least.tall) || (runs && most - kTurn - d.run_steps >= (tiles * kv_heads >= 64 ? least.many : least.few));
    return worth ? d : kWhole;
}
// behind the states: the deal, from the attention for the kernel that joins
__device__ __forceinline__ Deal* deal_of(const AttnArgs& A) { return reinterpret_cast<Deal*>(steps_of(A)); }

// the idx-th tile from the end (the last tiles of a prompt have the most keys and go first), whole; false: there is none
__device__ __forceinline__ bool find_whole(const Lens& H, const AttnArgs& A, int idx, AttnTile& t)
{
    Lanes L;
    int tiles = 0, s0 = 0;
    for (; s0 < H.seqs; s0 += 64) {
        L.load(H, s0);
        tiles += lane_sum(L.tiles);
    }
    int want = tiles - 1 - idx, cum;
    if (want < 0) return false;
    for (s0 = 0;; s0 += 64) {                                        // (fewer than the total)
        L.load(H, s0);
        cum = lane_scan(L.tiles);
        if (want < __builtin_amdgcn_readlane(cum, 63)) break;
        want -= __builtin_amdgcn_readlane(cum, 63);
    }
    const int at = __ffsll((unsigned long long)__ballot(want < cum)) - 1;
    set_tile(A, L, s0, at, want - __builtin_amdgcn_readlane(cum - L.tiles, at), 1 << 24, t);
    t.cuts = 1;
    return true;
}
// piece number idx of the long tiles; false: there is none
__device__ __forceinline__ bool find_tall(const Lens& H, const AttnArgs& A, const Deal& d, int idx, AttnTile& t)
{
    Lanes L;
    int want = idx;
    for (int s0 = 0; s0 < H.seqs; s0 += 64) {
        L.load(H, s0);
        const int all = tall_tiles(H, L) * L.cuts(d.tall_steps), cum = lane_scan(all);
        if (want >= __builtin_amdgcn_readlane(cum, 63)) {
            want -= __builtin_amdgcn_readlane(cum, 63);
            continue;
        }
        const int at = __ffsll((unsigned long long)__ballot(want < cum)) - 1, cuts = __builtin_amdgcn_readlane(L.cuts(d.tall_steps), at);
        want -= __builtin_amdgcn_readlane(cum - all, at);
        set_tile(A, L, s0, at, want / cuts, d.tall_steps, t);
        t.slot = idx;
        const int keys = piece_keys(t), begin = t.lo + want % cuts * keys;
        t.hi = min(begin + keys, t.hi);
        t.lo = begin;
        return true;
    }
    return false;
}
// Step `at` of the short tiles' and what follows of its tile up to the end of run number `run` (its first kTurn are no keys'); how many steps these are, 0: there
// are no more.
__device__ __forceinline__ int find_run(const Lens& H, const AttnArgs& A, const Deal& d, int run, int at, AttnTile& t)
{
    Lanes L;
    int want = at, number = 0;
    for (int s0 = 0; s0 < H.seqs; s0 += 64) {
        L.load(H, s0);
        const int all = short_steps(H, L), cum = lane_scan(all);
        const uint64_t tiles = __ballot(all > 0);
        if (want >= __builtin_amdgcn_readlane(cum, 63)) {
            want -= __builtin_amdgcn_readlane(cum, 63);
            number += __popcll(tiles);
            continue;
        }
        const int lane = __ffsll((unsigned long long)__ballot(want < cum)) - 1, steps = __builtin_amdgcn_readlane(all, lane);
        const int x0 = want - __builtin_amdgcn_readlane(cum - all, lane), x1 = min(steps, x0 + (run + 1) * d.run_steps - at), start = at - x0;
        set_tile(A, L, s0, lane, 0, 1 << 24, t);
        t.cuts = (start + steps - 1) / d.run_steps - (start + kTurn) / d.run_steps + 1;
        t.slot = d.tall + run + number + __popcll(tiles & ((1ull << lane) - 1));
        t.mine = x1 > kTurn;
        const int begin = t.lo + 128 * max(0, x0 - kTurn);
        t.hi = x1 == steps ? t.hi : min(t.hi, t.lo + 128 * max(0, x1 - kTurn));
        t.lo = begin;
        return x1 - x0;
    }
    return 0;
}
// the tile of a row and head as it was dealt out and its first part; false: of no sequence
__device__ __forceinline__ bool find_dealt_row(const Lens& H, const AttnArgs& A, int row, int head, AttnTile& t, int* in_tile)
{
    const Deal d = *deal_of(A);
    t.cuts = 1;
    if (d.tall < 0) return true;
    Lanes L;
    int pieces = 0, before = 0, numbers = 0;
    for (int s0 = 0; s0 < H.seqs; s0 += 64) {
        L.load(H, s0);
        const int all = tall_tiles(H, L) * L.cuts(d.tall_steps), n = short_steps(H, L), cum = lane_scan(all), steps_cum = lane_scan(n);
        const uint64_t has = __ballot(row >= L.start && row < L.start + L.n), tiles = __ballot(n > 0);
        if (has) {
            const int at = __ffsll((unsigned long long)has) - 1;
            const int r = (row - __builtin_amdgcn_readlane(L.start, at)) * H.group + head % H.group, steps = __builtin_amdgcn_readlane(n, at);
            if (steps == 0) {
                const int tile = r / kTileRows;
                t.cuts = __builtin_amdgcn_readlane(L.cuts(d.tall_steps), at);
                t.slot = pieces + __builtin_amdgcn_readlane(cum - all, at) + tile * t.cuts;
                *in_tile = r - tile * kTileRows;
            } else {
                const int start = before + __builtin_amdgcn_readlane(steps_cum - n, at);
                t.cuts = (start + steps - 1) / d.run_steps - (start + kTurn) / d.run_steps + 1;
                t.slot = d.tall + (start + kTurn) / d.run_steps + numbers + __popcll(tiles & ((1ull << at) - 1));
                *in_tile = r;
            }
            return true;
        }
        pieces += __builtin_amdgcn_readlane(cum, 63);
        before += __builtin_amdgcn_readlane(steps_cum, 63);
        numbers += __popcll(tiles);
    }
    return false;
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
// two floats as three times two bf16 that sum up to them
__device__ __forceinline__ void cut3_pair(float x0, float x1, u4_t (&part)[3], int i)
{
    const float y0 = below_bf16(x0), y1 = below_bf16(x1);
    part[0][i] = high_halves(x0, x1);
    part[1][i] = high_halves(y0, y1);
    part[2][i] = high_halves(below_bf16(y0), below_bf16(y1));
}
// and eight
__device__ __forceinline__ void cut3(const float (&x)[8], u4_t (&part)[3])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) cut3_pair(x[2 * i], x[2 * i + 1], part, i);
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

// the attention over a cache in four bits (paged_mx.hip)
bool launch_mx_attention(const Lens& H, const AttnArgs& args, const MxScales& scales, const dim3& grid, hipStream_t stream);

}  // namespace tship
