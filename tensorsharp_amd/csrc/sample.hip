// The next token of each row of logits: temperature, top-k, top-p, min-p and a draw from a given random number.
//
// Candidates are ranked by (logit, lower index first); what top-k and top-p keep is a prefix of that order, so each is a logit and how
// many of its equals stay.  Weights e^((l - l_max) / T) are formed in 64-bit floating point and held as whole multiples of 2^-43:
// sums of them are exact and the same in every order, so that neither a tile nor an atomic can move the border of a prefix or the
// place of a draw.  (What is rounded away is below 2^-44 of the likeliest candidate's weight.)
#include "tship_internal.h"

#include <algorithm>

namespace tship {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr double kOne = 8796093022208.0;                             // 2^43: 2^20 of them stay below 2^63
constexpr uint32_t kLowestKey = 0x007fffffu;                         // of -infinity; NaN has 0

// larger logit, larger key; both zeros the same
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __float_as_uint(l + 0.0f);
    return l != l ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }

struct Settings {
    double temperature;
    float top;                   // largest logit
    uint32_t top_key;
};
__device__ __forceinline__ double weight_of(uint32_t key, const Settings& S)
{
    if (key <= kLowestKey) return 0.0;
    if (key == S.top_key) return 1.0;                                // (an infinite maximum too)
    return exp(((double)logit_of(key) - (double)S.top) / S.temperature);
}
__device__ __forceinline__ uint64_t whole(double w) { return (uint64_t)(w * kOne + 0.5); }

__device__ __forceinline__ uint64_t wave_max(uint64_t v)
{
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, o));
    return v;
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v)
{
    for (int o = 32; o > 0; o >>= 1) v += (uint64_t)__shfl_xor((unsigned long long)v, o);
    return v;
}

struct Prefix {
    uint32_t key;                // logits above stay, and `ties` of the equal ones (UINT32_MAX: all of them)
    uint32_t ties;
};

__global__ void __launch_bounds__(kThreads) sample_kernel(const float* logits, int64_t ld, int vocab, const float* uniforms, const float* temperature,
                                                          const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
                                                          float* probabilities)
{
    __shared__ uint64_t hist[256], red[kWaves], found[2];
    __shared__ uint32_t count[256];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = logits + row * ld;

    // the largest logit, and its lowest index
    uint64_t best = 0;
    for (int i = tid; i < vocab; i += kThreads) best = max(best, (uint64_t)key_of(x[i]) << 32 | (uint32_t)~i);
    best = wave_max(best);
    if (lane == 0) red[wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) best = max(best, red[w]);
    const int top_index = (int)~(uint32_t)best;
    Settings S;
    S.top_key = (uint32_t)(best >> 32);
    S.top = logit_of(S.top_key);
    const float T = temperature[row];
    S.temperature = T;
    if (S.top_key <= kLowestKey || !(T > 0.f)) {
        if (tid == 0) {
            tokens[row] = S.top_key <= kLowestKey ? -1 : top_index;
            if (probabilities) probabilities[row] = S.top_key <= kLowestKey ? 0.f : 1.f;
        }
        return;
    }

    Prefix P{kLowestKey, 0};
    auto each = [&](auto&& f) {
        for (int i = tid; i < vocab; i += kThreads) f(i, key_of(x[i]));
    };
    // top-k: the key of the k-th candidate, eight bits at a time
    const int k = top_k ? top_k[row] : 0;
    if (k > 0 && k < vocab) {
        uint32_t prefix = 0, left = k;
        bool cut = true;
        for (int shift = 24; shift >= 0 && cut; shift -= 8) {
            if (tid < 256) count[tid] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            each([&](int, uint32_t key) {
                if (key > kLowestKey && (key & mask) == prefix) atomicAdd(&count[(key >> shift) & 255], 1u);
            });
            __syncthreads();
            int d = 255;
            while (d > 0 && count[d] < left) left -= count[d--];
            if (d == 0 && count[0] < left) cut = false;              // fewer candidates than k
            prefix |= (uint32_t)d << shift;
            __syncthreads();
        }
        if (cut) P = {prefix, left};
    }
    auto block_sum = [&](uint64_t v) {
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) red[wave] = v;
        __syncthreads();
        uint64_t s = 0;
        for (int w = 0; w < kWaves; ++w) s += red[w];
        return s;
    };
    // top-p: the same over the weights
    const double p = top_p ? (double)top_p[row] : 1.0;
    const uint64_t tied = P.ties ? whole(weight_of(P.key, S)) * P.ties : 0;
    if (p < 1.0) {
        uint64_t total = 0;
        each([&](int, uint32_t key) { total += key > P.key ? whole(weight_of(key, S)) : 0; });
        total = block_sum(total) + tied;
        uint64_t left = (uint64_t)fmin((double)total, fmax(1.0, ceil(p * (double)total)));
        left = min(left, total);
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            each([&](int, uint32_t key) {
                if (key > P.key && (key & mask) == prefix) atomicAdd((unsigned long long*)&hist[(key >> shift) & 255], (unsigned long long)whole(weight_of(key, S)));
            });
            if (tid == 0 && tied && (P.key & mask) == prefix) atomicAdd((unsigned long long*)&hist[(P.key >> shift) & 255], (unsigned long long)tied);
            __syncthreads();
            int d = 255;
            while (d > 0 && hist[d] < left) left -= hist[d--];
            prefix |= (uint32_t)d << shift;
            __syncthreads();
        }
        const uint64_t w = whole(weight_of(prefix, S));
        const uint32_t ties = (uint32_t)((left + w - 1) / max(w, (uint64_t)1));
        if (prefix > P.key) P = {prefix, ties};
        else P.ties = min(P.ties, ties);
    }
    // the index behind the last of the equal ones that stay
    int tie_end = vocab;
    if (P.ties) {
        uint32_t seen = 0;
        for (int i0 = 0; i0 < vocab; i0 += kThreads) {
            const bool is = i0 + tid < vocab && key_of(x[i0 + tid]) == P.key;
            const uint64_t lanes = __ballot(is);
            __syncthreads();
            if (lane == 0) count[wave] = __popcll(lanes);
            __syncthreads();
            uint32_t before = seen, all = 0;
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) before += count[w];
                all += count[w];
            }
            if (is && before + __popcll(lanes & ((1ull << lane) - 1)) + 1 == P.ties) found[0] = i0 + tid + 1;
            seen += all;
            if (seen >= P.ties) break;                               // uniform
        }
        __syncthreads();
        tie_end = (int)found[0];
    }
    const double least = min_p ? (double)min_p[row] : 0.0;
    auto kept = [&](int i) -> uint64_t {
        const uint32_t key = key_of(x[i]);
        if (key < P.key || (key == P.key && (P.ties == 0 || i >= tie_end))) return 0;
        const double w = weight_of(key, S);
        return w >= least || i == top_index ? whole(w) : 0;
    };
    // the draw: ranges of indices, cut in sixteen until one is left
    int begin = 0, end = vocab;
    uint64_t left = 0, total = 0;
    while (end - begin > 64) {
        const int part = ((end - begin + kWaves - 1) / kWaves + 63) / 64 * 64;
        uint64_t sum = 0;
        const int b = begin + wave * part, e = min(end, b + part);
        for (int i = b + lane; i < e; i += 64) sum += kept(i);
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 0) red[wave] = sum;
        __syncthreads();
        if (total == 0) {
            for (int w = 0; w < kWaves; ++w) total += red[w];
            const double u = fmin(fmax((double)uniforms[row], 0.0), 1.0);
            left = min((uint64_t)(u * (double)total) + 1, total);    // the first index that brings the sum to this
        }
        int w = 0;
        while (w < kWaves - 1 && red[w] < left) left -= red[w++];
        begin += w * part;
        end = min(end, begin + part);
        __syncthreads();
    }
    if (wave == 0) {
        const bool in = begin + lane < end;
        uint64_t v = in ? kept(begin + lane) : 0, cum = v;
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t below = (uint64_t)__shfl_up((unsigned long long)cum, o);
            if (lane >= o) cum += below;
        }
        if (total == 0) {                                            // (a vocabulary of 64 or less)
            total = (uint64_t)__shfl((unsigned long long)cum, 63);
            const double u = fmin(fmax((double)uniforms[row], 0.0), 1.0);
            left = min((uint64_t)(u * (double)total) + 1, total);
        }
        const int at = __ffsll((unsigned long long)__ballot(in && cum >= left)) - 1;
        if (lane == at) {
            tokens[row] = begin + at;
            if (probabilities) probabilities[row] = (float)(weight_of(key_of(x[begin + at]), S) * kOne / (double)total);
        }
    }
}

}  // namespace

size_t sample_ws_bytes(int, int) { return 0; }

bool launch_sample(const float* logits, int64_t ld, int rows, int vocab, const float* uniforms, const float* temperature, const int32_t* top_k,
                   const float* top_p, const float* min_p, int32_t* tokens, float* probabilities, void*, hipStream_t stream)
{
    hipLaunchKernelGGL(sample_kernel, dim3(rows), dim3(kThreads), 0, stream, logits, ld, vocab, uniforms, temperature, top_k, top_p, min_p, tokens,
                       probabilities);
    return hip_ok(hipGetLastError(), "sample launch");
}

}  // namespace tship
