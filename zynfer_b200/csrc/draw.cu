// Draw of the next tokens of `rows` rows of logits from given random numbers,
// over the whole vocabulary and with a rule per row (zynfer_cu_sample_rows).
//
// Definition, for a row with the largest logit m, temperature T, top_k, top_p,
// min_p and the random number u:
//   weight   w_i = rint(exp((l_i - m) / T) 2^33), 0 where exp(..) < min_p and
//            for logits that are NaN or -inf;
//   order    descending logits, the lower index first among equals;
//   kept     of the first top_k (0: all) the shortest run whose weight sum
//            reaches top_p of theirs;
//   drawn    the first token of that order whose running sum exceeds
//            floor(u S), S the kept run's sum; its log-probability is
//            (l - m) / T - ln(S / 2^33).
// T <= 0 takes the largest logit. The weights are whole numbers, so every sum
// is exact and independent of its order: a parallel selection by sums gives
// the token that the sorted definition names, run after run. 2^33 keeps a
// weight of 2^-34 of the largest apart from 0 and the sum of 2^18 of them
// below 2^53, so products with top_p and u are single f64 roundings.
#include "common.cuh"
#include "kernels.h"

namespace zc {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / kWarp;

// Larger key = earlier in the order, equal logits (-0 and 0 among them) alike;
// 0 for NaN and -inf.
__device__ __forceinline__ uint32_t order_key(float l) {
    const unsigned long long k = argmax_key(l + 0.0f, 0u);
    return (uint32_t)(k >> 32);
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ float load_logit(const DrawArgs& a, size_t i) {
    return a.bf16 ? bf16lo(static_cast<const uint16_t*>(a.logits)[i]) : static_cast<const float*>(a.logits)[i];
}

__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, unsigned long long* sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    __syncthreads();
    if (threadIdx.x % kWarp == 0) sh[threadIdx.x / kWarp] = v;
    __syncthreads();
    v = sh[threadIdx.x % kWarp];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

struct RowRule {
    float m, inv_t, min_p;
    __device__ __forceinline__ float exponent(float l) const { return l == m ? 0.0f : (l - m) * inv_t; }
    __device__ __forceinline__ unsigned long long weight(uint32_t key) const {
        if (key == 0u) return 0ull;
        const float e = expf(exponent(key_logit(key)));
        return e >= min_p ? (unsigned long long)__float2ll_rn(e * 8589934592.0f) : 0ull;
    }
};

__global__ void __launch_bounds__(kThreads) draw_simple_kernel(DrawArgs a) {
    __shared__ unsigned long long sh[kWarps];
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x;
    const size_t base = (size_t)r * a.stride;
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = !(T > 0.0f);
    int k = greedy ? 1 : (a.top_k ? a.top_k[r] : 0);
    float p = a.top_p ? a.top_p[r] : 1.0f;
    if (!(p < 1.0f)) p = 1.0f;
    float min_p = a.min_p ? a.min_p[r] : 0.0f;
    min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
    float u = a.uniforms[r];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;

    // sum over the row of f(key)
    auto total = [&](auto f) {
        unsigned long long s = 0ull;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) s += f(order_key(load_logit(a, base + i)));
        return block_sum(s, sh);
    };
    // largest key K with sum over keys >= K of f(key) at least `want`
    auto select = [&](unsigned long long want, auto f) {
        uint32_t K = 0u;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t c = K | (1u << bit);
            if (total([&](uint32_t key) { return key >= c ? f(key) : 0ull; }) >= want) K = c;
        }
        return K;
    };
    const uint32_t top = select(1ull, [](uint32_t key) { return key ? 1ull : 0ull; });
    if (top == 0u) {  // nothing but NaN and -inf
        if (threadIdx.x == 0) {
            a.ids[r] = 0u;
            if (a.logprobs) a.logprobs[r] = -INFINITY;
        }
        return;
    }
    const RowRule rule{key_logit(top), greedy ? 1.0f : 1.0f / T, min_p};
    auto mass = [&](uint32_t key) { return rule.weight(key); };
    auto live = [&](uint32_t key) { return rule.weight(key) ? 1ull : 0ull; };
    unsigned long long S = total(mass);
    if (k > 0 && total(live) > (unsigned long long)k) {
        const uint32_t K = select((unsigned long long)k, live);
        const unsigned long long n = total([&](uint32_t key) { return key > K ? live(key) : 0ull; });
        S = total([&](uint32_t key) { return key > K ? mass(key) : 0ull; }) + ((unsigned long long)k - n) * rule.weight(K);
    }
    if (p < 1.0f) {
        const double reach = ceil((double)S * (double)p);
        const unsigned long long R = reach > 1.0 ? (unsigned long long)reach : 1ull;
        const uint32_t K = select(R, mass);
        const unsigned long long above = total([&](uint32_t key) { return key > K ? mass(key) : 0ull; });
        const unsigned long long w = rule.weight(K);
        S = above + (R - above + w - 1) / w * w;
    }
    unsigned long long t = (unsigned long long)((double)u * (double)S);
    if (t >= S) t = S - 1;
    const uint32_t K = select(t + 1, mass);
    const unsigned long long above = total([&](uint32_t key) { return key > K ? mass(key) : 0ull; });
    const unsigned long long nth = (t - above) / rule.weight(K);  // of the tokens with this logit, by index
    // index of that token: the smallest i with nth + 1 of them at or before it
    int lo = 0, hi = a.vocab - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        unsigned long long s = 0ull;
        for (int i = threadIdx.x; i <= mid; i += kThreads) s += order_key(load_logit(a, base + i)) == K;
        if (block_sum(s, sh) > nth) hi = mid;
        else lo = mid + 1;
    }
    if (threadIdx.x == 0) {
        a.ids[r] = (uint32_t)lo;
        if (a.logprobs) a.logprobs[r] = rule.exponent(key_logit(K)) - (float)log((double)S / 8589934592.0);
    }
}

}  // namespace

void launch_draw(const DrawArgs& a, cudaStream_t st) { launch_pdl(draw_simple_kernel, a.rows, kThreads, 0, st, a); }

void prepare_draw_kernels() { configure_kernel((const void*)draw_simple_kernel, 0); }

}  // namespace zc
