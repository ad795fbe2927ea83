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
//
// One pass over HBM: a cluster of C CTAs holds a row's logits in registers (E
// per thread, as order keys) and selects by sums.
//   1. the largest and smallest key of the row (one exchange over distributed
//      shared memory; top_k = 1 is done here);
//   2. every CTA adds its tokens' weights and counts into NB bins even in
//      (m - l) / T, between 0 and where weights end; the CTAs then take a slice
//      of the bins each, add up the C copies and scan them;
//   3. a question (the top_k-th token, the token where top_p is reached, the
//      drawn one) is answered by the bin that holds it, then by the tokens of
//      that bin alone, which all CTAs collect in a list and rank by counting.
//      A bin that holds more than the list (many equal logits) is divided
//      again, by (logit, index) itself, until it fits.
// What bounds it is the chain of exchanges and barriers, about ten of them,
// not the bytes; so a row is spread over 8 SMs and rows run side by side.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace zc {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / kWarp;
constexpr int kList = 512;        // tokens of a bin that are ranked by counting
constexpr float kOne = 8589934592.0f;  // 2^33, the weight of the largest logit
constexpr float kEnd = 23.6f;     // exp(-kEnd) 2^33 < 1/2: weights beyond are 0
constexpr int kIndexBits = 18;    // vocab <= 2^18
constexpr unsigned kAll = 0xFFFFFFFFu;
using u64 = unsigned long long;
static_assert(kDrawMaxVocab == 1 << kIndexBits, "composite keys");

// Larger key = earlier in the order, equal logits (-0 and 0 among them) alike;
// 0 for NaN and -inf.
__device__ __forceinline__ uint32_t order_key(float l) { return (uint32_t)(argmax_key(l + 0.0f, 0u) >> 32); }
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ float load_logit(const DrawArgs& a, size_t i) {
    return a.bf16 ? bf16lo(__ldg(static_cast<const uint16_t*>(a.logits) + i)) : __ldg(static_cast<const float*>(a.logits) + i);
}
// The place of a token in the order as one number: larger = earlier.
__device__ __forceinline__ u64 composite(uint32_t key, int idx) {
    return ((u64)key << kIndexBits) | (u64)((1 << kIndexBits) - 1 - idx);
}

struct RowRule {
    float m, inv_t, min_p;
    __device__ __forceinline__ float exponent(float l) const { return l == m ? 0.0f : (l - m) * inv_t; }
    __device__ __forceinline__ u64 weight_at(float x) const {
        const float e = expf(x);
        return e >= min_p ? (u64)__float2ll_rn(e * kOne) : 0ull;
    }
    __device__ __forceinline__ u64 weight(uint32_t key) const { return key ? weight_at(exponent(key_logit(key))) : 0ull; }
};

// What CTAs of a cluster tell one another.
struct Note {
    u64 a, b;
    uint32_t c, d;
};

template <int C>
struct Shared {
    static constexpr int NB = C == 1 ? 1024 : 4096;  // bins
    uint32_t count[NB], lo[NB], hi[NB];              // tokens, and their weights' low 17 and remaining bits
    u64 list_c[kList], list_w[kList];
    Note note[2][C];
    uint32_t list_n;                                  // of rank 0
    u64 scan_m[kWarps];
    uint32_t scan_c[kWarps], red_a[kWarps], red_b[kWarps], red_i[kWarps];
    u64 res[2];
};

__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t ld_rank(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_rank(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t add_rank(uint32_t addr, uint32_t v) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
}

template <int C, int E>
__global__ void __launch_bounds__(kThreads, 1) draw_kernel(const __grid_constant__ DrawArgs a) {
    using Sh = Shared<C>;
    constexpr int NB = Sh::NB, SLICE = NB / C;
    static_assert(SLICE <= kThreads, "a thread per bin of a slice");
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Sh& sh = *reinterpret_cast<Sh*>(smem_raw);
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const int rank = C == 1 ? 0 : blockIdx.x % C, r = blockIdx.x / C;
    int parity = 0;

    auto barrier = [&]() {
        if constexpr (C == 1) {
            __syncthreads();
        } else {
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
    };
    // every CTA's note (thread 0's) to every CTA; returns the slots
    auto exchange = [&](const Note& n) -> const Note* {
        Note* slots = sh.note[parity];
        parity ^= 1;
        if constexpr (C == 1) {
            if (tid == 0) slots[0] = n;
        } else if (warp == 0) {
            const u64 x = __shfl_sync(kAll, n.a, 0), y = __shfl_sync(kAll, n.b, 0);
            const uint32_t z = __shfl_sync(kAll, n.c, 0), w = __shfl_sync(kAll, n.d, 0);
            if (lane < C) {
                const uint32_t at = at_rank(&slots[rank], lane);
                st_rank(at, x);
                st_rank(at + 8, y);
                st_rank(at + 16, (u64)z | ((u64)w << 32));
            }
        }
        barrier();
        return slots;
    };

    for (int i = tid; i < NB; i += kThreads) sh.count[i] = sh.lo[i] = sh.hi[i] = 0u;
    if (tid == 0) sh.list_n = 0u;
    pdl_wait();
    pdl_launch_dependents();
    const float T = a.temperature ? a.temperature[r] : 1.0f;
    const bool greedy = !(T > 0.0f);
    const int k = greedy ? 1 : (a.top_k ? a.top_k[r] : 0);
    float p = a.top_p ? a.top_p[r] : 1.0f;
    if (!(p < 1.0f)) p = 1.0f;
    float min_p = a.min_p ? a.min_p[r] : 0.0f;
    min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
    float u = a.uniforms[r];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;

    // ---- the row: CTA `rank` holds [i0, i1), thread t the tokens i0 + 1024 e + t
    const int chunk = (a.vocab + C - 1) / C;
    const int i0 = rank * chunk + tid, i1 = min(a.vocab, (rank + 1) * chunk);
    uint32_t key[E];
    {
        const size_t base = (size_t)r * a.stride;
        float l[E];
#pragma unroll
        for (int e = 0; e < E; ++e) l[e] = i0 + e * kThreads < i1 ? load_logit(a, base + i0 + e * kThreads) : -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) key[e] = order_key(l[e]);
    }
    uint32_t top = 0u, least = 0xFFFFFFFFu, first = 0u;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (key[e] > top) {
            top = key[e];
            first = (uint32_t)(i0 + e * kThreads);
        }
        if (key[e]) least = min(least, key[e]);
    }
    auto warp_best = [&](uint32_t& t, uint32_t& f, uint32_t& m) {  // largest t with its least f, least m
        const uint32_t w = __reduce_max_sync(kAll, t);
        f = __reduce_min_sync(kAll, t == w ? f : 0xFFFFFFFFu);
        t = w;
        m = __reduce_min_sync(kAll, m);
    };
    warp_best(top, first, least);
    if (lane == 0) {
        sh.red_a[warp] = top;
        sh.red_i[warp] = first;
        sh.red_b[warp] = least;
    }
    __syncthreads();
    top = sh.red_a[lane];
    first = sh.red_i[lane];
    least = sh.red_b[lane];
    warp_best(top, first, least);
    {
        const Note* n = exchange(Note{top, first, least, 0u});
        const Note x = n[C == 1 ? 0 : lane % C];
        top = (uint32_t)x.a;
        first = (uint32_t)x.b;
        least = x.c;
        warp_best(top, first, least);
    }
    if (top == 0u || k == 1) {  // nothing but NaN and -inf; or the largest alone
        if (rank == 0 && tid == 0) {
            a.ids[r] = top ? first : 0u;
            if (a.logprobs) a.logprobs[r] = top ? 0.0f : -INFINITY;
        }
        return;
    }
    const RowRule rule{key_logit(top), greedy ? 1.0f : 1.0f / T, min_p};

    // ---- bins even in (m - l) / T, up to the last weight
    float end = fminf(-rule.exponent(key_logit(least)), kEnd);
    if (!(end >= 0.0f)) end = kEnd;
    if (min_p > 0.0f) end = fminf(end, 0.01f - logf(min_p));
    const float bin_scale = end > 0.0f ? (float)(NB - 1) / end : 0.0f;
    auto bin_at = [&](float x) { return min((int)(-x * bin_scale), NB - 1); };

    // Adds this CTA's tokens into the bins (bin0 >= 0: those of that bin between
    // c_hi and c_lo, into bins of 2^shift places) and scans the sums: thread
    // t < SLICE has bin rank SLICE + t.
    u64 mass_ex, mass, all_mass;
    uint32_t count_ex, count, all_count;
    u64 c_hi = ~0ull, c_lo = 0ull;
    int bin0 = -1, shift = 0;
    auto histogram = [&]() {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!key[e]) continue;
            const float x = rule.exponent(key_logit(key[e]));
            int b = bin_at(x);
            if (bin0 >= 0) {
                const u64 c = composite(key[e], i0 + e * kThreads);
                if (b != bin0 || c < c_lo || c > c_hi) continue;
                b = (int)((c_hi - c) >> shift);
            }
            const u64 w = rule.weight_at(x);
            if (w) {
                atomicAdd(&sh.count[b], 1u);
                atomicAdd(&sh.lo[b], (uint32_t)w & 0x1FFFFu);
                atomicAdd(&sh.hi[b], (uint32_t)(w >> 17));
            }
        }
        barrier();
        mass = 0ull;
        count = 0u;
        if (tid < SLICE) {
            const int b = rank * SLICE + tid;
            if constexpr (C == 1) {
                count = sh.count[b];
                mass = ((u64)sh.hi[b] << 17) + sh.lo[b];
            } else {
                uint32_t x[C], y[C], z[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint32_t at = at_rank(&sh.count[b], c);
                    x[c] = ld_rank(at);
                    y[c] = ld_rank(at + NB * 4);
                    z[c] = ld_rank(at + 2 * NB * 4);
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    count += x[c];
                    mass += ((u64)z[c] << 17) + y[c];
                }
            }
        }
        // scan over the CTA's slice
        u64 m = mass;
        uint32_t n = count;
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const u64 mm = __shfl_up_sync(kAll, m, o);
            const uint32_t nn = __shfl_up_sync(kAll, n, o);
            if (lane >= o) {
                m += mm;
                n += nn;
            }
        }
        if (lane == kWarp - 1) {
            sh.scan_m[warp] = m;
            sh.scan_c[warp] = n;
        }
        __syncthreads();
        u64 before_m = 0ull, cta_m = 0ull;
        uint32_t before_n = 0u, cta_n = 0u;
        {
            u64 x = sh.scan_m[lane];
            uint32_t y = sh.scan_c[lane];
            const u64 x0 = x;
            const uint32_t y0 = y;
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
                const u64 mm = __shfl_up_sync(kAll, x, o);
                const uint32_t nn = __shfl_up_sync(kAll, y, o);
                if (lane >= o) {
                    x += mm;
                    y += nn;
                }
            }
            before_m = __shfl_sync(kAll, x - x0, warp);
            before_n = __shfl_sync(kAll, y - y0, warp);
            cta_m = __shfl_sync(kAll, x, kWarp - 1);
            cta_n = __shfl_sync(kAll, y, kWarp - 1);
        }
        const Note* t = exchange(Note{cta_m, cta_n, 0u, 0u});  // (all bins are read)
        all_mass = 0ull;
        all_count = 0u;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c < rank) {
                before_m += t[c].a;
                before_n += (uint32_t)t[c].b;
            }
            all_mass += t[c].a;
            all_count += (uint32_t)t[c].b;
        }
        mass_ex = before_m + m - mass;
        count_ex = before_n + n - count;
    };

    // ---- the questions: where the running count (of top_k) or weight sum (of
    // top_p, of the draw) reaches `want`
    u64 S = 0ull, drawn = 0ull;
    int held = 0;  // bins: 0 clear, 1 of the whole row, 2 of a divided bin
    for (int q = 0; q < 3; ++q) {
        const bool by_mass = q > 0;
        u64 want = (u64)k;
        if (q > 0 && held) {
            if (q == 1) {
                if (!(p < 1.0f)) continue;
                const double reach = ceil((double)S * (double)p);
                want = reach > 1.0 ? (u64)reach : 1ull;
            } else {
                want = (u64)((double)u * (double)S);
                want = min(want, S - 1) + 1;
            }
        }
        u64 before_m = 0ull;
        uint32_t before_n = 0u;
        bin0 = -1;
        for (;;) {
            if (bin0 >= 0 || held != 1) {
                if (held) {
                    for (int i = tid; i < NB; i += kThreads) sh.count[i] = sh.lo[i] = sh.hi[i] = 0u;
                    __syncthreads();
                }
                histogram();
                held = bin0 < 0 ? 1 : 2;
                if (q == 0 && bin0 < 0) {
                    S = all_mass;
                    if (!(k > 0 && all_count > (uint32_t)k)) break;  // every token stays
                }
            }
            // the bin that holds it: only its thread speaks up
            const bool mine = tid < SLICE && (by_mass ? before_m + mass_ex < want && want <= before_m + mass_ex + mass
                                                      : before_n + count_ex < want && want <= before_n + count_ex + count);
            Note n{0ull, 0ull, 0u, 0u};
            if (mine) {
                sh.res[0] = mass_ex;
                sh.res[1] = ((u64)(uint32_t)(rank * SLICE + tid + 1) << 32) | count;
                sh.red_a[0] = count_ex;
            }
            const bool here = __syncthreads_or(mine);
            if (here) n = Note{sh.res[0], sh.res[1], sh.red_a[0], 1u};
            const Note* t = exchange(n);
            u64 m_ex = 0ull, bc = 0ull;
            uint32_t n_ex = 0u;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (t[c].d) {
                    m_ex = t[c].a;
                    bc = t[c].b;
                    n_ex = t[c].c;
                }
            const int b = (int)(bc >> 32) - 1;
            const uint32_t inside = (uint32_t)bc;
            auto chosen = [&](int e) {  // token e of this thread is in the bin
                if (!key[e]) return false;
                const u64 c = composite(key[e], i0 + e * kThreads);
                if (c < c_lo || c > c_hi) return false;
                return bin_at(rule.exponent(key_logit(key[e]))) == bin0;
            };
            before_m += m_ex;
            before_n += n_ex;
            if (bin0 < 0) {
                bin0 = b;
                c_hi = ~0ull;
                c_lo = 0ull;
            } else {
                // bin b of the composites c_hi down to c_lo
                const u64 hi = c_hi - ((u64)b << shift);
                c_lo = max(c_lo, hi - ((1ull << shift) - 1ull));
                c_hi = hi;
            }
            if (inside <= kList) {
                // collect the bin's tokens in every CTA's list, then rank them
                const uint32_t counter = C == 1 ? 0u : at_rank(&sh.list_n, 0);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (!chosen(e)) continue;
                    const u64 w = rule.weight(key[e]);
                    if (!w) continue;
                    const u64 c = composite(key[e], i0 + e * kThreads);
                    if constexpr (C == 1) {
                        const uint32_t s = atomicAdd(&sh.list_n, 1u);
                        sh.list_c[s] = c;
                        sh.list_w[s] = w;
                    } else {
                        const uint32_t s = add_rank(counter, 1u);
#pragma unroll
                        for (int q = 0; q < C; ++q) {
                            st_rank(at_rank(&sh.list_c[s], q), c);
                            st_rank(at_rank(&sh.list_w[s], q), w);
                        }
                    }
                }
                barrier();
                if (rank == 0 && tid == 0) sh.list_n = 0u;  // (added to again after the next exchange)
                for (uint32_t i = warp; i < inside; i += kWarps) {
                    const u64 c = sh.list_c[i], w = sh.list_w[i];
                    u64 m = 0ull;
                    uint32_t n2 = 0u;
                    for (uint32_t j = lane; j < inside; j += kWarp)
                        if (sh.list_c[j] > c) {
                            m += sh.list_w[j];
                            n2 += 1u;
                        }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(kAll, m, o);
                    n2 = __reduce_add_sync(kAll, n2);
                    m += before_m;
                    n2 += before_n;
                    if (by_mass ? m < want && want <= m + w : n2 + 1u == want) {
                        if (lane == 0) {
                            sh.scan_m[0] = c;
                            sh.scan_m[1] = m + w;
                        }
                    }
                }
                __syncthreads();
                drawn = sh.scan_m[0];
                if (q < 2) S = sh.scan_m[1];
                __syncthreads();
                break;
            }
            // too many: divide the bin by (logit, index) between its extremes
            u64 mx = 0ull, mn = ~0ull;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (chosen(e) && rule.weight(key[e])) {
                    const u64 c = composite(key[e], i0 + e * kThreads);
                    mx = max(mx, c);
                    mn = min(mn, c);
                }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                mx = max(mx, __shfl_xor_sync(kAll, mx, o));
                mn = min(mn, __shfl_xor_sync(kAll, mn, o));
            }
            __syncthreads();
            if (lane == 0) {
                sh.scan_m[warp] = mx;
                sh.list_c[warp] = mn;
            }
            __syncthreads();
            mx = sh.scan_m[lane];
            mn = sh.list_c[lane];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                mx = max(mx, __shfl_xor_sync(kAll, mx, o));
                mn = min(mn, __shfl_xor_sync(kAll, mn, o));
            }
            const Note* x = exchange(Note{mx, mn, 0u, 0u});
#pragma unroll
            for (int c = 0; c < C; ++c) {
                mx = max(mx, x[c].a);
                mn = min(mn, x[c].b);
            }
            c_hi = mx;
            c_lo = mn;
            shift = max(0, 64 - __clzll((long long)(c_hi - c_lo)) - (C == 1 ? 10 : 12));
        }
    }
    if (rank == 0 && tid == 0) {
        a.ids[r] = (uint32_t)((1 << kIndexBits) - 1) - (uint32_t)(drawn & ((1u << kIndexBits) - 1u));
        if (a.logprobs)
            a.logprobs[r] = rule.exponent(key_logit((uint32_t)(drawn >> kIndexBits))) - (float)log((double)S / (double)kOne);
    }
}

template <int C, int E>
void launch(const DrawArgs& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared<C>);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C == 1 ? 1 : 2;
    cudaLaunchKernelEx(&cfg, draw_kernel<C, E>, a);
}

template <int C, int E>
void prepare() {
    configure_kernel((const void*)draw_kernel<C, E>, sizeof(Shared<C>));
}

}  // namespace

void launch_draw(const DrawArgs& a, cudaStream_t st) {
    if (a.vocab <= 4 * kThreads) launch<1, 4>(a, st);
    else if (a.vocab <= 16 * kThreads) launch<1, 16>(a, st);
    else if (a.vocab <= 8 * 8 * kThreads) launch<8, 8>(a, st);
    else if (a.vocab <= 8 * 20 * kThreads) launch<8, 20>(a, st);
    else launch<8, 32>(a, st);
}

void prepare_draw_kernels() {
    prepare<1, 4>();
    prepare<1, 16>();
    prepare<8, 8>();
    prepare<8, 20>();
    prepare<8, 32>();
}

}  // namespace zc
