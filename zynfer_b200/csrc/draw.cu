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
// A cluster of C CTAs takes a row, each CTA its C-th part, and selects by sums. It
// goes over the row for its range, for the bins and once for each question, the
// first time from HBM and then from shared memory or, mostly, L2.
//   1. the largest and smallest logit of the row (one exchange over distributed
//      shared memory);
//   2. every CTA adds its tokens' weights (and counts) into NB bins even in
//      (m - l) / T, from 0 to where weights end; the CTAs then take a slice of
//      the bins each, add up the C copies and scan them;
//   3. a question (the top_k-th token, the token where top_p is reached, the
//      drawn one) is answered by the bin that holds it, then by the tokens of
//      that bin, which all CTAs send to the first, where they are sorted and
//      their weights scanned. A bin of more tokens than that list holds (many
//      equal logits) is divided again, by (logit, index) itself, until it fits.
// A few rows are bound by the chain of loads, exchanges and barriers (20 us for
// one row of 151936), many rows by the instructions per logit (about 55, an
// accurate exponential among them), not by the bytes. So a row has the more CTAs
// the fewer rows there are: 16 for up to 4, 8 for up to 37, then 4, 2 and 1 (256
// rows of bf16, calls overlapping: 123 us a call with one CTA a row against 206 with
// eight, whose barriers left the SMs idle; 88 with half the instructions since, and
// 116 one after another on a stream); weights are
// split into two 32-bit words without integer conversions; and two CTAs share an
// SM. Eight CTAs or more hold their parts of a row in shared memory, fewer read
// them again from L2.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace zc {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / kWarp;
constexpr int kList = kThreads;        // tokens of a bin that are sorted
constexpr float kOne = 8589934592.0f;  // 2^33, the weight of the largest logit
constexpr float kEnd = 23.6f;          // exp(-kEnd) 2^33 < 1/2: weights beyond are 0
constexpr float kTiny = 1e-30f;        // exp(-kTiny) is 1
constexpr int kIndexBits = 18;         // vocab <= 2^18
constexpr float kMagic = 8388608.0f;   // 2^23: x + 2^23 holds rint(x) in its low bits
constexpr unsigned kAll = 0xFFFFFFFFu;
using u64 = unsigned long long;
static_assert(kDrawMaxVocab == 1 << kIndexBits, "composite keys");

// The place of a token in the order as one number: larger = earlier.
__device__ __forceinline__ u64 composite(float l, int idx) {
    return ((argmax_key(l + 0.0f, 0u) >> 32) << kIndexBits) | (u64)((1 << kIndexBits) - 1 - idx);  // (-0 is 0)
}
__device__ __forceinline__ float composite_logit(u64 c) {
    const uint32_t k = (uint32_t)(c >> kIndexBits);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// rint(e 2^33) = hi 2^17 + lo, lo in [-2^16, 2^16]: both parts by adding 2^23
// (1.5 2^23 for the signed one). e 2^16 and the remainder are exact, and hi 2^17
// is even, so rounding the remainder alone rounds the whole the same way. The
// sums of kBatch such words fit 32 bits.
struct Weight {
    uint32_t hi;
    int lo;
    __device__ __forceinline__ u64 whole() const { return ((u64)hi << 17) + (u64)(long long)lo; }
};

struct RowRule {
    float m, inv_t, end, bin_scale;
    float least;  // the smallest exponential with weight: min_p, or the float after 2^-34 (which rounds to 0)
    bool odd;     // m is infinite: l - m is not 0 where l is m
    __device__ __forceinline__ float exponent(float l) const {
        const float d = l - m;
        return (odd && l == m ? 0.0f : d) * inv_t;
    }
    // (0 <= fminf(-x, end) <= end, which bin_scale takes to NB - 1; `last` holds it there whatever x is)
    __device__ __forceinline__ int bin(float x, int last) const {
        return (int)min((uint32_t)(__float_as_int(__fmaf_rn(fminf(-x, end), bin_scale, kMagic)) - 0x4B000000), (uint32_t)last);
    }
    // does a token of exponential e weigh anything? (NaN does not)
    __device__ __forceinline__ bool weighs(float e) const { return e >= least; }
    __device__ __forceinline__ Weight weight(float e) const {
        const float s = e * 65536.0f, t = s + kMagic;
        return Weight{(uint32_t)(__float_as_int(t) - 0x4B000000),
                      __float_as_int(__fmaf_rn(s - (t - kMagic), 131072.0f, 12582912.0f)) - 0x4B400000};
    }
};

// What CTAs of a cluster tell one another.
struct Note {
    u64 a, b;
    uint32_t c, d;
};

// HOLD: the row's part stays in shared memory (of at most kBatch tokens);
// otherwise it is read again, and the bins' 32-bit sums are carried over into
// 64-bit ones every kBatch tokens.
constexpr int kBatch = (1 << 15) - 2;
template <int NB, bool HOLD>
struct Bins {
    uint32_t count[NB], hi[NB];  // tokens, and their weights' parts
    int lo[NB];
};
template <int NB>
struct Bins<NB, false> {
    uint32_t count[NB], hi[NB];
    int lo[NB];
    u64 mass[NB];
};
template <int C, bool HOLD>
struct Shared {
    static constexpr int NB_LOG = C == 1 && HOLD ? 9 : 11, NB = 1 << NB_LOG;  // bins
    Bins<NB, HOLD> bins;
    u64 list[kList];
    Note note[2][C];
    uint32_t list_n;  // of rank 0
    u64 scan_m[kWarps], scan_x[kWarps], res[3];
    uint32_t scan_c[kWarps];
    float red_a[kWarps], red_b[kWarps];
    alignas(16) float row[1];  // HOLD: this CTA's logits
};
template <int C, bool HOLD>
constexpr size_t smem_bytes(int chunk) {
    return sizeof(Shared<C, HOLD>) + (HOLD ? (size_t)chunk * sizeof(float) : 0);
}

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
__device__ __forceinline__ u64 ld_rank64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
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
__device__ __forceinline__ u64 warp_scan(u64 v) {
#pragma unroll
    for (int o = 1; o < kWarp; o <<= 1) {
        const u64 x = __shfl_up_sync(kAll, v, o);
        if ((int)(threadIdx.x % kWarp) >= o) v += x;
    }
    return v;
}

template <int C, bool HOLD>
__global__ void __launch_bounds__(kThreads, 2) draw_kernel(const __grid_constant__ DrawArgs a) {
    using Sh = Shared<C, HOLD>;
    constexpr int NB = Sh::NB, SLICE = NB / C, PER = SLICE > kThreads ? SLICE / kThreads : 1;  // bins: of a CTA, of a thread
    static_assert(PER * kThreads == SLICE || PER == 1, "bins of a slice");
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
    // every CTA's note (thread 0's) to every CTA; returns the slots. Two sets of
    // slots in turn: a set is written again only after everyone passed the
    // barrier behind its reading.
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
    auto clear_bins = [&]() {
        for (int i = tid; i < NB; i += kThreads) {
            sh.bins.count[i] = sh.bins.hi[i] = 0u;
            sh.bins.lo[i] = 0;
            if constexpr (!HOLD) sh.bins.mass[i] = 0ull;
        }
    };

    // no CTA writes into another before that one runs: this barrier's other half
    // is in front of the first exchange
    if constexpr (C > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    }
    clear_bins();
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

    // ---- the row: this CTA holds tokens i0 .. i0 + n - 1 (chunk is even)
    const int i0 = min(a.vocab, rank * a.chunk), n = min(a.vocab, i0 + a.chunk) - i0;
    const size_t base = (size_t)r * a.stride + i0;
    // f(logit, i) for this CTA's tokens i0 + i, i in [from, to), kAhead loads before any is used
    auto from_memory = [&](int from, int to, auto f) {
        constexpr int kAhead = 8;
        const uint16_t* half = static_cast<const uint16_t*>(a.logits) + base;
        if (a.bf16 && reinterpret_cast<uintptr_t>(half) % 4 == 0) {
            const uint32_t* two = reinterpret_cast<const uint32_t*>(half);
            const int end = to / 2;  // (from is even)
            int j = from / 2 + tid;
            for (; j + (kAhead - 1) * kThreads < end; j += kAhead * kThreads) {
                uint32_t x[kAhead];
#pragma unroll
                for (int v = 0; v < kAhead; ++v) x[v] = __ldg(two + j + v * kThreads);
#pragma unroll
                for (int v = 0; v < kAhead; ++v) {
                    f(bf16lo(x[v]), 2 * (j + v * kThreads));
                    f(bf16hi(x[v]), 2 * (j + v * kThreads) + 1);
                }
            }
#pragma unroll 1
            for (; j < end; j += kThreads) {
                const uint32_t x = __ldg(two + j);
                f(bf16lo(x), 2 * j);
                f(bf16hi(x), 2 * j + 1);
            }
            if ((to & 1) && tid == 0) f(bf16lo(__ldg(half + to - 1)), to - 1);
        } else if (a.bf16) {
#pragma unroll 4
            for (int i = from + tid; i < to; i += kThreads) f(bf16lo(__ldg(half + i)), i);
        } else {
            const float* src = static_cast<const float*>(a.logits) + base;
            int j = from + tid;
            for (; j + (kAhead - 1) * kThreads < to; j += kAhead * kThreads) {
                float x[kAhead];
#pragma unroll
                for (int v = 0; v < kAhead; ++v) x[v] = __ldg(src + j + v * kThreads);
#pragma unroll
                for (int v = 0; v < kAhead; ++v) f(x[v], j + v * kThreads);
            }
#pragma unroll 4
            for (; j < to; j += kThreads) f(__ldg(src + j), j);
        }
    };
    auto each = [&](int from, int to, auto f) {
        if constexpr (HOLD) {
#pragma unroll 4
            for (int i = from + tid; i < to; i += kThreads) f(sh.row[i], i);
        } else {
            from_memory(from, to, f);
        }
    };
    float top = -INFINITY, least = INFINITY;
    from_memory(0, n, [&](float l, int i) {
        if constexpr (HOLD) sh.row[i] = l;
        top = fmaxf(top, l);  // (NaN is passed over)
        least = fminf(least, l);
    });
    auto warp_range = [&]() {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
            least = fminf(least, __shfl_xor_sync(kAll, least, o));
        }
    };
    warp_range();
    if (lane == 0) {
        sh.red_a[warp] = top;
        sh.red_b[warp] = least;
    }
    __syncthreads();
    top = sh.red_a[lane % kWarps];
    least = sh.red_b[lane % kWarps];
    warp_range();
    if constexpr (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    {
        const Note* x = exchange(Note{0ull, 0ull, __float_as_uint(top), __float_as_uint(least)});
        top = __uint_as_float(x[lane % C].c);
        least = __uint_as_float(x[lane % C].d);
        warp_range();
    }
    if (top == -INFINITY) {  // nothing but NaN and -inf
        if (rank == 0 && tid == 0) {
            a.ids[r] = 0u;
            if (a.logprobs) a.logprobs[r] = -INFINITY;
        }
        return;
    }
    if (k == 1) {  // the first of the largest
        uint32_t first = 0xFFFFFFFFu;
        each(0, n, [&](float l, int i) {
            if (l == top) first = min(first, (uint32_t)(i0 + i));
        });
        first = __reduce_min_sync(kAll, first);
        if (lane == 0) sh.scan_c[warp] = first;
        __syncthreads();
        first = __reduce_min_sync(kAll, sh.scan_c[lane % kWarps]);
        const Note* x = exchange(Note{0ull, 0ull, first, 0u});
        first = __reduce_min_sync(kAll, x[lane % C].c);
        if (rank == 0 && tid == 0) {
            a.ids[r] = first;
            if (a.logprobs) a.logprobs[r] = 0.0f;
        }
        return;
    }

    // ---- bins even in (m - l) / T, up to the last weight
    // (1 / T beyond the floats: the largest of them, as for a temperature of 2^-128)
    RowRule rule{top, fminf(1.0f / T, 3.402823466e38f), 0.0f, 0.0f, fmaxf(min_p, 5.8207667e-11f), top == INFINITY};
    rule.end = fminf(-rule.exponent(least), kEnd);  // (with a logit of -inf in the row: where weights end)
    if (!(rule.end >= 0.0f)) rule.end = kEnd;
    if (min_p > 0.0f) rule.end = fminf(rule.end, 0.01f - logf(min_p));
    // (a range below kTiny weighs one, and its bins' scale could leave the floats: one bin, which the order divides)
    rule.bin_scale = rule.end > kTiny ? (float)(NB - 1) / rule.end : 0.0f;
    const bool counts = k > 0;

    // Adds this CTA's tokens into the bins (bin0 >= 0: those of that bin between
    // c_hi and c_lo, into bins of 2^shift places) and scans the sums: thread t has
    // bins rank SLICE + PER t .. of the whole row.
    u64 mass_ex = 0ull, mass[PER], all_mass, c_hi = ~0ull, c_lo = 0ull;
    uint32_t count_ex = 0u, count[PER], all_count;
    int bin0 = -1, shift = 0;
    auto histogram = [&]() {
        const bool counted = counts || bin0 >= 0;
        for (int from = 0; from < n; from += kBatch) {
            each(from, min(n, from + kBatch), [&](float l, int i) {
                const float x = rule.exponent(l), e = expf(x);
                int b = rule.bin(x, NB - 1);
                if (bin0 >= 0) {
                    if (b != bin0) return;
                    const u64 c = composite(l, i0 + i);
                    if (c < c_lo || c > c_hi) return;
                    b = (int)((c_hi - c) >> shift);
                }
                if (rule.weighs(e)) {
                    const Weight w = rule.weight(e);
                    atomicAdd(&sh.bins.hi[b], w.hi);
                    atomicAdd(&sh.bins.lo[b], w.lo);
                    if (counted) atomicAdd(&sh.bins.count[b], 1u);
                }
            });
            if constexpr (!HOLD) {
                __syncthreads();
                for (int i = tid; i < NB; i += kThreads) {
                    sh.bins.mass[i] += ((u64)sh.bins.hi[i] << 17) + (u64)(long long)sh.bins.lo[i];
                    sh.bins.hi[i] = 0u;
                    sh.bins.lo[i] = 0;
                }
                __syncthreads();
            }
        }
        barrier();
        u64 own_mass = 0ull;
        uint32_t own_count = 0u;
#pragma unroll
        for (int k2 = 0; k2 < PER; ++k2) {
            mass[k2] = 0ull;
            count[k2] = 0u;
            if (PER * tid < SLICE) {
                const int b = rank * SLICE + PER * tid + k2;
                uint32_t x[C], y[C], z[C];
                u64 s[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    x[c] = ld_rank(at_rank(&sh.bins.count[b], c));
                    if constexpr (HOLD) {
                        y[c] = ld_rank(at_rank(&sh.bins.hi[b], c));
                        z[c] = ld_rank(at_rank(&sh.bins.lo[b], c));
                    } else {
                        s[c] = ld_rank64(at_rank(&sh.bins.mass[b], c));
                    }
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    count[k2] += x[c];
                    mass[k2] += HOLD ? ((u64)y[c] << 17) + (u64)(long long)(int)z[c] : s[c];
                }
            }
            own_mass += mass[k2];
            own_count += count[k2];
        }
        const u64 m = warp_scan(own_mass), nn = warp_scan(own_count);
        if (lane == kWarp - 1) {
            sh.scan_m[warp] = m;
            sh.scan_c[warp] = (uint32_t)nn;
        }
        __syncthreads();
        const u64 x0 = lane < kWarps ? sh.scan_m[lane] : 0ull, y0 = lane < kWarps ? sh.scan_c[lane] : 0u;
        const u64 x = warp_scan(x0), y = warp_scan(y0);
        u64 before_m = __shfl_sync(kAll, x - x0, warp), before_n = __shfl_sync(kAll, y - y0, warp);
        const Note* t = exchange(Note{__shfl_sync(kAll, x, kWarp - 1), __shfl_sync(kAll, y, kWarp - 1), 0u, 0u});  // (all bins are read)
        all_mass = 0ull;
        all_count = 0u;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (c < rank) {
                before_m += t[c].a;
                before_n += t[c].b;
            }
            all_mass += t[c].a;
            all_count += (uint32_t)t[c].b;
        }
        mass_ex = before_m + m - own_mass;
        count_ex = (uint32_t)(before_n + nn) - own_count;
    };

    // ---- the questions: where the running count (of top_k) or weight sum (of
    // top_p, of the draw) reaches `want`. S becomes the sum up to and with that
    // token.
    u64 S = 0ull, drawn = 0ull;
    int held = 0;  // bins: 0 clear, 1 of the whole row, 2 of a divided bin
    for (int q = 0; q < 3; ++q) {
        const bool by_mass = q > 0;
        u64 want = (u64)(uint32_t)k;
        if (q == 1) {
            if (!(p < 1.0f)) continue;
            const double reach = ceil((double)S * (double)p);
            want = reach > 1.0 ? (u64)reach : 1ull;
        } else if (q == 2) {
            want = min((u64)((double)u * (double)S), S - 1) + 1;
        }
        u64 before_m = 0ull;
        uint32_t before_n = 0u;
        bin0 = -1;
        for (;;) {
            if (bin0 >= 0 || held != 1) {
                if (held) {
                    clear_bins();
                    __syncthreads();
                }
                histogram();
                held = bin0 < 0 ? 1 : 2;
                if (q == 0 && bin0 < 0) {
                    S = all_mass;
                    if (!(counts && all_count > (uint32_t)k)) break;  // every token stays
                }
            }
            // the bin that holds it: only its thread speaks up
            bool mine = false;
            {
                u64 m_ex = mass_ex;
                uint32_t n_ex = count_ex;
#pragma unroll
                for (int k2 = 0; k2 < PER; ++k2) {
                    if (by_mass ? before_m + m_ex < want && want <= before_m + m_ex + mass[k2]
                                : before_n + n_ex < want && want <= before_n + n_ex + count[k2]) {
                        mine = true;
                        sh.res[0] = m_ex;
                        sh.res[1] = ((u64)(uint32_t)(rank * SLICE + PER * tid + k2 + 1) << 32) | count[k2];
                        sh.res[2] = n_ex;
                    }
                    m_ex += mass[k2];
                    n_ex += count[k2];
                }
            }
            const bool here = __syncthreads_or(mine);
            Note note{0ull, 0ull, 0u, 0u};
            if (here) note = Note{sh.res[0], sh.res[1], (uint32_t)sh.res[2], 1u};
            const Note* t = exchange(note);
            u64 bc = 0ull;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (t[c].d) {
                    before_m += t[c].a;
                    bc = t[c].b;
                    before_n += t[c].c;
                }
            const int b = (int)(bc >> 32) - 1;
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
            // the bin's logits lie between these (a bin's width, of the 1 / T that the
            // exponents take, and a few roundings of slack, those of a width below the
            // normal numbers among them): a comparison leaves few tokens to look at closely
            const float width = rule.bin_scale > 0.0f ? (1.0f / rule.bin_scale) / rule.inv_t : INFINITY;
            const float slack = width + 1e-6f * fabsf(top) + 1e-41f;
            const float l_hi = bin0 < 2 ? INFINITY : top - ((float)bin0 * width - slack) * (1.0f - 1e-6f);
            const float l_lo = bin0 >= NB - 2 ? -INFINITY : top - ((float)bin0 * width + slack) * (1.0f + 1e-6f);
            u64 mx = 0ull, mn = ~0ull;
            uint32_t sent = 0u;
            // f(place, its logit) of each of this CTA's tokens in the bin
            auto chosen = [&](auto f) {
                each(0, n, [&](float l, int i) {
                    if (!(l <= l_hi) || l < l_lo) return;
                    const float x = rule.exponent(l);
                    if (rule.bin(x, NB - 1) != bin0 || !rule.weighs(expf(x))) return;
                    const u64 c = composite(l, i0 + i);
                    if (c >= c_lo && c <= c_hi) f(c);
                });
            };
            const bool counted = counts || held == 2;
            const uint32_t counter = C == 1 ? 0u : at_rank(&sh.list_n, 0), list = C == 1 ? 0u : at_rank(sh.list, 0);
            const bool fits = counted && (uint32_t)bc <= kList;
            if (!counted || fits) {
                // to the first CTA's list, as far as it goes
                chosen([&](u64 c) {
                    if constexpr (C == 1) {
                        const uint32_t s = atomicAdd(&sh.list_n, 1u);
                        if (s < kList) sh.list[s] = c;
                    } else {
                        const uint32_t s = add_rank(counter, 1u);
                        if (s < kList) st_rank(list + 8 * s, c);
                    }
                });
                barrier();
                sent = C == 1 ? sh.list_n : ld_rank(counter);
            }
            if (fits || (!counted && sent <= kList)) {
                if (rank == 0) {
                    // sort the list (largest first), scan the weights
                    const uint32_t len = sent;
                    int size2 = kWarp;
                    while (size2 < (int)len) size2 <<= 1;
                    u64 c = tid < (int)len ? sh.list[tid] : 0ull;
                    for (int size = 2; size <= size2; size <<= 1)
                        for (int stride = size >> 1; stride > 0; stride >>= 1) {
                            u64 other;
                            if (stride < kWarp) {
                                other = __shfl_xor_sync(kAll, c, stride);
                            } else {
                                __syncthreads();
                                sh.list[tid] = c;
                                __syncthreads();
                                other = sh.list[tid ^ stride];
                            }
                            const bool larger = ((tid & size) == 0) == ((tid & stride) == 0);
                            c = larger ? max(c, other) : min(c, other);
                        }
                    const float l = composite_logit(c);
                    const u64 w = c ? rule.weight(expf(rule.exponent(l))).whole() : 0ull;
                    const u64 m = warp_scan(w);
                    if (lane == kWarp - 1) sh.scan_x[warp] = m;
                    __syncthreads();
                    const u64 x0 = lane < kWarps ? sh.scan_x[lane] : 0ull;
                    const u64 upto = before_m + m + __shfl_sync(kAll, warp_scan(x0) - x0, warp);
                    if (c && (by_mass ? upto - w < want && want <= upto : before_n + (uint32_t)tid + 1u == (uint32_t)want)) {
                        sh.res[0] = upto;
                        sh.res[1] = c;
                    }
                    __syncthreads();
                }
                if (q < 2) {
                    S = exchange(Note{sh.res[0], 0ull, 0u, 0u})[0].a;
                    if (rank == 0 && tid == 0) sh.list_n = 0u;  // (every CTA has read it)
                } else {
                    if constexpr (C > 1) barrier();  // no CTA leaves while its counter may be read
                    if (rank == 0) drawn = sh.res[1];
                }
                break;
            }
            // too many: divide the bin by (logit, index) between its extremes
            chosen([&](u64 c) {
                mx = max(mx, c);
                mn = min(mn, c);
            });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                mx = max(mx, __shfl_xor_sync(kAll, mx, o));
                mn = min(mn, __shfl_xor_sync(kAll, mn, o));
            }
            __syncthreads();
            if (lane == 0) {
                sh.scan_m[warp] = mx;
                sh.scan_x[warp] = mn;
            }
            __syncthreads();
            mx = sh.scan_m[lane % kWarps];
            mn = sh.scan_x[lane % kWarps];
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
            if (rank == 0 && tid == 0) sh.list_n = 0u;  // (every CTA has read it)
            c_hi = mx;
            c_lo = mn;
            shift = max(0, 64 - __clzll((long long)(c_hi - c_lo)) - Sh::NB_LOG);
        }
    }
    if (rank == 0 && tid == 0) {
        a.ids[r] = (uint32_t)((1 << kIndexBits) - 1) - (uint32_t)(drawn & ((1u << kIndexBits) - 1u));
        if (a.logprobs) a.logprobs[r] = rule.exponent(composite_logit(drawn)) - (float)log((double)S / (double)kOne);
    }
}

template <int C, bool HOLD>
cudaLaunchConfig_t config(const DrawArgs& a, cudaLaunchAttribute* attr, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem_bytes<C, HOLD>(a.chunk);
    cfg.stream = st;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = C;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C == 1 ? 1 : 2;
    return cfg;
}

template <int C, bool HOLD>
void launch(DrawArgs a, cudaStream_t st) {
    a.chunk = (((a.vocab + C - 1) / C) + 1) & ~1;
    cudaLaunchAttribute attr[2];
    const cudaLaunchConfig_t cfg = config<C, HOLD>(a, attr, st);
    cudaLaunchKernelEx(&cfg, draw_kernel<C, HOLD>, a);
}

constexpr int kOneCta = 16384;  // largest vocabulary that one CTA holds
// A few rows of a large vocabulary take 16 CTAs each (one row of 151936: 19.8 us
// against 22.1 with 8; 4 rows 24.9 / 27.8; but 8 rows 30.7 / 27.9, and one row of
// 32000 17.0 / 16.6). Clusters of 16 are more than every GPU must offer.
constexpr int kWideRows = 4, kWideVocab = 65536;
bool wide_clusters_fit() {
    static int fit[64] = {0};  // by device: 0 not asked, 1 yes, 2 no
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return false;
    if (!fit[dev]) {
        DrawArgs a{};
        a.rows = 1;
        a.chunk = kDrawMaxVocab / 16;
        cudaLaunchAttribute attr[2];
        const cudaLaunchConfig_t cfg = config<16, true>(a, attr, nullptr);
        int n = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, draw_kernel<16, true>, &cfg);
        if (e != cudaSuccess) cudaGetLastError();
        fit[dev] = e == cudaSuccess && n >= kWideRows ? 1 : 2;
    }
    return fit[dev] == 1;
}

}  // namespace

// Two CTAs fit an SM: with the largest C whose CTAs run all at once, every SM
// has work and a row's barriers are few.
void launch_draw(const DrawArgs& a, cudaStream_t st) {
    const int slots = 2 * device_sm_count();
    if (a.vocab <= kOneCta) launch<1, true>(a, st);
    else if (a.rows <= kWideRows && a.vocab > kWideVocab && wide_clusters_fit()) launch<16, true>(a, st);
    else if (8 * a.rows <= slots && a.vocab <= 8 * kBatch) launch<8, true>(a, st);
    else if (4 * a.rows <= slots) launch<4, false>(a, st);
    else if (2 * a.rows <= slots) launch<2, false>(a, st);
    else launch<1, false>(a, st);
}

void prepare_draw_kernels() {
    configure_kernel((const void*)draw_kernel<1, true>, smem_bytes<1, true>(kOneCta));
    configure_kernel((const void*)draw_kernel<16, true>, smem_bytes<16, true>(kDrawMaxVocab / 16));
    cudaFuncSetAttribute(draw_kernel<16, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    wide_clusters_fit();  // (asked now, never during a graph capture)
    configure_kernel((const void*)draw_kernel<8, true>, smem_bytes<8, true>(kBatch));
    configure_kernel((const void*)draw_kernel<4, false>, smem_bytes<4, false>(0));
    configure_kernel((const void*)draw_kernel<2, false>, smem_bytes<2, false>(0));
    configure_kernel((const void*)draw_kernel<1, false>, smem_bytes<1, false>(0));
}

}  // namespace zc
