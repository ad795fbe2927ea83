// Pieces of the serving attention kernels (serve_attn.cu, attn_tile.cu): which
// cache blocks a query sees, partial results, and one row taken position by
// position.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace zc {
namespace serve {

constexpr int kD = 128, kG = 2;  // head dim, query heads per kv head
constexpr int kBlockElems = kKvBlock * kD;
constexpr float kLog2e = 1.4426950408889634f;
// A partial result of one query head: reference point (log2 units) and sum of
// its exponentials, a count (below) and a word of padding, the weighted sum of V.
constexpr int kRecord = kServeRecord;
static_assert(kRecord == kD + 4, "record: m, l, -, -, acc");

// A kernel parameter as ordinary memory: indexed by lane, constant-bank loads
// would be taken one index after another.
template <typename T>
__device__ __forceinline__ const T& as_memory(const T& param) {
    const T* p = &param;
    asm volatile("" : "+l"(p));
    return *p;
}

// First position inside the window of a query at `pos` (pos + 1: none).
__host__ __device__ __forceinline__ int window_low(int pos, uint32_t window) {
    const long long low = (long long)pos - (long long)window + 1;
    return low > 0 ? (int)low : 0;
}

// The cache blocks that queries at positions p0 .. p1 see, in order: the
// sinks' first nsb blocks, then those from the window's start on.
struct Span {
    int nsb, off, total;
    __host__ __device__ __forceinline__ int block(int v) const { return v < nsb ? v : v + off; }
};
__host__ __device__ __forceinline__ Span span_of(int p0, int p1, uint32_t window, int sinks, int skip) {
    const int end = p1 / kKvBlock + 1;
    const int s = sinks < p1 + 1 ? sinks : p1 + 1;
    const int nsb = (s + kKvBlock - 1) / kKvBlock;
    int wb = window ? window_low(p0, window) / kKvBlock : end;
    if (skip > 0) return Span{0, skip, end > skip ? end - skip : 0};
    if (wb <= nsb) return Span{0, 0, window ? end : nsb};
    return Span{nsb, wb - nsb, nsb + end - wb};
}

// Bit c: the query at `pos` with window start `low` sees position 16 block + c.
__device__ __forceinline__ uint32_t first_bits(int n) { return n >= 16 ? 0xFFFFu : (n <= 0 ? 0u : (1u << n) - 1u); }
__device__ __forceinline__ uint32_t seen_bits(int block, int pos, int low, int sinks) {
    const int base = block * kKvBlock;
    return first_bits(pos + 1 - base) & (first_bits(sinks - base) | ~first_bits(low - base));
}

// 2^x (flushing results below 2^-126): the tensor-core kernels' exponential.
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two f32 -> packed bf16x2 (x0 in the low half), round to nearest even.
__device__ __forceinline__ uint32_t pack_bf16(float x0, float x1) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x1), "f"(x0));
    return r;
}
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// mbar_wait_bounded with the barrier tried once in line: most are complete when they
// are asked for, and the loop costs such a wait 245 cycles (the tile kernel's MMA
// thread, which waits three times per tile) where one try costs 41.
static __device__ __noinline__ bool mbar_wait_loop(uint64_t* bar, uint32_t parity, uint32_t* err) {
    return mbar_wait_bounded(bar, parity, err);
}
__device__ __forceinline__ bool mbar_wait_try(uint64_t* bar, uint32_t parity, uint32_t* err) {
    return mbar_try_wait(bar, parity) || mbar_wait_loop(bar, parity, err);
}

// A partial result of one query head held by a warp: lane l has dims 4 l ..
// 4 l + 3.
struct Partial {
    float m, l, acc[4];
};
using SlowRow = Partial;
__device__ __forceinline__ Partial no_partial() { return Partial{-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}}; }

// x joined with `cnt` records in global memory, in order: 2^(m - M) weighs each. A
// record of nothing seen is m = -inf with zeros; one of NaN scores alone is m = -inf
// with l NaN, and that goes into the sum as a NaN or infinity does whose weight is 0.
// Lane j reads the (m, l) of record j and weighs it, so a batch of up to 32
// costs one exponential and, with kAhead accumulators requested before any is
// used, about cnt / kAhead round trips.
// counted >= 0: record `counted` says how many there are from it on.
__device__ __forceinline__ void join_records(Partial& x, const float* base, int cnt, int counted = -1) {
    const int lane = threadIdx.x % kWarp;
    if (counted >= 0) cnt = counted + __ldcg(reinterpret_cast<const int*>(base + (size_t)counted * kRecord + 2));
    constexpr int kAhead = 8;
    for (int j0 = 0; j0 < cnt; j0 += kWarp) {
        const int some = min(kWarp, cnt - j0);
        const float* rec = base + (size_t)j0 * kRecord;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (lane < some) ml = __ldcg(reinterpret_cast<const float2*>(rec + (size_t)lane * kRecord));
        float c = 0.0f;
#pragma unroll 1
        for (int i = 0; i < some; i += kAhead) {
            float4 v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                v[k] = __ldcg(reinterpret_cast<const float4*>(rec + (size_t)min(i + k, some - 1) * kRecord + 4 + 4 * lane));
            if (i == 0) {
                const float M = fmaxf(x.m, warp_max(ml.x));
                c = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - M);
                const float cx = x.m == -INFINITY ? 0.0f : exp2_fast(x.m - M);
                x.m = M;
                x.l = x.l * cx + warp_sum(ml.y * c);
#pragma unroll
                for (int e = 0; e < 4; ++e) x.acc[e] *= cx;
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const float ck = __shfl_sync(0xFFFFFFFFu, c, (i + k) & (kWarp - 1));
                if (i + k < some) {
                    x.acc[0] += v[k].x * ck;
                    x.acc[1] += v[k].y * ck;
                    x.acc[2] += v[k].z * ck;
                    x.acc[3] += v[k].w * ck;
                }
            }
        }
    }
}

// One query head over blocks [v0, v1) of its span, a warp together: lane l
// holds dims 4 l .. 4 l + 3. Positions that are not seen are not read.
__device__ __forceinline__ SlowRow slow_row(const ServeAttnArgs& a, int qrow, int hq, int slot, int pos, int low,
                                            int sinks, const Span& span, int v0, int v1) {
    const int lane = threadIdx.x % kWarp, head = hq / kG;
    const int* table = a.block_table + (size_t)slot * a.max_blocks;
    const size_t qat = (size_t)qrow * a.q_stride + (size_t)hq * kD + 4 * lane;
    const float scale2 = kLog2e / sqrtf((float)kD);
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        q[e] = a.bf16 ? bf16lo(static_cast<const uint16_t*>(a.q)[qat + e]) : static_cast<const float*>(a.q)[qat + e];
    SlowRow r{-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
    for (int v = v0; v < v1; ++v) {
        const int b = span.block(v);
        uint32_t bits = seen_bits(b, pos, low, sinks);
        if (!bits) continue;
        const int id = table[b];
        if (id < 0 || id >= a.n_pool_blocks) {
            if (lane == 0 && a.err) atomicOr(a.err, kErrBadIndex);
            continue;
        }
        const uint16_t* k = a.kv_layer + ((size_t)head * a.n_pool_blocks + id) * 2 * kBlockElems;
        for (; bits; bits &= bits - 1) {
            const int t = __ffs(bits) - 1;
            const uint2 kb = *reinterpret_cast<const uint2*>(k + kv_swizzle(t, 4 * lane));
            const uint2 vb = *reinterpret_cast<const uint2*>(k + kBlockElems + kv_swizzle(t, 4 * lane));
            const float s = warp_sum(q[0] * bf16lo(kb.x) + q[1] * bf16hi(kb.x) + q[2] * bf16lo(kb.y) + q[3] * bf16hi(kb.y)) * scale2;
            const float mn = fmaxf(r.m, s);
            const float c = mn == -INFINITY ? 1.0f : exp2f(r.m - mn);
            const float p = s == -INFINITY ? 0.0f : exp2f(s - mn);
            r.m = mn;
            r.l = r.l * c + p;
            const float f[4] = {bf16lo(vb.x), bf16hi(vb.x), bf16lo(vb.y), bf16hi(vb.y)};
#pragma unroll
            for (int e = 0; e < 4; ++e) r.acc[e] = r.acc[e] * c + p * f[e];
        }
    }
    return r;
}
// acc / l of one query head into the output (0 where nothing was seen)
__device__ __forceinline__ void store_out4(const ServeAttnArgs& a, int qrow, int hq, const float (&acc)[4], float l) {
    const size_t at = (size_t)qrow * a.out_stride + (size_t)hq * kD + 4 * (threadIdx.x % kWarp);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.bf16)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
            make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
    else
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
            make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
}
__device__ __forceinline__ void store_row(const ServeAttnArgs& a, int qrow, int hq, const SlowRow& r) {
    store_out4(a, qrow, hq, r.acc, r.l);
}
__device__ __forceinline__ void store_record(float* rec, const Partial& r, int count = 0) {
    const int lane = threadIdx.x % kWarp;
    if (lane == 0) *reinterpret_cast<float4*>(rec) = make_float4(r.m, r.l, __int_as_float(count), 0.0f);
    *reinterpret_cast<float4*>(rec + 4 + 4 * lane) = make_float4(r.acc[0], r.acc[1], r.acc[2], r.acc[3]);
}

}  // namespace serve
}  // namespace zc
