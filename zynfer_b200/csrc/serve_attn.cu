// Attention of the serving paths over the paged bf16 cache:
//   attn_shared: one query per sequence over all its positions, where sequences
//     made from one prompt (zynfer_cu_seq_fork) hold the same leading blocks;
//   attn_window: the last `tokens` positions of each sequence are queries, and
//     the query at position i sees j <= i with j < sinks or j > i - window.
// Both compute o = sum_j softmax_j(q . k_j / sqrt(d)) v_j per query head, with
// the maximum, the sum and the accumulators in f32 (attentionInto,
// src/backends/cpu/ops.zig:285-354, is the case without sharing or window).
#include "common.cuh"
#include "kernels.h"

namespace zc {

namespace {

constexpr int kD = 128, kG = 2;  // head dim, query heads per kv head
constexpr int kBlockElems = kKvBlock * kD;

__device__ __forceinline__ float load_q(const void* p, size_t i, int bf16) {
    return bf16 ? bf16lo(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
}

// One warp per (query row, kv head): every visible position in turn, lane l
// holding dims 4 l .. 4 l + 3 of both query heads.
__global__ void __launch_bounds__(128) serve_attn_simple_kernel(const __grid_constant__ ServeRows rows, ServeAttnArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x % kWarp;
    const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / kWarp;
    if (w >= (long long)a.batch * a.tokens * a.n_kv) return;
    const int head = (int)(w % a.n_kv);
    const long long qrow = w / a.n_kv;
    const int b = (int)(qrow / a.tokens), t = (int)(qrow % a.tokens);
    const int len = rows.len[b], pos = len - a.tokens + t;
    const int* table = a.block_table + (size_t)rows.slot[b] * a.max_blocks;
    float q[kG][4], acc[kG][4] = {}, m[kG], l[kG] = {0.0f, 0.0f};
    const float scale = 1.0f / sqrtf((float)kD);
#pragma unroll
    for (int h = 0; h < kG; ++h) {
        m[h] = -INFINITY;
        for (int e = 0; e < 4; ++e)
            q[h][e] = load_q(a.q, (size_t)qrow * a.q_stride + (head * kG + h) * kD + 4 * lane + e, a.bf16) * scale;
    }
    const long long low = (long long)pos - a.window + 1;  // first position inside the window
    for (int j = 0; j <= pos; ++j) {
        if (j >= a.sinks && j < low) {
            j = (int)low - 1;
            continue;
        }
        const int id = table[j / kKvBlock];
        if (id < 0 || id >= a.n_pool_blocks) {
            if (lane == 0 && a.err) atomicOr(a.err, kErrBadIndex);
            return;
        }
        const uint16_t* k = a.kv_layer + ((size_t)head * a.n_pool_blocks + id) * 2 * kBlockElems;
        const uint2 kb = *reinterpret_cast<const uint2*>(k + kv_swizzle(j % kKvBlock, 4 * lane));
        const uint2 vb = *reinterpret_cast<const uint2*>(k + kBlockElems + kv_swizzle(j % kKvBlock, 4 * lane));
        const float kf[4] = {bf16lo(kb.x), bf16hi(kb.x), bf16lo(kb.y), bf16hi(kb.y)};
        const float vf[4] = {bf16lo(vb.x), bf16hi(vb.x), bf16lo(vb.y), bf16hi(vb.y)};
#pragma unroll
        for (int h = 0; h < kG; ++h) {
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) s += q[h][e] * kf[e];
            s = warp_sum(s);
            const float mn = fmaxf(m[h], s);
            const float c = mn == -INFINITY ? 1.0f : expf(m[h] - mn), p = mn == -INFINITY ? 0.0f : expf(s - mn);
            m[h] = mn;
            l[h] = l[h] * c + p;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[h][e] = acc[h][e] * c + p * vf[e];
        }
    }
#pragma unroll
    for (int h = 0; h < kG; ++h)
        for (int e = 0; e < 4; ++e) {
            const float o = l[h] > 0.0f ? acc[h][e] / l[h] : (l[h] == 0.0f ? 0.0f : acc[h][e] / l[h]);
            const size_t at = (size_t)qrow * a.out_stride + (head * kG + h) * kD + 4 * lane + e;
            if (a.bf16) static_cast<uint16_t*>(a.out)[at] = f32_to_bf16_rne(o);
            else static_cast<float*>(a.out)[at] = o;
        }
}

// K and V rows [n_kv][n][128] (f32 rounded to nearest even, or bf16) into
// positions pos .. pos + n - 1 of one sequence's cache of one layer: a thread
// per 16-byte chunk of a row.
__global__ void __launch_bounds__(256) kv_write_kernel(KvWriteArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const long long chunks = 2ll * a.n_kv * a.n * (kD / 8);
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < chunks; i += (long long)gridDim.x * blockDim.x) {
        const int c = (int)(i % (kD / 8));
        const long long r = i / (kD / 8);
        const int t = (int)(r % a.n);
        const int hw = (int)(r / a.n), head = hw % a.n_kv, which = hw / a.n_kv;
        const int p = a.pos + t;
        const int id = a.table_row[p / kKvBlock];
        if (id < 0 || id >= a.n_pool_blocks) {
            if (a.err) atomicOr(a.err, kErrBadIndex);
            continue;
        }
        const size_t from = ((size_t)head * a.n + t) * kD + 8 * c;
        const void* src = which ? a.v : a.k;
        uint4 o;
        if (a.bf16) {
            o = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + from);
        } else {
            const float4 x = *reinterpret_cast<const float4*>(static_cast<const float*>(src) + from);
            const float4 y = *reinterpret_cast<const float4*>(static_cast<const float*>(src) + from + 4);
            auto two = [](float lo, float hi) { return (uint32_t)f32_to_bf16_rne(lo) | ((uint32_t)f32_to_bf16_rne(hi) << 16); };
            o = make_uint4(two(x.x, x.y), two(x.z, x.w), two(y.x, y.y), two(y.z, y.w));
        }
        uint16_t* dst = a.kv_layer + (((size_t)head * a.n_pool_blocks + id) * 2 + which) * kBlockElems;
        *reinterpret_cast<uint4*>(dst + kv_swizzle(p % kKvBlock, 8 * c)) = o;
    }
}

}  // namespace

void launch_serve_attn(const ServeRows& rows, const ServeAttnArgs& a, cudaStream_t st) {
    const long long warps = (long long)a.batch * a.tokens * a.n_kv;
    launch_pdl(serve_attn_simple_kernel, (unsigned)((warps + 3) / 4), 128, 0, st, rows, a);
}

void launch_kv_write(const KvWriteArgs& a, cudaStream_t st) {
    const long long chunks = 2ll * a.n_kv * a.n * (kD / 8);
    const long long ctas = (chunks + 255) / 256;
    launch_pdl(kv_write_kernel, (unsigned)(ctas < 4096 ? ctas : 4096), 256, 0, st, a);
}

void prepare_serve_attn_kernels() {
    configure_kernel((const void*)serve_attn_simple_kernel, 0);
    configure_kernel((const void*)kv_write_kernel, 0);
}

}  // namespace zc
