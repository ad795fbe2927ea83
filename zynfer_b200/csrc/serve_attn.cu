// Attention of the serving paths over the paged bf16 cache:
//   attn_shared: one query per sequence over all its positions, where sequences
//     made from one prompt (zynfer_cu_seq_fork) hold the same leading blocks;
//   attn_window: the last `tokens` positions of each sequence are queries, and
//     the query at position i sees j <= i with j < sinks or j > i - window.
// Both compute o = sum_j softmax_j(q . k_j / sqrt(d)) v_j per query head, with
// the maximum, the sum and the accumulators in f32 (attentionInto,
// src/backends/cpu/ops.zig:285-354, is the case without sharing or window).
#include <algorithm>

#include "serve_common.cuh"

namespace zc {

namespace {

using namespace serve;

// The records of a (row, query head) joined, a warp each: a chunk's (rows.n
// == 0), or those of the rows that share a prompt: the prompt's, then the row's
// own, whose first says how many they are. A launch of its own because a row's
// join is a chain of round trips: inside the kernel that streams the rows' own
// blocks it held up the warps that have many short rows (64 rows sharing 4096
// positions: 64 us a call with it there, 30 so, calls overlapping).
template <int N>
__global__ void __launch_bounds__(128) serve_merge_kernel(const __grid_constant__ ServeRowsT<N> rows_param,
                                                          const __grid_constant__ ServeAttnArgs a) {
    const ServeRowsT<N>& rows = as_memory(rows_param);
    const int n_q = a.n_kv * kG;
    const long long w = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / kWarp;
    if (w >= (long long)a.batch * a.tokens * n_q) return;
    const int hq = (int)(w % n_q), i = (int)(w / n_q);
    const float* base = a.part + ((size_t)i * n_q + hq) * a.max_segs * kRecord;
    Partial x = no_partial();
    if (a.nsplit > 1) {
        pdl_wait();
        pdl_launch_dependents();
        join_records(x, base, a.nsplit);
        store_out4(a, i, hq, x.acc, x.l);
    } else {
        const int4 r = *reinterpret_cast<const int4*>(&rows.r[i]);
        const int nrec = (int)((uint32_t)r.w & 1023u);
        pdl_wait();
        pdl_launch_dependents();
        if (nrec == 0) return;
        join_records(x, base, 0, nrec);
        store_out4(a, r.z, hq, x.acc, x.l);
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

int serve_tile_blocks(int p0, int p1, uint32_t window, int sinks) { return span_of(p0, p1, window, sinks, 0).total; }
int serve_span_blocks(int pos, uint32_t window, int sinks, int skip) { return span_of(pos, pos, window, sinks, skip).total; }

void launch_serve_merge(const ServeRows& rows, const ServeAttnArgs& a, cudaStream_t st) {
    const long long warps = (long long)a.batch * a.tokens * a.n_kv * kG;
    const unsigned ctas = (unsigned)((warps + 3) / 4);
    if (a.batch <= kServeSmallBatch)
        with_rows<kServeSmallBatch>(rows, [&](const ServeRowsT<kServeSmallBatch>& r) {
            launch_pdl(serve_merge_kernel<kServeSmallBatch>, ctas, 128, 0, st, r, a);
        });
    else if (a.batch <= kServeMidBatch)
        with_rows<kServeMidBatch>(rows, [&](const ServeRowsT<kServeMidBatch>& r) {
            launch_pdl(serve_merge_kernel<kServeMidBatch>, ctas, 128, 0, st, r, a);
        });
    else launch_pdl(serve_merge_kernel<kServeMaxBatch>, ctas, 128, 0, st, rows, a);
}

void launch_kv_write(const KvWriteArgs& a, cudaStream_t st) {
    const long long chunks = 2ll * a.n_kv * a.n * (kD / 8);
    const long long ctas = (chunks + 255) / 256;
    launch_pdl(kv_write_kernel, (unsigned)(ctas < 4096 ? ctas : 4096), 256, 0, st, a);
}

void prepare_serve_attn_kernels() {
    configure_kernel((const void*)serve_merge_kernel<kServeSmallBatch>, 0);
    configure_kernel((const void*)serve_merge_kernel<kServeMidBatch>, 0);
    configure_kernel((const void*)serve_merge_kernel<kServeMaxBatch>, 0);
    configure_kernel((const void*)kv_write_kernel, 0);
}

}  // namespace zc
