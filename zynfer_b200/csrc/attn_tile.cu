// Attention of many query rows over the paged cache on the tensor cores
// (tcgen05, accumulators and probabilities in TMEM), the dense part of the
// serving attention (serve_attn.cu): chunks of a prompt with a sliding window
// and sinks, and the common prompt of sequences that share it.
//
// A CTA takes 128 query rows of one kv head (64 queries x 2 query heads: the
// MMA's M) and a range of the visible 16-token cache blocks, TILE tokens at a
// time: S = Q K^T into TMEM, softmax in registers with one thread per row,
// P back into TMEM as the next MMA's A operand, O += P V into TMEM.
// Two warpgroups take the tiles in turn, each with an accumulator, a running
// maximum and a sum of its own (joined at the end), so the tensor cores work
// on one tile while the exponentials of the other are taken. Warp 8 loads
// K and V, warp 9 issues the MMAs.
//
// The cache's layout is the MMA's: a block row is 256 bytes whose 16-byte
// chunks are XOR-swizzled by token & 7 inside each 128-byte half, so 16-row
// boxes of half a row, copied as they lie (TMA without a swizzle of its own),
// form the 128-byte-swizzled atoms of K (K-major) and of V (token-major, read
// as the transposed operand). A block that is not there is a box past the end
// of the tensor: zeros.
//
// bf16 queries: one MMA term, P rounded to bf16 (8 bits, the output's own
// precision; its sum is taken from the f32 values). f32 queries: Q and P are
// split into three bf16 terms each (24 bits, nothing is lost) against the
// exact bf16 K and V: three times the MMAs, and f32 sums throughout.
// The accumulator is rescaled only when a row's maximum grows by more than
// 2^8 (the reference point of its exponentials may lag behind by that much).
//
// A row whose result is not finite is taken again position by position: a
// masked position's weight 0 times an infinite or NaN V would otherwise reach
// rows that do not see it.
#include <cuda.h>

#include <algorithm>

#include "serve_common.cuh"
#include "tc_gemm.h"

namespace zc {

namespace {

using namespace serve;

constexpr int kRows = 128;       // MMA M: 64 queries x 2 query heads, row 2 m + h
constexpr int kMembers = kRows / kG;
constexpr int kThreads = 384;    // warps 0-3 and 4-7: softmax; 8: TMA; 9: MMA; 10, 11 fill the third warpgroup
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;  // 2 x 128 x 208 + 128 x 88 = 384 x 168, the launch's registers
constexpr int kHalfDims = 64;    // dims of a 128-byte half row
constexpr float kLag = 8.0f;     // log2 of the growth of a row's maximum that is left to lag

template <int TERMS>
struct Lay {
    static constexpr int TILE = TERMS == 1 ? 128 : 64;  // tokens per tile
    static constexpr int BLOCKS = TILE / kKvBlock;
    static constexpr int STAGES = TERMS == 1 ? 3 : 4;
    static constexpr int HALF = TILE * 128;             // bytes of one half (64 dims) of a K or V tile
    static constexpr int KV = 2 * HALF;
    static constexpr int QTERM = kRows * 256;
    static constexpr int Q = TERMS * QTERM;
    static constexpr int BARS = Q + STAGES * 2 * KV;
    static constexpr int SMEM = BARS + 512 + 1024;      // 1024: alignment of the first atom
    static_assert(SMEM <= 232448, "tile attention shared memory");
    // TMEM columns: two accumulators, then per warpgroup S with P over it
    static constexpr int O_COL = 0, S_COL = 256, S_STEP = 128;
};

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(taddr)
        : "memory");
}

// Shared-memory operand of 128-byte-swizzled atoms (8 rows x 128 bytes):
// K-major, 8-row groups 1024 bytes apart; or, for V, rows along K with the
// 64-dim halves `lead` bytes apart.
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
           ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
// kind::f16, bf16 operands, f32 accumulators, M = 128; b_rows: B's rows run along K
constexpr uint32_t idesc(int n, bool b_rows) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
                 : "memory");
}

// What a CTA works on.
struct Job {
    int first, count;  // queries: the tile's first (chunk: global query index; shared: member) and how many
    int head, slot;
    int p0, p1;        // chunk: positions of the first and last query
    Span span;         // the visible blocks
    int t_lo, n;       // first tile and number of tiles of this CTA
    int seg, nseg;     // its record among the tile's (nseg 1: the output itself)
};

template <int TILE_BLOCKS, int N>
__device__ __forceinline__ Job find_job(const ServeRowsT<N>& rows, const TileListT<N>& list, const ServeAttnArgs& a) {
    Job j;
    if (list.n == 0) {  // chunk: the tiles that see most first
        const int per_seq = (a.tokens + kMembers - 1) / kMembers;
        int x = blockIdx.x;
        j.head = x % a.n_kv;
        x /= a.n_kv;
        j.seg = x % a.nsplit;
        x /= a.nsplit;
        j.nseg = a.nsplit;
        const int b = x % a.batch, ti = per_seq - 1 - x / a.batch;
        j.first = b * a.tokens + ti * kMembers;
        j.count = min(kMembers, a.tokens - ti * kMembers);
        j.slot = rows.slot[b];
        j.p0 = rows.len[b] - a.tokens + ti * kMembers;
        j.p1 = j.p0 + j.count - 1;
        j.span = span_of(j.p0, j.p1, a.window, a.sinks, 0);
    } else {
        int lo = 0, hi = list.n - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (list.item0[mid] <= (int)blockIdx.x) lo = mid;
            else hi = mid - 1;
        }
        const int x = blockIdx.x - list.item0[lo];
        j.head = x % a.n_kv;
        j.seg = x / a.n_kv;
        j.nseg = (list.item0[lo + 1] - list.item0[lo]) / a.n_kv;
        j.first = list.first[lo];
        j.count = list.count[lo];
        j.slot = rows.slot[j.first];
        j.p0 = j.p1 = list.blocks[lo] * kKvBlock - 1;  // every row sees every position of the common blocks
        j.span = Span{0, 0, list.blocks[lo]};
    }
    const int tiles = (j.span.total + TILE_BLOCKS - 1) / TILE_BLOCKS;
    j.t_lo = (int)((long long)j.seg * tiles / j.nseg);
    j.n = (int)((long long)(j.seg + 1) * tiles / j.nseg) - j.t_lo;
    return j;
}

// Three (or one) bf16 terms of p, packed in pairs: nothing is left of p after
// the third.
template <int TERMS>
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t (&t)[TERMS]) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        t[i] = pack_bf16(x0, x1);
        if (i + 1 < TERMS) {
            x0 -= bf16lo(t[i]);
            x1 -= bf16hi(t[i]);
        }
    }
}

template <int TERMS, int N>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tile_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ ServeRowsT<N> rows,
                     const __grid_constant__ TileListT<N> list, const __grid_constant__ ServeAttnArgs a) {
    using L = Lay<TERMS>;
    constexpr int TILE = L::TILE;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_k = reinterpret_cast<uint64_t*>(smem + L::BARS);
    uint64_t* full_v = full_k + L::STAGES;
    uint64_t* empty = full_v + L::STAGES;
    uint64_t* s_full = empty + L::STAGES;  // [2] S of warpgroup w is in TMEM
    uint64_t* p_full = s_full + 2;         // [2] its P is
    uint64_t* o_full = p_full + 2;         // [2] its last product is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
    uint32_t* bad_rows = tmem_slot + 1;    // [4] bit per row: not finite

    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(&full_k[s], 1);
            mbar_init(&full_v[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(&s_full[w], 1);
            mbar_init(&p_full[w], 128);
            mbar_init(&o_full[w], 1);
        }
        for (int w = 0; w < 4; ++w) bad_rows[w] = 0u;
        fence_barrier_init();
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const Job job = find_job<L::BLOCKS>(rows, list, a);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();
    const int n = job.n;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 8) {
            // ---------------- K and V: one lane per half of a block of K or of V
            constexpr int PER = 2 * L::BLOCKS;
            const int* table = a.block_table + (size_t)job.slot * a.max_blocks;
            const int is_v = lane / PER, blk = (lane % PER) >> 1, half = lane & 1;
            for (int i = 0; i < n; ++i) {
                const int s = i % L::STAGES, round = i / L::STAGES;
                int y = a.kv_rows;  // past the end: zeros
                const int v = (job.t_lo + i) * L::BLOCKS + blk;
                if (lane < 2 * PER && v < job.span.total) {
                    const int id = table[job.span.block(v)];
                    if (id >= 0 && id < a.n_pool_blocks)
                        y = a.kv_row0 + ((job.head * a.n_pool_blocks + id) * 2 + is_v) * kKvBlock;
                    else if (a.err) atomicOr(a.err, kErrBadIndex);
                }
                bool ok = true;
                if (round > 0) ok = mbar_wait_bounded(&empty[s], (uint32_t)((round - 1) & 1), a.err);
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    // the copies in flight land before the CTA ends
                    for (int k = max(0, i - L::STAGES); k < i; ++k) {
                        mbar_wait_bounded(&full_k[k % L::STAGES], (uint32_t)((k / L::STAGES) & 1), nullptr);
                        mbar_wait_bounded(&full_v[k % L::STAGES], (uint32_t)((k / L::STAGES) & 1), nullptr);
                    }
                    break;
                }
                uint8_t* ks = smem + L::Q + s * 2 * L::KV;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&full_k[s], L::KV);
                    mbar_arrive_expect_tx(&full_v[s], L::KV);
                }
                __syncwarp();
                if (lane < 2 * PER)
                    tma_box(smem_addr(ks + is_v * L::KV + half * L::HALF + blk * (kKvBlock * 128)), &kv_map,
                            half * kHalfDims, y, is_v ? &full_v[s] : &full_k[s]);
            }
        } else if (warp == 9) {
            asm volatile("bar.sync 1, 288;" ::: "memory");  // Q is in shared memory
            if (lane == 0) {
                // ---------------- MMA issuer: S of tile i, then P V of tile i - 1.
                // MMAs run in issue order, so S(i) overwrites the P of tile i - 2
                // after it was read.
                constexpr uint32_t id_s = idesc(TILE, false), id_o = idesc(kD, true);
                const uint32_t qs = smem_addr(smem);
                for (int i = 0; i <= n; ++i) {
                    if (i < n) {
                        const int s = i % L::STAGES;
                        if (!mbar_wait_bounded(&full_k[s], (uint32_t)((i / L::STAGES) & 1), a.err)) break;
                        tc_fence_after();
                        const uint32_t ks = smem_addr(smem + L::Q + s * 2 * L::KV);
                        const uint32_t d = tmem + L::S_COL + (i & 1) * L::S_STEP;
#pragma unroll
                        for (int t = TERMS - 1; t >= 0; --t)  // the small terms first: fewer roundings at the sum's size
#pragma unroll
                            for (int kk = 0; kk < 8; ++kk)
                                mma_ss(d, sdesc(qs + t * L::QTERM + (kk >> 2) * (kRows * 128) + (kk & 3) * 32, 16),
                                       sdesc(ks + (kk >> 2) * L::HALF + (kk & 3) * 32, 16), id_s, t < TERMS - 1 || kk);
                        mma_commit(&s_full[i & 1]);
                    }
                    if (i > 0) {
                        const int j = i - 1, w = j & 1, s = j % L::STAGES;
                        if (!mbar_wait_bounded(&full_v[s], (uint32_t)((j / L::STAGES) & 1), a.err)) break;
                        if (!mbar_wait_bounded(&p_full[w], (uint32_t)((j >> 1) & 1), a.err)) break;
                        tc_fence_after();
                        const uint32_t vs = smem_addr(smem + L::Q + s * 2 * L::KV + L::KV);
                        const uint32_t p = tmem + L::S_COL + w * L::S_STEP, d = tmem + L::O_COL + w * kD;
#pragma unroll
                        for (int t = TERMS - 1; t >= 0; --t)
#pragma unroll
                            for (int kk = 0; kk < TILE / 16; ++kk)
                                mma_ts(d, p + t * (TILE / 2) + kk * 8, sdesc(vs + kk * 2048, L::HALF), id_o,
                                       j > 1 || t < TERMS - 1 || kk);
                        mma_commit(&empty[s]);
                        if (j + 2 >= n) mma_commit(&o_full[w]);
                    }
                }
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        // ---------------- softmax: thread = one query row, warpgroup w takes tiles w, w + 2, ..
        const int w = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        {
            // Q: two threads per row, 64 dims each, split into terms
            const int qr = threadIdx.x >> 1, half = threadIdx.x & 1;
            const int m = qr >> 1, hh = qr & 1;
            const bool live = m < job.count;
            size_t at = 0;
            if (live) at = (size_t)(list.n ? rows.row[job.first + m] : job.first + m) * a.q_stride +
                           (size_t)(job.head * kG + hh) * kD + half * kHalfDims;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                uint32_t t[TERMS][4];
                if constexpr (TERMS == 1) {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (live) x = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + at + 8 * c));
                    t[0][0] = x.x; t[0][1] = x.y; t[0][2] = x.z; t[0][3] = x.w;
                } else {
                    float4 x = make_float4(0, 0, 0, 0), y = x;
                    if (live) {
                        x = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at + 8 * c));
                        y = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at + 8 * c + 4));
                    }
                    const float f[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t u[TERMS];
                        split_pair<TERMS>(f[2 * e], f[2 * e + 1], u);
#pragma unroll
                        for (int k = 0; k < TERMS; ++k) t[k][e] = u[k];
                    }
                }
#pragma unroll
                for (int k = 0; k < TERMS; ++k)
                    *reinterpret_cast<uint4*>(smem + k * L::QTERM + half * (kRows * 128) + qr * 128 + ((c ^ (qr & 7)) << 4)) =
                        make_uint4(t[k][0], t[k][1], t[k][2], t[k][3]);
            }
            fence_proxy_async_smem();
            asm volatile("bar.sync 1, 288;" ::: "memory");
        }
        const int pos = min(job.p0 + (r >> 1), job.p1);  // this row's position (chunk)
        const int low = window_low(pos, a.window);
        const float scale2 = kLog2e / sqrtf((float)kD);
        const uint32_t s_at = tmem + L::S_COL + w * L::S_STEP + lane_base;
        const uint32_t o_at = tmem + L::O_COL + w * kD + lane_base;
        float m_ref = -INFINITY, l = 0.0f;  // reference point (log2 units) and sum of the exponentials
        bool alive = true;
        for (int i = w; i < n; i += 2) {
            alive = __all_sync(0xFFFFFFFFu, mbar_wait_bounded(&s_full[w], (uint32_t)((i >> 1) & 1), a.err));
            if (!alive) break;
            tc_fence_after();
            float s[TILE];
#pragma unroll
            for (int c = 0; c < TILE; c += 32) tmem_ld32(s_at + c, reinterpret_cast<uint32_t*>(s + c));
            tmem_wait_ld();
            const int v0 = (job.t_lo + i) * L::BLOCKS;
            const int b0 = job.span.block(v0), b1 = job.span.block(v0 + L::BLOCKS - 1);
            const bool whole = v0 + L::BLOCKS <= job.span.total && v0 >= job.span.nsb && b1 * kKvBlock + kKvBlock - 1 <= job.p0 &&
                               (list.n || b0 * kKvBlock >= window_low(job.p1, a.window));
            if (!whole) {
#pragma unroll
                for (int u = 0; u < L::BLOCKS; ++u) {
                    const uint32_t bits = v0 + u < job.span.total
                                              ? (list.n ? 0xFFFFu : seen_bits(job.span.block(v0 + u), pos, low, a.sinks))
                                              : 0u;
#pragma unroll
                    for (int c = 0; c < kKvBlock; ++c)
                        if (!((bits >> c) & 1u)) s[u * kKvBlock + c] = -INFINITY;
                }
            }
            float mx[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) mx[c] = fmaxf(s[c], s[c + 8]);
#pragma unroll
            for (int c = 16; c < TILE; c += 16)
#pragma unroll
                for (int e = 0; e < 8; ++e) mx[e] = fmaxf(mx[e], fmaxf(s[c + e], s[c + 8 + e]));
            const float mt = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * scale2;
            const bool grow = mt > m_ref + kLag || (m_ref == -INFINITY && mt > -INFINITY);
            if (__any_sync(0xFFFFFFFFu, grow)) {
                const float m_new = grow ? mt : m_ref;
                const float c = grow ? exp2f(m_ref - m_new) : 1.0f;
                l *= c;
                m_ref = m_new;
                if (i > 1) {  // the accumulator holds tiles up to i - 2, whose products are done (S(i) came after them)
#pragma unroll
                    for (int d = 0; d < kD; d += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_at + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * c);
                        tmem_st32(o_at + d, o);
                    }
                }
            }
            const float neg = m_ref == -INFINITY ? 0.0f : -m_ref;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c0 = 0; c0 < TILE; c0 += 64) {
                uint32_t p[TERMS][32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    const float x0 = exp2_fast(fmaf(s[c0 + 2 * e], scale2, neg));
                    const float x1 = exp2_fast(fmaf(s[c0 + 2 * e + 1], scale2, neg));
                    sum[(2 * e) & 3] += x0;
                    sum[(2 * e + 1) & 3] += x1;
                    uint32_t u[TERMS];
                    split_pair<TERMS>(x0, x1, u);
#pragma unroll
                    for (int k = 0; k < TERMS; ++k) p[k][e] = u[k];
                }
#pragma unroll
                for (int k = 0; k < TERMS; ++k) tmem_st32(s_at + k * (TILE / 2) + c0 / 2, p[k]);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[w]);
        }
        // ---- join the two warpgroups' parts: maxima and sums through the Q
        // buffer (its last reader is done), warpgroup w then takes dims 64 w ..
        for (int k = 0; k < min(n, 2); ++k) alive = __all_sync(0xFFFFFFFFu, alive && mbar_wait_bounded(&o_full[k], 0u, a.err));
        tc_fence_after();
        float2* ml = reinterpret_cast<float2*>(smem);
        if (alive) ml[w * kRows + r] = make_float2(m_ref, l);
        asm volatile("bar.sync 2, 256;" ::: "memory");
        if (alive) {
            const float2 x0 = ml[r], x1 = ml[kRows + r];
            const float M = fmaxf(x0.x, x1.x);
            const float c0 = x0.x == -INFINITY ? 0.0f : exp2f(x0.x - M), c1 = x1.x == -INFINITY ? 0.0f : exp2f(x1.x - M);
            const float lsum = x0.y * c0 + x1.y * c1;
            const bool live = (r >> 1) < job.count;
            const bool direct = list.n == 0 && job.nseg == 1;
            float inv = 1.0f;
            if (direct) inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
            bool finite = true;
            const int member = job.first + (r >> 1), qrow = list.n ? rows.row[live ? member : job.first] : member;
            const int hq = job.head * kG + (r & 1);
            float* rec = a.part + (((size_t)member * (a.n_kv * kG) + hq) * a.max_segs + job.seg) * kRecord;
            if (!direct && live && w == 0) *reinterpret_cast<float2*>(rec) = make_float2(M, lsum);
#pragma unroll
            for (int d = 0; d < kHalfDims; d += 32) {
                __syncwarp();
                uint32_t u0[32], u1[32];
                if (n > 0) tmem_ld32(tmem + L::O_COL + lane_base + w * kHalfDims + d, u0);
                if (n > 1) tmem_ld32(tmem + L::O_COL + kD + lane_base + w * kHalfDims + d, u1);
                tmem_wait_ld();
                float o[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    o[e] = n > 0 ? __uint_as_float(u0[e]) * c0 : 0.0f;
                    if (n > 1) o[e] += __uint_as_float(u1[e]) * c1;
                    finite = finite && fabsf(o[e]) < INFINITY;
                    o[e] *= inv;
                }
                if (!live) {
                } else if (!direct) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4*>(rec + 4 + w * kHalfDims + d + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                } else if (TERMS == 1) {
                    uint16_t* op = static_cast<uint16_t*>(a.out) + (size_t)qrow * a.out_stride + (size_t)hq * kD + w * kHalfDims + d;
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *reinterpret_cast<uint4*>(op + e) = make_uint4(pack_bf16(o[e], o[e + 1]), pack_bf16(o[e + 2], o[e + 3]),
                                                                       pack_bf16(o[e + 4], o[e + 5]), pack_bf16(o[e + 6], o[e + 7]));
                } else {
                    float* op = static_cast<float*>(a.out) + (size_t)qrow * a.out_stride + (size_t)hq * kD + w * kHalfDims + d;
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4*>(op + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if (live && !(finite && fabsf(lsum) < INFINITY)) atomicOr(&bad_rows[quarter], 1u << lane);
        }
        asm volatile("bar.sync 2, 256;" ::: "memory");
        // rows that are not finite, position by position over this CTA's blocks
        for (int x = warp; x < kRows; x += 8) {
            if (!((bad_rows[x >> 5] >> (x & 31)) & 1u)) continue;
            const int m = job.first + (x >> 1), qrow = list.n ? rows.row[m] : m, hq = job.head * kG + (x & 1);
            const int p = list.n ? job.p1 : job.p0 + (x >> 1);
            SlowRow row = slow_row(a, qrow, hq, job.slot, p, list.n ? 0 : window_low(p, a.window), list.n ? 0 : a.sinks, job.span,
                                   job.t_lo * L::BLOCKS, min((job.t_lo + n) * L::BLOCKS, job.span.total));
            if (list.n == 0 && job.nseg == 1) store_row(a, qrow, hq, row);
            else store_record(a.part + (((size_t)m * (a.n_kv * kG) + hq) * a.max_segs + job.seg) * kRecord, row);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace

void launch_attn_tile(const CUtensorMap& kv_map, const ServeRows& rows, const TileList& list, const ServeAttnArgs& a,
                      int items, cudaStream_t st) {
    if (a.batch <= kServeSmallBatch) {
        TileListT<kServeSmallBatch> small;
        small.n = list.n;
        for (int e = 0; e < list.n; ++e) {
            small.item0[e] = list.item0[e];
            small.first[e] = list.first[e];
            small.count[e] = list.count[e];
            small.blocks[e] = list.blocks[e];
        }
        small.item0[list.n] = items;
        if (a.bf16) launch_pdl(attn_tile_kernel<1, kServeSmallBatch>, items, kThreads, Lay<1>::SMEM, st, kv_map, small_rows(rows), small, a);
        else launch_pdl(attn_tile_kernel<3, kServeSmallBatch>, items, kThreads, Lay<3>::SMEM, st, kv_map, small_rows(rows), small, a);
    } else {
        if (a.bf16) launch_pdl(attn_tile_kernel<1, kServeMaxBatch>, items, kThreads, Lay<1>::SMEM, st, kv_map, rows, list, a);
        else launch_pdl(attn_tile_kernel<3, kServeMaxBatch>, items, kThreads, Lay<3>::SMEM, st, kv_map, rows, list, a);
    }
}

void prepare_attn_tile_kernels() {
    configure_kernel((const void*)attn_tile_kernel<1, kServeSmallBatch>, Lay<1>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<3, kServeSmallBatch>, Lay<3>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<1, kServeMaxBatch>, Lay<1>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<3, kServeMaxBatch>, Lay<3>::SMEM);
}

}  // namespace zc
