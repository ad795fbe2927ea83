// Attention of many query rows over the paged cache on the tensor cores
// (tcgen05, accumulators and probabilities in TMEM), the dense part of the
// serving attention (serve_attn.cu): chunks of a prompt with a sliding window
// and sinks, and the common prompt of sequences that share it.
//
// A CTA takes 128 query rows of one kv head (64 queries x 2 query heads: the
// MMA's M) and a range of the visible 16-token cache blocks, 64 tokens at a
// time: S = Q K^T into TMEM, softmax in registers with one thread per row,
// P back into TMEM over S as the next MMA's A operand, O += P V into TMEM.
// S has two buffers: the tensor cores form tile i + 1 while the exponentials of
// tile i are taken. Warps 0-3: softmax; 4, 7 and 5: loads of K and of V, each a ring
// of two (K's places are free again after S, V's after P V); 6: MMAs, one thread.
// With bf16 queries two CTAs share an SM, so that the start and the end of one run
// beside the middle of the other.
//
// Measured: 8192 bf16 queries, 8 kv heads, window 1024: 115 us a call, 0.57 PFLOP/s,
// 35 % of the card's dense rate (0.72 and 44 % with P as one term, which cost the
// results half their precision); 64 f32 rows over 4096 common positions: 18 us of a
// lone call's 60 (4 tiles of keys a CTA). Bound by the two chains of a tile, with two
// CTAs on an SM: the MMA thread's (three barriers, sixteen MMAs queued behind the
// other CTA's, 912 cycles of tensor pipe each CTA: the pipe is active 55 % of the
// time) and the softmax's (S out of TMEM and the maximum 550, the exponentials 700,
// of which the special-function units need 512). So a barrier is tried before it is
// waited for, what ends together shares a commit, and the MMA loop's descriptors are
// constants (with one term of P: 101 us before these three and the asynchronous
// copies of Q, 89 after).
//
// The cache's layout is the MMA's: a block row is 256 bytes whose 16-byte
// chunks are XOR-swizzled by token & 7 inside each 128-byte half, so 16-row
// boxes of half a row, copied as they lie (TMA without a swizzle of its own),
// form the 128-byte-swizzled atoms of K (K-major) and of V (token-major, read
// as the transposed operand). A block that is not there is a box past the end
// of the tensor: zeros.
//
// bf16 queries: Q is one MMA term as it lies, P two (16 bits; its sum is taken from
// the f32 values), so that the result has one rounding, its own. With P as one term
// the error was that of two roundings: 2.3e-3 of the result against 1.7e-3. f32
// queries: Q and P are split into three bf16 terms each (24 bits, nothing is lost)
// against the exact bf16 K and V: three times the MMAs, and f32 sums throughout.
// The accumulator is rescaled only when a row's maximum grows by more than
// 2^8 (the reference point of its exponentials may lag behind by that much).
//
// A row whose result is not finite is taken again position by position: a
// masked position's weight 0 times an infinite or NaN V would otherwise reach
// rows that do not see it.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "serve_common.cuh"
#include "tc_gemm.h"

namespace zc {

namespace {

using namespace serve;

constexpr int kRows = 128;       // MMA M: 64 queries x 2 query heads, row 2 m + h
constexpr int kMembers = kRows / kG;
constexpr int kThreads = 256;    // warps 0-3: softmax; 4, 7: K; 5: V; 6: MMA
constexpr int TILE = 64, kTileBlocks = TILE / kKvBlock;  // tokens of a tile
constexpr int kHalf = TILE * 128, kTileBytes = 2 * kHalf;  // a K or V tile: two 64-dim halves
constexpr int kHalfDims = 64;
// Tiles that an f32 accumulator takes before it is added to a sum in shared memory:
// the MMA rounds its sums toward 0, an error that grows with their number.
// Measured relative error over 8192 keys: 8.6e-6 without, 1.4e-6 with (a plain f32
// computation 1.7e-6).
constexpr int kFlush = 16;
constexpr float kLag = 8.0f;     // log2 of the growth of a row's maximum that is left to lag
constexpr unsigned kAll = 0xFFFFFFFFu;
using u64x2 = unsigned long long;

template <int TERMS>
struct Lay {
    static constexpr int CTAS = TERMS == 1 ? 2 : 1;      // per SM
    static constexpr int PTERMS = TERMS == 1 ? 2 : 3;    // of P (TERMS: of Q)
    static constexpr int KST = 2, VST = 2;  // K's ring is S's: one barrier tells that S is there and K's place free
    static constexpr int QTERM = kRows * 256;
    static constexpr int K = TERMS * QTERM, V = K + KST * kTileBytes;
    // f32 queries: what the accumulators held after every kFlush tiles, added up [dim][row]
    static constexpr int TOTAL = V + VST * kTileBytes;
    static constexpr int BARS = TOTAL + (TERMS == 1 ? 0 : kRows * kD * 4);
    static constexpr int SMEM = BARS + 512;
    static_assert(CTAS * (SMEM + 1024) <= 233472, "tile attention shared memory");
    static_assert(TOTAL >= kRows * kD * 4, "the results are staged over Q, K and V");
    // TMEM columns: the accumulator (f32 queries: another for the products of P's
    // small terms, so that a sum is rounded, toward 0 by the MMA, 4 times per tile at
    // its full size instead of 12), then two regions of S with P over it
    static constexpr int ACCS = TERMS == 1 ? 1 : 2;
    static constexpr int S_COL = ACCS * kD, S_STEP = TERMS == 1 ? 64 : 128;
    static constexpr int COLS = TERMS == 1 ? 256 : 512;
    static_assert(PTERMS * (TILE / 2) <= S_STEP && S_COL + 2 * S_STEP <= COLS, "P lies over S");
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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

// Two f32 operations in one instruction.
__device__ __forceinline__ u64x2 fma2(u64x2 a, u64x2 b, u64x2 c) {
    u64x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ u64x2 add2(u64x2 a, u64x2 b) {
    u64x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64x2 pack2(float x, float y) {
    u64x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(u64x2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }

// What a CTA works on.
struct Job {
    int first, count;  // queries: the tile's first (chunk: global query index; shared: member) and how many
    int head, slot;
    int p0, p1;        // chunk: positions of the first and last query
    Span span;         // the visible blocks
    int t_lo, n;       // first tile and number of tiles of this CTA
    int seg, nseg;     // its record among the tile's (nseg 1: the output itself)
};

template <int N>
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
        j.slot = rows.r[b].slot;
        j.p0 = rows.r[b].len - a.tokens + ti * kMembers;
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
        j.slot = rows.r[j.first].slot;
        j.p0 = j.p1 = list.blocks[lo] * kKvBlock - 1;  // every row sees every position of the common blocks
        j.span = Span{0, 0, list.blocks[lo]};
    }
    const int tiles = (j.span.total + kTileBlocks - 1) / kTileBlocks;
    j.t_lo = (int)((long long)j.seg * tiles / j.nseg);
    j.n = (int)((long long)(j.seg + 1) * tiles / j.nseg) - j.t_lo;
    return j;
}

// bf16 terms of x0 and x1, packed in pairs: nothing is left after the third.
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
__global__ void __launch_bounds__(kThreads, Lay<TERMS>::CTAS)
    attn_tile_kernel(const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ ServeRowsT<N> rows,
                     const __grid_constant__ TileListT<N> list, const __grid_constant__ ServeAttnArgs a) {
    using L = Lay<TERMS>;
    extern __shared__ __align__(1024) uint8_t smem[];
    // A barrier per buffer: no waiter can be two phases behind. (A commit costs the MMA thread
    // 65 cycles, so what ends at once shares one.)
    uint64_t* full_k = reinterpret_cast<uint64_t*>(smem + L::BARS);
    uint64_t* s_full = full_k + L::KST;   // S of tile i (buffer i & 1) is in TMEM, its K read
    uint64_t* full_v = s_full + L::KST;
    uint64_t* o_full = full_v + L::VST;   // P V of tile i (buffer i % VST) is done, its V read
    uint64_t* p_full = o_full + L::VST;   // [2] P of tile i (buffer i & 1) is in TMEM
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(p_full + 2);
    uint32_t* bad_rows = tmem_slot + 1;   // [4] bit per row: not finite

    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::KST; ++s) {
            mbar_init(&full_k[s], 2);
            mbar_init(&s_full[s], 1);
            mbar_init(&p_full[s], 128);
        }
        for (int s = 0; s < L::VST; ++s) {
            mbar_init(&full_v[s], 1);
            mbar_init(&o_full[s], 1);
        }
        for (int w = 0; w < 4; ++w) bad_rows[w] = 0u;
        fence_barrier_init();
    }
    if (warp == 6) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                     "n"(L::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const Job job = find_job(rows, list, a);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();
    const int n = job.n;

    if (warp == 4 || warp == 5 || warp == 7) {
        // ---------------- K (warps 4 and 7, a half of the dims each) or V (warp 5):
        // a lane per half of a block. A copy costs its warp about 100 cycles, so the
        // eight of a K tile, which S waits for, are shared.
        const int is_v = warp == 5, stages = is_v ? L::VST : L::KST;
        uint64_t* full = is_v ? full_v : full_k;
        uint64_t* empty = is_v ? o_full : s_full;
        uint8_t* ring = smem + (is_v ? L::V : L::K);
        const int* table = a.block_table + (size_t)job.slot * a.max_blocks;
        const int v0 = job.t_lo * kTileBlocks, row0 = a.kv_row0 + job.head * a.n_pool_blocks * 2 * kKvBlock + is_v * kKvBlock;
        // rows of the pool of 32 blocks, a lane each (past the end: zeros), read a chunk ahead
        auto rows_of = [&](int c) {
            const int v = v0 + 32 * c + lane;
            if (v >= job.span.total) return a.kv_rows;
            const int id = table[job.span.block(v)];
            if (id >= 0 && id < a.n_pool_blocks) return row0 + id * 2 * kKvBlock;
            if (a.err) atomicOr(a.err, kErrBadIndex);
            return a.kv_rows;
        };
        constexpr int kChunk = 32 / kTileBlocks;  // tiles of a chunk
        int now = rows_of(0), next = n > kChunk ? rows_of(1) : 0;
        const int copies = is_v ? 2 * kTileBlocks : kTileBlocks;
        const int blk = lane & (kTileBlocks - 1), half = is_v ? (lane / kTileBlocks) & 1 : (warp == 7);
        for (int i = 0, s = 0, round = 0; i < n; ++i) {
            if (i > 0 && i % kChunk == 0) {
                now = next;
                if (i + kChunk < n) next = rows_of(i / kChunk + 1);
            }
            bool ok = true;
            if (round > 0) ok = mbar_wait_try(&empty[s], (uint32_t)((round - 1) & 1), a.err);
            if (!__all_sync(kAll, ok)) {
                // the copies in flight land before the CTA ends
                for (int k = max(0, i - stages); k < i; ++k)
                    mbar_wait_try(&full[k % stages], (uint32_t)((k / stages) & 1), nullptr);
                break;
            }
            const int y = __shfl_sync(kAll, now, (i % kChunk) * kTileBlocks + blk);
            if (lane == 0) mbar_arrive_expect_tx(&full[s], copies * (kTileBytes / (2 * kTileBlocks)));
            __syncwarp();
            if (lane < copies)
                tma_box(smem_addr(ring + s * kTileBytes + half * kHalf + blk * (kKvBlock * 128)), &kv_map, half * kHalfDims, y,
                        &full[s]);
            if (++s == stages) {
                s = 0;
                ++round;
            }
        }
    } else if (warp == 6) {
        asm volatile("bar.sync 1, 160;" ::: "memory");  // Q is in shared memory
        if (lane == 0) {
            // ---------------- MMA issuer: S of tile i, then P V of tile i - 1.
            // MMAs run in issue order, so S(i) overwrites the P of tile i - 2
            // after it was read.
            constexpr uint32_t id_s = idesc(TILE, false), id_o = idesc(kD, true);
            const uint32_t qs = smem_addr(smem);
            // tile i with buffer `s` known, so that descriptors are constants
            auto step = [&](int i, auto buffer) -> bool {
                constexpr int s = decltype(buffer)::value, o = 1 - s;
                if (i < n) {
                    if (!mbar_wait_try(&full_k[s], (uint32_t)((i >> 1) & 1), a.err)) return false;
                    tc_fence_after();
                    const uint32_t k = qs + L::K + s * kTileBytes;
#pragma unroll
                    for (int t = TERMS - 1; t >= 0; --t)  // the small terms first: fewer roundings at the sum's size
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            mma_ss(tmem + L::S_COL + s * L::S_STEP,
                                   sdesc(qs + t * L::QTERM + (kk >> 2) * (kRows * 128) + (kk & 3) * 32, 16),
                                   sdesc(k + (kk >> 2) * kHalf + (kk & 3) * 32, 16), id_s, t < TERMS - 1 || kk);
                    mma_commit(&s_full[s]);
                }
                if (i > 0) {
                    const int j = i - 1;
                    if (!mbar_wait_try(&full_v[o], (uint32_t)((j >> 1) & 1), a.err)) return false;
                    if (!mbar_wait_try(&p_full[o], (uint32_t)((j >> 1) & 1), a.err)) return false;
                    tc_fence_after();
                    const uint32_t v = qs + L::V + o * kTileBytes;
                    const bool more = TERMS == 1 ? j > 0 : j % kFlush > 0;
#pragma unroll
                    for (int t = L::PTERMS - 1; t >= 0; --t) {
                        const int apart = L::ACCS == 2 && t > 0;  // in the small terms' accumulator
                        const bool begins = t == L::PTERMS - 1 || (L::ACCS == 2 && t == 0);  // the first product of its accumulator
#pragma unroll
                        for (int kk = 0; kk < TILE / 16; ++kk)
                            mma_ts(tmem + apart * kD, tmem + L::S_COL + o * L::S_STEP + t * (TILE / 2) + kk * 8,
                                   sdesc(v + kk * 2048, kHalf), id_o, more || !begins || kk);
                    }
                    mma_commit(&o_full[o]);
                }
                return true;
            };
            for (int i = 0; i <= n; i += 2)
                if (!step(i, std::integral_constant<int, 0>{}) ||
                    (i < n && !step(i + 1, std::integral_constant<int, 1>{})))
                    break;
        }
        __syncwarp();
    } else if (warp < 4) {
        // ---------------- softmax: thread = one query row
        const int r = threadIdx.x;
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        {
            // Q, 16 lanes per row: 8 dims each, split into terms
            const int c = lane & 15, half = c >> 3;
            auto place = [&](int qr, int k) {
                return reinterpret_cast<uint4*>(smem + k * L::QTERM + half * (kRows * 128) + qr * 128 + (((c & 7) ^ (qr & 7)) << 4));
            };
            if constexpr (TERMS == 1) {
                // as they lie: asynchronous copies, all in flight at once (rows that are not there: zeros)
#pragma unroll
                for (int g = 0; g < 16; ++g) {
                    const int qr = 8 * g + 2 * warp + (lane >> 4), m = min(qr >> 1, job.count - 1);
                    const size_t at = (size_t)(list.n ? rows.r[job.first + m].row : job.first + m) * a.q_stride +
                                      (size_t)(job.head * kG + (qr & 1)) * kD + 8 * c;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(place(qr, 0))),
                                 "l"(static_cast<const uint16_t*>(a.q) + at), "r"((qr >> 1) < job.count ? 16 : 0)
                                 : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
            } else {
                constexpr int kAhead = 4;
#pragma unroll 1
                for (int g = 0; g < 16; g += kAhead) {
                    float4 x[kAhead][2];
#pragma unroll
                    for (int e = 0; e < kAhead; ++e) {
                        const int qr = 8 * (g + e) + 2 * warp + (lane >> 4), m = qr >> 1;
                        x[e][0] = x[e][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (m < job.count) {
                            const size_t at = (size_t)(list.n ? rows.r[job.first + m].row : job.first + m) * a.q_stride +
                                              (size_t)(job.head * kG + (qr & 1)) * kD + 8 * c;
                            x[e][0] = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at));
                            x[e][1] = __ldcg(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at + 4));
                        }
                    }
#pragma unroll
                    for (int e = 0; e < kAhead; ++e) {
                        const int qr = 8 * (g + e) + 2 * warp + (lane >> 4);
                        uint32_t t[4][TERMS];
                        split_pair<TERMS>(x[e][0].x, x[e][0].y, t[0]);
                        split_pair<TERMS>(x[e][0].z, x[e][0].w, t[1]);
                        split_pair<TERMS>(x[e][1].x, x[e][1].y, t[2]);
                        split_pair<TERMS>(x[e][1].z, x[e][1].w, t[3]);
#pragma unroll
                        for (int k = 0; k < TERMS; ++k) *place(qr, k) = make_uint4(t[0][k], t[1][k], t[2][k], t[3][k]);
                    }
                }
            }
            fence_proxy_async_smem();
            asm volatile("bar.sync 1, 160;" ::: "memory");
        }
        const int pos = min(job.p0 + (r >> 1), job.p1);  // this row's position (chunk)
        const int low = window_low(pos, a.window), low1 = window_low(job.p1, a.window);
        const float scale2 = kLog2e / sqrtf((float)kD);
        float m_ref = -INFINITY, l = 0.0f;  // reference point (log2 units) and sum of the exponentials
        float* total = reinterpret_cast<float*>(smem + L::TOTAL) + r;  // this row's (f32 queries)
        bool alive = true;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            alive = __all_sync(kAll, mbar_wait_try(&s_full[i & 1], (uint32_t)((i >> 1) & 1), a.err));
            if (!alive) break;
            tc_fence_after();
            const uint32_t s_at = tmem + L::S_COL + (i & 1) * L::S_STEP + lane_base;
            float s[TILE];
            tmem_ld32(s_at, reinterpret_cast<uint32_t*>(s));
            tmem_ld32(s_at + 32, reinterpret_cast<uint32_t*>(s + 32));
            tmem_wait_ld();
            const int v0 = (job.t_lo + i) * kTileBlocks;
            const int b0 = job.span.block(v0), b1 = job.span.block(v0 + kTileBlocks - 1);
            const bool whole = v0 + kTileBlocks <= job.span.total && v0 >= job.span.nsb &&
                               b1 * kKvBlock + kKvBlock - 1 <= job.p0 && (list.n || b0 * kKvBlock >= low1);
            if (!whole) {
#pragma unroll
                for (int u = 0; u < kTileBlocks; ++u) {
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
            if (__any_sync(kAll, grow)) {
                const float m_new = grow ? mt : m_ref;
                const float c = grow ? exp2f(m_ref - m_new) : 1.0f;
                l *= c;
                m_ref = m_new;
                if (i > 0) {
                    // the accumulator, once P V of the tile before is done (that of tile
                    // i waits for this warp)
                    const int j = i - 1;
                    alive = __all_sync(kAll, mbar_wait_try(&o_full[j % L::VST], (uint32_t)((j / L::VST) & 1), a.err));
                    if (!alive) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int d = 0; d < L::ACCS * kD; d += 32) {
                        uint32_t o[32];
                        tmem_ld32(tmem + lane_base + d, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * c);
                        tmem_st32(tmem + lane_base + d, o);
                    }
                    if (TERMS > 1 && i > kFlush)
#pragma unroll 8
                        for (int d = 0; d < kD; ++d) total[d * kRows] *= c;
                }
            }
            if (TERMS > 1 && i > 0 && i % kFlush == 0) {
                const int j = i - 1;
                alive = __all_sync(kAll, mbar_wait_try(&o_full[j % L::VST], (uint32_t)((j / L::VST) & 1), a.err));
                if (!alive) break;
                tc_fence_after();
                tmem_wait_st();  // of the rescaling
#pragma unroll 1
                for (int d = 0; d < kD; d += 16) {
                    uint32_t o[16], low_o[16];
                    tmem_ld16(tmem + lane_base + d, o);
                    tmem_ld16(tmem + kD + lane_base + d, low_o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float x = __uint_as_float(o[e]) + __uint_as_float(low_o[e]);
                        total[(d + e) * kRows] = i == kFlush ? x : total[(d + e) * kRows] + x;
                    }
                }
            }
            const float neg = m_ref == -INFINITY ? 0.0f : -m_ref;
            const u64x2 scale_2 = pack2(scale2, scale2), neg_2 = pack2(neg, neg);
            u64x2 sum[2] = {0ull, 0ull};
            uint32_t p[L::PTERMS][32];
#pragma unroll
            for (int e = 0; e < 32; ++e) {
                float x0, x1;
                unpack2(fma2(pack2(s[2 * e], s[2 * e + 1]), scale_2, neg_2), x0, x1);
                x0 = exp2_fast(x0);
                x1 = exp2_fast(x1);
                sum[e & 1] = add2(sum[e & 1], pack2(x0, x1));
                uint32_t u[L::PTERMS];
                split_pair<L::PTERMS>(x0, x1, u);
#pragma unroll
                for (int k = 0; k < L::PTERMS; ++k) p[k][e] = u[k];
            }
#pragma unroll
            for (int k = 0; k < L::PTERMS; ++k) tmem_st32(s_at + k * (TILE / 2), p[k]);
            float l0, l1;
            unpack2(add2(sum[0], sum[1]), l0, l1);
            l += l0 + l1;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[i & 1]);
        }
        // ---- the result: through shared memory (Q, K and V are read), so that
        // whole rows are stored together
        if (n > 0) alive = __all_sync(kAll, alive && mbar_wait_try(&o_full[(n - 1) % L::VST], (uint32_t)(((n - 1) / L::VST) & 1), a.err));
        tc_fence_after();
        const bool direct = list.n == 0 && job.nseg == 1;
        const int n_q = a.n_kv * kG;
        if (alive) {
            const float inv = !direct ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
            bool finite = fabsf(l) < INFINITY;
#pragma unroll 1
            for (int d = 0; d < kD; d += 32) {
                uint32_t u[32], low_u[32];
                if (n > 0) {
                    tmem_ld32(tmem + lane_base + d, u);
                    if (L::ACCS == 2) tmem_ld32(tmem + kD + lane_base + d, low_u);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) u[e] = low_u[e] = 0u;
                }
                tmem_wait_ld();
                float o[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    o[e] = __uint_as_float(u[e]);
                    if (L::ACCS == 2) o[e] += __uint_as_float(low_u[e]);
                    if (TERMS > 1 && n > kFlush) o[e] += total[(d + e) * kRows];
                    finite = finite && fabsf(o[e]) < INFINITY;
                    o[e] *= inv;
                }
                if (TERMS == 1 && direct) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        *reinterpret_cast<uint4*>(smem + r * 256 + ((((d + e) >> 3) ^ (r & 7)) << 4)) =
                            make_uint4(pack_bf16(o[e], o[e + 1]), pack_bf16(o[e + 2], o[e + 3]), pack_bf16(o[e + 4], o[e + 5]),
                                       pack_bf16(o[e + 6], o[e + 7]));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<float4*>(smem + r * 512 + ((((d + e) >> 2) ^ (r & 7)) << 4)) =
                            make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
            if ((r >> 1) < job.count) {
                if (!finite) atomicOr(&bad_rows[warp], 1u << lane);
                if (!direct) {
                    float* rec = a.part + (((size_t)(job.first + (r >> 1)) * n_q + job.head * kG + (r & 1)) * a.max_segs + job.seg) * kRecord;
                    *reinterpret_cast<float2*>(rec) = make_float2(m_ref, l);
                }
            }
            __syncwarp();
            // this warp's 32 rows
            if (TERMS == 1 && direct) {
#pragma unroll 4
                for (int g = 0; g < 16; ++g) {
                    const int qr = 32 * warp + 2 * g + (lane >> 4), c = lane & 15, m = job.first + (qr >> 1);
                    if ((qr >> 1) < job.count)
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (size_t)m * a.out_stride +
                                                  (size_t)(job.head * kG + (qr & 1)) * kD + 8 * c) =
                            *reinterpret_cast<const uint4*>(smem + qr * 256 + ((c ^ (qr & 7)) << 4));
                }
            } else {
#pragma unroll 4
                for (int g = 0; g < 32; ++g) {
                    const int qr = 32 * warp + g, m = job.first + (qr >> 1), hq = job.head * kG + (qr & 1);
                    const float4 x = *reinterpret_cast<const float4*>(smem + qr * 512 + ((lane ^ (qr & 7)) << 4));
                    if ((qr >> 1) < job.count) {
                        float* to = direct ? static_cast<float*>(a.out) + (size_t)m * a.out_stride + (size_t)hq * kD + 4 * lane
                                           : a.part + (((size_t)m * n_q + hq) * a.max_segs + job.seg) * kRecord + 4 + 4 * lane;
                        *reinterpret_cast<float4*>(to) = x;
                    }
                }
            }
        }
        __syncwarp();
        // rows that are not finite, position by position over this CTA's blocks
        for (uint32_t bad = bad_rows[warp]; bad; bad &= bad - 1) {
            const int x = 32 * warp + __ffs(bad) - 1;
            const int m = job.first + (x >> 1), qrow = list.n ? rows.r[m].row : m, hq = job.head * kG + (x & 1);
            const int p = list.n ? job.p1 : job.p0 + (x >> 1);
            const SlowRow row = slow_row(a, qrow, hq, job.slot, p, list.n ? 0 : window_low(p, a.window), list.n ? 0 : a.sinks,
                                         job.span, job.t_lo * kTileBlocks, min((job.t_lo + n) * kTileBlocks, job.span.total));
            if (direct) store_row(a, qrow, hq, row);
            else store_record(a.part + (((size_t)m * n_q + hq) * a.max_segs + job.seg) * kRecord, row);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 6) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(L::COLS) : "memory");
    }
}

}  // namespace

template <int N>
void launch_sized(const CUtensorMap& kv_map, const ServeRowsT<N>& rows, const TileListT<N>& list, const ServeAttnArgs& a,
                  int items, cudaStream_t st) {
    if (a.bf16) launch_pdl(attn_tile_kernel<1, N>, items, kThreads, Lay<1>::SMEM, st, kv_map, rows, list, a);
    else launch_pdl(attn_tile_kernel<3, N>, items, kThreads, Lay<3>::SMEM, st, kv_map, rows, list, a);
}

void launch_attn_tile(const CUtensorMap& kv_map, const ServeRows& rows, const TileList& list, const ServeAttnArgs& a,
                      int items, cudaStream_t st) {
    if (a.batch <= kServeSmallBatch)
        with_rows<kServeSmallBatch>(rows, [&](const ServeRowsT<kServeSmallBatch>& r) {
            launch_sized(kv_map, r, first_tiles<kServeSmallBatch>(list, items), a, items, st);
        });
    else if (a.batch <= kServeMidBatch)
        with_rows<kServeMidBatch>(rows, [&](const ServeRowsT<kServeMidBatch>& r) {
            launch_sized(kv_map, r, first_tiles<kServeMidBatch>(list, items), a, items, st);
        });
    else launch_sized(kv_map, rows, list, a, items, st);
}

void prepare_attn_tile_kernels() {
    configure_kernel((const void*)attn_tile_kernel<1, kServeSmallBatch>, Lay<1>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<3, kServeSmallBatch>, Lay<3>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<1, kServeMidBatch>, Lay<1>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<3, kServeMidBatch>, Lay<3>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<1, kServeMaxBatch>, Lay<1>::SMEM);
    configure_kernel((const void*)attn_tile_kernel<3, kServeMaxBatch>, Lay<3>::SMEM);
}

}  // namespace zc
