// Serving attention of single tokens: one query per sequence over the blocks
// of its cache that it sees (sinks and window, or what is left of it after a
// common prompt that attn_tile.cu takes).
//
// Bound by the bytes of K and V, so built to stream: persistent and
// warp-granular. The work is the list of (row, kv head, visible 16-token
// block), row-major; every warp of the grid takes a contiguous share of equal
// cost, whatever the rows' lengths (a (row, kv head) costs kSpanLead blocks beside its
// own: its query's way in and its result's way out; without them warps with many
// short rows finished last, 36 against 13 us), through a private ring of kRing 8 KB slots (K
// then V of one block and head are contiguous) filled by cp.async.bulk. Two
// blocks of one (row, kv head) are taken per step, on the tensor cores
// (mma.sync m16n8k16, bf16 in, f32 out; a query's 2 heads are too few rows for
// a tcgen05 tile, and the products are a tenth of the streaming time):
//   S[16 tokens][8] = K . Q columns, the columns being three bf16 terms of each
//     head's q (24 bits: nothing of an f32 q is lost; K is exact bf16), then
//   O[8 rows][128] += P . V with P's rows the three terms of each head's p.
// Maximum, sum and accumulators are f32, exponentials in powers of two.
// The pieces of a (row, kv head) that meet in one CTA are joined in shared
// memory; what crosses CTAs meets in global records that the last CTA of the
// row joins in a fixed order (an atomic counter tells which is last; nothing
// waits). A row with a common prompt leaves its records to serve_attn.cu's join.
//
// Measured: 64 rows that see 1028 positions each, 8 kv heads: 53.1 us a call, one after
// another on a stream, 5.1 TB/s, 78 % of the card's copy rate; 46.4 us and 89 % where
// calls on other streams fill the start and the end. One such row: 28 us for a lone
// call, of which the kernel's chain (parameters, block table, K and V, joins in and
// across CTAs) is 11.4.
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "serve_common.cuh"

namespace zc {

namespace {

using namespace serve;
using attn::ldsm_x4;
using attn::ldsm_x4_trans;
using attn::mma_bf16;

constexpr int kWarps = 8, kThreads = kWarps * kWarp;
constexpr int kRing = 3;
constexpr int kBlockBytes = kBlockElems * 2, kSlotBytes = 2 * kBlockBytes;
constexpr int kIdRing = 64;  // block places of a warp's share, two chunks of 32
// Blocks after which the accumulators are added to sums of their own: the MMA rounds
// its sums toward 0, an error that grows with their number. The sums lie in the
// accumulators' rows 8 - 15, to which P's rows of zeros there add nothing. Measured
// relative error, 16 rows of 65536 positions: 8.2e-6 without, 7e-7 with.
constexpr int kFlush = 32;
constexpr int kPair = kG * kRecord;  // a record of both query heads of a kv head
constexpr unsigned kAll = 0xFFFFFFFFu;

struct Smem {
    unsigned char ring[kWarps][kRing][kSlotBytes];
    float rec[2][kWarps][kPair];  // piece that began before the warp's share (0) or goes on past it (1)
    uint64_t full[kWarps][kRing];
    uint32_t kidx[kWarps][kIdRing];
    int rec_gid[2][kWarps];
    long long bound[kWarps + 1];  // first block of each warp's share
    int pref[kServeMaxBatch + 1];
    ServeRow info[kServeMidBatch];  // the rows, where they fit
};
static_assert(sizeof(Smem) + 1024 <= 232448, "span attention shared memory");

// Two values' bf16 term `term` (0 high, 1 middle, 2 low), packed.
__device__ __forceinline__ uint32_t term_of(float x0, float x1, int term) {
    uint32_t t = pack_bf16(x0, x1);
    if (term > 0) {
        x0 -= bf16lo(t);
        x1 -= bf16hi(t);
        t = pack_bf16(x0, x1);
        if (term > 1) t = pack_bf16(x0 - bf16lo(t), x1 - bf16hi(t));
    }
    return t;
}

// x joined with a record in shared memory (NaN and infinities as in join_records).
__device__ __forceinline__ void join_shared(Partial& x, const float* rec) {
    const float m = rec[0], l = rec[1];
    if (m == -INFINITY && l == 0.0f) return;  // nothing seen
    const float4 v = *reinterpret_cast<const float4*>(rec + 4 + 4 * (threadIdx.x % kWarp));
    const float mn = fmaxf(x.m, m);
    const float c0 = x.m == -INFINITY ? 0.0f : exp2_fast(x.m - mn), c1 = exp2_fast(m - mn);
    x.m = mn;
    x.l = x.l * c0 + l * c1;
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x.acc[e] = x.acc[e] * c0 + f[e] * c1;
}

// A piece whose result is not finite once more, position by position, a warp together:
// P's rows and terms that are 0 make a NaN of an infinite V, and the terms of an
// infinite q one of its scores. rec: the records of both heads; null: the output.
// (All by value: what a call passes by address would be kept in local memory.)
static __device__ __noinline__ void redo_piece(const ServeAttnArgs& a, int row, int slot, int pos, int head, int v0, int v1,
                                               int skip, float* rec, size_t rec_step) {
    const Span span = span_of(pos, pos, a.window, a.sinks, skip);
#pragma unroll 1
    for (int h = 0; h < kG; ++h) {
        const Partial x = slow_row(a, row, head * kG + h, slot, pos, window_low(pos, a.window), a.sinks, span, v0, min(v1, span.total));
        if (rec) store_record(rec + h * rec_step, x, 1);
        else store_row(a, row, head * kG + h, x);
    }
}

template <int N>
__global__ void __launch_bounds__(kThreads, 1)
    attn_span_kernel(const __grid_constant__ ServeRowsT<N> rows_param, const __grid_constant__ ServeAttnArgs a) {
    const ServeRowsT<N>& rows = as_memory(rows_param);
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    unsigned char* ring = sm.ring[warp][0];
    uint64_t* full = sm.full[warp];
    uint32_t* kidx = sm.kidx[warp];
    const int B = a.batch;
    auto info = [&](int b) {
        const int4 x = *reinterpret_cast<const int4*>(N <= kServeMidBatch ? &sm.info[b] : &rows.r[b]);
        return ServeRow{x.x, x.y, x.z, (uint32_t)x.w};
    };
    auto span_row = [&](const ServeRow& r) { return span_of(r.len - 1, r.len - 1, a.window, a.sinks, r.skip()); };

    // prefix of the rows' block counts; a row that sees nothing here counts one
    if (warp == 0) {
        int carry = 0;
        constexpr int kAhead = N < 256 ? N / kWarp : 8;
        for (int base0 = 0; base0 < B; base0 += kAhead * kWarp) {
            int4 w[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (base0 + k * kWarp + lane < B) w[k] = *reinterpret_cast<const int4*>(&rows.r[base0 + k * kWarp + lane]);
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int b = base0 + k * kWarp + lane;
                int x = 0;
                if (b < B) {
                    const ServeRow r{w[k].x, w[k].y, w[k].z, (uint32_t)w[k].w};
                    if (N <= kServeMidBatch) sm.info[b] = r;
                    x = max(1, span_row(r).total);
                }
#pragma unroll
                for (int o = 1; o < kWarp; o <<= 1) {
                    const int y = __shfl_up_sync(kAll, x, o);
                    if (lane >= o) x += y;
                }
                if (b < B) sm.pref[b + 1] = carry + x;
                carry += __shfl_sync(kAll, x, kWarp - 1);
            }
        }
        if (lane == 0) sm.pref[0] = 0;
    }
    if (lane == 0) {
        for (int s = 0; s < kRing; ++s) mbar_init(&full[s], 1);
        fence_barrier_init();
    }
    if (lane < 2) sm.rec_gid[lane][warp] = -1;
    __syncthreads();
    const int* pref = sm.pref;
    // cost units: kSpanLead of every (row, kv head), then its blocks. Block f of row b
    // is unit f + kSpanLead (b n_kv + head + 1); first_block(u) is the first block at
    // or after unit u.
    const long long total = (long long)pref[B] * a.n_kv, units = total + (long long)kSpanLead * B * a.n_kv;
    auto first_block = [&](long long u) -> long long {
        if (u >= units) return total;
        int l = 0, h = B - 1;
        while (l < h) {
            const int mid = (l + h + 1) / 2;
            if ((long long)a.n_kv * (pref[mid] + kSpanLead * mid) <= u) l = mid;
            else h = mid - 1;
        }
        const int nblk = pref[l + 1] - pref[l], r = (int)(u - (long long)a.n_kv * (pref[l] + kSpanLead * l));
        return (long long)a.n_kv * pref[l] + (long long)(r / (nblk + kSpanLead)) * nblk + max(0, r % (nblk + kSpanLead) - kSpanLead);
    };
    const int nwarps = gridDim.x * kWarps;
    const int per = (int)((units + nwarps - 1) / nwarps);
    const long long reach = (long long)kWarps * per;  // units of a CTA
    if (warp == 0 && lane <= kWarps) sm.bound[lane] = first_block(blockIdx.x * reach + (long long)lane * per);
    __syncthreads();
    const long long* bound = sm.bound;
    const long long c_lo = bound[0], c_hi = bound[kWarps];
    const long long lo = bound[warp];
    const int n = (int)(bound[warp + 1] - lo);

    struct Cursor {
        int b, head, blk, nblk;
    };
    auto locate = [&](long long f, Cursor& c) {
        int l = 0, h = B - 1;
        while (l < h) {
            const int mid = (l + h + 1) / 2;
            if ((long long)a.n_kv * pref[mid] <= f) l = mid;
            else h = mid - 1;
        }
        c.b = l;
        c.nblk = pref[l + 1] - pref[l];
        const int r = (int)(f - (long long)a.n_kv * pref[l]);
        c.head = r / c.nblk;
        c.blk = r % c.nblk;
    };
    auto advance = [&](Cursor& c) {
        if (++c.blk < c.nblk) return;
        c.blk = 0;
        if (++c.head < a.n_kv) return;
        c.head = 0;
        ++c.b;
        c.nblk = c.b < B ? pref[c.b + 1] - pref[c.b] : 1;
    };
    // places of this warp's blocks in the pool, 32 at a time, one lane each
    auto fill_chunk = [&](int c) {
        const int j = kWarp * c + lane;
        if (j < n) {
            Cursor x;
            locate(lo + j, x);
            const ServeRow r = info(x.b);
            const Span span = span_row(r);
            int id = 0;  // a row that sees nothing reads some block and weighs none of it
            if (x.blk < span.total) {
                id = a.block_table[(size_t)r.slot * a.max_blocks + span.block(x.blk)];
                if (id < 0 || id >= a.n_pool_blocks) {
                    if (a.err) atomicOr(a.err, kErrBadIndex);
                    id = 0;
                }
            }
            kidx[j % kIdRing] = (uint32_t)x.head * (uint32_t)a.n_pool_blocks + (uint32_t)id;
        }
        __syncwarp();
    };
    auto issue = [&](int j, int s) {  // lane 0: K and V of block j of the share, read once: evict-first in L2
        mbar_arrive_expect_tx(&full[s], kSlotBytes);
        bulk_g2s_hint(ring + s * kSlotBytes, a.kv_layer + (size_t)kidx[j % kIdRing] * (2 * kBlockElems), kSlotBytes, &full[s],
                      l2_evict_first_policy());
    };

    const int g = lane >> 2, t = lane & 3;
    const int mi = lane >> 3, ri = lane & 7;
    const int tok_a = ri + (mi & 1) * 8;             // row this lane addresses for ldmatrix
    const int hsel = (g >> 1) & 1, term = (g & 4) ? ((g & 1) ? 3 : 2) : (g & 1);  // head and term of row / column g (3: none)
    const float scale2 = kLog2e / sqrtf((float)kD);

    // this lane's values of a row's query: dims 16 ks + 8 hf + 2 t, + 1 of head hsel
    float2 qv[8][2];
    auto load_q = [&](int row, int head) {
        const size_t at = (size_t)row * a.q_stride + (size_t)(head * kG + hsel) * kD + 2 * t;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const size_t x = at + 16 * ks + 8 * hf;
                if (a.bf16) {
                    const uint32_t two = __ldcg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) + x));
                    qv[ks][hf] = make_float2(bf16lo(two), bf16hi(two));
                } else {
                    qv[ks][hf] = __ldcg(reinterpret_cast<const float2*>(static_cast<const float*>(a.q) + x));
                }
            }
    };

    // The cache was written by earlier kernels. After a tile kernel (which
    // waited for those before it let this one start) it may be read at once;
    // the tile's records and the buffers are touched after the wait below.
    if (!a.early) pdl_wait();
    Cursor cc;
    locate(min(lo, total - 1), cc);
    ServeRow cur = info(cc.b);
    if (n > 0) load_q(cur.row, cc.head);  // in front of the blocks, not behind them
    fill_chunk(0);
    if (lane == 0)
        for (int j = 0; j < min(kRing, n); ++j) issue(j, j);
    pdl_launch_dependents();

    uint32_t qf[8][2];
    float acc[16][4];
    float m_run = -INFINITY, l_run = 0.0f;  // lanes t = 0, 1: head t
    int pos = 0, low = 0, since = 0, blk0 = 0;  // since: blocks since the last flush; blk0: the piece's first
    Span span{};
    bool seg_start = true;

    // blocks i and, if nb is 2, i + 1 of the share, both of one (row, kv head); a
    // lone block is taken twice, the second time with no position seen
    auto run_blocks = [&](int i, int nb) -> bool {
        constexpr int NB = 2;
        bool ok = true;
        for (int u = 0; u < nb; ++u)
            ok = mbar_wait_bounded(&full[(i + u) % kRing], (uint32_t)(((i + u) / kRing) & 1), a.err) && ok;
        if (!__all_sync(kAll, ok)) return false;
        uint32_t kbase[NB], bits[NB];
        bool patched = false;
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            unsigned char* kb = ring + ((i + (u < nb ? u : 0)) % kRing) * kSlotBytes;
            kbase[u] = smem_addr(kb);
            const int v = cc.blk + u;
            bits[u] = u < nb && v < span.total ? seen_bits(span.block(v), pos, low, a.sinks) : 0u;
            if (u < nb && bits[u] != 0xFFFFu) {
                // positions that are not seen: p = 0 there, but 0 times a NaN that lies there is NaN
                for (int x = lane; x < kKvBlock * (kD * 2 / 16); x += kWarp)
                    if (!((bits[u] >> (x / 16)) & 1u)) reinterpret_cast<uint4*>(kb + kBlockBytes)[x] = make_uint4(0, 0, 0, 0);
                patched = true;
            }
        }
        __syncwarp();
        float sc[NB][4], sd[NB][4];  // even / odd k-steps
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[u][e] = sd[u][e] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            const int ch = 2 * ks + (mi >> 1);
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                uint32_t a0, a1, a2, a3;
                ldsm_x4(kbase[u] + tok_a * (kD * 2) + ((ch ^ ri) << 4), a0, a1, a2, a3);
                if (ks & 1) mma_bf16(sd[u], a0, a1, a2, a3, qf[ks][0], qf[ks][1]);
                else mma_bf16(sc[u], a0, a1, a2, a3, qf[ks][0], qf[ks][1]);
            }
        }
        // columns: (h0 high, middle), (h1 high, middle), (h0 low, 0), (h1 low, 0):
        // lanes t = 0, 1 take head t's scores for tokens g and g + 8
        float s0[NB], s1[NB], mt = -INFINITY;
#pragma unroll
        for (int u = 0; u < NB; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[u][e] += sd[u][e];
            const float x0 = __shfl_xor_sync(kAll, sc[u][0], 2), x1 = __shfl_xor_sync(kAll, sc[u][2], 2);
            s0[u] = t < 2 && ((bits[u] >> g) & 1u) ? (sc[u][0] + (sc[u][1] + x0)) * scale2 : -INFINITY;
            s1[u] = t < 2 && ((bits[u] >> (g + 8)) & 1u) ? (sc[u][2] + (sc[u][3] + x1)) * scale2 : -INFINITY;
            mt = fmaxf(mt, fmaxf(s0[u], s1[u]));
        }
        mt = fmaxf(mt, __shfl_xor_sync(kAll, mt, 4));
        mt = fmaxf(mt, __shfl_xor_sync(kAll, mt, 8));
        mt = fmaxf(mt, __shfl_xor_sync(kAll, mt, 16));
        const float m_new = fmaxf(m_run, mt);
        if (__any_sync(kAll, m_new > m_run)) {
            const float corr = m_new > m_run ? exp2f(m_run - m_new) : 1.0f;
            l_run *= corr;
            const float ca = __shfl_sync(kAll, corr, hsel);
#pragma unroll
            for (int nt = 0; nt < 16; ++nt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][e] *= ca;
            }
            m_run = m_new;
        }
        const float ref = m_run == -INFINITY ? 0.0f : m_run;
        // P as the A operand: lane (g, t) holds row g at tokens 2t, 2t + 1 (a0)
        // and 2t + 8, 2t + 9 (a2); p(h, token) sits in lane 4 (token % 8) + h
        const int src0 = 8 * t + hsel, src1 = src0 + 4;
        uint32_t pa0[NB], pa2[NB];
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            const float p0 = exp2f(s0[u] - ref), p1 = exp2f(s1[u] - ref);
            l_run += p0 + p1;
            const float x0 = __shfl_sync(kAll, p0, src0), x8 = __shfl_sync(kAll, p1, src0);
            const float x1 = __shfl_sync(kAll, p0, src1), x9 = __shfl_sync(kAll, p1, src1);
            pa0[u] = term < 3 ? term_of(x0, x1, term) : 0u;
            pa2[u] = term < 3 ? term_of(x8, x9, term) : 0u;
        }
#pragma unroll
        for (int np = 0; np < 8; ++np) {
            const int ch = 2 * np + (mi >> 1);
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4_trans(kbase[u] + kBlockBytes + tok_a * (kD * 2) + ((ch ^ ri) << 4), b0, b1, b2, b3);
                mma_bf16(acc[2 * np], pa0[u], 0u, pa2[u], 0u, b0, b1);
                mma_bf16(acc[2 * np + 1], pa0[u], 0u, pa2[u], 0u, b2, b3);
            }
        }
        if (patched) fence_proxy_async_smem();  // generic writes above, bulk copy next
        __syncwarp();
        for (int u = 0; u < nb; ++u) {
            const int jn = i + u + kRing;
            if (jn < n && jn % kWarp == 0) fill_chunk(jn / kWarp);
            if (lane == 0 && jn < n) issue(jn, (i + u) % kRing);
        }
        return true;
    };

    bool waited = !a.early;
    for (int i = 0; i < n;) {
        if (seg_start) {
            // this row's query as the B operand: column g holds term(g) of head hsel(g)
            if (i > 0) {
                cur = info(cc.b);
                load_q(cur.row, cc.head);
            }
            pos = cur.len - 1;
            low = window_low(pos, a.window);
            span = span_row(cur);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) qf[ks][hf] = term < 3 ? term_of(qv[ks][hf].x, qv[ks][hf].y, term) : 0u;
#pragma unroll
            for (int nt = 0; nt < 16; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
            m_run = -INFINITY;
            l_run = 0.0f;
            since = 0;
            blk0 = cc.blk;
            seg_start = false;
        }
        const int nb = (i + 1 < n && cc.blk + 1 < cc.nblk) ? 2 : 1;
        if (!run_blocks(i, nb)) {
            // the copies in flight land before the warp stops; the error word reports the launch
            if (lane == 0)
                for (int j = i; j < min(n, i + kRing); ++j)
                    mbar_wait_bounded(&full[j % kRing], (uint32_t)((j / kRing) & 1), nullptr);
            __syncwarp();
            break;
        }
        if (nb == 2) advance(cc);
        i += nb;
        since += nb;
        if (since >= kFlush) {
            since = 0;
#pragma unroll
            for (int nt = 0; nt < 16; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    acc[nt][2 + e] += acc[nt][e];
                    acc[nt][e] = 0.0f;
                }
        }
        if (cc.blk == cc.nblk - 1 || i == n) {
            // end of this warp's piece: to the output if it is the whole row, else to its record
            float L = l_run;
            L += __shfl_xor_sync(kAll, L, 4);
            L += __shfl_xor_sync(kAll, L, 8);
            L += __shfl_xor_sync(kAll, L, 16);
            const float Lh = __shfl_sync(kAll, L, hsel), Mh = __shfl_sync(kAll, m_run, hsel);
#pragma unroll
            for (int nt = 0; nt < 16; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {  // the terms' rows added up, the small ones first: rows 0 and 2 hold the heads
                    const float x = acc[nt][e] + acc[nt][2 + e];
                    const float lo_sum = __shfl_xor_sync(kAll, x, 16), mid = __shfl_xor_sync(kAll, x, 4);
                    acc[nt][e] = x + (mid + lo_sum);
                }
            const bool writer = (g & 5) == 0 && g < 4;
            bool finite = fabsf(Lh) < INFINITY;
#pragma unroll
            for (int nt = 0; nt < 16; ++nt) finite = finite && fabsf(acc[nt][0]) < INFINITY && fabsf(acc[nt][1]) < INFINITY;
            const bool redo = !__all_sync(kAll, finite || !writer);
            const long long f0 = (long long)a.n_kv * pref[cc.b] + (long long)cc.head * cc.nblk;
            const bool whole = f0 >= lo && f0 + cc.nblk <= lo + n;
            const int nrec = cur.nrec();
            if (whole && nrec == 0 && !waited) {
                pdl_wait();  // (the output may still be read)
                waited = true;
            }
            if (redo) {
                const int k = f0 < lo ? 0 : 1;
                const size_t at = ((size_t)cc.b * (a.n_kv * kG) + cc.head * kG) * a.max_segs + nrec;
                redo_piece(a, cur.row, cur.slot, pos, cc.head, blk0, cc.blk + 1, cur.skip(),
                           !whole ? sm.rec[k][warp] : (nrec > 0 ? a.part + at * kRecord : nullptr),
                           whole ? (size_t)a.max_segs * kRecord : (size_t)kRecord);
                if (!whole && lane == 0) sm.rec_gid[k][warp] = cc.b * a.n_kv + cc.head;
            } else if (whole && nrec == 0) {
                if (writer) {
                    const size_t at = (size_t)cur.row * a.out_stride + (size_t)(cc.head * kG + hsel) * kD + 2 * t;
                    const float inv = Lh == 0.0f ? 0.0f : 1.0f / Lh;
#pragma unroll
                    for (int nt = 0; nt < 16; ++nt) {
                        if (a.bf16)
                            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at + 8 * nt) = pack_bf16(acc[nt][0] * inv, acc[nt][1] * inv);
                        else
                            *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at + 8 * nt) = make_float2(acc[nt][0] * inv, acc[nt][1] * inv);
                    }
                }
            } else {
                // (the records of the call before were joined before the tile kernel started)
                const int k = f0 < lo ? 0 : 1;
                float* rec = whole ? a.part + (((size_t)cc.b * (a.n_kv * kG) + cc.head * kG + hsel) * a.max_segs + nrec) * kRecord
                                   : sm.rec[k][warp] + hsel * kRecord;
                if (writer) {
                    if (t == 0) *reinterpret_cast<float4*>(rec) = make_float4(Mh, Lh, __int_as_float(1), 0.0f);
#pragma unroll
                    for (int nt = 0; nt < 16; ++nt) *reinterpret_cast<float2*>(rec + 4 + 8 * nt + 2 * t) = make_float2(acc[nt][0], acc[nt][1]);
                }
                if (!whole && lane == 0) sm.rec_gid[k][warp] = cc.b * a.n_kv + cc.head;
            }
            seg_start = true;
        }
        advance(cc);
    }
    if (!waited) pdl_wait();

    // ---- join the warps' records of each (row, kv head) of this CTA, in warp
    // order, a warp per query head; a row that goes on in other CTAs through the
    // global records
    __syncthreads();
    Cursor gc;
    locate(min(c_lo, total - 1), gc);
    long long g0 = (long long)a.n_kv * pref[gc.b] + (long long)gc.head * gc.nblk;
#pragma unroll 1
    for (int gi = 0; g0 < c_hi; ++gi) {
        const long long g1 = g0 + gc.nblk;
        const int gb = gc.b, gh = gc.head;
        int wa = kWarps, wb = -1;  // warps with blocks of it
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
            if (max(bound[w], g0) < min(bound[w + 1], g1)) {
                wa = min(wa, w);
                wb = w;
            }
        const int h = (warp - 2 * gi) & (kWarps - 1);  // warps 2 gi, 2 gi + 1 (mod 8) take the two heads
        if (h < kG && wb >= 0 && !(wa == wb && g0 >= bound[wa] && g1 <= bound[wa + 1])) {  // (else its warp stored it)
            const ServeRow r = info(gb);
            const int nrec = r.nrec(), hq = gh * kG + h;
            Partial x = no_partial();
            for (int w = wa; w <= wb; ++w) {
                const int k = g0 >= bound[w] ? 1 : 0;
                if (sm.rec_gid[k][w] == gb * a.n_kv + gh) join_shared(x, sm.rec[k][w] + h * kRecord);  // (else it stopped early)
            }
            const long long lead = (long long)kSpanLead * ((long long)gb * a.n_kv + gh + 1);
            const int first = (int)((g0 + lead) / reach), nown = (int)((g1 - 1 + lead) / reach) - first + 1, seg = (int)blockIdx.x - first;
            float* base = a.part + ((size_t)gb * (a.n_kv * kG) + hq) * a.max_segs * kRecord;
            bool last = true;
            if (nrec + nown > a.max_segs) {
                if (lane == 0 && a.err) atomicOr(a.err, kErrBadIndex);
                last = false;
            } else if (nrec > 0) {
                store_record(base + (size_t)(nrec + seg) * kRecord, x, nown);
                last = false;
            } else if (nown > 1) {
                store_record(base + (size_t)seg * kRecord, x);
                __threadfence();
                __syncwarp();
                unsigned prev = 0;
                unsigned* counter = a.counters + (size_t)gb * (a.n_kv * kG) + hq;
                if (lane == 0) {
                    prev = atomicAdd(counter, 1u);
                    if (prev == (unsigned)(nown - 1)) *counter = 0u;
                }
                last = __shfl_sync(kAll, prev, 0) == (unsigned)(nown - 1);
                __threadfence();
                x = no_partial();
            }
            if (last) {
                if (nown > 1) join_records(x, base, nown);  // the CTAs', in order
                store_out4(a, r.row, hq, x.acc, x.l);
            }
        }
        g0 = g1;
        if (++gc.head == a.n_kv) {
            gc.head = 0;
            ++gc.b;
        }
        gc.nblk = gc.b < B ? pref[gc.b + 1] - pref[gc.b] : 1;
    }
}

}  // namespace

void launch_attn_span(const ServeRows& rows, const ServeAttnArgs& a, int ctas, cudaStream_t st) {
    if (a.batch <= kServeSmallBatch)
        with_rows<kServeSmallBatch>(rows, [&](const ServeRowsT<kServeSmallBatch>& r) {
            launch_pdl(attn_span_kernel<kServeSmallBatch>, ctas, kThreads, sizeof(Smem), st, r, a);
        });
    else if (a.batch <= kServeMidBatch)
        with_rows<kServeMidBatch>(rows, [&](const ServeRowsT<kServeMidBatch>& r) {
            launch_pdl(attn_span_kernel<kServeMidBatch>, ctas, kThreads, sizeof(Smem), st, r, a);
        });
    else launch_pdl(attn_span_kernel<kServeMaxBatch>, ctas, kThreads, sizeof(Smem), st, rows, a);
}

void prepare_attn_span_kernels() {
    configure_kernel((const void*)attn_span_kernel<kServeSmallBatch>, sizeof(Smem));
    configure_kernel((const void*)attn_span_kernel<kServeMidBatch>, sizeof(Smem));
    configure_kernel((const void*)attn_span_kernel<kServeMaxBatch>, sizeof(Smem));
}

}  // namespace zc
