// Serving attention of single tokens: one query per sequence over the blocks
// of its cache that it sees (sinks and window, or what is left of it after a
// common prompt that attn_tile.cu takes).
//
// Bound by the bytes of K and V, so built to stream: persistent and
// warp-granular. The work is the list of (row, kv head, visible 16-token
// block), row-major; every warp of the grid takes an equal contiguous share,
// whatever the rows' lengths, through a private ring of kRing 8 KB slots (K
// then V of one block and head are contiguous) filled by cp.async.bulk. Two
// blocks of one (row, kv head) are taken per step, on the tensor cores
// (mma.sync m16n8k16, bf16 in, f32 out; a query's 2 heads are too few rows for
// a tcgen05 tile, and the products are a tenth of the streaming time):
//   S[16 tokens][8] = K . Q columns, the columns being three bf16 terms of each
//     head's q (24 bits: nothing of an f32 q is lost; K is exact bf16), then
//   O[8 rows][128] += P . V with P's rows the three terms of each head's p.
// Maximum, sum and accumulators are f32, exponentials in powers of two.
// The pieces of a (row, kv head) that meet in one CTA are joined in shared
// memory; what crosses CTAs, and a common prompt's partial results, meet in
// global records that the last CTA of the row joins in a fixed order (an
// atomic counter tells which is last; nothing waits).
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
constexpr int kPair = kG * kRecord;  // a record of both query heads of a kv head
constexpr unsigned kAll = 0xFFFFFFFFu;

struct Smem {
    unsigned char ring[kWarps][kRing][kSlotBytes];
    float rec[2][kWarps][kPair];  // piece that began before the warp's share (0) or goes on past it (1)
    uint64_t full[kWarps][kRing];
    uint32_t kidx[kWarps][kIdRing];
    int rec_gid[2][kWarps];
    int pref[kServeMaxBatch + 1];
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

// A merged piece: lane l holds dims 4 l .. 4 l + 3 of both heads.
struct Piece {
    float m[kG], l[kG], acc[kG][4];
};
__device__ __forceinline__ void clear(Piece& p) {
#pragma unroll
    for (int h = 0; h < kG; ++h) {
        p.m[h] = -INFINITY;
        p.l[h] = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) p.acc[h][e] = 0.0f;
    }
}
__device__ __forceinline__ void join(Piece& p, int h, float m, float l, const float4& x) {
    const float mn = fmaxf(p.m[h], m);
    const float c0 = p.m[h] == -INFINITY ? 0.0f : exp2f(p.m[h] - mn), c1 = m == -INFINITY ? 0.0f : exp2f(m - mn);
    p.m[h] = mn;
    p.l[h] = p.l[h] * c0 + l * c1;
    const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) p.acc[h][e] = (c0 == 0.0f ? 0.0f : p.acc[h][e] * c0) + (c1 == 0.0f ? 0.0f : f[e] * c1);
}

template <int N>
__global__ void __launch_bounds__(kThreads, 1)
    attn_span_kernel(const __grid_constant__ ServeRowsT<N> rows, const __grid_constant__ ServeAttnArgs a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    unsigned char* ring = sm.ring[warp][0];
    uint64_t* full = sm.full[warp];
    uint32_t* kidx = sm.kidx[warp];
    const int B = a.batch;
    auto span_row = [&](int b) { return span_of(rows.len[b] - 1, rows.len[b] - 1, a.window, a.sinks, rows.skip[b]); };

    // prefix of the rows' block counts; a row that sees nothing here counts one
    if (warp == 0) {
        int carry = 0;
        for (int base = 0; base < B; base += kWarp) {
            const int b = base + lane;
            int x = b < B ? max(1, span_row(b).total) : 0;
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
                const int y = __shfl_up_sync(kAll, x, o);
                if (lane >= o) x += y;
            }
            if (b < B) sm.pref[b + 1] = carry + x;
            carry += __shfl_sync(kAll, x, kWarp - 1);
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
    const long long total = (long long)pref[B] * a.n_kv;
    const int nwarps = gridDim.x * kWarps;
    const int per = (int)max((total + nwarps - 1) / nwarps, (long long)a.min_per);
    const long long c_lo = (long long)blockIdx.x * kWarps * per, c_hi = min(total, c_lo + (long long)kWarps * per);
    if (c_lo >= total) return;
    const long long lo = c_lo + (long long)warp * per;
    const int n = (int)max(0ll, min(c_hi, lo + per) - lo);

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
            const Span span = span_row(x.b);
            int id = 0;  // a row that sees nothing reads some block and weighs none of it
            if (x.blk < span.total) {
                id = a.block_table[(size_t)rows.slot[x.b] * a.max_blocks + span.block(x.blk)];
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

    // The cache was written by earlier kernels. After a tile kernel (which
    // waited for those before it let this one start) it may be read at once;
    // the tile's records and the buffers are touched after the wait below.
    if (!a.early) pdl_wait();
    Cursor cc;
    locate(lo, cc);
    fill_chunk(0);
    if (lane == 0)
        for (int j = 0; j < min(kRing, n); ++j) issue(j, j);
    pdl_launch_dependents();

    const int g = lane >> 2, t = lane & 3;
    const int mi = lane >> 3, ri = lane & 7;
    const int tok_a = ri + (mi & 1) * 8;             // row this lane addresses for ldmatrix
    const int hsel = (g >> 1) & 1, term = (g & 4) ? ((g & 1) ? 3 : 2) : (g & 1);  // head and term of row / column g (3: none)
    const float scale2 = kLog2e / sqrtf((float)kD);

    uint32_t qf[8][2];
    float acc[16][4];
    float m_run = -INFINITY, l_run = 0.0f;  // lanes t = 0, 1: head t
    int pos = 0, low = 0;
    Span span{};
    bool seg_start = true;

    auto run_blocks = [&](int i, auto nb_c) -> bool {
        constexpr int NB = decltype(nb_c)::value;
        bool ok = true;
#pragma unroll
        for (int u = 0; u < NB; ++u)
            ok = mbar_wait_bounded(&full[(i + u) % kRing], (uint32_t)(((i + u) / kRing) & 1), a.err) && ok;
        if (!__all_sync(kAll, ok)) return false;
        uint32_t kbase[NB], bits[NB];
        bool patched = false;
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            unsigned char* kb = ring + ((i + u) % kRing) * kSlotBytes;
            kbase[u] = smem_addr(kb);
            const int v = cc.blk + u;
            bits[u] = v < span.total ? seen_bits(span.block(v), pos, low, a.sinks) : 0u;
            if (bits[u] != 0xFFFFu) {
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
                acc[nt][0] *= ca;
                acc[nt][1] *= ca;
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
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            const int jn = i + u + kRing;
            if (jn < n && jn % kWarp == 0) fill_chunk(jn / kWarp);
            if (lane == 0 && jn < n) issue(jn, (i + u) % kRing);
        }
        return true;
    };

    // the first `cnt` global records of (row, kv head) into x, kAhead requested at a time
    auto join_global = [&](Piece& x, int b, int head, int cnt) {
        const float* base = a.part + ((size_t)b * (a.n_kv * kG) + head * kG) * a.max_segs * kRecord;
        const size_t head_step = (size_t)a.max_segs * kRecord;
        constexpr int kAhead = 4;
        for (int j0 = 0; j0 < cnt; j0 += kAhead) {
            float2 ml[kAhead][kG];
            float4 v[kAhead][kG];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
#pragma unroll
                for (int h = 0; h < kG; ++h) {
                    const float* r = base + h * head_step + (size_t)min(j0 + j, cnt - 1) * kRecord;
                    ml[j][h] = __ldcg(reinterpret_cast<const float2*>(r));
                    v[j][h] = __ldcg(reinterpret_cast<const float4*>(r + 4 + 4 * lane));
                }
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (j0 + j < cnt)
#pragma unroll
                    for (int h = 0; h < kG; ++h) join(x, h, ml[j][h].x, ml[j][h].y, v[j][h]);
        }
    };
    bool waited = !a.early;
    for (int i = 0; i < n;) {
        if (seg_start) {
            // this row's query as the B operand: column g holds term(g) of head hsel(g)
            pos = rows.len[cc.b] - 1;
            low = window_low(pos, a.window);
            span = span_row(cc.b);
            const size_t at = (size_t)rows.row[cc.b] * a.q_stride + (size_t)(cc.head * kG + hsel) * kD + 2 * t;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const size_t x = at + 16 * ks + 8 * hf;
                    if (a.bf16) {
                        qf[ks][hf] = term == 0 ? __ldcg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) + x)) : 0u;
                    } else {
                        const float2 q2 = __ldcg(reinterpret_cast<const float2*>(static_cast<const float*>(a.q) + x));
                        qf[ks][hf] = term < 3 ? term_of(q2.x, q2.y, term) : 0u;
                    }
                }
#pragma unroll
            for (int nt = 0; nt < 16; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
            m_run = -INFINITY;
            l_run = 0.0f;
            seg_start = false;
        }
        const int nb = (i + 1 < n && cc.blk + 1 < cc.nblk) ? 2 : 1;
        const bool ok = nb == 2 ? run_blocks(i, std::integral_constant<int, 2>{}) : run_blocks(i, std::integral_constant<int, 1>{});
        if (!ok) {
            // the copies in flight land before the warp stops; the error word reports the launch
            if (lane == 0)
                for (int j = i; j < min(n, i + kRing); ++j)
                    mbar_wait_bounded(&full[j % kRing], (uint32_t)((j / kRing) & 1), nullptr);
            __syncwarp();
            break;
        }
        if (nb == 2) advance(cc);
        i += nb;
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
                    const float x = acc[nt][e];
                    const float lo_sum = __shfl_xor_sync(kAll, x, 16), mid = __shfl_xor_sync(kAll, x, 4);
                    acc[nt][e] = x + (mid + lo_sum);
                }
            const bool writer = (g & 5) == 0 && g < 4;
            const long long f0 = (long long)a.n_kv * pref[cc.b] + (long long)cc.head * cc.nblk;
            const bool whole = f0 >= lo && f0 + cc.nblk <= lo + n;
            const int nrec = rows.nrec[cc.b];
            if (whole && !waited) {
                pdl_wait();
                waited = true;
            }
            if (whole && nrec == 0) {
                if (writer) {
                    const size_t at = (size_t)rows.row[cc.b] * a.out_stride + (size_t)(cc.head * kG + hsel) * kD + 2 * t;
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
                const int k = f0 < lo ? 0 : 1;
                float* rec = sm.rec[k][warp] + hsel * kRecord;
                if (writer) {
                    if (t == 0) *reinterpret_cast<float2*>(rec) = make_float2(Mh, Lh);
#pragma unroll
                    for (int nt = 0; nt < 16; ++nt) *reinterpret_cast<float2*>(rec + 4 + 8 * nt + 2 * t) = make_float2(acc[nt][0], acc[nt][1]);
                }
                if (whole) {  // all of the row's own part: with its prompt's records at once
                    __syncwarp();
                    Piece x;
                    clear(x);
                    const float* r = sm.rec[1][warp];
#pragma unroll
                    for (int h = 0; h < kG; ++h)
                        join(x, h, r[h * kRecord], r[h * kRecord + 1], *reinterpret_cast<const float4*>(r + h * kRecord + 4 + 4 * lane));
                    join_global(x, cc.b, cc.head, nrec);
#pragma unroll
                    for (int h = 0; h < kG; ++h) store_out4(a, rows.row[cc.b], cc.head * kG + h, x.acc[h], x.l[h]);
                    __syncwarp();
                } else if (lane == 0) {
                    sm.rec_gid[k][warp] = cc.b * a.n_kv + cc.head;
                }
            }
            seg_start = true;
        }
        advance(cc);
    }
    if (!waited) pdl_wait();

    // ---- join the warps' records of each (row, kv head) of this CTA, in warp
    // order; a row that goes on in other CTAs, or has a common prompt, through
    // the global records
    __syncthreads();
    Cursor gc;
    locate(c_lo, gc);
    long long g0 = (long long)a.n_kv * pref[gc.b] + (long long)gc.head * gc.nblk;
    for (int gi = 0; g0 < c_hi; ++gi) {
        const long long g1 = g0 + gc.nblk;
        const int gb = gc.b, gh = gc.head, nrec = rows.nrec[gb];
        if (gi % kWarps == warp) {
            const int wa = (int)(max(0ll, g0 - c_lo) / per), wb = (int)min((long long)kWarps - 1, (g1 - 1 - c_lo) / per);
            const long long lo_a = c_lo + (long long)wa * per;
            if (!(wa == wb && g0 >= lo_a && g1 <= lo_a + per)) {  // else its warp stored it
                Piece x;
                clear(x);
                for (int w = wa; w <= wb; ++w) {
                    const int k = g0 >= c_lo + (long long)w * per ? 1 : 0;
                    if (sm.rec_gid[k][w] != gb * a.n_kv + gh) continue;  // a warp that stopped early
                    const float* r = sm.rec[k][w];
#pragma unroll
                    for (int h = 0; h < kG; ++h)
                        join(x, h, r[h * kRecord], r[h * kRecord + 1], *reinterpret_cast<const float4*>(r + h * kRecord + 4 + 4 * lane));
                }
                const long long reach = (long long)kWarps * per;
                const int first = (int)(g0 / reach), nown = (int)((g1 - 1) / reach) - first + 1, seg = (int)blockIdx.x - first;
                bool store = nown == 1 && nrec == 0;
                if (!store && nrec + nown <= a.max_segs) {
                    float* base = a.part + ((size_t)gb * (a.n_kv * kG) + gh * kG) * a.max_segs * kRecord;
                    const size_t head_step = (size_t)a.max_segs * kRecord;
                    bool last = true;
                    if (nown > 1) {
#pragma unroll
                        for (int h = 0; h < kG; ++h) {
                            float* r = base + h * head_step + (size_t)(nrec + seg) * kRecord;
                            if (lane == 0) *reinterpret_cast<float2*>(r) = make_float2(x.m[h], x.l[h]);
                            *reinterpret_cast<float4*>(r + 4 + 4 * lane) = make_float4(x.acc[h][0], x.acc[h][1], x.acc[h][2], x.acc[h][3]);
                        }
                        __threadfence();
                        __syncwarp();
                        unsigned prev = 0;
                        unsigned* counter = a.counters + (size_t)gb * a.n_kv + gh;
                        if (lane == 0) prev = atomicAdd(counter, 1u);
                        prev = __shfl_sync(kAll, prev, 0);
                        last = prev == (unsigned)(nown - 1);
                        if (last && lane == 0) *counter = 0u;
                        __threadfence();
                        if (last) clear(x);
                    }
                    if (last) {
                        // every record: the prompt's, then (if this row crosses CTAs) the CTAs' in order
                        join_global(x, gb, gh, nown > 1 ? nrec + nown : nrec);
                        store = true;
                    }
                } else if (!store && lane == 0 && a.err) {
                    atomicOr(a.err, kErrBadIndex);
                }
                if (store)
#pragma unroll
                    for (int h = 0; h < kG; ++h) store_out4(a, rows.row[gb], gh * kG + h, x.acc[h], x.l[h]);
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
        launch_pdl(attn_span_kernel<kServeSmallBatch>, ctas, kThreads, sizeof(Smem), st, small_rows(rows), a);
    else
        launch_pdl(attn_span_kernel<kServeMaxBatch>, ctas, kThreads, sizeof(Smem), st, rows, a);
}

void prepare_attn_span_kernels() {
    configure_kernel((const void*)attn_span_kernel<kServeSmallBatch>, sizeof(Smem));
    configure_kernel((const void*)attn_span_kernel<kServeMaxBatch>, sizeof(Smem));
}

}  // namespace zc
