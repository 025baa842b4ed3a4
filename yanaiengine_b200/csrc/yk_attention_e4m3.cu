// yk_attention_e4m3.cu -- causal attention of a ragged batch over an e4m3 paged
// KV cache (yk_attention_e4m3): the kernel for fp32 queries, and the host side.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "yk_attention_e4m3.cuh"

namespace yk {

// ---------------------------------------------------------------------------
// One launch; 2 CTAs of 4 warps per SM, all resident.  The work is the list of
// (sequence, query tile, KV head) spans, each a run of pages; laid end to end it
// is cut into equal ranges of pages, one per CTA, so that long and short
// sequences, one or many, load every SM alike.  Each CTA finds its range from
// the lengths on the device (a block-wide prefix sum over the sequences: no plan
// to keep, and a captured launch follows lengths that change).
//
// A tile's rows are the (token, query head) pairs of one GQA group: R = 8 * NT
// rows for one warp, or 16 * NT with the warps in two row groups.  The pages of
// the range go round robin to the warps (to the two pairs of warps), each with
// its own ring of pages filled by TMA: K and V of one (block, layer, head) come
// as one box of 32 rows.
//
// Per page, with m16n8k16 f16 products and fp32 sums:
//   S^T[16 keys x rows] = K Q^T, O^T[dims x rows] += V^T P^T.
// Queries and weights are two f16 terms each, 22 bits: no floating-point input of
// the matrix instructions has more than 11, and the e4m3 side is exact in f16.
// Keys and dims are the products' M side, so 8 rows cost one n-tile: decoding
// (4 or 8 rows) pays for 8, not 16 or 64.  e4m3 converts exactly to f16, and the
// fragments come straight from 16-byte shared-memory reads: a product does not
// care in which order its K dimension runs, nor its M dimension as long as the
// result is read back the same way, so each thread takes consecutive bytes of
// its rows and the orders are matched on the other operand (queries: in the
// order the K bytes dictate; weights: keys in the order sigma).
//
// The blocks' scales: K's multiplies the scores; V's joins the weights, p =
// 2^(x + e_V - m), so that O needs no correction, and the sum adds p * 2^-e_V.
// m follows the largest x + e_V of a row lazily: weights may exceed 1 by 2^8
// before O is rescaled (their f16 form is biased by 2^7, the rest is room).
// Measured: 9 sequences of 300-1900 keys, 5 tokens, 12 heads of 64, window 333: 11
// us, nearly all of it latency (launch, plan, first pages, join).
// Queries go to f16 terms after a shift of each row by a power of two that brings
// its largest value next to 2^15.
// ---------------------------------------------------------------------------
constexpr int A8_THREADS = 128, A8_CTAS = 2;  // per SM
constexpr int A8_COST = 8;                    // a span's own cost, in pages (11 sequences of 3 tokens: 23.9 -> 6.7 us, 16 of 500-2500 keys: 31.5 -> 28.6)

// n-tiles of a warp at most: the O^T accumulators take 4 * DH / 16 registers each.
template <int DH>
__host__ __device__ constexpr int a8_max_nt() {
    return DH == 256 ? 1 : 2;
}

template <int DH, int NT>
struct A8Cfg {
    static constexpr int TERMS = 2;  // of queries and weights
    static constexpr int KS = DH / 16, MT = DH / 16;  // k-steps of S^T, m-tiles of O^T
    static constexpr int ROWB = DH == 64 ? 64 : 128;  // bytes of a row in a TMA box
    static constexpr int BOX = 32 * ROWB;             // one box: 16 rows of K, 16 of V
    static constexpr int BOXES = DH / ROWB;
    static constexpr int PAGE = 32 * DH;
    static constexpr int DEPTH = DH == 64 ? 8 : DH == 128 ? 3 : 2;  // pages of a warp's share of the ring
    static constexpr int RING = 4 * DEPTH * PAGE;
    static constexpr bool QREG = TERMS * NT * KS * 2 <= 48;  // queries in registers through the page loop
    static constexpr int ROWS = 8 * NT;                      // of a warp
    static constexpr int QBYTES = 2 * TERMS * NT * KS * 256;  // fragments of two row groups
    static constexpr int LDO = (DH < 128 ? DH : 128) + 4;    // floats of an accumulator row in shared memory
    static constexpr int DUMP = 4 * ROWS * LDO * 4;          // the warps' accumulators (128 dims at a time)
    // queries and accumulators share their room only where both do not fit beside the ring
    static constexpr bool APART = A8_CTAS * (RING + QBYTES + DUMP + 6144) <= 227 * 1024;
    static constexpr int QOFF = APART ? DUMP : 0;
    static constexpr int SHARED = APART ? QBYTES + DUMP : QBYTES > DUMP ? QBYTES : DUMP;
    static constexpr int NANS = 2 * ROWS * (DH / 32) * 4;    // bit per (row, dim)
    static constexpr size_t SMEM = 1024 + RING + SHARED + NANS + 4 * ROWS * 8 + 2 * ROWS * 4 +
                                   2 * 4 * DEPTH * 8 + (A8_SEGS + 2) * sizeof(Seg) + 320;
};

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8x8 matrix of 16-bit values over the warp
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int x, int head, int layer, int blk,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(head * 16), "r"(0), "r"(layer), "r"(blk), "r"(bar)
        : "memory");
}

template <int DH, int NT>
__global__ void __launch_bounds__(A8_THREADS, A8_CTAS) attn8_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ Attn8Params p) {
    using C = A8Cfg<DH, NT>;
    constexpr int TERMS = C::TERMS, KS = C::KS, MT = C::MT, NH = DH / 64;
    constexpr float LOWEST = -3.402823466e38f, LARGEST = 3.402823466e38f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const shared = ring + C::RING;  // accumulators at a span's end, and its queries
    float* const s_o = reinterpret_cast<float*>(shared);                     // [4 warps][ROWS][LDO]
    uint32_t* const s_nan = reinterpret_cast<uint32_t*>(shared + C::SHARED);  // [2 * ROWS][DH / 32]
    float2* const s_ml = reinterpret_cast<float2*>(s_nan + C::NANS / 4);      // [4 warps][ROWS] (m, l)
    float* const s_rf = reinterpret_cast<float*>(s_ml + 4 * C::ROWS);         // [2 * ROWS] score factor
    uint64_t* const bars = reinterpret_cast<uint64_t*>(s_rf + 2 * C::ROWS);
    Seg* const segs = reinterpret_cast<Seg*>(bars + 2 * 4 * C::DEPTH);
    unsigned* const s_scan = reinterpret_cast<unsigned*>(segs + A8_SEGS);  // [A8_SCAN]
    int* const s_flag = reinterpret_cast<int*>(s_scan + A8_SCAN);           // NaN cells seen
    int* const s_last = s_flag + 2;   // [2] this CTA joins the parts of s_cut[i]
    Seg* const s_cut = reinterpret_cast<Seg*>(s_last + 2);  // [2]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = lane >> 2, c = lane & 3;
    const int RG = 1 << p.lg, nparts = 4 >> p.lg;
    const int part = warp >> p.lg, rg = warp & (RG - 1);
    const int depth = C::DEPTH << p.lg;
    const int R = C::ROWS * RG, rep = p.H / p.G;
    const int my0 = rg * C::ROWS;  // this warp's first row of a tile
    const uint32_t my_ring = smem_u32(ring) + (uint32_t)(part * depth * C::PAGE);
    const uint32_t full = smem_u32(bars + part * depth), empty = smem_u32(bars + 4 * C::DEPTH + part * depth);

    for (int i = threadIdx.x; i < 4 * C::DEPTH; i += A8_THREADS) {
        mbar_init(smem_u32(bars + i), 1);
        mbar_init(smem_u32(bars + 4 * C::DEPTH + i), (uint32_t)RG);
    }
    for (int i = threadIdx.x; i < C::NANS / 4; i += A8_THREADS) s_nan[i] = 0;
    if (threadIdx.x == 0) {
        mbar_fence_init();
        s_flag[0] = s_last[0] = s_last[1] = 0;
    }
    pdl_trigger();
    pdl_wait();

    A8Work work;
    if (!a8_plan<A8_THREADS, 1, A8_COST, 8>(p, R, rep, s_scan, work)) return;

    // per-thread places in a page: K rows sigma(r), sigma(r) + 8; V rows c, c + 4, c + 8, c + 12
    const int sigma = (r & 1) * 4 + (r >> 1);
    uint32_t k_off[2], v_off[2];  // (two 16-byte columns of K; V rows of even and odd index)
    int v_dim;                    // first of this thread's consecutive V dims
    if constexpr (DH == 64) {
        const int piece = (r & 1) | ((r & 2) << 1) | ((r & 4) >> 1);  // 8 bytes
        k_off[0] = k_off[1] = (uint32_t)(sigma * 64 + ((c ^ ((sigma >> 1) & 3)) << 4));
        v_dim = 8 * piece;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            v_off[j] = (uint32_t)(1024 + (c + 4 * j) * 64 + (((piece >> 1) ^ (((c + 4 * j) >> 1) & 3)) << 4) + (piece & 1) * 8);
    } else {
        const int chunk = ((r & 1) << 2) | (r >> 1);
        v_dim = 16 * chunk;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            k_off[j] = (uint32_t)(sigma * 128 + (((c + 4 * j) ^ (sigma & 7)) << 4));
            v_off[j] = (uint32_t)(2048 + (c + 4 * j) * 128 + ((chunk ^ ((c + 4 * j) & 7)) << 4));
        }
    }

    bool dead = false;  // a bounded wait ran out: nothing more is loaded or computed
    int in_slot = 0, in_phase = 1, out_slot = 0, out_phase = 0;  // of the ring: next to fill, next to read
    // the spans of this CTA's range, A8_SEGS of them at a time
    for (int seg0 = 0; seg0 < work.nspans; seg0 += A8_SEGS) {
        a8_list<1, A8_COST>(p, R, rep, work, seg0, segs);
        __syncthreads();
        const int nseg = min(A8_SEGS, work.nspans - seg0);
        if (threadIdx.x == 0)
            for (int i = 0, at = 0; i < nseg; ++i) {
                segs[i].v = at;
                at += segs[i].n;
            }
        __syncthreads();
        const int v0 = segs[0].v, v1 = segs[nseg - 1].v + segs[nseg - 1].n;
        const int nk = (v1 - v0 - part + nparts - 1) / nparts;  // pages of this part

        // lane i of a batch: block id (-1: nothing to read), head, scale bytes of page 32 * batch + i
        int bid = -1, bid2 = -1, gk = 0, gk2 = 0;
        uint32_t kb = 0, kb2 = 0, vb = 0, vb2 = 0;
        const auto fetch = [&](int batch, int& id, int& g, uint32_t& k_byte, uint32_t& v_byte) {
            const int k = batch * 32 + lane;
            id = -1;
            if (k >= nk) return;
            const int v = v0 + part + nparts * k;
            int a = 0, z = nseg - 1;  // the last span with segs[].v <= v
            while (a < z) {
                const int mid = (a + z + 1) >> 1;
                if (segs[mid].v <= v) a = mid; else z = mid - 1;
            }
            const int page = segs[a].page + (v - segs[a].v);
            if (page >= segs[a].pend) return;
            g = segs[a].g;
            id = p.tables[(size_t)segs[a].b * p.max_blocks + page];
            if (id < 0 || id >= p.num_blocks) {
                raise_err(p.err, YK_DEV_ERR_BOUNDS);
                id = -1;
                return;
            }
            const uint8_t* s = p.scales + (size_t)id * p.block_scales + p.layer_scale + g;
            k_byte = *s;
            v_byte = s[p.G];
        };
        // page k of this part into its ring slot, once every warp of the part is done with the slot
        // (the first time round the slot is free: the phase before a barrier's first counts as complete)
        int base = 0;  // first page of the batch in bid, ...; the next one is in bid2, ...
        const auto issue = [&](int k) {
            const int id = __shfl_sync(0xffffffffu, k - base < 32 ? bid : bid2, k & 31);
            const int g = __shfl_sync(0xffffffffu, k - base < 32 ? gk : gk2, k & 31);
            if (lane == 0 && !dead) {
                const uint32_t bar = full + in_slot * 8;
                if (!mbar_wait_bounded(empty + in_slot * 8, (uint32_t)in_phase)) {
                    raise_err(p.err, YK_DEV_ERR_TIMEOUT);
                    dead = true;
                } else if (id < 0) {
                    mbar_arrive(bar);
                } else {
                    mbar_arrive_expect_tx(bar, C::PAGE);
#pragma unroll
                    for (int x = 0; x < C::BOXES; ++x)
                        tma_load_page(my_ring + in_slot * C::PAGE + x * C::BOX, &map, x * 128, g, p.layer, id, bar);
                }
            }
            __syncwarp();
            if (++in_slot == depth) {
                in_slot = 0;
                in_phase ^= 1;
            }
        };
        fetch(0, bid, gk, kb, vb);
        if (rg == 0)
#pragma unroll 1
            for (int k = 0; k < min(depth, nk); ++k) issue(k);
        fetch(1, bid2, gk2, kb2, vb2);

        // rows 8 u .. 8 u + 7 of a span's tile: lane's dims 64 h + 16 c .. + 15 of row 8 u + r
        constexpr int QW = NH * 4;
        uint4 qw[QW];
        const auto load_q = [&](const Seg& sg, int u) {
            const int row = u * 8 + r, i = div_rep(p, sg.rem + row);
            const float* src = reinterpret_cast<const float*>(p.q) + (size_t)(sg.tok + i) * p.q_stride +
                            (size_t)(sg.g * rep + sg.rem + row - i * rep) * DH + 16 * c;
#pragma unroll
            for (int h = 0; h < QW; ++h) {
                qw[h] = make_uint4(0, 0, 0, 0);
                if (row < sg.rows)
                    qw[h] = __ldcg(reinterpret_cast<const uint4*>(src + 64 * (h / (QW / NH))) + h % (QW / NH));
            }
        };
        int k = 0, issued = min(depth, nk);
#pragma unroll 1
        for (int si = 0; si < nseg; ++si) {
            const Seg sg = segs[si];
            const int rows = sg.rows;
            const int pos_last = sg.pos + div_rep(p, sg.rem + rows - 1);
            const bool active = my0 < rows;
            // row i of the tile: token and query head of the group
            const auto row_token = [&](int i) { return div_rep(p, sg.rem + i); };

            // ---- queries to B fragments in shared memory, 8 rows at a time: column n = lane / 4,
            // dims 64 h + 16 c + 4 s + {0, 1 | 2, 3} of k-step 4 h + s
            // (rows that the span does not fill are zeros: what lay there before must not decide when a warp moves its
            // references, which shows in the last bit)
#pragma unroll 1
            for (int u = warp; u * 8 < R; u += 4) {
                const int row = u * 8 + r;
                load_q(sg, u);
                float amax = 0.f;
#pragma unroll
                for (int h = 0; h < QW; ++h)
                    amax = fmaxf(fmaxf(fmaxf(amax, fabsf(__uint_as_float(qw[h].x))), fabsf(__uint_as_float(qw[h].y))),
                                 fmaxf(fabsf(__uint_as_float(qw[h].z)), fabsf(__uint_as_float(qw[h].w))));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                // shift by 2^up: amax = m * 2^E, 1 <= m < 2, to m * 2^14 (an infinite element: its second term is NaN,
                // and so are the row's scores)
                const int up = amax == 0.f ? 0 : min(126, 14 + 127 - (int)(__float_as_uint(amax) >> 23));  // -114 at least
                const float f = exp2_int(up);
                if (c == 0) s_rf[row] = p.scale_log2 * exp2_int(-up);
                const uint32_t dst = smem_u32(shared + C::QOFF) + (uint32_t)(u * TERMS * KS * 256 + lane * 16);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    float x[4] = {__uint_as_float(qw[ks].x), __uint_as_float(qw[ks].y), __uint_as_float(qw[ks].z), __uint_as_float(qw[ks].w)};
#pragma unroll
                    for (int z = 0; z < 4; ++z) x[z] *= f;
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint32_t y0 = pack_f16(x[0], x[1]), y1 = pack_f16(x[2], x[3]);
                        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(
                                         dst + (uint32_t)(t * KS * 256 + (ks >> 1) * 512 + (ks & 1) * 8)),
                                     "r"(y0), "r"(y1)
                                     : "memory");
                        const float2 a = f32x2(y0), b = f32x2(y1);  // (what this term leaves)
                        x[0] -= a.x; x[1] -= a.y; x[2] -= b.x; x[3] -= b.y;
                    }
                }
            }
            __syncthreads();
            const uint32_t q_smem = smem_u32(shared + C::QOFF) + (uint32_t)(rg * NT * TERMS * KS * 256 + lane * 16);
            uint4 qf[C::QREG ? NT * TERMS * KS / 2 : 1];
            if constexpr (C::QREG) {
                if (active)
#pragma unroll
                    for (int i = 0; i < NT * TERMS * KS / 2; ++i) qf[i] = lds128(q_smem + i * 512);
            }
            float2 rf[NT];  // scores of rows 2c, 2c + 1 -> log2 domain

            float o[MT][NT][4];
            float m[NT][2], l[NT][2];  // m: the row's reference, less the bias of 7
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                rf[nt] = *reinterpret_cast<const float2*>(s_rf + my0 + nt * 8 + 2 * c);
                m[nt][0] = m[nt][1] = LOWEST;
                l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
                for (int t = 0; t < MT; ++t) o[t][nt][0] = o[t][nt][1] = o[t][nt][2] = o[t][nt][3] = 0.f;
            }

            // ---- this part's pages of the span.  The scores of the page after next come with the
            // product of weights and values of this one: two independent streams of instructions
            const int k_end = (sg.v + sg.n - v0 - part + nparts - 1) >> (2 - p.lg);
            int j0 = 0, ek = 0, ev = 0;
            uint32_t page = my_ring;
            // page i has arrived: its place, first key (-1: a page that is not there, no row sees its cells,
            // whatever its slot holds) and exponents
            const auto take = [&](int i) {
                if (i >= base + 32) {
                    base += 32;
                    bid = bid2;
                    gk = gk2;
                    kb = kb2;
                    vb = vb2;
                    fetch(base / 32 + 1, bid2, gk2, kb2, vb2);
                }
                const int id = __shfl_sync(0xffffffffu, bid, i & 31);
                ek = kv8_exponent(__shfl_sync(0xffffffffu, kb, i & 31));
                ev = kv8_exponent(__shfl_sync(0xffffffffu, vb, i & 31));
                page = my_ring + (uint32_t)(out_slot * C::PAGE);
                j0 = id >= 0 ? (sg.page + (v0 + part + nparts * i - sg.v)) * 16 : -1;
                if (!dead && !mbar_wait_bounded(full + out_slot * 8, (uint32_t)out_phase)) {
                    if (lane == 0) raise_err(p.err, YK_DEV_ERR_TIMEOUT);
                    dead = true;
                }
                dead = __any_sync(0xffffffffu, dead);
                if (++out_slot == depth) {
                    out_slot = 0;
                    out_phase ^= 1;
                }
            };
            float s[NT][4];
            const auto scores = [&]() {  // s = K Q^T of the page taken last
                float s2[2][NT][4];
#pragma unroll
                for (int ch = 0; ch < 2; ++ch)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s2[ch][nt][0] = s2[ch][nt][1] = s2[ch][nt][2] = s2[ch][nt][3] = 0.f;
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    const uint32_t ka = page + (uint32_t)((h >> 1) * C::BOX) + k_off[h & 1];
                    const uint4 x4 = lds128(ka), y4 = lds128(ka + 8 * C::ROWB);
                    const uint32_t x[4] = {x4.x, x4.y, x4.z, x4.w}, y[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const uint32_t a0[4] = {f16x2_lo(x[i]), f16x2_lo(y[i]), f16x2_hi(x[i]), f16x2_hi(y[i])};
                        const uint32_t a1[4] = {f16x2_lo(x[i + 1]), f16x2_lo(y[i + 1]), f16x2_hi(x[i + 1]), f16x2_hi(y[i + 1])};
#pragma unroll
                        for (int t = 0; t < TERMS; ++t)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const int at = ((nt * TERMS + t) * KS + h * 4 + i) / 2;
                                const uint4 b = C::QREG ? qf[C::QREG ? at : 0] : lds128(q_smem + at * 512);
                                mma_f16(s2[0][nt], a0, b.x, b.y);
                                mma_f16(s2[1][nt], a1, b.z, b.w);
                            }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[nt][i] = s2[0][nt][i] + s2[1][nt][i];
            };
            if (k < k_end) {
                take(k);
                if (active) scores();
            }
#pragma unroll 1
            while (k < k_end) {
                const uint32_t held = page;
                const int held_j0 = j0, slot = (out_slot == 0 ? depth : out_slot) - 1;
                const bool plain = p.cap <= 0.f && j0 >= 0 && j0 + 15 <= sg.pos && (p.window <= 0 || pos_last - j0 < p.window);
                uint32_t pb[TERMS][NT][2];
                if (active) {
                    // scores -> x + e_V in the log2 domain; row 2c: s[0], s[2], row 2c + 1: s[1], s[3]
                    const float fk = exp2_int(ek), shift = (float)ev, inv = exp2_int(-ev);
                    if (plain) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float f0 = fminf(rf[nt].x * fk, LARGEST), f1 = fminf(rf[nt].y * fk, LARGEST);
                            s[nt][0] = fmaf(s[nt][0], f0, shift);
                            s[nt][1] = fmaf(s[nt][1], f1, shift);
                            s[nt][2] = fmaf(s[nt][2], f0, shift);
                            s[nt][3] = fmaf(s[nt][3], f1, shift);
                        }
                    } else {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[nt][i] *= fminf((i & 1 ? rf[nt].y : rf[nt].x) * fk, LARGEST);
                        if (p.cap > 0.f)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int i = 0; i < 4; ++i) s[nt][i] = p.cap_log2 * tanh_cap(s[nt][i] * p.inv_cap_log2);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const int row = my0 + nt * 8 + 2 * c + j;
                                const unsigned back = (unsigned)(sg.pos + row_token(row) - sigma - j0);  // query minus key
                                const unsigned w = row < rows && j0 >= 0 ? (p.window > 0 ? (unsigned)p.window : 0x80000000u) : 0u;
                                s[nt][j] = back < w ? s[nt][j] + shift : -INFINITY;
                                s[nt][j + 2] = back - 8 < w ? s[nt][j + 2] + shift : -INFINITY;
                            }
                    }
                    // raise a row's reference once a weight would pass 2^15
                    bool over = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        over |= fmaxf(s[nt][0], s[nt][2]) - m[nt][0] > 15.f || fmaxf(s[nt][1], s[nt][3]) - m[nt][1] > 15.f;
                    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                float x = fmaxf(s[nt][j], s[nt][j + 2]);
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                                const float mn = fmaxf(m[nt][j], x - 7.f), f = ex2(m[nt][j] - mn);
                                m[nt][j] = mn;
                                l[nt][j] *= f;
#pragma unroll
                                for (int t = 0; t < MT; ++t) {
                                    o[t][nt][j] *= f;
                                    o[t][nt][j + 2] *= f;
                                }
                            }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][i] = ex2(s[nt][i] - m[nt][i & 1]);
                        l[nt][0] = fmaf(s[nt][0] + s[nt][2], inv, l[nt][0]);
                        l[nt][1] = fmaf(s[nt][1] + s[nt][3], inv, l[nt][1]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t x = pack_f16(s[nt][2 * j], s[nt][2 * j + 1]);
                            pb[0][nt][j] = transpose8(x);
                            const float2 a = f32x2(x);
                            pb[1][nt][j] = transpose8(pack_f16(s[nt][2 * j] - a.x, s[nt][2 * j + 1] - a.y));
                        }
                    }
                }
                if (k + 1 < k_end) take(k + 1);
                if (active) {
                    scores();  // (after the last page: of that one again, not used)
                    // O^T += V^T P^T
#pragma unroll
                    for (int bx = 0; bx < C::BOXES; ++bx) {
                        constexpr int W = DH == 64 ? 2 : 4;  // words of a thread's V bytes per key
                        uint32_t v[4][W];
                        const uint32_t va = held + (uint32_t)(bx * C::BOX);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t a = va + (uint32_t)((j >> 1) * 8 * C::ROWB) + v_off[j & 1];
                            if constexpr (DH == 64) {
                                const uint2 t = lds64(a);
                                v[j][0] = t.x; v[j][1] = t.y;
                            } else {
                                const uint4 t = lds128(a);
                                v[j][0] = t.x; v[j][1] = t.y; v[j][2] = t.z; v[j][3] = t.w;
                            }
                        }
                        if (!plain) {
                            // a NaN cell must reach the rows that see its key and no others: it is taken
                            // out of the product, and noted for the rows it belongs to
                            uint32_t any = 0;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
#pragma unroll
                                for (int i = 0; i < W; ++i) any |= (v[j][i] & 0x7f7f7f7fu) + 0x01010101u;
                            if (any & 0x80808080u) {
#pragma unroll
                                for (int j = 0; j < 4; ++j)
#pragma unroll
                                    for (int i = 0; i < W; ++i) {
                                        const uint32_t bad = ((v[j][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                                        v[j][i] &= ~(bad | (bad - (bad >> 7)));
                                    }
#pragma unroll 1
                                for (int z = 0; z < 16 * W; ++z) {
                                    const int key = c + 4 * (z / (4 * W)), byte = z % (4 * W);
                                    uint32_t x;
                                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(x) : "r"(
                                        va + (uint32_t)((key >> 3) * 8 * C::ROWB) + v_off[key >> 2 & 1] + (uint32_t)byte));
                                    if ((x & 0x7f) != 0x7f) continue;
                                    const int dim = bx * 128 + v_dim + byte;
                                    for (int row = my0; row < min(rows, my0 + C::ROWS); ++row) {
                                        const int back = sg.pos + row_token(row) - held_j0 - key;
                                        if (held_j0 >= 0 && back >= 0 && (p.window <= 0 || back < p.window)) {
                                            atomicOr(&s_nan[row * (DH / 32) + (dim >> 5)], 1u << (dim & 31));
                                            s_flag[0] = 1;
                                        }
                                    }
                                }
                            }
                            __syncwarp();
                        }
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            const uint32_t lo01 = __byte_perm(v[0][i], v[1][i], 0x5140), hi01 = __byte_perm(v[0][i], v[1][i], 0x7362);
                            const uint32_t lo23 = __byte_perm(v[2][i], v[3][i], 0x5140), hi23 = __byte_perm(v[2][i], v[3][i], 0x7362);
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const uint32_t w0 = half ? hi01 : lo01, w1 = half ? hi23 : lo23;
                                const uint32_t a[4] = {f16x2_lo(w0), f16x2_hi(w0), f16x2_lo(w1), f16x2_hi(w1)};
                                const int t = bx * 8 + 2 * i + half;
#pragma unroll
                                for (int tm = 0; tm < TERMS; ++tm)
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) mma_f16(o[t][nt], a, pb[tm][nt][0], pb[tm][nt][1]);
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + slot * 8);
                ++k;
                // the slot just freed takes the next page (of two row groups the first stays a page behind,
                // so that it does not wait for the other)
                if (rg == 0 && issued < min(nk, k - p.lg + depth)) issue(issued++);
            }

            // ---- end of the span: the parts of a row group are joined in shared memory
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
                    l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
                    l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
                    if (r == 0) s_ml[warp * C::ROWS + nt * 8 + 2 * c + j] = make_float2(m[nt][j], l[nt][j]);
                }
            if (!C::APART) __syncthreads();  // (every warp is done with the queries in `shared`)
            const bool whole = sg.c0 == sg.c1;
            const size_t part_row = (size_t)(2 * blockIdx.x + ((int)blockIdx.x == sg.c0 ? 1 : 0)) * R;
            bool nans = false;
#pragma unroll
            for (int bx = 0; bx < C::BOXES; ++bx) {
                if (bx) __syncthreads();
                if (active) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float* const dst = s_o + (warp * C::ROWS + nt * 8 + 2 * c + j) * C::LDO + v_dim;
#pragma unroll
                            for (int t = 0; t < MT / C::BOXES; t += 2)  // 4 consecutive dims
                                *reinterpret_cast<float4*>(dst + 2 * t) =
                                    make_float4(o[bx * 8 + t][nt][j], o[bx * 8 + t][nt][j + 2], o[bx * 8 + t + 1][nt][j],
                                                o[bx * 8 + t + 1][nt][j + 2]);
                        }
                }
                __syncthreads();
                nans = s_flag[0] != 0;
                constexpr int W4 = (DH < 128 ? DH : 128) / 4;
#pragma unroll 1
                for (int i = threadIdx.x; i < rows * W4; i += A8_THREADS) {
                    const int row = i / W4, d = bx * 128 + i % W4 * 4;
                    // the parts that hold the row: warps w0, w0 + RG, ...
                    const int w0 = row >= C::ROWS ? 1 : 0, at = row - w0 * C::ROWS;
                    float2 t[4];
                    float4 x[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int w = min((q << p.lg) + w0, 3);
                        t[q] = s_ml[w * C::ROWS + at];
                        x[q] = *reinterpret_cast<const float4*>(s_o + (w * C::ROWS + at) * C::LDO + i % W4 * 4);
                    }
                    float M = fmaxf(t[0].x, t[1].x), L = 0.f;
                    if (nparts == 4) M = fmaxf(M, fmaxf(t[2].x, t[3].x));
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (q < nparts) {
                            const float f = ex2(t[q].x - M);
                            L = fmaf(t[q].y, f, L);
                            a.x = fmaf(x[q].x, f, a.x); a.y = fmaf(x[q].y, f, a.y);
                            a.z = fmaf(x[q].z, f, a.z); a.w = fmaf(x[q].w, f, a.w);
                        }
                    }
                    if (nans) {
                        const uint32_t bad = s_nan[row * (DH / 32) + (d >> 5)] >> (d & 31);
                        const float nan = __int_as_float(0x7fffffff);
                        if (bad & 1) a.x = nan;
                        if (bad & 2) a.y = nan;
                        if (bad & 4) a.z = nan;
                        if (bad & 8) a.w = nan;
                    }
                    if (whole) {
                        const float z = L == 0.f ? 0.f : 1.0f / L;
                        const int tok = row_token(row);
                        store4(reinterpret_cast<float*>(p.out) + (size_t)(sg.tok + tok) * p.out_stride +
                                   (size_t)(sg.g * rep + sg.rem + row - tok * rep) * DH + d, a.x * z, a.y * z, a.z * z, a.w * z);
                    } else {
                        __stcg(reinterpret_cast<float4*>(p.ws_o + (part_row + row) * DH + d), a);
                        if (d == 0) __stcg(p.ws_ml + part_row + row, make_float2(M, L));
                    }
                }
            }
            if (nans) {
                __syncthreads();
                for (int i = threadIdx.x; i < C::NANS / 4; i += A8_THREADS) s_nan[i] = 0;
                if (threadIdx.x == 0) s_flag[0] = 0;
            }
            if (!C::APART || !whole || si + 1 == nseg) __syncthreads();  // (else the next span's first barrier serves)
            if (!whole && threadIdx.x == 0) {
                a8_arrive(p, sg, s_last, s_cut);
            }
        }
        __syncthreads();  // (the span list too)
    }
    a8_join<float, DH, A8_THREADS>(p, R, rep, s_last, s_cut);
    // every copy asked for has landed: the loop above waited for each, unless it gave up
    if (dead && rg == 0 && lane == 0)
        for (int i = 0; i < depth; ++i)
            for (int ph = 0; ph < 2; ++ph) (void)mbar_wait_bounded_ns(full + i * 8, (uint32_t)ph, 100000000ull);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// The workspace holds the rows of two cut spans per CTA (its first, begun
// elsewhere, and its last, ended elsewhere): CTAs per SM * tile rows at most
// A8_WS / head_dim, for every shape.
static size_t ws_rows(int num_sms, int head_dim) { return (size_t)2 * num_sms * (A8_WS / head_dim); }
size_t attention_e4m3_ws_bytes(int num_sms, int head_dim) {
    return A8_COUNTERS + ws_rows(num_sms, head_dim) * (8 + 4 * (size_t)head_dim);
}

static PFN_tmapEncodeTiled tensor_map_encoder() {
    static const PFN_tmapEncodeTiled fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            f = nullptr;
        }
        return (PFN_tmapEncodeTiled)f;
    }();
    return fn;
}

// (head dim, row of a head group, K|V, layer, block); one box: a head's 16 K rows, and its 16 V rows with both.
static yk_status page_map(const yk_kv_pages& g, bool both, CUtensorMap* map) {
    const PFN_tmapEncodeTiled encode = tensor_map_encoder();
    if (!encode) {
        yk_set_error("cuTensorMapEncodeTiled not available from the driver");
        return YK_ERR_CUDA;
    }
    const cuuint64_t dh = g.head_dim, rows = (cuuint64_t)16 * g.n_kv_heads;
    const cuuint64_t dims[5] = {dh, rows, 2, (cuuint64_t)g.n_layers, (cuuint64_t)g.num_blocks};
    const cuuint64_t strides[4] = {dh, dh * rows, 2 * dh * rows, 2 * dh * rows * g.n_layers};
    const cuuint32_t box[5] = {(cuuint32_t)std::min<cuuint64_t>(dh, 128), 16, both ? 2u : 1u, 1, 1};
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, g.data, dims, strides, box, one,
                              CU_TENSOR_MAP_INTERLEAVE_NONE,
                              g.head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        yk_set_error("cuTensorMapEncodeTiled(e4m3 pages) failed: " + std::to_string((int)r));
        return YK_ERR_CUDA;
    }
    return YK_OK;
}

yk_status attention_e4m3_check(const yk_attention_e4m3_args& a) {
    YK_TRY(kv_pages_check(a.pages, a.layer));
    YK_ARG(a.pages.kind == YK_KV_E4M3, "pages.kind must be YK_KV_E4M3");
    YK_ARG(a.dtype == YK_DTYPE_F32 || a.dtype == YK_DTYPE_BF16, "dtype");
    YK_ARG(a.T >= 0 && a.B >= (a.T > 0 ? 1 : 0) && a.B <= (1 << 20), "T must not be negative, B in 1..2^20 (0 where T is)");
    YK_ARG(a.n_heads > 0 && a.n_heads <= 65536 && a.n_heads % a.pages.n_kv_heads == 0,
           "n_heads must be a positive multiple of n_kv_heads");
    YK_ARG(a.n_heads / a.pages.n_kv_heads <= 1024, "at most 1024 query heads share a KV head");
    YK_ARG(a.max_blocks > 0 && a.max_blocks <= (1 << 25), "max_blocks must be in 1..2^25");
    YK_ARG(a.max_new >= 0 && a.window >= 0, "max_new / window must not be negative");
    YK_ARG(std::isfinite(a.scale) && a.scale >= 0.f && std::isfinite(a.cap) && a.cap >= 0.f,
           "scale and cap must be finite and not negative");
    if (a.T == 0) return YK_OK;
    YK_ARG(a.q && a.out && a.q_starts && a.context_lens && a.block_tables, "null q / out / q_starts / context_lens / block_tables");
    YK_ARG(a.workspace && ((uintptr_t)a.workspace & 15u) == 0, "workspace must be a 16-byte aligned device pointer");
    YK_ARG(((uintptr_t)a.q & 15u) == 0 && ((uintptr_t)a.out & 15u) == 0, "q and out must be 16-byte aligned");
    const int64_t es = a.dtype == YK_DTYPE_F32 ? 4 : 2, row = (int64_t)a.n_heads * a.pages.head_dim;
    YK_ARG(a.q_stride >= row && a.q_stride * es % 16 == 0 && a.out_stride >= row && a.out_stride * es % 16 == 0,
           "q_stride / out_stride must cover a row and be multiples of 16 bytes");
    // (tiles have 8 rows at least, and their pages and costs are counted in 32 bits)
    const int64_t tiles = (int64_t)a.T * (a.n_heads / a.pages.n_kv_heads) / 8 + a.B, heads = a.pages.n_kv_heads;
    if ((int64_t)a.T * a.n_heads >= (int64_t)1 << 31 || (double)tiles * (double)heads * (a.max_blocks + (double)A8_COST) >= 2147483648.0) {
        yk_set_error("unsupported: T * n_heads or (T * n_heads / 8 + B * n_kv_heads) * (max_blocks + 8) is 2^31 or more; "
                     "split the batch");
        return YK_ERR_UNSUPPORTED;
    }
    return YK_OK;
}

template <int DH, int NT>
static yk_status launch_a8(cudaStream_t st, bool pdl, int num_sms, const CUtensorMap& map, const Attn8Params& p) {
    using C = A8Cfg<DH, NT>;
    static_assert(A8_CTAS * C::ROWS * (2 * NT > a8_max_nt<DH>() ? 2 : 1) <= A8_WS / DH,
                  "cut spans' rows in the workspace");
    int dev = 0;
    YK_CHECK_CUDA(cudaGetDevice(&dev));
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {
        YK_CHECK_CUDA(cudaFuncSetAttribute(attn8_kernel<DH, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
        ready.fetch_or(bit, std::memory_order_release);
    }
    YK_CHECK_CUDA(launch_on(st, pdl, attn8_kernel<DH, NT>, num_sms * A8_CTAS, A8_THREADS, C::SMEM, map, p));
    return YK_OK;
}

// The tile: as few n-tiles as hold the rows of a sequence's new tokens; beyond a
// warp's most, two row groups share the pages.
template <int DH>
static yk_status launch_a8_rows(cudaStream_t st, bool pdl, int num_sms, const CUtensorMap& map, Attn8Params& p,
                                long long rows) {
    constexpr int MOST = a8_max_nt<DH>();
    p.lg = rows > 8 * MOST ? 1 : 0;
    const int nt = (int)std::min<long long>(MOST, (rows + (8 << p.lg) - 1) / (8 << p.lg));
    if constexpr (MOST >= 2) {
        if (nt == 2) return launch_a8<DH, 2>(st, pdl, num_sms, map, p);
    }
    return launch_a8<DH, 1>(st, pdl, num_sms, map, p);
}

yk_status attention_e4m3_launch(cudaStream_t st, bool pdl, int num_sms, const yk_attention_e4m3_args& a) {
    if (a.T == 0) return YK_OK;
    YK_ARG(num_sms * A8_CTAS * 4 <= A8_COUNTERS, "device has more SMs than the workspace's counters");
    CUtensorMap map;
    YK_TRY(page_map(a.pages, a.dtype == YK_DTYPE_F32, &map));
    Attn8Params p;
    p.q = a.q;
    p.out = a.out;
    p.pool = reinterpret_cast<const uint8_t*>(a.pages.data);
    p.scales = a.pages.scales;
    p.q_starts = a.q_starts;
    p.ctx = a.context_lens;
    p.tables = a.block_tables;
    p.err = a.err;
    p.q_stride = a.q_stride;
    p.out_stride = a.out_stride;
    p.layer_scale = 2LL * a.pages.n_kv_heads * a.layer;
    p.block_scales = 2LL * a.pages.n_kv_heads * a.pages.n_layers;
    p.block_cells = p.block_scales * YK_BLOCK_SIZE * a.pages.head_dim;
    p.layer_off = p.layer_scale * YK_BLOCK_SIZE * a.pages.head_dim;
    p.T = a.T;
    p.B = a.B;
    p.H = a.n_heads;
    p.G = a.pages.n_kv_heads;
    p.layer = a.layer;
    p.max_blocks = a.max_blocks;
    p.num_blocks = a.pages.num_blocks;
    p.window = a.window;
    const float scale = a.scale > 0.f ? a.scale : 1.0f / std::sqrt((float)a.pages.head_dim), log2e = 1.4426950408889634f;
    p.scale_log2 = scale * log2e;
    // (a cap of 2^125 changes no score that fp32 holds apart, one of 2^-125 makes all weights equal: beyond them
    // cap * log2(e) or its inverse has no place in fp32)
    p.cap = a.cap > 0.f ? std::min(std::max(a.cap, 0x1p-125f), 0x1p125f) : 0.f;
    p.cap_log2 = p.cap * log2e;
    p.inv_cap_log2 = p.cap > 0.f ? 1.0f / p.cap_log2 : 0.f;
    uint8_t* const ws = reinterpret_cast<uint8_t*>(a.workspace);
    const unsigned rep = (unsigned)(a.n_heads / a.pages.n_kv_heads);
    p.rep_magic = rep == 1 ? 0u : (unsigned)((0x100000000ull + rep - 1) / rep);
    const int dh = a.pages.head_dim;
    p.counters = reinterpret_cast<int32_t*>(ws);
    p.ws_ml = reinterpret_cast<float2*>(ws + A8_COUNTERS);
    p.ws_o = reinterpret_cast<float*>(ws + A8_COUNTERS + ws_rows(num_sms, dh) * 8);
    // rows of the longest sequence's new tokens, as far as the caller says
    const long long most = a.max_new > 0 ? std::min(a.max_new, a.T) : (a.T + a.B - 1) / a.B;
    const long long rows = most * (a.n_heads / a.pages.n_kv_heads);
    if (a.dtype == YK_DTYPE_BF16) return attention_e4m3_launch_bf16(st, pdl, num_sms, dh, map, p, rows);
    switch (dh) {
        case 64: return launch_a8_rows<64>(st, pdl, num_sms, map, p, rows);
        case 128: return launch_a8_rows<128>(st, pdl, num_sms, map, p, rows);
        default: return launch_a8_rows<256>(st, pdl, num_sms, map, p, rows);
    }
}

}  // namespace yk
