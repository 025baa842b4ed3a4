// yk_attention_e4m3.cu -- causal attention of a ragged batch over an e4m3 paged
// KV cache (yk_attention_e4m3).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "yk_epilogue.cuh"
#include "yk_kvcache.cuh"

namespace yk {

struct Attn8Params {
    const void* q;
    void* out;
    const uint8_t* scales;
    const int32_t *q_starts, *ctx, *tables;
    uint32_t* err;
    int32_t* counters;  // workspace: arrivals at a cut span, by its first CTA (zero between calls)
    float2* ws_ml;      // workspace: (m, l) and O of the parts of cut spans, [2 per CTA][R]
    float* ws_o;
    long long q_stride, out_stride;
    long long block_scales, layer_scale;
    int T, B, H, G, layer, max_blocks, num_blocks;
    int lg;             // log2 of the row groups
    uint32_t rep_magic;  // ceil(2^32 / (H / G)), 0 where that is 1
    unsigned long long grid_magic;  // the same for the grid size and 64-bit x
    int window;
    float scale_log2, cap, cap_log2, inv_cap_log2;  // _log2: times log2(e)
};

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
// Queries go to f16 (fp32 queries and weights: to two f16 terms) after a shift of
// each row by a power of two that brings its largest value next to 2^15.
// ---------------------------------------------------------------------------
constexpr int A8_THREADS = 128, A8_CTAS_PER_SM = 2, A8_RING = 65536;
constexpr int A8_SEGS = 32;      // spans a CTA lists at a time
constexpr int A8_COUNTERS = 4096;  // bytes of arrival counters, one per CTA
constexpr int A8_MIN_UNITS = 4;  // pages of a CTA's range, at least

// n-tiles of a warp at most: the O^T accumulators take 4 * DH / 16 registers each.
template <typename AT, int DH>
__host__ __device__ constexpr int a8_max_nt() {
    return DH == 256 ? (sizeof(AT) == 4 ? 1 : 2) : (sizeof(AT) == 4 ? 2 : 4);
}

struct Seg {
    int b, g;
    int tok, rem;    // first row of the tile: token tok of the batch, query head rem of the group
    int rows;
    int pos;         // position of that token
    int page, pend;  // first page of this CTA's part; pages of the span's keys end here
    int v, n;        // its place and length (pages) in the CTA's range
    int c0, c1;      // first and last CTA of the span
};

template <typename AT, int DH, int NT>
struct A8Cfg {
    static constexpr int TERMS = sizeof(AT) == 4 ? 2 : 1;
    static constexpr int KS = DH / 16, MT = DH / 16;  // k-steps of S^T, m-tiles of O^T
    static constexpr int ROWB = DH == 64 ? 64 : 128;  // bytes of a row in a TMA box
    static constexpr int BOX = 32 * ROWB;             // one box: 16 rows of K, 16 of V
    static constexpr int BOXES = DH / ROWB;
    static constexpr int PAGE = 32 * DH;
    static constexpr int DEPTH = A8_RING / 4 / PAGE;  // pages of a warp's share of the ring
    static constexpr bool QREG = TERMS * NT * KS * 2 <= 48;  // queries in registers through the page loop
    static constexpr int ROWS = 8 * NT;                      // of a warp
    static constexpr int QBYTES = 2 * TERMS * NT * KS * 256;  // fragments of two row groups
    static constexpr int LDO = DH + 4;                       // floats of an accumulator row
    static constexpr int DUMP = 2 * ROWS * LDO * 4;          // accumulators of two warps
    static constexpr int SHARED = QBYTES > DUMP ? QBYTES : DUMP;  // used in turn
    static constexpr int NANS = 2 * ROWS * (DH / 32) * 4;    // bit per (row, dim)
    static constexpr size_t SMEM = 1024 + A8_RING + SHARED + NANS + 4 * ROWS * 8 + 2 * ROWS * 8 + 2 * ROWS * 4 +
                                   2 * 4 * DEPTH * 8 + A8_SEGS * sizeof(Seg) + 128;
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
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int x, int head, int layer, int blk,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(head * 16), "r"(0), "r"(layer), "r"(blk), "r"(bar)
        : "memory");
}

// tanh to a few 2^-24 of its value: 1 - 2 / (1 + e^2z) away from 0, the odd
// series z - z^3/3 + 2z^5/15 - 17z^7/315 near it.
__device__ __forceinline__ float tanh_cap(float z) {
    const float e = 1.f - __fdividef(2.f, 1.f + ex2(fminf(z * 2.8853900817779268f, 126.f)));
    const float q = z * z, t = fmaf(fmaf(fmaf(-17.f / 315.f, q, 2.f / 15.f), q, -1.f / 3.f), q, 1.f) * z;
    return fabsf(z) < 0.25f ? t : e;
}

// x / (H / G), x below 64 + H / G (exact: x * (H / G) < 2^32).
__device__ __forceinline__ int div_rep(const Attn8Params& p, int x) {
    return p.rep_magic ? (int)__umulhi((unsigned)x, p.rep_magic) : x;
}

// A span's pages: [page, pend), at least one (page == pend: a tile without keys).
struct Span {
    int rows, page, pend, tok, rem;  // tok: of the sequence
    __device__ __forceinline__ int units() const { return max(1, pend - page); }
};
__device__ __forceinline__ Span span_of(const Attn8Params& p, int n, int ctx, int qt, int R, int rep) {
    const long long lo = (long long)qt * R;
    Span s;
    s.rows = (int)min((long long)n * rep - lo, (long long)R);
    s.tok = (int)((unsigned)lo / (unsigned)rep);
    s.rem = (int)lo - s.tok * rep;
    const int first = ctx - n + s.tok;
    const int last = first + div_rep(p, s.rem + s.rows - 1);
    s.pend = (int)((min(max((long long)last + 1, 0LL), (long long)p.max_blocks * 16) + 15) >> 4);
    s.page = p.window > 0 ? min(max(0, first - p.window + 1) >> 4, s.pend) : 0;
    return s;
}

// New tokens of sequence b; 0 where q_starts does not fit.
__device__ __forceinline__ int new_tokens(const Attn8Params& p, int b, int& start) {
    start = p.q_starts[b];
    const int end = p.q_starts[b + 1];
    return start >= 0 && end >= start && end <= p.T && (b > 0 || start == 0) ? end - start : -1;
}

template <typename AT, int DH, int NT>
__global__ void __launch_bounds__(A8_THREADS, A8_CTAS_PER_SM)
    attn8_kernel(const __grid_constant__ CUtensorMap map, Attn8Params p) {
    using C = A8Cfg<AT, DH, NT>;
    constexpr int TERMS = C::TERMS, KS = C::KS, MT = C::MT, NH = DH / 64, D4 = DH / 4;
    constexpr float LOWEST = -3.402823466e38f, LARGEST = 3.402823466e38f;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const shared = ring + A8_RING;  // queries at the start of a span, accumulators at its end
    float* const s_o = reinterpret_cast<float*>(shared);                     // [2][ROWS][LDO]
    uint32_t* const s_nan = reinterpret_cast<uint32_t*>(shared + C::SHARED);  // [2 * ROWS][DH / 32]
    float2* const s_ml = reinterpret_cast<float2*>(s_nan + C::NANS / 4);      // [4 warps][ROWS] (m, l)
    float2* const s_row = s_ml + 4 * C::ROWS;                                 // [2 * ROWS] joined (m, l)
    float* const s_rf = reinterpret_cast<float*>(s_row + 2 * C::ROWS);        // [2 * ROWS] score factor
    uint64_t* const bars = reinterpret_cast<uint64_t*>(s_rf + 2 * C::ROWS);
    Seg* const segs = reinterpret_cast<Seg*>(bars + 2 * 4 * C::DEPTH);
    long long* const s_units = reinterpret_cast<long long*>(segs + A8_SEGS);  // [4]
    int* const s_spans = reinterpret_cast<int*>(s_units + 4);                 // [4]
    int* const s_flag = s_spans + 4;  // [0] first span, [1] last span, [2] last arriver, [3] NaN cells seen

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
        s_flag[3] = 0;
    }
    pdl_trigger();
    pdl_wait();

    // ---- this CTA's range of pages: [lo, hi) of the spans laid end to end
    const int per_thread = (p.B + A8_THREADS - 1) / A8_THREADS;
    const int b_lo = min(p.B, (int)threadIdx.x * per_thread), b_hi = min(p.B, b_lo + per_thread);
    long long units = 0;
    int spans = 0;
    for (int b = b_lo; b < b_hi; ++b) {
        int start;
        const int n = new_tokens(p, b, start), ctx = p.ctx[b];
        if (n < 0 || (n > 0 && ctx > p.max_blocks * 16LL)) raise_err(p.err, YK_DEV_ERR_BOUNDS);
        for (int qt = 0; (long long)qt * R < (long long)n * rep; ++qt) {
            units += (long long)span_of(p, n, ctx, qt, R, rep).units() * p.G;
            spans += p.G;
        }
    }
    long long at0 = units;  // exclusive prefixes over the threads
    int ord0 = spans;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, at0, o);
        const int y = __shfl_up_sync(0xffffffffu, ord0, o);
        if (lane >= o) {
            at0 += x;
            ord0 += y;
        }
    }
    if (lane == 31) {
        s_units[warp] = at0;
        s_spans[warp] = ord0;
    }
    __syncthreads();
    long long total = 0;
    at0 -= units;
    ord0 -= spans;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < warp) {
            at0 += s_units[w];
            ord0 += s_spans[w];
        }
        total += s_units[w];
    }
    const long long per = max((long long)A8_MIN_UNITS, (long long)__umul64hi((unsigned long long)(total + gridDim.x - 1), p.grid_magic));
    const long long lo = (long long)blockIdx.x * per, hi = min(total, lo + per);
    if (lo >= hi) return;

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
    int done = 0;       // pages this part has been through (ring slots and phases follow from it)
    int first = 0, nspans = 0;
    // the spans of [lo, hi), A8_SEGS of them at a time; the first turn only counts them
    for (int seg0 = -A8_SEGS; seg0 < nspans; seg0 += A8_SEGS) {
        if (at0 < hi && at0 + units > lo) {
            long long at = at0;
            int ord = ord0;
            for (int b = b_lo; b < b_hi; ++b) {
                int start;
                const int n = new_tokens(p, b, start), ctx = p.ctx[b];
                for (int qt = 0; (long long)qt * R < (long long)n * rep; ++qt) {
                    const Span s = span_of(p, n, ctx, qt, R, rep);
                    const int u = s.units();
                    const long long end = at + (long long)u * p.G;
                    if (end > lo && at < hi) {
                        // heads [g0, g1) overlap (a tile's heads hold less than 2^31 pages)
                        const int g0 = at >= lo ? 0 : (int)((unsigned)(lo - at) / (unsigned)u);
                        const int g1 = end <= hi ? p.G : (int)((unsigned)(hi - at + u - 1) / (unsigned)u);
                        if (seg0 < 0) {
                            if (at <= lo) s_flag[0] = ord + g0;
                            if (end >= hi) s_flag[1] = ord + g1 - 1;
                        } else {
                            for (int g = max(g0, first + seg0 - ord); g < min(g1, first + seg0 + A8_SEGS - ord); ++g) {
                                const long long from = at + (long long)g * u, to = from + u;
                                Seg x;
                                x.b = b;
                                x.g = g;
                                x.tok = start + s.tok;
                                x.rem = s.rem;
                                x.rows = s.rows;
                                x.pos = ctx - n + s.tok;
                                x.page = s.page + (int)(max(from, lo) - from);
                                x.pend = s.pend;
                                x.v = (int)(max(from, lo) - lo);
                                x.n = (int)(min(to, hi) - max(from, lo));
                                x.c0 = (int)blockIdx.x - (from >= lo ? 0 : (int)((unsigned)(lo - from + per - 1) / (unsigned)per));
                                x.c1 = (int)blockIdx.x + (to <= hi ? 0 : (int)((unsigned)(to - 1 - lo) / (unsigned)per));
                                segs[ord + g - first - seg0] = x;
                            }
                        }
                    }
                    at = end;
                    ord += p.G;
                }
            }
        }
        __syncthreads();
        if (seg0 < 0) {
            first = s_flag[0];
            nspans = s_flag[1] - first + 1;
            continue;
        }
        const int nseg = min(A8_SEGS, nspans - seg0);
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
        const auto issue = [&](int k, int base) {
            const int id = __shfl_sync(0xffffffffu, k - base < 32 ? bid : bid2, k & 31);
            const int g = __shfl_sync(0xffffffffu, k - base < 32 ? gk : gk2, k & 31);
            if (lane == 0 && !dead) {
                const int kk = done + k, slot = kk & (depth - 1);
                if (kk >= depth && !mbar_wait_bounded(empty + slot * 8, (uint32_t)((kk / depth - 1) & 1))) {
                    raise_err(p.err, YK_DEV_ERR_TIMEOUT);
                    dead = true;
                } else if (id < 0) {
                    mbar_arrive(full + slot * 8);
                } else {
                    mbar_arrive_expect_tx(full + slot * 8, C::PAGE);
#pragma unroll
                    for (int x = 0; x < C::BOXES; ++x)
                        tma_load_page(my_ring + slot * C::PAGE + x * C::BOX, &map, x * 128, g, p.layer, id, full + slot * 8);
                }
            }
            dead = __shfl_sync(0xffffffffu, (int)dead, 0);
        };
        fetch(0, bid, gk, kb, vb);
        if (rg == 0)
#pragma unroll 1
            for (int k = 0; k < min(depth, nk); ++k) issue(k, 0);
        fetch(1, bid2, gk2, kb2, vb2);

        int k = 0;
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
#pragma unroll 1
            for (int u = warp; u * 8 < rows; u += 4) {
                const int row = u * 8 + r, i = row_token(row);
                const AT* src = reinterpret_cast<const AT*>(p.q) + (size_t)(sg.tok + i) * p.q_stride +
                                (size_t)(sg.g * rep + sg.rem + row - i * rep) * DH + 16 * c;
                float amax = 0.f;
                uint4 w[sizeof(AT) == 2 ? NH * 2 : 1];
                if constexpr (sizeof(AT) == 2) {
#pragma unroll
                    for (int h = 0; h < NH * 2; ++h) {
                        w[h] = make_uint4(0, 0, 0, 0);
                        if (row < rows) w[h] = __ldcg(reinterpret_cast<const uint4*>(src + 64 * (h >> 1)) + (h & 1));
                    }
#pragma unroll
                    for (int h = 0; h < NH * 2; ++h) {
                        const uint32_t t[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
                        for (int z = 0; z < 4; ++z)
                            amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(t[z] << 16)), fabsf(__uint_as_float(t[z] & 0xffff0000u))));
                    }
                } else if (row < rows) {
#pragma unroll
                    for (int h = 0; h < NH * 4; ++h) {
                        const float4 t = __ldcg(reinterpret_cast<const float4*>(src + 64 * (h >> 2)) + (h & 3));
                        amax = fmaxf(fmaxf(fmaxf(amax, fabsf(t.x)), fmaxf(fabsf(t.y), fabsf(t.z))), fabsf(t.w));
                    }
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                // shift by 2^up: amax = m * 2^E, 1 <= m < 2, to m * 2^14
                const int up = amax == 0.f ? 0 : max(-100, min(100, 14 + 127 - (int)(__float_as_uint(amax) >> 23)));
                const float f = exp2_int(up);
                if (c == 0) s_rf[row] = p.scale_log2 * exp2_int(-up);
                const uint32_t dst = smem_u32(shared) + (uint32_t)(u * TERMS * KS * 256 + lane * 16);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    float x[4];
                    if constexpr (sizeof(AT) == 2) {
                        const uint4 q = w[ks >> 1];
                        const uint32_t a = ks & 1 ? q.z : q.x, b = ks & 1 ? q.w : q.y;
                        x[0] = __uint_as_float(a << 16);
                        x[1] = __uint_as_float(a & 0xffff0000u);
                        x[2] = __uint_as_float(b << 16);
                        x[3] = __uint_as_float(b & 0xffff0000u);
                    } else {
                        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (row < rows) t = __ldcg(reinterpret_cast<const float4*>(src + 64 * (ks >> 2)) + (ks & 3));
                        x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
                    }
#pragma unroll
                    for (int z = 0; z < 4; ++z) x[z] *= f;
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint32_t y0 = pack_f16(x[0], x[1]), y1 = pack_f16(x[2], x[3]);
                        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(
                                         dst + (uint32_t)(t * KS * 256 + (ks >> 1) * 512 + (ks & 1) * 8)),
                                     "r"(y0), "r"(y1)
                                     : "memory");
                        if (TERMS == 2) {  // what this term leaves
                            const float2 a = f32x2(y0), b = f32x2(y1);
                            x[0] -= a.x; x[1] -= a.y; x[2] -= b.x; x[3] -= b.y;
                        }
                    }
                }
            }
            __syncthreads();
            const uint32_t q_smem = smem_u32(shared) + (uint32_t)(rg * NT * TERMS * KS * 256 + lane * 16);
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

            // ---- this part's pages of the span
            const int v_end = sg.v + sg.n;
#pragma unroll 1
            for (; k < nk && v0 + part + nparts * k < v_end; ++k) {
                const int base = k & ~31;
                if (k == base && k > 0) {
                    bid = bid2;
                    gk = gk2;
                    kb = kb2;
                    vb = vb2;
                    fetch(k / 32 + 1, bid2, gk2, kb2, vb2);
                }
                if (rg == 0 && k > 0 && k - 1 + depth < nk) issue(k - 1 + depth, base);
                const int kk = done + k, slot = kk & (depth - 1);
                const int id = __shfl_sync(0xffffffffu, bid, k & 31);
                const int ek = kv8_exponent(__shfl_sync(0xffffffffu, kb, k & 31));
                const int ev = kv8_exponent(__shfl_sync(0xffffffffu, vb, k & 31));
                if (!dead && !mbar_wait_bounded(full + slot * 8, (uint32_t)(kk / depth & 1))) {
                    if (lane == 0) raise_err(p.err, YK_DEV_ERR_TIMEOUT);
                    dead = true;
                }
                dead = __any_sync(0xffffffffu, dead);
                const int j0 = (sg.page + (v0 + part + nparts * k - sg.v)) * 16;
                if (active && !dead && id >= 0) {
                    const uint32_t page = my_ring + (uint32_t)(slot * C::PAGE);
                    float s[NT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
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
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int t = 0; t < TERMS; ++t) {
                                    const int at = ((nt * TERMS + t) * KS + h * 4 + i) / 2;
                                    const uint4 b = C::QREG ? qf[C::QREG ? at : 0] : lds128(q_smem + at * 512);
                                    mma_f16(s[nt], a0, b.x, b.y);
                                    mma_f16(s[nt], a1, b.z, b.w);
                                }
                        }
                    }
                    // scores -> x + e_V in the log2 domain; row 2c: s[0], s[2], row 2c + 1: s[1], s[3]
                    const float fk = exp2_int(ek), shift = (float)ev, inv = exp2_int(-ev);
                    const bool plain = p.cap <= 0.f && j0 + 15 <= sg.pos && (p.window <= 0 || pos_last - j0 < p.window);
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
                                const int back = sg.pos + row_token(row) - (j0 + sigma);  // query minus first key
                                const unsigned w = row < rows ? (p.window > 0 ? (unsigned)p.window : 0x80000000u) : 0u;
                                s[nt][j] = (unsigned)back < w ? s[nt][j] + shift : -INFINITY;
                                s[nt][j + 2] = (unsigned)(back - 8) < w ? s[nt][j + 2] + shift : -INFINITY;
                            }
                    }
                    // raise a row's reference once a weight would pass 2^15
                    bool over = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        over |= fmaxf(s[nt][0], s[nt][2]) > m[nt][0] + 15.f || fmaxf(s[nt][1], s[nt][3]) > m[nt][1] + 15.f;
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
                    uint32_t pb[TERMS][NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][i] = ex2(s[nt][i] - m[nt][i & 1]);
                        l[nt][0] = fmaf(s[nt][0] + s[nt][2], inv, l[nt][0]);
                        l[nt][1] = fmaf(s[nt][1] + s[nt][3], inv, l[nt][1]);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t w = pack_f16(s[nt][2 * j], s[nt][2 * j + 1]);
                            pb[0][nt][j] = transpose8(w);
                            if constexpr (TERMS == 2) {
                                const float2 a = f32x2(w);
                                pb[TERMS - 1][nt][j] = transpose8(pack_f16(s[nt][2 * j] - a.x, s[nt][2 * j + 1] - a.y));
                            }
                        }
                    }
                    // O^T += V^T P^T
#pragma unroll
                    for (int bx = 0; bx < C::BOXES; ++bx) {
                        constexpr int W = DH == 64 ? 2 : 4;  // words of a thread's V bytes per key
                        uint32_t v[4][W];
                        const uint32_t va = page + (uint32_t)(bx * C::BOX);
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
                                        const int back = sg.pos + row_token(row) - (j0 + key);
                                        if (back >= 0 && (p.window <= 0 || back < p.window)) {
                                            atomicOr(&s_nan[row * (DH / 32) + (dim >> 5)], 1u << (dim & 31));
                                            s_flag[3] = 1;
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
            __syncthreads();  // (and every warp is done with the queries in `shared`)
            if ((int)threadIdx.x < rows) {
                const int row = threadIdx.x, w0 = row >= C::ROWS ? 1 : 0;  // (w0: the row group)
                float M = LOWEST, L = 0.f;
                for (int q = 0; q < nparts; ++q) M = fmaxf(M, s_ml[((q << p.lg) + w0) * C::ROWS + row - w0 * C::ROWS].x);
                for (int q = 0; q < nparts; ++q) {
                    const float2 t = s_ml[((q << p.lg) + w0) * C::ROWS + row - w0 * C::ROWS];
                    L += t.y * ex2(t.x - M);
                }
                s_row[row] = make_float2(M, L);
            }
            __syncthreads();
            // warps 0, 1 write, 2, 3 add: buffer warp & 1 (its row group, or half of the parts)
#pragma unroll 1
            for (int turn = 0; turn < 2; ++turn) {
                if (warp >> 1 == turn && active) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int row = nt * 8 + 2 * c + j;
                            const float f = ex2(m[nt][j] - s_row[my0 + row].x);
                            float* const dst = s_o + ((warp & 1) * C::ROWS + row) * C::LDO + v_dim;
#pragma unroll
                            for (int t = 0; t < MT; t += 2) {  // 4 consecutive dims
                                float4* const d = reinterpret_cast<float4*>(dst + (t >> 3) * 128 + 2 * (t & 7));
                                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (turn) x = *d;
                                x.x = fmaf(o[t][nt][j], f, x.x);
                                x.y = fmaf(o[t][nt][j + 2], f, x.y);
                                x.z = fmaf(o[t + 1][nt][j], f, x.z);
                                x.w = fmaf(o[t + 1][nt][j + 2], f, x.w);
                                *d = x;
                            }
                        }
                }
                __syncthreads();
            }
            const bool whole = sg.c0 == sg.c1, nans = s_flag[3] != 0;
            const size_t part_row = (size_t)(2 * blockIdx.x + ((int)blockIdx.x == sg.c0 ? 1 : 0)) * R;
#pragma unroll 1
            for (int i = threadIdx.x; i < rows * D4; i += A8_THREADS) {
                const int row = i / D4, d = i % D4 * 4;
                float4 x = *reinterpret_cast<const float4*>(s_o + row * C::LDO + d);
                if (RG == 1) {
                    const float4 y = *reinterpret_cast<const float4*>(s_o + (C::ROWS + row) * C::LDO + d);
                    x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
                }
                if (nans) {
                    const uint32_t bad = s_nan[row * (DH / 32) + (d >> 5)] >> (d & 31);
                    const float nan = __int_as_float(0x7fffffff);
                    if (bad & 1) x.x = nan;
                    if (bad & 2) x.y = nan;
                    if (bad & 4) x.z = nan;
                    if (bad & 8) x.w = nan;
                }
                const float2 ml = s_row[row];
                if (whole) {
                    const float z = ml.y == 0.f ? 0.f : 1.0f / ml.y;
                    const int tok = row_token(row);
                    store4(reinterpret_cast<AT*>(p.out) + (size_t)(sg.tok + tok) * p.out_stride +
                               (size_t)(sg.g * rep + sg.rem + row - tok * rep) * DH + d, x.x * z, x.y * z, x.z * z, x.w * z);
                } else {
                    __stcg(reinterpret_cast<float4*>(p.ws_o + (part_row + row) * DH + d), x);
                    if (d == 0) __stcg(p.ws_ml + part_row + row, ml);
                }
            }
            if (nans) {
                __syncthreads();
                for (int i = threadIdx.x; i < C::NANS / 4; i += A8_THREADS) s_nan[i] = 0;
                if (threadIdx.x == 0) s_flag[3] = 0;
            }
            if (!whole) {
                // ---- a span cut across CTAs: the last of them to finish joins the parts, in order
                __threadfence();
                __syncthreads();
                if (threadIdx.x == 0) s_flag[2] = atomicAdd(&p.counters[sg.c0], 1) == sg.c1 - sg.c0;
                __syncthreads();
                if (s_flag[2]) {
                    __threadfence();
                    const int nq = sg.c1 - sg.c0 + 1;
                    const auto from = [&](int q) { return (size_t)(2 * (sg.c0 + q) + (q == 0)) * R; };
                    if ((int)threadIdx.x < rows) {
                        const int row = threadIdx.x;
                        float M = LOWEST, L = 0.f;
#pragma unroll 8
                        for (int q = 0; q < nq; ++q) {  // (no branch: the loads go out together)
                            const float2 t = __ldcg(p.ws_ml + from(q) + row);
                            const float mn = fmaxf(M, t.x);
                            L = fmaf(L, ex2(M - mn), t.y * ex2(t.x - mn));
                            M = mn;
                        }
                        s_row[row] = make_float2(M, L == 0.f ? 0.f : 1.0f / L);
                    }
                    __syncthreads();
#pragma unroll 1
                    for (int i = threadIdx.x; i < rows * D4; i += A8_THREADS) {
                        const int row = i / D4, d = i % D4 * 4;
                        const float2 M = s_row[row];
                        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                        for (int q = 0; q < nq; ++q) {
                            const size_t at = from(q) + row;
                            const float f = ex2(__ldcg(&p.ws_ml[at].x) - M.x);
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * DH + d));
                            a.x = fmaf(x.x, f, a.x); a.y = fmaf(x.y, f, a.y); a.z = fmaf(x.z, f, a.z); a.w = fmaf(x.w, f, a.w);
                        }
                        const int tok = row_token(row);
                        store4(reinterpret_cast<AT*>(p.out) + (size_t)(sg.tok + tok) * p.out_stride +
                                   (size_t)(sg.g * rep + sg.rem + row - tok * rep) * DH + d,
                               a.x * M.y, a.y * M.y, a.z * M.y, a.w * M.y);
                    }
                    if (threadIdx.x == 0) p.counters[sg.c0] = 0;
                }
            }
            __syncthreads();  // `shared` and the rows' values are free again
        }
        done += nk;
        __syncthreads();  // (the span list too)
    }
    // every copy asked for has landed: the loop above waited for each, unless it gave up
    if (dead && rg == 0 && lane == 0)
        for (int i = 0; i < depth; ++i)
            for (int ph = 0; ph < 2; ++ph) (void)mbar_wait_bounded_ns(full + i * 8, (uint32_t)ph, 100000000ull);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
// Partial rows of two spans per CTA (its first, begun elsewhere, and its last,
// ended elsewhere): at most two row groups of 8 * a8_max_nt rows.
size_t attention_e4m3_ws_bytes(int num_sms, int head_dim) {
    const size_t rows = 16 * (head_dim == 256 ? 2 : 4), slots = (size_t)2 * A8_CTAS_PER_SM * num_sms;
    return A8_COUNTERS + slots * rows * (8 + 4 * (size_t)head_dim);
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

// (head dim, row of a head group, K|V, layer, block); one box: a head's 16 K rows and 16 V rows.
static yk_status page_map(const yk_kv_pages& g, CUtensorMap* map) {
    const PFN_tmapEncodeTiled encode = tensor_map_encoder();
    if (!encode) {
        yk_set_error("cuTensorMapEncodeTiled not available from the driver");
        return YK_ERR_CUDA;
    }
    const cuuint64_t dh = g.head_dim, rows = (cuuint64_t)16 * g.n_kv_heads;
    const cuuint64_t dims[5] = {dh, rows, 2, (cuuint64_t)g.n_layers, (cuuint64_t)g.num_blocks};
    const cuuint64_t strides[4] = {dh, dh * rows, 2 * dh * rows, 2 * dh * rows * g.n_layers};
    const cuuint32_t box[5] = {(cuuint32_t)std::min<cuuint64_t>(dh, 128), 16, 2, 1, 1};
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
    YK_ARG(a.T >= 0 && a.B > 0 && a.B <= (1 << 20), "T must not be negative, B in 1..2^20");
    YK_ARG(a.n_heads > 0 && a.n_heads <= 65536 && a.n_heads % a.pages.n_kv_heads == 0,
           "n_heads must be a positive multiple of n_kv_heads");
    YK_ARG(a.n_heads / a.pages.n_kv_heads <= 1024, "at most 1024 query heads share a KV head");
    YK_ARG(a.max_blocks > 0 && a.max_blocks <= (1 << 27), "max_blocks must be in 1..2^27");
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
    // the kernel counts tiles (of 8 rows at least) and their pages in 31 and 38 bits
    const int64_t rep = a.n_heads / a.pages.n_kv_heads, tiles = ((int64_t)a.T * rep / 8 + a.B) * a.pages.n_kv_heads;
    if ((int64_t)a.T * a.n_heads > (int64_t)1 << 31 || tiles >= (int64_t)1 << 31 ||
        (int64_t)a.pages.n_kv_heads * a.max_blocks >= (int64_t)1 << 31 ||
        (double)tiles * a.max_blocks >= 274877906944.0) {
        yk_set_error("unsupported: T, B, n_heads and max_blocks together are too large for one call");
        return YK_ERR_UNSUPPORTED;
    }
    return YK_OK;
}

template <typename AT, int DH, int NT>
static yk_status launch_a8(cudaStream_t st, bool pdl, int num_sms, const CUtensorMap& map, const Attn8Params& p) {
    using C = A8Cfg<AT, DH, NT>;
    int dev = 0;
    YK_CHECK_CUDA(cudaGetDevice(&dev));
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {
        YK_CHECK_CUDA(cudaFuncSetAttribute(attn8_kernel<AT, DH, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
        ready.fetch_or(bit, std::memory_order_release);
    }
    YK_CHECK_CUDA(launch_on(st, pdl, attn8_kernel<AT, DH, NT>, num_sms * A8_CTAS_PER_SM, A8_THREADS, C::SMEM, map, p));
    return YK_OK;
}

// The tile: as few n-tiles as hold the rows of a sequence's new tokens; beyond a
// warp's most, two row groups share the pages.
template <typename AT, int DH>
static yk_status launch_a8_rows(cudaStream_t st, bool pdl, int num_sms, const CUtensorMap& map, Attn8Params& p,
                                long long rows) {
    constexpr int MOST = a8_max_nt<AT, DH>();
    p.lg = rows > 8 * MOST ? 1 : 0;
    const int nt = (int)std::min<long long>(MOST, (rows + (8 << p.lg) - 1) / (8 << p.lg));
    if constexpr (MOST >= 4) {
        if (nt == 4) return launch_a8<AT, DH, 4>(st, pdl, num_sms, map, p);
        if (nt == 3) return launch_a8<AT, DH, 3>(st, pdl, num_sms, map, p);
    }
    if constexpr (MOST >= 2) {
        if (nt == 2) return launch_a8<AT, DH, 2>(st, pdl, num_sms, map, p);
    }
    return launch_a8<AT, DH, 1>(st, pdl, num_sms, map, p);
}

yk_status attention_e4m3_launch(cudaStream_t st, bool pdl, int num_sms, const yk_attention_e4m3_args& a) {
    if (a.T == 0) return YK_OK;
    YK_ARG(num_sms * A8_CTAS_PER_SM * 4 <= A8_COUNTERS, "device has more SMs than the workspace's counters");
    CUtensorMap map;
    YK_TRY(page_map(a.pages, &map));
    Attn8Params p;
    p.q = a.q;
    p.out = a.out;
    p.scales = a.pages.scales;
    p.q_starts = a.q_starts;
    p.ctx = a.context_lens;
    p.tables = a.block_tables;
    p.err = a.err;
    p.q_stride = a.q_stride;
    p.out_stride = a.out_stride;
    p.layer_scale = 2LL * a.pages.n_kv_heads * a.layer;
    p.block_scales = 2LL * a.pages.n_kv_heads * a.pages.n_layers;
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
    p.cap = a.cap;
    p.cap_log2 = a.cap * log2e;
    p.inv_cap_log2 = a.cap > 0.f ? 1.0f / p.cap_log2 : 0.f;
    uint8_t* const ws = reinterpret_cast<uint8_t*>(a.workspace);
    const unsigned rep = (unsigned)(a.n_heads / a.pages.n_kv_heads);
    p.rep_magic = rep == 1 ? 0u : (unsigned)((0x100000000ull + rep - 1) / rep);
    const unsigned grid = (unsigned)(num_sms * A8_CTAS_PER_SM);
    p.grid_magic = 0xffffffffffffffffull / grid + 1;
    const int dh = a.pages.head_dim;
    const size_t ws_rows = (size_t)16 * (dh == 256 ? 2 : 4) * 2 * A8_CTAS_PER_SM * num_sms;
    p.counters = reinterpret_cast<int32_t*>(ws);
    p.ws_ml = reinterpret_cast<float2*>(ws + A8_COUNTERS);
    p.ws_o = reinterpret_cast<float*>(ws + A8_COUNTERS + ws_rows * 8);
    // rows of the longest sequence's new tokens, as far as the caller says
    const long long most = a.max_new > 0 ? std::min(a.max_new, a.T) : (a.T + a.B - 1) / a.B;
    const long long rows = most * (a.n_heads / a.pages.n_kv_heads);
    if (a.dtype == YK_DTYPE_BF16) {
        switch (dh) {
            case 64: return launch_a8_rows<__nv_bfloat16, 64>(st, pdl, num_sms, map, p, rows);
            case 128: return launch_a8_rows<__nv_bfloat16, 128>(st, pdl, num_sms, map, p, rows);
            default: return launch_a8_rows<__nv_bfloat16, 256>(st, pdl, num_sms, map, p, rows);
        }
    }
    switch (dh) {
        case 64: return launch_a8_rows<float, 64>(st, pdl, num_sms, map, p, rows);
        case 128: return launch_a8_rows<float, 128>(st, pdl, num_sms, map, p, rows);
        default: return launch_a8_rows<float, 256>(st, pdl, num_sms, map, p, rows);
    }
}

}  // namespace yk
