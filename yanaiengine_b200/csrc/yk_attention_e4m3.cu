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
    int b, qt, g;
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
    static constexpr bool QREG = TERMS * NT * KS * 2 <= 48;  // queries in registers, else shared memory
    static constexpr int QBYTES = QREG ? 0 : 2 * TERMS * NT * KS * 256;  // (two row groups)
    static constexpr int DUMP = 2 * NT * MT * 512;           // two warps' accumulators
    static constexpr int SHARED = QBYTES > DUMP ? QBYTES : DUMP;  // used in turn
    static constexpr size_t SMEM = 1024 + A8_RING + SHARED + 4 * NT * 8 * 8 + A8_SEGS * sizeof(Seg) + 2 * 4 * DEPTH * 8 + 256;
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

// A span's pages: [page, pend), at least one (page == pend: a tile without keys).
struct Span {
    int rows, page, pend;
    __device__ __forceinline__ int units() const { return max(1, pend - page); }
};
__device__ __forceinline__ Span span_of(const Attn8Params& p, int n, int ctx, int qt, int R, int rep) {
    const int lo = (int)((long long)qt * R), hi = (int)min((long long)n * rep, (long long)lo + R);
    const int first = ctx - n + lo / rep, last = ctx - n + (hi - 1) / rep;
    Span s;
    s.rows = hi - lo;
    s.pend = (int)((min(max((long long)last + 1, 0LL), (long long)p.max_blocks * 16) + 15) >> 4);
    s.page = p.window > 0 ? min(max(0, first - p.window + 1) >> 4, s.pend) : 0;
    return s;
}

// New tokens of sequence b; 0 (and the error word) where q_starts does not fit.
__device__ __forceinline__ int new_tokens(const Attn8Params& p, int b, int& start) {
    start = p.q_starts[b];
    const int end = p.q_starts[b + 1];
    const bool ok = start >= 0 && end >= start && end <= p.T && (b > 0 || start == 0);
    if (!ok) raise_err(p.err, YK_DEV_ERR_BOUNDS);
    return ok ? end - start : 0;
}

template <typename AT, int DH, int NT>
__global__ void __launch_bounds__(A8_THREADS, A8_CTAS_PER_SM)
    attn8_kernel(const __grid_constant__ CUtensorMap map, Attn8Params p) {
    using C = A8Cfg<AT, DH, NT>;
    constexpr int TERMS = C::TERMS, KS = C::KS, MT = C::MT, NH = DH / 64;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const shared = ring + A8_RING;  // queries during a span, accumulators at its end
    float2* const s_ml = reinterpret_cast<float2*>(shared + C::SHARED);  // [4 warps][8 * NT] (m, l)
    Seg* const segs = reinterpret_cast<Seg*>(s_ml + 4 * 8 * NT);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(segs + A8_SEGS);
    long long* const s_scan = reinterpret_cast<long long*>(bars + 2 * 4 * C::DEPTH);  // [4] + [4]
    int* const s_flag = reinterpret_cast<int*>(s_scan + 8);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = lane >> 2, c = lane & 3;
    const int RG = 1 << p.lg, nparts = 4 >> p.lg;
    const int part = warp >> p.lg, rg = warp & (RG - 1);
    const int depth = C::DEPTH << p.lg;
    const int R = 8 * NT * RG, rep = p.H / p.G;
    const uint32_t my_ring = smem_u32(ring) + (uint32_t)(part * depth * C::PAGE);
    const uint32_t full = smem_u32(bars + part * depth), empty = smem_u32(bars + 4 * C::DEPTH + part * depth);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4 * C::DEPTH; ++i) {
            mbar_init(smem_u32(bars + i), 1);
            mbar_init(smem_u32(bars + 4 * C::DEPTH + i), (uint32_t)RG);
        }
        mbar_fence_init();
    }
    pdl_trigger();
    pdl_wait();

    // ---- this CTA's range of pages: [lo, hi) of the spans laid end to end
    const int per_thread = (p.B + A8_THREADS - 1) / A8_THREADS;
    const int b_lo = min(p.B, (int)threadIdx.x * per_thread), b_hi = min(p.B, b_lo + per_thread);
    long long mine = 0;
    for (int b = b_lo; b < b_hi; ++b) {
        int start;
        const int n = new_tokens(p, b, start), ctx = p.ctx[b];
        if (n > 0 && ctx > p.max_blocks * 16LL) raise_err(p.err, YK_DEV_ERR_BOUNDS);
        const int tiles = (int)(((long long)n * rep + R - 1) / R);
        for (int qt = 0; qt < tiles; ++qt) mine += (long long)span_of(p, n, ctx, qt, R, rep).units() * p.G;
    }
    long long before = mine;  // inclusive, then exclusive prefix over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
    }
    if (lane == 31) s_scan[warp] = before;
    __syncthreads();
    long long total = 0;
    before -= mine;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    const long long per = max((long long)A8_MIN_UNITS, (total + gridDim.x - 1) / gridDim.x);
    const long long lo = (long long)blockIdx.x * per, hi = min(total, lo + per);
    if (lo >= hi) return;

    // the spans of [lo, hi), numbered in order, A8_SEGS of them at a time
    const auto each_span = [&](auto&& f) {
        if (before >= hi || before + mine <= lo) return;
        long long at = before;
        for (int b = b_lo; b < b_hi; ++b) {
            const int s0 = p.q_starts[b], s1 = p.q_starts[b + 1];
            const int n = s0 >= 0 && s1 >= s0 && s1 <= p.T && (b > 0 || s0 == 0) ? s1 - s0 : 0, ctx = p.ctx[b];
            const int tiles = (int)(((long long)n * rep + R - 1) / R);
            for (int qt = 0; qt < tiles; ++qt) {
                const Span s = span_of(p, n, ctx, qt, R, rep);
                const long long u = s.units(), end = at + u * p.G;
                if (end > lo && at < hi) {
                    const int g0 = (int)(at >= lo ? 0 : (lo - at) / u);
                    const int g1 = (int)(end <= hi ? p.G : (hi - at + u - 1) / u);
                    for (int g = g0; g < g1; ++g) f(b, qt, g, s, at + g * u, u);
                }
                at = end;
            }
        }
    };
    int count = 0;
    each_span([&](int, int, int, const Span&, long long, long long) { ++count; });
    int first = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, first, o);
        if (lane >= o) first += x;
    }
    if (lane == 31) s_scan[4 + warp] = first;
    __syncthreads();
    int nspans = 0;
    first -= count;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < warp) first += (int)s_scan[4 + w];
        nspans += (int)s_scan[4 + w];
    }

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
    for (int seg0 = 0; seg0 < nspans; seg0 += A8_SEGS) {
        __syncthreads();
        {
            int i = first - seg0;
            each_span([&](int b, int qt, int g, const Span& s, long long at, long long u) {
                if (i >= 0 && i < A8_SEGS) {
                    const long long from = max(at, lo), to = min(at + u, hi);
                    segs[i] = Seg{b, qt, g, s.page + (int)(from - at), s.pend, (int)(from - lo), (int)(to - from),
                                  (int)(at / per), (int)((at + u - 1) / per)};
                }
                ++i;
            });
        }
        __syncthreads();
        const int nseg = min(A8_SEGS, nspans - seg0);
        const int v0 = segs[0].v, v1 = segs[nseg - 1].v + segs[nseg - 1].n;
        const int nk = (v1 - v0 - part + nparts - 1) / nparts;  // pages of this part

        // lane i of a batch: block id (-1: nothing to read) and scale exponents of page 32 * batch + i
        int bid = -1, bid2 = -1, sc = 0, sc2 = 0;
        const auto fetch = [&](int batch, int& id, int& e) {
            const int k = batch * 32 + lane;
            id = -1;
            e = 0;
            if (k >= nk) return;
            const int v = v0 + part + nparts * k;
            int a = 0, z = nseg - 1;  // the last span with segs[].v <= v
            while (a < z) {
                const int mid = (a + z + 1) >> 1;
                if (segs[mid].v <= v) a = mid; else z = mid - 1;
            }
            const int page = segs[a].page + (v - segs[a].v);
            if (page >= segs[a].pend) return;
            id = p.tables[(size_t)segs[a].b * p.max_blocks + page];
            if (id < 0 || id >= p.num_blocks) {
                raise_err(p.err, YK_DEV_ERR_BOUNDS);
                id = -1;
                return;
            }
            const uint8_t* s = p.scales + (size_t)id * p.block_scales + p.layer_scale + segs[a].g;
            e = (kv8_exponent(__ldg(s)) + 128) | (kv8_exponent(__ldg(s + p.G)) + 128) << 8 | segs[a].g << 16;
        };
        fetch(0, bid, sc);
        fetch(1, bid2, sc2);
        // page k of this part into its ring slot, once every warp of the part is done with the slot
        const auto issue = [&](int k, int base) {
            const int id = __shfl_sync(0xffffffffu, k - base < 32 ? bid : bid2, k & 31);
            const int g = __shfl_sync(0xffffffffu, k - base < 32 ? sc : sc2, k & 31) >> 16;
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
        if (rg == 0)
            for (int k = 0; k < min(depth, nk); ++k) issue(k, 0);

        int k = 0;
        for (int si = 0; si < nseg; ++si) {
            const Seg sg = segs[si];
            int start = p.q_starts[sg.b];
            const int n = p.q_starts[sg.b + 1] - start, ctx = p.ctx[sg.b];
            const int rows = (int)min((long long)R, (long long)n * rep - (long long)sg.qt * R);
            const int row0 = sg.qt * R, my0 = rg * 8 * NT;  // first row of the tile, of this warp within it
            const int pos_first = ctx - n + row0 / rep, pos_last = ctx - n + (row0 + rows - 1) / rep;
            const bool active = my0 < rows;

            // ---- queries: B fragments, column n = lane / 4, dims 64 h + 16 c + 4 s + {0, 1 | 2, 3}
            uint32_t qf[C::QREG ? TERMS * NT * KS * 2 : 1];
            const uint32_t q_smem = smem_u32(shared) + (uint32_t)(rg * TERMS * NT * KS * 256 + lane * 8);
            float rf[NT][2];  // score of rows 2c, 2c + 1 -> log2 domain
            if (active) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int row = my0 + nt * 8 + r, rr = row0 + row;
                    const AT* src = reinterpret_cast<const AT*>(p.q) + (size_t)(start + rr / rep) * p.q_stride +
                                    (size_t)(sg.g * rep + rr % rep) * DH + 16 * c;
                    float amax = 0.f;
                    uint32_t w[sizeof(AT) == 2 ? NH * 8 : 1];
                    if constexpr (sizeof(AT) == 2) {
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            uint4 x = make_uint4(0, 0, 0, 0), y = x;
                            if (row < rows) {
                                x = __ldcg(reinterpret_cast<const uint4*>(src + 64 * h));
                                y = __ldcg(reinterpret_cast<const uint4*>(src + 64 * h + 8));
                            }
                            const uint32_t t[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                w[h * 8 + i] = t[i];
                                amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(t[i] << 16)),
                                                         fabsf(__uint_as_float(t[i] & 0xffff0000u))));
                            }
                        }
                    } else {
                        if (row < rows)
#pragma unroll
                            for (int h = 0; h < NH; ++h)
#pragma unroll
                                for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(to_f32(src[64 * h + i])));
                    }
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                    // shift by 2^up: amax = m * 2^E, 1 <= m < 2, to m * 2^14
                    const int E = (int)(__float_as_uint(amax) >> 23) - 127;
                    const int up = amax == 0.f ? 0 : max(-100, min(100, 14 - E));
                    const float f = exp2_int(up);
                    const int down = -up;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        rf[nt][j] = p.scale_log2 * exp2_int(__shfl_sync(0xffffffffu, down, 8 * c + 4 * j));
#pragma unroll
                    for (int h = 0; h < NH; ++h)
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            float x[4];
                            if constexpr (sizeof(AT) == 2) {
                                const uint32_t a = w[h * 8 + 2 * s], b = w[h * 8 + 2 * s + 1];
                                x[0] = __uint_as_float(a << 16);
                                x[1] = __uint_as_float(a & 0xffff0000u);
                                x[2] = __uint_as_float(b << 16);
                                x[3] = __uint_as_float(b & 0xffff0000u);
                            } else {
                                float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (row < rows) t = __ldcg(reinterpret_cast<const float4*>(src + 64 * h + 4 * s));
                                x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[i] *= f;
                            uint32_t hi2[2] = {pack_f16(x[0], x[1]), pack_f16(x[2], x[3])};
#pragma unroll
                            for (int t = 0; t < TERMS; ++t) {
                                if (t == 1) {  // what the first term leaves
                                    const float2 a = f32x2(hi2[0]), b = f32x2(hi2[1]);
                                    hi2[0] = pack_f16(x[0] - a.x, x[1] - a.y);
                                    hi2[1] = pack_f16(x[2] - b.x, x[3] - b.y);
                                }
                                const int ks = h * 4 + s;
                                if constexpr (C::QREG) {
                                    qf[((t * NT + nt) * KS + ks) * 2] = hi2[0];
                                    qf[((t * NT + nt) * KS + ks) * 2 + 1] = hi2[1];
                                } else if (part == 0) {
                                    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(
                                                     q_smem + (uint32_t)(((t * NT + nt) * KS + ks) * 256)),
                                                 "r"(hi2[0]), "r"(hi2[1])
                                                 : "memory");
                                }
                            }
                        }
                }
            }
            if constexpr (!C::QREG) __syncthreads();

            float o[MT][NT][4];
            float m[NT][2], l[NT][2];  // m: the row's reference, less the bias of 7
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m[nt][0] = m[nt][1] = -3.402823466e38f;
                l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
                for (int t = 0; t < MT; ++t) o[t][nt][0] = o[t][nt][1] = o[t][nt][2] = o[t][nt][3] = 0.f;
            }

            // ---- this part's pages of the span
            const int v_end = sg.v + sg.n;
            for (; k < nk && v0 + part + nparts * k < v_end; ++k) {
                const int base = k & ~31;
                if (k == base && k > 0) {
                    bid = bid2;
                    sc = sc2;
                    fetch(k / 32 + 1, bid2, sc2);
                }
                if (rg == 0 && k > 0 && k - 1 + depth < nk) issue(k - 1 + depth, base);
                const int kk = done + k, slot = kk & (depth - 1);
                const int id = __shfl_sync(0xffffffffu, bid, k & 31);
                const int e = __shfl_sync(0xffffffffu, sc, k & 31);
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
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t a[4] = {f16x2_lo(x[i]), f16x2_lo(y[i]), f16x2_hi(x[i]), f16x2_hi(y[i])};
                            const int ks = h * 4 + i;
#pragma unroll
                            for (int t = 0; t < TERMS; ++t)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    if constexpr (C::QREG) {
                                        mma_f16(s[nt], a, qf[((t * NT + nt) * KS + ks) * 2], qf[((t * NT + nt) * KS + ks) * 2 + 1]);
                                    } else {
                                        const uint2 b = lds64(q_smem + (uint32_t)(((t * NT + nt) * KS + ks) * 256));
                                        mma_f16(s[nt], a, b.x, b.y);
                                    }
                                }
                        }
                    }
                    // scores -> x + e_V in the log2 domain; row 2c: s[0], s[2], row 2c + 1: s[1], s[3]
                    const int ek = (e & 255) - 128, ev = (e >> 8 & 255) - 128;
                    const float fk = exp2_int(ek), shift = (float)ev, inv = exp2_int(-ev);
                    const bool plain = p.cap <= 0.f && j0 + 15 <= pos_first && (p.window <= 0 || pos_last - j0 < p.window);
                    uint32_t seen = 0xffffffffu;  // bit nt * 4 + i: s[nt][i]'s key is visible to its row
                    if (plain) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                s[nt][i] = fmaf(s[nt][i], fminf(rf[nt][i & 1] * fk, 3.402823466e38f), shift);
                    } else {
                        seen = 0;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int row = my0 + nt * 8 + 2 * c + (i & 1);
                                const int pos = ctx - n + (row0 + row) / rep, j = j0 + sigma + (i >> 1) * 8;
                                const bool vis = row < rows && j <= pos && (p.window <= 0 || pos - j < p.window);
                                float x = s[nt][i] * fminf(rf[nt][i & 1] * fk, 3.402823466e38f);
                                if (p.cap > 0.f) x = p.cap_log2 * tanhf(x * p.inv_cap_log2);
                                s[nt][i] = vis ? x + shift : -INFINITY;
                                seen |= (vis ? 1u : 0u) << (nt * 4 + i);
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
                        bool nan = false;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t va = page + (uint32_t)(bx * C::BOX + (j >> 1) * 8 * C::ROWB) + v_off[j & 1];
                            if constexpr (DH == 64) {
                                const uint2 t = lds64(va);
                                v[j][0] = t.x; v[j][1] = t.y;
                            } else {
                                const uint4 t = lds128(va);
                                v[j][0] = t.x; v[j][1] = t.y; v[j][2] = t.z; v[j][3] = t.w;
                            }
                            if (!plain)
#pragma unroll
                                for (int i = 0; i < W; ++i)
                                    nan |= ((v[j][i] & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u) != 0;
                        }
                        nan = !plain && __any_sync(0xffffffffu, nan);
#pragma unroll
                        for (int i = 0; i < W; ++i) {
                            const uint32_t lo01 = __byte_perm(v[0][i], v[1][i], 0x5140), hi01 = __byte_perm(v[0][i], v[1][i], 0x7362);
                            const uint32_t lo23 = __byte_perm(v[2][i], v[3][i], 0x5140), hi23 = __byte_perm(v[2][i], v[3][i], 0x7362);
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const uint32_t w0 = half ? hi01 : lo01, w1 = half ? hi23 : lo23;
                                uint32_t a[4] = {f16x2_lo(w0), f16x2_hi(w0), f16x2_lo(w1), f16x2_hi(w1)};
                                const int t = bx * 8 + 2 * i + half;
                                if (nan) {
                                    // a NaN cell reaches the rows that see its key, and no others: it counts as 0
                                    // here, and rows with a visible one become NaN (a product of flags finds them)
                                    uint32_t flag[4];
#pragma unroll
                                    for (int z = 0; z < 4; ++z) {
                                        const uint32_t bad = __hneu2_mask(*reinterpret_cast<__half2*>(&a[z]), *reinterpret_cast<__half2*>(&a[z]));
                                        flag[z] = bad & 0x3c003c00u;  // 1.0
                                        a[z] &= ~bad;
                                    }
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) {
                                        float hit[4] = {0.f, 0.f, 0.f, 0.f};
                                        const uint32_t f0 = (seen >> (nt * 4) & 1) * 0x3c00u | (seen >> (nt * 4 + 1) & 1) * 0x3c000000u;
                                        const uint32_t f1 = (seen >> (nt * 4 + 2) & 1) * 0x3c00u | (seen >> (nt * 4 + 3) & 1) * 0x3c000000u;
                                        mma_f16(hit, flag, transpose8(f0), transpose8(f1));
#pragma unroll
                                        for (int z = 0; z < 4; ++z)
                                            if (hit[z] > 0.f) o[t][nt][z] = __int_as_float(0x7fffffff);
                                    }
                                }
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

            // ---- end of the span: the parts of a row group are joined
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
                    l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
                    l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
                    if (r == 0) s_ml[warp * 8 * NT + nt * 8 + 2 * c + j] = make_float2(m[nt][j], l[nt][j]);
                }
            __syncthreads();  // (and every warp is done with the queries in `shared`)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = nt * 8 + 2 * c + j;
                    float M = -3.402823466e38f, L = 0.f;
                    for (int q = 0; q < nparts; ++q) M = fmaxf(M, s_ml[((q << p.lg) + rg) * 8 * NT + at].x);
                    for (int q = 0; q < nparts; ++q) {
                        const float2 t = s_ml[((q << p.lg) + rg) * 8 * NT + at];
                        L += t.y * ex2(t.x - M);
                    }
                    const float f = ex2(m[nt][j] - M);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        o[t][nt][j] *= f;
                        o[t][nt][j + 2] *= f;
                    }
                    m[nt][j] = M;
                    l[nt][j] = L;
                }
            // warps 2, 3 -> 0, 1 (their row group's part with the same index mod 2); then, with four
            // parts, 0 and 1 swap halves so that both finish half of the dims
            float4* const dump = reinterpret_cast<float4*>(shared);  // [2 warps][MT][NT][32 lanes]
            if (warp >= 2) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        dump[(((warp - 2) * MT + t) * NT + nt) * 32 + lane] = make_float4(o[t][nt][0], o[t][nt][1], o[t][nt][2], o[t][nt][3]);
            }
            __syncthreads();
            if (warp < 2) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float4 x = dump[((warp * MT + t) * NT + nt) * 32 + lane];
                        o[t][nt][0] += x.x; o[t][nt][1] += x.y; o[t][nt][2] += x.z; o[t][nt][3] += x.w;
                    }
            }
            int t0 = 0, t1 = MT;  // the m-tiles this warp finishes
            if (RG == 1) {
                __syncthreads();
                if (warp < 2) {
#pragma unroll
                    for (int t = 0; t < MT; ++t)
                        if ((t >= MT / 2) == (warp == 0))
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                dump[(t * NT + nt) * 32 + lane] = make_float4(o[t][nt][0], o[t][nt][1], o[t][nt][2], o[t][nt][3]);
                }
                __syncthreads();
                if (warp < 2) {
#pragma unroll
                    for (int t = 0; t < MT; ++t)
                        if ((t >= MT / 2) == (warp == 1))
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                const float4 x = dump[(t * NT + nt) * 32 + lane];
                                o[t][nt][0] += x.x; o[t][nt][1] += x.y; o[t][nt][2] += x.z; o[t][nt][3] += x.w;
                            }
                    t0 = warp * (MT / 2);
                    t1 = t0 + MT / 2;
                }
            }
            const bool whole = sg.c0 == sg.c1;
            const int mine_slot = 2 * (int)blockIdx.x + ((int)blockIdx.x == sg.c0 ? 1 : 0);
            if (warp < 2 && active) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int row = my0 + nt * 8 + 2 * c + j, rr = row0 + row;
                        if (row < rows) {
                            const float z = whole ? (l[nt][j] == 0.f ? 0.f : 1.0f / l[nt][j]) : 1.f;
                            AT* dst = reinterpret_cast<AT*>(p.out) + (size_t)(start + rr / rep) * p.out_stride +
                                      (size_t)(sg.g * rep + rr % rep) * DH;
                            float* ws = p.ws_o + ((size_t)mine_slot * R + row) * DH;
                            if (!whole && r == 0 && t0 == 0)
                                __stcg(p.ws_ml + (size_t)mine_slot * R + row, make_float2(m[nt][j], l[nt][j]));
#pragma unroll
                            for (int t = 0; t < MT; t += 2) {  // 4 consecutive dims
                                if (t < t0 || t >= t1) continue;
                                const int d = (t >> 3) * 128 + v_dim + 2 * (t & 7);
                                const float a0 = o[t][nt][j] * z, a1 = o[t][nt][j + 2] * z;
                                const float a2 = o[t + 1][nt][j] * z, a3 = o[t + 1][nt][j + 2] * z;
                                if (whole) store4(dst + d, a0, a1, a2, a3);
                                else __stcg(reinterpret_cast<float4*>(ws + d), make_float4(a0, a1, a2, a3));
                            }
                        }
                    }
            }
            if (whole) {
                __syncthreads();  // `shared` and s_ml are free again
                continue;
            }
            // ---- a span cut across CTAs: the last of them to finish joins the parts, in order
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) s_flag[0] = atomicAdd(&p.counters[sg.c0], 1) == sg.c1 - sg.c0;
            __syncthreads();
            if (s_flag[0]) {
                __threadfence();
                constexpr int D4 = DH / 4;
                for (int i = threadIdx.x; i < rows * D4; i += A8_THREADS) {
                    const int row = i / D4, d = i % D4 * 4;
                    float M = -3.402823466e38f, L = 0.f;
                    for (int q = sg.c0; q <= sg.c1; ++q)
                        M = fmaxf(M, __ldcg(p.ws_ml + (size_t)(2 * q + (q == sg.c0)) * R + row).x);
                    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int q = sg.c0; q <= sg.c1; ++q) {
                        const size_t at = (size_t)(2 * q + (q == sg.c0)) * R + row;
                        const float2 t = __ldcg(p.ws_ml + at);
                        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * DH + d));
                        const float f = ex2(t.x - M);
                        L += t.y * f;
                        a.x = fmaf(x.x, f, a.x); a.y = fmaf(x.y, f, a.y); a.z = fmaf(x.z, f, a.z); a.w = fmaf(x.w, f, a.w);
                    }
                    const float z = L == 0.f ? 0.f : 1.0f / L;
                    const int rr = row0 + row;
                    store4(reinterpret_cast<AT*>(p.out) + (size_t)(start + rr / rep) * p.out_stride +
                               (size_t)(sg.g * rep + rr % rep) * DH + d, a.x * z, a.y * z, a.z * z, a.w * z);
                }
                if (threadIdx.x == 0) p.counters[sg.c0] = 0;
            }
            __syncthreads();
        }
        done += nk;
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
    YK_ARG((int64_t)a.T * a.n_heads <= (int64_t)1 << 31, "T * n_heads too large");
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
