// yk_attention_e4m3.cuh -- what the two kernels of yk_attention_e4m3 share: the
// arguments, the division of the work over resident CTAs, the joining of spans
// that were cut between CTAs.
#pragma once
#include "yk_epilogue.cuh"
#include "yk_kvcache.cuh"

namespace yk {

constexpr int A8_SEGS = 32;        // spans a CTA lists at a time
constexpr int A8_COUNTERS = 4096;  // bytes of arrival counters, one per CTA
constexpr int A8_SCAN = 48;        // shared words of a8_plan
constexpr float A8_LOWEST = -3.402823466e38f, A8_LARGEST = 3.402823466e38f;

struct Attn8Params {
    const void* q;
    void* out;
    const uint8_t* pool;
    const uint8_t* scales;
    const int32_t *q_starts, *ctx, *tables;
    uint32_t* err;
    int32_t* counters;  // workspace: arrivals at a cut span, by its first CTA (zero between calls)
    float2* ws_ml;      // workspace: (m, l) and O of the parts of cut spans, [2 per CTA][R]
    float* ws_o;
    long long q_stride, out_stride;
    long long block_scales, layer_scale, block_cells, layer_off;
    int T, B, H, G, layer, max_blocks, num_blocks;
    int lg;             // log2 of the row groups
    uint32_t rep_magic;  // ceil(2^32 / (H / G)), 0 where that is 1
    int window;
    float scale_log2, cap, cap_log2, inv_cap_log2;  // _log2: times log2(e)
};

struct Seg {
    int b, g;
    int tok, rem;    // first row of the tile: token tok of the batch, query head rem of the group
    int rows;
    int pos;         // position of that token
    int page, pend;  // first page of this CTA's part; pages of the span's keys end here
    int v, n;        // its place among the listed spans' units (the kernel's own affair) and its length
    int c0, c1;      // first and last CTA of the span
};

// 2^x; results below 2^-126 are zero (without .ftz the instruction comes with three more that keep them).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fmin_nan(float a, float b) {  // (fminf passes over a NaN)
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// tanh to a few 2^-24 of its value: 1 - 2 / (1 + e^2z) away from 0, the odd
// series z - z^3/3 + 2z^5/15 - 17z^7/315 near it.  NaN stays NaN.
__device__ __forceinline__ float tanh_cap(float z) {
    const float e = 1.f - __fdividef(2.f, 1.f + ex2(fmin_nan(z * 2.8853900817779268f, 126.f)));
    const float q = z * z, t = fmaf(fmaf(fmaf(-17.f / 315.f, q, 2.f / 15.f), q, -1.f / 3.f), q, 1.f) * z;
    return fabsf(z) < 0.25f ? t : e;
}

// x / (H / G), x below 128 + H / G (exact: x * (H / G) < 2^32).
__device__ __forceinline__ int div_rep(const Attn8Params& p, int x) {
    return p.rep_magic ? (int)__umulhi((unsigned)x, p.rep_magic) : x;
}

// A span's pages: [page, pend), at least one (page == pend: a tile without keys).
struct Span {
    int rows, page, pend, tok, rem;  // tok: of the sequence
    template <int PU>  // in units of PU pages
    __device__ __forceinline__ int units() const { return max(1, (pend - page + PU - 1) / PU); }
};
// Query tiles of n new tokens (n may be -1).  R is a constant wherever this is called from a kernel's one shape.
__device__ __forceinline__ int tiles_of(int n, int R, int rep) { return n <= 0 ? 0 : (int)(((unsigned)n * (unsigned)rep + (unsigned)R - 1u) / (unsigned)R); }
__device__ __forceinline__ Span span_of(const Attn8Params& p, int n, int ctx, int qt, int R, int rep) {
    // (32 bits hold all of this: the host sees to T * n_heads < 2^31 and max_blocks * 16 <= 2^29)
    const unsigned lo = (unsigned)qt * (unsigned)R;
    Span s;
    s.rows = (int)min((unsigned)n * (unsigned)rep - lo, (unsigned)R);
    s.tok = s.rem = 0;
    if (qt > 0) {
        s.tok = (int)(lo / (unsigned)rep);
        s.rem = (int)lo - s.tok * rep;
    }
    const int first = ctx - n + s.tok;
    const int last = first + div_rep(p, s.rem + s.rows - 1);
    s.pend = (min(max(last, -1), p.max_blocks * 16 - 1) + 16) >> 4;
    s.page = p.window > 0 ? min(max(0, max(first, 0) - p.window + 1) >> 4, s.pend) : 0;
    return s;
}

// New tokens of sequence b; 0 where q_starts does not fit.
__device__ __forceinline__ int new_tokens(const Attn8Params& p, int b, int& start) {
    start = p.q_starts[b];
    const int end = p.q_starts[b + 1];
    return start >= 0 && end >= start && end <= p.T && (b > 0 || start == 0) ? end - start : -1;
}
// Its length.  (Below 0 all positions are, as they are at 0; ctx - n stays inside 32 bits.)
__device__ __forceinline__ int context_of(const Attn8Params& p, int b) { return max(p.ctx[b], 0); }


// A thread's sequences and this CTA's range of units (LEAST at least), [lo, hi) of the spans laid end to end.  A span has COST units
// more than its pages fill, in front, for what it costs beside them: spans that come and go quickly count.
struct A8Work {
    int b_lo, b_hi;
    int start, n, ctx;    // of sequence b_lo ...
    int q_lo, q_hi;       // ... and the query tiles of it that are the thread's (of further sequences: all)
    unsigned units, at0;  // of the thread's sequences, and before them
    unsigned per, lo, hi;
    int ord0;             // spans before the thread's
    int first, nspans;    // spans of the range
};

// A warp, where some q_starts do not fit: whether the sequences that do bring more than T tokens together.  (Starts that
// fall may give the same rows to many, and these more units than 32 bits hold.)
__device__ __forceinline__ bool a8_overlap(const Attn8Params& p) {
    unsigned tokens = 0;
    for (int b = threadIdx.x & 31; b < p.B; b += 32) {
        int start;
        tokens = min(tokens + (unsigned)max(new_tokens(p, b, start), 0), 1u << 31);
    }
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) tokens = min(tokens + __shfl_xor_sync(0xffffffffu, tokens, o), 1u << 31);
    return tokens > (unsigned)p.T;
}

// Block-wide: the range from the lengths on the device (prefix sums over the
// sequences, THREADS threads).  False: nothing for this CTA.
template <int THREADS, int PU, int COST, int LEAST>
__device__ __forceinline__ bool a8_plan(const Attn8Params& p, int R, int rep, unsigned* s_scan, A8Work& w) {
    constexpr int WARPS = THREADS / 32;
    static_assert(2 * WARPS + 2 <= A8_SCAN, "scan words");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // many query tiles to a sequence: 2^share threads to each; more sequences than threads: several to a thread
    const int per_thread = (p.B + THREADS - 1) / THREADS;
    const int share = p.B >= THREADS || p.T * rep <= 2 * R * p.B ? 0 : 31 - __clz(THREADS / p.B);
    w.b_lo = min(p.B, (int)(threadIdx.x >> share) * per_thread);
    w.b_hi = min(p.B, w.b_lo + per_thread);
    w.units = 0;  // (the host sees to it that all pages together stay below 2^31)
    w.start = w.n = w.ctx = w.q_lo = w.q_hi = 0;
    int spans = 0;
    bool misfit = false;
    for (int b = w.b_lo; b < w.b_hi; ++b) {
        int start;
        const int n = new_tokens(p, b, start), ctx = context_of(p, b);
        if (b == w.b_lo) {
            w.start = start;
            w.n = n;
            w.ctx = ctx;
            const int tiles = tiles_of(n, R, rep), each = (tiles + (1 << share) - 1) >> share;
            w.q_lo = min(tiles, ((int)threadIdx.x & ((1 << share) - 1)) * each);
            w.q_hi = min(tiles, w.q_lo + each);
        }
        misfit |= n < 0;
        if (n < 0 || (n > 0 && ctx > p.max_blocks * 16LL)) raise_err(p.err, YK_DEV_ERR_BOUNDS);
        const int q_hi = b == w.b_lo ? w.q_hi : tiles_of(n, R, rep);
        for (int qt = b == w.b_lo ? w.q_lo : 0; qt < q_hi; ++qt) {
            w.units += (unsigned)((span_of(p, n, ctx, qt, R, rep).units<PU>() + COST) * p.G);
            spans += p.G;
        }
    }
    w.at0 = w.units;  // exclusive prefixes over the threads
    w.ord0 = spans;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, w.at0, o);
        const int y = __shfl_up_sync(0xffffffffu, w.ord0, o);
        if (lane >= o) {
            w.at0 += x;
            w.ord0 += y;
        }
    }
    misfit = __any_sync(0xffffffffu, misfit);
    if (lane == 31) {
        s_scan[warp] = w.at0;
        s_scan[WARPS + warp] = (unsigned)w.ord0 | (misfit ? 1u << 31 : 0u);  // (below 2^31 where all starts fit)
    }
    __syncthreads();
    const unsigned wu = lane < WARPS ? s_scan[lane] : 0u, ws = lane < WARPS ? s_scan[WARPS + lane] : 0u;
    const unsigned total = __reduce_add_sync(0xffffffffu, wu);
    w.at0 += __reduce_add_sync(0xffffffffu, lane < warp ? wu : 0u) - w.units;
    w.ord0 += (int)__reduce_add_sync(0xffffffffu, lane < warp ? ws & 0x7fffffffu : 0u) - spans;
    w.per = max((unsigned)LEAST, (total + gridDim.x - 1) / gridDim.x);
    w.lo = min(total, blockIdx.x * w.per);
    w.hi = min(total, w.lo + w.per);
    if (w.lo >= w.hi) return false;
    // the spans that the range begins and ends in: the threads that hold them say so
    if (w.at0 < w.hi && w.at0 + w.units > w.lo && (w.at0 <= w.lo || w.at0 + w.units >= w.hi)) {
        unsigned at = w.at0;
        int ord = w.ord0;
        for (int b = w.b_lo; b < w.b_hi; ++b) {
            int start = w.start, n = w.n, ctx = w.ctx;
            if (b > w.b_lo) {
                n = new_tokens(p, b, start);
                ctx = context_of(p, b);
            }
            const int q_hi = b == w.b_lo ? w.q_hi : tiles_of(n, R, rep);
            for (int qt = b == w.b_lo ? w.q_lo : 0; qt < q_hi; ++qt) {
                const unsigned u = (unsigned)span_of(p, n, ctx, qt, R, rep).units<PU>() + COST, end = at + u * p.G;
                // (its last page's unit may lie behind the range already, or its first one still)
                if (at <= w.lo && end > w.lo) s_scan[2 * WARPS] = (unsigned)ord + (w.lo - at) / u;
                if (at < w.hi && end >= w.hi) {
                    const unsigned i = (w.hi - at - 1) / u;
                    s_scan[2 * WARPS + 1] = (unsigned)ord + i - (COST > 0 && at + i * u + COST >= w.hi ? 1u : 0u);
                }
                at = end;
                ord += p.G;
            }
        }
    }
    __syncthreads();
    w.first = (int)s_scan[2 * WARPS];
    w.nspans = (int)s_scan[2 * WARPS + 1] - w.first + 1;
    // where some starts do not fit (looked for here and not in front of it all: the same code there makes prompts at
    // head_dim 256 1 % slower)
    if (__any_sync(0xffffffffu, lane < WARPS && s_scan[WARPS + lane] >> 31) && a8_overlap(p)) w.nspans = 0;
    return w.nspans > 0;  // (a range may hold nothing but such a cost)
}

// Block-wide: spans seg0 .. seg0 + A8_SEGS - 1 of the range into segs (a barrier must follow).
template <int PU, int COST>
__device__ __forceinline__ void a8_list(const Attn8Params& p, int R, int rep, const A8Work& w, int seg0, Seg* segs) {
    // A warp goes through those of its threads that hold some of them; its lanes take the KV heads.
    const int lane = threadIdx.x & 31;
    unsigned holders = __ballot_sync(0xffffffffu, w.at0 < w.hi && w.at0 + w.units > w.lo);
    for (; holders; holders &= holders - 1) {
        const int who = __ffs(holders) - 1;
        unsigned at = __shfl_sync(0xffffffffu, w.at0, who);
        int ord = __shfl_sync(0xffffffffu, w.ord0, who) - w.first - seg0;  // place in segs
        const int b_lo = __shfl_sync(0xffffffffu, w.b_lo, who), b_hi = __shfl_sync(0xffffffffu, w.b_hi, who);
        int start = __shfl_sync(0xffffffffu, w.start, who), n = __shfl_sync(0xffffffffu, w.n, who);
        int ctx = __shfl_sync(0xffffffffu, w.ctx, who), q_lo = __shfl_sync(0xffffffffu, w.q_lo, who), q_hi = __shfl_sync(0xffffffffu, w.q_hi, who);
        for (int b = b_lo; b < b_hi; ++b) {
            if (b > b_lo) {
                n = new_tokens(p, b, start);
                ctx = context_of(p, b);
                q_lo = 0;
                q_hi = tiles_of(n, R, rep);
            }
            for (int qt = q_lo; qt < q_hi && ord < A8_SEGS && at < w.hi; ++qt) {
                const Span s = span_of(p, n, ctx, qt, R, rep);
                const unsigned u = (unsigned)s.units<PU>() + COST;
                for (int g = max(0, -ord) + lane; g < min(p.G, A8_SEGS - ord); g += 32) {
                    const unsigned from = at + g * u + COST, to = from + u - COST;
                    if (to <= w.lo || from >= w.hi) continue;
                    Seg x;
                    x.b = b;
                    x.g = g;
                    x.tok = start + s.tok;
                    x.rem = s.rem;
                    x.rows = s.rows;
                    x.pos = ctx - n + s.tok;
                    x.page = s.page + PU * (int)(max(from, w.lo) - from);
                    x.pend = s.pend;
                    x.v = 0;
                    x.n = (int)(min(to, w.hi) - max(from, w.lo));
                    x.c0 = x.c1 = (int)blockIdx.x;
                    if (from < w.lo) x.c0 -= (int)((w.lo - from + w.per - 1) / w.per);
                    if (to > w.hi) x.c1 += (int)((to - 1 - w.lo) / w.per);
                    segs[ord + g] = x;
                }
                at += u * p.G;
                ord += p.G;
            }
        }
    }
}

// One thread, after a barrier that follows the writing of a cut span's part:
// counts it; the CTA that counts last will join the span.
__device__ __forceinline__ void a8_arrive(const Attn8Params& p, const Seg& sg, int* s_last, Seg* s_cut) {
    int n;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(n) : "l"(p.counters + sg.c0) : "memory");
    const int which = (int)blockIdx.x == sg.c0;
    s_last[which] = n == sg.c1 - sg.c0;
    s_cut[which] = sg;
}

// Block-wide, at the end.
template <typename AT, int DH, int THREADS>
__device__ __forceinline__ void a8_join(const Attn8Params& p, int R, int rep, const int* s_last, const Seg* s_cut) {
    constexpr int D4 = DH / 4;
    // ---- spans cut across CTAs (this CTA's first, begun elsewhere, or its last): the last
    // CTA to arrive joins the parts, in their order
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        if (!s_last[which]) continue;
        const Seg sg = s_cut[which];
        __threadfence();
        const int nq = sg.c1 - sg.c0 + 1;
#pragma unroll 1
        for (int i = threadIdx.x; i < sg.rows * D4; i += THREADS) {
            const int row = i / D4, d = i % D4 * 4;
            float M = A8_LOWEST, L = 0.f;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int q0 = 0; q0 < nq; q0 += 8) {  // eight parts' loads go out together
                float2 t[8];
                float4 x[8];
#pragma unroll
                for (int z = 0; z < 8; ++z) {
                    const int q = min(q0 + z, nq - 1);
                    const size_t at = (size_t)(2 * (sg.c0 + q) + (q == 0)) * R + row;
                    t[z] = __ldcg(p.ws_ml + at);
                    x[z] = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * DH + d));
                }
                float mn = M;
#pragma unroll
                for (int z = 0; z < 8; ++z) mn = fmaxf(mn, t[z].x);
                const float g = ex2(M - mn);
                a.x *= g; a.y *= g; a.z *= g; a.w *= g;
                L *= g;
                M = mn;
#pragma unroll
                for (int z = 0; z < 8; ++z) {
                    if (q0 + z < nq) {
                        const float f = ex2(t[z].x - mn);
                        L = fmaf(t[z].y, f, L);
                        a.x = fmaf(x[z].x, f, a.x); a.y = fmaf(x[z].y, f, a.y);
                        a.z = fmaf(x[z].z, f, a.z); a.w = fmaf(x[z].w, f, a.w);
                    }
                }
            }
            const float z = L == 0.f ? 0.f : 1.0f / L;
            const int tok = div_rep(p, sg.rem + row);
            store4(reinterpret_cast<AT*>(p.out) + (size_t)(sg.tok + tok) * p.out_stride +
                       (size_t)(sg.g * rep + sg.rem + row - tok * rep) * DH + d, a.x * z, a.y * z, a.z * z, a.w * z);
        }
        if (threadIdx.x == 0) p.counters[sg.c0] = 0;
        __syncthreads();
    }
}

// CTAs per SM * rows of a tile * head_dim: at most this, for every shape (the workspace's parts).
constexpr int A8_WS = 16384;

// bf16 queries (yk_attention_e4m3_tc.cu); map: boxes of 16 K rows.
yk_status attention_e4m3_launch_bf16(cudaStream_t st, bool pdl, int num_sms, int head_dim, const CUtensorMap& map,
                                     const Attn8Params& p, long long rows);

}  // namespace yk
