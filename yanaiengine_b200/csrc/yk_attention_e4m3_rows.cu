// yk_attention_e4m3_rows.cu -- yk_attention_e4m3 for bf16 queries and many rows
// (prompts), on the tcgen05 tensor cores.
//
// The pipeline of the kernel for few rows, with the products the other way round:
//   S[128 rows x 128 keys] = Q K^T (kind::f8f6f4, Q in two terms),
//   O[128 rows x dims] += P V (kind::f16, P from TMEM, V as f16).
// A softmax thread holds a row, so its maximum, its sum and its reference need no
// other thread.  Two groups of four warps take the tiles in turn; a row's
// reference m passes between its two threads, tile by tile: a group reads the
// scores for their maximum, waits for the other's decision on the tile before,
// decides (m moves as in the kernel for few rows), and goes on to the weights.
// Weights go to TMEM as f16, where the second product reads them.
//
// Scores go out two tiles ahead of their values' product, so that a group finds its
// next tile ready; a moved reference rescales O only after the weights, when the
// product that it has to wait for is mostly done; the page loops are short (8 KB of
// code: unrolled they ran 4 % slower, from instruction fetch).
// Measured: three prompts of 1500 tokens over up to 5000 keys, 32 query and 8 KV
// heads of 128, 340 us, 0.61 PFLOP/s (43 % of the matrix product's sustained rate;
// the kernel for few rows: 813 us).  A tile of 128 x 128 takes about 2800 cycles, of
// which the two products need 1080 and the exponentials 1024 of their unit's; the
// softmax warps' instructions (1500 issued a tile by each scheduler) bound it.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "yk_attention_e4m3_tc.cuh"

namespace yk {

constexpr int TCR_THREADS = 512;  // warps 0-7 softmax, 8-11 V and results, 12 K and 13 V copies, 14 MMA, 15 queries
constexpr int TCR_ROWS = 128;

template <int DH>
struct TcrCfg {
    static constexpr int R = TCR_ROWS;
    static constexpr int ROWB = DH == 64 ? 64 : 128;  // bytes of a row of K or Q in one block
    static constexpr int KT = TCA_TILE * DH;          // bytes of a K (or V) tile
    static constexpr int V16 = 2 * KT, QB = 2 * R * DH;
    static constexpr int SMALL = (2 + 1 + 4 + 4) * R * 4 + R * (DH / 32) * 4 + 2 * TCA_INFO * TCA_PAGES * 4 +
                                 (A8_SEGS + 2) * (int)sizeof(Seg) + A8_SCAN * 4 + 64 * 8 + 128;
    static constexpr int ROOM = 227 * 1024 - 1024 - SMALL - 2 * V16 - 2 * QB;
    static constexpr int TILES = ROOM / KT;           // K and V tiles that fit
    static constexpr int NV = TILES / 2 < 6 ? TILES / 2 : 6, NK = TILES - NV < 6 ? TILES - NV : 6;
    static constexpr int SMEM = 1024 + (NK + NV) * KT + 2 * V16 + 2 * QB + SMALL;
    static constexpr int TMEM = 512;                  // two S of 128 columns, two P of 64, O
    static_assert(NK >= 2 && NV >= 2 && R * DH <= A8_WS, "tile shapes; cut spans' rows in the workspace");
};

// d += A B, A (f16, two keys a column) from TMEM.
__device__ __forceinline__ void mma_tc_ta(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Keeps what uses x behind the wait that precedes this.
__device__ __forceinline__ void settle(uint32_t (&x)[16]) {
    asm volatile("" : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]),
                      "+r"(x[9]), "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]));
}
// Raw scores of a page with this word -> log2 domain (above zero: masked ones stay -inf).
__device__ __forceinline__ float score_factor(int word, float rf) { return fmaxf(fminf(exp2_int((word & 255) - 128) * rf, A8_LARGEST), 1.18e-38f); }
// Barriers of the two warps of 32 rows: barrier 3 + quad says that an even tile's references are decided, 7 + quad an odd one's.
__device__ __forceinline__ void pair_wait(int group, int quad) { asm volatile("bar.sync %0, 64;" ::"r"(3 + 4 * group + quad) : "memory"); }
__device__ __forceinline__ void pair_tell(int group, int quad) { asm volatile("bar.arrive %0, 64;" ::"r"(3 + 4 * group + quad) : "memory"); }

// Scores that are capped (then in the log2 domain) or masked: -inf where the row does not see the key.
static __device__ __noinline__ void finish_scores(uint32_t s_at, const int* info, float rf, int pos, int j0, unsigned window, float cap, float cap_log2,
                                                  float inv_cap_log2) {
#pragma unroll 1
    for (int b = 0; b < TCA_PAGES; ++b) {
        uint32_t x[16];
        const int w = info[b];
        const unsigned wk = w >= 0 ? window : 0u;
        // (a page that all rows of the warp see whole stays as it is)
        if (cap <= 0.f && __all_sync(0xffffffffu, (unsigned)(pos - j0 - 16 * b) < wk && (unsigned)(pos - j0 - 16 * b - 15) < wk)) continue;
        tmem_ld<16>(s_at + 16 * b, x);
        const float f = cap > 0.f ? score_factor(w >= 0 ? w : 128, rf) : 1.f;
        tmem_wait_ld();
        settle(x);
#pragma unroll
        for (int z = 0; z < 16; ++z) {
            float v = __uint_as_float(x[z]) * f;
            if (cap > 0.f) v = cap_log2 * tanh_cap(v * inv_cap_log2);
            x[z] = __float_as_uint((unsigned)(pos - (j0 + 16 * b + z)) < wk ? v : -INFINITY);
        }
        tmem_st<16>(s_at + 16 * b, x);
    }
    tmem_wait_st();
}

// Scores -> what the weights are 2^ of, in TMEM: rounded as the row's largest was when its reference was taken from it.
// (Where fp32 holds scores to whole numbers or worse, a product that is not rounded before the reference is taken off may
// lie above the largest by more than f16 has room for.)
static __device__ __noinline__ void settle_scores(uint32_t s_at, const int* info, float rf, bool raw, float now) {
#pragma unroll 1
    for (int b = 0; b < TCA_PAGES; ++b) {
        uint32_t x[16];
        const int w = info[b];
        tmem_ld<16>(s_at + 16 * b, x);
        const float f = raw ? score_factor(w, rf) : 1.f, ev = (float)(w >= 0 ? (w >> 8) - 128 : 0);
        tmem_wait_ld();
        settle(x);
#pragma unroll
        for (int z = 0; z < 16; ++z) x[z] = __float_as_uint(fmaf(__uint_as_float(x[z]), f, ev) - now);
        tmem_st<16>(s_at + 16 * b, x);
    }
    tmem_wait_st();
}

template <int DH>
__global__ void __launch_bounds__(TCR_THREADS, 1) attn8_rows_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ Attn8Params p) {
    using C = TcrCfg<DH>;
    constexpr int R = C::R, NK = C::NK, NV = C::NV;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const k_ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const v_ring = k_ring + NK * C::KT;
    uint8_t* const v16 = v_ring + NV * C::KT;
    uint8_t* const s_q = v16 + 2 * C::V16;
    float* const s_rf = reinterpret_cast<float*>(s_q + 2 * C::QB);  // [2][R] score factors of a span's rows
    float* const s_m = s_rf + 2 * R;                                // [R] references
    float* const s_l = s_m + R;                                     // [2][2 groups][R] sums ...
    float* const s_mo = s_l + 4 * R;                                // ... and the references they go with
    uint32_t* const s_nan = reinterpret_cast<uint32_t*>(s_mo + 4 * R);  // [R][DH / 32]
    // [2][INFO][8]: exponents of a tile's pages, -1: no page (for the softmax warps, for the V warps)
    int* const s_info = reinterpret_cast<int*>(s_nan + R * (DH / 32));
    uint64_t* const bars = reinterpret_cast<uint64_t*>((reinterpret_cast<uintptr_t>(s_info + 2 * TCA_INFO * TCA_PAGES) + 7) & ~uintptr_t(7));
    Seg* const segs = reinterpret_cast<Seg*>(bars + 64);
    Seg* const s_cut = segs + A8_SEGS;  // [2]
    unsigned* const s_scan = reinterpret_cast<unsigned*>(s_cut + 2);
    int* const s_last = reinterpret_cast<int*>(s_scan + A8_SCAN);  // [2]
    int* const s_flag = s_last + 2;                                 // NaN cells seen
    uint32_t* const s_tmem = reinterpret_cast<uint32_t*>(s_flag + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rep = p.H / p.G;
    const uint32_t b0 = smem_u32(bars);
    const uint32_t k_full = b0, k_empty = k_full + 8 * NK, v_full = k_empty + 8 * NK, v_empty = v_full + 8 * NV;
    const uint32_t s_full = v_empty + 8 * NV, s_empty = s_full + 16, p_full = s_empty + 16, p_empty = p_full + 16;
    const uint32_t w_full = p_empty + 16, w_empty = w_full + 16;  // f16 V
    const uint32_t q_full = w_empty + 16, q_empty = q_full + 16, l_full = q_empty + 16, l_empty = l_full + 16;
    const uint32_t o_full = l_empty + 16, o_empty = o_full + 8;
    static_assert(2 * NK + 2 * NV + 22 <= 64, "barriers");
    if (threadIdx.x == 480) {  // (not of the warps that plan first)
        const auto init = [](uint32_t bar, int n, int count) {
            for (int i = 0; i < n; ++i) mbar_init(bar + 8 * i, (uint32_t)count);
        };
        init(k_full, NK, 1);
        init(k_empty, NK, 1);
        init(v_full, NV, 1);
        init(v_empty, NV, 4);
        init(s_full, 2, 2);   // the products, and the MMA thread itself (it passes on what it has seen)
        init(s_empty, 2, 4);
        init(p_full, 2, 4);
        init(p_empty, 2, 1);
        init(w_full, 2, 4);
        init(w_empty, 2, 1);
        init(q_full, 2, 1);
        init(q_empty, 2, 9);  // the products, and the softmax warps (score factors)
        init(l_full, 2, 8);
        init(l_empty, 2, 4);
        init(o_full, 1, 1);
        init(o_empty, 1, 4);
        mbar_fence_init();
        *s_flag = s_last[0] = s_last[1] = 0;
    }
    for (int i = threadIdx.x; i < R * (DH / 32); i += TCR_THREADS) s_nan[i] = 0;
    pdl_wait();
    A8Work work;
    if (warp == 14) tmem_alloc(smem_u32(s_tmem), C::TMEM);
    const bool busy = a8_plan<TCR_THREADS, TCA_PAGES, TCA_COST, 1>(p, R, rep, s_scan, work);  // (block-uniform)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    if (!busy) {
        if (warp == 14) tmem_dealloc(tmem, C::TMEM);
        return;
    }
    pdl_trigger();  // (after the TMEM is taken: a kernel that starts early does not take it first)
    const auto col_s = [&](int b) { return tmem + (uint32_t)(b * 128); };
    const auto col_p = [&](int b) { return tmem + (uint32_t)(256 + b * 64); };
    const uint32_t col_o = tmem + 384;

    // per role, through all rounds
    bool dead = false;  // a bounded wait ran out: the role goes through the motions without touching memory
    const auto wait = [&](uint32_t bar, int parity) {
        if (!dead && !mbar_test(bar, (uint32_t)parity)) dead = !wait_longer(bar, (uint32_t)parity, p.err);
    };
    const auto wait2 = [&](uint32_t bar_a, int parity_a, uint32_t bar_b, int parity_b) {
        const bool a = mbar_test(bar_a, (uint32_t)parity_a), b = mbar_test(bar_b, (uint32_t)parity_b);
        if (!dead && !a) dead = !wait_longer(bar_a, (uint32_t)parity_a, p.err);
        if (!dead && !b) dead = !wait_longer(bar_b, (uint32_t)parity_b, p.err);
    };
    Turn<NK> kt;
    Turn<NV> vt;
    Turn<2> st, pt, qt, wt, lt;
    Turn<1> ot;
    int tile = 0;  // of this CTA

    for (int seg0 = 0; seg0 < work.nspans; seg0 += A8_SEGS) {
        __syncwarp();
        __syncthreads();
        a8_list<TCA_PAGES, TCA_COST>(p, R, rep, work, seg0, segs);
        __syncthreads();
        const int nseg = min(A8_SEGS, work.nspans - seg0);
        // Queries of 128 rows are 32 steps of one warp, about 8 tiles' time: behind a shorter span the V warps convert
        // their share while it begins (200 tokens over 2000 keys: 48 -> 31 us; done for every span, the long
        // prompts lose 6 %).
        const auto shared_queries = [&](int si) { return si == 0 || segs[si - 1].n < 8; };
        if (warp < 8) {
            // ---------------- softmax: row 32 * quad + lane; group 0 takes the even tiles, group 1 the odd ones ----------------
            const int quad = warp & 3, group = warp >> 2, row = 32 * quad + lane;
            const uint32_t lanes = (uint32_t)(32 * quad) << 16;
            const uint32_t s_at = col_s(group) + lanes, p_at = col_p(group) + lanes, o_at = col_o + lanes;
            const unsigned window = p.window > 0 ? (unsigned)p.window : 0x80000000u;
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const Seg& sg = segs[si];
                const int n = sg.n, tile0 = tile;
                const int pos = sg.pos + div_rep(p, sg.rem + row), pos_last = sg.pos + div_rep(p, sg.rem + sg.rows - 1);
                float m = A8_LOWEST, l = 0.f;  // this thread's sum goes with this reference
#pragma unroll 1
                for (int i = (tile0 ^ group) & 1; i < n; i += 2) {
                    const int t = tile0 + i, j0 = (sg.page + TCA_PAGES * i) * 16, use = t >> 1;
                    const int* const info = s_info + (t & (TCA_INFO - 1)) * TCA_PAGES;
                    wait(s_full + 8 * group, use & 1);
                    tc_fence_after();
                    uint32_t x[2][16];
                    const float rf = s_rf[qt.slot * R + row];
                    bool raw = p.cap <= 0.f;  // the scores in TMEM are not in the log2 domain yet
                    {
                        const int4 a = *reinterpret_cast<const int4*>(info), b = *reinterpret_cast<const int4*>(info + 4);
                        if (!raw || !all_seen(p, sg, pos_last, j0) || (a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) < 0)
                            finish_scores(s_at, info, rf, pos, j0, window, p.cap, p.cap_log2, p.inv_cap_log2);
                    }
                    // the row's largest score + e_V (two pages a turn; the next page's scores come while one's are used)
                    float top = -INFINITY;
                    tmem_ld<16>(s_at, x[0]);
#pragma unroll 1
                    for (int b = 0; b < TCA_PAGES; b += 2) {
                        const int2 w = *reinterpret_cast<const int2*>(info + b);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            uint32_t(&y)[16] = x[u];
                            tmem_wait_ld();
                            settle(y);
                            tmem_ld<16>(s_at + (uint32_t)(16 * (b + u + 1) & 127), x[u ^ 1]);
                            float most = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
#pragma unroll
                            for (int z = 2; z < 16; z += 2) most = fmaxf(most, fmaxf(__uint_as_float(y[z]), __uint_as_float(y[z + 1])));
                            const int word = u ? w.y : w.x;
                            top = fmaxf(top, fmaf(most, raw ? score_factor(word, rf) : 1.f, (float)(word >= 0 ? (word >> 8) - 128 : 0)));
                        }
                    }
                    // the reference, after the tile before has decided: 2^3 below a row's first weights, and again before one
                    // would pass 2^15
                    if (t > 0) pair_wait(group ^ 1, quad);
                    float now = i == 0 ? A8_LOWEST : s_m[row];
                    const bool over = top - now > 15.f, moves = __any_sync(0xffffffffu, over) && i > 0;
                    const float was = now;
                    if (over) now = top - 3.f;
                    s_m[row] = now;
                    if (i + 1 < n || si + 1 < nseg || seg0 + A8_SEGS < work.nspans) pair_tell(group, quad);  // (not after the last tile)
                    l *= ex2(m - now);
                    m = now;
                    // (one reference of the warp's 32 from 2^22 on: all of them the long way)
                    const bool far = __any_sync(0xffffffffu, fabsf(now) >= 4194304.f && now != A8_LOWEST);
                    if (far) {
                        tmem_wait_ld();
                        settle_scores(s_at, info, rf, raw, now);
                        tmem_ld<16>(s_at, x[0]);
                        raw = false;
                    }
                    wait(p_empty + 8 * group, (use & 1) ^ 1);
                    tc_fence_after();
#pragma unroll 1
                    for (int b = 0; b < TCA_PAGES; b += 2) {
                        const int2 w = *reinterpret_cast<const int2*>(info + b);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            uint32_t(&y)[16] = x[u];
                            tmem_wait_ld();
                            settle(y);
                            if (u == 0 || b + 2 < TCA_PAGES) tmem_ld<16>(s_at + (uint32_t)(16 * (b + u + 1)), x[u ^ 1]);
                            const int word = u ? w.y : w.x, ev = word >= 0 ? (word >> 8) - 128 : 0;
                            const float f = raw ? score_factor(word, rf) : 1.f, c = far ? 0.f : (float)ev - now;
                            const float2 ff = make_float2(f, f), cc = make_float2(c, c);
                            float2 sum = make_float2(0.f, 0.f);
                            uint32_t h[8];
#pragma unroll
                            for (int z = 0; z < 16; z += 2) {
                                const float2 d = fma2(make_float2(__uint_as_float(y[z]), __uint_as_float(y[z + 1])), ff, cc);
                                const float2 e = make_float2(ex2(d.x), ex2(d.y));
                                sum = add2(sum, e);
                                h[z / 2] = f16x2_of(e.x, e.y);
                            }
                            l = fmaf(sum.x + sum.y, exp2_int(-ev), l);
                            tmem_st<8>(p_at + (uint32_t)(8 * (b + u)), h);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_empty + 8 * group);
                    if (moves) {
                        // O follows, once the products of the tile before are done (by now they mostly are)
                        const float g = ex2(was - now);
                        wait(p_empty + 8 * (group ^ 1), ((t - 1) >> 1) & 1);
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < DH; c += 16) {
                            tmem_ld<16>(o_at + (uint32_t)c, x[0]);
                            tmem_wait_ld();
                            settle(x[0]);
#pragma unroll
                            for (int z = 0; z < 16; ++z) x[0][z] = __float_as_uint(__uint_as_float(x[0][z]) * g);
                            tmem_st<16>(o_at + (uint32_t)c, x[0]);
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full + 8 * group);
                }
                tile += n;
                wait(l_empty + 8 * lt.slot, lt.phase ^ 1);
                s_l[(2 * lt.slot + group) * R + row] = l;
                s_mo[(2 * lt.slot + group) * R + row] = m;
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(l_full + 8 * lt.slot);
                    mbar_arrive(q_empty + 8 * qt.slot);
                }
                qt.next();
                lt.next();
            }
        } else if (warp < 12) {
            // ---------------- V: e4m3 -> f16, and the results ----------------
            const int tid = threadIdx.x - 256, quad = warp & 3;
            const uint32_t lanes = (uint32_t)(32 * quad) << 16;
            const auto queries = [&](int si) {
                if (shared_queries(si)) {
                    convert_queries<DH, R, true>(p, segs[si], rep, lane, quad, 5, s_q + qt.slot * C::QB, s_rf + qt.slot * R,
                                                 [&] { wait(q_empty + 8 * qt.slot, qt.phase ^ 1); return !dead; });
                    fence_proxy_async_smem();
                    queries_bar();
                }
                qt.next();
            };
            queries(0);
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const Seg sg = segs[si];
                const int pos_last = sg.pos + div_rep(p, sg.rem + sg.rows - 1);
#pragma unroll 1
                for (int i = 0; i < sg.n; ++i, ++tile) {
                    const int j0 = (sg.page + TCA_PAGES * i) * 16;
                    wait2(v_full + 8 * vt.slot, vt.phase, w_empty + 8 * wt.slot, wt.phase ^ 1);
                    if (!dead)
                        convert_tile<DH>(p, sg, pos_last, j0, tid, v_ring + vt.slot * C::KT, v16 + wt.slot * C::V16,
                                         s_info + (TCA_INFO + (tile & (TCA_INFO - 1))) * TCA_PAGES, s_nan, s_flag);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(v_empty + 8 * vt.slot);
                        mbar_arrive(w_full + 8 * wt.slot);
                    }
                    vt.next();
                    wt.next();
                    if (i == 0 && si + 1 < nseg) queries(si + 1);
                }
                // ---- the span's result: this thread's row is tid
                const bool whole = sg.c0 == sg.c1, mine = tid < sg.rows;
                wait(l_full + 8 * lt.slot, lt.phase);
                const float* const lp = s_l + 2 * lt.slot * R + tid;
                const float* const mp = s_mo + 2 * lt.slot * R + tid;
                const float M = fmaxf(mp[0], mp[R]), L = fmaf(lp[0], ex2(mp[0] - M), lp[R] * ex2(mp[R] - M));
                const float inv = !whole ? 1.f : L == 0.f ? 0.f : 1.0f / L;
                const int tok = div_rep(p, sg.rem + tid);
                const long long part_row = (long long)(2 * blockIdx.x + ((int)blockIdx.x == sg.c0 ? 1 : 0)) * R + tid;
                const long long off = whole ? (long long)(sg.tok + tok) * p.out_stride + (long long)(sg.g * rep + sg.rem + tid - tok * rep) * DH
                                            : part_row * DH;
                if (!whole && mine && !dead) __stcg(p.ws_ml + part_row, make_float2(L == 0.f ? A8_LOWEST : M, L));
                v_bar();
                const bool nans = *s_flag != 0;
                wait(o_full, ot.phase);
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < DH; c += 16) {
                    uint32_t x[16];
                    tmem_ld<16>(col_o + lanes + (uint32_t)c, x);
                    tmem_wait_ld();
                    settle(x);
                    if (mine && !dead) {
                        const uint32_t bad = nans ? s_nan[tid * (DH / 32) + (c >> 5)] >> (c & 31) : 0u;
                        float v[16];
#pragma unroll
                        for (int z = 0; z < 16; ++z) v[z] = bad >> z & 1 ? __int_as_float(0x7fffffff) : __uint_as_float(x[z]) * inv;
                        if (whole) {
#pragma unroll
                            for (int z = 0; z < 16; z += 4)
                                store4(reinterpret_cast<__nv_bfloat16*>(p.out) + off + c + z, v[z], v[z + 1], v[z + 2], v[z + 3]);
                        } else {
#pragma unroll
                            for (int z = 0; z < 16; z += 4)
                                __stcg(reinterpret_cast<float4*>(p.ws_o + off + c + z), make_float4(v[z], v[z + 1], v[z + 2], v[z + 3]));
                        }
                    }
                    __syncwarp();
                }
                tc_fence_before();
                v_bar();  // (a cut span's part is written; the NaN notes have been read)
                if (nans) {
                    for (int z = tid; z < R * (DH / 32); z += 128) s_nan[z] = 0;
                    if (tid == 0) *s_flag = 0;
                    v_bar();
                }
                if (lane == 0) {
                    mbar_arrive(o_empty);
                    mbar_arrive(l_empty + 8 * lt.slot);
                }
                ot.next();
                lt.next();
                if (!whole && tid == 0) a8_arrive(p, sg, s_last, s_cut);
            }
        } else if (warp == 12) {
            copy_tiles<DH, false, NK>(p, map, segs, nseg, lane, k_ring, k_full, k_empty, s_info, kt, tile, wait, dead);
        } else if (warp == 13) {
            copy_tiles<DH, true, NV>(p, map, segs, nseg, lane, v_ring, v_full, v_empty, s_info + TCA_INFO * TCA_PAGES, vt, tile, wait, dead);
        } else if (warp == 14) {
            // ---------------- MMA: the warp waits together, one elected lane issues ----------------
            // f32 accumulators; S: Q (e4m3, then e5m2: bit 7) and K (e4m3); O: f16 both, B (V) with its outer side contiguous
            constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(TCA_TILE >> 3) << 17) | ((uint32_t)(R >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(DH >> 3) << 17) | ((uint32_t)(R >> 4) << 24);
            constexpr uint32_t hi_s = desc_hi(8 * C::ROWB, DH == 64 ? 4 : 2), hi_v = desc_hi(1024, 2);
            // O of a tile comes after S of the second tile behind it: the scores' room is free a little before the
            // weights are there.  What is still to come: tiles that begin or end their span, the older in bit 1
            int pending = 0;
            unsigned begin_bits = 0, end_bits = 0;
            const auto values = [&]() {
                const bool begins = begin_bits >> (pending - 1) & 1, ends = end_bits >> (pending - 1) & 1;
                if (begins) wait(o_empty, ot.phase ^ 1);
                wait2(p_full + 8 * pt.slot, pt.phase, w_full + 8 * wt.slot, wt.phase);
                tc_fence_after();
                if (!dead && elected()) {
                    const uint32_t va = desc_lo(smem_u32(v16 + wt.slot * C::V16), DH == 64 ? 0 : 16384);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks)
                        mma_tc_ta(col_o, col_p(pt.slot) + (uint32_t)(8 * ks), va + (uint32_t)(ks * 128), hi_v, idesc_o, begins && ks == 0 ? 0u : 1u);
                    tc_commit(p_empty + 8 * pt.slot);
                    tc_commit(w_empty + 8 * wt.slot);
                    if (ends) tc_commit(o_full);
                }
                __syncwarp();
                pt.next();
                wt.next();
                if (ends) ot.next();
                --pending;
            };
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const int n = segs[si].n;
                // (queries come from the V warps too, which first write the results before them: nothing may wait here for those)
                if (!__all_sync(0xffffffffu, mbar_test(q_full + 8 * qt.slot, (uint32_t)qt.phase)))
                    while (pending > 0) values();
                wait(q_full + 8 * qt.slot, qt.phase);
#pragma unroll 1
                for (int i = 0; i < n; ++i) {
                    wait2(k_full + 8 * kt.slot, kt.phase, s_empty + 8 * st.slot, st.phase ^ 1);
                    tc_fence_after();
                    if (!dead && elected()) {
                        const uint32_t ka = desc_lo(smem_u32(k_ring + kt.slot * C::KT)), qa = desc_lo(smem_u32(s_q + qt.slot * C::QB));
#pragma unroll
                        for (int ks = 0; ks < DH / 32; ++ks)
#pragma unroll
                            for (int z = 0; z < 2; ++z)
                                mma_tc<true>(col_s(st.slot), qa + (uint32_t)((z * R * C::ROWB) / 16 + ks * 2), hi_s,
                                             ka + (uint32_t)(ks * 2), hi_s, idesc_s | (uint32_t)z << 7, ks + z == 0 ? 0u : 1u);
                        tc_commit(s_full + 8 * st.slot);
                        tc_commit(k_empty + 8 * kt.slot);
                        if (i == n - 1) tc_commit(q_empty + 8 * qt.slot);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_full + 8 * st.slot);  // (passes on what this warp has seen: page words, factors)
                    kt.next();
                    st.next();
                    if (pending == 2) values();
                    ++pending;
                    begin_bits = begin_bits << 1 | (i == 0 ? 1u : 0u);
                    end_bits = end_bits << 1 | (i == n - 1 ? 1u : 0u);
                }
                qt.next();
            }
            while (pending > 0) values();
        } else {
            // ---------------- queries: two terms of each row ----------------
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const bool shared = shared_queries(si);
                convert_queries<DH, R, true>(p, segs[si], rep, lane, shared ? 4 : 0, shared ? 5 : 1, s_q + qt.slot * C::QB, s_rf + qt.slot * R,
                                             [&] { wait(q_empty + 8 * qt.slot, qt.phase ^ 1); return !dead; });
                fence_proxy_async_smem();
                if (shared) queries_bar();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full + 8 * qt.slot);
                qt.next();
            }
        }
    }
    // every copy asked for has landed before the CTA ends (its readers waited for it, unless they gave up)
    if (dead && (warp == 12 || warp == 13) && lane == 0)
        for (int i = 0; i < (warp == 12 ? NK : NV); ++i)
            for (int ph = 0; ph < 2; ++ph)
                (void)mbar_wait_bounded_ns((warp == 12 ? k_full : v_full) + 8 * i, (uint32_t)ph, 100000000ull);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 14) tmem_dealloc(tmem, C::TMEM);
    a8_join<__nv_bfloat16, DH, TCR_THREADS>(p, R, rep, s_last, s_cut);
}

template <int DH>
static yk_status launch_tcr(cudaStream_t st, bool pdl, int num_sms, const CUtensorMap& map, const Attn8Params& p) {
    using C = TcrCfg<DH>;
    int dev = 0;
    YK_CHECK_CUDA(cudaGetDevice(&dev));
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {
        YK_CHECK_CUDA(cudaFuncSetAttribute(attn8_rows_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        ready.fetch_or(bit, std::memory_order_release);
    }
    YK_CHECK_CUDA(launch_on(st, pdl, attn8_rows_kernel<DH>, num_sms, TCR_THREADS, C::SMEM, map, p));
    return YK_OK;
}

yk_status attention_e4m3_launch_rows(cudaStream_t st, bool pdl, int num_sms, int head_dim, const CUtensorMap& map, const Attn8Params& p) {
    return head_dim == 64 ? launch_tcr<64>(st, pdl, num_sms, map, p) : launch_tcr<128>(st, pdl, num_sms, map, p);
}

}  // namespace yk
