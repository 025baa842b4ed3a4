// yk_attention_e4m3_tc.cu -- yk_attention_e4m3 for bf16 queries, on the
// tcgen05 tensor cores.
//
// One CTA per SM, resident; each takes an equal range of 128-key tiles of the
// spans (sequence, query tile, KV head) laid end to end, found from the lengths
// on the device.  Its warps are a pipeline:
//   producers  one warp for K, one for V (a warp issues a copy in about 85 cycles,
//              whatever its size): table entries and scale bytes; K pages by TMA
//              (128- or 64-byte swizzle), V pages by bulk copy, into rings of tiles
//   queries    the next span's queries into pairs of 8-bit terms
//   MMA        S^T[128 keys x 2R] = K Q^T (kind::f8f6f4), O^T[dims x R] += V^T P^T
//              (kind::f16), accumulators in TMEM, S^T and O^T double-buffered
//   softmax    two groups of 4 warps, half of the rows each, one key a thread: scores
//              from TMEM, weights to shared memory
//   V          4 warps: e4m3 V to f16, still [key][dim] (the MN-major operand of
//              O^T); at a span's end they read O^T and write the result
// K goes to the tensor core as it lies in the cache: no conversion at all.  The
// queries, as bf16, are 8 bits wide: two terms hold them exactly (to 2^-21 of a
// row's largest value at least).  For few rows both are e4m3, the second scaled by
// 16, as separate columns of one product; from 24 rows on the second is e5m2 (the
// remainder is at most 8 units of the last bit, 3 bits wide) and its product adds
// to the first's: half the scores to read back (64 rows: 835 -> 813 us).  V
// converts once for all rows of the tile (R up to 48).
//
// Weights as in the other kernel: p = 2^(x + e_V - m), f16.  The reference m of a
// row is kept by its group, lazily: it is set 2^3 below a row's first weights
// and moves when one would pass 2^15 (each move waits for the products before it
// and rescales O^T in TMEM).  What lies 2^-28 below a row's largest weight is
// lost: f16 ends at 2^-25, rounded.
//
// Measured, 32 query and 8 KV heads of 128: one token over 131,000 keys 57 us (268
// MB, 4.7 TB/s: 72 % of a copy's rate); 64 sequences of 2k-8k keys, 5 tokens, 16
// heads of 256, capped, 280 us (73 %); 32 sequences of 512-2048 keys, 6 tokens, 41
// us (88 MB, 33 %).  Long ranges run at 1800 cycles a tile where the bytes alone
// need 1400; a tile's fixed cost bounds them (every role is busy for 1100-1500
// cycles of barriers, fences and conversions).  Short ranges pay for their start
// besides: plan 2 us, first scores another 4 us, and a span's end and beginning
// cost as much as two tiles (TCA_COST).
#include <algorithm>
#include <atomic>
#include <cmath>
#include <string>

#include "yk_attention_e4m3_tc.cuh"

namespace yk {

constexpr int TCA_THREADS = 512;  // warps 0-7 softmax, 8-11 V, 12 K and 13 V copies, 14 MMA, 15 queries

template <int DH, int RN>
struct TcaCfg {
    static constexpr int R = 8 * RN, RP = R <= 16 ? 16 : R <= 32 ? 32 : 64;  // rows; columns of O^T
    static constexpr int RH = R / 2;                           // rows of a softmax thread
    static constexpr int ROWB = DH == 64 ? 64 : 128;           // bytes of a K row in one TMA box
    static constexpr int BOXES = DH / ROWB;
    static constexpr int HALVES = DH == 256 ? 2 : 1;           // 128-dim products of O^T
    static constexpr int KT = TCA_TILE * DH;                   // bytes of a K (or V) tile
    static constexpr int NV16 = DH == 256 ? 1 : 2, V16 = 2 * KT;
    static constexpr int PROW = 2 * RP;                        // bytes of a key's weights
    static constexpr int PB = PROW * TCA_TILE, QB = 2 * R * DH;
    static constexpr int LDL = 33;
    static constexpr int SMALL = 8 * 4 * LDL * 4 + (2 + 1 + 1 + 1 + 1 + 4 + 8 + 2 + 1 + 3) * R * 4 + R * (DH / 32) * 4 +
                                 2 * TCA_INFO * TCA_PAGES * 4 + (A8_SEGS + 2) * (int)sizeof(Seg) + A8_SCAN * 4 + 64 * 8 + 128;
    static constexpr int ROOM = 227 * 1024 - 1024 - SMALL - NV16 * V16 - 2 * PB - 2 * QB;
    static constexpr int TILES = ROOM / KT;                    // K and V tiles that fit
    static constexpr int NV = TILES / 2 < 6 ? TILES / 2 : 6, NK = TILES - NV < 6 ? TILES - NV : 6;
    static constexpr int SMEM = 1024 + (NK + NV) * KT + NV16 * V16 + 2 * PB + 2 * QB + SMALL;
    static constexpr bool JOINED = R >= 24;                    // the queries' second terms: a product of their own
    static constexpr int S_COLS = JOINED ? (R + 15) / 16 * 16 : 2 * R, O_COLS = HALVES * RP;
    static constexpr int COLS = 2 * S_COLS + 2 * O_COLS;
    static constexpr int TMEM = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static_assert(NK >= 2 && NV >= 1 && COLS <= 512, "tile shapes");
};

// Barriers of the 4 warps of a softmax group (true if any thread says so).
__device__ __forceinline__ bool softmax_or(int group, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(3 + group), "r"((uint32_t)v)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void softmax_bar(int group) { asm volatile("bar.sync %0, 128;" ::"r"(3 + group) : "memory"); }
__device__ __forceinline__ float warp_fmax(float v) {  // (NaN is passed over)
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
template <int DH, int RN>
__global__ void __launch_bounds__(TCA_THREADS, 1) attn8_tc_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ Attn8Params p) {
    using C = TcaCfg<DH, RN>;
    constexpr int R = C::R, RP = C::RP, NK = C::NK, NV = C::NV, NV16 = C::NV16;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const k_ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const v_ring = k_ring + NK * C::KT;
    uint8_t* const v16 = v_ring + NV * C::KT;
    uint8_t* const s_p = v16 + NV16 * C::V16;
    uint8_t* const s_q = s_p + 2 * C::PB;
    float* const s_lt = reinterpret_cast<float*>(s_q + 2 * C::QB);  // [8 warps][4][LDL]
    float* const s_rf = s_lt + 8 * 4 * C::LDL;                      // [2][R] score factors of a span's rows
    float* const s_neg = s_rf + 2 * R;                              // [R] references, negated
    int* const s_set = reinterpret_cast<int*>(s_neg + R);             // [R] a row has seen a key
    float* const s_f = reinterpret_cast<float*>(s_set + R);         // [R] factor and ...
    float* const s_dm = s_f + R;                                    // [R] ... step of a row's last move
    float* const s_mx = s_dm + R;                                   // [4][R]
    float* const s_l = s_mx + 4 * R;                                // [2][4][R] sums
    float* const s_mo = s_l + 8 * R;                                // [2][R] references at a span's end
    int* const s_pos = reinterpret_cast<int*>(s_mo + 2 * R);        // [R] positions, for the softmax warps
    float* const s_inv = reinterpret_cast<float*>(s_pos + R);       // [R] 1 / sum and ...
    long long* const s_off = reinterpret_cast<long long*>(s_inv + R);       // [R] ... place of a result row
    uint32_t* const s_nan = reinterpret_cast<uint32_t*>(s_off + R);         // [R][DH / 32]
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
    // barriers
    const uint32_t b0 = smem_u32(bars);
    const uint32_t k_full = b0, k_empty = k_full + 8 * NK, v_full = k_empty + 8 * NK, v_empty = v_full + 8 * NV;
    const uint32_t s_full = v_empty + 8 * NV, s_empty = s_full + 16, p_full = s_empty + 16, p_empty = p_full + 16;
    const uint32_t w_full = p_empty + 16, w_empty = w_full + 8 * NV16;  // f16 V
    const uint32_t q_full = w_empty + 8 * NV16, q_empty = q_full + 16, o_full = q_empty + 16, o_empty = o_full + 16;
    const uint32_t l_full = o_empty + 16, l_empty = l_full + 16;
    static_assert(2 * NK + 2 * NV + 2 * NV16 + 18 <= 64, "barriers");
    if (threadIdx.x == 480) {  // (not of the warps that plan first)
        const auto init = [](uint32_t bar, int n, int count) {
            for (int i = 0; i < n; ++i) mbar_init(bar + 8 * i, (uint32_t)count);
        };
        init(k_full, NK, 1);
        init(k_empty, NK, 1);
        init(v_full, NV, 1);
        init(v_empty, NV, 4);
        init(s_full, 2, 2);   // the products, and the MMA thread itself (it passes on what it has seen)
        init(s_empty, 2, 8);
        init(p_full, 2, 8);
        init(p_empty, 2, 1);
        init(w_full, NV16, 4);
        init(w_empty, NV16, 1);
        init(q_full, 2, 1);
        init(q_empty, 2, 9);  // the products, and the softmax warps (score factors)
        init(o_full, 2, 1);
        init(o_empty, 2, 4);
        init(l_full, 2, 8);
        init(l_empty, 2, 4);
        mbar_fence_init();
        *s_flag = s_last[0] = s_last[1] = 0;
    }
    for (int i = threadIdx.x; i < R * (DH / 32); i += TCA_THREADS) s_nan[i] = 0;
    pdl_wait();
    A8Work work;
    if (warp == 14) tmem_alloc(smem_u32(s_tmem), C::TMEM);
    const bool busy = a8_plan<TCA_THREADS, TCA_PAGES, TCA_COST, 1>(p, R, rep, s_scan, work);  // (block-uniform)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *s_tmem;
    if (!busy) {
        if (warp == 14) tmem_dealloc(tmem, C::TMEM);
        return;
    }
    pdl_trigger();  // (after the TMEM is taken: a kernel that starts early does not take it first)
    const auto col_s = [&](int b) { return tmem + (uint32_t)(b * C::S_COLS); };
    const auto col_o = [&](int b) { return tmem + (uint32_t)(2 * C::S_COLS + b * C::O_COLS); };

    // per role, through all rounds
    bool dead = false;  // a bounded wait ran out: the role goes through the motions without touching memory
    const auto wait = [&](uint32_t bar, int parity) {
        if (!dead && !mbar_test(bar, (uint32_t)parity)) dead = !wait_longer(bar, (uint32_t)parity, p.err);
    };
    // two at once: the first looks at both go out together (one that finds its barrier ready takes ~100 cycles)
    const auto wait2 = [&](uint32_t bar_a, int parity_a, uint32_t bar_b, int parity_b) {
        const bool a = mbar_test(bar_a, (uint32_t)parity_a), b = mbar_test(bar_b, (uint32_t)parity_b);
        if (!dead && !a) dead = !wait_longer(bar_a, (uint32_t)parity_a, p.err);
        if (!dead && !b) dead = !wait_longer(bar_b, (uint32_t)parity_b, p.err);
    };
    Turn<NK> kt;
    Turn<NV> vt;
    Turn<2> st, pt, qt, ot;
    Turn<NV16> wt;
    int tile = 0;           // of this CTA (page words)

    for (int seg0 = 0; seg0 < work.nspans; seg0 += A8_SEGS) {
        __syncwarp();
        __syncthreads();
        a8_list<TCA_PAGES, TCA_COST>(p, R, rep, work, seg0, segs);
        __syncthreads();
        const int nseg = min(A8_SEGS, work.nspans - seg0);
        if (warp < 8) {
            // ---------------- softmax: key 32 * quad + lane of each tile, rows r0 .. r0 + RH - 1 ----------------
            constexpr int RH = C::RH, BATCH = RH % 16 == 0 ? 16 : RH > 16 ? 8 : RH;  // rows read from TMEM at a time
            const int quad = warp & 3, group = warp >> 2, r0 = group * RH, key = 32 * quad + lane;
            const int own = key < RH ? r0 + key : -1;  // a row whose reference this thread keeps
            const uint32_t lanes = (uint32_t)(32 * quad) << 16;
            // this key's weights in P, [key][row], 16-byte chunks swizzled by the key
            const uint32_t p_sw = (uint32_t)(C::PROW == 128 ? key & 7 : C::PROW == 64 ? key >> 1 & 3 : key >> 2 & 1) << 4;
            const uint32_t p_at = smem_u32(s_p) + (uint32_t)(key * C::PROW);
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const Seg sg = segs[si];
                const int rows = sg.rows, pos_last = sg.pos + div_rep(p, sg.rem + rows - 1);
                if (own >= 0) {
                    const int n = own;
                    s_neg[n] = 0.f;
                    s_set[n] = 0;
                    s_pos[n] = n < rows ? sg.pos + div_rep(p, sg.rem + n) : -0x40000000;  // (no key is seen)
                }
                softmax_bar(group);
                const unsigned w = p.window > 0 ? (unsigned)p.window : 0x80000000u;
                bool force = true;  // some row has not seen a key yet
                float2 l[RH / 2];
#pragma unroll
                for (int n = 0; n < RH / 2; ++n) l[n] = make_float2(0.f, 0.f);
#pragma unroll 1
                for (int i = 0; i < sg.n; ++i, ++tile) {
                    const int j0 = (sg.page + TCA_PAGES * i) * 16;
                    wait(s_full + 8 * st.slot, st.phase);
                    tc_fence_after();
                    const bool p_free = mbar_test(p_empty + 8 * pt.slot, (uint32_t)(pt.phase ^ 1));
                    const int info = s_info[(tile & (TCA_INFO - 1)) * TCA_PAGES + 2 * quad + (lane >> 4)];
                    const bool here = info >= 0;
                    const int ek = here ? (info & 255) - 128 : 0, ev = here ? (info >> 8) - 128 : 0;
                    const float fk = exp2_int(ek), inv = exp2_int(-ev);
                    const float2 fk2 = make_float2(fk, fk), shift = make_float2((float)ev, (float)ev), inv2 = make_float2(inv, inv);
                    // (soft-capped scores are capped, then shifted, below)
                    const float2 now = p.cap <= 0.f ? make_float2(1.f, 1.f) : make_float2(0.f, 0.f), first = mul2(shift, now);
                    const bool plain = p.cap <= 0.f && all_seen(p, sg, pos_last, j0) && __all_sync(0xffffffffu, here);
                    const float* const rf = s_rf + qt.slot * R + r0;
                    const uint32_t at = col_s(st.slot) + lanes + (uint32_t)r0;
                    float2 d[RH / 2];  // score + e_V - reference, rows r0 + 2 n, + 1
#pragma unroll
                    for (int b0 = 0; b0 < RH; b0 += BATCH) {
                        uint32_t x[BATCH], y[C::JOINED ? 1 : BATCH];
                        tmem_ld<BATCH>(at + (uint32_t)b0, x);
                        if constexpr (!C::JOINED) tmem_ld<BATCH>(at + (uint32_t)(R + b0), y);
                        // (these come while the scores do; a score is rounded before its reference, which was taken from a rounded
                        // one, is taken off: where fp32 holds scores to whole numbers the difference counts)
                        float4 f[BATCH / 4], m[BATCH / 4];
#pragma unroll
                        for (int n = 0; n < BATCH / 4; ++n) {
                            f[n] = *reinterpret_cast<const float4*>(rf + b0 + 4 * n);
                            m[n] = *reinterpret_cast<const float4*>(s_neg + r0 + b0 + 4 * n);
                        }
                        tmem_wait_ld();
#pragma unroll
                        for (int n = 0; n < BATCH; n += 2) {
                            const float4 ff = f[n / 4], mm = m[n / 4];
                            float2 s = make_float2(__uint_as_float(x[n]), __uint_as_float(x[n + 1]));
                            if constexpr (!C::JOINED)
                                s = fma2(make_float2(__uint_as_float(y[n]), __uint_as_float(y[n + 1])), make_float2(0.0625f, 0.0625f), s);
                            const float2 r = n & 2 ? make_float2(ff.z, ff.w) : make_float2(ff.x, ff.y);
                            d[(b0 + n) / 2] = fma2(n & 2 ? make_float2(mm.z, mm.w) : make_float2(mm.x, mm.y), now, fma2(mul2(s, fk2), r, first));
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_empty + 8 * st.slot);
                    st.next();
                    if (p.cap > 0.f) {
#pragma unroll
                        for (int n = 0; n < RH; n += 2) {
                            const float2 m = *reinterpret_cast<const float2*>(s_neg + r0 + n);
                            d[n / 2] = add2(add2(make_float2(cap_score(p, d[n / 2].x), cap_score(p, d[n / 2].y)), shift), m);
                        }
                    }
                    if (!plain) {
                        const int kj = j0 + key;
                        const unsigned wk = here ? w : 0u;
#pragma unroll
                        for (int n = 0; n < RH; n += 4) {
                            const int4 q = *reinterpret_cast<const int4*>(s_pos + r0 + n);
                            float2 &a = d[n / 2], &b = d[n / 2 + 1];
                            a.x = (unsigned)(q.x - kj) < wk ? a.x : -INFINITY;
                            a.y = (unsigned)(q.y - kj) < wk ? a.y : -INFINITY;
                            b.x = (unsigned)(q.z - kj) < wk ? b.x : -INFINITY;
                            b.y = (unsigned)(q.w - kj) < wk ? b.y : -INFINITY;
                        }
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int n = 0; n < RH / 2; ++n) top = fmaxf(top, fmaxf(d[n].x, d[n].y));
                    // move the references: at a row's first keys, and before a weight would pass 2^15
                    if (softmax_or(group, force || top > 15.f)) {
                        float most = 0.f;  // lane n: the warp's largest of row r0 + n
#pragma unroll
                        for (int n = 0; n < RH; ++n) {
                            const float x = warp_fmax(n & 1 ? d[n / 2].y : d[n / 2].x);
                            most = lane == n ? x : most;
                        }
                        if (lane < RH) s_mx[quad * R + r0 + lane] = most;
                        softmax_bar(group);
                        bool unset = false;
                        if (own >= 0) {
                            const int n = own;
                            const float x = fmaxf(fmaxf(s_mx[n], s_mx[R + n]), fmaxf(s_mx[2 * R + n], s_mx[3 * R + n]));
                            const float was = -s_neg[n];
                            const bool set = s_set[n] != 0;
                            const float now = x == -INFINITY ? was : set ? fmaxf(was, was + (x - 3.f)) : was + (x - 3.f);
                            s_f[n] = set ? ex2(was - now) : 1.f;
                            s_dm[n] = was - now;
                            s_neg[n] = -now;
                            if (x > -INFINITY) s_set[n] = 1;
                            unset = n < rows && !set && x == -INFINITY;
                        }
                        force = softmax_or(group, unset);
#pragma unroll
                        for (int n = 0; n < RH; n += 4) {
                            const float4 a = *reinterpret_cast<const float4*>(s_dm + r0 + n), f = *reinterpret_cast<const float4*>(s_f + r0 + n);
                            d[n / 2] = add2(d[n / 2], make_float2(a.x, a.y));
                            d[n / 2 + 1] = add2(d[n / 2 + 1], make_float2(a.z, a.w));
                            l[n / 2] = mul2(l[n / 2], make_float2(f.x, f.y));
                            l[n / 2 + 1] = mul2(l[n / 2 + 1], make_float2(f.z, f.w));
                        }
                        if (i > 0) {
                            // O^T follows, once the products of the tile before are done
                            wait(p_empty + 8 * (pt.slot ^ 1), pt.slot ? pt.phase : pt.phase ^ 1);
                            tc_fence_after();
#pragma unroll 1
                            for (int half = 0; half < C::HALVES; ++half) {
                                const uint32_t o_at = col_o(ot.slot) + lanes + (uint32_t)(half * RP + r0);
#pragma unroll 1
                                for (int n = 0; n < RH; n += BATCH) {
                                    uint32_t x[BATCH];
                                    tmem_ld<BATCH>(o_at + (uint32_t)n, x);
                                    tmem_wait_ld();
#pragma unroll
                                    for (int z = 0; z < BATCH; ++z) x[z] = __float_as_uint(__uint_as_float(x[z]) * s_f[r0 + n + z]);
                                    tmem_st<BATCH>(o_at + (uint32_t)n, x);
                                }
                            }
                            tmem_wait_st();
                            tc_fence_before();
                        }
                    }
                    // weights
                    if (!p_free) wait(p_empty + 8 * pt.slot, pt.phase ^ 1);
                    const uint32_t pa = p_at + (uint32_t)(pt.slot * C::PB);
                    if (!dead) {
                        constexpr int PER = RH % 8 == 0 ? 8 : 4;  // rows a store
#pragma unroll
                        for (int n = 0; n < RH; n += PER) {
                            uint32_t h[PER / 2];
#pragma unroll
                            for (int z = 0; z < PER / 2; ++z) {
                                const float2 x = make_float2(ex2(d[n / 2 + z].x), ex2(d[n / 2 + z].y));
                                l[n / 2 + z] = fma2(x, inv2, l[n / 2 + z]);
                                h[z] = f16x2_of(x.x, x.y);
                            }
                            const uint32_t at_row = (uint32_t)(r0 + n) * 2;
                            const uint32_t a = pa + ((at_row & ~15u) ^ p_sw) + (at_row & 8u);
                            if constexpr (PER == 8) sts128(a, h[0], h[1], h[2], h[3]);
                            else sts64(a, h[0], h[1]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full + 8 * pt.slot);
                    pt.next();
                }
                // the span's sums over the warp's keys, and its references, for the warps that write the result
                wait(l_empty + 8 * ot.slot, ot.phase ^ 1);
                float* const lt = s_lt + warp * 4 * C::LDL;
#pragma unroll
                for (int n = 0; n < RH; n += 4) {
#pragma unroll
                    for (int z = 0; z < 4; ++z) lt[z * C::LDL + lane] = z & 1 ? l[(n + z) / 2].y : l[(n + z) / 2].x;
                    __syncwarp();
                    const float* const at = lt + (lane >> 3) * C::LDL + (lane & 7) * 4;
                    float x = (at[0] + at[1]) + (at[2] + at[3]);
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    if ((lane & 7) == 0) s_l[(ot.slot * 4 + quad) * R + r0 + n + (lane >> 3)] = x;
                    __syncwarp();
                }
                if (own >= 0) s_mo[ot.slot * R + own] = -s_neg[own];
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(l_full + 8 * ot.slot);
                    mbar_arrive(q_empty + 8 * qt.slot);
                }
                qt.next();
                ot.next();
                softmax_bar(group);  // (s_neg has been read)
            }
        } else if (warp < 12) {
            // ---------------- V: e4m3 -> f16, and the results ----------------
            const int tid = threadIdx.x - 256, quad = warp & 3;
            const uint32_t lanes = (uint32_t)(32 * quad) << 16;
            if (seg0 == 0 && RN > 1) {
                convert_queries<DH, R, C::JOINED>(p, segs[0], rep, lane, quad, 5, s_q, s_rf, [] { return true; });
                fence_proxy_async_smem();
                queries_bar();
            }
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const Seg sg = segs[si];
                const int rows = sg.rows, pos_last = sg.pos + div_rep(p, sg.rem + rows - 1);
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
                }
                // ---- the span's result: this thread's dim is 32 * quad + lane of each half
                const bool whole = sg.c0 == sg.c1;
                wait(l_full + 8 * ot.slot, ot.phase);
                if (tid < rows) {
                    const float* const lp = s_l + ot.slot * 4 * R + tid;
                    const float L = (lp[0] + lp[R]) + (lp[2 * R] + lp[3 * R]);
                    const long long part_row = (long long)(2 * blockIdx.x + ((int)blockIdx.x == sg.c0 ? 1 : 0)) * R + tid;
                    const int tok = div_rep(p, sg.rem + tid);
                    s_inv[tid] = !whole ? 1.f : L == 0.f ? 0.f : 1.0f / L;
                    s_off[tid] = whole ? (long long)(sg.tok + tok) * p.out_stride + (long long)(sg.g * rep + sg.rem + tid - tok * rep) * DH
                                       : part_row * DH;
                    if (!whole) __stcg(p.ws_ml + part_row, make_float2(L == 0.f ? A8_LOWEST : s_mo[ot.slot * R + tid], L));
                }
                v_bar();
                const bool nans = *s_flag != 0;
                wait(o_full + 8 * ot.slot, ot.phase);
                tc_fence_after();
#pragma unroll 1
                for (int half = 0; half < C::HALVES; ++half) {
                    const int dim = half * 128 + 32 * quad + lane;
#pragma unroll 1
                    for (int n0 = 0; n0 < rows; n0 += 8) {
                        uint32_t x[8];
                        tmem_ld<8>(col_o(ot.slot) + lanes + (uint32_t)(half * RP + n0), x);
                        tmem_wait_ld();
                        if (dim >= DH || dead) continue;
#pragma unroll
                        for (int z = 0; z < 8; ++z) {
                            if (n0 + z < rows) {
                                float v = __uint_as_float(x[z]) * s_inv[n0 + z];
                                if (nans && (s_nan[(n0 + z) * (DH / 32) + (dim >> 5)] >> (dim & 31) & 1)) v = __int_as_float(0x7fffffff);
                                if (whole) reinterpret_cast<__nv_bfloat16*>(p.out)[s_off[n0 + z] + dim] = __float2bfloat16_rn(v);
                                else __stcg(p.ws_o + s_off[n0 + z] + dim, v);
                            }
                        }
                    }
                }
                tc_fence_before();
                v_bar();  // (a cut span's part is written; s_inv, s_off and the NaN notes have been read)
                if (nans) {
                    for (int z = tid; z < R * (DH / 32); z += 128) s_nan[z] = 0;
                    if (tid == 0) *s_flag = 0;
                    v_bar();
                }
                if (lane == 0) {
                    mbar_arrive(o_empty + 8 * ot.slot);
                    mbar_arrive(l_empty + 8 * ot.slot);
                }
                ot.next();
                if (!whole && tid == 0) a8_arrive(p, sg, s_last, s_cut);
            }
        } else if (warp < 14) {
            // ---------------- copies: K (warp 12) and V (warp 13) ----------------
            if (warp == 12)
                copy_tiles<DH, false, NK>(p, map, segs, nseg, lane, k_ring, k_full, k_empty, s_info, kt, tile, wait, dead);
            else
                copy_tiles<DH, true, NV>(p, map, segs, nseg, lane, v_ring, v_full, v_empty, s_info + TCA_INFO * TCA_PAGES, vt, tile, wait, dead);
        } else if (warp == 14) {
            // ---------------- MMA: the warp waits together, one elected lane issues ----------------
            // (a branch on the lane number instead makes the twelve products of a tile take 740 cycles to issue, not 470)
            // f32 accumulators; S^T: e4m3 both; O^T: f16 both, A (V) and B (weights) with their outer side contiguous
            constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(C::S_COLS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | (1u << 15) | (1u << 16) | ((uint32_t)(RP >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
            constexpr uint32_t hi_s = desc_hi(8 * C::ROWB, DH == 64 ? 4 : 2), hi_v = desc_hi(1024, 2);
            constexpr uint32_t hi_p = desc_hi(8 * C::PROW, C::PROW == 128 ? 2 : C::PROW == 64 ? 4 : 6);
            constexpr uint32_t v_lbo = DH == 64 ? 0 : 16384;  // (64 dims: the product's other 64 rows repeat them)
            // O^T of the tile before: whether it is still to come, and begins or ends its span
            bool pending = false, begins = false, ends = false;
            const auto values = [&]() {
                if (begins) wait(o_empty + 8 * ot.slot, ot.phase ^ 1);
                wait2(p_full + 8 * pt.slot, pt.phase, w_full + 8 * wt.slot, wt.phase);
                tc_fence_after();
                if (!dead && elected()) {
                    const uint32_t va = desc_lo(smem_u32(v16 + wt.slot * C::V16), v_lbo), pa = desc_lo(smem_u32(s_p + pt.slot * C::PB));
                    const uint32_t d = col_o(ot.slot);
#pragma unroll
                    for (int half = 0; half < C::HALVES; ++half)
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            mma_tc<false>(d + (uint32_t)(half * RP), va + (uint32_t)(half * 2048 + ks * 128), hi_v,
                                          pa + (uint32_t)(ks * C::PROW), hi_p, idesc_o, begins && ks == 0 ? 0u : 1u);
                    tc_commit(p_empty + 8 * pt.slot);
                    tc_commit(w_empty + 8 * wt.slot);
                    if (ends) tc_commit(o_full + 8 * ot.slot);
                }
                __syncwarp();
                pt.next();
                wt.next();
                if (ends) ot.next();
                pending = false;
            };
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const int n = segs[si].n;
                wait(q_full + 8 * qt.slot, qt.phase);
#pragma unroll 1
                for (int i = 0; i < n; ++i) {
                    wait2(k_full + 8 * kt.slot, kt.phase, s_empty + 8 * st.slot, st.phase ^ 1);
                    tc_fence_after();
                    if (!dead && elected()) {
                        const uint32_t ka = desc_lo(smem_u32(k_ring + kt.slot * C::KT)), qa = desc_lo(smem_u32(s_q + qt.slot * C::QB));
                        const uint32_t d = col_s(st.slot);
#pragma unroll
                        for (int ks = 0; ks < DH / 32; ++ks)
#pragma unroll
                            for (int t = 0; t < (C::JOINED ? 2 : 1); ++t)  // (bit 10: B is e5m2)
                                mma_tc<true>(d, ka + (uint32_t)((ks >> 2) * (TCA_TILE * 8) + (ks & 3) * 2), hi_s,
                                             qa + (uint32_t)((ks >> 2) * (2 * R * 8) + t * (R * C::ROWB / 16) + (ks & 3) * 2), hi_s,
                                             idesc_s | (uint32_t)t << 10, ks + t == 0 ? 0u : 1u);
                        tc_commit(s_full + 8 * st.slot);
                        tc_commit(k_empty + 8 * kt.slot);
                        if (i == n - 1) tc_commit(q_empty + 8 * qt.slot);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_full + 8 * st.slot);  // (passes on what this warp has seen: page words, factors)
                    kt.next();
                    st.next();
                    if (pending) values();
                    pending = true;
                    begins = i == 0;
                    ends = i == n - 1;
                }
                qt.next();
            }
            if (pending) values();
        } else {
            // ---------------- queries: two terms of each row ----------------
#pragma unroll 1
            for (int si = 0; si < nseg; ++si) {
                const bool first = RN > 1 && seg0 + si == 0;
                convert_queries<DH, R, C::JOINED>(p, segs[si], rep, lane, first ? 4 : 0, first ? 5 : 1, s_q + qt.slot * C::QB, s_rf + qt.slot * R,
                                             [&] { wait(q_empty + 8 * qt.slot, qt.phase ^ 1); return !dead; });
                fence_proxy_async_smem();
                if (first) queries_bar();
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
    a8_join<__nv_bfloat16, DH, TCA_THREADS>(p, R, rep, s_last, s_cut);
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
template <int DH, int RN>
static yk_status launch_tca(cudaStream_t st, bool pdl, int num_sms, const CUtensorMap& map, const Attn8Params& p) {
    using C = TcaCfg<DH, RN>;
    static_assert(C::R <= A8_WS / DH, "cut spans' rows in the workspace");
    int dev = 0;
    YK_CHECK_CUDA(cudaGetDevice(&dev));
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    const uint64_t bit = 1ull << (dev & 63);
    if (!(ready.load(std::memory_order_acquire) & bit)) {
        YK_CHECK_CUDA(cudaFuncSetAttribute(attn8_tc_kernel<DH, RN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        ready.fetch_or(bit, std::memory_order_release);
    }
    YK_CHECK_CUDA(launch_on(st, pdl, attn8_tc_kernel<DH, RN>, num_sms, TCA_THREADS, C::SMEM, map, p));
    return YK_OK;
}

// rows: (token, head) rows of a sequence's new tokens, as far as the caller says.
// The tile holds them all up to 48 (head_dim 64 and 256: 32), rounded up
// to the next shape; beyond, the kernel for many rows takes over.  16 sequences of
// 500 to 3000 keys, 8 KV heads, this kernel and the other: head_dim 128, 40 rows 43
// and 45 us, 48 rows 46 and 45, 64 rows 58 and 49; head_dim 64, 32 rows 32 and 33,
// 40 rows 38 and 33, 64 rows 48 and 34.  (The other has no room for head_dim 256, whose
// prompts take tiles of 32 rows: 700 tokens over 700-3000 keys 185 us, of 16 rows
// 260.)
template <int DH>
static yk_status launch_tca_rows(cudaStream_t st, bool pdl, int num_sms, const CUtensorMap& map, const Attn8Params& p,
                                 long long rows) {
    if (DH != 256 && rows > (DH == 64 ? 32 : 48)) return attention_e4m3_launch_rows(st, pdl, num_sms, DH, map, p);
    if (rows <= 8) return launch_tca<DH, 1>(st, pdl, num_sms, map, p);
    if (rows <= 16) return launch_tca<DH, 2>(st, pdl, num_sms, map, p);
    if constexpr (DH == 256) return launch_tca<DH, 4>(st, pdl, num_sms, map, p);
    if constexpr (DH != 256) {
        if (rows <= 24) return launch_tca<DH, 3>(st, pdl, num_sms, map, p);
        if (rows <= 32) return launch_tca<DH, 4>(st, pdl, num_sms, map, p);
    }
    if constexpr (DH == 128) return launch_tca<DH, 6>(st, pdl, num_sms, map, p);
    return YK_OK;
}

yk_status attention_e4m3_launch_bf16(cudaStream_t st, bool pdl, int num_sms, int head_dim, const CUtensorMap& map,
                                     const Attn8Params& p, long long rows) {
    switch (head_dim) {
        case 64: return launch_tca_rows<64>(st, pdl, num_sms, map, p, rows);
        case 128: return launch_tca_rows<128>(st, pdl, num_sms, map, p, rows);
        default: return launch_tca_rows<256>(st, pdl, num_sms, map, p, rows);
    }
}

}  // namespace yk
