// yk_attention_e4m3_tc.cuh -- what the two tcgen05 kernels of yk_attention_e4m3
// share: instructions, the copies of K and V tiles, the conversion of V.
#pragma once
#include "yk_attention_e4m3.cuh"

namespace yk {

constexpr int TCA_TILE = 128;  // keys
constexpr int TCA_PAGES = TCA_TILE / YK_BLOCK_SIZE;
constexpr int TCA_COST = 2;    // a span's own cost, in tiles (verify: 6000 cycles and 2700 for a tile; head_dim 64: 2700 and 1600)
constexpr int TCA_INFO = 16;   // tiles whose page words are kept

// ---------------------------------------------------------------------------
// Small wrappers.
// ---------------------------------------------------------------------------
// N columns of this thread's TMEM lane (the values are there after tmem_wait_ld).
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t* r) {
    if constexpr (N >= 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(a));
        if constexpr (N > 16) tmem_ld<N - 16>(a + 16, r + 16);
    } else if constexpr (N >= 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(a));
        if constexpr (N > 8) tmem_ld<N - 8>(a + 8, r + 8);
    } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(a));
    }
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t* r) {
    if constexpr (N >= 8) {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                     "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                     : "memory");
        if constexpr (N > 8) tmem_st<N - 8>(a + 8, r + 8);
    } else {
        asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                     : "memory");
    }
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Shared-memory matrix descriptors (sm_100), as two words: the low one holds the
// address and the leading stride, the high one the other stride and the swizzle
// (2: 128 B, 4: 64 B, 6: 32 B).
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo, uint32_t swizzle) { return sbo >> 4 | 1u << 14 | swizzle << 29; }
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo = 0) { return addr >> 4 | lbo >> 4 << 16; }
template <bool F8>
__device__ __forceinline__ void mma_tc(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                       uint32_t accumulate) {
    if constexpr (F8)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %5, p;\n\t}" ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi),
            "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi),
            "r"(idesc), "r"(accumulate)
            : "memory");
}
__device__ __forceinline__ uint32_t f16x2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ uint32_t e5m2x2_from(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void sts64(uint32_t a, uint32_t x, uint32_t y) {
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(a), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// The rare ends of a wait and of a NaN cell, kept out of line: the kernel's loops
// have to stay in the instruction cache.
static __device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, uint32_t* err) {
    const bool ok = mbar_wait_bounded(bar, parity);
    if (!ok) raise_err(err, YK_DEV_ERR_TIMEOUT);
    return ok;
}
// Notes the NaN cells among the 16 of a key at `cells` (dims dim0 ..) for the rows that see it.
static __device__ __noinline__ void note_nans(uint32_t cells, int dim0, int key, int pos, int rem, uint32_t rep_magic, int rows,
                                       int window, int words, uint32_t* s_nan, int* s_flag) {
#pragma unroll 1
    for (int z = 0; z < 16; ++z) {
        uint32_t x;
        asm volatile("ld.shared.u8 %0, [%1];" : "=r"(x) : "r"(cells + (uint32_t)z));
        if ((x & 0x7f) != 0x7f) continue;
#pragma unroll 1
        for (int row = 0; row < rows; ++row) {
            const int back = pos + (rep_magic ? (int)__umulhi((unsigned)(rem + row), rep_magic) : rem + row) - key;
            if (back >= 0 && (window <= 0 || back < window)) {
                atomicOr(&s_nan[row * words + ((dim0 + z) >> 5)], 1u << ((dim0 + z) & 31));
                *s_flag = 1;
            }
        }
    }
}

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {  // (does not wait)
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool elected() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// A ring's next place: slot and the parity of its use.
template <int N>
struct Turn {
    int slot = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++slot == N) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// The V warps and the queries' warp, where all five convert a span's queries: those of a CTA's first span, which
// everything waits for, and with many rows every span's.
__device__ __forceinline__ void queries_bar() { asm volatile("bar.sync 1, 160;" ::: "memory"); }
__device__ __forceinline__ void v_bar() { asm volatile("bar.sync 2, 128;" ::: "memory"); }
__device__ __forceinline__ float cap_score(const Attn8Params& p, float x) { return p.cap_log2 * tanh_cap(x * p.inv_cap_log2); }

// Whether every row of the span's tile sees all keys j0 .. j0 + 127.
__device__ __forceinline__ bool all_seen(const Attn8Params& p, const Seg& sg, int pos_last, int j0) {
    return j0 + TCA_TILE - 1 <= sg.pos && (p.window <= 0 || pos_last - j0 < p.window);
}


// The V warps (128 threads, tid): a tile of e4m3 cells to f16, [64-dim block][key][128 bytes, swizzled].
template <int DH>
__device__ __forceinline__ void convert_tile(const Attn8Params& p, const Seg& sg, int pos_last, int j0, int tid, uint8_t* cells, uint8_t* f16,
                                             const int* info, uint32_t* s_nan, int* s_flag) {
    constexpr int C16 = DH / 16, KEYS = 128 / C16;  // 16-byte pieces of a key; keys the warps take at a time
    const int c16 = tid % C16, key0 = tid / C16;
    // places of a piece's two 16-byte chunks in a 128-byte row of f16, by key & 7 (swizzle); lanes of one
    // 64-dim block store them in the other order (bank conflicts)
    const int sw = (c16 >> 2) & 1;
    const uint32_t chunk = (uint32_t)(((2 * c16) & 7) << 4);
    const int4 i0 = *reinterpret_cast<const int4*>(info), i1 = *reinterpret_cast<const int4*>(info + 4);
    const bool plain = all_seen(p, sg, pos_last, j0) && (i0.x | i0.y | i0.z | i0.w | i1.x | i1.y | i1.z | i1.w) >= 0;
    const uint32_t src = smem_u32(cells) + (uint32_t)(tid * 16);
    const uint32_t dst = smem_u32(f16) + (uint32_t)((c16 >> 2) * 16384);
    if (!plain) {
        // cells without a page hold whatever the ring held: zeros instead.  A NaN cell must reach
        // the rows that see its key and no others: it is taken out of the product, and noted for
        // the rows it belongs to
#pragma unroll 1
        for (int it = 0; it < 128 / KEYS; ++it) {
            const int key = it * KEYS + key0;
            const uint32_t at = src + (uint32_t)(it * 2048);
            uint32_t w[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
            if (info[key >> 4] < 0) w[0] = w[1] = w[2] = w[3] = 0;
            uint32_t any = 0;
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const uint32_t bad = ((w[z] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                w[z] &= ~(bad | (bad - (bad >> 7)));
                any |= bad;
            }
            if (any)
                note_nans(at, c16 * 16, j0 + key, sg.pos, sg.rem, p.rep_magic, sg.rows, p.window, DH / 32, s_nan, s_flag);
            sts128(at, w[0], w[1], w[2], w[3]);
        }
    }
    // 8 bytes to one 16-byte chunk, twice
    const uint32_t from = src + (uint32_t)(sw * 8), to = dst + (chunk ^ (uint32_t)(sw << 4));
#pragma unroll 4
    for (int it = 0; it < 128 / KEYS; ++it) {
        const int key = it * KEYS + key0;
        const uint32_t at = from + (uint32_t)(it * 2048);
        uint32_t w[4];
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[2]), "=r"(w[3]) : "r"(at ^ 8u));
        const uint32_t a = (to ^ (uint32_t)((key & 7) << 4)) + (uint32_t)((key >> 3) * 1024 + (key & 7) * 128);
        sts128(a, f16x2_lo(w[0]), f16x2_hi(w[0]), f16x2_lo(w[1]), f16x2_hi(w[1]));
        sts128(a ^ 16u, f16x2_lo(w[2]), f16x2_hi(w[2]), f16x2_lo(w[3]), f16x2_hi(w[3]));
    }
}

// One warp: the K (or V) pages of the listed spans' tiles into a ring of N tiles,
// and each tile's page words, exponents or -1: no page.
template <int DH, bool V, int N, typename Wait>
__device__ __forceinline__ void copy_tiles(const Attn8Params& p, const CUtensorMap& map, const Seg* segs, int nseg, int lane, uint8_t* ring,
                                           uint32_t full, uint32_t empty, int* info, Turn<N>& t, int& tile, const Wait& wait, const bool& dead) {
    constexpr int ROWB = DH == 64 ? 64 : 128;  // bytes of a K row in one TMA box
    // lane: page lane & 7 of tile lane / 8 of a batch of four tiles of one span
    // (block ids are asked for two batches ahead, scale bytes one: nobody waits for either)
    int id = -1, id2 = -1, id3 = -1, g3 = 0;
    bool has3 = false;
    uint32_t kb = 0, vb = 0, kb2 = 0, vb2 = 0;
    int fsi = 0, fi = 0;  // the batch to ask for next
    const auto ids = [&]() {
        has3 = false;
        if (fsi >= nseg) return;
        const Seg& sg = segs[fsi];
        const int page = sg.page + TCA_PAGES * fi + lane;
        has3 = fi + (lane >> 3) < sg.n && page < sg.pend;
        g3 = sg.g;
        if (has3) id3 = p.tables[(size_t)sg.b * p.max_blocks + page];
        fi += 4;
        if (fi >= sg.n) {
            fi = 0;
            ++fsi;
        }
    };
    const auto scales = [&]() {
        id2 = -1;
        if (!has3) return;
        if (id3 < 0 || id3 >= p.num_blocks) {
            raise_err(p.err, YK_DEV_ERR_BOUNDS);
            return;
        }
        id2 = id3;
        if (!V) {
            const uint8_t* const s = p.scales + (size_t)id3 * p.block_scales + p.layer_scale + g3;
            kb2 = s[0];
            vb2 = s[p.G];
        }
    };
    ids();
    scales();
    ids();
#pragma unroll 1
    for (int si = 0; si < nseg; ++si) {
        const int n = segs[si].n, g = segs[si].g;
#pragma unroll 1
        for (int i = 0; i < n; ++i, ++tile) {
            if ((i & 3) == 0) {
                id = id2;
                kb = kb2;
                vb = vb2;
                scales();
                ids();
            }
            const bool mine = lane >> 3 == (i & 3);  // this lane's page belongs to the tile
            const int pages = __popc(__ballot_sync(0xffffffffu, mine && id >= 0));
            const uint32_t bar = full + 8 * t.slot;
            wait(empty + 8 * t.slot, t.phase ^ 1);
            __syncwarp();
            // (the copies first: the scale bytes may still be on their way, and the barrier's one arrival comes after both)
            if (mine && id >= 0 && !dead) {
                const uint32_t dst = smem_u32(ring + t.slot * TCA_TILE * DH) + (uint32_t)((lane & 7) * 16 * (V ? DH : ROWB));
                if constexpr (V) {
                    bulk_load(dst, p.pool + (size_t)id * p.block_cells + p.layer_off + (size_t)(p.G + g) * 16 * DH, 16 * DH, bar);
                } else {
#pragma unroll
                    for (int x = 0; x < DH / ROWB; ++x)
                        asm volatile(
                            "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
                            " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst + (uint32_t)(x * TCA_TILE * 128)),
                            "l"((uint64_t)&map), "r"(x * 128), "r"(g * 16), "r"(0), "r"(p.layer), "r"(id), "r"(bar)
                            : "memory");
                }
            }
            if (mine)
                info[(tile & (TCA_INFO - 1)) * TCA_PAGES + (lane & 7)] =
                    id < 0 ? -1 : (kv8_exponent(kb) + 128) | (kv8_exponent(vb) + 128) << 8;
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(bar, dead ? 0u : (uint32_t)(pages * 16 * DH));
            t.next();
        }
    }
}

// A warp, part of `parts`: a span's queries as two terms that sum to them, [128-dim block][term][R rows][128 bytes] (head_dim 64:
// 64 bytes), swizzled, and the rows' score factors.  JOINED: the second term is e5m2, else e4m3 times 16.
// `free` waits until the room is, and says whether to write.
template <int DH, int R, bool JOINED, typename Free>
__device__ __forceinline__ void convert_queries(const Attn8Params& p, const Seg& sg, int rep, int lane, int part, int parts, uint8_t* room,
                                                float* s_rf, const Free& free) {
    constexpr int LPR = DH / 16, RPI = 32 / LPR;  // lanes a row, rows at a time
    const int c16 = lane % LPR;
    uint4 x[2], y[2];  // 16 values; the next rows' come while these convert
    const auto load = [&](int r0, uint4 (&v)[2]) {
        const int row = r0 + lane / LPR;
        v[0] = v[1] = make_uint4(0, 0, 0, 0);
        if (row < sg.rows) {
            const int tok = div_rep(p, sg.rem + row);
            const uint4* const src = reinterpret_cast<const uint4*>(
                reinterpret_cast<const __nv_bfloat16*>(p.q) + (size_t)(sg.tok + tok) * p.q_stride +
                (size_t)(sg.g * rep + sg.rem + row - tok * rep) * DH + c16 * 16);
            v[0] = __ldcg(src);
            v[1] = __ldcg(src + 1);
        }
    };
    load(part * RPI, x);
    const bool live = free();
#pragma unroll 1
    for (int r0 = part * RPI; r0 < R; r0 += parts * RPI) {
        load(r0 + parts * RPI, y);
        const int row = r0 + lane / LPR;
        float f[16];
        const uint32_t w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
        float amax = 0.f;
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            f[2 * z] = __uint_as_float(w[z] << 16);
            f[2 * z + 1] = __uint_as_float(w[z] & 0xffff0000u);
            amax = fmaxf(amax, fmaxf(fabsf(f[2 * z]), fabsf(f[2 * z + 1])));
        }
#pragma unroll
        for (int o = 1; o < LPR; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        // 2^-e brings the row's largest value to at most 448.  An infinite one has no place in the terms, which
        // saturate: its row's become NaN, as the softmax of its scores is
        const uint32_t bits = __float_as_uint(amax);
        const int e = amax == 0.f ? 0 : max(-126, (int)(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));  // 120 at most
        const float g = bits == 0x7f800000u ? __int_as_float(0x7fffffff) : exp2_int(-e);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            hi[z] = lo[z] = 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float a = f[4 * z + 2 * k] * g, b = f[4 * z + 2 * k + 1] * g;
                const uint32_t h = e4m3x2_from(a, b);
                const float2 back = f32x2(f16x2_lo(h));
                hi[z] |= h << (16 * k);
                lo[z] |= (JOINED ? e5m2x2_from(a - back.x, b - back.y)
                                 : e4m3x2_from((a - back.x) * 16.f, (b - back.y) * 16.f)) << (16 * k);
            }
        }
        if (row < R && live) {
            if (c16 == 0) s_rf[row] = fminf(p.scale_log2 * exp2_int(e), A8_LARGEST);  // (finite: a score of 0 stays 0)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int n = row + t * R;
                const uint32_t at = DH == 64 ? (uint32_t)(n * 64 + ((c16 ^ ((n >> 1) & 3)) << 4))
                                             : (uint32_t)((c16 >> 3) * (2 * R * 128) + n * 128 + (((c16 & 7) ^ (n & 7)) << 4));
                const uint32_t* const v = t ? lo : hi;
                sts128(smem_u32(room) + at, v[0], v[1], v[2], v[3]);
            }
        }
        x[0] = y[0];
        x[1] = y[1];
    }
}

// Many rows (yk_attention_e4m3_rows.cu).
yk_status attention_e4m3_launch_rows(cudaStream_t st, bool pdl, int num_sms, int head_dim, const CUtensorMap& map, const Attn8Params& p);

}  // namespace yk
