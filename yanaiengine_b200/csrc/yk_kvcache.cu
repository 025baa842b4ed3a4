// yk_kvcache.cu -- yk_kv_append: per-head norms, rotation and the store into a
// paged KV cache, in one pass over the QKV projections.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "yk_epilogue.cuh"
#include "yk_kvcache.cuh"

namespace yk {

struct AppendParams {
    const void* qkv;
    void* q_out;
    void* pool;
    uint8_t* scales;
    const int32_t* slots;
    const float2* rope;
    const float *q_gain, *k_gain;
    uint32_t* err;
    long long qkv_stride, q_stride;   // elements
    long long block_cells, layer_off;  // cells per block, of the layers before this one
    long long block_scales, layer_scale;
    int T, H, G, num_blocks;
    float eps;
};

// Eight consecutive elements as fp32, and back.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&x);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// One head of one token, spread over DH / 8 lanes (8 consecutive dims each: a
// warp holds 32 * 8 / DH rows): the norm over the head, then the rotation of its
// pairs.  gain, cs: this lane's gains and (cos, sin) of its 4 pairs.  Every lane
// of the warp calls it.
template <int DH>
__device__ __forceinline__ void norm_rotate(bool norm, bool turn, float eps, const float (&gain)[8], const float (&cs)[8], float (&v)[8]) {
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(v[i], v[i], ss);
#pragma unroll
        for (int o = DH / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss * (1.0f / DH) + eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * inv * gain[i];
    }
    if (turn) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 r = rope_rot(v[i], v[i + 1], cs[i], cs[i + 1]);
            v[i] = r.x;
            v[i + 1] = r.y;
        }
    }
}

// The rows that stand alone: query heads, and with fp32 / bf16 pools key and
// value heads too.  A warp takes STEPS * (32 * 8 / DH) consecutive heads of one
// token: their loads go out together, angles and gains are loaded once.
template <typename SRC, typename DST, bool E4M3, int DH, int STEPS>
__device__ __forceinline__ void append_rows(const AppendParams& p, long long task, int lane) {
    constexpr int LPR = DH / 8, RPW = 32 / LPR;
    const int heads = E4M3 ? p.H : p.H + 2 * p.G, chunks = (heads + STEPS * RPW - 1) / (STEPS * RPW);
    const int t = (int)(task / chunks), h0 = (int)(task - (long long)t * chunks) * (STEPS * RPW) + lane / LPR, d = lane % LPR * 8;
    if (t >= p.T) return;
    const int slot = p.slots[t];
    const SRC* const src = reinterpret_cast<const SRC*>(p.qkv) + (size_t)t * p.qkv_stride + d;
    float v[STEPS][8], cs[8], gain[8];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int h = h0 + i * RPW;
        if (h < heads) load8(src + (size_t)h * DH, v[i]);
    }
    if (p.rope) load8(reinterpret_cast<const float*>(p.rope + (size_t)t * (DH / 2)) + d, cs);
    if (E4M3 && p.q_gain) load8(p.q_gain + d, gain);
    if (slot < 0) return;  // padding
    const bool inside = (slot >> 4) < p.num_blocks;
    if (!inside && lane == 0 && h0 == 0) raise_err(p.err, YK_DEV_ERR_BOUNDS);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
        const int h = h0 + i * RPW;
        bool norm = p.q_gain != nullptr, turn = p.rope != nullptr;
        if constexpr (!E4M3) {
            // (rows of a warp may be of different kinds: those without a norm or a turn get gains and angles that
            // change nothing, applied by selection)
            const float* const g = h < p.H ? p.q_gain : h < p.H + p.G ? p.k_gain : nullptr;
            const bool mine = g != nullptr;
            if (mine) load8(g + d, gain);
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = v[i][k];
            norm_rotate<DH>(__any_sync(0xffffffffu, mine), false, p.eps, gain, cs, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[i][k] = mine ? w[k] : v[i][k];
            norm = false;
            turn = turn && h < p.H + p.G;
        }
        norm_rotate<DH>(norm, turn, p.eps, gain, cs, v[i]);
        if (h >= heads) continue;
        if (h < p.H) {
            store8(reinterpret_cast<DST*>(p.q_out) + (size_t)t * p.q_stride + (size_t)h * DH + d, v[i]);
        } else if (inside) {
            store8(reinterpret_cast<DST*>(p.pool) + (size_t)(slot >> 4) * p.block_cells + p.layer_off +
                       ((size_t)(h - p.H) * 16 + (slot & 15)) * DH + d,
                   v[i]);
        }
    }
}

// Whether the 256 rows from `at` on are padding (a warp's eight loads go out together: a tail of thousands of
// rows, read 32 at a time, is a chain of hundreds of loads).
__device__ __forceinline__ bool all_padding(const int32_t* slots, int at, int lane) {
    int s = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) s &= slots[at + 32 * i + lane];
    return __all_sync(0xffffffffu, s < 0);
}

// e4m3 pools: the block's scale couples its tokens, so one warp takes a block's
// new tokens (at most 16) of one head together: the first of them, and the rows
// that follow it.  Their values wait in shared memory (fp32) for the scale.
template <typename SRC, int DH>
__device__ __forceinline__ void append_block(const AppendParams& p, int t, int slot, int h, int lane, float* stage) {
    constexpr int LPR = DH / 8, RPW = 32 / LPR;
    const bool key = h < p.G;
    const int sub = lane / LPR, d = lane % LPR * 8;
    // the block's rows from here on: lane i holds the i-th one's row and offset
    int run = 0, row_i = t, off_i = 0;
    for (int at = t; at < p.T; at += 32) {
        const int s = at + lane < p.T ? p.slots[at + lane] : -1;
        const uint32_t mine = __ballot_sync(0xffffffffu, s >= 0 && s >> 4 == slot >> 4);
        const uint32_t other = __ballot_sync(0xffffffffu, s >= 0 && s >> 4 != slot >> 4);
        const uint32_t here = other ? mine & ((1u << (__ffs(other) - 1)) - 1) : mine;
        const int n = __popc(here), k = lane - run;
        const int from = k >= 0 && k < n ? (int)__fns(here, 0, k + 1) : 0;
        const int o = __shfl_sync(0xffffffffu, s, from) & 15;
        if (k >= 0 && k < n) {
            row_i = at + from;
            off_i = o;
        }
        run += n;
        if (other) break;
        while (at + 32 <= p.T - 256 && all_padding(p.slots, at + 32, lane)) at += 256;
    }
    if (run > 16) {  // a slot appears twice
        if (lane == 0) raise_err(p.err, YK_DEV_ERR_BOUNDS);
        run = 16;
    }
    const uint32_t fresh = __reduce_or_sync(0xffffffffu, lane < run ? 1u << off_i : 0u);
    const uint32_t older = ((1u << (31 - __clz(fresh))) - 1) & ~fresh;  // cells below the last new one
    uint8_t* const sc = p.scales + (size_t)(slot >> 4) * p.block_scales + p.layer_scale + h;
    const uint32_t had_byte = *sc;
    const SRC* const src = reinterpret_cast<const SRC*>(p.qkv) + (size_t)(p.H + h) * DH + d;
    float* const mine = stage + sub * DH + d;
    const bool norm = key && p.k_gain, turn = key && p.rope;
    float amax = 0.f, gain[8];
    if (norm) load8(p.k_gain + d, gain);
    constexpr int U = 2;  // steps whose loads go out together
#pragma unroll 1
    for (int i0 = 0; i0 < run; i0 += U * RPW) {
        float v[U][8], cs[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * RPW + sub, row = __shfl_sync(0xffffffffu, row_i, i & 31);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[u][k] = cs[u][k] = 0.f;
            if (i < run) {
                load8(src + (size_t)row * p.qkv_stride, v[u]);
                if (turn) load8(reinterpret_cast<const float*>(p.rope + (size_t)row * (DH / 2)) + d, cs[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * RPW + sub;
            norm_rotate<DH>(norm, turn, p.eps, gain, cs[u], v[u]);
            if (i < run) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float a = fabsf(v[u][k]);
                    amax = a <= 3.402823466e38f ? fmaxf(amax, a) : amax;  // finite values only
                }
                store8(mine + (i0 + u * RPW) * DH, v[u]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    int e = kv8_cover(amax);
    uint8_t* const cells = reinterpret_cast<uint8_t*>(p.pool) + (size_t)(slot >> 4) * p.block_cells + p.layer_off +
                           (size_t)h * 16 * DH;  // K heads, then V heads: the pool's order
    if (older) {
        const int had = kv8_exponent(had_byte);
        if (e > had) {
            // older tokens' cells move to the larger scale
            const float f = exp2_int(max(had - e, -126));
            for (int c = lane; c < DH; c += 32) {  // 16-byte chunks of the block's 16 cells
                if (!(older >> (c / (DH / 16)) & 1)) continue;
                uint4* const w = reinterpret_cast<uint4*>(cells) + c;
                uint4 x = *w;
                uint32_t* const xs = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 a = f32x2(f16x2_lo(xs[k])), b = f32x2(f16x2_hi(xs[k]));
                    xs[k] = e4m3x2_from(a.x * f, a.y * f) | (e4m3x2_from(b.x * f, b.y * f) << 16);
                }
                *w = x;
            }
        }
        e = max(e, had);
    }
    __syncwarp();  // (every lane has read the old byte)
    if (lane == 0) *sc = (uint8_t)(e + KV8_BIAS);
    const float f = exp2_int(-e);
#pragma unroll 2
    for (int i0 = 0; i0 < run; i0 += RPW) {
        const int i = i0 + sub, off = __shfl_sync(0xffffffffu, off_i, i & 31);
        if (i < run) {
            float v[8];
            load8(mine + i0 * DH, v);  // (this lane's own values)
            uint32_t w[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                w[k] = e4m3x2_from(v[4 * k] * f, v[4 * k + 1] * f) | (e4m3x2_from(v[4 * k + 2] * f, v[4 * k + 3] * f) << 16);
            *reinterpret_cast<uint2*>(cells + (size_t)off * DH + d) = make_uint2(w[0], w[1]);
        }
    }
}

// The first row_blocks CTAs take single rows, the others (e4m3) blocks: a warp
// looks at `tile` consecutive rows (at most 16) for those that begin a block.
// Bytes bound it: every row is read once.  What the shape is after is loads in
// flight and few instructions a byte: 16 bytes of bf16 a lane, STEPS rows of
// loads a warp where there are rows enough, one where there are not (decode).
// Measured, 32 query and 8 KV heads of 128: 8,197 tokens of bf16 into e4m3 cells 52
// us (162 MB, 3.1 TB/s, 47 % of a copy's rate: a third of the warps fit beside 8 KB
// of staging each, and wait for loads; bound to 72 registers for a seventh CTA that
// the staging does not leave room for, 56 us); 2,048 tokens into bf16 cells 10.6 us
// (68 MB, 97 % with what stays in L2); 192 tokens 5.6 us and one token 2.7 us, the
// launch.  Eight tokens in front of 8,184 rows of padding 35 us, of 32,760 124 us (98 and
// 1,130 while every warp of the padding looked for a row before it, 32 rows at a time).
template <typename SRC, typename DST, bool E4M3, int DH, int STEPS>
__global__ void __launch_bounds__(128, DH == 256 ? 3 : 6) kv_append_kernel(const __grid_constant__ AppendParams p, unsigned row_blocks, int tile) {
    extern __shared__ __align__(16) float append_stage[];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x < row_blocks) {
        append_rows<SRC, DST, E4M3, DH, STEPS>(p, (long long)blockIdx.x * 4 + warp, lane);
        return;
    }
    if constexpr (E4M3) {
        const long long task = (long long)(blockIdx.x - row_blocks) * 4 + warp;
        const int t0 = (int)(task / (2 * p.G)) * tile, h = (int)(task % (2 * p.G));
        if (t0 >= p.T) return;
        const int s = lane < tile && t0 + lane < p.T ? p.slots[t0 + lane] : -1;
        uint32_t live = __ballot_sync(0xffffffffu, s >= 0);
        if (!live) return;
        // the nearest earlier row that is not padding: of the same block, it (or one before it) stores this row too
        int before = -1;
        for (int back = t0 - 1; back >= 0; back -= 32) {
            const int x = back - lane >= 0 ? p.slots[back - lane] : -1;
            const uint32_t m = __ballot_sync(0xffffffffu, x >= 0);
            if (m) {
                before = __shfl_sync(0xffffffffu, x, __ffs(m) - 1) >> 4;
                break;
            }
            while (back >= 287 && all_padding(p.slots, back - 287, lane)) back -= 256;
        }
        for (; live; live &= live - 1) {
            const int i = __ffs(live) - 1, slot = __shfl_sync(0xffffffffu, s, i), block = slot >> 4;
            if (block != before && block < p.num_blocks)
                append_block<SRC, DH>(p, t0 + i, slot, h, lane, append_stage + warp * 16 * DH);
            before = block;
        }
    }
}

template <typename SRC, typename DST, bool E4M3, int DH>
static cudaError_t launch_append_dh(cudaStream_t st, bool pdl, int sms, const AppendParams& p) {
    constexpr int RPW = 256 / DH, STEPS = 4;
    const int heads = E4M3 ? p.H : p.H + 2 * p.G;
    // Several rows a warp, and several rows to look through, once that leaves this many warps an SM.  16-bit and fp32
    // pools: 24, as many as run at once (384 tokens, 32 + 16 heads of 128 into bf16 cells: 4.1 us, 4.9 with 12).
    // e4m3 pools, whose block warps take half of the room: 12 (768 tokens 10.4 us, 12.1 with 24; 1,536 tokens 14.4
    // and 14.7; heads of 256 15.8 and 20.8, 21.1 and 23.7; heads of 64 7.4 and 7.9, 8.5 and 10.4).  Up to 192 tokens
    // and from 8,192 on the two are the same.
    const long long warps = (long long)sms * (E4M3 ? 12 : 24);
    const auto tasks = [&](int steps) { return (long long)p.T * ((heads + steps * RPW - 1) / (steps * RPW)); };
    const int steps = tasks(STEPS) >= warps ? STEPS : 1;  // (several rows a warp once that still fills the device)
    const unsigned row_blocks = (unsigned)((tasks(steps) + 3) / 4);
    // rows a warp looks through for blocks: by the same rule
    int tile = 1;
    while (tile < 16 && (long long)p.T * 2 * p.G >= 2 * tile * warps) tile *= 2;
    const unsigned blocks = E4M3 ? (unsigned)((((long long)p.T + tile - 1) / tile * 2 * p.G + 3) / 4) : 0;
    constexpr size_t smem = E4M3 ? 4 * 16 * DH * 4 : 0;
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    if (smem > 48 * 1024) {
        int dev = 0;
        if (const cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
        const uint64_t bit = 1ull << (dev & 63);
        if (!(ready.load(std::memory_order_acquire) & bit)) {
            for (auto* f : {kv_append_kernel<SRC, DST, E4M3, DH, STEPS>, kv_append_kernel<SRC, DST, E4M3, DH, 1>})
                if (const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); e != cudaSuccess)
                    return e;
            ready.fetch_or(bit, std::memory_order_release);
        }
    }
    if (steps > 1)
        return launch_on(st, pdl, kv_append_kernel<SRC, DST, E4M3, DH, STEPS>, row_blocks + blocks, 128, smem, p, row_blocks, tile);
    return launch_on(st, pdl, kv_append_kernel<SRC, DST, E4M3, DH, 1>, row_blocks + blocks, 128, smem, p, row_blocks, tile);
}

// N(0, std) into every cell of an e4m3 pool: one warp per (block, layer, K|V, head).
__global__ void __launch_bounds__(128) fill_e4m3_kernel(uint8_t* cells, uint8_t* scales, long long heads, int dh, uint64_t seed, float std) {
    const long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= heads) return;
    const auto four = [&](int q) {  // values 4 q .. 4 q + 3 of this head (Box-Muller)
        const uint4 r = philox4x32_10(make_uint4((uint32_t)i, (uint32_t)(i >> 32), (uint32_t)q, 0x4B38u),
                                      make_uint2((uint32_t)seed, (uint32_t)(seed >> 32)));
        float4 v;
        const float a = sqrtf(-2.f * logf(u24(r.x) + 2.98e-8f)) * std, b = sqrtf(-2.f * logf(u24(r.z) + 2.98e-8f)) * std;
        sincospif(2.f * u24(r.y), &v.y, &v.x);
        sincospif(2.f * u24(r.w), &v.w, &v.z);
        return make_float4(v.x * a, v.y * a, v.z * b, v.w * b);
    };
    float amax = 0.f;
    for (int q = lane; q < 4 * dh; q += 32) {
        const float4 v = four(q);
        amax = fmaxf(fmaxf(fmaxf(amax, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const int e = kv8_cover(amax);
    const float f = exp2_int(-e);
    for (int q = lane; q < 4 * dh; q += 32) {
        const float4 v = four(q);
        reinterpret_cast<uint32_t*>(cells + i * 16 * dh)[q] = e4m3x2_from(v.x * f, v.y * f) | e4m3x2_from(v.z * f, v.w * f) << 16;
    }
    if (lane == 0) scales[i] = (uint8_t)(e + KV8_BIAS);
}
yk_status launch_fill_e4m3(yk_kv_pool* p, uint64_t seed, float std) {
    const long long heads = (long long)p->num_blocks * p->n_pool_layers * 2 * p->cfg.n_kv_heads;
    fill_e4m3_kernel<<<(unsigned)((heads + 3) / 4), 128, 0, p->e->stream>>>((uint8_t*)p->data, p->scales, heads, p->cfg.head_dim, seed, std);
    p->e->launches++;
    YK_CHECK_CUDA(cudaGetLastError());
    return YK_OK;
}

template <typename SRC, typename DST, bool E4M3>
static cudaError_t launch_append(cudaStream_t st, bool pdl, int sms, int dh, const AppendParams& p) {
    switch (dh) {
        case 64: return launch_append_dh<SRC, DST, E4M3, 64>(st, pdl, sms, p);
        case 128: return launch_append_dh<SRC, DST, E4M3, 128>(st, pdl, sms, p);
        default: return launch_append_dh<SRC, DST, E4M3, 256>(st, pdl, sms, p);
    }
}

yk_status kv_append_launch(cudaStream_t st, bool pdl, int sms, const yk_kv_append_args& a) {
    if (a.T == 0) return YK_OK;
    AppendParams p;
    p.qkv = a.qkv;
    p.q_out = a.q_out;
    p.pool = a.pages.data;
    p.scales = a.pages.scales;
    p.slots = a.slots;
    p.rope = reinterpret_cast<const float2*>(a.rope);
    p.q_gain = a.q_gain;
    p.k_gain = a.k_gain;
    p.err = a.err;
    p.qkv_stride = a.qkv_stride;
    p.q_stride = a.q_stride;
    const long long layer_scales = 2LL * a.pages.n_kv_heads, layer_cells = layer_scales * YK_BLOCK_SIZE * a.pages.head_dim;
    p.block_cells = layer_cells * a.pages.n_layers;
    p.layer_off = layer_cells * a.layer;
    p.block_scales = layer_scales * a.pages.n_layers;
    p.layer_scale = layer_scales * a.layer;
    p.T = a.T;
    p.H = a.n_heads;
    p.G = a.pages.n_kv_heads;
    p.num_blocks = a.pages.num_blocks;
    p.eps = a.eps;
    const int dh = a.pages.head_dim;
    const bool e4 = a.pages.kind == YK_KV_E4M3;
    cudaError_t r;
    if (a.src_dtype == YK_DTYPE_BF16) {
        r = e4 ? launch_append<__nv_bfloat16, __nv_bfloat16, true>(st, pdl, sms, dh, p)
               : launch_append<__nv_bfloat16, __nv_bfloat16, false>(st, pdl, sms, dh, p);
    } else if (a.q_dtype == YK_DTYPE_BF16) {
        r = e4 ? launch_append<float, __nv_bfloat16, true>(st, pdl, sms, dh, p)
               : launch_append<float, __nv_bfloat16, false>(st, pdl, sms, dh, p);
    } else {
        r = e4 ? launch_append<float, float, true>(st, pdl, sms, dh, p) : launch_append<float, float, false>(st, pdl, sms, dh, p);
    }
    YK_CHECK_CUDA(r);
    return YK_OK;
}

// ---------------------------------------------------------------------------
// Argument checks.
// ---------------------------------------------------------------------------
static bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

yk_status kv_pages_check(const yk_kv_pages& p, int32_t layer) {
    YK_ARG(p.kind >= YK_KV_F32 && p.kind <= YK_KV_E4M3, "pages.kind (YK_KV_*)");
    YK_ARG(p.data && aligned16(p.data), "pages.data must be a 16-byte aligned device pointer");
    YK_ARG((p.scales != nullptr) == (p.kind == YK_KV_E4M3), "pages.scales belongs to YK_KV_E4M3 pools, and only to them");
    YK_ARG(p.head_dim == 64 || p.head_dim == 128 || p.head_dim == 256, "head_dim must be 64, 128 or 256");
    YK_ARG(p.num_blocks > 0 && p.num_blocks <= (1 << 27), "pages.num_blocks must be in 1..2^27 (slots are 32-bit)");
    YK_ARG(p.n_layers > 0 && p.n_kv_heads > 0 && p.n_kv_heads <= 4096, "pages.n_layers / n_kv_heads");
    YK_ARG(layer >= 0 && layer < p.n_layers, "layer outside the pool's");
    return YK_OK;
}

yk_status kv_append_check(const yk_kv_append_args& a) {
    YK_TRY(kv_pages_check(a.pages, a.layer));
    YK_ARG(a.T >= 0, "T");
    YK_ARG(a.n_heads > 0 && a.n_heads <= 65536 && a.n_heads % a.pages.n_kv_heads == 0,
           "n_heads must be a positive multiple of n_kv_heads");
    const bool f2f = a.src_dtype == YK_DTYPE_F32 && a.q_dtype == YK_DTYPE_F32;
    const bool f2b = a.src_dtype == YK_DTYPE_F32 && a.q_dtype == YK_DTYPE_BF16;
    const bool b2b = a.src_dtype == YK_DTYPE_BF16 && a.q_dtype == YK_DTYPE_BF16;
    if (!f2f && !f2b && !b2b) {
        yk_set_error("unsupported: src_dtype -> q_dtype must be F32 -> F32, F32 -> BF16 or BF16 -> BF16");
        return YK_ERR_UNSUPPORTED;
    }
    YK_ARG(a.pages.kind == YK_KV_E4M3 || a.pages.kind == (f2f ? YK_KV_F32 : YK_KV_BF16),
           "fp32 / bf16 cells must have q_dtype's type");
    YK_ARG(std::isfinite(a.eps) && a.eps >= 0.f, "eps must be finite and not negative");
    if (a.T == 0) return YK_OK;
    YK_ARG(a.qkv && a.q_out && a.slots, "null qkv / q_out / slots");
    const int64_t dh = a.pages.head_dim;
    const int64_t src = a.src_dtype == YK_DTYPE_F32 ? 4 : 2, dst = a.q_dtype == YK_DTYPE_F32 ? 4 : 2;
    YK_ARG(aligned16(a.qkv) && aligned16(a.q_out), "qkv and q_out must be 16-byte aligned");
    YK_ARG(a.qkv_stride >= (a.n_heads + 2 * (int64_t)a.pages.n_kv_heads) * dh && a.qkv_stride * src % 16 == 0,
           "qkv_stride must cover a row and be a multiple of 16 bytes");
    YK_ARG(a.q_stride >= a.n_heads * dh && a.q_stride * dst % 16 == 0,
           "q_stride must cover a row and be a multiple of 16 bytes");
    YK_ARG(aligned16(a.rope) && aligned16(a.q_gain) && aligned16(a.k_gain), "rope and gains must be 16-byte aligned");
    YK_ARG((int64_t)a.T * (a.n_heads + 2 * (int64_t)a.pages.n_kv_heads) <= (int64_t)1 << 32, "T * heads too large");
    return YK_OK;
}

// SMs of `device`, asked for once.
static yk_status device_sms(int32_t device, const char* what, int* sms) {
    static std::atomic<int> known[64];
    if (device >= 0 && device < 64 && (*sms = known[device].load(std::memory_order_relaxed)) > 0) return YK_OK;
    int n = 0;
    if (const cudaError_t e = cudaGetDeviceCount(&n); e != cudaSuccess) {
        cudaGetLastError();  // (not left pending for the next call)
        yk_set_error(std::string(what) + ": " + cudaGetErrorString(e));
        return YK_ERR_CUDA;
    }
    YK_ARG(device >= 0 && device < n, "device index");
    YK_CHECK_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
    if (device < 64) known[device].store(*sms, std::memory_order_relaxed);
    return YK_OK;
}

// The operators' launches may begin before the kernel ahead of them in the stream
// has ended: they wait for its end (griddepcontrol.wait) before they touch memory,
// whatever kernel it is.
// Runs body(SMs of `device`) with `device` current; a CUDA error that earlier work
// left pending on this thread is returned before anything is launched.
template <typename F>
static yk_status on_device(int32_t device, const char* what, F body) {
    const cudaError_t pending = cudaGetLastError();
    if (pending != cudaSuccess) {
        yk_set_error(std::string(what) + ": a CUDA error from earlier work was pending before this call (nothing "
                                         "launched): " + cudaGetErrorString(pending));
        return YK_ERR_CUDA;
    }
    int prev = 0, sms = 0;
    YK_TRY(device_sms(device, what, &sms));
    YK_CHECK_CUDA(cudaGetDevice(&prev));
    if (prev != device) YK_CHECK_CUDA(cudaSetDevice(device));
    const yk_status s = body(sms);
    if (prev != device) cudaSetDevice(prev);
    return s;
}

}  // namespace yk

extern "C" yk_status yk_kv_append(int32_t device, void* stream, const yk_kv_append_args* args) {
    YK_ARG(args, "args is null");
    YK_TRY(yk::kv_append_check(*args));
    return yk::on_device(device, "yk_kv_append", [&](int sms) {
        return yk::kv_append_launch(static_cast<cudaStream_t>(stream), true, sms, *args);
    });
}

extern "C" yk_status yk_attention_e4m3_workspace(int32_t device, int32_t head_dim, uint64_t* bytes) {
    YK_ARG(bytes, "bytes is null");
    YK_ARG(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256");
    return yk::on_device(device, "yk_attention_e4m3_workspace", [&](int sms) -> yk_status {
        *bytes = yk::attention_e4m3_ws_bytes(sms, head_dim);
        return YK_OK;
    });
}

extern "C" yk_status yk_attention_e4m3(int32_t device, void* stream, const yk_attention_e4m3_args* args) {
    YK_ARG(args, "args is null");
    YK_TRY(yk::attention_e4m3_check(*args));
    return yk::on_device(device, "yk_attention_e4m3", [&](int sms) -> yk_status {
        YK_ARG(args->T == 0 || args->workspace_bytes >= yk::attention_e4m3_ws_bytes(sms, args->pages.head_dim),
               "workspace_bytes is below yk_attention_e4m3_workspace's");
        return yk::attention_e4m3_launch(static_cast<cudaStream_t>(stream), true, sms, *args);
    });
}
