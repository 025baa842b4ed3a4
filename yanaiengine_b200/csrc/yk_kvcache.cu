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

// N consecutive elements at p (N * size <= 16 bytes per load) as fp32.
template <int N>
__device__ __forceinline__ void load_row(const float* p, float (&v)[N]) {
    if constexpr (N == 2) {
        const float2 a = *reinterpret_cast<const float2*>(p);
        v[0] = a.x; v[1] = a.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 a = *reinterpret_cast<const float4*>(p + i);
            v[i] = a.x; v[i + 1] = a.y; v[i + 2] = a.z; v[i + 3] = a.w;
        }
    }
}
template <int N>
__device__ __forceinline__ void load_row(const __nv_bfloat16* p, float (&v)[N]) {
    uint32_t w[N / 2];
    if constexpr (N == 2) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 4) {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        w[0] = a.x; w[1] = a.y;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <int N, typename AT>
__device__ __forceinline__ void store_row(AT* p, const float (&v)[N]) {
    if constexpr (N == 2) {
        store2(p, v[0], v[1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) store4(p + i, v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
}

// One head of one token, spread over a warp (lane: N = DH / 32 consecutive
// dims): the norm over the head, then the rotation of its pairs.
template <int DH, int N>
__device__ __forceinline__ void norm_rotate(const AppendParams& p, const float* gain, int t, int lane, float (&v)[N]) {
    if (gain) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(v[i], v[i], ss);
        const float inv = rsqrtf(warp_sum_f(ss) * (1.0f / DH) + p.eps);
        float g[N];
        load_row<N>(gain + lane * N, g);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] * inv * g[i];
    }
    if (p.rope) {
        float cs[N];  // (cos, sin) of N / 2 pairs
        load_row<N>(reinterpret_cast<const float*>(p.rope + (size_t)t * (DH / 2)) + lane * N, cs);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 r = rope_rot(v[i], v[i + 1], cs[i], cs[i + 1]);
            v[i] = r.x;
            v[i + 1] = r.y;
        }
    }
}

// The rows that stand alone: query heads, and with fp32 / bf16 pools key and
// value heads too.  A warp takes ROWS of them, consecutive in (token, head)
// order, their loads in flight together.
template <typename SRC, typename DST, bool E4M3, int DH, int ROWS>
__device__ __forceinline__ void append_rows(const AppendParams& p, long long first, int lane) {
    constexpr int N = DH / 32;
    const int all = p.H + 2 * p.G, heads = E4M3 ? p.H : all;
    int t = (int)(first / heads), h = (int)(first - (long long)t * heads);
    float v[ROWS][N];
    int ts[ROWS], hs[ROWS], slot[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        ts[i] = t;
        hs[i] = h;
        slot[i] = -1;
        if (t < p.T) {
            slot[i] = p.slots[t];
            load_row<N>(reinterpret_cast<const SRC*>(p.qkv) + (size_t)t * p.qkv_stride + (size_t)h * DH + lane * N, v[i]);
        }
        if (++h == heads) {
            h = 0;
            ++t;
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        if (slot[i] < 0) continue;  // padding
        const bool query = hs[i] < p.H;
        if (query || hs[i] < p.H + p.G) norm_rotate<DH, N>(p, query ? p.q_gain : p.k_gain, ts[i], lane, v[i]);
        if (query) {
            store_row<N>(reinterpret_cast<DST*>(p.q_out) + (size_t)ts[i] * p.q_stride + (size_t)hs[i] * DH + lane * N, v[i]);
        } else if ((slot[i] >> 4) < p.num_blocks) {
            store_row<N>(reinterpret_cast<DST*>(p.pool) + (size_t)(slot[i] >> 4) * p.block_cells + p.layer_off +
                             ((size_t)(hs[i] - p.H) * 16 + (slot[i] & 15)) * DH + lane * N,
                         v[i]);
        }
        if (hs[i] == 0 && lane == 0 && (slot[i] >> 4) >= p.num_blocks) raise_err(p.err, YK_DEV_ERR_BOUNDS);
    }
}

// e4m3 pools: the block's scale couples its tokens, so one warp takes a block's
// new tokens (at most 16) of one head together: the first of them, and the rows
// that follow it.  Their values wait in shared memory (fp32) for the scale.
template <typename SRC, int DH>
__device__ __forceinline__ void append_block(const AppendParams& p, int t, int slot, int h, int lane, float* stage) {
    constexpr int N = DH / 32;
    const bool key = h < p.G;
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
    }
    if (run > 16) {  // a slot appears twice
        if (lane == 0) raise_err(p.err, YK_DEV_ERR_BOUNDS);
        run = 16;
    }
    const uint32_t fresh = __reduce_or_sync(0xffffffffu, lane < run ? 1u << off_i : 0u);
    const uint32_t older = ((1u << (31 - __clz(fresh))) - 1) & ~fresh;  // cells below the last new one
    uint8_t* const sc = p.scales + (size_t)(slot >> 4) * p.block_scales + p.layer_scale + h;
    const uint32_t had_byte = *sc;
    const SRC* const src = reinterpret_cast<const SRC*>(p.qkv) + (size_t)(p.H + h) * DH + lane * N;
    float* const mine = stage + lane * N;
    float amax = 0.f;
    constexpr int U = 4;  // rows loaded together
#pragma unroll 1
    for (int i0 = 0; i0 < run; i0 += U) {
        float v[U][N];
        int row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            row[u] = __shfl_sync(0xffffffffu, row_i, (i0 + u) & 31);
            if (i0 + u < run) load_row<N>(src + (size_t)row[u] * p.qkv_stride, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u < run) {
                if (key) norm_rotate<DH, N>(p, p.k_gain, row[u], lane, v[u]);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float a = fabsf(v[u][j]);
                    amax = a <= 3.402823466e38f ? fmaxf(amax, a) : amax;  // finite values only
                }
                store_row<N>(mine + (i0 + u) * DH, v[u]);
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
    for (int i = 0; i < run; ++i) {
        float v[N];
        load_row<N>(mine + i * DH, v);  // (this lane's own values)
        uint8_t* const o = cells + (size_t)__shfl_sync(0xffffffffu, off_i, i) * DH + lane * N;
        const uint32_t a = e4m3x2_from(v[0] * f, v[1] * f);
        if constexpr (N == 2) {
            *reinterpret_cast<uint16_t*>(o) = (uint16_t)a;
        } else {
            const uint32_t b = a | (e4m3x2_from(v[2] * f, v[3] * f) << 16);
            if constexpr (N == 4) {
                *reinterpret_cast<uint32_t*>(o) = b;
            } else {
                const uint32_t c = e4m3x2_from(v[4] * f, v[5] * f) | (e4m3x2_from(v[6] * f, v[7] * f) << 16);
                *reinterpret_cast<uint2*>(o) = make_uint2(b, c);
            }
        }
    }
}

// The first row_blocks CTAs take single rows, the others (e4m3) blocks: a warp
// looks at `tile` consecutive rows (at most 16) for those that begin a block.
// Bytes bound it: every row is read once.  What the shape is after is loads in
// flight: ROWS rows a warp where there are rows enough (4: 8192 tokens), one
// where there are not (decode), and values in shared memory rather than
// registers so that 28 warps share an SM.
template <typename SRC, typename DST, bool E4M3, int DH, int ROWS>
__global__ void __launch_bounds__(128, DH == 256 ? 3 : 7) kv_append_kernel(const __grid_constant__ AppendParams p, unsigned row_blocks, int tile) {
    extern __shared__ __align__(16) float append_stage[];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x < row_blocks) {
        append_rows<SRC, DST, E4M3, DH, ROWS>(p, ((long long)blockIdx.x * 4 + warp) * ROWS, lane);
        return;
    }
    if constexpr (E4M3) {
        const long long task = (long long)(blockIdx.x - row_blocks) * 4 + warp;
        const int t0 = (int)(task / (2 * p.G)) * tile, h = (int)(task % (2 * p.G));
        if (t0 >= p.T) return;
        const int s = lane < tile && t0 + lane < p.T ? p.slots[t0 + lane] : -1;
        uint32_t live = __ballot_sync(0xffffffffu, s >= 0);
        // the nearest earlier row that is not padding: of the same block, it (or one before it) stores this row too
        int before = -1;
        for (int back = t0 - 1; back >= 0; back -= 32) {
            const int x = back - lane >= 0 ? p.slots[back - lane] : -1;
            const uint32_t m = __ballot_sync(0xffffffffu, x >= 0);
            if (m) {
                before = __shfl_sync(0xffffffffu, x, __ffs(m) - 1) >> 4;
                break;
            }
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
    const long long rows = (long long)p.T * (E4M3 ? p.H : p.H + 2 * p.G);
    const long long warps = (long long)sms * 28;
    const int per_warp = rows >= 4 * warps ? 4 : 1;
    const unsigned row_blocks = (unsigned)((rows + 4 * per_warp - 1) / (4 * per_warp));
    // rows a warp looks through: 16 once that still fills the device
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
            for (auto* f : {kv_append_kernel<SRC, DST, E4M3, DH, 4>, kv_append_kernel<SRC, DST, E4M3, DH, 1>})
                if (const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); e != cudaSuccess)
                    return e;
            ready.fetch_or(bit, std::memory_order_release);
        }
    }
    if (per_warp == 4)
        return launch_on(st, pdl, kv_append_kernel<SRC, DST, E4M3, DH, 4>, row_blocks + blocks, 128, smem, p, row_blocks, tile);
    return launch_on(st, pdl, kv_append_kernel<SRC, DST, E4M3, DH, 1>, row_blocks + blocks, 128, smem, p, row_blocks, tile);
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
        return yk::kv_append_launch(static_cast<cudaStream_t>(stream), false, sms, *args);
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
        return yk::attention_e4m3_launch(static_cast<cudaStream_t>(stream), false, sms, *args);
    });
}
