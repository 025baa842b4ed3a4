// yk_kvcache.cu -- yk_kv_append: per-head norms, rotation and the store into a
// paged KV cache, in one pass over the QKV projections.
#include <algorithm>
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

// One warp per (token, head).  Query heads: norm, rotation, store.  Key and
// value heads of fp32 / bf16 pools: the same into the token's slot.  e4m3 pools:
// the block's scale couples its tokens, so the warp of a block's first new token
// takes all of them (at most 16, held in registers) and the warps of the others
// have nothing to do.
template <typename SRC, typename DST, bool E4M3, int DH>
__global__ void __launch_bounds__(128) kv_append_kernel(AppendParams p) {
    constexpr int N = DH / 32;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int heads = p.H + 2 * p.G;
    const long long task = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(task / heads), h = (int)(task % heads);
    if (t >= p.T) return;
    const int slot = p.slots[t];
    if (slot < 0) return;  // padding
    if ((slot >> 4) >= p.num_blocks) {
        if (lane == 0) raise_err(p.err, YK_DEV_ERR_BOUNDS);
        if (h >= p.H) return;  // its query is computed all the same
    }
    const SRC* src = reinterpret_cast<const SRC*>(p.qkv) + (size_t)t * p.qkv_stride + (size_t)h * DH + lane * N;
    if (h < p.H) {
        float v[N];
        load_row<N>(src, v);
        norm_rotate<DH, N>(p, p.q_gain, t, lane, v);
        store_row<N>(reinterpret_cast<DST*>(p.q_out) + (size_t)t * p.q_stride + (size_t)h * DH + lane * N, v);
        return;
    }
    const bool key = h < p.H + p.G;
    const int cell_head = h - p.H;  // K heads, then V heads: the pool's order
    const int off = slot & 15;
    const size_t page = (size_t)(slot >> 4) * p.block_cells + p.layer_off + (size_t)cell_head * 16 * DH;
    if constexpr (!E4M3) {
        float v[N];
        load_row<N>(src, v);
        if (key) norm_rotate<DH, N>(p, p.k_gain, t, lane, v);
        store_row<N>(reinterpret_cast<DST*>(p.pool) + page + (size_t)off * DH + lane * N, v);
    } else {
        // the nearest earlier row that is not padding: of this block, it (or one
        // before it) stores this token too
        for (int back = t - 1; back >= 0; back -= 32) {
            const int s = back - lane >= 0 ? p.slots[back - lane] : -1;
            const uint32_t live = __ballot_sync(0xffffffffu, s >= 0);
            if (live) {
                if (__shfl_sync(0xffffffffu, s, __ffs(live) - 1) >> 4 == slot >> 4) return;
                break;
            }
        }
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
        const uint32_t older = (1u << (31 - __clz(fresh))) - 1 & ~fresh;  // cells below the last new one
        float v[16][N];
        int row[16], cell[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            row[i] = __shfl_sync(0xffffffffu, row_i, i);
            cell[i] = __shfl_sync(0xffffffffu, off_i, i);
            if (i < run) load_row<N>(src + (size_t)(row[i] - t) * p.qkv_stride, v[i]);
        }
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i < run) {
                if (key) norm_rotate<DH, N>(p, p.k_gain, row[i], lane, v[i]);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float a = fabsf(v[i][j]);
                    amax = a <= 3.402823466e38f ? fmaxf(amax, a) : amax;  // finite values only
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        int e = kv8_cover(amax);
        uint8_t* const sc = p.scales + (size_t)(slot >> 4) * p.block_scales + p.layer_scale + cell_head;
        uint8_t* const cells = reinterpret_cast<uint8_t*>(p.pool) + page;
        if (older) {
            const int had = kv8_exponent(*sc);
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
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i < run) {
                uint8_t* const o = cells + (size_t)cell[i] * DH + lane * N;
                const uint32_t a = e4m3x2_from(v[i][0] * f, v[i][1] * f);
                if constexpr (N == 2) {
                    *reinterpret_cast<uint16_t*>(o) = (uint16_t)a;
                } else {
                    const uint32_t b = a | (e4m3x2_from(v[i][2] * f, v[i][3] * f) << 16);
                    if constexpr (N == 4) {
                        *reinterpret_cast<uint32_t*>(o) = b;
                    } else {
                        const uint32_t c = e4m3x2_from(v[i][4] * f, v[i][5] * f) |
                                           (e4m3x2_from(v[i][6] * f, v[i][7] * f) << 16);
                        *reinterpret_cast<uint2*>(o) = make_uint2(b, c);
                    }
                }
            }
        }
    }
}

template <typename SRC, typename DST, bool E4M3>
static cudaError_t launch_append(cudaStream_t st, bool pdl, int dh, const AppendParams& p) {
    const long long tasks = (long long)p.T * (p.H + 2 * p.G);
    const unsigned blocks = (unsigned)((tasks + 3) / 4);
    switch (dh) {
        case 64: return launch_on(st, pdl, kv_append_kernel<SRC, DST, E4M3, 64>, blocks, 128, 0, p);
        case 128: return launch_on(st, pdl, kv_append_kernel<SRC, DST, E4M3, 128>, blocks, 128, 0, p);
        default: return launch_on(st, pdl, kv_append_kernel<SRC, DST, E4M3, 256>, blocks, 128, 0, p);
    }
}

yk_status kv_append_launch(cudaStream_t st, bool pdl, const yk_kv_append_args& a) {
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
        r = e4 ? launch_append<__nv_bfloat16, __nv_bfloat16, true>(st, pdl, dh, p)
               : launch_append<__nv_bfloat16, __nv_bfloat16, false>(st, pdl, dh, p);
    } else if (a.q_dtype == YK_DTYPE_BF16) {
        r = e4 ? launch_append<float, __nv_bfloat16, true>(st, pdl, dh, p)
               : launch_append<float, __nv_bfloat16, false>(st, pdl, dh, p);
    } else {
        r = e4 ? launch_append<float, float, true>(st, pdl, dh, p) : launch_append<float, float, false>(st, pdl, dh, p);
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
    int n = 0, prev = 0, sms = 0;
    if (const cudaError_t e = cudaGetDeviceCount(&n); e != cudaSuccess) {
        cudaGetLastError();  // (not left pending for the next call)
        yk_set_error(std::string(what) + ": " + cudaGetErrorString(e));
        return YK_ERR_CUDA;
    }
    YK_ARG(device >= 0 && device < n, "device index");
    YK_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
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
    return yk::on_device(device, "yk_kv_append", [&](int) {
        return yk::kv_append_launch(static_cast<cudaStream_t>(stream), false, *args);
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
