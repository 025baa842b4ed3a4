// yk_attention_e4m3.cu -- causal attention of a ragged batch over an e4m3 paged
// KV cache (yk_attention_e4m3).
#include <algorithm>
#include <cmath>

#include "yk_epilogue.cuh"
#include "yk_kvcache.cuh"

namespace yk {

struct Attn8Params {
    const void* q;
    void* out;
    const uint8_t* pool;
    const uint8_t* scales;
    const int32_t *q_starts, *ctx, *tables;
    uint32_t* err;
    long long q_stride, out_stride;
    long long block_cells, layer_off, block_scales, layer_scale;
    int T, B, H, G, max_blocks, num_blocks;
    int window;
    float scale, cap;
};

// One warp per (token, head), one key at a time.
template <typename AT, int DH>
__global__ void __launch_bounds__(128) attn8_simt_kernel(Attn8Params p) {
    constexpr int N = DH / 32;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    if (blockIdx.x == 0) {  // q_starts must run from 0, never fall, and end within T
        bool bad = threadIdx.x == 0 && p.q_starts[0] != 0;
        for (int b = threadIdx.x; b < p.B; b += 128)
            bad |= p.q_starts[b + 1] < p.q_starts[b] || p.q_starts[b + 1] > p.T;
        if (bad) raise_err(p.err, YK_DEV_ERR_BOUNDS);
    }
    const long long task = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int t = (int)(task / p.H), h = (int)(task % p.H);
    if (t >= p.T || t >= p.q_starts[p.B]) return;
    int lo = 0, hi = p.B - 1;  // the sequence: the first b with q_starts[b + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (p.q_starts[mid + 1] > t) hi = mid; else lo = mid + 1;
    }
    const int b = lo;
    const int pos = p.ctx[b] - (p.q_starts[b + 1] - t);
    const int g = h / (p.H / p.G);
    float q[N], o[N];
    const AT* qr = reinterpret_cast<const AT*>(p.q) + (size_t)t * p.q_stride + (size_t)h * DH + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        q[i] = to_f32(qr[i]);
        o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int jend = min(pos + 1, p.max_blocks * 16);
    if (jend < pos + 1 && lane == 0) raise_err(p.err, YK_DEV_ERR_BOUNDS);
    for (int j = p.window > 0 ? max(0, pos - p.window + 1) : 0; j < jend; ++j) {
        const int blk = p.tables[(size_t)b * p.max_blocks + (j >> 4)];
        if (blk < 0 || blk >= p.num_blocks) {
            if (lane == 0) raise_err(p.err, YK_DEV_ERR_BOUNDS);
            continue;
        }
        const uint8_t* sc = p.scales + (size_t)blk * p.block_scales + p.layer_scale + g;
        const uint8_t* kc = p.pool + (size_t)blk * p.block_cells + p.layer_off + ((size_t)g * 16 + (j & 15)) * DH + lane * N;
        const uint8_t* vc = kc + (size_t)p.G * 16 * DH;
        float dot = 0.f, v[N];
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 k2 = f32x2(f16x2_lo(*reinterpret_cast<const uint16_t*>(kc + i)));
            const float2 v2 = f32x2(f16x2_lo(*reinterpret_cast<const uint16_t*>(vc + i)));
            dot = fmaf(q[i], k2.x, fmaf(q[i + 1], k2.y, dot));
            v[i] = v2.x;
            v[i + 1] = v2.y;
        }
        float s = warp_sum_f(dot) * exp2_int(kv8_exponent(sc[0])) * p.scale;
        if (p.cap > 0.f) s = p.cap * tanhf(s / p.cap);
        const float mn = fmaxf(m, s);
        const float c = expf(m - mn), w = expf(s - mn);  // m = -inf at first: c = 0
        const float vs = exp2_int(kv8_exponent(sc[p.G]));
        l = l * c + w;
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(w, v[i] * vs, o[i] * c);
        m = mn;
    }
    AT* orow = reinterpret_cast<AT*>(p.out) + (size_t)t * p.out_stride + (size_t)h * DH + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) orow[i] = from_f32<AT>(l == 0.f ? 0.f : o[i] / l);
}

size_t attention_e4m3_ws_bytes(int num_sms, int head_dim) {
    (void)num_sms;
    (void)head_dim;
    return 16;
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

template <typename AT>
static cudaError_t launch_simt8(cudaStream_t st, bool pdl, int dh, const Attn8Params& p) {
    const unsigned blocks = (unsigned)(((long long)p.T * p.H + 3) / 4);
    switch (dh) {
        case 64: return launch_on(st, pdl, attn8_simt_kernel<AT, 64>, blocks, 128, 0, p);
        case 128: return launch_on(st, pdl, attn8_simt_kernel<AT, 128>, blocks, 128, 0, p);
        default: return launch_on(st, pdl, attn8_simt_kernel<AT, 256>, blocks, 128, 0, p);
    }
}

yk_status attention_e4m3_launch(cudaStream_t st, bool pdl, int num_sms, const yk_attention_e4m3_args& a) {
    (void)num_sms;
    if (a.T == 0) return YK_OK;
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
    p.layer_off = p.layer_scale * YK_BLOCK_SIZE * a.pages.head_dim;
    p.block_cells = p.block_scales * YK_BLOCK_SIZE * a.pages.head_dim;
    p.T = a.T;
    p.B = a.B;
    p.H = a.n_heads;
    p.G = a.pages.n_kv_heads;
    p.max_blocks = a.max_blocks;
    p.num_blocks = a.pages.num_blocks;
    p.window = a.window;
    p.scale = a.scale > 0.f ? a.scale : 1.0f / std::sqrt((float)a.pages.head_dim);
    p.cap = a.cap;
    YK_CHECK_CUDA(a.dtype == YK_DTYPE_BF16 ? launch_simt8<__nv_bfloat16>(st, pdl, a.pages.head_dim, p)
                                           : launch_simt8<float>(st, pdl, a.pages.head_dim, p));
    return YK_OK;
}

}  // namespace yk
