// What stands between two blocks of a residual stream, as one pass over the rows (any part may be left out):
//     u = x silu(gate)                 the block's gate
//     p = w_post u / rms(u)            the norm after the block        rms(v) = sqrt(mean v^2 + eps)
//     r = residual + scale p           the stream                      (the output p if there is no residual)
//     n = w_pre r / rms(r)             the norm before the next block
// Rows are read once and written once (three inputs, two outputs: ten bytes a bfloat16 element, about 16 operations), so
// HBM bounds both directions.  A thread holds eight elements of a row in fp32: rows of up to 512 elements are one wave, wider
// ones a block of up to sixteen.  Blocks walk over rows.  Forward, the weights stay in registers; backward in LDS (a wave a SIMD
// more, and bfloat16 rows of 8192 without spills: 4096 x 8192 299 -> 114 us; fp32 rows above 4096, at the 128 registers that a
// block of 1024 threads leaves, still spill 18: 4096 x 8192 221 us, 4.9 TB/s), the weights' gradients as partial sums in
// registers, added up in a fixed order by a second kernel.  Measured (medians): forward 16387 x 2048 bf16 63 us (5.3 TB/s),
// 16032 x 1285 fp32 77 us (5.3 TB/s), backward 111 us (4.8 TB/s) and 139 us (4.7 TB/s) and 5 for the sums; 64 rows of 2048 in 4 us.
#include "seq_common.hpp"

#include <type_traits>

namespace unetmi {

constexpr int kElems = 8;                // of a row, per thread

struct NormArgs {
    const void *x, *gate;                 // gate may be null
    const float *post, *scale, *pre;      // null: that part is left out (scale: 1)
    const void* residual;
    long long xs, gs, rs;                 // elements between rows
    long long rows;
    int D;
    float eps;
    void *out_r, *out_n;                  // r (or p without a residual), n
    float* stats;                         // [rows, 2]: 1 / rms(u), 1 / rms(r); null in inference
    // backward
    const void *d_r, *d_n;                // null: zero
    void *dx, *dgate, *dres;
    float* partial;                       // [workers, 3, D]: post, scale, pre
};

__device__ __forceinline__ float row_sum16(float v) {                 // over the lane's row of 16
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x124>(v);
    return v + dpp<0x128>(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    v = row_sum16(v);
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// threadIdx.y, which is the same for a wave: a block has one row, or a row per wave
__device__ __forceinline__ int wave_row() { return __builtin_amdgcn_readfirstlane(threadIdx.y); }

// Sums over a row's threads.  One wave: no LDS.  More: the two halves of `red` are used in turn, so that one barrier per
// call is enough.
struct RowSum {
    float* red;                           // [2][16][3]
    int waves, wave, turn = 0;
    template <int M>
    __device__ __forceinline__ void operator()(float (&v)[M]) {
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = wave_sum(v[m]);
        if (waves == 1) return;
        float* mine = red + turn * 48;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int m = 0; m < M; ++m) mine[wave * 3 + m] = v[m];
        __syncthreads();
        const int w = threadIdx.x & 15;                               // every sixteen lanes add up the waves' sums
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = w < waves ? mine[w * 3 + m] : 0.f;
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = row_sum16(v[m]);
    }
};

// a thread's elements of a row: E / V vectors, `width` threads apart.  The row's start is the same for a wave (scalar registers)
// and a thread's place in it an offset of 32 bits: a dozen 64-bit addresses a thread would cost the backward kernel a wave a SIMD.
template <class T>
__device__ __forceinline__ T* within(T* row, int c) {
    typedef std::conditional_t<std::is_const_v<T>, const char, char> byte;
    return reinterpret_cast<T*>(reinterpret_cast<byte*>(row) + (unsigned)c * (unsigned)sizeof(T));
}
template <class T, int V, int E>
__device__ __forceinline__ void load_row(float (&o)[E], const void* p, long long row, int D, int col, int width) {
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
        const int c = (j * width + col) * V;
        Pack<T, V> k;
        k.zero();
        if (c < D) k.load_n(within(static_cast<const T*>(p) + row, c), D - c);
#pragma unroll
        for (int v = 0; v < V; ++v) o[j * V + v] = k.get(v);
    }
}
template <class T, int V, int E>
__device__ __forceinline__ void store_row(const float (&o)[E], void* p, long long row, int D, int col, int width) {
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
        const int c = (j * width + col) * V;
        Pack<T, V> k;
#pragma unroll
        for (int v = 0; v < V; ++v) k.set(v, o[j * V + v]);
        if (c < D) k.store_n(within(static_cast<T*>(p) + row, c), D - c);
    }
}

template <class T, class RT>
__global__ __launch_bounds__(1024) void block_norm_fwd_kernel(NormArgs a) {
    constexpr int V = kVector<T>, E = kElems;
    __shared__ float red[96];
    const int width = blockDim.x, col = threadIdx.x;
    RowSum sum{red, width >> 6, col >> 6};
    float post[E], scale[E], pre[E];
    if (a.post) load_row<float, V, E>(post, a.post, 0, a.D, col, width);
    if (a.scale) load_row<float, V, E>(scale, a.scale, 0, a.D, col, width);
    if (a.pre) load_row<float, V, E>(pre, a.pre, 0, a.D, col, width);
    const float inv_d = 1.f / (float)a.D;
    for (long long row = (long long)blockIdx.x * blockDim.y + wave_row(); row < a.rows; row += (long long)gridDim.x * blockDim.y) {
        float u[E], r[E];
        load_row<T, V, E>(u, a.x, row * a.xs, a.D, col, width);
        if (a.residual) load_row<RT, V, E>(r, a.residual, row * a.rs, a.D, col, width);
        if (a.gate) {
            float z[E];
            load_row<T, V, E>(z, a.gate, row * a.gs, a.D, col, width);
#pragma unroll
            for (int i = 0; i < E; ++i) u[i] *= z[i] * sigmoid_hw(z[i]);
        }
        if (a.post) {
            float s[1] = {0.f};
#pragma unroll
            for (int i = 0; i < E; ++i) s[0] = fmaf(u[i], u[i], s[0]);
            sum(s);
            const float inv = __builtin_amdgcn_rsqf(fmaf(s[0], inv_d, a.eps));
            if (a.stats && col == 0) a.stats[2 * row] = inv;
#pragma unroll
            for (int i = 0; i < E; ++i) u[i] *= inv * post[i];
        }
        if (!a.residual) {
            store_row<T, V, E>(u, a.out_r, row * a.D, a.D, col, width);
            continue;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) r[i] = a.scale ? fmaf(scale[i], u[i], r[i]) : r[i] + u[i];
        store_row<RT, V, E>(r, a.out_r, row * a.D, a.D, col, width);
        if (a.pre) {
            float s[1] = {0.f};
#pragma unroll
            for (int i = 0; i < E; ++i) s[0] = fmaf(r[i], r[i], s[0]);
            sum(s);
            const float inv = __builtin_amdgcn_rsqf(fmaf(s[0], inv_d, a.eps));
            if (a.stats && col == 0) a.stats[2 * row + 1] = inv;
#pragma unroll
            for (int i = 0; i < E; ++i) r[i] *= inv * pre[i];
            store_row<T, V, E>(r, a.out_n, row * a.D, a.D, col, width);
        }
    }
}

// Backward.  With f = 1 / rms(r), e = 1 / rms(u) as the forward call saved them:
//     dr = d_r + f (g - r f^2 mean(g r)),  g = d_n w_pre          dw_pre = sum_rows d_n r f
//     dresidual = dr,  dscale = sum dr p,  dp = scale dr            (without a residual dp = d_r)
//     du = e (q - u e^2 mean(q u)),  q = dp w_post                  dw_post = sum dp u e
//     dx = du silu(gate),  dgate = du x silu'(gate)
// With the rows in units of their rms, v = u e and n = r f, and w = scale w_post, the second mean is linear in the first one,
//     m = f mean(g n),  dr = d_r + f g - m n,  sum(q v) = sum(w v (d_r + f g)) - m sum(w v n),
// so the three sums are taken together and a row waits once (16032 x 1285 fp32: 175 us with e, f and the means one after the
// other).  r is computed again from the residual, which has to be read anyway: a stream stored in 16 bits would leave its
// rounding in the weights' gradients (2e-3 of dscale and dw_pre over a few rows).
template <class T, class RT, int THREADS>
__global__ __launch_bounds__(THREADS) void block_norm_bwd_kernel(NormArgs a) {
    constexpr int V = kVector<T>, E = kElems;
    __shared__ float red[96];
    extern __shared__ f32x4 own[];        // [post, scale, pre][half][thread of a row]
    const int width = blockDim.x, col = threadIdx.x;
    RowSum sum{red, width >> 6, col >> 6};
    float d_post[E], d_scale[E], d_pre[E];
#pragma unroll
    for (int i = 0; i < E; ++i) d_post[i] = d_scale[i] = d_pre[i] = 0.f;
    if (threadIdx.y == 0) {
        const float* const w[3] = {a.post, a.scale, a.pre};
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            float v[E];
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = 1.f;
            if (w[k]) load_row<float, V, E>(v, w[k], 0, a.D, col, width);
            own[2 * k * width + col] = f32x4{v[0], v[1], v[2], v[3]};
            own[(2 * k + 1) * width + col] = f32x4{v[4], v[5], v[6], v[7]};
        }
    }
    __syncthreads();
    auto weight = [&](int k, int half) { return own[(2 * k + half) * width + col]; };
    const float inv_d = 1.f / (float)a.D;
    const bool with_pre = a.pre && a.d_n;
    const long long worker = (long long)blockIdx.x * blockDim.y + wave_row();
    for (long long row = worker; row < a.rows; row += (long long)gridDim.x * blockDim.y) {
        float x[E], z[E], g[E], r[E], dn[E];
        load_row<T, V, E>(x, a.x, row * a.xs, a.D, col, width);
#pragma unroll
        for (int i = 0; i < E; ++i) g[i] = 0.f;
        if (a.d_r) {
            if (a.dres) load_row<RT, V, E>(g, a.d_r, row * a.D, a.D, col, width);
            else load_row<T, V, E>(g, a.d_r, row * a.D, a.D, col, width);
        }
        if (a.gate) load_row<T, V, E>(z, a.gate, row * a.gs, a.D, col, width);
        if (with_pre) {
            load_row<RT, V, E>(r, a.residual, row * a.rs, a.D, col, width);
            load_row<T, V, E>(dn, a.d_n, row * a.D, a.D, col, width);
        }
        const float e = a.post ? a.stats[2 * row] : 1.f, f = with_pre ? a.stats[2 * row + 1] : 0.f;
        float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 w = weight(0, h) * weight(1, h), pre = weight(2, h);
            float wv[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) wv[k] = w[k] * (x[4 * h + k] * e);
            if (a.gate) {
#pragma unroll
                for (int k = 0; k < 4; ++k) wv[k] *= z[4 * h + k] * sigmoid_hw(z[4 * h + k]);
            }
            if (with_pre) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i = 4 * h + k;
                    r[i] = (r[i] + wv[k]) * f;
                    d_pre[i] = fmaf(dn[i], r[i], d_pre[i]);
                    const float dp = dn[i] * pre[k];
                    s[0] = fmaf(dp, r[i], s[0]);
                    g[i] = fmaf(f, dp, g[i]);
                    s[2] = fmaf(wv[k], r[i], s[2]);
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) s[1] = fmaf(wv[k], g[4 * h + k], s[1]);
        }
        if (with_pre || a.post) sum(s);
        const float m = f * (s[0] * inv_d), mv = a.post ? (s[1] - m * s[2]) * inv_d : 0.f;
        if (with_pre) {
#pragma unroll
            for (int i = 0; i < E; ++i) g[i] = fmaf(-r[i], m, g[i]);
        }
        if (a.dres) store_row<RT, V, E>(g, a.dres, row * a.D, a.D, col, width);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const f32x4 post = weight(0, h), scale = weight(1, h);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = 4 * h + k;
                const float sg = a.gate ? sigmoid_hw(z[i]) : 1.f, silu = a.gate ? z[i] * sg : 1.f;
                const float v = x[i] * e * silu, dp = g[i] * scale[k];
                d_scale[i] = fmaf(g[i], v * post[k], d_scale[i]);
                d_post[i] = fmaf(dp, v, d_post[i]);
                const float du = e * fmaf(-v, mv, dp * post[k]);
                g[i] = du * silu;
                if (a.gate) z[i] = du * x[i] * sg * fmaf(z[i], 1.f - sg, 1.f);
            }
        }
        if (a.gate) store_row<T, V, E>(z, a.dgate, row * a.D, a.D, col, width);
        store_row<T, V, E>(g, a.dx, row * a.D, a.D, col, width);
    }
    float* out = a.partial + worker * 3 * a.D;
    store_row<float, V, E>(d_post, out, 0, a.D, col, width);
    store_row<float, V, E>(d_scale, out, a.D, a.D, col, width);
    store_row<float, V, E>(d_pre, out, 2 * (long long)a.D, a.D, col, width);
}

namespace {

struct NormPlan {
    int width, per_block;                 // threads per row, rows per block
    unsigned blocks;
};

NormPlan norm_plan(const UnetmiNormDesc& d, long long most_blocks) {
    NormPlan p;
    p.width = ((d.channels + kElems - 1) / kElems + 63) / 64 * 64;
    p.per_block = p.width == 64 ? 4 : 1;
    long long n = (d.rows + p.per_block - 1) / p.per_block;
    p.blocks = (unsigned)(n < 1 ? 1 : (n > most_blocks ? most_blocks : n));
    return p;
}

// Waves per CU: forward 64, about three times what is resident, so that CUs that end early find work (16387 x 2048 bf16: 61 us,
// 67 with 32 and 65 with 16; 16032 x 1285 fp32: 81, 78 and 85).
long long fwd_blocks(const UnetmiNormDesc& d) { const NormPlan p = norm_plan(d, 1); return 256 * 64 / (p.width * p.per_block / 64); }
// Backward: whole blocks a CU, all resident (every block more costs 12 bytes a column of partial sums, and 1.2 blocks a CU take
// as long as two), sixteen waves of them with 16-bit activations and eight with fp32, whose rows are twice the bytes: 16387 x 2048
// bf16 145, 119 and 110 us with 8, 12 and 16 waves, 16032 x 1285 bf16 194, 127 and 115, fp32 139, 151 and 156.  More where a
// thread would add up more than 1024 rows of the weights' gradients in one running sum, which may be off by a rounding a row.
long long bwd_blocks(const UnetmiNormDesc& d) {
    const NormPlan p = norm_plan(d, 1);
    const int per_cu = (d.dtype == UNETMI_DTYPE_BF16 ? 16 : 8) / (p.width * p.per_block / 64);
    const long long resident = 256 * (per_cu ? per_cu : 1), long_sums = (d.rows + 1024 * p.per_block - 1) / (1024 * p.per_block);
    return resident > long_sums ? resident : long_sums;
}

int norm_check(const UnetmiNormDesc* d, const char* what) {
    const std::string w = what;
    if (!d) return api_fail(UNETMI_E_BAD_ARG, w + ": null descriptor");
    if (d->rows < 0 || d->channels < 1) return api_fail(UNETMI_E_BAD_DESC, w + ": bad sizes");
    if (d->channels > 8192) return api_fail(UNETMI_E_UNSUPPORTED, w + ": rows of at most 8192 elements are built");
    if (d->dtype != UNETMI_DTYPE_F32 && d->dtype != UNETMI_DTYPE_BF16) return api_fail(UNETMI_E_UNSUPPORTED, w + ": fp32 or bfloat16 activations");
    if (d->residual_dtype != d->dtype && d->residual_dtype != UNETMI_DTYPE_F32)
        return api_fail(UNETMI_E_UNSUPPORTED, w + ": the residual stream is fp32 or of the activations' type");
    if (!(d->eps >= 0.f)) return api_fail(UNETMI_E_BAD_DESC, w + ": eps must not be negative");
    if (d->x_stride < 0 || d->gate_stride < 0 || d->residual_stride < 0) return api_fail(UNETMI_E_BAD_DESC, w + ": negative stride");
    return UNETMI_OK;
}

template <class T, class RT, bool BWD>
int norm_launch(const NormArgs& a, const NormPlan& p, hipStream_t s) {
    const dim3 block(p.width, p.per_block);
    const size_t lds = 6 * sizeof(f32x4) * p.width;
    if (BWD && p.width <= 512) hipLaunchKernelGGL((block_norm_bwd_kernel<T, RT, 512>), dim3(p.blocks), block, lds, s, a);
    else if (BWD) hipLaunchKernelGGL((block_norm_bwd_kernel<T, RT, 1024>), dim3(p.blocks), block, lds, s, a);
    else hipLaunchKernelGGL((block_norm_fwd_kernel<T, RT>), dim3(p.blocks), block, 0, s, a);
    return launched(BWD ? "block_norm_bwd" : "block_norm_fwd");
}

template <bool BWD>
int norm_dispatch(const UnetmiNormDesc& d, const NormArgs& a, const NormPlan& p, hipStream_t s) {
    if (d.dtype == UNETMI_DTYPE_F32) return norm_launch<float, float, BWD>(a, p, s);
    return d.residual_dtype == UNETMI_DTYPE_F32 ? norm_launch<__bf16, float, BWD>(a, p, s) : norm_launch<__bf16, __bf16, BWD>(a, p, s);
}

NormArgs norm_args(const UnetmiNormDesc& d, const void* x, const void* gate, const float* post, const void* residual, const float* scale,
                   const float* pre) {
    NormArgs a = {};
    a.x = x; a.gate = gate; a.post = post; a.residual = residual; a.scale = scale; a.pre = pre;
    a.xs = d.x_stride; a.gs = gate ? d.gate_stride : 0; a.rs = residual ? d.residual_stride : 0;
    a.rows = d.rows; a.D = d.channels; a.eps = d.eps;
    return a;
}

}  // namespace
}  // namespace unetmi

using namespace unetmi;

extern "C" {

int unetmi_block_norm_fwd(const UnetmiNormDesc* d, const void* x, const void* gate, const float* post_weight, const void* residual,
                          const float* scale, const float* pre_weight, void* out, void* out_norm, float* stats, void* stream) {
    const int rc = norm_check(d, "block_norm_fwd");
    if (rc != UNETMI_OK) return rc;
    if (d->rows == 0) return UNETMI_OK;
    if (!x || !out || (pre_weight && !out_norm)) return api_fail(UNETMI_E_BAD_ARG, "block_norm_fwd: null tensor pointer");
    if (!residual && (pre_weight || scale)) return api_fail(UNETMI_E_BAD_ARG, "block_norm_fwd: scale and pre_weight belong to a residual stream");
    NormArgs a = norm_args(*d, x, gate, post_weight, residual, scale, pre_weight);
    a.out_r = out; a.out_n = out_norm; a.stats = stats;
    return norm_dispatch<false>(*d, a, norm_plan(*d, fwd_blocks(*d)), static_cast<hipStream_t>(stream));
}

size_t unetmi_block_norm_bwd_workspace_bytes(const UnetmiNormDesc* d) {
    if (norm_check(d, "block_norm_bwd_workspace_bytes") != UNETMI_OK) return 0;
    const NormPlan p = norm_plan(*d, bwd_blocks(*d));
    return (size_t)p.blocks * p.per_block * 3 * d->channels * sizeof(float);
}

int unetmi_block_norm_bwd(const UnetmiNormDesc* d, const void* x, const void* gate, const float* post_weight, const void* residual,
                          const float* scale, const float* pre_weight, const float* stats, const void* d_out, const void* d_norm, void* dx, void* dgate,
                          void* dresidual, float* dweights, void* ws, size_t ws_bytes, void* stream) {
    const int rc = norm_check(d, "block_norm_bwd");
    if (rc != UNETMI_OK) return rc;
    if (d->rows == 0) return api_fail(UNETMI_E_BAD_DESC, "block_norm_bwd: no rows");
    if (!x || !dx || !dweights || !ws || (gate && !dgate) || (pre_weight && d_norm && !residual) || ((post_weight || (pre_weight && d_norm)) && !stats))
        return api_fail(UNETMI_E_BAD_ARG, "block_norm_bwd: null tensor pointer");
    if (!dresidual && (pre_weight || scale)) return api_fail(UNETMI_E_BAD_ARG, "block_norm_bwd: scale and pre_weight belong to a residual stream");
    if (ws_bytes < unetmi_block_norm_bwd_workspace_bytes(d)) return api_fail(UNETMI_E_BAD_ARG, "block_norm_bwd: workspace too small");
    NormArgs a = norm_args(*d, x, gate, post_weight, residual, scale, pre_weight);
    a.stats = const_cast<float*>(stats); a.d_r = d_out; a.d_n = d_norm; a.dx = dx; a.dgate = dgate; a.dres = dresidual;
    a.partial = static_cast<float*>(ws);
    const NormPlan p = norm_plan(*d, bwd_blocks(*d));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int done = norm_dispatch<true>(*d, a, p, s);
    if (done != UNETMI_OK) return done;
    return launch_sum_rows(a.partial, (int)(p.blocks * p.per_block), {dweights, 3 * d->channels, 1, 1}, {nullptr, 0, 1, 0}, {nullptr, 0, 1, 0}, s);
}

}  // extern "C"
