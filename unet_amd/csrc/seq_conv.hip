// Short causal convolution along time, channels innermost (x [batch, length, channels]):
//     y_t = act(bias + sum_k w_k x_{t-K+1+k}),   K = 2..4, act = SiLU or none,
// over the K-1 inputs before the first one (a state, or zeros), its gradients and its form for single tokens.
// Two or three operations per tap against one read and one write of HBM: the traffic bounds all three kernels.  A thread
// keeps four channels and walks along time with the last K-1 inputs in registers, so a row is read once per time segment plus
// K-1 rows that the caches still hold.  Four also of 16 bits, 512 bytes a wave and row: eight take so many registers that two
// waves a SIMD remain of four (8 x 4096 x 2048 bf16 forward 54 -> 47 us, backward 113 -> 98; 32 x 501 x 768 13.8 -> 11.1 and 31
// -> 27).  Measured (medians): forward 32 x 501 x 768 fp32 20 us (4.9 TB/s), 8 x 4096 x 2048 bf16 of lengths 0..4096 40 us;
// backward of the former 36 us (4.1 TB/s) and 4 for the sums; 256 tokens x 2048 channels bf16 4 us.
#include "seq_common.hpp"

namespace unetmi {

constexpr int kConvV = 4;               // channels per thread

struct ConvSeqArgs {
    const void* x;
    long long xb, xt;                  // elements between sequences / steps of x
    const float *w, *bias;             // [D, K], [D] or null
    const void* state;                 // [B, K-1, D] or null
    const int* lengths;                // [B] or null
    int B, L, D;
    int steps;                         // time steps per thread
    int cw_log2;                       // threads along the channel vectors = 1 << cw_log2
};

template <bool ACT>
__device__ __forceinline__ float conv_act(float v) { return ACT ? v * sigmoid_hw(v) : v; }

// input at time t (t < 0: the state's rows, or zero)
template <class T, int V, int K>
__device__ __forceinline__ Pack<T, V> conv_input(const ConvSeqArgs& a, int b, int t, int ch) {
    Pack<T, V> p;
    if (t >= 0) p.load_n(static_cast<const T*>(a.x) + b * a.xb + t * a.xt + ch, a.D - ch);
    else if (a.state) p.load_n(static_cast<const T*>(a.state) + ((size_t)b * (K - 1) + (t + K - 1)) * a.D + ch, a.D - ch);
    else p.zero();
    return p;
}
// the taps and bias of the n channels (at most V) from ch on
template <int V, int K>
__device__ __forceinline__ void conv_weights(const float* w, const float* bias, int ch, int n, float (&wk)[K][V], float (&b)[V]) {
    Pack<float, V * K> rows;
    rows.load_n(w + (size_t)ch * K, n >= V ? V * K : n * K);
    Pack<float, V> bs;
    bs.zero();
    if (bias) bs.load_n(bias + ch, n);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        b[v] = bs.get(v);
#pragma unroll
        for (int k = 0; k < K; ++k) wk[k][v] = rows.get(v * K + k);
    }
}

// TAIL: the channels are no multiple of V, the last vector of a row holds fewer (guarded accesses for every width took 51 us
// where the whole vectors take 43).
template <class T, int V, int K, bool ACT, bool TAIL>
__global__ __launch_bounds__(256) void conv_seq_kernel(ConvSeqArgs a, T* __restrict__ y, T* __restrict__ state_out) {
    const int cw = 1 << a.cw_log2;
    const int ch = (blockIdx.x * cw + (threadIdx.x & (cw - 1))) * V;
    const int seg = blockIdx.y * (256 >> a.cw_log2) + (threadIdx.x >> a.cw_log2);
    const int b = blockIdx.z;
    if (ch >= a.D) return;
    const int t0 = seg * a.steps, t1 = min(t0 + a.steps, a.L);
    const int len = seq_len(a.lengths, b, a.L);
    // the state after the sequence: the last K-1 of [state, x[:len]]; the first time segment writes it
    if (state_out && seg == 0) {
#pragma unroll
        for (int i = 0; i < K - 1; ++i)
            conv_input<T, V, K>(a, b, len - (K - 1) + i, ch).store_n(state_out + ((size_t)b * (K - 1) + i) * a.D + ch, a.D - ch);
    }
    if (t0 >= t1) return;
    const int n = TAIL ? a.D - ch : V;
    float w[K][V], bias[V];
    conv_weights<V, K>(a.w, a.bias, ch, n, w, bias);
    T* out = y + ((size_t)b * a.L + t0) * a.D + ch;
    const int tend = min(t1, len);
    float win[K - 1][V];
    if (t0 < tend) {
#pragma unroll
        for (int i = 0; i < K - 1; ++i) {
            const Pack<T, V> p = conv_input<T, V, K>(a, b, t0 - (K - 1) + i, ch);
#pragma unroll
            for (int v = 0; v < V; ++v) win[i][v] = p.get(v);
        }
    }
    const T* in = static_cast<const T*>(a.x) + b * a.xb + t0 * a.xt + ch;
    int t = t0;
    for (; t + 4 <= tend; t += 4) {                     // four rows in flight
        Pack<T, V> r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { r[i].load_n(in, n); in += a.xt; }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Pack<T, V> o;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x = r[i].get(v);
                float s = bias[v];
#pragma unroll
                for (int k = 0; k < K - 1; ++k) s = fmaf(w[k][v], win[k][v], s);
                s = fmaf(w[K - 1][v], x, s);
#pragma unroll
                for (int k = 0; k + 1 < K - 1; ++k) win[k][v] = win[k + 1][v];
                win[K - 2][v] = x;
                o.set(v, conv_act<ACT>(s));
            }
            o.store_n(out, n);
            out += a.D;
        }
    }
    for (; t < tend; ++t) {
        Pack<T, V> r, o;
        r.load_n(in, n);
        in += a.xt;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float x = r.get(v);
            float s = bias[v];
#pragma unroll
            for (int k = 0; k < K - 1; ++k) s = fmaf(w[k][v], win[k][v], s);
            s = fmaf(w[K - 1][v], x, s);
#pragma unroll
            for (int k = 0; k + 1 < K - 1; ++k) win[k][v] = win[k + 1][v];
            win[K - 2][v] = x;
            o.set(v, conv_act<ACT>(s));
        }
        o.store_n(out, n);
        out += a.D;
    }
    Pack<T, V> zero;
    zero.zero();
    for (; t < t1; ++t, out += a.D) zero.store_n(out, n);    // behind the sequence's end
}

// Gradients.  A thread owns the steps [t0, t1): it adds their share of dw and db, and writes dx there, for which it
// needs the pre-activation gradients of [t0, t1 + K-1): K-1 rows more at each end than the forward kernel.
//     dpre_t = dy_t act'(pre_t),   dx_t = sum_k w_k dpre_{t+K-1-k},   dw_k = sum dpre_t x_{t-K+1+k},   db = sum dpre_t
// The time segments of a block are added up through LDS and a block writes one row of partial sums [K+1][D]; a second
// kernel adds the rows in a fixed order.
template <class T, int V, int K, bool ACT, bool TAIL>
__global__ __launch_bounds__(256) void conv_seq_bwd_kernel(ConvSeqArgs a, const T* __restrict__ dy, long long dyb, long long dyt,
                                                           const T* __restrict__ dstate_out, T* __restrict__ dx,
                                                           float* __restrict__ partial) {
    const int cw = 1 << a.cw_log2, nseg = 256 >> a.cw_log2;
    const int lane_c = threadIdx.x & (cw - 1), row = threadIdx.x >> a.cw_log2;
    const int ch0 = (blockIdx.x * cw + lane_c) * V;
    const bool live = ch0 < a.D;
    const int ch = live ? ch0 : 0;
    const int b = blockIdx.z;
    const int t0 = min((int)(blockIdx.y * nseg + row) * a.steps, a.L), t1 = min(t0 + a.steps, a.L);
    const int len = seq_len(a.lengths, b, a.L);
    const int n = TAIL ? a.D - ch : V;
    float w[K][V], bias[V], dw[K][V], db[V];
    conv_weights<V, K>(a.w, a.bias, ch, n, w, bias);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        db[v] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) dw[k][v] = 0.f;
    }
    const int tend = min(t1, len);
    T* out = dx + ((size_t)b * a.L) * a.D + ch;
    if (live && t0 < tend) {
        float win[K - 1][V], dp[K - 1][V];
#pragma unroll
        for (int i = 0; i < K - 1; ++i) {
            const Pack<T, V> p = conv_input<T, V, K>(a, b, t0 - (K - 1) + i, ch);
#pragma unroll
            for (int v = 0; v < V; ++v) { win[i][v] = p.get(v); dp[i][v] = 0.f; }
        }
        const T* in = static_cast<const T*>(a.x) + b * a.xb + t0 * a.xt + ch;
        const T* gin = dy + b * dyb + t0 * dyt + ch;
        // step t brings dpre_t; dx_{t-K+1} is then complete
        for (int t = t0; t < tend + K - 1; ++t) {
            Pack<T, V> r, g;
            r.zero();
            g.zero();
            if (t < len) { r.load_n(in, n); g.load_n(gin, n); }
            in += a.xt;
            gin += dyt;
            Pack<T, V> o;
            const int to = t - (K - 1);
            Pack<T, V> extra;
            const int si = to - len + (K - 1);          // dx of the last K-1 inputs also comes from the state behind them
            const bool has_extra = dstate_out && si >= 0 && to >= t0;
            if (has_extra) extra.load_n(dstate_out + ((size_t)b * (K - 1) + si) * a.D + ch, n);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x = r.get(v);
                float pre = bias[v];
#pragma unroll
                for (int k = 0; k < K - 1; ++k) pre = fmaf(w[k][v], win[k][v], pre);
                pre = fmaf(w[K - 1][v], x, pre);
                float d = g.get(v);
                if (ACT) {
                    const float s = sigmoid_hw(pre);
                    d *= s * fmaf(pre, 1.f - s, 1.f);
                }
                if (t >= len) d = 0.f;
                if (t < tend) {
                    db[v] += d;
#pragma unroll
                    for (int k = 0; k < K - 1; ++k) dw[k][v] = fmaf(d, win[k][v], dw[k][v]);
                    dw[K - 1][v] = fmaf(d, x, dw[K - 1][v]);
                }
                float sum = w[0][v] * d;                // dpre_t, dpre_{t-1}, ... meet w_0, w_1, ...
#pragma unroll
                for (int k = 1; k < K; ++k) sum = fmaf(w[k][v], dp[K - 1 - k][v], sum);
                if (has_extra) sum += extra.get(v);
                o.set(v, sum);
#pragma unroll
                for (int k = 0; k + 1 < K - 1; ++k) { win[k][v] = win[k + 1][v]; dp[k][v] = dp[k + 1][v]; }
                win[K - 2][v] = x;
                dp[K - 2][v] = d;
            }
            if (to >= t0) o.store_n(out + (size_t)to * a.D, n);
        }
    }
    if (live) {
        Pack<T, V> zero;
        zero.zero();
        for (int t = max(t0, tend); t < t1; ++t) zero.store_n(out + (size_t)t * a.D, n);
    }
    // add the block's time segments: [segment][tap or bias][thread along channels][V]
    extern __shared__ float red[];
    float* mine = red + (size_t)threadIdx.x * (K + 1) * V;
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int k = 0; k < K; ++k) mine[k * V + v] = dw[k][v];
        mine[K * V + v] = db[v];
    }
    __syncthreads();
    const size_t base = ((size_t)b * gridDim.y + blockIdx.y) * (size_t)a.D * (K + 1);
    for (int e = threadIdx.x; e < cw * (K + 1) * V; e += 256) {
        const int c = (blockIdx.x * cw + e / ((K + 1) * V)) * V + e % V;
        if (c >= a.D) continue;
        float s = 0.f;
        for (int i = 0; i < nseg; ++i) s += red[(size_t)i * cw * (K + 1) * V + e];
        const int k = (e / V) % (K + 1);
        partial[base + (k < K ? (size_t)c * K + k : (size_t)a.D * K + c)] = s;
    }
}

// Gradient of the initial state: row j of it is the input at time j - (K-1) < 0.
template <class T, int K, bool ACT>
__global__ __launch_bounds__(256) void conv_seq_dstate_kernel(ConvSeqArgs a, const T* __restrict__ dy, long long dyb, long long dyt,
                                                              const T* __restrict__ dstate_out, T* __restrict__ dstate) {
    const int ch = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    if (ch >= a.D) return;
    const int len = seq_len(a.lengths, b, a.L);
    float w[K], in[2 * K - 2], d[K - 1], g[K - 1];
#pragma unroll
    for (int k = 0; k < K; ++k) w[k] = a.w[ch * K + k];
#pragma unroll
    for (int i = 0; i < 2 * K - 2; ++i) {
        const int t = i - (K - 1);
        in[i] = t >= 0 ? (t < len ? widen(static_cast<const T*>(a.x)[b * a.xb + t * a.xt + ch]) : 0.f)
                       : (a.state ? widen(static_cast<const T*>(a.state)[((size_t)b * (K - 1) + i) * a.D + ch]) : 0.f);
    }
#pragma unroll
    for (int t = 0; t < K - 1; ++t) {                    // the steps whose window reaches before the first input
        float pre = a.bias ? a.bias[ch] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) pre = fmaf(w[k], in[t + k], pre);
        float v = t < len ? widen(dy[b * dyb + t * dyt + ch]) : 0.f;
        if (ACT) {
            const float s = sigmoid_hw(pre);
            v *= s * fmaf(pre, 1.f - s, 1.f);
        }
        d[t] = t < len ? v : 0.f;
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        g[j] = 0.f;
#pragma unroll
        for (int t = 0; t <= j; ++t) g[j] = fmaf(w[j - t], d[t], g[j]);
        const int si = j - len;                          // a short sequence leaves rows of the old state in the new one
        if (dstate_out && si >= 0) g[j] += widen(dstate_out[((size_t)b * (K - 1) + si) * a.D + ch]);
        dstate[((size_t)b * (K - 1) + j) * a.D + ch] = (T)g[j];
    }
}

// One token of every row: the window is the slot's K-1 old inputs and the new one; the slot is shifted in place.
template <class T, int V, int K, bool ACT>
__global__ __launch_bounds__(256) void conv_seq_step_kernel(const T* __restrict__ x, long long xb, const float* __restrict__ w,
                                                            const float* __restrict__ bias, const int* __restrict__ slots,
                                                            int nslots, T* __restrict__ state, T* __restrict__ y, int D) {
    const int row = blockIdx.y;
    bool bad;
    const int slot = claim_slot(slots, row, nslots, &bad);
    const int ch = (blockIdx.x * 256 + threadIdx.x) * V;
    if (ch >= D) return;
    Pack<T, V> o;
    if (bad || slot < 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) o.set(v, bad ? __builtin_nanf("") : 0.f);
        o.store_n(y + (size_t)row * D + ch, D - ch);
        return;
    }
    T* st = state + (size_t)slot * (K - 1) * D + ch;
    const int n = D - ch;
    Pack<T, V> r[K];
#pragma unroll
    for (int i = 0; i < K - 1; ++i) r[i].load_n(st + (size_t)i * D, n);
    r[K - 1].load_n(x + row * xb + ch, n);
    float wk[K][V], b[V];
    conv_weights<V, K>(w, bias, ch, n, wk, b);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float s = b[v];
#pragma unroll
        for (int k = 0; k < K; ++k) s = fmaf(wk[k][v], r[k].get(v), s);
        o.set(v, conv_act<ACT>(s));
    }
    o.store_n(y + (size_t)row * D + ch, n);
#pragma unroll
    for (int i = 0; i < K - 1; ++i) r[i + 1].store_n(st + (size_t)i * D, n);
}

// ---------------------------------------------------------------------------------------------------------------------
// sums of partial rows (shared by the sequence operators)
// ---------------------------------------------------------------------------------------------------------------------
// 32 columns a block, the rows over 32 groups of threads, eight loads of each in flight: one row of partial sums is a few
// thousand columns, so columns alone would leave most of the chip idle (683 rows of 3855: 24 us with 8 groups).
__global__ __launch_bounds__(1024) void sum_rows_kernel(const float* __restrict__ rows, int R, SumPiece a, SumPiece b, SumPiece c) {
    const int width = a.columns + b.columns + c.columns;
    const int part = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int col = blockIdx.x * 32 + lane;
    float s = 0.f;
    if (col < width) {
        int r = part;
        for (; r + 7 * 32 < R; r += 8 * 32) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = rows[(size_t)(r + k * 32) * width + col];
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; r < R; r += 32) s += rows[(size_t)r * width + col];
    }
    __shared__ float red[32][33];
    red[part][lane] = s;
    __syncthreads();
    if (part != 0 || col >= width) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += red[k][lane];
    SumPiece p = a;
    if (col >= p.columns) { col -= p.columns; p = b; }
    if (col >= p.columns) { col -= p.columns; p = c; }
    const int g = col / p.padded, n = col - g * p.padded;
    if (n < p.used) p.out[(size_t)g * p.used + n] = s;
}

int launch_sum_rows(const float* rows, int R, SumPiece a, SumPiece b, SumPiece c, hipStream_t s) {
    const int width = a.columns + b.columns + c.columns;
    hipLaunchKernelGGL(sum_rows_kernel, dim3((width + 31) / 32), dim3(1024), 0, s, rows, R, a, b, c);
    return launched("sum of partial rows");
}

namespace {

struct ConvSeqPlan {
    int cw_log2, steps, nblk_t, nblk_c;
};

// threads along the channels: as many (a power of two, at most a wave) as there are channel vectors; the rest of the
// block along time.  steps = rows per thread: 32 as long as that leaves two blocks a CU, down to 8 on short or narrow
// inputs, where each row that two threads share is read twice (backward of 32 x 501 x 768 fp32: 36 us with 16 rows and 768
// blocks, 41 with 8; forward of 8 x 4096 x 2048 bf16: 43.5 us with 32 rows, 45.6 with 16).
ConvSeqPlan conv_plan(const UnetmiSeqConvDesc& d) {
    ConvSeqPlan p;
    const int nv = (d.channels + kConvV - 1) / kConvV;
    p.cw_log2 = 0;
    while ((1 << p.cw_log2) < nv && p.cw_log2 < 6) ++p.cw_log2;
    p.nblk_c = (nv + (1 << p.cw_log2) - 1) >> p.cw_log2;
    const int nseg = 256 >> p.cw_log2;
    p.steps = 32;
    while (p.steps > 8 && (long long)d.batch * p.nblk_c * ((d.length + p.steps * nseg - 1) / (p.steps * nseg)) < 512) p.steps /= 2;
    p.nblk_t = (d.length + p.steps * nseg - 1) / (p.steps * nseg);
    return p;
}

int conv_check(const UnetmiSeqConvDesc* d, const char* what) {
    if (!d) return api_fail(UNETMI_E_BAD_ARG, std::string(what) + ": null descriptor");
    if (d->batch < 0 || d->length < 0 || d->channels < 1) return api_fail(UNETMI_E_BAD_DESC, std::string(what) + ": bad sizes");
    if (d->taps < 2 || d->taps > 4) return api_fail(UNETMI_E_UNSUPPORTED, std::string(what) + ": 2, 3 or 4 taps are built");
    if (d->act != UNETMI_ACT_NONE && d->act != UNETMI_ACT_SILU) return api_fail(UNETMI_E_UNSUPPORTED, std::string(what) + ": activation none or SiLU");
    if (d->dtype != UNETMI_DTYPE_F32 && d->dtype != UNETMI_DTYPE_BF16) return api_fail(UNETMI_E_UNSUPPORTED, std::string(what) + ": fp32 or bfloat16 activations");
    if (d->batch > 65535) return api_fail(UNETMI_E_UNSUPPORTED, std::string(what) + ": more than 65535 sequences");
    if (d->channels > (1 << 24) || d->length > (1 << 28)) return api_fail(UNETMI_E_UNSUPPORTED, std::string(what) + ": more than 2^24 channels or 2^28 steps");
    if (d->x_stride[0] < 0 || d->x_stride[1] < 0 || d->dy_stride[0] < 0 || d->dy_stride[1] < 0) return api_fail(UNETMI_E_BAD_DESC, std::string(what) + ": negative stride");
    return UNETMI_OK;
}

ConvSeqArgs conv_args(const UnetmiSeqConvDesc& d, const ConvSeqPlan& p, const void* x, const float* w, const float* bias,
                      const void* state, const int* lengths) {
    ConvSeqArgs a;
    a.x = x; a.xb = d.x_stride[0]; a.xt = d.x_stride[1];
    a.w = w; a.bias = bias; a.state = state; a.lengths = lengths;
    a.B = d.batch; a.L = d.length; a.D = d.channels;
    a.steps = p.steps; a.cw_log2 = p.cw_log2;
    return a;
}

// F<T, V, K, ACT>() for the descriptor's type, vector width, taps and activation
template <template <class, int, int, bool> class F, class T, int V, class... A>
int conv_taps(const UnetmiSeqConvDesc& d, A&&... args) {
    const bool act = d.act == UNETMI_ACT_SILU;
    switch (d.taps) {
        case 2: return act ? F<T, V, 2, true>::run(args...) : F<T, V, 2, false>::run(args...);
        case 3: return act ? F<T, V, 3, true>::run(args...) : F<T, V, 3, false>::run(args...);
        default: return act ? F<T, V, 4, true>::run(args...) : F<T, V, 4, false>::run(args...);
    }
}
template <template <class, int, int, bool> class F, class... A>
int conv_dispatch(const UnetmiSeqConvDesc& d, A&&... args) {
    return d.dtype == UNETMI_DTYPE_BF16 ? conv_taps<F, __bf16, kConvV>(d, args...) : conv_taps<F, float, kConvV>(d, args...);
}

template <class T, int V, int K, bool ACT>
struct RunFwd {
    static int run(const ConvSeqArgs& a, const ConvSeqPlan& p, void* y, void* state_out, hipStream_t s) {
        const dim3 grid(p.nblk_c, p.nblk_t > 0 ? p.nblk_t : 1, a.B), block(256);
        T *out = static_cast<T*>(y), *after = static_cast<T*>(state_out);
        if (a.D % V) hipLaunchKernelGGL((conv_seq_kernel<T, V, K, ACT, true>), grid, block, 0, s, a, out, after);
        else hipLaunchKernelGGL((conv_seq_kernel<T, V, K, ACT, false>), grid, block, 0, s, a, out, after);
        return launched("seq_conv_fwd");
    }
};
template <class T, int V, int K, bool ACT>
struct RunBwd {
    static int run(const ConvSeqArgs& a, const ConvSeqPlan& p, const UnetmiSeqConvDesc& d, const void* dy, const void* dstate_out,
                   void* dx, void* dstate, float* dw, float* db, float* partial, hipStream_t s) {
        const T* g = static_cast<const T*>(dy);
        const T* gs = static_cast<const T*>(dstate_out);
        const int nt = p.nblk_t > 0 ? p.nblk_t : 1;
        const dim3 grid(p.nblk_c, nt, a.B), block(256);
        const size_t lds = 256 * (K + 1) * V * sizeof(float);
        const long long yb = d.dy_stride[0], yt = d.dy_stride[1];
        if (a.D % V) hipLaunchKernelGGL((conv_seq_bwd_kernel<T, V, K, ACT, true>), grid, block, lds, s, a, g, yb, yt, gs, static_cast<T*>(dx), partial);
        else hipLaunchKernelGGL((conv_seq_bwd_kernel<T, V, K, ACT, false>), grid, block, lds, s, a, g, yb, yt, gs, static_cast<T*>(dx), partial);
        int rc = launched("seq_conv_bwd");
        if (rc != UNETMI_OK) return rc;
        if (dstate) {
            hipLaunchKernelGGL((conv_seq_dstate_kernel<T, K, ACT>), dim3((a.D + 255) / 256, a.B), dim3(256), 0, s, a, g,
                               d.dy_stride[0], d.dy_stride[1], gs, static_cast<T*>(dstate));
            rc = launched("seq_conv_bwd state");
            if (rc != UNETMI_OK) return rc;
        }
        return launch_sum_rows(partial, a.B * nt, {dw, a.D * K, 1, 1}, {db, a.D, 1, 1}, {nullptr, 0, 1, 0}, s);
    }
};
template <class T, int V, int K, bool ACT>
struct RunStep {
    static int run(const UnetmiSeqConvDesc& d, const void* x, const float* w, const float* bias, const int* slots, int nslots,
                   void* state, void* y, hipStream_t s) {
        hipLaunchKernelGGL((conv_seq_step_kernel<T, V, K, ACT>), dim3((d.channels + 256 * V - 1) / (256 * V), d.batch), dim3(256), 0, s,
                           static_cast<const T*>(x), (long long)d.x_stride[0], w, bias, slots, nslots, static_cast<T*>(state),
                           static_cast<T*>(y), d.channels);
        return launched("seq_conv_step");
    }
};

}  // namespace
}  // namespace unetmi

using namespace unetmi;

extern "C" {

int unetmi_seq_conv_fwd(const UnetmiSeqConvDesc* d, const void* x, const float* weight, const float* bias, const void* state,
                        const int32_t* lengths, void* y, void* state_out, void* stream) {
    const int rc = conv_check(d, "seq_conv_fwd");
    if (rc != UNETMI_OK) return rc;
    if (d->batch == 0) return UNETMI_OK;
    if (!weight || (d->length > 0 && (!x || !y))) return api_fail(UNETMI_E_BAD_ARG, "seq_conv_fwd: null tensor pointer");
    if (d->length == 0 && !state_out) return UNETMI_OK;
    const ConvSeqPlan p = conv_plan(*d);
    if (p.nblk_t > 65535) return api_fail(UNETMI_E_UNSUPPORTED, "seq_conv_fwd: too many steps");
    return conv_dispatch<RunFwd>(*d, conv_args(*d, p, x, weight, bias, state, lengths), p, y, state_out,
                                 static_cast<hipStream_t>(stream));
}

size_t unetmi_seq_conv_bwd_workspace_bytes(const UnetmiSeqConvDesc* d) {
    if (conv_check(d, "seq_conv_bwd") != UNETMI_OK) return 0;
    const ConvSeqPlan p = conv_plan(*d);
    return (size_t)(d->batch > 0 ? d->batch : 1) * (p.nblk_t > 0 ? p.nblk_t : 1) * d->channels * (d->taps + 1) * sizeof(float);
}

int unetmi_seq_conv_bwd(const UnetmiSeqConvDesc* d, const void* x, const float* weight, const float* bias, const void* state,
                        const int32_t* lengths, const void* dy, const void* dstate_out, void* dx, float* dweight, float* dbias,
                        void* dstate, void* ws, size_t ws_bytes, void* stream) {
    const int rc = conv_check(d, "seq_conv_bwd");
    if (rc != UNETMI_OK) return rc;
    if (d->batch == 0) return api_fail(UNETMI_E_BAD_DESC, "seq_conv_bwd: empty batch");
    if (!weight || !dweight || !dbias || !ws || (d->length > 0 && (!x || !dy || !dx)))
        return api_fail(UNETMI_E_BAD_ARG, "seq_conv_bwd: null tensor pointer");
    if (ws_bytes < unetmi_seq_conv_bwd_workspace_bytes(d)) return api_fail(UNETMI_E_BAD_ARG, "seq_conv_bwd: workspace too small");
    const ConvSeqPlan p = conv_plan(*d);
    if (p.nblk_t > 65535) return api_fail(UNETMI_E_UNSUPPORTED, "seq_conv_bwd: too many steps");
    return conv_dispatch<RunBwd>(*d, conv_args(*d, p, x, weight, bias, state, lengths), p, *d, dy, dstate_out, dx, dstate,
                                 dweight, dbias, static_cast<float*>(ws), static_cast<hipStream_t>(stream));
}

int unetmi_seq_conv_step(const UnetmiSeqConvDesc* d, const void* x, const float* weight, const float* bias, const int32_t* slots,
                         int num_slots, void* state, void* y, void* stream) {
    const int rc = conv_check(d, "seq_conv_step");
    if (rc != UNETMI_OK) return rc;
    if (d->batch == 0) return UNETMI_OK;
    if (!x || !weight || !state || !y) return api_fail(UNETMI_E_BAD_ARG, "seq_conv_step: null tensor pointer");
    if (num_slots < 0 || (!slots && num_slots < d->batch)) return api_fail(UNETMI_E_BAD_ARG, "seq_conv_step: fewer slots than rows");
    return conv_dispatch<RunStep>(*d, *d, x, weight, bias, slots, num_slots, state, y, static_cast<hipStream_t>(stream));
}

}  // extern "C"
