// Selective state space scan, channels innermost (x, dt, z [batch, length, channels], B, C [batch, length, groups, state]):
//     dt  = softplus(raw + bias)                     (or raw + bias)
//     h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t       A [channels, N], N <= 64
//     y_t = (C_t . h_t + D x_t) silu(z_t)
// its gradients, and its form for single tokens.
//
// Lanes: the four lanes of a quad share one channel and hold N/4 states each, so 64 channels make a block of 256 threads.
// (One lane per channel would save the quad's exchanges but leave a batch of 8 with 2048 channels at 256 waves, a quarter
// of the chip.)  Per time step and state: a product and an exponential for the decay, a product and two multiply-adds --
// N of them against eight bytes of traffic per step and channel, so the vector units bound the kernel, not HBM.  What is
// per step and channel (softplus, gate) is done by one lane of the quad for one of four consecutive steps and handed to the
// others by DPP operands; the four partial sums of y are transposed and added the same way.  B and C of a tile of steps,
// the same for all channels, are widened into LDS once per block.  States and sums are fp32.
#include "seq_common.hpp"

namespace unetmi {

constexpr int kTile = 16;                 // steps per tile of the forward kernels
constexpr int kCh = 64;                   // channels per block

// steps between two saved states, = the steps the backward kernel keeps in registers
template <int S> constexpr int mark_steps() { return S <= 4 ? 16 : 64 / S; }
static int mark_steps_of(int S) { return S <= 4 ? 16 : 64 / S; }

struct ScanArgs {
    const void *x, *dt, *z, *Bm, *Cm;     // z may be null
    const float *A, *Dp, *bias, *h0;      // Dp, bias, h0 may be null
    const int* lengths;
    long long xb, xt, dtb, dtt, zb, zt, bb, bt, bg, cb, ct, cg;      // element strides
    int L, D, N, Dg, tpg;                 // channels per group, blocks per group
    int chunk, nchunk;                    // steps per chunk (a multiple of kTile)
    int nmark;
    bool softplus;
    void* y;
    float *hT, *marks;                    // [B, D, N]; [B, nmark, D, 4S]
    float *hend, *sdt;                    // chunk summaries [B, nchunk, D, 4S], [B, nchunk, D]
    // backward
    const void* dy;
    long long dyb, dyt;
    const float* dhT;
    void *dx, *ddt, *dz;
    float *dh0, *pBC, *pA, *pD;           // [B, L, G, tpg, 2, 4S]; [B nchunk, D, 4S]; [B nchunk, 2, D]
};

struct Place {                            // what a thread works on
    int b, g, ch, q, len;
    bool live;
    int row0;                             // thread's place in the block's 64 channels
};

__device__ __forceinline__ Place place(const ScanArgs& a, int b) {
    Place p;
    p.b = b;
    p.g = blockIdx.x / a.tpg;
    p.q = threadIdx.x & 3;
    p.row0 = threadIdx.x >> 2;
    const int in_group = (blockIdx.x - p.g * a.tpg) * kCh + p.row0;
    p.live = in_group < a.Dg;
    p.ch = p.g * a.Dg + (p.live ? in_group : 0);
    p.len = seq_len(a.lengths, b, a.L);
    return p;
}

// a lane's states: elements q*S .. q*S+S-1 of a row of N (0 beyond)
template <int S>
__device__ __forceinline__ void load_states(float (&h)[S], const float* p, int q, int N) {
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = q * S + s < N ? p[q * S + s] : 0.f;
}
template <int S>
__device__ __forceinline__ void store_states(const float (&h)[S], float* p, int q, int N) {
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (q * S + s < N) p[q * S + s] = h[s];
}
// the same on the padded rows of 4S that only these kernels see
template <int S>
__device__ __forceinline__ void load_padded(float (&h)[S], const float* p, int q) {
    Pack<float, S> v;
    v.load(p + q * S);
#pragma unroll
    for (int s = 0; s < S; ++s) h[s] = v.get(s);
}
template <int S>
__device__ __forceinline__ void store_padded(const float (&h)[S], float* p, int q) {
    Pack<float, S> v;
#pragma unroll
    for (int s = 0; s < S; ++s) v.set(s, h[s]);
    v.store(p + q * S);
}

// B (and C) of STEPS steps from t on into LDS as fp32 [step][4S], zero beyond tend and beyond N
template <class T, int S, int STEPS>
__device__ __forceinline__ void stage_rows(float* lds, const void* src, long long base, long long stride, int t, int tend, int N) {
    constexpr int NP = 4 * S;
#pragma unroll
    for (int e = threadIdx.x; e < STEPS * NP; e += 256) {
        const int i = e / NP, n = e % NP;
        lds[e] = (t + i < tend && n < N) ? widen(static_cast<const T*>(src)[base + (t + i) * stride + n]) : 0.f;
    }
}

template <class T>
__device__ __forceinline__ float at(const void* p, long long i) { return widen(static_cast<const T*>(p)[i]); }

// Forward.  STATE_ONLY: the first pass over a time axis that is split into chunks: the chunk's last state from zero and
// the sum of its steps (the product of its decays is exp(A sum dt)).  Else the whole operator on a chunk, starting from
// the states of the chunks before it.
template <class T, int S, bool STATE_ONLY>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanArgs a) {
    constexpr int NP = 4 * S, MK = mark_steps<S>();
    __shared__ float lds_b[kTile * NP], lds_c[STATE_ONLY ? 1 : kTile * NP];
    const Place p = place(a, blockIdx.z);
    const int chunk = blockIdx.y, t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.L), tend = min(t1, p.len);
    float A2[S], h[S];
    load_states<S>(A2, a.A + (size_t)p.ch * a.N, p.q, a.N);
#pragma unroll
    for (int s = 0; s < S; ++s) { A2[s] *= kLog2e; h[s] = 0.f; }
    const float bias = a.bias ? a.bias[p.ch] : 0.f, dskip = a.Dp ? a.Dp[p.ch] : 0.f;
    if (!STATE_ONLY) {
        if (a.h0) load_states<S>(h, a.h0 + ((size_t)p.b * a.D + p.ch) * a.N, p.q, a.N);
        for (int k = 0; k < chunk; ++k) {
            const size_t row = ((size_t)p.b * a.nchunk + k) * a.D + p.ch;
            float e[S];
            load_padded<S>(e, a.hend + row * NP, p.q);
            const float sd = a.sdt[row];
#pragma unroll
            for (int s = 0; s < S; ++s) h[s] = fmaf(exp2_hw(A2[s] * sd), h[s], e[s]);
        }
    }
    float sdt = 0.f;
    for (int t = t0; t < tend; t += kTile) {
        __syncthreads();
        stage_rows<T, S, kTile>(lds_b, a.Bm, p.b * a.bb + p.g * a.bg, a.bt, t, tend, a.N);
        if (!STATE_ONLY) stage_rows<T, S, kTile>(lds_c, a.Cm, p.b * a.cb + p.g * a.cg, a.ct, t, tend, a.N);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i) {
            if (!STATE_ONLY && a.marks && (4 * i) % MK == 0 && t + 4 * i < tend && p.live)
                store_padded<S>(h, a.marks + (((size_t)p.b * a.nmark + (t + 4 * i) / MK) * a.D + p.ch) * NP, p.q);
            const int own = t + 4 * i + p.q;
            const bool in = own < tend && p.live;
            float x = 0.f, dt = 0.f;
            if (in) {
                x = at<T>(a.x, p.b * a.xb + own * a.xt + p.ch);
                dt = at<T>(a.dt, p.b * a.dtb + own * a.dtt + p.ch) + bias;
                if (a.softplus) dt = softplus_exact(dt);
            }
            const float u = dt * x;
            sdt += dt;
            float part[4];
            auto step = [&](int j, float dtj, float uj) {
                const float* bj = lds_b + (4 * i + j) * NP + p.q * S;
                const float* cj = lds_c + (STATE_ONLY ? 0 : (4 * i + j) * NP + p.q * S);
                float y = 0.f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    h[s] = fmaf(exp2_hw(A2[s] * dtj), h[s], uj * bj[s]);
                    if (!STATE_ONLY) y = fmaf(h[s], cj[s], y);
                }
                part[j] = y;
            };
            step(0, quad_lane<0>(dt), quad_lane<0>(u));
            step(1, quad_lane<1>(dt), quad_lane<1>(u));
            step(2, quad_lane<2>(dt), quad_lane<2>(u));
            step(3, quad_lane<3>(dt), quad_lane<3>(u));
            if (!STATE_ONLY) {
                float y = fmaf(dskip, x, quad_sum_of_own(part[0], part[1], part[2], part[3], p.q));
                if (in) {
                    if (a.z) {
                        const float z = at<T>(a.z, p.b * a.zb + own * a.zt + p.ch);
                        y *= z * sigmoid_hw(z);
                    }
                    static_cast<T*>(a.y)[((size_t)p.b * a.L + own) * a.D + p.ch] = (T)y;
                }
            }
        }
    }
    if (STATE_ONLY) {
        const size_t row = ((size_t)p.b * a.nchunk + chunk) * a.D + p.ch;
        sdt = quad_sum(sdt);
        if (p.live) {
            store_padded<S>(h, a.hend + row * NP, p.q);
            if (p.q == 0) a.sdt[row] = sdt;
        }
        return;
    }
    if (a.hT && chunk == a.nchunk - 1 && p.live) store_states<S>(h, a.hT + ((size_t)p.b * a.D + p.ch) * a.N, p.q, a.N);
    if (p.live)                                                       // behind the sequence's end
        for (int t = max(t0, tend) + p.q; t < t1; t += 4) static_cast<T*>(a.y)[((size_t)p.b * a.L + t) * a.D + p.ch] = (T)0.f;
}

// The first backward pass over a split time axis: the adjoint that a chunk hands to the chunk before it, from zero,
// and the sum of its steps.
template <class T, int S>
__global__ __launch_bounds__(256) void scan_bwd_state_kernel(ScanArgs a) {
    constexpr int NP = 4 * S;
    __shared__ float lds_c[kTile * NP];
    const Place p = place(a, blockIdx.z);
    const int chunk = blockIdx.y, t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.L), tend = min(t1, p.len);
    float A2[S], g[S];
    load_states<S>(A2, a.A + (size_t)p.ch * a.N, p.q, a.N);
#pragma unroll
    for (int s = 0; s < S; ++s) { A2[s] *= kLog2e; g[s] = 0.f; }
    const float bias = a.bias ? a.bias[p.ch] : 0.f;
    float sdt = 0.f;
    for (int k = (tend - t0 + kTile - 1) / kTile - 1; k >= 0; --k) {
        const int t = t0 + k * kTile;
        __syncthreads();
        stage_rows<T, S, kTile>(lds_c, a.Cm, p.b * a.cb + p.g * a.cg, a.ct, t, tend, a.N);
        __syncthreads();
#pragma unroll
        for (int i = kTile / 4 - 1; i >= 0; --i) {
            const int own = t + 4 * i + p.q;
            const bool in = own < tend && p.live;
            float dt = 0.f, dy = 0.f;
            if (in) {
                dt = at<T>(a.dt, p.b * a.dtb + own * a.dtt + p.ch) + bias;
                if (a.softplus) dt = softplus_exact(dt);
                dy = at<T>(a.dy, p.b * a.dyb + own * a.dyt + p.ch);
                if (a.z) {
                    const float z = at<T>(a.z, p.b * a.zb + own * a.zt + p.ch);
                    dy *= z * sigmoid_hw(z);
                }
            }
            sdt += dt;
            auto step = [&](int j, float dtj, float dyj) {
                const float* cj = lds_c + (4 * i + j) * NP + p.q * S;
#pragma unroll
                for (int s = 0; s < S; ++s) g[s] = exp2_hw(A2[s] * dtj) * fmaf(dyj, cj[s], g[s]);
            };
            step(3, quad_lane<3>(dt), quad_lane<3>(dy));
            step(2, quad_lane<2>(dt), quad_lane<2>(dy));
            step(1, quad_lane<1>(dt), quad_lane<1>(dy));
            step(0, quad_lane<0>(dt), quad_lane<0>(dy));
        }
    }
    const size_t row = ((size_t)p.b * a.nchunk + chunk) * a.D + p.ch;
    sdt = quad_sum(sdt);
    if (p.live) {
        store_padded<S>(g, a.hend + row * NP, p.q);
        if (p.q == 0) a.sdt[row] = sdt;
    }
}

// sum over the 16 channels of a wave (lanes of one place in their quads); every lane gets it
__device__ __forceinline__ float channel_sum(float v) {
    v += dpp<0x124>(v);                   // row_ror:4
    v += dpp<0x128>(v);                   // row_ror:8
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Backward on a chunk, tile after tile from its end.  A tile's states are computed again from the state saved in front
// of it (a_t and h_t of the tile stay in registers), then the adjoint runs back through it:
//     g_t = C_t dy'_t + a_{t+1} g_{t+1},  dy' = dy silu(z)
//     dC_t = sum_d dy' h_t,  dB_t = sum_d g_t u_t,  du = g_t . B_t,  w = g_t a_t h_{t-1}
//     d raw = (A . w + du x) sigmoid(raw),  dx = du dt + D dy',  dA = sum w dt
template <class T, int S>
__global__ __launch_bounds__(256) void scan_bwd_kernel(ScanArgs a) {
    constexpr int NP = 4 * S, MK = mark_steps<S>(), NI = MK / 4;
    __shared__ float lds_b[MK * NP], lds_c[MK * NP], red[4 * MK * 2 * NP];       // red: [wave][step][B, C][state]
    const Place p = place(a, blockIdx.z);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int chunk = blockIdx.y, t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.L), tend = min(t1, p.len);
    float A2[S], g[S], dA[S];
    load_states<S>(A2, a.A + (size_t)p.ch * a.N, p.q, a.N);
#pragma unroll
    for (int s = 0; s < S; ++s) { A2[s] *= kLog2e; g[s] = 0.f; dA[s] = 0.f; }
    const float bias = a.bias ? a.bias[p.ch] : 0.f, dskip = a.Dp ? a.Dp[p.ch] : 0.f;
    if (a.dhT) load_states<S>(g, a.dhT + ((size_t)p.b * a.D + p.ch) * a.N, p.q, a.N);
    for (int k = a.nchunk - 1; k > chunk; --k) {
        const size_t row = ((size_t)p.b * a.nchunk + k) * a.D + p.ch;
        float e[S];
        load_padded<S>(e, a.hend + row * NP, p.q);
        const float sd = a.sdt[row];
#pragma unroll
        for (int s = 0; s < S; ++s) g[s] = fmaf(exp2_hw(A2[s] * sd), g[s], e[s]);
    }
    float dD = 0.f, dbias = 0.f;
    for (int k = (tend - t0 + MK - 1) / MK - 1; k >= 0; --k) {
        const int t = t0 + k * MK;
        __syncthreads();
        stage_rows<T, S, MK>(lds_b, a.Bm, p.b * a.bb + p.g * a.bg, a.bt, t, tend, a.N);
        stage_rows<T, S, MK>(lds_c, a.Cm, p.b * a.cb + p.g * a.cg, a.ct, t, tend, a.N);
        float h0[S];
        load_padded<S>(h0, a.marks + (((size_t)p.b * a.nmark + t / MK) * a.D + p.ch) * NP, p.q);
        float raw[NI], dt[NI], u[NI], x[NI], dy[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int own = t + 4 * i + p.q;
            const bool in = own < tend && p.live;
            raw[i] = dt[i] = x[i] = dy[i] = 0.f;
            if (in) {
                x[i] = at<T>(a.x, p.b * a.xb + own * a.xt + p.ch);
                raw[i] = at<T>(a.dt, p.b * a.dtb + own * a.dtt + p.ch) + bias;
                dt[i] = a.softplus ? softplus_exact(raw[i]) : raw[i];
                dy[i] = at<T>(a.dy, p.b * a.dyb + own * a.dyt + p.ch);
            }
            u[i] = dt[i] * x[i];
        }
        __syncthreads();
        float av[MK][S], h[MK][S];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            float part[4];
            auto step = [&](int j, float dtj, float uj) {
                const int m = 4 * i + j;
                const float *bj = lds_b + m * NP + p.q * S, *cj = lds_c + m * NP + p.q * S;
                float y = 0.f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    av[m][s] = exp2_hw(A2[s] * dtj);
                    h[m][s] = fmaf(av[m][s], m ? h[m - 1][s] : h0[s], uj * bj[s]);
                    y = fmaf(h[m][s], cj[s], y);
                }
                part[j] = y;
            };
            step(0, quad_lane<0>(dt[i]), quad_lane<0>(u[i]));
            step(1, quad_lane<1>(dt[i]), quad_lane<1>(u[i]));
            step(2, quad_lane<2>(dt[i]), quad_lane<2>(u[i]));
            step(3, quad_lane<3>(dt[i]), quad_lane<3>(u[i]));
            if (a.z) {
                const float y = fmaf(dskip, x[i], quad_sum_of_own(part[0], part[1], part[2], part[3], p.q));
                const int own = t + 4 * i + p.q;
                if (own < tend && p.live) {
                    const float z = at<T>(a.z, p.b * a.zb + own * a.zt + p.ch), sg = sigmoid_hw(z);
                    static_cast<T*>(a.dz)[((size_t)p.b * a.L + own) * a.D + p.ch] = (T)(dy[i] * y * sg * fmaf(z, 1.f - sg, 1.f));
                    dy[i] *= z * sg;
                }
            }
        }
#pragma unroll
        for (int i = NI - 1; i >= 0; --i) {
            float pu[4], pt[4];
            auto step = [&](int j, float dtj, float uj, float dyj) {
                const int m = 4 * i + j;
                const float *bj = lds_b + m * NP + p.q * S, *cj = lds_c + m * NP + p.q * S;
                float du = 0.f, dd = 0.f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    g[s] = fmaf(dyj, cj[s], g[s]);
                    du = fmaf(g[s], bj[s], du);
                    const float ga = g[s] * av[m][s], w = ga * (m ? h[m - 1][s] : h0[s]);
                    dd = fmaf(A2[s], w, dd);
                    dA[s] = fmaf(dtj, w, dA[s]);
                    av[m][s] = g[s] * uj;                 // dB of this channel
                    h[m][s] *= dyj;                       // dC of this channel
                    g[s] = ga;
                }
                pu[j] = du;
                pt[j] = dd;
            };
            step(3, quad_lane<3>(dt[i]), quad_lane<3>(u[i]), quad_lane<3>(dy[i]));
            step(2, quad_lane<2>(dt[i]), quad_lane<2>(u[i]), quad_lane<2>(dy[i]));
            step(1, quad_lane<1>(dt[i]), quad_lane<1>(u[i]), quad_lane<1>(dy[i]));
            step(0, quad_lane<0>(dt[i]), quad_lane<0>(u[i]), quad_lane<0>(dy[i]));
            const float du = quad_sum_of_own(pu[0], pu[1], pu[2], pu[3], p.q);
            float dr = kLn2 * quad_sum_of_own(pt[0], pt[1], pt[2], pt[3], p.q) + du * x[i];
            if (a.softplus) dr *= sigmoid_hw(raw[i]);
            const int own = t + 4 * i + p.q;
            if (own < tend && p.live) {
                const size_t o = ((size_t)p.b * a.L + own) * a.D + p.ch;
                static_cast<T*>(a.dx)[o] = (T)fmaf(du, dt[i], dskip * dy[i]);
                static_cast<T*>(a.ddt)[o] = (T)dr;
                dbias += dr;
                dD = fmaf(dy[i], x[i], dD);
            }
        }
#pragma unroll
        for (int m = 0; m < MK; ++m)
#pragma unroll
            for (int s = 0; s < S; ++s) {
                const float vb = channel_sum(av[m][s]), vc = channel_sum(h[m][s]);
                if (lane < 4) {
                    float* r = red + (wave * MK + m) * 2 * NP + p.q * S + s;
                    r[0] = vb;
                    r[NP] = vc;
                }
            }
        __syncthreads();
        for (int e = threadIdx.x; e < MK * 2 * NP; e += 256) {
            const int m = e / (2 * NP), r = e % (2 * NP);
            if (t + m < tend)
                a.pBC[(((size_t)p.b * a.L + t + m) * gridDim.x + blockIdx.x) * 2 * NP + r] =
                    (red[e] + red[e + MK * 2 * NP]) + (red[e + 2 * MK * 2 * NP] + red[e + 3 * MK * 2 * NP]);
        }
    }
    dD = quad_sum(dD);
    dbias = quad_sum(dbias);
    if (!p.live) return;
    const size_t part = (size_t)p.b * a.nchunk + chunk;
    store_padded<S>(dA, a.pA + (part * a.D + p.ch) * NP, p.q);
    if (p.q == 0) {
        a.pD[(part * 2 + 0) * a.D + p.ch] = dD;
        a.pD[(part * 2 + 1) * a.D + p.ch] = dbias;
    }
    if (chunk == 0 && a.dh0) store_states<S>(g, a.dh0 + ((size_t)p.b * a.D + p.ch) * a.N, p.q, a.N);
    for (int t = max(t0, tend) + p.q; t < t1; t += 4) {                // behind the sequence's end
        const size_t o = ((size_t)p.b * a.L + t) * a.D + p.ch;
        static_cast<T*>(a.dx)[o] = (T)0.f;
        static_cast<T*>(a.ddt)[o] = (T)0.f;
        if (a.dz) static_cast<T*>(a.dz)[o] = (T)0.f;
    }
}

// dB, dC [B, L, G, N] from the blocks' partial sums [B, L, G, tpg, 2, NP]
template <class T>
__global__ __launch_bounds__(256) void scan_bc_kernel(const float* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC,
                                                      const int* __restrict__ lengths, long long rows, int L, int G, int tpg, int N, int NP) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;             // (row, which, n)
    const int per = 2 * NP;
    const long long row = i / per;
    if (row >= rows) return;
    const int r = (int)(i - row * per), n = r % NP;
    if (n >= N) return;
    const long long bt = row / G;
    float s = 0.f;
    if (!lengths || bt % L < lengths[bt / L])
        for (int k = 0; k < tpg; ++k) s += part[(row * tpg + k) * per + r];
    (r < NP ? dB : dC)[row * N + n] = (T)s;
}

// rows of NP with N used -> [D, N], summed over R partials
__global__ __launch_bounds__(256) void scan_dA_kernel(const float* __restrict__ part, float* __restrict__ dA, int R, int D, int N, int NP) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= D * N) return;
    const int d = i / N, n = i - d * N;
    float s = 0.f;
    for (int r = 0; r < R; ++r) s += part[((size_t)r * D + d) * NP + n];
    dA[i] = s;
}

// One token of every row; state [slots, D, N] is read and written once: 8N bytes a channel against 7N operations.
template <class T, int S>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a, const int* __restrict__ slots, int nslots, float* __restrict__ state) {
    const int row = blockIdx.y;
    bool bad;
    const int slot = claim_slot(slots, row, nslots, &bad);
    const Place p = place(a, row);
    if (!p.live) return;
    T* out = static_cast<T*>(a.y) + (size_t)row * a.D + p.ch;
    if (bad || slot < 0) {
        if (p.q == 0) *out = (T)(bad ? __builtin_nanf("") : 0.f);
        return;
    }
    float* st = state + ((size_t)slot * a.D + p.ch) * a.N;
    float h[S], A2[S], B[S], C[S];
    load_states<S>(h, st, p.q, a.N);
    load_states<S>(A2, a.A + (size_t)p.ch * a.N, p.q, a.N);
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int n = p.q * S + s;
        B[s] = n < a.N ? at<T>(a.Bm, row * a.bb + p.g * a.bg + n) : 0.f;
        C[s] = n < a.N ? at<T>(a.Cm, row * a.cb + p.g * a.cg + n) : 0.f;
    }
    const float x = at<T>(a.x, row * a.xb + p.ch);
    float dt = at<T>(a.dt, row * a.dtb + p.ch) + (a.bias ? a.bias[p.ch] : 0.f);
    if (a.softplus) dt = softplus_exact(dt);
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        h[s] = fmaf(exp2_hw(A2[s] * kLog2e * dt), h[s], dt * x * B[s]);
        y = fmaf(h[s], C[s], y);
    }
    store_states<S>(h, st, p.q, a.N);
    y = quad_sum(y);
    if (p.q == 0) {
        if (a.Dp) y = fmaf(a.Dp[p.ch], x, y);
        if (a.z) {
            const float z = at<T>(a.z, row * a.zb + p.ch);
            y *= z * sigmoid_hw(z);
        }
        *out = (T)y;
    }
}

namespace {

int lane_states(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

struct ScanPlan {
    int S, NP, tpg, nchunk, chunk, nmark;
};

// Time is split where the channels of the batch alone do not fill the chip.
ScanPlan scan_plan(const UnetmiScanDesc& d) {
    ScanPlan p;
    p.S = lane_states(d.state);
    p.NP = 4 * p.S;
    const int Dg = d.channels / d.groups;
    p.tpg = (Dg + kCh - 1) / kCh;
    const long long blocks = (long long)d.batch * d.groups * p.tpg;
    long long want = blocks > 0 ? 512 / blocks : 1;
    const long long most = (d.length + 63) / 64;
    if (want > most) want = most;
    if (want > 64) want = 64;
    if (want < 1) want = 1;
    p.chunk = (int)((d.length + want - 1) / want);
    p.chunk = (p.chunk + kTile - 1) / kTile * kTile;
    if (p.chunk < kTile) p.chunk = kTile;
    p.nchunk = (d.length + p.chunk - 1) / p.chunk;
    if (p.nchunk < 1) p.nchunk = 1;
    const int mk = mark_steps_of(p.S);
    p.nmark = (d.length + mk - 1) / mk;
    return p;
}

int scan_check(const UnetmiScanDesc* d, const char* what) {
    const std::string w = what;
    if (!d) return api_fail(UNETMI_E_BAD_ARG, w + ": null descriptor");
    if (d->batch < 0 || d->length < 0 || d->channels < 1 || d->state < 1 || d->groups < 1) return api_fail(UNETMI_E_BAD_DESC, w + ": bad sizes");
    if (d->channels % d->groups) return api_fail(UNETMI_E_BAD_DESC, w + ": the groups do not divide the channels");
    if (d->state > 64) return api_fail(UNETMI_E_UNSUPPORTED, w + ": at most 64 states per channel are built");
    if (d->dtype != UNETMI_DTYPE_F32 && d->dtype != UNETMI_DTYPE_BF16) return api_fail(UNETMI_E_UNSUPPORTED, w + ": fp32 or bfloat16 activations");
    if (d->batch > 65535) return api_fail(UNETMI_E_UNSUPPORTED, w + ": more than 65535 sequences");
    if (d->channels > (1 << 24) || d->length > (1 << 28)) return api_fail(UNETMI_E_UNSUPPORTED, w + ": more than 2^24 channels or 2^28 steps");
    for (const int64_t* s : {d->x_stride, d->dt_stride, d->z_stride, d->dy_stride})
        if (s[0] < 0 || s[1] < 0) return api_fail(UNETMI_E_BAD_DESC, w + ": negative stride");
    for (const int64_t* s : {d->b_stride, d->c_stride})
        if (s[0] < 0 || s[1] < 0 || s[2] < 0) return api_fail(UNETMI_E_BAD_DESC, w + ": negative stride");
    return UNETMI_OK;
}

ScanArgs scan_args(const UnetmiScanDesc& d, const ScanPlan& p, const void* x, const void* dt, const float* A, const void* B, const void* C,
                   const float* D, const void* z, const float* bias) {
    ScanArgs a = {};
    a.x = x; a.dt = dt; a.z = z; a.Bm = B; a.Cm = C; a.A = A; a.Dp = D; a.bias = bias;
    a.xb = d.x_stride[0]; a.xt = d.x_stride[1]; a.dtb = d.dt_stride[0]; a.dtt = d.dt_stride[1];
    a.zb = d.z_stride[0]; a.zt = d.z_stride[1]; a.dyb = d.dy_stride[0]; a.dyt = d.dy_stride[1];
    a.bb = d.b_stride[0]; a.bt = d.b_stride[1]; a.bg = d.b_stride[2];
    a.cb = d.c_stride[0]; a.ct = d.c_stride[1]; a.cg = d.c_stride[2];
    a.L = d.length; a.D = d.channels; a.N = d.state; a.Dg = d.channels / d.groups; a.tpg = p.tpg;
    a.chunk = p.chunk; a.nchunk = p.nchunk; a.nmark = p.nmark; a.softplus = d.softplus != 0;
    return a;
}

template <template <class, int> class F, class T, class... A>
int scan_states(int S, A&&... args) {
    switch (S) {
        case 1: return F<T, 1>::run(args...);
        case 2: return F<T, 2>::run(args...);
        case 4: return F<T, 4>::run(args...);
        case 8: return F<T, 8>::run(args...);
        default: return F<T, 16>::run(args...);
    }
}
template <template <class, int> class F, class... A>
int scan_dispatch(const UnetmiScanDesc& d, int S, A&&... args) {
    return d.dtype == UNETMI_DTYPE_BF16 ? scan_states<F, __bf16>(S, args...) : scan_states<F, float>(S, args...);
}

template <class T, int S>
struct RunScan {
    static int run(const UnetmiScanDesc& d, const ScanPlan& p, const ScanArgs& a, hipStream_t s) {
        const dim3 block(256);
        if (p.nchunk > 1) {
            // the last chunk's summary is never read
            hipLaunchKernelGGL((scan_fwd_kernel<T, S, true>), dim3(d.groups * p.tpg, p.nchunk - 1, d.batch), block, 0, s, a);
            const int rc = launched("ssm_scan_fwd states");
            if (rc != UNETMI_OK) return rc;
        }
        hipLaunchKernelGGL((scan_fwd_kernel<T, S, false>), dim3(d.groups * p.tpg, p.nchunk, d.batch), block, 0, s, a);
        return launched("ssm_scan_fwd");
    }
};
template <class T, int S>
struct RunScanBwd {
    static int run(const UnetmiScanDesc& d, const ScanPlan& p, const ScanArgs& a, void* dB, void* dC, float* dA, float* dD, float* dbias, hipStream_t s) {
        const dim3 block(256), grid(d.groups * p.tpg, p.nchunk, d.batch);
        int rc;
        if (p.nchunk > 1) {
            hipLaunchKernelGGL((scan_bwd_state_kernel<T, S>), grid, block, 0, s, a);
            if ((rc = launched("ssm_scan_bwd states")) != UNETMI_OK) return rc;
        }
        hipLaunchKernelGGL((scan_bwd_kernel<T, S>), grid, block, 0, s, a);
        if ((rc = launched("ssm_scan_bwd")) != UNETMI_OK) return rc;
        const long long rows = (long long)d.batch * d.length * d.groups, threads = rows * 2 * p.NP;
        if (threads) {
            hipLaunchKernelGGL((scan_bc_kernel<T>), dim3((unsigned)((threads + 255) / 256)), block, 0, s, a.pBC, static_cast<T*>(dB),
                               static_cast<T*>(dC), a.lengths, rows, d.length, d.groups, p.tpg, d.state, p.NP);
            if ((rc = launched("ssm_scan_bwd B C")) != UNETMI_OK) return rc;
        }
        const int parts = d.batch * p.nchunk;
        hipLaunchKernelGGL(scan_dA_kernel, dim3((d.channels * d.state + 255) / 256), block, 0, s, a.pA, dA, parts, d.channels, d.state, p.NP);
        if ((rc = launched("ssm_scan_bwd A")) != UNETMI_OK) return rc;
        return launch_sum_rows(a.pD, dD, dbias, d.channels, parts, 2 * d.channels, s);
    }
};
template <class T, int S>
struct RunScanStep {
    static int run(const UnetmiScanDesc& d, const ScanPlan& p, const ScanArgs& a, const int* slots, int nslots, float* state, hipStream_t s) {
        hipLaunchKernelGGL((scan_step_kernel<T, S>), dim3(d.groups * p.tpg, d.batch), dim3(256), 0, s, a, slots, nslots, state);
        return launched("ssm_scan_step");
    }
};

size_t summary_floats(const UnetmiScanDesc& d, const ScanPlan& p) {
    return p.nchunk > 1 ? (size_t)d.batch * p.nchunk * d.channels * (p.NP + 1) : 0;
}

}  // namespace
}  // namespace unetmi

using namespace unetmi;

extern "C" {

size_t unetmi_ssm_scan_marks_bytes(const UnetmiScanDesc* d) {
    if (scan_check(d, "ssm_scan_marks_bytes") != UNETMI_OK) return 0;
    const ScanPlan p = scan_plan(*d);
    return (size_t)d->batch * p.nmark * d->channels * p.NP * sizeof(float);
}

size_t unetmi_ssm_scan_fwd_workspace_bytes(const UnetmiScanDesc* d) {
    if (scan_check(d, "ssm_scan_fwd_workspace_bytes") != UNETMI_OK) return 0;
    return summary_floats(*d, scan_plan(*d)) * sizeof(float);
}

int unetmi_ssm_scan_fwd(const UnetmiScanDesc* d, const void* x, const void* dt, const float* A, const void* B, const void* C,
                        const float* D, const void* z, const float* dt_bias, const float* state, const int32_t* lengths, void* y,
                        float* state_out, float* marks, void* ws, size_t ws_bytes, void* stream) {
    const int rc = scan_check(d, "ssm_scan_fwd");
    if (rc != UNETMI_OK) return rc;
    if (d->batch == 0 || (d->length == 0 && !state_out)) return UNETMI_OK;
    if (!A || (d->length > 0 && (!x || !dt || !B || !C || !y))) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_fwd: null tensor pointer");
    const ScanPlan p = scan_plan(*d);
    const size_t need = summary_floats(*d, p);
    if (need && (!ws || ws_bytes < need * sizeof(float))) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_fwd: workspace too small");
    ScanArgs a = scan_args(*d, p, x, dt, A, B, C, D, z, dt_bias);
    a.h0 = state; a.lengths = lengths; a.y = y; a.hT = state_out; a.marks = marks;
    a.hend = static_cast<float*>(ws);
    a.sdt = a.hend ? a.hend + (size_t)d->batch * p.nchunk * d->channels * p.NP : nullptr;
    return scan_dispatch<RunScan>(*d, p.S, *d, p, a, static_cast<hipStream_t>(stream));
}

size_t unetmi_ssm_scan_bwd_workspace_bytes(const UnetmiScanDesc* d) {
    if (scan_check(d, "ssm_scan_bwd_workspace_bytes") != UNETMI_OK) return 0;
    const ScanPlan p = scan_plan(*d);
    const size_t parts = (size_t)d->batch * p.nchunk;
    return (summary_floats(*d, p) + (size_t)d->batch * d->length * d->groups * p.tpg * 2 * p.NP + parts * d->channels * (p.NP + 2)) * sizeof(float);
}

int unetmi_ssm_scan_bwd(const UnetmiScanDesc* d, const void* x, const void* dt, const float* A, const void* B, const void* C,
                        const float* D, const void* z, const float* dt_bias, const int32_t* lengths, const float* marks, const void* dy,
                        const float* dstate_out, void* dx, void* ddt, float* dA, void* dB, void* dC, float* dD, float* ddt_bias,
                        void* dz, float* dstate, void* ws, size_t ws_bytes, void* stream) {
    const int rc = scan_check(d, "ssm_scan_bwd");
    if (rc != UNETMI_OK) return rc;
    if (d->batch == 0) return api_fail(UNETMI_E_BAD_DESC, "ssm_scan_bwd: empty batch");
    if (!A || !dA || !dD || !ddt_bias || !ws || (d->length > 0 && (!x || !dt || !B || !C || !marks || !dy || !dx || !ddt || !dB || !dC)))
        return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_bwd: null tensor pointer");
    if (d->length > 0 && (z != nullptr) != (dz != nullptr)) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_bwd: z and dz go together");
    if (ws_bytes < unetmi_ssm_scan_bwd_workspace_bytes(d)) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_bwd: workspace too small");
    const ScanPlan p = scan_plan(*d);
    ScanArgs a = scan_args(*d, p, x, dt, A, B, C, D, z, dt_bias);
    a.lengths = lengths; a.marks = const_cast<float*>(marks);
    a.dy = dy; a.dhT = dstate_out; a.dx = dx; a.ddt = ddt; a.dz = dz; a.dh0 = dstate;
    const size_t parts = (size_t)d->batch * p.nchunk;
    a.pA = static_cast<float*>(ws);                                   // padded rows first: they stay 16-byte aligned
    a.pBC = a.pA + parts * d->channels * p.NP;
    a.hend = a.pBC + (size_t)d->batch * d->length * d->groups * p.tpg * 2 * p.NP;
    a.sdt = a.hend + (p.nchunk > 1 ? parts * d->channels * p.NP : 0);
    a.pD = a.sdt + (p.nchunk > 1 ? parts * d->channels : 0);
    return scan_dispatch<RunScanBwd>(*d, p.S, *d, p, a, dB, dC, dA, dD, ddt_bias, static_cast<hipStream_t>(stream));
}

int unetmi_ssm_scan_step(const UnetmiScanDesc* d, const void* x, const void* dt, const float* A, const void* B, const void* C,
                         const float* D, const void* z, const float* dt_bias, const int32_t* slots, int num_slots, float* state,
                         void* y, void* stream) {
    const int rc = scan_check(d, "ssm_scan_step");
    if (rc != UNETMI_OK) return rc;
    if (d->batch == 0) return UNETMI_OK;
    if (!x || !dt || !A || !B || !C || !state || !y) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_step: null tensor pointer");
    if (num_slots < 0 || (!slots && num_slots < d->batch)) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_step: fewer slots than rows");
    const ScanPlan p = scan_plan(*d);
    ScanArgs a = scan_args(*d, p, x, dt, A, B, C, D, z, dt_bias);
    a.y = y;
    return scan_dispatch<RunScanStep>(*d, p.S, *d, p, a, slots, num_slots, state, static_cast<hipStream_t>(stream));
}

}  // extern "C"
