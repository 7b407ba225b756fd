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

constexpr int kAlign = 16;                // chunks of the time axis start at multiples of this, itself one of every mark_steps
constexpr int kCh = 64;                   // channels per block

// Steps per tile of the forward kernels: a tile's computation has to cover the next one's loads, and with few states a step
// is short (16 x 1024 x 2048 bf16: 138 us for 4 and 148 for 8 states with 32 steps, 186 and 196 with 16; 16 states: 207 and 202).
template <int S> constexpr int tile_steps() { return S <= 2 ? 32 : 16; }

// steps between two saved states, = the steps the backward kernel keeps in registers
template <int S> constexpr int mark_steps() { return S <= 2 ? 16 : S == 4 ? 8 : 4; }
static int mark_steps_of(int S) { return S <= 2 ? 16 : S == 4 ? 8 : 4; }

// The backward kernel's running sums of dA, dD and ddt_bias go to memory every kPiece steps: a running sum of n terms is off by
// up to n roundings, and a channel whose time axis is not split would take all its steps in one (65536 steps of equal terms:
// dA off by 7e-4 of itself, 7e-6 in pieces).
constexpr int kPiece = 1024;

struct ScanArgs {
    const void *x, *dt, *z, *Bm, *Cm;     // z may be null
    const float *A, *Dp, *bias, *h0;      // Dp, bias, h0 may be null
    const int* lengths;
    long long xb, xt, dtb, dtt, zb, zt, bb, bt, bg, cb, ct, cg;      // element strides
    int L, D, N, Dg, tpg;                 // channels per group, blocks per group
    int chunk, nchunk;                    // steps per chunk: a multiple of kAlign; its last tile may hold fewer steps than a tile's
    int npiece;                           // kPiece steps per chunk
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
    float *dh0, *pBC, *pA;                // partial sums: [B, L, G tpg, 2, 4S]; [B nchunk npiece, (D, 4S), (D), (D)] of A, D, bias
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

// Rows of a sequence are reached through buffer descriptors that start at a tile's first row: the lane's offset inside a
// tile and the uniform one of its step are 32 bits (the host refuses steps that are further apart), and an offset beyond
// the window reads zero and stores nothing, which is how steps behind the end and dead lanes are kept out.
constexpr int kOutside = (int)0x80000000;

template <class T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t window(const T* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, 0x7fffffff, 0x00020000);
}
template <class T>
__device__ __forceinline__ T window_load(__amdgpu_buffer_rsrc_t rs, int voff, int soff) {
    if constexpr (sizeof(T) == 2) return __builtin_bit_cast(T, (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rs, voff, soff, 0));
    else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rs, voff, soff, 0));
}
template <class T>
__device__ __forceinline__ void window_store(T v, __amdgpu_buffer_rsrc_t rs, int voff, int soff) {
    if constexpr (sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, v), rs, voff, soff, 0);
    else __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, v), rs, voff, soff, 0);
}

template <int S>
__device__ __forceinline__ void window_store_states(const float (&h)[S], __amdgpu_buffer_rsrc_t rs, int voff) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    if constexpr (S == 1) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, h[0]), rs, voff, 0, 0);
    else if constexpr (S == 2) __builtin_amdgcn_raw_buffer_store_b64(i32x2{__builtin_bit_cast(int, h[0]), __builtin_bit_cast(int, h[1])}, rs, voff, 0, 0);
    else {
#pragma unroll
        for (int s = 0; s < S; s += 4)
            __builtin_amdgcn_raw_buffer_store_b128(i32x4{__builtin_bit_cast(int, h[s]), __builtin_bit_cast(int, h[s + 1]),
                                                         __builtin_bit_cast(int, h[s + 2]), __builtin_bit_cast(int, h[s + 3])}, rs, voff, 4 * s, 0);
    }
}

// A lane's steps of a tile: 4i + q of its channel, i = 0..STEPS/4-1.
template <class T, int STEPS>
struct Column {
    const T* base;                        // the chunk's first row
    long long stride;
    int off;                              // of the lane's first element of a tile, in bytes
    T v[STEPS / 4];
    __device__ __forceinline__ Column(const void* p, long long sb, long long st, const Place& pl, int t0)
        : base(static_cast<const T*>(p) + pl.b * sb + t0 * st), stride(st), off((pl.q * (int)st + pl.ch) * (int)sizeof(T)) {}
    // steps dt .. dt+STEPS-1 of the chunk, of which `left` are there
    __device__ __forceinline__ void load(int dt, int left, int q) {
        const auto rs = window(base + dt * stride);
        const int next = 4 * (int)stride * (int)sizeof(T);
        if (left >= STEPS) {
#pragma unroll
            for (int i = 0; i < STEPS / 4; ++i) v[i] = window_load<T>(rs, off, i * next);
        } else {
#pragma unroll
            for (int i = 0; i < STEPS / 4; ++i) v[i] = window_load<T>(rs, 4 * i + q < left ? off : kOutside, i * next);
        }
    }
};
// the same for a dense output [.., D]
template <class T, int STEPS>
struct OutColumn {
    T* base;
    int D, off;
    bool live;
    __device__ __forceinline__ OutColumn(void* p, int D, size_t first_row, const Place& pl)
        : base(static_cast<T*>(p) + first_row * D), D(D), off((pl.q * D + pl.ch) * (int)sizeof(T)), live(pl.live) {}
    __device__ __forceinline__ void store(int dt, int left, int q, int i, float f) const {
        window_store<T>((T)f, window(base + (size_t)dt * D), live && 4 * i + q < left ? off : kOutside, 4 * i * D * (int)sizeof(T));
    }
};

// B or C of a tile of steps, on its way from HBM to LDS: [step][4S] as fp32, zero behind the end and beyond N
template <class T, int S, int STEPS>
struct Shared {
    static constexpr int NP = 4 * S, E = (STEPS * NP + 255) / 256, ROWS = 256 / NP;
    const T* base;
    long long stride;
    int off, row;                         // of the thread's first element of a tile; its step
    T v[E];
    __device__ __forceinline__ Shared(const void* p, long long sb, long long st, long long sg, const Place& pl, int t0, int N)
        : base(static_cast<const T*>(p) + pl.b * sb + pl.g * sg + t0 * st), stride(st), row(threadIdx.x / NP) {
        const int n = threadIdx.x % NP;
        off = n < N && row < STEPS ? (row * (int)st + n) * (int)sizeof(T) : kOutside;
    }
    __device__ __forceinline__ void load(int dt, int left) {
        const auto rs = window(base + dt * stride);
#pragma unroll
        for (int k = 0; k < E; ++k) {
            v[k] = window_load<T>(rs, row + k * ROWS < left ? off : kOutside, k * ROWS * (int)stride * (int)sizeof(T));
        }
    }
    __device__ __forceinline__ void store(float* lds) const {
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int e = threadIdx.x + 256 * k;
            if (STEPS * NP % 256 == 0 || e < STEPS * NP) lds[e] = widen(v[k]);
        }
    }
};

template <class T>
__device__ __forceinline__ float at(const void* p, long long i) { return widen(static_cast<const T*>(p)[i]); }

// Forward.  kStates: the first pass over a time axis that is split into chunks: the chunk's last state from zero and the
// sum of its steps (the product of its decays is exp(A sum dt)).  Else the whole operator on a chunk, starting from the
// states of the chunks before it; kMarks also saves the states that the backward kernel starts its tiles from.  A tile's
// inputs are loaded while the tile before it is computed, B and C go into the other half of LDS: one barrier a tile.
// Measured (medians): 1 x 8192 x 2048 channels x 16 states bf16 62 + 95 us in 32 chunks, the vector units 87 and 86 % busy with
// 23 and 34 instructions a step and wave; 128 x 501 x 256 fp32 with marks 122 us (3.2 TB/s); 4 x 4096 x 2048 bf16 117 + 190 us.
enum ScanPass { kStates, kOutputs, kMarks };

template <class T, int S, ScanPass PASS>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanArgs a) {
    constexpr int NP = 4 * S, MK = mark_steps<S>(), kTile = tile_steps<S>();
    constexpr bool STATE_ONLY = PASS == kStates;
    __shared__ float lds_b[2][kTile * NP], lds_c[STATE_ONLY ? 1 : 2][STATE_ONLY ? 1 : kTile * NP];
    const Place p = place(a, blockIdx.z);
    const int chunk = blockIdx.y, t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.L), tend = min(t1, p.len);
    const int left = tend - t0;                                       // steps of this chunk
    Column<T, kTile> xs(a.x, a.xb, a.xt, p, t0), dts(a.dt, a.dtb, a.dtt, p, t0), zs(a.z, a.zb, a.zt, p, t0);
    Shared<T, S, kTile> bs(a.Bm, a.bb, a.bt, a.bg, p, t0, a.N), cs(a.Cm, a.cb, a.ct, a.cg, p, t0, a.N);
    auto fetch = [&](int dt) {
        dts.load(dt, left - dt, p.q);
        xs.load(dt, left - dt, p.q);
        if (!STATE_ONLY && a.z) zs.load(dt, left - dt, p.q);
        bs.load(dt, left - dt);
        if (!STATE_ONLY) cs.load(dt, left - dt);
    };
    if (left > 0) fetch(0);
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
            for (int s = 0; s < S; ++s) h[s] = h[s] == 0.f ? e[s] : fmaf(exp2_hw(A2[s] * sd), h[s], e[s]);   // A > 0: 0, not 0 inf
        }
    }
    const OutColumn<T, kTile> out(a.y, a.D, (size_t)p.b * a.L + t0, p);
    float sdt = 0.f;
    int half = 0;
    for (int dt0 = 0; dt0 < left; dt0 += kTile, half ^= 1) {
        float *lb = lds_b[half], *lc = lds_c[STATE_ONLY ? 0 : half];
        bs.store(lb);
        if (!STATE_ONLY) cs.store(lc);
        float x[kTile / 4], dt[kTile / 4], z[kTile / 4], y[kTile / 4];
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i) {
            x[i] = widen(xs.v[i]);
            dt[i] = widen(dts.v[i]) + bias;
            z[i] = !STATE_ONLY && a.z ? widen(zs.v[i]) : 0.f;
        }
        __syncthreads();
        if (dt0 + kTile < left) fetch(dt0 + kTile);
        if (a.softplus) {
#pragma unroll
            for (int i = 0; i < kTile / 4; ++i) dt[i] = softplus_exact(dt[i]);
        }
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i) {
            if (PASS == kMarks && (4 * i) % MK == 0)
                window_store_states<S>(h, window(a.marks + ((size_t)p.b * a.nmark + (t0 + dt0 + 4 * i) / MK) * a.D * NP),
                                       p.live && dt0 + 4 * i < left ? (p.ch * NP + p.q * S) * 4 : kOutside);
            dt[i] = dt0 + 4 * i + p.q < left ? dt[i] : 0.f;
            const float u = dt[i] * x[i];
            sdt += dt[i];
            float part[4];
            auto step = [&](int j, float dtj, float uj) {
                const float* bj = lb + (4 * i + j) * NP + p.q * S;
                const float* cj = lc + (STATE_ONLY ? 0 : (4 * i + j) * NP + p.q * S);
                float y = 0.f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    h[s] = fmaf(exp2_hw(A2[s] * dtj), h[s], uj * bj[s]);
                    if (!STATE_ONLY) y = fmaf(h[s], cj[s], y);
                }
                part[j] = y;
            };
            step(0, quad_lane<0>(dt[i]), quad_lane<0>(u));
            step(1, quad_lane<1>(dt[i]), quad_lane<1>(u));
            step(2, quad_lane<2>(dt[i]), quad_lane<2>(u));
            step(3, quad_lane<3>(dt[i]), quad_lane<3>(u));
            if (!STATE_ONLY) y[i] = fmaf(dskip, x[i], quad_sum_of_own(part[0], part[1], part[2], part[3], p.q));
        }
        if (!STATE_ONLY) {
            if (a.z) {
#pragma unroll
                for (int i = 0; i < kTile / 4; ++i) y[i] *= z[i] * sigmoid_hw(z[i]);
            }
#pragma unroll
            for (int i = 0; i < kTile / 4; ++i) out.store(dt0, left - dt0, p.q, i, y[i]);
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
// and the sum of its steps.  Built like the forward pass, from the chunk's last tile to its first.  4 x 4096 x 2048 bf16 in
// eight chunks: 132 us, vector units 90 % busy.
template <class T, int S>
__global__ __launch_bounds__(256) void scan_bwd_state_kernel(ScanArgs a) {
    constexpr int NP = 4 * S, kTile = tile_steps<S>();
    __shared__ float lds_c[2][kTile * NP];
    const Place p = place(a, blockIdx.z);
    const int chunk = blockIdx.y + 1;                                 // nobody stands before the first chunk
    const int t0 = chunk * a.chunk, tend = min(min(t0 + a.chunk, a.L), p.len), left = tend - t0;
    Column<T, kTile> dys(a.dy, a.dyb, a.dyt, p, t0), dts(a.dt, a.dtb, a.dtt, p, t0), zs(a.z, a.zb, a.zt, p, t0);
    Shared<T, S, kTile> cs(a.Cm, a.cb, a.ct, a.cg, p, t0, a.N);
    auto fetch = [&](int dt) {
        dts.load(dt, left - dt, p.q);
        dys.load(dt, left - dt, p.q);
        if (a.z) zs.load(dt, left - dt, p.q);
        cs.load(dt, left - dt);
    };
    int dt0 = left > 0 ? (left - 1) / kTile * kTile : -1;
    if (dt0 >= 0) fetch(dt0);
    float A2[S], g[S];
    load_states<S>(A2, a.A + (size_t)p.ch * a.N, p.q, a.N);
#pragma unroll
    for (int s = 0; s < S; ++s) { A2[s] *= kLog2e; g[s] = 0.f; }
    const float bias = a.bias ? a.bias[p.ch] : 0.f;
    float sdt = 0.f;
    for (int half = 0; dt0 >= 0; dt0 -= kTile, half ^= 1) {
        float* lc = lds_c[half];
        cs.store(lc);
        float dt[kTile / 4], dy[kTile / 4], z[kTile / 4];
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i) {
            dt[i] = widen(dts.v[i]) + bias;
            dy[i] = widen(dys.v[i]);
            z[i] = a.z ? widen(zs.v[i]) : 0.f;
        }
        __syncthreads();
        if (dt0 > 0) fetch(dt0 - kTile);
        if (a.softplus) {
#pragma unroll
            for (int i = 0; i < kTile / 4; ++i) dt[i] = softplus_exact(dt[i]);
        }
        if (a.z) {
#pragma unroll
            for (int i = 0; i < kTile / 4; ++i) dy[i] *= z[i] * sigmoid_hw(z[i]);
        }
#pragma unroll
        for (int i = kTile / 4 - 1; i >= 0; --i) {
            const bool in = dt0 + 4 * i + p.q < left;
            dt[i] = in ? dt[i] : 0.f;
            dy[i] = in ? dy[i] : 0.f;
            sdt += dt[i];
            auto step = [&](int j, float dtj, float dyj) {
                const float* cj = lc + (4 * i + j) * NP + p.q * S;
#pragma unroll
                for (int s = 0; s < S; ++s) g[s] = exp2_hw(A2[s] * dtj) * fmaf(dyj, cj[s], g[s]);
            };
            step(3, quad_lane<3>(dt[i]), quad_lane<3>(dy[i]));
            step(2, quad_lane<2>(dt[i]), quad_lane<2>(dy[i]));
            step(1, quad_lane<1>(dt[i]), quad_lane<1>(dy[i]));
            step(0, quad_lane<0>(dt[i]), quad_lane<0>(dy[i]));
        }
    }
    const size_t row = ((size_t)p.b * a.nchunk + chunk) * a.D + p.ch;
    sdt = quad_sum(sdt);
    if (p.live) {
        store_padded<S>(g, a.hend + row * NP, p.q);
        if (p.q == 0) a.sdt[row] = sdt;
    }
}

// Sums over the 16 channels of a wave of v[m][s], m = 0..MK-1 steps: an exchange of lane halves sums two steps at a time
// (each half of the lanes keeps one of them), then of rows of 16 lanes, then the four quads of a row are summed in place.
// Afterwards v[m][s], m < MK/4, holds the sums of step m + MK/4 * r in row r of lanes.
template <int MK, int S>
__device__ __forceinline__ void channel_sums(float (&v)[MK][S]) {
    constexpr int H = MK / 2, Q = MK / 4;
#pragma unroll
    for (int e = 0; e < H * S; e += 4) {
        float *a[4], *b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a[k] = &v[(e + k) / S][(e + k) % S];
            b[k] = &v[(e + k) / S + H][(e + k) % S];
        }
        swap32(*a[0], *b[0], *a[1], *b[1], *a[2], *b[2], *a[3], *b[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) *a[k] += *b[k];
    }
#pragma unroll
    for (int e = 0; e < Q * S; e += 4) {
        float *a[4], *b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a[k] = &v[(e + k) / S][(e + k) % S];
            b[k] = &v[(e + k) / S + Q][(e + k) % S];
        }
        swap16(*a[0], *b[0], *a[1], *b[1], *a[2], *b[2], *a[3], *b[3]);
#pragma unroll
        for (int k = 0; k < 4; ++k) *a[k] += *b[k];
    }
#pragma unroll
    for (int m = 0; m < Q; ++m)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            v[m][s] += dpp<0x128>(v[m][s]);           // row_ror:8
            v[m][s] += dpp<0x124>(v[m][s]);           // row_ror:4
        }
}

// Backward on a chunk, tile after tile from its end.  A tile's states are computed again from the state saved in front
// of it (a_t and h_t of the tile stay in registers), then the adjoint runs back through it:
//     g_t = C_t dy'_t + a_{t+1} g_{t+1},  dy' = dy silu(z)
//     dC_t = sum_d dy' h_t,  dB_t = sum_d g_t u_t,  du = g_t . B_t,  w = g_t a_t h_{t-1}
//     d raw = (A . w + du x) sigmoid(raw),  dx = du dt + D dy',  dA = sum w dt
// A channel's shares of dB and dC take the registers of its a_t and h_t; they are summed over the wave by lane exchanges
// and over the block's waves through LDS, and the block writes one row of partial sums per step.  One barrier a tile: the
// LDS areas are used in turn, and a tile's sums are taken after the next one's barrier.  Tiles of eight steps (16 states)
// keep the kernel at 193 registers and two waves a SIMD; sixteen steps spilled there (817 us for 128 x 501 x 256 fp32 where
// eight took 257) and took 357 us at one wave.  33 to 64 states take all 256 registers and 81 accumulation registers, one wave a
// SIMD, and spill 4.  Measured (medians): 285 us there, 499 us for 4 x 4096 x 2048 bf16, vector units 83 and 88 % busy with 100
// instructions a step and wave (16 of them the exchanges; the same sums as fp32 matrix products took 373 and 694 us where these
// took 257 and 473); 8 x 2048 x 2048 bf16 251 us with 4 states, 818 with 32, 2140 with 64.
template <class T, int S>
__global__ __launch_bounds__(256, S <= 8 ? 2 : 1) void scan_bwd_kernel(ScanArgs a) {
    constexpr int NP = 4 * S, MK = mark_steps<S>(), NI = MK / 4, RED = MK * 2 * NP;
    __shared__ float lds_b[2][MK * NP], lds_c[2][MK * NP];
    __shared__ __attribute__((aligned(16))) float red[2][4 * RED];    // [wave][step][B, C][state]
    const Place p = place(a, blockIdx.z);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int chunk = blockIdx.y, t0 = chunk * a.chunk, t1 = min(t0 + a.chunk, a.L), tend = min(t1, p.len), left = tend - t0;
    Column<T, MK> xs(a.x, a.xb, a.xt, p, t0), dts(a.dt, a.dtb, a.dtt, p, t0), zs(a.z, a.zb, a.zt, p, t0), dys(a.dy, a.dyb, a.dyt, p, t0);
    Shared<T, S, MK> bs(a.Bm, a.bb, a.bt, a.bg, p, t0, a.N), cs(a.Cm, a.cb, a.ct, a.cg, p, t0, a.N);
    float h0[S];
    auto fetch = [&](int dt) {
        dts.load(dt, left - dt, p.q);
        xs.load(dt, left - dt, p.q);
        dys.load(dt, left - dt, p.q);
        if (a.z) zs.load(dt, left - dt, p.q);
        bs.load(dt, left - dt);
        cs.load(dt, left - dt);
        load_padded<S>(h0, a.marks + ((size_t)p.b * a.nmark + (t0 + dt) / MK) * a.D * NP + (unsigned)p.ch * NP, p.q);
    };
    int dt0 = left > 0 ? (left - 1) / MK * MK : -1;
    if (dt0 >= 0) fetch(dt0);
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
        for (int s = 0; s < S; ++s) g[s] = g[s] == 0.f ? e[s] : fmaf(exp2_hw(A2[s] * sd), g[s], e[s]);
    }
    const size_t first = (size_t)p.b * a.L + t0;                      // row of the chunk's first step
    const OutColumn<T, MK> dx(a.dx, a.D, first, p), ddt(a.ddt, a.D, first, p), dz(a.dz, a.D, first, p);
    auto write_sums = [&](int dt, const float* r) {                   // of the tile at dt
        float* dst = a.pBC + ((first + dt) * gridDim.x + blockIdx.x) * (2 * NP);
        for (int e = threadIdx.x; e < RED; e += 256)
            if (dt + e / (2 * NP) < left)
                dst[(size_t)(e / (2 * NP)) * gridDim.x * (2 * NP) + e % (2 * NP)] = (r[e] + r[e + RED]) + (r[e + 2 * RED] + r[e + 3 * RED]);
    };
    float dD = 0.f, dbias = 0.f;
    auto write_piece = [&](int piece) {                               // its row of partial sums: [D][4S] of A, [D] of D, [D] of ddt_bias
        const auto part = window(a.pA + (((size_t)p.b * a.nchunk + chunk) * a.npiece + piece) * a.D * (NP + 2));
        window_store_states<S>(dA, part, p.live ? (p.ch * NP + p.q * S) * 4 : kOutside);
        const float sum_D = quad_sum(dD), sum_bias = quad_sum(dbias);
        window_store<float>(p.q == 0 ? sum_D : sum_bias, part, p.live && p.q < 2 ? (a.D * (NP + p.q) + p.ch) * 4 : kOutside, 0);
    };
    for (int piece = (max(left, 0) + kPiece - 1) / kPiece; piece < a.npiece; ++piece) write_piece(piece);      // behind the end: zeros
    int half = 0, before = -1;                                        // before: the tile whose sums wait in the other half
    auto tile = [&] {
        float *lb = lds_b[half], *lc = lds_c[half];
        bs.store(lb);
        cs.store(lc);
        float sg[NI], dt[NI], x[NI], dy[NI], z[NI], h1[S];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            x[i] = widen(xs.v[i]);
            dt[i] = widen(dts.v[i]) + bias;
            dy[i] = widen(dys.v[i]);
            z[i] = a.z ? widen(zs.v[i]) : 0.f;
        }
#pragma unroll
        for (int s = 0; s < S; ++s) h1[s] = h0[s];
        __syncthreads();
        if (before >= 0) write_sums(before, red[half ^ 1]);
        before = dt0;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const bool in = dt0 + 4 * i + p.q < left && p.live;
            sg[i] = a.softplus ? sigmoid_hw(dt[i]) : 1.f;
            if (a.softplus) dt[i] = softplus_exact(dt[i]);
            dt[i] = in ? dt[i] : 0.f;
            x[i] = in ? x[i] : 0.f;
            dy[i] = in ? dy[i] : 0.f;
        }
        float av[MK][S], h[MK][S], y[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            float part[4];
            const float u = dt[i] * x[i];
            auto step = [&](int j, float dtj, float uj) {
                const int m = 4 * i + j;
                const float *bj = lb + m * NP + p.q * S, *cj = lc + m * NP + p.q * S;
                float yj = 0.f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    av[m][s] = exp2_hw(A2[s] * dtj);
                    h[m][s] = fmaf(av[m][s], m ? h[m - 1][s] : h1[s], uj * bj[s]);
                    yj = fmaf(h[m][s], cj[s], yj);
                }
                part[j] = yj;
            };
            step(0, quad_lane<0>(dt[i]), quad_lane<0>(u));
            step(1, quad_lane<1>(dt[i]), quad_lane<1>(u));
            step(2, quad_lane<2>(dt[i]), quad_lane<2>(u));
            step(3, quad_lane<3>(dt[i]), quad_lane<3>(u));
            y[i] = fmaf(dskip, x[i], quad_sum_of_own(part[0], part[1], part[2], part[3], p.q));
        }
        if (a.z) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const float s = sigmoid_hw(z[i]);
                dz.store(dt0, left - dt0, p.q, i, dy[i] * y[i] * s * fmaf(z[i], 1.f - s, 1.f));
                dy[i] *= z[i] * s;
            }
        }
        if (dt0 > 0) fetch(dt0 - MK);
#pragma unroll
        for (int i = NI - 1; i >= 0; --i) {
            __builtin_amdgcn_sched_barrier(0);
            float pu[4], pt[4];
            const float u = dt[i] * x[i];
            auto step = [&](int j, float dtj, float uj, float dyj) {
                const int m = 4 * i + j;
                const float *bj = lb + m * NP + p.q * S, *cj = lc + m * NP + p.q * S;
                float du = 0.f, dd = 0.f;
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    g[s] = fmaf(dyj, cj[s], g[s]);
                    du = fmaf(g[s], bj[s], du);
                    const float ga = g[s] * av[m][s], w = ga * (m ? h[m - 1][s] : h1[s]);
                    dd = fmaf(A2[s], w, dd);
                    dA[s] = fmaf(dtj, w, dA[s]);
                    av[m][s] = g[s] * uj;                 // dB of this channel
                    h[m][s] *= dyj;                       // dC of this channel
                    g[s] = ga;
                }
                pu[j] = du;
                pt[j] = dd;
            };
            step(3, quad_lane<3>(dt[i]), quad_lane<3>(u), quad_lane<3>(dy[i]));
            step(2, quad_lane<2>(dt[i]), quad_lane<2>(u), quad_lane<2>(dy[i]));
            step(1, quad_lane<1>(dt[i]), quad_lane<1>(u), quad_lane<1>(dy[i]));
            step(0, quad_lane<0>(dt[i]), quad_lane<0>(u), quad_lane<0>(dy[i]));
            const float du = quad_sum_of_own(pu[0], pu[1], pu[2], pu[3], p.q);
            const float dr = sg[i] * fmaf(kLn2, quad_sum_of_own(pt[0], pt[1], pt[2], pt[3], p.q), du * x[i]);
            dx.store(dt0, left - dt0, p.q, i, fmaf(du, dt[i], dskip * dy[i]));
            ddt.store(dt0, left - dt0, p.q, i, dr);
            dbias += dt0 + 4 * i + p.q < left ? dr : 0.f;
            dD = fmaf(dy[i], x[i], dD);
        }
        channel_sums<MK, S>(av);
        channel_sums<MK, S>(h);
        if ((lane & 12) == 0) {
            const int m0 = (lane >> 4) * (MK / 4);
            float* r = red[half] + (wave * MK + m0) * 2 * NP + p.q * S;
#pragma unroll
            for (int m = 0; m < MK / 4; ++m) {
                Pack<float, S> vb, vc;
#pragma unroll
                for (int s = 0; s < S; ++s) { vb.set(s, av[m][s]); vc.set(s, h[m][s]); }
                vb.store(r + m * 2 * NP);
                vc.store(r + m * 2 * NP + NP);
            }
        }
    };
    while (dt0 >= 0) {
        const int piece = dt0 / kPiece;
        for (; dt0 >= piece * kPiece; dt0 -= MK, half ^= 1) tile();
        write_piece(piece);
#pragma unroll
        for (int s = 0; s < S; ++s) dA[s] = 0.f;
        dD = dbias = 0.f;
    }
    __syncthreads();
    if (before >= 0) write_sums(before, red[half ^ 1]);
    if (!p.live) return;
    if (chunk == 0 && a.dh0) store_states<S>(g, a.dh0 + ((size_t)p.b * a.D + p.ch) * a.N, p.q, a.N);
    for (int t = max(t0, tend) + p.q; t < t1; t += 4) {                // behind the sequence's end
        const size_t o = ((size_t)p.b * a.L + t) * a.D + p.ch;
        static_cast<T*>(a.dx)[o] = (T)0.f;
        static_cast<T*>(a.ddt)[o] = (T)0.f;
        if (a.dz) static_cast<T*>(a.dz)[o] = (T)0.f;
    }
}

// dB, dC [B, L, G, N] from the blocks' partial sums [B, L, G, tpg, 2, NP]: 4 x 4096 steps of 32 blocks, 67 MB in 20 us
template <class T>
__global__ __launch_bounds__(256) void scan_bc_kernel(const float* __restrict__ part, T* __restrict__ dB, T* __restrict__ dC,
                                                      const int* __restrict__ lengths, long long rows, int L, int G, int tpg, int N, int NP) {
    const int per = 2 * NP;                                           // a power of two: (which, n)
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (long long)gridDim.x * 256) {
        const long long row = i / per;
        const int r = (int)(i - row * per), n = r & (NP - 1);
        if (n >= N) continue;
        const long long bt = row / G;
        float s = 0.f;
        if (!lengths || bt % L < lengths[bt / L])
            for (int k = 0; k < tpg; ++k) s += part[(row * tpg + k) * per + r];
        (r < NP ? dB : dC)[row * N + n] = (T)s;
    }
}

// The token kernel's lanes take their states four at a time, so that a quad's accesses are 64 bytes in a row, and as vectors
// for any number of states (256 x 2048, one cache over and over: 64 states 62 -> 48 us, 61 states 114 -> 51; on caches that HBM
// has to bring, 75 and 89).
template <int S>
__device__ __forceinline__ int token_state(int q, int s) { return S <= 4 ? q * S + s : s / 4 * 16 + q * 4 + s % 4; }
template <int S>
__device__ __forceinline__ void load_token(float (&h)[S], const float* p, int q, int N) {
    constexpr int V = S < 4 ? S : 4;
#pragma unroll
    for (int s = 0; s < S; s += V) {
        Pack<float, V> v;
        v.load_n(p + token_state<S>(q, s), N - token_state<S>(q, s));
#pragma unroll
        for (int k = 0; k < V; ++k) h[s + k] = v.get(k);
    }
}
template <int S>
__device__ __forceinline__ void store_token(const float (&h)[S], float* p, int q, int N) {
    constexpr int V = S < 4 ? S : 4;
#pragma unroll
    for (int s = 0; s < S; s += V) {
        Pack<float, V> v;
#pragma unroll
        for (int k = 0; k < V; ++k) v.set(k, h[s + k]);
        v.store_n(p + token_state<S>(q, s), N - token_state<S>(q, s));
    }
}

// One token of every row; state [slots, D, N] is read and written once: 8N bytes a channel against 7N operations, HBM
// bound: 256 rows x 2048 channels x 16 states in 17 us (4.2 TB/s; 39 with a block per 64 channels and single loads); one row
// of 1280 channels in 4.  A block takes a row's blocks of 64 channels in turn (of one group: B and C are loaded once), so that
// the check of the row's slot against the rows before it is paid once for several of them.
template <class T, int S>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a, int parts, const int* __restrict__ slots, int nslots, float* __restrict__ state) {
    const int row = blockIdx.y, g = blockIdx.x / parts, part = blockIdx.x - g * parts;
    const int q = threadIdx.x & 3, lane_ch = threadIdx.x >> 2;
    float B[S], C[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int n = token_state<S>(q, s);
        B[s] = n < a.N ? at<T>(a.Bm, row * a.bb + g * a.bg + n) : 0.f;
        C[s] = n < a.N ? at<T>(a.Cm, row * a.cb + g * a.cg + n) : 0.f;
    }
    bool bad;
    const int slot = claim_slot(slots, row, nslots, &bad);
    for (int tile = part; tile < a.tpg; tile += parts) {
        if (tile * kCh + lane_ch >= a.Dg) break;
        const int ch = g * a.Dg + tile * kCh + lane_ch;
        T* out = static_cast<T*>(a.y) + (size_t)row * a.D + ch;
        if (bad || slot < 0) {
            if (q == 0) *out = (T)(bad ? __builtin_nanf("") : 0.f);
            continue;
        }
        float* st = state + ((size_t)slot * a.D + ch) * a.N;
        const float* Ap = a.A + (size_t)ch * a.N;
        float h[S], A2[S];
        load_token<S>(h, st, q, a.N);
        load_token<S>(A2, Ap, q, a.N);
        const float x = at<T>(a.x, row * a.xb + ch), z = a.z ? at<T>(a.z, row * a.zb + ch) : 0.f;
        float dt = at<T>(a.dt, row * a.dtb + ch) + (a.bias ? a.bias[ch] : 0.f);
        if (a.softplus) dt = softplus_exact(dt);
        float y = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            h[s] = fmaf(exp2_hw(A2[s] * kLog2e * dt), h[s], dt * x * B[s]);
            y = fmaf(h[s], C[s], y);
        }
        store_token<S>(h, st, q, a.N);
        y = quad_sum(y);
        if (a.Dp) y = fmaf(a.Dp[ch], x, y);
        if (a.z) y *= z * sigmoid_hw(z);
        if (q == 0) *out = (T)y;
    }
}

namespace {

int lane_states(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

struct ScanPlan {
    int S, NP, tpg, nchunk, chunk, npiece, nmark;
};

// Time is split where the blocks of the batch's channels alone do not fill the chip's 256 CUs: the first pass over the
// chunks costs about 0.6 of the second, so it does not pay before (128 sequences of 501 steps, 512 blocks: 115 us in one
// chunk, 36 + 99 us in two; 1 x 8192 steps x 2048 channels, 32 blocks: 66 + 103 us in 16 chunks, 64 + 97 in 32, 65 + 111 in
// 64).  With up to 8 states, where a step is short and one wave a SIMD waits for its loads, a split still pays at 256 blocks
// (8 x 2048 x 2048 x 4: 215 us in one chunk, 57 + 127 in four).  The backward kernel, two blocks a CU, gains from a split up to
// 384 blocks.  Sequences that end early (`ragged`) leave their last chunks empty, and finer chunks even that out (8 x 2001 x
// 1280, 26 chunks by this rule: 197 us in 3 chunks, 163 in 6, 126 in 21, 135 in 26).  Blocks do not span groups: a group of
// fewer than 64 channels leaves lanes idle, and counts here as if it did not.
ScanPlan scan_plan(const UnetmiScanDesc& d, bool ragged, bool backward) {
    ScanPlan p;
    p.S = lane_states(d.state);
    p.NP = 4 * p.S;
    const int Dg = d.channels / d.groups;
    p.tpg = (Dg + kCh - 1) / kCh;
    const long long blocks = (long long)d.batch * d.groups * p.tpg;
    long long want = 1;
    if (blocks > 0 && blocks < (backward ? 384 : p.S <= 2 ? 320 : 256)) want = ((ragged ? 4096 : 1024) + blocks - 1) / blocks;
    const long long most = (d.length + 63) / 64;                      // chunks of at least 64 steps
    if (want > most) want = most;
    if (want > 64) want = 64;
    if (want < 1) want = 1;
    p.chunk = (int)((d.length + want - 1) / want);
    p.chunk = (p.chunk + kAlign - 1) / kAlign * kAlign;
    if (p.chunk < kAlign) p.chunk = kAlign;
    p.nchunk = (d.length + p.chunk - 1) / p.chunk;
    if (p.nchunk < 1) p.nchunk = 1;
    p.npiece = (p.chunk + kPiece - 1) / kPiece;
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
    if (d->channels > (1 << 22) || d->length > (1 << 28)) return api_fail(UNETMI_E_UNSUPPORTED, w + ": more than 2^22 channels or 2^28 steps");
    for (const int64_t* s : {d->x_stride, d->dt_stride, d->z_stride, d->dy_stride}) {
        if (s[0] < 0 || s[1] < 0) return api_fail(UNETMI_E_BAD_DESC, w + ": negative stride");
        if (s[1] > UNETMI_SEQ_MAX_STEP) return api_fail(UNETMI_E_UNSUPPORTED, w + ": steps more than 2^24 elements apart");
    }
    for (const int64_t* s : {d->b_stride, d->c_stride})
        if (s[0] < 0 || s[1] < 0 || s[2] < 0) return api_fail(UNETMI_E_BAD_DESC, w + ": negative stride");
    for (const int64_t* s : {d->b_stride, d->c_stride})
        if (s[1] > UNETMI_SEQ_MAX_STEP) return api_fail(UNETMI_E_UNSUPPORTED, w + ": steps more than 2^24 elements apart");
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
    a.chunk = p.chunk; a.nchunk = p.nchunk; a.npiece = p.npiece; a.nmark = p.nmark; a.softplus = d.softplus != 0;
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
            hipLaunchKernelGGL((scan_fwd_kernel<T, S, kStates>), dim3(d.groups * p.tpg, p.nchunk - 1, d.batch), block, 0, s, a);
            const int rc = launched("ssm_scan_fwd states");
            if (rc != UNETMI_OK) return rc;
        }
        const dim3 grid(d.groups * p.tpg, p.nchunk, d.batch);
        if (a.marks) hipLaunchKernelGGL((scan_fwd_kernel<T, S, kMarks>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((scan_fwd_kernel<T, S, kOutputs>), grid, block, 0, s, a);
        return launched("ssm_scan_fwd");
    }
};
template <class T, int S>
struct RunScanBwd {
    static int run(const UnetmiScanDesc& d, const ScanPlan& p, const ScanArgs& a, void* dB, void* dC, float* dA, float* dD, float* dbias, hipStream_t s) {
        const dim3 block(256), grid(d.groups * p.tpg, p.nchunk, d.batch);
        int rc;
        if (p.nchunk > 1) {
            hipLaunchKernelGGL((scan_bwd_state_kernel<T, S>), dim3(d.groups * p.tpg, p.nchunk - 1, d.batch), block, 0, s, a);
            if ((rc = launched("ssm_scan_bwd states")) != UNETMI_OK) return rc;
        }
        hipLaunchKernelGGL((scan_bwd_kernel<T, S>), grid, block, 0, s, a);
        if ((rc = launched("ssm_scan_bwd")) != UNETMI_OK) return rc;
        const long long rows = (long long)d.batch * d.length * d.groups, threads = rows * 2 * p.NP;
        if (threads) {
            const long long blocks = (threads + 255) / 256;
            hipLaunchKernelGGL((scan_bc_kernel<T>), dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), block, 0, s, a.pBC, static_cast<T*>(dB),
                               static_cast<T*>(dC), a.lengths, rows, d.length, d.groups, p.tpg, d.state, p.NP);
            if ((rc = launched("ssm_scan_bwd B C")) != UNETMI_OK) return rc;
        }
        return launch_sum_rows(a.pA, d.batch * p.nchunk * p.npiece, {dA, d.channels * p.NP, p.NP, d.state}, {dD, d.channels, 1, 1},
                               {dbias, d.channels, 1, 1}, s);
    }
};
template <class T, int S>
struct RunScanStep {
    static int run(const UnetmiScanDesc& d, const ScanPlan& p, const ScanArgs& a, const int* slots, int nslots, float* state, hipStream_t s) {
        // about eight blocks a CU, as long as that many rows and channels are there (256 x 2048 x 16: 17.1 us, four 19.6, sixteen 20.2)
        long long parts = (2048 + (long long)d.batch * d.groups - 1) / ((long long)d.batch * d.groups);
        if (parts > p.tpg) parts = p.tpg;
        hipLaunchKernelGGL((scan_step_kernel<T, S>), dim3(d.groups * (int)parts, d.batch), dim3(256), 0, s, a, (int)parts, slots, nslots, state);
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
    const ScanPlan p = scan_plan(*d, false, false);
    return (size_t)d->batch * p.nmark * d->channels * p.NP * sizeof(float);
}

size_t unetmi_ssm_scan_fwd_workspace_bytes(const UnetmiScanDesc* d, int ragged) {
    if (scan_check(d, "ssm_scan_fwd_workspace_bytes") != UNETMI_OK) return 0;
    return summary_floats(*d, scan_plan(*d, ragged != 0, false)) * sizeof(float);
}

int unetmi_ssm_scan_fwd(const UnetmiScanDesc* d, const void* x, const void* dt, const float* A, const void* B, const void* C,
                        const float* D, const void* z, const float* dt_bias, const float* state, const int32_t* lengths, void* y,
                        float* state_out, float* marks, void* ws, size_t ws_bytes, void* stream) {
    const int rc = scan_check(d, "ssm_scan_fwd");
    if (rc != UNETMI_OK) return rc;
    if (d->batch == 0 || (d->length == 0 && !state_out)) return UNETMI_OK;
    if (!A || (d->length > 0 && (!x || !dt || !B || !C || !y))) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_fwd: null tensor pointer");
    const ScanPlan p = scan_plan(*d, lengths != nullptr, false);
    const size_t need = summary_floats(*d, p);
    if (need && (!ws || ws_bytes < need * sizeof(float))) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_fwd: workspace too small");
    ScanArgs a = scan_args(*d, p, x, dt, A, B, C, D, z, dt_bias);
    a.h0 = state; a.lengths = lengths; a.y = y; a.hT = state_out; a.marks = marks;
    a.hend = static_cast<float*>(ws);
    a.sdt = a.hend ? a.hend + (size_t)d->batch * p.nchunk * d->channels * p.NP : nullptr;
    return scan_dispatch<RunScan>(*d, p.S, *d, p, a, static_cast<hipStream_t>(stream));
}

size_t unetmi_ssm_scan_bwd_workspace_bytes(const UnetmiScanDesc* d, int ragged) {
    if (scan_check(d, "ssm_scan_bwd_workspace_bytes") != UNETMI_OK) return 0;
    const ScanPlan p = scan_plan(*d, ragged != 0, true);
    const size_t parts = (size_t)d->batch * p.nchunk * p.npiece;
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
    if (ws_bytes < unetmi_ssm_scan_bwd_workspace_bytes(d, lengths != nullptr)) return api_fail(UNETMI_E_BAD_ARG, "ssm_scan_bwd: workspace too small");
    const ScanPlan p = scan_plan(*d, lengths != nullptr, true);
    ScanArgs a = scan_args(*d, p, x, dt, A, B, C, D, z, dt_bias);
    a.lengths = lengths; a.marks = const_cast<float*>(marks);
    a.dy = dy; a.dhT = dstate_out; a.dx = dx; a.ddt = ddt; a.dz = dz; a.dh0 = dstate;
    const size_t chunks = (size_t)d->batch * p.nchunk;
    a.hend = static_cast<float*>(ws);                                 // multiples of four floats first: they stay 16-byte aligned
    a.pBC = a.hend + (p.nchunk > 1 ? chunks * d->channels * p.NP : 0);
    a.pA = a.pBC + (size_t)d->batch * d->length * d->groups * p.tpg * 2 * p.NP;
    a.sdt = a.pA + chunks * p.npiece * d->channels * (p.NP + 2);
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
    const ScanPlan p = scan_plan(*d, false, false);
    ScanArgs a = scan_args(*d, p, x, dt, A, B, C, D, z, dt_bias);
    a.y = y;
    return scan_dispatch<RunScanStep>(*d, p.S, *d, p, a, slots, num_slots, state, static_cast<hipStream_t>(stream));
}

}  // extern "C"
