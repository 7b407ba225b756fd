// Shared by the sequence operators (state space scan, causal convolution, block norm): element access in fp32 or
// bfloat16 storage, lane exchanges inside a quad, softplus / SiLU in fp32, and the fixed-order sum of partial rows.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/unetmi.h"
#include "io_types.hpp"

namespace unetmi {

int api_fail(int code, const std::string& msg);

typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__bf16 v) { return bf16_bits_to_f32(__builtin_bit_cast(unsigned short, v)); }

// V consecutive elements as one access of up to 16 bytes, widened to fp32.  The access needs no more alignment than its
// elements have (the hardware takes a vector access at any address), so rows of any width, stride or offset use it; the
// *_n forms are for the last vector of a row, which may hold fewer.
template <class T, int V>
struct Pack {
    typedef T raw __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    raw v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const raw*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<raw*>(p) = v; }
    __device__ __forceinline__ void load_n(const T* p, int n) {
        if (n >= V) return load(p);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < n ? p[i] : (T)0.f;
    }
    __device__ __forceinline__ void store_n(T* p, int n) const {
        if (n >= V) return store(p);
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = v[i];
    }
    __device__ __forceinline__ float get(int i) const { return widen(v[i]); }
    __device__ __forceinline__ void set(int i, float f) { v[i] = (T)f; }      // to nearest, ties to even
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)0.f;
    }
};
template <class T>
struct Pack<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *p; }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    __device__ __forceinline__ void load_n(const T* p, int n) { v = n > 0 ? *p : (T)0.f; }
    __device__ __forceinline__ void store_n(T* p, int n) const { if (n > 0) *p = v; }
    __device__ __forceinline__ float get(int) const { return widen(v); }
    __device__ __forceinline__ void set(int, float f) { v = (T)f; }
    __device__ __forceinline__ void zero() { v = (T)0.f; }
};
template <class T> constexpr int kVector = 16 / sizeof(T);

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// lane J of each quad to all four of its lanes; the lane one / two away inside the quad
template <int J>
__device__ __forceinline__ float quad_lane(float v) { return dpp<J * 0x55>(v); }
__device__ __forceinline__ float quad_xor1(float v) { return dpp<0xB1>(v); }
__device__ __forceinline__ float quad_xor2(float v) { return dpp<0x4E>(v); }

// lane q of a quad gets the quad's sum of p_q
__device__ __forceinline__ float quad_sum_of_own(float p0, float p1, float p2, float p3, int q) {
    const bool odd = q & 1, high = q & 2;
    const float r0 = (odd ? p1 : p0) + quad_xor1(odd ? p0 : p1);
    const float r1 = (odd ? p3 : p2) + quad_xor1(odd ? p2 : p3);
    return (high ? r1 : r0) + quad_xor2(high ? r0 : r1);
}
__device__ __forceinline__ float quad_sum(float p) {
    p += quad_xor1(p);
    return p + quad_xor2(p);
}

// a's odd rows of 16 lanes and b's even rows change places, / a's upper and b's lower 32 lanes: afterwards a + b holds a's sum
// over the exchanged lanes in the one half of the lanes and b's in the other.  Four pairs at a time, with the wait states
// that the compiler puts around its own.
__device__ __forceinline__ void swap16(float& a0, float& b0, float& a1, float& b1, float& a2, float& b2, float& a3, float& b3) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3\n\tv_permlane16_swap_b32 %4, %5\n\t"
                 "v_permlane16_swap_b32 %6, %7\n\ts_nop 1"
                 : "+v"(a0), "+v"(b0), "+v"(a1), "+v"(b1), "+v"(a2), "+v"(b2), "+v"(a3), "+v"(b3));
}
__device__ __forceinline__ void swap32(float& a0, float& b0, float& a1, float& b1, float& a2, float& b2, float& a3, float& b3) {
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\tv_permlane32_swap_b32 %2, %3\n\tv_permlane32_swap_b32 %4, %5\n\t"
                 "v_permlane32_swap_b32 %6, %7\n\ts_nop 1"
                 : "+v"(a0), "+v"(b0), "+v"(a1), "+v"(b1), "+v"(a2), "+v"(b2), "+v"(a3), "+v"(b3));
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float sigmoid_hw(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_hw(-kLog2e * v)); }

// log(1 + e^v) = max(v, 0) + log1p(t), t = e^-|v|: log1p(t) = 2 atanh(s), s = t / (2 + t) <= 1/3, with atanh(s) / s as the
// polynomial of degree 4 in s^2 through its values at the five Chebyshev nodes of [0, 1/9]: 8e-9 of the value.  Relative
// error stays at a few 2^-24 where the value is small -- step sizes live around 1e-3 -- where log(1 + t) itself would lose it.
__device__ __forceinline__ float softplus_exact(float v) {
    const float t = exp2_hw(-kLog2e * fabsf(v));
    const float s = t * __builtin_amdgcn_rcpf(2.f + t), s2 = s * s;
    float r = fmaf(s2, 0.14078889787197113f, 0.13982579112052917f);
    r = fmaf(r, s2, 0.20012298226356506f);
    r = fmaf(r, s2, 0.3333316147327423f);
    r = fmaf(r, s2, 1.f);
    return fmaf(2.f * s, r, fmaxf(v, 0.f));
}

// a sequence's length: lengths[b] held inside [0, L], or L
__device__ __forceinline__ int seq_len(const int* lengths, int b, int L) {
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > L ? L : n);
}

// The cache slot of a row of single tokens.  Negative: a padding row (zeros out, no state touched).  bad: out of range, or
// the slot of an earlier row of the same call -- two rows cannot both advance one stream -- : NaN out, no state touched.
// Every thread of the block calls it.
__device__ __forceinline__ int claim_slot(const int* slots, int row, int nslots, bool* bad) {
    const int s = slots ? slots[row] : row;
    int taken = 0;
    if (slots) {
        for (int i = threadIdx.x; i < row; i += blockDim.x) taken |= slots[i] == s;
        taken = __syncthreads_or(taken);
    }
    *bad = s >= nslots || (s >= 0 && taken);
    return s;
}

// Sums of R partial rows in one fixed order (bit-reproducible).  A row holds up to three pieces one after the other; a piece's
// columns come in groups of `padded`, of which the first `used` are kept, and go to `out`.
struct SumPiece {
    float* out;
    int columns, padded, used;
};
int launch_sum_rows(const float* rows, int R, SumPiece a, SumPiece b, SumPiece c, hipStream_t s);

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? UNETMI_OK : api_fail(UNETMI_E_HIP, std::string(what) + " launch: " + hipGetErrorString(e));
}

}  // namespace unetmi
