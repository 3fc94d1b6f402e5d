// Shared by the selective-scan, short-convolution and 8-bit checkpoint kernels (ssm_*.hip, ckpt8.hip).
#pragma once
#include "gmt_common.h"

namespace gmt_ssm {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// ---- element types.  Q8 is the 8-bit checkpoint (ckpt8.hip): int8 codes of a contiguous tensor and one exponent byte s per
// 32 channels of a row; an element is code * 2^(s - 127).  s = 255 marks a block that held an infinity or a NaN: its codes
// are 0, and 0 * inf = NaN for every element without a test.
struct F32 { using raw = float; };
struct B16 { using raw = unsigned short; };
struct Q8 { struct raw { signed char q; unsigned char s; }; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
__device__ __forceinline__ float to_f(Q8::raw v) { return (float)v.q * __uint_as_float((unsigned)v.s << 23); }

__device__ __forceinline__ unsigned short f_to_bf16(float v) {                // round to nearest even
    return __builtin_bit_cast(unsigned short, (__bf16)v);
}
template <class M> __device__ __forceinline__ typename M::raw from_f(float v);
template <> __device__ __forceinline__ float from_f<F32>(float v) { return v; }
template <> __device__ __forceinline__ unsigned short from_f<B16>(float v) { return f_to_bf16(v); }

// softplus(v) = max(v, 0) + log(1 + u), u = exp(-|v|) in (0, 1].  log(1 + u) = 2 atanh(s), s = u / (2 + u) <= 1/3, by its odd
// power series (the first term left out is below 2^-29 of the sum): steps of 0.001 come out to fp32 precision, where
// log2(1 + exp) on the hardware units keeps only the digits of 1 + u (6e-5 off at 0.001).  sig = its derivative.
__device__ __forceinline__ float softplus(float v, float& sig) {
    const float u = __builtin_amdgcn_exp2f(-fabsf(v) * LOG2E);
    const float s = u * __builtin_amdgcn_rcpf(2.0f + u);
    const float q = s * s;
    float p = 1.0f / 15.0f;
    p = fmaf(p, q, 1.0f / 13.0f);
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    p = p * q;
    const float r = __builtin_amdgcn_rcpf(1.0f + u);
    sig = v >= 0.f ? r : u * r;
    return fmaxf(v, 0.f) + 2.0f * fmaf(s, p, s);
}
// silu(v) = v / (1 + exp(-v)).  exp(-v) overflows to inf below -88: rcp gives 0 and v * 0 = -0, the limit.
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * LOG2E)); }

// A pointer to device memory that is the same on all lanes, kept in scalar registers: `at(uniform(p), 32-bit byte offset)` is then
// one global memory instruction (otherwise the compiler adds the lane's offset first, in 64-bit vector arithmetic, and keeps the
// results).
typedef const __attribute__((address_space(1))) char* Uniform;
__device__ __forceinline__ Uniform uniform(const void* p) {
    Uniform g = (Uniform)p;
    asm("" : "+s"(g));
    return g;
}
template <class E> __device__ __forceinline__ E load_at(Uniform p, unsigned off) {
    return *reinterpret_cast<const __attribute__((address_space(1))) E*>(p + off);
}
template <class E> __device__ __forceinline__ void store_at(Uniform p, unsigned off, E v) {
    *(__attribute__((address_space(1))) E*)(p + off) = v;
}

// steps of a sequence, at most: sums of a step and a segment's length (fewer than 2^18 beyond the last step) are 32-bit
constexpr int MAX_STEPS = 0x7fffffff - (1 << 18) + 1;

__device__ __forceinline__ int length_of(const int* lengths, int b, int L) {
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : n > L ? L : n;               // a length outside 0 .. L cannot lead outside the buffers
}

// The row whose length is number `rank` in descending order (rows of one length: the lower number first), found by every wave
// for itself: bit by bit the largest key that more than `rank` keys reach.  For up to ORDERED rows of fewer than 2^21 steps; 16 keys a lane.
constexpr int ORDERED = 1024;
__device__ __forceinline__ int row_of_rank(const int* lengths, int rank, int B, int L) {
    const int lane = threadIdx.x & 63;
    unsigned key[ORDERED / 64];
#pragma unroll
    for (int k = 0; k < ORDERED / 64; ++k) {
        const int i = k * 64 + lane;
        key[k] = i < B ? (unsigned)length_of(lengths, i, L) * ORDERED + (ORDERED - 1 - i) : 0;
    }
    unsigned top = 0;
    for (int bit = 41 - __builtin_clz(L); bit >= 0; --bit) {
        const unsigned want = top | 1u << bit;
        int n = 0;
#pragma unroll
        for (int k = 0; k < ORDERED / 64; ++k)
            if (k * 64 < B) n += __popcll(__ballot(key[k] >= want));
        if (n > rank) top = want;
    }
    return ORDERED - 1 - (int)(top % ORDERED);
}

// ---- sum of P slabs, `pitch` floats apart, in a fixed order: out[i] = sum_p slab[p][i], i < n.  64 columns x 16 slab groups a workgroup,
// eight loads in flight a thread.
static __global__ __launch_bounds__(1024) void slab_reduce_kernel(const float* __restrict__ slab, float* __restrict__ out, long long n, long long pitch, int P)
{
    __shared__ float part[16][64];
    const int col = threadIdx.x & 63, grp = threadIdx.x >> 6;
    for (long long i0 = (long long)blockIdx.x * 64; i0 < n; i0 += (long long)gridDim.x * 64) {
        const long long i = i0 + col;
        float s = 0.f;
        if (i < n) {
            int p = grp;
            for (; p + 7 * 16 < P; p += 8 * 16) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = slab[(p + 16 * j) * pitch + i];
#pragma unroll
                for (int j = 0; j < 8; ++j) s += v[j];
            }
            for (; p < P; p += 16) s += slab[p * pitch + i];
        }
        part[grp][col] = s;
        __syncthreads();
        if (grp == 0 && i < n) {
#pragma unroll
            for (int g = 1; g < 16; ++g) s += part[g][col];
            out[i] = s;
        }
        __syncthreads();                                // before `part` is written again
    }
}
static inline int launch_slab_reduce(const float* slab, float* out, long long n, long long pitch, int P, hipStream_t stream)
{
    const int grid = gmt_grid_1d(n, 64, 1 << 20);       // (below 2^32 threads)
    hipLaunchKernelGGL(slab_reduce_kernel, dim3(grid), dim3(1024), 0, stream, slab, out, n, pitch, P);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}

}  // namespace gmt_ssm
