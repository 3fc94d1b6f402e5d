// Selective scan: what its forward and backward kernels share (ssm_scan_fwd.hip, ssm_scan_bwd.hip).
//
//     step[t] = softplus(dt[t] + dt_bias)                                                         per channel
//     h[t][n] = exp(step[t] A[n]) h[t-1][n] + step[t] x[t] B[t][n]                                N states per channel
//     y[t]    = (sum_n C[t][n] h[t][n] + D x[t]) silu(z[t])
//
// B and C are shared by the channels of a group.  Time-major [L][B][..]; a LANE is a channel and keeps its N states in
// registers, a wave is 64 channels of one row, a workgroup up to 4 waves of one group, which share B[t] and C[t] through LDS.
// Time runs in chunks of CH steps: the chunk's elements are requested one chunk ahead, its B and C sit in LDS as fp32.
//
// Few rows (long prompts) do not fill 1024 SIMDs: time is then cut into segments.  A segment maps its incoming state
// linearly, h_out = exp(A S) h_in + h_loc, S = the sum of its steps - one float per channel holds the whole decay.  Pass 1 finds
// (h_loc, S) of every segment, pass 2 chains them, pass 3 runs the segments from their incoming states; the backward pass
// does the same with the adjoint.  It costs the recurrence twice, so segments are cut only where half of the machine or more
// would stand idle (scan_plan).
#pragma once
#include "ssm_common.h"

namespace gmt_ssm {

constexpr int CH = 8;                    // steps per chunk = steps between kept states

struct ScanPlan { int np, waves, width, cblk, nseg, seglen, nck; };   // cblk: workgroups across a group's channels

// Padded state count, workgroup width and time segments
static inline ScanPlan scan_plan(int L, int B, int C, int N, int G)
{
    ScanPlan p;
    p.np = N <= 8 ? 8 : N <= 16 ? 16 : 32;
    const int cg = C / G;
    p.waves = cg <= 64 ? 1 : cg <= 128 ? 2 : 4;
    p.width = 64 * p.waves;
    p.cblk = (cg + p.width - 1) / p.width;
    const long long waves = (long long)B * G * p.cblk * p.waves;
    long long nseg = 1;
    if (waves <= 512) {
        nseg = 4096 / waves;
        const long long most = L / (4 * CH);
        if (nseg > most) nseg = most;
        if (nseg < 4) nseg = 1;          // the recurrence runs twice: two or three segments gain nothing
    }
    p.seglen = (int)(((L + nseg - 1) / nseg + CH - 1) / CH * CH);
    p.nseg = (L + p.seglen - 1) / p.seglen;
    p.nck = (L - 1) / CH;                // states kept before steps CH, 2 CH, ...
    return p;
}

static inline int scan_check(const gmt_scan_args* a)
{
    GMT_CHECK_ARG(a && a->x && a->dt && a->A && a->Bm && a->Cm && a->L > 0 && a->B > 0 && a->C > 0 && a->N > 0 && a->G > 0);
    GMT_CHECK_ARG(a->C % a->G == 0);
    GMT_CHECK_ARG((a->x_scale != nullptr) == (a->dt_scale != nullptr) && (a->z == nullptr || (a->x_scale != nullptr) == (a->z_scale != nullptr)));
    if (a->N > 32) return GMT_ERR_UNSUPPORTED;
    const ScanPlan p = scan_plan(a->L, a->B, a->C, a->N, a->G);
    if ((long long)p.cblk * a->G * a->B * p.nseg >= (1LL << 24)) return GMT_ERR_UNSUPPORTED;
    return GMT_OK;
}

// pointers and pitches of one launch by value; T / M: element types of x, dt, z / of everything else
template <class T, class M> struct ScanArgs {
    const typename T::raw* x; const typename T::raw* dt; const typename T::raw* z;
    const void *xq, *dtq, *zq; const unsigned char *xs, *dts, *zs;        // 8-bit checkpoints: codes, exponents
    const typename M::raw* Bm; const typename M::raw* Cm;
    const float *A, *D, *dt_bias, *state; const int* lengths;
    typename M::raw* y; float* state_out; float* ck; float* seg_h; float* seg_s;
    const typename M::raw* dy; const float* dstate_out;
    typename M::raw *dx, *ddt, *dz, *dB, *dC; float* dstate; float* part; float* bc_part;
    long long x_t, x_b, dt_t, dt_b, z_t, z_b, B_t, B_b, B_g, C_t, C_b, C_g, dy_t, dy_b;
    int L, B, C, N, G, P;
    ScanPlan p;
};

template <class T, class M> ScanArgs<T, M> scan_args(const gmt_scan_args* a)
{
    ScanArgs<T, M> s;
    s.x = (const typename T::raw*)a->x; s.dt = (const typename T::raw*)a->dt; s.z = (const typename T::raw*)a->z;
    s.xq = a->x; s.dtq = a->dt; s.zq = a->z; s.xs = a->x_scale; s.dts = a->dt_scale; s.zs = a->z_scale;
    s.Bm = (const typename M::raw*)a->Bm; s.Cm = (const typename M::raw*)a->Cm;
    s.A = a->A; s.D = a->D; s.dt_bias = a->dt_bias; s.state = a->state; s.lengths = a->lengths;
    s.y = (typename M::raw*)a->y; s.state_out = a->state_out; s.ck = a->ck; s.seg_h = s.seg_s = nullptr;
    s.dy = (const typename M::raw*)a->dy; s.dstate_out = a->dstate_out;
    s.dx = (typename M::raw*)a->dx; s.ddt = (typename M::raw*)a->ddt; s.dz = (typename M::raw*)a->dz;
    s.dB = (typename M::raw*)a->dB; s.dC = (typename M::raw*)a->dC; s.dstate = a->dstate; s.part = s.bc_part = nullptr;
    s.x_t = a->x_t; s.x_b = a->x_b; s.dt_t = a->dt_t; s.dt_b = a->dt_b; s.z_t = a->z_t; s.z_b = a->z_b;
    s.B_t = a->B_t; s.B_b = a->B_b; s.B_g = a->B_g; s.C_t = a->C_t; s.C_b = a->C_b; s.C_g = a->C_g;
    s.dy_t = a->dy_t; s.dy_b = a->dy_b;
    s.L = a->L; s.B = a->B; s.C = a->C; s.N = a->N; s.G = a->G; s.P = 0;
    s.p = scan_plan(a->L, a->B, a->C, a->N, a->G);
    return s;
}

// Between unrolled steps: B and C of the next step are read from LDS when it comes to them, not 8 steps ahead into registers.
__device__ __forceinline__ void step_fence() { asm volatile("" ::: "memory"); __builtin_amdgcn_sched_barrier(0); }

// ... and what a step computes from v stays behind this point.
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// which = 0: x, 1: dt, 2: z at (t, b, c)
template <class T, class M, int WHICH> __device__ __forceinline__ typename T::raw load_elem(const ScanArgs<T, M>& a, int t, int b, int c)
{
    if constexpr (__is_same(T, Q8)) {
        const long long row = (long long)t * a.B + b;
        const void* q = WHICH == 0 ? a.xq : WHICH == 1 ? a.dtq : a.zq;
        const unsigned char* s = WHICH == 0 ? a.xs : WHICH == 1 ? a.dts : a.zs;
        Q8::raw r;
        r.q = ((const signed char*)q)[row * a.C + c];
        r.s = s[row * ((a.C + 31) / 32) + c / 32];
        return r;
    } else {
        return WHICH == 0 ? a.x[t * a.x_t + b * a.x_b + c] : WHICH == 1 ? a.dt[t * a.dt_t + b * a.dt_b + c] : a.z[t * a.z_t + b * a.z_b + c];
    }
}

// N floats of a channel's row (state buffers [B][C][N], A [C][N]) <-> NP registers, zero-padded
template <int NP> __device__ __forceinline__ void load_states(const float* p, int N, float (&h)[NP])
{
    if (N == NP && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int n = 0; n < NP; n += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + n);
            h[n] = v.x; h[n + 1] = v.y; h[n + 2] = v.z; h[n + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int n = 0; n < NP; ++n) h[n] = n < N ? p[n] : 0.f;
    }
}
template <int NP> __device__ __forceinline__ void store_states(float* p, int N, const float (&h)[NP])
{
    if (N == NP && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int n = 0; n < NP; n += 4) *reinterpret_cast<float4*>(p + n) = make_float4(h[n], h[n + 1], h[n + 2], h[n + 3]);
    } else {
#pragma unroll
        for (int n = 0; n < NP; ++n) if (n < N) p[n] = h[n];
    }
}

// The kept states and the segments' states: [..][B][NP][C], N padded to NP with zeros.
template <int NP> __device__ __forceinline__ void load_kept(const float* p, long long slot, int B, int b, int C, int c, float (&h)[NP])
{
    const float* k = p + (slot * B + b) * NP * C + c;
#pragma unroll
    for (int n = 0; n < NP; ++n) h[n] = k[(long long)n * C];
}
template <int NP> __device__ __forceinline__ void store_kept(float* p, long long slot, int B, int b, int C, int c, const float (&h)[NP])
{
    float* k = p + (slot * B + b) * NP * C + c;
#pragma unroll
    for (int n = 0; n < NP; ++n) k[(long long)n * C] = h[n];
}

// The chunk's B (or C) as fp32 [CH][NP] in LDS, by all threads of the workgroup: request() one chunk ahead, put() behind the wait.
template <class M, int NP> struct MapTile {
    static constexpr int PER = CH * NP / 64;            // (one wave; wider workgroups need fewer)
    typename M::raw v[PER];
    __device__ __forceinline__ void request(const typename M::raw* p, long long pt, int t0, int t1, int N) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * blockDim.x, s = i / NP, n = i % NP;
            v[j] = from_f<M>(0.f);
            if (s < CH && n < N && t0 + s < t1) v[j] = p[(t0 + s) * pt + n];
        }
    }
    __device__ __forceinline__ void put(float* lds) const {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * blockDim.x;
            if (i < CH * NP) lds[i] = to_f(v[j]);
        }
    }
};

// host functions of one file that the other calls
int scan_chain(float* seg_h, const float* seg_s, const float* A, const float* first, int nseg, int np, int B, int C, int N,
               int reverse, hipStream_t stream);
int scan_states_q8(const gmt_scan_args* a, hipStream_t stream);
long long scan_bwd_floats(const gmt_scan_args* a);

}  // namespace gmt_ssm
