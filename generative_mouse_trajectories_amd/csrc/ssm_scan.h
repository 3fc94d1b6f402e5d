// Selective scan: what its forward and backward kernels share (ssm_scan_fwd.hip, ssm_scan_bwd.hip).
//
//     step[t] = softplus(dt[t] + dt_bias)                                                         per channel
//     h[t][n] = exp(step[t] A[n]) h[t-1][n] + step[t] x[t] B[t][n]                                N states per channel
//     y[t]    = (sum_n C[t][n] h[t][n] + D x[t]) silu(z[t])
//
// B and C are shared by the channels of a group.  Time-major [L][B][..].  PARTS = 1, 2 or 4 lanes hold a channel with N / PARTS
// states each in registers; a workgroup is up to 8 waves of one row and one group, which share B[t] and C[t] through LDS as fp32.
// Time runs in chunks of CH steps, requested one chunk ahead, in three phases: what depends on (t, channel) alone - softplus,
// gate - for all steps at once, divided between a channel's lanes; the recurrence, step by step; the outputs, divided again.
// The recurrence is 5 instructions a state and step, one of them an exponential at half rate, and VALU issue is what bounds these
// kernels: N = 16 forward with kept states 165 issue slots for a step of 64 channels, 88 % of them filled (L=256 B=256 C=512 bf16 155 us =
// 216e9 elements a second); backward 434, 80 % filled (455 us).  Pairs of times beside a choice below compare both sides in one build on one
// card when it was made; later steps moved both.
//
// Few rows (long prompts) do not fill 1024 SIMDs: time is then cut into segments.  A segment maps its incoming state
// linearly, h_out = exp(A S) h_in + h_loc, S = the sum of its steps - one float per channel holds the whole decay.  Pass 1 finds
// (h_loc, S) of every segment, pass 2 chains them, pass 3 runs the segments from their incoming states; the backward pass
// does the same with the adjoint.  It costs the recurrence twice, so segments are cut only where few waves run (scan_plan).
#pragma once
#include <cfloat>
#include "ssm_common.h"

namespace gmt_ssm {

constexpr int BWD_WAVES = 8;              // waves a workgroup of the backward pass, at most
constexpr int CH = 8;                    // steps per chunk; the state before every chunk is kept for the backward pass

struct ScanPlan { int np, parts, waves, width, chans, cblk, nseg, seglen, nck; };   // chans: channels a workgroup; cblk: workgroups a group

// Padded state count, lanes per channel, workgroup width (at most max_waves waves) and time segments: up to 512 waves (the idle ones of a
// workgroup with fewer channels counted) and four segments of 32 steps or more.  From 513 waves on time is not cut, although up to 1023 waves of the
// forward pass leave SIMDs idle, and 65 .. 255 workgroups of 8 waves of the backward pass leave CUs idle.
static inline ScanPlan scan_plan(int L, int B, int C, int N, int G, int parts, int max_waves)
{
    ScanPlan p;
    p.np = N <= 8 ? 8 : N <= 16 ? 16 : 32;
    p.parts = parts;
    const int cg = C / G, per = 64 / parts;
    p.waves = 1;
    while (p.waves < max_waves && p.waves * per < cg) p.waves *= 2;
    p.width = 64 * p.waves;
    p.chans = p.waves * per;
    p.cblk = (cg + p.chans - 1) / p.chans;
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
    p.nck = (L + CH - 1) / CH;
    return p;
}
// One lane per channel costs the fewest instructions; two lanes fill the machine with half of the rows
static inline ScanPlan fwd_plan(int L, int B, int C, int N, int G)
{
    const ScanPlan p = scan_plan(L, B, C, N, G, 1, 4);
    return (long long)B * G * p.cblk * p.waves >= 4096 ? p : scan_plan(L, B, C, N, G, 2, 4);
}
// 4 .. 8 states a lane: what the backward pass can keep of a chunk in registers (N=32, L=256 B=128 C=512 bf16: 16 states a lane 760 us,
// 8 states 505 us; N=16, B=256: 4 states a lane 536 us, 8 states 473 us)
static inline ScanPlan bwd_plan(int L, int B, int C, int N, int G) { return scan_plan(L, B, C, N, G, N > 16 ? 4 : 2, BWD_WAVES); }

// what holds of whole sequences and of a single step
static inline int scan_check_any(const gmt_scan_args* a)
{
    GMT_CHECK_ARG(a && a->x && a->dt && a->A && a->Bm && a->Cm && a->L > 0 && a->B > 0 && a->C > 0 && a->N > 0 && a->G > 0);
    GMT_CHECK_ARG(a->C % a->G == 0);
    GMT_CHECK_ARG((a->x_scale != nullptr) == (a->dt_scale != nullptr) && (a->z == nullptr || (a->x_scale != nullptr) == (a->z_scale != nullptr)));
    return a->N > 32 ? GMT_ERR_UNSUPPORTED : GMT_OK;
}
static inline int scan_check(const gmt_scan_args* a)
{
    if (int rc = scan_check_any(a)) return rc;
    if (a->L > MAX_STEPS) return GMT_ERR_UNSUPPORTED;
    // byte offsets within four steps (B and C: a chunk) and within a row's kept states are 31 bits
    const long long lim = 1LL << 27;
    if ((long long)a->C * 128 >= 1LL << 31 || a->x_t < 0 || a->dt_t < 0 || a->z_t < 0 || a->dy_t < 0 ||
        a->B_t < 0 || a->C_t < 0 || a->B_t >= lim / 2 || a->C_t >= lim / 2) return GMT_ERR_UNSUPPORTED;
    if (a->C >= lim || a->x_t >= lim || a->dt_t >= lim || a->z_t >= lim || a->dy_t >= lim || (long long)a->B * a->C >= lim ||
        (long long)a->B * a->G * a->N >= lim / 2) return GMT_ERR_UNSUPPORTED;
    // A launch stays below 2^32 threads: B G C / G channels padded to whole waves, at most 64 for each of fewer than 2^26 (row, group) pairs of
    // up to 64 channels, at most twice the 2^27 channels of wider groups; segments and two lanes a channel come with few waves only.
    return GMT_OK;
}

// Rows of unequal length, if they fill more than 2048 waves (what the backward pass keeps on the machine), are taken in descending order,
// so that the last ones are short: L=129 B=512 C=256 fp32 with lengths of 64 .. 129, backward 276 -> 256 us, forward 88 -> 85 us (rows that
// come in descending order: 247 and 78 us).
static inline bool by_length(const gmt_scan_args* a, const ScanPlan& p)
{
    return a->lengths && p.nseg == 1 && a->B <= ORDERED && a->L < 1 << 21 && (long long)a->B * a->G * p.cblk * p.waves > 2048;
}

// pointers and pitches of one launch by value; T / M: element types of x, dt, z / of everything else
template <class T, class M> struct ScanArgs {
    const void *x, *dt, *z; const unsigned char *xs, *dts, *zs;           // elements, or codes and exponents of 8-bit checkpoints
    const typename M::raw* Bm; const typename M::raw* Cm;
    const float *A, *D, *dt_bias, *state; const int* lengths;
    typename M::raw* y; float* state_out; float* ck; float* seg_h; float* seg_s;
    const typename M::raw* dy; const float* dstate_out;
    typename M::raw *dx, *ddt, *dz, *dB, *dC; float* dstate; float* part; float* bc_part;
    long long x_t, x_b, dt_t, dt_b, z_t, z_b, B_t, B_b, B_g, C_t, C_b, C_g, dy_t, dy_b;
    int L, B, C, N, G, P;
    int sorted;                                         // rows are taken by length
    ScanPlan p;
};

template <class T, class M> ScanArgs<T, M> scan_args(const gmt_scan_args* a, const ScanPlan& p)
{
    ScanArgs<T, M> s;
    s.x = a->x; s.dt = a->dt; s.z = a->z; s.xs = a->x_scale; s.dts = a->dt_scale; s.zs = a->z_scale;
    s.Bm = (const typename M::raw*)a->Bm; s.Cm = (const typename M::raw*)a->Cm;
    s.A = a->A; s.D = a->D; s.dt_bias = a->dt_bias; s.state = a->state; s.lengths = a->lengths;
    s.y = (typename M::raw*)a->y; s.state_out = a->state_out; s.ck = a->ck; s.seg_h = s.seg_s = nullptr;
    s.dy = (const typename M::raw*)a->dy; s.dstate_out = a->dstate_out;
    s.dx = (typename M::raw*)a->dx; s.ddt = (typename M::raw*)a->ddt; s.dz = (typename M::raw*)a->dz;
    s.dB = (typename M::raw*)a->dB; s.dC = (typename M::raw*)a->dC; s.dstate = a->dstate; s.part = s.bc_part = nullptr;
    s.x_t = a->x_t; s.x_b = a->x_b; s.dt_t = a->dt_t; s.dt_b = a->dt_b; s.z_t = a->z_t; s.z_b = a->z_b;
    if (a->x_scale) { s.x_t = s.dt_t = s.z_t = (long long)a->B * a->C; s.x_b = s.dt_b = s.z_b = a->C; }
    s.B_t = a->B_t; s.B_b = a->B_b; s.B_g = a->B_g; s.C_t = a->C_t; s.C_b = a->C_b; s.C_g = a->C_g;
    s.dy_t = a->dy_t; s.dy_b = a->dy_b;
    s.L = a->L; s.B = a->B; s.C = a->C; s.N = a->N; s.G = a->G; s.P = 0;
    s.sorted = by_length(a, p);
    s.p = p;
    return s;
}

// Between unrolled steps: B and C of the next step are read from LDS when it comes to them, not 8 steps ahead into registers.
__device__ __forceinline__ void step_fence() { asm volatile("" ::: "memory"); __builtin_amdgcn_sched_barrier(0); }
// ... and v is computed before this point, what follows from it behind it (a sum is not put off with its terms in registers).
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// The workgroup's LDS writes before it are seen behind it.  __syncthreads() would also wait for the stores of the chunk before.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E;             // quad_perm

// (a, b) -> lanes 0 - 31: a summed over bit 5 of the lane, lanes 32 - 63: b
__device__ __forceinline__ float half32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// (a, b) -> lanes with bit 4 clear: a summed over that bit, set: b
__device__ __forceinline__ float half16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ---- lanes of a channel.  With PARTS parts, the halves or quarters of the wave: neighbouring channels each, whole memory sectors.
// Few permlane swaps spread the values of PARTS steps over the parts or gather their sums.
template <int PARTS> struct Lanes {
    static constexpr int OWN = CH / PARTS;              // a lane's own steps of a chunk: j * PARTS + part
    int part; unsigned chan;                            // chan: channel within the workgroup
    __device__ __forceinline__ Lanes() {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        part = lane / (64 / PARTS);
        chan = wave * (64 / PARTS) + lane % (64 / PARTS);
    }
    // a lane's value for its own step -> those of the PARTS neighbouring steps, on every lane of the channel
    __device__ __forceinline__ void spread(float own, float (&v)[PARTS]) const {
        if constexpr (PARTS == 1) v[0] = own;
        else {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(own), __float_as_uint(own), false, false);
            if constexpr (PARTS == 2) {
                v[0] = __uint_as_float(r[0]);
                v[1] = __uint_as_float(r[1]);
            } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const auto q = __builtin_amdgcn_permlane16_swap(r[k], r[k], false, false);
                    v[2 * k] = __uint_as_float(q[0]);
                    v[2 * k + 1] = __uint_as_float(q[1]);
                }
            }
        }
    }
    // the lanes' terms for PARTS neighbouring steps -> the sum for a lane's own step
    __device__ __forceinline__ float gather(const float (&v)[PARTS]) const {
        if constexpr (PARTS == 1) return v[0];
        else if constexpr (PARTS == 2) return half32(v[0], v[1]);
        else return half16(half32(v[0], v[2]), half32(v[1], v[3]));
    }
    __device__ __forceinline__ float sum(float v) const {
        if constexpr (PARTS > 1) v = half32(v, v);
        if constexpr (PARTS > 2) v = half16(v, v);
        return v;
    }
};

// One sequence of a row, as a lane sees it.  Uniform base of a step plus a 32-bit byte offset of the lane (its part's step and its
// channel): the scalar-base form of the memory instructions, no 64-bit vector arithmetic.
template <class T> struct Seq {
    const char* p; int pt; unsigned off, off0;          // (at step 0), pitch of a step in bytes; off0: of the first part
    const char* sp; int spt; unsigned soff, soff0;      // exponents of an 8-bit checkpoint
    __device__ __forceinline__ Seq(const void* base, const unsigned char* scale, long long t, long long b, int row, int part, unsigned c,
                                   int rows, int channels) {
        constexpr int E = __is_same(T, Q8) ? 1 : (int)sizeof(typename T::raw);
        p = (const char*)base + row * b * E;
        pt = (int)t * E;
        off0 = c * E;
        off = (unsigned)(part * pt) + off0;
        const int n_sc = (channels + 31) / 32;
        sp = (const char*)scale + (long long)row * n_sc;
        spt = rows * n_sc;
        soff0 = c / 32;
        soff = (unsigned)(part * spt) + soff0;
    }
};
// A lane's own elements for one chunk.  Steps behind the end repeat the last one and are masked by the caller.
template <class T, int PARTS> struct Own {
    static constexpr int OWN = CH / PARTS;
    typename T::raw v[OWN];
    __device__ __forceinline__ void request(const Seq<T>& q, int tc, int te, int part) {
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
            const int t = min(tc + j * PARTS, te - 1);
            // (uniform) every part's step exists; else the parts without one take the last one that does
            const bool all = t + PARTS <= te;
            const int back = PARTS > 2 ? min(part, te - 1 - t) : 0;
            const unsigned off = all ? q.off : q.off0 + back * q.pt, soff = all ? q.soff : q.soff0 + back * q.spt;
            const Uniform p = uniform(q.p + (long long)t * q.pt);
            if constexpr (__is_same(T, Q8)) {
                v[j].q = load_at<signed char>(p, off);
                v[j].s = load_at<unsigned char>(uniform(q.sp + (long long)t * q.spt), soff);
            } else v[j] = load_at<typename T::raw>(p, off);
        }
    }
};
// the same for an output [L][B][C]
template <class M> __device__ __forceinline__ void put_out(typename M::raw* base, long long uniform_elem, unsigned off_bytes, float v) {
    store_at<typename M::raw>(uniform(base + uniform_elem), off_bytes, from_f<M>(v));
}

// NS floats of a channel's row, states n0 .. n0 + NS - 1 (state buffers [B][C][N], A [C][N]) <-> registers, zero-padded
template <int NS> __device__ __forceinline__ void load_states(const float* p, int n0, int N, float (&h)[NS])
{
    if ((N & 3) == 0 && n0 + NS <= N && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int n = 0; n < NS; n += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + n0 + n);
            h[n] = v.x; h[n + 1] = v.y; h[n + 2] = v.z; h[n + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = n0 + n < N ? p[n0 + n] : 0.f;
    }
}
template <int NS> __device__ __forceinline__ void store_states(float* p, int n0, int N, const float (&h)[NS])
{
    if ((N & 3) == 0 && n0 + NS <= N && ((uintptr_t)p & 15) == 0) {
#pragma unroll
        for (int n = 0; n < NS; n += 4) *reinterpret_cast<float4*>(p + n0 + n) = make_float4(h[n], h[n + 1], h[n + 2], h[n + 3]);
    } else {
#pragma unroll
        for (int n = 0; n < NS; ++n) if (n0 + n < N) p[n0 + n] = h[n];
    }
}
// A for exponentials in base 2.  A masked step is one of length 0, which must leave a state as it is: -inf (a state without memory, or what
// base 2 makes of the lowest numbers) becomes the lowest number, because 0 * -inf is NaN.
__device__ __forceinline__ float base2(float A) {
    const float a = A * LOG2E;
    return a < -FLT_MAX ? -FLT_MAX : a;
}
// The kept states (slot k: before step k CH) and the segments' states: [..][B][NP][C], N padded to NP with zeros.  off: (n0 C + c) * 4
template <int NP, int NS> __device__ __forceinline__ void load_kept(const float* p, long long slot, int B, int b, int C, unsigned off, float (&h)[NS])
{
    const char* k = reinterpret_cast<const char*>(p + (slot * B + b) * NP * C);
#pragma unroll
    for (int n = 0; n < NS; ++n) h[n] = load_at<float>(uniform(k + (long long)n * C * 4), off);
}
template <int NP, int NS> __device__ __forceinline__ void store_kept(float* p, long long slot, int B, int b, int C, unsigned off, const float (&h)[NS])
{
    char* k = reinterpret_cast<char*>(p + (slot * B + b) * NP * C);
#pragma unroll
    for (int n = 0; n < NS; ++n) store_at<float>(uniform(k + (long long)n * C * 4), off, h[n]);
}

// The chunk's B (or C) as fp32 [CH][NP] in LDS, by all threads of the workgroup: request() one chunk ahead, put() behind the wait.
template <class M, int NP> struct MapTile {
    static constexpr int PER = CH * NP / 64;            // (one wave; wider workgroups need fewer)
    typename M::raw v[PER];
    __device__ __forceinline__ void request(const typename M::raw* p, int pt, int t0, int t1, int N) {
        const Uniform q = uniform(p + (long long)t0 * pt);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int i = threadIdx.x + j * blockDim.x, s = i / NP, n = i % NP;
            v[j] = from_f<M>(0.f);
            if (s < CH && n < N && t0 + s < t1)
                v[j] = load_at<typename M::raw>(q, (unsigned)((s * pt + n) * (int)sizeof(typename M::raw)));
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
