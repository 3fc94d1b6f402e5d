// Selective scan, forward (ssm_scan.h has the formulas and the layout), its single-step form, and the segment chain that the
// backward pass shares.
#include <type_traits>
#include "ssm_scan.h"

namespace {

using namespace gmt_ssm;

// what a launch writes: y; y and the kept states; the kept states alone; a segment's (h_loc, S)
enum Mode { OUT = 0, TRAIN = 1, STATES = 2, LOCAL = 3 };

template <class T, class M, int NP, int PARTS, int MODE, bool GATED>
__global__ __launch_bounds__(256)
void scan_fwd_kernel(ScanArgs<T, M> a)
{
    constexpr bool Y = MODE == OUT || MODE == TRAIN, KEEP = MODE == TRAIN || MODE == STATES;
    constexpr int NS = NP / PARTS, OWN = CH / PARTS;
    __shared__ __align__(16) float sB[2][CH * NP], sC[Y ? 2 : 1][Y ? CH * NP : 1];
    const int cb = blockIdx.x % a.p.cblk, rest = blockIdx.x / a.p.cblk;
    const int g = rest % a.G, rest2 = rest / a.G;
    const int seg = rest2 / a.B, b = a.sorted ? row_of_rank(a.lengths, rest2, a.B, a.L) : rest2 % a.B;
    const Lanes<PARTS> ln;
    const int cg = a.C / a.G, ci = cb * a.p.chans + ln.chan, n0 = ln.part * NS;
    const bool on = ci < cg, wave_on = cb * a.p.chans + (int)(threadIdx.x >> 6) * (64 / PARTS) < cg;
    const unsigned c = g * cg + (on ? ci : cg - 1);     // lanes beyond the group repeat its last channel
    const int len = length_of(a.lengths, b, a.L);
    const int t0 = seg * a.p.seglen, t1 = min(t0 + a.p.seglen, a.L), te = min(t1, len);

    float A2[NS], h[NS];
    load_states<NS>(a.A + (long long)c * a.N, n0, a.N, A2);
#pragma unroll
    for (int n = 0; n < NS; ++n) { A2[n] = base2(A2[n]); h[n] = 0.f; }
    const long long row = (long long)b * a.C + c;
    const unsigned koff = (unsigned)(n0 * a.C + c) * 4, yoff = (unsigned)((ln.part * a.B * a.C + c) * sizeof(typename M::raw));
    if (MODE != LOCAL) {
        if (a.p.nseg > 1) load_kept<NP, NS>(a.seg_h, seg, a.B, b, a.C, koff, h);
        else if (a.state) load_states<NS>(a.state + row * a.N, n0, a.N, h);
    }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = Y && a.D ? a.D[c] : 0.f;
    const typename M::raw* Bp = a.Bm + b * a.B_b + g * a.B_g;
    const typename M::raw* Cp = a.Cm + b * a.C_b + g * a.C_g;
    const Seq<T> xq(a.x, a.xs, a.x_t, a.x_b, b, ln.part, c, a.B, a.C), dq(a.dt, a.dts, a.dt_t, a.dt_b, b, ln.part, c, a.B, a.C),
        zq(a.z, a.zs, a.z_t, a.z_b, b, ln.part, c, a.B, a.C);

    Own<T, PARTS> xr, dr, zr;
    MapTile<M, NP> mB, mC;
    auto request = [&](int tc) {
        xr.request(xq, tc, te, ln.part);
        dr.request(dq, tc, te, ln.part);
        if (GATED) zr.request(zq, tc, te, ln.part);
        mB.request(Bp, a.B_t, tc, te, a.N);
        if (Y) mC.request(Cp, a.C_t, tc, te, a.N);
    };
    float S = 0.f;
    if (te > t0) request(t0);
    int buf = 0;
    for (int tc = t0; tc < te; tc += CH, buf ^= 1) {
        const Own<T, PARTS> xc = xr, dc = dr, zc = zr;
        mB.put(sB[buf]);
        if (Y) mC.put(sC[Y ? buf : 0]);
        // one barrier a chunk: a buffer is written again two chunks later, behind the next barrier, which its readers have passed
        lds_barrier();
        if (tc + CH < te) request(tc + CH);
        if (KEEP && wave_on) store_kept<NP, NS>(a.ck, tc / CH, a.B, b, a.C, koff, h);
        if (MODE == STATES && tc + CH >= te) break;     // nothing is kept behind the last chunk
        if (wave_on) {
            float xv[OWN], st[OWN];                     // st: the step, then (its step done) the sum over the states
#pragma unroll
            for (int j = 0; j < OWN; ++j) {
                const bool live = tc + j * PARTS + ln.part < te;        // behind the row's end: a step of 0, which changes nothing
                float sig;
                xv[j] = live ? to_f(xc.v[j]) : 0.f;
                st[j] = softplus(to_f(dc.v[j]) + bias, sig);
                st[j] = live ? st[j] : 0.f;
                if (MODE == LOCAL) S += st[j];
            }
            float sts[PARTS], xs[PARTS], ys[PARTS];
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                const int j = s / PARTS, k = s % PARTS;
                if (k == 0) { ln.spread(st[j], sts); ln.spread(xv[j], xs); }
                pin(sts[k]);
                const float sx = sts[k] * xs[k];
                float y0 = 0.f, y1 = 0.f;
                const float* Bt = sB[buf] + s * NP + n0;
                const float* Ct = sC[Y ? buf : 0] + (Y ? s * NP + n0 : 0);
#pragma unroll
                for (int n = 0; n < NS; ++n) {
                    const float e = __builtin_amdgcn_exp2f(sts[k] * A2[n]);
                    h[n] = fmaf(e, h[n], sx * Bt[n]);
                    if (Y) { if (n & 1) y1 = fmaf(h[n], Ct[n], y1); else y0 = fmaf(h[n], Ct[n], y0); }
                }
                if (Y) {
                    ys[k] = y0 + y1;
                    pin(ys[k]);
                    if (k == PARTS - 1) st[j] = ln.gather(ys);
                }
                step_fence();
            }
            if (Y) {
#pragma unroll
                for (int j = 0; j < OWN; ++j) {
                    const int t = tc + j * PARTS + ln.part;
                    float o = fmaf(Dc, xv[j], st[j]);
                    if (GATED) { const float zv = to_f(zc.v[j]); o *= zv * sigmoid(zv); }
                    if (t < t1) put_out<M>(a.y, ((long long)(tc + j * PARTS) * a.B + b) * a.C, yoff, t < te ? o : 0.f);
                }
            }
        }
    }
    if (!on) return;
    if (MODE == LOCAL) {
        store_kept<NP, NS>(a.seg_h, seg, a.B, b, a.C, koff, h);
        S = ln.sum(S);
        if (ln.part == 0) a.seg_s[(long long)(seg * a.B + b) * a.C + c] = S;
        return;
    }
    // the segment in which the row ends (the first one for an empty row) holds its final state
    if (Y && a.state_out && ((len > t0 && len <= t1) || (len == 0 && seg == 0))) store_states<NS>(a.state_out + row * a.N, n0, a.N, h);
    if (Y)
        for (int t = t0 + (max(te - t0, 0) + CH - 1) / CH * CH + ln.part; t < t1; t += PARTS) a.y[((long long)t * a.B + b) * a.C + c] = from_f<M>(0.f);
}

// exp(A S) h + loc of a segment, x = A S in base 2.  A growing state (A > 0) can have a decay beyond fp32 over a segment while the state itself,
// zero or small, stays finite, as it does step by step: the factor is then taken in three parts (x >= 378 overflows for every h but 0).
template <bool GROWS> __device__ __forceinline__ float chain_step(float x, float h, float loc) {
    if (!GROWS) return fmaf(__builtin_amdgcn_exp2f(x), h, loc);
    const float e = __builtin_amdgcn_exp2f(fminf(x, 378.f) * (1.0f / 3.0f));
    return fmaf(e, e * (e * h), loc);
}

// seg_h: (h_loc of every segment) -> (its incoming state), in place.  The chain of a state is cut into 8 runs: each is joined to one
// link by a thread of its own, the 8 links are chained through LDS, and each thread walks its run again from where it
// starts.  Latency is all of the cost: 16 segments are requested at once (128 segments x 16384 states: a single walk 78 us, with 16
// requested ahead 14 us, in 8 runs 6 us).
constexpr int RUNS = 8;
__global__ __launch_bounds__(32 * RUNS)
void scan_chain_kernel(float* seg_h, const float* __restrict__ seg_s, const float* __restrict__ A, const float* __restrict__ first,
                       int nseg, int np, int B, int C, int N, int reverse)
{
    __shared__ float run_h[RUNS][32], run_s[RUNS][32];
    const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
    const long long n_all = (long long)B * np * C, i = (long long)blockIdx.x * 32 + lane;
    const int c = (int)(i % C), n = (int)(i / C % np);
    const long long b = i / C / np;
    const bool on = i < n_all && n < N;                 // (padding: zeros in every segment)
    const float A2 = on ? base2(A[(long long)c * N + n]) : 0.f;
    const int per = (nseg + RUNS - 1) / RUNS, k0 = run * per, k1 = min(k0 + per, nseg);
    constexpr int AHEAD = 16;
    float loc[AHEAD], step[AHEAD];
    auto request = [&](int kb) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int k = min(kb + j, k1 - 1), s = reverse ? nseg - 1 - k : k;
            loc[j] = seg_h[s * n_all + i];
            step[j] = seg_s[((long long)s * B + b) * C + c];
        }
    };
    auto walk = [&](float& h, float& S, bool store, auto grows) {       // (a run of AHEAD segments or fewer is requested once)
        for (int kb = k0; kb < k1; kb += AHEAD) {
            if (!store || per > AHEAD) request(kb);
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                if (kb + j >= k1) break;
                const int s = reverse ? nseg - 1 - (kb + j) : kb + j;
                if (store) seg_h[s * n_all + i] = h;
                h = chain_step<grows>(A2 * step[j], h, loc[j]);
                S += step[j];
            }
        }
    };
    auto chain = [&](auto grows) {
        float h = 0.f, S = 0.f;
        if (on) walk(h, S, false, grows);
        run_h[run][lane] = h;
        run_s[run][lane] = S;
        __syncthreads();
        if (!on) return;
        h = first ? first[(b * C + c) * N + n] : 0.f;
        for (int r = 0; r < run; ++r) h = chain_step<grows>(A2 * run_s[r][lane], h, run_h[r][lane]);
        walk(h, S, true, grows);
    };
    // the same for the whole workgroup (it has a barrier inside): its runs hold the same 32 states
    if (__any(A2 > 0.f)) chain(std::true_type{});
    else chain(std::false_type{});
}

// One step of every row: state [B][C][N] -> state_out (may be the same buffer).  The state, read and written once, is all of the
// traffic: LPC lanes hold a channel, V = 4 or 1 states each, whole lines of it, and a sum over LPC neighbouring lanes.  A workgroup
// keeps the parameters of its 256 / LPC channels in registers and walks down the rows, ROWS at a time, so that as many
// lines are in flight from each lane.
template <class M, int V> __device__ __forceinline__ void load_map(const typename M::raw* p, bool wide, int n0, int N, float (&o)[V])
{
    if constexpr (V == 4) {
        if (wide) {                                     // (uniform) 4 elements at once
            typedef typename M::raw vec __attribute__((ext_vector_type(4)));
            const vec v = *reinterpret_cast<const vec*>(p + n0);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = to_f((typename M::raw)v[k]);
            return;
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) o[k] = to_f(p[n0 + k]);
}

template <class M, int V, int LPC, int ROWS>
__global__ __launch_bounds__(256)
void scan_step_kernel(const typename M::raw* __restrict__ x, long long x_b, const typename M::raw* __restrict__ dt, long long dt_b,
                      const typename M::raw* __restrict__ z, long long z_b, const typename M::raw* __restrict__ Bm, long long B_b,
                      long long B_g, const typename M::raw* __restrict__ Cm, long long C_b, long long C_g, const float* __restrict__ A,
                      const float* __restrict__ D, const float* __restrict__ dt_bias, const float* state, float* state_out,
                      const unsigned char* __restrict__ active, typename M::raw* __restrict__ y, int B, int C, int N, int G, int gx, int wide)
{
    constexpr int CHANS = 256 / LPC;
    const int part = threadIdx.x % LPC, ci = blockIdx.x % gx * CHANS + threadIdx.x / LPC;
    const bool on = ci < C;
    const int c = on ? ci : C - 1, g = c / (C / G);
    // lanes beyond the states or the channels repeat the last ones, add nothing and store nothing
    const bool has = part * V < N;
    const int n0 = has ? part * V : N - V;
    float A2[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A2[v] = A[(long long)c * N + n0 + v] * LOG2E;
    const float bias = dt_bias ? dt_bias[c] : 0.f, Dc = D ? D[c] : 0.f;
    const long long at0 = (long long)c * N + n0, pitch = (long long)C * N;
    const int groups = gridDim.x / gx;
    for (int b0 = blockIdx.x / gx * ROWS; b0 < B; b0 += groups * ROWS) {
        float h[ROWS][V], Bv[ROWS][V], Cv[ROWS][V];
        typename M::raw xr[ROWS], dr[ROWS], zr[ROWS];
        bool act[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int b = min(b0 + r, B - 1);
            const float* sp = state + b * pitch + at0;
            if constexpr (V == 4) *reinterpret_cast<float4*>(h[r]) = *reinterpret_cast<const float4*>(sp);
            else h[r][0] = *sp;
            xr[r] = x[b * x_b + c];
            dr[r] = dt[b * dt_b + c];
            zr[r] = z ? z[b * z_b + c] : from_f<M>(0.f);
            load_map<M, V>(Bm + b * B_b + g * B_g, wide, n0, N, Bv[r]);
            load_map<M, V>(Cm + b * C_b + g * C_g, wide, n0, N, Cv[r]);
            act[r] = !active || active[b];
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int b = b0 + r;
            if (b >= B) break;
            float yv = 0.f;
            if (act[r]) {                               // (an inactive row's state stays as it is)
                const float xv = to_f(xr[r]);
                float sig;
                const float st = softplus(to_f(dr[r]) + bias, sig), sx = st * xv;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    h[r][v] = fmaf(__builtin_amdgcn_exp2f(st * A2[v]), h[r][v], sx * Bv[r][v]);
                    yv = fmaf(h[r][v], Cv[r][v], yv);
                }
                yv = has ? yv : 0.f;
#pragma unroll
                for (int o = 1; o < LPC; o <<= 1) yv += __shfl_xor(yv, o, 64);
                yv = fmaf(Dc, xv, yv);
                if (z) { const float zv = to_f(zr[r]); yv *= zv * sigmoid(zv); }
            }
            if (on && has && (act[r] || state_out != state)) {
                float* sp = state_out + b * pitch + at0;
                if constexpr (V == 4) *reinterpret_cast<float4*>(sp) = *reinterpret_cast<float4*>(h[r]);
                else *sp = h[r][0];
            }
            if (on && part == 0) y[(long long)b * C + c] = from_f<M>(yv);
        }
    }
}

template <class T, class M, int NP, int PARTS, int MODE> int launch(const ScanArgs<T, M>& a, hipStream_t stream)
{
    const dim3 grid((unsigned)((long long)a.p.cblk * a.G * a.B * a.p.nseg));
    if constexpr (MODE == OUT || MODE == TRAIN) {
        if (a.z) hipLaunchKernelGGL((scan_fwd_kernel<T, M, NP, PARTS, MODE, true>), grid, dim3(a.p.width), 0, stream, a);
        else hipLaunchKernelGGL((scan_fwd_kernel<T, M, NP, PARTS, MODE, false>), grid, dim3(a.p.width), 0, stream, a);
    } else {
        hipLaunchKernelGGL((scan_fwd_kernel<T, M, NP, PARTS, MODE, false>), grid, dim3(a.p.width), 0, stream, a);
    }
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}
template <class T, class M, int NP, int MODE> int by_parts(const ScanArgs<T, M>& a, hipStream_t stream)
{
    return a.p.parts == 1 ? launch<T, M, NP, 1, MODE>(a, stream) : launch<T, M, NP, 2, MODE>(a, stream);
}
template <class T, class M, int MODE> int by_np(const ScanArgs<T, M>& a, hipStream_t stream)
{
    return a.p.np == 8 ? by_parts<T, M, 8, MODE>(a, stream) : a.p.np == 16 ? by_parts<T, M, 16, MODE>(a, stream) : by_parts<T, M, 32, MODE>(a, stream);
}

// segments (if any), then the pass itself
template <class T, class M, int MODE> int run(const gmt_scan_args* args, hipStream_t stream)
{
    ScanArgs<T, M> a = scan_args<T, M>(args, fwd_plan(args->L, args->B, args->C, args->N, args->G));
    if (a.p.nseg > 1) {
        const long long nh = (long long)a.p.nseg * a.B * a.p.np * a.C, ns = (long long)a.p.nseg * a.B * a.C;
        if (!args->workspace || args->workspace_floats < nh + ns) return GMT_ERR_WORKSPACE;
        a.seg_h = args->workspace;
        a.seg_s = args->workspace + nh;
        if (int rc = by_np<T, M, LOCAL>(a, stream)) return rc;
        if (int rc = scan_chain(a.seg_h, a.seg_s, a.A, a.state, a.p.nseg, a.p.np, a.B, a.C, a.N, 0, stream)) return rc;
    }
    return by_np<T, M, MODE>(a, stream);
}

template <class M, int V, int LPC> int launch_step(const gmt_scan_args* a, const unsigned char* active, hipStream_t stream)
{
    using R = typename M::raw;
    const int chans = 256 / LPC, gx = (a->C + chans - 1) / chans;
    // 4 rows at a time once 8 workgroups a CU are at work, 16 workgroups a CU at most
    const int rows = (long long)gx * a->B >= 4 * 8 * 256 ? 4 : 1;
    long long groups = (a->B + rows - 1) / rows;
    const long long most = (16 * 256 + gx - 1) / gx;
    if (groups > most) groups = most;
    const int esz = sizeof(R);
    const int wide = (((uintptr_t)a->Bm | (uintptr_t)a->Cm) % (4 * esz)) == 0 && ((a->B_b | a->B_g | a->C_b | a->C_g) & 3) == 0;
    auto k = rows == 4 ? scan_step_kernel<M, V, LPC, 4> : scan_step_kernel<M, V, LPC, 1>;
    hipLaunchKernelGGL(k, dim3((unsigned)(gx * groups)), dim3(256), 0, stream, (const R*)a->x, a->x_b, (const R*)a->dt, a->dt_b,
                       (const R*)a->z, a->z_b, (const R*)a->Bm, a->B_b, a->B_g, (const R*)a->Cm, a->C_b, a->C_g, a->A, a->D, a->dt_bias,
                       a->state, a->state_out, active, (R*)a->y, a->B, a->C, a->N, a->G, gx, wide);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}
template <class M> int step(const gmt_scan_args* a, const unsigned char* active, hipStream_t stream)
{
    const int N = a->N;
    if (N % 4 == 0 && (((uintptr_t)a->state | (uintptr_t)a->state_out) & 15) == 0)
        return N <= 4 ? launch_step<M, 4, 1>(a, active, stream) : N <= 8 ? launch_step<M, 4, 2>(a, active, stream)
             : N <= 16 ? launch_step<M, 4, 4>(a, active, stream) : launch_step<M, 4, 8>(a, active, stream);
    return N <= 4 ? launch_step<M, 1, 4>(a, active, stream) : N <= 8 ? launch_step<M, 1, 8>(a, active, stream)
         : N <= 16 ? launch_step<M, 1, 16>(a, active, stream) : launch_step<M, 1, 32>(a, active, stream);
}

}  // namespace

namespace gmt_ssm {
int scan_chain(float* seg_h, const float* seg_s, const float* A, const float* first, int nseg, int np, int B, int C, int N,
               int reverse, hipStream_t stream)
{
    const long long n = (long long)B * np * C;
    hipLaunchKernelGGL(scan_chain_kernel, dim3((unsigned)((n + 31) / 32)), dim3(32 * RUNS), 0, stream, seg_h, seg_s, A, first, nseg, np, B, C,
                       N, reverse);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}
// the states before every chunk, from 8-bit checkpoints (backward pass)
int scan_states_q8(const gmt_scan_args* a, hipStream_t stream)
{
    return a->bf16 ? run<Q8, B16, STATES>(a, stream) : run<Q8, F32, STATES>(a, stream);
}
}  // namespace gmt_ssm

extern "C" int gmt_selective_scan_workspace(const gmt_scan_args* a, long long* ck_floats, long long* fwd_floats, long long* bwd_floats)
{
    if (int rc = scan_check(a)) return rc;
    GMT_CHECK_ARG(ck_floats && fwd_floats && bwd_floats);
    const ScanPlan p = fwd_plan(a->L, a->B, a->C, a->N, a->G);
    *ck_floats = (long long)p.nck * a->B * p.np * a->C;
    *fwd_floats = p.nseg > 1 ? (long long)p.nseg * a->B * a->C * (p.np + 1) : 0;
    const long long bwd = scan_bwd_floats(a);
    *bwd_floats = bwd > *fwd_floats ? bwd : *fwd_floats;    // from 8-bit checkpoints the states are found again in it first
    return GMT_OK;
}

extern "C" int gmt_selective_scan_fwd(const gmt_scan_args* a, hipStream_t stream)
{
    if (int rc = scan_check(a)) return rc;
    GMT_CHECK_ARG(a->y && !a->x_scale);
    if (a->ck) return a->bf16 ? run<B16, B16, TRAIN>(a, stream) : run<F32, F32, TRAIN>(a, stream);
    return a->bf16 ? run<B16, B16, OUT>(a, stream) : run<F32, F32, OUT>(a, stream);
}

extern "C" int gmt_selective_scan_step(const gmt_scan_args* a, const unsigned char* active, hipStream_t stream)
{
    if (int rc = scan_check_any(a)) return rc;
    // rows are 64-bit offsets and a loop; 8 channels a workgroup or more, fewer than 2^24 workgroups of 256 threads
    if (a->C >= 1 << 26 || a->B > MAX_STEPS) return GMT_ERR_UNSUPPORTED;
    GMT_CHECK_ARG(a->y && a->state && a->state_out && a->L == 1 && !a->x_scale);
    return a->bf16 ? step<B16>(a, active, stream) : step<F32>(a, active, stream);
}
