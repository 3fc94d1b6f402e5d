// Selective scan, backward (ssm_scan.h has the formulas and the layout).  With dy' = dy silu(z) and g[t] = d(loss)/d(h[t]):
//     g[t][n]  = C[t][n] dy'[t] + exp(step[t+1] A[n]) g[t+1][n]
//     dB[t][n] = sum_c g step x,     dC[t][n] = sum_c h dy'          over the channels of the group
//     q        = g exp(step A) h[t-1]:  dA[n] += q step,  dstep = sum_n q A + x sum_n g B
//     dx = step sum_n g B + D dy',   dz = dy (sum_n C h + D x) silu'(z),   ddt = dstep softplus'(dt + dt_bias)
// A chunk is walked forward from its kept state with all its h in registers, then backward.  The forward pass keeps the state
// before every chunk (or, from 8-bit checkpoints, scan_states_q8 finds them first, so that every gradient is that of the
// operator at the values the checkpoints stand for).
//
// dB and dC are sums over lanes: 2 N values a step.  They leave by halving exchanges - a lane hands half of its values to its
// partner and keeps the partner's other half, v_permlane32/16_swap then DPP - 70 instructions for 32 values where 32 separate
// wave sums take 192.  The waves of a workgroup meet in LDS, workgroups of one group through slabs: no float atomics, results
// do not depend on the order of execution.
#include "ssm_scan.h"

namespace {

using namespace gmt_ssm;

template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_XOR7 = 0x141, DPP_XOR8 = 0x128;     // quad_perm, row_half_mirror, row_ror:8

// (a, b) -> lanes with bit 5 (16 lanes: bit 4) clear: a summed over that bit, set: b
__device__ __forceinline__ float half32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float half16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int CTRL> __device__ __forceinline__ float half_dpp(float a, float b, bool upper) {
    const float keep = upper ? b : a, send = upper ? a : b;
    return keep + dpp<CTRL>(send);
}
// v[0 .. NV) summed over the wave: lane l returns value index_of(l)
template <int NV> __device__ __forceinline__ float wave_sums(float (&v)[NV], int lane)
{
    static_assert(NV == 16 || NV == 32, "values per lane");
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) v[i] = half32(v[i], v[i + NV / 2]);
#pragma unroll
    for (int i = 0; i < NV / 4; ++i) v[i] = half16(v[i], v[i + NV / 4]);
    const bool b3 = lane & 8, b2 = lane & 4, b1 = lane & 2;
#pragma unroll
    for (int i = 0; i < NV / 8; ++i) v[i] = half_dpp<DPP_XOR8>(v[i], v[i + NV / 8], b3);
#pragma unroll
    for (int i = 0; i < NV / 16; ++i) v[i] = half_dpp<DPP_XOR7>(v[i], v[i + NV / 16], b2);
    float s = v[0];
    if constexpr (NV == 32) s = half_dpp<DPP_XOR2>(v[0], v[1], b1);
    else s += dpp<DPP_XOR2>(s);
    return s + dpp<DPP_XOR1>(s);
}
template <int NV> __device__ __forceinline__ int index_of(int lane) { return NV == 32 ? lane >> 1 : lane >> 2; }

// a segment's adjoint: (adjoint of its incoming state for a zero adjoint behind it, S)
template <class T, class M, int NP, bool GATED>
__global__ __launch_bounds__(256)
void scan_bwd_local_kernel(ScanArgs<T, M> a)
{
    __shared__ __align__(16) float sC[2][CH * NP];
    const int cb = blockIdx.x % a.p.cblk, rest = blockIdx.x / a.p.cblk;
    const int gr = rest % a.G, rest2 = rest / a.G;
    const int b = rest2 % a.B, seg = rest2 / a.B;
    const int cg = a.C / a.G, ci = cb * a.p.width + threadIdx.x;
    const bool on = ci < cg;
    const int c = gr * cg + (on ? ci : cg - 1);
    const int len = length_of(a.lengths, b, a.L);
    const int t0 = seg * a.p.seglen, t1 = min(t0 + a.p.seglen, a.L), te = min(t1, len);
    float A2[NP], g[NP];
    load_states<NP>(a.A + (long long)c * a.N, a.N, A2);
#pragma unroll
    for (int n = 0; n < NP; ++n) { A2[n] *= LOG2E; g[n] = 0.f; }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    const typename M::raw* Cp = a.Cm + b * a.C_b + gr * a.C_g;
    float S = 0.f;
    int buf = 0;
    for (int k = te > t0 ? (te - t0 + CH - 1) / CH - 1 : -1; k >= 0; --k, buf ^= 1) {
        const int tc = t0 + k * CH;
        typename T::raw dr[CH], zr[CH];
        typename M::raw yr[CH];
        MapTile<M, NP> mC;
#pragma unroll
        for (int s = 0; s < CH; ++s) {
            const int t = min(tc + s, te - 1);
            dr[s] = load_elem<T, M, 1>(a, t, b, c);
            if (GATED) zr[s] = load_elem<T, M, 2>(a, t, b, c);
            yr[s] = a.dy[t * a.dy_t + b * a.dy_b + c];
        }
        mC.request(Cp, a.C_t, tc, te, a.N);
        mC.put(sC[buf]);
        __syncthreads();
#pragma unroll
        for (int s = CH - 1; s >= 0; --s) {
            const bool live = tc + s < te;
            float sig, st = softplus(to_f(dr[s]) + bias, sig);
            st = live ? st : 0.f;
            pin(st);
            float d = live ? to_f(yr[s]) : 0.f;
            if (GATED) { const float zv = live ? to_f(zr[s]) : 0.f; d *= zv * sigmoid(zv); }
            S += st;
#pragma unroll
            for (int n = 0; n < NP; ++n) g[n] = __builtin_amdgcn_exp2f(st * A2[n]) * fmaf(d, sC[buf][s * NP + n], g[n]);
            step_fence();
        }
    }
    if (!on) return;
    store_kept<NP>(a.seg_h, seg, a.B, b, a.C, c, g);
    a.seg_s[(long long)(seg * a.B + b) * a.C + c] = S;
}

template <class T, class M, int NP, bool GATED>
__global__ __launch_bounds__(256, 1)
void scan_bwd_kernel(ScanArgs<T, M> a)
{
    constexpr int NV = NP == 8 ? 16 : 32;               // values per wave_sums call: dB and dC together, or one after the other
    __shared__ __align__(16) float sB[2][CH * NP], sC[2][CH * NP];
    __shared__ float red[2][4][CH][2 * NP];
    const int cb = blockIdx.x % a.p.cblk, rest = blockIdx.x / a.p.cblk;
    const int gr = rest % a.G, slab = rest / a.G;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int cg = a.C / a.G, ci = cb * a.p.width + threadIdx.x;
    const bool on = ci < cg, wave_on = ci - lane < cg;
    const int c = gr * cg + (on ? ci : cg - 1);         // lanes beyond the group repeat its last channel, outside the sums
    float A2[NP], dA[NP], dD = 0.f, dbias = 0.f;
    load_states<NP>(a.A + (long long)c * a.N, a.N, A2);
#pragma unroll
    for (int n = 0; n < NP; ++n) { A2[n] *= LOG2E; dA[n] = 0.f; }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
    const long long tbg = (long long)a.L * a.B * a.G * a.N;

    auto put_bc = [&](int t, int b, int j, float v) {   // j < NP: dB, else dC
        const int n = j % NP;
        const long long at = (((long long)t * a.B + b) * a.G + gr) * a.N + n;
        if (a.p.cblk > 1) a.bc_part[(long long)cb * 2 * tbg + (j < NP ? 0 : tbg) + at] = v;
        else (j < NP ? a.dB : a.dC)[at] = from_f<M>(v);
    };
    int buf = 0, p_tc = 0, p_te = 0, p_b = 0;           // the chunk whose sums wait in red[buf ^ 1]: steps p_tc .. p_te - 1
    auto flush = [&]() {
        for (int i = threadIdx.x; i < CH * 2 * NP; i += a.p.width) {
            const int s = i / (2 * NP), j = i % (2 * NP);
            if (p_tc + s >= p_te || j % NP >= a.N) continue;
            float v = 0.f;
            for (int w = 0; w < a.p.waves; ++w) v += red[buf ^ 1][w][s][j];
            put_bc(p_tc + s, p_b, j, v);
        }
    };

    const int units = a.B * a.p.nseg;
    for (int u = slab; u < units; u += a.P) {
        const int b = u % a.B, seg = u / a.B;
        const int len = length_of(a.lengths, b, a.L);
        const int t0 = seg * a.p.seglen, t1 = min(t0 + a.p.seglen, a.L), te = min(t1, len);
        const long long row = (long long)b * a.C + c;
        const typename M::raw* Bp = a.Bm + b * a.B_b + gr * a.B_g;
        const typename M::raw* Cp = a.Cm + b * a.C_b + gr * a.C_g;
        float gc[NP];                                   // exp(step[t+1] A) g[t+1]
#pragma unroll
        for (int n = 0; n < NP; ++n) gc[n] = 0.f;
        {
            if (a.p.nseg > 1) load_kept<NP>(a.seg_h, seg, a.B, b, a.C, c, gc);
            else if (a.dstate_out) load_states<NP>(a.dstate_out + row * a.N, a.N, gc);
        }
        typename T::raw xr[CH], dr[CH], zr[CH];
        typename M::raw yr[CH];
        MapTile<M, NP> mB, mC;
        float hk[NP];
        auto request = [&](int tc) {
#pragma unroll
            for (int s = 0; s < CH; ++s) {
                const int t = min(tc + s, te - 1);
                xr[s] = load_elem<T, M, 0>(a, t, b, c);
                dr[s] = load_elem<T, M, 1>(a, t, b, c);
                if (GATED) zr[s] = load_elem<T, M, 2>(a, t, b, c);
                yr[s] = a.dy[t * a.dy_t + b * a.dy_b + c];
            }
            mB.request(Bp, a.B_t, tc, te, a.N);
            mC.request(Cp, a.C_t, tc, te, a.N);
            if (tc > 0) load_kept<NP>(a.ck, tc / CH - 1, a.B, b, a.C, c, hk);
            else if (a.state) load_states<NP>(a.state + row * a.N, a.N, hk);
            else {
#pragma unroll
                for (int n = 0; n < NP; ++n) hk[n] = 0.f;
            }
        };
        int k = te > t0 ? (te - t0 + CH - 1) / CH - 1 : -1;
        if (k >= 0) request(t0 + k * CH);
        for (; k >= 0; --k) {
            const int tc = t0 + k * CH;
            typename T::raw xc[CH], dc[CH], zc[CH];
            typename M::raw yc[CH];
            float h[CH + 1][NP], st[CH], sig[CH], out[CH];
#pragma unroll
            for (int s = 0; s < CH; ++s) { xc[s] = xr[s]; dc[s] = dr[s]; zc[s] = zr[s]; yc[s] = yr[s]; }
#pragma unroll
            for (int n = 0; n < NP; ++n) h[0][n] = hk[n];
            mB.put(sB[buf]);
            mC.put(sC[buf]);
            __syncthreads();
            flush();                                    // the sums of the chunk before, written before the barrier
            if (k > 0) request(tc - CH);
            const float *tB = sB[buf], *tC = sC[buf];
            if (wave_on) {
#pragma unroll
                for (int s = 0; s < CH; ++s) {
                    const bool live = tc + s < te;      // behind the row's end: a step of 0 with no adjoint of its own
                    const float xv = live ? to_f(xc[s]) : 0.f, v = softplus(to_f(dc[s]) + bias, sig[s]);
                    st[s] = live ? v : 0.f;
                    sig[s] = live ? sig[s] : 0.f;
                    pin(st[s]);
                    const float sx = st[s] * xv;
                    float o = Dc * xv;
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const float e = __builtin_amdgcn_exp2f(st[s] * A2[n]);
                        h[s + 1][n] = fmaf(e, h[s][n], sx * tB[s * NP + n]);
                        if (GATED) o = fmaf(h[s + 1][n], tC[s * NP + n], o);
                    }
                    out[s] = o;
                    step_fence();
                }
#pragma unroll
                for (int s = CH - 1; s >= 0; --s) {
                    const int t = tc + s;
                    const bool live = t < te;
                    pin(st[s]);                         // the exponentials again, not kept in 128 registers
                    const float xv = live ? to_f(xc[s]) : 0.f, dyv = live ? to_f(yc[s]) : 0.f, sx = st[s] * xv;
                    float d = dyv, dz = 0.f;
                    if (GATED) {
                        const float zv = live ? to_f(zc[s]) : 0.f, sz = sigmoid(zv);
                        d = dyv * zv * sz;
                        dz = dyv * out[s] * sz * fmaf(zv, 1.0f - sz, 1.0f);
                    }
                    dD = fmaf(d, xv, dD);
                    const float sxm = on ? sx : 0.f, dm = on ? d : 0.f;
                    float gB = 0.f, qA = 0.f, vB[NP], vC[NP];
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        const float e = __builtin_amdgcn_exp2f(st[s] * A2[n]);
                        const float gn = fmaf(d, tC[s * NP + n], gc[n]);
                        vB[n] = gn * sxm;
                        vC[n] = h[s + 1][n] * dm;
                        gB = fmaf(gn, tB[s * NP + n], gB);
                        gc[n] = gn * e;
                        const float q = gc[n] * h[s][n];
                        qA = fmaf(q, A2[n], qA);
                        dA[n] = fmaf(q, st[s], dA[n]);
                    }
                    const float dstep = fmaf(gB, xv, qA * LN2) * sig[s];
                    dbias += dstep;
                    if (t < t1) {
                        const long long at = ((long long)t * a.B + b) * a.C + c;
                        a.dx[at] = from_f<M>(fmaf(gB, st[s], Dc * d));
                        a.ddt[at] = from_f<M>(dstep);
                        if (GATED) a.dz[at] = from_f<M>(dz);
                    }
                    if constexpr (NP <= 16) {
                        float v[NV];
#pragma unroll
                        for (int n = 0; n < NP; ++n) { v[n] = vB[n]; v[NP + n] = vC[n]; }
                        red[buf][wave][s][index_of<NV>(lane)] = wave_sums<NV>(v, lane);
                    } else {
                        red[buf][wave][s][index_of<NV>(lane)] = wave_sums<NV>(vB, lane);
                        red[buf][wave][s][NP + index_of<NV>(lane)] = wave_sums<NV>(vC, lane);
                    }
                    step_fence();
                }
            }
            else {
#pragma unroll
                for (int s = 0; s < CH; ++s)
                    for (int j = lane; j < 2 * NP; j += 64) red[buf][wave][s][j] = 0.f;
            }
            p_tc = tc; p_te = te; p_b = b;
            buf ^= 1;
        }
        if (on) {
            if (a.dstate && seg == 0) store_states<NP>(a.dstate + row * a.N, a.N, gc);
            for (int t = t0 + (max(te - t0, 0) + CH - 1) / CH * CH; t < t1; ++t) {       // chunks behind the row's end
                const long long at = ((long long)t * a.B + b) * a.C + c;
                a.dx[at] = from_f<M>(0.f);
                a.ddt[at] = from_f<M>(0.f);
                if (GATED) a.dz[at] = from_f<M>(0.f);
            }
        }
        const int z0 = max(t0, len);
        for (int i = threadIdx.x; i < (t1 - z0) * 2 * NP; i += a.p.width)
            if (i % NP < a.N) put_bc(z0 + i / (2 * NP), b, i % (2 * NP), 0.f);
    }
    __syncthreads();
    flush();
    if (!on) return;
    float* part = a.part + (long long)slab * a.C * (a.N + 2);
#pragma unroll
    for (int n = 0; n < NP; ++n) if (n < a.N) part[(long long)c * a.N + n] = dA[n];
    part[(long long)a.C * a.N + c] = dD;
    part[(long long)a.C * (a.N + 1) + c] = dbias;
}

// dB and dC of several workgroups across a group's channels: sums in a fixed order
template <class M> __global__ __launch_bounds__(256)
void bc_reduce_kernel(const float* __restrict__ part, typename M::raw* __restrict__ dB, typename M::raw* __restrict__ dC, long long n, int cblk)
{
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += (long long)gridDim.x * 256) {
        float s = 0.f;
        for (int k = 0; k < cblk; ++k) s += part[k * 2 * n + i];
        if (i < n) dB[i] = from_f<M>(s); else dC[i - n] = from_f<M>(s);
    }
}

// Slabs of parameter-gradient sums: enough workgroups for two a CU, no more than rows x segments
int slabs(const ScanPlan& p, int B, int G)
{
    const long long units = (long long)B * p.nseg, want = (2048 / p.waves + p.cblk * G - 1) / (p.cblk * G);
    return (int)(units < want ? units : want);
}

struct BwdSpace { long long part, bc, seg_h, seg_s, total; };
BwdSpace bwd_space(const gmt_scan_args* a)
{
    const ScanPlan p = scan_plan(a->L, a->B, a->C, a->N, a->G);
    BwdSpace s;
    s.part = 0;
    s.bc = s.part + (long long)slabs(p, a->B, a->G) * a->C * (a->N + 2);
    s.seg_h = s.bc + (p.cblk > 1 ? 2LL * p.cblk * a->L * a->B * a->G * a->N : 0);
    s.seg_s = s.seg_h + (p.nseg > 1 ? (long long)p.nseg * a->B * a->C * p.np : 0);
    s.total = s.seg_s + (p.nseg > 1 ? (long long)p.nseg * a->B * a->C : 0);
    return s;
}

template <class T, class M, int NP, bool GATED> int launch(const ScanArgs<T, M>& a, hipStream_t stream)
{
    if (a.p.nseg > 1) {
        const dim3 grid((unsigned)((long long)a.p.cblk * a.G * a.B * a.p.nseg));
        hipLaunchKernelGGL((scan_bwd_local_kernel<T, M, NP, GATED>), grid, dim3(a.p.width), 0, stream, a);
        GMT_LAUNCH_CHECK();
        if (int rc = scan_chain(a.seg_h, a.seg_s, a.A, a.dstate_out, a.p.nseg, NP, a.B, a.C, a.N, 1, stream)) return rc;
    }
    hipLaunchKernelGGL((scan_bwd_kernel<T, M, NP, GATED>), dim3((unsigned)(a.p.cblk * a.G * a.P)), dim3(a.p.width), 0, stream, a);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}
template <class T, class M, int NP> int by_gate(const ScanArgs<T, M>& a, hipStream_t stream)
{
    return a.zq ? launch<T, M, NP, true>(a, stream) : launch<T, M, NP, false>(a, stream);
}

template <class T, class M> int run(const gmt_scan_args* args, hipStream_t stream)
{
    ScanArgs<T, M> a = scan_args<T, M>(args);
    const BwdSpace s = bwd_space(args);
    if (args->workspace_floats < s.total) return GMT_ERR_WORKSPACE;
    a.P = slabs(a.p, a.B, a.G);
    a.part = args->workspace + s.part;
    a.bc_part = args->workspace + s.bc;
    a.seg_h = args->workspace + s.seg_h;
    a.seg_s = args->workspace + s.seg_s;
    const int rc = a.p.np == 8 ? by_gate<T, M, 8>(a, stream) : a.p.np == 16 ? by_gate<T, M, 16>(a, stream) : by_gate<T, M, 32>(a, stream);
    if (rc) return rc;
    if (a.p.cblk > 1) {
        const long long n = (long long)a.L * a.B * a.G * a.N;
        hipLaunchKernelGGL(bc_reduce_kernel<M>, dim3(gmt_grid_1d(2 * n, 256, 256 * 16)), dim3(256), 0, stream, a.bc_part, a.dB, a.dC, n, a.p.cblk);
        GMT_LAUNCH_CHECK();
    }
    const long long n = (long long)a.C * (a.N + 2);
    return launch_slab_reduce(a.part, args->dparam, n, n, a.P, stream);
}

}  // namespace

long long gmt_ssm::scan_bwd_floats(const gmt_scan_args* a) { return bwd_space(a).total; }

extern "C" int gmt_selective_scan_bwd(const gmt_scan_args* a, hipStream_t stream)
{
    if (int rc = scan_check(a)) return rc;
    GMT_CHECK_ARG(a->dy && a->dx && a->ddt && a->dB && a->dC && a->dparam && a->workspace && (!a->z || a->dz));
    GMT_CHECK_ARG(a->ck || a->L <= CH);
    GMT_CHECK_ARG((long long)a->B * scan_plan(a->L, a->B, a->C, a->N, a->G).nseg < (1LL << 31));
    if (a->x_scale) {
        if (a->L > CH) { if (int rc = scan_states_q8(a, stream)) return rc; }
        return a->bf16 ? run<Q8, B16>(a, stream) : run<Q8, F32>(a, stream);
    }
    return a->bf16 ? run<B16, B16>(a, stream) : run<F32, F32>(a, stream);
}
