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
// partner and keeps the partner's other half, by DPP and v_permlane16_swap - 32 instructions for 16 values over 32 lanes where 16
// separate sums take 80.  The waves of a workgroup meet in LDS, workgroups of one group through slabs: no float atomics, results
// do not depend on the order of execution.
#include "ssm_scan.h"

namespace {

using namespace gmt_ssm;

template <int CTRL> __device__ __forceinline__ float half_dpp(float a, float b, bool upper) {
    const float keep = upper ? b : a, send = upper ? a : b;
    return keep + dpp<CTRL>(send);
}
// The same for bits 3 and 2 of the lane, which are banks of four lanes that a DPP instruction can leave out: a + its partner on all
// lanes, then b + its partner on the upper ones - two instructions a value instead of three.  The waits at the front (and at the end of
// half_rows4, whose results go to permlane swaps) are those that a DPP or permlane operand needs behind the instruction that wrote
// it; the compiler does not see into these blocks.
__device__ __forceinline__ void half_rows8(float& a0, float& a1, float& a2, float& a3, float b0, float b1, float b2, float b3) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %1, %1, %1 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %2, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %3, %3, %3 row_ror:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %3, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xc"
        : "+&v"(a0), "+&v"(a1), "+&v"(a2), "+&v"(a3) : "v"(b0), "v"(b1), "v"(b2), "v"(b3));
}
__device__ __forceinline__ void half_rows4(float& a0, float& a1, float b0, float b1) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %0, %0 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %1, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf\n\t"
        "v_add_f32_dpp %0, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %1, %3, %3 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "s_nop 1"
        : "+&v"(a0), "+&v"(a1) : "v"(b0), "v"(b1));
}
// v[0 .. NV) summed over the lanes of one part: lane l returns value index_of(l).  (row_half_mirror also turns bits 0 and 1 round: all
// lanes that it mixes are summed later on.)
template <int NV, int PARTS> __device__ __forceinline__ float part_sums(float (&v)[NV], int lane)
{
    static_assert((PARTS == 2 || PARTS == 4) && (NV == 8 || NV == 16), "values per lane");
    constexpr int N4 = NV / 4, N2 = PARTS == 2 ? N4 / 2 : N4;          // values left behind bits 3 and 2, and behind bit 4
#pragma unroll
    for (int i = 0; i < NV / 2; i += 4)
        half_rows8(v[i], v[i + 1], v[i + 2], v[i + 3], v[i + NV / 2], v[i + NV / 2 + 1], v[i + NV / 2 + 2], v[i + NV / 2 + 3]);
#pragma unroll
    for (int i = 0; i < N4; i += 2) half_rows4(v[i], v[i + 1], v[i + N4], v[i + N4 + 1]);
    if constexpr (PARTS == 2) {
#pragma unroll
        for (int i = 0; i < N2; ++i) v[i] = half16(v[i], v[i + N2]);
    }
    if constexpr (N2 == 1) v[0] += dpp<DPP_XOR2>(v[0]);
    else {
#pragma unroll
        for (int i = 0; i < N2 / 2; ++i) v[i] = half_dpp<DPP_XOR2>(v[i], v[i + N2 / 2], lane & 2);
    }
    if constexpr (N2 == 4) return half_dpp<DPP_XOR1>(v[0], v[1], lane & 1);
    else return v[0] + dpp<DPP_XOR1>(v[0]);
}
template <int NV, int PARTS> __device__ __forceinline__ int index_of(int lane) {     // bits 3, 2, (4,) 1, 0, the first log2(NV) of them
    constexpr int LOG = NV == 8 ? 3 : 4;
    const int hi = lane >> 2 & 3;
    const int all = PARTS == 2 ? hi << 3 | (lane >> 4 & 1) << 2 | (lane & 3) : hi << 2 | (lane & 3);
    return all >> ((PARTS == 2 ? 5 : 4) - LOG);
}

// a segment's adjoint: (adjoint of its incoming state for a zero adjoint behind it, S)
template <class T, class M, int NP, bool GATED>
__global__ __launch_bounds__(64 * BWD_WAVES)
void scan_bwd_local_kernel(ScanArgs<T, M> a)
{
    constexpr int PARTS = NP == 32 ? 4 : 2, NS = NP / PARTS, OWN = CH / PARTS;
    __shared__ __align__(16) float sC[2][CH * NP];
    const int cb = blockIdx.x % a.p.cblk, rest = blockIdx.x / a.p.cblk;
    const int gr = rest % a.G, rest2 = rest / a.G;
    const int b = rest2 % a.B, seg = rest2 / a.B;
    const Lanes<PARTS> ln;
    const int cg = a.C / a.G, ci = cb * a.p.chans + ln.chan, n0 = ln.part * NS;
    const bool on = ci < cg;
    const unsigned c = gr * cg + (on ? ci : cg - 1);
    const int len = length_of(a.lengths, b, a.L);
    const int t0 = seg * a.p.seglen, t1 = min(t0 + a.p.seglen, a.L), te = min(t1, len);
    float A2[NS], g[NS];
    load_states<NS>(a.A + (long long)c * a.N, n0, a.N, A2);
#pragma unroll
    for (int n = 0; n < NS; ++n) { A2[n] = base2(A2[n]); g[n] = 0.f; }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f;
    const typename M::raw* Cp = a.Cm + b * a.C_b + gr * a.C_g;
    const Seq<T> dq(a.dt, a.dts, a.dt_t, a.dt_b, b, ln.part, c, a.B, a.C), zq(a.z, a.zs, a.z_t, a.z_b, b, ln.part, c, a.B, a.C);
    const Seq<M> yq(a.dy, nullptr, a.dy_t, a.dy_b, b, ln.part, c, a.B, a.C);
    float S = 0.f;
    Own<T, PARTS> dr, zr;
    Own<M, PARTS> yr;
    MapTile<M, NP> mC;
    auto request = [&](int tc) {
        dr.request(dq, tc, te, ln.part);
        if (GATED) zr.request(zq, tc, te, ln.part);
        yr.request(yq, tc, te, ln.part);
        mC.request(Cp, a.C_t, tc, te, a.N);
    };
    int buf = 0, k = te > t0 ? (te - t0 + CH - 1) / CH - 1 : -1;
    if (k >= 0) request(t0 + k * CH);
    for (; k >= 0; --k, buf ^= 1) {
        const int tc = t0 + k * CH;
        float st[OWN], d[OWN];
#pragma unroll
        for (int j = 0; j < OWN; ++j) {
            const bool live = tc + j * PARTS + ln.part < te;
            float sig;
            st[j] = softplus(to_f(dr.v[j]) + bias, sig);
            st[j] = live ? st[j] : 0.f;
            d[j] = live ? to_f(yr.v[j]) : 0.f;
            if (GATED) { const float zv = live ? to_f(zr.v[j]) : 0.f; d[j] *= zv * sigmoid(zv); }
            S += st[j];
        }
        mC.put(sC[buf]);
        lds_barrier();
        if (k > 0) request(tc - CH);
        float sts[PARTS], ds[PARTS];
#pragma unroll
        for (int s = CH - 1; s >= 0; --s) {
            const int j = s / PARTS, q = s % PARTS;
            if (q == PARTS - 1) { ln.spread(st[j], sts); ln.spread(d[j], ds); }
            pin(sts[q]);
#pragma unroll
            for (int n = 0; n < NS; ++n) g[n] = __builtin_amdgcn_exp2f(sts[q] * A2[n]) * fmaf(ds[q], sC[buf][s * NP + n0 + n], g[n]);
            step_fence();
        }
    }
    S = ln.sum(S);
    if (!on) return;
    store_kept<NP, NS>(a.seg_h, seg, a.B, b, a.C, (unsigned)(n0 * a.C + c) * 4, g);
    if (ln.part == 0) a.seg_s[(long long)(seg * a.B + b) * a.C + c] = S;
}

template <class T, class M, int NP, bool GATED>
__global__ __launch_bounds__(64 * BWD_WAVES, 2)
void scan_bwd_kernel(ScanArgs<T, M> a)
{
    constexpr int PARTS = NP == 32 ? 4 : 2, NS = NP / PARTS, OWN = CH / PARTS;
    // The exponentials of the last KE steps of a chunk stay in registers, those of the others are computed twice: as many as fit
    // beside the states (N = 16, L=256 B=256 C=512 bf16: 8 kept 478 us, 4 kept 504 us; from 8-bit codes, whose exponents take
    // registers too, L=129 B=256 C=512: 8 kept 425 us, 6 375, 5 372, 4 388).
    constexpr int KE = NS == 8 && __is_same(T, Q8) ? 5 : CH;
    __shared__ __align__(16) float sB[2][CH * NP], sC[2][CH * NP];
    __shared__ float red[2][BWD_WAVES][CH][2 * NP];             // [wave][step][part][dB, dC of the part's states]
    const int cb = blockIdx.x % a.p.cblk, rest = blockIdx.x / a.p.cblk;
    const int gr = rest % a.G, slab = rest / a.G;
    __shared__ unsigned short rows[ORDERED];            // the slab's rows, if they are taken by length
    if (a.sorted) {                                     // every other round from the other end: a slab's sum of lengths evens out
        for (int lo = 0; lo + slab < a.B; lo += a.P) {
            const int r = lo / a.P & 1 ? min(lo + a.P, a.B) - 1 - slab : lo + slab;
            rows[lo / a.P] = (unsigned short)row_of_rank(a.lengths, r, a.B, a.L);     // every wave the same
        }
        lds_barrier();
    }
    step_fence();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Lanes<PARTS> ln;
    const int cg = a.C / a.G, ci = cb * a.p.chans + ln.chan, n0 = ln.part * NS;
    const bool on = ci < cg, wave_on = cb * a.p.chans + wave * (64 / PARTS) < cg;
    const unsigned c = gr * cg + (on ? ci : cg - 1);    // lanes beyond the group repeat its last channel with x = dy = 0
    float A2[NS], dA[NS], dD = 0.f, dbias = 0.f;
    load_states<NS>(a.A + (long long)c * a.N, n0, a.N, A2);
#pragma unroll
    for (int n = 0; n < NS; ++n) { A2[n] = base2(A2[n]); dA[n] = 0.f; }
    const float bias = a.dt_bias ? a.dt_bias[c] : 0.f, Dc = a.D ? a.D[c] : 0.f;
    const long long tbg = (long long)a.L * a.B * a.G * a.N;
    const unsigned koff = (unsigned)(n0 * a.C + c) * 4;
    const int o_t = a.B * a.C;                          // pitch of a step of the outputs

    auto put_bc = [&](int t, int b, bool is_c, int n, float v) {
        const long long at = (((long long)t * a.B + b) * a.G + gr) * a.N + n;
        if (a.p.cblk > 1) a.bc_part[(long long)cb * 2 * tbg + (is_c ? tbg : 0) + at] = v;
        else (is_c ? a.dC : a.dB)[at] = from_f<M>(v);
    };
    int buf = 0, p_tc = 0, p_te = 0, p_b = 0;           // the chunk whose sums wait in red[buf ^ 1]: steps p_tc .. p_te - 1
    const int bc_t = a.B * a.G * a.N;                   // pitch of a step of dB and dC
    auto flush = [&]() {
        static_assert(CH * NP % 64 == 0, "a wave's 64 sums are all dB or all dC");
        const long long row = (((long long)p_tc * a.B + p_b) * a.G + gr) * a.N;
        for (int i0 = wave * 64; i0 < 2 * CH * NP; i0 += a.p.width) {
            const bool is_c = i0 >= CH * NP;
            const int i = i0 % (CH * NP) + lane, s = i / NP, n = i % NP;
            if (p_tc + s >= p_te || n >= a.N) continue;
            float v = 0.f;
            for (int w = 0; w < a.p.waves; ++w) v += red[buf ^ 1][w][s][n / NS * 2 * NS + (is_c ? NS : 0) + n % NS];
            const unsigned at = (unsigned)(s * bc_t + n);
            if (a.p.cblk > 1) store_at<float>(uniform(a.bc_part + (long long)cb * 2 * tbg + (is_c ? tbg : 0) + row), at * 4, v);
            else store_at<typename M::raw>(uniform((is_c ? a.dC : a.dB) + row), at * (unsigned)sizeof(typename M::raw), from_f<M>(v));
        }
    };

    const int units = a.B * a.p.nseg;
    for (int u = slab; u < units; u += a.P) {
        const int seg = u / a.B;
        int b = u % a.B;
        if (a.sorted) b = __builtin_amdgcn_readfirstlane(rows[u / a.P]);
        const int len = length_of(a.lengths, b, a.L);
        const int t0 = seg * a.p.seglen, t1 = min(t0 + a.p.seglen, a.L), te = min(t1, len);
        const long long row = (long long)b * a.C + c;
        const typename M::raw* Bp = a.Bm + b * a.B_b + gr * a.B_g;
        const typename M::raw* Cp = a.Cm + b * a.C_b + gr * a.C_g;
        const Seq<T> xq(a.x, a.xs, a.x_t, a.x_b, b, ln.part, c, a.B, a.C), dq(a.dt, a.dts, a.dt_t, a.dt_b, b, ln.part, c, a.B, a.C),
            zq(a.z, a.zs, a.z_t, a.z_b, b, ln.part, c, a.B, a.C);
        const Seq<M> yq(a.dy, nullptr, a.dy_t, a.dy_b, b, ln.part, c, a.B, a.C);
        const unsigned ooff = (unsigned)((ln.part * o_t + b * a.C + c) * sizeof(typename M::raw));
        float gc[NS];                                   // exp(step[t+1] A) g[t+1]
#pragma unroll
        for (int n = 0; n < NS; ++n) gc[n] = 0.f;
        if (on) {
            if (a.p.nseg > 1) load_kept<NP, NS>(a.seg_h, seg, a.B, b, a.C, koff, gc);
            else if (a.dstate_out) load_states<NS>(a.dstate_out + row * a.N, n0, a.N, gc);
        }
        Own<T, PARTS> xr, dr, zr;
        Own<M, PARTS> yr;
        MapTile<M, NP> mB, mC;
        float hk[NS];
        auto request = [&](int tc) {
            xr.request(xq, tc, te, ln.part);
            dr.request(dq, tc, te, ln.part);
            if (GATED) zr.request(zq, tc, te, ln.part);
            yr.request(yq, tc, te, ln.part);
            mB.request(Bp, a.B_t, tc, te, a.N);
            mC.request(Cp, a.C_t, tc, te, a.N);
            load_kept<NP, NS>(a.ck, tc / CH, a.B, b, a.C, koff, hk);
        };
        int k = te > t0 ? (te - t0 + CH - 1) / CH - 1 : -1;
        if (k >= 0) request(t0 + k * CH);
        for (; k >= 0; --k) {
            const int tc = t0 + k * CH;
            float h[CH + 1][NS], ex[KE][NS];
            float xv[OWN], st[OWN], sig[OWN], d[OWN], dzf[OWN], out[OWN], gBk[OWN], qAk[OWN];        // dzf: dy silu'(z)
#pragma unroll
            for (int j = 0; j < OWN; ++j) {
                const bool live = tc + j * PARTS + ln.part < te;        // behind the row's end: a step of 0 with no adjoint of its own
                xv[j] = live && on ? to_f(xr.v[j]) : 0.f;
                const float v = softplus(to_f(dr.v[j]) + bias, sig[j]);
                st[j] = live ? v : 0.f;
                sig[j] = live ? sig[j] : 0.f;
                d[j] = live && on ? to_f(yr.v[j]) : 0.f;
                if (GATED) {
                    const float zv = live ? to_f(zr.v[j]) : 0.f, sz = sigmoid(zv);
                    dzf[j] = d[j] * sz * fmaf(zv, 1.0f - sz, 1.0f);
                    d[j] *= zv * sz;
                }
                out[j] = gBk[j] = qAk[j] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < NS; ++n) h[0][n] = hk[n];
            mB.put(sB[buf]);
            mC.put(sC[buf]);
            lds_barrier();
            flush();                                    // the sums of the chunk before, written before the barrier
            if (wave_on) {
                float sts[PARTS], xs[PARTS], ds[PARTS], va[PARTS], vb[PARTS];
#pragma unroll
                for (int s = 0; s < CH; ++s) {
                    const int j = s / PARTS, q = s % PARTS;
                    if (q == 0) { ln.spread(st[j], sts); ln.spread(xv[j], xs); }
                    pin(sts[q]);
                    const float sx = sts[q] * xs[q];
                    const float *Bt = sB[buf] + s * NP + n0, *Ct = sC[buf] + s * NP + n0;
                    va[q] = 0.f;
#pragma unroll
                    for (int n = 0; n < NS; ++n) {
                        const float e = __builtin_amdgcn_exp2f(sts[q] * A2[n]);
                        if (s >= CH - KE) ex[s >= CH - KE ? s - (CH - KE) : 0][n] = e;
                        h[s + 1][n] = fmaf(e, h[s][n], sx * Bt[n]);
                        if (GATED) va[q] = fmaf(h[s + 1][n], Ct[n], va[q]);
                    }
                    if (GATED) {
                        pin(va[q]);
                        if (q == PARTS - 1) out[j] = ln.gather(va);
                    }
                    step_fence();
                }
                if (GATED) {
#pragma unroll
                    for (int j = 0; j < OWN; ++j)
                        if (tc + j * PARTS + ln.part < t1 && on)
                            put_out<M>(a.dz, (long long)(tc + j * PARTS) * o_t, ooff, dzf[j] * fmaf(Dc, xv[j], out[j]));
                    step_fence();
                }
#pragma unroll
                for (int s = CH - 1; s >= 0; --s) {
                    // the next chunk's elements: by now half of h and ex is free again
                    if (s == CH / 2 - 1 && k > 0) request(tc - CH);
                    const int j = s / PARTS, q = s % PARTS;
                    if (q == PARTS - 1) { ln.spread(st[j], sts); ln.spread(xv[j], xs); ln.spread(d[j], ds); }
                    pin(sts[q]);
                    const float sx = sts[q] * xs[q];
                    const float *Bt = sB[buf] + s * NP + n0, *Ct = sC[buf] + s * NP + n0;
                    float v[2 * NS];
                    va[q] = vb[q] = 0.f;
#pragma unroll
                    for (int n = 0; n < NS; ++n) {
                        const float e = s >= CH - KE ? ex[s >= CH - KE ? s - (CH - KE) : 0][n] : __builtin_amdgcn_exp2f(sts[q] * A2[n]);
                        const float gn = fmaf(ds[q], Ct[n], gc[n]);
                        v[n] = gn * sx;
                        v[NS + n] = h[s + 1][n] * ds[q];
                        va[q] = fmaf(gn, Bt[n], va[q]);
                        gc[n] = gn * e;
                        const float p = gc[n] * h[s][n];
                        vb[q] = fmaf(p, A2[n], vb[q]);
                        dA[n] = fmaf(p, sts[q], dA[n]);
                    }
                    pin(va[q]); pin(vb[q]);
#pragma unroll
                    for (int n = 0; n < NS; ++n) pin(dA[n]);
                    if (q == 0) { gBk[j] = ln.gather(va); qAk[j] = ln.gather(vb); }
                    red[buf][wave][s][ln.part * 2 * NS + index_of<2 * NS, PARTS>(lane)] = part_sums<2 * NS, PARTS>(v, lane);
                    step_fence();
                }
#pragma unroll
                for (int j = 0; j < OWN; ++j) {
                    const int t = tc + j * PARTS + ln.part;
                    // (a masked step's sum over A may overflow: 0, not 0 * inf)
                    const float dstep = sig[j] == 0.f ? 0.f : fmaf(gBk[j], xv[j], qAk[j] * LN2) * sig[j];
                    dbias += dstep;
                    dD = fmaf(d[j], xv[j], dD);
                    if (t < t1 && on) {
                        const long long base = (long long)(tc + j * PARTS) * o_t;
                        put_out<M>(a.dx, base, ooff, fmaf(gBk[j], st[j], Dc * d[j]));
                        put_out<M>(a.ddt, base, ooff, dstep);
                    }
                }
            } else {
                if (k > 0) request(tc - CH);            // (its share of B and C)
#pragma unroll
                for (int s = 0; s < CH; ++s)
                    for (int j = lane; j < 2 * NP; j += 64) red[buf][wave][s][j] = 0.f;
            }
            p_tc = tc; p_te = te; p_b = b;
            buf ^= 1;
        }
        if (on) {
            if (a.dstate && seg == 0) store_states<NS>(a.dstate + row * a.N, n0, a.N, gc);
            for (int t = t0 + (max(te - t0, 0) + CH - 1) / CH * CH + ln.part; t < t1; t += PARTS) {     // chunks behind the row's end
                const long long at = ((long long)t * a.B + b) * a.C + c;
                a.dx[at] = from_f<M>(0.f);
                a.ddt[at] = from_f<M>(0.f);
                if (GATED) a.dz[at] = from_f<M>(0.f);
            }
        }
        const int z0 = max(t0, len);
        for (int i = threadIdx.x; i < (t1 - z0) * 2 * NP; i += a.p.width)
            if (i % NP < a.N) put_bc(z0 + i / (2 * NP), b, i % (2 * NP) >= NP, i % NP, 0.f);
    }
    lds_barrier();
    flush();
    dD = ln.sum(dD);
    dbias = ln.sum(dbias);
    if (!on) return;
    float* part = a.part + (long long)slab * a.C * (a.N + 2);
#pragma unroll
    for (int n = 0; n < NS; ++n) if (n0 + n < a.N) part[(long long)c * a.N + n0 + n] = dA[n];
    if (ln.part == 0) {
        part[(long long)a.C * a.N + c] = dD;
        part[(long long)a.C * (a.N + 1) + c] = dbias;
    }
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

// Slabs of parameter-gradient sums, a workgroup each: rows x segments, at most 512 workgroups of 8 waves (two rounds of the machine:
// rows in descending order of length even out, L=129 B=512 C=256 fp32 with lengths of 64 .. 129 256 us against 263 us with one).
int slabs(const ScanPlan& p, int B, int G)
{
    const long long units = (long long)B * p.nseg, want = (4096 / p.waves + p.cblk * G - 1) / (p.cblk * G);
    return (int)(units < want ? units : want);
}

struct BwdSpace { long long part, bc, seg_h, seg_s, total; };
BwdSpace bwd_space(const gmt_scan_args* a)
{
    const ScanPlan p = bwd_plan(a->L, a->B, a->C, a->N, a->G);
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
    return a.z ? launch<T, M, NP, true>(a, stream) : launch<T, M, NP, false>(a, stream);
}

template <class T, class M> int run(const gmt_scan_args* args, hipStream_t stream)
{
    ScanArgs<T, M> a = scan_args<T, M>(args, bwd_plan(args->L, args->B, args->C, args->N, args->G));
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
    GMT_CHECK_ARG(a->ck);
    if (a->x_scale) {
        if (int rc = scan_states_q8(a, stream)) return rc;
        return a->bf16 ? run<Q8, B16>(a, stream) : run<Q8, F32>(a, stream);
    }
    return a->bf16 ? run<B16, B16>(a, stream) : run<F32, F32>(a, stream);
}
