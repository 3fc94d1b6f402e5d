// Short causal convolution over time, one filter per channel, with the SiLU behind it - the operator in front of the
// selective scan (ssm_scan_fwd.hip).  Time-major: x [L][B][C], K taps, past = [state (K - 1 steps); x]:
//     pre[t] = bias + sum_k w[k] past[t + k],     y[t] = silu(pre[t])  (or pre itself)
// and with g = dy silu'(pre):  dx[s] = sum_k w[k] g[s + K-1-k],  dw[k] = sum_{b,t} g[t] past[t + k],  dbias = sum g.
//
// Bound by HBM (2 K + 6 operations per 4 - 8 bytes).  A thread owns V neighbouring channels (16 bytes) of one row and walks
// along time with the last K - 1 inputs in registers: every element is read once.  A workgroup is 2^k channel vectors x rows,
// so that narrow rows share a wave.  When rows x channels do not fill the machine, time is cut into segments of 16 steps or
// a little fewer (conv_map); a segment reads the K - 1 inputs before it again (and the backward pass K - 1 steps behind it).
#include "ssm_common.h"

namespace {

using namespace gmt_ssm;

constexpr int THREADS = 256;

// V elements of type T at p (aligned to V elements) as floats
template <class T, int V> struct Vec;
template <int V> struct Vec<F32, V> {
    typedef float type __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ void load(const float* p, float (&o)[V]) {
        const type v = *reinterpret_cast<const type*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = v[i];
    }
    static __device__ __forceinline__ void store(float* p, const float (&o)[V]) {
        type v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = o[i];
        *reinterpret_cast<type*>(p) = v;
    }
};
template <> struct Vec<F32, 1> {
    static __device__ __forceinline__ void load(const float* p, float (&o)[1]) { o[0] = *p; }
    static __device__ __forceinline__ void store(float* p, const float (&o)[1]) { *p = o[0]; }
};
template <int V> struct Vec<B16, V> {
    typedef unsigned short type __attribute__((ext_vector_type(V)));
    static __device__ __forceinline__ void load(const unsigned short* p, float (&o)[V]) {
        const type v = *reinterpret_cast<const type*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = to_f((unsigned short)v[i]);
    }
    static __device__ __forceinline__ void store(unsigned short* p, const float (&o)[V]) {
        type v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = f_to_bf16(o[i]);
        *reinterpret_cast<type*>(p) = v;
    }
};
template <> struct Vec<B16, 1> {
    static __device__ __forceinline__ void load(const unsigned short* p, float (&o)[1]) { o[0] = to_f(*p); }
    static __device__ __forceinline__ void store(unsigned short* p, const float (&o)[1]) { *p = f_to_bf16(o[0]); }
};
// 8-bit codes: V <= 8 channels never straddle a block of 32 (V divides 32 and c is a multiple of V)
template <int V> __device__ __forceinline__ void load_q8(const signed char* p, const unsigned char* s, float (&o)[V]) {
    typedef signed char type __attribute__((ext_vector_type(V)));
    const float scale = __uint_as_float((unsigned)*s << 23);
    if constexpr (V == 1) {
        o[0] = (float)*p * scale;
    } else {
        const type v = *reinterpret_cast<const type*>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = (float)v[i] * scale;
    }
}

struct Map { int cv, cvb, rpb, gx, P; long long units; int nseg, seglen; };   // see conv_map

// channel vector and first unit of this thread; units are (row, segment) pairs
struct Place { int c, row0, lane_row; };
__device__ __forceinline__ Place place(const Map& m, int V) {
    Place p;
    p.c = (blockIdx.x % m.gx * m.cvb + threadIdx.x % m.cvb) * V;
    p.row0 = blockIdx.x / m.gx;
    p.lane_row = threadIdx.x / m.cvb;
    return p;
}

template <class T, int V, int K>
__global__ __launch_bounds__(THREADS)
void conv_fwd_kernel(const typename T::raw* __restrict__ x, long long x_t, long long x_b, const float* __restrict__ w,
                     const float* __restrict__ bias, const typename T::raw* __restrict__ state, const int* __restrict__ lengths,
                     typename T::raw* __restrict__ y, typename T::raw* __restrict__ state_out, int L, int B, int C, int silu, Map m)
{
    const Place pl = place(m, V);
    const long long u = (long long)pl.row0 * m.rpb + pl.lane_row;
    if (pl.c >= C || u >= m.units) return;
    const int b = (int)(u % B), seg = (int)(u / B), c = pl.c;
    const int len = length_of(lengths, b, L);
    const int t0 = seg * m.seglen, t1 = min(t0 + m.seglen, L), te = min(t1, len);
    float wk[K][V], bi[V], win[K][V];                  // win[K-1]: the current input
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bi[v] = bias ? bias[c + v] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) wk[k][v] = w[(long long)(c + v) * K + k];
    }
    const typename T::raw* xp = x + b * x_b + c;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
        const int s = t0 + k - (K - 1);
#pragma unroll
        for (int v = 0; v < V; ++v) win[k][v] = 0.f;
        if (s >= 0) { if (s < len) Vec<T, V>::load(xp + s * x_t, win[k]); }
        else if (state) Vec<T, V>::load(state + ((long long)(s + K - 1) * B + b) * C + c, win[k]);
    }
    typename T::raw* yp = y + (long long)b * C + c;
    const long long y_t = (long long)B * C;
    auto step = [&](int t) {
        float o[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float p = bi[v];
#pragma unroll
            for (int k = 0; k < K; ++k) p = fmaf(wk[k][v], win[k][v], p);
            o[v] = silu ? p * sigmoid(p) : p;
        }
        Vec<T, V>::store(yp + t * y_t, o);
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) win[k][v] = win[k + 1][v];
    };
    int t = t0;
    for (; t + 8 <= te; t += 8) {                       // eight loads in flight
        float nx[8][V];
#pragma unroll
        for (int j = 0; j < 8; ++j) Vec<T, V>::load(xp + (t + j) * x_t, nx[j]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int v = 0; v < V; ++v) win[K - 1][v] = nx[j][v];
            step(t + j);
        }
    }
    for (; t < te; ++t) {
        Vec<T, V>::load(xp + t * x_t, win[K - 1]);
        step(t);
    }
    // the segment in which the row ends holds its last K - 1 inputs
    if (state_out && ((len > t0 && len <= t1) || (len == 0 && seg == 0))) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) Vec<T, V>::store(state_out + ((long long)k * B + b) * C + c, win[k]);
    }
    const float zero[V] = {};
    for (t = max(t0, len); t < t1; ++t) Vec<T, V>::store(yp + t * y_t, zero);
}

// Q: x is read from its 8-bit checkpoint
template <class T, int V, int K, bool Q>
__global__ __launch_bounds__(THREADS)
void conv_bwd_kernel(const void* __restrict__ x_, const unsigned char* __restrict__ x_scale, long long x_t, long long x_b,
                     const float* __restrict__ w, const float* __restrict__ bias, const typename T::raw* __restrict__ state,
                     const int* __restrict__ lengths, const typename T::raw* __restrict__ dy, long long dy_t, long long dy_b,
                     const typename T::raw* __restrict__ dlast, typename T::raw* __restrict__ dx, float* __restrict__ part,
                     typename T::raw* __restrict__ dstate, int L, int B, int C, int silu, Map m)
{
    __shared__ float red[THREADS][V];
    const Place pl = place(m, V);
    const int c = pl.c;
    const bool on = c < C;
    float wk[K][V], bi[V], dw[K][V] = {}, db[V] = {};
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bi[v] = on && bias ? bias[c + v] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) wk[k][v] = on ? w[(long long)(c + v) * K + k] : 0.f;
    }
    const int n_sc = (C + 31) / 32;
    const long long dx_t = (long long)B * C;
    if (on)
    for (long long u = (long long)pl.row0 * m.rpb + pl.lane_row; u < m.units; u += (long long)m.P * m.rpb) {
        const int b = (int)(u % B), seg = (int)(u / B);
        const int len = length_of(lengths, b, L);
        const int t0 = seg * m.seglen, t1 = min(t0 + m.seglen, L), te = min(t1, len);
        auto load_x = [&](int s, float (&o)[V]) {
            if constexpr (Q) {
                const long long row = (long long)s * B + b;
                load_q8<V>((const signed char*)x_ + row * C + c, x_scale + row * n_sc + c / 32, o);
            } else {
                Vec<T, V>::load((const typename T::raw*)x_ + s * x_t + b * x_b + c, o);
            }
        };
        float win[K][V], g[K][V] = {};                  // g[k] = the adjoint of pre at t - k
#pragma unroll
        for (int k = 0; k < K - 1; ++k) {
            const int s = t0 + k - (K - 1);
#pragma unroll
            for (int v = 0; v < V; ++v) win[k][v] = 0.f;
            if (s >= 0) { if (s < len) load_x(s, win[k]); }
            else if (state) Vec<T, V>::load(state + ((long long)(s + K - 1) * B + b) * C + c, win[k]);
        }
        const typename T::raw* dyp = dy + b * dy_b + c;
        // step t gives g[t] and finishes dx[t - (K-1)]; `own`: t belongs to this segment
        auto step = [&](int t, const float (&dyv)[V], bool live, bool own) {
#pragma unroll
            for (int k = K - 1; k > 0; --k)
#pragma unroll
                for (int v = 0; v < V; ++v) g[k][v] = g[k - 1][v];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float p = bi[v];
#pragma unroll
                for (int k = 0; k < K; ++k) p = fmaf(wk[k][v], win[k][v], p);
                const float s = silu ? sigmoid(p) : 0.f;
                g[0][v] = live ? (silu ? dyv[v] * s * fmaf(p, 1.0f - s, 1.0f) : dyv[v]) : 0.f;
                if (own) {
                    db[v] += g[0][v];
#pragma unroll
                    for (int k = 0; k < K; ++k) dw[k][v] = fmaf(g[0][v], win[k][v], dw[k][v]);
                }
            }
            const int s = t - (K - 1);
            if (s >= t0 || (seg == 0 && s < 0)) {
                float o[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    o[v] = 0.f;
#pragma unroll
                    for (int k = 0; k < K; ++k) o[v] = fmaf(wk[k][v], g[k][v], o[v]);
                }
                const int j = t - len;                  // past[len + j] is entry j of the final state
                if (dlast && j >= 0 && j < K - 1) {
                    float d[V];
                    Vec<T, V>::load(dlast + ((long long)j * B + b) * C + c, d);
#pragma unroll
                    for (int v = 0; v < V; ++v) o[v] += d[v];
                }
                if (s >= 0) Vec<T, V>::store(dx + s * dx_t + (long long)b * C + c, o);
                else if (dstate) Vec<T, V>::store(dstate + ((long long)(s + K - 1) * B + b) * C + c, o);
            }
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) win[k][v] = win[k + 1][v];
        };
        int t = t0;
        for (; t + 4 <= te; t += 4) {
            float nx[4][V], nd[4][V];
#pragma unroll
            for (int j = 0; j < 4; ++j) { load_x(t + j, nx[j]); Vec<T, V>::load(dyp + (t + j) * dy_t, nd[j]); }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int v = 0; v < V; ++v) win[K - 1][v] = nx[j][v];
                step(t + j, nd[j], true, true);
            }
        }
        // the rest of the segment, and K - 1 steps behind it that dx of its last steps needs (zero beyond the row's end)
        const int tx = min(t1, max(len, t0)) + K - 1;
        for (; t < tx; ++t) {
            float d[V] = {};
            const bool live = t < len;
            if (live) { load_x(t, win[K - 1]); Vec<T, V>::load(dyp + t * dy_t, d); }
            else {
#pragma unroll
                for (int v = 0; v < V; ++v) win[K - 1][v] = 0.f;
            }
            step(t, d, live, t < te);
        }
        const float zero[V] = {};
        for (int s = max(t0, len); s < t1; ++s) Vec<T, V>::store(dx + s * dx_t + (long long)b * C + c, zero);
    }
    // sums over the workgroup's rows, then one slab of [K + 1][C] for every group of workgroups across the channels
    float* out = part + (long long)pl.row0 * (K + 1) * C;
#pragma unroll
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) red[threadIdx.x][v] = k < K ? dw[k < K ? k : 0][v] : db[v];
        __syncthreads();
        if (pl.lane_row == 0 && on) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float s = 0.f;
                for (int r = 0; r < m.rpb; ++r) s += red[r * m.cvb + threadIdx.x][v];
                out[(long long)k * C + c + v] = s;
            }
        }
    }
}

// one step: state [K-1][B][C] -> state_out (may be the same buffer: a thread reads its K - 1 entries before it writes)
template <class T, int K>
__global__ __launch_bounds__(THREADS)
void conv_step_kernel(const typename T::raw* __restrict__ x, long long x_b, const typename T::raw* state, typename T::raw* state_out,
                      const float* __restrict__ w, const float* __restrict__ bias, const unsigned char* __restrict__ active,
                      typename T::raw* __restrict__ y, int B, int C, int silu)
{
    const long long n = (long long)B * C;
    for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < n; i += (long long)gridDim.x * THREADS) {
        const int b = (int)(i / C), c = (int)(i % C);
        const bool act = !active || active[b];
        typename T::raw win[K];
#pragma unroll
        for (int k = 0; k < K - 1; ++k) win[k] = state[k * n + i];
        if (!act) {                                     // the row's state stays as it is
            if (state_out != state) {
#pragma unroll
                for (int k = 0; k < K - 1; ++k) state_out[k * n + i] = win[k];
            }
            y[i] = from_f<T>(0.f);
            continue;
        }
        win[K - 1] = x[b * x_b + c];
        float p = bias ? bias[c] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) p = fmaf(w[(long long)c * K + k], to_f(win[k]), p);
        y[i] = from_f<T>(silu ? p * sigmoid(p) : p);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) state_out[k * n + i] = win[k + 1];
    }
}

// widest vector (16 bytes, 2 elements, 1) that every pointer and pitch allows
int conv_vec(const gmt_conv_args* a, bool backward)
{
    const int esz = a->bf16 ? 2 : 4, full = 16 / esz;
    const bool q8 = a->x_scale != nullptr;
    for (int V : {full, 2}) {
        long long m = a->C | (q8 && backward ? 0 : (a->x_t | a->x_b));
        uintptr_t p = (uintptr_t)a->state | (uintptr_t)a->state_out;
        if (backward) {
            m |= a->dy_t | a->dy_b;
            p |= (uintptr_t)a->dy | (uintptr_t)a->dx | (uintptr_t)a->dstate | (uintptr_t)a->dstate_out;
            if (q8 && ((uintptr_t)a->x % V)) continue;
        } else p |= (uintptr_t)a->y;
        if (!(q8 && backward)) p |= (uintptr_t)a->x;
        if (m % V == 0 && p % (uintptr_t)(V * esz) == 0) return V;
    }
    return 1;
}

// Threads are 2^k channel vectors (at most 64) x rows.  Time is cut so that about 2^17 threads run (2 waves on each SIMD, all that
// the backward pass's registers admit), into ceil(L / 16) segments at most: of 16 steps for long sequences, where the K - 1 inputs read twice
// are under a fifth, of 9 at the least (L = 17: a third at K = 4).  L=128 B=1024 C=512 bf16, forward / backward, when the number was chosen:
// 2^16 threads 80 / 130 us, 2^17 59 / 111 us, 2^18 60 / 129 us.
Map conv_map(int L, int B, int C, int V)
{
    Map m;
    m.cv = (C + V - 1) / V;
    m.cvb = 1;
    while (m.cvb < m.cv && m.cvb < 64) m.cvb *= 2;
    m.rpb = THREADS / m.cvb;
    const long long threads = (long long)B * m.cv;
    long long nseg = ((1LL << 17) + threads - 1) / threads;
    const long long most = (L + 15) / 16;
    if (nseg > most) nseg = most;
    m.seglen = (int)((L + nseg - 1) / nseg);
    m.nseg = (L + m.seglen - 1) / m.seglen;
    m.units = (long long)B * m.nseg;
    const long long rows = (m.units + m.rpb - 1) / m.rpb;
    m.gx = (m.cv + m.cvb - 1) / m.cvb;
    long long P = (4096 + m.gx - 1) / m.gx;                 // backward: slabs of weight-gradient sums (16 workgroups a CU in all)
    if (P > rows) P = rows;
    m.P = (int)P;
    return m;
}

int check_any(const gmt_conv_args* a)
{
    GMT_CHECK_ARG(a && a->x && a->w && a->L > 0 && a->B > 0 && a->C > 0);
    return a->K < 2 || a->K > 4 ? GMT_ERR_UNSUPPORTED : GMT_OK;
}
// Whole sequences: a launch stays below 2^24 workgroups (vectors and rows are padded to at most twice as many threads; segments come with few
// threads only).  A single step walks over any number of elements.
int check(const gmt_conv_args* a)
{
    if (int rc = check_any(a)) return rc;
    if (a->L > MAX_STEPS || (long long)a->B * a->C >= (1LL << 31) || a->C > (1 << 30) - 64) return GMT_ERR_UNSUPPORTED;
    return GMT_OK;
}

template <class T, int V, int K> int run_fwd(const gmt_conv_args* a, hipStream_t stream)
{
    using R = typename T::raw;
    const Map m = conv_map(a->L, a->B, a->C, V);
    const long long blocks = (m.units + m.rpb - 1) / m.rpb * m.gx;
    auto k = conv_fwd_kernel<T, V, K>;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(THREADS), 0, stream, (const R*)a->x, a->x_t, a->x_b, a->w, a->bias,
                       (const R*)a->state, a->lengths, (R*)a->y, (R*)a->state_out, a->L, a->B, a->C, a->silu, m);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}

template <class T, int V, int K> int run_bwd(const gmt_conv_args* a, hipStream_t stream)
{
    using R = typename T::raw;
    const Map m = conv_map(a->L, a->B, a->C, V);
    const long long n = (long long)(K + 1) * a->C;
    if (a->workspace_floats < n * m.P) return GMT_ERR_WORKSPACE;
    const dim3 grid((unsigned)m.gx * m.P);
    if (a->x_scale) {
        auto k = conv_bwd_kernel<T, V, K, true>;
        hipLaunchKernelGGL(k, grid, dim3(THREADS), 0, stream, a->x, a->x_scale, 0LL, 0LL, a->w, a->bias, (const R*)a->state, a->lengths,
                           (const R*)a->dy, a->dy_t, a->dy_b, (const R*)a->dstate_out, (R*)a->dx, a->workspace, (R*)a->dstate, a->L, a->B,
                           a->C, a->silu, m);
    } else {
        auto k = conv_bwd_kernel<T, V, K, false>;
        hipLaunchKernelGGL(k, grid, dim3(THREADS), 0, stream, a->x, a->x_scale, a->x_t, a->x_b, a->w, a->bias, (const R*)a->state,
                           a->lengths, (const R*)a->dy, a->dy_t, a->dy_b, (const R*)a->dstate_out, (R*)a->dx, a->workspace,
                           (R*)a->dstate, a->L, a->B, a->C, a->silu, m);
    }
    GMT_LAUNCH_CHECK();
    return launch_slab_reduce(a->workspace, a->dparam, n, n, m.P, stream);
}

template <class T, int V> int fwd_k(const gmt_conv_args* a, hipStream_t s)
{
    return a->K == 2 ? run_fwd<T, V, 2>(a, s) : a->K == 3 ? run_fwd<T, V, 3>(a, s) : run_fwd<T, V, 4>(a, s);
}
template <class T, int V> int bwd_k(const gmt_conv_args* a, hipStream_t s)
{
    return a->K == 2 ? run_bwd<T, V, 2>(a, s) : a->K == 3 ? run_bwd<T, V, 3>(a, s) : run_bwd<T, V, 4>(a, s);
}

}  // namespace

extern "C" int gmt_causal_conv_fwd(const gmt_conv_args* a, hipStream_t stream)
{
    if (int rc = check(a)) return rc;
    GMT_CHECK_ARG(a->y);
    const int V = conv_vec(a, false);
    if (a->bf16) return V == 8 ? fwd_k<B16, 8>(a, stream) : V == 2 ? fwd_k<B16, 2>(a, stream) : fwd_k<B16, 1>(a, stream);
    return V == 4 ? fwd_k<F32, 4>(a, stream) : V == 2 ? fwd_k<F32, 2>(a, stream) : fwd_k<F32, 1>(a, stream);
}

extern "C" int gmt_causal_conv_bwd_workspace_floats(const gmt_conv_args* a, long long* floats_out)
{
    if (int rc = check(a)) return rc;
    GMT_CHECK_ARG(floats_out);
    *floats_out = (long long)(a->K + 1) * a->C * conv_map(a->L, a->B, a->C, conv_vec(a, true)).P;
    return GMT_OK;
}

extern "C" int gmt_causal_conv_bwd(const gmt_conv_args* a, hipStream_t stream)
{
    if (int rc = check(a)) return rc;
    GMT_CHECK_ARG(a->dy && a->dx && a->dparam && a->workspace);
    const int V = conv_vec(a, true);
    if (a->bf16) return V == 8 ? bwd_k<B16, 8>(a, stream) : V == 2 ? bwd_k<B16, 2>(a, stream) : bwd_k<B16, 1>(a, stream);
    return V == 4 ? bwd_k<F32, 4>(a, stream) : V == 2 ? bwd_k<F32, 2>(a, stream) : bwd_k<F32, 1>(a, stream);
}

extern "C" int gmt_causal_conv_step(const gmt_conv_args* a, const unsigned char* active, hipStream_t stream)
{
    if (int rc = check_any(a)) return rc;
    GMT_CHECK_ARG(a->y && a->state && a->state_out);
    const int grid = gmt_grid_1d((long long)a->B * a->C, THREADS, 256 * 16);
#define GMT_STEP(T, K)                                                                                                     \
    hipLaunchKernelGGL((conv_step_kernel<T, K>), dim3(grid), dim3(THREADS), 0, stream, (const T::raw*)a->x, a->x_b,        \
                       (const T::raw*)a->state, (T::raw*)a->state_out, a->w, a->bias, active, (T::raw*)a->y, a->B, a->C, a->silu)
    if (a->bf16) { if (a->K == 2) GMT_STEP(B16, 2); else if (a->K == 3) GMT_STEP(B16, 3); else GMT_STEP(B16, 4); }
    else { if (a->K == 2) GMT_STEP(F32, 2); else if (a->K == 3) GMT_STEP(F32, 3); else GMT_STEP(F32, 4); }
#undef GMT_STEP
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}
