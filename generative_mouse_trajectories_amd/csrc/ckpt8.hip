// 8-bit activation checkpoints, and the weight gradient that reads them.
//
// A row is cut into blocks of 32 channels.  A block is stored as int8 codes q and one exponent byte s = e + 127 and stands for
// q 2^e:  e = the smallest exponent in -118 .. 121 with max|x| <= 127 * 2^e, q = x 2^-e rounded to nearest even (|q| <= 127).  The
// scale is a power of two, so that packing rounds once, a code's value is exact in fp32 and in bf16 (7 bits), and its error
// is at most 2^(e-1), that is max|x| / 127 - but at the ends of the range: a block whose maximum is below 127 2^-119 (1.9e-34) is off by
// up to 2^-119 (numbers below that become 0), one above 127.5 2^121, where 127 is the largest code, by up to 2^121.  The exponent's range
// keeps 2^-e, and every value that a block of normal numbers stands for, a normal number.  A block that holds an infinity or a NaN
// stands for NaN throughout: s = 255, q = 0.
//
// Weight gradient: dW[n][i] = sum_r dY[r][n] Xhat[r][i], db[n] = sum_r dY[r][n].  Xhat is exact in bf16; an fp32 dY is exactly
// the sum of three bf16 numbers (its 24 mantissa bits cut into 8 + 8 + 8; all of them normal numbers from |dY| = 2^-102 on, below
// up to 2^-126 of each may be lost), so three bf16 MFMAs give the products without a rounding, accumulated in fp32, at 16 / 3 the
// rate of the fp32 matrix instruction.  A bf16 dY is one, and so is an infinite one.
#include "ssm_common.h"
#include "bf16_maps.h"

namespace {

using namespace gmt_ssm;

constexpr int BLK = 32;

// several elements at any address: one memory instruction, which need not be aligned on this hardware
template <class V, class E> __device__ __forceinline__ V load_any(const E* p) { V v; __builtin_memcpy(&v, p, sizeof(V)); return v; }
template <class V, class E> __device__ __forceinline__ void store_any(E* p, const V& v) { __builtin_memcpy(p, &v, sizeof(V)); }

// A lane takes 16 bytes of elements, 32 / V lanes share a block; a row's last lanes take what is left of it one by one.
// Bound by HBM: 105 MB of bf16 in, 54 MB of codes and exponents out, and back (200 x 512 rows of 512 channels): 35 and 26 us.
template <class T>
__global__ __launch_bounds__(256)
void pack_kernel(const typename T::raw* __restrict__ x, long long x_t, long long x_b, signed char* __restrict__ codes,
                 unsigned char* __restrict__ scale, long long rows, int B, int C, int nb)
{
    using R = typename T::raw;
    constexpr int V = 16 / sizeof(R), LPB = BLK / V;
    typedef R vec __attribute__((ext_vector_type(V)));
    typedef signed char qvec __attribute__((ext_vector_type(V)));
    const long long total = rows * nb * LPB, step = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const long long blk = i / LPB, row = blk / nb;
        const int part = (int)(i % LPB), c = (int)(blk % nb) * BLK + part * V;
        const R* p = x + row / B * x_t + row % B * x_b + c;
        vec v = {};
        if (c + V <= C) v = load_any<vec>(p);
        else {
#pragma unroll
            for (int k = 0; k < V; ++k) if (c + k < C) v[k] = p[k];
        }
        unsigned m = 0;                                 // largest magnitude by its bits: NaN > infinity > numbers
#pragma unroll
        for (int k = 0; k < V; ++k) m = max(m, __float_as_uint(to_f((R)v[k])) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < LPB; o <<= 1) m = max(m, (unsigned)__shfl_xor((int)m, o, 64));
        int e = (int)(m >> 23) - 133 + ((m & 0x7fffffu) > 0x7e0000u);
        e = min(max(e, -118), 121);
        const bool bad = m >= 0x7f800000u;
        const float inv = __uint_as_float((unsigned)(127 - e) << 23);
        qvec q;
#pragma unroll
        for (int k = 0; k < V; ++k) q[k] = bad ? 0 : (signed char)(int)fminf(fmaxf(rintf(to_f((R)v[k]) * inv), -127.f), 127.f);
        signed char* o = codes + row * C + c;
        if (c + V <= C) store_any(o, q);
        else {
#pragma unroll
            for (int k = 0; k < V; ++k) if (c + k < C) o[k] = q[k];
        }
        if (part == 0) scale[blk] = bad ? 255 : (unsigned char)(e + 127);
    }
}

template <class T>
__global__ __launch_bounds__(256)
void unpack_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ scale, typename T::raw* __restrict__ out,
                   long long rows, int C, int nb)
{
    using R = typename T::raw;
    constexpr int V = 16 / sizeof(R);
    typedef R vec __attribute__((ext_vector_type(V)));
    typedef signed char qvec __attribute__((ext_vector_type(V)));
    const int cv = (C + V - 1) / V;
    const long long total = rows * cv, step = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const long long row = i / cv;
        const int c = (int)(i % cv) * V;
        const unsigned char s = scale[row * nb + c / BLK];
        const signed char* p = codes + row * C + c;
        R* o = out + row * C + c;
        if (c + V <= C) {
            const qvec q = load_any<qvec>(p);
            vec v;
#pragma unroll
            for (int k = 0; k < V; ++k) v[k] = from_f<T>(to_f(Q8::raw{(signed char)q[k], s}));
            store_any(o, v);
        } else {
            for (int k = 0; c + k < C; ++k) o[k] = from_f<T>(to_f(Q8::raw{p[k], s}));
        }
    }
}

// ---- weight gradient.  A workgroup owns a 128 (n) x 128 (i) tile for one slab of rows, 4 waves of 64 x 64 (2 x 2 accumulators of
// 32 x 32).  Both operands have the contraction index as their ROW: stages of 32 rows go global -> registers -> LDS as bf16
// [32][128] images (dY as PL of them), requested one stage ahead, and the fragments (8 consecutive rows of one column a lane)
// come out of ds_read_b64_tr_b16.  Chunk c (16 bytes) of row r sits at c ^ ((r & 3) << 2): the four rows that half a wave reads
// together fall on different banks.  Slabs are summed in a fixed order.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int WG_K = 32, WG_T = 128, WG_IMG = WG_K * WG_T * 2;     // rows a stage, tile width, bytes an image

__device__ __forceinline__ int img_addr(int row, int col) { return row * 256 + (((col >> 3) ^ ((row & 3) << 2)) << 4) + (col & 7) * 2; }

__device__ __forceinline__ bf16x8 tr_frag(const char* img, int col0, int s, int lane)
{
    s16x4 h[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        int row, col;
        gmt_bf16_maps::wg_tr_lane(lane, col0, s, half, row, col);
        h[half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(img + img_addr(row, col)));
    }
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

// the high halves of two floats as a pair of bf16 (cut, not rounded)
__device__ __forceinline__ unsigned hi_pair(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }

// T: type of dY
template <class T>
__global__ __launch_bounds__(256, 3)
void wgrad8_kernel(const typename T::raw* __restrict__ dY, long long ldy, const signed char* __restrict__ codes,
                   const unsigned char* __restrict__ scale, float* __restrict__ out, long long R, int N, int I, int ks, int want_db)
{
    constexpr int PL = __is_same(T, F32) ? 3 : 1;
    __shared__ __align__(16) char lds[(PL + 1) * WG_IMG];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wp = wave >> 1, wq = wave & 1;
    const int n_t = (N + WG_T - 1) / WG_T, i_t = (I + WG_T - 1) / WG_T, tiles = n_t * i_t;
    // 8 slabs or more (then a multiple of 8): block = xcd + 8 (tile + tiles * group), slab = 8 group + xcd, so that the tiles of one slab
    // share an XCD's L2.  Fewer: there are tiles enough for all XCDs.
    const int rest = blockIdx.x >> 3;
    const int tile = ks >= 8 ? rest % tiles : blockIdx.x % tiles, slab = ks >= 8 ? rest / tiles * 8 + (blockIdx.x & 7) : blockIdx.x / tiles;
    const int n0 = tile % n_t * WG_T, i0 = tile / n_t * WG_T;
    const long long r1 = R;
    const int all = (int)((R + WG_K - 1) / WG_K);       // stages, dealt to the slabs in turn
    const int nb = (I + BLK - 1) / BLK;

    const int yc = (tid & 31) * 4, yr = tid >> 5;       // dY: 4 columns, rows yr + 8 j
    const int xc = (tid & 7) * 16, xr = tid >> 3;       // codes: 16 columns of one row (half a block)
    typedef typename T::raw yvec __attribute__((ext_vector_type(4)));
    typedef signed char qvec __attribute__((ext_vector_type(16)));
    typedef yvec yvec_any __attribute__((aligned(sizeof(typename T::raw))));        // loads need not be aligned
    typedef qvec qvec_any __attribute__((aligned(1)));
    struct Stage { yvec y[4]; qvec q; unsigned char s; };
    float colsum[4] = {};
    const bool y_in = n0 + yc + 4 <= N, x_in = i0 + xc + 16 <= I;
    // uniform base of a stage + 32-bit offsets of the thread (launch_wgrad8 checks that they fit)
    const unsigned yoff = (unsigned)(yr * (int)ldy + yc) * sizeof(typename T::raw);
    const unsigned qoff = xr * I + xc, soff = xr * nb + xc / BLK;
    auto request = [&](Stage& st, long long r) {
        const Uniform qp = uniform(codes + r * I + i0), sp = uniform(scale + r * nb + i0 / BLK);
        // (uniform) Whole rows of tiles whose last element lies within the buffers.  Beyond column N or I of a row that reads the next
        // row (or what lies between rows): it ends in rows and columns of the tile that are not stored.
        const long long last = r + WG_K - 1;
        if (last < r1 && last * ldy + n0 + WG_T <= (R - 1) * ldy + N && last * I + i0 + WG_T <= R * I &&
            last * nb + i0 / BLK + WG_T / BLK <= R * nb) {
#pragma unroll
            for (int j = 0; j < 4; ++j) st.y[j] = load_at<yvec_any>(uniform(dY + (r + 8 * j) * ldy + n0), yoff);
            st.q = load_at<qvec_any>(qp, qoff);
            st.s = load_at<unsigned char>(sp, soff);
            return;
        }
        const int left = (int)(r1 - r < WG_K ? r1 - r : WG_K);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const Uniform yp = uniform(dY + (r + 8 * j) * ldy + n0);
            st.y[j] = yvec{};
            if (yr + 8 * j < left) {
                if (y_in) st.y[j] = load_at<yvec_any>(yp, yoff);
                else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) if (n0 + yc + k < N) st.y[j][k] = load_at<typename T::raw>(yp, yoff + k * sizeof(typename T::raw));
                }
            }
        }
        st.s = 127;
        st.q = qvec{};
        if (xr < left && i0 + xc < I) {
            st.s = load_at<unsigned char>(sp, soff);
            if (x_in) st.q = load_at<qvec_any>(qp, qoff);
            else {
#pragma unroll
                for (int k = 0; k < 16; ++k) if (i0 + xc + k < I) st.q[k] = load_at<signed char>(qp, qoff + k);
            }
        }
    };
    auto put = [&](const Stage& st, char* img) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int row = yr + 8 * j;
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = to_f((typename T::raw)st.y[j][k]); colsum[k] += v[k]; }
#pragma unroll
            for (int pl = 0; pl < PL; ++pl) {
                uint2 w = make_uint2(hi_pair(v[0], v[1]), hi_pair(v[2], v[3]));
                *reinterpret_cast<uint2*>(img + pl * WG_IMG + img_addr(row, yc)) = w;
                if (pl + 1 < PL) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] -= __uint_as_float(__float_as_uint(v[k]) & 0xffff0000u);
                }
            }
        }
        if constexpr (PL > 1) {
            // An infinity is its first number alone, but inf - inf was a NaN.  Looked for only where the column sums show one (or a NaN, or
            // overflow): 345 -> 347 us at R=524288 N=512 I=128 with the packing, where a test of every value takes 352.
            if (__any(!(fabsf(colsum[0]) + fabsf(colsum[1]) + fabsf(colsum[2]) + fabsf(colsum[3]) < __builtin_inff()))) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (__builtin_isinf(to_f((typename T::raw)st.y[j][k]))) {
#pragma unroll
                            for (int pl = 1; pl < PL; ++pl)
                                *reinterpret_cast<unsigned short*>(img + pl * WG_IMG + img_addr(yr + 8 * j, yc + k)) = 0;
                        }
            }
        }
        const float sc = __uint_as_float((unsigned)st.s << 23);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            unsigned w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = hi_pair((float)st.q[8 * h + 2 * k] * sc, (float)st.q[8 * h + 2 * k + 1] * sc);
            *reinterpret_cast<uint4*>(img + PL * WG_IMG + img_addr(xr, xc + 8 * h)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    };
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const int nk = (all - slab + ks - 1) / ks;
    auto at = [&](int t) { return (long long)(slab + t * ks) * WG_K; };
    auto contract = [&](const char* img) {
#pragma unroll
        for (int s = 0; s < WG_K / 16; ++s) {
            bf16x8 q[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) q[j] = tr_frag(img + PL * WG_IMG, wq * 64 + j * 32, s, lane);
#pragma unroll
            for (int pl = 0; pl < PL; ++pl) {
                bf16x8 p[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) p[i] = tr_frag(img + pl * WG_IMG, wp * 64 + i * 32, s, lane);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[i], q[j], acc[i][j], 0, 0, 0);
            }
        }
    };
    Stage st;
    if (nk > 0) { request(st, at(0)); put(st, lds); }
    __syncthreads();
    for (int t = 0; t < nk; ++t) {
        if (t + 1 < nk) request(st, at(t + 1));
        contract(lds);
        __syncthreads();                                // everybody is done with stage t
        if (t + 1 < nk) put(st, lds);
        __syncthreads();                                // stage t + 1 is written
    }
    const int lo = lane & 31, hi = lane >> 5;
    float* slab_out = out + (long long)slab * ((long long)N * I + N);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int col = i0 + wq * 64 + j * 32 + lo;
        if (col < I) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int n = n0 + wp * 64 + i * 32 + (r & 3) + 8 * (r >> 2) + 4 * hi;
                    if (n < N) slab_out[(long long)n * I + col] = acc[i][j][r];
                }
        }
    }
    if (want_db && i0 == 0) {                           // (uniform) column sums: 8 row groups of 32 threads x 4 columns
        float (*sum)[WG_T] = reinterpret_cast<float (*)[WG_T]>(lds);
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[yr][yc + k] = colsum[k];
        __syncthreads();
        if (tid < WG_T && n0 + tid < N) {
            float v = 0.f;
#pragma unroll
            for (int r = 0; r < 8; ++r) v += sum[r][tid];
            slab_out[(long long)N * I + n0 + tid] = v;
        }
    }
}

// Slabs of four stages or more, three workgroups a CU in all (R=524288 N=512 I=128 fp32, in one build when it was chosen: three with one LDS
// image each 314 us, two 359 us, two with two images, which need one barrier a stage, 362 us; now 267 us).
int wgrad8_slabs(long long R, int N, int I)
{
    const long long tiles = (long long)((N + WG_T - 1) / WG_T) * ((I + WG_T - 1) / WG_T);
    long long k = (768 + tiles - 1) / tiles;
    const long long most = (R + 4 * WG_K - 1) / (4 * WG_K);
    if (k > most) k = most;
    return (int)(k < 1 ? 1 : k >= 8 ? k / 8 * 8 : k);
}

template <class T> int launch_wgrad8(const void* dY, long long ldy, const signed char* codes, const unsigned char* scale, float* slab, long long R,
                                     int N, int I, int ks, int want_db, hipStream_t stream)
{
    const long long tiles = (long long)((N + WG_T - 1) / WG_T) * ((I + WG_T - 1) / WG_T), grid = tiles * ks;
    hipLaunchKernelGGL(wgrad8_kernel<T>, dim3((unsigned)grid), dim3(256), 0, stream, (const typename T::raw*)dY, ldy, codes, scale, slab, R, N, I,
                       ks, want_db);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}

}  // namespace

extern "C" int gmt_ckpt8_pack(const void* x, long long x_t, long long x_b, signed char* codes, unsigned char* scale, long long T, int B,
                              int C, int bf16, hipStream_t stream)
{
    GMT_CHECK_ARG(x && codes && scale && T > 0 && B > 0 && C > 0);
    const int V = bf16 ? 8 : 4, nb = (C + BLK - 1) / BLK;
    const long long rows = T * B;
    const int grid = gmt_grid_1d(rows * nb * (BLK / V), 256, 256 * 16);
    if (bf16) hipLaunchKernelGGL(pack_kernel<B16>, dim3(grid), dim3(256), 0, stream, (const unsigned short*)x, x_t, x_b, codes, scale, rows, B, C, nb);
    else hipLaunchKernelGGL(pack_kernel<F32>, dim3(grid), dim3(256), 0, stream, (const float*)x, x_t, x_b, codes, scale, rows, B, C, nb);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}

extern "C" int gmt_ckpt8_unpack(const signed char* codes, const unsigned char* scale, void* out, long long rows, int C, int bf16, hipStream_t stream)
{
    GMT_CHECK_ARG(out && codes && scale && rows > 0 && C > 0);
    const int V = bf16 ? 8 : 4, nb = (C + BLK - 1) / BLK;
    const int grid = gmt_grid_1d(rows * ((C + V - 1) / V), 256, 256 * 16);
    if (bf16) hipLaunchKernelGGL(unpack_kernel<B16>, dim3(grid), dim3(256), 0, stream, codes, scale, (unsigned short*)out, rows, C, nb);
    else hipLaunchKernelGGL(unpack_kernel<F32>, dim3(grid), dim3(256), 0, stream, codes, scale, (float*)out, rows, C, nb);
    GMT_LAUNCH_CHECK();
    return GMT_OK;
}

extern "C" int gmt_ckpt8_wgrad_workspace_floats(long long R, int N, int I, long long* floats_out)
{
    GMT_CHECK_ARG(R > 0 && N > 0 && I > 0 && floats_out);
    const int ks = wgrad8_slabs(R, N, I);
    *floats_out = ks > 1 ? ks * ((long long)N * I + N) : 0;
    return GMT_OK;
}

extern "C" int gmt_ckpt8_wgrad(const void* dY, long long ldy, const signed char* codes, const unsigned char* scale, float* dW_db, long long R,
                               int N, int I, int bf16, int want_db, float* workspace, long long workspace_floats, hipStream_t stream)
{
    GMT_CHECK_ARG(dY && codes && scale && dW_db && R > 0 && N > 0 && I > 0 && ldy >= N);
    const int ks = wgrad8_slabs(R, N, I);
    // 32-bit offsets within a stage of rows; fewer than 2^32 threads; 32-bit numbers of stages
    const long long tiles = (long long)((N + WG_T - 1) / WG_T) * ((I + WG_T - 1) / WG_T);
    if (ldy >= (1LL << 24) || I >= (1 << 24) || tiles * ks >= (1LL << 24) || R >= (1LL << 35)) return GMT_ERR_UNSUPPORTED;
    const long long n = (long long)N * I + (want_db ? N : 0), pitch = (long long)N * I + N;
    if (ks > 1 && (!workspace || workspace_floats < ks * pitch)) return GMT_ERR_WORKSPACE;
    float* slab = ks > 1 ? workspace : dW_db;
    const int rc = bf16 ? launch_wgrad8<B16>(dY, ldy, codes, scale, slab, R, N, I, ks, want_db, stream)
                        : launch_wgrad8<F32>(dY, ldy, codes, scale, slab, R, N, I, ks, want_db, stream);
    if (rc || ks == 1) return rc;
    return launch_slab_reduce(workspace, dW_db, n, pitch, ks, stream);
}
