// Layer normalisation of rows, with the residual sum before it, forward and backward with the parameters' gradients.
//
//   s = x + r in the tensors' type;  y = (s - mean) rstd w + b
//   dh = dy w;  dx = rstd (dh - mean(dh) - h mean(dh h)) + ds,  h = (s - mean) rstd;  dw = sum dy h,  db = sum dy over rows
//
// A row is held in registers, by 8, 16 or 32 lanes of a warp or by a CTA, as its length asks; mean first, then the squares about it.  The mean is
// taken about the row's first value, so that equal values have that value for a mean, whatever its size.  In the backward pass a thread
// has the same columns in every row that it meets: it sums their parameter gradients in registers, CTAs write their sums side by side, and a second
// launch adds those up in a fixed order.  Rows too long for registers are read again where they are needed.
#include "follow.cuh"
#include "plan.cuh"
#include "m2d_seq.h"

namespace m2d {

struct LnArgs {
    const void *x, *r, *w, *b, *dy, *ds;
    long long xp, rp, dyp, dsp;        // rows apart, in elements
    void *s, *y, *dx, *dw, *db;
    float2* stats;                     // mean, rstd of each row
    float* partial;                    // [CTAs][2][C]
    long long N;
    int C, params_f32, parts;
    float eps;
};

template <typename T, int V> struct Lane;
template <> struct Lane<float, 4> {
    using Raw = float4;
    static __device__ __forceinline__ void get(const Raw& r, float* v) { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
    static __device__ __forceinline__ Raw put(const float* v) { return make_float4(v[0], v[1], v[2], v[3]); }
};
template <> struct Lane<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ void get(Raw r, float* v) { v[0] = r; }
    static __device__ __forceinline__ Raw put(const float* v) { return v[0]; }
};
template <> struct Lane<__nv_bfloat16, 8> {
    using Raw = uint4;
    static __device__ __forceinline__ void get(const Raw& r, float* v) {
        const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ Raw put(const float* v) {
        return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
};
template <> struct Lane<__nv_bfloat16, 1> {
    using Raw = unsigned short;
    static __device__ __forceinline__ void get(Raw r, float* v) { v[0] = bf16_bits_to_float(r); }
    static __device__ __forceinline__ Raw put(const float* v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v[0])); }
};
// V neighbouring values of a parameter (fp32 or T); `none` where there is no such parameter.
template <typename T, int V>
__device__ __forceinline__ void parameter(const void* p, int f32, int c, float none, float* v) {
    if (!p) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = none;
    } else if (f32) {
        const float* q = static_cast<const float*>(p) + c;
        if constexpr (V % 4 == 0) {
#pragma unroll
            for (int k = 0; k < V; k += 4) Lane<float, 4>::get(__ldg(reinterpret_cast<const float4*>(q + k)), v + k);
        } else {
            v[0] = __ldg(q);
        }
    } else {
        using P = Lane<T, V>;
        P::get(__ldg(reinterpret_cast<const typename P::Raw*>(static_cast<const T*>(p) + c)), v);
    }
}
template <typename T> __device__ __forceinline__ float value_of(const T* p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return __bfloat162float(*p);
}
// The sum of x and r in the tensors' type.
template <typename T> __device__ __forceinline__ float sum_as(float a, float b) {
    if constexpr (sizeof(T) == 4) return a + b;
    else return __bfloat162float(__float2bfloat16_rn(a + b));
}
// R lanes (R = 0: the CTA) add up K values each; all have the sums.  `slot` alternates between calls of a CTA.
template <int R, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], int& slot) {
#pragma unroll
    for (int m = (R ? R : 32) / 2; m; m >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], m);
    if constexpr (R == 0) {
        __shared__ float part[2][32][K];
        const int warps = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) part[slot][threadIdx.x >> 5][k] = v[k];
        __syncthreads();
        const int i = threadIdx.x & 31;
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = i < warps ? part[slot][i][k] : 0.f;
#pragma unroll
        for (int m = 16; m; m >>= 1)
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], m);
        slot ^= 1;
    }
}
constexpr int kLnThreads = 256;        // of a CTA whose rows are held by parts of warps

template <typename T, int V, int R, int NV>
__global__ void __launch_bounds__(R ? kLnThreads : 1024) ln_fwd_kernel(const LnArgs p) {
    using P = Lane<T, V>;
    using Raw = typename P::Raw;
    const int span = R ? R : blockDim.x, l = R ? threadIdx.x % R : threadIdx.x;
    const long long row = R ? (long long)blockIdx.x * (kLnThreads / (R ? R : 1)) + threadIdx.x / (R ? R : 1) : blockIdx.x;
    const bool on = row < p.N;
    const T *const x = static_cast<const T*>(p.x) + (on ? row : 0) * p.xp, *const r = p.r ? static_cast<const T*>(p.r) + (on ? row : 0) * p.rp : nullptr;
    float v[NV][V];
    int slot = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * span + l) * V;
        Raw a{};
        if (on && c < p.C) a = __ldcs(reinterpret_cast<const Raw*>(x + c));
        P::get(a, v[i]);
    }
    float first = value_of(x);
    if (r) {
        first = sum_as<T>(first, value_of(r));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * span + l) * V;
            if (!on || c >= p.C) continue;
            float t[V];
            P::get(__ldcs(reinterpret_cast<const Raw*>(r + c)), t);
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] = sum_as<T>(v[i][k], t[k]);
            *reinterpret_cast<Raw*>(static_cast<T*>(p.s) + row * p.C + c) = P::put(v[i]);
        }
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * span + l) * V < p.C)
#pragma unroll
            for (int k = 0; k < V; ++k) sum[0] += v[i][k] - first;
    row_sum<R>(sum, slot);
    const float mean = first + sum[0] / (float)p.C;
    sum[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if ((i * span + l) * V < p.C)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[i][k] -= mean;
                sum[0] = fmaf(v[i][k], v[i][k], sum[0]);
            }
    row_sum<R>(sum, slot);
    const float rstd = rsqrtf(sum[0] / (float)p.C + p.eps);
    if (!on) return;
    if (p.stats && l == 0) p.stats[row] = make_float2(mean, rstd);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * span + l) * V;
        if (c >= p.C) continue;
        float w[V], b[V];
        parameter<T, V>(p.w, p.params_f32, c, 1.f, w);
        parameter<T, V>(p.b, p.params_f32, c, 0.f, b);
#pragma unroll
        for (int k = 0; k < V; ++k) v[i][k] = fmaf(v[i][k] * rstd, w[k], b[k]);
        *reinterpret_cast<Raw*>(static_cast<T*>(p.y) + row * p.C + c) = P::put(v[i]);
    }
}

template <typename T, int V, int R, int NV>
__global__ void __launch_bounds__(R ? kLnThreads : 512) ln_bwd_kernel(const LnArgs p) {
    using P = Lane<T, V>;
    using Raw = typename P::Raw;
    extern __shared__ float sums[];                // where parts of warps hold rows: [columns of all lanes][2]
    let_follow();
    const int span = R ? R : blockDim.x, l = R ? threadIdx.x % R : threadIdx.x, rows = R ? kLnThreads / (R ? R : 1) : 1;
    float dw[NV][V] = {}, db[NV][V] = {};
    int slot = 0;
    const float per = 1.f / (float)p.C;
    for (long long first = (long long)blockIdx.x * rows; first < p.N; first += (long long)gridDim.x * rows) {
        const long long row = first + (R ? threadIdx.x / (R ? R : 1) : 0);
        const bool on = row < p.N;
        const T *const x = static_cast<const T*>(p.x) + (on ? row : 0) * p.xp, *const dy = static_cast<const T*>(p.dy) + (on ? row : 0) * p.dyp;
        Raw rx[NV], rd[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * span + l) * V;
            rx[i] = rd[i] = Raw{};
            if (on && c < p.C) {
                rx[i] = __ldcs(reinterpret_cast<const Raw*>(x + c));
                rd[i] = __ldcs(reinterpret_cast<const Raw*>(dy + c));
            }
        }
        const float2 st = on ? p.stats[row] : make_float2(0.f, 0.f);
        float h[NV][V], dh[NV][V], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * span + l) * V;
            float w[V];
            P::get(rx[i], h[i]);
            P::get(rd[i], dh[i]);
            if (c < p.C) parameter<T, V>(p.w, p.params_f32, c, 1.f, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                h[i][k] = (h[i][k] - st.x) * st.y;
                if (!on || c >= p.C) h[i][k] = 0.f, w[k] = 0.f;
                db[i][k] += dh[i][k];
                dw[i][k] = fmaf(dh[i][k], h[i][k], dw[i][k]);
                dh[i][k] *= w[k];
                sum[0] += dh[i][k];
                sum[1] = fmaf(dh[i][k], h[i][k], sum[1]);
            }
        }
        row_sum<R>(sum, slot);
        if (!on) continue;
        const float m0 = sum[0] * per, m1 = sum[1] * per;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * span + l) * V;
            if (c >= p.C) continue;
            float g[V] = {};
            if (p.ds) P::get(__ldcs(reinterpret_cast<const Raw*>(static_cast<const T*>(p.ds) + row * p.dsp + c)), g);
#pragma unroll
            for (int k = 0; k < V; ++k) g[k] = fmaf(st.y, fmaf(-h[i][k], m1, dh[i][k] - m0), g[k]);
            *reinterpret_cast<Raw*>(static_cast<T*>(p.dx) + row * p.C + c) = P::put(g);
        }
    }
    if (!p.partial) return;
    float* const out = p.partial + (long long)blockIdx.x * 2 * p.C;
    if constexpr (R == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int c = (i * span + l) * V + k;
                if (c < p.C) { out[c] = dw[i][k]; out[p.C + c] = db[i][k]; }
            }
    } else {
        // lanes of one warp that have the same columns, then the warps in turn
        constexpr int cols = R * NV * V;
#pragma unroll
        for (int m = R; m < 32; m <<= 1)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    dw[i][k] += __shfl_xor_sync(0xffffffffu, dw[i][k], m);
                    db[i][k] += __shfl_xor_sync(0xffffffffu, db[i][k], m);
                }
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        if (lane < R)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    sums[(warp * 2) * cols + (i * R + l) * V + k] = dw[i][k];
                    sums[(warp * 2 + 1) * cols + (i * R + l) * V + k] = db[i][k];
                }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * cols; c += kLnThreads) {
            float v = 0.f;
            for (int w = 0; w < kLnThreads / 32; ++w) v += sums[w * 2 * cols + c];
            const int col = c % cols;
            if (col < p.C) out[(c / cols) * p.C + col] = v;
        }
    }
}

// Rows of any length: every value is read three times.
constexpr int kLongThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kLongThreads) ln_long_fwd_kernel(const LnArgs p) {
    int slot = 0;
    for (long long row = blockIdx.x; row < p.N; row += gridDim.x) {
        const T *const x = static_cast<const T*>(p.x) + row * p.xp, *const r = p.r ? static_cast<const T*>(p.r) + row * p.rp : nullptr;
        auto at = [&](int c) { return r ? sum_as<T>(value_of(x + c), value_of(r + c)) : value_of(x + c); };
        const float first = at(0);
        float sum[1] = {0.f};
        for (int c = threadIdx.x; c < p.C; c += kLongThreads) sum[0] += at(c) - first;
        row_sum<0>(sum, slot);
        const float mean = first + sum[0] / (float)p.C;
        sum[0] = 0.f;
        for (int c = threadIdx.x; c < p.C; c += kLongThreads) { const float d = at(c) - mean; sum[0] = fmaf(d, d, sum[0]); }
        row_sum<0>(sum, slot);
        const float rstd = rsqrtf(sum[0] / (float)p.C + p.eps);
        if (p.stats && threadIdx.x == 0) p.stats[row] = make_float2(mean, rstd);
        for (int c = threadIdx.x; c < p.C; c += kLongThreads) {
            const float v = at(c);
            float w, b;
            parameter<T, 1>(p.w, p.params_f32, c, 1.f, &w);
            parameter<T, 1>(p.b, p.params_f32, c, 0.f, &b);
            store1(static_cast<T*>(p.y), row * p.C + c, fmaf((v - mean) * rstd, w, b));
            if (r) store1(static_cast<T*>(p.s), row * p.C + c, v);
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(kLongThreads) ln_long_bwd_kernel(const LnArgs p) {
    let_follow();
    int slot = 0;
    for (long long row = blockIdx.x; row < p.N; row += gridDim.x) {
        const T *const x = static_cast<const T*>(p.x) + row * p.xp, *const dy = static_cast<const T*>(p.dy) + row * p.dyp;
        const float2 st = p.stats[row];
        float sum[2] = {0.f, 0.f}, w;
        for (int c = threadIdx.x; c < p.C; c += kLongThreads) {
            parameter<T, 1>(p.w, p.params_f32, c, 1.f, &w);
            const float dh = value_of(dy + c) * w;
            sum[0] += dh;
            sum[1] = fmaf(dh, (value_of(x + c) - st.x) * st.y, sum[1]);
        }
        row_sum<0>(sum, slot);
        const float m0 = sum[0] / (float)p.C, m1 = sum[1] / (float)p.C;
        for (int c = threadIdx.x; c < p.C; c += kLongThreads) {
            parameter<T, 1>(p.w, p.params_f32, c, 1.f, &w);
            const float h = (value_of(x + c) - st.x) * st.y, g = p.ds ? value_of(static_cast<const T*>(p.ds) + row * p.dsp + c) : 0.f;
            store1(static_cast<T*>(p.dx), row * p.C + c, fmaf(st.y, fmaf(-h, m1, value_of(dy + c) * w - m0), g));
        }
    }
    // the parameters' sums: this CTA's rows, column by column
    if (!p.partial) return;
    float* const out = p.partial + (long long)blockIdx.x * 2 * p.C;
    for (int c = threadIdx.x; c < p.C; c += kLongThreads) {
        float dw = 0.f, db = 0.f;
        for (long long row = blockIdx.x; row < p.N; row += gridDim.x) {
            const float2 st = p.stats[row];
            const float g = value_of(static_cast<const T*>(p.dy) + row * p.dyp + c);
            dw = fmaf(g, (value_of(static_cast<const T*>(p.x) + row * p.xp + c) - st.x) * st.y, dw);
            db += g;
        }
        out[c] = dw;
        out[p.C + c] = db;
    }
}

// Adds up the CTAs' sums: 32 columns of one of the two gradients a CTA, a warp every 32nd of the sums.
template <typename W>
__global__ void __launch_bounds__(1024) ln_params_kernel(const LnArgs p) {
    __shared__ float part[32][33];
    follow_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float v = 0.f;
    if (c < p.C)
        for (int i = warp; i < p.parts; i += 32) v += p.partial[((long long)i * 2 + blockIdx.y) * p.C + c];
    part[warp][lane] = v;
    __syncthreads();
    v = part[lane][warp];
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    const int col = blockIdx.x * 32 + warp;
    void* const out = blockIdx.y ? p.db : p.dw;
    if (lane == 0 && col < p.C && out) store1(static_cast<W*>(out), col, v);
}

// ---- host ---------------------------------------------------------------------------------------

static int check_ln(const m2d_ln_desc* d) {
    if (!d) return M2D_ERR_NULL;
    if (d->struct_bytes != sizeof(m2d_ln_desc)) return M2D_ERR_ABI;
    if (d->dtype != M2D_F32 && d->dtype != M2D_BF16) return M2D_ERR_DTYPE;
    if (d->N < 1 || d->C < 1) return M2D_ERR_SHAPE;
    if (d->N > INT32_MAX || d->C > (1 << 30)) return M2D_ERR_TOO_LARGE;
    return M2D_OK;
}
// Whether every row of a tensor begins at a 16-byte boundary (rows may be one and the same).
static bool whole(const void* p, long long pitch, int es) { return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch * es % 16 == 0); }
struct LnPlan {
    int lanes, vec, nv, threads;       // lanes of a row (0: the CTA, -1: too long for registers), values of a load, loads of a lane
    int rows() const { return lanes > 0 ? threads / lanes : 1; }
};
static LnPlan plan_ln(const m2d_ln_desc* d, bool bwd) {
    const int es = d->dtype == M2D_F32 ? 4 : 2, pes = d->params_f32 ? 4 : es;
    bool v = (long long)d->C * es % 16 == 0 && whole(d->x, d->x_row, es) && whole(d->weight, 0, pes);
    if (bwd) v = v && whole(d->d_y, d->d_y_row, es) && whole(d->d_sum, d->d_sum_row, es) && whole(d->d_x, 0, es);
    else v = v && whole(d->residual, d->residual_row, es) && whole(d->bias, 0, pes) && whole(d->y, 0, es) && whole(d->sum, 0, es);
    LnPlan pl{};
    pl.vec = v ? 16 / es : 1;
    pl.threads = kLnThreads;
    // up to 16 values a lane
    const int most = 16 / pl.vec;
    static const int wide[][2] = {{8, 1}, {8, 2}, {16, 2}, {32, 2}, {32, 4}}, narrow[][2] = {{32, 4}, {32, 16}};
    for (int i = 0; i < (v ? 5 : 2); ++i) {
        pl.lanes = v ? wide[i][0] : narrow[i][0];
        pl.nv = v ? wide[i][1] : narrow[i][1];
        if (pl.nv <= most && d->C <= pl.lanes * pl.vec * pl.nv) return pl;
    }
    pl.lanes = 0;
    pl.nv = most;
    pl.threads = (d->C + pl.vec * pl.nv * 32 - 1) / (pl.vec * pl.nv * 32) * 32;
    if (pl.threads > (bwd ? 512 : 1024)) { pl.lanes = -1; pl.threads = kLongThreads; }
    return pl;
}
// Calls fn(element, values of a load, lanes, loads of a lane) with the plan's.
template <typename F>
static int for_ln(const m2d_ln_desc* d, const LnPlan& pl, F fn) {
    auto go = [&](auto elem, auto full) {
        using std::integral_constant;
        constexpr int V = decltype(full)::value;
        auto with = [&](auto v, auto lanes, auto nv) { return fn(elem, v, lanes, nv); };
        constexpr integral_constant<int, 0> cta{};
        constexpr integral_constant<int, 8> l8{};
        constexpr integral_constant<int, 16> l16{};
        constexpr integral_constant<int, 32> l32{};
        constexpr integral_constant<int, 1> n1{};
        constexpr integral_constant<int, 2> n2{};
        constexpr integral_constant<int, 16 / V> most{};
        if (pl.vec == 1) return pl.lanes == 0 ? with(n1, cta, l16) : pl.nv == 4 ? with(n1, l32, integral_constant<int, 4>{}) : with(n1, l32, l16);
        if (pl.lanes == 0) return with(full, cta, most);
        if (pl.lanes == 32) return pl.nv == 2 ? with(full, l32, n2) : with(full, l32, most);
        return pl.lanes == 16 ? with(full, l16, n2) : pl.nv == 2 ? with(full, l8, n2) : with(full, l8, n1);
    };
    return d->dtype == M2D_F32 ? go(float{}, std::integral_constant<int, 4>{}) : go(__nv_bfloat16{}, std::integral_constant<int, 8>{});
}
static LnArgs ln_args(const m2d_ln_desc* d) {
    LnArgs a{};
    a.x = d->x; a.r = d->residual; a.w = d->weight; a.b = d->bias; a.dy = d->d_y; a.ds = d->d_sum;
    a.xp = d->x_row; a.rp = d->residual_row; a.dyp = d->d_y_row; a.dsp = d->d_sum_row;
    a.s = d->sum; a.y = d->y; a.dx = d->d_x; a.dw = d->d_weight; a.db = d->d_bias;
    a.stats = reinterpret_cast<float2*>(d->stats);
    a.N = d->N; a.C = d->C; a.params_f32 = d->params_f32; a.eps = d->eps;
    return a;
}
// CTAs of the backward pass: what the SMs hold at once, so that a CTA meets many rows.
static long long ln_parts(const m2d_ln_desc* d, const LnPlan& pl) {
    const long long tasks = (d->N + pl.rows() - 1) / pl.rows();
    const int held = std::max(1, 768 / pl.threads);
    return std::min<long long>(tasks, (long long)held * sm_count());
}

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_ln_bwd_workspace(const m2d_ln_desc* d) {
    if (check_ln(d) != M2D_OK || (!d->d_weight && !d->d_bias)) return 0;
    return (uint64_t)ln_parts(d, plan_ln(d, true)) * 2 * d->C * sizeof(float);
}

extern "C" int m2d_ln_fwd(const m2d_ln_desc* d, void* stream) {
    const int rc = check_ln(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->y || (d->residual && !d->sum)) return M2D_ERR_NULL;
    const LnArgs a = ln_args(d);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const LnPlan pl = plan_ln(d, false);
    if (pl.lanes < 0) {
        const unsigned grid = (unsigned)std::min<long long>(d->N, 4ll * sm_count());
        if (d->dtype == M2D_F32) ln_long_fwd_kernel<float><<<grid, kLongThreads, 0, st>>>(a);
        else ln_long_fwd_kernel<__nv_bfloat16><<<grid, kLongThreads, 0, st>>>(a);
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    }
    return for_ln(d, pl, [&](auto elem, auto vec, auto lanes, auto nv) {
        ln_fwd_kernel<decltype(elem), decltype(vec)::value, decltype(lanes)::value, decltype(nv)::value><<<(unsigned)((d->N + pl.rows() - 1) / pl.rows()), pl.threads, 0, st>>>(a);
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    });
}

extern "C" int m2d_ln_bwd(const m2d_ln_desc* d, void* stream) {
    const int rc = check_ln(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->stats || !d->d_y || !d->d_x) return M2D_ERR_NULL;
    LnArgs a = ln_args(d);
    const bool params = d->d_weight || d->d_bias;
    if (params && (!d->workspace || d->workspace_bytes < m2d_ln_bwd_workspace(d) || (reinterpret_cast<uintptr_t>(d->workspace) & 255))) return M2D_ERR_WORKSPACE;
    a.partial = params ? static_cast<float*>(d->workspace) : nullptr;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const LnPlan pl = plan_ln(d, true);
    a.parts = (int)ln_parts(d, pl);
    int done = M2D_OK;
    if (pl.lanes < 0) {
        if (d->dtype == M2D_F32) ln_long_bwd_kernel<float><<<a.parts, kLongThreads, 0, st>>>(a);
        else ln_long_bwd_kernel<__nv_bfloat16><<<a.parts, kLongThreads, 0, st>>>(a);
    } else {
        done = for_ln(d, pl, [&](auto elem, auto vec, auto lanes, auto nv) {
            constexpr int V = decltype(vec)::value, R = decltype(lanes)::value, NV = decltype(nv)::value;
            const size_t smem = R && params ? (size_t)kLnThreads / 32 * 2 * R * NV * V * sizeof(float) : 0;
            if (!allow_smem(reinterpret_cast<const void*>(ln_bwd_kernel<decltype(elem), V, R, NV>), smem)) return (int)M2D_ERR_LAUNCH;
            ln_bwd_kernel<decltype(elem), V, R, NV><<<a.parts, pl.threads, smem, st>>>(a);
            return (int)M2D_OK;
        });
    }
    if (done != M2D_OK || cudaGetLastError() != cudaSuccess) return M2D_ERR_LAUNCH;
    if (!params) return M2D_OK;
    const dim3 grid((d->C + 31) / 32, 2);
    const bool f32 = d->params_f32 || d->dtype == M2D_F32;
    if (!(f32 ? launch_following(ln_params_kernel<float>, grid, dim3(1024), 0, st, a) : launch_following(ln_params_kernel<__nv_bfloat16>, grid, dim3(1024), 0, st, a))) return M2D_ERR_LAUNCH;
    return M2D_OK;
}
