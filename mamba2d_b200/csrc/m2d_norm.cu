// Group normalisation with an activation, channels last: entry points and kernels.
#include "plan.cuh"
#include "m2d_seq.h"

namespace m2d {

struct NormArgs {
    const void *x, *weight, *bias, *d_y;
    void *y, *d_x;
    float* stats;              // (N,groups,2): mean, rstd
    float *sums, *partial;     // backward: (N,groups,2) means of dh and dh h; [splits][2][C] sums of dz h and dz
    long long N, S;
    int C, groups, per;        // per: channels of a group
    int act, params_f32;
    float eps;
};

// z = act's argument; its value, and its slope
__device__ __forceinline__ float act_value(float z, int act) {
    if (act == M2D_ACT_SILU) return z * __fdividef(1.f, 1.f + ex2(-z * kLog2e));
    if (act == M2D_ACT_GELU) return gelu_erf(z);
    return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == M2D_ACT_SILU) {
        const float s = __fdividef(1.f, 1.f + ex2(-z * kLog2e));
        return s * fmaf(z, 1.f - s, 1.f);
    }
    if (act == M2D_ACT_GELU) {
        // Phi(z) + z phi(z)
        return fmaf(z * 0.3989422804014327f, ex2(z * z * (-0.5f * kLog2e)), normcdff(z));
    }
    return 1.f;
}
template <typename io_t>
__device__ __forceinline__ float norm_param(const void* p, int c, int f32, float none) {
    if (!p) return none;
    return f32 ? __ldg(static_cast<const float*>(p) + c) : load1(static_cast<const io_t*>(p), c);
}

// Sums over a block of 256 threads, the same in every thread.
__device__ __forceinline__ float2 block_sum2(float2 v) {
    __shared__ float2 part[8];
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, m);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, m);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float2 s = part[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        s.x += part[i].x;
        s.y += part[i].y;
    }
    return s;
}

// Any shape: a CTA owns a group of an image and reads it three times (mean, variance about it, values).
template <typename io_t>
__global__ void __launch_bounds__(256) norm_fwd_any(const NormArgs a) {
    const long long n = blockIdx.x / a.groups, count = a.S * a.per;
    const int c0 = (int)(blockIdx.x % a.groups) * a.per;
    const io_t* const x = static_cast<const io_t*>(a.x) + n * a.S * a.C + c0;
    io_t* const y = static_cast<io_t*>(a.y) + n * a.S * a.C + c0;
    float2 v = make_float2(0.f, 0.f);
    for (long long i = threadIdx.x; i < count; i += 256) v.x += load1(x, i / a.per * a.C + i % a.per);
    const float mean = block_sum2(v).x / (float)count;
    v.x = 0.f;
    for (long long i = threadIdx.x; i < count; i += 256) {
        const float d = load1(x, i / a.per * a.C + i % a.per) - mean;
        v.x = fmaf(d, d, v.x);
    }
    const float rstd = rsqrtf(block_sum2(v).x / (float)count + a.eps);
    if (a.stats && threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[blockIdx.x] = make_float2(mean, rstd);
    for (long long i = threadIdx.x; i < count; i += 256) {
        const int c = (int)(i % a.per);
        const long long at = i / a.per * a.C + c;
        const float z = fmaf((load1(x, at) - mean) * rstd, norm_param<io_t>(a.weight, c0 + c, a.params_f32, 1.f), norm_param<io_t>(a.bias, c0 + c, a.params_f32, 0.f));
        store1(y, at, act_value(z, a.act));
    }
}

// dh = dy act'(z) w;  dx = rstd (dh - mean(dh) - h mean(dh h))
template <typename io_t>
__global__ void __launch_bounds__(256) norm_bwd_any(const NormArgs a) {
    const long long n = blockIdx.x / a.groups, count = a.S * a.per;
    const int c0 = (int)(blockIdx.x % a.groups) * a.per;
    const long long base = n * a.S * a.C + c0;
    const io_t *const x = static_cast<const io_t*>(a.x) + base, *const dy = static_cast<const io_t*>(a.d_y) + base;
    io_t* const dx = static_cast<io_t*>(a.d_x) + base;
    const float2 st = reinterpret_cast<const float2*>(a.stats)[blockIdx.x];
    auto at = [&](long long i, float& h, float& dh) {
        const int c = (int)(i % a.per);
        const long long o = i / a.per * a.C + c;
        const float w = norm_param<io_t>(a.weight, c0 + c, a.params_f32, 1.f);
        h = (load1(x, o) - st.x) * st.y;
        // (rounded before it meets its mean: a group of one value has a gradient of exactly zero)
        dh = __fmul_rn(load1(dy, o) * act_slope(fmaf(h, w, norm_param<io_t>(a.bias, c0 + c, a.params_f32, 0.f)), a.act), w);
        return o;
    };
    float2 v = make_float2(0.f, 0.f);
    float h, dh;
    for (long long i = threadIdx.x; i < count; i += 256) {
        at(i, h, dh);
        v.x += dh;
        v.y = fmaf(dh, h, v.y);
    }
    const float2 s = block_sum2(v);
    const float m0 = s.x / (float)count, m1 = s.y / (float)count;
    for (long long i = threadIdx.x; i < count; i += 256) {
        const long long o = at(i, h, dh);
        store1(dx, o, st.y * (dh - m0 - h * m1));
    }
}

// Sums over pixels and images for each channel: a CTA owns 32 channels of every gridDim.y-th row block.
template <typename io_t>
__global__ void __launch_bounds__(256) norm_wgrad_any(const NormArgs a) {
    __shared__ float2 part[8][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), row0 = threadIdx.x >> 5;
    float2 v = make_float2(0.f, 0.f);
    if (c < a.C) {
        const float w = norm_param<io_t>(a.weight, c, a.params_f32, 1.f), bias = norm_param<io_t>(a.bias, c, a.params_f32, 0.f);
        const int group = c / a.per;
        for (long long r = blockIdx.y * 8ll + row0; r < a.N * a.S; r += gridDim.y * 8ll) {
            const float2 st = reinterpret_cast<const float2*>(a.stats)[r / a.S * a.groups + group];
            const float h = (load1(static_cast<const io_t*>(a.x), r * a.C + c) - st.x) * st.y;
            const float dz = load1(static_cast<const io_t*>(a.d_y), r * a.C + c) * act_slope(fmaf(h, w, bias), a.act);
            v.x = fmaf(dz, h, v.x);
            v.y += dz;
        }
    }
    part[row0][threadIdx.x & 31] = v;
    __syncthreads();
    if (row0 == 0 && c < a.C) {
        for (int i = 1; i < 8; ++i) {
            v.x += part[i][threadIdx.x].x;
            v.y += part[i][threadIdx.x].y;
        }
        a.partial[(2ll * blockIdx.y) * a.C + c] = v.x;
        a.partial[(2ll * blockIdx.y + 1) * a.C + c] = v.y;
    }
}

// The sum of the splits' partial results, in order: [splits][2][C] -> d_weight, d_bias.  A warp's worth of splits at a time.
template <typename io_t>
__global__ void __launch_bounds__(256) norm_wgrad_sum(const float* __restrict__ partial, int splits, int C, int f32, void* d_weight, void* d_bias) {
    __shared__ float part[8][33];
    const int i = blockIdx.x * 32 + (threadIdx.x & 31), row0 = threadIdx.x >> 5;
    float v = 0.f;
    if (i < 2 * C)
        for (int s = row0; s < splits; s += 8) v += partial[(size_t)s * 2 * C + i];
    part[row0][threadIdx.x & 31] = v;
    __syncthreads();
    if (row0 == 0 && i < 2 * C) {
        for (int j = 1; j < 8; ++j) v += part[j][threadIdx.x];
        void* to = i < C ? d_weight : d_bias;
        const int c = i < C ? i : i - C;
        if (f32) static_cast<float*>(to)[c] = v;
        else store1(static_cast<io_t*>(to), c, v);
    }
}

static int check_norm(const m2d_norm_desc* d) {
    if (!d) return M2D_ERR_NULL;
    if (d->struct_bytes != sizeof(m2d_norm_desc)) return M2D_ERR_ABI;
    if (d->dtype != M2D_F32 && d->dtype != M2D_BF16) return M2D_ERR_DTYPE;
    if (d->act < M2D_ACT_NONE || d->act > M2D_ACT_GELU) return M2D_ERR_FLAGS;
    if (d->N < 1 || d->S < 1 || d->C < 1 || d->groups < 1 || d->C % d->groups) return M2D_ERR_SHAPE;
    if (d->N > (1ll << 40) || d->S > (1ll << 40) || d->N * d->groups >= (1ll << 31)) return M2D_ERR_TOO_LARGE;
    return M2D_OK;
}
static NormArgs norm_args(const m2d_norm_desc* d) {
    NormArgs a{};
    a.x = d->x; a.weight = d->weight; a.bias = d->bias; a.d_y = d->d_y;
    a.y = d->y; a.d_x = d->d_x; a.stats = d->stats;
    a.N = d->N; a.S = d->S; a.C = d->C; a.groups = d->groups; a.per = d->C / d->groups;
    a.act = d->act; a.params_f32 = d->params_f32; a.eps = d->eps;
    return a;
}
static int wgrad_splits(const m2d_norm_desc* d) {
    const long long blocks = (d->C + 31) / 32, rows = (d->N * d->S + 63) / 64;
    return (int)std::max<long long>(1, std::min<long long>({rows, 8ll * sm_count() / blocks + 1, 4096ll}));
}
static int norm_workspace_ok(const m2d_norm_desc* d, size_t need) {
    if (!need) return M2D_OK;
    return d->workspace && d->workspace_bytes >= need && (reinterpret_cast<uintptr_t>(d->workspace) & 255) == 0 ? M2D_OK : M2D_ERR_WORKSPACE;
}

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_norm_fwd_workspace(const m2d_norm_desc*) { return 0; }
extern "C" uint64_t m2d_norm_bwd_workspace(const m2d_norm_desc* d) {
    if (check_norm(d) != M2D_OK || !d->d_weight) return 0;
    return (uint64_t)wgrad_splits(d) * 2 * d->C * sizeof(float);
}

extern "C" int m2d_norm_fwd(const m2d_norm_desc* d, void* stream) {
    const int rc = check_norm(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->y) return M2D_ERR_NULL;
    const NormArgs a = norm_args(d);
    const unsigned grid = (unsigned)(d->N * d->groups);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d->dtype == M2D_F32) norm_fwd_any<float><<<grid, 256, 0, st>>>(a);
    else norm_fwd_any<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}

extern "C" int m2d_norm_bwd(const m2d_norm_desc* d, void* stream) {
    int rc = check_norm(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->d_y || !d->d_x || !d->stats || !d->d_weight != !d->d_bias) return M2D_ERR_NULL;
    if ((rc = norm_workspace_ok(d, m2d_norm_bwd_workspace(d))) != M2D_OK) return rc;
    NormArgs a = norm_args(d);
    a.partial = static_cast<float*>(d->workspace);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f32 = d->dtype == M2D_F32;
    const unsigned grid = (unsigned)(d->N * d->groups);
    if (f32) norm_bwd_any<float><<<grid, 256, 0, st>>>(a);
    else norm_bwd_any<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
    if (d->d_weight) {
        const int splits = wgrad_splits(d);
        const dim3 wgrid((d->C + 31) / 32, splits);
        const unsigned sgrid = (2 * d->C + 31) / 32;
        if (f32) {
            norm_wgrad_any<float><<<wgrid, 256, 0, st>>>(a);
            norm_wgrad_sum<float><<<sgrid, 256, 0, st>>>(a.partial, splits, d->C, 1, d->d_weight, d->d_bias);
        } else {
            norm_wgrad_any<__nv_bfloat16><<<wgrid, 256, 0, st>>>(a);
            norm_wgrad_sum<__nv_bfloat16><<<sgrid, 256, 0, st>>>(a.partial, splits, d->C, d->params_f32, d->d_weight, d->d_bias);
        }
    }
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}
