// Group normalisation with an activation, channels last: entry points and kernels.
#include <cooperative_groups.h>

#include "follow.cuh"
#include "plan.cuh"
#include "m2d_seq.h"

namespace m2d {

struct NormArgs {
    const void *x, *weight, *bias, *d_y;
    void *y, *d_x;
    float* stats;              // (N,groups,2): mean, rstd
    float* partial;            // backward: [CTAs][2][C] sums of dz h and dz
    float2* pieces;            // images in pieces: (N,pieces,groups) mean and sum of squares about it
    float2* group_sums;        // images in pieces, backward: (N,groups) means of dh and dh h
    long long N, S;
    int C, groups, per;        // per: channels of a group
    int act, params_f32;
    float eps;
    int rows, pieces_n;        // rows of a CTA (at most), CTAs of an image
};

__device__ __forceinline__ float rcp_of(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// The smaller of the two (the larger), NaN where z is.
__device__ __forceinline__ float at_most(float z, float top) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(top));
    return r;
}
__device__ __forceinline__ float at_least(float z, float bottom) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(bottom));
    return r;
}
// Phi(-|z|) = erfc(|z| / sqrt 2) / 2 and exp(-z^2 / 2), by formula 7.1.26 of Abramowitz and Stegun's Handbook of Mathematical Functions,
// erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2) with t = 1 / (1 + p x), within 1.5e-7: the exponential is the one that phi needs.  (In
// scalars: a packed multiply-add takes no constant, and the constants' registers cost more than it saves.)
__device__ __forceinline__ float gauss_tail(float z, float* e) {
    const float t = rcp_of(fmaf(fabsf(z), 0.3275911f * 0.70710678f, 1.f));
    *e = ex2(z * (z * (-0.5f * kLog2e)));
    float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    q = fmaf(q, t, 0.5f * 1.421413741f);
    q = fmaf(q, t, 0.5f * -0.284496736f);
    q = fmaf(q, t, 0.5f * 0.254829592f);
    return q * t * *e;
}
// act(z) and act'(z).  A NaN stays one.  Value and slope at an infinity are their limits: z is bounded where an infinity would meet a
// zero, at a value beyond which exp has long been zero or infinite.
constexpr float kActFar = 256.f;
template <int ACT>
__device__ __forceinline__ float act_value1(float z) {
    if constexpr (ACT == M2D_ACT_SILU) {
        z = at_least(z, -kActFar);
        return z * rcp_of(1.f + ex2(z * -kLog2e));
    }
    if constexpr (ACT == M2D_ACT_GELU) {
        float e;
        const float tail = gauss_tail(z, &e);
        return fmaf(-at_most(fabsf(z), kActFar), tail, z < 0.f ? 0.f : z);      // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    }
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope1(float z) {
    if constexpr (ACT != M2D_ACT_NONE) z = at_least(at_most(z, kActFar), -kActFar);
    if constexpr (ACT == M2D_ACT_SILU) {
        const float s = rcp_of(1.f + ex2(z * -kLog2e));
        return s * fmaf(z, 1.f - s, 1.f);                     // s (1 + z (1 - s)), s the logistic function
    }
    if constexpr (ACT == M2D_ACT_GELU) {
        float e;
        const float tail = gauss_tail(z, &e);
        return fmaf(z * 0.3989422804f, e, z < 0.f ? tail : 1.f - tail);      // Phi(z) + z phi(z)
    }
    return 1.f;
}
template <int ACT>
__device__ __forceinline__ float2 act_value2(float2 z) { return make_float2(act_value1<ACT>(z.x), act_value1<ACT>(z.y)); }
template <int ACT>
__device__ __forceinline__ float2 act_slope2(float2 z) { return make_float2(act_slope1<ACT>(z.x), act_slope1<ACT>(z.y)); }
__device__ __forceinline__ float act_value(float z, int act) {
    return act == M2D_ACT_SILU ? act_value1<M2D_ACT_SILU>(z) : act == M2D_ACT_GELU ? act_value1<M2D_ACT_GELU>(z) : z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
    return act == M2D_ACT_SILU ? act_slope1<M2D_ACT_SILU>(z) : act == M2D_ACT_GELU ? act_slope1<M2D_ACT_GELU>(z) : 1.f;
}
template <typename io_t>
__device__ __forceinline__ float norm_param(const void* p, int c, int f32, float none) {
    if (!p) return none;
    return f32 ? __ldg(static_cast<const float*>(p) + c) : load1(static_cast<const io_t*>(p), c);
}

// 16 bytes: eight bf16 or four fp32 values, as pairs
template <typename io_t>
struct Vec {
    static constexpr int n = 16 / sizeof(io_t), pairs = n / 2;
    uint4 u;
    __device__ __forceinline__ float2 get(int i) const {
        if constexpr (sizeof(io_t) == 2) {
            const uint32_t w = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
            return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        } else {
            return i == 0 ? make_float2(__uint_as_float(u.x), __uint_as_float(u.y)) : make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
        }
    }
    __device__ __forceinline__ void set(int i, float2 v) {
        if constexpr (sizeof(io_t) == 2) {
            const uint32_t w = pack_bf16x2(v.x, v.y);
            if (i == 0) u.x = w; else if (i == 1) u.y = w; else if (i == 2) u.z = w; else u.w = w;
        } else if (i == 0) {
            u.x = __float_as_uint(v.x); u.y = __float_as_uint(v.y);
        } else {
            u.z = __float_as_uint(v.x); u.w = __float_as_uint(v.y);
        }
    }
};

// Sums over a block of 256 threads, the same in every thread.
__device__ __forceinline__ double2 block_sum2(double2 v) {
    __shared__ double2 part[8];
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, m);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, m);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    double2 s = part[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) {
        s.x += part[i].x;
        s.y += part[i].y;
    }
    return s;
}

// ------------------------------------------------------------------------------------------------
// S = 1, groups of whole 16-byte vectors, at most 32: a group is that many neighbouring lanes of a warp (a warp holds as
// many groups as fit).  A thread keeps its channels over all the rows that it walks: their parameters stay in registers, and
// so do the sums of their gradients.  One read of x (and dy), one write: at 16384x16x128 bf16 with SiLU 39 us forward (3.5 TB/s),
// 67 us backward with the parameters' sums (3.0 TB/s); what holds it up is the activation's instructions and the groups' shuffles at 16
// (backward) and 32 warps an SM, which issue in 51 and 66 % of the cycles.
// ------------------------------------------------------------------------------------------------
template <typename io_t, int ACT, bool BWD>
__global__ void __launch_bounds__(256, BWD ? 2 : 4) norm_rows_kernel(const NormArgs a, int lanes, int cols) {      // lanes of a group, groups of a row in this block
    using V = Vec<io_t>;
    extern __shared__ float red[];
    const int per_row = a.C / V::n, lane = threadIdx.x & 31, fit = 32 / lanes, pos = lane % lanes;
    const int slot = (threadIdx.x >> 5) * fit + lane / lanes, row0 = slot / cols, rows = 8 * fit / cols;
    const int group = blockIdx.y * cols + slot % cols, col = group * lanes + pos;
    const bool on = lane < fit * lanes && row0 < rows && group < a.groups;
    const unsigned mask = __ballot_sync(0xffffffffu, on);       // (whole groups)
    const int c0 = col * V::n;
    const bool even = (lanes & (lanes - 1)) == 0;
    let_follow();
    float2 w[V::pairs], bias[V::pairs], dw[V::pairs] = {}, db[V::pairs] = {};
#pragma unroll
    for (int i = 0; i < V::pairs; ++i) {
        w[i] = on ? make_float2(norm_param<io_t>(a.weight, c0 + 2 * i, a.params_f32, 1.f), norm_param<io_t>(a.weight, c0 + 2 * i + 1, a.params_f32, 1.f)) : make_float2(0.f, 0.f);
        bias[i] = on ? make_float2(norm_param<io_t>(a.bias, c0 + 2 * i, a.params_f32, 0.f), norm_param<io_t>(a.bias, c0 + 2 * i + 1, a.params_f32, 0.f)) : make_float2(0.f, 0.f);
    }
    const float inv = 1.f / (float)a.per;
    auto group_sum = [&](float v) {
        if (even) {
            for (int m = lanes / 2; m; m >>= 1) v += __shfl_xor_sync(mask, v, m);
            return v;
        }
        for (int m = 1; m < lanes; m <<= 1) {
            const float o = __shfl_down_sync(mask, v, m);
            if (pos + m < lanes) v += o;
        }
        return __shfl_sync(mask, v, lane - pos);
    };
    if (on) {
        constexpr int kRows = 2;                                // in flight
        const long long step = (long long)gridDim.x * rows;
        const size_t ahead = (size_t)step * per_row, ahead_g = (size_t)step * a.groups;
        size_t at = (size_t)(blockIdx.x * (long long)rows + row0) * per_row + col, at_g = (size_t)(blockIdx.x * (long long)rows + row0) * a.groups + group;
        for (long long first = blockIdx.x * (long long)rows; first < a.N; first += step * kRows, at += ahead * kRows, at_g += ahead_g * kRows) {      // (as often for every lane)
            const bool live[kRows] = {first + row0 < a.N, first + step + row0 < a.N};      // (all lanes of a group agree; the others take part in the sums)
            V xv[kRows], gv[kRows];
            float2 st[kRows];
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                xv[j].u = live[j] ? __ldg(static_cast<const uint4*>(a.x) + at + j * ahead) : make_uint4(0, 0, 0, 0);
                if (BWD) {
                    gv[j].u = live[j] ? __ldg(static_cast<const uint4*>(a.d_y) + at + j * ahead) : make_uint4(0, 0, 0, 0);
                    st[j] = live[j] ? __ldg(reinterpret_cast<const float2*>(a.stats) + at_g + j * ahead_g) : make_float2(0.f, 0.f);
                }
            }
            float s0[kRows], s1[kRows];
            if constexpr (!BWD) {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    float2 sum = xv[j].get(0);
#pragma unroll
                    for (int i = 1; i < V::pairs; ++i) sum = __fadd2_rn(sum, xv[j].get(i));
                    s0[j] = sum.x + sum.y;
                }
                if (even) {
#pragma unroll
                    for (int j = 0; j < kRows; ++j) s0[j] = group_sum(s0[j]) * inv;
                } else {          // about the group's first value: where the size is no power of two, equal values' sum and its share are rounded
#pragma unroll
                    for (int j = 0; j < kRows; ++j) {
                        const float base = __shfl_sync(mask, xv[j].get(0).x, lane - pos);
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int i = 0; i < V::pairs; ++i) sum = __fadd2_rn(sum, __fadd2_rn(xv[j].get(i), make_float2(-base, -base)));
                        s0[j] = fmaf(group_sum(sum.x + sum.y), inv, base);
                    }
                }
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i) {
                        const float2 d = __fadd2_rn(xv[j].get(i), make_float2(-s0[j], -s0[j]));
                        sum = __ffma2_rn(d, d, sum);
                    }
                    s1[j] = sum.x + sum.y;
                }
#pragma unroll
                for (int j = 0; j < kRows; ++j) s1[j] = rsqrtf(group_sum(s1[j]) * inv + a.eps);
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    V out;
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i) {
                        const float2 h = __fmul2_rn(__fadd2_rn(xv[j].get(i), make_float2(-s0[j], -s0[j])), make_float2(s1[j], s1[j]));
                        out.set(i, act_value2<ACT>(__ffma2_rn(h, w[i], bias[i])));
                    }
                    if (live[j]) {
                        static_cast<uint4*>(a.y)[at + j * ahead] = out.u;
                        if (a.stats && pos == 0) reinterpret_cast<float2*>(a.stats)[at_g + j * ahead_g] = make_float2(s0[j], s1[j]);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < kRows; ++j) {
                    float2 h[V::pairs], dh[V::pairs], t0 = make_float2(0.f, 0.f), t1 = make_float2(0.f, 0.f);
                    const float2 minus = make_float2(-st[j].x, -st[j].x), rr = make_float2(st[j].y, st[j].y);
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i) {
                        h[i] = __fmul2_rn(__fadd2_rn(xv[j].get(i), minus), rr);
                        const float2 dz = __fmul2_rn(gv[j].get(i), act_slope2<ACT>(__ffma2_rn(h[i], w[i], bias[i])));
                        dw[i] = __ffma2_rn(dz, h[i], dw[i]);
                        db[i] = __fadd2_rn(db[i], dz);
                        dh[i] = __fmul2_rn(dz, w[i]);
                        t0 = __fadd2_rn(t0, dh[i]);
                        t1 = __ffma2_rn(dh[i], h[i], t1);
                    }
                    const float m0 = group_sum(t0.x + t0.y) * inv, m1 = group_sum(t1.x + t1.y) * inv;
                    V out;
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i)
                        out.set(i, __fmul2_rn(rr, __ffma2_rn(h[i], make_float2(-m1, -m1), __fadd2_rn(dh[i], make_float2(-m0, -m0)))));
                    if (live[j]) static_cast<uint4*>(a.d_x)[at + j * ahead] = out.u;
                }
            }
        }
    }
    if (BWD && a.partial) {
        // the block's rows, in order
        for (int k = 0; k < 2; ++k) {
            if (on)
#pragma unroll
                for (int i = 0; i < V::pairs; ++i) *reinterpret_cast<float2*>(red + ((size_t)row0 * cols * lanes + (slot % cols) * lanes + pos) * V::n + 2 * i) = k ? db[i] : dw[i];
            __syncthreads();
            const int width = cols * lanes * V::n;
            for (int c = threadIdx.x; c < width; c += 256) {
                const int at = blockIdx.y * width + c;
                if (at < a.C) {
                    float v = 0.f;
                    for (int r = 0; r < rows; ++r) v += red[r * width + c];
                    a.partial[((size_t)blockIdx.x * 2 + k) * a.C + at] = v;
                }
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------------------------------
// Images.  A CTA holds some rows of an image in shared memory (x, and dy in the backward pass), so that sums and values take one read.  Either a cluster of up to eight CTAs holds a whole image and exchanges its
// groups' sums through distributed shared memory (PHASE 0; it walks a list of images; every CTA
// writes its groups' results into all the others' inboxes, two in turn, so that one barrier an image is enough), or, for images larger than that,
// the CTAs' sums go to memory (PHASE 1), a small kernel joins them, and a second pass reads the image again (PHASE 2).
// A thread keeps a vector of channels and walks rows, with the channels' parameters and statistics in registers.
// In the backward pass act' dy replaces dy in shared memory, in fp32; with bf16 tensors act' is evaluated twice (kept in bf16 the
// product would carry a rounding as large as dx's own).
// 128x3136x64 bf16 with GELU, in pieces: sums 18 and values 31 us forward (the second read comes from L2: 9 of its 51 MB from memory),
// 36 and 42 backward (the second read comes from memory again: 100 of 103 MB), 130 with what joins them.  The schedulers issue in 54 to
// 64 % of the cycles and memory moves at 2.4 to 2.9 TB/s: neither is the bound, loads in flight at 16 warps an SM (backward) are too few.
// ------------------------------------------------------------------------------------------------
constexpr int kNormThreads = 256, kNormWarps = kNormThreads / 32;

template <typename io_t, int ACT, bool BWD, int PHASE>
__global__ void __launch_bounds__(kNormThreads, BWD ? 2 : 4) norm_image_kernel(const __grid_constant__ NormArgs a) {
    namespace cg = cooperative_groups;
    using V = Vec<io_t>;
    extern __shared__ uint4 tile[];                             // [rows][C] of x (and of dy), then the sums
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = PHASE == 0 ? a.pieces_n : 1, rank = PHASE == 0 ? (int)(blockIdx.x % ranks) : 0;
    const int cv = a.C / V::n, rp = kNormThreads / cv;          // vectors of a row, rows at once
    const int tid = threadIdx.x, col = tid % cv, row0 = tid / cv, c0 = col * V::n;
    const bool on = row0 < rp;
    constexpr bool kDirect = PHASE > 0;     // one pass over the tensors: from memory
    constexpr int kAhead = kDirect ? 4 : 2;
    const size_t slice = kDirect ? 0 : (size_t)a.rows * cv;
    uint4* const xs = tile;
    uint4* const gs = tile + slice;
    const float inv_per = 1.f / (float)a.per;
    const bool fold = cv < 32 && (cv & (cv - 1)) == 0;          // lanes that hold the same channels are summed in the warp
    const int parts = fold ? kNormWarps : rp;
    float* const red = reinterpret_cast<float*>(tile + slice * (BWD ? 2 : 1));      // [parts][C]
    float* const chan = red + (size_t)parts * a.C;                                  // [2][C]: of this image
    float* const sums = chan + 2 * a.C;                                             // [2][C]: dw, db of all images (backward)
    float2* const all = reinterpret_cast<float2*>(sums + (BWD ? 2 * a.C : 0));      // [groups]
    float2* const inbox = all + a.groups;                                           // [2][ranks][groups]
    int turn = 0;
    // (Short loops whose count only the launch knows are not unrolled: small images spend their time on fetching code that runs once,
    // 14x14x320 fp32 9.6 -> 8.5 us, 2000x36x64 bf16 27.4 -> 23.5.)
    // No CTA writes to another that has not begun: all arrive here, and wait for the rest behind the first image's requests.
    bool met = PHASE > 0 || ranks == 1;
    if (!met) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    auto meet = [&] {
        if (!met) asm volatile("barrier.cluster.wait;" ::: "memory");
        met = true;
    };
    auto send = [&](int g, float2 v) {                          // (one thread per group)
#pragma unroll 1
        for (int q = 0; q < ranks; ++q) (ranks > 1 ? cluster.map_shared_rank(inbox, q) : inbox)[(turn * ranks + rank) * a.groups + g] = v;
    };
    auto receive = [&] { if (ranks > 1) cluster.sync(); else __syncthreads(); };

    float2 w[V::pairs], bias[V::pairs];
#pragma unroll
    for (int i = 0; i < V::pairs; ++i) {
        w[i] = make_float2(norm_param<io_t>(a.weight, c0 + 2 * i, a.params_f32, 1.f), norm_param<io_t>(a.weight, c0 + 2 * i + 1, a.params_f32, 1.f));
        bias[i] = make_float2(norm_param<io_t>(a.bias, c0 + 2 * i, a.params_f32, 0.f), norm_param<io_t>(a.bias, c0 + 2 * i + 1, a.params_f32, 0.f));
    }
    let_follow();
    if (PHASE == 2) follow_wait();
    // chan[k][c] = sum over the threads of channel c
    auto channel_sums = [&](float2 (&v)[V::pairs], int k) {
        if (fold)
            for (int m = 16; m >= cv; m >>= 1)
#pragma unroll
                for (int i = 0; i < V::pairs; ++i) {
                    v[i].x += __shfl_xor_sync(0xffffffffu, v[i].x, m);
                    v[i].y += __shfl_xor_sync(0xffffffffu, v[i].y, m);
                }
        if (fold ? (tid & 31) < cv : on)
#pragma unroll
            for (int i = 0; i < V::pairs; ++i) *reinterpret_cast<float2*>(red + (size_t)(fold ? tid >> 5 : row0) * a.C + c0 + 2 * i) = v[i];
        __syncthreads();
        for (int c = tid; c < a.C; c += kNormThreads) {
            float s0 = 0.f, s1 = 0.f;
            int r = 0;
            for (; r + 1 < parts; r += 2) {
                s0 += red[r * a.C + c];
                s1 += red[(r + 1) * a.C + c];
            }
            if (r < parts) s0 += red[r * a.C + c];
            chan[k * a.C + c] = s0 + s1;
        }
        __syncthreads();
    };
    // a warp's sum over the channels of group g of value(c), in every lane
    auto over_group = [&](int g, auto value) {
        float v = 0.f;
#pragma unroll 1
        for (int c = g * a.per + (tid & 31); c < (g + 1) * a.per; c += 32) v += value(c);
#pragma unroll
        for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
        return v;
    };
    if (BWD) {
        for (int c = tid; c < 2 * a.C; c += kNormThreads) sums[c] = 0.f;
    }

    const long long lists = PHASE == 0 ? gridDim.x / ranks : gridDim.x / a.pieces_n;
    for (long long n = PHASE == 0 ? blockIdx.x / ranks : blockIdx.x / a.pieces_n; n < a.N; n += PHASE == 0 ? lists : a.N) {
        const int piece = PHASE == 0 ? rank : (int)(blockIdx.x % a.pieces_n);
        const long long s0 = (long long)piece * a.rows;
        const int rows = (int)max(0ll, min((long long)a.rows, a.S - s0));
        const auto rows_of = [&](int p) { return (float)max(0ll, min((long long)a.rows, a.S - (long long)p * a.rows)); };
        const size_t at = ((size_t)n * a.S + s0) * cv;
        const uint4* const xg = static_cast<const uint4*>(a.x) + at;
        const uint4* const dg = static_cast<const uint4*>(a.d_y) + at;
        if (!kDirect) {
            const unsigned xa = smem_u32(xs), ga = smem_u32(gs);
            for (int i = tid; i < rows * cv; i += kNormThreads) {
                cp_async16(xa + 16 * i, xg + i);
                if (BWD) cp_async16(ga + 16 * i, dg + i);
            }
            meet();
            cp_async_wait_all();
            __syncthreads();
        }
        auto x_at = [&](int i) { return kDirect ? __ldg(xg + i) : xs[i]; };
        auto g_at = [&](int i) { return kDirect ? __ldg(dg + i) : gs[i]; };
        const float count = (float)((double)a.S * a.per);
        // c / per, without a division: half a channel from the next whole number at least, of at most 2048
        auto group_of = [&](int c) { return (int)(((float)c + 0.5f) * inv_per); };
        if constexpr (!BWD) {
            float2 A[V::pairs], B[V::pairs];
            if constexpr (PHASE < 2) {
                // one pass: sums of x - p and its square, p the thread's own first value of the channel.  As p is one of the n
                // values, the sum of squares is at most n times what is left of it about their mean: no cancellation to speak of.
                float2 sum[V::pairs] = {}, sq[V::pairs] = {}, pivot[V::pairs] = {};
                float n_own = 0.f;
                if (on && row0 < rows) {
                    V v;
                    v.u = x_at(row0 * cv + col);
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i) pivot[i] = make_float2(-v.get(i).x, -v.get(i).y);
                    n_own = (float)((rows - row0 + rp - 1) / rp);
#pragma unroll kAhead
                    for (int r = row0 + rp; r < rows; r += rp) {
                        v.u = x_at(r * cv + col);
#pragma unroll
                        for (int i = 0; i < V::pairs; ++i) {
                            const float2 d = __fadd2_rn(v.get(i), pivot[i]);
                            sum[i] = __fadd2_rn(sum[i], d);
                            sq[i] = __ffma2_rn(d, d, sq[i]);
                        }
                    }
                }
                // sum -> that of x - base, base the group's first value in this CTA (of x itself, equal values far from zero gave a
                // mean some steps away from theirs); sq -> that about the thread's mean, which pivot becomes (negated)
                auto base = [&](int first) {
                    if (rows == 0) return 0.f;
                    if constexpr (kDirect) return load1(reinterpret_cast<const io_t*>(xg), first);
                    else if constexpr (sizeof(io_t) == 4) return reinterpret_cast<const float*>(xs)[first];
                    else return bf16_bits_to_float(reinterpret_cast<const unsigned short*>(xs)[first]);
                };
                const float each = n_own > 0.f ? 1.f / n_own : 0.f;
#pragma unroll
                for (int i = 0; i < V::pairs; ++i) {
                    const float2 d = __fmul2_rn(sum[i], make_float2(each, each));
                    sq[i] = __ffma2_rn(make_float2(-sum[i].x, -sum[i].y), d, sq[i]);      // (below zero by rounding, at most)
                    pivot[i] = make_float2(pivot[i].x - d.x, pivot[i].y - d.y);
                    sum[i] = __fmul2_rn(__fadd2_rn(pivot[i], make_float2(base(group_of(c0 + 2 * i) * a.per), base(group_of(c0 + 2 * i + 1) * a.per))), make_float2(-n_own, -n_own));
                }
                channel_sums(sum, 0);
                // this CTA's groups: mean, then sum of squares about it
                const float here = 1.f / fmaxf((float)rows * (float)a.per, 1.f);
                for (int g = tid >> 5; g < a.groups; g += kNormWarps) {
                    const float first = base(g * a.per), v = over_group(g, [&](int c) { return chan[c]; });
                    if ((tid & 31) == 0) all[g].x = fmaf(v, here, first);
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < V::pairs; ++i) {
                    const float2 d = make_float2(pivot[i].x + all[group_of(c0 + 2 * i)].x, pivot[i].y + all[group_of(c0 + 2 * i + 1)].x);
                    sum[i] = make_float2(fmaf(n_own * d.x, d.x, sq[i].x < 0.f ? 0.f : sq[i].x), fmaf(n_own * d.y, d.y, sq[i].y < 0.f ? 0.f : sq[i].y));
                }
                channel_sums(sum, 0);
                for (int g = tid >> 5; g < a.groups; g += kNormWarps) {
                    const float v = over_group(g, [&](int c) { return chan[c]; });
                    if ((tid & 31) == 0) {
                        const float2 own = make_float2(all[g].x, v);
                        if constexpr (PHASE == 1) a.pieces[((size_t)n * a.pieces_n + piece) * a.groups + g] = own;
                        else send(g, own);
                    }
                }
                if constexpr (PHASE == 1) return;
                receive();
                for (int g = tid; g < a.groups; g += kNormThreads) {
                    const float2* const in = inbox + (size_t)turn * ranks * a.groups + g;
                    float mean = 0.f, sq_all = 0.f;              // (about the first CTA's, for the same reason)
#pragma unroll 1
                    for (int q = 1; q < ranks; ++q) mean = fmaf(rows_of(q), in[q * a.groups].x - in[0].x, mean);
                    mean = in[0].x + mean / (float)a.S;
#pragma unroll 1
                    for (int q = 0; q < ranks; ++q) {
                        const float2 v = in[q * a.groups];
                        const float d = v.x - mean;
                        sq_all += rows_of(q) > 0.f ? fmaf(rows_of(q) * (float)a.per * d, d, v.y) : 0.f;
                    }
                    all[g] = make_float2(mean, rsqrtf(sq_all / count + a.eps));
                    if (a.stats && rank == 0) reinterpret_cast<float2*>(a.stats)[n * a.groups + g] = all[g];
                }
                __syncthreads();
            } else {
                for (int g = tid; g < a.groups; g += kNormThreads) all[g] = reinterpret_cast<const float2*>(a.stats)[n * a.groups + g];
                __syncthreads();
            }
            if (on) {
#pragma unroll
                for (int i = 0; i < V::pairs; ++i) {
                    const float2 g0 = all[group_of(c0 + 2 * i)], g1 = all[group_of(c0 + 2 * i + 1)];
                    A[i] = __fmul2_rn(make_float2(g0.y, g1.y), w[i]);
                    B[i] = make_float2(-g0.x, -g1.x);
                }
#pragma unroll kAhead
                for (int r = row0; r < rows; r += rp) {
                    V v, o;
                    v.u = x_at(r * cv + col);
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i) o.set(i, act_value2<ACT>(__ffma2_rn(__fadd2_rn(v.get(i), B[i]), A[i], bias[i])));
                    static_cast<uint4*>(a.y)[at + (size_t)r * cv + col] = o.u;
                }
            }
        } else {
            float2 mean[V::pairs], rstd[V::pairs];
#pragma unroll
            for (int i = 0; i < V::pairs; ++i) {
                const float2* const st = reinterpret_cast<const float2*>(a.stats) + n * a.groups;
                const float2 g0 = __ldg(st + group_of(min(c0 + 2 * i, a.C - 1))), g1 = __ldg(st + group_of(min(c0 + 2 * i + 1, a.C - 1)));
                mean[i] = make_float2(-g0.x, -g1.x);
                rstd[i] = make_float2(g0.y, g1.y);
            }
            constexpr bool kKeep = sizeof(io_t) == 4 && ACT != M2D_ACT_NONE && PHASE == 0;
            float2 sw[V::pairs] = {}, sb[V::pairs] = {};
            if (on && PHASE < 2)
#pragma unroll kAhead
                for (int r = row0; r < rows; r += rp) {
                    V v, g;
                    v.u = x_at(r * cv + col);
                    g.u = g_at(r * cv + col);
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i) {
                        const float2 h = __fmul2_rn(__fadd2_rn(v.get(i), mean[i]), rstd[i]);
                        const float2 dz = __fmul2_rn(g.get(i), act_slope2<ACT>(__ffma2_rn(h, w[i], bias[i])));
                        sw[i] = __ffma2_rn(dz, h, sw[i]);
                        sb[i] = __fadd2_rn(sb[i], dz);
                        if (kKeep) g.set(i, dz);
                    }
                    if (kKeep) gs[r * cv + col] = g.u;
                }
            if constexpr (PHASE == 1) {
                channel_sums(sw, 0);
                channel_sums(sb, 1);
                for (int i = tid; i < 2 * a.C; i += kNormThreads) a.partial[(size_t)blockIdx.x * 2 * a.C + i] = chan[i];
                return;
            }
            if constexpr (PHASE == 0) {
                channel_sums(sw, 0);
                channel_sums(sb, 1);
                for (int c = tid; c < 2 * a.C; c += kNormThreads) sums[c] += chan[c];
                for (int g = tid >> 5; g < a.groups; g += kNormWarps) {
                    const float v0 = over_group(g, [&](int c) { return norm_param<io_t>(a.weight, c, a.params_f32, 1.f) * chan[a.C + c]; });
                    const float v1 = over_group(g, [&](int c) { return norm_param<io_t>(a.weight, c, a.params_f32, 1.f) * chan[c]; });
                    if ((tid & 31) == 0) send(g, make_float2(v0, v1));
                }
                receive();
                for (int g = tid; g < a.groups; g += kNormThreads) {
                    const float2* const in = inbox + (size_t)turn * ranks * a.groups + g;
                    float2 v = make_float2(0.f, 0.f);
                    for (int q = 0; q < ranks; ++q) {
                        v.x += in[q * a.groups].x;
                        v.y += in[q * a.groups].y;
                    }
                    all[g] = make_float2(v.x / count, v.y / count);
                }
            } else {
                for (int g = tid; g < a.groups; g += kNormThreads) all[g] = a.group_sums[n * a.groups + g];
            }
            __syncthreads();
            if (on) {
                float2 m0[V::pairs], m1[V::pairs];
#pragma unroll
                for (int i = 0; i < V::pairs; ++i) {
                    const float2 g0 = all[group_of(c0 + 2 * i)], g1 = all[group_of(c0 + 2 * i + 1)];
                    m0[i] = make_float2(-g0.x, -g1.x);
                    m1[i] = make_float2(-g0.y, -g1.y);
                }
#pragma unroll kAhead
                for (int r = row0; r < rows; r += rp) {
                    V v, g, o;
                    v.u = x_at(r * cv + col);
                    g.u = g_at(r * cv + col);
#pragma unroll
                    for (int i = 0; i < V::pairs; ++i) {
                        const float2 h = __fmul2_rn(__fadd2_rn(v.get(i), mean[i]), rstd[i]);
                        float2 dz = g.get(i);
                        if (!kKeep) dz = __fmul2_rn(dz, act_slope2<ACT>(__ffma2_rn(h, w[i], bias[i])));
                        o.set(i, __fmul2_rn(rstd[i], __ffma2_rn(h, m1[i], __fadd2_rn(__fmul2_rn(dz, w[i]), m0[i]))));
                    }
                    static_cast<uint4*>(a.d_x)[at + (size_t)r * cv + col] = o.u;
                }
            }
        }
        __syncthreads();                                        // the tile is free again
        turn ^= 1;
    }
    meet();                                                     // (of a CTA without an image)
    if (PHASE == 0 && ranks > 1) cluster.sync();                // (no CTA leaves while another writes to it)
    if (BWD && PHASE == 0 && a.partial) {
        for (int i = tid; i < 2 * a.C; i += kNormThreads) a.partial[(size_t)blockIdx.x * 2 * a.C + i] = sums[i];
    }
}

// Images in pieces: (mean, sum of squares about it) of the pieces' groups -> (mean, rstd).  A warp per image and group.
__global__ void __launch_bounds__(256) norm_join_kernel(const NormArgs a) {
    let_follow();
    follow_wait();
    const long long at = blockIdx.x * 8ll + (threadIdx.x >> 5);
    if (at >= a.N * a.groups) return;
    const long long n = at / a.groups;
    const int g = (int)(at % a.groups), lane = threadIdx.x & 31;
    const double whole = (double)a.S * a.per;
    auto rows_of = [&](int p) { return (double)min((long long)a.rows, a.S - (long long)p * a.rows) * a.per; };
    double sum = 0.0, sq = 0.0;
    for (int p = lane; p < a.pieces_n; p += 32) sum += (double)a.pieces[((size_t)n * a.pieces_n + p) * a.groups + g].x * rows_of(p);
#pragma unroll
    for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const double mean = sum / whole;
    for (int p = lane; p < a.pieces_n; p += 32) {
        const float2 v = a.pieces[((size_t)n * a.pieces_n + p) * a.groups + g];
        const double d = (double)v.x - mean;
        sq += (double)v.y + d * d * rows_of(p);
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
    if (lane == 0) reinterpret_cast<float2*>(a.stats)[at] = make_float2((float)mean, rsqrtf((float)(sq / whole) + a.eps));
}
// Images in pieces, backward: the pieces' channel sums ([N][pieces][2][C], dz h and dz) -> means of dh and dh h.  A warp per image and group.
template <typename io_t>
__global__ void __launch_bounds__(256) norm_join_bwd_kernel(const NormArgs a) {
    let_follow();
    follow_wait();
    const long long at = blockIdx.x * 8ll + (threadIdx.x >> 5);
    if (at >= a.N * a.groups) return;
    const long long n = at / a.groups;
    const int g = (int)(at % a.groups), lane = threadIdx.x & 31;
    double s0 = 0.0, s1 = 0.0;
    for (int i = lane; i < a.pieces_n * a.per; i += 32) {
        const int p = i / a.per, c = g * a.per + i % a.per;
        const float w = norm_param<io_t>(a.weight, c, a.params_f32, 1.f);
        const float* const from = a.partial + ((size_t)n * a.pieces_n + p) * 2 * a.C + c;
        s1 += (double)(w * from[0]);
        s0 += (double)(w * from[a.C]);
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        s0 += __shfl_xor_sync(0xffffffffu, s0, m);
        s1 += __shfl_xor_sync(0xffffffffu, s1, m);
    }
    const double whole = (double)a.S * a.per;
    if (lane == 0) a.group_sums[at] = make_float2((float)(s0 / whole), (float)(s1 / whole));
}

// A thread's values of a group, every 256th: f(place in the image, channel of the group).  No divisions.
template <typename F>
__device__ __forceinline__ void walk_group(const NormArgs& a, F f) {
    const int rows = 256 / a.per, columns = 256 % a.per;
    int c = (int)threadIdx.x % a.per;
    for (long long r = (int)threadIdx.x / a.per; r < a.S;) {
        f(r * a.C + c, c);
        r += rows;
        c += columns;
        if (c >= a.per) {
            c -= a.per;
            ++r;
        }
    }
}
// Any shape: a CTA owns a group of an image and reads it three times (mean, variance about it, values).  One group per token, C = 320,
// 100352 tokens: 310 us forward, 520 ... 530 backward, fp32 or bf16; 128x3136x30 bf16 90 and 167 (floors 20 ... 39, 29 ... 59; 7 and 11).  A thread adds up a 256th of
// it one by one, without bound, so here and in the two kernels below that is done in 64 bits: in 32, values around 1000 left a mean
// off by 0.2 after 49000 terms.
template <typename io_t>
__global__ void __launch_bounds__(256) norm_fwd_any(const NormArgs a) {
    const long long n = blockIdx.x / a.groups, count = a.S * a.per;
    const int c0 = (int)(blockIdx.x % a.groups) * a.per;
    const io_t* const x = static_cast<const io_t*>(a.x) + n * a.S * a.C + c0;
    io_t* const y = static_cast<io_t*>(a.y) + n * a.S * a.C + c0;
    double2 v = make_double2(0.0, 0.0);
    walk_group(a, [&](long long at, int) { v.x += (double)load1(x, at); });
    const float mean = (float)(block_sum2(v).x / (double)count);
    v.x = 0.0;
    walk_group(a, [&](long long at, int) {
        const float d = load1(x, at) - mean;
        v.x += (double)(d * d);
    });
    const float rstd = rsqrtf((float)(block_sum2(v).x / (double)count) + a.eps);
    if (a.stats && threadIdx.x == 0) reinterpret_cast<float2*>(a.stats)[blockIdx.x] = make_float2(mean, rstd);
    walk_group(a, [&](long long at, int c) {
        const float z = fmaf((load1(x, at) - mean) * rstd, norm_param<io_t>(a.weight, c0 + c, a.params_f32, 1.f), norm_param<io_t>(a.bias, c0 + c, a.params_f32, 0.f));
        store1(y, at, act_value(z, a.act));
    });
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
    double2 v = make_double2(0.0, 0.0);
    float h, dh;
    for (long long i = threadIdx.x; i < count; i += 256) {
        at(i, h, dh);
        v.x += (double)dh;
        v.y += (double)(dh * h);
    }
    const double2 s = block_sum2(v);
    const float m0 = (float)(s.x / (double)count), m1 = (float)(s.y / (double)count);
    for (long long i = threadIdx.x; i < count; i += 256) {
        const long long o = at(i, h, dh);
        store1(dx, o, st.y * (dh - m0 - h * m1));
    }
}

// Sums over pixels and images for each channel: a CTA owns 32 channels of every gridDim.y-th row block.
template <typename io_t>
__global__ void __launch_bounds__(256) norm_wgrad_any(const NormArgs a) {
    __shared__ double2 part[8][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), row0 = threadIdx.x >> 5;
    double2 v = make_double2(0.0, 0.0);
    if (c < a.C) {
        const float w = norm_param<io_t>(a.weight, c, a.params_f32, 1.f), bias = norm_param<io_t>(a.bias, c, a.params_f32, 0.f);
        const int group = c / a.per;
        for (long long r = blockIdx.y * 8ll + row0; r < a.N * a.S; r += gridDim.y * 8ll) {
            const float2 st = reinterpret_cast<const float2*>(a.stats)[r / a.S * a.groups + group];
            const float h = (load1(static_cast<const io_t*>(a.x), r * a.C + c) - st.x) * st.y;
            const float dz = load1(static_cast<const io_t*>(a.d_y), r * a.C + c) * act_slope(fmaf(h, w, bias), a.act);
            v.x += (double)(dz * h);
            v.y += (double)dz;
        }
    }
    part[row0][threadIdx.x & 31] = v;
    __syncthreads();
    if (row0 == 0 && c < a.C) {
        for (int i = 1; i < 8; ++i) {
            v.x += part[i][threadIdx.x].x;
            v.y += part[i][threadIdx.x].y;
        }
        a.partial[(2ll * blockIdx.y) * a.C + c] = (float)v.x;
        a.partial[(2ll * blockIdx.y + 1) * a.C + c] = (float)v.y;
    }
}

// The sum of the splits' partial results, in order: [splits][2][C] -> d_weight, d_bias.  32 rows of splits a block, four reads of a
// thread under way at once.
constexpr int kSumRows = 32;
template <typename io_t>
__global__ void __launch_bounds__(32 * kSumRows) norm_wgrad_sum(const float* partial, int splits, int C, int f32, void* d_weight, void* d_bias) {
    follow_wait();
    __shared__ float part[kSumRows][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, i = blockIdx.x * 32 + lane;
    float v[4] = {};
    if (i < 2 * C)
        for (int s = row; s < splits; s += 4 * kSumRows)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (s + j * kSumRows < splits) v[j] += partial[(size_t)(s + j * kSumRows) * 2 * C + i];
    part[row][lane] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    float sum = part[lane][row];                        // (warp `row` adds column `row` up)
#pragma unroll
    for (int m = 16; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const int o = blockIdx.x * 32 + row;
    if (lane == 0 && o < 2 * C) {
        void* to = o < C ? d_weight : d_bias;
        const int c = o < C ? o : o - C;
        if (f32) static_cast<float*>(to)[c] = sum;
        else store1(static_cast<io_t*>(to), c, sum);
    }
}

static int check_norm(const m2d_norm_desc* d) {
    if (!d) return M2D_ERR_NULL;
    if (d->struct_bytes != sizeof(m2d_norm_desc)) return M2D_ERR_ABI;
    if (d->dtype != M2D_F32 && d->dtype != M2D_BF16) return M2D_ERR_DTYPE;
    if (d->act < M2D_ACT_NONE || d->act > M2D_ACT_GELU) return M2D_ERR_FLAGS;
    if (d->N < 1 || d->S < 1 || d->C < 1 || d->groups < 1 || d->C % d->groups) return M2D_ERR_SHAPE;
    if (d->C > (1 << 29) || d->N > (1ll << 40) || d->S > (1ll << 40) || d->N * d->groups >= (1ll << 31)) return M2D_ERR_TOO_LARGE;
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

struct NormPlan {
    enum { kAny, kRows, kImage, kPieces } kind = kAny;
    int lanes = 0, cols = 0;              // kRows
    int rows = 0, pieces = 1, grid = 1;   // rows of a CTA, CTAs of an image, CTAs (kRows: blocks along the rows)
    int grid_y = 1;
    size_t smem = 0;
    size_t partial = 0;                   // CTAs that write sums of the parameters' gradients
};
static size_t image_smem(const m2d_norm_desc* d, bool bwd, long long rows, int ranks = 1) {
    const int es = d->dtype == M2D_F32 ? 4 : 2, cv = d->C * es / 16, parts = cv < 32 && (cv & (cv - 1)) == 0 ? kNormWarps : kNormThreads / cv;
    return (size_t)rows * d->C * es * (bwd ? 2 : 1) + sizeof(float) * ((size_t)parts * d->C + (bwd ? 4 : 2) * d->C) + sizeof(float2) * (1 + 2 * ranks) * d->groups;
}
static NormPlan plan_norm(const m2d_norm_desc* d, bool bwd) {
    NormPlan p;
    const int es = d->dtype == M2D_F32 ? 4 : 2, v = 16 / es, per = d->C / d->groups;
    p.partial = wgrad_splits(d);
    if (d->C % v) return p;
    const int cv = d->C / v;
    if (d->S == 1) {
        const int lanes = per / v;
        if (per % v || lanes < 1 || lanes > 32) return p;
        const int slots = 8 * (32 / lanes);              // groups of a block
        p.cols = std::min(d->groups, slots);
        p.grid_y = (d->groups + p.cols - 1) / p.cols;
        if (p.grid_y > 65535) return p;                  // (not a grid)
        p.kind = NormPlan::kRows;
        p.lanes = lanes;
        const long long rows = slots / p.cols, steps = (d->N + rows - 1) / rows;
        // as many blocks as run at once; few rows: a block for each of its steps
        p.grid = (int)std::max<long long>(1, std::min<long long>(steps, (bwd ? 2ll : 4ll) * sm_count() / p.grid_y));
        p.smem = bwd ? (size_t)rows * p.cols * lanes * v * sizeof(float) : 0;
        p.partial = p.grid;
        return p;
    }
    if (cv > kNormThreads || image_smem(d, bwd, 1) > kMaxSmem) return p;
    // CTAs of an image: as few as leave room for four (backward two) on an SM, more where there are few images, none with less
    // than 16 rows
    const int per_sm = bwd ? 2 : 4;
    const size_t room = kMaxSmem / per_sm - 1024;
    int ranks = 1;
    while (ranks < 8 && (image_smem(d, bwd, (d->S + ranks - 1) / ranks, ranks) > room || (d->N * ranks < sm_count() && d->S / (2 * ranks) >= 16))) ranks *= 2;
    p.rows = (int)std::min<long long>(1 << 30, (d->S + ranks - 1) / ranks);
    p.pieces = ranks;
    p.smem = image_smem(d, bwd, (d->S + ranks - 1) / ranks, ranks);
    // A cluster holds an image, one launch, where all images' clusters run at once or an image needs one CTA only; not where a few
    // clusters would be all that works.  us, cluster / pieces, forward: 128x784x128 bf16 (one round) 20 / 24, fp32 (two) 39 / 27,
    // 512x64x512 fp32 64 / 47, 128x3136x64 bf16 52 / 50 (with the backward 171 / 131), 16x3136x96 fp32 (150 KB a CTA) 27 / 19,
    // 2000x36x64 bf16 (one CTA an image) 24 / 38, 32x3136x64 fp32 14 / 18.
    const int fit = std::max<int>(1, std::min<int>(per_sm, (int)((kMaxSmem + 1024) / (p.smem + 1024))));
    if (p.smem <= kMaxSmem / 2 && (ranks == 1 || d->N * ranks <= (long long)fit * sm_count()) &&
        (d->N * ranks >= sm_count() / 2 || (long long)d->S * d->C * es <= 512 * 1024)) {
        p.kind = NormPlan::kImage;
        p.grid = ranks * (int)std::max<long long>(1, std::min<long long>(d->N, (long long)fit * sm_count() / ranks));
        p.partial = p.grid;
        return p;
    }
    // pieces: as many as run at once, of 16 rows and 4 KB at least; they are not staged
    p.kind = NormPlan::kPieces;
    const long long slots = (long long)per_sm * sm_count(), least = std::max<long long>(16, 4096 / ((long long)d->C * es));
    const long long rows = std::max<long long>(least, (d->S + std::max<long long>(1, slots / d->N) - 1) / std::max<long long>(1, slots / d->N));
    p.rows = (int)std::min<long long>({rows, d->S, 1ll << 30});
    const long long pieces = (d->S + p.rows - 1) / p.rows;
    if (pieces * d->N >= (1ll << 30) || (long long)p.rows * cv >= (1ll << 31) || image_smem(d, bwd, 0) > kMaxSmem) { p.kind = NormPlan::kAny; return p; }
    p.pieces = (int)pieces;
    p.grid = (int)(pieces * d->N);
    p.smem = image_smem(d, bwd, 0);
    p.partial = p.grid;
    return p;
}
// Scratch: partial sums of the parameters' gradients; in pieces also the groups' statistics or sums.
struct NormScratch {
    size_t partial = 0, pieces = 0, stats = 0, bytes = 0;
    NormScratch(const m2d_norm_desc* d, const NormPlan& p, bool bwd) {
        auto take = [&](size_t n) {
            const size_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        const bool split = p.kind == NormPlan::kPieces;
        if (bwd && (d->d_weight || split)) partial = take(p.partial * 2 * d->C * sizeof(float));
        if (split) pieces = take(sizeof(float2) * d->N * d->groups * (bwd ? 1 : p.pieces));
        if (split && !bwd) stats = take(sizeof(float2) * d->N * d->groups);
    }
};

template <typename io_t, int ACT, bool BWD, int PHASE>
static int launch_image(const NormArgs& a, const NormPlan& p, cudaStream_t st) {
    auto kern = norm_image_kernel<io_t, ACT, BWD, PHASE>;
    if (!allow_smem(reinterpret_cast<const void*>(kern), p.smem)) return M2D_ERR_LAUNCH;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(p.grid);
    c.blockDim = dim3(kNormThreads);
    c.dynamicSmemBytes = p.smem;
    c.stream = st;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = PHASE == 0 ? p.pieces : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = attr;
    c.numAttrs = PHASE == 2 ? 2 : 1;
    return cudaLaunchKernelEx(&c, kern, a) == cudaSuccess ? M2D_OK : (cudaGetLastError(), M2D_ERR_LAUNCH);
}
template <typename io_t, int ACT, bool BWD>
static int launch_norm(NormArgs a, const NormPlan& p, cudaStream_t st) {
    if (p.kind == NormPlan::kRows) {
        norm_rows_kernel<io_t, ACT, BWD><<<dim3(p.grid, p.grid_y), 256, p.smem, st>>>(a, p.lanes, p.cols);
        return M2D_OK;
    }
    if (p.kind == NormPlan::kImage) return launch_image<io_t, ACT, BWD, 0>(a, p, st);
    if (p.kind == NormPlan::kPieces) {
        int rc = launch_image<io_t, ACT, BWD, 1>(a, p, st);
        if (rc != M2D_OK) return rc;
        const unsigned grid = (unsigned)((a.N * a.groups + 7) / 8);
        if (!launch_following(BWD ? norm_join_bwd_kernel<io_t> : norm_join_kernel, dim3(grid), dim3(256), 0, st, a)) return M2D_ERR_LAUNCH;
        return launch_image<io_t, ACT, BWD, 2>(a, p, st);
    }
    const unsigned grid = (unsigned)(a.N * a.groups);
    if (!BWD) {
        norm_fwd_any<io_t><<<grid, 256, 0, st>>>(a);
    } else {
        norm_bwd_any<io_t><<<grid, 256, 0, st>>>(a);
        if (a.partial) norm_wgrad_any<io_t><<<dim3((a.C + 31) / 32, (unsigned)p.partial), 256, 0, st>>>(a);
    }
    return M2D_OK;
}
template <bool BWD>
static int launch_norm(const m2d_norm_desc* d, const NormArgs& a, const NormPlan& p, cudaStream_t st) {
    const bool f32 = d->dtype == M2D_F32;
    if (d->act == M2D_ACT_SILU) return f32 ? launch_norm<float, M2D_ACT_SILU, BWD>(a, p, st) : launch_norm<__nv_bfloat16, M2D_ACT_SILU, BWD>(a, p, st);
    if (d->act == M2D_ACT_GELU) return f32 ? launch_norm<float, M2D_ACT_GELU, BWD>(a, p, st) : launch_norm<__nv_bfloat16, M2D_ACT_GELU, BWD>(a, p, st);
    return f32 ? launch_norm<float, M2D_ACT_NONE, BWD>(a, p, st) : launch_norm<__nv_bfloat16, M2D_ACT_NONE, BWD>(a, p, st);
}
static bool norm_aligned(const m2d_norm_desc* d, bool bwd) {
    auto ok = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    return ok(d->x) && (bwd ? ok(d->d_y) && ok(d->d_x) : ok(d->y));
}
// What either kind of kernel may need: a query does not depend on the tensors' addresses.
static size_t norm_scratch(const m2d_norm_desc* d, bool bwd) {
    NormPlan any;
    any.partial = wgrad_splits(d);
    return std::max(NormScratch(d, plan_norm(d, bwd), bwd).bytes, NormScratch(d, any, bwd).bytes);
}

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_norm_fwd_workspace(const m2d_norm_desc* d) { return check_norm(d) == M2D_OK ? norm_scratch(d, false) : 0; }
extern "C" uint64_t m2d_norm_bwd_workspace(const m2d_norm_desc* d) { return check_norm(d) == M2D_OK ? norm_scratch(d, true) : 0; }

static NormPlan plan_call(const m2d_norm_desc* d, bool bwd, NormArgs* a) {
    NormPlan p;
    p.partial = wgrad_splits(d);
    if (norm_aligned(d, bwd)) p = plan_norm(d, bwd);
    const NormScratch at(d, p, bwd);
    char* const ws = static_cast<char*>(d->workspace);
    *a = norm_args(d);
    a->rows = p.rows; a->pieces_n = p.pieces;
    const bool split = p.kind == NormPlan::kPieces;
    if (bwd && (d->d_weight || split)) a->partial = reinterpret_cast<float*>(ws + at.partial);
    if (split && bwd) a->group_sums = reinterpret_cast<float2*>(ws + at.pieces);
    if (split && !bwd) {
        a->pieces = reinterpret_cast<float2*>(ws + at.pieces);
        if (!a->stats) a->stats = reinterpret_cast<float*>(ws + at.stats);
    }
    return p;
}

extern "C" int m2d_norm_fwd(const m2d_norm_desc* d, void* stream) {
    int rc = check_norm(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->y) return M2D_ERR_NULL;
    if ((rc = norm_workspace_ok(d, m2d_norm_fwd_workspace(d))) != M2D_OK) return rc;
    NormArgs a;
    const NormPlan p = plan_call(d, false, &a);
    if ((rc = launch_norm<false>(d, a, p, static_cast<cudaStream_t>(stream))) != M2D_OK) return rc;
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}

extern "C" int m2d_norm_bwd(const m2d_norm_desc* d, void* stream) {
    int rc = check_norm(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->d_y || !d->d_x || !d->stats || !d->d_weight != !d->d_bias) return M2D_ERR_NULL;
    if ((rc = norm_workspace_ok(d, m2d_norm_bwd_workspace(d))) != M2D_OK) return rc;
    NormArgs a;
    const NormPlan p = plan_call(d, true, &a);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if ((rc = launch_norm<true>(d, a, p, st)) != M2D_OK) return rc;
    if (d->d_weight) {
        const unsigned grid = (2 * d->C + 31) / 32;
        const bool f32 = d->dtype == M2D_F32;
        if (!launch_following(f32 ? norm_wgrad_sum<float> : norm_wgrad_sum<__nv_bfloat16>, dim3(grid), dim3(32 * kSumRows), 0, st, (const float*)a.partial, (int)p.partial, d->C,
                              f32 ? 1 : d->params_f32, d->d_weight, d->d_bias))
            return M2D_ERR_LAUNCH;
    }
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}
