// Linear attention: entry points, and the kernels for any head size, type and alignment (attn_tc.cuh has the tcgen05 form).
#include <climits>

#include "attn_core.cuh"
#include "attn_tc.cuh"
#include "follow.cuh"
#include "launch.cuh"
#include "packed.cuh"

namespace m2d {

// ------------------------------------------------------------------------------------------------
// attn_core.cuh's computation on chunks of 64 tokens.  A CTA owns a sequence's head, VT columns of z and of the
// state, and one segment of the tokens; its products run on mma.sync in tf32, every operand split into two tf32 parts
// and three products per term, which leaves an error of about 2^-21 (operands in bf16 are exact in one part).
//
// What bounds it: at 6x1395x3x64 fp32 (training, 129 us) two CTAs on an SM issue in 39 % of their cycles, a third of that for the
// operands' splitting, and the longest sequences' CTAs end last; at 196 tokens (16 us) two launches of one chunk each.  64 tokens and
// 64 columns: larger tiles leave one CTA on an SM.
// ------------------------------------------------------------------------------------------------
constexpr int kC = 64, kAttnThreads = 256, kPStride = kC + 4;

__device__ __forceinline__ void mma_tf32(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// v = hi + lo exactly; hi is v rounded to tf32's 11 bits, of lo the first 11 are read (its sign varies: no bias)
struct Split {
    unsigned hi, lo;
    __device__ __forceinline__ Split(float v) {
        hi = (__float_as_uint(v) + 0x1000u) & 0xffffe000u;
        lo = __float_as_uint(v - __uint_as_float(hi));
    }
};
// acc[n] += A (16 x 8) B_n (8 x 8) over steps of 8 in [from, to), n < NT; fa(kk, i): the four values of A's fragment, fb(kk, n, i):
// the two of B's.  (The unit cuts off what it adds to an accumulator: the small products have one of their own, which leaves the large
// ones a third of the steps.  One of the three products for all n before the next: those of one accumulator wait for one another.)
// A1, B1: A's or B's values are bf16, exact in one part; the products with its second one are left out.
template <int NT, bool A1, bool B1, typename FA, typename FB>
__device__ __forceinline__ void mma_chain(float (&acc)[NT][4], int from, int to, FA fa, FB fb) {
    float low[NT][4] = {};
#pragma unroll 2
    for (int kk = from; kk < to; kk += 8) {
        unsigned ah[4], al[4], bh[NT][2], bl[NT][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (A1) {
                ah[i] = __float_as_uint(fa(kk, i));
            } else {
                const Split s(fa(kk, i));
                ah[i] = s.hi; al[i] = s.lo;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (B1) {
                    bh[n][i] = __float_as_uint(fb(kk, n, i));
                } else {
                    const Split s(fb(kk, n, i));
                    bh[n][i] = s.hi; bl[n][i] = s.lo;
                }
            }
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if constexpr (!B1) mma_tf32(low[n], ah, bl[n][0], bl[n][1]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_tf32(acc[n], ah, bh[n][0], bh[n][1]);
#pragma unroll
        for (int n = 0; n < NT; ++n)
            if constexpr (!A1) mma_tf32(low[n], al, bh[n][0], bh[n][1]);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] += low[n][i];
}

// rows [0, 64) x cols [0, width) of a tile, zero behind `valid` rows and `n` columns.  fp32 goes straight to shared memory (the caller
// waits for it); of bf16 four pieces a thread are under way at once.
template <typename io_t>
__device__ __forceinline__ void load_rows(float* dst, int stride, const io_t* src, long long st, int valid, int n, int width, int vec) {
    const int r = threadIdx.x >> 2, c0 = (threadIdx.x & 3) * 4;      // four threads a row (no division: it took a third of this)
    const io_t* const p = src + (long long)r * st;
    float* const to = dst + r * stride;
    static_assert(kAttnThreads == 4 * kC, "rows of a tile");
#pragma unroll 4
    for (int c = c0; c < width; c += 16) {
        if (r < valid && vec && c + 4 <= n) {
            if constexpr (sizeof(io_t) == 4) {
                cp_async16(smem_u32(to + c), p + c);
            } else {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(p + c));
                *reinterpret_cast<float4*>(to + c) =
                    make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
            }
        } else {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < valid) {
                if (c < n) v.x = load1(p, c);
                if (c + 1 < n) v.y = load1(p, c + 1);
                if (c + 2 < n) v.z = load1(p, c + 2);
                if (c + 3 < n) v.w = load1(p, c + 3);
            }
            *reinterpret_cast<float4*>(to + c) = v;
        }
    }
}

__host__ __device__ inline int attn_pad(int d) { return (d + 15) / 16 * 16; }
inline size_t attn_smem(int Kd, int VT) {
    const int kd = attn_pad(Kd);
    return sizeof(float) * ((size_t)2 * kC * (kd + 4) + (size_t)(kC + kd) * (VT + 8) + (size_t)kC * kPStride + 7 * kC);
}

template <typename io_t, int VT, bool STATE_ONLY>
__global__ void __launch_bounds__(kAttnThreads) attn_core_kernel(const __grid_constant__ AttnLaunch a) {
    const AttnCore& k = a.core[blockIdx.z];
    const int v0 = blockIdx.y * VT;
    if (v0 >= k.Vd) return;
    extern __shared__ float4 smem4[];
    const int kd = attn_pad(k.Kd), ks = kd + 4;
    constexpr int VS = VT + 8, NT = VT / 16;
    constexpr bool kOne = sizeof(io_t) == 2;
    float* X = reinterpret_cast<float*>(smem4);
    float* Y = X + kC * ks;
    float* Z = Y + kC * ks;
    float* S = Z + kC * VS;
    float* P = S + kd * VS;
    float* c_hi = P + kC * kPStride;
    float *c_lo = c_hi + kC, *w = c_lo + kC, *u = w + kC, *dot = u + kC, *whole = dot + 2 * kC;

    const int seg = blockIdx.x % a.nseg, bh = blockIdx.x / a.nseg, h = bh % a.H, b = bh / a.H;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
    const int wm = (warp & 3) * 16, wn = (warp >> 2) * (VT / 2);
    const int len = attn_length(a, b), t_lo = seg * a.seg_len, t_hi = t_lo + min(a.seg_len, a.T - t_lo);      // (t_lo + seg_len may lie beyond 2^31)
    const bool pairs = k.Vd % 2 == 0 && (reinterpret_cast<uintptr_t>(k.out) & 7) == 0;      // out may be written two columns at a time
    const int nv = min(VT, k.Vd - v0), chunks = (t_hi - t_lo + kC - 1) / kC;
    const io_t* const x = static_cast<const io_t*>(attn_at(k.x, b, h, sizeof(io_t)));
    const io_t* const y = static_cast<const io_t*>(attn_at(k.y, b, h, sizeof(io_t)));
    const io_t* const z = static_cast<const io_t*>(attn_at(k.z, b, h, sizeof(io_t))) + v0;
    const float* const g = a.g + (long long)b * a.gb + (long long)h * a.gh;

    // The state before the segment, where it is needed first: until then this launch may run beside the one over the segments' own
    // states.  A few segments are joined here, else attn_join_kernel has done it.
    bool begun = false;
    auto begin = [&] {
        if (begun) return;
        begun = true;
        const float* init = k.init.p ? k.init.p + b * k.init.sb + h * k.init.sh : nullptr;
        long long sr = k.init.sr, sc = k.init.sc;
        if (!STATE_ONLY) follow_wait();
        if (!STATE_ONLY && a.nseg > 1 && !a.join_here) {
            init = k.seg_state + ((size_t)bh * a.nseg + seg) * k.Kd * k.Vd;
            sr = k.Vd; sc = 1;
        }
        for (int i = tid; i < kd * VT; i += kAttnThreads) {
            const int r = i / VT, c = i % VT;
            S[r * VS + c] = !STATE_ONLY && init && r < k.Kd && c < nv ? init[r * sr + (v0 + c) * sc] : 0.f;
        }
        if (!STATE_ONLY && a.join_here)
            for (int j = k.rev ? a.nseg - 1 : 0; j != seg; j += k.rev ? -1 : 1) {
                const size_t at = (size_t)bh * a.nseg + j;
                const float decay = ex2(k.seg_decay[at]);
                const float* own = k.seg_state + at * k.Kd * k.Vd + v0;
#pragma unroll 8
                for (int i = tid; i < k.Kd * VT; i += kAttnThreads) {
                    const int r = i / VT, c = i % VT;
                    if (c < nv) S[r * VS + c] = fmaf(S[r * VS + c], decay, own[(size_t)r * k.Vd + c]);
                }
            }
    };
    if (STATE_ONLY) begin();
    let_follow();
    const bool last_wanted = STATE_ONLY || (k.fin.p && seg == (k.rev ? 0 : a.nseg - 1));
    double total = 0.0;

    for (int it = 0; it < chunks; ++it) {
        const int t0 = t_lo + (k.rev ? chunks - 1 - it : it) * kC;
        const int rows = min(kC, t_hi - t0), valid = max(0, min(rows, len - t0));
        const bool run_end = !STATE_ONLY && k.anchors && ((t0 + kC) % kAnchor == 0 || t0 + kC >= a.T);
        auto keep_state = [&] {
            float* to = k.anchors + ((size_t)bh * a.runs + t0 / kAnchor) * k.Kd * k.Vd + v0;
            for (int i = tid; i < k.Kd * VT; i += kAttnThreads) {
                const int r = i / VT, c = i % VT;
                if (c < nv) to[(size_t)r * k.Vd + c] = S[r * VS + c];
            }
        };
        __syncthreads();
        if (run_end && k.rev) {
            begin();
            __syncthreads();
            keep_state();
        }
        if (valid == 0) {
            if (!STATE_ONLY) {
                for (int i = tid; i < rows * nv; i += kAttnThreads) {
                    const long long at = b * k.ob + (long long)(t0 + i / nv) * k.ot + h * k.oh + v0 + i % nv;
                    if (k.out_f32) static_cast<float*>(k.out)[at] = 0.f;
                    else store1(static_cast<io_t*>(k.out), at, 0.f);
                }
                if (k.dots && tid < rows) k.dots[(((size_t)blockIdx.y * a.B + b) * a.T + t0 + tid) * a.H + h] = 0.f;
                if (run_end && !k.rev) {
                    begin();
                    __syncthreads();
                    keep_state();
                }
            }
            continue;
        }
        float g2[2] = {0.f, 0.f};
        if (warp == 0) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (2 * lane + j < valid) g2[j] = __ldg(g + (long long)(t0 + 2 * lane + j) * a.gt);
        }
        if (!STATE_ONLY) load_rows(X, ks, x + (long long)t0 * k.x.st, k.x.st, valid, k.Kd, kd, k.x.vec);
        load_rows(Y, ks, y + (long long)t0 * k.y.st, k.y.st, valid, k.Kd, kd, k.y.vec);
        load_rows(Z, VS, z + (long long)t0 * k.z.st, k.z.st, valid, nv, VT, k.z.vec);
        if (warp == 0) {
            double d[2], up;
#pragma unroll
            for (int j = 0; j < 2; ++j) d[j] = attn_decay(g2[j]);
            up = d[0] + d[1];
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, up, s);
                if (lane >= s) up += o;
            }
            const double end = __shfl_sync(0xffffffffu, up, 31);
            d[0] = up - d[1];      // inclusive sums of the lane's two tokens
            d[1] = up;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int t = 2 * lane + j;
                const float hi = (float)d[j];
                c_hi[t] = hi;
                c_lo[t] = (float)(d[j] - hi);
                const float from_start = ex2((float)d[j]), to_end = ex2((float)(end - d[j]));
                w[t] = k.rev ? to_end : from_start;
                u[t] = (k.rev ? from_start : to_end) * k.s_update;
            }
            if (lane == 0) *whole = ex2((float)end);
            total += end;
        }
        if (sizeof(io_t) == 4) cp_async_wait_all();
        __syncthreads();

        if (!STATE_ONLY) {
            // P = s_intra D (X Y^T), 16 rows x 32 columns a warp
            const int pn = (warp >> 2) * 32;
            float acc[4][4] = {};
            if (k.rev ? pn + 31 >= wm : pn <= wm + 15)
                mma_chain<4, kOne, kOne>(acc, 0, kd, [&](int kk, int i) { return X[(wm + gq + (i & 1) * 8) * ks + kk + tq + (i >> 1) * 4]; },
                             [&](int kk, int n, int i) { return Y[(pn + n * 8 + gq) * ks + kk + tq + i * 4]; });
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = wm + gq + (i >> 1) * 8, c = pn + n * 8 + tq * 2 + (i & 1);
                    const float d = (c_hi[r] - c_hi[c]) + (c_lo[r] - c_lo[c]);
                    const bool on = (k.rev ? c >= r : c <= r) && c < valid && r < valid;
                    P[r * kPStride + c] = on ? k.s_intra * ex2(k.rev ? -d : d) * acc[n][i] : 0.f;
                }
            begin();
            __syncthreads();
            // out, 16 rows x VT / 2 columns a warp
            float o1[NT][4] = {}, o2[NT][4] = {};
            mma_chain<NT, false, kOne>(o1, k.rev ? wm : 0, k.rev ? kC : wm + 16, [&](int kk, int i) { return P[(wm + gq + (i & 1) * 8) * kPStride + kk + tq + (i >> 1) * 4]; },
                          [&](int kk, int n, int i) { return Z[(kk + tq + i * 4) * VS + wn + n * 8 + gq]; });
            mma_chain<NT, kOne, false>(o2, 0, kd, [&](int kk, int i) { return X[(wm + gq + (i & 1) * 8) * ks + kk + tq + (i >> 1) * 4]; },
                          [&](int kk, int n, int i) { return S[(kk + tq + i * 4) * VS + wn + n * 8 + gq]; });
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int r = wm + gq + half * 8;
                const float wr = k.s_inter * w[r];
                const long long row = b * k.ob + (long long)(t0 + r) * k.ot + h * k.oh + v0;
                const io_t* e = k.dots ? static_cast<const io_t*>(attn_at(k.e, b, h, sizeof(io_t))) + (long long)(t0 + r) * k.e.st + v0 : nullptr;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int c = wn + n * 8 + tq * 2;
                    const float a0 = r < valid ? fmaf(wr, o2[n][half * 2], o1[n][half * 2]) : 0.f, a1 = r < valid ? fmaf(wr, o2[n][half * 2 + 1], o1[n][half * 2 + 1]) : 0.f;
                    if (r < rows && c < nv) {
                        if (pairs) {
                            if (sizeof(io_t) == 4 || k.out_f32) *reinterpret_cast<float2*>(static_cast<float*>(k.out) + row + c) = make_float2(a0, a1);
                            else *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(k.out) + row + c) = pack_bf16x2(a0, a1);
                        } else {
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                if (c + i < nv) {
                                    if (k.out_f32) static_cast<float*>(k.out)[row + c + i] = i ? a1 : a0;
                                    else store1(static_cast<io_t*>(k.out), row + c + i, i ? a1 : a0);
                                }
                        }
                        if (e && r < valid) {
                            sum = fmaf(a0, load1(e, c), sum);
                            if (c + 1 < nv) sum = fmaf(a1, load1(e, c + 1), sum);
                        }
                    }
                }
                if (k.dots) {
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    if (tq == 0) dot[(warp >> 2) * kC + r] = sum;
                }
            }
            __syncthreads();
            if (k.dots && tid < rows) k.dots[(((size_t)blockIdx.y * a.B + b) * a.T + t0 + tid) * a.H + h] = dot[tid] + dot[kC + tid];
        }
        // state: 16 rows x VT / 2 columns at a time (after a segment's last chunk only where somebody takes it)
        const float decay = *whole;
        for (int m = (warp & 3) * 16; m < kd && (it + 1 < chunks || last_wanted || run_end); m += 64) {
            float acc[NT][4] = {};
            mma_chain<NT, false, kOne>(acc, 0, kC,
                          [&](int kk, int i) {
                              const int c = kk + tq + (i >> 1) * 4;
                              return Y[c * ks + m + gq + (i & 1) * 8] * u[c];
                          },
                          [&](int kk, int n, int i) { return Z[(kk + tq + i * 4) * VS + wn + n * 8 + gq]; });
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float& s = S[(m + gq + (i >> 1) * 8) * VS + wn + n * 8 + tq * 2 + (i & 1)];
                    s = fmaf(s, decay, acc[n][i]);
                }
        }
        if (run_end && !k.rev) {
            __syncthreads();
            keep_state();
        }
    }
    begin();
    __syncthreads();
    float* fin = nullptr;
    long long sr = k.fin.sr, sc = k.fin.sc;
    if (STATE_ONLY) {
        fin = k.seg_state + ((size_t)bh * a.nseg + seg) * k.Kd * k.Vd;
        sr = k.Vd; sc = 1;
        if (tid == 0 && v0 == 0) k.seg_decay[(size_t)bh * a.nseg + seg] = (float)total;
    } else if (k.fin.p && seg == (k.rev ? 0 : a.nseg - 1)) {
        fin = k.fin.p + b * k.fin.sb + h * k.fin.sh;
    }
    if (fin)
        for (int i = tid; i < k.Kd * VT; i += kAttnThreads) {
            const int r = i / VT, c = i % VT;
            if (c < nv) fin[r * sr + (v0 + c) * sc] = S[r * VS + c];
        }
}

// The segments' own states become the states that they start from.  A thread has one element of the states; the reads of
// eight segments are under way at once (one by one, their latency was 50 us for 16 segments).
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnLaunch a) {
    const AttnCore& k = a.core[blockIdx.z];
    const int bh = blockIdx.x, h = bh % a.H, b = bh / a.H, n = k.Kd * k.Vd;
    const int i = blockIdx.y * 128 + threadIdx.x;
    let_follow();
    if (i >= n) return;
    const int row = a.seg_columns ? i % k.Kd : i / k.Vd, col = a.seg_columns ? i / k.Kd : i % k.Vd;
    float carry = k.init.p ? k.init.p[b * k.init.sb + h * k.init.sh + row * k.init.sr + col * k.init.sc] : 0.f;
    for (int j0 = 0; j0 < a.nseg; j0 += 8) {
        float own[8], decay[8];
        auto at = [&](int j) { return (size_t)bh * a.nseg + (k.rev ? a.nseg - 1 - j : j); };
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j0 + j < a.nseg) {
                own[j] = k.seg_state[at(j0 + j) * n + i];
                decay[j] = k.seg_decay[at(j0 + j)];
            }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j0 + j < a.nseg) {
                k.seg_state[at(j0 + j) * n + i] = carry;
                carry = fmaf(carry, ex2(decay[j]), own[j]);
            }
    }
}

// The decay's gradient from the dots and the anchors: suffix sums over a run, and <S, R> of its two kept states (n elements each), which
// is what it reads: 71 MB at 8x2048x16x128, 18 us (a launch of its own for <S, R>: 16 and 7 us).
// Dots: [blocks][B][T][H], one of dq and one of dk.
__global__ void __launch_bounds__(kAnchor) attn_decay_kernel(const float* rq, const float* rk, int blocks, const float* anchor_s, const float* anchor_r, int n,
                                                             const int* __restrict__ lengths, float* dg, int B, int T, int H, int runs) {
    __shared__ double part[kAnchor / 32], whole[kAnchor / 32];
    const int run = blockIdx.x % runs, bh = blockIdx.x / runs, h = bh % H, b = bh / H;
    const int t = run * kAnchor + (kAnchor - 1 - threadIdx.x), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;      // from the last token on
    const float *const s = anchor_s + (size_t)blockIdx.x * n, *const r = anchor_r + (size_t)blockIdx.x * n;
    float e = 0.f;
    let_follow();
    follow_wait();
    if (n % 4 == 0) {
#pragma unroll 8
        for (int i = threadIdx.x; i < n / 4; i += kAnchor) {
            const float4 x = reinterpret_cast<const float4*>(s)[i], y = reinterpret_cast<const float4*>(r)[i];
            e = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, e))));
        }
    } else {
        for (int i = threadIdx.x; i < n; i += kAnchor) e = fmaf(s[i], r[i], e);
    }
    double v = 0.0, sum = (double)e;
    if (t < T)
        for (int j = 0; j < blocks; ++j) {
            const size_t at = (((size_t)j * B + b) * T + t) * H + h;
            v += (double)rq[at] - (double)rk[at];
        }
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
        const double o = __shfl_up_sync(0xffffffffu, v, m);
        if (lane >= m) v += o;
        sum += __shfl_xor_sync(0xffffffffu, sum, m);
    }
    if (lane == 31) {
        part[warp] = v;
        whole[warp] = sum;
    }
    __syncthreads();
    for (int i = 0; i < kAnchor / 32; ++i) v += (i < warp ? part[i] : 0.0) + whole[i];
    const int len = lengths ? min(max(lengths[b], 0), T) : T;
    if (t < T) dg[((size_t)b * T + t) * H + h] = t < len ? (float)v : 0.f;
}

// Gradients of shared queries or keys: (rows,H,K) fp32 -> (rows,G,K), heads summed in order.
template <typename io_t>
__global__ void __launch_bounds__(256) attn_share_kernel(const float* p0, const float* p1, io_t* o0, io_t* o1, long long n,
                                                         int K, int per) {
    follow_wait();
    const float* p = blockIdx.y ? p1 : p0;
    io_t* o = blockIdx.y ? o1 : o0;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const long long rg = i / K, c = i - rg * K;
        float sum = 0.f;
        for (int j = 0; j < per; ++j) sum += p[(rg * per + j) * K + c];
        store1(o, i, sum);
    }
}

// ------------------------------------------------------------------------------------------------
// One token.  The state is read and written once and nothing else is large: a CTA owns a head's state rows (or, where
// there are few heads, some of its columns), a warp every eighth row of it, all of a thread's rows requested
// before the first is used.  256x16x128x128: 537 MB in 89 us, 6.1 TB/s (93 % of a copy's rate); 1x8x64x64: 6 us, a launch and one round trip.
// ------------------------------------------------------------------------------------------------
template <typename io_t, int NV>      // NV columns a lane
__global__ void __launch_bounds__(256) attn_step_kernel(AttnTensor q, AttnTensor k, AttnTensor v, const float* __restrict__ g, long long gb, long long gh, float scale, int H, int K, int V,
                                                        const float* state, float* state_out, long long sb, long long sh, void* out) {
    __shared__ float qs[M2D_ATTN_MAX_DIM], ks[M2D_ATTN_MAX_DIM], part[8][32 * NV];
    const int h = blockIdx.x % H, b = blockIdx.x / H, c = (blockIdx.y * 32 + (threadIdx.x & 31)) * NV, warp = threadIdx.x >> 5;
    const io_t* const qp = static_cast<const io_t*>(attn_at(q, b, h, sizeof(io_t)));
    const io_t* const kp = static_cast<const io_t*>(attn_at(k, b, h, sizeof(io_t)));
    const io_t* const vp = static_cast<const io_t*>(attn_at(v, b, h, sizeof(io_t)));
    const size_t at = (size_t)(b * sb + h * sh) + c;
    const bool on = c < V;
    constexpr int kAhead = 16;
    using N = Num<NV == 4 ? 2 : 1>;       // (packed arithmetic for pairs of columns)
    constexpr int P = NV == 4 ? 2 : 1;
    N s[kAhead][P];
    auto request = [&](int r0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int r = r0 + warp + j * 8;
            if (on && r < K) {
                const float* p = state + at + (size_t)r * V;
                if constexpr (NV == 4) { const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(p); s[j][0].v = t.x; s[j][1].v = t.y; }
                else s[j][0].v = *p;
            }
        }
    };
    const float gv = __ldg(g + b * gb + h * gh);          // (first: the state's rows are on their way meanwhile)
    request(0);
    if (threadIdx.x < K) {
        qs[threadIdx.x] = load1(qp, threadIdx.x);
        ks[threadIdx.x] = load1(kp, threadIdx.x);
    }
    // The decay in two parts, of which the first is below it and the second above zero (a state of infinity stays one): rounded to one, what it is off by would come
    // back with every token of the same decay and add up over its memory (8192 tokens: 7.5e-5 of the state after 2000 of them, now at most 8e-6 after 20000).
    const bool near = fabsf(gv) <= kLn2;
    const float less = near ? expm1f(gv) : 0.f, a = near ? 1.f + less : ex2((float)attn_decay(gv));
    float hi = fmaf(a, -0x1p-22f, a), lo = near ? less - (hi - 1.f) : a - hi;
    if (!(a <= 3.402823466e38f)) hi = lo = a;
    const N first = N::all(hi), rest = N::all(lo);
    N vv[P], o[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
#pragma unroll
        for (int k = 0; k < NV / P; ++k) vv[i].set(k, on ? load1(vp, c + i * (NV / P) + k) : 0.f);
        o[i] = N::all(0.f);
    }
    __syncthreads();
    for (int r0 = 0; r0 < K; r0 += 8 * kAhead) {
        if (r0) request(r0);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int r = r0 + warp + j * 8;
            if (on && r < K) {
                const N kr = N::all(ks[r]), qr = N::all(qs[r]);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    s[j][i] = fma_(s[j][i], first, fma_(s[j][i], rest, mul_(kr, vv[i])));
                    o[i] = fma_(qr, s[j][i], o[i]);
                }
                float* p = state_out + at + (size_t)r * V;
                if constexpr (NV == 4) *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(s[j][0].v, s[j][1].v);
                else *p = s[j][0].v;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) part[warp][(threadIdx.x & 31) * NV + i] = o[i / (NV / P)].get(i % (NV / P));
    __syncthreads();
    const int n0 = blockIdx.y * 32 * NV;
    for (int i = threadIdx.x; i < 32 * NV; i += 256)
        if (n0 + i < V) {
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += part[j][i];
            store1(static_cast<io_t*>(out), (size_t)blockIdx.x * V + n0 + i, scale * sum);
        }
}

// ---- host ------------------------------------------------------------------------------------------

static int check_attn(const m2d_attn_desc* d, bool ptrs) {
    if (!d) return M2D_ERR_NULL;
    if (d->struct_bytes != sizeof(m2d_attn_desc)) return M2D_ERR_ABI;
    if (d->dtype != M2D_F32 && d->dtype != M2D_BF16) return M2D_ERR_DTYPE;
    if (d->flags && ((d->flags & ~M2D_ATTN_TEST_GIVE_UP) || !test_hooks_enabled())) return M2D_ERR_FLAGS;
    if (d->B < 1 || d->T < 1 || d->H < 1 || d->G < 1 || d->H % d->G || d->K < 1 || d->V < 1 || d->K > M2D_ATTN_MAX_DIM || d->V > M2D_ATTN_MAX_DIM) return M2D_ERR_SHAPE;
    if (d->T > INT_MAX - 4 * kAnchor) return M2D_ERR_TOO_LARGE;      // (token numbers go up to the end of the last chunk)
    if ((int64_t)d->B * d->H > (1 << 24) || (int64_t)d->B * d->H * ((d->T + kAnchor - 1) / kAnchor) >= (1ll << 31)) return M2D_ERR_TOO_LARGE;
    if (ptrs && (!d->q.data || !d->k.data || !d->v.data || !d->log_decay)) return M2D_ERR_NULL;
    return M2D_OK;
}

static AttnTensor attn_tensor(const m2d_attn_desc* d, const m2d_attn_tensor& t, int per, int dim) {
    const uintptr_t bytes = d->dtype == M2D_F32 ? 16 : 8;
    const bool vec = dim % 4 == 0 && (reinterpret_cast<uintptr_t>(t.data) % bytes) == 0 && t.batch % 4 == 0 && t.token % 4 == 0 && t.head % 4 == 0;
    return {t.data, t.batch, t.token, t.head, per, vec ? 1 : 0};
}
static AttnState dense_state(const m2d_attn_desc* d, const float* p, bool transposed) {
    const long long n = (long long)d->K * d->V;
    return {const_cast<float*>(p), n * d->H, n, 0, transposed ? 1 : d->V, transposed ? d->V : 1};
}

// Segments: as many as fill the GPU, of `least` chunks of `chunk` tokens at least.  A second pass over y and z and two launches
// more: taken where it at least halves the time of the first.
static void plan_segments(const m2d_attn_desc* d, long long ctas, int per_sm, int chunk, int least, AttnLaunch* a) {
    a->runs = (d->T + kAnchor - 1) / kAnchor;
    const long long chunks = (d->T + chunk - 1) / chunk, want = std::min<long long>((long long)sm_count() * per_sm / ctas, chunks / least);
    a->nseg = 1;
    a->seg_len = (int)(chunks * chunk);
    if (want < 2) return;
    const long long per = (chunks + want - 1) / want;
    a->seg_len = (int)(per * chunk);
    a->nseg = (int)((chunks + per - 1) / per);
}

struct AttnPlan {
    AttnLaunch a{};
    bool tc = false;
    int cores = 1, col_blocks = 1, VT = 64, dot_blocks = 1;
    size_t smem = 0, bytes = 0;
    size_t at_seg[3] = {}, at_decay[3] = {}, at_dots[2] = {}, at_anchor[2] = {}, at_heads[2] = {};
};
// Of the forward pass's one core, or of `cores` of the backward's; its scratch begins at `base`.
static AttnPlan plan_attn(const m2d_attn_desc* d, bool bwd, bool tc, int cores = 3, size_t base = 0) {
    AttnPlan p;
    p.tc = tc;
    p.cores = bwd ? cores : 1;
    p.bytes = base;
    int per_sm = 1;
    if (!tc) {
        const int big = bwd ? std::max(d->K, d->V) : d->K, out = bwd ? big : d->V;
        p.VT = big > 192 ? 32 : 64;
        p.smem = attn_smem(big, p.VT);
        p.col_blocks = (out + p.VT - 1) / p.VT;
        p.dot_blocks = (d->K + p.VT - 1) / p.VT;
        per_sm = std::max<int>(1, (int)((kMaxSmem + 1024) / (p.smem + 1024)));
    }
    p.a.seg_columns = tc;
    // lengths: only the GPU knows how much of T there is, so twice as many as run at once (6x1395x3x64 fp32, training: 138 us for 153;
    // a segment of the tcgen05 form costs too much for that, 8x2048x16x128 forward: 19 us more)
    plan_segments(d, (long long)d->B * d->H * p.col_blocks * p.cores, per_sm * (d->lengths && !tc ? 2 : 1), tc ? 128 : 64, tc ? 4 : 1, &p.a);
    // Joined by the kernels that start from them, or by a launch.  tcgen05 form, two segments: 128 us against 139 with a launch; 18: a
    // CTA would read up to 17 states one after another.  The other form, four segments of single chunks: 16 us against 27, 11 and 5: 166 against 182.
    p.a.join_here = p.a.nseg > 1 && p.a.nseg <= (tc ? 4 : 12);
    // Nothing needs the own state of the last segment: where the others leave half of the GPU free (two segments), their states are
    // computed in parts (of two chunks at least, four states at most to read): 4x4096x16x128 131 -> 121 us.
    int states = p.a.nseg;
    p.a.parts = 1;
    if (tc && p.a.join_here) {
        const int per = p.a.seg_len / 128, others = p.a.nseg - 1;
        p.a.parts = (int)std::max<long long>(1, std::min<long long>({(long long)sm_count() / ((long long)d->B * d->H * p.cores * others), per / 2, 4 / others}));
        p.a.part_len = (per + p.a.parts - 1) / p.a.parts * 128;
        states = others * p.a.parts;
    }
    auto take = [&](size_t n) {
        const size_t at = p.bytes;
        p.bytes += (n + 255) / 256 * 256;
        return at;
    };
    const size_t bh = (size_t)d->B * d->H, kv = (size_t)d->K * d->V, tokens = bh * d->T;
    if (p.a.nseg > 1)
        for (int i = 0; i < p.cores; ++i) {
            p.at_seg[i] = take(4 * bh * states * kv);
            p.at_decay[i] = take(4 * bh * states);
        }
    if (bwd && d->d_log_decay) {
        for (size_t& at : p.at_dots) at = take(4 * tokens * p.dot_blocks);
        for (size_t& at : p.at_anchor) at = take(4 * bh * p.a.runs * kv);
    }
    if (bwd && d->G != d->H)
        for (size_t& at : p.at_heads) at = take(4 * tokens * d->K);
    return p;
}

// Whether the tcgen05 form takes the call: bf16, head sizes of whole 16-byte pieces up to 128, and tensors that TMA can address.
static bool tc_applies(const m2d_attn_desc* d, bool bwd) {
    if (d->dtype != M2D_BF16 || d->K > 128 || d->V > 128 || d->K % 8 || d->V % 8 || !tc_encoder()) return false;
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    auto fits = [&](const m2d_attn_tensor& t, int heads) {
        auto stride = [](int n, int64_t s) { return n == 1 || (s > 0 && s % 8 == 0 && s < (1ll << 36)); };
        return aligned(t.data) && stride(d->B, t.batch) && stride(d->T, t.token) && stride(heads, t.head);
    };
    if (!fits(d->q, d->G) || !fits(d->k, d->G) || !fits(d->v, d->H)) return false;
    return bwd ? fits(d->d_o, d->H) && aligned(d->d_q) && aligned(d->d_k) && aligned(d->d_v) : aligned(d->o);
}

static bool attn_map(CUtensorMap* map, const m2d_attn_desc* d, const AttnTensor& t, int dim) {
    const int heads = d->H / t.per;
    // (a stride that no step is taken along may be anything: the map gets a valid one)
    auto bytes = [](int n, long long s) { return n == 1 ? (cuuint64_t)16 : (cuuint64_t)s * 2; };
    const cuuint64_t dims[4] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)d->T, (cuuint64_t)d->B};
    const cuuint64_t strides[3] = {bytes(heads, t.sh), bytes(d->T, t.st), bytes(d->B, t.sb)};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)kTc, 1}, step[4] = {1, 1, 1, 1};
    return tc_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(t.p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A launch of `count` cores from `first` on, all with the same head sizes.
template <int KD, int VD, TcMode MODE>
static int launch_tc(const m2d_attn_desc* d, const AttnPlan& p, int first, int count, cudaStream_t st) {
    TcLaunch L;
    TcMaps maps;
    L.a = p.a;
    L.cores = count;
    L.host_flag = wait_failure_flag();
    L.give_up = (d->flags & M2D_ATTN_TEST_GIVE_UP) != 0;
    for (int i = 0; i < count; ++i) {
        const AttnCore& c = L.a.core[i] = p.a.core[first + i];
        if (!(MODE == kTcStateOnly || attn_map(&maps.m[i][0], d, c.x, c.Kd)) || !attn_map(&maps.m[i][1], d, c.y, c.Kd) || !attn_map(&maps.m[i][2], d, c.z, c.Vd)) return M2D_ERR_LAUNCH;
        if (MODE != kTcStateOnly && !c.out_f32 && !attn_map(&maps.m[i][3], d, {c.out, c.ob, c.ot, c.oh, 1, 1}, c.Vd)) return M2D_ERR_LAUNCH;
    }
    constexpr TcLayout lay(KD, VD, MODE);
    constexpr size_t smem = lay.small + sizeof(TcSmall);
    static_assert(smem <= kMaxSmem, "shared memory of a CTA");
    auto kern = attn_tc_kernel<KD, VD, MODE>;
    if (!allow_smem(reinterpret_cast<const void*>(kern), smem)) return M2D_ERR_LAUNCH;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(d->B * d->H * (MODE == kTcStateOnly && p.a.join_here ? (p.a.nseg - 1) * p.a.parts : p.a.nseg) * count));
    c.blockDim = dim3(kTcThreads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    // what follows another group of the same pass needs nothing of it
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &attr;
    c.numAttrs = first > 0 ? 1 : 0;
    return cudaLaunchKernelEx(&c, kern, maps, L) == cudaSuccess ? M2D_OK : (cudaGetLastError(), M2D_ERR_LAUNCH);
}
template <TcMode MODE>
static int launch_tc(const m2d_attn_desc* d, const AttnPlan& p, int first, int count, cudaStream_t st) {
    const bool k64 = p.a.core[first].Kd <= 64, v64 = p.a.core[first].Vd <= 64;
    if (k64) return v64 ? launch_tc<64, 64, MODE>(d, p, first, count, st) : launch_tc<64, 128, MODE>(d, p, first, count, st);
    return v64 ? launch_tc<128, 64, MODE>(d, p, first, count, st) : launch_tc<128, 128, MODE>(d, p, first, count, st);
}

// (Not as a launch that follows: its CTAs would gather on the few SMs that the states leave free, 1x65536x8: 180 us against 174.)
static void launch_join(const AttnPlan& p, cudaStream_t st) {
    const int n = p.a.core[0].Kd * p.a.core[0].Vd;
    attn_join_kernel<<<dim3(p.a.B * p.a.H, (n + 127) / 128, p.cores), 128, 0, st>>>(p.a);
}
template <typename io_t, int VT>
static int launch_any(const AttnPlan& p, cudaStream_t st) {
    const dim3 grid((unsigned)(p.a.B * p.a.H * p.a.nseg), p.col_blocks, p.cores);
    auto full = attn_core_kernel<io_t, VT, false>;
    if (!allow_smem(reinterpret_cast<const void*>(full), p.smem)) return M2D_ERR_LAUNCH;
    if (p.a.nseg > 1) {
        auto part = attn_core_kernel<io_t, VT, true>;
        if (!allow_smem(reinterpret_cast<const void*>(part), p.smem)) return M2D_ERR_LAUNCH;
        part<<<grid, kAttnThreads, p.smem, st>>>(p.a);
        if (!p.a.join_here) launch_join(p, st);
    }
    if (p.a.nseg > 1) return launch_following(full, grid, dim3(kAttnThreads), p.smem, st, p.a) ? M2D_OK : M2D_ERR_LAUNCH;
    full<<<grid, kAttnThreads, p.smem, st>>>(p.a);
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}
static int launch_core(const m2d_attn_desc* d, const AttnPlan& p, cudaStream_t st) {
    if (p.tc) {
        // dq and dk have (V,K) states, dv a (K,V) one: one launch where the kernel is the same
        const bool together = p.cores == 1 || ((d->K <= 64) == (d->V <= 64) && !p.a.core[0].out_f32);
        const int counts[2] = {together ? p.cores : 2, together ? 0 : 1};
        for (int pass = p.a.nseg > 1 ? 0 : 1; pass < 2; ++pass) {
            for (int i = 0; i < 2; ++i) {
                if (!counts[i]) continue;
                const int first = i ? counts[0] : 0;
                const AttnCore& c = p.a.core[first];                // (dv, which wants least, is never the first of several)
                const int rc = !pass ? launch_tc<kTcStateOnly>(d, p, first, counts[i], st)
                               : c.out_f32 ? launch_tc<kTcHeads>(d, p, first, counts[i], st) : launch_tc<kTcPlain>(d, p, first, counts[i], st);
                if (rc != M2D_OK) return rc;
            }
            if (!pass && !p.a.join_here) launch_join(p, st);
        }
        return M2D_OK;
    }
    if (d->dtype == M2D_F32) return p.VT == 64 ? launch_any<float, 64>(p, st) : launch_any<float, 32>(p, st);
    return p.VT == 64 ? launch_any<__nv_bfloat16, 64>(p, st) : launch_any<__nv_bfloat16, 32>(p, st);
}

static void fill_launch(const m2d_attn_desc* d, AttnPlan& p) {
    AttnLaunch& a = p.a;
    a.g = d->log_decay; a.gb = d->g_batch; a.gt = d->g_token; a.gh = d->g_head;
    a.lengths = d->lengths;
    a.B = d->B; a.T = d->T; a.H = d->H;
    char* const ws = static_cast<char*>(d->workspace);
    for (int i = 0; i < p.cores; ++i) {
        a.core[i].seg_state = reinterpret_cast<float*>(ws + p.at_seg[i]);
        a.core[i].seg_decay = reinterpret_cast<float*>(ws + p.at_decay[i]);
    }
}
static int check_workspace(const m2d_attn_desc* d, size_t bytes) {
    if (!bytes) return M2D_OK;
    return d->workspace && d->workspace_bytes >= bytes && (reinterpret_cast<uintptr_t>(d->workspace) & 255) == 0 ? M2D_OK : M2D_ERR_WORKSPACE;
}
// What either form may need, with lengths or without: a query does not depend on the tensors' addresses.
static size_t attn_workspace(const m2d_attn_desc* desc, bool bwd) {
    size_t most = 0;
    for (const int32_t* lengths : {(const int32_t*)nullptr, (const int32_t*)&desc->B}) {      // (whether there are any is all that a plan looks at)
        m2d_attn_desc d = *desc;
        d.lengths = lengths;
        size_t tc = 0;
        if (d.dtype == M2D_BF16) tc = bwd && d.d_log_decay ? plan_attn(&d, false, true, 1, plan_attn(&d, true, false, 2).bytes).bytes : plan_attn(&d, bwd, true).bytes;
        most = std::max({most, plan_attn(&d, bwd, false).bytes, tc});
    }
    return most;
}

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_attn_fwd_workspace(const m2d_attn_desc* d) { return check_attn(d, false) == M2D_OK ? attn_workspace(d, false) : 0; }
extern "C" uint64_t m2d_attn_bwd_workspace(const m2d_attn_desc* d) { return check_attn(d, false) == M2D_OK ? attn_workspace(d, true) : 0; }

extern "C" int m2d_attn_fwd(const m2d_attn_desc* d, void* stream) {
    int rc = check_attn(d, true);
    if (rc != M2D_OK) return rc;
    if (!d->o) return M2D_ERR_NULL;
    AttnPlan p = plan_attn(d, false, tc_applies(d, false));
    if ((rc = check_workspace(d, attn_workspace(d, false))) != M2D_OK) return rc;
    fill_launch(d, p);
    AttnCore& c = p.a.core[0];
    const int per = d->H / d->G;
    c.x = attn_tensor(d, d->q, per, d->K); c.y = attn_tensor(d, d->k, per, d->K); c.z = attn_tensor(d, d->v, 1, d->V);
    c.Kd = d->K; c.Vd = d->V;
    c.out = d->o; c.oh = d->V; c.ot = (long long)d->H * d->V; c.ob = c.ot * d->T;
    c.s_intra = c.s_inter = d->scale; c.s_update = 1.f;
    c.init = dense_state(d, d->state, false);
    c.fin = dense_state(d, d->state_out, false);
    return launch_core(d, p, static_cast<cudaStream_t>(stream));
}

extern "C" int m2d_attn_bwd(const m2d_attn_desc* d, void* stream) {
    int rc = check_attn(d, true);
    if (rc != M2D_OK) return rc;
    if (!d->d_o.data || !d->d_q || !d->d_k || !d->d_v) return M2D_ERR_NULL;
    // The decay's gradient sums dots of 512 tokens that cancel: dq and dk with operands in two bf16 parts left it at up to 4e-5
    // (2x1000x4x128), split tf32 ones leave it at 1e-6.  (8x2048x16x128, training: 2690 us, 3525 with dv in this form too, 430 with the parts.)
    const bool tc = tc_applies(d, true), apart = tc && d->d_log_decay;       // dv, which has no part in it, in the tcgen05 form
    AttnPlan p = plan_attn(d, true, tc && !apart, apart ? 2 : 3), pv = p;
    if (apart) pv = plan_attn(d, false, true, 1, p.bytes);
    if ((rc = check_workspace(d, attn_workspace(d, true))) != M2D_OK) return rc;
    fill_launch(d, p);
    if (apart) fill_launch(d, pv);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    char* const ws = static_cast<char*>(d->workspace);
    const int per = d->H / d->G;
    const AttnTensor q = attn_tensor(d, d->q, per, d->K), k = attn_tensor(d, d->k, per, d->K), v = attn_tensor(d, d->v, 1, d->V), go = attn_tensor(d, d->d_o, 1, d->V);
    AttnCore &dq = p.a.core[0], &dk = p.a.core[1], &dv = apart ? pv.a.core[0] : p.a.core[2];
    dq.x = go; dq.y = v; dq.z = k; dq.e = q; dq.rev = 0;
    dk.x = v; dk.y = go; dk.z = q; dk.e = k; dk.rev = 1;
    dv.x = k; dv.y = q; dv.z = go; dv.rev = 1;
    dq.Kd = dk.Kd = dv.Vd = d->V;
    dq.Vd = dk.Vd = dv.Kd = d->K;
    dq.s_intra = dq.s_inter = d->scale; dq.s_update = 1.f;
    dk.s_intra = dv.s_intra = dk.s_update = dv.s_update = d->scale;
    dk.s_inter = dv.s_inter = 1.f;
    for (int i = 0; i < 2; ++i) {
        AttnCore& c = i ? dk : dq;
        c.out = d->G == d->H ? (i ? d->d_k : d->d_q) : ws + p.at_heads[i];
        c.out_f32 = d->G != d->H;
        c.oh = d->K; c.ot = (long long)d->H * d->K; c.ob = c.ot * d->T;
        if (d->d_log_decay) {
            c.dots = reinterpret_cast<float*>(ws + p.at_dots[i]);
            c.anchors = reinterpret_cast<float*>(ws + p.at_anchor[i]);
        }
    }
    dv.out = d->d_v; dv.oh = d->V; dv.ot = (long long)d->H * d->V; dv.ob = dv.ot * d->T;
    dq.init = dense_state(d, d->state, true);
    dk.init = dense_state(d, d->d_state_out, true);
    dv.init = dense_state(d, d->d_state_out, false);
    dv.fin = dense_state(d, d->d_state, false);
    if (apart && (rc = launch_core(d, pv, st)) != M2D_OK) return rc;
    if ((rc = launch_core(d, p, st)) != M2D_OK) return rc;
    if (d->d_log_decay) {
        const unsigned n = (unsigned)(d->B * d->H * p.a.runs);
        if (!launch_following(attn_decay_kernel, dim3(n), dim3(kAnchor), 0, st, (const float*)dq.dots, (const float*)dk.dots, p.dot_blocks,
                              (const float*)dq.anchors, (const float*)dk.anchors, d->K * d->V, d->lengths, d->d_log_decay, d->B, d->T, d->H, p.a.runs))
            return M2D_ERR_LAUNCH;
    }
    if (d->G != d->H) {
        const long long n = (long long)d->B * d->T * d->G * d->K;
        const dim3 grid((unsigned)std::min<long long>((n + 255) / 256, 16ll * sm_count()), 2);
        const float *h0 = reinterpret_cast<const float*>(ws + p.at_heads[0]), *h1 = reinterpret_cast<const float*>(ws + p.at_heads[1]);
        if (d->dtype == M2D_F32) rc = launch_following(attn_share_kernel<float>, grid, dim3(256), 0, st, h0, h1, static_cast<float*>(d->d_q), static_cast<float*>(d->d_k), n, d->K, per) ? M2D_OK : M2D_ERR_LAUNCH;
        else rc = launch_following(attn_share_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, h0, h1, static_cast<__nv_bfloat16*>(d->d_q), static_cast<__nv_bfloat16*>(d->d_k), n, d->K, per) ? M2D_OK : M2D_ERR_LAUNCH;
        if (rc != M2D_OK) return rc;
    }
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}

extern "C" int m2d_attn_step(const m2d_attn_desc* d, int64_t state_batch, int64_t state_head, void* stream) {
    const int rc = check_attn(d, true);
    if (rc != M2D_OK) return rc;
    if (d->T != 1) return M2D_ERR_SHAPE;
    if (!d->o || !d->state || !d->state_out) return M2D_ERR_NULL;
    const int per = d->H / d->G;
    const AttnTensor q = attn_tensor(d, d->q, per, d->K), k = attn_tensor(d, d->k, per, d->K), v = attn_tensor(d, d->v, 1, d->V);
    auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
    const bool vec = d->V % 4 == 0 && state_batch % 4 == 0 && state_head % 4 == 0 && aligned(d->state) && aligned(d->state_out);
    const dim3 grid(d->B * d->H, (d->V + (vec ? 127 : 31)) / (vec ? 128 : 32));
    auto launch = [&](auto kern) {
        kern<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(q, k, v, d->log_decay, d->g_batch, d->g_head, d->scale, d->H, d->K, d->V, d->state, d->state_out, state_batch, state_head, d->o);
    };
    if (d->dtype == M2D_F32) vec ? launch(attn_step_kernel<float, 4>) : launch(attn_step_kernel<float, 1>);
    else vec ? launch(attn_step_kernel<__nv_bfloat16, 4>) : launch(attn_step_kernel<__nv_bfloat16, 1>);
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}
