// Layer normalisation of rows, with the residual sum before it, forward and backward with the parameters' gradients.
//
//   s = x + r in the tensors' type;  y = (s - mean) rstd w + b
//   dh = dy w;  dx = rstd (dh - mean(dh) - h mean(dh h)) + ds,  h = (s - mean) rstd;  dw = sum dy h,  db = sum dy over rows
//
// A row is held in registers, by 8, 16 or 32 lanes of a warp or by a CTA, as its length asks; mean first, then the squares about it.  The mean is
// taken about the row's first value, so that equal values have that value for a mean, whatever its size.  In the backward pass a thread
// has the same columns in every row that it meets: it sums their parameter gradients in registers, CTAs write their sums side by side, and a second
// launch adds those up in a fixed order.  Rows too long for registers are read again where they are needed.  Measured, bf16: 100352x320 forward 28 us
// (4.6 TB/s), backward 35 (5.5) and 7 for the parameters' sums; 8192x4096 with a residual 47 (5.7) and 57 (4.7): a row's two sums, one after the other.
#include "follow.cuh"
#include "packed.cuh"
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
    int C, params_f32, parts, stages;  // stages: rows on their way, where those are not whole pieces
    float eps;
};

// V neighbouring values as they are in memory, and as V / W packed numbers.
template <typename T, int V> struct Lane;
template <> struct Lane<float, 4> {
    using Raw = float4;
    using N = Num<2>;
    static constexpr int n = 2;
    static __device__ __forceinline__ void get(const Raw& r, N* v) { v[0] = N::make(r.x, r.y); v[1] = N::make(r.z, r.w); }
    static __device__ __forceinline__ Raw put(const N* v) { return make_float4(v[0].get(0), v[0].get(1), v[1].get(0), v[1].get(1)); }
};
template <> struct Lane<float, 1> {
    using Raw = float;
    using N = Num<1>;
    static constexpr int n = 1;
    static __device__ __forceinline__ void get(Raw r, N* v) { v[0].v = r; }
    static __device__ __forceinline__ Raw put(const N* v) { return v[0].v; }
};
template <> struct Lane<__nv_bfloat16, 8> {
    using Raw = uint4;
    using N = Num<2>;
    static constexpr int n = 4;
    static __device__ __forceinline__ void get(const Raw& r, N* v) {
        const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = N::make(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    }
    static __device__ __forceinline__ Raw put(const N* v) {
        return make_uint4(pack_bf16x2(v[0].get(0), v[0].get(1)), pack_bf16x2(v[1].get(0), v[1].get(1)), pack_bf16x2(v[2].get(0), v[2].get(1)), pack_bf16x2(v[3].get(0), v[3].get(1)));
    }
};
template <> struct Lane<__nv_bfloat16, 1> {
    using Raw = unsigned short;
    using N = Num<1>;
    static constexpr int n = 1;
    static __device__ __forceinline__ void get(Raw r, N* v) { v[0].v = bf16_bits_to_float(r); }
    static __device__ __forceinline__ Raw put(const N* v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v[0].v)); }
};
// V neighbouring values of a parameter (fp32 or T); `none` where there is no such parameter.
template <typename T, int V>
__device__ __forceinline__ void parameter(const void* p, int f32, int c, float none, typename Lane<T, V>::N* v) {
    using P = Lane<T, V>;
    if (!p) {
#pragma unroll
        for (int k = 0; k < P::n; ++k) v[k] = P::N::all(none);
    } else if (f32) {
        const float* q = static_cast<const float*>(p) + c;
        if constexpr (V % 4 == 0) {
#pragma unroll
            for (int k = 0; k < V; k += 4) Lane<float, 4>::get(__ldg(reinterpret_cast<const float4*>(q + k)), v + k / 2);
        } else {
            v[0].v = __ldg(q);
        }
    } else {
        P::get(__ldg(reinterpret_cast<const typename P::Raw*>(static_cast<const T*>(p) + c)), v);
    }
}
__device__ __forceinline__ float total(Num<1> n) { return n.v; }
__device__ __forceinline__ float total(Num<2> n) { return n.get(0) + n.get(1); }
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
constexpr int kLnThreads = 128;        // of a CTA whose rows are held by parts of warps
constexpr size_t kLnStatic = 1024;     // row_sum's shared memory counts towards what a kernel has without asking

// A thread's share of the rows: columns (i span + l) V ..., i < NV, of every `step`-th row from `row` on, as many rows at a time as `step` says
// all CTAs have.  The loads of its next row are under way while it works on one, and the parameters stay in registers.
template <int V, int R>
struct Share {
    static constexpr int lanes = R ? R : 1;
    int span, l;
    long long row, step;
    __device__ __forceinline__ Share() {
        span = R ? R : blockDim.x;
        l = R ? threadIdx.x % lanes : threadIdx.x;
        const int rows = R ? kLnThreads / lanes : 1;
        row = (long long)blockIdx.x * rows + (R ? threadIdx.x / lanes : 0);
        step = (long long)gridDim.x * rows;
    }
    __device__ __forceinline__ int column(int i) const { return (i * span + l) * V; }
    // rows that a CTA still meets: the same number for all of its threads, which reduce together
    __device__ __forceinline__ bool more(long long N, long long at) const { return at - (R ? threadIdx.x / lanes : 0) < N; }
};

// Rows on their way, through shared memory: what is wanted are 40 KB and more of an SM under way, which registers have no room for.
// Whole pieces (V > 1): each thread its own, two or three rows ahead; nobody else looks at them.  Others: the 16-byte pieces that a row touches, by all of
// its lanes, one to three rows ahead, as they have room; a value is then where it lies in them.
template <typename T, int V, int R, int NV, int TENSORS>
struct Rows {
    using Raw = typename Lane<T, V>::Raw;
    static constexpr int room = 224 * 1024 / (TENSORS * NV * 16 * (R ? kLnThreads : 512)), fixed = room < 3 ? room : 3;
    static constexpr int groups = R ? kLnThreads / (R ? R : 1) : 1;            // rows of a CTA at a time
    static int stages(int C) { return V > 1 ? fixed : (int)std::max<size_t>(1, std::min<size_t>(3, 200 * 1024 / (TENSORS * groups * span_bytes(C)))); }
    static size_t bytes(int C, int threads) { return V > 1 ? (size_t)fixed * TENSORS * NV * threads * 16 : stages(C) * TENSORS * groups * span_bytes(C); }
    __host__ __device__ static size_t span_bytes(int C) { return (((size_t)C * sizeof(T) + 15) / 16 + 1) * 16; }

    const T* from[TENSORS];
    long long pitch[TENSORS];
    unsigned base, slot, span, off[TENSORS];
    int C, ahead, l, lanes;
    template <typename S>
    __device__ __forceinline__ Rows(void* smem, const S& at, const LnArgs& p) {
        C = p.C;
        slot = 0;
        l = at.l;
        lanes = at.span;
        if constexpr (V > 1) {
            ahead = fixed;
            base = smem_u32(smem) + threadIdx.x * 16;
        } else {
            ahead = p.stages;
            span = (unsigned)span_bytes(C);
            base = smem_u32(smem) + (R ? threadIdx.x / (R ? R : 1) : 0) * (unsigned)ahead * TENSORS * span;
        }
    }
    __device__ __forceinline__ unsigned place(int t, int i) const {
        if constexpr (V > 1) return base + ((slot * TENSORS + t) * NV + i) * blockDim.x * 16;
        else return base + (slot * TENSORS + t) * span;
    }
    // asks for a row (an empty one where it is not `on`)
    __device__ __forceinline__ void order(long long row, bool on) {
#pragma unroll
        for (int t = 0; t < TENSORS; ++t) {
            const T* const p = from[t] + (on ? row : 0) * pitch[t];
            if constexpr (V > 1) {
#pragma unroll
                for (int i = 0; i < NV; ++i) cp_async16_if(on && (i * lanes + l) * V < C, place(t, i), p + (i * lanes + l) * V);
            } else if (on) {
                const int head = (int)(reinterpret_cast<uintptr_t>(p) & 15), all = head + C * (int)sizeof(T);
                const char* const q = reinterpret_cast<const char*>(p) - head;
                for (int j = l * 16; j < all; j += lanes * 16) {
                    const unsigned to = place(t, 0) + j;
                    if (q + j >= reinterpret_cast<const char*>(from[t])) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(q + j), "r"(min(16, all - j)) : "memory");
                    } else {                       // (the piece begins before the tensor)
                        for (int k = head; k < min(16, all); k += (int)sizeof(T)) {
                            if constexpr (sizeof(T) == 4) asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + k), "r"(*reinterpret_cast<const unsigned*>(q + k)) : "memory");
                            else asm volatile("st.shared.b16 [%0], %1;" ::"r"(to + k), "h"(*reinterpret_cast<const unsigned short*>(q + k)) : "memory");
                        }
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++slot == (unsigned)ahead) slot = 0;
    }
    static __device__ __forceinline__ void together() {
        if constexpr (R == 0) __syncthreads();
        else __syncwarp();
    }
    // waits for the oldest row that was asked for; its slot is the next to be filled, after release()
    __device__ __forceinline__ void arrived(long long row) {
        if constexpr (V > 1) {
            asm volatile("cp.async.wait_group %0;" ::"n"(fixed - 1) : "memory");
        } else {
            if (ahead == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
            else if (ahead == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 0;" ::: "memory");
            together();
#pragma unroll
            for (int t = 0; t < TENSORS; ++t) off[t] = place(t, 0) + (unsigned)(reinterpret_cast<uintptr_t>(from[t] + row * pitch[t]) & 15);
        }
    }
    __device__ __forceinline__ Raw take(int t, int i) const {
        if constexpr (V > 1) {
            uint4 r;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(place(t, i)) : "memory");
            return *reinterpret_cast<const Raw*>(&r);
        } else {
            const int c = i * lanes + l;
            Raw r{};
            if (c >= C) return r;
            if constexpr (sizeof(T) == 4) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(off[t] + c * 4) : "memory");
            else asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(off[t] + c * 2) : "memory");
            return r;
        }
    }
    __device__ __forceinline__ void release() const {
        if constexpr (V == 1) together();
    }
};

template <typename T, int V, int R, int NV, bool RES>
__global__ void __launch_bounds__(R ? kLnThreads : 512) ln_fwd_kernel(const LnArgs p) {
    using P = Lane<T, V>;
    using Raw = typename P::Raw;
    using N = typename P::N;
    const Share<V, R> at;
    N w[NV][P::n], b[NV][P::n];
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at.column(i) < p.C) {
            parameter<T, V>(p.w, p.params_f32, at.column(i), 1.f, w[i]);
            parameter<T, V>(p.b, p.params_f32, at.column(i), 0.f, b[i]);
        }
    extern __shared__ __align__(16) char smem[];
    Rows<T, V, R, NV, RES ? 2 : 1> rows(smem, at, p);
    rows.from[0] = static_cast<const T*>(p.x);
    rows.pitch[0] = p.xp;
    if constexpr (RES) {
        rows.from[1] = static_cast<const T*>(p.r);
        rows.pitch[1] = p.rp;
    }
    T lead, lead_r;                         // the next row's first values (as they are: nothing waits for them here)
    auto load = [&](long long row) { rows.order(row, row < p.N); };
    auto look = [&](long long row) {
        lead = static_cast<const T*>(p.x)[(row < p.N ? row : 0) * p.xp];
        if constexpr (RES) lead_r = static_cast<const T*>(p.r)[(row < p.N ? row : 0) * p.rp];
    };
    int slot = 0;
    long long row = at.row;
    for (int k = 0; k < rows.ahead; ++k) load(row + k * at.step);
    look(row);
    const float per = 1.f / (float)p.C;
    for (; at.more(p.N, row); row += at.step) {
        N v[NV][P::n];
        rows.arrived(row < p.N ? row : 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            P::get(rows.take(0, i), v[i]);
            if constexpr (RES) {
                N r[P::n];
                P::get(rows.take(1, i), r);
#pragma unroll
                for (int k = 0; k < P::n; ++k) v[i][k] = add_(v[i][k], r[k]);
                const Raw sum = P::put(v[i]);
                if (row < p.N && at.column(i) < p.C) *reinterpret_cast<Raw*>(static_cast<T*>(p.s) + row * p.C + at.column(i)) = sum;
                P::get(sum, v[i]);           // (rounded)
            }
        }
        const float first = RES ? sum_as<T>(value_of(&lead), value_of(&lead_r)) : value_of(&lead);
        rows.release();
        load(row + rows.ahead * at.step);
        look(row + at.step);
        N acc = N::all(0.f);
        const N less = N::all(-first);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.column(i) < p.C)
#pragma unroll
                for (int k = 0; k < P::n; ++k) acc = add_(acc, add_(v[i][k], less));
        float sum[1] = {total(acc)};
        row_sum<R>(sum, slot);
        const float mean = first + sum[0] / (float)p.C;
        const N off = N::all(-mean);
        acc = N::all(0.f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.column(i) < p.C)
#pragma unroll
                for (int k = 0; k < P::n; ++k) {
                    v[i][k] = add_(v[i][k], off);
                    acc = fma_(v[i][k], v[i][k], acc);
                }
        sum[0] = total(acc);
        row_sum<R>(sum, slot);
        const float rstd = rsqrtf(fmaf(sum[0], per, p.eps));
        if (row >= p.N) continue;
        if (p.stats && at.l == 0) p.stats[row] = make_float2(mean, rstd);
        const N scale = N::all(rstd);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.column(i) < p.C) {
#pragma unroll
                for (int k = 0; k < P::n; ++k) v[i][k] = fma_(mul_(v[i][k], scale), w[i][k], b[i][k]);
                *reinterpret_cast<Raw*>(static_cast<T*>(p.y) + row * p.C + at.column(i)) = P::put(v[i]);
            }
    }
}

template <typename T, int V, int R, int NV, bool DS>
__global__ void __launch_bounds__(R ? kLnThreads : 512) ln_bwd_kernel(const LnArgs p) {
    using P = Lane<T, V>;
    using Raw = typename P::Raw;
    using N = typename P::N;
    let_follow();
    const Share<V, R> at;
    N w[NV][P::n], dw[NV][P::n], db[NV][P::n];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int k = 0; k < P::n; ++k) w[i][k] = dw[i][k] = db[i][k] = N::all(0.f);
        if (at.column(i) < p.C) parameter<T, V>(p.w, p.params_f32, at.column(i), 1.f, w[i]);
    }
    extern __shared__ __align__(16) char smem[];   // the rows on their way; at the end sums, where parts of warps hold rows: [warps][2][columns of R lanes]
    Rows<T, V, R, NV, DS ? 3 : 2> rows(smem, at, p);
    rows.from[0] = static_cast<const T*>(p.x);
    rows.from[1] = static_cast<const T*>(p.dy);
    rows.pitch[0] = p.xp;
    rows.pitch[1] = p.dyp;
    if constexpr (DS) {
        rows.from[2] = static_cast<const T*>(p.ds);
        rows.pitch[2] = p.dsp;
    }
    float2 st;
    auto load = [&](long long row) { rows.order(row, row < p.N); };
    auto look = [&](long long row) { st = row < p.N ? p.stats[row] : make_float2(0.f, 0.f); };
    int slot = 0;
    long long row = at.row;
    for (int k = 0; k < rows.ahead; ++k) load(row + k * at.step);
    look(row);
    const float per = 1.f / (float)p.C;
    for (; at.more(p.N, row); row += at.step) {
        N h[NV][P::n], dh[NV][P::n], s0 = N::all(0.f), s1 = N::all(0.f);
        Raw keep[DS ? NV : 1];
        const N off = N::all(-st.x), scale = N::all(st.y);
        rows.arrived(row < p.N ? row : 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            P::get(rows.take(0, i), h[i]);
            P::get(rows.take(1, i), dh[i]);
            if constexpr (DS) keep[i] = rows.take(2, i);
        }
        const float rstd = st.y;
        rows.release();
        load(row + rows.ahead * at.step);
        look(row + at.step);
        if (row < p.N)
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.column(i) < p.C)
#pragma unroll
                for (int k = 0; k < P::n; ++k) {
                    h[i][k] = mul_(add_(h[i][k], off), scale);
                    db[i][k] = add_(db[i][k], dh[i][k]);
                    dw[i][k] = fma_(dh[i][k], h[i][k], dw[i][k]);
                    dh[i][k] = mul_(dh[i][k], w[i][k]);
                    s0 = add_(s0, dh[i][k]);
                    s1 = fma_(dh[i][k], h[i][k], s1);
                }
        float sum[2] = {total(s0), total(s1)};
        row_sum<R>(sum, slot);
        if (row >= p.N) continue;
        const N m0 = N::all(-sum[0] * per), m1 = N::all(-sum[1] * per), factor = N::all(rstd);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at.column(i) < p.C) {
                N g[P::n];
                if constexpr (DS) P::get(keep[i], g);
#pragma unroll
                for (int k = 0; k < P::n; ++k) {
                    const N t = fma_(h[i][k], m1, add_(dh[i][k], m0));
                    g[k] = DS ? fma_(factor, t, g[k]) : mul_(factor, t);
                }
                *reinterpret_cast<Raw*>(static_cast<T*>(p.dx) + row * p.C + at.column(i)) = P::put(g);
            }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!p.partial) return;
    float* const out = p.partial + (long long)blockIdx.x * 2 * p.C;
    constexpr int W = V / P::n;
    if constexpr (R == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int c = at.column(i) + k;
                if (c < p.C) { out[c] = dw[i][k / W].get(k % W); out[p.C + c] = db[i][k / W].get(k % W); }
            }
    } else {
        // lanes of one warp that have the same columns, then the warps in turn
        constexpr int cols = R * NV * V;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        float* const sums = reinterpret_cast<float*>(smem);
        __syncthreads();                           // (no row is on its way any more, for any thread)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float a = dw[i][k / W].get(k % W), b = db[i][k / W].get(k % W);
#pragma unroll
                for (int m = R; m < 32; m <<= 1) {
                    a += __shfl_xor_sync(0xffffffffu, a, m);
                    b += __shfl_xor_sync(0xffffffffu, b, m);
                }
                if (lane < R) {
                    sums[(warp * 2) * cols + at.column(i) + k] = a;
                    sums[(warp * 2 + 1) * cols + at.column(i) + k] = b;
                }
            }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * cols; c += kLnThreads) {
            float v = 0.f;
            for (int k = 0; k < kLnThreads / 32; ++k) v += sums[k * 2 * cols + c];
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
            Num<1> w, b;
            parameter<T, 1>(p.w, p.params_f32, c, 1.f, &w);
            parameter<T, 1>(p.b, p.params_f32, c, 0.f, &b);
            store1(static_cast<T*>(p.y), row * p.C + c, fmaf((v - mean) * rstd, w.v, b.v));
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
        float sum[2] = {0.f, 0.f};
        Num<1> w;
        for (int c = threadIdx.x; c < p.C; c += kLongThreads) {
            parameter<T, 1>(p.w, p.params_f32, c, 1.f, &w);
            const float dh = value_of(dy + c) * w.v;
            sum[0] += dh;
            sum[1] = fmaf(dh, (value_of(x + c) - st.x) * st.y, sum[1]);
        }
        row_sum<0>(sum, slot);
        const float m0 = sum[0] / (float)p.C, m1 = sum[1] / (float)p.C;
        for (int c = threadIdx.x; c < p.C; c += kLongThreads) {
            parameter<T, 1>(p.w, p.params_f32, c, 1.f, &w);
            const float h = (value_of(x + c) - st.x) * st.y, g = p.ds ? value_of(static_cast<const T*>(p.ds) + row * p.dsp + c) : 0.f;
            store1(static_cast<T*>(p.dx), row * p.C + c, fmaf(st.y, fmaf(-h, m1, value_of(dy + c) * w.v - m0), g));
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
    if (c < p.C) {
        constexpr int U = 16;                      // loads under way at once: some 500 sums in one go
        const float* const q = p.partial + (long long)blockIdx.y * p.C + c;
        for (int i = warp; i < p.parts; i += 32 * U) {
            float t[U];
#pragma unroll
            for (int k = 0; k < U; ++k) t[k] = i + 32 * k < p.parts ? q[(long long)(i + 32 * k) * 2 * p.C] : 0.f;
#pragma unroll
            for (int k = 0; k < U; ++k) v += t[k];
        }
    }
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
    const uintptr_t es = d->dtype == M2D_F32 ? 4 : 2, pes = d->params_f32 ? 4 : es;
    for (const void* t : {d->x, d->residual, static_cast<const void*>(d->sum), static_cast<const void*>(d->y), d->d_y, d->d_sum, static_cast<const void*>(d->d_x)})
        if (reinterpret_cast<uintptr_t>(t) % es) return M2D_ERR_PITCH;
    for (const void* t : {d->weight, d->bias, static_cast<const void*>(d->d_weight), static_cast<const void*>(d->d_bias)})
        if (reinterpret_cast<uintptr_t>(t) % pes) return M2D_ERR_PITCH;
    if (reinterpret_cast<uintptr_t>(d->stats) % sizeof(float2)) return M2D_ERR_PITCH;
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
    // whole pieces: one to three of bf16 a lane, twice as many of fp32, by parts of warps that leave the fewest lanes without work
    const int unit = es == 4 ? 2 : 1;
    long long least = INT64_MAX;
    if (v)
        for (int lanes = 32; lanes >= 8; lanes /= 2)
            for (int n = 1; n <= 3; ++n) {
                const long long room = (long long)lanes * n * unit * pl.vec;
                if (room >= d->C && room < least) { least = room; pl.lanes = lanes; pl.nv = n * unit; }
            }
    else
        for (int n : {4, 16})
            if (!pl.lanes && d->C <= 32 * n) { pl.lanes = 32; pl.nv = n; }
    if (pl.lanes) return pl;
    pl.nv = v ? 2 * unit : d->C <= 4096 ? 8 : 16;         // (single values: fewer a lane leave registers for more warps)
    pl.threads = (d->C + pl.vec * pl.nv * 32 - 1) / (pl.vec * pl.nv * 32) * 32;
    if (pl.threads > 512) { pl.lanes = -1; pl.threads = kLongThreads; }
    return pl;
}
// Calls fn(element, values of a load, lanes, loads of a lane, flag) with the plan's.
template <typename F>
static int for_ln(const m2d_ln_desc* d, const LnPlan& pl, bool flag, F fn) {
    using std::integral_constant;
    auto go = [&](auto elem, auto full) {
        constexpr int V = decltype(full)::value, unit = V == 4 ? 2 : 1;
        auto with = [&](auto v, auto lanes, auto nv) { return flag ? fn(elem, v, lanes, nv, std::true_type{}) : fn(elem, v, lanes, nv, std::false_type{}); };
        constexpr integral_constant<int, 0> cta{};
        constexpr integral_constant<int, 1> one{};
        constexpr integral_constant<int, 4> four{};
        constexpr integral_constant<int, 16> sixteen{};
        constexpr integral_constant<int, 32> warp{};
        if (pl.vec == 1) return pl.lanes == 0 ? (pl.nv == 8 ? with(one, cta, integral_constant<int, 8>{}) : with(one, cta, sixteen)) : pl.nv == 4 ? with(one, warp, four) : with(one, warp, sixteen);
        if (pl.lanes == 0) return with(full, cta, integral_constant<int, 2 * unit>{});
        auto with_lanes = [&](auto lanes) {
            return pl.nv == unit ? with(full, lanes, integral_constant<int, unit>{}) : pl.nv == 2 * unit ? with(full, lanes, integral_constant<int, 2 * unit>{}) : with(full, lanes, integral_constant<int, 3 * unit>{});
        };
        return pl.lanes == 8 ? with_lanes(integral_constant<int, 8>{}) : pl.lanes == 16 ? with_lanes(sixteen) : with_lanes(warp);
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
// CTAs of a launch: what the SMs hold at once.
static long long ln_grid(const m2d_ln_desc* d, const LnPlan& pl, int per_sm) { return std::min<long long>((d->N + pl.rows() - 1) / pl.rows(), (long long)std::max(1, per_sm) * sm_count()); }
// Calls fn(kernel, CTAs) of the backward pass.
template <typename F>
static int with_ln_bwd(const m2d_ln_desc* d, F fn) {
    const LnPlan pl = plan_ln(d, true);
    const bool params = d->d_weight || d->d_bias;
    if (pl.lanes < 0) {
        const long long grid = ln_grid(d, pl, 2);
        return d->dtype == M2D_F32 ? fn(ln_long_bwd_kernel<float>, pl, grid, (size_t)0, 0) : fn(ln_long_bwd_kernel<__nv_bfloat16>, pl, grid, (size_t)0, 0);
    }
    return for_ln(d, pl, d->d_sum != nullptr, [&](auto elem, auto vec, auto lanes, auto nv, auto ds) {
        auto kern = ln_bwd_kernel<decltype(elem), decltype(vec)::value, decltype(lanes)::value, decltype(nv)::value, decltype(ds)::value>;
        constexpr int V = decltype(vec)::value, R = decltype(lanes)::value, NV = decltype(nv)::value;
        using Way = Rows<decltype(elem), V, R, NV, decltype(ds)::value ? 3 : 2>;
        const size_t rows = Way::bytes(d->C, pl.threads), last = R && params ? (size_t)kLnThreads / 32 * 2 * R * NV * V * sizeof(float) : 0;
        const size_t smem = std::max(rows, last);
        if (!allow_smem(reinterpret_cast<const void*>(kern), smem + kLnStatic)) return (int)M2D_ERR_LAUNCH;
        return fn(kern, pl, ln_grid(d, pl, resident_ctas(reinterpret_cast<const void*>(kern), pl.threads, smem)), smem, Way::stages(d->C));
    });
}

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_ln_bwd_workspace(const m2d_ln_desc* d) {
    if (check_ln(d) != M2D_OK || (!d->d_weight && !d->d_bias)) return 0;
    uint64_t bytes = 0;
    with_ln_bwd(d, [&](auto, const LnPlan&, long long grid, size_t, int) {
        bytes = (uint64_t)grid * 2 * d->C * sizeof(float);
        return (int)M2D_OK;
    });
    return bytes;
}

extern "C" int m2d_ln_fwd(const m2d_ln_desc* d, void* stream) {
    const int rc = check_ln(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->y || (d->residual && !d->sum)) return M2D_ERR_NULL;
    LnArgs a = ln_args(d);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const LnPlan pl = plan_ln(d, false);
    if (pl.lanes < 0) {
        const unsigned grid = (unsigned)ln_grid(d, pl, 4);
        if (d->dtype == M2D_F32) ln_long_fwd_kernel<float><<<grid, kLongThreads, 0, st>>>(a);
        else ln_long_fwd_kernel<__nv_bfloat16><<<grid, kLongThreads, 0, st>>>(a);
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    }
    return for_ln(d, pl, d->residual != nullptr, [&](auto elem, auto vec, auto lanes, auto nv, auto res) {
        auto kern = ln_fwd_kernel<decltype(elem), decltype(vec)::value, decltype(lanes)::value, decltype(nv)::value, decltype(res)::value>;
        using Way = Rows<decltype(elem), decltype(vec)::value, decltype(lanes)::value, decltype(nv)::value, decltype(res)::value ? 2 : 1>;
        const size_t smem = Way::bytes(d->C, pl.threads);
        a.stages = Way::stages(d->C);
        if (!allow_smem(reinterpret_cast<const void*>(kern), smem + kLnStatic)) return (int)M2D_ERR_LAUNCH;
        kern<<<(unsigned)ln_grid(d, pl, resident_ctas(reinterpret_cast<const void*>(kern), pl.threads, smem)), pl.threads, smem, st>>>(a);
        return cudaGetLastError() == cudaSuccess ? (int)M2D_OK : (int)M2D_ERR_LAUNCH;
    });
}

extern "C" int m2d_ln_bwd(const m2d_ln_desc* d, void* stream) {
    const int rc = check_ln(d);
    if (rc != M2D_OK) return rc;
    if (!d->x || !d->stats || !d->d_y || !d->d_x) return M2D_ERR_NULL;
    LnArgs a = ln_args(d);
    const bool params = d->d_weight || d->d_bias;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int done = with_ln_bwd(d, [&](auto kern, const LnPlan& pl, long long grid, size_t smem, int stages) {
        if (params && (!d->workspace || d->workspace_bytes < (uint64_t)grid * 2 * d->C * sizeof(float) || (reinterpret_cast<uintptr_t>(d->workspace) & 255))) return (int)M2D_ERR_WORKSPACE;
        a.partial = params ? static_cast<float*>(d->workspace) : nullptr;
        a.parts = (int)grid;
        a.stages = stages;
        kern<<<a.parts, pl.threads, smem, st>>>(a);
        return cudaGetLastError() == cudaSuccess ? (int)M2D_OK : (int)M2D_ERR_LAUNCH;
    });
    if (done != M2D_OK || !params) return done;
    const dim3 grid((d->C + 31) / 32, 2);
    const bool f32 = d->params_f32 || d->dtype == M2D_F32;
    if (!(f32 ? launch_following(ln_params_kernel<float>, grid, dim3(1024), 0, st, a) : launch_following(ln_params_kernel<__nv_bfloat16>, grid, dim3(1024), 0, st, a))) return M2D_ERR_LAUNCH;
    return M2D_OK;
}
