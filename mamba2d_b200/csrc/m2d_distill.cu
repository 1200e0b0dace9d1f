// Distillation from a teacher's top logits, forward and backward.
//
//   q = softmax(z / tau) over all classes,  p = softmax(t / tau) over the teacher's entries
//   loss = (1 - w) tau^2 sum_k p_k (log p_k - log q_{i_k}) + w (log sum_j exp(z_j) - z_label)
//   dz_j = up ((1 - w) tau (q_j - sum_{k: i_k = j} p_k) + w (softmax(z)_j - [j = label]))
//
// One pass over the rows with running maxima and sums: by a warp each where rows are short; else all rows are cut into pieces, every CTA takes as
// many neighbouring ones as any other, whatever rows they belong to, and a second launch joins what they found.  The backward pass reads a row once more
// and writes its gradient; the few entries that the teacher or the label touch are written again
// behind it, the first of entries with one index for all of them, so that every value is rounded once and does not depend on
// any order.  Exponents are (z - max) c with c = log2(e) / tau: exact where all values are equal, also at the type's lowest.  What is left of a row
// (its sums' logarithms, the teacher's entries) is summed in 64 bits: a loss is a small difference of large logarithms.
// Measured, bf16: 2048x131072 forward 95 us (5.7 TB/s), backward 176 (6.1); 2047x50001 with labels at temperature 2 44 (4.6; its exponentials alone 23) and 76
// us (5.4).
#include "follow.cuh"
#include "packed.cuh"
#include "plan.cuh"
#include "m2d_seq.h"

#include <cfloat>

namespace m2d {

struct DistillArgs {
    const void *z, *t, *index, *labels;
    long long zp, tp, ip;              // rows apart, in elements
    const float* up;
    long long upp;
    float *loss, *stats;
    void* dz;
    long long N;
    int V, K, t_f32, index64, labels64, same_phase;
    float tau, w, c, c1;               // log2(e) / tau, log2(e)
    double exact_c;                    // c for what is summed in 64 bits
    float4* found;                     // forward by pieces: largest value and sums of a CTA's share of a row, at [row + CTA]
    int pieces, ctas;                  // pieces of a row
};
// Exponentials of a value: at one temperature, at tau and at 1, or at 2 and at 1, whose second is the first one's square.
enum { kOne = 0, kTwo = 1, kSquare = 2 };
// Of a row, for the backward pass: max, 1 / sum at tau, 1 / sum at 1, the teacher's largest logit, 1 / the teacher's sum (0: no entries).
constexpr int kRowStats = 8;
constexpr int kRowCta = 256;           // threads of a CTA that works on one row
constexpr int kRowWarps = 4;           // rows of a CTA whose warps work on one row each

template <typename T> struct Vec16;    // 16 bytes
template <> struct Vec16<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }       // -inf: adds nothing
    static __device__ __forceinline__ void get(const uint4& r, Num<2>* v) { v[0] = Num<2>::make(__uint_as_float(r.x), __uint_as_float(r.y)); v[1] = Num<2>::make(__uint_as_float(r.z), __uint_as_float(r.w)); }
    static __device__ __forceinline__ uint4 put(const Num<2>* v) {
        return make_uint4(__float_as_uint(v[0].get(0)), __float_as_uint(v[0].get(1)), __float_as_uint(v[1].get(0)), __float_as_uint(v[1].get(1)));
    }
    static __device__ __forceinline__ float most(const uint4& r, float m) {
        return fmaxf(fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w))), m);
    }
};
template <> struct Vec16<__nv_bfloat16> {
    static constexpr int n = 8;
    static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
    static __device__ __forceinline__ void get(const uint4& r, Num<2>* v) {
        const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = Num<2>::make(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    }
    static __device__ __forceinline__ uint4 put(const Num<2>* v) {
        return make_uint4(pack_bf16x2(v[0].get(0), v[0].get(1)), pack_bf16x2(v[1].get(0), v[1].get(1)), pack_bf16x2(v[2].get(0), v[2].get(1)), pack_bf16x2(v[3].get(0), v[3].get(1)));
    }
    static __device__ __forceinline__ unsigned two(unsigned a, unsigned b) {
        unsigned r;
        asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float most(const uint4& r, float m) {
        const unsigned t = two(two(r.x, r.y), two(r.z, r.w));
        return fmaxf(fmaxf(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u)), m);
    }
};
__device__ __forceinline__ float number(const float* p) { return *p; }
__device__ __forceinline__ float number(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// A row cut into a head before the first 16-byte boundary, whole pieces, and a tail.
template <typename T>
struct RowCut {
    int head, pieces, tail;            // elements, pieces, first element of the tail
    __device__ __forceinline__ RowCut(const T* row, int V) {
        head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T));
        pieces = (V - head) / Vec16<T>::n;
        tail = head + pieces * Vec16<T>::n;
    }
};

// Largest value so far, and sums of exp2((z - max) c) at tau and at 1.
template <int MODE>
struct Running {
    float m = -3.402823466e38f;
    Num<2> s = Num<2>::all(0.f), s1 = Num<2>::all(0.f);
    __device__ __forceinline__ void raise(float to, float c, float c1) {
        const float n = fmaxf(m, to), f = ex2((m - n) * c);
        s = mul_(s, Num<2>::all(f));
        if constexpr (MODE == kTwo) s1 = mul_(s1, Num<2>::all(ex2((m - n) * c1)));
        if constexpr (MODE == kSquare) s1 = mul_(s1, Num<2>::all(f * f));
        m = n;
    }
    __device__ __forceinline__ void add(Num<2> z, float c, float c1) {
        const Num<2> d = add_(z, Num<2>::all(-m)), x = mul_(d, Num<2>::all(c)), e = Num<2>::make(ex2(x.get(0)), ex2(x.get(1)));
        s = add_(s, e);
        if constexpr (MODE == kTwo) {
            const Num<2> x1 = mul_(d, Num<2>::all(c1));
            s1 = add_(s1, Num<2>::make(ex2(x1.get(0)), ex2(x1.get(1))));
        }
        if constexpr (MODE == kSquare) s1 = fma_(e, e, s1);
    }
    __device__ __forceinline__ void one(float z, float c, float c1) {
        raise(z, c, c1);
        add(Num<2>::make(z, -__int_as_float(0x7f800000)), c, c1);
    }
    __device__ __forceinline__ float4 found() const { return make_float4(m, s.get(0) + s.get(1), s1.get(0) + s1.get(1), 0.f); }
};
// Two shares of a row as one; the same on both sides of an exchange, to the last bit.
template <int MODE>
__device__ __forceinline__ float4 joined(const float4& a, const float4& b, float c, float c1) {
    const float n = fmaxf(a.x, b.x), f = ex2((a.x - n) * c), g = ex2((b.x - n) * c);
    float4 r = make_float4(n, __fadd_rn(__fmul_rn(a.y, f), __fmul_rn(b.y, g)), 0.f, 0.f);
    if constexpr (MODE != kOne) {
        const float f1 = MODE == kSquare ? f * f : ex2((a.x - n) * c1), g1 = MODE == kSquare ? g * g : ex2((b.x - n) * c1);
        r.z = __fadd_rn(__fmul_rn(a.z, f1), __fmul_rn(b.z, g1));
    }
    return r;
}
template <int MODE>
__device__ __forceinline__ float4 join_lanes(float4 r, float c, float c1, int lanes = 32) {
    for (int k = lanes / 2; k; k >>= 1) {
        const float4 o = make_float4(__shfl_xor_sync(0xffffffffu, r.x, k), __shfl_xor_sync(0xffffffffu, r.y, k), MODE != kOne ? __shfl_xor_sync(0xffffffffu, r.z, k) : 0.f, 0.f);
        r = joined<MODE>(r, o, c, c1);
    }
    return r;
}

__device__ __forceinline__ long long whole_at(const void* p, int is64, long long i) { return is64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i]; }
__device__ __forceinline__ float teacher_at(const DistillArgs& p, long long row, int k) {
    return p.t_f32 ? static_cast<const float*>(p.t)[row * p.tp + k] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.t)[row * p.tp + k]);
}
__device__ __forceinline__ int entry_at(const DistillArgs& p, long long row, int k) {        // -1: absent
    const long long i = whole_at(p.index, p.index64, row * p.ip + k);
    return i >= 0 && i < p.V ? (int)i : -1;
}
__device__ __forceinline__ int label_of(const DistillArgs& p, long long row) {               // -1: none
    if (!p.labels) return -1;
    const long long i = whole_at(p.labels, p.labels64, row);
    return i >= 0 && i < p.V ? (int)i : -1;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int k = 16; k; k >>= 1) v += __shfl_xor_sync(0xffffffffu, v, k);
    return v;
}

// What the teacher's entries give, by a warp and without the row's own sums: the largest logits, its and the student's, among them, the sum of
// 2^(t - top) and that of 2^(t - top) (log2 p + log2 of the sum - (z - high) c).
struct Taught {
    float top, high;
    double sum, dot;
    bool any;
};
template <typename T>
__device__ __forceinline__ Taught teach(const DistillArgs& p, long long row, const T* z) {
    const int lane = threadIdx.x & 31;
    const float low = -__int_as_float(0x7f800000);
    Taught r{low, low, 0.0, 0.0, false};
    for (int k = lane; k < p.K; k += 32) {
        const int i = entry_at(p, row, k);
        if (i < 0) continue;
        const float t = teacher_at(p, row, k);
        r.any = r.any || t != low;                     // (a NaN is there too)
        r.top = fmaxf(r.top, t);
        r.high = fmaxf(r.high, number(z + i));
    }
#pragma unroll
    for (int k = 16; k; k >>= 1) {
        r.top = fmaxf(r.top, __shfl_xor_sync(0xffffffffu, r.top, k));
        r.high = fmaxf(r.high, __shfl_xor_sync(0xffffffffu, r.high, k));
    }
    if (r.high == low) r.high = 0.f;
    r.any = __any_sync(0xffffffffu, r.any) && p.w < 1.f;
    if (r.any) {
        for (int k = lane; k < p.K; k += 32) {
            const int i = entry_at(p, row, k);
            if (i < 0) continue;
            const double a = ((double)teacher_at(p, row, k) - (double)r.top) * p.exact_c, e = exp2(a);
            r.sum += e;
            if (e != 0.0) r.dot += e * (a - ((double)number(z + i) - (double)r.high) * p.exact_c);
        }
        r.sum = warp_sum(r.sum);
        r.dot = warp_sum(r.dot);
    }
    return r;
}
// The loss of a row from its sums, by a warp.
template <int MODE>
__device__ __forceinline__ void finish_row(const DistillArgs& p, long long row, const Taught& t, int label, float at_label, const float4& r) {
    const float at_one = MODE != kOne ? r.z : r.y;
    if ((threadIdx.x & 31) != 0) return;
    double loss = 0.0;
    if (t.any)       // (dot is about `high`: exact where everything is at the type's lowest)
        loss = (1.0 - (double)p.w) * (double)p.tau * (double)p.tau * 0.6931471805599453 * (t.dot / t.sum + ((double)r.x - (double)t.high) * p.exact_c - log2(t.sum) + log2((double)r.y));
    if (label >= 0) loss += (double)p.w * (log((double)at_one) - ((double)at_label - (double)r.x));
    p.loss[row] = (float)loss;
    if (p.stats) {
        float* const s = p.stats + row * kRowStats;
        s[0] = r.x;
        s[1] = 1.f / r.y;
        s[2] = 1.f / at_one;
        s[3] = t.top;
        s[4] = t.any ? (float)(1.0 / t.sum) : 0.f;
    }
}

// 16-byte pieces first, first + step, ... below `end` of a row's body.
template <typename T, int MODE>
__device__ __forceinline__ void read_pieces(const uint4* body, int first, int step, int end, float c, float c1, Running<MODE>& r) {
    using W = Vec16<T>;
    constexpr int U = 4;
    auto batch = [&](int i, auto whole) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!whole.value) raw[u] = W::none();
            if (whole.value || i + u * step < end) raw[u] = __ldcs(body + i + u * step);
        }
        float top = r.m;
#pragma unroll
        for (int u = 0; u < U; ++u) top = W::most(raw[u], top);
        r.raise(top, c, c1);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Num<2> v[W::n / 2];
            W::get(raw[u], v);
#pragma unroll
            for (int k = 0; k < W::n / 2; ++k) r.add(v[k], c, c1);
        }
    };
    int i = first;
    for (; i < end - (U - 1) * step; i += U * step) batch(i, std::true_type{});
    if (i < end) batch(i, std::false_type{});
}
// A row's head and tail, by threads of which this is number `me`.
template <typename T, int MODE>
__device__ __forceinline__ void read_ends(const T* z, const RowCut<T>& cut, int V, int me, float c, float c1, Running<MODE>& r) {
    if (me < cut.head) r.one(number(z + me), c, c1);
    if (me < V - cut.tail) r.one(number(z + cut.tail + me), c, c1);
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kRowWarps * 32) distill_fwd_warp_kernel(const DistillArgs p) {
    const long long row = (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    if (row >= p.N) return;
    const int lane = threadIdx.x & 31;
    const T* const z = static_cast<const T*>(p.z) + row * p.zp;
    const RowCut<T> cut(z, p.V);
    Running<MODE> r;
    read_pieces<T, MODE>(reinterpret_cast<const uint4*>(z + cut.head), lane, 32, cut.pieces, p.c, p.c1, r);
    read_ends<T, MODE>(z, cut, p.V, lane, p.c, p.c1, r);
    const float4 all = join_lanes<MODE>(r.found(), p.c, p.c1);
    const Taught t = teach(p, row, z);
    const int label = label_of(p, row);
    finish_row<MODE>(p, row, t, label, label >= 0 ? number(z + label) : 0.f, all);
}

// All rows' pieces of kRowCta * UNIT times 16 bytes in order; CTA k of n has those from k total / n on.
template <typename T, int MODE, int UNIT>
__global__ void __launch_bounds__(kRowCta) distill_fwd_kernel(const DistillArgs p) {
    __shared__ float4 part[2][kRowCta / 32];
    let_follow();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long total = p.N * p.pieces, end = (blockIdx.x + 1ll) * total / p.ctas;
    long long at = blockIdx.x * total / p.ctas;
    for (int buf = 0; at < end; buf ^= 1) {
        const long long row = at / p.pieces;
        const int first = (int)(at - row * p.pieces), last = (int)min((long long)p.pieces, first + end - at);
        const T* const z = static_cast<const T*>(p.z) + row * p.zp;
        const RowCut<T> cut(z, p.V);
        Running<MODE> r;
        read_pieces<T, MODE>(reinterpret_cast<const uint4*>(z + cut.head), first * kRowCta * UNIT + threadIdx.x, kRowCta, min(cut.pieces, last * kRowCta * UNIT), p.c, p.c1, r);
        if (first == 0) read_ends<T, MODE>(z, cut, p.V, threadIdx.x, p.c, p.c1, r);
        const float4 f = join_lanes<MODE>(r.found(), p.c, p.c1);
        if (lane == 0) part[buf][warp] = f;
        __syncthreads();
        if (warp == 0) {
            const float4 whole = join_lanes<MODE>(part[buf][lane % (kRowCta / 32)], p.c, p.c1, kRowCta / 32);
            if (lane == 0) p.found[row + blockIdx.x] = whole;
        }
        at += last - first;
    }
}
// Joins the shares of a row, a warp a row.
template <typename T, int MODE>
__global__ void __launch_bounds__(kRowWarps * 32) distill_join_kernel(const DistillArgs p) {
    const long long row = (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    if (row >= p.N) return follow_wait();
    const int lane = threadIdx.x & 31;
    // (inputs: written before the launch that this one follows)
    const T* const z = static_cast<const T*>(p.z) + row * p.zp;
    const int label = label_of(p, row);
    const float at_label = label >= 0 ? number(z + label) : 0.f;
    const Taught t = teach(p, row, z);
    follow_wait();
    const long long total = p.N * p.pieces;
    // the CTAs of its first piece and of its last: k total / n <= piece < (k + 1) total / n
    const long long a = ((row * p.pieces + 1) * p.ctas - 1) / total, b = ((row + 1) * p.pieces * p.ctas - 1) / total;
    float4 r = make_float4(-3.402823466e38f, 0.f, 0.f, 0.f);
    for (long long k = a + lane; k <= b; k += 32) r = joined<MODE>(r, p.found[row + k], p.c, p.c1);
    finish_row<MODE>(p, row, t, label, at_label, join_lanes<MODE>(r, p.c, p.c1));
}

// ---- backward -------------------------------------------------------------------------------------

// dz_j of a row: a * 2^((z - m) c) + b * 2^((z - m) c1), less what the teacher and the label take.
template <int MODE>
struct Slope {
    float m, a, b, c, c1;
    __device__ __forceinline__ Num<2> operator()(Num<2> z) const {
        const Num<2> d = add_(z, Num<2>::all(-m)), x = mul_(d, Num<2>::all(c)), e = Num<2>::make(ex2(x.get(0)), ex2(x.get(1)));
        if constexpr (MODE == kOne) return mul_(e, Num<2>::all(a));
        if constexpr (MODE == kSquare) return mul_(e, fma_(e, Num<2>::all(b), Num<2>::all(a)));
        const Num<2> x1 = mul_(d, Num<2>::all(c1));
        return fma_(Num<2>::make(ex2(x1.get(0)), ex2(x1.get(1))), Num<2>::all(b), mul_(e, Num<2>::all(a)));
    }
    __device__ __forceinline__ float operator()(float z) const { return (*this)(Num<2>::all(z)).get(0); }
};

// What a row's gradient is made of.
template <int MODE>
struct RowSlope {
    Slope<MODE> f;
    float teach, hard, top, share;         // of the teacher's and of the label's share of the loss; the teacher's largest logit and 1 / its sum
    int label;                             // -1: none
    bool has, zero;                        // whether there is a teacher; whether there is nothing to learn from
    __device__ __forceinline__ RowSlope(const DistillArgs& p, long long row) {
        const float* const st = p.stats + row * kRowStats;
        const float up = p.up[row * p.upp];
        teach = up * (1.f - p.w) * p.tau;
        hard = up * p.w;
        top = st[3];
        share = st[4];
        label = label_of(p, row);
        has = share != 0.f;                // (NaN: there is one)
        zero = !has && label < 0;
        f = Slope<MODE>{st[0], has ? teach * st[1] : 0.f, label >= 0 ? hard * st[2] : 0.f, p.c, p.c1};
        if (MODE == kOne) f.a += f.b;
    }
};
// 16-byte pieces [b0, b1) of a row's body and, where `ends`, its head and tail, by `threads` threads of which this is number `me`: as if there were
// neither list nor label.
template <typename T, int MODE>
__device__ __forceinline__ void write_dense(const DistillArgs& p, const RowSlope<MODE>& s, const T* z, T* out, const RowCut<T>& cut, int b0, int b1, bool ends, int me, int threads) {
    using W = Vec16<T>;
    if (p.same_phase) {
        const uint4* const body = reinterpret_cast<const uint4*>(z + cut.head);
        uint4* const to = reinterpret_cast<uint4*>(out + cut.head);
        constexpr int U = 4;
        for (int i = b0 + me; i < b1; i += U * threads) {
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * threads < b1) raw[u] = __ldcs(body + i + u * threads);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u * threads >= b1) break;
                Num<2> v[W::n / 2];
                W::get(raw[u], v);
#pragma unroll
                for (int k = 0; k < W::n / 2; ++k) v[k] = s.f(v[k]);
                to[i + u * threads] = s.zero ? make_uint4(0, 0, 0, 0) : W::put(v);
            }
        }
    } else {
        for (int i = cut.head + b0 * W::n + me; i < cut.head + b1 * W::n; i += threads) store1(out, i, s.zero ? 0.f : s.f(number(z + i)));
    }
    if (!ends) return;
    if (me < cut.head) store1(out, me, s.zero ? 0.f : s.f(number(z + me)));
    if (me < p.V - cut.tail) store1(out, cut.tail + me, s.zero ? 0.f : s.f(number(z + cut.tail + me)));
}
// The entries that the teacher or the label touch, by a warp, of those that are mine(index): the first of entries with one index for all of them.
// list: 2 K words of shared memory.
template <typename T, int MODE, typename Mine>
__device__ __forceinline__ void write_listed(const DistillArgs& p, const RowSlope<MODE>& s, long long row, const T* z, T* out, int* list, Mine mine) {
    const int lane = threadIdx.x & 31;
    float* const shares = reinterpret_cast<float*>(list + p.K);
    if (s.has)
        for (int k = lane; k < p.K; k += 32) {
            const int i = entry_at(p, row, k);
            list[k] = i;
            shares[k] = i >= 0 ? ex2((teacher_at(p, row, k) - s.top) * p.c) * s.share : 0.f;
        }
    __syncwarp();
    bool listed = false;
    if (s.has)
        for (int k = lane; k < p.K; k += 32) {
            const int i = list[k];
            if (i < 0 || !mine(i)) continue;
            listed = listed || i == s.label;
            const float value = s.f(number(z + i));
            float take = 0.f;
            bool first = true;
#pragma unroll 4
            for (int j = 0; j < p.K; ++j)
                if (list[j] == i) {
                    first = first && j >= k;
                    take += shares[j];
                }
            if (first) store1(out, i, value - s.teach * take - (i == s.label ? s.hard : 0.f));
        }
    if (s.label >= 0 && mine(s.label) && !__any_sync(0xffffffffu, listed) && lane == 0) store1(out, s.label, s.f(number(z + s.label)) - s.hard);
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kRowWarps * 32) distill_bwd_warp_kernel(const DistillArgs p) {
    extern __shared__ int lists[];
    const int warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * kRowWarps + warp;
    if (row >= p.N) return;
    const T* const z = static_cast<const T*>(p.z) + row * p.zp;
    T* const out = static_cast<T*>(p.dz) + row * p.V;
    const RowSlope<MODE> s(p, row);
    const RowCut<T> cut(z, p.V);
    write_dense<T, MODE>(p, s, z, out, cut, 0, cut.pieces, true, threadIdx.x & 31, 32);
    __syncwarp();
    write_listed<T, MODE>(p, s, row, z, out, lists + warp * 2 * p.K, [](int) { return true; });
}
// CTAs of a row have p.pieces loads of 16 bytes each; the listed entries among a CTA's own are written by its first warp behind the rest.
template <typename T, int MODE>
__global__ void __launch_bounds__(kRowCta) distill_bwd_kernel(const DistillArgs p) {
    extern __shared__ int lists[];
    const long long row = blockIdx.x / p.ctas;
    const int part = blockIdx.x % p.ctas;
    const T* const z = static_cast<const T*>(p.z) + row * p.zp;
    T* const out = static_cast<T*>(p.dz) + row * p.V;
    const RowCut<T> cut(z, p.V);
    const int b0 = min(cut.pieces, part * p.pieces), b1 = part + 1 < p.ctas ? min(cut.pieces, b0 + p.pieces) : cut.pieces;
    const RowSlope<MODE> s(p, row);
    write_dense<T, MODE>(p, s, z, out, cut, b0, b1, part == 0, threadIdx.x, kRowCta);
    __syncthreads();
    if (threadIdx.x < 32)
        write_listed<T, MODE>(p, s, row, z, out, lists, [&](int i) {
            const int piece = (i - cut.head) / Vec16<T>::n;
            return i < cut.head || i >= cut.tail ? part == 0 : piece >= b0 && piece < b1;
        });
}

// ---- host ---------------------------------------------------------------------------------------

static int check_distill(const m2d_distill_desc* d) {
    if (!d) return M2D_ERR_NULL;
    if (d->struct_bytes != sizeof(m2d_distill_desc)) return M2D_ERR_ABI;
    for (int t : {d->dtype, d->teacher_dtype})
        if (t != M2D_F32 && t != M2D_BF16) return M2D_ERR_DTYPE;
    if (d->N < 1 || d->V < 1 || d->K < 1) return M2D_ERR_SHAPE;
    if (d->N > INT32_MAX / 64 || d->V > INT32_MAX - (1 << 16) || d->K > M2D_DISTILL_MAX_TOP) return M2D_ERR_TOO_LARGE;
    if (!(d->temperature > 0.f) || d->temperature > 3.4e38f || !(d->label_weight >= 0.f && d->label_weight <= 1.f)) return M2D_ERR_FLAGS;
    if (!d->logits || !d->teacher || !d->index || (d->label_weight > 0.f && !d->labels)) return M2D_ERR_NULL;
    const uintptr_t es = d->dtype == M2D_F32 ? 4 : 2;
    auto off = [](const void* p, uintptr_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
    if (off(d->logits, es) || off(d->d_logits, es) || off(d->teacher, d->teacher_dtype == M2D_F32 ? 4 : 2) || off(d->index, d->index_64 ? 8 : 4) || off(d->labels, d->labels_64 ? 8 : 4) ||
        off(d->loss, 4) || off(d->stats, 4) || off(d->d_loss, 4))
        return M2D_ERR_PITCH;
    return M2D_OK;
}
static DistillArgs distill_args(const m2d_distill_desc* d) {
    DistillArgs a{};
    a.z = d->logits; a.zp = d->logits_row;
    a.t = d->teacher; a.tp = d->teacher_row; a.t_f32 = d->teacher_dtype == M2D_F32;
    a.index = d->index; a.ip = d->index_row; a.index64 = d->index_64;
    a.labels = d->label_weight > 0.f ? d->labels : nullptr; a.labels64 = d->labels_64;
    a.up = d->d_loss; a.upp = d->d_loss_row;
    a.loss = d->loss; a.stats = d->stats; a.dz = d->d_logits;
    a.N = d->N; a.V = d->V; a.K = d->K;
    a.tau = d->temperature; a.w = d->label_weight;
    a.c1 = kLog2e; a.exact_c = 1.4426950408889634 / (double)d->temperature; a.c = std::min((float)a.exact_c, FLT_MAX);        // (an infinite one would make NaN of the largest value's zero)
    return a;
}
// A warp for a row of up to 8 KB, whose loads would be two of a CTA's threads at most, and of up to 32 KB where rows are enough to fill the
// GPU with warps (7361x7552 bf16, forward and backward: 100 us, by CTAs 150).
static bool short_rows(const m2d_distill_desc* d) {
    const long long bytes = (long long)d->V * (d->dtype == M2D_F32 ? 4 : 2);
    return bytes <= 8192 || (bytes <= 32768 && d->N >= 24ll * sm_count());
}
template <typename F>
static int for_distill(const m2d_distill_desc* d, F fn) {
    using std::integral_constant;
    auto with = [&](auto elem) {
        // two exponentials where temperatures differ and both are wanted
        if (d->label_weight == 0.f || d->temperature == 1.f) return fn(elem, integral_constant<int, kOne>{});
        return d->temperature == 2.f ? fn(elem, integral_constant<int, kSquare>{}) : fn(elem, integral_constant<int, kTwo>{});
    };
    return d->dtype == M2D_F32 ? with(float{}) : with(__nv_bfloat16{});
}
// Pieces of 16 KB and CTAs as many as the GPU may hold; pieces of 4 KB where there are too few of those.
struct DistillPlan { int unit, pieces, ctas; };
static DistillPlan plan_distill(const m2d_distill_desc* d) {
    const int loads = d->V / (d->dtype == M2D_F32 ? 4 : 8);
    const long long most = 8ll * sm_count();
    DistillPlan pl{};
    for (pl.unit = 4; pl.unit >= 1; pl.unit -= 3) {
        pl.pieces = std::max(1, (loads + kRowCta * pl.unit - 1) / (kRowCta * pl.unit));
        pl.ctas = (int)std::min<long long>(most, d->N * pl.pieces);
        if (pl.ctas == most) break;
    }
    pl.unit = std::max(1, pl.unit);
    return pl;
}

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_distill_stats(const m2d_distill_desc* d) { return d && d->N > 0 ? (uint64_t)d->N * kRowStats : 0; }

extern "C" uint64_t m2d_distill_fwd_workspace(const m2d_distill_desc* d) {
    return d && d->N > 0 && d->V > 0 && !short_rows(d) ? (uint64_t)(d->N + plan_distill(d).ctas) * sizeof(float4) : 0;
}

extern "C" int m2d_distill_fwd(const m2d_distill_desc* d, void* stream) {
    const int rc = check_distill(d);
    if (rc != M2D_OK) return rc;
    if (!d->loss) return M2D_ERR_NULL;
    if (!short_rows(d) && (!d->workspace || d->workspace_bytes < m2d_distill_fwd_workspace(d) || (reinterpret_cast<uintptr_t>(d->workspace) & 255))) return M2D_ERR_WORKSPACE;
    DistillArgs a = distill_args(d);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return for_distill(d, [&](auto elem, auto mode) {
        using T = decltype(elem);
        constexpr int MODE = decltype(mode)::value;
        const unsigned warps = (unsigned)((d->N + kRowWarps - 1) / kRowWarps);
        if (short_rows(d)) {
            distill_fwd_warp_kernel<T, MODE><<<warps, kRowWarps * 32, 0, st>>>(a);
            return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
        }
        const DistillPlan pl = plan_distill(d);
        auto kern = pl.unit == 4 ? distill_fwd_kernel<T, MODE, 4> : distill_fwd_kernel<T, MODE, 1>;
        const long long held = (long long)std::max(1, resident_ctas(reinterpret_cast<const void*>(kern), kRowCta, 0)) * sm_count();
        a.pieces = pl.pieces;
        a.ctas = (int)std::min<long long>(pl.ctas, held);            // one wave
        a.found = static_cast<float4*>(d->workspace);
        kern<<<a.ctas, kRowCta, 0, st>>>(a);
        if (cudaGetLastError() != cudaSuccess || !launch_following(distill_join_kernel<T, MODE>, dim3(warps), dim3(kRowWarps * 32), 0, st, a)) return M2D_ERR_LAUNCH;
        return M2D_OK;
    });
}

extern "C" int m2d_distill_bwd(const m2d_distill_desc* d, void* stream) {
    const int rc = check_distill(d);
    if (rc != M2D_OK) return rc;
    if (!d->stats || !d->d_loss || !d->d_logits) return M2D_ERR_NULL;
    DistillArgs a = distill_args(d);
    const int es = d->dtype == M2D_F32 ? 4 : 2;
    // a row and its gradient begin at the same distance from a 16-byte boundary
    a.same_phase = (reinterpret_cast<uintptr_t>(d->logits) - reinterpret_cast<uintptr_t>(d->d_logits)) % 16 == 0 && (d->logits_row - d->V) * es % 16 == 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return for_distill(d, [&](auto elem, auto mode) {
        using T = decltype(elem);
        constexpr int MODE = decltype(mode)::value;
        const size_t smem = (size_t)kRowWarps * 2 * d->K * 4;
        const unsigned warps = (unsigned)((d->N + kRowWarps - 1) / kRowWarps);
        if (short_rows(d)) {
            distill_bwd_warp_kernel<T, MODE><<<warps, kRowWarps * 32, smem, st>>>(a);
        } else {
            // whole loads of all threads, 96 KB a CTA where there is enough to do and 16 KB where not, and a rest: 2048x131072 bf16 176 us, in equal
            // parts of about that size 194, in parts of 16 KB 212
            const long long loads = std::max(1, d->V / Vec16<T>::n);
            for (int times = 6; times >= 1; --times) {
                a.pieces = 4 * kRowCta * times;
                a.ctas = (int)((loads + a.pieces - 1) / a.pieces);
                if (d->N * a.ctas >= 8ll * sm_count()) break;
            }
            distill_bwd_kernel<T, MODE><<<(unsigned)(d->N * a.ctas), kRowCta, (size_t)2 * d->K * 4, st>>>(a);
        }
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    });
}
