// Distillation from a teacher's top logits, forward and backward.
//
//   q = softmax(z / tau) over all classes,  p = softmax(t / tau) over the teacher's entries
//   loss = (1 - w) tau^2 sum_k p_k (log p_k - log q_{i_k}) + w (log sum_j exp(z_j) - z_label)
//   dz_j = up ((1 - w) tau (q_j - sum_{k: i_k = j} p_k) + w (softmax(z)_j - [j = label]))
//
// One pass over a row with the running maximum and sums: by a warp where rows are short, by a CTA, or by a cluster of CTAs where there are few
// rows.  The backward pass reads a row once more and writes its gradient; the few entries that the teacher or the label touch are written again
// behind it by the same CTA, the first of entries with one index for all of them, so that every value is rounded once and does not depend on
// any order.  Exponents are (z - max) c with c = log2(e) / tau: exact where all values are equal, also at the type's lowest.  What is left of a row
// (its sums' logarithms, the teacher's entries) is summed in 64 bits: a loss is a small difference of large logarithms.
#include <cooperative_groups.h>

#include "follow.cuh"
#include "plan.cuh"
#include "m2d_seq.h"

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
    int parts;
};
// Of a row, for the backward pass: max, 1 / sum at tau, 1 / sum at 1, the teacher's largest logit, 1 / the teacher's sum (0: no entries).
constexpr int kRowStats = 8;
constexpr int kRowCta = 256;           // threads of a CTA that works on one row
constexpr int kRowWarps = 4;           // rows of a CTA whose warps work on one row each

template <typename T> struct Vec16;    // 16 bytes
template <> struct Vec16<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ void get(const uint4& r, float* v) { v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w); }
    static __device__ __forceinline__ uint4 put(const float* v) { return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])); }
};
template <> struct Vec16<__nv_bfloat16> {
    static constexpr int n = 8;
    static __device__ __forceinline__ void get(const uint4& r, float* v) {
        const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ uint4 put(const float* v) {
        return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
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

// Largest value so far, and sums of exp2((z - max) c) at tau and (TWO) at 1.
template <bool TWO>
struct Running {
    float m = -3.402823466e38f, s = 0.f, s1 = 0.f;
    __device__ __forceinline__ void raise(float to, float c, float c1) {
        const float n = fmaxf(m, to);
        s *= ex2((m - n) * c);
        if constexpr (TWO) s1 *= ex2((m - n) * c1);
        m = n;
    }
    __device__ __forceinline__ void add(float z, float c, float c1) {
        const float d = z - m;
        s += ex2(d * c);
        if constexpr (TWO) s1 += ex2(d * c1);
    }
    __device__ __forceinline__ void join(float om, float os, float os1, float c, float c1) {
        raise(om, c, c1);
        s = fmaf(os, ex2((om - m) * c), s);
        if constexpr (TWO) s1 = fmaf(os1, ex2((om - m) * c1), s1);
    }
};
template <bool TWO>
__device__ __forceinline__ void join_lanes(Running<TWO>& r, float c, float c1, int lanes = 32) {
    for (int k = lanes / 2; k; k >>= 1) {
        const float m = __shfl_xor_sync(0xffffffffu, r.m, k), s = __shfl_xor_sync(0xffffffffu, r.s, k), s1 = TWO ? __shfl_xor_sync(0xffffffffu, r.s1, k) : 0.f;
        // (both sides do the same operations: the lanes agree to the last bit)
        const float n = fmaxf(r.m, m), f = ex2((r.m - n) * c), g = ex2((m - n) * c);
        r.s = __fadd_rn(__fmul_rn(r.s, f), __fmul_rn(s, g));
        if constexpr (TWO) r.s1 = __fadd_rn(__fmul_rn(r.s1, ex2((r.m - n) * c1)), __fmul_rn(s1, ex2((m - n) * c1)));
        r.m = n;
    }
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

// The loss of a row from its sums, by a warp.
template <typename T, bool TWO>
__device__ __forceinline__ void finish_row(const DistillArgs& p, long long row, const T* z, const Running<TWO>& r) {
    const int lane = threadIdx.x & 31;
    const double c = p.c, m = r.m;
    float top = -__int_as_float(0x7f800000);
    bool any = false;
    for (int k = lane; k < p.K; k += 32)
        if (entry_at(p, row, k) >= 0) {
            const float t = teacher_at(p, row, k);
            any = any || t != -__int_as_float(0x7f800000);        // (a NaN is there too)
            top = fmaxf(top, t);
        }
#pragma unroll
    for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    any = __any_sync(0xffffffffu, any) && p.w < 1.f;
    double loss = 0.0;
    float part = 0.f;
    if (any) {
        double sum = 0.0, dot = 0.0;                  // of 2^(t - top) and of that times (log2 p + log2 of its sum - (z - max) c)
        for (int k = lane; k < p.K; k += 32) {
            const int i = entry_at(p, row, k);
            if (i < 0) continue;
            const double a = ((double)teacher_at(p, row, k) - (double)top) * c, e = exp2(a);
            sum += e;
            if (e != 0.0) dot += e * (a - ((double)number(z + i) - m) * c);
        }
        sum = warp_sum(sum);
        dot = warp_sum(dot);
        loss = (1.0 - (double)p.w) * (double)p.tau * (double)p.tau * 0.6931471805599453 * (dot / sum - log2(sum) + log2((double)r.s));
        part = (float)(1.0 / sum);
    }
    const int label = label_of(p, row);
    if (label >= 0) loss += (double)p.w * (log((double)(TWO ? r.s1 : r.s)) - ((double)number(z + label) - m));
    if (lane == 0) {
        p.loss[row] = (float)loss;
        if (p.stats) {
            float* const s = p.stats + row * kRowStats;
            s[0] = r.m;
            s[1] = 1.f / r.s;
            s[2] = 1.f / (TWO ? r.s1 : r.s);
            s[3] = top;
            s[4] = part;
        }
    }
}

// Every step-th piece of a row from piece `first` on, and its head and tail where `ends`.
template <typename T, bool TWO>
__device__ __forceinline__ void read_row(const T* z, int V, int first, int step, bool ends, float c, float c1, Running<TWO>& r) {
    using W = Vec16<T>;
    const RowCut<T> cut(z, V);
    const uint4* const body = reinterpret_cast<const uint4*>(z + cut.head);
    constexpr int U = 4;
    int i = first;
    for (; i < cut.pieces - (U - 1) * step; i += U * step) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = __ldcs(body + i + u * step);
        float top = r.m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[W::n];
            W::get(raw[u], v);
#pragma unroll
            for (int k = 0; k < W::n; ++k) top = fmaxf(top, v[k]);
        }
        r.raise(top, c, c1);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[W::n];
            W::get(raw[u], v);
#pragma unroll
            for (int k = 0; k < W::n; ++k) r.add(v[k], c, c1);
        }
    }
    for (; i < cut.pieces; i += step) {
        float v[W::n], top = r.m;
        W::get(__ldcs(body + i), v);
#pragma unroll
        for (int k = 0; k < W::n; ++k) top = fmaxf(top, v[k]);
        r.raise(top, c, c1);
#pragma unroll
        for (int k = 0; k < W::n; ++k) r.add(v[k], c, c1);
    }
    if (ends) {
        if (first < cut.head) { const float v = number(z + first); r.raise(v, c, c1); r.add(v, c, c1); }
        if (first < V - cut.tail) { const float v = number(z + cut.tail + first); r.raise(v, c, c1); r.add(v, c, c1); }
    }
}

template <typename T, bool TWO>
__global__ void __launch_bounds__(kRowWarps * 32) distill_fwd_warp_kernel(const DistillArgs p) {
    const long long row = (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
    if (row >= p.N) return;
    const T* const z = static_cast<const T*>(p.z) + row * p.zp;
    Running<TWO> r;
    read_row<T, TWO>(z, p.V, threadIdx.x & 31, 32, true, p.c, p.c1, r);
    join_lanes<TWO>(r, p.c, p.c1);
    finish_row<T, TWO>(p, row, z, r);
}

template <typename T, bool TWO>
__global__ void __launch_bounds__(kRowCta) distill_fwd_kernel(const DistillArgs p) {
    namespace cg = cooperative_groups;
    __shared__ float part[kRowCta / 32][3], whole[16][3];
    cg::cluster_group cluster = cg::this_cluster();
    if (p.parts > 1) cluster.barrier_arrive();           // (all have begun before one writes to another)
    const long long row = blockIdx.x / p.parts;
    const int rank = blockIdx.x % p.parts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* const z = static_cast<const T*>(p.z) + row * p.zp;
    Running<TWO> r;
    read_row<T, TWO>(z, p.V, rank * kRowCta + threadIdx.x, p.parts * kRowCta, rank == 0, p.c, p.c1, r);
    join_lanes<TWO>(r, p.c, p.c1);
    if (lane == 0) { part[warp][0] = r.m; part[warp][1] = r.s; part[warp][2] = r.s1; }
    __syncthreads();
    if (warp == 0) {
        constexpr int n = kRowCta / 32;
        r.m = part[lane % n][0]; r.s = part[lane % n][1]; r.s1 = part[lane % n][2];
        join_lanes<TWO>(r, p.c, p.c1, n);
    }
    if (p.parts > 1) {
        cluster.barrier_wait();
        if (threadIdx.x == 0) {
            float* const to = cluster.map_shared_rank(&whole[0][0], 0) + rank * 3;
            to[0] = r.m; to[1] = r.s; to[2] = r.s1;
        }
        cluster.sync();
        if (rank != 0 || warp != 0) return;
        r.m = whole[0][0]; r.s = whole[0][1]; r.s1 = whole[0][2];
        for (int k = 1; k < p.parts; ++k) r.join(whole[k][0], whole[k][1], whole[k][2], p.c, p.c1);
    }
    if (warp == 0) finish_row<T, TWO>(p, row, z, r);
}

// ---- backward -------------------------------------------------------------------------------------

// dz_j of a row: a * 2^((z - m) c) + b * 2^((z - m) c1), less what the teacher and the label take.
template <bool TWO>
struct Slope {
    float m, a, b, c, c1;
    __device__ __forceinline__ float operator()(float z) const {
        const float d = z - m, f = a * ex2(d * c);
        if constexpr (TWO) return fmaf(b, ex2(d * c1), f);
        return f;
    }
};

// A row's entries [lo, hi), by `threads` threads of which this is number `me`; sync() is theirs.  list: 2 K words of shared memory.
template <typename T, bool TWO, typename Sync>
__device__ __forceinline__ void write_row(const DistillArgs& p, long long row, int lo, int hi, int me, int threads, int* list, Sync sync) {
    using W = Vec16<T>;
    const T* const z = static_cast<const T*>(p.z) + row * p.zp;
    T* const out = static_cast<T*>(p.dz) + row * p.V;
    const float* const st = p.stats + row * kRowStats;
    const float up = p.up[row * p.upp], teach = up * (1.f - p.w) * p.tau, iP = st[4];
    const int label = label_of(p, row);
    const bool has = iP != 0.f;                           // (NaN: there is one)
    Slope<TWO> f{st[0], has ? teach * st[1] : 0.f, label >= 0 ? up * p.w * st[2] : 0.f, p.c, p.c1};
    if (!TWO) f.a += f.b;
    const bool zero = !has && label < 0;                  // nothing to learn from in this row
    int* const at = list;
    float* const share = reinterpret_cast<float*>(list + p.K);
    if (has)
        for (int k = me; k < p.K; k += threads) {
            const int i = entry_at(p, row, k);
            at[k] = i;
            share[k] = i >= 0 ? ex2((teacher_at(p, row, k) - st[3]) * p.c) * iP : 0.f;
        }
    const RowCut<T> cut(z, p.V);
    // (lo and hi lie on pieces' borders, or at the row's ends)
    const int b0 = lo ? (lo - cut.head) / W::n : 0, b1 = hi < p.V ? (hi - cut.head) / W::n : cut.pieces;
    if (p.same_phase) {
        const uint4* const body = reinterpret_cast<const uint4*>(z + cut.head);
        uint4* const to = reinterpret_cast<uint4*>(out + cut.head);
        constexpr int U = 4;
        for (int i = b0 + me; i < b1; i += U * threads) {
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = i + u * threads < b1 ? __ldcs(body + i + u * threads) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u * threads >= b1) break;
                float v[W::n];
                W::get(raw[u], v);
#pragma unroll
                for (int k = 0; k < W::n; ++k) v[k] = zero ? 0.f : f(v[k]);
                to[i + u * threads] = W::put(v);
            }
        }
    } else {
        for (int i = cut.head + b0 * W::n + me; i < cut.head + b1 * W::n; i += threads) store1(out, i, zero ? 0.f : f(number(z + i)));
    }
    if (lo == 0 && me < cut.head) store1(out, me, zero ? 0.f : f(number(z + me)));
    if (hi == p.V && me < p.V - cut.tail) store1(out, cut.tail + me, zero ? 0.f : f(number(z + cut.tail + me)));
    sync();
    if (has)
        for (int k = me; k < p.K; k += threads) {
            const int i = at[k];
            if (i < lo || i >= hi) continue;
            float take = 0.f;
            bool first = true;
            for (int j = 0; j < p.K; ++j)
                if (at[j] == i) {
                    first = first && j >= k;
                    take += share[j];
                }
            if (first) store1(out, i, f(number(z + i)) - teach * take - (i == label ? up * p.w : 0.f));
        }
    if (label >= lo && label < hi && me == 0) {
        bool listed = false;
        if (has)
            for (int j = 0; j < p.K; ++j) listed = listed || at[j] == label;
        if (!listed) store1(out, label, f(number(z + label)) - up * p.w);
    }
}

template <typename T, bool TWO>
__global__ void __launch_bounds__(kRowWarps * 32) distill_bwd_warp_kernel(const DistillArgs p) {
    extern __shared__ int lists[];
    const int warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * kRowWarps + warp;
    if (row < p.N) write_row<T, TWO>(p, row, 0, p.V, threadIdx.x & 31, 32, lists + warp * 2 * p.K, [] { __syncwarp(); });
}
template <typename T, bool TWO>
__global__ void __launch_bounds__(kRowCta) distill_bwd_kernel(const DistillArgs p) {
    extern __shared__ int lists[];
    const long long row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    const RowCut<T> cut(static_cast<const T*>(p.z) + row * p.zp, p.V);
    const int per = (cut.pieces + p.parts - 1) / p.parts;
    const int lo = part ? min(cut.tail, cut.head + part * per * Vec16<T>::n) : 0, hi = part + 1 < p.parts ? min(cut.tail, cut.head + (part + 1) * per * Vec16<T>::n) : p.V;
    write_row<T, TWO>(p, row, lo, hi, threadIdx.x, kRowCta, lists, [] { __syncthreads(); });
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
    const int es = d->dtype == M2D_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(d->logits) % es) return M2D_ERR_PITCH;
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
    a.c1 = kLog2e; a.c = (float)(1.4426950408889634 / (double)d->temperature);
    return a;
}
// A warp for a row of up to 8 KB: a CTA's threads would have less than two pieces each.
static bool short_rows(const m2d_distill_desc* d) { return (long long)d->V * (d->dtype == M2D_F32 ? 4 : 2) <= 8192; }
template <typename F>
static int for_distill(const m2d_distill_desc* d, F fn) {
    // both temperatures where they differ and both are wanted
    const bool two = d->label_weight > 0.f && d->temperature != 1.f;
    if (d->dtype == M2D_F32) return two ? fn(float{}, std::true_type{}) : fn(float{}, std::false_type{});
    return two ? fn(__nv_bfloat16{}, std::true_type{}) : fn(__nv_bfloat16{}, std::false_type{});
}

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_distill_stats(const m2d_distill_desc* d) { return d && d->N > 0 ? (uint64_t)d->N * kRowStats : 0; }

extern "C" int m2d_distill_fwd(const m2d_distill_desc* d, void* stream) {
    const int rc = check_distill(d);
    if (rc != M2D_OK) return rc;
    if (!d->loss) return M2D_ERR_NULL;
    DistillArgs a = distill_args(d);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return for_distill(d, [&](auto elem, auto two) {
        using T = decltype(elem);
        constexpr bool TWO = decltype(two)::value;
        if (short_rows(d)) {
            distill_fwd_warp_kernel<T, TWO><<<(unsigned)((d->N + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, st>>>(a);
            return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
        }
        // few rows: up to eight CTAs each, while a thread has two pieces or more
        a.parts = 1;
        while (a.parts < 8 && d->N * a.parts * 2 <= 2ll * sm_count() && (long long)d->V * (int)sizeof(T) / 16 / (a.parts * 2 * kRowCta) >= 2) a.parts *= 2;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)(d->N * a.parts));
        cfg.blockDim = dim3(kRowCta);
        cfg.stream = st;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = a.parts; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, distill_fwd_kernel<T, TWO>, a) != cudaSuccess) { cudaGetLastError(); return M2D_ERR_LAUNCH; }
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
    return for_distill(d, [&](auto elem, auto two) {
        using T = decltype(elem);
        constexpr bool TWO = decltype(two)::value;
        if (short_rows(d)) {
            const size_t smem = (size_t)kRowWarps * 2 * d->K * 4;
            distill_bwd_warp_kernel<T, TWO><<<(unsigned)((d->N + kRowWarps - 1) / kRowWarps), kRowWarps * 32, smem, st>>>(a);
        } else {
            a.parts = (int)std::min<long long>(32, std::max<long long>(1, (long long)d->V * (int)sizeof(T) / 32768));
            distill_bwd_kernel<T, TWO><<<(unsigned)(d->N * a.parts), kRowCta, (size_t)2 * d->K * 4, st>>>(a);
        }
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    });
}
