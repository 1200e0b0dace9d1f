// Gated recurrence per channel: h_t = a_t h_{t-1} + u_t, forward, backward and for single tokens.
//
//   form decay:   a = exp(gate), u = x;          form forget: f = sigmoid(gate), a = f, u = (1 - f) x
//   backward:     D_t = dy_t + R_{t+1}, R_t = a_t D_t;   decay: dx = D, dgate = R_t h_{t-1};
//                 forget: dx = (1 - f) D, dgate = (1 - f) R_t (h_{t-1} - x_t)
//
// A CTA owns the channels of 32 lanes and walks a sequence in tiles.  Inside a tile a warp takes kSteps tokens: it finds what they do
// to any state, h -> A h + b, from registers; the warps' pairs (A, b) are joined in shared memory; then each warp goes over its tokens
// again from the state before them, still from registers, and stores.  So memory is read once and written once, and the loads of the
// next tile are under way meanwhile.
//
// Precision: states and sums are fp32.  A channel may remember thousands of tokens: 1 - A of a warp's tokens is small then, and A
// rounded to fp32 would be off by the same amount at every step, 2^-24 against a 1 - A of 2^-12 at a memory of 4096 tokens.  So a join has
// E = A - 1 beside A, computed without cancellation (expm1 of the summed gates, or a sum of 1 - f), and adds E h to h.
#include "follow.cuh"
#include "plan.cuh"
#include "m2d_seq.h"

namespace m2d {

constexpr int kMark = 64;            // tokens between the states that the forward pass leaves for the backward pass
constexpr int kRecurWarps = 8;       // warps of a CTA, at most

struct RecurArgs {
    const void *x, *gate, *dy;
    long long xb, xt, gb, gt, db, dt;
    const int* lengths;
    const float *state, *d_state_out;
    float *state_out, *d_state, *marks;
    void *y, *dx, *dgate;
    int B, T, C, groups;
};

// VEC neighbouring values of a row as they are in memory, and as numbers.
template <typename T, int VEC> struct Piece;
template <> struct Piece<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ void get(Raw r, float* v) { v[0] = r; }
    static __device__ __forceinline__ Raw put(const float* v) { return v[0]; }
};
template <> struct Piece<__nv_bfloat16, 1> {
    using Raw = unsigned short;
    static __device__ __forceinline__ void get(Raw r, float* v) { v[0] = bf16_bits_to_float(r); }
    static __device__ __forceinline__ Raw put(const float* v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v[0])); }
};
template <> struct Piece<__nv_bfloat16, 2> {
    using Raw = unsigned;
    static __device__ __forceinline__ void get(Raw r, float* v) { v[0] = __uint_as_float(r << 16); v[1] = __uint_as_float(r & 0xffff0000u); }
    static __device__ __forceinline__ Raw put(const float* v) { return pack_bf16x2(v[0], v[1]); }
};

__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// a = exp(gate), or f = sigmoid(gate) and 1 - f, each to its own precision: from exp(-|gate|), which is at most 1.
template <int FORM>
__device__ __forceinline__ void open_gate(float g, float& a, float& rest) {
    if constexpr (FORM == M2D_GATE_DECAY) {
        a = ex2(g * kLog2e);
        rest = 1.f;
    } else {
        const float t = ex2(fabsf(g) * -kLog2e), r = rcp_approx(1.f + t), s = t * r;
        a = g >= 0.f ? r : s;
        rest = g >= 0.f ? s : r;
    }
}
// What some tokens do to a state: h -> A h + b, with E = A - 1.
struct Step {
    float A, E;
    __device__ __forceinline__ void then(const Step& n) {
        A *= n.A;
        E = fmaf(E, n.E, E + n.E);
    }
    __device__ __forceinline__ float apply(float h, float b) const {
        const bool near = A >= 0.5f;
        return fmaf(near ? E : A, h, b) + (near ? h : 0.f);
    }
};
// The same for a run of tokens, collected token by token: the sum of the gates, or the product of f and the sum that is 1 - A.
template <int FORM>
struct Collect {
    float s = 0.f, p = 1.f;
    __device__ __forceinline__ void add(float g, float a, float rest) {
        if constexpr (FORM == M2D_GATE_DECAY) {
            s += g;
        } else {
            p *= a;
            s = fmaf(-s, rest, s + rest);
        }
    }
    __device__ __forceinline__ Step done() const {
        if constexpr (FORM == M2D_GATE_DECAY) return {ex2(s * kLog2e), expm1f(s)};
        else return {p, -s};
    }
};

template <typename T, int VEC, int FORM, int L>
__global__ void __launch_bounds__(kRecurWarps * 32) recur_fwd_kernel(const RecurArgs p) {
    using P = Piece<T, VEC>;
    using Raw = typename P::Raw;
    __shared__ float part[2][kRecurWarps][3][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, tile = warps * L;
    const int b = blockIdx.x / p.groups, c = (blockIdx.x % p.groups) * 32 * VEC + lane * VEC;
    const bool mine = c < p.C;
    const int len = p.lengths ? max(0, min(p.T, p.lengths[b])) : p.T;
    const T* const x = static_cast<const T*>(p.x) + b * p.xb + c;
    const T* const g = static_cast<const T*>(p.gate) + b * p.gb + c;
    T* const y = static_cast<T*>(p.y) + (long long)b * p.T * p.C + c;
    Raw rx[L], rg[L];
    auto load = [&](int t0) {
        const T *px = x + t0 * p.xt, *pg = g + t0 * p.gt;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const bool on = mine && t0 + i < len;
            rx[i] = on ? __ldcs(reinterpret_cast<const Raw*>(px + i * p.xt)) : Raw(0);
            rg[i] = on ? __ldcs(reinterpret_cast<const Raw*>(pg + i * p.gt)) : Raw(0);
        }
    };
    float carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = p.state && mine ? p.state[(long long)b * p.C + c + v] : 0.f;
    load(warp * L);
    for (int t1 = 0, buf = 0; t1 < len; t1 += tile, buf ^= 1) {
        const int t0 = t1 + warp * L;
        float a[L][VEC], u[L][VEC];
        Collect<FORM> all[VEC];
        float h[VEC] = {};
#pragma unroll
        for (int i = 0; i < L; ++i) {
            float xv[VEC], gv[VEC];
            P::get(rx[i], xv);
            P::get(rg[i], gv);
            const bool on = t0 + i < len;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float rest;
                open_gate<FORM>(gv[v], a[i][v], rest);
                if (!on) { a[i][v] = 1.f; rest = 0.f; }            // (its gate and x are 0: the state stays as it is)
                u[i][v] = FORM == M2D_GATE_DECAY ? xv[v] : rest * xv[v];
                all[v].add(gv[v], a[i][v], rest);
                h[v] = fmaf(a[i][v], h[v], u[i][v]);
            }
        }
        if (t1 + tile < len) load(t0 + tile);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Step s = all[v].done();
            part[buf][warp][0][lane * VEC + v] = s.A;
            part[buf][warp][1][lane * VEC + v] = s.E;
            part[buf][warp][2][lane * VEC + v] = h[v];
        }
        __syncthreads();                      // (one barrier a tile: what is read below is written over two tiles on)
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = carry[v];
        for (int w = 0; w < warps; ++w) {
            if (w == warp) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) h[v] = carry[v];
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Step s{part[buf][w][0][lane * VEC + v], part[buf][w][1][lane * VEC + v]};
                carry[v] = s.apply(carry[v], part[buf][w][2][lane * VEC + v]);
            }
        }
        if (p.marks && mine && t0 < len && t0 % kMark == 0) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) p.marks[((long long)b * ((p.T + kMark - 1) / kMark) + t0 / kMark) * p.C + c + v] = h[v];
        }
        T* py = y + (long long)t0 * p.C;
#pragma unroll
        for (int i = 0; i < L; ++i) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = fmaf(a[i][v], h[v], u[i][v]);
            if (mine && t0 + i < len) *reinterpret_cast<Raw*>(py + (long long)i * p.C) = P::put(h);
        }
    }
    if (!mine) return;
    const float zero[VEC] = {};
    for (long long t = len + warp; t < p.T; t += warps) *reinterpret_cast<Raw*>(y + t * p.C) = P::put(zero);
    if (p.state_out && warp == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.state_out[(long long)b * p.C + c + v] = carry[v];
    }
}

// Tiles from the last to the first.  The states inside a tile come from the forward pass's mark before it.
template <typename T, int VEC, int FORM, int L>
__global__ void __launch_bounds__(kRecurWarps * 32) recur_bwd_kernel(const RecurArgs p) {
    using P = Piece<T, VEC>;
    using Raw = typename P::Raw;
    __shared__ float part[2][kRecurWarps][4][32 * VEC];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    constexpr int tile = kMark;
    const int b = blockIdx.x / p.groups, c = (blockIdx.x % p.groups) * 32 * VEC + lane * VEC;
    const bool mine = c < p.C;
    const int len = p.lengths ? max(0, min(p.T, p.lengths[b])) : p.T;
    const T* const x = static_cast<const T*>(p.x) + b * p.xb + c;
    const T* const g = static_cast<const T*>(p.gate) + b * p.gb + c;
    const T* const dy = static_cast<const T*>(p.dy) + b * p.db + c;
    const long long out = (long long)b * p.T * p.C + c;
    T *const dx = static_cast<T*>(p.dx) + out, *const dgate = static_cast<T*>(p.dgate) + out;
    const float* const marks = p.marks + (long long)b * ((p.T + kMark - 1) / kMark) * p.C + c;
    Raw rx[L], rg[L], rd[L];
    float mark[VEC] = {};
    auto load = [&](int t1) {
        const int t0 = t1 + warp * L;
        const T *px = x + t0 * p.xt, *pg = g + t0 * p.gt, *pd = dy + t0 * p.dt;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const bool on = mine && t0 + i < len;
            rx[i] = on ? __ldcs(reinterpret_cast<const Raw*>(px + i * p.xt)) : Raw(0);
            rg[i] = on ? __ldcs(reinterpret_cast<const Raw*>(pg + i * p.gt)) : Raw(0);
            rd[i] = on ? __ldcs(reinterpret_cast<const Raw*>(pd + i * p.dt)) : Raw(0);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) mark[v] = mine ? marks[(long long)(t1 / kMark) * p.C + v] : 0.f;
    };
    float carry[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) carry[v] = p.d_state_out && mine ? p.d_state_out[(long long)b * p.C + c + v] : 0.f;
    int t1 = (len - 1) / tile * tile;         // (of no tokens: none)
    if (len > 0) load(t1);
    for (int buf = 0; len > 0 && t1 >= 0; t1 -= tile, buf ^= 1) {
        const int t0 = t1 + warp * L;
        float a[L][VEC], rest[L][VEC], xv[L][VEC], dv[L][VEC], before[L][VEC];
        Collect<FORM> all[VEC];
        float h[VEC] = {}, R[VEC] = {};
#pragma unroll
        for (int i = 0; i < L; ++i) {
            float gv[VEC];
            P::get(rx[i], xv[i]);
            P::get(rg[i], gv);
            P::get(rd[i], dv[i]);
            const bool on = t0 + i < len;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                open_gate<FORM>(gv[v], a[i][v], rest[i][v]);
                if (!on) { a[i][v] = 1.f; rest[i][v] = 0.f; }
                all[v].add(gv[v], a[i][v], rest[i][v]);
                h[v] = fmaf(a[i][v], h[v], FORM == M2D_GATE_DECAY ? xv[i][v] : rest[i][v] * xv[i][v]);
            }
        }
#pragma unroll
        for (int i = L - 1; i >= 0; --i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) R[v] = a[i][v] * (dv[i][v] + R[v]);
        float first[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) first[v] = mark[v];
        if (t1 >= tile) load(t1 - tile);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const Step s = all[v].done();
            part[buf][warp][0][lane * VEC + v] = s.A;
            part[buf][warp][1][lane * VEC + v] = s.E;
            part[buf][warp][2][lane * VEC + v] = h[v];
            part[buf][warp][3][lane * VEC + v] = R[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = first[v];
        for (int w = 0; w < warp; ++w)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Step s{part[buf][w][0][lane * VEC + v], part[buf][w][1][lane * VEC + v]};
                h[v] = s.apply(h[v], part[buf][w][2][lane * VEC + v]);
            }
        for (int w = warps - 1; w >= 0; --w) {
            if (w == warp) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) R[v] = carry[v];
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const Step s{part[buf][w][0][lane * VEC + v], part[buf][w][1][lane * VEC + v]};
                carry[v] = s.apply(carry[v], part[buf][w][3][lane * VEC + v]);
            }
        }
#pragma unroll
        for (int i = 0; i < L; ++i)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                before[i][v] = h[v];
                h[v] = fmaf(a[i][v], h[v], FORM == M2D_GATE_DECAY ? xv[i][v] : rest[i][v] * xv[i][v]);
            }
        const long long at = (long long)t0 * p.C;
#pragma unroll
        for (int i = L - 1; i >= 0; --i) {
            float gx[VEC], gg[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float D = dv[i][v] + R[v];
                R[v] = a[i][v] * D;
                if constexpr (FORM == M2D_GATE_DECAY) {
                    gx[v] = D;
                    gg[v] = R[v] * before[i][v];
                } else {
                    gx[v] = rest[i][v] * D;
                    gg[v] = rest[i][v] * R[v] * (before[i][v] - xv[i][v]);
                }
            }
            if (mine && t0 + i < len) {
                *reinterpret_cast<Raw*>(dx + at + (long long)i * p.C) = P::put(gx);
                *reinterpret_cast<Raw*>(dgate + at + (long long)i * p.C) = P::put(gg);
            }
        }
    }
    if (!mine) return;
    const float zero[VEC] = {};
    for (long long t = len + warp; t < p.T; t += warps) {
        *reinterpret_cast<Raw*>(dx + t * p.C) = P::put(zero);
        *reinterpret_cast<Raw*>(dgate + t * p.C) = P::put(zero);
    }
    if (p.d_state && warp == 0) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.d_state[(long long)b * p.C + c + v] = carry[v];
    }
}

// One token of every sequence.  state and state_out may be the same array.
template <typename T, int VEC, int FORM>
__global__ void __launch_bounds__(128) recur_step_kernel(const RecurArgs p, long long sb) {
    using P = Piece<T, VEC>;
    using Raw = typename P::Raw;
    const int c = (blockIdx.x * 128 + threadIdx.x) * VEC;
    if (c >= p.C) return;
    for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
        float xv[VEC], gv[VEC], h[VEC];
        P::get(*reinterpret_cast<const Raw*>(static_cast<const T*>(p.x) + b * p.xb + c), xv);
        P::get(*reinterpret_cast<const Raw*>(static_cast<const T*>(p.gate) + b * p.gb + c), gv);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float a, rest;
            open_gate<FORM>(gv[v], a, rest);
            h[v] = fmaf(a, p.state[b * sb + c + v], FORM == M2D_GATE_DECAY ? xv[v] : rest * xv[v]);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.state_out[b * sb + c + v] = h[v];
        *reinterpret_cast<Raw*>(static_cast<T*>(p.y) + (long long)b * p.C + c) = P::put(h);
    }
}

static int check_recur(const m2d_recur_desc* d, bool step) {
    if (!d) return M2D_ERR_NULL;
    if (d->struct_bytes != sizeof(m2d_recur_desc)) return M2D_ERR_ABI;
    if (d->dtype != M2D_F32 && d->dtype != M2D_BF16) return M2D_ERR_DTYPE;
    if (d->form != M2D_GATE_DECAY && d->form != M2D_GATE_FORGET) return M2D_ERR_FLAGS;
    if (d->B < 1 || d->T < 1 || d->C < 1 || (step && d->T != 1)) return M2D_ERR_SHAPE;
    // (tokens are counted in 32 bits, a tile beyond the last included; CTAs too)
    if (d->T > INT32_MAX - 1024 || (long long)d->B * ((d->C + 31) / 32) > INT32_MAX / 16) return M2D_ERR_TOO_LARGE;
    const uintptr_t es = d->dtype == M2D_F32 ? 4 : 2;
    for (const void* t : {d->x.data, d->gate.data}) {
        if (!t) return M2D_ERR_NULL;
        if (reinterpret_cast<uintptr_t>(t) % es) return M2D_ERR_PITCH;
    }
    return M2D_OK;
}
static bool pairs_ok(const void* p, long long a, long long b) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 4 == 0 && a % 2 == 0 && b % 2 == 0); }
static RecurArgs recur_args(const m2d_recur_desc* d) {
    RecurArgs a{};
    a.x = d->x.data; a.xb = d->x.batch; a.xt = d->x.token;
    a.gate = d->gate.data; a.gb = d->gate.batch; a.gt = d->gate.token;
    a.dy = d->d_y.data; a.db = d->d_y.batch; a.dt = d->d_y.token;
    a.lengths = d->lengths; a.state = d->state; a.d_state_out = d->d_state_out;
    a.state_out = d->state_out; a.d_state = d->d_state; a.marks = d->marks;
    a.y = d->y; a.dx = d->d_x; a.dgate = d->d_gate;
    a.B = d->B; a.T = d->T; a.C = d->C;
    return a;
}
// Calls fn(element, channels of a lane, form): two channels of bf16 where rows are whole 4-byte pieces.
template <typename F>
static int for_recur(const m2d_recur_desc* d, bool pairs, F fn) {
    auto with_form = [&](auto elem, auto vec) {
        return d->form == M2D_GATE_DECAY ? fn(elem, vec, std::integral_constant<int, M2D_GATE_DECAY>{}) : fn(elem, vec, std::integral_constant<int, M2D_GATE_FORGET>{});
    };
    if (d->dtype == M2D_F32) return with_form(float{}, std::integral_constant<int, 1>{});
    if (pairs) return with_form(__nv_bfloat16{}, std::integral_constant<int, 2>{});
    return with_form(__nv_bfloat16{}, std::integral_constant<int, 1>{});
}
constexpr int kFwdSteps = 16, kBwdSteps = 8;

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_recur_marks(const m2d_recur_desc* d) {
    if (!d || d->B < 1 || d->T < 1 || d->C < 1) return 0;
    return (uint64_t)d->B * ((d->T + kMark - 1) / kMark) * d->C;
}

extern "C" int m2d_recur_fwd(const m2d_recur_desc* d, void* stream) {
    const int rc = check_recur(d, false);
    if (rc != M2D_OK) return rc;
    if (!d->y) return M2D_ERR_NULL;
    RecurArgs a = recur_args(d);
    const bool pairs = d->C % 2 == 0 && pairs_ok(a.x, a.xb, a.xt) && pairs_ok(a.gate, a.gb, a.gt) && pairs_ok(a.y, 0, 0);
    return for_recur(d, pairs, [&](auto elem, auto vec, auto form) {
        using T = decltype(elem);
        constexpr int VEC = decltype(vec)::value, FORM = decltype(form)::value;
        a.groups = (d->C + 32 * VEC - 1) / (32 * VEC);
        const int warps = std::min(kRecurWarps, (d->T + kFwdSteps - 1) / kFwdSteps);
        recur_fwd_kernel<T, VEC, FORM, kFwdSteps><<<d->B * a.groups, warps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    });
}

extern "C" int m2d_recur_bwd(const m2d_recur_desc* d, void* stream) {
    const int rc = check_recur(d, false);
    if (rc != M2D_OK) return rc;
    if (!d->d_y.data || !d->d_x || !d->d_gate || !d->marks) return M2D_ERR_NULL;
    RecurArgs a = recur_args(d);
    const bool pairs = d->C % 2 == 0 && pairs_ok(a.x, a.xb, a.xt) && pairs_ok(a.gate, a.gb, a.gt) && pairs_ok(a.dy, a.db, a.dt) && pairs_ok(a.dx, 0, 0) && pairs_ok(a.dgate, 0, 0);
    return for_recur(d, pairs, [&](auto elem, auto vec, auto form) {
        using T = decltype(elem);
        constexpr int VEC = decltype(vec)::value, FORM = decltype(form)::value;
        a.groups = (d->C + 32 * VEC - 1) / (32 * VEC);
        recur_bwd_kernel<T, VEC, FORM, kBwdSteps><<<d->B * a.groups, kMark / kBwdSteps * 32, 0, static_cast<cudaStream_t>(stream)>>>(a);
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    });
}

extern "C" int m2d_recur_step(const m2d_recur_desc* d, int64_t state_batch, void* stream) {
    const int rc = check_recur(d, true);
    if (rc != M2D_OK) return rc;
    if (!d->y || !d->state || !d->state_out) return M2D_ERR_NULL;
    const RecurArgs a = recur_args(d);
    const bool pairs = d->C % 2 == 0 && pairs_ok(a.x, a.xb, 0) && pairs_ok(a.gate, a.gb, 0) && pairs_ok(a.y, 0, 0);
    return for_recur(d, pairs, [&](auto elem, auto vec, auto form) {
        using T = decltype(elem);
        constexpr int VEC = decltype(vec)::value, FORM = decltype(form)::value;
        const dim3 grid((d->C + 128 * VEC - 1) / (128 * VEC), std::min(d->B, 65535));
        recur_step_kernel<T, VEC, FORM><<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(a, (long long)state_batch);
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    });
}
