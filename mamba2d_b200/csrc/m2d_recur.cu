// Gated recurrence per channel: h_t = a_t h_{t-1} + u_t, forward, backward and for single tokens.
//
//   form decay:   a = exp(gate), u = x;          form forget: f = sigmoid(gate), a = f, u = (1 - f) x
//   backward:     D_t = dy_t + R_{t+1}, R_t = a_t D_t;   decay: dx = D, dgate = R_t h_{t-1};
//                 forget: dx = (1 - f) D, dgate = (1 - f) R_t (h_{t-1} - x_t)
//
// A cluster of CTAs owns the channels of LANES lanes and walks a sequence in strides, a tile of it for each CTA.  Inside a tile the lanes of a row
// take L tokens: they find what those do to any state, h -> A h + b, from registers; the runs' pairs (A, b) are joined in shared memory, the tiles' in
// that of every CTA of the cluster; then each goes over its tokens again from the state before them, still from registers, and stores.  So
// memory is read once and written once.  Tiles come by TMA, one to three ahead of the one that is worked on (two forward and one backward where tiles are as large as in the cases below); where rows are not whole 16-byte pieces, or
// there is but one stride, by plain loads into registers, the next tile's while one is worked on.  Where sequences and channels are too few for all SMs, rows are
// split into shorter pieces and the sequence over up to 8 CTAs (plan_recur).  Measured, bf16: 4x4096x2048 forget gates 47 us (201 MB at 4.3 TB/s: half
// of the issue slots, two CTAs an SM), 1x65536x512 decays 57 us (the chain of waits of 16 strides), 8x4096x2048 forward 75 and backward 126 us (5.4 and 5.3 TB/s).
//
// Precision: states and sums are fp32.  A channel may remember thousands of tokens: 1 - A of a run is small then, and A
// rounded to fp32 would be off by the same amount at every step, 2^-24 against a 1 - A of 2^-12 at a memory of 4096 tokens.  So A is held in two
// parts, from E = A - 1 computed without cancellation (a series in the summed gates, or a sum of 1 - f).
#include <cooperative_groups.h>

#include "launch.cuh"
#include "packed.cuh"
#include "tc_ptx.cuh"
#include "m2d_seq.h"

namespace m2d {

constexpr int kMark = 64;            // tokens between the states that the forward pass leaves for the backward pass
constexpr int kRecurWarps = 16;      // warps of a CTA, at most
constexpr int kRecurCluster = 8;     // CTAs of a cluster, at most

struct RecurArgs {
    const void *x, *gate, *dy;
    long long xb, xt, gb, gt, db, dt;
    const int* lengths;
    const float *state, *d_state_out;
    float *state_out, *d_state, *marks;
    void *y, *dx, *dgate;
    int B, T, C, groups, ctas;         // channel groups, CTAs of a cluster
    int stages, box;                   // tiles in shared memory; tokens of one TMA copy
    int give_up;                       // test hook
    int* host_flag;
};
struct RecurMaps { CUtensorMap x, gate, dy; };

// VEC neighbouring values of a row as they are in memory, and as numbers.
template <typename T, int VEC> struct Piece;
template <> struct Piece<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ Raw fill(float f) { return f; }
    static __device__ __forceinline__ Num<1> get(Raw r) { return {r}; }
    static __device__ __forceinline__ Raw put(Num<1> n) { return n.v; }
};
template <> struct Piece<float, 2> {
    using Raw = float2;
    static __device__ __forceinline__ Raw fill(float f) { return make_float2(f, f); }
    static __device__ __forceinline__ Num<2> get(Raw r) { return Num<2>::make(r.x, r.y); }
    static __device__ __forceinline__ Raw put(Num<2> n) { return make_float2(n.get(0), n.get(1)); }
};
template <> struct Piece<__nv_bfloat16, 1> {
    using Raw = unsigned short;
    static __device__ __forceinline__ Raw fill(float f) { return (unsigned short)(__float_as_uint(f) >> 16); }
    static __device__ __forceinline__ Num<1> get(Raw r) { return {bf16_bits_to_float(r)}; }
    static __device__ __forceinline__ Raw put(Num<1> n) { return __bfloat16_as_ushort(__float2bfloat16_rn(n.v)); }
};
template <> struct Piece<__nv_bfloat16, 2> {
    using Raw = unsigned;
    static __device__ __forceinline__ Raw fill(float f) { return __float_as_uint(f) | __float_as_uint(f) >> 16; }
    static __device__ __forceinline__ Num<2> get(Raw r) { return Num<2>::make(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u)); }
    static __device__ __forceinline__ Raw put(Num<2> n) { return pack_bf16x2(n.get(0), n.get(1)); }
};
// A gate that leaves the state as it is, where x is 0.  (Its lower 16 bits are zero.)
template <int FORM> __device__ __forceinline__ float kept() { return FORM == M2D_GATE_DECAY ? 0.f : __int_as_float(0x7f800000); }

__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float most(float a, float b) {          // a NaN stays one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// A gate as it is in memory.  Forget gates below -87 count as -87, whose f is 1.6e-38, so that exp(-gate) stays finite.
template <typename T, int VEC, int FORM>
__device__ __forceinline__ Num<VEC> gate_of(typename Piece<T, VEC>::Raw r) {
    using P = Piece<T, VEC>;
    if constexpr (FORM == M2D_GATE_DECAY) {
        return P::get(r);
    } else if constexpr (sizeof(T) == 2 && VEC == 2) {
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(r), "r"(0xc2aec2aeu));
        return P::get(r);
    } else {
        Num<VEC> g = P::get(r);
#pragma unroll
        for (int v = 0; v < VEC; ++v) g.set(v, most(g.get(v), -87.f));
        return g;
    }
}
// a = exp(gate), or f = sigmoid(gate) and 1 - f, each to its own precision: e = exp(-gate), f = 1 / (1 + e), 1 - f = e f.
template <int FORM, int VEC>
__device__ __forceinline__ void open_gate(Num<VEC> g, Num<VEC>& a, Num<VEC>& rest) {
    if constexpr (FORM == M2D_GATE_DECAY) {
        const Num<VEC> s = mul_(g, Num<VEC>::all(kLog2e));
#pragma unroll
        for (int v = 0; v < VEC; ++v) a.set(v, ex2(s.get(v)));
        rest = Num<VEC>::all(1.f);
    } else {
        Num<VEC> e = mul_(g, Num<VEC>::all(-kLog2e));
#pragma unroll
        for (int v = 0; v < VEC; ++v) e.set(v, ex2(e.get(v)));
        const Num<VEC> d = add_(e, Num<VEC>::all(1.f));
#pragma unroll
        for (int v = 0; v < VEC; ++v) a.set(v, rcp_approx(d.get(v)));
        rest = mul_(e, a);
    }
}
// exp(s) - 1 by its series, used for |s| <= log 2: the tenth power's term is below 2^-26 of the sum.
template <int VEC>
__device__ __forceinline__ Num<VEC> less_one(Num<VEC> s) {
    using N = Num<VEC>;
    N e = N::all(1.f / 362880);
    constexpr float c[] = {1.f / 40320, 1.f / 5040, 1.f / 720, 1.f / 120, 1.f / 24, 1.f / 6, 0.5f, 1.f};
#pragma unroll
    for (int k = 0; k < 8; ++k) e = fma_(e, s, N::all(c[k]));
    return mul_(e, s);
}
// What some tokens do to a state: h -> (hi + lo) h + b.
template <int VEC>
struct Step {
    Num<VEC> hi, lo;
    __device__ __forceinline__ Num<VEC> apply(Num<VEC> h, Num<VEC> b) const { return fma_(hi, h, fma_(lo, h, b)); }
    __device__ __forceinline__ void times(const Step& n) {          // the product of both, in two parts
        const Num<VEC> p = mul_(hi, n.hi), rest = fma_(hi, n.hi, neg_(p));
        lo = fma_(hi, n.lo, fma_(lo, n.hi, rest));
        hi = p;
    }
};
// The same for a run of tokens, collected token by token: the sum of the gates, or the product of f and the sum that is 1 - A (every token takes
// its 1 - f of what those before it left).
template <int FORM, int VEC>
struct Collect {
    using N = Num<VEC>;
    Num<VEC> s = Num<VEC>::all(0.f), p = Num<VEC>::all(1.f);
    __device__ __forceinline__ void add(Num<VEC> g, Num<VEC> a, Num<VEC> rest) {
        if constexpr (FORM == M2D_GATE_DECAY) {
            s = add_(s, g);
        } else {
            s = fma_(rest, p, s);
            p = mul_(p, a);
        }
    }
    __device__ __forceinline__ Step<VEC> done() const {
        Step<VEC> r;
        N e = neg_(s);
        if constexpr (FORM == M2D_GATE_DECAY) e = less_one(s);
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const float A = FORM == M2D_GATE_DECAY ? ex2(s.get(v) * kLog2e) : p.get(v), E = e.get(v);
            const bool near = A >= 0.5f && A <= 2.f;
            const float hi = near ? 1.f + E : A;
            r.hi.set(v, hi);
            r.lo.set(v, near ? E - (hi - 1.f) : 0.f);
        }
        return r;
    }
};
// Two Nums of VEC channels side by side in shared memory: hi and lo of a step, or what goes with it.
template <int VEC> struct Two { Num<VEC> a, b; };
template <int VEC> __device__ __forceinline__ Two<VEC> take2(const float* p) {
    if constexpr (VEC == 1) {
        const float2 f = *reinterpret_cast<const float2*>(p);
        return {{f.x}, {f.y}};
    } else {
        const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(p);
        return {{f.x}, {f.y}};
    }
}
template <int VEC> __device__ __forceinline__ void give2(float* p, Num<VEC> a, Num<VEC> b) {
    if constexpr (VEC == 1) *reinterpret_cast<float2*>(p) = make_float2(a.v, b.v);
    else *reinterpret_cast<ulonglong2*>(p) = make_ulonglong2(a.v, b.v);
}
// VEC neighbouring floats of shared memory
template <int VEC> __device__ __forceinline__ Num<VEC> take(const float* p) {
    if constexpr (VEC == 1) return {*p};
    else return Num<2>{*reinterpret_cast<const unsigned long long*>(p)};
}
template <int VEC> __device__ __forceinline__ void give(float* p, Num<VEC> n) {
    if constexpr (VEC == 1) *p = n.v;
    else *reinterpret_cast<unsigned long long*>(p) = n.v;
}
template <int VEC> __device__ __forceinline__ Num<VEC> load_state(const float* p, bool on) {
    Num<VEC> n = Num<VEC>::all(0.f);
    if (on)
#pragma unroll
        for (int v = 0; v < VEC; ++v) n.set(v, p[v]);
    return n;
}
template <int VEC> __device__ __forceinline__ void store_state(float* p, Num<VEC> n) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) p[v] = n.get(v);
}

// Rows of fewer lanes than a warp has: its runs are joined by shuffles first.
template <int VEC> __device__ __forceinline__ Num<VEC> moved(Num<VEC> n, int lanes, bool up) {
    if constexpr (VEC == 1) return {up ? __shfl_up_sync(0xffffffffu, n.v, lanes) : __shfl_down_sync(0xffffffffu, n.v, lanes)};
    else return Num<2>{up ? __shfl_up_sync(0xffffffffu, n.v, lanes) : __shfl_down_sync(0xffffffffu, n.v, lanes)};
}
// step and b of all runs of the warp up to and with the lane's own (UP: in the order of time, else against it).
template <int VEC, int LANES, bool UP>
__device__ __forceinline__ void join_warp(Step<VEC>& step, Num<VEC>& b) {
    const int run = (threadIdx.x & 31) / LANES, before = UP ? run : 32 / LANES - 1 - run;
#pragma unroll
    for (int k = 1; k < 32 / LANES; k *= 2) {
        const Step<VEC> first{moved<VEC>(step.hi, k * LANES, UP), moved<VEC>(step.lo, k * LANES, UP)};
        const Num<VEC> c = moved<VEC>(b, k * LANES, UP);
        if (before >= k) {
            b = step.apply(c, b);
            step.times(first);
        }
    }
}
// The state before the lane's own run, from that before the warp's runs and what join_warp left.
template <int VEC, int LANES, bool UP>
__device__ __forceinline__ Num<VEC> after_others(const Step<VEC>& step, Num<VEC> b, Num<VEC> h) {
    if constexpr (LANES == 32) return h;
    const int run = (threadIdx.x & 31) / LANES;
    const Num<VEC> there = moved<VEC>(step.apply(h, b), LANES, UP);
    return run == (UP ? 0 : 32 / LANES - 1) ? h : there;
}

// Where a thread stands: its channels, its run of a tile, its CTA of the cluster.
template <int VEC, int LANES>
struct Place {
    static constexpr int width = LANES * VEC;      // channels of a CTA
    int at, runs, run, warps, warp, b, c, rank, ctas, len;         // at: first of the thread's channels among the CTA's
    bool mine, first, last;                        // first, last: of the runs of its warp
    __device__ __forceinline__ Place(const RecurArgs& p) {
        const int lane = threadIdx.x & 31, per = 32 / LANES;
        at = lane % LANES * VEC;
        warps = blockDim.x >> 5;
        warp = threadIdx.x >> 5;
        runs = warps * per;
        run = warp * per + lane / LANES;
        first = lane < LANES;
        last = lane >= 32 - LANES;
        ctas = p.ctas;
        rank = blockIdx.x % ctas;
        const int chain = blockIdx.x / ctas;
        b = chain / p.groups;
        c = chain % p.groups * width + at;
        mine = c < p.C;
        len = p.lengths ? max(0, min(p.T, p.lengths[b])) : p.T;
    }
};

// Shared memory: with TMA first [stages][TENSORS][tile][width] of the tensors; [2][warps][PARTS][width] of the CTA's warps, [2][ctas][3][width] of
// the cluster's tiles (two of each: one barrier lies between what is read of a tile and what is written of the next but one); last the
// barriers of the stages and of the cluster's tiles, and the word that tells that a wait gave up.
constexpr int kRecurStages = 4;
inline size_t recur_joins(int parts, int warps, int ctas, int width) { return sizeof(float) * 2 * width * ((size_t)warps * parts + (ctas > 1 ? (size_t)ctas * 3 : 0)); }
inline size_t recur_stage(int tensors, int tile, int width, int es) { return (size_t)tensors * tile * width * es; }
constexpr size_t kRecurTail = (kRecurStages + 3) * 8;

// Waits for a barrier's phase, so many times 32 tries of at most about a microsecond; gives up and tells so in *abort, or where that has been told.
// CLUSTER: of what other CTAs send.
template <bool CLUSTER>
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, int limit, volatile int* abort) {
    for (int n = 0; n < limit; ++n) {
        if (mbar_try_wait32<CLUSTER>(bar, parity)) return true;
        if (*abort) return false;
    }
    *abort = 1;
    return false;
}
// For a copy about a quarter of a second; for other CTAs' joins four times that, since one of them may be giving up a copy.
constexpr int kCopyLimit = 1 << 13, kJoinLimit = 1 << 15;

// Barriers and the abort words of a CTA.  A tile's join reaches every CTA of the cluster by stores that count towards the receiver's barrier:
// nothing else is waited for.  All waits are bounded; where one gives up, what depends on it is NaN.  A CTA that has given up a copy asks for no more
// of them, but goes on joining and sending (NaN) like all others: the joins' barriers are armed once a phase, whatever happens to copies.  One that has given up
// a join arms, waits and sends no more, and the others run out of its joins a tile later.
struct Waits {
    uint32_t stage_bars, join_bars;
    volatile int *abort, *apart;              // a copy was given up; a join was
    __device__ __forceinline__ Waits(const RecurArgs& p, char* tail) {
        stage_bars = smem_u32(tail);
        join_bars = stage_bars + 8 * kRecurStages;
        abort = reinterpret_cast<volatile int*>(tail + 8 * (kRecurStages + 2));
        apart = abort + 1;
        if (threadIdx.x == 0) {
            for (int k = 0; k < kRecurStages + 2; ++k) mbar_init(stage_bars + 8 * k, 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
            *abort = p.give_up && blockIdx.x == 0;
            *apart = 0;
        }
        __syncthreads();
    }
    static __device__ __forceinline__ uint32_t there(uint32_t addr, int rank) {
        uint32_t r;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
        return r;
    }
    // a lane's channels of a tile's join, to CTA `rank`: hi and lo, and what goes with them
    template <int VEC>
    __device__ __forceinline__ void send(int rank, const float* pair, const float* add, const Step<VEC>& s, Num<VEC> b, int buf) const {
        const uint32_t p = there(smem_u32(pair), rank), a = there(smem_u32(add), rank), bar = there(join_bars + 8 * buf, rank);
        if constexpr (VEC == 2) {
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(p), "l"(s.hi.v), "l"(s.lo.v), "r"(bar) : "memory");
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(a), "l"(b.v), "r"(bar) : "memory");
        } else {
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(p), "r"(__float_as_uint(s.hi.v)), "r"(__float_as_uint(s.lo.v)), "r"(bar) : "memory");
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(a), "r"(__float_as_uint(b.v)), "r"(bar) : "memory");
        }
    }
    // all CTAs' joins are there; `turn` counts the tiles
    __device__ __forceinline__ bool joined(int turn, uint32_t bytes) const {
        const uint32_t bar = join_bars + 8 * (turn & 1);
        if (*apart) return false;
        if (threadIdx.x == 0) mbar_expect_tx(bar, bytes);
        return wait_for<true>(bar, (turn >> 1) & 1, kJoinLimit, apart);
    }
};

// A thread's tokens of a tile: TENSORS raw values of each.  order() asks for a tile (thread 0), ready() waits for the oldest one that was asked for, raw()
// reads it, next() goes on; or, without TMA, load() and raw().
template <typename T, int VEC, int FORM, int L, int LANES, int TENSORS, bool TMA>
struct Feed {
    using P = Piece<T, VEC>;
    using Raw = typename P::Raw;
    static constexpr int width = LANES * VEC;
    Raw reg[TMA ? 1 : TENSORS][TMA ? 1 : L];
    char* ring;
    uint32_t bars;
    volatile int *abort, *apart;
    int stage, stages, tile, box, at, run, ordered, turned;
    unsigned parity;
    template <typename W>
    __device__ __forceinline__ Feed(const RecurArgs& p, const W& w, char* smem, const Waits& waits) {
        abort = waits.abort;
        apart = waits.apart;
        if constexpr (TMA) {
            ring = smem;
            bars = waits.stage_bars;
            stage = ordered = 0;
            parity = 0;
            stages = p.stages;
            tile = w.runs * L;
            box = p.box;
            at = w.at;
            run = w.run;
            turned = (threadIdx.x & 31) / LANES;
        }
    }
    static __device__ __forceinline__ Raw nothing(int t) { return P::fill(t == 1 ? kept<FORM>() : 0.f); }
    // the tile that begins at token t1 of sequence b, to channel c0 on
    __device__ __forceinline__ void order(const RecurMaps& maps, int c0, int t1, int b) {
        if (threadIdx.x != 0 || *abort) return;
        const int k = ordered % stages;
        const uint32_t bar = bars + 8 * k, one = (uint32_t)box * width * sizeof(T);
        uint32_t to = smem_u32(ring) + (uint32_t)k * TENSORS * tile * width * sizeof(T);
        mbar_expect_tx(bar, TENSORS * tile * width * sizeof(T));
#pragma unroll
        for (int t = 0; t < TENSORS; ++t) {
            const CUtensorMap* const map = t == 0 ? &maps.x : t == 1 ? &maps.gate : &maps.dy;
            for (int i = 0; i < tile; i += box, to += one)
                asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                             ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(t1 + i), "r"(b), "r"(bar) : "memory");
        }
        ++ordered;
    }
    __device__ __forceinline__ Raw* place(int t, int i) const { return reinterpret_cast<Raw*>(ring + (((size_t)(stage * TENSORS + t) * tile + run * L + i) * width + at) * sizeof(T)); }
    // false: gave up.  n: tokens that there are of the thread's run; the others' places get what changes nothing.
    __device__ __forceinline__ bool ready(int n) {
        if (!wait_for<false>(bars + 8 * stage, parity, kCopyLimit, abort)) return false;
        if (n < L) {
#pragma unroll
            for (int t = 0; t < TENSORS; ++t)
                for (int i = max(0, n); i < L; ++i) *place(t, i) = nothing(t);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // (a later copy comes here)
        }
        return true;
    }
    __device__ __forceinline__ void next() {
        if (++stage == stages) { stage = 0; parity ^= 1; }
    }
    // Tokens i ... i + 3.  Where a warp has several rows at once, those of its runs lie in the same banks, 16 tokens apart: run q reads its tokens in
    // the order i ^ q and sorts them in registers.
    __device__ __forceinline__ void four(int t, int i, Raw (&r)[4]) const {
        if constexpr (!TMA) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = reg[t][i + j];
        } else if constexpr (LANES == 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = *place(t, i + j);
        } else {
            const char* const p = reinterpret_cast<const char*>(place(t, i));
            Raw q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const Raw*>(p + (j ^ turned) * (width * (int)sizeof(T)));
            const bool one = turned & 1, two = turned & 2;
            const Raw a0 = one ? q[1] : q[0], a1 = one ? q[0] : q[1], a2 = one ? q[3] : q[2], a3 = one ? q[2] : q[3];
            r[0] = two ? a2 : a0;
            r[1] = two ? a3 : a1;
            r[2] = two ? a0 : a2;
            r[3] = two ? a1 : a3;
        }
    }
    // bounded wait for what is still on its way, after a wait that gave up; tells the host
    __device__ __forceinline__ void leave(int* host_flag) {
        if (threadIdx.x != 0 || !(*abort || *apart)) return;
        if constexpr (TMA)
            for (int j = max(0, ordered - stages); j < ordered; ++j)
                for (int n = 0; n < kCopyLimit && !mbar_try_wait32(bars + 8 * (j % stages), (j / stages) & 1); ++n) {}
        if (host_flag) *reinterpret_cast<volatile int*>(host_flag) = 1;
    }
};

template <typename T, int VEC, int FORM, int L, int LANES, bool TMA>
__global__ void __launch_bounds__(kRecurWarps * 32) recur_fwd_kernel(const RecurArgs p, const __grid_constant__ RecurMaps maps) {
    namespace cg = cooperative_groups;
    using P = Piece<T, VEC>;
    using Raw = typename P::Raw;
    using N = Num<VEC>;
    constexpr int width = LANES * VEC;
    extern __shared__ __align__(128) char ring[];
    const Place<VEC, LANES> w(p);
    cg::cluster_group cluster = cg::this_cluster();
    const int tile = w.runs * L, stride = w.ctas * tile;
    float* const smem = reinterpret_cast<float*>(ring + (TMA ? p.stages * (size_t)2 * tile * width * sizeof(T) : 0));
    const Waits waits(p, reinterpret_cast<char*>(smem + 2 * width * (w.warps * 3 + (w.ctas > 1 ? w.ctas * 3 : 0))));
    if (w.ctas > 1) cluster.barrier_arrive();             // (all have begun, their barriers too, before one writes to another)
    Feed<T, VEC, FORM, L, LANES, 2, TMA> feed(p, w, ring, waits);
    const uint32_t join_bytes = (uint32_t)w.ctas * 3 * width * sizeof(float);
    int turn = 0;
    const T* const x = static_cast<const T*>(p.x) + w.b * p.xb + w.c;
    const T* const g = static_cast<const T*>(p.gate) + w.b * p.gb + w.c;
    T* const y = static_cast<T*>(p.y) + (long long)w.b * p.T * p.C + w.c;
    auto load = [&](int t0) {
        const T *px = x + t0 * p.xt, *pg = g + t0 * p.gt;
        const int n = w.mine ? w.len - t0 : 0;
        if (n >= L) {
#pragma unroll
            for (int i = 0; i < L; ++i, px += p.xt, pg += p.gt) {
                feed.reg[0][i] = __ldcs(reinterpret_cast<const Raw*>(px));
                feed.reg[1][i] = __ldcs(reinterpret_cast<const Raw*>(pg));
            }
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i, px += p.xt, pg += p.gt) {
                feed.reg[0][i] = i < n ? __ldcs(reinterpret_cast<const Raw*>(px)) : feed.nothing(0);
                feed.reg[1][i] = i < n ? __ldcs(reinterpret_cast<const Raw*>(pg)) : feed.nothing(1);
            }
        }
    };
    float* const cluster_part = smem + (size_t)2 * w.warps * 3 * width;
    N carry = load_state<VEC>(p.state + (long long)w.b * p.C + w.c, p.state && w.mine);
    int t0 = w.rank * tile + w.run * L;
    // (tokens are counted in 64 bits where a stride may end beyond 2^31)
    auto order = [&](long long s0) {
        if (s0 < w.len) feed.order(maps, w.c - w.at, (int)s0 + w.rank * tile, w.b);
    };
    if constexpr (TMA) {
        for (int k = 0; k < p.stages; ++k) order((long long)k * stride);
    } else {
        load(t0);
    }
    if (w.ctas > 1) cluster.barrier_wait();
    for (int s0 = 0, buf = 0; s0 < w.len; s0 += stride, t0 += stride, buf ^= 1) {
        bool ok = true;
        if constexpr (TMA) ok = feed.ready(w.mine ? w.len - t0 : 0);
        float *const steps = smem + (size_t)buf * w.warps * 3 * width + 2 * w.at, *const adds = smem + (size_t)(buf * 3 + 2) * w.warps * width + w.at;
        N a[L], u[L], h = N::all(0.f);
        Collect<FORM, VEC> all;
#pragma unroll
        for (int i0 = 0; i0 < L; i0 += 4) {
            Raw rx[4], rg[4];
            feed.four(0, i0, rx);
            feed.four(1, i0, rg);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = i0 + j;
                const N gate = gate_of<T, VEC, FORM>(rg[j]), x = P::get(rx[j]);
                N rest;
                open_gate<FORM, VEC>(gate, a[i], rest);
                u[i] = FORM == M2D_GATE_DECAY ? x : mul_(rest, x);
                all.add(gate, a[i], rest);
                h = fma_(a[i], h, u[i]);
            }
        }
        if (!TMA && s0 + stride < w.len) load(t0 + stride);
        Step<VEC> step = all.done();
        N add = ok ? h : N::all(__int_as_float(0x7fc00000));
        join_warp<VEC, LANES, true>(step, add);
        if (w.last) {
            give2(steps + 2 * w.warp * width, step.hi, step.lo);
            give(adds + w.warp * width, add);
        }
        __syncthreads();
        if constexpr (TMA) feed.next();
        if (w.ctas > 1) {
            // one warp joins the tile's runs and tells every CTA of the cluster
            float* const tiles = cluster_part + (size_t)buf * w.ctas * 3 * width;
            if (threadIdx.x < LANES && !*waits.apart) {
                Step<VEC> whole{N::all(1.f), N::all(0.f)};
                N sum = N::all(0.f);
#pragma unroll 8
                for (int k = 0; k < w.warps; ++k) {
                    const Two<VEC> s = take2<VEC>(steps + 2 * k * width);
                    const Step<VEC> next{s.a, s.b};
                    sum = next.apply(sum, take<VEC>(adds + k * width));
                    whole.times(next);
                }
                const float* const to = tiles + w.rank * 3 * width;
                for (int k = 0; k < w.ctas; ++k) waits.send<VEC>(k, to + 2 * w.at, to + 2 * width + w.at, whole, sum, turn & 1);
            }
            if (!waits.joined(turn++, join_bytes)) ok = false;
            h = carry;
            for (int k = 0; k < w.ctas; ++k) {
                if (k == w.rank) h = carry;
                const Two<VEC> s = take2<VEC>(tiles + k * 3 * width + 2 * w.at);
                carry = Step<VEC>{s.a, s.b}.apply(carry, take<VEC>(tiles + k * 3 * width + 2 * width + w.at));
            }
            if (!ok) carry = N::all(__int_as_float(0x7fc00000));
        } else {
            h = carry;
        }
#pragma unroll 4
        for (int k = 0; k < w.warp; ++k) {
            const Two<VEC> s = take2<VEC>(steps + 2 * k * width);
            h = Step<VEC>{s.a, s.b}.apply(h, take<VEC>(adds + k * width));
        }
        if (w.ctas == 1) {
            carry = h;
#pragma unroll 4
            for (int k = w.warp; k < w.warps; ++k) {
                const Two<VEC> s = take2<VEC>(steps + 2 * k * width);
                carry = Step<VEC>{s.a, s.b}.apply(carry, take<VEC>(adds + k * width));
            }
        }
        h = after_others<VEC, LANES, true>(step, add, h);
        if (!ok) h = N::all(__int_as_float(0x7fc00000));
        const int n = w.mine ? w.len - t0 : 0;
        if (p.marks && n > 0 && t0 % kMark == 0) store_state<VEC>(p.marks + ((long long)w.b * ((p.T + kMark - 1) / kMark) + t0 / kMark) * p.C + w.c, h);
        char* const py = reinterpret_cast<char*>(y + (long long)t0 * p.C);
        const unsigned row = (unsigned)p.C * (unsigned)sizeof(T);
        if (n >= L) {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                h = fma_(a[i], h, u[i]);
                *reinterpret_cast<Raw*>(py + (unsigned long long)row * (unsigned)i) = P::put(h);
            }
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i) {
                h = fma_(a[i], h, u[i]);
                if (i < n) *reinterpret_cast<Raw*>(py + (unsigned long long)row * (unsigned)i) = P::put(h);
            }
        }
        // (all have read the stage; asked for last, since the others wait for what this thread's warp joins)
        if constexpr (TMA) order((long long)s0 + (long long)p.stages * stride);
    }
    feed.leave(p.host_flag);
    if (w.ctas > 1) cluster.sync();                       // (none leaves while another may still write to it)
    if (!w.mine) return;
    for (long long t = (long long)w.len + w.rank * w.runs + w.run; t < p.T; t += w.ctas * w.runs) *reinterpret_cast<Raw*>(y + t * p.C) = P::fill(0.f);
    if (p.state_out && w.rank == 0 && w.run == 0) store_state<VEC>(p.state_out + (long long)w.b * p.C + w.c, carry);
}

// Tiles from the last to the first.  The states inside a tile come from the forward pass's mark before it: only what flows back is joined
// between CTAs.
template <typename T, int VEC, int FORM, int L, int LANES, bool TMA>
__global__ void __launch_bounds__(kRecurWarps * 32) recur_bwd_kernel(const RecurArgs p, const __grid_constant__ RecurMaps maps) {
    namespace cg = cooperative_groups;
    using P = Piece<T, VEC>;
    using Raw = typename P::Raw;
    using N = Num<VEC>;
    constexpr int width = LANES * VEC;
    extern __shared__ __align__(128) char ring[];
    const Place<VEC, LANES> w(p);
    cg::cluster_group cluster = cg::this_cluster();
    const int tile = w.runs * L, stride = w.ctas * tile;
    float* const smem = reinterpret_cast<float*>(ring + (TMA ? p.stages * (size_t)3 * tile * width * sizeof(T) : 0));
    const Waits waits(p, reinterpret_cast<char*>(smem + 2 * width * (w.warps * 4 + (w.ctas > 1 ? w.ctas * 3 : 0))));
    if (w.ctas > 1) cluster.barrier_arrive();             // (all have begun, their barriers too, before one writes to another)
    Feed<T, VEC, FORM, L, LANES, 3, TMA> feed(p, w, ring, waits);
    const uint32_t join_bytes = (uint32_t)w.ctas * 3 * width * sizeof(float);
    int turn = 0;
    const T* const x = static_cast<const T*>(p.x) + w.b * p.xb + w.c;
    const T* const g = static_cast<const T*>(p.gate) + w.b * p.gb + w.c;
    const T* const dy = static_cast<const T*>(p.dy) + w.b * p.db + w.c;
    const long long out = (long long)w.b * p.T * p.C + w.c;
    T *const dx = static_cast<T*>(p.dx) + out, *const dgate = static_cast<T*>(p.dgate) + out;
    const float* const marks = p.marks + (long long)w.b * ((p.T + kMark - 1) / kMark) * p.C + w.c;
    float mark[VEC];                                      // (packed where it is used: nothing waits for it before)
    auto load = [&](int t1) {
        if constexpr (!TMA) {
            const int t0 = t1 + w.run * L, n = w.mine ? w.len - t0 : 0;
            const T *px = x + t0 * p.xt, *pg = g + t0 * p.gt, *pd = dy + t0 * p.dt;
            if (n >= L) {
#pragma unroll
                for (int i = 0; i < L; ++i, px += p.xt, pg += p.gt, pd += p.dt) {
                    feed.reg[0][i] = __ldcs(reinterpret_cast<const Raw*>(px));
                    feed.reg[1][i] = __ldcs(reinterpret_cast<const Raw*>(pg));
                    feed.reg[2][i] = __ldcs(reinterpret_cast<const Raw*>(pd));
                }
            } else {
#pragma unroll
                for (int i = 0; i < L; ++i, px += p.xt, pg += p.gt, pd += p.dt) {
                    feed.reg[0][i] = i < n ? __ldcs(reinterpret_cast<const Raw*>(px)) : feed.nothing(0);
                    feed.reg[1][i] = i < n ? __ldcs(reinterpret_cast<const Raw*>(pg)) : feed.nothing(1);
                    feed.reg[2][i] = i < n ? __ldcs(reinterpret_cast<const Raw*>(pd)) : feed.nothing(2);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) mark[v] = w.mine && t1 < w.len ? marks[(long long)(t1 / kMark) * p.C + v] : 0.f;
    };
    float* const cluster_part = smem + (size_t)2 * w.warps * 4 * width;
    N carry = load_state<VEC>(p.d_state_out + (long long)w.b * p.C + w.c, p.d_state_out && w.mine);
    int s0 = w.len > 0 ? (w.len - 1) / stride * stride : -1;
    auto order = [&](int s0) {
        if (s0 >= 0) feed.order(maps, w.c - w.at, s0 + w.rank * tile, w.b);
    };
    int asked = s0;                                       // the next stride to ask for
    if constexpr (TMA)
        for (int k = 0; k < p.stages && asked >= 0; ++k, asked -= stride) order(asked);
    if (s0 >= 0) load(s0 + w.rank * tile);
    if (w.ctas > 1) cluster.barrier_wait();
    bool again = false;                                   // from the second stride on the stage of the one before is free
    for (int buf = 0; s0 >= 0; s0 -= stride, buf ^= 1) {
        const int t0 = s0 + w.rank * tile + w.run * L;
        bool ok = true;
        if constexpr (TMA) ok = feed.ready(w.mine ? w.len - t0 : 0);
        float *const steps = smem + (size_t)buf * w.warps * 4 * width + 2 * w.at, *const adds = steps + (size_t)w.warps * 2 * width;
        N a[L], rest[L], before[L], h = N::all(0.f), R = N::all(0.f);
        Collect<FORM, VEC> all;
#pragma unroll
        for (int i0 = 0; i0 < L; i0 += 4) {
            Raw rx[4], rg[4];
            feed.four(0, i0, rx);
            feed.four(1, i0, rg);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = i0 + j;
                const N gate = gate_of<T, VEC, FORM>(rg[j]), x = P::get(rx[j]);
                open_gate<FORM, VEC>(gate, a[i], rest[i]);
                all.add(gate, a[i], rest[i]);
                h = fma_(a[i], h, FORM == M2D_GATE_DECAY ? x : mul_(rest[i], x));
            }
        }
#pragma unroll
        for (int i0 = L - 4; i0 >= 0; i0 -= 4) {
            Raw rd[4];
            feed.four(2, i0, rd);
#pragma unroll
            for (int j = 3; j >= 0; --j) R = mul_(a[i0 + j], add_(P::get(rd[j]), R));
        }
        Raw xs[TMA ? 1 : L], ds[TMA ? 1 : L];             // (of a tile in shared memory x and dy are read again instead)
        if constexpr (!TMA)
#pragma unroll
            for (int i = 0; i < L; ++i) {
                xs[i] = feed.reg[0][i];
                ds[i] = feed.reg[2][i];
            }
        auto four = [&](int t, int i, Raw (&r)[4]) {
            if constexpr (TMA) {
                feed.four(t, i, r);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = t == 0 ? xs[i + j] : ds[i + j];
            }
        };
        N first = N::all(mark[0]);
        if constexpr (VEC == 2) first.set(1, mark[1]);
        if (s0 >= stride) load(s0 - stride + w.rank * tile);
        Step<VEC> up = all.done(), down = up;
        const N nan = N::all(__int_as_float(0x7fc00000));
        N add = ok ? h : nan, flow = ok ? R : nan;
        join_warp<VEC, LANES, true>(up, add);
        join_warp<VEC, LANES, false>(down, flow);
        if (w.last) {
            give2(steps + 2 * w.warp * width, up.hi, up.lo);
            give(adds + 2 * w.warp * width, add);
        }
        if (w.first) give(adds + 2 * w.warp * width + VEC, flow);
        __syncthreads();
        if constexpr (TMA)                    // (at once: there may be but two stages)
            if (again && asked >= 0) {
                order(asked);
                asked -= stride;
            }
        again = true;
        auto back = [&](int k, N from) {
            const Two<VEC> s = take2<VEC>(steps + 2 * k * width);
            return Step<VEC>{s.a, s.b}.apply(from, take<VEC>(adds + 2 * k * width + VEC));
        };
        if (w.ctas > 1) {
            float* const tiles = cluster_part + (size_t)buf * w.ctas * 3 * width;
            if (threadIdx.x < LANES && !*waits.apart) {
                Step<VEC> whole{N::all(1.f), N::all(0.f)};
                N sum = N::all(0.f);
#pragma unroll 8
                for (int k = w.warps - 1; k >= 0; --k) {
                    const Two<VEC> s = take2<VEC>(steps + 2 * k * width);
                    const Step<VEC> next{s.a, s.b};
                    sum = next.apply(sum, take<VEC>(adds + 2 * k * width + VEC));
                    whole.times(next);
                }
                const float* const to = tiles + w.rank * 3 * width;
                for (int k = 0; k < w.ctas; ++k) waits.send<VEC>(k, to + 2 * w.at, to + 2 * width + w.at, whole, sum, turn & 1);
            }
            if (!waits.joined(turn++, join_bytes)) ok = false;
            R = carry;
            for (int k = w.ctas - 1; k >= 0; --k) {
                if (k == w.rank) R = carry;
                const Two<VEC> s = take2<VEC>(tiles + k * 3 * width + 2 * w.at);
                carry = Step<VEC>{s.a, s.b}.apply(carry, take<VEC>(tiles + k * 3 * width + 2 * width + w.at));
            }
            if (!ok) carry = nan;
        } else {
            R = carry;
        }
#pragma unroll 4
        for (int k = w.warps - 1; k > w.warp; --k) R = back(k, R);
        if (w.ctas == 1) {
            carry = R;
#pragma unroll 4
            for (int k = w.warp; k >= 0; --k) carry = back(k, carry);
        }
        R = after_others<VEC, LANES, false>(down, flow, R);
        h = first;
#pragma unroll 4
        for (int k = 0; k < w.warp; ++k) {
            const Two<VEC> s = take2<VEC>(steps + 2 * k * width);
            h = Step<VEC>{s.a, s.b}.apply(h, take<VEC>(adds + 2 * k * width));
        }
        h = after_others<VEC, LANES, true>(up, add, h);
        if (!ok) h = R = nan;
#pragma unroll
        for (int i0 = 0; i0 < L; i0 += 4) {
            Raw rx[4];
            four(0, i0, rx);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const N x = P::get(rx[j]);
                before[i0 + j] = FORM == M2D_GATE_DECAY ? h : fma_(x, N::all(-1.f), h);        // (forget: h_{t-1} - x_t)
                h = fma_(a[i0 + j], h, FORM == M2D_GATE_DECAY ? x : mul_(rest[i0 + j], x));
            }
        }
        const int n = w.mine ? w.len - t0 : 0;
        char *const px = reinterpret_cast<char*>(dx + (long long)t0 * p.C), *const pg = reinterpret_cast<char*>(dgate + (long long)t0 * p.C);
        const unsigned row = (unsigned)p.C * (unsigned)sizeof(T);
        auto write = [&](auto whole) {
#pragma unroll
            for (int i0 = L - 4; i0 >= 0; i0 -= 4) {
                Raw rd[4];
                four(2, i0, rd);
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    const int i = i0 + j;
                    const N D = add_(P::get(rd[j]), R);
                    R = mul_(a[i], D);
                    const N gx = FORM == M2D_GATE_DECAY ? D : mul_(rest[i], D);
                    const N gg = FORM == M2D_GATE_DECAY ? mul_(R, before[i]) : mul_(mul_(rest[i], R), before[i]);
                    if (whole.value || i < n) {
                        *reinterpret_cast<Raw*>(px + (unsigned long long)row * (unsigned)i) = P::put(gx);
                        *reinterpret_cast<Raw*>(pg + (unsigned long long)row * (unsigned)i) = P::put(gg);
                    }
                }
            }
        };
        if (n >= L) write(std::true_type{});
        else write(std::false_type{});
        if constexpr (TMA) feed.next();
    }
    feed.leave(p.host_flag);
    if (w.ctas > 1) cluster.sync();                       // (none leaves while another may still write to it)
    if (!w.mine) return;
    for (long long t = (long long)w.len + w.rank * w.runs + w.run; t < p.T; t += w.ctas * w.runs) {
        *reinterpret_cast<Raw*>(dx + t * p.C) = P::fill(0.f);
        *reinterpret_cast<Raw*>(dgate + t * p.C) = P::fill(0.f);
    }
    if (p.d_state && w.rank == 0 && w.run == 0) store_state<VEC>(p.d_state + (long long)w.b * p.C + w.c, carry);
}

// One token of every sequence.  state and state_out may be the same array.  Where half or more of the state stays, it is moved by its increment, (a - 1) h + u or
// (1 - f) (x - h), instead of multiplied by a: a's rounding would come back with every token of the same gate, and add up over its memory (8192 tokens
// long: the state was off by 1.0e-4 to 1.5e-4 after 2000 tokens, by increments it is off by at most 6e-6 after 20000).  An increment that is not finite is not taken.
template <typename T, int VEC, int FORM>
__global__ void __launch_bounds__(128) recur_step_kernel(const RecurArgs p, long long sb) {
    using P = Piece<T, VEC>;
    using Raw = typename P::Raw;
    const int c = (blockIdx.x * 128 + threadIdx.x) * VEC;
    if (c >= p.C) return;
    for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
        using N = Num<VEC>;
        const N x = P::get(*reinterpret_cast<const Raw*>(static_cast<const T*>(p.x) + b * p.xb + c)), g = gate_of<T, VEC, FORM>(*reinterpret_cast<const Raw*>(static_cast<const T*>(p.gate) + b * p.gb + c));
        const N h = load_state<VEC>(p.state + b * sb + c, true);
        N a, rest;
        open_gate<FORM, VEC>(g, a, rest);
        N to = fma_(a, h, FORM == M2D_GATE_DECAY ? x : mul_(rest, x)), move, moved;
        if constexpr (FORM == M2D_GATE_DECAY) {
            move = fma_(less_one(g), h, x);
            moved = add_(h, move);
        } else {
            move = add_(x, neg_(h));
            moved = fma_(rest, move, h);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (a.get(v) >= 0.5f && a.get(v) <= 2.f && fabsf(move.get(v)) <= 3.402823466e38f) to.set(v, moved.get(v));
        store_state<VEC>(p.state_out + b * sb + c, to);
        *reinterpret_cast<Raw*>(static_cast<T*>(p.y) + (long long)b * p.C + c) = P::put(to);
    }
}

static int check_recur(const m2d_recur_desc* d, bool step) {
    if (!d) return M2D_ERR_NULL;
    if (d->struct_bytes != sizeof(m2d_recur_desc)) return M2D_ERR_ABI;
    if (d->dtype != M2D_F32 && d->dtype != M2D_BF16) return M2D_ERR_DTYPE;
    if (d->form != M2D_GATE_DECAY && d->form != M2D_GATE_FORGET) return M2D_ERR_FLAGS;
    if (d->flags && !(d->flags == M2D_RECUR_TEST_GIVE_UP && test_hooks_enabled())) return M2D_ERR_FLAGS;
    if (d->B < 1 || d->T < 1 || d->C < 1 || (step && d->T != 1)) return M2D_ERR_SHAPE;
    // (tokens are counted in 32 bits, a tile beyond the last included; CTAs and the bytes of a row too)
    if (d->T > INT32_MAX - (1 << 17) || d->C > (1 << 29) || (long long)d->B * ((d->C + 31) / 32) > INT32_MAX / 16) return M2D_ERR_TOO_LARGE;
    const uintptr_t es = d->dtype == M2D_F32 ? 4 : 2;
    for (const void* t : {d->x.data, d->gate.data})
        if (!t) return M2D_ERR_NULL;
    for (const void* t : {d->x.data, d->gate.data, d->d_y.data, static_cast<const void*>(d->y), static_cast<const void*>(d->d_x), static_cast<const void*>(d->d_gate)})
        if (reinterpret_cast<uintptr_t>(t) % es) return M2D_ERR_PITCH;
    for (const void* t : {static_cast<const void*>(d->lengths), static_cast<const void*>(d->state), static_cast<const void*>(d->state_out), static_cast<const void*>(d->marks),
                          static_cast<const void*>(d->d_state_out), static_cast<const void*>(d->d_state)})
        if (reinterpret_cast<uintptr_t>(t) % 4) return M2D_ERR_PITCH;
    return M2D_OK;
}
static bool pairs_ok(const void* p, long long a, long long b, int es) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (2 * es) == 0 && a % 2 == 0 && b % 2 == 0); }
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
// Calls fn(element, channels of a lane, form): two channels where rows are whole pieces of two.
template <typename F>
static int for_recur(const m2d_recur_desc* d, bool pairs, F fn) {
    using std::integral_constant;
    auto with_form = [&](auto elem, auto vec) {
        return d->form == M2D_GATE_DECAY ? fn(elem, vec, integral_constant<int, M2D_GATE_DECAY>{}) : fn(elem, vec, integral_constant<int, M2D_GATE_FORGET>{});
    };
    if (d->dtype == M2D_F32) return pairs ? with_form(float{}, integral_constant<int, 2>{}) : with_form(float{}, integral_constant<int, 1>{});
    return pairs ? with_form(__nv_bfloat16{}, integral_constant<int, 2>{}) : with_form(__nv_bfloat16{}, integral_constant<int, 1>{});
}
// Lanes of a row, warps of a CTA and CTAs of a cluster: the least time by a model of it.  An SM holds 16 warps (128 registers a
// thread); clusters of 4 and 8 leave some SMs of a GPC over (of CTAs of 16 warps 33 and 15 fit 148 SMs, of 8 warps 71 and 33).  All clusters run in so many waves, and each takes so many
// strides; a stride takes about a time of 10 for its chain of load, joins and store and 1 for each warp of the SM (its instructions), the start of a wave 30
// (some 3 us).
// Rows in pieces of 16 or 8 lanes (64 and 32 bytes of bf16), larger clusters and CTAs that have an SM for themselves cost a little more; the
// backward pass without TMA spills registers there and takes twice as long.
struct RecurPlan { int lanes, warps, ctas; };
// Tiles that a CTA's share of an SM's memory has room for, beside the joins.
static int recur_stages(const RecurPlan& pl, int vec, int steps, int tensors, int es) {
    const int width = pl.lanes * vec, tile = pl.warps * (32 / pl.lanes) * steps;
    const size_t used = recur_joins(tensors + 1, pl.warps, pl.ctas, width) + kRecurTail, share = pl.warps > 8 ? kMaxSmem : kMaxSmem * pl.warps / kRecurWarps - 512;
    return share > used ? (int)std::min<size_t>(kRecurStages, (share - used) / recur_stage(tensors, tile, width, es)) : 0;
}
// By TMA (fed) there is room for the tile, and for two where there are several strides.
static RecurPlan plan_recur(const m2d_recur_desc* d, int vec, int steps, int tensors, bool fed) {
    const long long runs = (d->T + steps - 1) / steps, sms = sm_count();
    const bool bwd = tensors == 3;
    RecurPlan best{32, 0, 1};
    double least = 1e300;
    for (int lanes = 32; lanes >= (vec == 2 ? 8 : 32); lanes /= 2) {
        const long long chains = (long long)d->B * ((d->C + lanes * vec - 1) / (lanes * vec));
        for (int warps = 1; warps <= kRecurWarps; warps *= 2)
            for (int ctas = 1; ctas <= kRecurCluster; ctas *= 2) {
                const long long tile = (long long)warps * (32 / lanes);            // in runs
                if (ctas > 1 && tile * (ctas / 2) >= runs) break;                  // (half of them would do)
                if (bwd && tile * steps % kMark && (ctas > 1 || tile < runs)) continue;        // (a tile begins at a mark)
                if (fed && recur_stages({lanes, warps, ctas}, vec, steps, tensors, d->dtype == M2D_F32 ? 4 : 2) < (tile * ctas < runs ? 2 : 1)) continue;
                const long long eights = (ctas == 8 ? 33 : ctas == 4 ? 71 : 296 / ctas) * sms / 148;            // clusters of CTAs of eight warps
                const long long held = std::max(1ll, warps == 16 ? (ctas == 8 ? 15 : ctas == 4 ? 33 : 148 / ctas) * sms / 148 : eights * 8 / warps);
                const long long waves = (chains + held - 1) / held, strides = (runs + tile * ctas - 1) / (tile * ctas);
                const long long per_sm = std::min<long long>(kRecurWarps, (chains * ctas + sms - 1) / sms * warps);
                const double t = (double)waves * (30 + strides * (10 + per_sm)) * (warps == 16 ? 1.1 : 1.0) * (lanes == 32 ? 1.0 : bwd && !fed ? 2.0 : lanes == 16 ? 1.05 : 1.15) * (ctas == 1 ? 1.0 : 1.1 + 0.02 * ctas);
                if (t < least) { least = t; best = {lanes, warps, ctas}; }
            }
    }
    return best;
}
// Whether a tensor can be fetched by TMA: 16-byte aligned rows.  (A stride that no step is taken along may be anything: the map gets a valid one.)
static bool recur_fits(const m2d_recur_desc* d, const m2d_recur_tensor& t, int es) {
    auto stride = [&](int n, int64_t s) { return n == 1 || (s > 0 && s * es % 16 == 0 && s * es < (1ll << 39)); };
    return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && stride(d->T, t.token) && stride(d->B, t.batch);
}
static bool recur_map(CUtensorMap* map, const m2d_recur_desc* d, const m2d_recur_tensor& t, int es, int width, int box) {
    const cuuint64_t dims[3] = {(cuuint64_t)d->C, (cuuint64_t)d->T, (cuuint64_t)d->B};
    const cuuint64_t strides[2] = {d->T == 1 ? 16 : (cuuint64_t)t.token * es, d->B == 1 ? 16 : (cuuint64_t)t.batch * es};
    const cuuint32_t boxes[3] = {(cuuint32_t)width, (cuuint32_t)box, 1}, step[3] = {1, 1, 1};
    return tc_encoder()(map, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(t.data), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Calls fn(plan, whether by TMA, maps, shared memory): TENSORS of two or three, runs of `fed` tokens by TMA and of `plain` without.
template <int TENSORS, typename F>
static int with_recur(const m2d_recur_desc* d, RecurArgs& a, int vec, int fed, int plain, F fn) {
    const int es = d->dtype == M2D_F32 ? 4 : 2;
    RecurMaps maps{};
    if (vec == 2 && recur_fits(d, d->x, es) && recur_fits(d, d->gate, es) && (TENSORS == 2 || recur_fits(d, d->d_y, es)) && tc_encoder()) {
        const RecurPlan pl = plan_recur(d, vec, fed, TENSORS, true);
        const int width = pl.lanes * vec, tile = pl.warps * (32 / pl.lanes) * fed;
        a.stages = pl.warps ? recur_stages(pl, vec, fed, TENSORS, es) : 0;
        a.box = std::min(tile, 256);
        // forward a single stride takes as long without; backward the form by TMA needs fewer registers (25x2010x192 bf16 32 us for 54)
        if (a.stages && ((long long)tile * pl.ctas < d->T || (TENSORS == 3 && d->T >= kMark)) && recur_map(&maps.x, d, d->x, es, width, a.box) &&
            recur_map(&maps.gate, d, d->gate, es, width, a.box) && (TENSORS == 2 || recur_map(&maps.dy, d, d->d_y, es, width, a.box))) {
            a.host_flag = wait_failure_flag();
            a.give_up = (d->flags & M2D_RECUR_TEST_GIVE_UP) != 0;
            return fn(pl, true, maps, recur_joins(TENSORS + 1, pl.warps, pl.ctas, width) + kRecurTail + a.stages * recur_stage(TENSORS, tile, width, es));
        }
    }
    const RecurPlan pl = plan_recur(d, vec, plain, TENSORS, false);
    a.host_flag = pl.ctas > 1 ? wait_failure_flag() : nullptr;
    return fn(pl, false, maps, recur_joins(TENSORS + 1, pl.warps, pl.ctas, pl.lanes * vec) + kRecurTail);
}
template <typename K>
static int launch_recur(K kern, const RecurArgs& a, const RecurMaps& maps, const RecurPlan& pl, size_t smem, cudaStream_t st) {
    if (!allow_smem(reinterpret_cast<const void*>(kern), smem)) return M2D_ERR_LAUNCH;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a.B * a.groups * pl.ctas));
    cfg.blockDim = dim3(pl.warps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = pl.ctas; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, a, maps) != cudaSuccess) { cudaGetLastError(); return M2D_ERR_LAUNCH; }
    return M2D_OK;
}
// Calls fn(lanes) with the plan's; rows of single values are not cut.
template <int VEC, typename F>
static int for_lanes(int lanes, F fn) {
    using std::integral_constant;
    if constexpr (VEC == 2) {
        if (lanes == 8) return fn(integral_constant<int, 8>{});
        if (lanes == 16) return fn(integral_constant<int, 16>{});
    }
    return fn(integral_constant<int, 32>{});
}
// Tokens of a run, by the registers that they take (and in the backward pass the shared memory).
template <typename T> constexpr int kFwdSteps = sizeof(T) == 4 ? 8 : 16;
template <typename T> constexpr int kBwdSteps = sizeof(T) == 4 ? 8 : 16;
constexpr int kBwdPlain = 8;

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
    const int es = d->dtype == M2D_F32 ? 4 : 2;
    const bool pairs = d->C % 2 == 0 && pairs_ok(a.x, a.xb, a.xt, es) && pairs_ok(a.gate, a.gb, a.gt, es) && pairs_ok(a.y, 0, 0, es);
    return for_recur(d, pairs, [&](auto elem, auto vec, auto form) {
        using T = decltype(elem);
        constexpr int VEC = decltype(vec)::value, FORM = decltype(form)::value, L = kFwdSteps<T>;
        return with_recur<2>(d, a, VEC, L, L, [&](const RecurPlan& pl, bool fed, const RecurMaps& maps, size_t smem) {
            return for_lanes<VEC>(pl.lanes, [&](auto lanes) {
                constexpr int LANES = decltype(lanes)::value;
                a.groups = (d->C + LANES * VEC - 1) / (LANES * VEC);
                a.ctas = pl.ctas;
                return launch_recur(fed ? recur_fwd_kernel<T, VEC, FORM, L, LANES, VEC == 2> : recur_fwd_kernel<T, VEC, FORM, L, LANES, false>, a, maps, pl, smem, static_cast<cudaStream_t>(stream));
            });
        });
    });
}

extern "C" int m2d_recur_bwd(const m2d_recur_desc* d, void* stream) {
    const int rc = check_recur(d, false);
    if (rc != M2D_OK) return rc;
    if (!d->d_y.data || !d->d_x || !d->d_gate || !d->marks) return M2D_ERR_NULL;
    RecurArgs a = recur_args(d);
    const int es = d->dtype == M2D_F32 ? 4 : 2;
    const bool pairs = d->C % 2 == 0 && pairs_ok(a.x, a.xb, a.xt, es) && pairs_ok(a.gate, a.gb, a.gt, es) && pairs_ok(a.dy, a.db, a.dt, es) && pairs_ok(a.dx, 0, 0, es) && pairs_ok(a.dgate, 0, 0, es);
    return for_recur(d, pairs, [&](auto elem, auto vec, auto form) {
        using T = decltype(elem);
        constexpr int VEC = decltype(vec)::value, FORM = decltype(form)::value, L = kBwdSteps<T>;
        return with_recur<3>(d, a, VEC, L, kBwdPlain, [&](const RecurPlan& pl, bool fed, const RecurMaps& maps, size_t smem) {
            return for_lanes<VEC>(pl.lanes, [&](auto lanes) {
                constexpr int LANES = decltype(lanes)::value;
                a.groups = (d->C + LANES * VEC - 1) / (LANES * VEC);
                a.ctas = pl.ctas;
                return launch_recur(fed ? recur_bwd_kernel<T, VEC, FORM, VEC == 2 ? L : kBwdPlain, LANES, VEC == 2> : recur_bwd_kernel<T, VEC, FORM, kBwdPlain, LANES, false>, a, maps, pl, smem,
                                    static_cast<cudaStream_t>(stream));
            });
        });
    });
}

extern "C" int m2d_recur_step(const m2d_recur_desc* d, int64_t state_batch, void* stream) {
    const int rc = check_recur(d, true);
    if (rc != M2D_OK) return rc;
    if (!d->y || !d->state || !d->state_out) return M2D_ERR_NULL;
    const RecurArgs a = recur_args(d);
    const int es = d->dtype == M2D_F32 ? 4 : 2;
    const bool pairs = d->C % 2 == 0 && pairs_ok(a.x, a.xb, 0, es) && pairs_ok(a.gate, a.gb, 0, es) && pairs_ok(a.y, 0, 0, es);
    return for_recur(d, pairs, [&](auto elem, auto vec, auto form) {
        using T = decltype(elem);
        constexpr int VEC = decltype(vec)::value, FORM = decltype(form)::value;
        const dim3 grid((d->C + 128 * VEC - 1) / (128 * VEC), std::min(d->B, 65535));
        recur_step_kernel<T, VEC, FORM><<<grid, 128, 0, static_cast<cudaStream_t>(stream)>>>(a, (long long)state_batch);
        return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
    });
}
