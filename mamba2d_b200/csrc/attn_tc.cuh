// attn_core.cuh's computation on the 5th-generation tensor cores: bf16 tensors, head sizes up to 128.
//
// A chunk is 128 tokens, the rows of one accumulator.  Per chunk, with the tiles of x, y, z in shared memory (TMA, 128-byte
// swizzle, blocks of 128 rows x 64 columns) and St in bf16 next to them:
//     (1)  pairs = x y^T            128 x 128    both operands as they arrived
//     (2)  O2    = x St             128 x VD
//     (3)  O1    = P z              128 x VD     P = s_intra D pairs, bf16 in tensor memory in the place of pairs
//     (4)  delta = (u y)^T z        KD x VD      u y scaled in place, in two bf16 parts: St is carried in fp32 and a state
//                                                is an output; one part would leave it at 2^-9
//     out = O1 + s_inter w O2,  St <- exp(c_end) St + delta
// The work is dealt to warps that wait on one another through mbarriers only:
//     warps 0 - 3   a token row a thread: pairs -> P, O1 and O2 -> out
//     warps 4 - 7   a token row a thread: y -> u y; a row of St a thread: St in registers, its bf16 copy in shared memory
//     warp 8        TMA loads into a ring of tiles        warp 9   issues the products       warp 10   the decays' tables
// Decays: c is summed in 64 bits; D_rc of one 32 x 32 block on the diagonal is exp of a difference that the table holds in
// two floats, and factors into exp(c_r - b) exp(b - c_c) elsewhere, b the sum up to the row block: both at most one, and
// 32 exponentials a row instead of 128.
//
// `fine` (wanted where the decay's gradient is): P and St also in two parts each, so that the dots that out is summed
// into are exact to 2^-17 like the states that they meet.
//
// Every wait is bounded: one that gives up makes all of the CTA's roles leave, rows not written yet become NaN, and a word in
// host memory says so.
#pragma once

#include "attn_core.cuh"
#include "tc_ptx.cuh"

namespace m2d {

constexpr int kTc = 128;                      // tokens of a chunk
constexpr int kTcThreads = 352;
constexpr int kTcBlock = kTc * 128;           // 128 rows x 64 columns of bf16
constexpr int kTcMaxSlots = 12;

struct TcMaps { CUtensorMap m[3][3]; };       // [core][x, y, z]
struct TcLaunch {
    AttnLaunch a;
    int cores, slots;
    int fine;                                 // bit per core
    int* host_flag;
};

// ---- PTX ---------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                   "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Operand descriptors of the 128-byte-swizzle layout (wgrad_tc.cuh): contraction along the 128-byte rows ("K-major"), or across
// them ("MN-major", `next` bytes to the next 64 columns).
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t next) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return desc_mn(addr, 16); }
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// Decay tables of a chunk, in log2 where they are not exponentials yet.
struct alignas(16) TcTable {
    float2 l[kTc];          // c within the 32-token block, in two floats
    float u[kTc];           // update weight times s_update
    float f[192];           // exp(b - c_c): columns of the blocks before (rev: behind) row block 1, 2, 3 (0, 1, 2)
    float2 base[4];         // forwards the sum before the block, backwards from its start to the end
    float2 total[4];        // of the block
    float whole;            // exp(c_end)
};
__device__ __forceinline__ int tc_f(int rev, int i) { return rev ? (i == 0 ? 0 : i == 1 ? 96 : 160) : (i <= 1 ? 0 : i == 2 ? 32 : 96); }

// (KD = 64: a block behind the ring, since (4) computes 128 rows: the upper 64, of whatever lies behind y, are not used)
inline size_t tc_fixed_smem(int KD, int VD, bool fine) { return (size_t)KD * VD * 2 * (fine ? 2 : 1) + (size_t)kTc * KD * 2 + 1024 + (KD == 64 ? kTcBlock : 0); }
inline int tc_slots(int KD, int VD, bool fine) {
    const size_t tile = (size_t)kTc * 2 * (KD > VD ? KD : VD);
    const int n = (int)((kMaxSmem - 2944 - tc_fixed_smem(KD, VD, fine)) / tile);
    return n < kTcMaxSlots ? n : kTcMaxSlots;
}
inline size_t tc_smem(int KD, int VD, bool fine, int slots) { return tc_fixed_smem(KD, VD, fine) + (size_t)slots * kTc * 2 * (KD > VD ? KD : VD); }

template <int KD, int VD, bool STATE_ONLY>
__global__ void __launch_bounds__(kTcThreads, 1) attn_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcLaunch L) {
    extern __shared__ uint8_t tc_smem_raw[];
    __shared__ TcTable tab;
    enum { kSc, kP, kY, kO, kOFree, kDelta, kS, kMma2, kTabFull, kTabFree, kBars };
    __shared__ uint64_t bars[kBars + 2 * kTcMaxSlots];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    constexpr int KB = KD / 64, VB = VD / 64;                     // 64-column blocks
    constexpr uint32_t kTile = kTc * 2 * (KD > VD ? KD : VD);
    constexpr uint32_t kSc0 = 0, kO1 = 128, kO2 = 128 + VD, kDl = 128 + 2 * VD;      // columns of tensor memory
    constexpr uint32_t kCols = STATE_ONLY ? (VD <= 64 ? 64 : 128) : 512;
    constexpr uint32_t kDelta0 = STATE_ONLY ? 0 : kDl;

    const AttnLaunch& a = L.a;
    const int ci = blockIdx.x % L.cores, unit = blockIdx.x / L.cores;
    const AttnCore& k = a.core[ci];
    const bool fine = !STATE_ONLY && (L.fine >> ci & 1);
    const int seg = unit % a.nseg, bh = unit / a.nseg, h = bh % a.H, b = bh / a.H;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rev = k.rev;
    const int len = attn_length(a, b), t_lo = seg * a.seg_len, t_hi = min(a.T, t_lo + a.seg_len);
    const int active = max(0, min(len, t_hi) - t_lo), chunks = (active + kTc - 1) / kTc;         // the others hold nothing

    const uint32_t smem0 = (smem_u32(tc_smem_raw) + 1023u) & ~1023u;
    const uint32_t s_hi = smem0, s_lo = s_hi + KD * VD * 2, y_lo = s_hi + KD * VD * 2 * (fine ? 2 : 1), ring = y_lo + kTc * KD * 2;
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    auto full = [&](int s) { return bar0 + 8u * (kBars + s); };
    auto empty = [&](int s) { return bar0 + 8u * (kBars + kTcMaxSlots + s); };
    volatile int* const abort = &abort_flag;
    constexpr int kTiles = STATE_ONLY ? 2 : 3;                    // a chunk's tiles in the ring: y, x, z
    constexpr int kTileX = 1, kTileZ = kTiles - 1;
    auto slot_of = [&](int it, int tile) { return (it * kTiles + tile) % L.slots; };
    auto phase_of = [&](int it, int tile) { return (uint32_t)((it * kTiles + tile) / L.slots) & 1u; };
    auto tile_at = [&](int it, int tile) { return ring + (uint32_t)slot_of(it, tile) * kTile; };
    auto chunk_at = [&](int it) { return t_lo + (rev ? chunks - 1 - it : it) * kTc; };
    auto wait = [&](uint32_t bar_, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar_, parity, abort)) != 0; };      // whole warps

    if (tid == 0) {
        for (int i = 0; i < kBars; ++i) {
            const int n = i == kP || i == kY || i == kOFree || i == kS ? 4 : i == kTabFree ? (STATE_ONLY ? 4 : 8) : 1;
            mbar_init(bar(i), n);
        }
        for (int s = 0; s < L.slots; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) tmem_alloc(smem_u32(&tmem_slot), kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp < 4) {
        // ---- token rows ----
        if constexpr (!STATE_ONLY) {
            const uint32_t mine = tmem + ((uint32_t)(warp * 32) << 16);
            for (int it = 0; it < chunks; ++it) {
                const int t0 = chunk_at(it), valid = min(kTc, len - t0), r = tid;
                const uint32_t ph = it & 1;
                if (!wait(bar(kTabFull), ph)) break;
                const float2 lr = tab.l[r], base = tab.base[warp], total = tab.total[warp];
                const float w = k.s_inter * (rev ? ex2((base.x - lr.x) + (base.y - lr.y)) : ex2((base.x + lr.x) + (base.y + lr.y)));
                const float e = k.s_intra * (rev ? ex2((total.x - lr.x) + (total.y - lr.y)) : ex2(lr.x + lr.y));
                if (!wait(bar(kSc), ph)) break;
                tc_fence_after();
                uint32_t lo[2][16];                               // second parts that wait for their columns to be read
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v[32];
                    uint32_t hi[16], low[16];
                    const bool on = rev ? j >= warp : j <= warp;
                    tmem_ld32(mine + kSc0 + 32 * j, v);
                    if (on && j == warp) {
                        const float4* const lp = reinterpret_cast<const float4*>(tab.l + 32 * j);
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const float4 lc = lp[c / 2];
                            float d0 = (lr.x - lc.x) + (lr.y - lc.y), d1 = (lr.x - lc.z) + (lr.y - lc.w);
                            if (rev) { d0 = -d0; d1 = -d1; }
                            v[c] = (rev ? c >= lane : c <= lane) ? v[c] * (k.s_intra * ex2(d0)) : 0.f;
                            v[c + 1] = (rev ? c + 1 >= lane : c + 1 <= lane) ? v[c + 1] * (k.s_intra * ex2(d1)) : 0.f;
                        }
                    } else if (on) {
                        const float4* const f = reinterpret_cast<const float4*>(tab.f + tc_f(rev, warp) + (rev ? 32 * (j - warp - 1) : 32 * j));
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            const float4 q = f[c / 4];
                            v[c] *= e * q.x; v[c + 1] *= e * q.y; v[c + 2] *= e * q.z; v[c + 3] *= e * q.w;
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; ++c) v[c] = 0.f;
                    }
                    if (valid < kTc) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) v[c] = 32 * j + c < valid ? v[c] : 0.f;
                    }
#pragma unroll
                    for (int c = 0; c < 16; ++c) hi[c] = pack_bf16x2(v[2 * c], v[2 * c + 1]);
                    tmem_st16(mine + kSc0 + 16 * j, hi);
                    if (fine) {
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            low[c] = pack_bf16x2(v[2 * c] - __uint_as_float(hi[c] << 16), v[2 * c + 1] - __uint_as_float(hi[c] & 0xffff0000u));
                        if (j == 2) {
                            tmem_st16(mine + kSc0 + 64, lo[0]);
                            tmem_st16(mine + kSc0 + 80, lo[1]);
                        }
                        if (j == 3) {
                            tmem_st16(mine + kSc0 + 96, lo[0]);
                            tmem_st16(mine + kSc0 + 112, low);
                        } else {
#pragma unroll
                            for (int c = 0; c < 16; ++c) lo[j & 1][c] = low[c];
                        }
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(kP));
                    mbar_arrive(bar(kTabFree));
                }
                if (!wait(bar(kO), ph)) break;
                tc_fence_after();
                const bool row = t0 + r < t_hi, live = r < valid;
                const long long at = b * k.ob + (long long)(t0 + r) * k.ot + h * k.oh;
                const __nv_bfloat16* const er = k.dots ? static_cast<const __nv_bfloat16*>(attn_at(k.e, b, h, 2)) + (long long)(t0 + r) * k.e.st : nullptr;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < VD / 32; ++j) {
                    float o[32], o2[32];
                    tmem_ld32(mine + kO1 + 32 * j, o);
                    tmem_ld32(mine + kO2 + 32 * j, o2);
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] = live ? fmaf(w, o2[c], o[c]) : 0.f;
                    if (row) {
#pragma unroll
                        for (int c = 0; c < 32; c += 8) {
                            if (32 * j + c >= k.Vd) continue;
                            if (k.out_f32) {
                                float4* p = reinterpret_cast<float4*>(static_cast<float*>(k.out) + at + 32 * j + c);
                                p[0] = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                                p[1] = make_float4(o[c + 4], o[c + 5], o[c + 6], o[c + 7]);
                            } else {
                                *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(k.out) + at + 32 * j + c) =
                                    make_uint4(pack_bf16x2(o[c], o[c + 1]), pack_bf16x2(o[c + 2], o[c + 3]), pack_bf16x2(o[c + 4], o[c + 5]), pack_bf16x2(o[c + 6], o[c + 7]));
                            }
                            if (er && live) {
                                const uint4 q = __ldg(reinterpret_cast<const uint4*>(er + 32 * j + c));
                                const uint32_t qq[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                                for (int i = 0; i < 4; ++i) sum = fmaf(o[c + 2 * i], __uint_as_float(qq[i] << 16), fmaf(o[c + 2 * i + 1], __uint_as_float(qq[i] & 0xffff0000u), sum));
                            }
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kOFree));
                if (k.dots && row) k.dots[((size_t)b * a.T + t0 + r) * a.H + h] = sum;
            }
        }
    } else if (warp < 8) {
        // ---- y and the state ----
        const int r = tid - 128, sw = warp - 4;
        const uint32_t mine = tmem + ((uint32_t)(sw * 32) << 16) + kDelta0;
        float S[VD];
        const bool have_row = r < k.Kd;
#pragma unroll
        for (int c = 0; c < VD; ++c) S[c] = 0.f;
        if (!STATE_ONLY && have_row) {
            const float* init = nullptr;
            long long sr = k.init.sr, sc = k.init.sc;
            if (a.nseg > 1) {
                init = k.seg_state + ((size_t)bh * a.nseg + seg) * k.Kd * k.Vd;
                sr = k.Vd; sc = 1;
            } else if (k.init.p) {
                init = k.init.p + b * k.init.sb + h * k.init.sh;
            }
            if (init && sc == 1 && (reinterpret_cast<uintptr_t>(init) & 15) == 0) {
#pragma unroll
                for (int c = 0; c < VD; c += 4)
                    if (c < k.Vd) {
                        const float4 v = *reinterpret_cast<const float4*>(init + r * sr + c);
                        S[c] = v.x; S[c + 1] = v.y; S[c + 2] = v.z; S[c + 3] = v.w;
                    }
            } else if (init) {
#pragma unroll
                for (int c = 0; c < VD; ++c)
                    if (c < k.Vd) S[c] = init[r * sr + c * sc];
            }
        }
        auto put = [&](float* to, long long sr, long long sc) {
            if (have_row && sc == 1 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
#pragma unroll
                for (int c = 0; c < VD; c += 4)
                    if (c < k.Vd) *reinterpret_cast<float4*>(to + r * sr + c) = make_float4(S[c], S[c + 1], S[c + 2], S[c + 3]);
            } else if (have_row) {
#pragma unroll
                for (int c = 0; c < VD; ++c)
                    if (c < k.Vd) to[r * sr + c * sc] = S[c];
            }
        };
        auto keep = [&](int t0) {                                 // if the chunk at t0 ends a run
            if (k.anchors && ((t0 + kTc) % kAnchor == 0 || t0 + kTc >= a.T)) put(k.anchors + ((size_t)bh * a.runs + t0 / kAnchor) * k.Kd * k.Vd, k.Vd, 1);
        };
        // 16-byte piece c of 64-column block j of this thread's row
        auto piece = [&](uint32_t base, int rows, int j, int c) { return base + (uint32_t)j * rows * 128 + (uint32_t)r * 128 + (uint32_t)((c ^ (r & 7)) << 4); };
        auto sts = [&](uint32_t addr, uint4 v) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); };
        auto publish = [&] {                                      // the state's bf16 copy
            if (r < KD) {
#pragma unroll
                for (int c = 0; c < VD / 8; ++c) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float v0 = S[8 * c + 2 * i], v1 = S[8 * c + 2 * i + 1];
                        hi[i] = pack_bf16x2(v0, v1);
                        lo[i] = pack_bf16x2(v0 - __uint_as_float(hi[i] << 16), v1 - __uint_as_float(hi[i] & 0xffff0000u));
                    }
                    sts(piece(s_hi, KD, c / 8, c % 8), make_uint4(hi[0], hi[1], hi[2], hi[3]));
                    if (fine) sts(piece(s_lo, KD, c / 8, c % 8), make_uint4(lo[0], lo[1], lo[2], lo[3]));
                }
            }
            async_fence();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kS));
        };
        if constexpr (!STATE_ONLY) {
            if (rev)
                for (int t0 = t_lo + chunks * kTc; t0 < t_hi; t0 += kTc) keep(t0);
            if (chunks) publish();
        }
        for (int it = 0; it < chunks; ++it) {
            const int t0 = chunk_at(it), valid = min(kTc, len - t0);
            const uint32_t ph = it & 1;
            if (!STATE_ONLY && rev) keep(t0);
            if (!wait(bar(kTabFull), ph)) break;
            const float u = r < valid ? tab.u[r] : 0.f, whole = tab.whole;
            const uint32_t y = tile_at(it, 0);
            // y is free to change once (1) has read it
            if (!wait(full(slot_of(it, 0)), phase_of(it, 0)) || (!STATE_ONLY && !wait(bar(kSc), ph))) break;
#pragma unroll 4
            for (int c = 0; c < KD / 8; ++c) {
                const uint32_t at = piece(y, kTc, c / 8, c % 8);
                uint32_t q[4], hi[4], lo[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q[0]), "=r"(q[1]), "=r"(q[2]), "=r"(q[3]) : "r"(at) : "memory");
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // (a row behind the last token may hold anything: it becomes zero, not a product with zero)
                    const float v0 = r < valid ? u * __uint_as_float(q[i] << 16) : 0.f, v1 = r < valid ? u * __uint_as_float(q[i] & 0xffff0000u) : 0.f;
                    hi[i] = pack_bf16x2(v0, v1);
                    lo[i] = pack_bf16x2(v0 - __uint_as_float(hi[i] << 16), v1 - __uint_as_float(hi[i] & 0xffff0000u));
                }
                sts(at, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                sts(piece(y_lo, kTc, c / 8, c % 8), make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            if (valid < kTc) {                                    // z's rows there meet zeros in P and in u y
                if (!wait(full(slot_of(it, kTileZ)), phase_of(it, kTileZ))) break;
                if (r >= valid) {
                    const uint32_t z = tile_at(it, kTileZ);
#pragma unroll
                    for (int c = 0; c < VD / 8; ++c) sts(piece(z, kTc, c / 8, c % 8), make_uint4(0, 0, 0, 0));
                }
            }
            async_fence();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(kY));
                mbar_arrive(bar(kTabFree));
            }
            if (!wait(bar(kDelta), ph)) break;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < VD / 32; ++j) {
                float d[32];
                tmem_ld32(mine + 32 * j, d);
#pragma unroll
                for (int c = 0; c < 32; ++c) S[32 * j + c] = fmaf(S[32 * j + c], whole, d[c]);
            }
            tc_fence_before();
            if (!STATE_ONLY) {
                if (it + 1 < chunks) {
                    if (!wait(bar(kMma2), ph)) break;             // (2) has read the copy
                    publish();
                }
                if (!rev) keep(t0);
            }
        }
        if constexpr (STATE_ONLY) {
            put(k.seg_state + ((size_t)bh * a.nseg + seg) * k.Kd * k.Vd, k.Vd, 1);
        } else {
            if (!rev)
                for (int t0 = t_lo + chunks * kTc; t0 < t_hi; t0 += kTc) keep(t0);
            if (k.fin.p && seg == (rev ? 0 : a.nseg - 1)) {
                if (*abort) {
#pragma unroll
                    for (int c = 0; c < VD; ++c) S[c] = __int_as_float(0x7fc00000);
                }
                put(k.fin.p + b * k.fin.sb + h * k.fin.sh, k.fin.sr, k.fin.sc);
            }
        }
    } else if (warp == 8) {
        // ---- loads ----
        if (lane == 0) {
            const CUtensorMap* const m = maps.m[ci];
            int armed = 0;
            for (int i = 0; i < chunks * kTiles; ++i) {
                const int it = i / kTiles, tile = i % kTiles, s = i % L.slots;
                if (!mbar_wait(empty(s), ((uint32_t)(i / L.slots) & 1u) ^ 1u, abort)) break;
                const int t0 = chunk_at(it);
                const int which = tile == 0 ? 1 : tile == kTileZ ? 2 : 0;
                const int blocks = which == 2 ? VB : KB, head = h / (which == 0 ? k.x.per : which == 1 ? k.y.per : k.z.per);
                mbar_expect_tx(full(s), (uint32_t)blocks * kTcBlock);
                for (int j = 0; j < blocks; ++j) tma_load_4d(ring + (uint32_t)s * kTile + j * kTcBlock, m + which, 64 * j, head, t0, b, full(s));
                armed = i + 1;
            }
            if (*abort)
                for (int i = max(0, armed - L.slots); i < armed; ++i)
                    for (int n = 0; n < kTcWaitLimit && !mbar_try_wait(full(i % L.slots), (uint32_t)(i / L.slots) & 1u); ++n) {}
        }
    } else if (warp == 9) {
        // ---- products ----
        if (lane == 0) {
            constexpr uint32_t i1 = tc_idesc(128, false, false), i2 = tc_idesc(VD, false, true), i4 = tc_idesc(VD, true, true);
            for (int it = 0; it < chunks; ++it) {
                const uint32_t ph = it & 1;
                const uint32_t y = tile_at(it, 0), x = tile_at(it, kTileX), z = tile_at(it, kTileZ);
                if constexpr (!STATE_ONLY) {
                    if (it > 0 && !mbar_wait(bar(kO), ph ^ 1u, abort)) break;          // P has been read
                    if (!mbar_wait(full(slot_of(it, 0)), phase_of(it, 0), abort) || !mbar_wait(full(slot_of(it, kTileX)), phase_of(it, kTileX), abort)) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < KD / 16; ++kk) {
                        const uint32_t off = (uint32_t)(kk / 4) * kTcBlock + (kk % 4) * 32;
                        umma_bf16(tmem + kSc0, desc_k(x + off), desc_k(y + off), i1, kk > 0);
                    }
                    umma_commit(bar(kSc));
                }
                // (4)
                if (!mbar_wait(full(slot_of(it, kTileZ)), phase_of(it, kTileZ), abort) || !mbar_wait(bar(kY), ph, abort)) break;
                tc_fence_after();
#pragma unroll
                for (int part = 0; part < 2; ++part)
#pragma unroll
                    for (int kk = 0; kk < kTc / 16; ++kk)
                        umma_bf16(tmem + kDelta0, desc_mn((part ? y_lo : y) + kk * 2048, kTcBlock), desc_mn(z + kk * 2048, kTcBlock), i4, part > 0 || kk > 0);
                umma_commit(bar(kDelta));
                umma_commit(empty(slot_of(it, 0)));
                if constexpr (STATE_ONLY) {
                    umma_commit(empty(slot_of(it, kTileZ)));
                } else {
                    // (2)
                    if (!mbar_wait(bar(kS), ph, abort) || (it > 0 && !mbar_wait(bar(kOFree), ph ^ 1u, abort))) break;
                    tc_fence_after();
                    for (int part = 0; part < (fine ? 2 : 1); ++part)
#pragma unroll
                        for (int kk = 0; kk < KD / 16; ++kk)
                            umma_bf16(tmem + kO2, desc_k(x + (uint32_t)(kk / 4) * kTcBlock + (kk % 4) * 32), desc_mn((part ? s_lo : s_hi) + kk * 2048, KD * 128), i2, part > 0 || kk > 0);
                    umma_commit(bar(kMma2));
                    umma_commit(empty(slot_of(it, kTileX)));
                    // (3)
                    if (!mbar_wait(bar(kP), ph, abort)) break;
                    tc_fence_after();
                    for (int part = 0; part < (fine ? 2 : 1); ++part)
#pragma unroll
                        for (int kk = 0; kk < kTc / 16; ++kk)
                            umma_bf16_ts(tmem + kO1, tmem + kSc0 + part * 64 + kk * 8, desc_mn(z + kk * 2048, kTcBlock), i2, part > 0 || kk > 0);
                    umma_commit(bar(kO));
                    umma_commit(empty(slot_of(it, kTileZ)));
                }
            }
        }
    } else {
        // ---- decays: four tokens a lane ----
        const float* const g = a.g + (long long)b * a.gb + (long long)h * a.gh;
        double whole = 0.0;
        for (int it = 0; it < chunks; ++it) {
            const int t0 = chunk_at(it), valid = min(kTc, len - t0), j = lane >> 3;
            double d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] = 4 * lane + i < valid ? attn_decay(__ldg(g + (long long)(t0 + 4 * lane + i) * a.gt)) : 0.0;
#pragma unroll
            for (int i = 1; i < 4; ++i) d[i] += d[i - 1];
            double up = d[3];
#pragma unroll
            for (int s = 1; s < 8; s <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, up, s);
                if ((lane & 7) >= s) up += o;
            }
            const double before = up - d[3];
#pragma unroll
            for (int i = 0; i < 4; ++i) d[i] += before;
            double start[5];
            start[0] = 0.0;
#pragma unroll
            for (int i = 0; i < 4; ++i) start[i + 1] = start[i] + __shfl_sync(0xffffffffu, up, 8 * i + 7);
            whole += start[4];
            if (it > 0 && !wait(bar(kTabFree), (uint32_t)(it & 1) ^ 1u)) break;
            double mine = 0.0;
#pragma unroll
            for (int i = 1; i < 4; ++i) mine = j == i ? start[i] : mine;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 4 * lane + i;
                const float hi = (float)d[i];
                tab.l[t] = make_float2(hi, (float)(d[i] - hi));
                const double c = mine + d[i];
                tab.u[t] = k.s_update * ex2((float)(rev ? c : start[4] - c));
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (!rev && q > j) tab.f[tc_f(0, q) + t] = ex2((float)(start[q] - c));
                    if (rev && q < j) tab.f[tc_f(1, q) + t - 32 * (q + 1)] = ex2((float)(c - start[q + 1]));
                }
            }
            if ((lane & 7) == 7) {
                const double base = rev ? start[4] - mine : mine, total = d[3];
                tab.base[j] = make_float2((float)base, (float)(base - (double)(float)base));
                tab.total[j] = make_float2((float)total, (float)(total - (double)(float)total));
            }
            if (lane == 0) tab.whole = ex2((float)start[4]);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kTabFull));
        }
        if (STATE_ONLY && lane == 0) k.seg_decay[(size_t)bh * a.nseg + seg] = (float)whole;
    }

    __syncthreads();
    if constexpr (!STATE_ONLY) {
        // rows of chunks behind the sequence's last token: zero; rows that a given-up wait has left: NaN
        if (warp < 4) {
            const bool lost = *abort != 0;
            auto fill = [&](int from, int to, float v) {
                for (int t = from + tid; t < to; t += 128) {
                    const long long at = b * k.ob + (long long)t * k.ot + h * k.oh;
                    for (int c = 0; c < k.Vd; ++c) {
                        if (k.out_f32) static_cast<float*>(k.out)[at + c] = v;
                        else static_cast<__nv_bfloat16*>(k.out)[at + c] = __float2bfloat16_rn(v);
                    }
                    if (k.dots) k.dots[((size_t)b * a.T + t) * a.H + h] = v;
                }
            };
            if (t_lo + chunks * kTc < t_hi) fill(t_lo + chunks * kTc, t_hi, 0.f);
            if (lost)
                for (int it = 0; it < chunks; ++it) fill(chunk_at(it), min(t_hi, chunk_at(it) + kTc), __int_as_float(0x7fc00000));
        }
    }
    if (tid == 0 && abort_flag && L.host_flag) *reinterpret_cast<volatile int*>(L.host_flag) = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == 8) tmem_dealloc(tmem, kCols);
}

}  // namespace m2d
