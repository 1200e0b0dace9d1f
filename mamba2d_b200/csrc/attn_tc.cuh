// attn_core.cuh's computation on the 5th-generation tensor cores: bf16 tensors, head sizes up to 128.
//
// A chunk is 128 tokens, the rows of one accumulator.  Per chunk, with the tiles of x, y, z in shared memory (TMA, 128-byte
// swizzle, blocks of 128 rows x 64 columns) and St in bf16 next to them:
//     (1)  pairs = x y^T            128 x 128    both operands as they arrived
//     (2)  O     = x St             128 x VD
//     (3)  O    += P z              128 x VD     P, from pairs, as bf16 in tensor memory in the place of pairs
//     (4)  delta = (u y)^T z        KD x VD      u y scaled in place, in two bf16 parts: St is carried in fp32 and a state
//                                                is an output; one part would leave it at 2^-9
// A decay D_rc = exp(c_r - c_c) is a product of exp(c_r - m) and f_c = exp(m - c_c), m half of the chunk's decay: P is pairs times
// f, the copy of St is scaled by exp(m), and out = exp(c_r - m) O; all factors lie within 2^+-48 or the chunk is not `mild`
// (m would have to lie further from its ends than that: decays of more than 0.52 a token on average, a sequence that starts
// anew inside).  P of such a chunk takes its D from differences of c, and O of (2) is scaled by its rows where it lies
// before (3) adds.  What the factors take of the range of values is missing at its ends: with 2^+-80 values of 1e-17 lost bits and such of
// 1e16 became infinite.  (If no chunk were mild: 4x4096x16x128 135 us for 124, 1x65536x8 194 for 178.)  c is summed in 64 bits.
// Rounded to bf16 on the way are P and St's copy, once each, of which one lies on a term's way: an output, itself rounded to bf16 after
// that, is off by 2.3e-3 where its own rounding alone would leave 1.7e-3.  q, k and v come with as large a rounding.  u y has two
// parts (16 bits; what a state is off by, 2.5e-6, is theirs): a third would be half as many products (4) again, on the longest chain, and take
// a tile of the ring.
// The work is dealt to warps that wait on one another through mbarriers only:
//     warps 0 - 7    a token row and half of the columns a thread: pairs -> P, O -> out
//     warps 8 - 15   half of a token row a thread: y -> u y; half of a row of St a thread: St in registers, its bf16 copy
//     warp 16  TMA loads    warps 17, 18  issue (1), (4) and (2), (3)     warp 19  the decays' tables
// pairs has two places, so that (1) of the next chunk runs beside (3) of this one.  The copy of St is written while (4) runs, after
// u y: what bounds a chunk is the chain u y -> (4) -> St.  out goes through shared memory and by TMA: rows stored from registers
// took 2000 cycles of a chunk, 32 lines a request.  It has a tile of its own where there is room (a head size of 64), else that of x,
// which nothing reads any more, but whose next load then waits for it.
//
// Measured, forward at 8x2048x16x128: 84 us for 128 CTAs of 16 chunks, 10000 cycles a chunk: the tensor cores are busy for 29 % of them,
// the schedulers issue in 26 %, and what most warps wait for, besides each other, is instructions (1.9 of the 6 cycles between
// two instructions of a warp).  The bytes would take 34 us.  At 96 registers a thread full passes spill 24 to 40 bytes (92 to 156 bytes of
// loads); a pass over states 8 at most.
//
// Every wait is bounded: one that gives up makes all of the CTA's roles leave, its rows become NaN (or, where it computes a segment's
// state, that does, and with it the rows that come of it), and a word in host memory says so.
#pragma once

#include "attn_core.cuh"
#include "tc_ptx.cuh"

namespace m2d {

constexpr int kTc = 128;                      // tokens of a chunk
constexpr int kTcThreads = 640;
constexpr int kTcBlock = kTc * 128;           // 128 rows x 64 columns of bf16
constexpr int kTcTiles = 3;                   // tiles of x, y, z each in flight, at most
constexpr float kTcMild = 48.f;

struct TcMaps { CUtensorMap m[3][4]; };       // [core][x, y, z, out]
struct TcLaunch {
    AttnLaunch a;
    int cores;
    int* host_flag;
    int give_up;                // test hook: the first CTA's, of a launch over states
};

// ---- PTX ---------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2, int c3) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2), "r"(c3) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// The issuing warps run as a whole and one lane's predicate is on: operands then stay in uniform registers, where the
// instruction wants them.  (One lane alone in a branch moved them there for every product, 160 cycles a product instead of its 64.)
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on;
}
// A descriptor's lower half (address and distance of blocks) in a uniform register, where a reduction over the warp leaves it; its
// upper half is a constant.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t next) { return uniform(((addr & 0x3ffffu) >> 4) | ((next >> 4) << 16)); }
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
template <uint32_t IDESC, bool ACCUMULATE>
__device__ __forceinline__ void umma_ss(uint32_t on, uint32_t tmem_d, uint32_t a, uint32_t b) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t.reg .b32 i;\n\tsetp.ne.b32 q, %3, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 da, {%1, %4};\n\tmov.b64 db, {%2, %4};\n\tmov.b32 i, %5;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, i, p;\n\t}"
        ::"r"(tmem_d), "r"(a), "r"(b), "r"(on), "n"(kDescHi), "n"(IDESC), "n"(ACCUMULATE ? 1 : 0) : "memory");
}
template <uint32_t IDESC, bool ACCUMULATE>
__device__ __forceinline__ void umma_ts(uint32_t on, uint32_t tmem_d, uint32_t tmem_a, uint32_t b) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t.reg .b32 i;\n\tsetp.ne.b32 q, %3, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 db, {%2, %4};\n\tmov.b32 i, %5;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, i, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "r"(b), "r"(on), "n"(kDescHi), "n"(IDESC), "n"(ACCUMULATE ? 1 : 0) : "memory");
}
// `n` products, one for each 16 of the contraction: a and b of the k-th; the first one starts the accumulator unless GO_ON
template <uint32_t IDESC, bool GO_ON, int N, typename FA, typename FB>
__device__ __forceinline__ void umma_chain(uint32_t on, uint32_t tmem_d, FA fa, FB fb) {
    if constexpr (GO_ON) umma_ss<IDESC, true>(on, tmem_d, fa(0), fb(0));
    else umma_ss<IDESC, false>(on, tmem_d, fa(0), fb(0));
#pragma unroll
    for (int k = 1; k < N; ++k) umma_ss<IDESC, true>(on, tmem_d, fa(k), fb(k));
}
__device__ __forceinline__ void commit_if(uint32_t on, uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(on) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                   "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr) : "memory");
}
// 16 columns of this thread's row
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Operand descriptors of the 128-byte-swizzle layout are wgrad_tc.cuh's; an operand is contracted along its 128-byte rows
// ("K-major"), or across them ("MN-major", `next` bytes to the next 64 columns).
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// Decay tables of a chunk.
struct alignas(16) TcTable {
    float f[kTc];           // mild: exp(m - c), times s_intra / s_inter; else c in log2
    float e[kTc];           // mild: exp(c - m), times s_inter; else what c lost to its rounding
    float u[kTc];           // update weight times s_update
    float2 end;             // c_end in log2, in two floats
    float whole, copy;      // exp(c_end); mild: exp(m), else one
    int mild;
};
struct alignas(16) TcSmall {
    TcTable tab;
    uint64_t bars[40];
    uint32_t tmem;
    int abort;
};

// What a launch is for.  kTcPlain: bf16 out and nothing else, the least code (20 warps in five roles miss the instruction caches
// often: with the branches of the others it takes 104 us where it takes 85).  kTcHeads: out in fp32, head by head.
enum TcMode { kTcPlain, kTcHeads, kTcStateOnly };

// Shared memory: St in bf16, the second part of u y, tiles, out's tile.  (KD = 64: (4) computes 128 rows; the upper
// 64, of whatever lies behind y, are not used, and a tile lies there.)  Tiles of x, y, z: x first, whose tile is held longest, z
// last, which is needed last; out's own tile before third ones.
struct TcLayout {
    int n[3] = {1, 1, 1};                     // tiles of x, y, z in flight
    bool own_stage = false;                   // out has a tile of its own, else it goes through x's
    uint32_t y_lo = 0, ring[3] = {}, stage = 0, small = 0;
    __host__ __device__ constexpr TcLayout(int KD, int VD, TcMode mode) {
        const bool state_only = mode == kTcStateOnly;
        const uint32_t tile[3] = {(uint32_t)kTc * KD * 2, (uint32_t)kTc * KD * 2, (uint32_t)kTc * VD * 2};
        if (state_only) n[0] = 0;
        y_lo = state_only ? 0 : KD * VD * 2;
        uint32_t bytes = y_lo + (state_only ? 2 : 1) * tile[0] + n[0] * tile[0] + tile[1] + tile[2];
        const uint32_t most = (uint32_t)(kMaxSmem - sizeof(TcSmall));
        for (int round = 1; round < kTcTiles; ++round) {
            if (round == 2 && !state_only && (KD < VD || bytes + tile[2] <= most)) {
                own_stage = true;
                bytes += tile[2];
            }
            for (int i = state_only ? 1 : 0; i < 3; ++i)
                if (n[i] == round && bytes + tile[i] <= most) {
                    ++n[i];
                    bytes += tile[i];
                }
        }
        ring[0] = y_lo + (state_only ? 2 : 1) * tile[0];
        ring[1] = ring[0] + n[0] * tile[0];
        ring[2] = ring[1] + n[1] * tile[1];
        stage = ring[2] + n[2] * tile[2];
        small = bytes;
    }
};

template <int KD, int VD, TcMode MODE>
__global__ void __launch_bounds__(kTcThreads, 1) attn_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcLaunch L) {
    extern __shared__ __align__(1024) uint8_t tc_smem_raw[];
    // (kSc, kY, kO, kDelta: one for even chunks, one for odd, where a barrier may complete again before all have seen it)
    enum { kSc, kP = kSc + 2, kY, kO = kY + 2, kOFree = kO + 2, kDelta, kS = kDelta + 2, kMma2, kTabFull, kTabFree, kFull, kEmpty = kFull + 3 * kTcTiles, kBars = kEmpty + 3 * kTcTiles };
    static_assert(kBars <= 40, "room for the barriers");
    constexpr bool STATE_ONLY = MODE == kTcStateOnly;
    constexpr TcLayout lay(KD, VD, MODE);
    constexpr int kHalf = VD / 2;                                 // columns of a thread
    constexpr uint32_t kTileX = kTc * KD * 2, kTileZ = kTc * VD * 2;
    constexpr uint32_t kO0 = 256;                                 // columns of tensor memory: pairs (2 x 128), O, delta
    constexpr uint32_t kCols = STATE_ONLY ? 2 * VD : 512;           // (two places for delta where states are all that is wanted)
    constexpr uint32_t kDelta0 = STATE_ONLY ? 0 : kO0 + VD;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // (a launch that needs nothing of this one may fill its last wave)
    const AttnLaunch& a = L.a;
    const int ci = blockIdx.x % L.cores, unit = blockIdx.x / L.cores;
    const AttnCore& k = a.core[ci];
    constexpr bool f32_out = MODE == kTcHeads;
    const int states = a.join_here ? (a.nseg - 1) * a.parts : a.nseg, units = STATE_ONLY ? states : a.nseg;
    const int seg = unit % units, bh = unit / units, h = bh % a.H, b = bh / a.H;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, rev = k.rev;
    const int len = attn_length(a, b);
    unsigned lo = seg * a.seg_len, hi = lo + a.seg_len;              // (may lie beyond 2^31)
    if (STATE_ONLY && a.join_here) {
        const unsigned from = (seg / a.parts + rev) * a.seg_len;
        lo = from + seg % a.parts * a.part_len;
        hi = min(from + a.seg_len, lo + a.part_len);
    }
    const int t_lo = STATE_ONLY ? (int)min(lo, (unsigned)a.T) : (int)lo, t_hi = (int)min(hi, (unsigned)a.T);
    const int active = max(0, min(len, t_hi) - t_lo), chunks = (active + kTc - 1) / kTc;         // the others hold nothing

    TcSmall& small = *reinterpret_cast<TcSmall*>(tc_smem_raw + lay.small);
    TcTable& tab = small.tab;
    const uint32_t smem0 = smem_u32(tc_smem_raw), s_hi = smem0, y_lo = smem0 + lay.y_lo;
    const uint32_t bar0 = smem_u32(small.bars);
    auto bar = [&](int i) { return bar0 + 8u * i; };
    enum { X, Y, Z };
    // (`which` is a constant wherever these are inlined; X has no tiles in a pass over states only)
    auto tiles_of = [&](int which) { return which == X ? (lay.n[X] ? lay.n[X] : 1) : which == Y ? lay.n[Y] : lay.n[Z]; };
    auto tile_at = [&](int which, int it) { return smem0 + lay.ring[which] + (uint32_t)(it % tiles_of(which)) * (which == Z ? kTileZ : kTileX); };
    auto full = [&](int which, int it) { return bar(kFull + which * kTcTiles + it % tiles_of(which)); };
    auto empty = [&](int which, int it) { return bar(kEmpty + which * kTcTiles + it % tiles_of(which)); };
    auto turn = [&](int which, int it) { return (uint32_t)(it / tiles_of(which)) & 1u; };
    auto chunk_at = [&](int it) { return t_lo + (rev ? chunks - 1 - it : it) * kTc; };
    volatile int* const abort = &small.abort;
    auto wait = [&](uint32_t bar_, uint32_t parity) {            // whole warps
        if (__builtin_expect(__all_sync(0xffffffffu, mbar_try_wait(bar_, parity)), 1)) return true;
        return __all_sync(0xffffffffu, mbar_wait(bar_, parity, abort)) != 0;
    };
    auto wait2 = [&](int bar_, int it) { return wait(bar(bar_ + (it & 1)), it >> 1 & 1); };                                          // of a pair
    auto loaded = [&](int which, int it) { return wait(full(which, it), turn(which, it)); };

    if (tid == 0) {
        for (int i = 0; i < kFull; ++i) mbar_init(bar(i), i == kP || i == kY || i == kY + 1 || i == kOFree || i == kS || (STATE_ONLY && (i == kO || i == kO + 1)) ? 8 : i == kTabFree ? 16 : 1);
        for (int i = kFull; i < kEmpty; ++i) mbar_init(bar(i), 1);
        // who gives a tile back: its two products, (1) and (4) counted as one; x's where out goes through it, whoever stores that
        for (int i = 0; i < 3 * kTcTiles; ++i) mbar_init(bar(kEmpty + i), STATE_ONLY || i / kTcTiles == Y || (i / kTcTiles == X && !lay.own_stage) ? 1 : 2);
        small.abort = (smem_u32(tc_smem_raw) & 1023u) != 0 || (STATE_ONLY && L.give_up && blockIdx.x == 0);      // (swizzled tiles have to be aligned; nothing runs if they are not)
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 16) tmem_alloc(smem_u32(&small.tmem), kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = small.tmem;

    // 16-byte piece c of a tile's row (64-column blocks of `rows` rows, swizzled)
    auto piece = [&](uint32_t base, int rows, int r, int c) { return base + (uint32_t)(c / 8) * rows * 128 + (uint32_t)r * 128 + (uint32_t)(((c ^ r) & 7) << 4); };
    auto sts = [&](uint32_t addr, uint32_t v0, uint32_t v1, uint32_t v2, uint32_t v3) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v0), "r"(v1), "r"(v2), "r"(v3) : "memory"); };

    // y -> u y, half of row r a thread; false if a wait has given up
    auto scale_y = [&](int it, int valid, int r, int half, float u) {
        const uint32_t y = tile_at(Y, it);
        // y is free to change once (1) has read it; its second part has two places where states are all that is wanted
        if (!loaded(Y, it) || (!STATE_ONLY && !wait2(kSc, it)) || (STATE_ONLY && it > 1 && !wait2(kDelta, it - 2))) return false;
#pragma unroll 2
        for (int i = 0; i < KD / 16; ++i) {
            const int c = half * (KD / 16) + i;
            const uint32_t at = piece(y, kTc, r, c);
            uint32_t g[4], hi[4], lo[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(g[0]), "=r"(g[1]), "=r"(g[2]), "=r"(g[3]) : "r"(at) : "memory");
            if (__builtin_expect(valid < kTc, 0) && r >= valid) g[0] = g[1] = g[2] = g[3] = 0;      // (such a row may hold anything: no product with zero)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 v = __fmul2_rn(make_float2(__uint_as_float(g[i] << 16), __uint_as_float(g[i] & 0xffff0000u)), make_float2(u, u));
                hi[i] = pack_bf16x2(v.x, v.y);
                const float2 rest = __ffma2_rn(make_float2(__uint_as_float(hi[i] << 16), __uint_as_float(hi[i] & 0xffff0000u)), make_float2(-1.f, -1.f), v);
                lo[i] = pack_bf16x2(rest.x, rest.y);
            }
            sts(at, hi[0], hi[1], hi[2], hi[3]);
            sts(piece(y_lo + (STATE_ONLY ? (it & 1) * kTileX : 0), kTc, r, c), lo[0], lo[1], lo[2], lo[3]);
        }
        if (__builtin_expect(valid < kTc, 0)) {               // z's rows there meet zeros in P and in u y
            if (!loaded(Z, it)) return false;
            if (r >= valid) {
#pragma unroll 1
                for (int c = 0; c < VD / 16; ++c) sts(piece(tile_at(Z, it), kTc, r, half * (VD / 16) + c), 0, 0, 0, 0);
            }
        }
        async_fence();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kY + (it & 1)));
        return true;
    };

    if (warp < 8) {
        // ---- token rows ----
        if constexpr (STATE_ONLY) {                               // (they scale y, so that warps 8 - 15 only add what comes of it)
            for (int it = 0; it < chunks; ++it) {
                const int r = tid & 127, valid = min(kTc, len - chunk_at(it));
                if (!wait(bar(kTabFull), it & 1)) break;
                const float u = r < valid ? tab.u[r] : 0.f;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kTabFree));
                if (!scale_y(it, valid, r, warp >> 2, u)) break;
            }
        }
        if constexpr (!STATE_ONLY) {
            const int q = warp & 3, half = warp >> 2, r = tid & 127;
            const uint32_t mine = tmem + ((uint32_t)(q * 32) << 16), oc = mine + kO0 + half * kHalf;
            for (int it = 0; it < chunks; ++it) {
                // pairs -> P
                const int t0 = chunk_at(it), valid = min(kTc, len - t0);
                const uint32_t pairs = mine + 128 * (it & 1);
                if (!wait(bar(kTabFull), it & 1)) break;
                const bool mild = tab.mild;
                float e = tab.e[r];
                if (!wait2(kSc, it)) break;
                tc_fence_after();
                // blocks of 32 columns: 0 and 3, or 1 and 2, so that no warp has more than two that are not masked
#pragma unroll 1
                for (int i = 0; i < 2; ++i) {
                    const int j = half ? 1 + i : 3 * i;
                    const uint32_t at = pairs + 32 * j;
                    const bool off = rev ? j < q : j > q;
                    float v[32];
                    if (off) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) v[c] = 0.f;
                    } else {
                        tmem_ld32(at, v);
                        const float4* const f = reinterpret_cast<const float4*>(tab.f + 32 * j);
                        if (__builtin_expect(mild, 1)) {
#pragma unroll
                            for (int c = 0; c < 32; c += 4) {
                                const float4 g = f[c / 4];
                                const float2 v0 = __fmul2_rn(make_float2(v[c], v[c + 1]), make_float2(g.x, g.y)), v1 = __fmul2_rn(make_float2(v[c + 2], v[c + 3]), make_float2(g.z, g.w));
                                v[c] = v0.x; v[c + 1] = v0.y; v[c + 2] = v1.x; v[c + 3] = v1.y;
                            }
                        } else {
                            const float cr = tab.f[r], ratio = rev ? k.s_intra : 1.f, sign = rev ? -1.f : 1.f;
#pragma unroll
                            for (int c = 0; c < 32; ++c) v[c] *= ratio * ex2(sign * ((cr - tab.f[32 * j + c]) + (e - tab.e[32 * j + c])));
                        }
                        unsigned on = 0xffffffffu;
                        if (j == q) on = rev ? 0xffffffffu << lane : 0xffffffffu >> (31 - lane);
                        if (valid < 32 * j + 32) on &= valid <= 32 * j ? 0u : 0xffffffffu >> (32 * j + 32 - valid);
                        if (__any_sync(0xffffffffu, on != 0xffffffffu)) {
#pragma unroll
                            for (int c = 0; c < 32; ++c) v[c] = on >> c & 1 ? v[c] : 0.f;
                        }
                    }
                    uint32_t p[16];
#pragma unroll
                    for (int c = 0; c < 16; ++c) p[c] = pack_bf16x2(v[2 * c], v[2 * c + 1]);
                    tmem_st16(at, p);
                }
                if (__builtin_expect(!mild, 0)) {                 // O2 -> w O2
                    const float c = tab.f[r], w = rev ? ex2((tab.end.x - c) + (tab.end.y - e)) : ex2(c + e);
                    e = k.s_inter;
                    if (!wait(bar(kMma2), it & 1)) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < kHalf; c0 += 16) {
                        float v[16];
                        uint32_t p[16];
                        tmem_ld16(oc + c0, v);
#pragma unroll
                        for (int c = 0; c < 16; ++c) p[c] = __float_as_uint(w * v[c]);
                        tmem_st16(oc + c0, p);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(bar(kP));
                    mbar_arrive(bar(kTabFree));
                }
                // O -> out
                const bool row = t0 + r < t_hi, live = r < valid;
                const uint32_t stage = lay.own_stage ? smem0 + lay.stage : tile_at(X, it);
                if (!wait2(kO, it)) break;
                tc_fence_after();
#pragma unroll 1
                for (int c0 = 0; c0 < kHalf; c0 += 32) {
                    float o[32];
                    const int col = half * kHalf + c0;
                    tmem_ld32(oc + c0, o);
#pragma unroll
                    for (int c = 0; c < 32; ++c) o[c] *= e;
                    if (__builtin_expect(valid < kTc, 0)) {
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = live ? o[c] : 0.f;
                    }
                    if (!f32_out) {
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            sts(piece(stage, kTc, r, (col + c) / 8), pack_bf16x2(o[c], o[c + 1]), pack_bf16x2(o[c + 2], o[c + 3]), pack_bf16x2(o[c + 4], o[c + 5]), pack_bf16x2(o[c + 6], o[c + 7]));
                    } else if (row) {
                        float4* const p = reinterpret_cast<float4*>(static_cast<float*>(k.out) + b * k.ob + (long long)(t0 + r) * k.ot + h * k.oh + col);
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            if (col + c < k.Vd) {
                                p[c / 4] = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                                p[c / 4 + 1] = make_float4(o[c + 4], o[c + 5], o[c + 6], o[c + 7]);
                            }
                    }
                }
                tc_fence_before();
                async_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kOFree));
            }
        }
    } else if (warp < 16) {
        // ---- y and the state ----
        const int r = tid & 127, half = (warp >> 2) & 1, v0 = half * kHalf;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kDelta0 + v0;
        float S[kHalf];
        const bool have_row = r < k.Kd;
#pragma unroll
        for (int c = 0; c < kHalf; ++c) S[c] = 0.f;
        if (!STATE_ONLY && have_row) {
            const float* init = nullptr;
            long long sr = k.init.sr, sc = k.init.sc;
            if (a.nseg > 1 && !a.join_here) {
                init = k.seg_state + ((size_t)bh * a.nseg + seg) * k.Kd * k.Vd;
                sr = 1; sc = k.Kd;
            } else if (k.init.p) {
                init = k.init.p + b * k.init.sb + h * k.init.sh;
            }
            if (init) {
                init += r * sr + v0 * sc;
#pragma unroll
                for (int c = 0; c < kHalf; ++c)
                    if (v0 + c < k.Vd) S[c] = init[c * sc];
            }
        }
        // a few segments: each joins the states of those before it itself, a launch less
        if (!STATE_ONLY && a.join_here && have_row)
            for (int j = rev ? states - 1 : 0; rev ? j >= seg * a.parts : j < seg * a.parts; j += rev ? -1 : 1) {
                const size_t at = (size_t)bh * states + j;
                const float decay = ex2(k.seg_decay[at]);
                const float* own = k.seg_state + at * k.Kd * k.Vd + r + (size_t)v0 * k.Kd;
#pragma unroll
                for (int c = 0; c < kHalf; ++c) {
                    if (v0 + c < k.Vd) S[c] = fmaf(S[c], decay, *own);
                    own += k.Kd;
                }
            }
        // (states kept between kernels and runs have a column's rows next to one another: a warp's store is one line, not 32, which
        // held the other warps' shared memory up for 7000 cycles every four chunks)
        auto put = [&](float* to, long long sr, long long sc) {
            to += r * sr + v0 * sc;
            if (have_row && sc == 1 && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
#pragma unroll
                for (int c = 0; c < kHalf; c += 4)
                    if (v0 + c < k.Vd) *reinterpret_cast<float4*>(to + c) = make_float4(S[c], S[c + 1], S[c + 2], S[c + 3]);
            } else if (have_row) {
#pragma unroll
                for (int c = 0; c < kHalf; ++c) {
                    if (v0 + c < k.Vd) *to = S[c];
                    to += sc;
                }
            }
        };
        for (int it = 0; it < chunks; ++it) {
            const int t0 = chunk_at(it), valid = min(kTc, len - t0);
            if (!wait(bar(kTabFull), it & 1)) break;
            const float u = !STATE_ONLY && r < valid ? tab.u[r] : 0.f, whole = tab.whole, copy = tab.copy;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kTabFree));
            if constexpr (!STATE_ONLY) {
                if (!scale_y(it, valid, r, half, u)) break;
            }
            if constexpr (!STATE_ONLY) {                          // the state's copy for (2)
                if (it > 0 && !wait(bar(kMma2), (it & 1) ^ 1)) break;
                if (r < KD) {
#pragma unroll
                    for (int c = 0; c < kHalf / 8; ++c) {
                        uint32_t hi[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) hi[i] = pack_bf16x2(copy * S[8 * c + 2 * i], copy * S[8 * c + 2 * i + 1]);
                        sts(piece(s_hi, KD, r, v0 / 8 + c), hi[0], hi[1], hi[2], hi[3]);
                    }
                }
                async_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kS));
            }
            if (!wait2(kDelta, it)) break;
            tc_fence_after();
#pragma unroll
            for (int c0 = 0; c0 < kHalf; c0 += 16) {
                float d[16];
                tmem_ld16(mine + (STATE_ONLY ? (it & 1) * VD : 0) + c0, d);
#pragma unroll
                for (int c = 0; c < 16; ++c) S[c0 + c] = fmaf(S[c0 + c], whole, d[c]);
            }
            tc_fence_before();
            if (STATE_ONLY) {
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(kO + (it & 1)));
            }
        }
        // a warp that has left its chunks early has seen (or made) the abort: what it has is no state
        auto void_it = [&] {
            if (*abort) {
#pragma unroll
                for (int c = 0; c < kHalf; ++c) S[c] = __int_as_float(0x7fc00000);
            }
        };
        if constexpr (STATE_ONLY) {
            void_it();
            put(k.seg_state + ((size_t)bh * states + seg) * k.Kd * k.Vd, 1, k.Kd);
        } else {
            if (k.fin.p && seg == (rev ? 0 : a.nseg - 1)) {
                void_it();
                put(k.fin.p + b * k.fin.sb + h * k.fin.sh, k.fin.sr, k.fin.sc);
            }
        }
    } else if (warp == 16) {
        // ---- loads ----
        if (lane == 0) {
            int armed[3] = {0, 0, 0};
            for (int it = 0; it < chunks && !*abort; ++it) {
                const int t0 = chunk_at(it);
                auto load = [&](int which, int per) {
                    if (!mbar_wait(empty(which, it), turn(which, it) ^ 1u, abort)) return;
                    const int blocks = (which == Z ? VD : KD) / 64;
                    mbar_expect_tx(full(which, it), (uint32_t)blocks * kTcBlock);
                    for (int j = 0; j < blocks; ++j) tma_load_4d(tile_at(which, it) + j * kTcBlock, &maps.m[ci][which], 64 * j, h / per, t0, b, full(which, it));
                    armed[which] = it + 1;
                };
                load(Y, k.y.per);                                 // (its tile comes free first)
                if (!STATE_ONLY) load(X, k.x.per);
                load(Z, k.z.per);
            }
            if (*abort)                                           // let the copies land (bounded)
                for (int which = STATE_ONLY ? Y : X; which <= Z; ++which)
                    for (int it = max(0, armed[which] - tiles_of(which)); it < armed[which]; ++it)
                        for (int n = 0; n < kTcWaitLimit && !mbar_try_wait(full(which, it), turn(which, it)); ++n) {}
        }
    } else if (warp == 17) {
        // ---- products (1) and (4) ----
        constexpr uint32_t i1 = tc_idesc(128, false, false), i4 = tc_idesc(VD, true, true);
        const uint32_t on = elect_one(), tm = uniform(tmem);
        const int count = __reduce_max_sync(0xffffffffu, chunks);
        for (int it = -1; it < count; ++it) {
            if (it >= 0) {
                if (!wait(full(Y, it), turn(Y, it)) || !wait(full(Z, it), turn(Z, it)) || !wait2(kY, it)) break;
                tc_fence_after();
                if (STATE_ONLY && it > 1 && !wait2(kO, it - 2)) break;      // delta of two chunks ago has been read
                const uint32_t y = desc_lo(tile_at(Y, it), kTcBlock), yl = desc_lo(y_lo + (STATE_ONLY ? (it & 1) * kTileX : 0), kTcBlock), z = desc_lo(tile_at(Z, it), kTcBlock);
                const uint32_t delta = uniform(tm + kDelta0 + (STATE_ONLY ? (it & 1) * VD : 0));
                umma_chain<i4, false, kTc / 16>(on, delta, [&](int k) { return y + k * 128; }, [&](int k) { return z + k * 128; });
                commit_if(on, empty(Y, it));
                umma_chain<i4, true, kTc / 16>(on, delta, [&](int k) { return yl + k * 128; }, [&](int k) { return z + k * 128; });
                commit_if(on, bar(kDelta + (it & 1)));
                commit_if(on, empty(Z, it));
            }
            const int n = it + 1;
            if (!STATE_ONLY && n < count) {
                if (n > 1 && !wait2(kO, n - 2)) break;            // P of two chunks ago has been read
                if (!wait(full(X, n), turn(X, n)) || !wait(full(Y, n), turn(Y, n))) break;
                tc_fence_after();
                const uint32_t x = desc_lo(tile_at(X, n), 16), y = desc_lo(tile_at(Y, n), 16);
                umma_chain<i1, false, KD / 16>(on, tm + 128 * (n & 1), [&](int k) { return x + (((k / 4) * kTcBlock + (k % 4) * 32) >> 4); },
                                               [&](int k) { return y + (((k / 4) * kTcBlock + (k % 4) * 32) >> 4); });
                commit_if(on, bar(kSc + (n & 1)));
                if (lay.own_stage) commit_if(on, empty(X, n));
            }
        }
    } else if (warp == 18) {
        // ---- products (2) and (3), and what becomes of out ----
        if constexpr (!STATE_ONLY) {
            constexpr uint32_t i2 = tc_idesc(VD, false, true);
            const uint32_t on = elect_one(), tm = uniform(tmem);
            const int count = __reduce_max_sync(0xffffffffu, chunks);
            // chunk n's rows are in their tile (or have been stored from registers)
            auto store = [&](int n) {
                if (on) {
                    if (!f32_out) {
                        for (int j = 0; 64 * j < k.Vd; ++j) tma_store_4d(&maps.m[ci][3], (lay.own_stage ? smem0 + lay.stage : tile_at(X, n)) + j * kTcBlock, 64 * j, h, chunk_at(n), b);
                        bulk_commit();
                        bulk_wait_read();
                    }
                    if (!lay.own_stage) mbar_arrive(empty(X, n));
                }
                __syncwarp();
            };
            int it = 0;
            for (; it < count; ++it) {
                const uint32_t ph = it & 1;
                if (it > 0) {
                    if (!wait(bar(kOFree), ph ^ 1u)) break;
                    store(it - 1);
                }
                if (!wait(full(X, it), turn(X, it)) || !wait(bar(kS), ph)) break;
                tc_fence_after();
                const uint32_t x = desc_lo(tile_at(X, it), 16), sh = desc_lo(s_hi, KD * 128);
                auto xk = [&](int k) { return x + (((k / 4) * kTcBlock + (k % 4) * 32) >> 4); };
                umma_chain<i2, false, KD / 16>(on, tm + kO0, xk, [&](int k) { return sh + k * 128; });
                commit_if(on, bar(kMma2));
                if (lay.own_stage) commit_if(on, empty(X, it));
                if (!wait(full(Z, it), turn(Z, it)) || !wait(bar(kP), ph)) break;
                if (len - chunk_at(it) < kTc && !wait2(kY, it)) break;          // z's last rows have been cleared
                tc_fence_after();
                const uint32_t z = desc_lo(tile_at(Z, it), kTcBlock), p = uniform(tm + 128 * ph);       // (a block of 32 columns is in its first 16)
#pragma unroll
                for (int k = 0; k < kTc / 16; ++k) umma_ts<i2, true>(on, tm + kO0, p + (k / 2) * 32 + (k % 2) * 8, z + k * 128);
                commit_if(on, bar(kO + (it & 1)));
                commit_if(on, empty(Z, it));
            }
            if (it == count && count && wait(bar(kOFree), (count & 1) ^ 1u)) store(count - 1);
            if (on) bulk_wait();
            __syncwarp();
        }
    } else {
        // ---- decays: four tokens a lane ----
        const float* const g = a.g + (long long)b * a.gb + (long long)h * a.gh;
        double whole = 0.0;
        const float ratio = rev ? k.s_intra : 1.f;                // s_intra / s_inter
        float next[4];                                            // the next chunk's decays, on their way
        auto fetch = [&](int it) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = it < chunks ? chunk_at(it) + 4 * lane + i : len;
                next[i] = t < len ? __ldg(g + (long long)t * a.gt) : 0.f;
            }
        };
        fetch(0);
        for (int it = 0; it < chunks; ++it) {
            double c[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = attn_decay(next[i]);
            fetch(it + 1);
#pragma unroll
            for (int i = 1; i < 4; ++i) c[i] += c[i - 1];
            double up = c[3];
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const double o = __shfl_up_sync(0xffffffffu, up, s);
                if (lane >= s) up += o;
            }
            const double before = up - c[3], end = __shfl_sync(0xffffffffu, up, 31), m = 0.5 * end;
            bool near = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[i] += before;
                near = near && fabsf((float)(c[i] - m)) <= kTcMild;       // (not where it is NaN)
            }
            const bool mild = __all_sync(0xffffffffu, near && fabsf((float)m) <= kTcMild);
            whole += end;
            if (it > 0 && !wait(bar(kTabFree), (uint32_t)(it & 1) ^ 1u)) break;
            float f[4], e[4], u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float hi = (float)c[i], from_m = (float)(rev ? m - c[i] : c[i] - m);      // backwards m - c takes the place of c - m
                f[i] = mild ? ratio * ex2(-from_m) : hi;
                e[i] = mild ? k.s_inter * ex2(from_m) : (float)(c[i] - hi);
                u[i] = k.s_update * ex2((float)(rev ? c[i] : end - c[i]));
            }
            reinterpret_cast<float4*>(tab.f)[lane] = make_float4(f[0], f[1], f[2], f[3]);
            reinterpret_cast<float4*>(tab.e)[lane] = make_float4(e[0], e[1], e[2], e[3]);
            reinterpret_cast<float4*>(tab.u)[lane] = make_float4(u[0], u[1], u[2], u[3]);
            if (lane == 0) {
                tab.whole = ex2((float)end);
                tab.copy = mild ? ex2((float)m) : 1.f;
                tab.end = make_float2((float)end, (float)(end - (double)(float)end));
                tab.mild = mild;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kTabFull));
        }
        if (STATE_ONLY && lane == 0) k.seg_decay[(size_t)bh * states + seg] = (float)whole;
    }

    __syncthreads();
    if constexpr (!STATE_ONLY) {
        // rows of chunks behind the sequence's last token: zero; where a wait has given up: NaN
        if (warp < 8) {
            auto fill = [&](int from, int to, float v) {
                for (int t = from + warp; t < to; t += 8) {
                    const long long at = b * k.ob + (long long)t * k.ot + h * k.oh;
                    for (int c = lane; c < k.Vd; c += 32) {
                        if (f32_out) static_cast<float*>(k.out)[at + c] = v;
                        else static_cast<__nv_bfloat16*>(k.out)[at + c] = __float2bfloat16_rn(v);
                    }
                }
            };
            if (t_lo + chunks * kTc < t_hi) fill(t_lo + chunks * kTc, t_hi, 0.f);
            if (*abort) fill(t_lo, min(t_hi, t_lo + chunks * kTc), __int_as_float(0x7fc00000));
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");                   // (but does not end before it)
    if (tid == 0 && *abort && L.host_flag) *reinterpret_cast<volatile int*>(L.host_flag) = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == 16) tmem_dealloc(tmem, kCols);
}

}  // namespace m2d
