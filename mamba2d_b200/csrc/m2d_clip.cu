// The global norm of many tensors, and clipping by it: two launches for up to kClipTensors tensors.
//
// The table of tensors travels in the kernels' parameters, so that nothing is copied to the device and a captured call
// holds its own.  A tensor is cut into pieces of kClipPiece bytes; CTAs take every gridDim.x-th piece.  The first kernel writes a
// partial sum per CTA; in the second every CTA adds the partial sums up for itself, in the same order, so that
// all have the same factor and no counter or flag is needed.  It walks the pieces backwards: what the
// first kernel read last is what the L2 still holds.  Where the factor is 1 nothing is written.
// Bound by memory: 1.39 GB of bf16 in 660 us, 6.3 TB/s over its three passes; 77 MB of fp32 in 308 tensors in 41 us, the host's checks and
// launches about as long as the two kernels.
#include "follow.cuh"
#include "plan.cuh"
#include "m2d_seq.h"

namespace m2d {

constexpr int kClipTensors = 512, kClipPiece = 32768, kClipThreads = 256;

struct ClipTable {
    char* p[kClipTensors];
    long long bytes[kClipTensors];                // bf16: with bit 62 set
    unsigned first[kClipTensors + 1];             // piece numbers
    int count;
};
constexpr long long kClipBf16 = 1ll << 62;

// Calls vec(16-byte pointer) and one(element pointer) for a piece, of the type it has.
template <typename V, typename O>
__device__ __forceinline__ void for_piece(char* p, int bytes, int es, V vec, O one) {
    const int head = min(bytes, (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15));
    const int body = (bytes - head) / 16;
    if ((int)threadIdx.x < head / es) one(p + threadIdx.x * es);
    const int tail0 = head + body * 16;
    if ((int)threadIdx.x < (bytes - tail0) / es) one(p + tail0 + threadIdx.x * es);
    p += head;
#pragma unroll 4
    for (int i = threadIdx.x; i < body; i += kClipThreads) vec(reinterpret_cast<uint4*>(p) + i);
}
__device__ __forceinline__ int clip_find(const ClipTable& t, unsigned piece) {
    int lo = 0, hi = t.count;                     // first[lo] <= piece < first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= piece) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ float sq2(unsigned u, float s) {
    const float a = __uint_as_float(u << 16), b = __uint_as_float(u & 0xffff0000u);
    return fmaf(a, a, fmaf(b, b, s));
}
__device__ __forceinline__ double clip_block_sum(double v) {
    __shared__ double part[kClipThreads / 32];
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < kClipThreads / 32; ++i) v += part[i];
    return v;
}

__global__ void __launch_bounds__(kClipThreads) clip_norm_kernel(const __grid_constant__ ClipTable t, double* __restrict__ partial) {
    let_follow();
    double total = 0.0;
    for (unsigned piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
        const int i = clip_find(t, piece);
        const bool bf16 = t.bytes[i] & kClipBf16;
        const long long off = (long long)(piece - t.first[i]) * kClipPiece, left = (t.bytes[i] & ~kClipBf16) - off;
        char* const p = t.p[i] + off;
        const int bytes = (int)min((long long)kClipPiece, left);
        float s0 = 0.f, s1 = 0.f;                 // (at most 64 squares each)
        if (bf16)
            for_piece(p, bytes, 2, [&](uint4* q) { const uint4 u = __ldg(q); s0 = sq2(u.x, sq2(u.y, s0)); s1 = sq2(u.z, sq2(u.w, s1)); },
                      [&](char* q) { const float v = bf16_bits_to_float(*reinterpret_cast<unsigned short*>(q)); s0 = fmaf(v, v, s0); });
        else
            for_piece(p, bytes, 4,
                      [&](uint4* q) {
                          const float4 u = __ldg(reinterpret_cast<float4*>(q));
                          s0 = fmaf(u.x, u.x, fmaf(u.y, u.y, s0));
                          s1 = fmaf(u.z, u.z, fmaf(u.w, u.w, s1));
                      },
                      [&](char* q) { const float v = *reinterpret_cast<float*>(q); s0 = fmaf(v, v, s0); });
        total += (double)s0 + (double)s1;
    }
    total = clip_block_sum(total);
    if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

__global__ void __launch_bounds__(kClipThreads) clip_scale_kernel(const __grid_constant__ ClipTable t, const double* partial, int partials, float max_norm, float* norm) {
    follow_wait();
    double total = 0.0;
    for (int i = threadIdx.x; i < partials; i += kClipThreads) total += partial[i];
    total = sqrt(clip_block_sum(total));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    const float f = (float)((double)max_norm / ((double)(float)total + 1e-6));
    if (f >= 1.f || max_norm == __int_as_float(0x7f800000)) return;      // (a NaN goes on, but not where there is no bound)
    const unsigned pieces = t.first[t.count];
    for (unsigned k = blockIdx.x; k < pieces; k += gridDim.x) {
        const unsigned piece = pieces - 1 - k;
        const int i = clip_find(t, piece);
        const bool bf16 = t.bytes[i] & kClipBf16;
        const long long off = (long long)(piece - t.first[i]) * kClipPiece, left = (t.bytes[i] & ~kClipBf16) - off;
        char* const p = t.p[i] + off;
        const int bytes = (int)min((long long)kClipPiece, left);
        if (bf16) {
            auto two = [&](unsigned u) { return pack_bf16x2(__uint_as_float(u << 16) * f, __uint_as_float(u & 0xffff0000u) * f); };
            for_piece(p, bytes, 2, [&](uint4* q) { uint4 u = *q; u.x = two(u.x); u.y = two(u.y); u.z = two(u.z); u.w = two(u.w); *q = u; },
                      [&](char* q) {
                          __nv_bfloat16* e = reinterpret_cast<__nv_bfloat16*>(q);
                          *e = __float2bfloat16_rn(__bfloat162float(*e) * f);
                      });
        } else {
            for_piece(p, bytes, 4,
                      [&](uint4* q) {
                          float4 u = *reinterpret_cast<float4*>(q);
                          u.x *= f; u.y *= f; u.z *= f; u.w *= f;
                          *reinterpret_cast<float4*>(q) = u;
                      },
                      [&](char* q) { *reinterpret_cast<float*>(q) *= f; });
        }
    }
}

static int check_clip(const m2d_clip_tensor* t, int32_t count) {
    if (count < 0) return M2D_ERR_SHAPE;
    if (count && !t) return M2D_ERR_NULL;
    for (int i = 0; i < count; ++i) {
        if (t[i].dtype != M2D_F32 && t[i].dtype != M2D_BF16) return M2D_ERR_DTYPE;
        if (t[i].elements < 0) return M2D_ERR_SHAPE;
        if (t[i].elements && !t[i].data) return M2D_ERR_NULL;
        if (t[i].elements > (1ll << 44)) return M2D_ERR_TOO_LARGE;
        if (reinterpret_cast<uintptr_t>(t[i].data) % (t[i].dtype == M2D_F32 ? 4 : 2)) return M2D_ERR_PITCH;
    }
    return M2D_OK;
}
// CTAs of one launch; a partial sum each
static int clip_grid() { return 8 * sm_count(); }
static int clip_launches(int32_t count) { return count > 0 ? (count + kClipTensors - 1) / kClipTensors : 1; }

}  // namespace m2d

using namespace m2d;

extern "C" uint64_t m2d_clip_workspace(const m2d_clip_tensor* tensors, int32_t count) {
    return check_clip(tensors, count) == M2D_OK ? (uint64_t)clip_launches(count) * clip_grid() * sizeof(double) : 0;
}

extern "C" int m2d_clip_grad_norm(const m2d_clip_tensor* tensors, int32_t count, float max_norm, float* norm, void* workspace, uint64_t workspace_bytes, void* stream) {
    const int rc = check_clip(tensors, count);
    if (rc != M2D_OK) return rc;
    if (!norm) return M2D_ERR_NULL;
    if (!workspace || workspace_bytes < m2d_clip_workspace(tensors, count) || (reinterpret_cast<uintptr_t>(workspace) & 255)) return M2D_ERR_WORKSPACE;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    double* const partial = static_cast<double*>(workspace);
    const int launches = clip_launches(count), grid = clip_grid();
    ClipTable t;
    for (int pass = 0; pass < 2; ++pass)
        for (int l = 0; l < launches; ++l) {
            if (!pass || launches > 1) {          // (one launch's worth: the table is still the one)
                t.count = 0;
                unsigned long long pieces = 0;
                for (int i = l * kClipTensors; i < std::min(count, (l + 1) * kClipTensors); ++i) {
                    if (!tensors[i].elements) continue;
                    const long long bytes = tensors[i].elements * (tensors[i].dtype == M2D_F32 ? 4 : 2);
                    t.p[t.count] = static_cast<char*>(tensors[i].data);
                    t.bytes[t.count] = bytes | (tensors[i].dtype == M2D_BF16 ? kClipBf16 : 0);
                    t.first[t.count++] = (unsigned)pieces;
                    pieces += (unsigned long long)((bytes + kClipPiece - 1) / kClipPiece);
                    if (pieces >= (1ull << 31)) return M2D_ERR_TOO_LARGE;
                }
                t.first[t.count] = (unsigned)pieces;
            }
            if (!pass) clip_norm_kernel<<<grid, kClipThreads, 0, st>>>(t, partial + (size_t)l * grid);
            else if (!launch_following(clip_scale_kernel, dim3(grid), dim3(kClipThreads), 0, st, t, (const double*)partial, launches * grid, max_norm, l ? (float*)nullptr : norm)) return M2D_ERR_LAUNCH;
        }
    return cudaGetLastError() == cudaSuccess ? M2D_OK : M2D_ERR_LAUNCH;
}
