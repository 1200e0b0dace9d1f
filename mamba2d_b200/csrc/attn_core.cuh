// Linear attention with a decay per head: the one computation that the forward pass and the three gradients share.
//
// With the decay c accumulated inside a chunk of tokens, and St (Kd,Vd) the state that is carried from chunk to chunk,
//     out_r = s_intra sum_{c <= r} D_rc (x_r . y_c) z_c  +  s_inter w_r x_r^T St,        D_rc = exp(c_r - c_c)
//     St   <- exp(c_end) St + s_update sum_c u_c y_c z_c^T
// with w_r = exp(c_r), u_c = exp(c_end - c_c) forwards in time; backwards the chunks are walked from the last to the
// first, the mask is c >= r (D_rc = exp(c_c - c_r)) and w and u change places.  That is
//     o   forwards  with (x, y, z) = (q, k, v)        dq  forwards  with (do, v, k)
//     dk  backwards with (v, do, q)                   dv  backwards with (k, q, do)
// where the carried states are S, S^T, R^T and R: S of the recurrence, R the gradient of the state from later tokens.
//
// The decay's own gradient: with e_i = <S, R> at the end of a run of kAnchor tokens (S after it, R from what follows),
//     dg_t = sum_{s >= t in the run} (q_s . dq_s - k_s . dk_s) + e_i,
// so that the rounding of a sum does not grow with the length of the sequence.  dq and dk write these dots and the
// states at the runs' ends.
#pragma once

#include "plan.cuh"
#include "m2d_seq.h"

namespace m2d {

constexpr int kAnchor = 512;          // tokens between two states kept for the decay's gradient
constexpr float kMinDecay = -1.0e4f;  // (natural) exp is zero long before; keeps sums of -inf apart from NaN

struct AttnTensor {
    const void* p;
    long long sb, st, sh;     // strides in elements: batch, token, head
    int per;                  // heads of z that share one of this tensor's
    int vec;                  // rows may be read in vectors of four elements
};
struct AttnState {            // (B,H,[segments],rows,cols) in fp32
    float* p;
    long long sb, sh, sg;     // strides: batch, head, segment
    long long sr, sc;         // strides: row, column
};
struct AttnCore {
    AttnTensor x, y, z, e;    // e: what out is multiplied with for `dots`
    void* out;
    long long ob, ot, oh;
    int out_f32, rev;
    int Kd, Vd;
    float s_intra, s_inter, s_update;
    float* dots;              // [column block][B][T][H], or nullptr
    AttnState init, fin;      // p may be nullptr
    float* anchors;           // [B][H][runs][Kd Vd], or nullptr; the same order for dq and dk
    float* seg_state;         // [B][H][segments][Kd Vd]
    float* seg_decay;         // [B][H][segments], log2
};
struct AttnLaunch {
    AttnCore core[3];
    const float* g;
    long long gb, gt, gh;
    const int* lengths;
    int B, T, H;
    int nseg, seg_len, runs;
    int join_here;            // the kernel joins the segments before its own, no launch has
    int parts, part_len;      // tcgen05 form where segments are joined so: states are those of the segments' parts, of all segments
                              // but the one that nothing comes after: (B,H,(nseg - 1) parts) of them.  Else one part a segment, of all.
    int seg_columns;          // segments' states have a column's rows next to one another, else a row's columns
};

__device__ __forceinline__ const void* attn_at(const AttnTensor& t, int b, int h, size_t elem) {
    return static_cast<const char*>(t.p) + (size_t)((long long)b * t.sb + (long long)(h / t.per) * t.sh) * elem;
}
__device__ __forceinline__ int attn_length(const AttnLaunch& a, int b) {
    return a.lengths ? min(max(__ldg(a.lengths + b), 0), a.T) : a.T;
}
// One decay in units of log2, in 64 bits: a chunk's sums and their differences are then exact to fp32.  (A NaN stays.)
__device__ __forceinline__ double attn_decay(float g) { return (double)(g < kMinDecay ? kMinDecay : g) * 1.4426950408889634; }

}  // namespace m2d
