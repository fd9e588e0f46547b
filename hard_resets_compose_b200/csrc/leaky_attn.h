// Internal declarations of leaky attention (leaky_attn.cu, leaky_attn_tc.cu).
//
// With b = exp(log_decay[h]) <= 1 a head's state and output are
//
//   S_t = b S_{t-1} + k_t v_t^T,   o_t = scale * S_t^T q_t
//
// The gradients are the same recurrence on other operands.  Written out,
// o_i = scale * sum_{j <= i} b^(i-j) (q_i . k_j) v_j + scale * b^(i+1) S^T q_i with
// S the state before token 0, so
//
//   dq_i = scale * sum_{j <= i} b^(i-j) (do_i . v_j) k_j + scale * b^(i+1) S do_i
//   dk_j = scale * sum_{i >= j} b^(i-j) (v_j . do_i) q_i + b^(n-1-j) G v_j
//   dv_j = scale * sum_{i >= j} b^(i-j) (k_j . q_i) do_i + b^(n-1-j) G^T k_j
//
// with G the gradient of the state after the last of n tokens.  dq runs forward
// with (do, v, k) in the place of (q, k, v) and the transposed state; dk and dv
// run backward in time with (v, do, q) and (k, q, do).  A backward pass carries
// the gradient of the state *before* the tokens it has seen, so its weights have
// one power of b less on the carried term and one more on the new one (`shift`).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "lifscan_b200.h"

namespace lifb {

// One pass of the recurrence over all sequences and heads.
struct AttnPass {
    const void *q, *k, *v;        // element strides below: sequence, token, head
    void *o;
    int64_t qs[3], ks[3], vs[3], os[3];
    int qg, kg, vg;               // heads that share one of the operand's heads
    int dq, dv;                   // widths of q and k, and of v and o
    const float *s_in;            // the carried state before the first chunk, or NULL (zeros)
    float *s_out;                 // after the last one, or NULL
    int64_t s_row, s_col;         // their strides: row (q's width), column (v's)
    float p_scale, i_scale, w_scale;  // of the chunk's products, the carried term, and the state's update
    int shift, rev, o_f32;
    float *seg;                   // [B*H][nseg + 1][dq][dv]: each time segment's starting state (0's unused);
                                  // the last is what the final state is joined from
    // of a pass over a part of the widths (leaky_attn_tc32.cu): elements between two heads' states,
    // a segment state's row, and whether o is added to
    int64_t mat, seg_row;
    int add;
};

constexpr int kAttnMaxPasses = 3;

template <int N>
struct AttnArgsOf {
    AttnPass p[N];
    const float *log_decay;       // [H]
    const int32_t *lengths;       // [B], or NULL: every sequence has T tokens
    int64_t B, T, H;
    int passes;                   // of this launch: the fastest part of the block's number, so that the
                                  // passes over one head run together and share its operands in L2
    int nseg;                     // time segments, each with a multiple of kAttnSegGrain tokens
    int64_t seg_tokens;
};
using AttnArgs = AttnArgsOf<kAttnMaxPasses>;

constexpr int kAttnSegGrain = 128;
constexpr int kAttnMaxDim = 128;  // of q, k and of v

#ifdef __CUDACC__
// b^n = exp(log_decay * n); b^0 = 1 for b = 0 (log_decay = -inf) too.
__device__ __forceinline__ float decay_pow(float ld, float n) { return n == 0.0f ? 1.0f : expf(ld * n); }

// b^n as a sum of two floats: the factor between chunks is applied once for each
// chunk, so an error in it grows with their number (in one float, b^32 near 1
// is off by up to 3e-8: 8e-6 after the 256 chunks that such a head remembers).
struct DecayFactor {
    float hi, lo;
    __device__ __forceinline__ DecayFactor(float ld, int64_t n)
    {
        const double b = n == 0 ? 1.0 : exp((double)ld * (double)n);
        hi = (float)b;
        lo = (float)(b - (double)hi);
    }
    __device__ __forceinline__ float times(float s) const { return fmaf(s, hi, s * lo); }
};

__device__ __forceinline__ int64_t attn_length(const int32_t *lengths, int64_t b, int64_t T)
{
    if (!lengths) return T;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > T ? T : n;
}
#endif

// leaky_attn.cu: chunks of 32 tokens on the fp32 pipe, any type and strides.
// state_only: the segments' own end states into seg (first launch of a split).
bool attn_simt(const AttnArgs &a, int passes, int dtype, bool state_only, cudaStream_t s);

// leaky_attn_tc.cu: chunks of 128 tokens on the tensor cores, bf16 operands that TMA
// can load (16-byte aligned strides, widths multiples of 8).
bool attn_tc_applies(const AttnArgs &a, int passes, int dtype);
bool attn_tc(const AttnArgs &a, int passes, cudaStream_t s);
// leaky_attn_state.cu: the segments' own end states for them (the last segment's where the
// pass returns its state).
bool attn_state(const AttnArgs &a, int passes, bool finish, cudaStream_t s);
// A tensor map of an operand in tiles of 64 columns by 128 tokens.
bool attn_operand_map(CUtensorMap *m, const void *base, const int64_t (&st)[3], int d, int64_t T, int64_t heads,
                      int64_t B);
// Whether attn_tc returns this pass's state itself.
bool attn_tc_returns_state(int dq, int dv);
// leaky_attn_tc32.cu: the same for fp32 operands in 16-byte aligned vectors.
constexpr int kT32W = 64;  // widths of its tiles; wider heads are several
bool attn_tc32_applies(const AttnArgs &a, int passes, int dtype);
bool attn_tc32(const AttnArgs &a, int passes, bool state_only, cudaStream_t s);

}  // namespace lifb
