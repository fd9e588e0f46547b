// What the bf16 kernels of leaky attention share (leaky_attn_tc.cu,
// leaky_attn_state.cu).
#pragma once

#include <cuda_bf16.h>

#include "leaky_attn.h"
#include "tc.cuh"

namespace lifb {

constexpr int kTcC = 128;             // tokens of a chunk
constexpr int kTcBlock = kTcC * 128;  // bytes of 128 rows of 64 bf16

// Registers a thread, moved between the warpgroups of a block.
template <int N>
__device__ __forceinline__ void regs_inc()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// A token's weight, as the pieces of its weighted key need it: two bf16 values
// (each twice in a word) whose sum is w to 2^-18, or w itself.
template <int NP>
struct TokenWeight {
    uint32_t wh, wm;
    __device__ __forceinline__ void set(float w)
    {
        wh = NP == 2 ? pack_bf16(w, w) : __float_as_uint(w);
        wm = NP == 2 ? pack_bf16(w - bf16_lo(wh), w - bf16_lo(wh)) : 0;
    }
    // w * x for eight bf16 elements x (four words) as NP bf16 pieces.  Two pieces: hi =
    // x wh rounded; what that dropped is exact in bf16 (the product has 16 bits), so
    // mid = x wm + it.
    __device__ __forceinline__ void split(const uint4 &x4, uint4 &hi4, uint4 &mid4, uint4 &lo4) const
    {
        const uint32_t in[4] = {x4.x, x4.y, x4.z, x4.w};
        uint32_t hi[4], mid[4], lo[4] = {};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (NP == 2) {
                const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162 *>(&in[e]);
                const __nv_bfloat162 h2 = *reinterpret_cast<const __nv_bfloat162 *>(&wh);
                const __nv_bfloat162 m2 = *reinterpret_cast<const __nv_bfloat162 *>(&wm);
                const __nv_bfloat162 h = __hmul2_rn(x, h2);
                const __nv_bfloat162 m = __hfma2(x, m2, __hfma2(x, h2, __hneg2(h)));
                hi[e] = *reinterpret_cast<const uint32_t *>(&h);
                mid[e] = *reinterpret_cast<const uint32_t *>(&m);
            } else {
                const float w = __uint_as_float(wh);
                const float f0 = bf16_lo(in[e]) * w, f1 = bf16_hi(in[e]) * w;
                hi[e] = pack_bf16(f0, f1);
                const float g0 = f0 - bf16_lo(hi[e]), g1 = f1 - bf16_hi(hi[e]);
                mid[e] = pack_bf16(g0, g1);
                lo[e] = pack_bf16(g0 - bf16_lo(mid[e]), g1 - bf16_hi(mid[e]));
            }
        }
        hi4 = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        mid4 = make_uint4(mid[0], mid[1], mid[2], mid[3]);
        lo4 = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
};

}  // namespace lifb
