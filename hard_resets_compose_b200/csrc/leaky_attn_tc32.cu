// Leaky attention in fp32 on the 5th-generation tensor cores.  leaky_attn.h has the
// recurrence, leaky_attn_tc.cu the chunked form in bf16.
//
// A block does 64 columns of q and k and 64 of v.  Everything is linear in the products
// of a column of k with one of v, so wider heads are two or four such parts, each with
// its own part of the state: the parts over v's columns run together, and those over
// the second half of q's and k's columns in a launch of their own that adds to o (in a
// fixed order).  128 x 128 costs a third more multiplications than whole tiles would
// (Q K^T twice), which would not fit an SM as three pieces.  Measured against the fp32
// pipe: B 8, T 1024, H 8, 128 x 128: forward 559 -> 136 us, backward 1308 -> 379 us; B 5,
// T 1336, 8 heads on one k/v head, 32 x 128: 250 -> 73, 688 -> 231 us.
//
// Each fp32 operand is the sum of three bf16 pieces, x = x0 + x1 + x2 (8 + 8 + 8 bits),
// and a product of two operands the six products of pieces down to 2^-16:
// x2 y0, x0 y2, x1 y1, x1 y0, x0 y1, x0 y0, added up in that order, the small ones
// first, so that the accumulator (which drops bits below its last place) is small
// while most of the additions happen.  What is left out is 2^-24 of the result.
//
// A chunk of 128 tokens costs 6 x (128 x 128 x 64 [Q K^T] + 128 x 64 x 64 [Q S] + 128 x
// 64 x 128 [P V] + 64 (M is 128 all the same) x 64 x 128 [the state]) multiply-adds:
// 6500 cycles of the tensor cores, 17 times the rate of the fp32 pipe (q, k, v, o are
// 128 KB: 5500 cycles of an SM's share of the memory).  Measured: 12000 a chunk (B 64, T
// 1024, H 4, 64 x 64: forward 465 us on the fp32 pipe, 120 us here); what is left is the
// making of the pieces, some 250 elements a thread and chunk, which runs one tile after
// another (the pieces' stores share the 128 bytes a cycle with the MMAs' operands).
//
// All tiles are there once (216 KB of pieces), so each is refilled while the MMAs that
// do not need it run: P(c), Q S(c), the state's(c), P V(c), P(c + 1), ...
//   scores   P: tensor memory -> decay -> three pieces, in tensor memory (A operand)
//   output   the epilogue;  state: as in the bf16 kernel, its copy in three pieces
//   keys     k's pieces, and those of the weighted k;  rows: q's and v's pieces
//   one warp issues the MMAs.
// Powers of the decay are exp of the product each (a chain of multiplications would
// be off by 2^-24 a step).  Every wait is bounded (status 101).
#include <algorithm>

#include "leaky_attn.h"
#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "seq_types.cuh"
#include "tc.cuh"

namespace lifb {

namespace {

constexpr int kT32C = 128, kT32Threads = 768;
constexpr uint32_t kT32Tile = kT32C * 128;       // one piece of 128 rows
constexpr uint32_t kT32S = kT32W * 128;          // one piece of the state
constexpr uint32_t kT32Q = 0, kT32K = 3 * kT32Tile, kT32Kw = 6 * kT32Tile, kT32V = 9 * kT32Tile,
                   kT32St = 12 * kT32Tile, kT32Bytes = kT32St + 3 * kT32S;
static_assert(kT32Bytes + 1024 + 512 <= 227 * 1024, "tiles fit an SM");
// tensor memory: the scores, their pieces, P V, Q S, the state's result
constexpr uint32_t kT32Pa = 128, kT32O1 = 320, kT32O2 = 384, kT32Ds = 448, kT32Cols = 512;
// warpgroups and their registers; 768 threads are launched with 80 each
enum T32Group { kScores, kOutput, kState, kKeys, kRows, kIssue };
constexpr int kT32Regs[6] = {72, 72, 120, 96, 96, 24};
static_assert(kT32Regs[0] + kT32Regs[1] + kT32Regs[2] + kT32Regs[3] + kT32Regs[4] + kT32Regs[5] <= 480,
              "no more registers than the block was launched with");

struct T32Bars {
    uint64_t q_ready, k_ready, kw_ready, v_ready, s_ready, p_ready, o_free, ds_free;  // 128 threads each
    uint64_t p_full, o2_full, ds_full, o1_full, done;                                // MMAs
};

// The parts of one launch.
using T32Args = AttnArgsOf<4 * kAttnMaxPasses>;

// The piece pairs of a product, small ones first: a nibble each.
constexpr uint32_t kPieceA = 0x001102, kPieceB = 0x010120;

// Eight fp32 values as three times eight bf16.
__device__ __forceinline__ void split_eight(const uint64_t (&x)[4], uint4 (&out)[3])
{
    uint32_t w[3][4];
    const uint64_t minus = two(-1.0f, -1.0f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint64_t r = x[i];
#pragma unroll
        for (int p = 0; p < 3; p++) {
            w[p][i] = pack2_bf16(r);
            if (p < 2) r = fma2(two(bf16_lo(w[p][i]), bf16_hi(w[p][i])), minus, r);  // exact
        }
    }
#pragma unroll
    for (int p = 0; p < 3; p++) out[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// This thread's eight vectors (eight columns each) of a [128, 64] fp32 tile: rows
// st / 8 + 16 i, columns 8 (st % 8) on; zeros past n rows and d columns.
struct TileRegs {
    float4 a[8], b[8];
    __device__ __forceinline__ void load(const float *src, int64_t stride, int n, int d, int st)
    {
        const int c = (st & 7) * 8;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int r = st / 8 + 16 * i;
            const float *at = src + r * stride + c;
            a[i] = r < n && c < d ? *reinterpret_cast<const float4 *>(at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            b[i] = r < n && c + 4 < d ? *reinterpret_cast<const float4 *>(at + 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    // as three pieces, rows scaled by w[i]; 128-byte swizzled
    template <bool SCALE>
    __device__ __forceinline__ void put(unsigned char *tile, const float (&w)[8], int st) const
    {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint64_t x[4] = {two(a[i].x, a[i].y), two(a[i].z, a[i].w), two(b[i].x, b[i].y), two(b[i].z, b[i].w)};
            if (SCALE) {
                const uint64_t ww = two(w[i], w[i]);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = mul2(x[e], ww);
            }
            uint4 piece[3];
            split_eight(x, piece);
            const int r = st / 8 + 16 * i;
            unsigned char *at = tile + r * 128 + (((st & 7) ^ (r & 7)) * 16);
#pragma unroll
            for (int p = 0; p < 3; p++) *reinterpret_cast<uint4 *>(at + p * kT32Tile) = piece[p];
        }
    }
};

}  // namespace

template <bool STATE_ONLY>
__global__ void __launch_bounds__(kT32Threads, 1) k_attn_tc32(const __grid_constant__ T32Args a, int *status)
{
    extern __shared__ unsigned char t32_raw[];
    unsigned char *base = (unsigned char *)(((uintptr_t)t32_raw + 1023) & ~(uintptr_t)1023);
    __shared__ T32Bars bars;
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0), group = warp >> 2;
    const int item = blockIdx.x / a.passes;
    const AttnPass &p = a.p[blockIdx.x % a.passes];
    const int64_t bh = item / a.nseg;
    const int u = (int)(item - bh * a.nseg);  // in the order of the pass
    if (STATE_ONLY && u == a.nseg - 1) return;      // nothing starts from the last one
    const int64_t b = bh / a.H, h = bh - b * a.H;
    const int64_t len = attn_length(a.lengths, b, a.T);
    const float ld = a.log_decay[h];
    const int64_t seg = p.rev ? a.nseg - 1 - u : u;  // in time
    const int s0 = (int)(seg * a.seg_tokens), s1 = (int)min(a.T, seg * a.seg_tokens + a.seg_tokens);
    const int end = min(s1, (int)len);
    const int chunks = max(0, end - s0 + kT32C - 1) / kT32C;  // with tokens in them
    const int t_first = p.rev ? s0 + (chunks - 1) * kT32C : s0, t_step = p.rev ? -kT32C : kT32C;

    if (warp == 0) tmem_alloc(&tmem_slot, kT32Cols);
    if (tid == 32) {
        uint64_t *many[] = {&bars.q_ready, &bars.k_ready, &bars.kw_ready, &bars.v_ready,
                            &bars.s_ready, &bars.p_ready, &bars.o_free,   &bars.ds_free};
        for (uint64_t *m : many) mbar_init(m, 128);
        uint64_t *one[] = {&bars.p_full, &bars.o2_full, &bars.ds_full, &bars.o1_full, &bars.done};
        for (uint64_t *m : one) mbar_init(m, 1);
        fence_barrier_init();
    }
    tcgen05_before();
    __syncthreads();
    tcgen05_after();
    const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
    // bounded; a role that gives up ends, and the others then run out of theirs
    auto wait = [&](uint64_t *bar, int phase) {  // a whole warp's, one decision for it
        if (__all_sync(~0u, mbar_wait(bar, (uint32_t)phase & 1))) return true;
        atomicExch(status, kStatusTmaWaitTimeout);
        return false;
    };
    const int st = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;

    if (group == kIssue) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kT32Regs[kIssue]));
        if ((warp & 3) == 0) {
            const uint32_t sb = smem_u32(base);
            constexpr uint32_t kIdP = umma_idesc_bf16(kT32C, kT32C, false, false);
            constexpr uint32_t kIdO = umma_idesc_bf16(kT32C, kT32W, false, true);
            constexpr uint32_t kIdS = umma_idesc_bf16(kT32C, kT32W, true, true);
            // D (columns d) = the six products of A's and B's pieces: `steps` MMAs each, descriptors
            // advancing by ka and kb (16-byte units), pieces pa and pb apart.  A's second 64 rows (the
            // state's MMA has only 64) lie a tile on, inside.
            auto product = [&](uint32_t d, uint32_t a_at, uint32_t pa, int ka, uint32_t b_at, uint32_t pb, int kb,
                               int steps, uint32_t id) {
#pragma unroll 1
                for (int t = 0; t < 6; t++) {
                    const uint64_t da = umma_desc_sw128(a_at + ((kPieceA >> (4 * t)) & 15) * pa, kT32Tile);
                    const uint64_t db = umma_desc_sw128(b_at + ((kPieceB >> (4 * t)) & 15) * pb, kT32Tile);
#pragma unroll 4
                    for (int k = 0; k < steps; k++) umma_bf16_ss(d, da + k * ka, db + k * kb, id, t > 0 || k > 0);
                }
            };
            bool ok = true;
            for (int c = 0; ok && c < chunks; c++) {
                if (!STATE_ONLY) {
                    ok = wait(&bars.q_ready, c) && wait(&bars.k_ready, c);  // P's columns: p_ready(c - 1), below
                    if (!ok) break;
                    tcgen05_after();
                    if (elect_lane()) {
                        product(tmem, sb + kT32Q, kT32Tile, 2, sb + kT32K, kT32Tile, 2, kT32W / 16, kIdP);
                        umma_arrive(&bars.p_full);
                    }
                    ok = wait(&bars.s_ready, c) && (c == 0 || wait(&bars.o_free, c - 1));
                    if (!ok) break;
                    tcgen05_after();
                    if (elect_lane()) {
                        product(tmem + kT32O2, sb + kT32Q, kT32Tile, 2, sb + kT32St, kT32S, 128, kT32W / 16, kIdO);
                        umma_arrive(&bars.o2_full);
                    }
                }
                ok = wait(&bars.v_ready, c) && wait(&bars.kw_ready, c) && (c == 0 || wait(&bars.ds_free, c - 1));
                if (!ok) break;
                tcgen05_after();
                if (elect_lane()) {
                    product(tmem + kT32Ds, sb + kT32Kw, kT32Tile, 128, sb + kT32V, kT32Tile, 128, kT32C / 16, kIdS);
                    umma_arrive(&bars.ds_full);
                }
                if (!STATE_ONLY) {
                    ok = wait(&bars.p_ready, c);
                    if (!ok) break;
                    tcgen05_after();
                    if (elect_lane()) {
#pragma unroll 1
                        for (int t = 0; t < 6; t++) {
                            const uint32_t pa = tmem + kT32Pa + ((kPieceA >> (4 * t)) & 15) * 64;
                            const uint64_t db = umma_desc_sw128(sb + kT32V + ((kPieceB >> (4 * t)) & 15) * kT32Tile, kT32Tile);
#pragma unroll 4
                            for (int k = 0; k < kT32C / 16; k++)
                                umma_bf16_ts(tmem + kT32O1, pa + k * 8, db + k * 128, kIdO, t > 0 || k > 0);
                        }
                        umma_arrive(&bars.o1_full);
                    }
                }
            }
            if (elect_lane()) {  // nothing of the tensor cores is left running
                umma_arrive(&bars.done);
                mbar_wait(&bars.done, 0);
            }
        }
    } else if (group == kScores) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kT32Regs[kScores]));
        if (!STATE_ONLY) {
            uint64_t pw[8];  // of 16 columns in their order, from the one nearest the diagonal
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float lo = decay_pow(ld, (float)(p.rev ? 2 * i : 15 - 2 * i));
                const float hi = decay_pow(ld, (float)(p.rev ? 2 * i + 1 : 14 - 2 * i));
                pw[i] = two(lo, hi);
            }
            const float near = decay_pow(ld, (float)lane);
            const int w4 = warp & 3;
            for (int c = 0; c < chunks; c++) {
                const int n = min(kT32C, end - (t_first + c * t_step));
                if (!wait(&bars.p_full, c)) break;
                tcgen05_after();
#pragma unroll 1
                for (int s = 0; s < 8; s++) {
                    const int c0 = s * 16, blk = s >> 1;
                    const bool past = p.rev ? blk < w4 : blk > w4;  // on the other side of the diagonal
                    if (past) {
                        const uint32_t zero[8] = {};
#pragma unroll
                        for (int q = 0; q < 3; q++) tmem_store8(tmem + lanes + kT32Pa + q * 64 + s * 8, zero);
                        continue;
                    }
                    uint32_t x[16];
                    tmem_load16(tmem + lanes + c0, x);
                    // the nearest column's power, then pw's of the others from there
                    const float f = p.p_scale * decay_pow(ld, (float)max(0, p.rev ? c0 - st : st - c0 - 15));
                    tmem_wait_ld();
                    if (blk == w4) {
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int d = p.rev ? c0 + e - st : st - c0 - e;  // -31 .. 31
                            const float g = __shfl_sync(~0u, near, d & 31);
                            x[e] = d >= 0 && c0 + e < n ? __float_as_uint(__uint_as_float(x[e]) * (p.p_scale * g)) : 0u;
                        }
                    } else {
                        const uint64_t ff = two(f, f);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            float lo, hi;
                            both(mul2(two(x[2 * i], x[2 * i + 1]), mul2(pw[i], ff)), lo, hi);
                            x[2 * i] = __float_as_uint(lo);
                            x[2 * i + 1] = __float_as_uint(hi);
                        }
                        if (c0 + 16 > n) {
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                if (c0 + e >= n) x[e] = 0;
                        }
                    }
                    uint32_t out[3][8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        uint64_t r = two(x[2 * i], x[2 * i + 1]);
#pragma unroll
                        for (int q = 0; q < 3; q++) {
                            out[q][i] = pack2_bf16(r);
                            if (q < 2) r = fma2(two(bf16_lo(out[q][i]), bf16_hi(out[q][i])), two(-1.0f, -1.0f), r);
                        }
                    }
#pragma unroll
                    for (int q = 0; q < 3; q++) tmem_store8(tmem + lanes + kT32Pa + q * 64 + s * 8, out[q]);
                }
                tmem_wait_st();
                tcgen05_before();
                mbar_arrive(&bars.p_ready);
            }
        }
    } else if (group == kOutput) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kT32Regs[kOutput]));
        if (!STATE_ONLY) {
            float *o = (float *)p.o + b * p.os[0] + h * p.os[2];
            for (int c = 0; c < chunks; c++) {
                const int t0 = t_first + c * t_step, n = min(kT32C, end - t0);
                const int r = p.rev ? n - 1 - st : st;
                const float w = st < n ? p.i_scale * decay_pow(ld, (float)(r + 1 - p.shift)) : 0.0f;
                if (!wait(&bars.o1_full, c)) break;
                tcgen05_after();
                float *dst = o + (int64_t)(t0 + st) * p.os[1];
#pragma unroll 1
                for (int g = 0; g < kT32W; g += 16) {
                    uint32_t x[16], y[16];
                    float4 had[4];
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        had[e / 4] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (p.add && st < n && g + e < p.dv) had[e / 4] = *reinterpret_cast<const float4 *>(dst + g + e);
                    }
                    tmem_load16(tmem + lanes + kT32O1 + g, x);
                    tmem_load16(tmem + lanes + kT32O2 + g, y);
                    tmem_wait_ld();
                    if (g == kT32W - 16) {
                        tcgen05_before();
                        mbar_arrive(&bars.o_free);
                    }
                    if (t0 + st < s1) {
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            float f[4];
#pragma unroll
                            for (int q = 0; q < 4; q++)
                                f[q] = st < n ? fmaf(w, __uint_as_float(y[e + q]), __uint_as_float(x[e + q])) : 0.0f;
                            const float4 z = had[e / 4];
                            if (g + e < p.dv)
                                *reinterpret_cast<float4 *>(dst + g + e) =
                                    make_float4(z.x + f[0], z.y + f[1], z.z + f[2], z.w + f[3]);
                        }
                    }
                    __syncwarp();
                }
            }
            // tokens past the sequence's end in chunks that have none of it
            const int z0 = s0 + chunks * kT32C, per = p.dv / 4;
            const int64_t nz = (int64_t)max(0, s1 - z0) * per;
            for (int64_t i = st; i < nz; i += 128) {
                const int64_t r = i / per;
                *reinterpret_cast<float4 *>(o + (z0 + r) * p.os[1] + (i - r * per) * 4) =
                    make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
    } else if (group == kState) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kT32Regs[kState]));
        const bool has_row = st < kT32W;  // uniform over a warp
        uint64_t S[kT32W / 2];            // pairs of columns of this thread's row
        const int64_t mat = p.mat;
        {
            const float *s_in = nullptr;
            int64_t row = p.s_row, col = p.s_col;
            if (!STATE_ONLY) {
                if (u == 0) {
                    if (p.s_in) s_in = p.s_in + bh * mat;
                } else {
                    s_in = p.seg + (bh * (a.nseg + 1) + u) * mat;
                    row = p.seg_row;
                    col = 1;
                }
            }
#pragma unroll
            for (int j = 0; j < kT32W / 2; j++) S[j] = 0;
            // (a branch, not a condition of each load: what is not there is not fetched either)
            if (s_in && st < p.dq) {
                s_in += st * row;
#pragma unroll
                for (int j = 0; j < kT32W; j += 2)
                    if (j < p.dv) S[j / 2] = two(s_in[j * col], s_in[(j + 1) * col]);
            }
        }
        const DecayFactor full(ld, kT32C);
        for (int c = 0; c < chunks; c++) {
            if (!STATE_ONLY) {
                if (c > 0 && !wait(&bars.o2_full, c - 1)) break;  // Q S has read the last copy
                if (has_row) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint64_t x[4] = {S[4 * j], S[4 * j + 1], S[4 * j + 2], S[4 * j + 3]};
                        uint4 piece[3];
                        split_eight(x, piece);
#pragma unroll
                        for (int q = 0; q < 3; q++)
                            *reinterpret_cast<uint4 *>(base + kT32St + q * kT32S + st * 128 + ((j ^ (st & 7)) * 16)) =
                                piece[q];
                    }
                }
                fence_proxy_async_shared();
                mbar_arrive(&bars.s_ready);
            }
            const int n = min(kT32C, end - (t_first + c * t_step));
            const DecayFactor bn = n == kT32C ? full : DecayFactor(ld, n);
            const uint64_t bn_hi = two(bn.hi, bn.hi), bn_lo = two(bn.lo, bn.lo);
            if (!wait(&bars.ds_full, c)) break;
            tcgen05_after();
            if (has_row) {
#pragma unroll
                for (int g = 0; g < kT32W; g += 16) {
                    uint32_t x[16];
                    tmem_load16(tmem + kT32Ds + lanes + g, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        uint64_t &z = S[g / 2 + e];
                        z = fma2(z, bn_hi, fma2(z, bn_lo, two(x[2 * e], x[2 * e + 1])));
                    }
                }
            }
            tcgen05_before();
            mbar_arrive(&bars.ds_free);
        }
        float *s_out = nullptr;
        int64_t row = p.seg_row, col = 1;
        if (STATE_ONLY) {
            s_out = p.seg + (bh * (a.nseg + 1) + u + 1) * mat;
        } else if (u == a.nseg - 1 && p.s_out) {
            s_out = p.s_out + bh * mat;
            row = p.s_row;
            col = p.s_col;
        }
        if (s_out && st < p.dq) {
#pragma unroll
            for (int j = 0; j < kT32W; j += 2) {
                float f[2];
                both(S[j / 2], f[0], f[1]);
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (j + e < p.dv) s_out[st * row + (j + e) * col] = f[e];
            }
        }
    } else if (group == kKeys) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kT32Regs[kKeys]));
        const float *k = (const float *)p.k + b * p.ks[0] + (h / p.kg) * p.ks[2];
        float wk[8];  // of this thread's rows
        int wn = -1;  // the chunk size that they are for
        TileRegs x;
        for (int c = 0; c < chunks; c++) {
            const int t0 = t_first + c * t_step, n = min(kT32C, end - t0);
            x.load(k + (int64_t)t0 * p.ks[1], p.ks[1], n, p.dq, st);
            if (!STATE_ONLY) {
                if (c > 0 && !wait(&bars.p_full, c - 1)) break;
                x.put<false>(base + kT32K, wk, st);
                fence_proxy_async_shared();
                mbar_arrive(&bars.k_ready);
            }
            if (n != wn) {  // the first chunk, the one with the sequence's end, and the one after it
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int row = st / 8 + 16 * i, r = p.rev ? n - 1 - row : row;
                    wk[i] = row < n ? p.w_scale * decay_pow(ld, (float)(n - 1 - r + p.shift)) : 0.0f;
                }
                wn = n;
            }
            if (c > 0 && !wait(&bars.ds_full, c - 1)) break;
            x.put<true>(base + kT32Kw, wk, st);
            fence_proxy_async_shared();
            mbar_arrive(&bars.kw_ready);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kT32Regs[kRows]));
        const float *q = (const float *)p.q + b * p.qs[0] + (h / p.qg) * p.qs[2];
        const float *v = (const float *)p.v + b * p.vs[0] + (h / p.vg) * p.vs[2];
        const float none[8] = {};
        TileRegs x;
        for (int c = 0; c < chunks; c++) {
            const int t0 = t_first + c * t_step, n = min(kT32C, end - t0);
            if (!STATE_ONLY) {
                x.load(q + (int64_t)t0 * p.qs[1], p.qs[1], n, p.dq, st);
                if (c > 0 && !wait(&bars.o2_full, c - 1)) break;
                x.put<false>(base + kT32Q, none, st);
                fence_proxy_async_shared();
                mbar_arrive(&bars.q_ready);
            }
            x.load(v + (int64_t)t0 * p.vs[1], p.vs[1], n, p.dv, st);
            if (c > 0 && !wait(STATE_ONLY ? &bars.ds_full : &bars.o1_full, c - 1)) break;
            x.put<false>(base + kT32V, none, st);
            fence_proxy_async_shared();
            mbar_arrive(&bars.v_ready);
        }
    }
    tcgen05_before();
    __syncthreads();
    if (warp == 0) {
        tcgen05_after();
        tmem_free(tmem, kT32Cols);
    }
}

bool attn_tc32_applies(const AttnArgs &a, int passes, int dtype)
{
    if (dtype != LIFB_F32) return false;
    auto four = [&](const void *p, const int64_t (&st)[3], int group) {  // (one element along it: never used)
        return aligned16(p) && (a.B == 1 || st[0] % 4 == 0) && (a.T == 1 || st[1] % 4 == 0) &&
               (a.H == group || st[2] % 4 == 0);
    };
    for (int i = 0; i < passes; i++) {
        const AttnPass &p = a.p[i];
        if (p.dq > kAttnMaxDim || p.dv > kAttnMaxDim || p.dq % 4 || p.dv % 4 || !aligned16(p.o) ||
            !four(p.q, p.qs, p.qg) || !four(p.k, p.ks, p.kg) || !four(p.v, p.vs, p.vg))
            return false;
    }
    return true;
}

namespace {

// The part of pass p with columns from 64 qi of q and k and 64 vi of v and o.
AttnPass part_of(const AttnPass &p, int qi, int vi)
{
    AttnPass x = p;
    const int q0 = qi * kT32W, v0 = vi * kT32W;
    x.q = (const float *)p.q + q0;
    x.k = (const float *)p.k + q0;
    x.v = (const float *)p.v + v0;
    x.o = (float *)p.o + v0;
    x.dq = std::min(p.dq - q0, kT32W);
    x.dv = std::min(p.dv - v0, kT32W);
    x.mat = (int64_t)p.dq * p.dv;
    x.seg_row = p.dv;
    if (p.s_in) x.s_in = p.s_in + q0 * p.s_row + v0 * p.s_col;
    if (p.s_out) x.s_out = p.s_out + q0 * p.s_row + v0 * p.s_col;
    if (p.seg) x.seg = p.seg + q0 * p.dv + v0;
    x.add = qi > 0;
    return x;
}

}  // namespace

bool attn_tc32(const AttnArgs &a, int passes, bool state_only, cudaStream_t s)
{
    auto kern = state_only ? k_attn_tc32<true> : k_attn_tc32<false>;
    const size_t smem = kT32Bytes + 1024;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return false;
    T32Args b = {};
    b.log_decay = a.log_decay, b.lengths = a.lengths;
    b.B = a.B, b.T = a.T, b.H = a.H;
    b.nseg = a.nseg, b.seg_tokens = a.seg_tokens;
    for (int qi = 0; qi * kT32W < kAttnMaxDim; qi++) {
        for (int i = 0; i < passes; i++)
            if (qi * kT32W < a.p[i].dq)
                for (int vi = 0; vi * kT32W < a.p[i].dv; vi++) b.p[b.passes++] = part_of(a.p[i], qi, vi);
        // states alone do not add up: all parts in one launch
        if (b.passes == 0 || (state_only && (qi + 1) * kT32W < kAttnMaxDim)) continue;
        count_launches(1);
        kern<<<(unsigned)(a.B * a.H * a.nseg * b.passes), kT32Threads, smem, s>>>(b, device_status_ptr());
        b.passes = 0;
    }
    return true;
}

}  // namespace lifb
