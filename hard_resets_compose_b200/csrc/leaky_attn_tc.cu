// Leaky attention on the 5th-generation tensor cores: bf16 operands, fp32
// accumulation and fp32 states.  leaky_attn.h has the recurrence; one launch runs
// one to three of its passes.
//
// A block owns one (pass, sequence, head, time segment) and walks its chunks of
// C = 128 tokens (128 = M of the MMA).  With the state S before the chunk, b the
// decay, r the tokens seen before one's own:
//   P  = mask(b^(i-j)) * Q K^T              128 x 128 x dq
//   O  = P V + b^(r+1) * (Q S)              128 x dv x (128 + dq)
//   S <- b^C S + K^T diag(b^(C-1-r)) V      dq x dv x 128
// The powers of b cannot be factored into q and k (b^-128 overflows for strong
// decays), so they are applied where the values are: to P between its two MMAs, to
// Q S in the epilogue, to k before the state's MMA, to S in registers.
//
// Precision: P and S enter their MMAs rounded to bf16, like the inputs are; S
// itself stays in fp32 registers of its warps, one row of the state a thread.  A
// rounded weighted k would put 2^-9 into the fp32 state, so b^(C-1-r) k is split
// into three bf16 pieces (24 bits) that three MMAs add up.
//
// Per chunk and head at dq = dv = 128: 6 x 128^3 multiply-adds (3 of them the
// state's pieces), 3072 cycles of the tensor cores at 4096 a cycle and SM, against
// 128 KB of q, k, v, o: 5500 cycles at 1/148 of 6.46 TB/s.  So memory should bound
// it, if loads, MMAs and the element-wise work overlap:
//   warps 0-3   P: tensor memory -> decay, bf16 -> tensor memory (A operand of P V);
//               O: the epilogue to global memory.  A thread owns a token.
//   4 or 8 more k's three pieces in shared memory (the first in k's place), then the
//               state: registers += MMA result, its bf16 copy to shared memory.
//   one warp    TMA loads: k two chunks deep, q and v reloaded as their MMAs end.
//   one warp    issues all MMAs.
// Every wait is bounded (status 101).
#include <algorithm>

#include "leaky_attn.h"
#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "seq_types.cuh"
#include "tc.cuh"

namespace lifb {

namespace {

constexpr int kTcC = 128;           // tokens of a chunk
constexpr int kTcBlock = kTcC * 128;  // bytes of 128 rows of 64 bf16

struct AttnMaps {
    CUtensorMap q[kAttnMaxPasses], k[kAttnMaxPasses], v[kAttnMaxPasses];
};

// Shared memory of a block: tiles of 64-column blocks.  What an MMA with fewer
// than 128 rows of A reads past its 64 columns (dq = 64) must lie inside: a piece is
// never the last tile.
template <int DQ, int DV>
struct TcLayout {
    static constexpr uint32_t kQ = DQ / 64 * kTcBlock, kV = DV / 64 * kTcBlock, kS = DV / 64 * DQ * 128;
    static constexpr uint32_t mid = 0, lo = kQ, k = 2 * kQ, q = 4 * kQ, v = 5 * kQ, s = 5 * kQ + kV;
    static constexpr uint32_t bytes = 5 * kQ + kV + kS;
    // columns of tensor memory.  dv = 64: the state's MMA result lies over the half
    // of P's scores that its bf16 form leaves free, so that two blocks share an SM.
    static constexpr uint32_t tmem_cols = DV == 64 ? 256 : 512;
    static constexpr uint32_t o1 = 128, o2 = 128 + DV, ds = 128 + 2 * DV;  // ds: dv = 128 only
    static constexpr int blocks_per_sm = DQ == 64 && DV == 64 ? 2 : 1;
    // warpgroups of the state: where one block has an SM, two, with half of the columns
    // each, so that the state stays in registers (128 a thread at 14 warps)
    static constexpr int state_groups = blocks_per_sm == 1 ? 2 : 1;
    static constexpr int tma_warp = 4 + 4 * state_groups, mma_warp = tma_warp + 1;
    static constexpr int threads = 32 * (mma_warp + 1);
};

struct TcBars {
    uint64_t q_full, q_free, k_full[2], k_free[2], v_full, v_free;
    uint64_t p_full, p_ready, kw_ready, s_ready, s_free, o_full, o_free, ds_full, ds_free, done;
};

}  // namespace

// This thread's row of P: scores from tensor memory, times p_scale * b^distance
// where the other token is not in the future (and is one of the n), else zero;
// packed to bf16 into 64 of the same 128 columns.  Powers of b (pw[i] = b^i) run
// from the diagonal outwards.  Forward passes walk the columns
// downwards and pack into the upper half, backward passes the other way round, so
// that nothing unread is overwritten.
template <bool REV>
__device__ __forceinline__ void attn_scores(uint32_t lane_cols, int warp, int lane, int n, float b16,
                                            const float (&pw)[16], float p_scale)
{
    float d = 0.0f;
    auto col = [&](int s) { return (REV ? s : 7 - s) * 16; };
    uint32_t x[2][16];
    const int first = 2 * (REV ? warp : 3 - warp);  // before it all columns are on the other side of the diagonal
    tmem_load16(lane_cols + col(first), x[0]);
    {
        const uint32_t zero[8] = {};
        for (int s = 0; s < first; s++) tmem_store8(lane_cols + (REV ? 0 : 64) + col(s) / 2, zero);
    }
    // the pair of column blocks with the diagonal, then the ones past it
#pragma unroll
    for (int half = 0; half < 2; half++) {
        tmem_wait_ld();
        if (half == 0) tmem_load16(lane_cols + col(first + 1), x[1]);
        else if (first < 6) tmem_load16(lane_cols + col(first + 2), x[0]);
        uint32_t w[8];
        float y[16];
#pragma unroll
        for (int t = 0; t < 16; t++) {
            const int e = REV ? t : 15 - t, c = (REV ? half : 1 - half) * 16 + e;  // of the pair's 32 columns
            d = c == lane ? p_scale : d * pw[1];
            y[e] = (REV ? c >= lane : c <= lane) ? __uint_as_float(x[half][e]) * d : 0.0f;
            if (REV && warp * 32 + c >= n) y[e] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = pack_bf16(y[2 * i], y[2 * i + 1]);
        tmem_store8(lane_cols + (REV ? 0 : 64) + col(first + half) / 2, w);
    }
    d *= pw[1];  // of the next block's nearest column
#pragma unroll 1
    for (int s = first + 2; s < 8; s += 2) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            tmem_wait_ld();
            if (half == 0) tmem_load16(lane_cols + col(s + 1), x[1]);
            else if (s < 6) tmem_load16(lane_cols + col(s + 2), x[0]);
            uint32_t w[8];
            float y[16];
#pragma unroll
            for (int t = 0; t < 16; t++) {
                const int e = REV ? t : 15 - t;
                y[e] = __uint_as_float(x[half][e]) * (d * pw[t]);
                if (REV && n < kTcC && col(s + half) + e >= n) y[e] = 0.0f;
            }
            d *= b16;
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = pack_bf16(y[2 * i], y[2 * i + 1]);
            tmem_store8(lane_cols + (REV ? 0 : 64) + col(s + half) / 2, w);
        }
    }
    tmem_wait_st();
}

// A 4 x 4 transposition of 16-byte elements among the four lanes of a quad:
// m[i] of lane j becomes m[j] of lane i.
__device__ __forceinline__ void quad_transpose(uint32_t (&m)[4][4], int lane)
{
#pragma unroll
    for (int step = 1; step <= 2; step *= 2) {
        const bool up = lane & step;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i & step) continue;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t send = up ? m[i][e] : m[i + step][e];
                const uint32_t got = __shfl_xor_sync(~0u, send, step);
                if (up) m[i][e] = got;
                else m[i + step][e] = got;
            }
        }
    }
}

template <int DQ, int DV, bool STATE_ONLY>
__global__ void __launch_bounds__((TcLayout<DQ, DV>::threads), (TcLayout<DQ, DV>::blocks_per_sm))
    k_attn_tc(const __grid_constant__ AttnArgs a, const __grid_constant__ AttnMaps maps, int *status)
{
    using L = TcLayout<DQ, DV>;
    extern __shared__ unsigned char tc_raw[];
    unsigned char *base = (unsigned char *)(((uintptr_t)tc_raw + 1023) & ~(uintptr_t)1023);
    __shared__ TcBars bars;
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pi = blockIdx.y;
    const AttnPass &p = a.p[pi];
    const int64_t bh = blockIdx.x / a.nseg;
    const int u = (int)(blockIdx.x - bh * a.nseg);  // in the order of the pass
    if (STATE_ONLY && u == a.nseg - 1) return;      // nothing starts from the last one
    const int64_t b = bh / a.H, h = bh - b * a.H;
    const int64_t len = attn_length(a.lengths, b, a.T);
    const float ld = a.log_decay[h];
    const int64_t seg = p.rev ? a.nseg - 1 - u : u;  // in time
    const int64_t s0 = seg * a.seg_tokens, s1 = min(a.T, s0 + a.seg_tokens);
    const int chunks = (int)(max((int64_t)0, min(s1, len) - s0 + kTcC - 1) / kTcC);  // with tokens in them
    auto first_token = [&](int c) { return s0 + (int64_t)(p.rev ? chunks - 1 - c : c) * kTcC; };
    auto tokens = [&](int64_t t0) { return (int)min((int64_t)kTcC, min(s1, len) - t0); };

    if (warp == L::mma_warp) tmem_alloc(&tmem_slot, L::tmem_cols);
    if (tid == 0) {
        mbar_init(&bars.q_full, 1);
        mbar_init(&bars.q_free, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.k_full[i], 1);
            mbar_init(&bars.k_free[i], 1);
        }
        mbar_init(&bars.v_full, 1);
        mbar_init(&bars.v_free, 1);
        mbar_init(&bars.p_full, 1);
        mbar_init(&bars.p_ready, 128);
        mbar_init(&bars.kw_ready, 128 * L::state_groups);
        mbar_init(&bars.s_ready, 128 * L::state_groups);
        mbar_init(&bars.s_free, 1);
        mbar_init(&bars.o_full, 1);
        mbar_init(&bars.o_free, 128);
        mbar_init(&bars.ds_full, 1);
        mbar_init(&bars.ds_free, 128 * L::state_groups);
        mbar_init(&bars.done, 1);
        fence_barrier_init();
    }
    tcgen05_before();
    __syncthreads();
    tcgen05_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t ds_cols = tmem + (DV == 64 ? (p.rev ? 64u : 0u) : L::ds);
    // bounded waits; a role that gives up ends, and the others then run out of theirs
    auto wait = [&](uint64_t *bar, uint32_t phase) {  // one thread's
        if (mbar_wait(bar, phase & 1)) return true;
        atomicExch(status, kStatusTmaWaitTimeout);
        return false;
    };
    auto wait_warp = [&](uint64_t *bar, uint32_t phase) {  // a whole warp's, one decision for it
        if (__all_sync(~0u, mbar_wait(bar, phase & 1))) return true;
        atomicExch(status, kStatusTmaWaitTimeout);
        return false;
    };

    if (warp == L::tma_warp) {
        // ---- loads
        if (lane == 0) {
            prefetch_tmap(&maps.k[pi]);
            prefetch_tmap(&maps.v[pi]);
            if (!STATE_ONLY) prefetch_tmap(&maps.q[pi]);
            const int hq = (int)(h / p.qg), hk = (int)(h / p.kg), hv = (int)(h / p.vg), ib = (int)b;
            auto load = [&](const CUtensorMap *m, uint32_t at, int blocks, int64_t t0, int head, uint64_t *bar) {
                mbar_arrive_expect_tx(bar, blocks * kTcBlock);
                for (int i = 0; i < blocks; i++)
                    tma_load_4d(base + at + i * kTcBlock, m, i * 64, (int)t0, head, ib, bar);
            };
            auto load_k = [&](int c) {
                load(&maps.k[pi], L::k + (c & 1) * L::kQ, DQ / 64, first_token(c), hk, &bars.k_full[c & 1]);
            };
            int nk = 0, nq = 0, nv = 0;  // loads issued
            if (chunks > 0) load_k(nk++);
            for (int c = 0; c < chunks; c++) {
                if (!STATE_ONLY) {
                    if (c > 0 && !wait(&bars.q_free, c - 1)) break;
                    load(&maps.q[pi], L::q, DQ / 64, first_token(c), hq, &bars.q_full);
                    nq++;
                }
                if (c > 0 && !wait(&bars.v_free, c - 1)) break;
                load(&maps.v[pi], L::v, DV / 64, first_token(c), hv, &bars.v_full);
                nv++;
                if (c + 1 < chunks) {
                    if (c > 0 && !wait(&bars.k_free[(c + 1) & 1], (c - 1) >> 1)) break;
                    load_k(nk++);
                }
            }
            // no copy is left in flight, whatever happened
            if (nq > 0) mbar_wait(&bars.q_full, (nq - 1) & 1);
            if (nv > 0) mbar_wait(&bars.v_full, (nv - 1) & 1);
            for (int i = std::max(0, nk - 2); i < nk; i++) mbar_wait(&bars.k_full[i & 1], (i >> 1) & 1);
        }
    } else if (warp == L::mma_warp) {
        // ---- MMAs
        if (lane == 0) {
            const uint32_t sb = smem_u32(base);
            constexpr uint32_t kIdP = umma_idesc_bf16(kTcC, kTcC, false, false);
            constexpr uint32_t kIdO = umma_idesc_bf16(kTcC, DV, false, true);
            constexpr uint32_t kIdS = umma_idesc_bf16(kTcC, DV, true, true);
            const uint32_t pb_cols = tmem + (p.rev ? 0u : 64u);  // P in bf16
            int c = 0;
            for (; c < chunks; c++) {
                const uint32_t k_at = sb + L::k + (c & 1) * L::kQ;
                const bool tail = tokens(first_token(c)) < kTcC;
                if (!STATE_ONLY) {
                    if (!wait(&bars.q_full, c) || !wait(&bars.k_full[c & 1], c >> 1)) break;
                    // P's columns: the last chunk's P V has read them, and (dv = 64) its state's result is out
                    if (c > 0 && !wait(&bars.o_full, c - 1)) break;
                    if (DV == 64 && c > 0 && !wait(&bars.ds_free, c - 1)) break;
                    tcgen05_after();
#pragma unroll
                    for (int k = 0; k < DQ / 16; k++) {
                        const uint32_t off = (k / 4) * kTcBlock + (k % 4) * 32;
                        umma_bf16_ss(tmem, umma_desc_sw128(sb + L::q + off, 16), umma_desc_sw128(k_at + off, 16), kIdP,
                                     k > 0);
                    }
                    umma_arrive(&bars.p_full);
                    if (!wait(&bars.s_ready, c)) break;
                    if (c > 0 && !wait(&bars.o_free, c - 1)) break;
                    tcgen05_after();
#pragma unroll
                    for (int k = 0; k < DQ / 16; k++)
                        umma_bf16_ss(tmem + L::o2, umma_desc_sw128(sb + L::q + (k / 4) * kTcBlock + (k % 4) * 32, 16),
                                     umma_desc_sw128(sb + L::s + k * 2048, DQ * 128), kIdO, k > 0);
                    umma_arrive(&bars.q_free);
                    umma_arrive(&bars.s_free);
                    if (!wait(&bars.v_full, c) || !wait(&bars.p_ready, c)) break;
                    if (tail && !wait(&bars.kw_ready, c)) break;  // v's rows past the end are cleared there
                    tcgen05_after();
#pragma unroll
                    for (int k = 0; k < kTcC / 16; k++)
                        umma_bf16_ts(tmem + L::o1, pb_cols + k * 8, umma_desc_sw128(sb + L::v + k * 2048, kTcBlock),
                                     kIdO, k > 0);
                    umma_arrive(&bars.o_full);
                } else {
                    if (!wait(&bars.v_full, c)) break;
                }
                if (!wait(&bars.kw_ready, c)) break;
                if ((STATE_ONLY || DV != 64) && c > 0 && !wait(&bars.ds_free, c - 1)) break;
                tcgen05_after();
#pragma unroll
                for (int piece = 0; piece < 3; piece++) {
                    const uint32_t at = piece == 0 ? k_at : sb + (piece == 1 ? L::mid : L::lo);
#pragma unroll
                    for (int k = 0; k < kTcC / 16; k++)
                        umma_bf16_ss(ds_cols, umma_desc_sw128(at + k * 2048, kTcBlock),
                                     umma_desc_sw128(sb + L::v + k * 2048, kTcBlock), kIdS, piece > 0 || k > 0);
                }
                umma_arrive(&bars.ds_full);
                umma_arrive(&bars.v_free);
                umma_arrive(&bars.k_free[c & 1]);
            }
            if (c > 0 || chunks > 0) {  // nothing of the tensor cores is left running
                umma_arrive(&bars.done);
                mbar_wait(&bars.done, 0);
            }
        }
    } else if (warp < 4) {
        // ---- P and O: one token a thread
        if (!STATE_ONLY) {
            const uint32_t lanes = (uint32_t)(warp * 32) << 16;
            const int row = warp * 32 + lane;
            float pw[16];
            pw[0] = 1.0f;
            pw[1] = decay_pow(ld, 1.0f);
#pragma unroll
            for (int i = 2; i < 16; i++) pw[i] = pw[i / 2] * pw[i - i / 2];
            const float b16 = pw[8] * pw[8];
            const int64_t o_at = b * p.os[0] + h * p.os[2];
            for (int c = 0; c < chunks; c++) {
                const int64_t t0 = first_token(c);
                const int n = tokens(t0);
                if (!wait_warp(&bars.p_full, c)) break;
                tcgen05_after();
                if (p.rev) attn_scores<true>(tmem + lanes, warp, lane, n, b16, pw, p.p_scale);
                else attn_scores<false>(tmem + lanes, warp, lane, n, b16, pw, p.p_scale);
                tcgen05_before();
                mbar_arrive(&bars.p_ready);

                const int r = p.rev ? n - 1 - row : row;
                const float w = row < n ? p.i_scale * decay_pow(ld, (float)(r + 1 - p.shift)) : 0.0f;
                if (!wait_warp(&bars.o_full, c)) break;
                tcgen05_after();
                const bool in = t0 + row < s1;
                const int64_t at = o_at + (t0 + row) * p.os[1];
#pragma unroll 1
                for (int g = 0; g < DV / 32; g++) {
                    uint32_t x[32], y[2][16];
                    tmem_load32(tmem + lanes + L::o1 + g * 32, x);
                    tmem_load16(tmem + lanes + L::o2 + g * 32, y[0]);
                    tmem_load16(tmem + lanes + L::o2 + g * 32 + 16, y[1]);
                    tmem_wait_ld();
                    if (g == DV / 32 - 1) {
                        tcgen05_before();
                        mbar_arrive(&bars.o_free);
                    }
                    float o[32];
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        o[e] = row < n ? fmaf(w, __uint_as_float(y[e / 16][e % 16]), __uint_as_float(x[e])) : 0.0f;
                    if (in && p.o_f32) {
                        float *dst = (float *)p.o + at + g * 32;
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            if (g * 32 + e < p.dv)
                                *reinterpret_cast<float4 *>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    } else if (!p.o_f32) {
                        // four lanes hold four rows of 64 bytes: transposed among them, so that they
                        // write 64 consecutive bytes of one row at a time
                        uint32_t m[4][4];
#pragma unroll
                        for (int e = 0; e < 16; e++) m[e / 4][e % 4] = pack_bf16(o[2 * e], o[2 * e + 1]);
                        quad_transpose(m, lane);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int r4 = (row & ~3) + i, col = g * 32 + (lane & 3) * 8;
                            if (t0 + r4 < s1 && col < p.dv)
                                *reinterpret_cast<uint4 *>((__nv_bfloat16 *)p.o + o_at + (t0 + r4) * p.os[1] + col) =
                                    make_uint4(m[i][0], m[i][1], m[i][2], m[i][3]);
                        }
                    }
                    __syncwarp();
                }
            }
            // tokens past the sequence's end in chunks that have none of it
            const int64_t z0 = s0 + (int64_t)chunks * kTcC, nz = max((int64_t)0, s1 - z0) * (p.dv / 8);
            for (int64_t i = tid; i < nz; i += 128) {
                const int64_t r = i / (p.dv / 8), at = o_at + (z0 + r) * p.os[1] + (i - r * (p.dv / 8)) * 8;
                if (p.o_f32) {
                    *reinterpret_cast<float4 *>((float *)p.o + at) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    *reinterpret_cast<float4 *>((float *)p.o + at + 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                } else {
                    *reinterpret_cast<uint4 *>((__nv_bfloat16 *)p.o + at) = make_uint4(0, 0, 0, 0);
                }
            }
        }
    } else {
        // ---- k's pieces and the state: one row of the state a thread, SC of its columns
        constexpr int NB = L::state_groups, SC = DV / NB;
        const int at = tid - 128, st = at & 127, c0 = (at >> 7) * SC;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const bool has_row = st < DQ;  // uniform over a warp
        float S[SC];
        const int64_t mat = (int64_t)p.dq * p.dv;
        {
            const float *s_in = nullptr;
            int64_t row = p.s_row, col = p.s_col;
            if (!STATE_ONLY) {
                if (u == 0) {
                    if (p.s_in) s_in = p.s_in + bh * mat;
                } else {
                    s_in = p.seg + (bh * a.nseg + u) * mat;
                    row = p.dv;
                    col = 1;
                }
            }
#pragma unroll
            for (int j = 0; j < SC; j++)
                S[j] = s_in && st < p.dq && c0 + j < p.dv ? s_in[st * row + (c0 + j) * col] : 0.0f;
        }
        auto put_state = [&] {  // its bf16 copy, the B operand of Q S
            if (has_row) {
#pragma unroll
                for (int j = 0; j < SC; j += 8) {
                    const int col = c0 + j;
                    *reinterpret_cast<uint4 *>(base + L::s + (col / 64) * (DQ * 128) + st * 128 +
                                               (((col % 64) / 8) ^ (st & 7)) * 16) =
                        make_uint4(pack_bf16(S[j], S[j + 1]), pack_bf16(S[j + 2], S[j + 3]),
                                   pack_bf16(S[j + 4], S[j + 5]), pack_bf16(S[j + 6], S[j + 7]));
                }
            }
            fence_proxy_async_shared();
            mbar_arrive(&bars.s_ready);
        };
        if (!STATE_ONLY && chunks > 0) put_state();
        const DecayFactor full(ld, kTcC);
        // the weights of the tokens whose columns this thread scales
        constexpr int NW = 8 / NB;
        float wk[NW];
        int wn = -1;  // the chunk size that they are for
        for (int c = 0; c < chunks; c++) {
            const int64_t t0 = first_token(c);
            const int n = tokens(t0);
            if (n != wn) {  // the first chunk, the one with the sequence's end, and the one after it
#pragma unroll
                for (int i = 0; i < NW; i++) {
                    const int row = at / 8 + 16 * NB * i, r = p.rev ? n - 1 - row : row;
                    wk[i] = row < n ? p.w_scale * decay_pow(ld, (float)(n - 1 - r + p.shift)) : 0.0f;
                }
                wn = n;
            }
            if (!wait_warp(&bars.k_full[c & 1], c >> 1)) break;
            if (!STATE_ONLY && !wait_warp(&bars.p_full, c)) break;  // Q K^T has read k
            if (t0 + n < min(t0 + kTcC, a.T)) {
                // what lies past the end may be anything: a zero weight does not remove it from v
                if (!wait_warp(&bars.v_full, c)) break;
                uint4 *v4 = reinterpret_cast<uint4 *>(base + L::v);
                for (int i = at; i < (int)L::kV / 16; i += 128 * NB)
                    if (i / 8 % kTcC >= n) v4[i] = make_uint4(0, 0, 0, 0);
            }
            uint4 *k4 = reinterpret_cast<uint4 *>(base + L::k + (c & 1) * L::kQ);
            uint4 *mid4 = reinterpret_cast<uint4 *>(base + L::mid), *lo4 = reinterpret_cast<uint4 *>(base + L::lo);
#pragma unroll 1
            for (int blk = 0; blk < DQ / 64; blk++) {
                // four loads first: a thread's vectors do not depend on one another
                const int i0 = blk * (kTcBlock / 16) + at;  // rows at / 8 + 16 NB it
#pragma unroll
                for (int j = 0; j < NW; j += 4) {
                uint4 x[4];
#pragma unroll
                for (int it = 0; it < 4; it++) x[it] = k4[i0 + (j + it) * 128 * NB];
#pragma unroll
                for (int it = 0; it < 4; it++) {
                    const int i = i0 + (j + it) * 128 * NB;
                    const float w = wk[j + it];
                    const bool zero = at / 8 + 16 * NB * (j + it) >= n;
                    uint32_t in[4] = {x[it].x, x[it].y, x[it].z, x[it].w}, hi[4], mid[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float f0 = zero ? 0.0f : bf16_lo(in[e]) * w, f1 = zero ? 0.0f : bf16_hi(in[e]) * w;
                        hi[e] = pack_bf16(f0, f1);
                        const float g0 = f0 - bf16_lo(hi[e]), g1 = f1 - bf16_hi(hi[e]);
                        mid[e] = pack_bf16(g0, g1);
                        lo[e] = pack_bf16(g0 - bf16_lo(mid[e]), g1 - bf16_hi(mid[e]));
                    }
                    k4[i] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    mid4[i] = make_uint4(mid[0], mid[1], mid[2], mid[3]);
                    lo4[i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                }
            }
            fence_proxy_async_shared();
            mbar_arrive(&bars.kw_ready);

            float bn_hi = full.hi, bn_lo = full.lo;
            if (n != kTcC) {
                const DecayFactor f(ld, n);
                bn_hi = f.hi;
                bn_lo = f.lo;
            }
            if (!wait_warp(&bars.ds_full, c)) break;
            tcgen05_after();
            if (has_row) {
#pragma unroll
                for (int g = 0; g < SC / 32; g++) {
                    uint32_t x[32];
                    tmem_load32(ds_cols + lanes + c0 + g * 32, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 32; e++) {
                        float &z = S[g * 32 + e];
                        z = fmaf(z, bn_hi, fmaf(z, bn_lo, __uint_as_float(x[e])));
                    }
                }
            }
            tcgen05_before();
            mbar_arrive(&bars.ds_free);
            if (!STATE_ONLY && c + 1 < chunks) {
                if (!wait_warp(&bars.s_free, c)) break;
                put_state();
            }
        }
        float *s_out = nullptr;
        int64_t row = p.dv, col = 1;
        if (STATE_ONLY) {
            s_out = p.seg + (bh * a.nseg + u + 1) * mat;
        } else if (u == a.nseg - 1 && p.s_out) {
            s_out = p.s_out + bh * mat;
            row = p.s_row;
            col = p.s_col;
        }
        if (s_out && st < p.dq) {
#pragma unroll
            for (int j = 0; j < SC; j++)
                if (c0 + j < p.dv) s_out[st * row + (c0 + j) * col] = S[j];
        }
    }
    tcgen05_before();
    __syncthreads();
    if (warp == L::mma_warp) {
        tcgen05_after();
        tmem_free(tmem, L::tmem_cols);
    }
}

namespace {

int width_class(int d) { return d <= 64 ? 64 : 128; }

bool operand_map(CUtensorMap *m, const void *base, const int64_t (&st)[3], int d, int64_t T, int64_t heads, int64_t B)
{
    const int64_t dims[4] = {d, T, heads, B}, strides[3] = {st[1], st[2], st[0]};
    return make_tmap_4d_bf16(m, base, dims, strides, 64, kTcC);
}

template <int DQ, int DV>
bool launch_tc(const AttnArgs &a, const AttnMaps &m, int passes, bool state_only, cudaStream_t s)
{
    const size_t smem = TcLayout<DQ, DV>::bytes + 1024;
    auto kern = state_only ? k_attn_tc<DQ, DV, true> : k_attn_tc<DQ, DV, false>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return false;
    count_launches(1);
    kern<<<dim3((unsigned)(a.B * a.H * a.nseg), (unsigned)passes), TcLayout<DQ, DV>::threads, smem, s>>>(a, m, device_status_ptr());
    return true;
}

}  // namespace

bool attn_tc_applies(const AttnArgs &a, int passes, int dtype)
{
    if (dtype != LIFB_BF16) return false;
    for (int i = 0; i < passes; i++) {
        const AttnPass &p = a.p[i];
        if (p.dq % 8 || p.dv % 8 || p.dq > kAttnMaxDim || p.dv > kAttnMaxDim || !aligned16(p.o)) return false;
        CUtensorMap m;
        if (!operand_map(&m, p.q, p.qs, p.dq, a.T, a.H / p.qg, a.B) ||
            !operand_map(&m, p.k, p.ks, p.dq, a.T, a.H / p.kg, a.B) ||
            !operand_map(&m, p.v, p.vs, p.dv, a.T, a.H / p.vg, a.B))
            return false;
    }
    return true;
}

int attn_tc_blocks_per_sm(int dq, int dv) { return width_class(dq) == 64 && width_class(dv) == 64 ? 2 : 1; }

bool attn_tc(const AttnArgs &a, int passes, bool state_only, cudaStream_t s)
{
    // passes of one pair of width classes share a launch
    bool launched[kAttnMaxPasses] = {};
    for (int i = 0; i < passes; i++) {
        if (launched[i]) continue;
        const int dq = width_class(a.p[i].dq), dv = width_class(a.p[i].dv);
        AttnArgs b = a;
        AttnMaps m = {};
        int n = 0;
        for (int j = i; j < passes; j++) {
            const AttnPass &p = a.p[j];
            if (launched[j] || width_class(p.dq) != dq || width_class(p.dv) != dv) continue;
            if (!operand_map(&m.q[n], p.q, p.qs, p.dq, a.T, a.H / p.qg, a.B) ||
                !operand_map(&m.k[n], p.k, p.ks, p.dq, a.T, a.H / p.kg, a.B) ||
                !operand_map(&m.v[n], p.v, p.vs, p.dv, a.T, a.H / p.vg, a.B))
                return false;
            launched[j] = true;
            b.p[n++] = p;
        }
        const bool ok = dq == 64 ? (dv == 64 ? launch_tc<64, 64>(b, m, n, state_only, s)
                                             : launch_tc<64, 128>(b, m, n, state_only, s))
                                 : (dv == 64 ? launch_tc<128, 64>(b, m, n, state_only, s)
                                             : launch_tc<128, 128>(b, m, n, state_only, s));
        if (!ok) return false;
    }
    return true;
}

}  // namespace lifb
