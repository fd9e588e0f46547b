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
// Precision: P and S enter their MMAs rounded to bf16, like the inputs are: 2^-9 each, as
// much as the output's own rounding, so that outputs are sqrt(2) times as far off as
// values rounded once (2.4e-3 against 1.7e-3, relative).  Calls of one chunk, and of
// 8192 rows (tokens of heads) or less, use two pieces of each, and their outputs are
// rounded once: roundings of few rows need not average out (one of 130 to 400 tokens and
// one to four heads in a hundred was 1.5 to 1.56 times as far off as one rounding; from
// 8192 rows on none was over 1.44), and such a call's time is mostly latency (B 1, T 1024, H 8,
// 128 x 128: forward 35 -> 37 us, backward 43 -> 45; four of T 256: 12.3 -> 14.4, 12.4 ->
// 16.5).  Two pieces in every call would cost more than half of
// the large ones again (B 8, T 4096, H 16, 128 x 128: 104 -> 164 us and 299 -> 494; 64 x 64 at B 16:
// 132 -> 156 and 443 -> 640).  S itself
// stays in fp32 registers of its warps, one row of the state a thread.  A rounded
// weighted k would put 2^-9 into the fp32 state, so b^(C-1-r) k is split into bf16
// pieces that as many MMAs add up: two (2^-18) where the state only feeds further bf16
// products, three (24 bits) where heads of 64 x 64 return it (wider ones have it from
// leaky_attn_state.cu).
//
// Per chunk and head at dq = dv = 128: q, k, v, o are 128 KB, 4800 cycles of the
// memory that 128 busy SMs share; the MMAs are 5 x 128^3 multiply-adds, 2560 cycles
// at 4096 a cycle and SM, but an MMA with both operands in shared memory reads 8 KB
// in 64 cycles, all that shared memory can give (128 bytes a cycle): with the loads
// and the element-wise writes 512 KB pass through it, 4000 cycles.  So no stage may
// wait for another (measured: with P, k's pieces, O and S done by 12 warps one after
// another 7400 cycles a chunk, spilling states 14000, as below 5200: B 8, T 4096, H 16
// in 103 us, 83 us at the copy rate):
//   scores      P: tensor memory -> decay, bf16 -> tensor memory (A operand of P V).
//               A thread owns a token.  Two warpgroups where heads of 64 x 64 leave
//               tensor memory for two P's, in turn.
//   output      the epilogue to global memory.  A thread owns a token.
//   state       the weighted k's pieces in shared memory, then the state: registers +=
//               MMA result, its bf16 copy to shared memory.  One warpgroup for each 64
//               columns.
//   one warp    TMA loads, as far ahead as there are tiles.
//   one warp    issues all MMAs: the state's, P V, the next Q K^T, Q S.
// Registers are moved from the other warpgroups to the state's (setmaxnreg).  What
// starts a block up (12 us before its first chunk was out, 8 us now) is mostly code
// fetched for the first time, so loops stay rolled where that costs nothing.
// Every wait is bounded (status 101).
#include <algorithm>

#include "leaky_attn_tc.cuh"
#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "seq_types.cuh"

namespace lifb {

namespace {

// Tensor maps of the passes of one launch.
struct AttnMaps {
    CUtensorMap q[kAttnMaxPasses], k[kAttnMaxPasses], v[kAttnMaxPasses];
};

// Shared memory of a block: tiles of 64-column blocks.  What an MMA with fewer
// than 128 rows of A reads past its 64 columns (dq = 64) must lie inside: a piece is
// never the last tile.
template <int DQ, int DV, int NP, bool FINE>
struct TcLayout {
    static constexpr uint32_t kQ = DQ / 64 * kTcBlock, kV = DV / 64 * kTcBlock, kS = DV / 64 * DQ * 128;
    static constexpr bool small = DQ == 64 && DV == 64;
    static constexpr int np = small ? 2 : 1;  // P's in flight, in tensor memory
    // tiles in flight: of q one more than P's, so that the next Q K^T need not wait for Q S
    // (where S's second piece leaves room for it)
    static constexpr int nq = FINE && DQ == 128 && DV == 128 ? np : np + 1, nk = np;
    static constexpr int nv = DQ == 128 && DV == 128 ? 1 : 2, nm = small ? 2 : 1;  // nm: sets of pieces
    static constexpr uint32_t pieces = 0, k = nm * NP * kQ, q = k + nk * kQ, v = q + nq * kQ, s = v + nv * kV,
                              s_fine = s + kS,  // S's second piece
                              bytes = s_fine + (FINE ? kS : 0);
    static_assert(bytes + 1024 + 512 <= 227 * 1024, "tiles fit an SM");
    // columns of tensor memory
    static constexpr uint32_t tmem_cols = 512, o1 = np * 128, o2 = o1 + DV, ds = o2 + DV;
    static_assert(ds + DV <= tmem_cols, "accumulators fit");
    // warpgroups: scores, output, state, and one with the loading and the issuing warp
    static constexpr int score_groups = np, state_groups = DV / 64;
    static constexpr int output_group = score_groups, first_state = score_groups + 1,
                         last_group = first_state + state_groups;
    static constexpr int threads = 640;  // five groups; one of them idles at dq = 128, dv = 64
    // registers a thread: 640 threads are launched with 96 each, 480 for the five groups
    static constexpr int score_regs = 80, output_regs = 80, state_regs = DV == 64 ? 152 : 128, last_regs = 64;
    static constexpr int idle_groups = 5 - (score_groups + 1 + state_groups + 1);
    static_assert(score_groups * score_regs + output_regs + state_groups * state_regs + last_regs + idle_groups * 24 <= 480,
                  "no more registers than the block was launched with");
};

struct TcBars {
    uint64_t q_full[3], q_free[3], k_full[2], k_free[2], v_full[2], v_free[2];
    uint64_t p_full[2], p_ready[2], kw_ready[2], s_ready, s_free, o_full, o_free, ds_full, ds_free, done;
};

}  // namespace

// This thread's row of P: scores from tensor memory, times p_scale * b^distance
// where the other token is not in the future (and is one of the n), else zero;
// packed to bf16 into 64 of the same 128 columns.  Powers of b run from the
// diagonal outwards, a product each (at most 128 of them: 2^-17, below the 2^-16 of two
// pieces) (pw: of 16 columns, in their order).  Forward passes walk the columns
// downwards and pack into the upper half, backward passes the other way round, so
// that nothing unread is overwritten.  FINE: two bf16 pieces (2^-18) in place of one,
// each 16 columns of scores becoming 8 of the first and 8 of the second.
template <bool REV, bool FINE>
__device__ __forceinline__ void attn_scores(uint32_t lane_cols, int warp, int lane, int n, float b, float b16,
                                            const uint64_t (&pw)[8], float p_scale)
{
    float d = 0.0f;
    auto col = [&](int s) { return (REV ? s : 7 - s) * 16; };
    auto out = [&](int s) { return lane_cols + (FINE ? col(s) : (REV ? 0 : 64) + col(s) / 2); };
    uint32_t x[2][16];
    const int first = 2 * (REV ? warp : 3 - warp);  // before it all columns are on the other side of the diagonal
    tmem_load16(lane_cols + col(first), x[0]);
    {
        const uint32_t zero[8] = {};
        for (int s = 0; s < first; s++) {
            tmem_store8(out(s), zero);
            if (FINE) tmem_store8(out(s) + 8, zero);
        }
    }
    // the two column blocks with the diagonal, then the ones past it, two at a time
#pragma unroll 1
    for (int s = first; s < 8; s += 2) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            tmem_wait_ld();
            if (half == 0) tmem_load16(lane_cols + col(s + 1), x[1]);
            else if (s < 6) tmem_load16(lane_cols + col(s + 2), x[0]);
            uint32_t w[8], fine[8];
            auto pack = [&](int i, uint64_t v) {
                w[i] = pack2_bf16(v);
                if (FINE) fine[i] = pack2_bf16(fma2(two(-1.0f, -1.0f), two(bf16_lo(w[i]), bf16_hi(w[i])), v));
            };
            if (s == first) {
#pragma unroll
                for (int t = 0; t < 16; t++) {
                    const int e = REV ? t : 15 - t, c = (REV ? half : 1 - half) * 16 + e;  // of the pair's 32
                    d = c == lane ? p_scale : d * b;
                    const bool on = (REV ? c >= lane : c <= lane) && !(REV && warp * 32 + c >= n);
                    x[half][e] = on ? __float_as_uint(__uint_as_float(x[half][e]) * d) : 0u;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) pack(i, two(x[half][2 * i], x[half][2 * i + 1]));
                if (half == 1) d *= b;  // of the next block's nearest column
            } else {
                const uint64_t dd = two(d, d);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    pack(i, mul2(two(x[half][2 * i], x[half][2 * i + 1]), mul2(pw[i], dd)));
                if (REV && n < kTcC) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const uint32_t on = col(s + half) + 2 * i >= n       ? 0u
                                            : col(s + half) + 2 * i + 1 >= n ? 0xFFFFu
                                                                             : ~0u;
                        w[i] &= on;
                        if (FINE) fine[i] &= on;
                    }
                }
                d *= b16;
            }
            tmem_store8(out(s + half), w);
            if (FINE) tmem_store8(out(s + half) + 8, fine);
        }
    }
    tmem_wait_st();
}

// 32 bytes, a whole sector, in one store.
__device__ __forceinline__ void store_32_bytes(void *p, const uint32_t (&m)[8])
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(m[0]), "r"(m[1]), "r"(m[2]),
                 "r"(m[3]), "r"(m[4]), "r"(m[5]), "r"(m[6]), "r"(m[7])
                 : "memory");
}

// FINE: P and S as two pieces each.
template <int DQ, int DV, int NP, bool FINE>
__global__ void __launch_bounds__((TcLayout<DQ, DV, NP, FINE>::threads), 1)
    k_attn_tc(const __grid_constant__ AttnArgs a, const __grid_constant__ AttnMaps maps, int *status)
{
    using L = TcLayout<DQ, DV, NP, FINE>;
    extern __shared__ unsigned char tc_raw[];
    unsigned char *base = (unsigned char *)(((uintptr_t)tc_raw + 1023) & ~(uintptr_t)1023);
    __shared__ TcBars bars;
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0), group = warp >> 2;
    const int pi = blockIdx.x % a.passes, item = blockIdx.x / a.passes;
    const AttnPass &p = a.p[pi];
    const int64_t bh = item / a.nseg;
    const int u = (int)(item - bh * a.nseg);  // in the order of the pass
    const int64_t b = bh / a.H, h = bh - b * a.H;
    const int64_t len = attn_length(a.lengths, b, a.T);
    const float ld = a.log_decay[h];
    const int64_t seg = p.rev ? a.nseg - 1 - u : u;  // in time
    // T < 2^31 - 2^7: a token's number, and one chunk past the last, fit an int
    const int s0 = (int)(seg * a.seg_tokens), s1 = (int)min(a.T, seg * a.seg_tokens + a.seg_tokens);
    const int end = min(s1, (int)len);                         // of the tokens that count
    const int chunks = max(0, end - s0 + kTcC - 1) / kTcC;     // with tokens in them
    const int t_first = p.rev ? s0 + (chunks - 1) * kTcC : s0, t_step = p.rev ? -kTcC : kTcC;

    if (warp == 0) tmem_alloc(&tmem_slot, L::tmem_cols);
    if (tid == 32) {
        for (int i = 0; i < 3; i++) {
            mbar_init(&bars.q_full[i], 1);
            mbar_init(&bars.q_free[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.k_full[i], 1);
            mbar_init(&bars.k_free[i], 1 + 128 * L::state_groups);
            mbar_init(&bars.v_full[i], 1);
            mbar_init(&bars.v_free[i], 1);
            mbar_init(&bars.p_full[i], 1);
            mbar_init(&bars.p_ready[i], 128);
            mbar_init(&bars.kw_ready[i], 128 * L::state_groups);
        }
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
    const uint32_t tmem = __shfl_sync(~0u, tmem_slot, 0);
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

    if (group == L::last_group) {
        regs_dec<L::last_regs>();
        if ((warp & 3) == 0 && lane == 0) {
            // ---- loads
            prefetch_tmap(&maps.k[pi]);
            prefetch_tmap(&maps.v[pi]);
            prefetch_tmap(&maps.q[pi]);
            const int hq = (int)(h / p.qg), hk = (int)(h / p.kg), hv = (int)(h / p.vg), ib = (int)b;
            // tile c of an operand with N buffers of `bytes` from `at`; false: gave up
            auto load = [&](const CUtensorMap *m, uint32_t at, uint32_t bytes, int N, int c, int head, uint64_t *full,
                            uint64_t *free) {
                const int i = c % N, use = c / N;
                if (use > 0 && !wait(&free[i], use - 1)) return false;
                mbar_arrive_expect_tx(&full[i], bytes);
                for (uint32_t j = 0; j < bytes / kTcBlock; j++)
                    tma_load_4d(base + at + i * bytes + j * kTcBlock, m, j * 64, t_first + c * t_step, head, ib, &full[i]);
                return true;
            };
            int nk = 0, nq = 0, nv = 0;  // loads issued
            for (int c = 0; c < chunks; c++) {
                if (!load(&maps.k[pi], L::k, L::kQ, L::nk, c, hk, bars.k_full, bars.k_free)) break;
                nk++;
                if (L::nq > L::np) {
                    if (!load(&maps.q[pi], L::q, L::kQ, L::nq, c, hq, bars.q_full, bars.q_free)) break;
                    nq++;
                }
                if (!load(&maps.v[pi], L::v, L::kV, L::nv, c, hv, bars.v_full, bars.v_free)) break;
                nv++;
                if (L::nq == L::np) {  // its tile is the last to be free
                    if (!load(&maps.q[pi], L::q, L::kQ, L::nq, c, hq, bars.q_full, bars.q_free)) break;
                    nq++;
                }
            }
            // no copy is left in flight, whatever happened
            for (int c = max(0, nk - L::nk); c < nk; c++) mbar_wait(&bars.k_full[c % L::nk], (c / L::nk) & 1);
            for (int c = max(0, nq - L::nq); c < nq; c++) mbar_wait(&bars.q_full[c % L::nq], (c / L::nq) & 1);
            for (int c = max(0, nv - L::nv); c < nv; c++) mbar_wait(&bars.v_full[c % L::nv], (c / L::nv) & 1);
        } else if ((warp & 3) == 1) {
            // ---- MMAs: the warp together, one lane issues
            const uint32_t sb = smem_u32(base);
            constexpr uint32_t kIdP = umma_idesc_bf16(kTcC, kTcC, false, false);
            constexpr uint32_t kIdO = umma_idesc_bf16(kTcC, DV, false, true);
            constexpr uint32_t kIdS = umma_idesc_bf16(kTcC, DV, true, true);
            auto p_cols = [&](int c) { return tmem + (c % L::np) * 128; };
            auto scores = [&](int c) {  // Q K^T; its columns are free
                if (!wait_warp(&bars.q_full[c % L::nq], c / L::nq)) return false;
                if (!wait_warp(&bars.k_full[c % L::nk], c / L::nk)) return false;
                tcgen05_after();
                const uint64_t dq = umma_desc_sw128(sb + L::q + (c % L::nq) * L::kQ, 16);
                const uint64_t dk = umma_desc_sw128(sb + L::k + (c % L::nk) * L::kQ, 16);
                if (elect_lane()) {
#pragma unroll
                    for (int k = 0; k < DQ / 16; k++) {
                        const uint32_t off = ((k / 4) * kTcBlock + (k % 4) * 32) >> 4;
                        umma_bf16_ss(p_cols(c), dq + off, dk + off, kIdP, k > 0);
                    }
                    umma_arrive(&bars.p_full[c % L::np]);
                    umma_arrive(&bars.k_free[c % L::nk]);
                }
                return true;
            };
            auto carried = [&](int c) {  // Q S
                if (!wait_warp(&bars.s_ready, c)) return false;
                tcgen05_after();
                const uint64_t dq = umma_desc_sw128(sb + L::q + (c % L::nq) * L::kQ, 16);
                const uint64_t ds = umma_desc_sw128(sb + L::s, DQ * 128);
                if (elect_lane()) {
#pragma unroll
                    for (int k = 0; k < DQ / 16; k++)
                        umma_bf16_ss(tmem + L::o2, dq + (((k / 4) * kTcBlock + (k % 4) * 32) >> 4), ds + k * 128, kIdO,
                                     k > 0);
                    if constexpr (FINE) {
                        const uint64_t lo = umma_desc_sw128(sb + L::s_fine, DQ * 128);
#pragma unroll 1
                        for (int k = 0; k < DQ / 16; k++)
                            umma_bf16_ss(tmem + L::o2, dq + (((k / 4) * kTcBlock + (k % 4) * 32) >> 4), lo + k * 128,
                                         kIdO, true);
                    }
                    umma_arrive(&bars.q_free[c % L::nq]);
                    umma_arrive(&bars.s_free);
                    umma_arrive(&bars.o_full);
                }
                return true;
            };
            auto body = [&](int c) {
                const uint64_t dv = umma_desc_sw128(sb + L::v + (c % L::nv) * L::kV, kTcBlock);
                if (!wait_warp(&bars.v_full[c % L::nv], c / L::nv)) return false;
                if (!wait_warp(&bars.kw_ready[c % L::nm], c / L::nm)) return false;
                if (c > 0 && !wait_warp(&bars.ds_free, c - 1)) return false;
                tcgen05_after();
                if (elect_lane()) {
#pragma unroll 1
                    for (int piece = 0; piece < NP; piece++) {
                        const uint64_t dk = umma_desc_sw128(sb + L::pieces + ((c % L::nm) * NP + piece) * L::kQ, kTcBlock);
#pragma unroll
                        for (int k = 0; k < kTcC / 16; k++)
                            umma_bf16_ss(tmem + L::ds, dk + k * 128, dv + k * 128, kIdS, piece > 0 || k > 0);
                    }
                    umma_arrive(&bars.ds_full);
                }
                if (!wait_warp(&bars.p_ready[c % L::np], c / L::np)) return false;
                if (c > 0 && !wait_warp(&bars.o_free, c - 1)) return false;
                tcgen05_after();
                const uint32_t pb = p_cols(c) + (p.rev ? 0u : 64u);  // P in bf16
                if (elect_lane()) {
                    if constexpr (FINE) {
#pragma unroll 1
                        for (int k = 0; k < kTcC / 8; k++)
                            umma_bf16_ts(tmem + L::o1, p_cols(c) + k * 8, dv + k / 2 * 128, kIdO, k > 0);
                    } else {
#pragma unroll
                        for (int k = 0; k < kTcC / 16; k++)
                            umma_bf16_ts(tmem + L::o1, pb + k * 8, dv + k * 128, kIdO, k > 0);
                    }
                    umma_arrive(&bars.v_free[c % L::nv]);
                }
                if (L::nq == L::np && !carried(c)) return false;  // the next q comes into this one's tile
                if (c + L::np < chunks) {
                    // P V is done: P's columns are free
                    if (!wait_warp(&bars.v_free[c % L::nv], c / L::nv)) return false;
                    if (!scores(c + L::np)) return false;
                }
                return L::nq == L::np || carried(c);
            };
            bool ok = true;
            for (int c = 0; ok && c < L::np && c < chunks; c++) ok = scores(c);
            for (int c = 0; ok && c < chunks; c++) ok = body(c);
            if (elect_lane()) {  // nothing of the tensor cores is left running
                umma_arrive(&bars.done);
                mbar_wait(&bars.done, 0);
            }
        }
    } else if (group < L::score_groups) {
        // ---- P: one token a thread
        regs_dec<L::score_regs>();
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float b1 = decay_pow(ld, 1.0f);
        uint64_t pw[8];
        float b16 = 1.0f;
        {
            float f[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                f[i] = b16;
                b16 *= b1;
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
                pw[i] = p.rev ? two(f[2 * i], f[2 * i + 1]) : two(f[15 - 2 * i], f[14 - 2 * i]);
        }
        for (int c = group; c < chunks; c += L::np) {
            const int n = min(kTcC, end - (t_first + c * t_step));
            if (!wait_warp(&bars.p_full[group], c / L::np)) break;
            tcgen05_after();
            const uint32_t cols = tmem + lanes + group * 128;
            if (p.rev) attn_scores<true, FINE>(cols, warp & 3, lane, n, b1, b16, pw, p.p_scale);
            else attn_scores<false, FINE>(cols, warp & 3, lane, n, b1, b16, pw, p.p_scale);
            tcgen05_before();
            mbar_arrive(&bars.p_ready[group]);
        }
    } else if (group == L::output_group) {
        // ---- O: one token a thread
        regs_dec<L::output_regs>();
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const int row = tid & 127;
        const int64_t o_at = b * p.os[0] + h * p.os[2];
        const bool sectors = p.dv % 16 == 0 && (uintptr_t)p.o % 32 == 0;  // rows of whole 32-byte sectors
        for (int c = 0; c < chunks; c++) {
            const int t0 = t_first + c * t_step, n = min(kTcC, end - t0);
            const int r = p.rev ? n - 1 - row : row;
            const float w = row < n ? p.i_scale * decay_pow(ld, (float)(r + 1 - p.shift)) : 0.0f;
            if (!wait_warp(&bars.o_full, c)) break;
            tcgen05_after();
            const uint64_t ww = two(w, w);
            char *o_row = (char *)p.o + (o_at + (int64_t)(t0 + row) * p.os[1]) * (p.o_f32 ? 4 : 2);
#pragma unroll 1
            for (int g = 0; g < DV; g += 32) {
                uint32_t x[32], y[32];
                tmem_load32(tmem + lanes + L::o1 + g, x);
                tmem_load32(tmem + lanes + L::o2 + g, y);
                tmem_wait_ld();
                if (g == DV - 32) {
                    tcgen05_before();
                    mbar_arrive(&bars.o_free);
                }
                uint64_t o[16];
#pragma unroll
                for (int e = 0; e < 16; e++)
                    o[e] = fma2(ww, two(y[2 * e], y[2 * e + 1]), two(x[2 * e], x[2 * e + 1]));
                if (row >= n) {
#pragma unroll
                    for (int e = 0; e < 16; e++) o[e] = 0;
                }
                if (t0 + row < s1) {
                    if (!p.o_f32) {
                        __nv_bfloat16 *dst = (__nv_bfloat16 *)o_row + g;
#pragma unroll
                        for (int e = 0; e < 16; e += 8) {
                            const uint32_t m[8] = {pack2_bf16(o[e]),     pack2_bf16(o[e + 1]), pack2_bf16(o[e + 2]),
                                                   pack2_bf16(o[e + 3]), pack2_bf16(o[e + 4]), pack2_bf16(o[e + 5]),
                                                   pack2_bf16(o[e + 6]), pack2_bf16(o[e + 7])};
                            if (sectors && g + 2 * e < p.dv) {
                                store_32_bytes(dst + 2 * e, m);
                            } else {
                                if (g + 2 * e < p.dv)
                                    *reinterpret_cast<uint4 *>(dst + 2 * e) = make_uint4(m[0], m[1], m[2], m[3]);
                                if (g + 2 * e + 8 < p.dv)
                                    *reinterpret_cast<uint4 *>(dst + 2 * e + 8) = make_uint4(m[4], m[5], m[6], m[7]);
                            }
                        }
                    } else {
                        float *dst = (float *)o_row + g;
#pragma unroll
                        for (int e = 0; e < 16; e += 2)
                            if (g + 2 * e < p.dv)
                                *reinterpret_cast<ulonglong2 *>(dst + 2 * e) = make_ulonglong2(o[e], o[e + 1]);
                    }
                }
                __syncwarp();
            }
        }
        // tokens past the sequence's end in chunks that have none of it
        const int z0 = s0 + chunks * kTcC;
        const int64_t nz = (int64_t)max(0, s1 - z0) * (p.dv / 8);
        for (int64_t i = row; i < nz; i += 128) {
            const int64_t r = i / (p.dv / 8), at = o_at + (z0 + r) * p.os[1] + (i - r * (p.dv / 8)) * 8;
            if (p.o_f32) {
                *reinterpret_cast<float4 *>((float *)p.o + at) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                *reinterpret_cast<float4 *>((float *)p.o + at + 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            } else {
                *reinterpret_cast<uint4 *>((__nv_bfloat16 *)p.o + at) = make_uint4(0, 0, 0, 0);
            }
        }
    } else if (group < L::last_group) {
        // ---- k's pieces and the state: one row of the state a thread, 64 of its columns
        regs_inc<L::state_regs>();
        constexpr int NB = L::state_groups, SC = 64;
        const int at = tid - L::first_state * 128, st = at & 127, c0 = (at >> 7) * SC;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const bool has_row = st < DQ;  // uniform over a warp
        uint64_t S[SC / 2];  // pairs of columns
        const int64_t mat = (int64_t)p.dq * p.dv;
        {
            const float *s_in = nullptr;
            int64_t row = p.s_row, col = p.s_col;
            if (u == 0) {
                if (p.s_in) s_in = p.s_in + bh * mat;
            } else {
                s_in = p.seg + (bh * (a.nseg + 1) + u) * mat;
                row = p.dv;
                col = 1;
            }
#pragma unroll
            for (int j = 0; j < SC / 2; j++) S[j] = 0;
            // (a branch, not a condition of each load: what is not there is not fetched either)
            if (s_in && st < p.dq) {
                s_in += st * row + c0 * col;
#pragma unroll
                for (int j = 0; j < SC; j += 2)
                    if (c0 + j < p.dv) S[j / 2] = two(s_in[j * col], s_in[(j + 1) * col]);
            }
        }
        auto put_state = [&] {  // its bf16 copy, the B operand of Q S
            if (has_row) {
                const uint32_t row = (at >> 7) * (DQ * 128) + st * 128;
#pragma unroll
                for (int j = 0; j < SC; j += 8)
                    *reinterpret_cast<uint4 *>(base + L::s + row + ((j / 8) ^ (st & 7)) * 16) =
                        make_uint4(pack2_bf16(S[j / 2]), pack2_bf16(S[j / 2 + 1]), pack2_bf16(S[j / 2 + 2]),
                                   pack2_bf16(S[j / 2 + 3]));
                if constexpr (FINE) {  // what the copy dropped
#pragma unroll
                    for (int j = 0; j < SC; j += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t m = pack2_bf16(S[j / 2 + i]);
                            w[i] = pack2_bf16(fma2(two(-1.0f, -1.0f), two(bf16_lo(m), bf16_hi(m)), S[j / 2 + i]));
                        }
                        *reinterpret_cast<uint4 *>(base + L::s_fine + row + ((j / 8) ^ (st & 7)) * 16) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            fence_proxy_async_shared();
            mbar_arrive(&bars.s_ready);
        };
        if (chunks > 0) put_state();
        const DecayFactor full(ld, kTcC);
        // the weights of the tokens whose columns this thread scales
        constexpr int NW = 8 / NB;
        TokenWeight<NP> wk[NW];
        int wn = -1;  // the chunk size that they are for
        auto weigh = [&](int c) {  // k's pieces of chunk c; the MMAs that read this set of them are done
            const int t0 = t_first + c * t_step, n = min(kTcC, end - t0);
            if (n != wn) {  // the first chunk, the one with the sequence's end, and the one after it
#pragma unroll
                for (int i = 0; i < NW; i++) {
                    const int row = at / 8 + 16 * NB * i, r = p.rev ? n - 1 - row : row;
                    wk[i].set(row < n ? p.w_scale * decay_pow(ld, (float)(n - 1 - r + p.shift)) : 0.0f);
                }
                wn = n;
            }
            if (!wait_warp(&bars.k_full[c % L::nk], c / L::nk)) return false;
            const uint4 *k4 = reinterpret_cast<const uint4 *>(base + L::k + (c % L::nk) * L::kQ) + at;
            uint4 *to = reinterpret_cast<uint4 *>(base + L::pieces + (c % L::nm) * NP * L::kQ) + at;
#pragma unroll 1
            for (int blk = 0; blk < DQ / 64; blk++) {
#pragma unroll
                for (int j = 0; j < NW; j += 4) {
                    // four loads first: a thread's vectors (rows at / 8 + 16 NB i) do not depend on one another
                    uint4 x[4];
#pragma unroll
                    for (int it = 0; it < 4; it++) {
                        x[it] = k4[(j + it) * 128 * NB];
                        // not a token: anything may be there
                        if (n < kTcC && at / 8 + 16 * NB * (j + it) >= n) x[it] = make_uint4(0, 0, 0, 0);
                    }
#pragma unroll
                    for (int it = 0; it < 4; it++) {
                        uint4 hi, mid, lo;
                        wk[j + it].split(x[it], hi, mid, lo);
                        uint4 *dst = to + (j + it) * 128 * NB;
                        dst[0] = hi;
                        dst[L::kQ / 16] = mid;
                        if (NP == 3) dst[2 * (L::kQ / 16)] = lo;
                    }
                }
                k4 += kTcBlock / 16;
                to += kTcBlock / 16;
            }
            mbar_arrive(&bars.k_free[c % L::nk]);
            if (t0 + n < min(t0 + kTcC, (int)a.T)) {
                // what lies past the end may be anything: a zero weight does not remove it from v
                if (!wait_warp(&bars.v_full[c % L::nv], c / L::nv)) return false;
                uint4 *v4 = reinterpret_cast<uint4 *>(base + L::v + (c % L::nv) * L::kV);
                for (int i = at; i < (int)L::kV / 16; i += 128 * NB)
                    if (i / 8 % kTcC >= n) v4[i] = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_shared();
            mbar_arrive(&bars.kw_ready[c % L::nm]);
            return true;
        };
        bool ok = chunks > 0 && weigh(0);
        for (int c = 0; ok && c < chunks; c++) {
            const int n = min(kTcC, end - (t_first + c * t_step));
            if (L::nm == 2 && c + 1 < chunks && !weigh(c + 1)) break;
            const DecayFactor bn = n == kTcC ? full : DecayFactor(ld, n);
            const uint64_t bn_hi = two(bn.hi, bn.hi), bn_lo = two(bn.lo, bn.lo);
            if (!wait_warp(&bars.ds_full, c)) break;
            tcgen05_after();
            if (has_row) {
#pragma unroll
                for (int g = 0; g < SC / 32; g++) {
                    uint32_t x[32];
                    tmem_load32(tmem + L::ds + lanes + c0 + g * 32, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        uint64_t &z = S[g * 16 + e];
                        z = fma2(z, bn_hi, fma2(z, bn_lo, two(x[2 * e], x[2 * e + 1])));
                    }
                }
            }
            tcgen05_before();
            mbar_arrive(&bars.ds_free);
            if (c + 1 == chunks) break;
            if (L::nm == 1 && !weigh(c + 1)) break;
            if (!wait_warp(&bars.s_free, c)) break;
            put_state();
        }
        float *s_out = nullptr;
        int64_t row = p.dv, col = 1;
        if (u == a.nseg - 1 && p.s_out) {
            s_out = p.s_out + bh * mat;
            row = p.s_row;
            col = p.s_col;
        }
        if (s_out && st < p.dq) {
#pragma unroll
            for (int j = 0; j < SC; j += 2) {
                float f[2];
                both(S[j / 2], f[0], f[1]);
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (c0 + j + e < p.dv) s_out[st * row + (c0 + j + e) * col] = f[e];
            }
        }
    } else {
        regs_dec<24>();  // a group without a role
    }
    tcgen05_before();
    __syncthreads();
    if (warp == 0) {
        tcgen05_after();
        tmem_free(tmem, L::tmem_cols);
    }
}

bool attn_operand_map(CUtensorMap *m, const void *base, const int64_t (&st)[3], int d, int64_t T, int64_t heads,
                      int64_t B)
{
    const int64_t dims[4] = {d, T, heads, B}, strides[3] = {st[1], st[2], st[0]};
    return make_tmap_4d_bf16(m, base, dims, strides, 64, kTcC);
}

namespace {

// Rows (tokens of heads) of a call up to which P and S have two pieces, whatever its length.
constexpr int64_t kTcFineRows = 8192;

int width_class(int d) { return d <= 64 ? 64 : 128; }

template <int DQ, int DV, int NP, bool FINE>
bool launch_kernel(const AttnArgs &a, const AttnMaps &m, int passes, cudaStream_t s)
{
    using L = TcLayout<DQ, DV, NP, FINE>;
    const size_t smem = L::bytes + 1024;
    auto kern = k_attn_tc<DQ, DV, NP, FINE>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return false;
    count_launches(1);
    kern<<<(unsigned)(a.B * a.H * a.nseg * passes), L::threads, smem, s>>>(a, m, device_status_ptr());
    return true;
}

// (As a condition in the kernel, the second pieces took 3 to 10% of the longer calls' time.)
template <int DQ, int DV, int NP>
bool launch_tc(const AttnArgs &a, const AttnMaps &m, int passes, cudaStream_t s)
{
    const bool fine = a.T <= kTcC || a.B * a.T * a.H <= kTcFineRows;
    return fine ? launch_kernel<DQ, DV, NP, true>(a, m, passes, s)
                : launch_kernel<DQ, DV, NP, false>(a, m, passes, s);
}

}  // namespace

bool attn_tc_applies(const AttnArgs &a, int passes, int dtype)
{
    if (dtype != LIFB_BF16) return false;
    for (int i = 0; i < passes; i++) {
        const AttnPass &p = a.p[i];
        if (p.dq % 8 || p.dv % 8 || p.dq > kAttnMaxDim || p.dv > kAttnMaxDim || !aligned16(p.o)) return false;
        CUtensorMap m;
        if (!attn_operand_map(&m, p.q, p.qs, p.dq, a.T, a.H / p.qg, a.B) ||
            !attn_operand_map(&m, p.k, p.ks, p.dq, a.T, a.H / p.kg, a.B) ||
            !attn_operand_map(&m, p.v, p.vs, p.dv, a.T, a.H / p.vg, a.B))
            return false;
    }
    return true;
}

bool attn_tc_returns_state(int dq, int dv) { return width_class(dq) == 64 && width_class(dv) == 64; }

bool attn_tc(const AttnArgs &a, int passes, cudaStream_t s)
{
    // passes of one pair of width classes, and with a returned state or without, share a launch
    bool launched[kAttnMaxPasses] = {};
    for (int i = 0; i < passes; i++) {
        if (launched[i]) continue;
        const int dq = width_class(a.p[i].dq), dv = width_class(a.p[i].dv);
        const bool exact_state = a.p[i].s_out != nullptr;
        AttnArgs b = a;
        AttnMaps m = {};
        int n = 0;
        for (int j = i; j < passes; j++) {
            const AttnPass &p = a.p[j];
            if (launched[j] || width_class(p.dq) != dq || width_class(p.dv) != dv ||
                (p.s_out != nullptr) != exact_state)
                continue;
            if (!attn_operand_map(&m.q[n], p.q, p.qs, p.dq, a.T, a.H / p.qg, a.B) ||
                !attn_operand_map(&m.k[n], p.k, p.ks, p.dq, a.T, a.H / p.kg, a.B) ||
                !attn_operand_map(&m.v[n], p.v, p.vs, p.dv, a.T, a.H / p.vg, a.B))
                return false;
            launched[j] = true;
            b.p[n++] = p;
        }
        b.passes = n;
        const bool ok = dq == 64 ? (dv != 64      ? launch_tc<64, 128, 2>(b, m, n, s)
                                    : exact_state ? launch_tc<64, 64, 3>(b, m, n, s)
                                                  : launch_tc<64, 64, 2>(b, m, n, s))
                                 : (dv == 64 ? launch_tc<128, 64, 2>(b, m, n, s) : launch_tc<128, 128, 2>(b, m, n, s));
        if (!ok) return false;
    }
    return true;
}

}  // namespace lifb
