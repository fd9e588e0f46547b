// Leaky attention: the states alone, bf16 operands (leaky_attn.h has the recurrence,
// leaky_attn_tc.cu the chunked form).  For the time segments' starting states, and for
// a state that is returned: there the weighted keys have three bf16 pieces (24 bits),
// else two (2^-18).
//
// A block owns one (pass, sequence, head, time segment) and forms S = sum of b^.. k v^T
// over its tokens from zero, 128 at a time: S <- b^128 S + (K^T diag(w)) V.
//
// At dq = dv = 128 with three pieces a chunk's MMAs read 192 KB of shared memory, its
// pieces are 128 KB of it read and written and its loads 64 KB: 3000 cycles at 128
// bytes a cycle, against 64 KB of k and v: 2800 cycles of an SM's share of the memory.
// Both want the pieces made while the MMAs run, so they come in halves of 64 tokens,
// three sets of them, the first piece in k's place:
//   two warpgroups  k's pieces;
//   one for each 64 columns of the state: registers += MMA result (two in tensor memory);
//   one warp TMA loads, one the MMAs.
// Measured: segments of 15 chunks of 16 heads (144 blocks) 56 us with these steps one
// after another in the main kernel's roles, 35 us so.
// Every wait is bounded (status 101).
#include <algorithm>

#include "leaky_attn_tc.cuh"
#include "lifb_common.cuh"
#include "lifb_internal.h"
#include "seq_types.cuh"

namespace lifb {

namespace {

struct StateMaps {
    CUtensorMap k[kAttnMaxPasses], v[kAttnMaxPasses];
};

// Tiles: 64-column blocks of 128 tokens (k, v) or of 64 (further pieces).  A piece is
// never the last tile (see TcLayout).
template <int DQ, int DV, int NP>
struct StateLayout {
    static constexpr uint32_t kK = DQ / 64 * kTcBlock, kV = DV / 64 * kTcBlock, kHalf = DQ / 64 * (kTcBlock / 2);
    static constexpr int nt = 2, nm = 3;  // k and v tiles, sets of pieces
    static constexpr uint32_t pieces = 0, k = nm * (NP - 1) * kHalf, v = k + nt * kK, bytes = v + nt * kV;
    static_assert(bytes + 1024 + 512 <= 227 * 1024, "tiles fit an SM");
    static constexpr int weigh_groups = 2, state_groups = DV / 64, last_group = weigh_groups + state_groups;
    static constexpr int threads = 128 * (last_group + 1);
    static constexpr uint32_t tmem_cols = DV == 64 ? 128 : 256;  // two results
};

struct StateBars {
    uint64_t k_full[2], v_full[2], kv_free[2], w_ready[3], w_free[3], ds_full[2], ds_free[2], done;
};

}  // namespace

template <int DQ, int DV, int NP>
__global__ void __launch_bounds__((StateLayout<DQ, DV, NP>::threads), 1)
    k_attn_state(const __grid_constant__ AttnArgs a, const __grid_constant__ StateMaps maps, int finish, int *status)
{
    using L = StateLayout<DQ, DV, NP>;
    extern __shared__ unsigned char st_raw[];
    unsigned char *base = (unsigned char *)(((uintptr_t)st_raw + 1023) & ~(uintptr_t)1023);
    __shared__ StateBars bars;
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0), group = warp >> 2;
    const int pi = blockIdx.x % a.passes, item = blockIdx.x / a.passes;
    const AttnPass &p = a.p[pi];
    const int64_t bh = item / a.nseg;
    const int u = (int)(item - bh * a.nseg);                // in the order of the pass
    if (u == a.nseg - 1 && !(finish && p.s_out)) return;          // nothing starts from the last one
    const int64_t b = bh / a.H, h = bh - b * a.H;
    const int64_t len = attn_length(a.lengths, b, a.T);
    const float ld = a.log_decay[h];
    const int64_t seg = p.rev ? a.nseg - 1 - u : u;  // in time
    const int s0 = (int)(seg * a.seg_tokens), s1 = (int)min(a.T, seg * a.seg_tokens + a.seg_tokens);
    const int end = min(s1, (int)len);
    const int chunks = max(0, end - s0 + kTcC - 1) / kTcC;  // with tokens in them
    const int t_first = p.rev ? s0 + (chunks - 1) * kTcC : s0, t_step = p.rev ? -kTcC : kTcC;

    if (warp == 0) tmem_alloc(&tmem_slot, L::tmem_cols);
    if (tid == 32) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&bars.k_full[i], 1);
            mbar_init(&bars.v_full[i], 1);
            mbar_init(&bars.kv_free[i], 1);
            mbar_init(&bars.ds_full[i], 1);
            mbar_init(&bars.ds_free[i], 128 * L::state_groups);
        }
        for (int i = 0; i < 3; i++) {
            mbar_init(&bars.w_ready[i], 128 * L::weigh_groups);
            mbar_init(&bars.w_free[i], 1);
        }
        mbar_init(&bars.done, 1);
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

    if (group == L::last_group) {
        if ((warp & 3) == 0) {
            // ---- loads: the warp waits together, one lane issues
            const int hk = (int)(h / p.kg), hv = (int)(h / p.vg), ib = (int)b;
            int c = 0;
            for (; c < chunks; c++) {
                const int i = c & 1, t0 = t_first + c * t_step;
                if (c >= 2 && !wait(&bars.kv_free[i], c / 2 - 1)) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&bars.k_full[i], L::kK);
                    for (int j = 0; j < DQ / 64; j++)
                        tma_load_4d(base + L::k + i * L::kK + j * kTcBlock, &maps.k[pi], j * 64, t0, hk, ib,
                                    &bars.k_full[i]);
                    mbar_arrive_expect_tx(&bars.v_full[i], L::kV);
                    for (int j = 0; j < DV / 64; j++)
                        tma_load_4d(base + L::v + i * L::kV + j * kTcBlock, &maps.v[pi], j * 64, t0, hv, ib,
                                    &bars.v_full[i]);
                }
                __syncwarp();
            }
            // no copy is left in flight, whatever happened
            for (int j = max(0, c - 2); j < c; j++) {
                mbar_wait(&bars.k_full[j & 1], (j >> 1) & 1);
                mbar_wait(&bars.v_full[j & 1], (j >> 1) & 1);
            }
        } else if ((warp & 3) == 1) {
            // ---- MMAs
            const uint32_t sb = smem_u32(base);
            constexpr uint32_t kIdS = umma_idesc_bf16(kTcC, DV, true, true);
            bool ok = true;
            for (int c = 0; ok && c < chunks; c++) {
                const int i = c & 1;
                ok = wait(&bars.v_full[i], c / 2) && (c < 2 || wait(&bars.ds_free[i], c / 2 - 1));
                for (int half = 0; ok && half < 2; half++) {
                    const int hh = 2 * c + half, set = hh % L::nm;
                    ok = wait(&bars.w_ready[set], hh / L::nm);
                    if (!ok) break;
                    tcgen05_after();
                    if (elect_lane()) {
                        const uint64_t dv = umma_desc_sw128(sb + L::v + i * L::kV + half * (kTcBlock / 2), kTcBlock);
#pragma unroll 1
                        for (int piece = 0; piece < NP; piece++) {
                            const uint64_t dk =
                                piece == 0 ? umma_desc_sw128(sb + L::k + i * L::kK + half * (kTcBlock / 2), kTcBlock)
                                           : umma_desc_sw128(sb + L::pieces + (set * (NP - 1) + piece - 1) * L::kHalf,
                                                             kTcBlock / 2);
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                umma_bf16_ss(tmem + i * DV, dk + k * 128, dv + k * 128, kIdS,
                                             half > 0 || piece > 0 || k > 0);
                        }
                        umma_arrive(&bars.w_free[set]);
                        if (half == 1) {
                            umma_arrive(&bars.ds_full[i]);
                            umma_arrive(&bars.kv_free[i]);
                        }
                    }
                    __syncwarp();
                }
            }
            if (elect_lane()) {  // nothing of the tensor cores is left running
                umma_arrive(&bars.done);
                mbar_wait(&bars.done, 0);
            }
        }
    } else if (group < L::weigh_groups) {
        // ---- k's pieces, 64 tokens at a time
        constexpr int NT = 128 * L::weigh_groups, NV = DQ / 64 * 512 / NT;  // vectors a thread and half
        const int at = tid;
        TokenWeight<NP> wk[2][2];  // of this thread's tokens: rows 64 half + at / 8 + 32 i
        int wn = -1;               // the chunk size that they are for
        bool ok = true;
        for (int c = 0; ok && c < chunks; c++) {
            const int i = c & 1, t0 = t_first + c * t_step, n = min(kTcC, end - t0);
            if (n != wn) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int row = 32 * j + at / 8, r = p.rev ? n - 1 - row : row;
                    wk[j / 2][j % 2].set(row < n ? p.w_scale * decay_pow(ld, (float)(n - 1 - r + p.shift)) : 0.0f);
                }
                wn = n;
            }
            ok = wait(&bars.k_full[i], c / 2);
            if (ok && t0 + n < min(t0 + kTcC, (int)a.T)) {
                // what lies past the end may be anything: a zero weight does not remove it from v
                ok = wait(&bars.v_full[i], c / 2);
                uint4 *v4 = reinterpret_cast<uint4 *>(base + L::v + i * L::kV);
                for (int j = at; ok && j < (int)L::kV / 16; j += NT)
                    if (j / 8 % kTcC >= n) v4[j] = make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (!ok) break;
                const int hh = 2 * c + half, set = hh % L::nm;
                if (hh >= L::nm) ok = wait(&bars.w_free[set], hh / L::nm - 1);
                if (!ok) break;
                uint4 *k4 = reinterpret_cast<uint4 *>(base + L::k + i * L::kK + half * (kTcBlock / 2)) + at;
                uint4 *to = reinterpret_cast<uint4 *>(base + L::pieces + set * (NP - 1) * L::kHalf) + at;
                uint4 x[NV];
#pragma unroll
                for (int j = 0; j < NV; j++) {  // 64 rows of a column block are 512 vectors: two a thread
                    x[j] = k4[j / 2 * (kTcBlock / 16) + j % 2 * NT];
                    if (n < kTcC && half * 64 + at / 8 + 32 * (j % 2) >= n) x[j] = make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < NV; j++) {
                    uint4 hi, mid, lo;
                    wk[half][j % 2].split(x[j], hi, mid, lo);
                    k4[j / 2 * (kTcBlock / 16) + j % 2 * NT] = hi;
                    uint4 *dst = to + j / 2 * (kTcBlock / 32) + j % 2 * NT;
                    dst[0] = mid;
                    if (NP == 3) dst[L::kHalf / 16] = lo;
                }
                fence_proxy_async_shared();
                mbar_arrive(&bars.w_ready[set]);
            }
        }
    } else {
        // ---- the state: one row a thread, 64 of its columns
        const int at = tid - 128 * L::weigh_groups, st = at & 127, c0 = (at >> 7) * 64;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const bool has_row = st < DQ;  // uniform over a warp
        uint64_t S[32];                // pairs of columns
#pragma unroll
        for (int j = 0; j < 32; j++) S[j] = 0;
        const DecayFactor full(ld, kTcC);
        for (int c = 0; c < chunks; c++) {
            const int i = c & 1, n = min(kTcC, end - (t_first + c * t_step));
            const DecayFactor bn = n == kTcC ? full : DecayFactor(ld, n);
            const uint64_t bn_hi = two(bn.hi, bn.hi), bn_lo = two(bn.lo, bn.lo);
            if (!wait(&bars.ds_full[i], c / 2)) break;
            tcgen05_after();
            if (has_row) {
#pragma unroll
                for (int g = 0; g < 64; g += 16) {
                    uint32_t x[16];
                    tmem_load16(tmem + i * DV + lanes + c0 + g, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        uint64_t &z = S[g / 2 + e];
                        z = fma2(z, bn_hi, fma2(z, bn_lo, two(x[2 * e], x[2 * e + 1])));
                    }
                }
            }
            tcgen05_before();
            mbar_arrive(&bars.ds_free[i]);
        }
        if (st < p.dq) {
            float *to = p.seg + (bh * (a.nseg + 1) + u + 1) * p.dq * p.dv + (int64_t)st * p.dv + c0;
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                float f[4];
                both(S[j / 2], f[0], f[1]);
                both(S[j / 2 + 1], f[2], f[3]);
                if (c0 + j < p.dv) *reinterpret_cast<float4 *>(to + j) = make_float4(f[0], f[1], f[2], f[3]);
            }
        }
    }
    tcgen05_before();
    __syncthreads();
    if (warp == 0) {
        tcgen05_after();
        tmem_free(tmem, L::tmem_cols);
    }
}

namespace {

template <int DQ, int DV>
bool launch_state(const AttnArgs &a, const StateMaps &m, int passes, bool finish, cudaStream_t s)
{
    auto go = [&](auto kern, size_t bytes, int threads) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes + 1024) != cudaSuccess)
            return false;
        count_launches(1);
        kern<<<(unsigned)(a.B * a.H * a.nseg * passes), threads, bytes + 1024, s>>>(a, m, finish,
                                                                                                 device_status_ptr());
        return true;
    };
    using L3 = StateLayout<DQ, DV, 3>;
    using L2 = StateLayout<DQ, DV, 2>;
    return finish ? go(k_attn_state<DQ, DV, 3>, L3::bytes, L3::threads) : go(k_attn_state<DQ, DV, 2>, L2::bytes, L2::threads);
}

}  // namespace

bool attn_state(const AttnArgs &a, int passes, bool finish, cudaStream_t s)
{
    // passes of one pair of width classes share a launch
    bool launched[kAttnMaxPasses] = {};
    for (int i = 0; i < passes; i++) {
        if (launched[i]) continue;
        const bool wq = a.p[i].dq > 64, wv = a.p[i].dv > 64;
        AttnArgs b = a;
        StateMaps m = {};
        int n = 0;
        for (int j = i; j < passes; j++) {
            const AttnPass &p = a.p[j];
            if (launched[j] || (p.dq > 64) != wq || (p.dv > 64) != wv) continue;
            if (!attn_operand_map(&m.k[n], p.k, p.ks, p.dq, a.T, a.H / p.kg, a.B) ||
                !attn_operand_map(&m.v[n], p.v, p.vs, p.dv, a.T, a.H / p.vg, a.B))
                return false;
            launched[j] = true;
            b.p[n++] = p;
        }
        b.passes = n;
        const bool ok = wq ? (wv ? launch_state<128, 128>(b, m, n, finish, s) : launch_state<128, 64>(b, m, n, finish, s))
                           : (wv ? launch_state<64, 128>(b, m, n, finish, s) : launch_state<64, 64>(b, m, n, finish, s));
        if (!ok) return false;
    }
    return true;
}

}  // namespace lifb
